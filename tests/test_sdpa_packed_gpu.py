"""Attention of packed sequences of different lengths, keys packed alike or in pages, against 64 bits."""
import math

import pytest
import torch

from tests import cache_harness as ch

pytestmark = pytest.mark.gpu
LENGTHS = {"one": [1], "short": [3, 1, 2], "around a tile": [63, 64, 65, 1, 128, 127, 129], "some are empty": [0, 70, 0, 0, 33, 0], "long and short": [700, 5, 1, 260], "many": [(7 * i) % 40 for i in range(150)]}


def ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def starts(lengths, behind=0):
    return ints([behind + sum(lengths[:i]) for i in range(len(lengths) + 1)])


class Problem:
    """q (and packed keys) for `lengths`, with rows around them that no sequence owns; `keys` of each, in pages or packed"""

    def __init__(self, lengths, heads, kv_heads, dim, dt, keys=None, page=0, by_head=False, seed=0, scale=1.0, ld=0, pad=0):
        self.lengths, self.keys, self.dt, self.dim = lengths, keys or lengths, dt, dim
        g, t = ch.generator(seed), ch.DTYPES[dt][1]
        around = 5
        total, total_kv = sum(lengths) + 2 * around, sum(self.keys) + 2 * around
        wide = torch.randn(total, heads + 1, dim + pad, generator=g).mul(scale).to(t).cuda()
        self.q, self.cu_q = wide[:, 1:, :dim], starts(lengths, around)
        self.k = self.v = self.kp = self.vp = self.table = self.lens = self.cu_kv = None
        if page:
            need = sum(-(-n // page) for n in self.keys)
            self.kp, self.vp = ch.pool(need + 4, page, kv_heads, dim, dt, by_head, seed=seed + 1, pad=pad)
            self.order = torch.randperm(need + 4, generator=g)
            table, used = ch.table_of(self.keys, page, self.order, columns=ld)
            self.host_table = table
            self.table, self.lens = table.cuda(), ints(self.keys)
            own = [ch.rows_of(p, r, n) for p in (self.kp, self.vp) for r, n in zip(table, self.keys)]
        else:
            kv = torch.randn(total_kv, 2 * kv_heads, dim + pad, generator=g).to(t).cuda()
            self.k, self.v, self.cu_kv = kv[:, :kv_heads, :dim], kv[:, kv_heads:, :dim], starts(self.keys, around)
            own = [x[a:a + n].cpu().double() for x in (self.k, self.v) for a, n in zip(self.cu_kv.tolist(), self.keys)]
        self.own_k, self.own_v = own[:len(lengths)], own[len(lengths):]

    def run(self, causal=True, **how):
        paged = dict(kp=self.kp, vp=self.vp, table=self.table, lengths=self.lens) if self.table is not None else dict(cu_kv=self.cu_kv)
        return ch.packed(self.q, self.k, self.v, self.cu_q, self.dt, causal=causal, **paged, **how)

    def check(self, o, causal=True, scale=None):
        at, owned = self.cu_q.tolist(), torch.zeros(o.shape[0], dtype=torch.bool)
        for s, (n, m) in enumerate(zip(self.lengths, self.keys)):
            rows = slice(at[s], at[s] + n)
            owned[rows] = True
            want, around, big = ch.attention(self.q[rows], self.own_k[s], self.own_v[s], m - n if causal else None, scale)
            off = (o[rows].cpu().double() - want).abs() - ch.attention_tolerance(want, around, big, m, self.dim, self.dt)
            assert n == 0 or float(off.max()) <= 0, (s, n, m, float(off.max()))
        assert bool((o.cpu()[~owned] == ch.LEFT).all())  # rows that no sequence owns


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lengths", LENGTHS, ids=list(LENGTHS))
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (8, 2, 128), (7, 1, 80)])
def test_prompts(dt, lengths, heads, kv_heads, dim):
    p = Problem(LENGTHS[lengths], heads, kv_heads, dim, dt, seed=dim)
    o, kernel = p.run()
    assert kernel != "generic"
    p.check(o)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,dim,page,by_head", [(4, 4, 64, 16, False), (8, 2, 128, 8, True), (12, 4, 96, 32, False), (6, 2, 128, 64, True), (3, 3, 40, 128, False)])
def test_chunks_over_pages(dt, causal, heads, kv_heads, dim, page, by_head):
    """Queries behind what the cache holds already; fewer keys than queries; sequences without keys, or without queries."""
    lengths, keys = [1, 70, 130, 5, 0, 9, 64], [200, 70, 700, 3, 50, 0, 129]
    p = Problem(lengths, heads, kv_heads, dim, dt, keys, page, by_head, seed=page)
    o, kernel = p.run(causal)
    assert kernel != "generic"
    p.check(o, causal)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [4, 8, 12, 24, 32, 36, 48, 56, 72, 88, 104, 112, 120, 136, 192, 200, 256])
def test_head_sizes(dt, dim):
    for page in (0, 16):
        p = Problem([40, 100, 3], 4, 2, dim, dt, page=page, seed=dim)
        o, kernel = p.run()
        assert (kernel == "generic") == (dim % 8 != 0 if dt == "bf16" else dim > 128)
        p.check(o)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,pad,page", [(33, 0, 0), (64, 1, 0), (64, 3, 16), (65, 0, 8), (128, 0, 4), (64, 0, 1), (128, 8, 2), (64, 8, 16), (128, 8, 0)])
def test_odd_sizes_and_strides(dt, dim, pad, page):
    p = Problem([17, 1, 50], 6, 2, dim, dt, page=page, seed=dim + pad, pad=pad)
    o, _ = p.run()
    p.check(o)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page", [0, 16])
def test_scale_large_scores_and_one_key_that_decides(dt, page):
    p = Problem([300, 20], 4, 2, 64, dt, page=page, scale=4.0)
    for scale in (1.0, 0.3, 0.001):
        o, _ = p.run(scale=scale)
        p.check(o, scale=scale)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [0, 16])
def test_what_lies_outside_a_sequence_does_not_matter(dt, dim, page):
    """NaN and infinities in other sequences' rows, behind the last row of a page, in pages that are not listed, and in K where a causal query does not look."""
    lengths = [70, 1, 33]
    p = Problem(lengths, 4, 2, dim, dt, page=page, seed=dim)
    clean, _ = p.run()
    p.check(clean)
    clean = clean.clone()
    if page:
        inside = torch.zeros(p.kp.shape[:2], dtype=torch.bool)
        for r, n in zip(p.host_table, lengths):
            i = torch.arange(n)
            inside[r.long()[i // page], i % page] = True
        for x, bad in ((p.kp, math.nan), (p.vp, math.inf)):
            x[~inside.cuda()] = bad
        o, _ = p.run()
        assert torch.equal(o, clean)
        return
    at = p.cu_kv.tolist()
    for s in range(3):  # every sequence among rows that hold nothing sensible
        k, v = p.k.clone(), p.v.clone()
        for x, bad in ((p.k, math.nan), (p.v, -math.inf)):
            x[:at[s]] = bad
            x[at[s + 1]:] = bad
        o, _ = p.run()
        rows = slice(p.cu_q.tolist()[s], p.cu_q.tolist()[s + 1])
        assert torch.equal(o[rows], clean[rows])
        p.k.copy_(k)
        p.v.copy_(v)
    p.k[at[1] - 1] = math.inf  # the last key of the first sequence, which only its last query sees
    o, _ = p.run()
    assert torch.equal(o[5:5 + 69], clean[5:5 + 69])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_pages_that_do_not_exist_and_numbers_out_of_range(dt):
    p = Problem([40, 30, 20], 4, 2, 64, dt, keys=[100, 90, 80], page=16, ld=9)
    clean = p.run()[0].clone()
    for bad in (-1, p.kp.shape[0], 2**31 - 1, -(2**31)):
        keep = p.table.clone()
        p.table[1, 4] = bad
        o, _ = p.run()
        at = p.cu_q.tolist()
        assert bool(torch.isnan(o[at[1]:at[2]]).all()) and torch.equal(o[:at[1]], clean[:at[1]]) and torch.equal(o[at[2]:], clean[at[2]:])
        p.table.copy_(keep)
    # a length beyond the table is the table's (144 keys, the last ones in pages -1: NaN); a negative one is none
    p.lens[0], p.lens[2] = 2**31 - 1, -5
    o, _ = p.run()
    assert bool(torch.isnan(o[at[0]:at[1]]).all()) and bool((o[at[2]:at[3]] == 0).all()) and torch.equal(o[at[1]:at[2]], clean[at[1]:at[2]])
    # borders outside the tensors are clamped to them
    q = Problem([40, 30], 4, 2, 64, dt)
    q.cu_q[0], q.cu_q[2] = -100, 10**6
    q.cu_kv[0], q.cu_kv[2] = -3, 10**6
    o, _ = q.run()
    q.lengths, q.keys, q.cu_q = [45, 35], [45, 35], ints([0, 45, 80])
    q.own_k, q.own_v = ([x[:45].cpu().double(), x[45:].cpu().double()] for x in (q.k, q.v))
    q.check(o)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("hint", [0, 1, 128, 700, 10**6])
def test_hints_are_hints(dt, page, hint):
    """Keys undivided and in as many parts as there may be: sequences longer and shorter than the hint says, and rows that no sequence owns."""
    p = Problem([40, 0, 3, 150], 4, 2, 96, dt, keys=[900, 5, 0, 1500] if page else None, page=page)
    o, kernel = p.run(max_kv=hint)
    assert kernel.endswith("parts") if page and hint == 10**6 else kernel in ("f32", "few") if hint <= 128 else kernel != "generic"
    p.check(o)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_every_run_gives_the_same_bits(dt):
    p = Problem([50, 700, 3], 8, 2, 128, dt, keys=[3000, 700, 1000], page=16)
    first = p.run(max_kv=3000)[0].clone()
    p.check(first)
    for _ in range(5):
        assert torch.equal(p.run(max_kv=3000)[0], first)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_more_sequences_than_a_wavefront_has_lanes(dt):
    for n in (64, 65, 300, 1100):
        lengths = [(i * 37) % 23 for i in range(n)]
        p = Problem(lengths, 2, 1, 64, dt, seed=n)
        p.check(p.run()[0])


def test_keys_behind_four_gigabytes():
    heads, dim, page = 2, 128, 16
    n_pages = (1 << 32) // (heads * dim * page) + 64
    kp = torch.zeros(n_pages, page, heads, dim, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    table = torch.tensor([[n_pages - 1 - i for i in range(20)]], dtype=torch.int32)
    for i, x in enumerate((kp, vp)):
        x[-20:] = torch.randn(20, page, heads, dim, generator=ch.generator(i)).bfloat16().cuda()
    q = torch.randn(50, 4, dim, generator=ch.generator(9)).bfloat16().cuda()
    o, kernel = ch.packed(q, None, None, ints([0, 50]), "bf16", kp=kp, vp=vp, table=table.cuda(), lengths=ints([313]))
    assert kernel != "generic"
    k, v = (x[-20:].cpu().double().flip(0).reshape(-1, heads, dim)[:313] for x in (kp, vp))
    want, around, big = ch.attention(q, k, v, 263)
    assert float(((o.cpu().double() - want).abs() - ch.attention_tolerance(want, around, big, 313, dim, "bf16")).max()) <= 0


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,dim,page,by_head", [(16, 8, 64, 0, False), (16, 8, 40, 16, True), (32, 8, 128, 0, False), (14, 7, 100, 8, False), (24, 12, 12, 32, True)])
def test_many_short_prompts_of_32_bits(causal, heads, kv_heads, dim, page, by_head):
    """Each wave walks the keys of its own 16 rows (max_kv, a hint, says that there are few): sequences of less than a work-group's 64, empty ones, more keys than queries and fewer."""
    lengths = [(13 * i) % 61 for i in range(55)] + [64, 65, 1, 0, 130]
    keys = [n + (3 * i) % 7 - 2 if n > 2 else n for i, n in enumerate(lengths)] if page else lengths
    p = Problem(lengths, heads, kv_heads, dim, "f32", keys=keys, page=page, by_head=by_head, seed=dim, ld=20)
    o, kernel = p.run(causal=causal, max_kv=40)
    assert kernel == "f32, apart"
    p.check(o, causal)
    first = o.clone()
    assert torch.equal(p.run(causal=causal, max_kv=40)[0], first)
    if page:  # what no sequence holds does not matter; a page that does not exist spoils its sequence alone
        inside = torch.zeros(p.kp.shape[:2], dtype=torch.bool)
        for r, n in zip(p.host_table, keys):
            i = torch.arange(n)
            inside[r.long()[i // page], i % page] = True
        p.kp[~inside.cuda()] = math.nan
        p.vp[~inside.cuda()] = math.inf
        assert torch.equal(p.run(causal=causal, max_kv=40)[0], first)
        p.table[55, 0] = p.kp.shape[0]  # (the one of 64)
        o, at = p.run(causal=causal, max_kv=40)[0], p.cu_q.tolist()
        assert torch.equal(o[:at[55]], first[:at[55]]) and torch.equal(o[at[56]:], first[at[56]:])
        sees = torch.arange(64) + keys[55] - 64 >= 0 if causal else torch.ones(64, dtype=torch.bool)
        assert bool(torch.isnan(o[at[55]:at[56]][sees.cuda()]).all())


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,dim,page,by_head", [(32, 8, 128, 0, False), (32, 8, 104, 16, True), (16, 8, 128, 64, False)])
def test_work_groups_of_eight_waves(dt, causal, heads, kv_heads, dim, page, by_head):
    """(max_kv, a hint, says that walks are long)"""
    lengths = [(37 * i) % 190 for i in range(40)] + [0, 63, 256, 257, 511] if heads == 32 else [(37 * i) % 190 for i in range(44)] + [1030]
    keys = [n + (5 * i) % 90 - 20 if n > 20 else n for i, n in enumerate(lengths)] if page else lengths
    p = Problem(lengths, heads, kv_heads, dim, dt, keys=keys, page=page, by_head=by_head, seed=dim, ld=80)
    o, kernel = p.run(causal=causal, max_kv=4000)
    assert kernel == "tile, eight waves"
    p.check(o, causal)
    first = o.clone()
    assert torch.equal(p.run(causal=causal, max_kv=4000)[0], first)
    if page:
        inside = torch.zeros(p.kp.shape[:2], dtype=torch.bool)
        for r, n in zip(p.host_table, keys):
            i = torch.arange(n)
            inside[r.long()[i // page], i % page] = True
        p.kp[~inside.cuda()] = math.nan
        p.vp[~inside.cuda()] = math.inf
        assert torch.equal(p.run(causal=causal, max_kv=4000)[0], first)


MORE = [35, 64, 30, 1, 31, 32, 33] * 6  # enough blocks of rows for work-groups of 128 of them


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths", LENGTHS, ids=list(LENGTHS))
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 16, 64), (16, 16, 128), (30, 15, 80), (16, 16, 24), (17, 17, 200)])
def test_prompts_on_tiles(dt, causal, lengths, heads, kv_heads, dim):
    p = Problem(LENGTHS[lengths] + MORE, heads, kv_heads, dim, dt, seed=dim)
    o, kernel = p.run(causal=causal)
    assert kernel == "tile"
    p.check(o, causal)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,dim,page,by_head", [(32, 16, 64, 16, False), (16, 16, 128, 8, True), (16, 16, 96, 32, False), (17, 17, 40, 128, True), (32, 16, 256, 16, False)])
def test_chunks_over_pages_on_tiles(dt, causal, heads, kv_heads, dim, page, by_head):
    """Queries behind what the cache holds, fewer keys than queries, nothing of either; what lies outside does not matter, and a page that does not exist spoils its sequence alone."""
    lengths = [17, 64, 0, 5, 130, 1, 33] + MORE
    keys = [300, 64, 40, 3, 141, 90, 0] + [n + (7 * i) % 60 for i, n in enumerate(MORE)]
    p = Problem(lengths, heads, kv_heads, dim, dt, keys=keys, page=page, by_head=by_head, seed=dim, ld=50)
    o, kernel = p.run(causal=causal)
    assert kernel == "tile"
    p.check(o, causal)
    first = o.clone()
    inside = torch.zeros(p.kp.shape[:2], dtype=torch.bool)
    for r, n in zip(p.host_table, keys):
        i = torch.arange(n)
        inside[r.long()[i // page], i % page] = True
    p.kp[~inside.cuda()] = math.nan
    p.vp[~inside.cuda()] = math.inf
    assert torch.equal(p.run(causal=causal)[0], first)
    p.table[4, 0] = -1
    o, at = p.run(causal=causal)[0], p.cu_q.tolist()
    assert torch.equal(o[:at[4]], first[:at[4]]) and torch.equal(o[at[5]:], first[at[5]:]) and bool(torch.isnan(o[at[4]:at[5]]).all())


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 16), (4, 4, 64, 0), (12, 2, 80, 32), (2, 1, 256, 8), (8, 8, 40, 0)])
def test_few_rows(dt, causal, heads, kv_heads, dim, page):
    lengths = [17, 64, 0, 5, 130, 1, 33]
    keys = [300, 64, 40, 3, 641, 90, 0] if page else lengths
    p = Problem(lengths, heads, kv_heads, dim, dt, keys=keys, page=page, seed=dim)
    o, kernel = p.run(causal=causal, max_kv=641)
    assert kernel == "few"
    p.check(o, causal)
    if page:  # divided: one long sequence beside short ones
        q = Problem([3, 1, 20], heads, kv_heads, dim, dt, keys=[1200, 1000, 20], page=page, seed=dim + 1)
        o, kernel = q.run(causal=causal, max_kv=1200)
        assert kernel == "few, parts"
        q.check(o, causal)
