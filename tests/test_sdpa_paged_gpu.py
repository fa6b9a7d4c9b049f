"""A decoding step over pages, with and without prefixes that sequences share, against 64 bits."""
import math

import pytest
import torch

from tests import cache_harness as ch

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


class Step:
    def __init__(self, lengths, new, heads, kv_heads, dim, page, dt, by_head=False, starts=None, prefixes=None, seed=0, pad=0, spare=4, ld=0):
        self.lengths, self.dt, self.dim, self.new, self.page = lengths, dt, dim, new, page
        self.starts, self.prefixes = starts, prefixes
        need = sum(-(-n // page) for n in lengths + (prefixes or []))
        self.kp, self.vp = ch.pool(need + spare, page, kv_heads, dim, dt, by_head, seed=seed, pad=pad)
        order = torch.randperm(need + spare, generator=ch.generator(seed))
        self.host_table, used = ch.table_of(lengths, page, order, columns=ld)
        self.table, self.lens = self.host_table.cuda(), ints(lengths)
        self.how = {}
        if starts is not None:
            self.host_prefix, more = ch.table_of(prefixes, page, order[used:])
            self.how = dict(starts=ints(starts), prefix_table=self.host_prefix.cuda(), prefix_lengths=ints(prefixes))
        self.q = torch.randn(len(lengths), new + 1, heads, dim + pad, generator=ch.generator(seed + 50)).mul(1.5).to(ch.DTYPES[dt][1]).cuda()[:, :new, :, :dim]

    def run(self, **more):
        return ch.paged(self.q, self.kp, self.vp, self.table, self.lens, self.dt, **self.how, **more)

    def check(self, o, scale=None):
        o = o.cpu().double()
        for s, n in enumerate(self.lengths):
            prefix, k, v = 0, ch.rows_of(self.kp, self.host_table[s], n), ch.rows_of(self.vp, self.host_table[s], n)
            if self.starts is not None and self.starts[0] <= s < self.starts[-1]:
                g = max(i for i in range(len(self.starts) - 1) if self.starts[i] <= s)
                prefix = self.prefixes[g]
                k, v = (torch.cat((ch.rows_of(p, self.host_prefix[g], prefix), x)) for p, x in ((self.kp, k), (self.vp, v)))
            # tokens that stand in front of the first own key see the prefix all the same
            for i in range(self.new):
                seen = prefix + max(0, n - self.new + i + 1)
                want, around, big = ch.attention(self.q[s, i:i + 1], k[:seen], v[:seen], None, scale)
                off = (o[s, i] - want[0]).abs() - ch.attention_tolerance(want, around, big, seen, self.dim, self.dt)[0]
                assert float(off.max()) <= 0, (s, i, n, prefix, float(off.max()))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("lengths,new,heads,kv_heads,dim,page", [([1], 1, 1, 1, 64, 16), ([5, 0, 1, 300], 1, 8, 2, 128, 16), ([1000, 33, 2500], 1, 32, 8, 128, 32), ([17, 31, 32, 33, 64, 65], 4, 12, 4, 96, 8),
                                                                 ([3, 1, 90], 5, 7, 1, 80, 64), ([9000], 2, 16, 2, 128, 16), ([50] * 70, 1, 4, 4, 64, 128), ([700, 20], 3, 40, 2, 40, 16)])
def test_steps(dt, by_head, lengths, new, heads, kv_heads, dim, page):
    s = Step(lengths, new, heads, kv_heads, dim, page, dt, by_head)
    o, kernel = s.run()
    assert kernel != "generic"
    s.check(o)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lengths,new,heads,kv_heads,dim,page,starts,prefixes", [
    ([5, 9, 300], 1, 8, 2, 128, 16, [0, 3], [500]), ([5, 9, 0, 40], 1, 8, 2, 64, 16, [1, 3], [70]), ([4] * 9, 2, 4, 4, 96, 8, [0, 2, 2, 7, 8], [100, 33, 0, 1]), ([20] * 40, 1, 16, 2, 128, 32, [0, 40], [2000]),
    ([1], 1, 1, 1, 64, 16, [0, 1], [1]), ([10, 20, 30], 3, 6, 6, 80, 64, [0, 1, 3], [65, 1300]), ([0, 1, 2, 3], 4, 8, 1, 128, 16, [0, 4], [200]), ([12] * 5, 1, 4, 2, 64, 16, [0, 0, 0], [50, 60])])
def test_shared_prefixes(dt, lengths, new, heads, kv_heads, dim, page, starts, prefixes):
    s = Step(lengths, new, heads, kv_heads, dim, page, dt, starts=starts, prefixes=prefixes)
    o, kernel = s.run()
    assert kernel != "generic"
    s.check(o)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("hint", [0, 1, 10**6])
def test_hints_are_hints(dt, hint):
    for starts in ([0, 2], None):
        s = Step([1500, 7, 300], 1, 8, 2, 64, 16, dt, starts=starts, prefixes=[900] if starts else None)
        o, kernel = s.run(max_kv=hint, max_prefix=hint)
        assert (kernel == "whole") == (hint < 10)
        s.check(o)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("starts,prefixes", [(None, None), ([0, 3], [100]), ([1, 3, 3, 5], [33, 40, 130])])
@pytest.mark.parametrize("heads,kv_heads,dim,new", [(8, 2, 128, 1), (4, 4, 64, 3), (12, 1, 80, 2), (2, 2, 128, 20)])
def test_short_sequences_undivided(dt, starts, prefixes, heads, kv_heads, dim, new):
    s = Step([5, 0, 130, 64, 1], new, heads, kv_heads, dim, 16, dt, starts=starts, prefixes=prefixes)
    o, kernel = s.run(max_kv=130, max_prefix=130)
    assert kernel == "whole"
    s.check(o)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [4, 8, 12, 24, 36, 48, 72, 104, 120, 136, 192, 256])
def test_head_sizes(dt, dim):
    s = Step([100, 3, 40], 2, 4, 2, dim, 16, dt, starts=[1, 3], prefixes=[77])
    o, kernel = s.run()
    s.check(o)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,pad,page", [(33, 0, 16), (64, 1, 16), (128, 0, 4), (64, 0, 1), (64, 8, 16), (128, 8, 2), (80, 2, 32)])
def test_odd_sizes_and_strides(dt, dim, pad, page):
    s = Step([100, 3, 40, 0], 2, 6, 2, dim, page, dt, starts=[0, 2], prefixes=[21], pad=pad)
    s.check(s.run()[0])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_what_lies_outside_a_sequence_does_not_matter(dt, dim):
    s = Step([70, 1, 33, 200], 1, 4, 2, dim, 16, dt, starts=[0, 2], prefixes=[37])
    clean = s.run()[0].clone()
    s.check(clean)
    inside = torch.zeros(s.kp.shape[:2], dtype=torch.bool)
    for r, n in list(zip(s.host_table, s.lengths)) + list(zip(s.host_prefix, s.prefixes)):
        i = torch.arange(n)
        inside[r.long()[i // 16], i % 16] = True
    s.kp[~inside.cuda()] = math.nan
    s.vp[~inside.cuda()] = math.inf
    assert torch.equal(s.run()[0], clean)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_large_scores_and_scale(dt):
    s = Step([400, 90], 1, 8, 2, 64, 16, dt, starts=[0, 1], prefixes=[300])
    s.q.mul_(3)
    for scale in (1.0, 0.01):
        s.check(s.run(scale=scale)[0], scale)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_pages_that_do_not_exist_and_numbers_out_of_range(dt):
    s = Step([100, 200, 30, 40], 1, 8, 2, 64, 16, dt, starts=[0, 2, 3], prefixes=[50, 60], ld=14)
    clean = s.run()[0].clone()
    for bad in (-1, s.kp.shape[0], 2**31 - 1, -(2**31)):
        keep = s.table.clone()
        s.table[1, 12] = bad
        o, _ = s.run()
        assert bool(torch.isnan(o[1]).all()) and torch.equal(o[0], clean[0]) and torch.equal(o[2:], clean[2:])
        s.table.copy_(keep)
        keep = s.how["prefix_table"].clone()
        s.how["prefix_table"][0, 3] = bad
        o, _ = s.run()
        assert bool(torch.isnan(o[:2]).all()) and torch.equal(o[2:], clean[2:])
        s.how["prefix_table"].copy_(keep)
    s.lens[0], s.lens[3], s.how["prefix_lengths"][1] = -3, -(2**31), -7  # no keys of their own; no prefix
    o, _ = s.run()
    t = Step([100, 200, 30, 40], 1, 8, 2, 64, 16, dt, starts=[0, 2, 3], prefixes=[50, 60], ld=14)
    t.lengths, t.prefixes = [0, 200, 30, 0], [50, 0]
    t.check(o)
    assert bool((o[3] == 0).all())
    s.lens[3] = 2**31 - 1  # the table's: pages -1 among them
    assert bool(torch.isnan(s.run()[0][3]).all())


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_every_run_gives_the_same_bits(dt):
    s = Step([3000, 10, 777, 4000], 1, 32, 8, 128, 16, dt, starts=[0, 4], prefixes=[3000])
    first = s.run()[0].clone()
    s.check(first)
    for _ in range(5):
        assert torch.equal(s.run()[0], first)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("groups,new", [(70, 1), (300, 1), (300, 3), (4200, 1)])
def test_more_groups_than_a_wavefront_has_lanes(dt, groups, new):
    """Of up to four sequences, every fifth of none, some behind a prefix of no keys; sequences without a group in front and behind."""
    starts, prefixes = [2], []
    for g in range(groups):
        starts.append(starts[-1] + (0 if g % 5 == 4 else (g * 7) % 5 if groups < 1000 else 1 if g % 9 == 0 else 0))
        prefixes.append(0 if g % 11 == 3 else 1 + (g * 29) % 90)
    n = starts[-1] + 3
    s = Step([(i * 37) % 60 for i in range(n)], new, 2, 1, 64, 16, dt, starts=starts, prefixes=prefixes, seed=groups, ld=64)
    o, kernel = s.run()
    assert kernel == "shares, prefix"
    s.kp, s.vp = s.kp.cpu().double(), s.vp.cpu().double()  # (once for all sequences)
    s.check(o)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_more_sequences_than_a_wavefront_has_lanes(dt):
    for n in (64, 65, 257, 1030):
        s = Step([(i * 37) % 90 for i in range(n)], 1, 2, 1, 64, 16, dt, starts=[0, 3, n], prefixes=[40, 200], seed=n)
        s.check(s.run()[0])


def test_keys_behind_four_gigabytes():
    heads, dim, page = 2, 128, 16
    n_pages = (1 << 32) // (heads * dim * page) + 64
    kp = torch.zeros(n_pages, page, heads, dim, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    table = torch.tensor([[n_pages - 1 - i for i in range(20)]], dtype=torch.int32)
    for i, x in enumerate((kp, vp)):
        x[-20:] = torch.randn(20, page, heads, dim, generator=ch.generator(i)).bfloat16().cuda()
    q = torch.randn(1, 1, 8, dim, generator=ch.generator(9)).bfloat16().cuda()
    k, v = (x[-20:].cpu().double().flip(0).reshape(-1, heads, dim) for x in (kp, vp))
    want, around, big = ch.attention(q[0], torch.cat((k[:313], k[:77])), torch.cat((v[:313], v[:77])), None)
    o, _ = ch.paged(q, kp, vp, table.cuda(), ints([77]), "bf16", starts=ints([0, 1]), prefix_table=table.cuda(), prefix_lengths=ints([313]))
    assert float(((o[0].cpu().double() - want).abs() - ch.attention_tolerance(want, around, big, 390, dim, "bf16")).max()) <= 0


def test_pages_four_gigabytes_apart():
    """(offsets from one page to the next beyond 32 bits: the generic kernel)"""
    page, heads, dim, apart = 16, 2, 64, (1 << 31) + 64
    pools = [torch.empty(apart + page * heads * dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    kp, vp = (p.as_strided((2, page, heads, dim), (apart, heads * dim, dim, 1)) for p in pools)
    for i, p in enumerate((kp, vp)):
        p.copy_(torch.randn(2, page, heads, dim, generator=ch.generator(i)).bfloat16())
    table = torch.tensor([[1, 0]], dtype=torch.int32)
    q = torch.randn(1, 2, 4, dim, generator=ch.generator(5)).bfloat16().cuda()
    k, v = (p.cpu().double().flip(0).reshape(-1, heads, dim)[:27] for p in (kp, vp))
    want, around, big = ch.attention(q[0], k, v, 25)
    o, kernel = ch.paged(q, kp, vp, table.cuda(), ints([27]), "bf16")
    assert kernel == "generic"
    o2, kernel = ch.packed(q[0], None, None, ints([0, 2]), "bf16", kp=kp, vp=vp, table=table.cuda(), lengths=ints([27]))
    assert kernel == "generic"
    for x in (o[0], o2):
        assert float(((x.cpu().double() - want).abs() - ch.attention_tolerance(want, around, big, 27, dim, "bf16")).max()) <= 0


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("starts,prefixes", [(None, None), ([0, 2], [5])])
def test_a_cache_without_pages(dt, starts, prefixes):
    """Every page is one that does not exist: sequences with keys are not numbers, those without are zeros."""
    none = torch.empty(0, 16, 2, 64, dtype=ch.DTYPES[dt][1], device="cuda")
    q = torch.randn(4, 1, 8, 64, generator=ch.generator(3)).to(none.dtype).cuda()
    table, lens = torch.zeros(4, 200, dtype=torch.int32, device="cuda"), ints([300, 0, 1, 0])
    how = dict(starts=ints(starts), prefix_table=torch.zeros(1, 8, dtype=torch.int32, device="cuda"), prefix_lengths=ints(prefixes)) if starts else {}
    o, _ = ch.paged(q, none, none, table, lens, dt, **how)
    bad = [0, 2] + ([1] if starts else [])
    good = [i for i in range(4) if i not in bad]
    assert bool(torch.isnan(o[bad]).all()) and bool((o[good] == 0).all())
    o, _ = ch.packed(q[:, 0], None, None, ints([0, 1, 2, 3, 4]), dt, kp=none, vp=none, table=table, lengths=lens)
    assert bool(torch.isnan(o[[0, 2]]).all()) and bool((o[[1, 3]] == 0).all())
