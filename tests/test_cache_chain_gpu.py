"""A decoder's passes with the operators together: rotated keys and values into pages, prompts from pages, pages copied for a fork, steps that share a prefix; on a stream, over
captured graphs with workspaces of their own, and through the forms without a workspace."""
import ctypes as C

import pytest
import torch

from axiom_amd import capi
from tests import cache_harness as ch

pytestmark = pytest.mark.gpu
PAGE, LAYERS = 16, 2


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype).cuda()


class Workspace:
    def __init__(self, need):
        self.need, (self.bytes, self.intact) = need, ch.workspace(need)

    def args(self):
        return (ch.at(self.bytes) if self.need else None, self.need)


class Decoder:
    """Two sequences side by side and one that forks the first: buffers and launches of a prompt pass and of a step, for a stream."""

    def __init__(self, dt, heads=8, kv_heads=2, dim=64, seed=0):
        self.dt, self.heads, self.kv_heads, self.dim, self.seed = dt, heads, kv_heads, dim, seed
        self.kp, self.vp = ch.pool(40, PAGE, kv_heads, dim, dt, layers=LAYERS, seed=seed)
        self.turns_host = ch.turns(dim)
        self.turns = ch.device_turns(self.turns_host)
        self.record = []

    def rows(self, tokens, seed):
        g = ch.generator(1000 * self.seed + seed)
        return [torch.randn(LAYERS, tokens, n, self.dim, generator=g).to(ch.DTYPES[self.dt][1]).cuda() for n in (self.heads, self.kv_heads, self.kv_heads)]

    def append(self, layer, x, q_out, slots, positions, stream):
        q, k, v = (t[layer] for t in x)
        p = ch.append_params(q, k, v, q_out, self.kp[layer], self.vp[layer], slots, self.dt, positions=positions, table=self.turns, rot=self.dim)
        capi.check(capi.lib().axhip_kv_append(ch.at(q), ch.at(k), ch.at(v), ch.at(q_out), C.byref(p), stream))

    def copy(self, src, dst, rows, stream):
        p = ch.copy_params(self.kp, self.vp, src, dst, self.dt, rows)
        capi.check(capi.lib().axhip_kv_copy_pages(C.byref(p), stream))

    def close(self, o, want, around, big, keys):
        # Queries and keys are the ones in memory, already rounded
        off = (o.cpu().double() - want).abs() - ch.attention_tolerance(want, around, big, keys, self.dim, self.dt)
        assert float(off.max()) <= 0, float(off.max())

    def keys(self, layer, table, n):
        return ch.rows_of(self.kp[layer], table.cpu(), n), ch.rows_of(self.vp[layer], table.cpu(), n)


def slots_of(table, first, n):
    return [int(table[i // PAGE]) * PAGE + i % PAGE for i in range(first, first + n)]


def prompt(d, stream):
    """Sequences of 50 and 23 tokens, the first in chunks of 30 and 20, padded with rows that belong to nobody; checked against 64 bits."""
    lib = capi.lib()
    tables = torch.full((2, 6), -1, dtype=torch.int32)
    tables[0, :4], tables[1, :2] = torch.tensor([7, 3, 11, 30]), torch.tensor([0, 39])
    table = tables.cuda()
    for turn, (lengths, new) in enumerate((([30, 23], [30, 23]), ([50, 23], [20, 0]))):
        total = sum(new) + 7
        x = d.rows(total, turn)
        q_out, o = torch.full_like(x[0], ch.LEFT), torch.full_like(x[0], ch.LEFT)
        positions = [p for n, m in zip(lengths, new) for p in range(n - m, n)]
        slots = [s for t, n, m in zip(tables, lengths, new) for s in slots_of(t, n - m, m)]
        padded = ints(slots + [-1] * 7, torch.int64)
        where = ints(positions + [0] * 7)
        starts, lens = ints([0, new[0], sum(new)]), ints(lengths)
        torch.cuda.synchronize()
        for layer in range(LAYERS):
            d.append(layer, x, q_out[layer], padded, where, stream)
            p = ch.packed_params(q_out[layer], None, None, o[layer], starts, d.dt, kp=d.kp[layer], vp=d.vp[layer], table=table, lengths=lens)
            ws = Workspace(lib.axhip_sdpa_packed_workspace_bytes(C.byref(p)))
            capi.check(lib.axhip_sdpa_packed_ws(ch.at(q_out[layer]), None, None, ch.at(o[layer]), C.byref(p), *ws.args(), stream))
            capi.check(lib.axhip_stream_sync(stream))
            assert ws.intact()
        torch.cuda.synchronize()
        assert bool((o[:, sum(new):] == ch.LEFT).all())  # rows behind the last sequence
        for layer in range(LAYERS):
            want_q, moved = ch.rotated(x[0][layer, :sum(new)], positions, d.turns_host, d.dim, False)
            assert bool(((q_out[layer, :sum(new)].cpu().double() - want_q).abs() <= ch.rotation_tolerance(want_q, moved, d.dt)).all())
            want_k, moved = ch.rotated(x[1][layer, :sum(new)], positions, d.turns_host, d.dim, False)
            at = 0
            for t, n, m in zip(tables, lengths, new):
                k, v = d.keys(layer, t, n)
                tolerance = ch.rotation_tolerance(want_k[at:at + m], moved[at:at + m], d.dt)
                assert bool(((k[n - m:] - want_k[at:at + m]).abs() <= tolerance).all()) and torch.equal(v[n - m:], x[2][layer, at:at + m].cpu().double())
                if m:
                    d.close(o[layer, at:at + m], *ch.attention(q_out[layer, at:at + m], k, v, n - m), n)
                at += m
    return table


class Step:
    """Buffers of a decoding step of three sequences, of which the first two share three pages; run() is what a graph captures.  `wide`: tables with room for long sequences,
    whose keys are divided among work-groups."""

    def __init__(self, d, shared, wide):
        self.d, self.shared = d, shared
        self.q = torch.empty(LAYERS, 3, d.heads, d.dim, dtype=ch.DTYPES[d.dt][1], device="cuda")
        self.k, self.v = (torch.empty(LAYERS, 3, d.kv_heads, d.dim, dtype=self.q.dtype, device="cuda") for _ in range(2))
        self.q_out, self.o = torch.empty_like(self.q), torch.empty_like(self.q)
        self.positions, self.lens = ints([0] * 3), ints([0] * 3)
        self.slots = ints([0] * 3, torch.int64)
        self.table = torch.full((3, 200 if wide else 8), -1, dtype=torch.int32, device="cuda")
        self.src, self.dst, self.copy_rows = ints([-1]), ints([-1]), ints([0])
        self.starts, self.prefix_lengths = ints([0, 2, 3]), ints([48, 0])
        self.prefix_table = torch.full((2, 200 if wide else 3), -1, dtype=torch.int32, device="cuda")
        self.prefix_table[0, :3] = ints([7, 3, 11])
        how = dict(starts=self.starts, prefix_table=self.prefix_table, prefix_lengths=self.prefix_lengths) if shared else {}
        lib = capi.lib()
        self.params = [ch.paged_params(self.q_out[i][:, None], self.o[i][:, None], d.kp[i], d.vp[i], self.table, self.lens, d.dt, **how) for i in range(LAYERS)]
        self.ws = Workspace(lib.axhip_sdpa_paged_workspace_bytes(C.byref(self.params[0])))
        assert (self.ws.need > 0) == wide

    def run(self, stream, plain=False):
        lib = capi.lib()
        self.d.copy(self.src, self.dst, self.copy_rows, stream)
        for i in range(LAYERS):
            self.d.append(i, (self.q, self.k, self.v), self.q_out[i], self.slots, self.positions, stream)
            if plain:
                capi.check(lib.axhip_sdpa_paged(ch.at(self.q_out[i]), ch.at(self.o[i]), C.byref(self.params[i]), stream))
            else:
                capi.check(lib.axhip_sdpa_paged_ws(ch.at(self.q_out[i]), ch.at(self.o[i]), C.byref(self.params[i]), *self.ws.args(), stream))

    def fill(self, turn):
        """The step's tokens: the first sequence goes on in page 30, the fork in its copy (page 20), the second sequence in page 39 and 21."""
        d = self.d
        for x, y in zip((self.q, self.k, self.v), d.rows(3, 100 + turn)):
            x.copy_(y)
        self.full = [[7, 3, 11, 30, 31], [7, 3, 11, 20, 22], [0, 39, 21, 23, 24]]
        self.lengths = [51 + turn, 51 + turn, 24 + turn]
        self.slots.copy_(ints([slots_of(t, n - 1, 1)[0] for t, n in zip(self.full, self.lengths)], torch.int64))
        self.positions.copy_(ints([n - 1 for n in self.lengths]))
        skip = [3, 3, 0] if self.shared else [0, 0, 0]
        self.table.fill_(-1)
        for i, (t, s) in enumerate(zip(self.full, skip)):
            self.table[i, :5 - s] = ints(t[s:])
        self.lens.copy_(ints([n - s * PAGE for n, s in zip(self.lengths, skip)]))
        fork = turn == 0
        self.src.fill_(30 if fork else -1)
        self.dst.fill_(20 if fork else -1)
        self.copy_rows.fill_(2 if fork else 0)
        self.o.fill_(ch.LEFT)
        torch.cuda.synchronize()

    def check(self):
        d = self.d
        assert self.ws.intact()
        for layer in range(LAYERS):
            for s, (t, n) in enumerate(zip(self.full, self.lengths)):
                k, v = d.keys(layer, torch.tensor(t), n)
                d.close(self.o[layer, s:s + 1], *ch.attention(self.q_out[layer, s:s + 1], k, v, n - 1), n)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("wide", [False, True])
def test_prompt_fork_and_steps(dt, shared, wide):
    stream = torch.cuda.Stream()
    d = Decoder(dt)
    prompt(d, stream.cuda_stream)
    step = Step(d, shared, wide)
    for turn in range(20):  # (past the end of a page)
        step.fill(turn)
        step.run(stream.cuda_stream)
        stream.synchronize()
        step.check()
        with_ws = step.o.clone()
        torch.cuda.synchronize()
        step.src.fill_(-1)
        step.run(None, plain=True)  # the same again, with memory that the call finds for itself
        ch.sync()
        assert torch.equal(step.o, with_ws)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_steps_captured_and_replayed(dt):
    """Three decoders, with and without a shared prefix, whose graphs are replayed with eager work between them and other lengths every time."""
    stream = torch.cuda.Stream()
    steps, graphs = [], []
    for seed, shared, wide in ((1, True, True), (2, False, True), (3, True, False)):
        d = Decoder(dt, seed=seed)
        prompt(d, stream.cuda_stream)
        step = Step(d, shared, wide)
        step.fill(0)
        step.run(stream.cuda_stream)  # (kernels loaded before the capture; the fork's copy made)
        stream.synchronize()
        step.check()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            step.run(stream.cuda_stream)
        steps.append(step)
        graphs.append(g)
    for turn in range(1, 18):
        for step, g in zip(steps, graphs):
            step.fill(turn)
            g.replay()
        torch.cuda.synchronize()
        for step in steps:
            step.check()
            replayed = step.o.clone()
            step.run(stream.cuda_stream)  # eager, the same inputs: the same bits
            stream.synchronize()
            assert torch.equal(step.o, replayed)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_prompts_captured_and_replayed(dt):
    """Lengths and rows of a captured prompt pass are read when it runs."""
    lib, stream = capi.lib(), torch.cuda.Stream()
    q, k, v = (torch.empty(300, n, 64, dtype=ch.DTYPES[dt][1], device="cuda") for n in (4, 2, 2))
    o, starts = torch.empty_like(q), ints([0] * 4)
    p = ch.packed_params(q, k, v, o, starts, dt, cu_kv=starts)
    ws = Workspace(lib.axhip_sdpa_packed_workspace_bytes(C.byref(p)))
    call = lambda s: capi.check(lib.axhip_sdpa_packed_ws(ch.at(q), ch.at(k), ch.at(v), ch.at(o), C.byref(p), *ws.args(), s))
    torch.cuda.synchronize()
    call(stream.cuda_stream)
    stream.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        call(stream.cuda_stream)
    for turn, cu in enumerate(([0, 100, 100, 300], [0, 1, 2, 3], [0, 299, 300, 300], [0, 0, 0, 0], [0, 64, 192, 256])):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=ch.generator(turn)).to(x.dtype))
        starts.copy_(ints(cu))
        o.fill_(ch.LEFT)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert ws.intact() and bool((o[cu[-1]:] == ch.LEFT).all())
        for a, b in zip(cu, cu[1:]):
            if b > a:
                want, around, big = ch.attention(q[a:b], k[a:b], v[a:b], 0)
                assert float(((o[a:b].cpu().double() - want).abs() - ch.attention_tolerance(want, around, big, b - a, 64, dt)).max()) <= 0
        replayed = o.clone()
        call(stream.cuda_stream)
        stream.synchronize()
        assert torch.equal(o, replayed)
        capi.check(lib.axhip_sdpa_packed(ch.at(q), ch.at(k), ch.at(v), ch.at(o), C.byref(p), None))
        ch.sync()
        assert torch.equal(o, replayed)


def test_too_small_workspaces_are_refused():
    lib = capi.lib()
    d = Decoder("bf16")
    step = Step(d, True, True)
    step.fill(1)
    need = step.ws.need
    for ptr, size in ((ch.at(step.ws.bytes), need - 1), (ch.at(step.ws.bytes), 0)):
        assert lib.axhip_sdpa_paged_ws(ch.at(step.q_out), ch.at(step.o), C.byref(step.params[0]), ptr, size, None) == capi.ERR_WORKSPACE
    ch.sync()
    assert bool((step.o == ch.LEFT).all())
    q = torch.randn(3000, 4, 64).bfloat16().cuda()
    starts = ints([0, 3000])
    p = ch.packed_params(q, q, q, torch.empty_like(q), starts, "bf16", cu_kv=starts, max_kv=3000)
    need = lib.axhip_sdpa_packed_workspace_bytes(C.byref(p))
    assert need > 0
    assert lib.axhip_sdpa_packed_ws(ch.at(q), ch.at(q), ch.at(q), ch.at(torch.empty_like(q)), C.byref(p), ch.at(step.ws.bytes), need - 1, None) == capi.ERR_WORKSPACE


def test_two_streams_at_once():
    """Two decoders' steps in flight together, each with its own buffers."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    decoders = [Decoder("bf16", seed=s, heads=16) for s in (5, 6)]
    for d, s in zip(decoders, streams):
        prompt(d, s.cuda_stream)
    steps = [Step(d, shared, True) for d, shared in zip(decoders, (True, False))]
    for turn in range(8):
        for step in steps:
            step.fill(turn)
        for _ in range(3):  # (the same tokens to the same places)
            for step, s in zip(steps, streams):
                step.run(s.cuda_stream)
        torch.cuda.synchronize()
        for step in steps:
            step.check()
