"""The 8-bit calls and sampling one after the other, as a decoding step ends: against the same step from their integers in 64 bits, on a stream
of its own, and captured into a graph that is replayed with the program's own work in between."""
import ctypes as C

import numpy as np
import pytest
import torch

from axiom_amd import capi
from tests import q8_harness as q8

pytestmark = pytest.mark.gpu
WIDTH, INNER, VOCAB = 512, 1408, 5003


class Step:
    """norm -> up (silu) -> quantize -> down + residual -> norm -> logits -> token, for `rows` sequences; outputs are made once"""

    def __init__(self, rows, seed=0):
        gen = torch.Generator()
        gen.manual_seed(seed)

        def normal(*shape, scale=1.0, dtype=torch.bfloat16):
            return (torch.randn(shape, generator=gen) * scale).to(dtype).cuda()

        self.lib, self.rows = capi.lib(), rows
        self.x, self.res, self.w = normal(rows, WIDTH), normal(rows, WIDTH), normal(WIDTH, scale=0.1) + 1
        self.u = torch.rand(rows, generator=gen).cuda()
        self.weights = [q8.quantize(normal(n, k, scale=k**-0.5), "bf16") for n, k in ((INNER, WIDTH), (WIDTH, INNER), (VOCAB, WIDTH))]
        e = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
        i8, f32 = torch.int8, torch.float32
        self.sum, self.hidden, self.out, self.logits = e(rows, WIDTH), e(rows, INNER), e(rows, WIDTH), e(rows, VOCAB, dtype=f32)
        self.q = [(e(rows, n, dtype=i8), e(rows, dtype=f32)) for n in (WIDTH, INNER, WIDTH)]
        self.tokens, self.probs = e(rows, dtype=torch.int64), e(rows, dtype=f32)
        self.top_k = torch.randint(1, 50, (rows,), generator=gen, dtype=torch.int32).cuda()
        self.temperature, self.top_p = torch.full((rows,), 0.8, device="cuda"), torch.full((rows,), 0.9, device="cuda")
        self.keep = []

    def gemm(self, a, w, c, dt, residual=None, act=None):
        p = capi.GemmQ8Params()
        p.dtype, p.epilogue_op = q8.DTYPES[dt][0], capi.OP[act] if act else 0
        p.m, p.n, p.k = a[0].shape[0], w[0].shape[0], w[0].shape[1]
        p.lda, p.ldb, p.ldc, p.scale_a, p.scale_b, p.residual = p.k, p.k, p.n, q8.at(a[1]), q8.at(w[1]), q8.at(residual)
        return self.lib.axhip_gemm_q8, (q8.at(a[0]), q8.at(w[0]), q8.at(c), C.byref(p))

    def calls(self):
        rows = q8.rows_params("bf16", self.rows, WIDTH, WIDTH, WIDTH)
        inner = q8.rows_params("bf16", self.rows, INNER, INNER, INNER)
        s = q8.sample_params(self.logits, "f32", self.u, self.temperature, self.top_k, self.top_p)
        self.keep = [rows, inner, s]
        (a, b, c), (up, down, head) = self.q, self.weights
        yield self.lib.axhip_rms_norm_q8, (q8.at(self.x), q8.at(self.res), q8.at(self.w), q8.at(self.sum), q8.at(a[0]), q8.at(a[1]), C.byref(rows))
        yield self.gemm(a, up, self.hidden, "bf16", act="silu")
        yield self.lib.axhip_quantize_q8, (q8.at(self.hidden), q8.at(b[0]), q8.at(b[1]), C.byref(inner))
        yield self.gemm(b, down, self.out, "bf16", residual=self.sum)
        yield self.lib.axhip_rms_norm_q8, (q8.at(self.out), None, q8.at(self.w), None, q8.at(c[0]), q8.at(c[1]), C.byref(rows))
        yield self.gemm(c, head, self.logits, "f32")
        assert self.lib.axhip_sample_workspace_bytes(C.byref(s)) == 0
        yield self.lib.axhip_sample_ws, (q8.at(self.logits), q8.at(self.tokens), q8.at(self.probs), C.byref(s), None, 0)

    def run(self, stream=None):
        for call, args in self.calls():
            capi.check(call(*args, stream))

    def results(self):
        return [t.clone() for t in (self.sum, self.q[0][0], self.hidden, self.q[1][0], self.out, self.q[2][0], self.logits, self.tokens, self.probs)]


@pytest.mark.parametrize("rows", [1, 2, 7, 40, 300])
def test_a_decoding_step(rows):
    s = Step(rows, rows)
    q8.sync()
    s.run()
    q8.sync()
    # each product from the integers that it was given; each row of integers from the values that it was given
    def product(a, w):
        return (a[0].cpu().double() @ w[0].cpu().double().T) * a[1].cpu().double()[:, None] * w[1].cpu().double()

    half = 1.01 * 2.0**-8
    (a, b, c), (up, down, head) = s.q, s.weights
    assert torch.equal(s.sum, (s.x.float() + s.res.float()).bfloat16())
    for q, values in ((a, q8.f64(s.sum) * q8.f64(s.w)), (b, q8.f64(s.hidden)), (c, q8.f64(s.out) * q8.f64(s.w))):
        assert np.array_equal(q[0].cpu().numpy(), q8.nearest(values)[1])
    y = product(a, up)
    y = y * torch.sigmoid(y)
    assert bool(((s.hidden.cpu().double() - y).abs() <= half * y.abs() + 4e-6).all())
    y = product(b, down) + s.sum.cpu().double()
    assert bool(((s.out.cpu().double() - y).abs() <= half * y.abs() + 4e-6).all())
    y = product(c, head)
    assert bool(((s.logits.cpu().double() - y).abs() <= 4 * 2.0**-24 * y.abs() + 1e-30).all())
    l, tokens = q8.f64(s.logits), s.tokens.cpu().numpy()
    for i in range(rows):
        token, prob, margin = q8.sampled(l[i], float(s.u[i]), float(np.float32(0.8)), int(s.top_k[i]), float(np.float32(0.9)))
        if margin > 1e-9:
            assert tokens[i] == token and abs(float(s.probs[i]) - prob) <= 1e-6


@pytest.mark.parametrize("rows", [1, 33])
def test_two_steps_captured_and_replayed(rows):
    """Two steps' calls in graphs of their own, replayed in turn with eager work and changed inputs between them."""
    s, other = Step(rows, 1), Step(rows, 2)
    stream = torch.cuda.Stream()
    graphs = []
    for step in (s, other):
        step.run(stream.cuda_stream)  # (kernels loaded before the capture)
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            step.run(stream.cuda_stream)
        graphs.append(g)
    for turn in range(4):
        for step, g in zip((s, other), graphs):
            step.x.copy_(torch.randn(rows, WIDTH, generator=torch.Generator().manual_seed(turn)).bfloat16())
            for t in (step.hidden, step.logits, step.tokens):
                t.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            got = step.results()
            torch.cuda.synchronize()
            step.run()
            q8.sync()
            assert all(torch.equal(x, y) for x, y in zip(got, step.results()))
