"""Sampling with one setting for every row, in the parameters: what is refused (no device is needed), and that it gives what the arrays give."""
import ctypes as C

import numpy as np
import pytest
import torch

from axiom_amd import capi
from tests import q8_harness as q8

X = 1 << 20  # an address that nothing reads
NAN = float("nan")


def uniform(p, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    p.uniform, p.all_temperature, p.all_top_k, p.all_top_p, p.all_min_p = 1, temperature, top_k, top_p, min_p
    return p


def test_what_is_refused():
    lib = capi.lib()
    assert lib.axhip_sizeof(7) == C.sizeof(capi.SampleParams)

    def params():
        p = capi.SampleParams()
        p.dtype, p.rows, p.vocab, p.ld, p.u = capi.DTYPE_F32, 4, 100, 100, X
        return p

    for value in (2, -1, 1 << 30):
        p = params()
        p.uniform = value
        assert lib.axhip_sample(X, X, X, C.byref(p), None) == capi.ERR_INVALID_ARG and b"uniform" in lib.axhip_last_error()
    for name in ("temperature", "top_k", "top_p", "min_p"):
        p = uniform(params())
        setattr(p, name, X)
        assert lib.axhip_sample(X, X, X, C.byref(p), None) == capi.ERR_INVALID_ARG and b"uniform" in lib.axhip_last_error()
    p = uniform(params())
    p.rows = 0
    capi.check(lib.axhip_sample(None, None, None, C.byref(p), None))


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 700, 0.8, 0.02), (0.0, 5, 0.5, 0.0), (NAN, 0, 1.0, 0.0), (1.0, -3, NAN, NAN), (0.9, 2**31 - 1, 2.0, 5.0), (0.05, 50, 1.0, 0.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [900, 5003, 70001])
def test_one_setting_is_that_of_an_array(dt, vocab):
    gen = torch.Generator()
    gen.manual_seed(vocab)
    rows = 7
    logits = (torch.randn(rows, vocab, generator=gen) * 2.5).to(q8.DTYPES[dt][1]).cuda()
    u = torch.rand(rows, generator=gen).clamp(max=1 - 2.0**-24)
    on = u.cuda()
    for temperature, top_k, top_p, min_p in SETTINGS:
        want, prob = q8.sample(logits, dt, u, temperature, top_k, top_p, min_p)
        tokens, probs = torch.full((rows,), -7, dtype=torch.int64, device="cuda"), torch.full((rows,), -7.0, device="cuda")
        p = uniform(q8.sample_params(logits, dt, on), temperature, top_k, top_p, min_p)
        q8.sync()
        capi.check(capi.lib().axhip_sample(q8.at(logits), q8.at(tokens), q8.at(probs), C.byref(p), None))
        q8.sync()
        assert np.array_equal(tokens.cpu().numpy(), want) and np.array_equal(probs.cpu().numpy(), prob)


@pytest.mark.gpu
def test_one_setting_captured_and_replayed():
    """The settings are the graph's, logits and random numbers whatever the device arrays hold at the replay."""
    gen = torch.Generator()
    gen.manual_seed(5)
    rows, vocab = 9, 5003
    logits, u = torch.empty(rows, vocab, device="cuda"), torch.empty(rows, device="cuda")
    tokens, probs = torch.empty(rows, dtype=torch.int64, device="cuda"), torch.empty(rows, device="cuda")
    p = uniform(q8.sample_params(logits, "f32", u), 0.8, 60, 0.95, 0.01)
    stream, lib = torch.cuda.Stream(), capi.lib()
    call = lambda: capi.check(lib.axhip_sample(q8.at(logits), q8.at(tokens), q8.at(probs), C.byref(p), stream.cuda_stream))  # noqa: E731
    logits.zero_(), u.zero_()
    torch.cuda.synchronize()
    call()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for _ in range(4):
        logits.copy_(torch.randn(rows, vocab, generator=gen) * 2.5)
        u.copy_(torch.rand(rows, generator=gen))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = tokens.cpu().numpy(), probs.cpu().numpy()
        want = q8.sample(logits, "f32", u.cpu(), 0.8, 60, 0.95, 0.01)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
