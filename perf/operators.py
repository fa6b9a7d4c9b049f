"""The 8-bit path of a decoder layer and the end of a decoding step, as cases that can be timed and compared.

    norm      the residual's addition and the RMS norm of the sum, out in 8 bits with a scale for each row (axhip_rms_norm_q8)
    quantize  rows in 8 bits with a scale each: weights by output channel, activations by token (axhip_quantize_q8)
    linear    x W^T of 8-bit integers with scales for each token and channel, bias, residual, activation (axhip_gemm_q8)
    sample    a token from each row of logits by temperature, top-k, top-p and min-p, from given random numbers (axhip_sample)

With `own` the passes go through the C ABI the way a program holding device buffers calls it: outputs, parameter structs and workspaces
are made once, a pass is the call, on the library's own stream.  Without it they are plain torch operations.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
ACTS = {"none": 0, "relu": 16, "gelu": 17, "silu": 24}  # AXHIP_OP_* of the epilogue


def listed():
    return [
        # one new token through a layer of the encoder example's largest width: launch and latency, nothing else
        dict(name="norm_1_row", kind="norm", dtype="bf16", rows=1, cols=1280, residual=True),
        # a batch of prompts between two blocks
        dict(name="norm_8192_rows", kind="norm", dtype="bf16", rows=8192, cols=4096, residual=True),
        # thirty seconds of audio in the reference's default type, a width that is no multiple of a vector
        dict(name="norm_f32_odd", kind="norm", dtype="f32", rows=1500, cols=1283, residual=False),
        # 64 conversations' activations before the second product of a feed-forward block
        dict(name="quantize_64_rows", kind="quantize", dtype="f16", rows=64, cols=5120),
        # a weight matrix as it is loaded, by output channel
        dict(name="quantize_weights", kind="quantize", dtype="f32", rows=4096, cols=4096),
        # one token against a weight matrix: one read of the weights
        dict(name="linear_1_row", kind="linear", dtype="bf16", m=1, n=4096, k=4096, bias=False, residual=False, act="none"),
        # 64 conversations decoding together
        dict(name="linear_64_rows", kind="linear", dtype="bf16", m=64, n=4096, k=4096, bias=True, residual=False, act="none"),
        # thirty seconds of audio through the first product of a feed-forward block
        dict(name="linear_1500_rows_gelu", kind="linear", dtype="f16", m=1500, n=5120, k=1280, bias=True, residual=False, act="gelu"),
        # a batch of prompts through a projection back into the residual stream
        dict(name="linear_8192_rows", kind="linear", dtype="bf16", m=8192, n=4096, k=4096, bias=False, residual=True, act="none"),
        # the next token of one conversation, the vocabulary of the encoder example's family
        dict(name="sample_1_row", kind="sample", dtype="f32", rows=1, vocab=51865, filters="k"),
        # 64 conversations, each with settings of its own
        dict(name="sample_64_rows", kind="sample", dtype="bf16", rows=64, vocab=51865, filters="kpm"),
        # a large batch over a large vocabulary, nucleus sampling
        dict(name="sample_256_rows", kind="sample", dtype="bf16", rows=256, vocab=128256, filters="p"),
    ]


# ---------------------------------------------------------------------- draws
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _ragged(rng, lo, hi, multiple=64):
    """A size over the whole range: in half of the draws a multiple of `multiple`, in the others any number."""
    n = _log(rng, lo, hi)
    return max(multiple, n // multiple * multiple) if rng.random() < 0.5 and n >= multiple else n


def draw(rng):
    kind = rng.choice(("norm", "quantize", "linear", "linear", "sample", "sample"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    while True:
        if kind == "norm":
            case = dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 16384), cols=_ragged(rng, 64, 16384), residual=rng.random() < 0.7)
        elif kind == "quantize":
            case = dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 16384), cols=_ragged(rng, 64, 16384))
        elif kind == "linear":
            case = dict(kind=kind, dtype=dtype, m=_ragged(rng, 1, 8192), n=_ragged(rng, 64, 8192), k=_ragged(rng, 64, 8192), bias=rng.random() < 0.6,
                        residual=rng.random() < 0.3, act=rng.choice(("none", "none", "relu", "gelu", "silu")))
        else:
            case = dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, 128256), filters=rng.choice(("", "k", "p", "m", "kp", "kpm")))
        need = work(case)
        if need["flops"] <= 2.7e11 and need["bytes"] <= 1.7e8:
            return case


# ----------------------------------------------------------------------- work
def work(case):
    c, es = case, SIZES[case["dtype"]]
    if c["kind"] == "norm":  # x, the residual and the weight in; the sum, the integers and the scales out
        size = c["rows"] * c["cols"]
        return {"bytes": size * (3 * es if c["residual"] else es) + es * c["cols"] + size + 4 * c["rows"], "flops": 6 * size}
    if c["kind"] == "quantize":
        size = c["rows"] * c["cols"]
        return {"bytes": size * es + size + 4 * c["rows"], "flops": 3 * size}
    if c["kind"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + es * (m * n * (2 if c["residual"] else 1) + (n if c["bias"] else 0)), "flops": 2 * m * n * k}
    size = c["rows"] * c["vocab"]
    return {"bytes": size * es + 12 * c["rows"] + 4 * c["rows"] * (2 + len(c["filters"])), "flops": 4 * size}


# --------------------------------------------------------------------- inputs
def prepare(case, seed):
    c, t = case, DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))

    def normal(*shape, scale=1.0, shift=0.0, dtype=t):
        return (torch.randn(shape, device="cuda", generator=gen) * scale + shift).to(dtype)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(shape, device="cuda", generator=gen) * (hi - lo) + lo

    s = dict(case)
    if c["kind"] in ("norm", "quantize"):
        rows, cols = c["rows"], c["cols"]
        x = normal(rows, cols)
        x[:, :: max(1, cols // 5)] *= 12  # the few channels that carry large values
        x[rows - rows // 16:] = 0  # the padded end of a batch
        s.update(x=x, q=torch.empty(rows, cols, dtype=torch.int8, device="cuda"), scales=torch.empty(rows, device="cuda"))
        if c["kind"] == "norm":
            s.update(weight=normal(cols, scale=0.2, shift=1.0), r=normal(rows, cols, scale=3.0) if c["residual"] else None,
                     sum=torch.empty_like(x) if c["residual"] else None)
    elif c["kind"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        for name, rows in (("a", m), ("b", n)):
            s[name] = normal(rows, k, scale=30.0, dtype=torch.float32).round_().clamp_(-127, 127).to(torch.int8)
            s["scale_" + name] = uniform(rows, lo=0.5, hi=1.5) / (30.0 * k**0.25)
        s.update(bias=normal(n, scale=0.1) if c["bias"] else None, r=normal(m, n) if c["residual"] else None, c=torch.empty(m, n, dtype=t, device="cuda"))
    else:
        rows, vocab = c["rows"], c["vocab"]
        s.update(logits=normal(rows, vocab, scale=2.5), u=uniform(rows).clamp_(max=1 - 2.0**-24), temperature=uniform(rows, lo=0.6, hi=1.2), top_k=None, top_p=None, min_p=None,
                 tokens=torch.empty(rows, dtype=torch.int64, device="cuda"), probs=torch.empty(rows, device="cuda"))
        if "k" in c["filters"]:
            s["top_k"] = torch.randint(1, 200, (rows,), device="cuda", generator=gen, dtype=torch.int32)
        if "p" in c["filters"]:
            s["top_p"] = uniform(rows, lo=0.7, hi=0.99)
        if "m" in c["filters"]:
            s["min_p"] = uniform(rows, lo=0.0, hi=0.1)
    return s


# ------------------------------------------------------------- the plain forms
def _integers(y):
    """Rows of values -> their largest magnitudes and the integers that stand for them, in 64 bits: which integer is nearest shows in no fewer."""
    y = y.double()
    largest = y.abs().amax(-1, keepdim=True)
    q = torch.round(127.0 * y / torch.where(largest > 0, largest, torch.ones_like(largest)))
    return largest[:, 0], q.to(torch.int8)


def _plain_norm(s):
    h = s["x"] if s["r"] is None else (s["x"].float() + s["r"].float()).to(s["x"].dtype)
    largest, q = _integers(h.double() * s["weight"].double())
    scales = largest.float() * torch.rsqrt(h.float().square().mean(-1) + EPS) / 127.0
    return {"q": q, "scales": scales} if s["r"] is None else {"q": q, "scales": scales, "sum": h}


def _plain_quantize(s):
    largest, q = _integers(s["x"])
    return {"q": q, "scales": largest.float() / 127.0}


def _plain_linear(s):
    y = (s["a"].float() @ s["b"].float().T) * (s["scale_a"][:, None] * s["scale_b"])
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["r"] is not None:
        y = y + s["r"].float()
    if s["act"] == "relu":
        y = y.clamp(min=0)
    elif s["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * 0.5**0.5))
    elif s["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    return y.to(s["c"].dtype)


def _plain_sample(s):
    """In 64 bits: which token a random number falls on is a comparison of long sums."""
    logits, ids = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)  # (equal ones: the lowest index first)
    w = torch.exp((logits - logits[:, :1]) / s["temperature"].double()[:, None])
    place = torch.arange(w.shape[1], device=w.device)
    kept = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        kept &= place < s["top_k"][:, None]
    if s["top_p"] is not None:
        mass = torch.where(kept, w, 0.0)
        before = torch.cumsum(mass, -1) - mass
        kept &= (before < s["top_p"].double()[:, None] * mass.sum(-1, keepdim=True)) | (place == 0)
    if s["min_p"] is not None:
        kept &= (w >= s["min_p"].double()[:, None]) | (place == 0)
    mass = torch.zeros_like(w).scatter_(1, ids, torch.where(kept, w, 0.0))  # by index again
    upto = torch.cumsum(mass, -1)
    total = upto[:, -1:]
    tokens = (upto > s["u"].double()[:, None] * total).to(torch.uint8).argmax(-1)
    return {"tokens": tokens, "probs": (mass.gather(1, tokens[:, None]) / total)[:, 0].float()}


# --------------------------------------------------------- the library's calls
def _own_call(s):
    """The call of a pass, its parameters filled in, and what it writes."""
    import ctypes as C

    from axiom_amd import capi

    lib = capi.lib()
    capi.check(lib.axhip_init(0))

    def at(t):
        return None if t is None else t.data_ptr()

    code = {"f32": capi.DTYPE_F32, "f16": capi.DTYPE_F16, "bf16": capi.DTYPE_BF16}[s["dtype"]]
    if s["kind"] in ("norm", "quantize"):
        p = capi.RowsQ8Params()
        p.dtype, p.eps, p.rows, p.cols = code, EPS, s["rows"], s["cols"]
        p.ld_x = p.ld_residual = p.ld_sum = p.ld_q = s["cols"]
        if s["kind"] == "quantize":
            return capi.check, lib.axhip_quantize_q8, (at(s["x"]), at(s["q"]), at(s["scales"]), C.byref(p), None), {"q": s["q"], "scales": s["scales"]}
        out = {"q": s["q"], "scales": s["scales"]}
        if s["r"] is not None:
            out["sum"] = s["sum"]
        return capi.check, lib.axhip_rms_norm_q8, (at(s["x"]), at(s["r"]), at(s["weight"]), at(s["sum"]), at(s["q"]), at(s["scales"]), C.byref(p), None), out
    if s["kind"] == "linear":
        p = capi.GemmQ8Params()
        p.dtype, p.epilogue_op, p.m, p.n, p.k = code, ACTS[s["act"]], s["m"], s["n"], s["k"]
        p.lda, p.ldb, p.ldc = s["k"], s["k"], s["n"]
        p.scale_a, p.scale_b, p.bias, p.residual = at(s["scale_a"]), at(s["scale_b"]), at(s["bias"]), at(s["r"])
        return capi.check, lib.axhip_gemm_q8, (at(s["a"]), at(s["b"]), at(s["c"]), C.byref(p), None), s["c"]
    p = capi.SampleParams()
    p.dtype, p.rows, p.vocab, p.ld = code, s["rows"], s["vocab"], s["vocab"]
    p.temperature, p.top_k, p.top_p, p.min_p, p.u = at(s["temperature"]), at(s["top_k"]), at(s["top_p"]), at(s["min_p"]), at(s["u"])
    need = lib.axhip_sample_workspace_bytes(C.byref(p))
    s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    return capi.check, lib.axhip_sample_ws, (at(s["logits"]), at(s["tokens"]), at(s["probs"]), C.byref(p), at(s["workspace"]), need, None), {"tokens": s["tokens"], "probs": s["probs"]}


def run(state):
    s = state
    if own:
        if "call" not in s:
            s["call"] = _own_call(s)
        check, call, args, out = s["call"]
        check(call(*args))
        return out
    return {"norm": _plain_norm, "quantize": _plain_quantize, "linear": _plain_linear, "sample": _plain_sample}[s["kind"]](s)


# ------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "linear":
        total = torch.mm(s["a"].to(torch.float64), s["b"].to(torch.float64).t()) * torch.outer(s["scale_a"].double(), s["scale_b"].double())
        for more in (s["bias"], s["r"]):
            if more is not None:
                total += more.double()
        if s["act"] == "relu":
            return torch.relu(total)
        if s["act"] == "gelu":
            return total * torch.special.ndtr(total)
        return total * torch.sigmoid(total) if s["act"] == "silu" else total
    if s["kind"] == "sample":
        # The probability of the token that is drawn, row by row: the kept ones are those before the first that a filter turns away.
        probs = []
        for i in range(s["rows"]):
            l = s["logits"][i].double()
            p = torch.softmax(l / s["temperature"][i].double(), 0)
            order = torch.argsort(-l, stable=True)
            n = len(order) if s["top_k"] is None else min(len(order), int(s["top_k"][i]))
            p = p / p[order[:n]].sum()
            if s["top_p"] is not None:
                reached = torch.cumsum(p[order[:n]], 0) >= s["top_p"][i].double()
                n = min(n, int(torch.nonzero(reached)[0]) + 1) if bool(reached.any()) else n
            if s["min_p"] is not None:
                n = max(1, int((p[order[:n]] >= s["min_p"][i].double() * p[order[0]]).sum()))
            chosen = torch.sort(order[:n]).values
            q = p[chosen] / p[chosen].sum()
            at = int(torch.searchsorted(torch.cumsum(q, 0), s["u"][i].double(), right=True))
            probs.append(q[min(at, n - 1)])
        return {"tokens": None, "probs": torch.stack(probs)}
    h = s["x"].double()
    if s["kind"] == "norm":
        if s["r"] is not None:
            h = (h + s["r"].double()).to(s["x"].dtype).double()  # (the sum is rounded to the type it is handed on in)
        y = h * s["weight"].double()
        spread = (h.pow(2).sum(1) / h.shape[1] + EPS).sqrt()
    else:
        y, spread = h, torch.ones(len(h), dtype=torch.float64, device=h.device)
    out = {"q": None, "scales": torch.linalg.vector_norm(y, ord=math.inf, dim=1) / (127 * spread)}
    if s["kind"] == "norm" and s["r"] is not None:
        out["sum"] = h
    return out
