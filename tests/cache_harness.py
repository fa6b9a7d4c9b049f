"""Calls of the rotary and cache entry points on torch tensors, and their definitions in 64 bits (torch, CPU)."""
from __future__ import annotations

import ctypes as C
import math

import torch

from axiom_amd import capi

DTYPES = {"f32": (capi.DTYPE_F32, torch.float32), "f16": (capi.DTYPE_F16, torch.float16), "bf16": (capi.DTYPE_BF16, torch.bfloat16)}
LEFT = 7.0  # what memory that a call must leave alone holds


def at(t):
    return None if t is None else t.data_ptr()


def sync():
    torch.cuda.synchronize()
    capi.check(capi.lib().axhip_stream_sync(None))


def half(dt):
    """Of a rounding, relative to the value."""
    return torch.finfo(DTYPES[dt][1]).eps / 2


def generator(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


# ------------------------------------------------------------------- rotation
def scaling(rot, theta=10000.0, kind=capi.ROPE_PLAIN, factor=1.0, low=1.0, high=4.0, length=8192.0):
    s = capi.RopeScaling()
    s.rot_dim, s.kind, s.theta, s.factor, s.low, s.high, s.length = rot, kind, theta, factor, low, high, length
    return s


def turns(rot, **how):
    table = (C.c_uint64 * (rot // 2))()
    capi.check(capi.lib().axhip_rope_turns(C.byref(scaling(rot, **how)), table))
    return list(table)


def device_turns(values):
    return torch.tensor([v - (1 << 64) if v >= 1 << 63 else v for v in values], dtype=torch.int64).cuda()


def rotated(x, positions, table, rot, interleaved, inverse=False, amplitude=1.0):
    """In 64 bits, by the fractions of a turn in whole numbers: [tokens, heads, dim], and what a relative error of a sine moves each result by"""
    x = x.detach().cpu().double()
    angle = torch.tensor([[((int(p) * t) % 2**64) / 2**64 * 2 * math.pi for t in table] for p in positions], dtype=torch.float64)[:, None]
    c, s = angle.cos() * amplitude, angle.sin() * (-amplitude if inverse else amplitude)
    y, moved = x.clone(), torch.zeros_like(x)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    moved[..., a] = moved[..., b] = (x[..., a].abs() + x[..., b].abs()) * abs(amplitude)
    return y, moved


def rotation_tolerance(want, moved, dt):
    """Sines are within 2^-22; the amplitude, two products and their sum round to 32 bits once each; then the result's own rounding."""
    return half(dt) * want.abs() + moved * (2.0**-22 + 4 * 2.0**-24) + 1e-30 + (2.0**-25 if dt == "f16" else 0.0)


def rope(x, positions, table, rot, interleaved, dt, inverse=False, amplitude=1.0, out=None, stream=None):
    y = torch.full_like(x, LEFT) if out is None else out
    p = capi.RopeParams()
    p.dtype, p.heads, p.head_dim, p.rot_dim, p.interleaved, p.inverse, p.amplitude = DTYPES[dt][0], x.shape[1], x.shape[2], rot, int(interleaved), int(inverse), amplitude
    p.position_bytes, p.positions, p.turns, p.tokens = positions.element_size(), at(positions), at(table), x.shape[0]
    p.x_strides[:], p.y_strides[:] = x.stride()[:2], y.stride()[:2]
    sync()
    capi.check(capi.lib().axhip_rope(at(x), at(y), C.byref(p), stream))
    sync()
    return y


# ---------------------------------------------------------------------- pages
def pool(n_pages, page, heads, dim, dt, by_head=False, seed=0, layers=None, scale=1.0, pad=0):
    """K and V pages as views [(layers,) page, row, head, dim]; `pad`: elements between one head's dims and the next."""
    lead = () if layers is None else (layers,)
    outside, inside = (heads, page) if by_head else (page, heads)
    got = []
    for i in range(2):
        x = (torch.randn(*lead, n_pages, outside, inside, dim + pad, generator=generator(2 * seed + i)) * scale).to(DTYPES[dt][1]).cuda()[..., :dim]
        got.append(x.transpose(-3, -2) if by_head else x)
    return got


def pages_of(k, v, dt, to=None):
    p = capi.KvPages() if to is None else to
    p.k, p.v, p.dtype, p.page_size, p.heads, p.head_dim, p.n_pages = at(k), at(v), DTYPES[dt][0], k.shape[-3], k.shape[-2], k.shape[-1], k.shape[-4]
    p.k_strides[:], p.v_strides[:] = k.stride()[-4:-1], v.stride()[-4:-1]
    return p


def append_params(q, k, v, q_out, kp, vp, slots, dt, positions=None, table=None, rot=0, interleaved=False, amplitude=1.0):
    p = capi.KvAppendParams()
    pages_of(kp, vp, dt, p.pages)
    p.heads, p.rot_dim, p.interleaved, p.amplitude, p.tokens = 0 if q is None else q.shape[1], rot, int(interleaved), amplitude, k.shape[0]
    p.position_bytes, p.positions, p.turns, p.slots = 0 if positions is None else positions.element_size(), at(positions), at(table), at(slots)
    for to, x in ((p.q_strides, q), (p.k_strides, k), (p.v_strides, v), (p.q_out_strides, q_out)):
        if x is not None:
            to[:] = x.stride()[:2]
    return p


def append(q, k, v, q_out, kp, vp, slots, dt, stream=None, **how):
    p = append_params(q, k, v, q_out, kp, vp, slots, dt, **how)
    sync()
    capi.check(capi.lib().axhip_kv_append(at(q), at(k), at(v), at(q_out), C.byref(p), stream))
    sync()


def copy_params(kp, vp, src, dst, dt, rows=None):
    p = capi.KvCopyParams()
    pages_of(kp, vp, dt, p.pages)
    p.layers, p.pairs, p.src, p.dst, p.rows = kp.shape[0], len(src), at(src), at(dst), at(rows)
    p.k_layer_stride, p.v_layer_stride = kp.stride(0), vp.stride(0)
    return p


def table_of(lengths, page, order, columns=None, behind=-1):
    """A page table with pages from `order` in turn; (table, how many were taken)."""
    need = [-(-n // page) for n in lengths]
    t = torch.full((len(lengths), max([1, columns or 0] + need)), behind, dtype=torch.int32)
    used = 0
    for i, n in enumerate(need):
        t[i, :n] = torch.as_tensor(order[used:used + n], dtype=torch.int32)
        used += n
    return t, used


def rows_of(pages, table, n):
    """[n, heads, dim] of a sequence, float64 on the CPU"""
    page = pages.shape[1]
    i = torch.arange(n)
    return pages.detach().cpu().double()[table.long()[i // page], i % page] if n else torch.zeros(0, *pages.shape[2:], dtype=torch.float64)


# ------------------------------------------------------------------ attention
def attention(q, k, v, first, scale=None):
    """One sequence in 64 bits: q [rows, heads, dim], k, v [keys, key heads, dim], query i sees keys up to first + i (None: all) -> (o, sum p |v| / sum p,
    the largest sum of |q k| scale of a row)"""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    rows, heads, dim = q.shape
    each = heads // k.shape[1] if k.shape[1] else 1
    scale = dim**-0.5 if not scale or scale <= 0 else scale
    k, v = k.repeat_interleave(each, 1), v.repeat_interleave(each, 1)
    s = torch.einsum("rhd,khd->hrk", q, k) * scale
    if first is not None:
        s.masked_fill_(torch.arange(k.shape[0]) > first + torch.arange(rows)[:, None], -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else torch.zeros(*s.shape[:2], 1, dtype=torch.float64)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / torch.where(total > 0, total, torch.ones_like(total)), torch.zeros_like(p))
    big = torch.einsum("rhd,khd->hrk", q.abs(), k.abs()).amax(-1) * scale if k.shape[0] else torch.zeros(heads, rows, dtype=torch.float64)
    return torch.einsum("hrk,khd->rhd", p, v), torch.einsum("hrk,khd->rhd", p, v.abs()), big.T


def attention_tolerance(o, around, big, keys, dim, dt):
    """A score is a sum of `dim` products in 32 bits (one rounding of at most 2^-24 of sum |q k| each, and its scaling); a weight then is off by that and by its own
    rounding to dtype, in the numerator and in the denominator; sums over the keys round once a key; then the result's own rounding."""
    u = 0.0 if dt == "f32" else half(dt)
    weight = u + ((dim + 4) * 2.0**-24 * big[:, :, None] + 4 * 2.0**-24)
    return half(dt) * o.abs() + (2 * weight + 2 * (keys + 8) * 2.0**-24) * around + 1e-30 + (2.0**-24 if dt == "f16" else 0.0)


def packed_params(q, k, v, o, cu_q, dt, cu_kv=None, causal=True, scale=0.0, kp=None, vp=None, table=None, lengths=None, kv_heads=None, max_kv=1000):
    p = capi.SdpaPackedParams()
    p.dtype, p.heads, p.head_dim, p.n_seqs, p.is_causal, p.scale, p.max_kv = DTYPES[dt][0], q.shape[1], q.shape[2], len(cu_q) - 1, int(causal), scale, max_kv
    p.total_q, p.cu_q = q.shape[0], at(cu_q)
    p.q_strides[:], p.o_strides[:] = q.stride()[:2], o.stride()[:2]
    if table is None:
        p.kv_heads, p.total_kv, p.cu_kv = k.shape[1], k.shape[0], at(cu_kv)
        p.k_strides[:], p.v_strides[:] = k.stride()[:2], v.stride()[:2]
    else:
        p.kv_heads = kp.shape[2]
        pages_of(kp, vp, dt, p.pages)
        p.page_table, p.table_ld, p.kv_lengths = at(table), table.stride(0), at(lengths)
    return p


def workspace(need):
    """`need` bytes with a border behind them that has to stay as it is."""
    ws = torch.full((need + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    return ws, lambda: bool((ws[need:] == 0x5A).all())


def packed(q, k, v, cu_q, dt, stream=None, out=None, **how):
    lib = capi.lib()
    o = torch.full_like(q, LEFT) if out is None else out
    p = packed_params(q, k, v, o, cu_q, dt, **how)
    need = lib.axhip_sdpa_packed_workspace_bytes(C.byref(p))
    ws, intact = workspace(need)
    sync()
    capi.check(lib.axhip_sdpa_packed_ws(at(q), at(k), at(v), at(o), C.byref(p), at(ws) if need else None, need, stream))
    sync()
    assert intact()
    return o, lib.axhip_sdpa_cache_last_kernel().decode()


def paged_params(q, o, kp, vp, table, lengths, dt, scale=0.0, starts=None, prefix_table=None, prefix_lengths=None, max_kv=1000, max_prefix=1000):
    p = capi.SdpaPagedParams()
    pages_of(kp, vp, dt, p.pages)
    p.n_seqs, p.new_tokens, p.heads, p.scale, p.max_kv = q.shape[0], q.shape[1], q.shape[2], scale, max_kv
    p.q_strides[:], p.o_strides[:] = q.stride()[:3], o.stride()[:3]
    p.page_table, p.table_ld, p.kv_lengths = at(table), table.stride(0), at(lengths)
    if starts is not None:
        p.n_groups, p.max_prefix, p.group_starts = len(starts) - 1, max_prefix, at(starts)
        p.prefix_table, p.prefix_ld, p.prefix_lengths = at(prefix_table), prefix_table.stride(0), at(prefix_lengths)
    return p


def paged(q, kp, vp, table, lengths, dt, stream=None, out=None, **how):
    lib = capi.lib()
    o = torch.full_like(q, LEFT) if out is None else out
    p = paged_params(q, o, kp, vp, table, lengths, dt, **how)
    need = lib.axhip_sdpa_paged_workspace_bytes(C.byref(p))
    ws, intact = workspace(need)
    sync()
    capi.check(lib.axhip_sdpa_paged_ws(at(q), at(o), C.byref(p), at(ws) if need else None, need, stream))
    sync()
    assert intact()
    return o, lib.axhip_sdpa_cache_last_kernel().decode()
