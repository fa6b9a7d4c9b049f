"""Rotary positions, new tokens into the pages of a cache and pages copied, against their definitions in 64 bits."""
import ctypes as C

import pytest
import torch

from axiom_amd import capi
from tests import cache_harness as ch

pytestmark = pytest.mark.gpu


def near(got, want, moved, dt):
    off = (got.cpu().double() - want).abs() - ch.rotation_tolerance(want, moved, dt)
    assert float(off.max()) <= 0, float(off.max())


def normal(*shape, dt, seed=0):
    return torch.randn(*shape, generator=ch.generator(seed)).to(ch.DTYPES[dt][1]).cuda()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 40, 20), (7, 3, 33, 6), (65, 8, 128, 64), (2, 1, 256, 256), (700, 48, 128, 128), (129, 7, 80, 80), (4000, 9, 96, 32)])
def test_rope(dt, interleaved, tokens, heads, dim, rot):
    x = normal(tokens, heads, dim, dt=dt, seed=tokens)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=ch.generator(rot)).to(torch.int32 if tokens % 2 else torch.int64)
    positions[0] = 0
    table = ch.turns(rot, theta=500000.0)
    y = ch.rope(x, positions.cuda(), ch.device_turns(table), rot, interleaved, dt)
    want, moved = ch.rotated(x, positions, table, rot, interleaved)
    near(y, want, moved, dt)
    assert torch.equal(y[0], x[0]) and torch.equal(y[..., rot:], x[..., rot:])  # position 0 turns nothing; dims behind rot are copied


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_far_and_negative_positions_and_amplitude(dt, interleaved):
    positions = torch.tensor([-1, -12345, 2**31 - 1, 2**31 + 7, -(2**33), 2**40 + 1, 2**62], dtype=torch.int64)
    x = normal(len(positions), 4, 64, dt=dt)
    table = ch.turns(64, theta=1e6, kind=capi.ROPE_BANDS, factor=8.0)
    for inverse, amplitude in ((False, 1.25), (True, 1.0), (True, 0.75)):
        y = ch.rope(x, positions.cuda(), ch.device_turns(table), 64, interleaved, dt, inverse=inverse, amplitude=amplitude)
        near(y, *ch.rotated(x, positions, table, 64, interleaved, inverse, amplitude), dt)


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shift,pad", [(0, 0), (1, 3), (2, 2), (4, 4)])
def test_rope_of_views(dt, interleaved, shift, pad):
    """Heads in the middle of wider rows, from any element on, in place and out of place; what lies around them stays."""
    tokens, heads, dim, rot = 37, 6, 48, 24
    wide = normal(tokens, heads + 2, dim + pad, dt=dt, seed=shift)
    flat = torch.cat((wide.new_zeros(shift), wide.flatten()))
    view = flat[shift:].view(wide.shape)[:, 1:-1, :dim]
    positions, table = torch.arange(tokens, dtype=torch.int32) * 977, ch.turns(rot)
    want, moved = ch.rotated(view, positions, table, rot, interleaved)
    out = torch.full_like(wide, ch.LEFT)
    ch.rope(view, positions.cuda(), ch.device_turns(table), rot, interleaved, dt, out=out[:, 1:-1, :dim])
    near(out[:, 1:-1, :dim], want, moved, dt)
    assert bool((out[:, 0] == ch.LEFT).all() and (out[:, -1] == ch.LEFT).all() and (out[..., dim:] == ch.LEFT).all())
    before = flat.clone()
    ch.rope(view, positions.cuda(), ch.device_turns(table), rot, interleaved, dt, out=view)
    assert torch.equal(view, out[:, 1:-1, :dim])
    view.copy_(before[shift:].view(wide.shape)[:, 1:-1, :dim])
    assert torch.equal(flat, before)


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_inverse_is_the_gradient(interleaved):
    """<g, d rope(x) / dx h> by a difference along h (rope is linear: of any length) is <rope_inverse(g), h>."""
    positions, table = torch.arange(50, dtype=torch.int64) * 131, ch.turns(32)
    x, h, g = (normal(50, 3, 40, dt="f32", seed=s) for s in (1, 2, 3))
    how = dict(positions=positions.cuda(), table=ch.device_turns(table), rot=32, interleaved=interleaved, dt="f32", amplitude=1.5)
    difference = (ch.rope(x + h, **how).double() - ch.rope(x, **how).double())
    back = ch.rope(g, **how, inverse=True).double()
    left, right = (g.double() * difference).sum(), (back * h.double()).sum()
    # each of the 6000 results rounds a few times, as do x + h: no more than 16 roundings of 2^-24 of sums of magnitudes below 8
    assert abs(float(left - right)) <= 6000 * 16 * 2.0**-24 * 8
    both = ch.rotated(g, positions, table, 32, interleaved, True, 1.5)
    near(back, *both, "f32")


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot,page,interleaved", [(1, 8, 2, 64, 64, 16, False), (5, 0, 3, 40, 20, 8, False), (64, 32, 8, 128, 128, 16, False), (33, 6, 6, 80, 32, 1, True), (20, 4, 1, 36, 0, 4, False),
                                                                            (1000, 32, 8, 128, 128, 64, True), (7, 2, 2, 33, 6, 32, True)])
def test_append(dt, by_head, tokens, heads, kv_heads, dim, rot, page, interleaved):
    n_pages = -(-tokens // page) + 3
    kp, vp = ch.pool(n_pages, page, kv_heads, dim, dt, by_head, seed=1)
    qkv = normal(tokens, heads + 2 * kv_heads, dim, dt=dt, seed=tokens)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    q_out = torch.full((tokens, heads, dim), ch.LEFT, dtype=qkv.dtype, device="cuda") if heads else None
    slots = torch.randperm(n_pages * page, generator=ch.generator(tokens))[:tokens]
    if tokens > 4:
        slots[-1], slots[1], slots[2], slots[3] = -1, n_pages * page, 2**62, -(2**62)  # padding, and slots that do not exist
    positions, table = torch.randint(0, 100000, (tokens,), generator=ch.generator(3)), ch.turns(rot) if rot else None
    want_k, want_v = kp.cpu().double(), vp.cpu().double()
    moved_k = torch.zeros_like(want_k)
    rows, moved = ch.rotated(k, positions, table, rot, interleaved) if rot else (k.cpu().double(), torch.zeros(tokens, kv_heads, dim, dtype=torch.float64))
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < n_pages * page:
            want_k[s // page, s % page], want_v[s // page, s % page], moved_k[s // page, s % page] = rows[t], v[t].cpu().double(), moved[t]
    ch.append(q if heads else None, k, v, q_out, kp, vp, slots.cuda(), dt, positions=positions.cuda() if rot else None, table=ch.device_turns(table) if rot else None, rot=rot, interleaved=interleaved)
    untouched = (moved_k == 0) & (want_k == kp.cpu().double())
    near(kp, want_k, moved_k, dt)
    assert bool((untouched | (moved_k > 0) | (torch.tensor(rot == 0))).all()) and torch.equal(vp.cpu().double(), want_v)
    if heads:
        near(q_out, *(ch.rotated(q, positions, table, rot, interleaved) if rot else (q.cpu().double(), torch.zeros_like(q, device="cpu").double())), dt)
        ch.append(q, k, v, q, kp, vp, slots.cuda(), dt, positions=positions.cuda() if rot else None, table=ch.device_turns(table) if rot else None, rot=rot, interleaved=interleaved)  # q in place
        assert torch.equal(q, q_out)


def test_append_behind_four_gigabytes():
    """Pages farther from the pool's start than 32 bits of bytes and of elements."""
    heads, dim, page = 2, 64, 16
    n_pages = (1 << 32) // (heads * dim * page) + 4
    kp = torch.empty(n_pages, page, heads, dim, dtype=torch.float16, device="cuda")
    vp = torch.empty_like(kp)
    k, v = normal(3, heads, dim, dt="f16"), normal(3, heads, dim, dt="f16", seed=1)
    slots = torch.tensor([n_pages * page - 1, (1 << 31) // (heads * dim) + 5, 0]).cuda()
    ch.append(None, k, v, None, kp, vp, slots, "f16")
    for t, s in enumerate(slots.tolist()):
        assert torch.equal(kp[s // page, s % page], k[t]) and torch.equal(vp[s // page, s % page], v[t])
    kp, vp = kp[None], vp[None]
    p = ch.copy_params(kp, vp, torch.tensor([n_pages - 1], dtype=torch.int32).cuda(), torch.tensor([n_pages - 2], dtype=torch.int32).cuda(), "f16")
    ch.sync()
    capi.check(capi.lib().axhip_kv_copy_pages(C.byref(p), None))
    ch.sync()
    assert torch.equal(kp[0, -1, -1], kp[0, -2, -1]) and torch.equal(vp[0, -1, -1], vp[0, -2, -1])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("by_head,pad", [(False, 0), (True, 0), (False, 8), (True, 3)])
@pytest.mark.parametrize("pairs,layers,heads,dim,page", [(1, 1, 1, 2, 1), (1, 3, 8, 128, 16), (40, 5, 3, 40, 8), (7, 2, 2, 33, 64), (300, 2, 8, 64, 32)])
@pytest.mark.parametrize("partial", [False, True])
def test_copy(dt, by_head, pad, pairs, layers, heads, dim, page, partial):
    n_pages = 2 * pairs + 3
    kp, vp = ch.pool(n_pages, page, heads, dim, dt, by_head, seed=pairs, layers=layers, pad=pad)
    order = torch.randperm(n_pages, generator=ch.generator(pairs)).to(torch.int32)
    src, dst = order[:pairs].clone(), order[pairs:2 * pairs].clone()
    rows = torch.randint(-1, page + 3, (pairs,), generator=ch.generator(page), dtype=torch.int32) if partial else None
    if pairs > 5:
        src[0], dst[1], src[2], dst[3], dst[4] = -1, n_pages, 2**31 - 1, -(2**31), src[4]  # pages that do not exist, and a page onto itself
    want = [kp.clone(), vp.clone()]
    for i, (a, b) in enumerate(zip(src.tolist(), dst.tolist())):
        n = page if rows is None else min(max(int(rows[i]), 0), page)
        if 0 <= a < n_pages and 0 <= b < n_pages:
            for w in want:
                w[:, b, :n] = w[:, a, :n]
    p = ch.copy_params(kp, vp, src.cuda(), dst.cuda(), dt, None if rows is None else rows.cuda())
    keep = [src.cuda(), dst.cuda(), rows.cuda() if partial else None]
    p.src, p.dst, p.rows = (ch.at(t) for t in keep)
    ch.sync()
    capi.check(capi.lib().axhip_kv_copy_pages(C.byref(p), None))
    ch.sync()
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


# 64 MiB and more of output, which are stored past the caches, are the same bits as in calls of less
@pytest.mark.parametrize("dt,heads,dim,rot,tokens", [("bf16", 9, 80, 32, 46700), ("f32", 7, 96, 96, 25001), ("f16", 5, 36, 20, 190001)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_of_large_outputs(dt, heads, dim, rot, tokens, interleaved):
    x = normal(tokens, heads, dim, dt=dt, seed=4)
    assert x.numel() * x.element_size() >= 64 << 20
    positions, table = torch.randint(0, 1 << 20, (tokens,), generator=ch.generator(5)).cuda(), ch.turns(rot)
    how = dict(table=ch.device_turns(table), rot=rot, interleaved=interleaved, dt=dt)
    y = ch.rope(x, positions, **how)
    for rows in torch.arange(tokens).split(-(-tokens // 3)):
        part = slice(int(rows[0]), int(rows[-1]) + 1)
        assert torch.equal(y[part], ch.rope(x[part], positions[part], **how))
    some = torch.tensor([0, 1, tokens // 2, tokens - 1])
    near(y[some.cuda()], *ch.rotated(x[some.cuda()], positions.cpu()[some], table, rot, interleaved), dt)
    ch.rope(x, positions, **how, out=x)
    assert torch.equal(x, y)


@pytest.mark.parametrize("dt,heads,kv_heads,dim,rot,tokens,page,by_head", [("bf16", 5, 3, 96, 64, 32003, 16, True), ("f32", 3, 1, 80, 80, 43000, 64, False), ("f16", 7, 2, 128, 0, 24001, 8, False)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_of_large_outputs(dt, heads, kv_heads, dim, rot, tokens, page, by_head, interleaved):
    n_pages = -(-tokens // page) + 3
    qkv = normal(tokens, heads + 2 * kv_heads, dim, dt=dt, seed=6)
    assert qkv.numel() * qkv.element_size() >= 64 << 20
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    slots = torch.randperm(n_pages * page, generator=ch.generator(7))[:tokens].cuda()
    slots[-tokens // 16:] = -1
    positions, table = torch.randint(0, 100000, (tokens,), generator=ch.generator(8)).cuda(), ch.device_turns(ch.turns(rot)) if rot else None
    got = []
    for parts in (1, 3):
        kp, vp = ch.pool(n_pages, page, kv_heads, dim, dt, by_head, seed=9)
        q_out = torch.full((tokens, heads, dim), ch.LEFT, dtype=qkv.dtype, device="cuda")
        for rows in torch.arange(tokens).split(-(-tokens // parts)):
            part = slice(int(rows[0]), int(rows[-1]) + 1)
            ch.append(q[part], k[part], v[part], q_out[part], kp, vp, slots[part], dt, positions=positions[part] if rot else None, table=table, rot=rot, interleaved=interleaved)
        got.append((kp, vp, q_out))
    for one, three in zip(*got):
        assert torch.equal(one, three)
    written = slots >= 0
    assert torch.equal(got[0][1][slots[written] // page, slots[written] % page], v[written])
    ch.append(q, k, v, q, kp, vp, slots, dt, positions=positions if rot else None, table=table, rot=rot, interleaved=interleaved)  # q in place
    assert torch.equal(q, q_out)
