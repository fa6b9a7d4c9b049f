"""What the rotary and cache entry points refuse, before any launch: no device is needed."""
import ctypes as C

import pytest

from axiom_amd import capi

X = 1 << 20  # an address that nothing reads


def refused(code, call, *args):
    with pytest.raises(capi.AxhipError) as e:
        capi.check(call(*args))
    assert e.value.code == code, str(e.value)
    return str(e.value)


def changed(p, change):
    for name, value in change.items():
        at = p
        *path, last = name.split("__")
        for part in path:
            at = getattr(at, part)
        if isinstance(value, tuple):
            getattr(at, last)[:] = value
        else:
            setattr(at, last, value)
    return p


def test_struct_layouts_match_the_compiled_library():
    for which, cls in ((8, capi.RopeScaling), (9, capi.RopeParams), (10, capi.KvPages), (11, capi.KvAppendParams), (12, capi.KvCopyParams), (13, capi.SdpaPackedParams), (14, capi.SdpaPagedParams)):
        assert capi.lib().axhip_sizeof(which) == C.sizeof(cls)


def rope_params():
    p = capi.RopeParams()
    p.dtype, p.heads, p.head_dim, p.rot_dim, p.tokens, p.position_bytes, p.positions, p.turns = capi.DTYPE_BF16, 4, 64, 64, 3, 8, X, X
    p.x_strides[:] = p.y_strides[:] = (256, 64)
    return p


@pytest.mark.parametrize("change", [dict(dtype=3), dict(dtype=-1), dict(tokens=-1), dict(heads=-1), dict(heads=1 << 20), dict(head_dim=1), dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=66), dict(interleaved=2),
                                    dict(inverse=-1), dict(amplitude=float("nan")), dict(amplitude=float("inf")), dict(position_bytes=2), dict(positions=None), dict(turns=None), dict(positions=X + 4), dict(turns=X + 4),
                                    dict(x_strides=(-1, 64)), dict(y_strides=(256, -64)), dict(y_strides=(0, 64)), dict(y_strides=(256, 63)), dict(x_strides=(1 << 41, 64))])
def test_rope(change):
    refused(capi.ERR_INVALID_ARG, capi.lib().axhip_rope, X, 2 * X, C.byref(changed(rope_params(), change)), None)


def test_rope_more():
    lib = capi.lib()
    refused(capi.ERR_INVALID_ARG, lib.axhip_rope, X, X, None, None)
    for args in ((None, X), (X, None), (X + 1, 2 * X), (X, 2 * X + 1)):
        refused(capi.ERR_INVALID_ARG, lib.axhip_rope, *args, C.byref(rope_params()), None)
    assert "in place" in refused(capi.ERR_INVALID_ARG, lib.axhip_rope, X, X, C.byref(changed(rope_params(), dict(x_strides=(512, 64)))), None)
    for nothing in (dict(tokens=0), dict(heads=0)):
        capi.check(lib.axhip_rope(None, None, C.byref(changed(rope_params(), nothing)), None))


def pages(p):
    p.k, p.v, p.dtype, p.page_size, p.heads, p.head_dim, p.n_pages = X, X, capi.DTYPE_BF16, 16, 2, 64, 10
    p.k_strides[:] = p.v_strides[:] = (2048, 128, 64)


BAD_PAGES = [dict(pages__dtype=3), dict(pages__page_size=0), dict(pages__page_size=-16), dict(pages__page_size=24), dict(pages__page_size=1 << 17), dict(pages__heads=0), dict(pages__head_dim=0),
             dict(pages__n_pages=-1), dict(pages__n_pages=1 << 31), dict(pages__k_strides=(-1, 0, 0)), dict(pages__v_strides=(0, 0, 1 << 40)), dict(pages__k=None), dict(pages__v=None), dict(pages__k=X + 1)]


def append_params():
    p = capi.KvAppendParams()
    pages(p.pages)
    p.heads, p.rot_dim, p.tokens, p.position_bytes, p.positions, p.turns, p.slots = 4, 64, 3, 4, X, X, X
    p.q_strides[:] = p.q_out_strides[:] = (256, 64)
    p.k_strides[:] = p.v_strides[:] = (128, 64)
    return p


@pytest.mark.parametrize("change", BAD_PAGES + [dict(tokens=-1), dict(heads=-1), dict(rot_dim=-2), dict(rot_dim=65), dict(rot_dim=66), dict(interleaved=2), dict(amplitude=float("inf")), dict(position_bytes=0),
                                                dict(positions=None), dict(turns=None), dict(slots=None), dict(slots=X + 4), dict(q_strides=(-1, 64)), dict(k_strides=(128, -1)), dict(v_strides=(1 << 40, 64)),
                                                dict(q_out_strides=(0, 64)), dict(q_out_strides=(256, 32))])
def test_append(change):
    refused(capi.ERR_INVALID_ARG, capi.lib().axhip_kv_append, X, X, X, 2 * X, C.byref(changed(append_params(), change)), None)


def test_append_more():
    lib = capi.lib()
    refused(capi.ERR_INVALID_ARG, lib.axhip_kv_append, X, X, X, X, None, None)
    for args in ((None, X, X, X), (X, None, X, X), (X, X, None, X), (X, X, X, None), (X + 1, X, X, X), (X, X + 1, X, X)):
        refused(capi.ERR_INVALID_ARG, lib.axhip_kv_append, *args, C.byref(append_params()), None)
    assert "in place" in refused(capi.ERR_INVALID_ARG, lib.axhip_kv_append, X, X, X, X, C.byref(changed(append_params(), dict(q_strides=(512, 64)))), None)
    capi.check(lib.axhip_kv_append(None, None, None, None, C.byref(changed(append_params(), dict(tokens=0))), None))


def copy_params():
    p = capi.KvCopyParams()
    pages(p.pages)
    p.layers, p.pairs, p.src, p.dst = 2, 3, X, X
    p.k_layer_stride = p.v_layer_stride = 20480
    return p


@pytest.mark.parametrize("change", BAD_PAGES + [dict(layers=-1), dict(pairs=-1), dict(k_layer_stride=-1), dict(v_layer_stride=1 << 41), dict(src=None), dict(dst=None), dict(src=X + 2), dict(rows=X + 1)])
def test_copy(change):
    refused(capi.ERR_INVALID_ARG, capi.lib().axhip_kv_copy_pages, C.byref(changed(copy_params(), change)), None)


def test_copy_more():
    refused(capi.ERR_INVALID_ARG, capi.lib().axhip_kv_copy_pages, None, None)
    for nothing in (dict(pairs=0), dict(layers=0), dict(pages__n_pages=0)):
        capi.check(capi.lib().axhip_kv_copy_pages(C.byref(changed(copy_params(), nothing)), None))


def packed_params(paged=False):
    p = capi.SdpaPackedParams()
    p.dtype, p.heads, p.kv_heads, p.head_dim, p.n_seqs, p.is_causal, p.total_q, p.total_kv = capi.DTYPE_BF16, 4, 2, 64, 3, 1, 50, 50
    p.q_strides[:] = p.o_strides[:] = (256, 64)
    p.k_strides[:] = p.v_strides[:] = (128, 64)
    p.cu_q, p.cu_kv = X, X
    if paged:
        pages(p.pages)
        p.page_table, p.kv_lengths, p.table_ld = X, X, 5
    return p


@pytest.mark.parametrize("change", [dict(dtype=3), dict(heads=0), dict(kv_heads=0), dict(heads=5), dict(heads=-4, kv_heads=-2), dict(head_dim=0), dict(n_seqs=-1), dict(n_seqs=1 << 24), dict(is_causal=2),
                                    dict(scale=float("nan")), dict(scale=float("inf")), dict(total_q=-1), dict(total_q=1 << 31), dict(total_kv=-1), dict(q_strides=(-1, 64)), dict(o_strides=(256, -1)),
                                    dict(k_strides=(1 << 40, 64)), dict(v_strides=(128, -64)), dict(cu_q=None), dict(cu_kv=None), dict(cu_q=X + 2), dict(cu_kv=X + 1)])
def test_packed(change):
    p = changed(packed_params(), change)
    refused(capi.ERR_INVALID_ARG, capi.lib().axhip_sdpa_packed, X, X, X, X, C.byref(p), None)
    refused(capi.ERR_INVALID_ARG, capi.lib().axhip_sdpa_packed_ws, X, X, X, X, C.byref(p), None, 0, None)
    assert capi.lib().axhip_sdpa_packed_workspace_bytes(C.byref(p)) == 0


@pytest.mark.parametrize("change", BAD_PAGES + [dict(pages__dtype=0), dict(pages__heads=4), dict(pages__head_dim=128), dict(table_ld=0), dict(table_ld=1 << 31), dict(kv_lengths=None), dict(page_table=X + 2)])
def test_packed_over_pages(change):
    refused(capi.ERR_INVALID_ARG, capi.lib().axhip_sdpa_packed, X, None, None, X, C.byref(changed(packed_params(True), change)), None)


def test_packed_more():
    lib = capi.lib()
    refused(capi.ERR_INVALID_ARG, lib.axhip_sdpa_packed, X, X, X, X, None, None)
    for args in ((None, X, X, X), (X, None, X, X), (X, X, None, X), (X, X, X, None), (X + 1, X, X, X), (X, X, X + 1, X)):
        refused(capi.ERR_INVALID_ARG, lib.axhip_sdpa_packed, *args, C.byref(packed_params()), None)
    assert "beside" in refused(capi.ERR_INVALID_ARG, lib.axhip_sdpa_packed, X, X, X, X, C.byref(packed_params(True)), None)
    refused(capi.ERR_UNSUPPORTED, lib.axhip_sdpa_packed, X, X, X, X, C.byref(changed(packed_params(), dict(head_dim=257))), None)
    for nothing in (dict(n_seqs=0), dict(total_q=0)):
        capi.check(lib.axhip_sdpa_packed(None, None, None, None, C.byref(changed(packed_params(), nothing)), None))
        assert lib.axhip_sdpa_cache_last_kernel() == b"empty"


def paged_params():
    p = capi.SdpaPagedParams()
    pages(p.pages)
    p.heads, p.n_seqs, p.new_tokens, p.table_ld, p.page_table, p.kv_lengths = 4, 3, 1, 5, X, X
    p.q_strides[:] = p.o_strides[:] = (256, 256, 64)
    p.n_groups, p.group_starts, p.prefix_table, p.prefix_lengths, p.prefix_ld = 1, X, X, X, 4
    return p


@pytest.mark.parametrize("change", BAD_PAGES + [dict(heads=3), dict(heads=0), dict(n_seqs=-1), dict(new_tokens=0), dict(new_tokens=1 << 20), dict(scale=float("nan")), dict(n_groups=-1), dict(reserved=1),
                                                dict(q_strides=(-1, 0, 0)), dict(o_strides=(0, 0, 1 << 40)), dict(page_table=None), dict(kv_lengths=None), dict(table_ld=0), dict(group_starts=None),
                                                dict(prefix_table=None), dict(prefix_lengths=None), dict(prefix_ld=0), dict(prefix_table=X + 1), dict(kv_lengths=X + 2)])
def test_paged(change):
    p = changed(paged_params(), change)
    refused(capi.ERR_INVALID_ARG, capi.lib().axhip_sdpa_paged, X, X, C.byref(p), None)
    refused(capi.ERR_INVALID_ARG, capi.lib().axhip_sdpa_paged_ws, X, X, C.byref(p), None, 0, None)
    assert capi.lib().axhip_sdpa_paged_workspace_bytes(C.byref(p)) == 0


def test_paged_more():
    lib = capi.lib()
    refused(capi.ERR_INVALID_ARG, lib.axhip_sdpa_paged, X, X, None, None)
    for args in ((None, X), (X, None), (X + 1, X), (X, X + 1)):
        refused(capi.ERR_INVALID_ARG, lib.axhip_sdpa_paged, *args, C.byref(paged_params()), None)
    refused(capi.ERR_UNSUPPORTED, lib.axhip_sdpa_paged, X, X, C.byref(changed(paged_params(), dict(pages__head_dim=264))), None)
    capi.check(lib.axhip_sdpa_paged(None, None, C.byref(changed(paged_params(), dict(n_seqs=0))), None))


@pytest.mark.parametrize("params,change", [
    (rope_params, dict(y_strides=(32, 64))), (append_params, dict(q_out_strides=(63, 256))), (append_params, dict(pages__k_strides=(2048, 128, 0))), (append_params, dict(pages__v_strides=(2048, 63, 64))),
    (append_params, dict(pages__k_strides=(0, 128, 64))), (copy_params, dict(pages__k_strides=(32, 128, 64))), (copy_params, dict(pages__v_strides=(2048, 0, 64))), (copy_params, dict(k_layer_stride=0)),
    (packed_params, dict(o_strides=(256, 32))), (packed_params, dict(o_strides=(0, 64))), (paged_params, dict(o_strides=(0, 256, 64))), (paged_params, dict(o_strides=(256, 256, 63))),
    (paged_params, dict(new_tokens=2, o_strides=(512, 32, 64)))])
def test_written_rows_that_overlap(params, change):
    lib = capi.lib()
    call = {rope_params: lambda p: lib.axhip_rope(X, 2 * X, p, None), append_params: lambda p: lib.axhip_kv_append(X, X, X, 2 * X, p, None), copy_params: lambda p: lib.axhip_kv_copy_pages(p, None),
            packed_params: lambda p: lib.axhip_sdpa_packed(X, X, X, X, p, None), paged_params: lambda p: lib.axhip_sdpa_paged(X, X, p, None)}[params]
    assert "overlap" in refused(capi.ERR_INVALID_ARG, call, C.byref(changed(params(), change)))


@pytest.mark.gpu
def test_more_than_a_launch_takes():
    """(nothing is launched)"""
    lib = capi.lib()
    for tokens in (1 << 33, 1 << 61):
        refused(capi.ERR_UNSUPPORTED, lib.axhip_rope, X, 2 * X, C.byref(changed(rope_params(), dict(tokens=tokens))), None)
        refused(capi.ERR_UNSUPPORTED, lib.axhip_kv_append, X, X, X, 2 * X, C.byref(changed(append_params(), dict(tokens=tokens))), None)
    refused(capi.ERR_UNSUPPORTED, lib.axhip_kv_copy_pages, C.byref(changed(copy_params(), dict(pairs=(1 << 31) - 1, layers=1 << 19))), None)
