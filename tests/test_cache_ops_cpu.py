"""CPU: what ops.window_attention / paged_kv_write / paged_decode_attention / kv_evict refuse, in the wrappers and at the C entries."""
import ctypes as C

import pytest
import torch

from valle_amd import _lib, ops


def _window(**kw):
    a = dict(q=torch.zeros(6, 4, 16), k=torch.zeros(6, 2, 16), v=torch.zeros(6, 2, 16), seq_off=torch.tensor([0, 6], dtype=torch.int32))
    a.update(kw)
    return ops.window_attention(**a)


def _cache(**kw):
    a = dict(k_pages=torch.zeros(3, 2, 8, 16), v_pages=torch.zeros(3, 2, 8, 16), page_table=torch.zeros(2, 2, dtype=torch.int32))
    a.update(kw)
    return a


I32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731


@pytest.mark.parametrize("kw,err", [
    (dict(q=torch.zeros(6, 64)), ValueError),
    (dict(k=torch.zeros(6, 3, 16), v=torch.zeros(6, 3, 16)), ValueError),
    (dict(k=torch.zeros(5, 2, 16), v=torch.zeros(5, 2, 16)), ValueError),
    (dict(v=torch.zeros(6, 2, 8)), ValueError),
    (dict(k=torch.zeros(6, 2, 16, dtype=torch.bfloat16)), TypeError),
    (dict(q=torch.zeros(6, 4, 16, dtype=torch.float16)), TypeError),
    (dict(seq_off=torch.tensor([0, 6])), TypeError),
    (dict(seq_off=torch.zeros(0, dtype=torch.int32)), ValueError),
    (dict(text_len=I32(1, 2)), ValueError),
    (dict(out=torch.zeros(6, 4, 8)), ValueError),
    (dict(out=torch.zeros(4, 6, 16).transpose(0, 1)), ValueError),
    (dict(q=torch.zeros(6, 4, 16, requires_grad=True)), RuntimeError),
    (dict(window=-1), ValueError),
    (dict(window=2 ** 32 + 5), ValueError),  # would arrive as 5 in 32 bits
    (dict(sinks=2 ** 31), ValueError),
    (dict(), AssertionError),  # no CPU path
])
def test_window_attention_refuses(kw, err):
    with pytest.raises(err):
        _window(**kw)


@pytest.mark.parametrize("kw,err", [
    (dict(k_pages=torch.zeros(3, 2, 8, 8)), ValueError),
    (dict(k_pages=torch.zeros(3, 8, 2, 16).transpose(1, 2)), ValueError),
    (dict(page_table=torch.zeros(2, 2)), TypeError),
    (dict(page_table=torch.zeros(4, dtype=torch.int32)), ValueError),
    (dict(page_table=torch.zeros(2, 4, dtype=torch.int32)[:, ::2]), ValueError),
    (dict(mass=torch.zeros(3, 2, 8, dtype=torch.float64)), TypeError),
    (dict(mass=torch.zeros(3, 2, 16)), ValueError),
    (dict(), AssertionError),
])
def test_every_cache_operator_refuses_a_bad_pool(kw, err):
    c = _cache(**kw)
    mass = c.pop("mass", torch.zeros(3, 2, 8))
    with pytest.raises(err):
        ops.paged_kv_write(torch.zeros(2, 2, 16), torch.zeros(2, 2, 16), start=I32(0, 0), mass=mass, **c)
    with pytest.raises(err):
        ops.paged_decode_attention(torch.zeros(2, 4, 16), lengths=I32(1, 1), mass=mass, **c)
    with pytest.raises(err):
        ops.kv_evict(mass=mass, lengths=I32(1, 1), budget=4, **c)


def test_cache_operators_refuse_bad_rows():
    c = _cache()
    kv = torch.zeros(2, 2, 16)
    with pytest.raises(ValueError):  # two sequences, three rows, no offsets
        ops.paged_kv_write(torch.zeros(3, 2, 16), torch.zeros(3, 2, 16), start=I32(0, 0), **c)
    with pytest.raises(ValueError):
        ops.paged_kv_write(torch.zeros(2, 1, 16), torch.zeros(2, 1, 16), start=I32(0, 0), **c)
    with pytest.raises(TypeError):
        ops.paged_kv_write(kv, kv, start=torch.tensor([0, 0]), **c)
    with pytest.raises(ValueError):
        ops.paged_kv_write(kv, kv, start=I32(0, 0), **dict(c, v_pages=c["k_pages"]))
    with pytest.raises(TypeError):
        ops.paged_kv_write(kv.bfloat16(), kv.bfloat16(), start=I32(0, 0), **c)
    with pytest.raises(ValueError):
        ops.paged_decode_attention(torch.zeros(3, 4, 16), lengths=I32(1, 1), **c)
    with pytest.raises(ValueError):
        ops.paged_decode_attention(torch.zeros(2, 3, 16), lengths=I32(1, 1), **c)
    with pytest.raises(ValueError):
        ops.paged_decode_attention(torch.zeros(2, 4, 16), lengths=I32(1), **c)
    with pytest.raises(RuntimeError):
        ops.paged_decode_attention(torch.zeros(2, 4, 16, requires_grad=True), lengths=I32(1, 1), **c)
    mass = torch.zeros(3, 2, 8)
    with pytest.raises(ValueError):
        ops.kv_evict(mass=None, lengths=I32(1, 1), budget=4, **c)
    for kw in (dict(budget=0), dict(budget=-3), dict(budget=2 ** 32 + 4), dict(budget=4, recent=-1), dict(budget=4, sinks=2 ** 32)):
        with pytest.raises(ValueError):
            ops.kv_evict(mass=mass, lengths=I32(1, 1), **kw, **c)
    with pytest.raises(ValueError):
        ops.paged_decode_attention(torch.zeros(2, 4, 16), lengths=I32(1, 1), window=2 ** 33, **c)
    with pytest.raises(ValueError):
        ops.kv_evict(mass=mass, lengths=I32(1, 1), budget=4, **dict(c, v_pages=c["k_pages"]))


# ---- C entries: refused before anything is launched, so no GPU is needed (the pointers are never followed) -----------------------------
P = C.c_void_p(4096)


def _c_window(dtype=0, q=P, rows=4, B=1, H=4, Hkv=2, dh=16, window=0, sinks=0, scale=0.25, q_row=64, off=P):
    return _lib.load().vle_op_window_attention(None, dtype, q, q_row, 16, P, 32, 16, P, 32, 16, P, off, None, rows, B, H, Hkv, dh, window, sinks, scale, 0)


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(Hkv=3), dict(Hkv=0), dict(dh=12), dict(dh=136), dict(dh=0), dict(window=-1), dict(sinks=-1),
                                dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(rows=-1), dict(B=-1),
                                dict(q=C.c_void_p(4100)), dict(q_row=66), dict(q=None), dict(off=None), dict(H=512, Hkv=1), dict(rows=2**31 - 1)])
def test_c_window_attention_refuses(kw):
    assert _c_window(**kw) == _lib.VLE_EINVAL
    assert b"vle_op_window_attention" in _lib.load().vle_last_error(None)


def _c_decode(dtype=0, k=P, B=2, H=4, Hkv=2, dh=16, n_pages=3, W=2, ps=8, window=0, sinks=0, scale=0.25, ws=None, ws_bytes=0, mass=None):
    return _lib.load().vle_op_paged_decode_attention(None, dtype, P, 64, 16, k, P, P, P, None, mass, ws, ws_bytes, P, B, H, Hkv, dh, n_pages, W, ps, window,
                                                     sinks, scale)


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(H=5), dict(dh=20), dict(n_pages=0), dict(W=0), dict(ps=4), dict(ps=24), dict(W=2**20, ps=1024),
                                dict(B=70000), dict(window=-1), dict(sinks=-2), dict(scale=0.0), dict(k=None), dict(k=C.c_void_p(4104)),
                                dict(mass=P, W=2000), dict(mass=P, W=2000, ws=P, ws_bytes=16), dict(W=4096, B=1), dict(Hkv=2, H=2, ps=2**24, W=1)])
def test_c_paged_decode_refuses(kw):
    assert _c_decode(**kw) == _lib.VLE_EINVAL
    assert b"vle_op_paged_decode_attention" in _lib.load().vle_last_error(None)


def test_c_workspace_query():
    lib = _lib.load()
    assert lib.vle_op_paged_decode_workspace_bytes(1, 1, 16, 16, 64, 8, 16, 0, 0, 0, 0) == 0  # short: one launch, no workspace
    assert lib.vle_op_paged_decode_workspace_bytes(1, 1, 16, 16, 64, 8, 16, 0, 0, 0, 1) == 0  # its scores fit the LDS
    assert lib.vle_op_paged_decode_workspace_bytes(1, 1, 16, 1, 64, 64, 16, 0, 0, 0, 1) >= 16 * 1024 * 4  # every score
    assert lib.vle_op_paged_decode_workspace_bytes(1, 1, 16, 16, 64, 8192, 16, 0, 0, 0, 0) > 0
    # a window bounds the scores kept, whatever the table's width; a text of unknown length does not
    wide, bounded = (lib.vle_op_paged_decode_workspace_bytes(1, 1, 16, 16, 64, 8192, 16, w, 4, 0, 1) for w in (0, 500))
    assert bounded < wide // 50 and lib.vle_op_paged_decode_workspace_bytes(1, 1, 16, 16, 64, 8192, 16, 500, 4, 1, 1) > wide // 2
    assert lib.vle_op_paged_decode_workspace_bytes(1, 1, 16, 16, 60, 8, 16, 0, 0, 0, 0) == _lib.VLE_EINVAL
    assert lib.vle_op_paged_decode_workspace_bytes(1, 0, 16, 16, 64, 8192, 16, 0, 0, 0, 1) == 0  # no sequence at all


def _c_write(dtype=0, rows=2, B=2, Hkv=2, dh=16, n_pages=3, W=2, ps=8, off=None, k=P, row=32):
    return _lib.load().vle_op_paged_kv_write(None, dtype, k, row, 16, P, 32, 16, P, P, None, P, P, off, rows, B, Hkv, dh, n_pages, W, ps)


@pytest.mark.parametrize("kw", [dict(dtype=5), dict(rows=3), dict(rows=-1, off=P), dict(dh=4), dict(Hkv=0), dict(n_pages=0), dict(ps=6), dict(k=None),
                                dict(k=C.c_void_p(4098)), dict(row=30)])
def test_c_paged_write_refuses(kw):
    assert _c_write(**kw) == _lib.VLE_EINVAL


def _c_evict(budget=8, recent=2, sinks=2, v=C.c_void_p(8192), mass=P, B=2, ps=8):
    return _lib.load().vle_op_kv_evict(None, 0, P, v, mass, P, P, None, P, P, B, 2, 16, 3, 2, ps, budget, recent, sinks)


@pytest.mark.parametrize("kw", [dict(budget=0), dict(budget=3), dict(recent=-1), dict(sinks=-1), dict(recent=7), dict(v=P), dict(mass=None), dict(ps=12),
                                dict(budget=2**26)])
def test_c_evict_refuses(kw):
    assert _c_evict(**kw) == _lib.VLE_EINVAL


def test_nothing_to_do_is_no_error():
    assert _c_window(rows=0) == 0 and _c_decode(B=0) == 0 and _c_write(B=0, rows=0) == 0 and _c_evict(B=0) == 0


@pytest.mark.parametrize("scale", [2.5e38, 3.0e38])
def test_c_scale_whose_base_2_form_overflows_is_refused(scale):
    # scale * log2(e) would be infinite, and 0 * inf not a number, where the softmax of equal scores is their mean
    assert _c_window(scale=scale) == _lib.VLE_EINVAL
    assert _c_decode(scale=scale) == _lib.VLE_EINVAL and b"scale" in _lib.load().vle_last_error(None)
