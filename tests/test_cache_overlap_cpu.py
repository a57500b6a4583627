"""CPU: the C entries of the cache operators refuse, before anything is launched, memory that a call would write while it is read or written as something else
(the pointers are never followed)."""
import ctypes as C

import pytest

from valle_amd import _lib

A = lambda i: C.c_void_p(i << 24)  # noqa: E731  (places 16 MB apart: nothing below is as large)
AT = lambda i, off: C.c_void_p((i << 24) + off)  # noqa: E731


def refused(rc, op):
    msg = _lib.load().vle_last_error(None)
    return rc == _lib.VLE_EINVAL and op in msg and b"overlap" in msg


def evict(k=A(1), v=A(2), mass=A(3), table=A(4), lengths=A(5), text=A(6), kept=A(7), left=A(8)):
    # 2 sequences, 2 heads of 16 (fp32), 3 pages of 8, a table of 2, a budget of 8: pools of 3072 bytes, weights 192, kept 128, tables 16, lengths 8
    return _lib.load().vle_op_kv_evict(None, 0, k, v, mass, table, lengths, text, kept, left, 2, 2, 16, 3, 2, 8, 8, 2, 2)


@pytest.mark.parametrize("kw", [dict(left=A(5)), dict(left=AT(5, 4)), dict(lengths=AT(8, 4))], ids=["same", "behind", "ahead"])
def test_evict_refuses_new_lengths_over_the_lengths(kw):
    """The lengths are read to the call's end: an eviction whose lengths change under it moves nothing and reports that it did."""
    assert refused(evict(**kw), b"vle_op_kv_evict")


@pytest.mark.parametrize("kw", [dict(kept=A(4)), dict(kept=AT(5, 0)), dict(kept=AT(6, 4)), dict(left=A(4)), dict(left=AT(6, 4)), dict(left=AT(7, 124)), dict(kept=AT(3, 188)),
                                dict(left=AT(1, 3068)), dict(kept=AT(2, 16)), dict(mass=AT(1, 3056)), dict(mass=AT(2, 0)), dict(table=AT(3, 64)), dict(lengths=AT(1, 64)),
                                dict(text=AT(2, 64)), dict(v=AT(1, 1024)), dict(k=AT(2, 3056))])
def test_evict_refuses_other_overlaps(kw):
    assert refused(evict(**kw), b"vle_op_kv_evict")


def window(q=A(1), k=A(2), v=A(3), out=A(4), off=A(5), text=A(6), q_row=64, kv_row=32, q_head=16, kv_head=16):
    # 4 rows, 4 heads on 2 of 16 (fp32): q and out 1024 bytes, k and v 512
    return _lib.load().vle_op_window_attention(None, 0, q, q_row, q_head, k, kv_row, kv_head, v, kv_row, kv_head, out, off, text, 4, 1, 4, 2, 16, 0, 0, 0.25, 0)


@pytest.mark.parametrize("kw", [dict(out=A(1)), dict(out=AT(1, 1008)), dict(q=AT(4, 1008)), dict(out=A(2)), dict(out=AT(2, 496)), dict(k=AT(4, 1008)), dict(out=AT(3, 496)), dict(v=AT(4, 512)),
                                dict(off=AT(4, 1020)), dict(text=AT(4, 0)), dict(q=AT(4, -1280), q_row=256),  # a strided view that reaches into out with its last row
                                dict(k=AT(4, -48), kv_row=0, kv_head=0)])                                     # one row for all
def test_window_attention_refuses_overlaps(kw):
    assert refused(window(**kw), b"vle_op_window_attention")


def decode(q=A(1), k=A(2), v=A(3), table=A(4), lengths=A(5), text=A(6), mass=A(7), ws=A(8), out=A(9), W=2000):
    # 2 sequences, 4 heads on 2 of 16 (fp32), 3 pages of 8: q and out 512 bytes, pools 3072, weights 192
    need = _lib.load().vle_op_paged_decode_workspace_bytes(0, 2, 4, 2, 16, W, 8, 0, 0, 1, 1)
    assert 0 < need < 1 << 24
    return _lib.load().vle_op_paged_decode_attention(None, 0, q, 64, 16, k, v, table, lengths, text, mass, ws, need, out, 2, 4, 2, 16, 3, W, 8, 0, 0, 0.25)


@pytest.mark.parametrize("kw", [dict(out=A(1)), dict(out=AT(1, 496)), dict(q=AT(9, 496)), dict(out=AT(2, 3056)), dict(out=AT(3, 0)), dict(out=AT(4, 15984)), dict(out=A(5)), dict(text=AT(9, 508)),
                                dict(out=AT(7, 176)), dict(mass=AT(2, 16)), dict(mass=AT(3, 3068)), dict(mass=AT(1, 508)), dict(mass=A(4)), dict(mass=AT(5, 4)), dict(ws=A(9)), dict(ws=A(7)),
                                dict(ws=AT(3, 3056)), dict(ws=A(1)), dict(lengths=AT(8, 64))])
def test_decode_refuses_overlaps(kw):
    assert refused(decode(**kw), b"vle_op_paged_decode_attention")


def write(k=A(1), v=A(2), kp=A(3), vp=A(4), mass=A(5), table=A(6), start=A(7), off=A(8)):
    return _lib.load().vle_op_paged_kv_write(None, 0, k, 32, 16, v, 32, 16, kp, vp, mass, table, start, off, 5, 2, 2, 16, 3, 2, 8)


@pytest.mark.parametrize("kw", [dict(vp=A(3)), dict(vp=AT(3, 1024)), dict(kp=AT(4, 3056)), dict(mass=AT(3, 0)), dict(mass=AT(4, 3068)), dict(mass=AT(6, 12)), dict(start=AT(5, 188)), dict(off=AT(3, 4)),
                                dict(table=AT(4, 64)), dict(mass=A(1)), dict(mass=AT(2, 4))])
def test_write_refuses_overlaps(kw):
    """(k and v may be views of the pools: what a row is read from is the caller's to keep apart from where rows are written.)"""
    assert refused(write(**kw), b"vle_op_paged_kv_write")


def test_shared_inputs_are_no_overlap():
    """Operands that are only read may be one: the call goes on to its launch, which has no device here."""
    import torch

    if torch.cuda.is_available():
        pytest.skip("would launch")
    for rc in (window(q=A(1), k=A(1), v=A(1)), window(k=A(2), v=A(2)), decode(v=A(2)), write(k=AT(3, 512), v=AT(3, 512)), decode(text=A(5)), evict(text=A(5)), write(start=A(8)),
               window(out=AT(1, 1024)), window(q=AT(4, 1024)), evict(left=AT(5, 8)), evict(kept=AT(8, 8))):
        assert not (rc == _lib.VLE_EINVAL and b"overlap" in _lib.load().vle_last_error(None)) and rc == _lib.VLE_EHIP
