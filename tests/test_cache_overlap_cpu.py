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
