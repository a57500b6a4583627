"""CPU: each bound of the cache operators' C entries by its own message, so that no other refusal stands in for it; one below the bound goes past that check."""
import ctypes as C

import pytest

from valle_amd import _lib

P = [C.c_void_p(i << 40) for i in range(1, 11)]  # far apart, never followed


def message(rc):
    assert rc == _lib.VLE_EINVAL
    return _lib.load().vle_last_error(None).decode()


def sizes(**kw):
    return dict(dict(dtype=0, B=2, H=4, Hkv=2, dh=16, n_pages=3, W=2, ps=8), **kw)


def decode(**kw):
    s = sizes(**kw)
    return _lib.load().vle_op_paged_decode_attention(None, s["dtype"], P[0], 64, 16, P[1], P[2], P[3], P[4], None, None, None, 0, P[5], s["B"], s["H"], s["Hkv"], s["dh"], s["n_pages"], s["W"],
                                                     s["ps"], 0, 0, 0.25)


def room(**kw):
    s = sizes(**kw)
    return _lib.load().vle_op_paged_decode_workspace_bytes(s["dtype"], s["B"], s["H"], s["Hkv"], s["dh"], s["W"], s["ps"], 0, 0, 0, 0)


def write(**kw):
    s = sizes(**kw)
    return _lib.load().vle_op_paged_kv_write(None, s["dtype"], P[0], 32, 16, P[1], 32, 16, P[2], P[3], None, P[4], P[5], P[6], s.get("rows", 2), s["B"], s["Hkv"], s["dh"], s["n_pages"], s["W"], s["ps"])


def evict(**kw):
    s = sizes(**kw)
    return _lib.load().vle_op_kv_evict(None, s["dtype"], P[0], P[1], P[2], P[3], P[4], None, P[5], P[6], s["B"], s["Hkv"], s["dh"], s["n_pages"], s["W"], s["ps"], s.get("budget", 8), s.get("recent", 2),
                                       s.get("sinks", 2))


CACHE = [("a page holds fewer than 2^30 elements", dict(H=64, Hkv=64, ps=2 ** 20, W=1)), ("a page holds fewer than 2^30 elements", dict(H=4096, Hkv=4096, dh=128, ps=2048, W=1)),
         ("a sequence holds fewer than 2^30 keys", dict(W=2 ** 20, ps=1024)), ("a sequence holds fewer than 2^30 keys", dict(W=2 ** 27, ps=8)), ("page size must be a power of two", dict(ps=24)),
         ("page size must be a power of two", dict(ps=4)), ("0 to 65535 sequences", dict(B=65536)), ("0 to 65535 sequences", dict(B=-1)), ("no pages", dict(W=0)),
         ("at most 4096 key-value heads", dict(H=4097, Hkv=4097)), ("head size must be a multiple of 8", dict(dh=12)), ("head size must be a multiple of 8", dict(dh=136)), ("dtype must be", dict(dtype=2))]


@pytest.mark.parametrize("text,kw", CACHE)
def test_every_entry_refuses_sizes_of_the_cache(text, kw):
    for entry in (decode, room, write, evict):
        assert text in message(entry(**kw)), entry.__name__


@pytest.mark.parametrize("text,kw", [("no pages", dict(n_pages=0))])
def test_entries_with_a_pool_refuse_an_empty_one(text, kw):
    for entry in (decode, write, evict):
        assert text in message(entry(**kw)), entry.__name__


def test_the_largest_sizes_pass_the_checks():
    """One step inside each bound the workspace is told, not an error."""
    for kw in (dict(H=64, Hkv=64, ps=2 ** 19, W=1), dict(W=2 ** 20, ps=512), dict(B=65535), dict(H=4096, Hkv=4096), dict(dh=128), dict(dh=8), dict(H=512)):
        assert room(**kw) >= 0, kw


@pytest.mark.parametrize("entry,text,kw", [
    (decode, "at most 256 query heads", dict(H=514)), (decode, "nhead must be a multiple", dict(H=5)), (decode, "workspace too small", dict(W=4096, B=1)), (write, "0 to 2^25 rows", dict(rows=2 ** 25 + 1)),
    (write, "0 to 2^25 rows", dict(rows=-1)), (evict, "budget must be 1 to 2^25", dict(budget=0)), (evict, "budget must be 1 to 2^25", dict(budget=2 ** 25 + 1)),
    (evict, "must fit the budget", dict(recent=7)), (evict, "must fit the budget", dict(sinks=-1)), (evict, "must fit the budget", dict(recent=-1))])
def test_refusals_of_one_entry(entry, text, kw):
    assert text in message(entry(**kw))
