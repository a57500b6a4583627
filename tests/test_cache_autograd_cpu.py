"""CPU: what the cache operators owe autograd, though they have no backward pass: gradients and tangents that would be lost are refused, tensors written in place
count as written.  (Refusals come before anything else; for the rest the C entries are left out.)"""
import pytest
import torch
from torch.autograd import forward_ad

from valle_amd import ops

I32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731


def operands():
    return dict(q=torch.zeros(2, 4, 16), k=torch.zeros(2, 2, 16), v=torch.zeros(2, 2, 16), k_pages=torch.zeros(3, 2, 8, 16), v_pages=torch.zeros(3, 2, 8, 16), mass=torch.zeros(3, 2, 8),
                out=torch.zeros(2, 4, 16))


def calls(t):
    table, n = torch.zeros(2, 2, dtype=torch.int32), I32(1, 1)
    return {
        "window": (lambda: ops.window_attention(t["q"], t["k"], t["v"], I32(0, 2), out=t["out"]), ("q", "k", "v", "out")),
        "write": (lambda: ops.paged_kv_write(t["k"], t["v"], t["k_pages"], t["v_pages"], table, n, mass=t["mass"]), ("k", "v", "k_pages", "v_pages", "mass")),
        "decode": (lambda: ops.paged_decode_attention(t["q"], t["k_pages"], t["v_pages"], table, n, mass=t["mass"], out=t["out"]), ("q", "k_pages", "v_pages", "mass", "out")),
        "evict": (lambda: ops.kv_evict(t["k_pages"], t["v_pages"], t["mass"], table, n, 4), ("k_pages", "v_pages", "mass")),
    }


EACH = [(op, name) for op, (_, names) in calls(operands()).items() for name in names]


@pytest.mark.parametrize("op,name", EACH)
def test_tensors_that_ask_for_a_gradient_are_refused(op, name, monkeypatch):
    t = operands()
    t[name].requires_grad_()
    call = calls(t)[op][0]
    with pytest.raises(RuntimeError, match="backward"):
        call()
    monkeypatch.setattr(ops, "_call", lambda *a: None)
    with torch.no_grad():
        call()


@pytest.mark.parametrize("op,name", EACH)
def test_tensors_with_a_tangent_are_refused(op, name, monkeypatch):
    t = operands()
    with forward_ad.dual_level():
        t[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
        call = calls(t)[op][0]
        with pytest.raises(RuntimeError, match="tangent"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):  # no_grad does not turn the forward mode off
            call()
        monkeypatch.setattr(ops, "_call", lambda *a: None)
        t[name] = forward_ad.unpack_dual(t[name]).primal
        call()


@pytest.mark.parametrize("op,written", [("window", {"out"}), ("write", {"k_pages", "v_pages", "mass"}), ("decode", {"mass", "out"}), ("evict", {"k_pages", "v_pages", "mass"})])
def test_tensors_written_in_place_count_as_written(op, written, monkeypatch):
    """Saved for a backward pass and overwritten by one of these operators, a tensor has to be found out."""
    monkeypatch.setattr(ops, "_call", lambda *a: None)
    t = operands()
    was = {n: x._version for n, x in t.items()}
    call, names = calls(t)[op]
    call()
    for n in names:
        assert (t[n]._version > was[n]) == (n in written), n
    x = torch.ones(3, requires_grad=True)
    for n in written:
        y = (x.sum() * t[n]).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        t = operands()
        calls(t)[op][0]()
    calls(t)[op][0]()  # tensors of inference mode, which count nothing


def test_optional_tensors_may_be_missing(monkeypatch):
    monkeypatch.setattr(ops, "_call", lambda *a: None)
    t = dict(operands(), mass=None, out=None)
    for op in ("window", "write", "decode"):
        calls(t)[op][0]()
