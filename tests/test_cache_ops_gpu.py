"""GPU: ops.window_attention, paged_kv_write, paged_decode_attention and kv_evict against plain 64-bit implementations.

Tolerances, per output element, from the operand values (u = half a step of the type relative to the value, finfo.eps / 2):
* a score is a sum of dh products in fp32: off by at most (dh + 2) 2^-24 sum |q k| scale, twice that for the difference to the maximum; with the
  rounding of the exponential's argument and value that makes each weight off by a relative  delta = 2 (dh + 4) 2^-24 max(sum |q k|) scale + 2^-20;
* the weighted sum over n keys in fp32 adds n 2^-24;  numerator and denominator: 2 (delta + n 2^-24) sum p |v|;
* window_attention in bf16 rounds each weight to bf16 in numerator and denominator alike: 2 u sum p |v| more; paged_decode_attention keeps 16 bits of them;
* the result is rounded once: u |out|."""
import math

import pytest
import torch

from valle_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def rnd(g, *shape, dtype=torch.float32, gain=1.0):
    return (torch.randn(shape, generator=g, dtype=torch.float32) * gain).to(dtype)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def sees(n, i, text, window, sinks):
    j = torch.arange(n)
    m = j <= i
    if window:
        m &= (i - j < window) | (j < sinks)
    return m | (j < text)


def attend(q, k, v, see, scale, weight_ulp=0.0):
    """One query (dh,) in 64 bits over the keys that `see` allows: (out, bound on |got - out|, weights)."""
    k, v, q = k[see].to(F64), v[see].to(F64), q.to(F64)
    s = (k @ q) * scale
    p = torch.softmax(s, 0)
    o = p @ v
    u = weight_ulp
    spread = float((k.abs() @ q.abs()).max()) * scale
    delta = 2 * (q.numel() + 4) * 2.0 ** -24 * spread + 2.0 ** -20
    return o, (2 * (delta + len(p) * 2.0 ** -24) + 2 * u) * (p @ v.abs()), p, delta


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def near(got, want, bound, what=""):
    off = (got.detach().cpu().to(F64) - want).abs()
    assert bool((off <= bound).all()), f"{what}: off by {float((off - bound).max()):.3g} more than allowed, at {int((off - bound).argmax())}"


# ---- window_attention -------------------------------------------------------------------------------------------------------------
def window_ref(q, k, v, off, text, window, sinks, scale=None):
    rows, H, dh = q.shape
    G = H // k.shape[1]
    scale = 1 / math.sqrt(dh) if scale is None else scale
    u = half_step(q.dtype)
    out, tol = torch.zeros(rows, H, dh, dtype=F64), torch.zeros(rows, H, dh, dtype=F64)
    wu = u if q.dtype == torch.bfloat16 else 0.0
    for b in range(len(off) - 1):
        n = off[b + 1] - off[b]
        r = slice(off[b], off[b + 1])
        for i in range(n):
            m = sees(n, i, min(text[b], n), window, sinks)
            for h in range(H):
                o, t, _, _ = attend(q[off[b] + i, h], k[r, h // G], v[r, h // G], m, scale, wu)
                out[off[b] + i, h], tol[off[b] + i, h] = o, t + u * o.abs()
    return out, tol


def offsets(lens):
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    return off


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,text,H,Hkv,dh,window,sinks", [
    ([1], [0], 1, 1, 64, 0, 0),
    ([1, 0, 2, 65, 0], [1, 0, 0, 7, 0], 4, 2, 64, 16, 2),
    ([130, 63, 64], [0, 63, 20], 2, 1, 128, 33, 4),
    ([200, 129], [0, 0], 2, 2, 96, 0, 0),          # no window: plain causal
    ([150], [90], 3, 1, 40, 5, 0),                 # text past the window, head size inside a wider tile
    ([190], [0], 2, 2, 32, 1, 0),                  # a row sees itself alone
    ([260], [0], 2, 1, 8, 64, 70),                 # sinks past the first tile
    ([257], [300], 1, 1, 120, 7, 3),               # text longer than the sequence: every row sees all
    ([100, 100], [100, 0], 2, 2, 64, 1000, 1000),  # window and sinks past the sequence
])
def test_window_attention(dtype, lens, text, H, Hkv, dh, window, sinks):
    g, off = gen(sum(lens) + dh), offsets(lens)
    q, k, v = rnd(g, off[-1], H, dh, dtype=dtype, gain=1.5), rnd(g, off[-1], Hkv, dh, dtype=dtype), rnd(g, off[-1], Hkv, dh, dtype=dtype)
    got = ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(off), window=window, sinks=sinks, text_len=i32(text))
    near(got, *window_ref(q, k, v, off, text, window, sinks), "window")


@pytest.mark.parametrize("B", [65, 300])
def test_window_attention_and_write_of_many_short_sequences(B):
    """More sequences than a wave has lanes, empty ones among them: attention of their prompts, the write of their keys, a step over the cache."""
    g, H, dh, ps = gen(B), 2, 32, 8
    lens = torch.randint(0, 9, (B,), generator=g).tolist()
    off, text = offsets(lens), [min(2, n) for n in lens]
    q, k, v = (rnd(g, off[-1], H, dh, dtype=torch.bfloat16) for _ in range(3))
    got = ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(off), window=3, sinks=1, text_len=i32(text))
    near(got, *window_ref(q, k, v, off, text, 3, 1), "window")
    pool = Pool(g, lens, H, dh, ps, torch.bfloat16)
    kp, vp, table, mass = pool.device()
    kp.fill_(float("nan")), vp.fill_(float("nan"))
    ops.paged_kv_write(k.to(DEV), v.to(DEV), kp, vp, table, i32([0] * B), seq_off=i32(off), mass=mass)
    for b in range(B):
        page, slot = pool.at(b)
        pool.k[page, :, slot], pool.v[page, :, slot], pool.mass[page, :, slot] = k[off[b]:off[b + 1]], v[off[b]:off[b + 1]], 0.0
    same = lambda a, w: bool(((a.cpu() == w) | (a.cpu().isnan() & w.isnan())).all())  # noqa: E731
    assert same(kp, pool.k) and same(vp, pool.v) and same(mass, pool.mass)
    one = rnd(g, B, H, dh, dtype=torch.bfloat16)
    out, tol, add, add_tol = decode_ref(pool, one, text, 3, 1)
    near(ops.paged_decode_attention(one.to(DEV), kp, vp, table, i32(lens), window=3, sinks=1, text_len=i32(text), mass=mass), out, tol, "step")
    near(mass, pool.mass.to(F64) + add, add_tol + 2.0 ** -22, "mass")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_window_attention_views_and_rows_of_no_sequence(dtype):
    """q / k / v as slices of one packed qkv, keys and values of one head broadcast over all, operands off the 16-byte grid; sequences that start behind row 0 and end
    ahead of the last one: those rows are 0, or as they were in a given output."""
    g, H, dh, rows, lens = gen(3), 4, 32, 150, [40, 30]
    off = [11, 51, 81]
    qkv = rnd(g, rows, 3 * H * dh, dtype=dtype).to(DEV)
    q, k, v = (x.view(rows, H, dh) for x in qkv.split(H * dh, 1))
    shift = lambda o, t: (torch.cat([torch.zeros(o, H, dh, dtype=F64), t, torch.zeros(rows - o - len(t), H, dh, dtype=F64)]))  # noqa: E731
    cut = slice(off[0], off[-1])
    want, tol = (shift(off[0], t) for t in window_ref(q[cut].cpu(), k[cut].cpu(), v[cut].cpu(), offsets(lens), [0, 0], 9, 2, 0.3))
    got = ops.window_attention(q, k, v, i32(off), window=9, sinks=2, scale=0.3)
    near(got, want, tol, "views")
    out = torch.full((rows, H, dh), 7.0, dtype=dtype, device=DEV)
    assert ops.window_attention(q, k, v, i32(off), window=9, sinks=2, scale=0.3, out=out) is out
    assert torch.equal(out[cut], got[cut]) and bool((out[: off[0]] == 7).all()) and bool((out[off[-1]:] == 7).all())
    one = k[:, :1].expand(rows, H, dh)  # head stride 0
    assert torch.equal(ops.window_attention(q, one, one, i32(off), window=9), ops.window_attention(q, k[:, :1], k[:, :1], i32(off), window=9))
    odd = torch.zeros(rows * H * dh + 1, dtype=dtype, device=DEV)[1:].view(rows, H, dh)
    odd.copy_(q)
    assert torch.equal(ops.window_attention(odd, k, v, i32(off), window=9), ops.window_attention(q, k, v, i32(off), window=9))
    none = ops.window_attention(q, k, v, i32([0]), window=9)
    assert none.shape == q.shape and bool((none == 0).all())
    assert ops.window_attention(q[:0], k[:0], v[:0], i32([0, 0])).shape == (0, H, dh)
    bad = ops.window_attention(q, k, v, i32([-5, 40, 20, 10 ** 9]), window=9)  # offsets past the rows are clamped
    assert torch.equal(bad[:20], ops.window_attention(q, k, v, i32([0, 40]), window=9)[:20])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_window_attention_rows_do_not_feel_keys_they_do_not_see(dtype, bad):
    g, n, H, dh, window = gen(5), 150, 2, 64, 20
    q, k, v = rnd(g, n, H, dh, dtype=dtype), rnd(g, n, H, dh, dtype=dtype), rnd(g, n, H, dh, dtype=dtype)
    clean = ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32([0, n]), window=window, sinks=1)
    at = 70
    v[at] = bad
    got = ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32([0, n]), window=window, sinks=1)
    want, tol = window_ref(q, torch.where(torch.isfinite(k), k, 0), torch.where(torch.isfinite(v), v, 0), [0, n], [0], window, 1)
    unseen = [i for i in range(n) if not sees(n, i, 0, window, 1)[at]]
    seen = [i for i in range(n) if i not in unseen]
    near(got[unseen], want[unseen], tol[unseen], "unseen values")
    assert not bool(torch.isfinite(got[seen]).any())
    k[at], v[at] = float("nan"), 0.5
    got = ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32([0, n]), window=window, sinks=1)
    assert bool(torch.isnan(got[seen]).all()) and bool(torch.isfinite(got[unseen]).all())
    near(got[:at], clean[:at].cpu().to(F64), 2 * tol[:at], "unseen keys")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_window_attention_largest_values(dtype):
    """Values whose unnormalised sums pass the largest number still average to themselves; scores of any size."""
    n, dh = 100, 64
    big = torch.full((n, 1, dh), 2.0 ** 127, dtype=dtype)
    z = torch.zeros(n, 1, dh, dtype=dtype)
    got = ops.window_attention(z.to(DEV), z.to(DEV), big.to(DEV), i32([0, n]))
    assert bool(((got.float() / 2.0 ** 127 - 1).abs() <= 2 ** -7).all())
    q = torch.full((n, 1, dh), 2.0 ** 40, dtype=dtype)
    k = torch.zeros(n, 1, dh, dtype=dtype)
    k[:, 0, 0] = torch.arange(n)  # each row's own key wins by far
    v = rnd(gen(1), n, 1, dh, dtype=dtype)
    assert torch.equal(ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32([0, n])).cpu(), v)
    assert torch.equal(ops.window_attention(-q.to(DEV), k.to(DEV), v.to(DEV), i32([0, n])).cpu()[1:], v[:1].expand(n - 1, 1, dh))


@pytest.mark.parametrize("dtype,rows,H,Hkv,dh,window,sinks,text", [
    (torch.bfloat16, 4200, 32, 8, 64, 700, 4, 0), (torch.bfloat16, 4111, 32, 4, 128, 0, 0, 100), (torch.float32, 2111, 8, 2, 96, 500, 0, 33)])
def test_window_attention_long(dtype, rows, H, Hkv, dh, window, sinks, text):
    """Enough work that a wide launch takes it; single heads and every 97th row against 64 bits on the device."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    q, k, v = (torch.randn(rows, h, dh, generator=g, device=DEV).to(dtype) for h in (H, Hkv, Hkv))
    got = ops.window_attention(q, k, v, i32([0, rows]), window=window, sinks=sinks, text_len=i32([text]))
    i, j = torch.arange(0, rows, 97, device=DEV)[:, None], torch.arange(rows, device=DEV)[None]
    m = j <= i
    if window:
        m = m & ((i - j < window) | (j < sinks))
    m = m | (j < text)
    u = half_step(dtype)
    for h in (0, H // 2, H - 1):
        kh, vh = k[:, h // (H // Hkv)].double(), v[:, h // (H // Hkv)].double()
        s = (q[::97, h].double() @ kh.T) / math.sqrt(dh)
        spread = float((q[::97, h].double().abs() @ kh.abs().T).max()) / math.sqrt(dh)
        p = torch.softmax(s.masked_fill(~m, -math.inf), 1)
        want = p @ vh
        delta = 2 * (dh + 4) * 2.0 ** -24 * spread + 2.0 ** -20
        tol = (2 * (delta + rows * 2.0 ** -24) + (2 * u if dtype == torch.bfloat16 else 0)) * (p @ vh.abs()) + u * want.abs()
        near(got[::97, h], want.cpu(), tol.cpu(), f"head {h}")


@pytest.mark.parametrize("dh,Hkv,window,sinks", [(128, 4, 33, 2), (120, 32, 150, 0), (104, 1, 0, 0), (96, 4, 70, 3)])
def test_window_attention_many_ragged_sequences_of_large_heads(dh, Hkv, window, sinks):
    """Work enough for the largest items, and sequences that end inside them; rows of no sequence; a key that is not a number reaches only the rows that see it."""
    g, H, dtype = gen(dh), 32, torch.bfloat16
    lens = [0, 1, 15, 16, 17, 127, 128, 129, 0, 200, 255, 256, 257, 63, 64, 65, 300]
    text = [0, 1, 3, 0, 17, 40, 0, 64, 0, 0, 65, 0, 9, 70, 0, 0, 120]
    off = offsets(lens)
    rows = off[-1] + 13
    q, k, v = rnd(g, rows, H, dh, dtype=dtype), rnd(g, rows, Hkv, dh, dtype=dtype), rnd(g, rows, Hkv, dh, dtype=dtype)
    poisoned = {9: 180, 16: 130}  # sequence: key
    for b, j in poisoned.items():
        k[off[b] + j] = float("nan")
    q, k, v = q.to(DEV), k.to(DEV), v.to(DEV)
    got = ops.window_attention(q, k, v, i32(off), window=window, sinks=sinks, text_len=i32(text))
    assert bool((got[off[-1]:] == 0).all())
    u = half_step(dtype)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        r = slice(off[b], off[b + 1])
        m = torch.stack([sees(n, i, min(text[b], n), window, sinks) for i in range(n)]).to(DEV)
        hit = m[:, poisoned[b]] if b in poisoned else torch.zeros(n, dtype=torch.bool, device=DEV)
        assert bool(got[r][hit].isnan().all())
        for h in range(H):
            qh, kh, vh = q[r, h].double(), k[r, h // (H // Hkv)].double().nan_to_num(0.0), v[r, h // (H // Hkv)].double()
            spread = float((qh.abs() @ kh.abs().T).max()) / math.sqrt(dh)
            w = torch.softmax(((qh @ kh.T) / math.sqrt(dh)).masked_fill(~m, -math.inf), 1)
            want, delta = w @ vh, 2 * (dh + 4) * 2.0 ** -24 * spread + 2.0 ** -20
            tol = (2 * (delta + n * 2.0 ** -24) + 2 * u) * (w @ vh.abs()) + u * want.abs()
            near(got[r, h][~hit], want[~hit].cpu(), tol[~hit].cpu(), f"sequence {b} head {h}")


def test_window_attention_offsets_whose_runs_overflow_their_count():
    """Offsets that go back and forth: 2^31 runs of rows and more, of which the launch has work items for a few.  Nothing outside `out` is written, and inside it
    only averages."""
    H, dh, B = 1024, 8, 5800
    rows = 64 * B
    assert (B // 2) * B * (H // 8) > 2 ** 31
    q = torch.zeros(rows, H, dh, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(rows, 4, dh, dtype=torch.bfloat16, device=DEV)
    room = torch.full(((rows + 256) * H * dh,), 7.0, dtype=torch.bfloat16, device=DEV)
    out = room[128 * H * dh: -128 * H * dh].view(rows, H, dh)
    ops.window_attention(q, k, k + 1, i32([0, rows] * (B // 2) + [0]), window=1, out=out)
    torch.cuda.synchronize()
    assert bool((room[: 128 * H * dh] == 7).all()) and bool((room[-128 * H * dh:] == 7).all())
    assert bool(((out == 1) | (out == 7)).all())


def test_window_attention_is_the_prefix_lm_attention_without_a_window():
    """window = 0 and one key-value head per query head: the mask of ops.attention (both bf16: weights and result rounded)."""
    g, H, dh, lens, text = gen(8), 4, 64, [90, 70], [20, 31]
    off = offsets(lens)
    qkv = rnd(g, off[-1], 3 * H * dh, dtype=torch.bfloat16).to(DEV)
    q, k, v = (x.view(off[-1], H, dh) for x in qkv.split(H * dh, 1))
    want, tol = window_ref(q.cpu(), k.cpu(), v.cpu(), off, text, 0, 0)
    near(ops.window_attention(q, k, v, i32(off), text_len=i32(text)), want, tol, "window")
    near(ops.attention(qkv, i32(off), i32(text), H, causal=True).view(-1, H, dh), want, 2 * tol, "attention")


# ---- a page pool and its mirror ---------------------------------------------------------------------------------------------------
class Pool:
    """Random pages for sequences of `lens` keys; what no sequence holds is NaN, as fresh memory may be."""

    def __init__(self, g, lens, Hkv, dh, ps, dtype, spare=2, width=None):
        need = [-(-n // ps) for n in lens]
        total = sum(need) + spare
        order = torch.randperm(total, generator=g).tolist()
        W = width or max(1, max(need, default=1))
        self.lens, self.ps, self.Hkv = lens, ps, Hkv
        self.table = torch.full((len(lens), W), -1, dtype=torch.int32)
        self.k, self.v = (torch.full((total, Hkv, ps, dh), float("nan"), dtype=dtype) for _ in range(2))
        self.mass = torch.rand(total, Hkv, ps, generator=g)
        for b, n in enumerate(need):
            for i in range(n):
                self.table[b, i] = order.pop()
            page, slot = self.at(b)
            self.k[page, :, slot], self.v[page, :, slot] = rnd(g, lens[b], Hkv, dh, dtype=dtype), rnd(g, lens[b], Hkv, dh, dtype=dtype)

    def at(self, b, n=None):
        j = torch.arange(self.lens[b] if n is None else n)
        return self.table[b][j // self.ps].long(), j % self.ps

    def device(self):
        return self.k.to(DEV), self.v.to(DEV), self.table.to(DEV), self.mass.to(DEV)


def decode_ref(pool, q, text, window, sinks, scale=None):
    B, H, dh = q.shape
    G = H // pool.Hkv
    scale = 1 / math.sqrt(dh) if scale is None else scale
    u = half_step(q.dtype)
    wu = 2.0 ** -16 if q.dtype == torch.bfloat16 else 0.0
    out, tol = torch.zeros(B, H, dh, dtype=F64), torch.zeros(B, H, dh, dtype=F64)
    add, add_tol = torch.zeros(pool.mass.shape, dtype=F64), torch.zeros(pool.mass.shape, dtype=F64)
    for b in range(B):
        n = pool.lens[b]
        page, slot = pool.at(b)
        there = (page >= 0) & (page < pool.k.shape[0])
        m = sees(n, n - 1, min(text[b], n), window, sinks) & there
        if not bool(m.any()):
            continue
        for h in range(H):
            kh, vh = (x[page.clamp(0, x.shape[0] - 1), h // G, slot] for x in (pool.k, pool.v))
            o, t, p, delta = attend(q[b, h], kh, vh, m, scale, wu)
            out[b, h], tol[b, h] = o, t + u * o.abs()
            add[page[m], h // G, slot[m]] += p
            add_tol[page[m], h // G, slot[m]] += (2 * delta + n * 2.0 ** -24) * p + 2.0 ** -23
    return out, tol, add, add_tol


# ---- paged_decode_attention ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,text,H,Hkv,dh,ps,window,sinks,width", [
    ([1], [0], 1, 1, 64, 16, 0, 0, None),
    ([0, 1, 31, 32, 33, 100, 0], [0] * 7, 4, 2, 64, 16, 0, 0, None),
    ([70, 200, 5], [10, 0, 5], 6, 2, 128, 8, 33, 2, None),
    ([700, 513], [0, 40], 3, 3, 96, 64, 100, 4, None),
    ([1500, 64], [0, 0], 16, 1, 40, 32, 0, 0, None),     # split and joined
    ([900], [0], 40, 2, 32, 16, 0, 0, 300),              # 20 heads a group, a table wider than the sequence
    ([300, 299], [0, 0], 4, 4, 8, 128, 1, 0, None),      # the newest key alone
    ([300], [299], 2, 2, 120, 256, 1, 0, None),          # text up to the newest key
    ([2100, 90, 1200], [64, 90, 3], 8, 2, 64, 16, 700, 0, None),
])
@pytest.mark.parametrize("with_mass", [False, True], ids=["", "mass"])
def test_paged_decode_attention(dtype, lens, text, H, Hkv, dh, ps, window, sinks, width, with_mass):
    g = gen(sum(lens) + dh + ps)
    pool = Pool(g, lens, Hkv, dh, ps, dtype, width=width)
    q = rnd(g, len(lens), H, dh, dtype=dtype, gain=1.5)
    k, v, table, mass = pool.device()
    got = ops.paged_decode_attention(q.to(DEV), k, v, table, i32(lens), window=window, sinks=sinks, text_len=i32(text), mass=mass if with_mass else None)
    out, tol, add, add_tol = decode_ref(pool, q, text, window, sinks)
    near(got, out, tol, "out")
    if with_mass:
        near(mass, pool.mass.to(F64) + add, add_tol + 2.0 ** -22, "mass")
    else:
        assert torch.equal(mass.cpu(), pool.mass)


def test_paged_decode_attention_views_scale_and_given_output():
    g, lens = gen(2), [37, 80]
    pool = Pool(g, lens, 2, 64, 16, torch.bfloat16)
    k, v, table, _ = pool.device()
    qkv = rnd(g, 2, 3 * 4 * 64, dtype=torch.bfloat16)
    q = qkv[:, 256:512].view(2, 4, 64)
    out = torch.empty(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    assert ops.paged_decode_attention(qkv.to(DEV)[:, 256:512].view(2, 4, 64), k, v, table, i32(lens), scale=0.05, out=out) is out
    want, tol, _, _ = decode_ref(pool, q, [0, 0], 0, 0, 0.05)
    near(out, want, tol)


@pytest.mark.parametrize("ps", [16, 64])
def test_paged_decode_attention_pages_that_are_not_there(ps):
    """Ids outside the pool are not followed, their keys are absent; a length past the table is clamped to it."""
    g, lens = gen(ps), [5 * ps + 3, 4 * ps, ps]
    pool = Pool(g, lens, 2, 64, ps, torch.bfloat16)
    pool.table[0, 1], pool.table[0, 4], pool.table[2, 0] = -7, pool.k.shape[0], 2 ** 31 - 1
    q = rnd(g, 3, 4, 64, dtype=torch.bfloat16)
    k, v, table, mass = pool.device()
    got = ops.paged_decode_attention(q.to(DEV), k, v, table, i32(lens), mass=mass)
    out, tol, add, add_tol = decode_ref(pool, q, [0] * 3, 0, 0)
    near(got, out, tol)
    near(mass, pool.mass.to(F64) + add, add_tol + 2.0 ** -22, "mass")
    assert bool((got[2] == 0).all())
    full = ops.paged_decode_attention(q.to(DEV), k, v, table[1:2].repeat(3, 1)[:, :4].contiguous(), i32([10 ** 9, 4 * ps, -3]))
    assert torch.equal(full[0], ops.paged_decode_attention(q.to(DEV), k, v, table[1:2].repeat(3, 1)[:, :4].contiguous(), i32([4 * ps] * 3))[0])
    assert bool((full[2] == 0).all())


def test_paged_decode_attention_shared_pages_and_one_sequence_twice():
    g, lens = gen(9), [96, 96, 96]
    pool = Pool(g, lens, 2, 64, 16, torch.bfloat16)
    pool.table[1] = pool.table[0]        # the same sequence twice
    pool.table[2, :3] = pool.table[0, :3]  # a common prefix
    q = rnd(g, 3, 2, 64, dtype=torch.bfloat16)
    k, v, table, mass = pool.device()
    got = ops.paged_decode_attention(q.to(DEV), k, v, table, i32(lens), mass=mass)
    out, tol, add, add_tol = decode_ref(pool, q, [0] * 3, 0, 0)
    near(got, out, tol)
    near(mass, pool.mass.to(F64) + add, add_tol + 3 * 2.0 ** -22, "mass")


def test_paged_decode_attention_offsets_past_32_bits():
    """Pools of more than 2^32 bytes and 2^31 elements: the last pages are written and read back where they are."""
    Hkv, ps, dh = 16, 64, 128
    n_pages = 2 ** 31 // (Hkv * ps * dh) + 40
    k, v = (torch.empty(n_pages, Hkv, ps, dh, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    g, n = gen(4), 150
    pages = [n_pages - 1, 3, n_pages - 30]
    table = i32([pages])
    kk, vv, q = rnd(g, n, Hkv, dh, dtype=torch.bfloat16), rnd(g, n, Hkv, dh, dtype=torch.bfloat16), rnd(g, 1, Hkv, dh, dtype=torch.bfloat16)
    ops.paged_kv_write(kk.to(DEV), vv.to(DEV), k, v, table, i32([0]), seq_off=i32([0, n]))
    for i, p in enumerate(pages):
        part = kk[i * ps:(i + 1) * ps]
        assert torch.equal(k[p, :, : len(part)].cpu(), part.transpose(0, 1))
    got = ops.paged_decode_attention(q.to(DEV), k, v, table, i32([n]))
    for h in range(Hkv):
        o, t, _, _ = attend(q[0, h], kk[:, h], vv[:, h], torch.ones(n, dtype=torch.bool), 1 / math.sqrt(dh), 2.0 ** -16)
        near(got[0, h], o, t + 2.0 ** -8 * o.abs(), f"head {h}")


# ---- paged_kv_write -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,start,Hkv,dh,ps,W", [
    ([1, 1, 1], [0, 17, 63], 2, 64, 16, 4), ([40, 0, 7, 1], [5, 2, 31, 0], 3, 40, 8, 8), ([300], [1], 1, 128, 64, 5), ([5, 9], [60, -3], 2, 8, 16, 4)])
def test_paged_kv_write(dtype, lens, start, Hkv, dh, ps, W):
    g, off = gen(dh + ps), [2] + [2 + x for x in offsets(lens)[1:]]
    rows, n_pages = off[-1] + 3, len(lens) * W + 2  # rows ahead of the first sequence and behind the last
    table = torch.randperm(n_pages, generator=g)[: len(lens) * W].view(len(lens), W).to(torch.int32)
    table[-1, 1] = -1
    k, v = rnd(g, rows, Hkv, dh, dtype=dtype), rnd(g, rows, Hkv, dh, dtype=dtype)
    kp, vp, mass = torch.zeros(n_pages, Hkv, ps, dh, dtype=dtype), torch.zeros(n_pages, Hkv, ps, dh, dtype=dtype), torch.ones(n_pages, Hkv, ps)
    got = kp.to(DEV), vp.to(DEV), mass.to(DEV)
    packed = torch.cat([k, v], 2).to(DEV)  # strided views
    ops.paged_kv_write(packed[..., :dh], packed[..., dh:], got[0], got[1], table.to(DEV), i32(start), seq_off=i32(off), mass=got[2])
    for b, n in enumerate(lens):
        for i in range(n):
            pos = start[b] + i
            if 0 <= pos < W * ps and table[b, pos // ps] >= 0:
                p = int(table[b, pos // ps])
                kp[p, :, pos % ps], vp[p, :, pos % ps], mass[p, :, pos % ps] = k[off[b] + i], v[off[b] + i], 0.0
    assert all(torch.equal(a.cpu(), w) for a, w in zip(got, (kp, vp, mass)))
    if all(n == 1 for n in lens):
        again = torch.zeros_like(got[0]), torch.zeros_like(got[1])
        ops.paged_kv_write(k[2:5].to(DEV), v[2:5].to(DEV), *again, table.to(DEV), i32(start))
        assert all(torch.equal(a.cpu(), w) for a, w in zip(again, (kp, vp)))


# ---- kv_evict -----------------------------------------------------------------------------------------------------------------------
def evict_ref(mass, n, budget, recent, first):
    """mass of one head's n keys -> the positions that stay."""
    if n <= budget:
        return list(range(n))
    first = min(budget, first)
    last = min(recent, budget - first)
    key = [(not math.isnan(m), 0.0 if math.isnan(m) else -m, j) for j, m in enumerate(mass.tolist())]  # NaN is the largest
    mid = sorted(key[first:n - last])[: budget - first - last]
    return list(range(first)) + sorted(j for _, _, j in mid) + list(range(n - last, n))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,text,Hkv,dh,ps,budget,recent,sinks,kind", [
    ([40, 0, 7, 20, 21], [0] * 5, 2, 64, 16, 20, 5, 2, "random"),
    ([100, 33], [30, 0], 3, 40, 8, 24, 10, 0, "random"),        # a text longer than the budget
    ([3000, 2500], [0, 41], 2, 128, 64, 1300, 100, 4, "random"),
    ([2111], [0], 1, 8, 32, 1, 0, 0, "random"),                 # one key
    ([2111], [0], 1, 8, 32, 2110, 0, 0, "random"),              # all but one
    ([500, 400], [0, 0], 2, 64, 16, 100, 0, 0, "ties"),
    ([1500], [0], 2, 64, 16, 700, 3, 1, "zeros"),
    ([600], [0], 2, 64, 16, 90, 0, 0, "odd"),
    ([300], [0], 1, 64, 16, 50, 50, 0, "random"),               # the newest alone
    ([300], [0], 1, 64, 16, 50, 20, 30, "random"),
    ([12000], [0], 1, 64, 128, 5000, 1, 1, "random"),
])
def test_kv_evict(dtype, lens, text, Hkv, dh, ps, budget, recent, sinks, kind):
    g = gen(sum(lens) + budget)
    pool = Pool(g, lens, Hkv, dh, ps, dtype)
    if kind == "ties":
        pool.mass = (pool.mass * 4).floor()
    elif kind == "zeros":
        pool.mass = torch.where(pool.mass < 0.3, pool.mass, torch.where(pool.mass < 0.6, 0.0, -0.0))
    elif kind == "odd":
        pool.mass = torch.where(pool.mass < 0.05, float("nan"), torch.where(pool.mass < 0.1, float("inf"), pool.mass - 0.5))
    k, v, table, mass = pool.device()
    kept, left = ops.kv_evict(k, v, mass, table, i32(lens), budget, recent=recent, sinks=sinks, text_len=i32(text))
    assert left.tolist() == [min(n, budget) for n in lens]
    want_k, want_v, want_m = pool.k.clone(), pool.v.clone(), pool.mass.clone()
    for b, n in enumerate(lens):
        page, slot = pool.at(b)
        for h in range(Hkv):
            stay = evict_ref(pool.mass[page, h, slot], n, budget, recent, max(text[b], sinks))
            assert kept[b, h].tolist() == stay + [-1] * (budget - len(stay)), (b, h)
            to = slice(0, len(stay))
            for new, old in ((want_k, pool.k), (want_v, pool.v), (want_m, pool.mass)):
                new[page[to], h, slot[to]] = old[page[stay], h, slot[stay]]
    same = lambda a, w: bool(((a.cpu() == w) | (a.cpu().isnan() & w.isnan())).all())  # noqa: E731
    assert same(k, want_k) and same(v, want_v) and same(mass, want_m)


def test_kv_evict_pages_that_are_not_there():
    """Keys of a page id outside the pool weigh nothing and nothing is read from or written to it."""
    g, lens, ps = gen(6), [100], 16
    pool = Pool(g, lens, 1, 64, ps, torch.bfloat16)
    k, v, table, mass = pool.device()
    table[0, 2], table[0, 5] = -1, 10 ** 6
    kept, left = ops.kv_evict(k, v, mass, table, i32(lens), 40, recent=4)
    w = pool.mass[pool.at(0)[0], 0, pool.at(0)[1]]
    w[32:48] = w[80:96] = 0.0
    stay = evict_ref(w, 100, 40, 4, 0)
    assert kept[0, 0].tolist() == stay and left.tolist() == [40]
    page, slot = pool.at(0)
    for i, j in enumerate(stay):
        if not 32 <= i < 48 and not (32 <= j < 48 or 80 <= j < 96):
            assert torch.equal(k[page[i], 0, slot[i]].cpu(), pool.k[page[j], 0, slot[j]])


# ---- together -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_a_bounded_cache_over_a_prompt_and_many_tokens(dtype):
    """Prompt attention and the write of its keys, single tokens that add up their weights, an eviction whenever a sequence is full, on and on: outputs, lengths and
    the keys that are left, against lists of keys kept on the host."""
    g, H, Hkv, dh, ps, budget, full, text, B = gen(12), 4, 2, 64, 16, 40, 56, [6, 9, 0], 3
    lens = [50, 17, 3]
    off = offsets(lens)
    q, k, v = rnd(g, off[-1], H, dh, dtype=dtype), rnd(g, off[-1], Hkv, dh, dtype=dtype), rnd(g, off[-1], Hkv, dh, dtype=dtype)
    near(ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(off), window=24, sinks=2, text_len=i32(text)),
         *window_ref(q, k, v, off, text, 24, 2), "prompt")
    W = full // ps + 1
    table = torch.randperm(B * W + 2, generator=g)[: B * W].view(B, W).to(torch.int32)
    kp, vp = (torch.full((B * W + 2, Hkv, ps, dh), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    mass = torch.full((B * W + 2, Hkv, ps), 5.0, device=DEV)
    tab = table.to(DEV)
    ops.paged_kv_write(k.to(DEV), v.to(DEV), kp, vp, tab, i32([0] * B), seq_off=i32(off), mass=mass)
    # the host's lists: keys[b][h] = [key, value] rows in order, weights beside them
    keys = [[k[off[b]:off[b + 1], h] for h in range(Hkv)] for b in range(B)]
    vals = [[v[off[b]:off[b + 1], h] for h in range(Hkv)] for b in range(B)]
    lengths = i32(lens)
    for step in range(60):
        nq, nk, nv = rnd(g, B, H, dh, dtype=dtype), rnd(g, B, Hkv, dh, dtype=dtype), rnd(g, B, Hkv, dh, dtype=dtype)
        ops.paged_kv_write(nk.to(DEV), nv.to(DEV), kp, vp, tab, lengths, mass=mass)
        lengths = lengths + 1
        lens = [n + 1 for n in lens]
        got = ops.paged_decode_attention(nq.to(DEV), kp, vp, tab, lengths, window=24, sinks=2, text_len=i32(text), mass=mass)
        for b in range(B):
            m = sees(lens[b], lens[b] - 1, text[b], 24, 2)
            for h in range(Hkv):
                keys[b][h], vals[b][h] = torch.cat([keys[b][h], nk[b, h][None]]), torch.cat([vals[b][h], nv[b, h][None]])
            for h in range(H):
                o, t, _, _ = attend(nq[b, h], keys[b][h // 2], vals[b][h // 2], m, 1 / math.sqrt(dh), 2.0 ** -16 if dtype == torch.bfloat16 else 0.0)
                near(got[b, h], o, t + half_step(dtype) * o.abs(), f"step {step}")
        if max(lens) >= full:
            old = mass.cpu()
            kept, lengths = ops.kv_evict(kp, vp, mass, tab, lengths, budget, recent=12, sinks=2, text_len=i32(text))
            for b in range(B):
                j = torch.arange(lens[b])
                for h in range(Hkv):
                    stay = evict_ref(old[table[b][j // ps].long(), h, j % ps], lens[b], budget, 12, max(text[b], 2))
                    assert kept[b, h, : len(stay)].tolist() == stay
                    keys[b][h], vals[b][h] = keys[b][h][stay], vals[b][h][stay]
            lens = [min(n, budget) for n in lens]
            assert lengths.tolist() == lens
    for b in range(B):
        j = torch.arange(lens[b])
        for h in range(Hkv):
            assert torch.equal(kp.cpu()[table[b][j // ps].long(), h, j % ps], keys[b][h])


def test_captured_and_replayed_steps():
    """A step (write, attention with weights, eviction) and a prompt pass in a graph each: replays with the program's own eager calls between them give the eager results."""
    g, lens = gen(21), [1500, 700]
    pool = Pool(g, lens, 2, 64, 16, torch.bfloat16)
    q, nk, nv = (rnd(g, 2, h, 64, dtype=torch.bfloat16).to(DEV) for h in (4, 2, 2))
    at = i32([n - 1 for n in lens])
    lengths = i32(lens)
    state = pool.device()

    def step(k, v, table, mass):
        ops.paged_kv_write(nk, nv, k, v, table, at, mass=mass)
        o = ops.paged_decode_attention(q, k, v, table, lengths, mass=mass)
        o2 = ops.window_attention(q, nk, nv, i2, window=1)
        kept, left = ops.kv_evict(k, v, mass, table, lengths, 600, recent=50)
        return o, o2, kept, left

    i2 = i32([0, 1, 2])
    eager = [t.clone() for t in state]
    captured = [t.clone() for t in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*[t.clone() for t in state])
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for gr in graphs:  # two graphs of the same call: neither has the other's workspace
        with torch.cuda.graph(gr):
            outs.append(step(*captured))
    for rep in range(4):
        want = step(*eager)
        torch.cuda.synchronize()
        for t, s in zip(captured, state if rep == 0 else before):
            t.copy_(s)
        graphs[rep % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs[rep % 2])), rep
        assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(eager, captured)), rep
        before = [t.clone() for t in eager]


def test_two_streams_at_once():
    """The same pages read by two streams at a time, with a split and its join: each call has a workspace of its own."""
    g, lens = gen(31), [3000]
    pool = Pool(g, lens, 2, 64, 16, torch.bfloat16)
    k, v, table, _ = pool.device()
    qs = [rnd(g, 1, 4, 64, dtype=torch.bfloat16).to(DEV) for _ in range(2)]
    n = i32(lens)
    want = [ops.paged_decode_attention(q, k, v, table, n) for q in qs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_decode_attention(qs[i], k, v, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
