"""GPU: what ops.paged_decode_attention makes of extreme values -- values near the largest number, infinities, large scores -- against 64 bits.

Tolerances as derived in test_cache_ops_gpu.py, where a tighter one does not hold by the construction of the inputs (said at each test)."""
import math

import pytest
import torch

from tests.test_cache_ops_gpu import DEV, F64, Pool, attend, gen, half_step, i32, near, rnd, sees
from tests.test_window_scores_gpu import LOG2E, scored
from valle_amd import ops

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])


def cache(lens, Hkv, dh, ps, dtype, seed, width=None):
    return Pool(gen(seed), lens, Hkv, dh, ps, dtype, width=width)


def plain_decode(pool, q):
    """Every head over all keys in 64 bits (infinities and NaN as they come), and sum p |v|, with the weights' bound."""
    B, H, dh = q.shape
    out, size = torch.zeros(B, H, dh, dtype=F64), torch.zeros(B, H, dh, dtype=F64)
    rel = 0.0
    for b in range(B):
        page, slot = pool.at(b)
        see = torch.ones(pool.lens[b], dtype=torch.bool)
        for h in range(H):
            kh, vh = (x[page, h // (H // pool.Hkv), slot] for x in (pool.k, pool.v))
            _, _, p, delta = attend(q[b, h], kh, vh.nan_to_num(0.0, 0.0, 0.0), see, 1 / math.sqrt(dh))
            rel = max(rel, 2 * (delta + len(p) * 2.0 ** -24))
            out[b, h], size[b, h] = (p[:, None] * vh.to(F64)).sum(0), (p[:, None] * vh.to(F64).abs()).sum(0)
    return out, size, rel


# one launch with 8 waves, with 4 (16 heads a group), a split and its join; heads that fill their registers and heads that do not
SHAPES = pytest.mark.parametrize("lens,H,Hkv,dh,ps,width", [
    ([100, 37], 2, 2, 64, 16, None), ([70], 16, 1, 128, 16, None), ([90, 5], 6, 2, 40, 8, None), ([1400, 300], 4, 2, 64, 16, None), ([900, 64], 2, 1, 120, 32, 80)])


@TYPES
@SHAPES
def test_paged_decode_attention_largest_values(dtype, lens, H, Hkv, dh, ps, width):
    """Values whose unnormalised sums pass the largest number still average to numbers below it; the weights that are added up are those of any values."""
    pool = cache(lens, Hkv, dh, ps, dtype, 3, width)
    q = rnd(gen(4), len(lens), H, dh, dtype=dtype)
    table = pool.table.to(DEV)
    k, mass = pool.k.to(DEV), [torch.zeros_like(pool.mass, device=DEV) for _ in range(2)]
    ops.paged_decode_attention(q.to(DEV), k, pool.v.to(DEV), table, i32(lens), mass=mass[0])
    there = pool.v.isfinite()
    pool.v = torch.where(there, 2.0 ** 127, float("nan")).to(dtype)
    got = ops.paged_decode_attention(q.to(DEV), k, pool.v.to(DEV), table, i32(lens), mass=mass[1])
    _, _, rel = plain_decode(pool, q)
    near(got / 2.0 ** 127, torch.ones(got.shape, dtype=F64), rel + half_step(dtype), "one value")
    assert torch.equal(*mass)
    pool.v = torch.where(there, torch.rand(pool.v.shape, generator=gen(5), dtype=F64).mul(2).sub(1).mul(3e38), float("nan")).to(dtype)
    got = ops.paged_decode_attention(q.to(DEV), k, pool.v.to(DEV), table, i32(lens))
    want, size, rel = plain_decode(pool, q)
    near(got, want, (rel + (2.0 ** -15 if dtype == torch.bfloat16 else 0.0)) * size + half_step(dtype) * want.abs(), "random")


@TYPES
@SHAPES
def test_paged_decode_attention_infinite_values(dtype, lens, H, Hkv, dh, ps, width):
    """A visible infinity comes through as one, opposite ones and NaN as NaN, each in its own element; the others are what they are without it."""
    pool = cache(lens, Hkv, dh, ps, dtype, 6, width)
    q = rnd(gen(7), len(lens), H, dh, dtype=dtype, gain=0.3)  # no weight underflows, so 0 * inf does not occur
    page, slot = pool.at(0)
    inf, at = float("inf"), lambda j, e, x: pool.v.__setitem__((int(page[j]), slice(None), int(slot[j]), e), x)
    at(3, 0, inf), at(4, 1, -inf), at(5, 2, inf), at(6, 2, -inf), at(9, 5, float("nan")), at(lens[0] - 1, dh - 1, inf)
    got = ops.paged_decode_attention(q.to(DEV), pool.k.to(DEV), pool.v.to(DEV), pool.table.to(DEV), i32(lens)).cpu().to(F64)
    want, size, rel = plain_decode(pool, q)
    fine = want.isfinite()
    assert int((~fine).sum()) == 5 * H
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0, 1.0, -1.0)[~fine], want.nan_to_num(0.0, 1.0, -1.0)[~fine])
    near(got[fine], want[fine], ((rel + (2.0 ** -15 if dtype == torch.bfloat16 else 0.0)) * size + half_step(dtype) * want.abs())[fine], "the others")


@TYPES
def test_paged_decode_attention_equal_scores_share_equally(dtype):
    """As for the prompt: the rounded scores of equal keys are equal, and so are their weights."""
    for n in (150, 1500):  # one launch; split and joined
        pool = cache([n], 1, 64, 16, dtype, 9)
        q, k = scored(n, 2, 64, [0] * 24, 1.0, dtype)
        page, slot = pool.at(0)
        pool.k[page, :, slot] = k
        for score in (2e6, 2e8, 1.5e9):
            got = ops.paged_decode_attention(q[:1].to(DEV), pool.k.to(DEV), pool.v.to(DEV), pool.table.to(DEV), i32([n]), scale=score / LOG2E / 3.7265625)
            v = pool.v[page, 0, slot].to(F64)
            want = v.mean(0)
            near(got[0], want.expand(2, 64), 2 * (n + 2) * 2.0 ** -24 * v.abs().mean(0) + half_step(dtype) * want.abs(), f"score {score}")


@TYPES
@pytest.mark.parametrize("lens,text,H,Hkv,dh,ps,window,sinks,width", [
    ([300, 33, 5], [20, 0, 5], 4, 2, 64, 16, 40, 2, None),       # a gap between the head and the window, where everything is NaN
    ([700, 150], [0, 60], 3, 1, 96, 64, 100, 4, None),
    ([1500, 900], [0, 17], 4, 2, 64, 8, 700, 3, None),           # split and joined
    ([900, 64], [70, 0], 40, 2, 40, 16, 333, 0, 300),            # 20 heads a group, a table wider than the sequences
    ([260], [259], 2, 2, 120, 32, 1, 0, None)])
def test_paged_decode_attention_extreme_values_behind_a_mask(dtype, lens, text, H, Hkv, dh, ps, window, sinks, width):
    """Values near the largest number where the newest token looks, infinities and NaN wherever it does not, pages that are not there, queries out of a packed row; then
    one visible infinity."""
    g = gen(sum(lens) + window)
    pool = Pool(g, lens, Hkv, dh, ps, dtype, width=width)
    pool.table[0, 1] = -3  # keys ps .. 2 ps - 1 of the first sequence
    n_pages = pool.k.shape[0]
    packed = rnd(g, len(lens), 3 * H * dh, dtype=dtype, gain=0.3)
    q = packed[:, H * dh:2 * H * dh].view(-1, H, dh)
    seen = []
    for b, n in enumerate(lens):
        page, slot = pool.at(b)
        m = sees(n, n - 1, min(text[b], n), window, sinks) & (page >= 0) & (page < n_pages)
        big = rnd(g, n, Hkv, dh).clamp(-1, 1).mul(3e38).to(dtype)
        gone, there = ~m & (page >= 0), page >= 0
        pool.v[page[there], :, slot[there]] = big[there]
        pool.v[page[gone], :, slot[gone]] = float("nan")
        pool.v[page[gone], 0, slot[gone]] = float("inf")
        pool.k[page[gone], :, slot[gone]] = float("nan")
        seen.append((page, slot, m))

    def check(what):
        got = ops.paged_decode_attention(packed.to(DEV)[:, H * dh:2 * H * dh].view(-1, H, dh), pool.k.to(DEV), pool.v.to(DEV), pool.table.to(DEV), i32(lens), window=window, sinks=sinks,
                                         text_len=i32(text)).cpu().to(F64)
        for b, (page, slot, m) in enumerate(seen):
            for h in range(H):
                kh, vh = (x[page.clamp(0), h // (H // Hkv), slot] for x in (pool.k, pool.v))
                _, _, p, delta = attend(q[b, h], kh, vh.nan_to_num(0.0, 0.0, 0.0), m, 1 / math.sqrt(dh))
                want, size = (p[:, None] * vh[m].to(F64)).sum(0), (p[:, None] * vh[m].to(F64).abs()).sum(0)
                fine = want.isfinite()
                assert torch.equal(got[b, h][~fine], want[~fine]), (what, b, h)
                rel = 2 * (delta + len(p) * 2.0 ** -24) + (2.0 ** -15 if dtype == torch.bfloat16 else 0.0)
                near(got[b, h][fine], want[fine], (rel * size + half_step(dtype) * want.abs())[fine], f"{what} {b} {h}")

    check("large")
    for b, (page, slot, m) in enumerate(seen):
        j = int(m.nonzero()[len(lens) - 1 if int(m.sum()) > len(lens) else 0])
        pool.v[page[j], :, slot[j], b] = float("inf")
    check("one infinity")
