"""GPU: the launches of the cache operators that only larger calls take, against 64 bits (tolerances as in test_cache_ops_gpu.py)."""
import math

import pytest
import torch

from tests.test_cache_ops_gpu import DEV, F64, Pool, decode_ref, evict_ref, gen, half_step, i32, near, offsets, rnd, sees
from valle_amd import _lib, ops

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])


# ---- window_attention in fp32 with one group of waves a workgroup (more than 448 work items; the other tests' calls have fewer) -----
@pytest.mark.parametrize("dh,Hkv,window,sinks", [(32, 32, 0, 0), (24, 4, 33, 2), (64, 8, 0, 0), (56, 32, 150, 0), (96, 4, 70, 3), (88, 1, 0, 0), (128, 4, 33, 2), (120, 32, 0, 0)])
def test_window_attention_fp32_many_ragged_sequences(dh, Hkv, window, sinks):
    """Every head size's kernel with sequences that end inside their runs, rows of no sequence, and a key that is not a number, which reaches only the rows that see it."""
    g, H = gen(dh), 32
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 200, 257, 300]
    text = [0, 1, 3, 0, 17, 0, 70, 9, 0, 40, 0, 64, 0, 65, 120]
    off = offsets(lens)
    rows = off[-1] + 13
    assert (-(-rows // 64) + len(lens) + 1) * H > 448
    q, k, v = rnd(g, rows, H, dh), rnd(g, rows, Hkv, dh), rnd(g, rows, Hkv, dh)
    poisoned = {12: 180, 14: 130}  # sequence: key
    for b, j in poisoned.items():
        k[off[b] + j] = float("nan")
    q, k, v = q.to(DEV), k.to(DEV), v.to(DEV)
    got = ops.window_attention(q, k, v, i32(off), window=window, sinks=sinks, text_len=i32(text))
    assert bool((got[off[-1]:] == 0).all())
    u = half_step(torch.float32)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        r = slice(off[b], off[b + 1])
        m = torch.stack([sees(n, i, min(text[b], n), window, sinks) for i in range(n)]).to(DEV)
        hit = m[:, poisoned[b]] if b in poisoned else torch.zeros(n, dtype=torch.bool, device=DEV)
        assert bool(got[r][hit].isnan().all())
        for h in range(0, H, 5):
            qh, kh, vh = q[r, h].double(), k[r, h // (H // Hkv)].double().nan_to_num(0.0), v[r, h // (H // Hkv)].double()
            spread = float((qh.abs() @ kh.abs().T).max()) / math.sqrt(dh)
            w = torch.softmax(((qh @ kh.T) / math.sqrt(dh)).masked_fill(~m, -math.inf), 1)
            want, delta = w @ vh, 2 * (dh + 4) * 2.0 ** -24 * spread + 2.0 ** -20
            tol = 2 * (delta + n * 2.0 ** -24) * (w @ vh.abs()) + u * want.abs()
            near(got[r, h][~hit], want[~hit].cpu(), tol[~hit].cpu(), f"sequence {b} head {h}")


# ---- paged_decode_attention -----------------------------------------------------------------------------------------------------------
def workspace(dtype, B, H, Hkv, dh, W, ps, mass):
    return _lib.load().vle_op_paged_decode_workspace_bytes(_lib.DTYPE_BF16 if dtype == torch.bfloat16 else _lib.DTYPE_F32, B, H, Hkv, dh, W, ps, 0, 0, 0, int(mass))


@TYPES
@pytest.mark.parametrize("B,H,Hkv,dh,ps,width", [
    (70, 8, 8, 64, 16, 70), (70, 8, 8, 128, 32, 35),       # one launch, weights added by the workgroup that has them
    (3, 16, 8, 64, 16, 1700), (3, 8, 8, 128, 64, 200),     # split and joined
])
@pytest.mark.parametrize("with_mass", [False, True], ids=["", "mass"])
def test_paged_decode_attention_that_reads_past_the_memory_side_cache(dtype, B, H, Hkv, dh, ps, width, with_mass):
    """Tables wide enough for more than 128 MB of keys and values: their loads are non-temporal."""
    assert width * ps * B * Hkv * dh * (4 if dtype == torch.bfloat16 else 8) > 128 << 20
    assert (workspace(dtype, B, H, Hkv, dh, width, ps, False) > 0) == (B == 3)
    g = gen(B + dh)
    lens = torch.randint(0, 260, (B,), generator=g).tolist() if B > 3 else [1500, 0, 77]
    pool = Pool(g, lens, Hkv, dh, ps, dtype, width=width)
    q = rnd(g, B, H, dh, dtype=dtype, gain=1.5)
    k, v, table, mass = pool.device()
    got = ops.paged_decode_attention(q.to(DEV), k, v, table, i32(lens), mass=mass if with_mass else None)
    out, tol, add, add_tol = decode_ref(pool, q, [0] * B, 0, 0)
    near(got, out, tol, "out")
    if with_mass:
        near(mass, pool.mass.to(F64) + add, add_tol + 2.0 ** -22, "mass")


@pytest.mark.parametrize("dtype,lens,H,Hkv,dh", [
    (torch.bfloat16, [600, 450], 16, 1, 64), (torch.bfloat16, [470], 24, 1, 96), (torch.bfloat16, [500, 0], 32, 2, 128),
    (torch.float32, [300], 24, 1, 96), (torch.float32, [270, 0, 310], 40, 2, 128)])
def test_paged_decode_attention_weights_of_one_launch_by_the_join(dtype, lens, H, Hkv, dh):
    """Not split, but more scores than fit beside the outputs, or more heads a group than one workgroup takes: the weights are added by a launch of their own."""
    ps = 16
    W = -(-max(lens) // ps)
    assert workspace(dtype, len(lens), H, Hkv, dh, W, ps, False) == 0 < workspace(dtype, len(lens), H, Hkv, dh, W, ps, True)
    g = gen(H + dh)
    pool = Pool(g, lens, Hkv, dh, ps, dtype)
    q = rnd(g, len(lens), H, dh, dtype=dtype, gain=1.5)
    k, v, table, mass = pool.device()
    got = ops.paged_decode_attention(q.to(DEV), k, v, table, i32(lens), mass=mass)
    out, tol, add, add_tol = decode_ref(pool, q, [0] * len(lens), 0, 0)
    near(got, out, tol, "out")
    near(mass, pool.mass.to(F64) + add, add_tol + 2.0 ** -22, "mass")


# ---- kv_evict -------------------------------------------------------------------------------------------------------------------------
@TYPES
@pytest.mark.parametrize("lens,text,Hkv,ps,budget,recent,sinks,kind,width", [
    ([20000, 17000, 300, 16385], [0, 30, 0, 0], 2, 8, 9000, 100, 4, "random", None),  # more candidates than a workgroup's registers hold
    ([1500, 0, 700], [0, 0, 41], 2, 16, 600, 10, 0, "ties", 1100),                    # few of them, under a table for many
    ([18000], [0], 1, 64, 17999, 0, 0, "zeros", None),
    ([18000], [0], 1, 64, 1, 0, 0, "ties", None),
    ([17000], [0], 1, 32, 2000, 7, 1, "odd", None),
    ([40000, 33000], [0, 5], 1, 8, 31000, 50, 2, "random", None),                     # more pages than a workgroup keeps
])
def test_kv_evict_long_tables(dtype, lens, text, Hkv, ps, budget, recent, sinks, kind, width):
    g, dh = gen(sum(lens) + budget), 8
    pool = Pool(g, lens, Hkv, dh, ps, dtype, width=width)
    assert pool.table.shape[1] * ps > 16384
    if kind == "ties":
        pool.mass = (pool.mass * 4).floor()
    elif kind == "zeros":
        pool.mass = torch.where(pool.mass < 0.3, pool.mass, torch.where(pool.mass < 0.6, 0.0, -0.0))
    elif kind == "odd":
        pool.mass = torch.where(pool.mass < 0.05, float("nan"), torch.where(pool.mass < 0.1, float("inf"), pool.mass - 0.5))
    k, v, table, mass = pool.device()
    kept, left = ops.kv_evict(k, v, mass, table, i32(lens), budget, recent=recent, sinks=sinks, text_len=i32(text))
    assert left.tolist() == [min(n, budget) for n in lens]
    want_k, want_v, want_m, kept = pool.k.clone(), pool.v.clone(), pool.mass.clone(), kept.cpu()
    for b, n in enumerate(lens):
        page, slot = pool.at(b)
        for h in range(Hkv):
            stay = torch.tensor(evict_ref(pool.mass[page, h, slot], n, budget, recent, max(text[b], sinks)), dtype=torch.int64)
            assert torch.equal(kept[b, h], torch.cat([stay, torch.full((budget - len(stay),), -1)]).to(torch.int32)), (b, h)
            to = slice(0, len(stay))
            for new, old in ((want_k, pool.k), (want_v, pool.v), (want_m, pool.mass)):
                new[page[to], h, slot[to]] = old[page[stay], h, slot[stay]]
    same = lambda a, w: bool(((a.cpu() == w) | (a.cpu().isnan() & w.isnan())).all())  # noqa: E731
    assert same(k, want_k) and same(v, want_v) and same(mass, want_m)
