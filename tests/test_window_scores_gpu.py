"""GPU: what ops.window_attention makes of large scores, against 64 bits.

Tolerances as derived in test_cache_ops_gpu.py, where a tighter one does not hold by the construction of the inputs (said at each test)."""
import pytest
import torch

from tests.test_cache_ops_gpu import DEV, F64, gen, half_step, i32, near, rnd
from valle_amd import ops

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
LOG2E = 1.4426950408889634


def scored(rows, H, dh, levels, step, dtype):
    """q, k of equal rows whose products are exactly 3 * 159 / 128 + level * step in any precision of 24 bits, level by the key's 64-key tile."""
    q, k = torch.zeros(rows, H, dh, dtype=dtype), torch.zeros(rows, 1, dh, dtype=dtype)
    q[..., 0], q[..., 1] = 3.0, 1.0
    k[..., 0] = 159 / 128
    k[:, 0, 1] = torch.tensor(levels).repeat_interleave(64)[:rows] * step
    return q, k


@TYPES
@pytest.mark.parametrize("dh,H", [(64, 2), (128, 2), (128, 128)])  # the last: two fragments of queries a wave in bf16
@pytest.mark.parametrize("score", [5.0, 2e6, 2e7, 2e8, 1.5e9])
def test_window_attention_equal_scores_share_equally(dtype, dh, H, score):
    """Keys of one score get one weight, whatever the score's size (in units of the exp2 argument) and whichever tile they stand in: the mean of the values.  The
    weights of equal scores are equal, their rounding included, so only the two sums' roundings are left, and the result's."""
    rows = 384
    q, k = scored(rows, H, dh, [0] * 6, 1.0, dtype)
    v = rnd(gen(7), rows, 1, dh, dtype=dtype)
    got = ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32([0, rows]), text_len=i32([rows]), scale=score / LOG2E / 3.7265625)
    want = v.to(F64).mean(0)
    tol = 2 * (rows + 2) * 2.0 ** -24 * v.to(F64).abs().mean(0) + half_step(dtype) * want.abs()
    near(got, want.expand(rows, H, dh), tol, f"score {score}")


@TYPES
@pytest.mark.parametrize("dh,H", [(64, 2), (128, 128)])
@pytest.mark.parametrize("score,step,levels", [(2e6, 2.0 ** -18, [0, 3, 1, 6, 6, 2]), (2e7, 2.0 ** -21, [0, 3, 1, 6, 6, 2]), (2e8, 2.0 ** -22, [0, 1, 0, 2, 2, 1]),
                                               (2e8, 2.0 ** -22, [2, 1, 2, 0, 1, 2])])
def test_window_attention_large_scores_a_few_units_apart(dtype, dh, H, score, step, levels):
    """Scores of any size whose differences are a few units of the exp2 argument, the largest in a late tile: the difference to the row's reference is one rounding of a
    small number, so a weight is off by 2^-20 (its argument below 64: 2^-18 / 4; the exponential) and its rounding to the type, as for small scores."""
    rows = 384
    q, k = scored(rows, H, dh, levels, step, dtype)
    v = rnd(gen(8), rows, 1, dh, dtype=dtype)
    scale = score / LOG2E / 3.7265625
    got = ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32([0, rows]), text_len=i32([rows]), scale=scale)
    s = k[:, 0, 1].to(F64) * float(torch.tensor(scale, dtype=torch.float32)) * LOG2E
    p = torch.exp2(s - s.max())
    p = p / p.sum()
    want, size = p @ v[:, 0].to(F64), p @ v[:, 0].to(F64).abs()
    u = half_step(dtype)
    tol = (2 * (2.0 ** -19 + rows * 2.0 ** -24) + (2 * u if dtype == torch.bfloat16 else 0.0)) * size + u * want.abs()
    near(got, want.expand(rows, H, dh), tol, f"score {score}")
