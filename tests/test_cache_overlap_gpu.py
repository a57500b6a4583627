"""GPU: calls of the cache operators through Python whose output lies over an operand are refused and write nothing; a copy inside the pools is not."""
import pytest
import torch

from tests.test_cache_ops_gpu import DEV, Pool, gen, i32, rnd
from valle_amd import _lib, ops

pytestmark = pytest.mark.gpu


def test_outputs_over_operands_are_refused():
    g, rows, H, dh = gen(1), 70, 2, 64
    q, k, v = (rnd(g, rows, H, dh, dtype=torch.bfloat16).to(DEV) for _ in range(3))
    room = torch.cat([q, k, v])
    was = room.clone()
    off = i32([0, rows])
    parts = [room[i * rows:(i + 1) * rows] for i in range(3)]
    for out in (parts[1], parts[2], room[rows - 1:2 * rows - 1], room[1:rows + 1]):
        with pytest.raises(_lib.VleError, match="overlap"):
            ops.window_attention(*parts, off, out=out)
    pool = Pool(g, [40, 7], H, dh, 16, torch.bfloat16)
    kp, vp, table, mass = pool.device()
    lengths, one = i32([40, 7]), room[:2]
    for out in (kp.view(-1, H, dh)[:2], vp.view(-1, H, dh)[-2:], room[1:3]):
        with pytest.raises(_lib.VleError, match="overlap"):
            ops.paged_decode_attention(one, kp, vp, table, lengths, out=out)
    both = torch.zeros(2 * kp.shape[0], *kp.shape[1:], dtype=kp.dtype, device=DEV)
    n = kp.shape[0]
    with pytest.raises(_lib.VleError, match="overlap"):
        ops.kv_evict(both[:n], both[1:n + 1], mass, table, lengths, 20)
    with pytest.raises(_lib.VleError, match="overlap"):
        ops.paged_kv_write(one, one, both[:n], both[n - 1:2 * n - 1], table, lengths)
    torch.cuda.synchronize()
    assert torch.equal(room, was) and bool((both == 0).all()) and torch.equal(mass.cpu(), pool.mass)
    assert torch.equal(kp.cpu().nan_to_num(), pool.k.nan_to_num()) and torch.equal(vp.cpu().nan_to_num(), pool.v.nan_to_num())


def test_a_page_copied_to_another_of_its_pool():
    g, H, dh, ps = gen(2), 2, 64, 16
    kp, vp = (rnd(g, 5, H, ps, dh, dtype=torch.bfloat16).to(DEV) for _ in range(2))
    want = kp.clone(), vp.clone()
    want[0][4], want[1][4] = kp[1], vp[1]
    ops.paged_kv_write(kp[1].transpose(0, 1), vp[1].transpose(0, 1), kp, vp, i32([[4]]), i32([0]), seq_off=i32([0, ps]))
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
