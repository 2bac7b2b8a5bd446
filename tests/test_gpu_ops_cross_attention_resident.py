"""GPU: cross attention whose workgroups keep all keys (two tiles of them at most) and walk several blocks of rows over them, forward and dq; ragged rows and keys.

Bounds: those of test_gpu_ops_cross_attention.py."""
import pytest
import torch

from test_gpu_ops_cross_attention import T, check, make

pytestmark = pytest.mark.gpu


def blocks(rows, d, dtype, dq):
    """Blocks of rows of a key head: 64 rows, or 128 where a wave takes two groups of 16 (head sizes below 5, for dq 4, steps of 64 bytes; fp32: 2, 4, 5, 8 steps)."""
    steps = -(-d * (4 if dtype == "f32" else 2) // 64)
    if dtype == "f32":
        steps = next(s for s in (2, 4, 5, 8, 10, 16) if s >= steps)
    return -(-rows // (64 if steps >= (4 if dq else 5) else 128))


@pytest.mark.parametrize("dtype,d", [("f16", 40), ("bf16", 40), ("f32", 40), ("f16", 64), ("bf16", 96), ("f32", 64), ("f16", 128), ("bf16", 128)])
@pytest.mark.parametrize("b,sq,skv,h,hkv", [(16, 1100, 77, 16, 16), (24, 700, 128, 16, 8), (16, 1937, 33, 8, 8)])
def test_many_blocks_of_rows_on_few_keys(b, sq, skv, h, hkv, d, dtype):
    rows = sq * (h // hkv)
    assert all(b * hkv * blocks(rows, d, dtype, dq) >= 2048 for dq in (False, True))          # two blocks and more to a workgroup
    check(*make(b, sq, skv, h, hkv, d, T[dtype], seed=d))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_many_blocks_of_ragged_rows(dtype):
    b, sq, skv = 24, 1100, 100
    q, k, v, do = make(b, sq, skv, 16, 16, 40, T[dtype], seed=2)
    n = lambda top, turn: torch.tensor([top * ((i * 7 + turn) % b) // (b - 1) for i in range(b)], dtype=torch.int32, device="cuda")
    mask = torch.rand(b, skv, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") < 0.8
    mask[5] = False
    check(q, k, v, do, n(sq, 0), n(skv, 5))
    check(q, k, v, do, n(sq, 3), n(skv, 1), mask)


def test_very_many_blocks():
    """16 blocks to a workgroup and a last workgroup with fewer."""
    b, sq = 64, 4200
    assert b * 16 * blocks(sq, 40, "f16", True) // 1024 >= 16
    check(*make(b, sq, 20, 16, 16, 40, torch.float16, seed=4))
