"""GPU: every tile of the gated feed-forward's three products, with and without a split contraction, with fewer and with more tiles than workgroups that run at once (a workgroup then
walks to a second tile), on sizes that are no multiple of a tile.  The sizes are those for which the library's rule takes these forms: the plan is asserted, so that a change of the rule
cannot lose one unseen.  Bounds: those of test_gpu_ops_gated_ff.py."""
import ctypes as C

import pytest
import torch

from diffusers_amd import _lib
from test_gpu_ops_gated_ff import T, check, make

pytestmark = pytest.mark.gpu
RESIDENT = (256, 512, 1024)             # workgroups of each tile that run at once
SIZES = {  # M, K, F, and (tile, splits) of x W^T, dx, dW
    "16": [((235, 40, 48), (2, 1), (2, 1), (2, 1)), ((1507, 48, 1032), (1, 1), (2, 7), (2, 6)), ((3087, 72, 2232), (0, 1), (1, 10), (1, 7)), ((1895, 1160, 1160), (2, 1), (1, 1), (1, 1)),
           ((6277, 144, 4424), (0, 1), (0, 10), (0, 7)), ((4005, 2072, 2120), (1, 1), (0, 1), (0, 1)), ((35137, 48, 4408), (0, 1), (2, 3), (2, 11)), ((36357, 80, 48), (2, 1), (2, 1), (2, 32)),
           ((2705, 3432, 40), (2, 1), (1, 1), (2, 2)), ((215, 552, 3736), (2, 1), (2, 7), (2, 1)), ((215, 1552, 2720), (2, 1), (2, 5), (1, 1)), ((19785, 1200, 40), (1, 1), (0, 1), (1, 24)),
           ((359, 3144, 3952), (1, 1), (1, 3), (0, 1)), ((33671, 72, 2168), (0, 1), (1, 3), (1, 7)), ((35739, 136, 3312), (0, 1), (0, 3), (0, 9))],
    "32": [((259, 44, 40), (2, 1), (2, 1), (2, 1)), ((2323, 44, 684), (1, 1), (2, 6), (2, 11)), ((2059, 80, 2856), (1, 1), (1, 15), (1, 5)), ((537, 948, 3744), (2, 1), (2, 9), (2, 1)),
           ((8953, 464, 804), (0, 1), (2, 1), (2, 6)), ((6861, 236, 2160), (0, 1), (0, 9), (0, 15)), ((1095, 3112, 560), (2, 1), (1, 1), (1, 1)), ((11797, 72, 4136), (1, 1), (1, 8), (1, 11)),
           ((6819, 1736, 928), (0, 1), (1, 1), (0, 9)), ((1161, 2804, 3576), (2, 1), (0, 9), (1, 1)), ((13363, 932, 40), (2, 1), (0, 1), (2, 17)), ((9019, 2924, 40), (2, 1), (0, 1), (1, 11)),
           ((203, 1756, 4048), (2, 1), (1, 9), (0, 1)), ((267, 3440, 4144), (2, 1), (2, 7), (0, 1))]}
ACTS = ("gelu", "silu", "gelu_tanh")


def plan(dtype, m, k, f, product):
    code = {"f16": 0, "bf16": 1, "f32": 2}[dtype]
    tile, splits, units = C.c_int(), C.c_int(), C.c_int64()
    a = _lib.GatedFfArgs(code, code, 0, m, k, f, k, k, f, f, k, k)
    _lib.check(_lib.lib().sde_test_gated_ff_plan(a, product, tile, splits, units))
    return tile.value, splits.value, units.value


def forms(dtype):
    return SIZES["32" if dtype == "f32" else "16"]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_the_sizes_take_every_form(dtype):
    seen = set()
    for size, *expected in forms(dtype):
        for product in range(3):
            tile, splits, units = plan(dtype, *size, product)
            assert (tile, splits) == expected[product], (size, product)
            seen.add((product, tile, splits > 1, units > RESIDENT[tile]))
    for tile in range(3):
        assert {(0, tile, False, False), (0, tile, False, True)} <= seen
        assert {(p, tile, split, False) for p in (1, 2) for split in (False, True)} <= seen
        assert {(p, tile, False, True) for p in (1, 2)} <= seen


@pytest.mark.parametrize("dtype,index", [(t, i) for t in ("f16", "bf16", "f32") for i in range(len(forms(t)))])
def test_gated_ff_in_every_form(dtype, index):
    check(*make(*forms(dtype)[index][0], T[dtype], seed=index), ACTS[index % 3])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("act", ACTS)
def test_the_largest_tile_with_each_activation(dtype, act):
    assert plan(dtype, 6277, 144, 4424, 0)[0] == 0
    check(*make(6277, 144, 4424, T[dtype], seed=40, bt=torch.float32), act)
