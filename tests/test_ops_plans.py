"""CPU: the plans of the operators' kernels keep to what the kernels can address."""
import ctypes as C
import random

import pytest
import torch  # noqa: F401 - before the library: both use its HIP runtime

from diffusers_amd import _lib

P = 4096
L = _lib.lib()
ROWS = (256, 128, 64)


def ff(dtype, m, k, f):
    return _lib.GatedFfArgs(dtype, dtype, 0, m, k, f, k, k, f, f, k, k, P, P, P, P, P, P, P, P)


def plan(a, product):
    tile, splits, units = C.c_int(), C.c_int(), C.c_int64()
    assert L.sde_test_gated_ff_plan(a, product, tile, splits, units) == 0, L.sde_last_error()
    return tile.value, splits.value, units.value


def test_a_tile_of_dag_lies_inside_the_window_of_its_loads():
    """dx reads rows of [da dg], 2 F values apart: the rows of a tile have to lie within 2^31 bytes (past that they would come as zeros)."""
    rng = random.Random(0)
    cases = [(2, 1024, 512, 1_100_000), (2, 100_000, 4096, (1 << 21) - 4), (1, 4096, 512, (1 << 21) - 8), (2, 4096, 2048, 1 << 20), (2, 4096, 2048, (1 << 20) - 4)]
    cases += [(rng.choice([0, 1, 2]), rng.randint(1, 1 << 17), rng.randint(1, 1024) * 8, rng.randint(1, (1 << 18) - 1) * 8) for _ in range(300)]
    for dtype, m, k, f in cases:
        tile, _, _ = plan(ff(dtype, m, k, f), 1)
        assert (ROWS[tile] - 1) * 2 * f * (4 if dtype == 2 else 2) + 128 <= 1 << 31, (dtype, m, k, f)


def test_plans_of_known_sizes_are_as_they_were():
    """The rule leaves alone what lies inside the window."""
    assert [plan(ff(1, 8191, 1280, 5120), i) for i in range(3)] == [(0, 1, 1280), (0, 3, 480), (0, 1, 200)]
    assert plan(ff(0, 65536, 320, 1280), 0)[0] == 0 and plan(ff(0, 2, 1280, 5120), 0)[0] == 2


@pytest.mark.parametrize("product", [-1, 3])
def test_the_plan_refuses_an_unknown_product(product):
    assert L.sde_test_gated_ff_plan(ff(0, 4, 64, 64), product, C.c_int(), C.c_int(), C.c_int64()) == 1
