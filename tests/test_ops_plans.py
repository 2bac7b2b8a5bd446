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


def xa(**kw):
    a = dict(dtype=1, B=2, Sq=3, Skv=7, H=4, Hkv=2, D=64, scale=0.125, q=P, k=P, v=P, o=P, lse=P, d_o=P, dq=P, dk=P, dv=P)
    return _lib.CrossAttentionArgs(**{**a, **kw})


@pytest.mark.parametrize("sizes,fits", [({"B": 1 << 20, "Hkv": 15, "H": 15, "D": 8, "Sq": 1, "Skv": 64}, True), ({"B": 1 << 20, "Hkv": 15, "H": 15, "D": 8, "Sq": 1, "Skv": 128}, True),
                                        ({"B": 1 << 20, "Hkv": 15, "H": 15, "D": 8, "Sq": 1, "Skv": 129}, False), ({"B": 1 << 20, "Hkv": 15, "H": 15, "D": 8, "Sq": 17, "Skv": 64}, True),
                                        ({"B": 1 << 20, "Hkv": 15, "H": 15, "D": 8, "Sq": 65, "Skv": 64}, True), ({"B": 1 << 20, "Hkv": 15, "H": 15, "D": 8, "Sq": 2049, "Skv": 200}, False),
                                        ({"B": 1 << 22, "Hkv": 1, "H": 1, "D": 256, "Sq": 1, "Skv": 320}, False), ({"B": 1 << 20, "Hkv": 15, "H": 15, "D": 8, "Sq": 0, "Skv": 10000}, True)])
def test_launches_that_the_hardware_does_not_take_are_refused_before_anything_runs(sizes, fits):
    """A launch has less than 2^32 threads: 256 of them to 64 or 128 keys of a key head, 64 or 256 to a block of rows."""
    n = C.c_size_t()
    status = L.sde_cross_attention_workspace(xa(**sizes), 1, n)
    assert status == (0 if fits else 1)
    if not fits:
        assert b"too many workgroups" in L.sde_last_error()


@pytest.mark.parametrize("m,fits", [((1 << 31) - 257, True), ((1 << 31) - 256, False), ((1 << 31) - 1, False)])
def test_rows_of_gated_ff_past_what_a_contraction_counts(m, fits):
    """dW runs over the rows in steps of 64 counted in 32 bits: the last 64 rows before 2^31 came out as no rows at all."""
    status = L.sde_gated_ff_workspace(ff(1, m, 8, 8), 1, C.c_size_t())
    assert status == (0 if fits else 1)
    if not fits:
        assert b"too large" in L.sde_last_error()
