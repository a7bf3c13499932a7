"""Which kernel ``gemm_act`` takes for a product (the library's own query; without a GPU the rule counts 256 CUs), on the CPU."""

from __future__ import annotations

import ctypes
import importlib
import random

import pytest

# The forms' codes, with their tiles' rows and columns and a workgroup's threads.
SPLIT16, SPLIT32, TILE64, FOLD, WIDE, TILE256, ANY64, ANY128 = range(1, 9)
FORMS = {SPLIT16: (16, 16, 512), SPLIT32: (32, 32, 512), TILE64: (64, 128, 512), FOLD: (128, 128, 512), WIDE: (128, 256, 512),
         TILE256: (256, 256, 512), ANY64: (64, 64, 256), ANY128: (128, 128, 256)}


@pytest.fixture(scope="module")
def native():
    return importlib.import_module("zonos3-mini_amd._native")


def form(native, M, N, K, wide=True):
    """(form, workgroups)."""
    groups = ctypes.c_int64(-1)
    return native.lib().zgdn_gemm_act_form(M, N, K, int(wide), ctypes.byref(groups)), groups.value


@pytest.mark.parametrize("wide", [True, False])
def test_grids_hold_their_tiles(native, wide):
    """Products of any size: a grid of fewer than 2^32 threads that holds every tile, or no form at all."""
    rng = random.Random(5)
    sizes = [(2**29, 8, 8), (2**30, 1, 8), (2**31 - 257, 1, 1), (8, 2**29, 8), (1, 2**31 - 257, 16), (2**20, 2**16, 8),
             (2**25, 2**10, 64), (2**18, 2**18, 2**15), (2**30, 2**30, 8)]
    sizes += [tuple(int(2 ** rng.uniform(0, 30.9)) for _ in range(3)) for _ in range(2000)]
    refused = 0
    for M, N, K in sizes:
        f, groups = form(native, M, N, K, wide)
        if f == 0:
            refused += 1
            assert -(-M // 64) * -(-N // 64) > 2**23  # (fewer always fit)
            continue
        rows, cols, threads = FORMS[f]
        assert wide == (f < ANY64) or f <= SPLIT32
        assert groups * threads < 2**32 and groups % 8 == 0
        tiles = -(-M // rows) * (N // cols if f == FOLD else -(-N // cols))
        assert 0 <= groups - tiles < 8, (M, N, K, f, groups)
        if f == FOLD:
            assert 0 < N % 128 <= 16 and N // 128 >= 8
    assert 0 < refused < len(sizes)
    assert form(native, 2**29, 8, 8, wide)[0] and form(native, 2**30, 1, 8, wide)[0]


def test_products_without_a_form_are_refused(native):
    at = [ctypes.c_void_p(1 << n) for n in (20, 40, 60)]  # never read
    with pytest.raises(RuntimeError, match="more tiles than a grid holds"):
        native.call("zlin_gemm_act", at[0], 8, at[1], 8, None, 0, 0, None, 0, at[2], 1 << 30, 1 << 30, 1 << 30, 8, 1, None)


def test_every_form_is_taken(native):
    """No form of the table that no product of a model's sizes takes."""
    rng = random.Random(2)
    taken = set()
    for _ in range(20000):
        M, N, K = (int(2 ** rng.uniform(0, b)) for b in (16, 13, 13))
        if rng.random() < 0.3:
            N = 128 * rng.randint(8, 40) + rng.randint(1, 16)
        for wide in (True, False):
            taken.add(form(native, M, N, K, wide)[0])
    assert taken == set(FORMS)
