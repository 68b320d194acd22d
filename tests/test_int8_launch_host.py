"""The kernels that linear_int8 chooses hold the call in a launch, also where the fastest one would not; what none holds is refused."""

import random

import pytest

from appcorr_amd import _lib
from appcorr_amd import kernels as K

THREADS = {(16, 16): 512, (64, 64): 256, (64, 128): 512, (128, 128): 256, (192, 256): 512, (256, 256): 512}


def threads(M, N, tile):
    return -(-M // tile[0]) * -(-N // tile[1]) * THREADS[tile]


LARGE = [(1 << 27, 16, 64), ((1 << 30) - 1, 64, 64), ((1 << 30) - 1, 8, 128), (16, (1 << 30) - 8, 64), (1, 1 << 29, 64),
         (40, 1 << 29, 4096), (1 << 20, 1 << 18, 64)]


@pytest.mark.parametrize("M,N,Kd", LARGE)
def test_a_large_products_launch_holds_it(M, N, Kd):
    rows, columns, first = K.linear_int8_tile(M, N, Kd)
    assert 0 < first <= M and threads(first, N, (rows, columns)) < 1 << 32


def test_every_launch_holds_its_rows():
    r = random.Random(3)
    for _ in range(4000):
        M, N = int(2 ** r.uniform(0, 30)), 8 * int(2 ** r.uniform(0, 26))
        Kd = 64 * int(2 ** r.uniform(0, 10))
        if -(-M // 16) * -(-N // 16) >= 1 << 30:
            continue
        rows, columns, first = K.linear_int8_tile(M, N, Kd)
        assert threads(first, N, (rows, columns)) < 1 << 32
        if first < M:  # the rest goes by what the remaining rows are given
            tile = K.linear_int8_tile(M - first, N, Kd)[:2]
            assert first % rows == 0 and threads(M - first, N, tile) < 1 << 32


@pytest.mark.parametrize("M,N", [((1 << 30) - 1, 496), (1 << 30, 8), (8, 1 << 30), (1 << 22, 1 << 22)])
def test_what_no_launch_holds_is_refused(M, N):
    with pytest.raises(_lib.OudjatKernelError) as e:
        K.linear_int8_tile(M, N, 64)
    assert e.value.status_name == "OUDJAT_ERR_TOO_LARGE"
