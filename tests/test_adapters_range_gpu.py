"""Linears with adapters whose x down^T lies beyond fp16 or far below 1, on the GPU: the outputs are in range and right.
Tolerances as in test_adapters_gpu.py (a rounding of x down^T is off by 2^-11 of it, or 2^-25 below 2^-14)."""
import math

import pytest

from test_adapters_gpu import Case
from test_adapters_nonfinite_gpu import elapsed
from chess_transformer_b200.build import build

pytestmark = pytest.mark.gpu

SHAPES = [  # lengths, ids, adapters, rank, K, N
    ([1], [0], 1, 8, 64, 8),
    ([1] * 20, [i % 5 - 1 for i in range(20)], 4, 24, 2048, 136),
    ([17, 0, 14], [1, 0, 1], 2, 128, 400, 40),
    ([70, 0, 1, 127, 130], [2, 1, 0, -1, 2], 3, 16, 768, 1440),
    ([64, 64, 128, 256, 512], [0, 1, 2, 3, -1], 4, 72, 128, 256),
    ([3000, 2500], [1, 0], 2, 32, 256, 2304),
    ([1] * 200, [i % 9 - 1 for i in range(200)], 8, 128, 208, 72),
]


@pytest.fixture(scope="module", autouse=True)
def built():
    build()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("power", [17, 15, 12, -12])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_the_adapters_two_factors_may_be_far_from_one(shape, power, int8):
    case = Case(int8, *SHAPES[shape], seed=60 + shape)
    most = math.floor(math.log2(65504 / case.down.abs().amax().item()))  # down itself stays in fp16
    factor = 2.0 ** min(power, most)
    case.down, case.up = case.down * factor, case.up / factor
    assert case.down.isfinite().all() and case.up.isfinite().all() and case.expected()[0].abs().max() < 65504
    if power == 17 and shape > 0:  # beyond fp16 for some of the rows at least
        x = case.x.double() * (case.scales[0].double()[:, None] if int8 else 1.0)
        assert (x @ case.down.double().flatten(0, 1).T).abs().max() > 65520
    case.check()


@pytest.mark.parametrize("int8", [False, True])
def test_sums_beyond_fp16_cost_no_more_than_a_neighbour_that_is_not_finite(int8):
    case = Case(int8, [700, 3, 250, 1000, 90, 1, 1200, 500], [0, 1, 2, 3, -1, 0, 1, 2], 4, 32, 2048, 2048, seed=51)
    clean = elapsed(case.run)
    case.down, case.up = case.down * 2.0 ** 17, case.up * 2.0 ** -17
    taken = elapsed(case.run)
    print(f"int8={int8}: {clean * 1e3:.1f} us, beyond fp16 {taken * 1e3:.1f} us")
    case.check()
    assert taken <= 30 * clean + 0.1
