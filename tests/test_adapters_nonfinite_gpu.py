"""Linears with adapters whose operands are not finite, on the GPU: a row answers what its own operands give, whatever its
tile's other requests hold, and the call does not take long over it. Tolerances as in test_adapters_gpu.py."""
import math

import pytest
import torch

from test_adapters_gpu import Case
from chess_transformer_b200.build import build

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def built():
    build()


def elapsed(call):
    for _ in range(3):
        call()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    start.record()
    for _ in range(5):
        call()
    end.record()
    torch.cuda.synchronize()
    return start.elapsed_time(end) / 5


@pytest.mark.parametrize("N", [136, 2304])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_row_that_is_not_finite_stays_in_its_row(N, bad):
    case = Case(False, [30, 40, 100, 1900], [0, 1, -1, 2], 4, 16, 64, N, seed=50)
    expected, tolerance = case.expected()
    case.x[35, 7] = bad
    found = case.run()
    others = [m for m in range(case.x.shape[0]) if m != 35]
    assert ((found[others].double() - expected[others]).abs() <= tolerance[others]).all()
    assert not torch.isfinite(found[35]).any()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("what", ["adapter", "down", "x", "weight"])
def test_operands_that_are_not_finite_cost_little(what, int8):
    """Where all of a request's sums are not finite, they are its own operands' and stand. Where a neighbour's adapter has
    reached a row, the row's sums are taken again: K products each, in 16-byte loads."""
    if int8 and what in ("x", "weight"):
        pytest.skip("int8 values are finite")
    lengths = [700, 3, 250, 1000, 90, 1, 1200, 500]
    case = Case(int8, lengths, [0, 1, 2, 3, -1, 0, 1, 2], 4, 32, 2048, 2048, seed=51)
    clean = elapsed(case.run)
    if what == "adapter":
        case.up[1] = math.nan
    elif what == "down":
        case.down[:, 3, 5] = math.inf
    elif what == "x":
        case.x[:, 11] = math.inf
    else:
        case.weight[:, 11] = math.nan
    taken = elapsed(case.run)
    print(f"{what} int8={int8}: {clean * 1e3:.1f} us, not finite {taken * 1e3:.1f} us")
    assert taken <= (30 if what == "adapter" else 5) * clean + 0.1
