"""Edges of the packed attention's shapes on the GPU: no width, no heads, no keys, no capacity."""
import pytest
import torch

from chess_transformer_b200 import ops
from chess_transformer_b200.build import build
from chess_transformer_b200.library import FryError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def built():
    build()


def half(*shape):
    return torch.zeros(*shape, device="cuda", dtype=torch.float16)


def int32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("heads, width, match", [(4, 0, "heads a multiple of 8"), (0, 64, "query heads")])
def test_no_width_and_no_heads_are_refused(heads, width, match):
    at = int32(0, 3)
    with pytest.raises(FryError, match=match):
        ops.packed_attention(half(3, heads, width), half(3, 2, width), half(3, 2, width), at, at)
    with pytest.raises(FryError, match=match):
        ops.cached_attention(half(3, heads, width), half(3, 5, 2, width), half(3, 5, 2, width), int32(1, 2, 3))


def test_no_keys_and_no_capacity_answer_zeros():
    q = half(3, 4, 64) + 1
    assert not ops.packed_attention(q, half(0, 2, 64), half(0, 2, 64), int32(0, 3), int32(0, 0)).any()
    assert not ops.cached_attention(q, half(3, 0, 2, 64), half(3, 0, 2, 64), int32(0, 0, 0)).any()
    assert ops.packed_attention(half(0, 4, 64), half(3, 2, 64), half(3, 2, 64), int32(0, 0), int32(0, 3)).shape == (0, 4, 64)
    assert ops.cached_attention(half(0, 4, 64), half(0, 7, 2, 64), half(0, 7, 2, 64), int32()).shape == (0, 4, 64)
