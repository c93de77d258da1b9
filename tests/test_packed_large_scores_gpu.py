"""Attention whose scores are far beyond what the exponential resolves, on the GPU: the softmax is then the mean of the keys
that share the largest score, whatever that is. Queries and keys of +-2^e have products and sums that fp32 holds exactly, so
that equal scores are equal, and others apart by 2^(2 e + 1) scale at least."""
import pytest
import torch

from chess_transformer_b200 import ops
from chess_transformer_b200.build import build

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def built():
    build()


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


SHAPES = [  # rows, keys, heads, kv_heads, width: the prompt kernel's three forms, the row warps, the key warps with and without a split
    (300, 300, 4, 2, 64), (700, 700, 4, 1, 128), (150, 6400, 6, 6, 72), (70, 70, 24, 12, 32), (3, 150, 8, 1, 128), (1, 5000, 2, 1, 40), (1, 30, 2, 2, 64)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("exponent, scale", [(15, None), (15, 1.0), (0, 2.0 ** 40), (0, 1e30), (7, 3.0)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_the_largest_scores_share_the_answer(shape, causal, exponent, scale, dtype):
    rows, keys, heads, kv_heads, width = SHAPES[shape]
    g = torch.Generator(device="cuda").manual_seed(shape)
    signs = lambda *size: (torch.randint(0, 2, size, generator=g, device="cuda") * 2.0 - 1).mul(2.0 ** exponent).to(dtype)  # noqa: E731
    q, k = signs(rows, heads, width), signs(keys, kv_heads, width)
    v = torch.randn(keys, kv_heads, width, generator=g, device="cuda").to(dtype)
    found = ops.packed_attention(q, k, v, int32([0, rows]), int32([0, keys]), causal, scale).double()
    scores = torch.einsum("ihd,jhd->hij", q.double(), k.double().repeat_interleave(heads // kv_heads, 1))
    if causal:
        seen = torch.ones(rows, keys, dtype=torch.bool, device="cuda").tril(keys - rows)
        scores = scores.masked_fill(~seen, -float("inf"))
    top = (scores == scores.amax(-1, keepdim=True)).double()
    values = v.double().repeat_interleave(heads // kv_heads, 1)
    p = top / top.sum(-1, keepdim=True)
    expected = torch.einsum("hij,jhd->ihd", p, values)
    u = torch.finfo(dtype).eps / 2
    # the tied probabilities are alike in every rounding; the output's own, and fp32 sums of up to `keys` of them
    tolerance = u * expected.abs() + (u + (keys + 8) * 2.0 ** -24) * torch.einsum("hij,jhd->ihd", p, values.abs())
    assert ((found - expected).abs() <= tolerance).all()
    if rows == 1:
        cached = ops.cached_attention(q, k[None], v[None], int32([keys]), scale).double()
        assert ((cached - expected).abs() <= tolerance).all()
