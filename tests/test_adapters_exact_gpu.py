"""The int8 linear with adapters sums its int8 products exactly, as int8_linear does, for any number of rows."""
import pytest
import torch

from chess_transformer_b200 import ops
from chess_transformer_b200.build import build

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def built():
    build()


@pytest.mark.parametrize("K, N", [(16, 8), (80, 24), (768, 1152), (1040, 264), (4096, 72), (16384, 40)])
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 32, 33, 70])
def test_without_adapters_it_is_the_int8_linear(M, K, N):
    """Sums of K products of up to 127 * 127: beyond 2^24, which fp32 holds exactly, from K = 1041 on."""
    g = torch.Generator(device="cuda").manual_seed(M * K + N)
    whole = lambda *shape: (127 - torch.randint(0, 9, shape, generator=g, device="cuda")).to(torch.int8)  # noqa: E731
    x, weight = whole(M, K), whole(N, K)
    x[:, 1::7] = -x[:, 1::7]
    weight[1::2] = -weight[1::2]
    x_scale, weight_scale = (torch.rand(n, generator=g, device="cuda") * 0.001 for n in (M, N))
    bias = torch.randn(N, generator=g, device="cuda").half()
    down, up = torch.ones(1, 8, K, device="cuda").half(), torch.ones(1, N, 8, device="cuda").half()
    at, ids = torch.tensor([0, M], dtype=torch.int32, device="cuda"), torch.tensor([-1], dtype=torch.int32, device="cuda")
    found = ops.int8_adapter_linear(x, x_scale, weight, weight_scale, bias, None, down, up, at, ids)
    assert torch.equal(found, ops.int8_linear(x, x_scale, weight, weight_scale, bias, None, False, "projection"))
