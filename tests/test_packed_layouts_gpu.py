"""Layouts and sizes that the packed operators' documentation allows: each gives the bits of the dense call, or its definition."""
import pytest
import torch

from chess_transformer_b200 import ops
from chess_transformer_b200.build import build
from test_adapters_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def built():
    build()


def offsets(lengths):
    return torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)


def heads_first(t):
    """The same values, heads in the outermost place of memory."""
    return t.transpose(-2, -3).contiguous().transpose(-2, -3)


def padded(t):
    """The same values, each row the beginning of a longer one."""
    return torch.cat([t, torch.full_like(t[..., :24], float("nan"))], -1)[..., : t.shape[-1]]


def spread(t):
    """The same values, every other head of twice as many."""
    return torch.stack([t, torch.full_like(t, float("nan"))], -2).flatten(-3, -2)[..., ::2, :]


LAYOUTS = [heads_first, padded, spread, lambda t: heads_first(padded(t))]
SHAPES = [  # queries, keys, heads, kv_heads, width: the prompt kernel's three forms, the row warps, the key warps
    ([300, 129], [300, 129], 8, 2, 64), ([700], [700], 8, 4, 128), ([150], [6400], 6, 6, 72), ([70, 3, 64], [70, 3, 64], 24, 12, 32),
    ([3, 1], [700, 900], 8, 1, 128), ([1], [5000], 1, 1, 40)]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
def test_attention_reads_any_layout(layout, shape):
    queries, keys, heads, kv_heads, width = SHAPES[shape]
    g = torch.Generator(device="cuda").manual_seed(shape)
    normal = lambda *size: torch.randn(*size, generator=g, device="cuda").half()  # noqa: E731
    q, k, v, at, k_at = normal(sum(queries), heads, width), normal(sum(keys), kv_heads, width), normal(sum(keys), kv_heads, width), offsets(queries), offsets(keys)
    lay = LAYOUTS[layout]
    expected = ops.packed_attention(q, k, v, at, k_at)
    for a, b, c in ((lay(q), k, v), (q, lay(k), v), (q, k, lay(v)), (lay(q), lay(k), lay(v))):
        assert torch.equal(ops.packed_attention(a, b, c, at, k_at), expected)


@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
@pytest.mark.parametrize("capacity, width", [(40, 64), (3000, 128), (700, 24)])
def test_a_cache_of_any_layout(layout, capacity, width):
    g = torch.Generator(device="cuda").manual_seed(capacity)
    normal = lambda *size: torch.randn(*size, generator=g, device="cuda").bfloat16()  # noqa: E731
    q, k, v = normal(5, 8, width), normal(5, capacity, 2, width), normal(5, capacity, 2, width)
    lengths = torch.tensor([capacity, 0, 1, capacity // 2, capacity - 1], dtype=torch.int32, device="cuda")
    lay = LAYOUTS[layout]
    assert torch.equal(ops.cached_attention(lay(q), lay(k), lay(v), lengths), ops.cached_attention(q, k, v, lengths))
    outer = lambda t: lay(t.transpose(0, 1).contiguous().transpose(0, 1))  # noqa: E731  (tokens outermost)
    assert torch.equal(ops.cached_attention(q, outer(k), outer(v), lengths), ops.cached_attention(q, k, v, lengths))


def test_offsets_by_a_stride():
    q = torch.randn(60, 4, 64, device="cuda").half()
    at = offsets([20, 3, 37])
    wide = torch.stack([at, torch.full_like(at, 7)], 1)
    assert torch.equal(ops.packed_attention(q, q, q, wide[:, 0], wide[:, 0]), ops.packed_attention(q, q, q, at, at))


@pytest.mark.parametrize("count", [1100, 70000])
def test_many_sequences(count):
    """Token s of sequence s sees two keys of scores 0, so it answers their mean; every fifth has none and answers 0."""
    q = torch.zeros(count, 2, 32, device="cuda", dtype=torch.float16)
    lengths = torch.full((count,), 2, device="cuda")
    lengths[::5] = 0
    k_at = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)]).to(torch.int32)
    total = int(k_at[-1])
    v = (torch.arange(total, device="cuda") % 512 * 2).half()[:, None, None].expand(-1, 1, 32).contiguous()
    found = ops.packed_attention(q, torch.zeros_like(v), v, torch.arange(count + 1, dtype=torch.int32, device="cuda"), k_at)
    first = k_at[:-1].long()
    mean = (v[first.clamp(max=total - 2), 0, 0] + v[(first + 1).clamp(max=total - 1), 0, 0]).float() / 2
    expected = torch.where(lengths > 0, mean, 0.0)
    assert torch.equal(found.float(), expected[:, None, None].expand(-1, 2, 32))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lengths, ids, rank, K, N", [
    ([1], [0], 8, 16, 8), ([33], [0], 8, 16, 8), ([200, 1], [0, 1], 16, 16, 8), ([129, 64], [1, 0], 128, 16, 16),
    ([0] * 900 + [40] + [0] * 700 + [50] + [0] * 300, [i % 2 for i in range(1902)], 16, 64, 72),
    ([0] * 900 + [4] + [0] * 700 + [5] + [0] * 300, [i % 2 for i in range(1902)], 16, 64, 72)])
def test_the_smallest_linears_and_many_empty_requests(lengths, ids, rank, K, N, int8):
    Case(int8, lengths, ids, 2, rank, K, N, seed=70).check()
    if not int8 and K == 16:
        Case(int8, lengths, ids, 2, rank, 8, N, seed=71).check()


def test_operands_of_the_linear_by_strides():
    case = Case(False, [40, 30], [0, 1], 2, 16, 64, 72, seed=72)
    expected = case.run()
    for name in ("x", "weight", "residual", "down", "up"):
        dense = getattr(case, name)
        for strided in (torch.cat([dense, dense], -1)[..., : dense.shape[-1]], dense.transpose(0, -1).contiguous().transpose(0, -1),
                        torch.cat([dense.flatten()[:1], dense.flatten()])[1:].view(dense.shape)):
            setattr(case, name, strided)
            assert torch.equal(case.run(), expected)
        setattr(case, name, dense)
