"""Values that are not finite, on the GPU: who sees one answers it, who does not see it is not reached, and neither takes
the attention long. Against the softmax in fp64: a column of a row is NaN if a seen value is NaN or if both infinities are
seen, an infinity if values of that sign are, else the finite sum. Tolerances as in test_packed_attention_gpu.py, the term
of an fp16 probability's subnormal range for fp16 alone."""
import math

import pytest
import torch

from chess_transformer_b200 import ops
from chess_transformer_b200.build import build

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def built():
    build()


def offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def check(found, q, k, v, causal):
    """One sequence, v with values that are not finite."""
    (nq, heads, width), (nk, kv_heads, _), u, scale = q.shape, k.shape, torch.finfo(q.dtype).eps / 2, q.shape[-1] ** -0.5
    group = heads // kv_heads
    q, k, v = (t.double().transpose(0, 1) for t in (q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)))
    seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(nk - nq)
    scores = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    p = torch.softmax(scores, -1).nan_to_num(0.0)  # rows that see no key
    finite_v = torch.where(torch.isfinite(v), v, 0.0)
    holds = [seen.double() @ kind(v).double() > 0 for kind in (torch.isnan, torch.isposinf, torch.isneginf)]
    expected = p @ finite_v
    weight, count = p @ finite_v.abs(), seen.sum(-1).double()[:, None]
    products = (q.abs() @ k.abs().transpose(1, 2)).masked_fill(~seen, 0.0).amax(-1, keepdim=True) * scale if nk else 0.0
    off = 2 * (width + 2) * 2.0 ** -24 * products + (count + 8) * 2.0 ** -24
    tolerance = u * expected.abs() + (u + off) * (1 + u) * weight
    if u == 2.0 ** -11 and nk:
        tolerance = tolerance + count * 2.0 ** -25 * finite_v.abs().amax(1, keepdim=True)
    nan = holds[0] | (holds[1] & holds[2])
    expected = torch.where(holds[1], math.inf, torch.where(holds[2], -math.inf, expected))
    found = found.double().transpose(0, 1)
    assert torch.equal(torch.isnan(found), nan)
    infinite = ~nan & torch.isinf(expected)
    assert torch.equal(found[infinite], expected[infinite])
    finite = ~nan & ~infinite
    assert ((found - expected).abs()[finite] <= tolerance[finite]).all()


def plant(v):
    """In one sequence's values: what all tokens see, what none but the last ones see, and both in one column."""
    n = v.shape[0]
    if n < 2:
        return
    v[0, :, 0] = math.inf
    v[n // 2, :, 1] = -math.inf
    v[n - 1, :, 2] = math.nan
    v[0, :, 3], v[n - 1, :, 3] = math.inf, math.nan
    v[n // 3, :, 4], v[n - 1, :, 4] = math.inf, -math.inf
    v[n - 2, :, 5] = math.inf
    v[0, 0, 6], v[n - 1, 0, 6] = math.nan, math.inf
    v[n - 1, :, 7] = -math.inf


SHAPES = [  # queries, keys (None: the queries' own), heads, kv_heads, width
    ([300, 129], None, 4, 2, 64),
    ([700], None, 4, 1, 128),
    ([150, 40], [7000, 6500], 8, 2, 128),
    ([600], [6200], 3, 1, 72),
    ([130], [1000], 2, 1, 64),
    ([200, 180], [150, 140], 2, 1, 64),          # more queries than keys: causal, the first see none
    ([70, 1, 64], None, 24, 12, 32),
    ([40, 9], [40, 130], 8, 2, 80),
    ([3, 1, 1], [700, 800, 900], 1, 1, 128),
    ([1, 2, 0, 1] * 3, [200, 130, 150, 333] * 3, 8, 4, 64),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("everywhere", [False, True])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_values_that_are_not_finite_reach_those_who_see_them(shape, everywhere, causal, dtype):
    queries, keys, heads, kv_heads, width = SHAPES[shape]
    keys = keys or queries
    g = torch.Generator(device="cuda").manual_seed(shape)
    normal = lambda *size: torch.randn(*size, generator=g, device="cuda").to(dtype)  # noqa: E731
    q, k, v = normal(sum(queries), heads, width), normal(sum(keys), kv_heads, width), normal(sum(keys), kv_heads, width)
    at = torch.tensor([0] + keys).cumsum(0).tolist()
    for first, last in zip(at, at[1:]):
        plant(v[first:last])
    if everywhere:  # and one value in 500
        v[torch.rand(v.shape, generator=g, device="cuda") < 0.002] = math.inf
    found = ops.packed_attention(q, k, v, offsets(queries), offsets(keys), causal)
    q0 = 0
    for nq, first, last in zip(queries, at, at[1:]):
        check(found[q0:q0 + nq], q[q0:q0 + nq], k[first:last], v[first:last], causal)
        q0 += nq


@pytest.mark.parametrize("capacity", [40, 3000])
def test_a_cache_with_values_that_are_not_finite(capacity):
    g = torch.Generator(device="cuda").manual_seed(capacity)
    normal = lambda *size: torch.randn(*size, generator=g, device="cuda").half()  # noqa: E731
    lengths = [capacity, capacity // 2 + 1, 1, 17]
    q, k, v = normal(4, 8, 64), normal(4, capacity, 2, 64), normal(4, capacity, 2, 64)
    for s, n in enumerate(lengths):
        plant(v[s, :n])
        v[s, n:] = math.nan
    found = ops.cached_attention(q, k, v, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    for s, n in enumerate(lengths):
        check(found[s:s + 1], q[s:s + 1], k[s, :n], v[s, :n], False)


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


@pytest.mark.parametrize("queries, keys, heads, width, causal", [
    ([4096], [4096], 8, 128, True), ([4096], [4096], 8, 128, False), ([1024] * 4, [1024] * 4, 8, 64, True),
    ([64] * 64, [64] * 64, 8, 64, True), ([64] * 64, [64] * 64, 8, 64, False), ([1] * 8, [6000] * 8, 8, 128, True)])
def test_a_value_that_all_see_costs_little(queries, keys, heads, width, causal):
    """An overflown value early in each sequence makes all its rows infinite. They are right as they come out, and at most the
    values behind each tile's first row are looked at, a few times the call's own work. A row summed again alone takes its keys
    times 2 * width scalar products: for all of 4096 causal tokens of 8 heads 1.7e10, in one warp a row a hundred times the call."""
    normal = lambda n: torch.randn(n, heads, width, device="cuda").half()  # noqa: E731
    q, k, v, at, k_at = normal(sum(queries)), normal(sum(keys)), normal(sum(keys)), offsets(queries), offsets(keys)
    call = lambda: ops.packed_attention(q, k, v, at, k_at, causal)  # noqa: E731
    clean = elapsed(call)
    v[k_at[:-1].long(), :, 5] = math.inf
    taken = elapsed(call)
    print(f"{clean * 1e3:.1f} us, with the value {taken * 1e3:.1f} us")
    assert torch.isposinf(call()[:, :, 5]).all()
    assert taken <= 10 * clean + 0.1


@pytest.mark.parametrize("queries, heads, kv_heads, width", [([4096], 8, 8, 128), ([4096], 8, 2, 64), ([1024] * 4, 8, 8, 64), ([64] * 64, 8, 8, 32)])
def test_a_value_that_only_the_last_sees_costs_little(queries, heads, kv_heads, width):
    """The rows before it in its tile are summed again: 16 rows by 32 columns of a warp at once, by width * 16 + 32 * 16 products
    a key, which is a few of the passes that a warp of the same tile makes anyway, and the rest of the call does not wait."""
    normal = lambda n: torch.randn(sum(queries), n, width, device="cuda").half()  # noqa: E731
    q, k, v, at = normal(heads), normal(kv_heads), normal(kv_heads), offsets(queries)
    call = lambda: ops.packed_attention(q, k, v, at, at)  # noqa: E731
    clean, right = elapsed(call), call()
    last = at[1:].long() - 1
    v[last, :, 5] = math.nan
    taken, found = elapsed(call), call()
    print(f"{clean * 1e3:.1f} us, with the value {taken * 1e3:.1f} us")
    assert torch.isnan(found[last, :, 5]).all()
    found[last, :, 5] = right[last, :, 5]
    # the sums again are of the same rounded factors, in another order and with probabilities against the last maximum
    assert (found.double() - right.double()).abs().max() <= 4 * 2.0 ** -11 * v[torch.isfinite(v)].abs().max()
    assert taken <= 20 * clean + 0.1
