"""Packed and cached attention on the GPU (the fry::packed_attention and fry::cached_attention ops) against the softmax's
definition in fp64.

The tolerance of one output, from u = eps / 2 of its type: each probability is rounded once (u of it), so their sum with
the values is off by u W, W = sum p |v| / sum p; the output is rounded once (u |out|); a score, a sum of `width` products in
fp32, is off by (width + 2) 2^-24 sum |q k| scale, which moves a probability and the sum it is divided by by that much each;
the exponentials and the fp32 sums over n keys by (n + 8) 2^-24 of W at most; and an fp16 probability below its normal range
by 2^-25, n of them of the largest |v| (their sum is at least 1)."""
import math

import pytest
import torch

from chess_transformer_b200 import ops
from chess_transformer_b200.build import build
from chess_transformer_b200.library import FryError, library

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def built():
    build()


def offsets(lengths, first=0):
    out = [first]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def one_sequence(q, k, v, causal, scale):
    """(out, tolerance) in fp64 of one sequence: q [nq, heads, width], k and v [nk, kv_heads, width]."""
    (nq, heads, width), (nk, kv_heads, _), u = q.shape, k.shape, torch.finfo(q.dtype).eps / 2
    if nk == 0:
        return torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    q, k, v = q.double(), k.double().repeat_interleave(heads // kv_heads, 1), v.double().repeat_interleave(heads // kv_heads, 1)
    seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(nk - nq)
    out, tolerance = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(nq):  # only what the query sees is read
        count = int(seen[i].sum())
        if count == 0:
            continue
        keys, values = k[:count], v[:count]
        scores = torch.einsum("hd,jhd->hj", q[i], keys) * scale
        p = torch.softmax(scores, -1)
        out[i] = torch.einsum("hj,jhd->hd", p, values)
        weight = torch.einsum("hj,jhd->hd", p, values.abs())
        products = torch.einsum("hd,jhd->hj", q[i].abs(), keys.abs()).amax(-1)[:, None] * scale
        off = 2 * (width + 2) * 2.0 ** -24 * products + (count + 8) * 2.0 ** -24
        tolerance[i] = u * out[i].abs() + (u + off) * (1 + u) * weight + count * 2.0 ** -25 * values.abs().amax(0)
    return out, tolerance


def check(found, expected, tolerance):
    assert found.shape == expected.shape
    finite = torch.isfinite(expected)
    assert torch.equal(torch.isfinite(found), finite)
    off = (found.double() - expected).abs()[finite] - tolerance[finite]
    assert off.numel() == 0 or off.max() <= 0, off.max()


def check_packed(found, q, k, v, queries, keys, causal, scale):
    q0 = k0 = 0
    for nq, nk in zip(queries, keys):
        check(found[q0:q0 + nq], *one_sequence(q[q0:q0 + nq], k[k0:k0 + nk], v[k0:k0 + nk], causal, scale))
        q0, k0 = q0 + nq, k0 + nk


def operands(queries, keys, heads, kv_heads, width, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda").to(dtype)  # noqa: E731
    return normal(sum(queries), heads, width), normal(sum(keys), kv_heads, width), normal(sum(keys), kv_heads, width)


SHAPES = [  # queries, keys (None: the queries' own), heads, kv_heads, width
    ([1], None, 1, 1, 8),
    ([70], None, 24, 12, 32),
    ([64, 0, 1, 65, 127, 128, 129], None, 4, 2, 64),
    ([3, 200, 17], None, 6, 1, 128),
    ([5, 33], None, 5, 5, 40),
    ([40, 0, 16, 9], [40, 12, 0, 130], 8, 2, 80),     # queries without keys, keys without queries
    ([20, 7], [4, 7], 3, 3, 16),                      # more queries than keys: causal, the first see none
    ([1, 1, 2, 1], [257, 1, 300, 64], 12, 3, 96),     # a few last tokens against longer keys
    ([2], [5000], 8, 1, 128),
    ([130], [1000], 2, 1, 64),
    ([9, 60], None, 40, 2, 24),                       # 20 query heads a key/value head
    ([300], None, 130, 1, 8),                         # 130 of them
    ([700, 513], None, 4, 1, 128),
    ([400], [1500], 6, 2, 128),
    ([150, 40], [7000, 6500], 8, 2, 128),
    ([600], [6200], 3, 1, 72),
    ([20], [700], 1, 1, 64),
    ([300, 310] * 10, None, 16, 8, 128),
    ([260] * 6, [6200] * 6, 32, 8, 128),
    ([1, 2, 0, 1] * 30, [200, 130, 150, 333] * 30, 8, 4, 64),
    ([1], [900], 1, 1, 24),          # 3 splits of one row: the partial results' places are odd
    ([3, 1, 1], [700, 800, 900], 1, 1, 128),
    ([47, 48, 49, 20, 30, 40, 33], [47, 48, 49, 95, 96, 97, 113], 6, 2, 32),  # keys about a stage's end
    ([20, 17, 35], [15, 47, 145], 3, 3, 24),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_packed_attention_is_the_softmax_of_each_sequence(shape, causal, dtype):
    queries, keys, heads, kv_heads, width = SHAPES[shape]
    keys = keys or queries
    q, k, v = operands(queries, keys, heads, kv_heads, width, dtype, shape)
    found = ops.packed_attention(q, k, v, offsets(queries), offsets(keys), causal)
    assert found.dtype == dtype
    check_packed(found, q, k, v, queries, keys, causal, width ** -0.5)


@pytest.mark.parametrize("scale", [0.02, 2.0])
def test_packed_attention_takes_a_scale(scale):
    q, k, v = operands([150], [150], 4, 2, 64, torch.float16, 1)
    check_packed(ops.packed_attention(q, k, v, offsets([150]), offsets([150]), True, scale), q, k, v, [150], [150], True, scale)


@pytest.mark.parametrize("queries, keys", [([150, 80], [150, 80]), ([600], [600])])
def test_scores_far_apart_and_rising(queries, keys):
    """Rows whose largest score comes last, and is far above the first ones: every running maximum is replaced."""
    q, k, v = operands(queries, keys, 2, 1, 64, torch.bfloat16, 2)
    k = k * torch.linspace(0.1, 6, k.shape[0], device="cuda")[:, None, None].to(k.dtype)
    check_packed(ops.packed_attention(q, k, v, offsets(queries), offsets(keys), False), q, k, v, queries, keys, False, 0.125)


def test_views_of_a_projection_are_read_in_place():
    queries, heads, kv_heads, width = [70, 31, 140], 8, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    rows = torch.randn(sum(queries), (heads + 2 * kv_heads) * width, generator=g, device="cuda").half()
    q, k, v = (t.unflatten(1, (-1, width)) for t in rows.split([heads * width, kv_heads * width, kv_heads * width], 1))
    at = offsets(queries)
    assert torch.equal(ops.packed_attention(q, k, v, at, at), ops.packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), at, at))
    # strides and starts that are not on 16 bytes are copied first
    odd = torch.randn(sum(queries), 8, 65, generator=g, device="cuda").half()[:, :, 1:]
    assert torch.equal(ops.packed_attention(odd, k, v, at, at), ops.packed_attention(odd.contiguous(), k, v, at, at))
    # one head of keys for all, by a stride of 0
    shared = k[:, :1].expand(-1, 2, -1)
    assert torch.equal(ops.packed_attention(q, shared, v, at, at), ops.packed_attention(q, shared.contiguous(), v, at, at))


@pytest.mark.parametrize("rows", [90, 900])
def test_rows_of_no_sequence_are_zero(rows):
    q, k, v = operands([rows], [rows], 4, 2, 64, torch.float16, 4)
    at = torch.tensor([11, rows // 2, rows - 20], dtype=torch.int32, device="cuda")
    found = ops.packed_attention(q, k, v, at, at)
    assert not found[:11].any() and not found[rows - 20:].any()
    check_packed(found[11:rows - 20], q[11:rows - 20], k[11:rows - 20], v[11:rows - 20], [rows // 2 - 11, rows - 20 - rows // 2],
                 [rows // 2 - 11, rows - 20 - rows // 2], True, 0.125)


def test_empty_calls():
    q, k, v = operands([0], [0], 4, 2, 64, torch.float16, 5)
    assert ops.packed_attention(q, k, v, offsets([0]), offsets([0])).shape == (0, 4, 64)
    assert ops.packed_attention(q, k, v, offsets([]), offsets([])).shape == (0, 4, 64)
    q, k, v = operands([7], [0], 4, 2, 64, torch.float16, 5)
    assert not ops.packed_attention(q, k, v, offsets([7]), offsets([0])).any()
    assert not ops.packed_attention(q, k, v, offsets([]), offsets([])).any()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("queries, keys", [([90, 90, 41], [90, 90, 41]), ([2, 3], [400, 333]), ([2], [2000]), ([700, 300], [700, 300]), ([300], [6500])])
def test_what_a_query_does_not_see_does_not_reach_it(queries, keys, bad, width):
    q, k, v = operands(queries, keys, 4, 2, width, torch.bfloat16, 6)
    k[keys[0] - 1, 0, 5] = bad      # the first sequence's last key and value: its last query alone sees them
    v[keys[0] - 1, 1, 7] = bad
    k[keys[0] - 1, 1] = 0
    found = ops.packed_attention(q, k, v, offsets(queries), offsets(keys))
    last = queries[0] - 1
    check(found[:last], *one_sequence(q[:last], k[:keys[0] - 1], v[:keys[0] - 1], True, width ** -0.5))
    assert not torch.isfinite(found[last, 2:, 7]).any() and torch.isfinite(found[last, 2:, 8:]).all()
    if len(queries) > 1:
        check_packed(found[queries[0]:], q[queries[0]:], k[keys[0]:], v[keys[0]:], queries[1:], keys[1:], True, width ** -0.5)


@pytest.mark.parametrize("bad_q, bad_k", [([0, 30, 20, 60], [0, 20, 40, 60]), ([0, 20, 40, 60], [0, 20, 40, 61]), ([-1, 20, 40, 60], [0, 20, 40, 60]),
                                          ([0, 20, 40, 2 ** 31 - 1], [0, 20, 40, 60]), ([0, 20, 40, 60], [0, -(2 ** 31), 40, 60])])
def test_bad_offsets_are_recorded(bad_q, bad_k):
    lib = library()
    lib.device_status(clear=True)
    q, k, v = operands([60], [60], 4, 2, 64, torch.float16, 7)
    at = [torch.tensor(o, dtype=torch.int32, device="cuda") for o in (bad_q, bad_k)]
    ops.packed_attention(q, k, v, *at)
    assert lib.device_status(clear=True)[0] == 7
    good = offsets([20, 20, 20])
    check_packed(ops.packed_attention(q, k, v, good, good), q, k, v, [20] * 3, [20] * 3, True, 0.125)
    assert lib.device_status()[0] == 0


CACHES = [  # lengths, capacity, heads, kv_heads, width
    ([1], 1, 1, 1, 8),
    ([0], 5, 2, 1, 64),
    ([70, 0, 1, 64, 65, 33, 128], 128, 24, 12, 32),
    ([5000], 5001, 8, 1, 128),
    ([2000, 17, 0, 1999], 2000, 12, 3, 96),
    ([300, 301], 400, 40, 2, 64),
    ([64] * 40, 64, 8, 8, 24),
    ([20000, 3], 20000, 16, 2, 128),
    ([600] * 50, 640, 4, 4, 128),
    ([900], 900, 1, 1, 40),          # 3 splits of one row: the partial results' places are odd
    ([1300, 7, 5], 1300, 3, 1, 8),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cache", range(len(CACHES)))
@pytest.mark.parametrize("heads_first", [False, True])
def test_cached_attention_is_the_softmax_of_each_cache(cache, dtype, heads_first):
    lengths, capacity, heads, kv_heads, width = CACHES[cache]
    S = len(lengths)
    q, k, v = operands([S], [S * capacity], heads, kv_heads, width, dtype, cache)
    k, v = k.view(S, capacity, kv_heads, width), v.view(S, capacity, kv_heads, width)
    if heads_first:
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    for s, n in enumerate(lengths):  # what lies behind a length is not read
        k[s, n:], v[s, n:] = math.nan, math.inf
    found = ops.cached_attention(q, k, v, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    for s, n in enumerate(lengths):
        check(found[s:s + 1], *one_sequence(q[s:s + 1], k[s, :n], v[s, :n], False, width ** -0.5))


def test_cached_lengths_out_of_range_are_recorded():
    lib = library()
    q, k, v = operands([3], [3 * 40], 4, 2, 64, torch.float16, 8)
    k, v = k.view(3, 40, 2, 64), v.view(3, 40, 2, 64)
    for lengths, read in (([40, 41, 3], [40, 40, 3]), ([-1, 5, 40], [0, 5, 40]), ([2 ** 31 - 1, 1, 1], [40, 1, 1])):
        lib.device_status(clear=True)
        found = ops.cached_attention(q, k, v, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        assert lib.device_status(clear=True)[0] == 7
        for s, n in enumerate(read):
            check(found[s:s + 1], *one_sequence(q[s:s + 1], k[s, :n], v[s, :n], False, 0.125))


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements, of which the last sequence's last keys lie behind them; and packed keys as far."""
    S, capacity, kv_heads, width = 9, 2 ** 21, 1, 128
    k = torch.zeros(S, capacity, kv_heads, width, device="cuda", dtype=torch.float16)
    g = torch.Generator(device="cuda").manual_seed(9)
    k[-1] = torch.randn(capacity, kv_heads, width, generator=g, device="cuda").half()
    v = k.flip(3)
    q = torch.randn(S, 2, width, generator=g, device="cuda").half()
    lengths = torch.tensor([1] * (S - 1) + [capacity], dtype=torch.int32, device="cuda")
    found = ops.cached_attention(q, k, v, lengths)
    expected, tolerance = one_sequence(q[-1:], k[-1], v[-1], False, width ** -0.5)
    check(found[-1:], expected, tolerance)
    flat = ops.packed_attention(q[-1:], k.view(-1, kv_heads, width), v.view(-1, kv_heads, width), offsets([1]),
                                torch.tensor([(S - 1) * capacity, S * capacity], dtype=torch.int32, device="cuda"))
    check(flat, expected, tolerance)


def test_packed_attention_over_one_token_each_is_cached_attention():
    lengths, capacity, heads, kv_heads, width = [50, 3, 200], 200, 8, 4, 64
    q, k, v = operands([3], [3 * capacity], heads, kv_heads, width, torch.float16, 10)
    k, v = k.view(3, capacity, kv_heads, width), v.view(3, capacity, kv_heads, width)
    packed_k, packed_v = (torch.cat([t[s, :n] for s, n in enumerate(lengths)]) for t in (k, v))
    cached = ops.cached_attention(q, k, v, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    packed = ops.packed_attention(q, packed_k, packed_v, offsets([1, 1, 1]), offsets(lengths))
    check_packed(cached, q, packed_k, packed_v, [1, 1, 1], lengths, True, 0.125)
    check_packed(packed, q, packed_k, packed_v, [1, 1, 1], lengths, True, 0.125)


@pytest.mark.parametrize("queries, keys", [([70, 3], [70, 3]), ([1, 2], [3000, 10]), ([900], [900])])
def test_recorded_into_graphs_on_a_side_stream(queries, keys):
    """Two graphs, replayed in turn on inputs that change between replays, answer as eager calls do."""
    q, k, v = operands(queries, keys, 4, 2, 64, torch.bfloat16, 11)
    at, to = offsets(queries), offsets(keys)
    lengths = torch.tensor([sum(keys)], dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(stream):
        ops.packed_attention(q, k, v, at, to)
        for call in (lambda: ops.packed_attention(q, k, v, at, to), lambda: ops.cached_attention(q[:1], k[None], v[None], lengths)):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(call())
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(stream)
    for seed in (12, 13):
        for mine, new in zip((q, k, v), operands(queries, keys, 4, 2, 64, torch.bfloat16, seed)):
            mine.copy_(new)
        for graph in graphs:
            graph.replay()
        assert torch.equal(outs[0], ops.packed_attention(q, k, v, at, to))
        assert torch.equal(outs[1], ops.cached_attention(q[:1], k[None], v[None], lengths))


def test_the_same_call_gives_the_same_bits():
    q, k, v = operands([5, 600, 64], [700, 600, 64], 8, 2, 128, torch.bfloat16, 14)
    at, to = offsets([5, 600, 64]), offsets([700, 600, 64])
    first = ops.packed_attention(q, k, v, at, to)
    assert all(torch.equal(first, ops.packed_attention(q, k, v, at, to)) for _ in range(20))


def test_under_torch_compile():
    q, k, v = operands([70, 3], [70, 3], 4, 2, 64, torch.float16, 15)
    at = offsets([70, 3])
    compiled = torch.compile(lambda q, k, v: ops.packed_attention(q * 2, k, v, at, at) + 1, fullgraph=True, backend="eager")
    assert torch.equal(compiled(q, k, v), ops.packed_attention(q * 2, k, v, at, at) + 1)


def test_refusals():
    q, k, v = operands([6], [6], 4, 2, 64, torch.float16, 16)
    at = offsets([6])
    for call, match in [
        (lambda: ops.packed_attention(q.float(), k, v, at, at), "one type"),
        (lambda: ops.packed_attention(q, k.bfloat16(), v, at, at), "one type"),
        (lambda: ops.packed_attention(q[:, :3], k, v, at, at), "multiple of kv_heads"),
        (lambda: ops.packed_attention(q, k, v[:5], at, at), "key rows"),
        (lambda: ops.packed_attention(q, k, v, at.long(), at), "int32"),
        (lambda: ops.packed_attention(q, k, v, at, offsets([3, 3])), "int32"),
        (lambda: ops.packed_attention(q, k, v, at.cpu(), at), "on cuda"),
        (lambda: ops.packed_attention(q, k, v, at, at, True, 0.0), "positive"),
        (lambda: ops.packed_attention(q, k, v, at, at, True, math.inf), "positive"),
        (lambda: ops.packed_attention(q[..., :12], k[..., :12], v[..., :12], at, at), "multiple of 8"),
        (lambda: ops.packed_attention(*(t.repeat(1, 1, 3) for t in (q, k, v)), at, at), "up to 128"),
        (lambda: ops.cached_attention(q, k, v, at), "capacity"),
        (lambda: ops.cached_attention(q[:1], k[None], v[None], at), "int32"),
    ]:
        with pytest.raises(FryError, match=match):
            call()
