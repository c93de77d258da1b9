"""Linears with low-rank adapters on the GPU (the fry::adapter_linear and fry::int8_adapter_linear ops) against their
definition in fp64, and a run of them with the attention as a serving step uses them.

The tolerance of one output, u = 2^-11 (half an fp16 step): the output's own rounding u |out| + 2^-25; x down^T is summed in
fp32 over K (K 2^-24 of its products' magnitudes), rounded (u of it, 2^-25 below the normal range) and meets |up|; and the
sums over K and the rank, the scales, bias and residual are fp32 (K + rank + 8 roundings of 2^-24 of all magnitudes)."""
import math

import pytest
import torch

from chess_transformer_b200 import ops
from chess_transformer_b200.build import build
from chess_transformer_b200.library import FryError, library

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


@pytest.fixture(scope="module", autouse=True)
def built():
    build()


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def offsets(lengths, first=0):
    out = [first]
    for n in lengths:
        out.append(out[-1] + n)
    return int32(out)


class Case:
    def __init__(self, int8, lengths, ids, adapters, rank, K, N, seed, bias=True, residual=True, first=0, behind=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
        self.int8, self.lengths, self.first, M = int8, lengths, first, first + sum(lengths) + behind
        self.ids, self.offsets = int32(ids), offsets(lengths, first)
        self.down, self.up = (normal(adapters, rank, K) / math.sqrt(K)).half(), (normal(adapters, N, rank) * 0.3).half()
        self.bias = normal(N).half() if bias else None
        self.residual = normal(M, N).half() if residual else None
        if int8:
            self.x = torch.randint(-127, 128, (M, K), generator=g, device="cuda", dtype=torch.int8)
            self.weight = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
            self.scales = (torch.rand(M, generator=g, device="cuda") * 0.03 + 0.001, torch.rand(N, generator=g, device="cuda") * 0.002)
        else:
            self.x, self.weight, self.scales = normal(M, K).half(), (normal(N, K) / math.sqrt(K)).half(), None

    def run(self):
        if self.int8:
            return ops.int8_adapter_linear(self.x, self.scales[0], self.weight, self.scales[1], self.bias, self.residual, self.down, self.up,
                                           self.offsets, self.ids)
        return ops.adapter_linear(self.x, self.weight, self.bias, self.residual, self.down, self.up, self.offsets, self.ids)

    def expected(self):
        x, weight = self.x.double(), self.weight.double()
        if self.int8:
            x, weight = x * self.scales[0].double()[:, None], weight * self.scales[1].double()[:, None]
        K, rank = x.shape[1], self.down.shape[1]
        out, magnitude = x @ weight.T, x.abs() @ weight.abs().T
        tolerance = torch.zeros_like(out)
        row = self.first
        for length, a in zip(self.lengths, self.ids.tolist()):
            rows, row = slice(row, row + length), row + length
            if a < 0 or a >= self.down.shape[0]:
                continue
            down, up = self.down[a].double(), self.up[a].double()
            low, low_magnitude = x[rows] @ down.T, x[rows].abs() @ down.abs().T
            out[rows] += low @ up.T
            magnitude[rows] += low.abs() @ up.abs().T
            tolerance[rows] += (U * low.abs() + 2.0 ** -25 + (K + 4) * 2.0 ** -24 * low_magnitude) @ up.abs().T * (1 + U)
        for added in (self.bias, self.residual):
            if added is not None:
                out, magnitude = out + added.double(), magnitude + added.double().abs()
        return out, (tolerance + (K + rank + 8) * 2.0 ** -24 * magnitude) * (1 + U) + U * out.abs() + 2.0 ** -25

    def check(self, found=None, rows=slice(None)):
        found = (self.run() if found is None else found)[rows]
        expected, tolerance = (t[rows] for t in self.expected())
        off = (found.double() - expected).abs() - tolerance
        assert off.numel() == 0 or off.max() <= 0, off.max()


SHAPES = [  # lengths, ids, adapters, rank, K, N
    ([1], [0], 1, 8, 16, 8),
    ([5], [-1], 1, 16, 64, 24),
    ([70, 0, 1, 127, 130], [2, 1, 0, -1, 2], 3, 16, 768, 1440),
    ([1] * 40, [i % 7 - 1 for i in range(40)], 6, 24, 256, 200),
    ([70] * 64, [i % 9 - 1 for i in range(64)], 8, 8, 768, 1152),
    ([300, 17, 900], [0, 1, 2], 3, 64, 528, 328),
    ([200, 3], [1, 0], 2, 128, 400, 136),
    ([64, 64, 128, 256, 512], [0, 1, 2, 3, -1], 4, 72, 128, 256),
    ([3000, 2500], [1, 0], 2, 32, 256, 2304),        # fp16: pairs of 256-row tiles
    ([37] * 150, [i % 11 - 1 for i in range(150)], 10, 40, 128, 2056),
    ([1] * 32, [i % 20 - 1 for i in range(32)], 20, 16, 2048, 2040),
    ([1] * 33, [i % 20 - 1 for i in range(33)], 20, 128, 1040, 264),
    ([17, 0, 14], [1, 0, 1], 2, 64, 4096, 40),
    ([2] * 300, [i % 290 for i in range(300)], 290, 8, 64, 72),
]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("bias, residual", [(True, True), (False, False)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_the_linear_with_adapters_is_its_definition(shape, bias, residual, int8):
    Case(int8, *SHAPES[shape], seed=shape, bias=bias, residual=residual).check()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("M", [2, 90, 6000])
def test_rows_of_no_request_have_no_adapter(M, int8):
    Case(int8, [M, 7], [1, 0], 2, 16, 64, 2304, seed=20, first=13, behind=150).check()
    Case(int8, [], [], 2, 16, 64, 2304, seed=20, behind=M).check()


def test_empty_calls_and_leading_axes():
    for int8 in (False, True):
        assert Case(int8, [], [], 1, 8, 32, 16, seed=21).run().shape == (0, 16)
        assert Case(int8, [0, 0], [0, 0], 1, 8, 32, 16, seed=21).run().shape == (0, 16)
        flat = Case(int8, [70, 70], [0, 1], 2, 8, 32, 16, seed=22)
        expected = flat.run()
        flat.x, flat.residual = flat.x.view(2, 70, 32), flat.residual.view(2, 70, 16)
        assert torch.equal(flat.run(), expected.view(2, 70, 16))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("N", [136, 2304])
def test_an_adapter_reaches_its_own_requests_alone(N, bad, int8):
    case = Case(int8, [30, 40, 100, 1900], [0, 1, -1, 2], 4, 16, 64, N, seed=23)
    clean = case.expected()
    case.up[1, 5, 3] = bad          # one column of request 1's
    case.up[2, :, 0] = bad          # all of request 3's
    case.up[3] = bad                # nobody's
    case.down[3] = bad
    found = case.run()
    rows = slice(70, 170)
    for part in (slice(0, 30), rows):
        assert ((found[part].double() - clean[0][part]).abs() <= clean[1][part]).all()
    assert not torch.isfinite(found[30:70, 5]).any() and not torch.isfinite(found[170:]).any()
    others = [c for c in range(N) if c != 5]
    assert ((found[30:70, others].double() - clean[0][30:70, others]).abs() <= clean[1][30:70, others]).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("int8", [False, True])
def test_an_adapter_reaches_its_own_single_row_alone(int8, bad):
    case = Case(int8, [1] * 9, [0, 1, -1] * 3, 2, 16, 64, 136, seed=33)
    clean = case.expected()
    case.up[1, 5, 3], case.down[1, 2, 1] = bad, bad
    found = case.run()
    others = [m for m in range(9) if m % 3 != 1]
    assert ((found[others].double() - clean[0][others]).abs() <= clean[1][others]).all()
    assert not torch.isfinite(found[1::3]).any()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("ids, bad_offsets", [([0, 2, 1], None), ([0, -2, 1], None), ([0, 1, 2 ** 31 - 1], None), ([0, 1, 1], [0, 200, 100, 300]),
                                              ([0, 1, 1], [0, 100, 200, 301]), ([0, 1, 1], [-5, 100, 200, 300])])
def test_ids_and_offsets_out_of_range_are_recorded(ids, bad_offsets, int8):
    lib = library()
    lib.device_status(clear=True)
    case = Case(int8, [100, 100, 100], ids, 2, 16, 64, 72, seed=24)
    if bad_offsets:
        case.offsets = int32(bad_offsets)
        case.run()
    else:
        case.check()  # as without an adapter
    assert lib.device_status(clear=True)[0] == 7
    Case(int8, [100, 100, 100], [0, 1, -1], 2, 16, 64, 72, seed=25).check()
    assert lib.device_status()[0] == 0


@pytest.mark.parametrize("int8", [False, True])
def test_recorded_into_two_graphs_on_a_side_stream(int8):
    cases = [Case(int8, [70, 1, 400], [0, 1, -1], 2, 16, 64, 72, seed=26), Case(int8, [3000, 5], [1, 0], 2, 32, 128, 2304, seed=27)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(stream):
        for case in cases:
            case.run()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(case.run())
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(3):
        for case in cases:  # other rows, and other adapters for the same requests
            case.x.copy_(case.x.flip(0))
            case.ids.copy_(case.ids.flip(0))
        for graph in graphs:
            graph.replay()
        for case, out in zip(cases, outs):
            case.check(out)
            assert torch.equal(out, case.run())


def test_two_streams_at_once():
    """Calls that overlap on the GPU have workspaces of their own."""
    cases = [Case(int8, [70] * 40 + [900], [i % 4 - 1 for i in range(41)], 3, 16, 768, 1440, seed=40 + i) for i, int8 in enumerate((False, True))]
    q = torch.randn(3, 8, 64, device="cuda").half()
    cache = torch.randn(3, 4000, 2, 64, device="cuda").half()
    lengths = int32([4000, 17, 2500])
    expected = [case.run() for case in cases] + [ops.cached_attention(q, cache, cache, lengths)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    found = [[], []]
    for _ in range(20):
        for stream, outs in zip(streams, found):
            with torch.cuda.stream(stream):
                outs.append([case.run() for case in cases] + [ops.cached_attention(q, cache, cache, lengths)])
    torch.cuda.synchronize()
    assert all(torch.equal(out, right) for outs in found for call in outs for out, right in zip(call, expected))


def test_the_same_call_gives_the_same_bits():
    for int8 in (False, True):
        case = Case(int8, [70] * 30, [i % 5 - 1 for i in range(30)], 4, 16, 768, 1440, seed=28)
        first = case.run()
        assert all(torch.equal(first, case.run()) for _ in range(20))


def test_under_torch_compile():
    case = Case(False, [70, 3], [0, 1], 2, 8, 64, 72, seed=29)
    compiled = torch.compile(lambda x: ops.adapter_linear(x * 2, case.weight, None, None, case.down, case.up, case.offsets, case.ids) + 1,
                             fullgraph=True, backend="eager")
    eager = ops.adapter_linear(case.x * 2, case.weight, None, None, case.down, case.up, case.offsets, case.ids) + 1
    assert torch.equal(compiled(case.x), eager)


def test_without_adapters_it_is_the_linear():
    case = Case(True, [70] * 64, [-1] * 64, 1, 8, 768, 1152, seed=30, residual=False)
    assert torch.equal(case.run(), ops.int8_linear(case.x, case.scales[0], case.weight, case.scales[1], case.bias, None, False, "projection"))


def test_refusals():
    case = Case(False, [6], [0], 1, 8, 64, 72, seed=31)
    args = [case.x, case.weight, case.bias, case.residual, case.down, case.up, case.offsets, case.ids]
    for at, value, match in [(0, case.x.float(), "x must be"), (1, case.weight.bfloat16(), "weight must be"), (1, case.weight[:, :32], "K"),
                             (2, case.bias[:8], "bias must be"), (3, case.residual[:5], "residual must be"), (4, case.down[:, :4], "down"),
                             (5, case.up.bfloat16(), "up must be"), (6, case.offsets.long(), "int32"), (6, case.offsets[:1], "int32"),
                             (7, case.ids.cpu(), "another operand"), (7, case.ids[None], "int32")]:
        with pytest.raises(FryError, match=match):
            ops.adapter_linear(*args[:at], value, *args[at + 1:])
    with pytest.raises(FryError, match="rank"):
        ops.adapter_linear(*args[:4], case.down[:, :4].contiguous(), case.up[:, :, :4].contiguous(), *args[6:])
    with pytest.raises(FryError, match="1 or more adapters"):
        ops.adapter_linear(*args[:4], case.down[:0], case.up[:0], *args[6:])
    case = Case(True, [6], [0], 1, 8, 64, 72, seed=31)
    with pytest.raises(FryError, match="scale a row"):
        ops.int8_adapter_linear(case.x, case.scales[0][:5], case.weight, case.scales[1], None, None, case.down, case.up, case.offsets, case.ids)


def test_a_serving_step_with_an_adapter_a_request():
    """Prompts of several requests through one layer: projections with each request's adapters, causal attention within each
    request, the output linear with the residual; then each request's next token over the cache the prompts left."""
    heads, kv_heads, width, d = 12, 4, 64, 768
    lengths, ids, capacity = [70, 1, 33, 200], [1, -1, 0, 1], 256
    g = torch.Generator(device="cuda").manual_seed(32)
    normal = lambda *shape, scale=1.0: (torch.randn(*shape, generator=g, device="cuda") * scale).half()  # noqa: E731
    columns = (heads + 2 * kv_heads) * width
    qkv, qkv_down, qkv_up = normal(columns, d, scale=d ** -0.5), normal(2, 16, d, scale=d ** -0.5), normal(2, columns, 16, scale=0.2)
    out, out_down, out_up = normal(d, d, scale=d ** -0.5), normal(2, 8, d, scale=d ** -0.5), normal(2, d, 8, scale=0.2)
    x, token, at, one = normal(sum(lengths), d), normal(len(lengths), d), offsets(lengths), offsets([1] * len(lengths))

    def layer(rows, where, attend):
        q, k, v = (t.unflatten(1, (-1, width)) for t in ops.adapter_linear(rows, qkv, None, None, qkv_down, qkv_up, where, int32(ids)).split(
            [heads * width, kv_heads * width, kv_heads * width], 1))
        return ops.adapter_linear(attend(q, k, v).flatten(1), out, None, rows, out_down, out_up, where, int32(ids))

    cache = torch.full((2, len(lengths), capacity, kv_heads, width), math.nan, device="cuda", dtype=torch.float16)

    def prompt(q, k, v):
        for s, n in enumerate(lengths):
            cache[0, s, :n], cache[1, s, :n] = k[at[s]:at[s + 1]], v[at[s]:at[s + 1]]
        return ops.packed_attention(q, k, v, at, at)

    def step(q, k, v):
        for s, n in enumerate(lengths):
            cache[0, s, n], cache[1, s, n] = k[s], v[s]
        return ops.cached_attention(q, cache[0], cache[1], int32([n + 1 for n in lengths]))

    first, second = layer(x, at, prompt), layer(token, one, step)
    for s, (n, a) in enumerate(zip(lengths, ids)):
        rows = torch.cat([x[at[s]:at[s + 1]], token[s:s + 1]]).double()  # the prompt and its next token at once
        linear = lambda r, w, down, up: r @ (w.double() + (up[a].double() @ down[a].double() if a >= 0 else 0)).T  # noqa: E731
        q, k, v = (t.unflatten(1, (-1, width)) for t in linear(rows, qkv, qkv_down, qkv_up).split([heads * width, kv_heads * width, kv_heads * width], 1))
        k, v = (t.repeat_interleave(heads // kv_heads, 1) for t in (k, v))
        scores = torch.einsum("ihd,jhd->hij", q, k) * width ** -0.5
        p = torch.softmax(scores.masked_fill(~torch.ones(n + 1, n + 1, dtype=torch.bool, device="cuda").tril(), -math.inf), -1)
        expected = rows + linear(torch.einsum("hij,jhd->ihd", p, v).flatten(1), out, out_down, out_up)
        found = torch.cat([first[at[s]:at[s + 1]], second[s:s + 1]]).double()
        # four fp16 roundings (q|k|v, p, the attention's output, the layer's), each half a step of values of order 1, through
        # a softmax of scores of order 1: their sum in the 2-norm is below ten half steps
        assert (found - expected).norm() <= 10 * U * expected.norm()
