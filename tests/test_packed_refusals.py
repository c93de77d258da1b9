"""What the packed operators refuse on the host, and the search that gives requests their tiles, on the CPU."""
import ctypes
import random

import pytest
import torch

from chess_transformer_b200 import ops
from chess_transformer_b200.build import build
from chess_transformer_b200.library import FryError, library


@pytest.fixture(scope="module")
def lib():
    build()
    return library()


def packed(lib, q_rows=4, k_rows=4, sequences=1, heads=4, kv_heads=2, width=64, strides=(256, 64, 128, 64, 128, 64), scale=0.125, q=16, out=16,
           offsets=16, workspace=None, size=0):
    pointer = ctypes.c_void_p
    return lib.fry_packed_attention(pointer(q), pointer(16), pointer(16), pointer(out), pointer(offsets), pointer(16), q_rows, k_rows, sequences, heads,
                                    kv_heads, width, *strides, scale, 1, 0, pointer(workspace), size, None)


@pytest.mark.parametrize("arguments, match", [
    ({"heads": 3}, "multiple of the key/value heads"), ({"kv_heads": 0}, "query heads"), ({"heads": 2048, "kv_heads": 1}, "1024"),
    ({"width": 12}, "multiple of 8"), ({"width": 136}, "up to 128"), ({"width": 0}, "up to 128"), ({"q_rows": -1}, ">= 0"), ({"sequences": -1}, ">= 0"),
    ({"scale": 0.0}, "positive"), ({"scale": -1.0}, "positive"), ({"scale": float("nan")}, "positive"), ({"scale": float("inf")}, "positive"),
    ({"strides": (256, 64, 128, 60, 128, 64)}, "strides"), ({"strides": (-256, 64, 128, 64, 128, 64)}, "strides"), ({"q": 24}, "16-byte"),
    ({"offsets": None}, "offsets"), ({"out": None}, "needs q"), ({"sequences": 1 << 27}, "2\\^24"), ({"k_rows": (1 << 30) + 1}, "2\\^30"),
    ({"scale": 3e38}, "2e38"),
    ({"q_rows": 2, "k_rows": 100000, "workspace": 16, "size": 8}, "workspace"), ({"q_rows": 2, "k_rows": 100000}, "workspace"),
])
def test_packed_attention_refuses(lib, arguments, match):
    with pytest.raises(FryError, match=match):
        packed(lib, **arguments)


def test_calls_without_rows_do_nothing(lib):
    assert packed(lib, q_rows=0) == 0


def test_workspaces_are_sized_by_the_shape(lib):
    assert lib.fry_packed_attention_workspace_bytes(8192, 8192, 1, 32, 4, 128) == 0
    one = lib.fry_packed_attention_workspace_bytes(1, 32768, 1, 32, 4, 128)
    assert one > 0 and one % (32 * 130 * 4) == 0
    assert lib.fry_cached_attention_workspace_bytes(1, 32768, 32, 4, 128) == one
    assert lib.fry_packed_attention_workspace_bytes(1, 32768, 1, 32, 5, 128) == 0  # a refused shape


def test_every_shape_has_a_plan(lib):
    """Fewer rows than sequences, none, or one of many keys: the choice of kernel and splits divides by none of them."""
    for rows in (0, 1, 3, 200, 100000):
        for keys in (0, 1, 127, 128, 5000, 1 << 20):
            for sequences in (0, 1, 7, 5000):
                for heads, kv_heads in ((1, 1), (24, 12), (130, 1)):
                    assert lib.fry_packed_attention_workspace_bytes(rows, keys, sequences, heads, kv_heads, 64) >= 0


def test_cpu_tensors_are_refused():
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    at = torch.tensor([0, 3], dtype=torch.int32)
    with pytest.raises(FryError, match="GPU only"):
        ops.packed_attention(q, q, q, at, at)
    with pytest.raises(FryError, match="GPU only"):
        ops.cached_attention(q, q[None], q[None], at)


def find_segment(starts, tile, slot):
    """csrc/segments.cuh's search, lane by lane."""
    low, count = 0, len(starts) - 1
    while count > 1:
        step = (count + 31) // 32
        reached = [lane for lane in range(32) if lane * step < count and starts[low + lane * step] // tile + low + lane * step <= slot]
        last = max(reached, default=0)
        low += last * step
        count = min(step, count - last * step)
    return low


def test_every_tile_has_one_slot():
    rng = random.Random(0)
    for _ in range(300):
        tile, requests = rng.choice([1, 2, 5, 16, 64, 128]), rng.choice([0, 1, 2, 7, 40, 1100])
        lengths = [rng.choice([0, 1, tile - 1, tile, tile + 1, rng.randrange(300)]) for _ in range(requests)]
        starts = [0, rng.choice([0, 3])]
        for n in lengths:
            starts.append(starts[-1] + n)
        rows = starts[-1] + rng.choice([0, 9])
        starts.append(rows)
        seen = []
        for slot in range(rows // tile + requests + 2):
            i = find_segment(starts, tile, slot)
            first = (slot - starts[i] // tile - i) * tile
            seen += range(starts[i] + first, min(starts[i] + first + tile, starts[i + 1]))
        assert seen == list(range(rows))


def test_descending_starts_end_the_search_in_range():
    rng = random.Random(1)
    for _ in range(300):
        starts = [0] + [rng.randrange(500) for _ in range(rng.choice([1, 5, 40, 1100]))] + [500]
        assert all(0 <= find_segment(starts, 16, slot) <= len(starts) - 2 for slot in range(0, 500, 7))


def adapters(lib, int8, M=4, N=16, K=32, requests=1, adapters=1, rank=8, x=16, scale=16, offsets=16, workspace=16, size=1 << 20):
    pointer = ctypes.c_void_p
    if int8:
        return lib.fry_int8_adapter_linear(pointer(x), pointer(scale), pointer(16), pointer(scale), None, None, pointer(16), pointer(16), pointer(offsets),
                                           pointer(16), pointer(16), M, N, K, requests, adapters, rank, pointer(workspace), size, None)
    return lib.fry_adapter_linear(pointer(x), pointer(16), None, None, pointer(16), pointer(16), pointer(offsets), pointer(16), pointer(16), M, N, K,
                                  requests, adapters, rank, pointer(workspace), size, None)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("arguments, match", [
    ({"N": 12}, "multiple of 8"), ({"N": 0}, "multiple of 8"), ({"K": 20}, "K of"), ({"rank": 4}, "rank"), ({"rank": 136}, "rank"), ({"rank": 0}, "rank"),
    ({"M": 1 << 23, "requests": (1 << 24) - 1, "size": 1 << 50}, "fewer requests"), ({"adapters": 0}, "1 or more"), ({"adapters": 1 << 28}, "2\\^31"), ({"M": -1}, "rows"), ({"requests": -1}, "requests"), ({"x": 8}, "16-byte"),
    ({"x": None}, "needs x"), ({"offsets": None}, "offsets"), ({"workspace": None}, "workspace"), ({"size": 100}, "workspace"),
])
def test_linears_with_adapters_refuse(lib, int8, arguments, match):
    with pytest.raises(FryError, match=match):
        adapters(lib, int8, **arguments)


def test_the_int8_linear_with_adapters_needs_its_scales(lib):
    with pytest.raises(FryError, match="both scales"):
        adapters(lib, True, scale=None)


def test_linears_with_adapters_take_no_rows(lib):
    assert adapters(lib, False, M=0) == adapters(lib, True, M=0) == 0
    x = torch.zeros(3, 64, dtype=torch.float16)
    with pytest.raises(FryError, match="GPU only"):
        ops.adapter_linear(x, x, None, None, x[None], x[None], torch.tensor([0, 3], dtype=torch.int32), torch.tensor([0], dtype=torch.int32))
