"""Attention over many keys on the GPU, where single keys decide the answer: one key of a sequence is aligned with the
queries so that its softmax weight is all but 1, and its value is recognisable. Wherever it lies (the first and the last key,
both sides of a stage, a tile and a split, both sides of each 2^31 elements of the cache), a key that is dropped, read from a
wrong place or taken twice shows, as it would not among thousands of keys of alike weights.

The planted key's score is `margin` above the others', whose weights are below n e^-margin in all: with margin 30 and n up to
2^21 below 2e-7. The answer is then the planted value to u |v| of its rounding, u |v| of its probability's, and n e^-margin of
(|v| + the largest other value)."""
import math

import pytest
import torch

from chess_transformer_b200 import ops
from chess_transformer_b200.build import build

pytestmark = pytest.mark.gpu
MARGIN = 30.0


@pytest.fixture(scope="module", autouse=True)
def built():
    build()


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def queries(rows, heads, width, dtype):
    """Each row of the same sign pattern for all heads of a group: q . k is width * |k| for a key of the same signs."""
    signs = torch.where(torch.arange(width, device="cuda") % 3 == 0, -1.0, 1.0)
    return signs.expand(rows, heads, width).contiguous().to(dtype), signs.to(dtype)


def planted_value(kv_heads, width, dtype, salt):
    at = torch.arange(kv_heads * width, device="cuda").view(kv_heads, width)
    return (((at * 7 + salt * 13) % 61 - 30) / 16).to(dtype)  # exact in fp16 and bf16


def check(found, value, group, count):
    """found [heads, width] against the planted value [kv_heads, width]; the other values are 0 to 1."""
    value, u = value.double().repeat_interleave(group, 0), torch.finfo(found.dtype).eps / 2
    others = count * math.exp(-MARGIN)
    tolerance = 2 * u * (1 + u) * value.abs() + 2 * others * (value.abs() + 1)
    # answers of nothing, or of the other keys alone, lie far outside
    assert tolerance.max() < 0.02 * value.abs().amax()
    assert ((found.double() - value).abs() <= tolerance).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads, kv_heads, width", [(8, 2, 128), (4, 4, 64), (6, 1, 32), (3, 3, 24)])
@pytest.mark.parametrize("rows, keys", [(1, 5000), (1, 130), (3, 777), (40, 6500), (300, 1500), (1, 20000), (17, 33)])
def test_each_key_counts_once(rows, keys, heads, kv_heads, width, dtype):
    q, signs = queries(rows, heads, width, dtype)
    scale = MARGIN / width
    k, v = torch.zeros(keys, kv_heads, width, device="cuda", dtype=dtype), torch.rand(keys, kv_heads, width, device="cuda").to(dtype)
    places = {0, 1, keys - rows, keys // 2} | {p for edge in (16, 32, 48, 64, 128, 256, 512, 1024, 4096, 6144) for p in (edge - 1, edge)} | {
        p for part in range(1, 8) for p in (keys * part // 8 // 128 * 128 - 1, keys * part // 8 // 128 * 128)}
    for causal in (False, True):
        for place in sorted(p for p in places if 0 <= p <= keys - rows):  # all rows see it
            value = planted_value(kv_heads, width, dtype, place)
            was = v[place].clone()
            k[place], v[place] = signs, value
            found = ops.packed_attention(q, k, v, int32([0, rows]), int32([0, keys]), causal, scale)
            for row in {0, rows // 2, rows - 1}:
                check(found[row], value, heads // kv_heads, keys)
            if rows == 1:
                cached = ops.cached_attention(q, k[None], v[None], int32([keys]), scale)
                check(cached[0], value, heads // kv_heads, keys)
                if place == keys - 1:  # and with a length that ends before it, not at all
                    cached = ops.cached_attention(q, k[None], v[None], int32([keys - 1]), scale)
                    assert (cached >= 0).all() and (cached <= 1).all()
            k[place], v[place] = 0, was


def test_keys_past_32_bit_offsets_of_a_cache():
    """A cache of more than 2^32 + 2^30 elements a tensor: 5 sequences of 2^21 + 4321 keys, 4 heads of 128. Keys on both sides
    of each 2^31 elements, which lie within a sequence, and of a stage's, a split's and a sequence's ends."""
    sequences, capacity, kv_heads, width = 5, (1 << 21) + 4321, 4, 128
    row = kv_heads * width
    q, signs = queries(sequences, 4, width, torch.float16)
    k = torch.zeros(sequences, capacity, kv_heads, width, device="cuda", dtype=torch.float16)
    v = torch.full_like(k, 0.5)
    keys = [k.view(-1, kv_heads, width), v.view(-1, kv_heads, width)]
    crossing = (1 << 31) // row  # rows of 2^31 elements
    rounds = [[crossing * i + offset for i in (1, 2)] for offset in (-1, 0, 1)] + [
        [capacity * s + place for s in range(sequences)] for place in (0, 1, 127, 128, capacity // 2, capacity - 129, capacity - 1)]
    lengths = int32([capacity] * sequences)
    for places in rounds:
        by_sequence = {}
        for salt, place in enumerate(places):  # one a sequence
            by_sequence[place // capacity] = (place, planted_value(kv_heads, width, torch.float16, salt + 1))
        for place, value in by_sequence.values():
            keys[0][place], keys[1][place] = signs, value
        found = ops.cached_attention(q, k, v, lengths, MARGIN / width)
        packed = ops.packed_attention(q, *keys, int32(list(range(sequences + 1))), int32([capacity * s for s in range(sequences + 1)]), True, MARGIN / width)
        for s, (place, value) in by_sequence.items():
            check(found[s], value, 1, capacity)
            check(packed[s], value, 1, capacity)
        for s in set(range(sequences)) - set(by_sequence):  # nothing planted: the mean of the others
            assert ((found[s].double() - 0.5).abs() <= 2.0 ** -10).all() and ((packed[s].double() - 0.5).abs() <= 2.0 ** -10).all()
        for place, _ in by_sequence.values():
            keys[0][place], keys[1][place] = 0, 0.5


def test_rows_past_32_bit_offsets_of_a_prompt():
    """The same through the prompt kernel: the last of 2^21 key rows of 8 heads of 256 elements apart, 2^32 elements a tensor."""
    rows, kv_heads, width, count = 300, 8, 128, 1500
    total = 1 << 21
    wide_k = torch.zeros(total, kv_heads, 2 * width, device="cuda", dtype=torch.float16)
    k, v = wide_k[:, :, :width], wide_k[:, :, width:]  # k beside v, strides of 2048 elements a row
    v[-count - 200:] = 0.5
    q, signs = queries(rows, kv_heads, width, torch.float16)
    at, k_at = int32([0, rows, rows]), int32([total - count - 100, total - 100, total])
    for place in (total - count - 100, total - count - 99, total - 900, total - 100 - rows, total - 100 - rows - 1):
        value = planted_value(kv_heads, width, torch.float16, place % 97)
        k[place], v[place] = signs, value
        found = ops.packed_attention(q, k, v, at, k_at, True, MARGIN / width)
        for row in (0, 150, rows - 1):
            check(found[row], value, 1, count)
        k[place], v[place] = 0, 0.5
