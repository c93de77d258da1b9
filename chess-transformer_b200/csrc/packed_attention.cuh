// Attention over packed sequences and over a cache: out = softmax(scale q k^T) v for each token and head, grouped heads
// (query head h reads key/value head h / group), causal or not. What the kernels of packed_attention.cu and
// prompt_attention.cu share.
//
//  packed: q [rows, heads, width], k and v [key rows, kv_heads, width], sequences one behind the other at q_offsets and
//          k_offsets. Causal: a sequence's queries are its last tokens, query i sees keys j <= i + nk - nq.
//  cached: q [sequences, heads, width], one token a sequence, k and v [sequences, capacity, kv_heads, width] of which the
//          first lengths[s] keys count.
//
// Softmax in one pass over the keys: with m the running maximum of a row's scores (times scale log2 e) and l the running
// sum of 2^(s - m), a tile of keys takes m to m' = max(m, its maximum), scales l and the row's sums o by 2^(m - m') and
// adds its own 2^(s - m') and 2^(s - m') v. out = o / l at the end; a row that sees no key has l = 0 and answers 0. Scores,
// m, l and o are fp32. The probabilities 2^(s - m') are rounded to the inputs' type for the second product (off by at most half a
// step each, about what rounding the output costs), l sums them unrounded.
//
// Rows. The `group` query heads of a key/value head share its keys, so they are rows of one tile: row r of a block is token
// r / group, head r % group, and one pass over the keys serves them all.
//
// What a query does not see does not reach it, whatever it holds: scores behind a row's last key count as -inf however
// they came out, and rows behind a sequence's last key are read as zeros. A value of a key that some rows of a tile see
// and others do not is multiplied by their probability 0; if it is not finite that product is NaN, so rows whose sum l is
// finite and whose output is not are looked at again (repair_rows).
#pragma once

#include <climits>

#include "common.cuh"
#include "kernels.h"
#include "segments.cuh"

namespace fry {

struct AttentionArgs {
    const uint16_t *q = nullptr, *k = nullptr, *v = nullptr;
    uint16_t* out = nullptr;                                         // [rows, heads, width] dense
    int64_t q_row = 0, q_head = 0, k_row = 0, k_head = 0, v_row = 0, v_head = 0;  // strides in elements
    int64_t k_sequence = 0, v_sequence = 0;                        // cached
    int heads = 0, kv_heads = 0, width = 0;
    int group = 1, tile_heads = 1, head_tiles = 1;  // query heads a key/value head, of which a block takes tile_heads in each of head_tiles
    int heads_inverse = 0;                // ceil(2^16 / tile_heads): a tile's row r is token (r heads_inverse) >> 16 (exact below 2^16 / tile_heads rows)
    FRY_DEVICE int token_of(int r) const { return (r * heads_inverse) >> 16; }
    FRY_DEVICE int head_in_tile(int r) const { return r - token_of(r) * tile_heads; }
    TileRows slot_tokens{1};            // the tokens of a slot
    void set_tile(int rows, int tiles = 1) {  // as many query heads as a tile of `rows` rows takes, `tiles` tiles a slot
        tile_heads = group < rows ? group : rows;
        head_tiles = (group + tile_heads - 1) / tile_heads;
        heads_inverse = (65536 + tile_heads - 1) / tile_heads;
        slot_tokens = TileRows(tiles * (rows / tile_heads));
    }
    PackedRows queries{};                // packed; cached: count sequences of one row
    const int32_t* k_offsets = nullptr;          // packed: [count + 1]
    int k_rows = 0;
    const int32_t* lengths = nullptr;            // cached: [count], else null
    int capacity = 0;
    int causal = 0;
    float scale_log2 = 0.0f;                 // scale * log2(e), positive
    int splits = 1;
    float* part_out = nullptr;                   // [splits][rows][heads][width], where splits > 1
    float* part_sums = nullptr;                  // [splits][rows][heads][2]: m, l
};

// A block's rows: tokens [first, first + tokens) of a sequence of nq queries and nk keys.
struct RowBlock {
    int row;     // the first token's row of q and out
    int first, tokens, nq, nk;
    int k_first;             // packed: the row of the sequence's first key
    int64_t k_base, v_base;  // the sequence's first key and value, in elements
    FRY_DEVICE int limit(int token, int causal) const {  // how many keys a token sees
        if (!causal) return nk;
        const int seen = nk - nq + first + token + 1;
        return seen < 0 ? 0 : seen > nk ? nk : seen;
    }
};

// The rows of block `slot` of tiles of `tile` tokens; false if it has none. Every thread of the warp calls it.
FRY_DEVICE bool find_rows(const AttentionArgs& a, const TileRows& tile, int slot, int lane, RowBlock& b) {
    b.k_first = 0, b.k_base = b.v_base = 0;
    if (a.lengths) {
        if (slot >= a.queries.count) return false;
        const int length = a.lengths[slot];
        b.row = slot, b.first = 0, b.tokens = 1, b.nq = 1;
        b.nk = length < 0 ? 0 : length > a.capacity ? a.capacity : length;
        if (b.nk != length && threadIdx.x == 0) record_error(kBadOffsets, slot);
        b.k_base = slot * a.k_sequence, b.v_base = slot * a.v_sequence;
        return true;
    }
    const int segment = find_segment(a.queries, tile, slot, lane);
    const int start = a.queries.start(segment), end = a.queries.start(segment + 1);
    b.nq = end > start ? end - start : 0;
    // a sequence's last tile first: later tokens see more keys, and the longest work is best started early
    b.first = ((b.nq + tile.rows - 1) / tile.rows - 1 - (slot - tile.of(start) - segment)) * tile.rows;
    b.tokens = b.first < 0 ? 0 : min(tile.rows, b.nq - b.first);
    if (b.tokens <= 0) return false;
    b.row = start + b.first;
    b.nk = 0;
    if (segment >= 1 && segment <= a.queries.count) {  // not the rows before the first or behind the last sequence
        const PackedRows keys{a.k_offsets, a.queries.count, a.k_rows};
        const int k_start = keys.start(segment), k_end = keys.start(segment + 1);
        b.nk = k_end > k_start ? k_end - k_start : 0;
        b.k_first = k_start, b.k_base = k_start * a.k_row, b.v_base = k_start * a.v_row;
    }
    return true;
}

// Records a sequence whose offsets descend or leave their tensor. One block of a launch does it for all, the last: it has
// the rows behind the last sequence, usually none.
FRY_DEVICE void check_offsets(const AttentionArgs& a) {
    if (a.lengths || blockIdx.x != gridDim.x - 1 || blockIdx.y != 0 || blockIdx.z != 0) return;
    const PackedRows keys{a.k_offsets, a.queries.count, a.k_rows};
    for (int s = threadIdx.x; s < a.queries.count; s += blockDim.x)
        if (a.queries.bad(s + 1) || keys.bad(s + 1)) record_error(kBadOffsets, s);
}

template <bool BF16>
FRY_DEVICE float widen16(uint16_t bits) {
    if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(bits) << 16);
    else return h2f_bits(bits);
}
template <bool BF16>
FRY_DEVICE uint32_t pack16(float lo, float hi) {
    if constexpr (BF16) return pack_bf162_rn(lo, hi);
    else return pack_half2_rn(lo, hi);
}
template <bool BF16>
FRY_DEVICE void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16) mma_bf16(c, a, b0, b1);
    else mma_f16(c, a[0], a[1], a[2], a[3], b0, b1);
}

// Whether a running maximum is so large that its rounding shows in the exponentials: s - m' as one FMA of the raw score, the
// scale and m' keeps the largest score's own rounding, up to half a step of m'. Below 2^22 that is 1/4 at most and alike for
// all of a row's weights; from 2^30 on it makes the largest probability 0 or infinite. There scores are scaled and rounded
// first, as m' was. The row kernels do so for all (product2; 1%), the prompts, which it would cost 2 to 5%, ask first (1 to 2%).
// product2: in mul.rn.f32x2 and add.rn.f32x2 one behind the other the product comes out in an FMA with the sum, and a zero
// addend keeps them apart.
FRY_DEVICE uint64_t product2(uint64_t a, uint64_t b) { return fma2(a, b, pair2(0.0f, 0.0f)); }
FRY_DEVICE bool rounds_apart(float m) { return fabsf(m) >= 4194304.0f && m != -INFINITY; }

FRY_DEVICE float max3(float a, float b, float c) {
    float m;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}

// Where a row's results go: out (o / l rounded), or with splits this split's m, l and o.
struct AttentionOut {
    uint16_t* out;
    float *part_out, *part_sums;
};
FRY_DEVICE AttentionOut attention_out(const AttentionArgs& a, int split, int row, int head) {
    const int64_t at = static_cast<int64_t>(row) * a.heads + head;
    const int64_t part = static_cast<int64_t>(split) * a.queries.rows * a.heads + at;
    return {a.out + at * a.width, a.part_out + part * a.width, a.part_sums + part * 2};
}

// Four 16-bit values, 8-byte aligned.
template <bool BF16>
FRY_DEVICE float4 load4(const uint16_t* from) {
    const uint2 words = __ldg(reinterpret_cast<const uint2*>(from));
    return make_float4(widen16<BF16>(words.x & 0xffff), widen16<BF16>(words.x >> 16), widen16<BF16>(words.y & 0xffff), widen16<BF16>(words.y >> 16));
}

// What a column's values hold beside finite ones.
constexpr uint32_t kHasInf = 1, kHasMinusInf = 2, kHasNan = 4;
FRY_DEVICE uint32_t not_finite(float v) { return isfinite(v) ? 0u : isnan(v) ? kHasNan : v > 0.0f ? kHasInf : kHasMinusInf; }

// A warp's first row in its tile, and the token and head that the tile's first row has.
struct RowsAt {
    int row, token, head;
};

// Puts right the rows of a warp whose sums l are finite and whose outputs, written already, are not: bit i of `rows` for its
// row i, whose m and l lane i holds. Their tile took the keys [low, taken); row i sees those up to its limit, at most
// `high`. A value at its limit or behind that is not finite has been multiplied by 0 and made its column NaN. A row without
// such a value keeps its output, which is its own operands'. Of the others' columns, one with a seen value that is not
// finite needs no sum, since its probability is above 0: it is NaN, or the infinity of one sign that it holds. Those whose
// seen values are finite are summed again, 16 rows and 32 columns at a time on mma.sync, with 0 for every value that is not
// finite. So an overflown value costs its head passes over the values, and sums in the one tile of rows that holds a
// column's first. 4096 causal tokens, 8 heads of 128, 72 us a call: with an infinity at the first token 83 us, at the last
// 1020, in one value of 500 1050 (a row at a time in scalars 69, 23 and 20 ms). Not inlined, and with b by value, so that the
// kernels keep their registers.
template <bool BF16, int WIDTH>
__device__ __noinline__ void repair_rows(const AttentionArgs& a, RowBlock b, uint32_t rows, RowsAt at, float m, float l, int low, int high,
                                         int taken, int split) {
    __syncwarp();  // the outputs are written
    const int lane = threadIdx.x & 31;
    int token, head;
    auto limit_of = [&](int i) {
        token = at.token + a.token_of(at.row + i), head = at.head + a.head_in_tile(at.row + i);
        return max(low, min(high, b.limit(token, a.causal)));
    };
    const int fewest = __reduce_min_sync(0xffffffffu, (rows >> lane) & 1 ? limit_of(lane) : INT_MAX);
    const int kv_head = at.head / a.group;
    const uint16_t *keys = a.k + b.k_base + kv_head * a.k_head, *values = a.v + b.v_base + kv_head * a.v_head;
    const bool mine = 4 * lane < a.width;  // this lane's columns: 4 lane to 4 lane + 3
    auto values4 = [&](int j) {
        const uint2 words = __ldg(reinterpret_cast<const uint2*>(values + j * a.v_row + (mine ? 4 * lane : 0)));
        return make_float4(widen16<BF16>(words.x & 0xffff), widen16<BF16>(words.x >> 16), widen16<BF16>(words.y & 0xffff), widen16<BF16>(words.y >> 16));
    };
    int last[4] = {-1, -1, -1, -1};  // the last key of [fewest, taken) whose value is not finite
#pragma unroll 8
    for (int j = fewest; j < taken; ++j) {
        const float4 x = values4(j);
        if (!isfinite(x.x)) last[0] = j;
        if (!isfinite(x.y)) last[1] = j;
        if (!isfinite(x.z)) last[2] = j;
        if (!isfinite(x.w)) last[3] = j;
    }
    auto scan = [&](int from, int to, uint32_t (&holds)[4]) {
#pragma unroll 8
        for (int j = from; j < to; ++j) {
            const float4 x = values4(j);
            holds[0] |= not_finite(x.x), holds[1] |= not_finite(x.y), holds[2] |= not_finite(x.z), holds[3] |= not_finite(x.w);
        }
    };
    uint32_t common[4] = {0, 0, 0, 0};  // of the keys that all these rows see
    bool scanned = false;
    uint32_t sum_rows = 0, sum_lanes = 0, sums[4] = {0, 0, 0, 0};  // to be summed: rows, columns / 4; of lane's row, columns e of each 4
    for (; rows != 0; rows &= rows - 1) {
        const int i = __ffs(rows) - 1, limit = limit_of(i);
        const bool empty = __shfl_sync(0xffffffffu, l, i) == 0.0f;  // no keys: zeros
        const AttentionOut to = attention_out(a, split, b.row + token, head);
        bool reached[4], any = false;
        for (int e = 0; e < 4; ++e) reached[e] = mine && (empty || last[e] >= limit), any = any || reached[e];
        if (!__any_sync(0xffffffffu, any)) continue;
        uint32_t holds[4] = {0, 0, 0, 0};
        if (!empty) {
            if (!scanned) scan(low, fewest, common);
            scanned = true;
            for (int e = 0; e < 4; ++e) holds[e] = common[e];
            scan(fewest, limit, holds);
        }
        for (int e = 0; e < 4; ++e) {
            const bool sum = reached[e] && holds[e] == 0 && !empty;
            if (reached[e] && !sum) {
                const float value = empty ? 0.0f : holds[e] == kHasInf ? INFINITY : holds[e] == kHasMinusInf ? -INFINITY : NAN;
                if (a.splits > 1) to.part_out[4 * lane + e] = value;
                else to.out[4 * lane + e] = static_cast<uint16_t>(pack16<BF16>(value, 0.0f) & 0xffff);
            }
            const uint32_t votes = __ballot_sync(0xffffffffu, sum);
            if (votes) sum_rows |= 1u << i;
            if (lane == i) sums[e] = votes;
            sum_lanes |= votes;
        }
    }

    const int g = lane >> 2, t = lane & 3;
#pragma unroll 1
    for (int first = 0; first < 32; first += 16) {
        if (((sum_rows >> first) & 0xffffu) == 0) continue;
        const uint16_t* q[2];
        AttentionOut to[2];
        int limit[2];
        float base[2], inverse[2];
        for (int half = 0; half < 2; ++half) {
            const int i = first + g + 8 * half;
            const float its_m = __shfl_sync(0xffffffffu, m, i), its_l = __shfl_sync(0xffffffffu, l, i);
            limit[half] = low, base[half] = 0.0f, inverse[half] = a.splits > 1 ? 1.0f : 1.0f / its_l;
            const bool summed = (sum_rows >> i) & 1;
            const int its_limit = limit_of(summed ? i : __ffs(sum_rows) - 1);  // (the others take a summed row's query, and no keys)
            q[half] = a.q + (b.row + token) * a.q_row + head * a.q_head;
            to[half] = attention_out(a, split, b.row + token, head);
            if (summed) limit[half] = its_limit, base[half] = its_m;
        }
        const int end = __reduce_max_sync(0xffffffffu, max(limit[0], limit[1]));
#pragma unroll 1
        for (int chunk = 0; chunk < WIDTH; chunk += 32) {
            if (((sum_lanes >> (chunk / 4)) & 0xffu) == 0) continue;
            float o[4][4] = {};
#pragma unroll 1
            for (int j0 = low; j0 < end; j0 += 16) {
                // every load is made, from the last key and column where its own is behind them, so that all are in flight at once
                auto key_at = [&](int j) { return j < end ? j : end - 1; };
                uint16_t bits[4][4];
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        bits[n][e] = __ldg(values + key_at(j0 + 8 * (e / 2) + 2 * t + e % 2) * a.v_row + min(chunk + 8 * n + g, a.width - 1));
                // the products' K index, 8 of a head's columns a lane and 32 columns, is assigned alike for q and k
                float s[2][4] = {};
#pragma unroll 1
                for (int w = 0; w < WIDTH; w += 32) {
                    const bool inside = w + 8 * t < a.width;
                    const int c = inside ? w + 8 * t : 0;
                    uint4 x[2], k[2];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        x[half] = __ldg(reinterpret_cast<const uint4*>(q[half] + c));
                        k[half] = __ldg(reinterpret_cast<const uint4*>(keys + key_at(j0 + 8 * half + g) * a.k_row + c));
                        if (!inside) x[half] = k[half] = make_uint4(0, 0, 0, 0);
                    }
                    const uint32_t near[4] = {x[0].x, x[1].x, x[0].y, x[1].y}, far[4] = {x[0].z, x[1].z, x[0].w, x[1].w};
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        mma16816<BF16>(s[n], near, k[n].x, k[n].y);
                        mma16816<BF16>(s[n], far, k[n].z, k[n].w);
                    }
                }
                uint32_t p[4];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int j = j0 + 8 * n + 2 * t;
                        const float even = ex2_approx_ftz(__fsub_rn(__fmul_rn(s[n][2 * half], a.scale_log2), base[half]));
                        const float odd = ex2_approx_ftz(__fsub_rn(__fmul_rn(s[n][2 * half + 1], a.scale_log2), base[half]));
                        p[2 * n + half] = pack16<BF16>(j < limit[half] ? even : 0.0f, j + 1 < limit[half] ? odd : 0.0f);
                    }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!isfinite(widen16<BF16>(bits[n][e]))) bits[n][e] = 0;
                    mma16816<BF16>(o[n], p, bits[n][0] | static_cast<uint32_t>(bits[n][1]) << 16, bits[n][2] | static_cast<uint32_t>(bits[n][3]) << 16);
                }
            }
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int half = e >> 1, c = chunk + 8 * n + 2 * t + (e & 1);  // c % 4 == 2 t % 4 + e % 2
                    const uint32_t even = __shfl_sync(0xffffffffu, sums[e & 1], first + g + 8 * half), odd = __shfl_sync(0xffffffffu, sums[2 + (e & 1)], first + g + 8 * half);
                    if (!(((t % 2 == 0 ? even : odd) >> (c / 4)) & 1)) continue;
                    if (a.splits > 1) to[half].part_out[c] = o[n][e];
                    else to[half].out[c] = static_cast<uint16_t>(pack16<BF16>(o[n][e] * inverse[half], 0.0f) & 0xffff);
                }
        }
    }
}

}  // namespace fry
