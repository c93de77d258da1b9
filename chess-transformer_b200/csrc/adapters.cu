// Low-rank adapters of many requests beside a shared linear: the rows of request s go through adapter a = ids[s] too,
//     out[m] = x[m] W^T + bias + residual[m] + (x[m] down[a]^T) up[a]^T,   down[a] [rank, K], up[a] [N, rank]
// Two kernels. adapter_low_kernel makes low[m] = x[m] down[a]^T, a thin product that reads x once and is bound by it. The
// linear's GEMM (gemm.cu) then takes low up[a]^T as further K steps of its tiles, on the tensor cores and in the same
// accumulators, so the output is written once and no second pass reads it.
//
// A tile of the GEMM may hold rows of several requests. low is therefore laid out by slots (segments.cuh): the block of a
// (tile, request) pair has the tile's rows, those of other requests zero, and the GEMM takes one step of rank columns a
// pair, low's block against up[a]'s rows. slot_adapter gives a slot's adapter (-1: none) and tile_slots a tile's slots.
// This suits requests of many rows. One row a request costs a step and a block of low each, shared adapter or not: 2048 x 2048,
// rank 16, 32 single rows (the thin kernel) 16 us, 33 26, 64 35, 128 52, 256 57, 1024 124.
//
// low's sums are fp32. The GEMM takes them rounded to fp16, as rounding the output costs: off by 2^-11 of a value from 2^-14
// on, by 2^-25 below that. Eight of a row's that hold a finite value beyond fp16 (65504) are kept in fp32 (low32), and
// kBeyondFp16 in the first's place makes the row's sums NaN, which take_sums_again makes good. Up to 32 rows take no GEMM
// and keep all of low in fp32.
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "rowops.cuh"
#include "segments.cuh"

namespace fry {

constexpr int kThinRows = 32, kThinWarps = 8;  // rows of x a block takes; its warps share K
constexpr uint16_t kBeyondFp16 = 0x7e2a;       // a NaN that no conversion gives (theirs is 0x7fff)

FRY_DEVICE void load8(const float* from, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(from)[0], b = reinterpret_cast<const float4*>(from)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// 16 bytes as fp16 pairs: 8 fp16 values, or 16 int8 values. int8 widens exactly: a byte with its sign bit flipped in the
// low bits of 1024.0's fp16 pattern is 1024 + 128 + value.
template <bool INT8>
FRY_DEVICE void widen_pairs(const uint4& raw, uint32_t* pairs) {
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (INT8) {
            const uint32_t flipped = words[i] ^ 0x80808080u;
            const __half2 offset = __floats2half2_rn(1152.0f, 1152.0f);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t biased = __byte_perm(flipped, 0x64646464u, h == 0 ? 0x4140 : 0x4342);
                const __half2 exact = __hsub2(*reinterpret_cast<const __half2*>(&biased), offset);
                pairs[2 * i + h] = *reinterpret_cast<const uint32_t*>(&exact);
            }
        } else {
            pairs[i] = words[i];
        }
    }
}

// c += a b^T, 16 rows by 8 columns over 32 int8 values
FRY_DEVICE void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A block's product of up to 32 rows of x, in `groups` of 16 (rows below `low` or from `high` on count as 0), with TILES * 8
// rows of w (those from `columns` on count as 0), K long both: the warps take runs of K in turn and leave their sums in
// partial [kThinWarps][kThinRows][TILES * 8]. A lane's MMA fragments come from 16-byte loads: of each run of K the four
// lanes of a quad read 16 (of int8 x against fp16 w, 16 and 32) bytes each, and the MMA's K index is assigned to what a lane
// holds, alike for x and w (a sum over K may take it in any order). Each block reads its x and w once, and the loads bound
// it: what a warp has in flight (kAhead runs), blocks an SM, and the search and the first load before them. Warps that
// share K rather than rows read each weight once a block (4333 rows of 2048, rank 32: 47.6 -> 17.3 us). The sums are fp32,
// of int8 x and w exact int32.
template <bool X_INT8, bool W_INT8>
using ThinSum = std::conditional_t<X_INT8 && W_INT8, int, float>;
template <bool X_INT8, bool W_INT8, int TILES, int GROUPS>
FRY_DEVICE void thin_product_of(const void* x, int first_row, int low, int high, int groups, const void* w, int columns, int K,
                                ThinSum<X_INT8, W_INT8>* partial) {
    static_assert(X_INT8 || !W_INT8, "int8 weights take int8 rows");
    constexpr int kSteps = X_INT8 ? 4 : 2;          // MMA K steps of 16 a run
    constexpr int kLane = kSteps * 4;               // K values a lane holds of a run
    constexpr int kRun = 4 * kLane;
    constexpr int kLoads = X_INT8 && !W_INT8 ? 2 : 1;
    // runs whose loads are in flight together: about 16 of 16 bytes a lane
    constexpr int kPerRun = 2 * GROUPS + kLoads * TILES, kAhead = kPerRun <= 4 ? 4 : kPerRun <= 12 ? 2 : 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint8_t* x_lane = static_cast<const uint8_t*>(x) + (static_cast<size_t>(first_row + g) * K + t * kLane) * (X_INT8 ? 1 : 2);
    const uint8_t* w_lane = static_cast<const uint8_t*>(w) + (static_cast<size_t>(g) * K + t * kLane) * (W_INT8 ? 1 : 2);
    const size_t x_step = static_cast<size_t>(K) * 8 * (X_INT8 ? 1 : 2), w_step = static_cast<size_t>(K) * 8 * (W_INT8 ? 1 : 2);
    using Sum = ThinSum<X_INT8, W_INT8>;
    struct alignas(8) Pair {
        Sum first, second;
    };
    Sum sums[GROUPS][TILES][4] = {};
    for (int run = warp * kRun; run < K; run += kThinWarps * kRun * kAhead) {
        uint4 raw[kAhead][GROUPS][2], weight[kAhead][TILES][kLoads];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int k = run + u * kThinWarps * kRun;
            const bool inside = k + t * kLane < K;
#pragma unroll
            for (int n = 0; n < TILES; ++n)
#pragma unroll
                for (int h = 0; h < kLoads; ++h)
                    weight[u][n][h] = inside && n * 8 + g < columns
                                          ? __ldg(reinterpret_cast<const uint4*>(w_lane + n * w_step + static_cast<size_t>(k) * (W_INT8 ? 1 : 2)) + h)
                                          : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < GROUPS; ++i)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int m = first_row + i * 16 + half * 8 + g;
                    raw[u][i][half] = i < groups && inside && m >= low && m < high
                                          ? *reinterpret_cast<const uint4*>(x_lane + (2 * i + half) * x_step + static_cast<size_t>(k) * (X_INT8 ? 1 : 2))
                                          : make_uint4(0, 0, 0, 0);
                }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if constexpr (W_INT8) {  // both int8: two steps of 32 a run
#pragma unroll
                for (int i = 0; i < GROUPS; ++i) {
                    if (i >= groups) break;
                    const uint4 &a0 = raw[u][i][0], &a1 = raw[u][i][1];
#pragma unroll
                    for (int n = 0; n < TILES; ++n) {
                        mma_s8(sums[i][n], a0.x, a1.x, a0.y, a1.y, weight[u][n][0].x, weight[u][n][0].y);
                        mma_s8(sums[i][n], a0.z, a1.z, a0.w, a1.w, weight[u][n][0].z, weight[u][n][0].w);
                    }
                }
            } else {
                uint32_t b[TILES][2 * kSteps];
#pragma unroll
                for (int n = 0; n < TILES; ++n)
#pragma unroll
                    for (int h = 0; h < kLoads; ++h) widen_pairs<false>(weight[u][n][h], b[n] + 4 * h);
#pragma unroll
                for (int i = 0; i < GROUPS; ++i) {
                    if (i >= groups) break;
                    uint32_t a[2][2 * kSteps];
                    widen_pairs<X_INT8>(raw[u][i][0], a[0]);
                    widen_pairs<X_INT8>(raw[u][i][1], a[1]);
#pragma unroll
                    for (int n = 0; n < TILES; ++n)
#pragma unroll
                        for (int s = 0; s < kSteps; ++s)
                            mma_f16(sums[i][n], a[0][2 * s], a[1][2 * s], a[0][2 * s + 1], a[1][2 * s + 1], b[n][2 * s], b[n][2 * s + 1]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        if (i >= groups) break;
#pragma unroll
        for (int n = 0; n < TILES; ++n)
#pragma unroll
            for (int half = 0; half < 2; ++half)
                *reinterpret_cast<Pair*>(partial + ((warp * kThinRows + i * 16 + half * 8 + g) * TILES + n) * 8 + 2 * t) = {sums[i][n][2 * half], sums[i][n][2 * half + 1]};
    }
}
template <bool X_INT8, bool W_INT8, int TILES>
FRY_DEVICE void thin_product(const void* x, int first_row, int low, int high, int groups, const void* w, int columns, int K,
                             ThinSum<X_INT8, W_INT8>* partial) {
    if (groups == 1) thin_product_of<X_INT8, W_INT8, TILES, 1>(x, first_row, low, high, 1, w, columns, K, partial);
    else thin_product_of<X_INT8, W_INT8, TILES, kThinRows / 16>(x, first_row, low, high, groups, w, columns, K, partial);
}
// The warps' sums of columns [column, column + COUNT) of a row, in the order of the warps.
template <int TILES, typename Sum, int COUNT>
FRY_DEVICE void thin_total(const Sum* partial, int row, int column, Sum (&total)[COUNT]) {
#pragma unroll
    for (int e = 0; e < COUNT; ++e) total[e] = 0;
#pragma unroll
    for (int q = 0; q < kThinWarps; ++q)
#pragma unroll
        for (int e = 0; e < COUNT; ++e) total[e] += partial[(q * kThinRows + row) * TILES * 8 + column + e];
}

// low of 32 rows of a slot and up to TILES * 8 columns of the rank.
template <bool INT8, int TILES>
__global__ void __launch_bounds__(kThinWarps * 32, TILES == 1 ? 3 : TILES <= 4 ? 2 : 1) adapter_low_kernel(const AdapterArgs p, int M, int K) {
    extern __shared__ __align__(16) float partial[];
    const int lane = threadIdx.x & 31, slot = blockIdx.x, part = blockIdx.y, rank_first = blockIdx.z * TILES * 8;
    grid_dependency_start();

    const PackedRows rows{p.offsets, p.requests, M};
    const int segment = find_segment(rows, TileRows(p.tile_rows), slot, lane);
    const int tile = slot - segment, tile_first = tile * p.tile_rows;
    const int first = max(rows.start(segment), tile_first), last = min(rows.start(segment + 1), min(M, tile_first + p.tile_rows));
    const bool request = segment >= 1 && segment <= p.requests;
    int adapter = -1;
    if (request && first < last) adapter = p.ids[segment - 1];
    const bool known = adapter >= 0 && adapter < p.adapters;
    if (part == 0 && blockIdx.z == 0) {
        if (slot == 0)  // one block records the requests that are not in range, for all
            for (int s = threadIdx.x; s < p.requests; s += kThinWarps * 32)
                if (rows.bad(s + 1) || p.ids[s] < -1 || p.ids[s] >= p.adapters) record_error(kBadOffsets, s);
        if (p.row_adapter)
            for (int m = first + threadIdx.x; m < last; m += kThinWarps * 32) p.row_adapter[m] = known ? adapter : -1;
        if (threadIdx.x == 0) {
            p.slot_adapter[slot] = known ? adapter : -1;
            if (first < last && first == tile_first) p.tile_slots[tile].x = slot;
            if (first < last && last == min(M, tile_first + p.tile_rows)) p.tile_slots[tile].y = slot + 1;
        }
    }
    if (!known) return;

    const int part_first = tile_first + part * kThinRows, columns = min(TILES * 8, p.rank - rank_first), units = columns / 8;
    const int low = max(first, part_first), high = min(last, part_first + kThinRows);  // this block's rows of the request
    uint16_t* out = p.low + (static_cast<size_t>(slot) * p.tile_rows + part * kThinRows) * p.rank + rank_first;
    if (low < high) {
        // the 16-row groups from the first with a row of the request
        const int group_first = (low - part_first) / 16, groups = (high - 1 - part_first) / 16 - group_first + 1;
        thin_product<INT8, false, TILES>(p.x, part_first + group_first * 16, low, high, groups,
                                         p.down + (static_cast<size_t>(adapter) * p.rank + rank_first) * K, columns, K, partial);
        __syncthreads();
        for (int i = threadIdx.x; i < kThinRows * units; i += kThinWarps * 32) {
            const int row = i / units, unit = i % units, m = part_first + row;
            uint4 packed = make_uint4(0, 0, 0, 0);
            if (m >= low && m < high) {
                float total[8];
                thin_total<TILES>(partial, row - group_first * 16, unit * 8, total);
                const float scale = INT8 ? p.x_scale[m] : 1.0f;
                bool beyond = false;  // finite, and infinite in fp16
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    total[e] = __fmul_rn(total[e], scale);
                    beyond = beyond || (fabsf(total[e]) >= 65520.0f && isfinite(total[e]));
                }
                if (beyond || p.row_adapter) {
                    float4* kept = reinterpret_cast<float4*>(p.low32 + static_cast<size_t>(m) * p.rank + rank_first + unit * 8);
                    kept[0] = make_float4(total[0], total[1], total[2], total[3]), kept[1] = make_float4(total[4], total[5], total[6], total[7]);
                }
                uint32_t* words = reinterpret_cast<uint32_t*>(&packed);
#pragma unroll
                for (int e = 0; e < 4; ++e) words[e] = pack_half2_rn(total[2 * e], total[2 * e + 1]);
                if (beyond) words[0] = kBeyondFp16;
            }
            if (p.row_adapter) continue;
            *reinterpret_cast<uint4*>(out + static_cast<size_t>(row) * p.rank + unit * 8) = packed;
        }
    } else if (!p.row_adapter) {  // none of its rows: zeros
        for (int i = threadIdx.x; i < kThinRows * units; i += kThinWarps * 32)
            *reinterpret_cast<uint4*>(out + static_cast<size_t>(i / units) * p.rank + i % units * 8) = make_uint4(0, 0, 0, 0);
    }
}

// The whole linear for up to 32 rows, 16 columns a block: there its weights are read once and bound it, and the tensor
// cores' 128-row tiles would be mostly empty (16 rows against 2048 x 2048 fp16 weights: 32 such tiles of 64 columns took
// 15.8 us). Each block's product of x and its 16 weight rows is this kernel's; an output then adds low . up of its row's
// adapter, rank products. The weights stream in while the kernel before this one still makes low.
template <bool INT8>
__global__ void __launch_bounds__(kThinWarps * 32) adapter_thin_kernel(const AdapterArgs p, const GemmArgs args, const void* weight, int M, int N, int K) {
    constexpr int kTiles = 2, kColumns = kTiles * 8;
    using Sum = ThinSum<INT8, INT8>;
    extern __shared__ __align__(16) uint8_t thin_smem[];
    Sum* partial = reinterpret_cast<Sum*>(thin_smem);
    const int n0 = blockIdx.x * kColumns, columns = min(kColumns, N - n0);
    thin_product<INT8, INT8, kTiles>(p.x, 0, 0, M, (M + 15) / 16, static_cast<const uint8_t*>(weight) + static_cast<size_t>(n0) * K * (INT8 ? 1 : 2), columns, K,
                                     partial);
    grid_dependency_start();  // low32 and row_adapter are made
    __syncthreads();
    for (int i = threadIdx.x; i < M * kColumns / 2; i += kThinWarps * 32) {
        const int m = i / (kColumns / 2), c = i % (kColumns / 2) * 2, n = n0 + c;
        if (c >= columns) continue;
        Sum total[2];
        float added[2] = {0.0f, 0.0f};
        thin_total<kTiles>(partial, m, c, total);
        const int adapter = p.row_adapter[m];  // (rows of offsets that descend may have none written)
        if (adapter >= 0 && adapter < p.adapters) {
            const float* low = p.low32 + static_cast<size_t>(m) * p.rank;
            const uint4* up = reinterpret_cast<const uint4*>(p.up + (static_cast<size_t>(adapter) * N + n) * p.rank);
            for (int j = 0; j < p.rank / 8; ++j) {
                float l[8], u[8];
                load8(low + 8 * j, l);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    unpack8(__ldg(up + h * (p.rank / 8) + j), u);
#pragma unroll
                    for (int e = 0; e < 8; ++e) added[h] = __fmaf_rn(l[e], u[e], added[h]);
                }
            }
        }
        float value[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float b = args.bias ? h2f_bits(args.bias[n + h]) : 0.0f;
            // as the GEMM's epilogues: the scales and bias then the adapter (int8), or the adapter in the sums then the bias
            value[h] = INT8 ? __fadd_rn(__fmaf_rn(__fmul_rn(static_cast<float>(total[h]), args.x_scale[m]), args.w_scale[n + h], b), added[h])
                            : __fadd_rn(__fadd_rn(total[h], added[h]), b);
        }
        const size_t at = static_cast<size_t>(m) * N + n;
        if (args.residual) {
            const __half2 residual = *reinterpret_cast<const __half2*>(args.residual + at);
            value[0] = __fadd_rn(value[0], __low2float(residual)), value[1] = __fadd_rn(value[1], __high2float(residual));
        }
        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(args.out) + at) = pack_half2_rn(value[0], value[1]);
    }
}

// Row m's low, in its slot, times up[.., n] of its adapter.
FRY_DEVICE float low_up(const AdapterArgs& p, const uint16_t* low, const uint16_t* up, int m) {
    float sum = 0.0f;
    for (int j = 0; j < p.rank; j += 8) {
        float l[8], u[8];
        if (low[j] == kBeyondFp16) load8(p.low32 + static_cast<size_t>(m) * p.rank + j, l);
        else unpack8(*reinterpret_cast<const uint4*>(low + j), l);
        unpack8(__ldg(reinterpret_cast<const uint4*>(up + j)), u);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __fmaf_rn(l[e], u[e], sum);
    }
    return sum;
}

// A sum that is not finite stands where no other request of the tile has an adapter that is not finite in its column and all
// of the row's low is in fp16: it is the row's own then. The others are the row's x . w (kEpiAdapterF16; a warp's 32 x 16 of
// them on mma.sync, its fragments as in thin_product_of) plus low . up of its own request. 3744 rows through 2048 x 2048, rank
// 32, 50 us a call: 86 us with an x that is not finite in every row; 1.08 ms (int8 0.27 and 0.51) with a quarter of the
// requests on a NaN adapter or with all of low beyond fp16, 79 ms when every such sum was taken again in scalars.
template <int EPI>
__device__ __noinline__ void take_sums_again(const AdapterGemmArgs& p, int m, int column, uint32_t* sums) {
    const int lane = threadIdx.x & 31, first_row = m - lane, tile_rows = p.adapters.tile_rows, tile = first_row / tile_rows, rank = p.adapters.rank;
    uint32_t bad = 0;  // of this lane's row, by column
    for (int e = 0; e < 16; ++e)
        if (m < p.M && column + e < p.N && !isfinite(__uint_as_float(sums[e]))) bad |= 1u << e;
    const int2 slots = adapter_slots(p, tile);
    uint32_t reached = 0;
    int own_slot = -1, own_adapter = 0;
    for (int slot = slots.x; slot < slots.y; ++slot) {
        const int adapter = p.adapters.slot_adapter[slot], request = slot - tile - 1;
        if (adapter < 0 || adapter >= p.adapters.adapters || request < 0 || request >= p.adapters.requests) continue;
        const bool mine = m >= p.adapters.offsets[request] && m < p.adapters.offsets[request + 1];
        if (mine) own_slot = slot, own_adapter = adapter;
        // lane i looks at half of the rank in column i % 16
        bool found = false;
        if (column + lane % 16 < p.N) {
            const uint16_t* up = p.adapters.up + (static_cast<size_t>(adapter) * p.N + column + lane % 16) * rank;
            for (int j = lane / 16 * 8; j < rank; j += 16) {
                const uint4 words = __ldg(reinterpret_cast<const uint4*>(up + j));
                for (uint32_t w : {words.x, words.y, words.z, words.w}) found = found || (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
            }
        }
        const uint32_t votes = __ballot_sync(0xffffffffu, found);
        if (!mine) reached |= (votes | votes >> 16) & 0xffffu;
    }
    const uint16_t* low = p.adapters.low + (static_cast<size_t>(own_slot < 0 ? 0 : own_slot) * tile_rows + m % tile_rows) * rank;
    if (bad && own_slot >= 0)
        for (int j = 0; j < rank; j += 8)
            if (low[j] == kBeyondFp16) reached = 0xffffu;
    const uint32_t again = bad & reached;
    if (!__any_sync(0xffffffffu, again != 0)) return;

    float total[2][2][4] = {};  // rows in two 16s, columns in two 8s
    if constexpr (EPI == kEpiAdapterF16) {
        const int g = lane >> 2, t = lane & 3;
        const uint16_t* x = static_cast<const uint16_t*>(p.adapters.x);
#pragma unroll 2
        for (int k = t * 8; k - t * 8 < p.K; k += 32) {
            uint4 a[2][2], b[2];
#pragma unroll
            for (int n = 0; n < 2; ++n)
                b[n] = k < p.K && column + n * 8 + g < p.N ? __ldg(reinterpret_cast<const uint4*>(p.weight + static_cast<size_t>(column + n * 8 + g) * p.K + k))
                                                           : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int row = first_row + i * 16 + half * 8 + g;
                    a[i][half] = k < p.K && row < p.M ? *reinterpret_cast<const uint4*>(x + static_cast<size_t>(row) * p.K + k) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    mma_f16(total[i][n], a[i][0].x, a[i][1].x, a[i][0].y, a[i][1].y, b[n].x, b[n].y);
                    mma_f16(total[i][n], a[i][0].z, a[i][1].z, a[i][0].w, a[i][1].w, b[n].z, b[n].w);
                }
        }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        // element (lane, e) is in lane (lane % 8) * 4 + e % 8 / 2, of its rows' 16 and 8
        float sum = 0.0f;
        if constexpr (EPI == kEpiAdapterF16) {
#pragma unroll
            for (int quarter = 0; quarter < 4; ++quarter) {
                const float found = __shfl_sync(0xffffffffu, total[quarter / 2][e / 8][quarter % 2 * 2 + e % 2], lane % 8 * 4 + e % 8 / 2);
                if (lane / 8 == quarter) sum = found;
            }
        }
        if (!((again >> e) & 1)) continue;
        if (own_slot >= 0)
            sum += low_up(p.adapters, low, p.adapters.up + (static_cast<size_t>(own_adapter) * p.N + column + e) * rank, m);
        sums[e] = __float_as_uint(sum);
    }
}

namespace {

constexpr int kThinMost = 32;  // rows up to which the thin kernel takes the linear

template <bool INT8, int TILES>
cudaError_t launch_low(const AdapterArgs& p, int M, int K, cudaStream_t stream) {
    constexpr int kSmem = kThinWarps * kThinRows * TILES * 8 * 4;
    auto kernel = adapter_low_kernel<INT8, TILES>;
    const cudaError_t status = ensure_smem(reinterpret_cast<const void*>(kernel), kSmem);
    if (status != cudaSuccess) return status;
    const dim3 grid(packed_slots(M, p.tile_rows, p.requests), (p.tile_rows + kThinRows - 1) / kThinRows, (p.rank + TILES * 8 - 1) / (TILES * 8));
    return launch_dependent(kernel, grid, dim3(kThinWarps * 32), kSmem, stream, p, M, K);
}

template <bool INT8>
cudaError_t low_rank_rows(const AdapterArgs& p, int M, int K, cudaStream_t stream) {
    return p.rank <= 8    ? launch_low<INT8, 1>(p, M, K, stream)
           : p.rank <= 16 ? launch_low<INT8, 2>(p, M, K, stream)
           : p.rank <= 32 ? launch_low<INT8, 4>(p, M, K, stream)
                          : launch_low<INT8, 8>(p, M, K, stream);
}

template <bool INT8>
cudaError_t launch_thin(const AdapterArgs& p, const GemmArgs& args, const void* weight, int M, int N, int K, cudaStream_t stream) {
    constexpr int kSmem = kThinWarps * kThinRows * 16 * 4;
    return launch_dependent(adapter_thin_kernel<INT8>, dim3((N + 15) / 16), dim3(kThinWarps * 32), kSmem, stream, p, args, weight, M, N, K);
}

// the row tiles the slots are laid out by: the GEMM's, or of the thin kernel's rows all
int slot_rows(int kind, int M, int N) { return M <= kThinMost ? kThinRows : adapter_tile_rows(kind, M, N); }

}  // namespace

AdapterWorkspace::AdapterWorkspace(int kind, int M, int N, int requests, int rank) : tile_rows(slot_rows(kind, M, N)) {
    const size_t tiles = (static_cast<size_t>(M) + tile_rows - 1) / tile_rows;
    auto up = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
    const bool thin = M <= kThinMost;
    slots = packed_slots(M, tile_rows, requests);
    tile_slots = thin ? 0 : up(slots * tile_rows * rank * 2);
    slot_adapter = tile_slots + up(tiles * sizeof(int2));
    low32 = slot_adapter + up(slots * sizeof(int32_t));
    row_adapter = low32 + up(static_cast<size_t>(M) * rank * sizeof(float));
    total = row_adapter + (thin ? up(M * sizeof(int32_t)) : 0);
}

cudaError_t adapter_linear(int kind, GemmArgs& gemm_args, AdapterArgs& p, const void* weight, int M, int N, int K, void* workspace, cudaStream_t stream,
                           std::string* error) {
    const AdapterWorkspace layout(kind, M, N, p.requests, p.rank);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    p.tile_rows = layout.tile_rows;
    p.low = reinterpret_cast<uint16_t*>(base);
    p.tile_slots = reinterpret_cast<int2*>(base + layout.tile_slots);
    p.slot_adapter = reinterpret_cast<int32_t*>(base + layout.slot_adapter);
    const bool thin = M <= kThinMost;
    p.low32 = reinterpret_cast<float*>(base + layout.low32);
    if (thin) p.row_adapter = reinterpret_cast<int32_t*>(base + layout.row_adapter);
    const cudaError_t status = kind == 0 ? low_rank_rows<true>(p, M, K, stream) : low_rank_rows<false>(p, M, K, stream);
    if (status != cudaSuccess) return status;
    if (thin) return kind == 0 ? launch_thin<true>(p, gemm_args, weight, M, N, K, stream) : launch_thin<false>(p, gemm_args, weight, M, N, K, stream);
    return adapter_gemm(kind, p, weight, gemm_args, static_cast<int>(layout.slots), M, N, K, stream, error);
}

}  // namespace fry
