// Low-rank adapters of many requests beside a shared linear: the rows of request s go through adapter a = ids[s] too,
//     out[m] = x[m] W^T + bias + residual[m] + (x[m] down[a]^T) up[a]^T,   down[a] [rank, K], up[a] [N, rank]
// Two kernels. adapter_low_kernel makes low[m] = x[m] down[a]^T, a thin product that reads x once and is bound by it. The
// linear's GEMM (gemm.cu) then takes low up[a]^T as further K steps of its tiles, on the tensor cores and in the same
// accumulators, so the output is written once and no second pass reads it.
//
// A tile of the GEMM may hold rows of several requests. low is therefore laid out by slots (segments.cuh): the block of a
// (tile, request) pair has the tile's rows, those of other requests zero, and the GEMM takes one step of rank columns a
// pair, low's block against up[a]'s rows. slot_adapter gives a slot's adapter (-1: none) and tile_slots a tile's slots.
//
// low is rounded to fp16 (at most half a step a value, 2^-12 of the adapter's part of the output, which rounding the
// output costs too); its sums are fp32.
#include "common.cuh"
#include "kernels.h"
#include "segments.cuh"

namespace fry {

constexpr int kLowRows = 64, kLowWarps = 8;  // rows a block; its warps share 16-row groups and, beyond those, K

// 16 bytes of x as fp16 pairs: 8 fp16 values, or 16 int8 values. int8 widens exactly: a byte with its sign bit flipped
// in the low bits of 1024.0's fp16 pattern is 1024 + 128 + value.
template <bool INT8>
FRY_DEVICE void low_pairs(const uint4& raw, uint32_t (&pairs)[INT8 ? 8 : 4]) {
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

// TILES: 8-column tiles of the rank. A lane's MMA fragments come from 16-byte loads: of each run of K columns the four
// lanes of a quad read 16 bytes each, and the MMA's K index is assigned to what a lane holds, alike for x and down (a sum
// over K may take it in any order).
template <bool INT8, int TILES>
__global__ void __launch_bounds__(kLowWarps * 32) adapter_low_kernel(const AdapterArgs p, int M, int K) {
    constexpr int kSteps = INT8 ? 4 : 2;          // MMA K steps of 16 a run
    constexpr int kLane = kSteps * 4;             // K columns a lane holds of a run
    constexpr int kRun = 4 * kLane;
    extern __shared__ __align__(16) float partial[];  // [kLowWarps][16][TILES * 8]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int slot = blockIdx.x, part = blockIdx.y;
    grid_dependency_start();

    const PackedRows rows{p.offsets, p.requests, M};
    const int segment = find_segment(rows, TileRows(p.tile_rows), slot, lane);
    const int tile = slot - segment, tile_first = tile * p.tile_rows;
    const int first = max(rows.start(segment), tile_first), last = min(rows.start(segment + 1), min(M, tile_first + p.tile_rows));
    const bool request = segment >= 1 && segment <= p.requests;
    int adapter = -1;
    if (request && first < last) adapter = p.ids[segment - 1];
    const bool known = adapter >= 0 && adapter < p.adapters;
    if (slot == 0 && part == 0)  // one block records the requests that are not in range, for all
        for (int s = threadIdx.x; s < p.requests; s += kLowWarps * 32)
            if (rows.bad(s + 1) || p.ids[s] < -1 || p.ids[s] >= p.adapters) record_error(kBadOffsets, s);
    if (part == 0 && threadIdx.x == 0) {
        p.slot_adapter[slot] = known ? adapter : -1;
        if (first < last && first == tile_first) p.tile_slots[tile].x = slot;
        if (first < last && last == min(M, tile_first + p.tile_rows)) p.tile_slots[tile].y = slot + 1;
    }
    if (!known) return;

    const int part_first = tile_first + part * kLowRows;
    const int low = max(first, part_first), high = min(last, part_first + kLowRows);  // this block's rows of the request
    uint16_t* out = p.low + (static_cast<size_t>(slot) * p.tile_rows + part * kLowRows) * p.rank;
    const int units = p.rank / 8;
    if (low >= high) {
        for (int i = threadIdx.x; i < kLowRows * units; i += kLowWarps * 32) reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
        return;
    }
    // the 16-row groups with rows of the request, and how many warps share each's K
    const int group_first = (low - part_first) / 16, groups = (high - 1 - part_first) / 16 - group_first + 1;
    const int shares = kLowWarps / groups, group = group_first + warp % groups, share = warp / groups;

    float sums[TILES][4] = {};
    if (share < shares) {
        const uint8_t* x_rows[2];
        bool mine[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int m = part_first + group * 16 + g + 8 * half;
            mine[half] = m >= low && m < high;
            x_rows[half] = static_cast<const uint8_t*>(p.x) + static_cast<size_t>(mine[half] ? m : 0) * K * (INT8 ? 1 : 2);
        }
        const uint16_t* down = p.down + static_cast<size_t>(adapter) * p.rank * K;
        constexpr int kAhead = TILES <= 4 ? 4 : 2;  // runs whose loads are in flight together
        for (int run = share * kRun; run < K; run += shares * kRun * kAhead) {
            uint4 raw[kAhead][2], weight[kAhead][TILES][INT8 ? 2 : 1];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int k = run + u * shares * kRun + t * kLane;
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    raw[u][half] = k < K && mine[half] ? *reinterpret_cast<const uint4*>(x_rows[half] + static_cast<size_t>(k) * (INT8 ? 1 : 2)) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int n = 0; n < TILES; ++n)
#pragma unroll
                    for (int h = 0; h < (INT8 ? 2 : 1); ++h)
                        weight[u][n][h] = k < K && n < units ? *reinterpret_cast<const uint4*>(down + static_cast<size_t>(n * 8 + g) * K + k + 8 * h)
                                                             : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                uint32_t a[2][INT8 ? 8 : 4];
                low_pairs<INT8>(raw[u][0], a[0]);
                low_pairs<INT8>(raw[u][1], a[1]);
#pragma unroll
                for (int n = 0; n < TILES; ++n) {
                    const uint32_t* b = reinterpret_cast<const uint32_t*>(weight[u][n]);
#pragma unroll
                    for (int s = 0; s < kSteps; ++s) mma_f16(sums[n], a[0][2 * s], a[1][2 * s], a[0][2 * s + 1], a[1][2 * s + 1], b[2 * s], b[2 * s + 1]);
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
        for (int half = 0; half < 2; ++half)
            *reinterpret_cast<float2*>(partial + ((warp * 16 + g + 8 * half) * TILES + n) * 8 + 2 * t) = make_float2(sums[n][2 * half], sums[n][2 * half + 1]);
    __syncthreads();
    // the shares in order, scaled and rounded; rows of other requests 0
    for (int i = threadIdx.x; i < kLowRows * units; i += kLowWarps * 32) {
        const int row = i / units, unit = i % units, m = part_first + row;
        uint4 packed = make_uint4(0, 0, 0, 0);
        if (m >= low && m < high) {
            const int from = row / 16 - group_first;
            float values[8] = {};
            for (int q = 0; q < shares; ++q) {
                const float* source = partial + (((from + q * groups) * 16 + row % 16) * TILES + unit) * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) values[e] = __fadd_rn(values[e], source[e]);
            }
            const float scale = INT8 ? p.x_scale[m] : 1.0f;
            uint32_t* words = reinterpret_cast<uint32_t*>(&packed);
#pragma unroll
            for (int e = 0; e < 4; ++e) words[e] = pack_half2_rn(__fmul_rn(values[2 * e], scale), __fmul_rn(values[2 * e + 1], scale));
        }
        reinterpret_cast<uint4*>(out)[i] = packed;
    }
}

namespace {

template <bool INT8, int TILES>
cudaError_t launch_low(const AdapterArgs& p, int M, int K, cudaStream_t stream) {
    constexpr int kSmem = kLowWarps * 16 * TILES * 8 * 4;
    auto kernel = adapter_low_kernel<INT8, TILES>;
    const cudaError_t status = ensure_smem(reinterpret_cast<const void*>(kernel), kSmem);
    if (status != cudaSuccess) return status;
    return launch_dependent(kernel, dim3(packed_slots(M, p.tile_rows, p.requests), p.tile_rows / kLowRows), dim3(kLowWarps * 32), kSmem, stream, p, M, K);
}

template <bool INT8>
cudaError_t low_rank_rows(const AdapterArgs& p, int M, int K, cudaStream_t stream) {
    return p.rank <= 16   ? launch_low<INT8, 2>(p, M, K, stream)
           : p.rank <= 32 ? launch_low<INT8, 4>(p, M, K, stream)
           : p.rank <= 64 ? launch_low<INT8, 8>(p, M, K, stream)
                          : launch_low<INT8, 16>(p, M, K, stream);
}

}  // namespace

// low [slots * tile_rows, rank] fp16, then tile_slots and slot_adapter, each 256-byte aligned
AdapterWorkspace::AdapterWorkspace(int M, int requests, int rank, int tile_rows) {
    const size_t slots = packed_slots(M, tile_rows, requests), tiles = (static_cast<size_t>(M) + tile_rows - 1) / tile_rows;
    auto up = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
    this->slots = slots;
    tile_slots = up(slots * tile_rows * rank * 2);
    slot_adapter = tile_slots + up(tiles * sizeof(int2));
    total = slot_adapter + up(slots * sizeof(int32_t));
}

cudaError_t adapter_linear(int kind, GemmArgs& gemm_args, AdapterArgs& p, const void* weight, int M, int N, int K, void* workspace, cudaStream_t stream,
                           std::string* error) {
    p.tile_rows = adapter_tile_rows(kind, M, N);
    const AdapterWorkspace layout(M, p.requests, p.rank, p.tile_rows);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    p.low = reinterpret_cast<uint16_t*>(base);
    p.tile_slots = reinterpret_cast<int2*>(base + layout.tile_slots);
    p.slot_adapter = reinterpret_cast<int32_t*>(base + layout.slot_adapter);
    const cudaError_t status = kind == 0 ? low_rank_rows<true>(p, M, K, stream) : low_rank_rows<false>(p, M, K, stream);
    if (status != cudaSuccess) return status;
    return adapter_gemm(kind, p, weight, gemm_args, static_cast<int>(layout.slots), M, N, K, stream, error);
}

}  // namespace fry
