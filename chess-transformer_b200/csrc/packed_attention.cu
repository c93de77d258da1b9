// Attention over packed sequences and over a cache (packed_attention.cuh) on warp-wide tensor steps (mma.sync), for
// sequences of few rows or few keys, and the choice between these kernels and those of prompt_attention.cu.
//
// Two forms. The block's warps of 16 rows each share tiles of keys (many queries), or KEY_WARPS warps hold the same 16 rows
// and take different keys, each with copies and a softmax of its own, joined at the end (few queries: there the loads
// bound the kernel, and warps that wait for no other keep them in flight). Where blocks are still fewer than the SMs, the
// keys are also split over blocks (`splits`): each writes its m, l and o to a workspace and attention_join_kernel joins
// them in order of the split, so results do not depend on the blocks' order.
#include "packed_attention.cuh"

namespace fry {

// Byte offset of 16-byte unit `unit` of row `row` in a tile of rows of WIDTH 16-bit values, so that eight rows' equal
// units lie in different banks: rows of 128 bytes and up swap units by the row within 8, rows of 64 bytes are paired.
template <int WIDTH>
FRY_DEVICE uint32_t tile_unit(int row, int unit) {
    if constexpr (WIDTH >= 64) return static_cast<uint32_t>(row * WIDTH * 2 + ((unit ^ (row & 7)) << 4));
    else return static_cast<uint32_t>((row >> 1) * 128 + ((((row & 1) * 4 + unit) ^ ((row >> 1) & 7)) << 4));
}
// 16 bytes global -> shared, or zeros without reading
FRY_DEVICE void cp_async16_or_zero(uint32_t shared, const void* global, bool read) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared), "l"(global), "r"(read ? 16 : 0) : "memory");
}

// WIDTH: the head width padded to 32, 64 or 128 with zeros. KEY_WARPS: 1, the block's warps have 16 rows each and share the
// keys; more, they have the same rows and KEYS keys each of a stage.
//
// What bounds them: the key warps HBM (64 full caches of 8192 keys, 8 heads of 128: 6.7 TB/s; of 2048, 12 heads of 64: 5.2
// TB/s, 4.3 to 4.8 with uneven lengths). The row warps the instructions: of 59 us for 256 x 70 tokens, 24 heads of 32, 20 go
// to the search, the queries and the outputs (no keys at all), 10 to the copies and 29 to products and softmax (256 x 64: 20, 6
// and 21 of 47).
constexpr int kMaxRowWarps = 8;
template <int WIDTH, int KEY_WARPS, int KEYS, int STAGES>
struct RowsShape {
    static constexpr int kMaxThreads = (KEY_WARPS > 1 ? KEY_WARPS : kMaxRowWarps) * 32;
    // blocks an SM: 8 warps of a narrow head in 64 registers a thread, 4 times over, hide the loads' latency; the key warps'
    // as many as their own registers allow, which keeps repair_rows' within them
    static constexpr int kBlocks = KEY_WARPS > 1 ? (WIDTH == 128 ? 2 : 4) : WIDTH == 32 ? 4 : WIDTH == 64 ? 2 : 1;
    static constexpr int kStageKeys = KEYS * KEY_WARPS;
    static constexpr int kTileBytes = kStageKeys * WIDTH * 2;  // the keys or the values of a stage
    static constexpr int kLoopBytes = STAGES * 2 * kTileBytes;
    // after the loop: a warp's 16 output rows, or with KEY_WARPS its 16 rows of fp32 sums, m and l
    static constexpr int kSumsPitch = WIDTH + 8;  // floats a row: the quads of a store in different banks
    __host__ __device__ static constexpr int join_bytes(int warps) { return KEY_WARPS > 1 ? KEY_WARPS * 16 * (kSumsPitch + 2) * 4 : warps * 16 * WIDTH * 2; }
    __host__ __device__ static constexpr int found_at(int warps) { return kLoopBytes > join_bytes(warps) ? kLoopBytes : join_bytes(warps); }  // the block's RowBlock
    static constexpr int smem_bytes(int warps) { return found_at(warps) + 64; }
    static_assert(sizeof(RowBlock) <= 64, "the block's rows fit their place");
};

template <int WIDTH, int KEY_WARPS, int KEYS, int STAGES, bool BF16>
__global__ void __launch_bounds__((RowsShape<WIDTH, KEY_WARPS, KEYS, STAGES>::kMaxThreads), (RowsShape<WIDTH, KEY_WARPS, KEYS, STAGES>::kBlocks))
    attention_rows_kernel(const __grid_constant__ AttentionArgs a) {
    using S = RowsShape<WIDTH, KEY_WARPS, KEYS, STAGES>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int row_warp = KEY_WARPS > 1 ? 0 : warp, key_warp = KEY_WARPS > 1 ? warp : 0;
    grid_dependency_start();
    check_offsets(a);

    // one warp searches for all
    RowBlock* found = reinterpret_cast<RowBlock*>(smem + S::found_at(static_cast<int>(blockDim.x) / 32));
    if (warp == 0) {
        RowBlock mine;
        if (!find_rows(a, a.slot_tokens, blockIdx.x, lane, mine)) mine.tokens = 0;
        if (lane == 0) *found = mine;
    }
    __syncthreads();
    const RowBlock b = *found;
    if (b.tokens <= 0) return;
    const int kv_head = blockIdx.y / a.head_tiles, first_head = kv_head * a.group + (blockIdx.y % a.head_tiles) * a.tile_heads;
    const int heads_here = min(a.tile_heads, (kv_head + 1) * a.group - first_head);
    // a row's token and head; rows past the block's tokens or heads compute on zeros and are not written
    auto token_of = [&](int r) { return a.token_of(r); };
    auto head_of = [&](int r) { return first_head + a.head_in_tile(r); };
    auto live = [&](int r) { return a.token_of(r) < b.tokens && a.head_in_tile(r) < heads_here; };
    const bool idle = row_warp * 16 >= b.tokens * a.tile_heads;  // no row of this warp's 16 is live

    // this block's keys: those its last token sees, of which a split takes whole stages
    const int seen = b.limit(b.tokens - 1, a.causal);
    const int stages = (seen + S::kStageKeys - 1) / S::kStageKeys, per_split = (stages + a.splits - 1) / a.splits;
    const int split = blockIdx.z;
    const int low = min(seen, split * per_split * S::kStageKeys), high = min(seen, (split + 1) * per_split * S::kStageKeys);
    const int steps = (high - low + S::kStageKeys - 1) / S::kStageKeys;

    const uint16_t* keys = a.k + b.k_base + kv_head * a.k_head;
    const uint16_t* values = a.v + b.v_base + kv_head * a.v_head;
    constexpr int kUnits = WIDTH / 8;
    const int units = a.width / 8;
    auto load = [&](int step) {
        if (step < steps) {
            uint8_t* stage = smem + (step % STAGES) * 2 * S::kTileBytes;
            const uint32_t k_tile = smem_addr(stage), v_tile = k_tile + S::kTileBytes;
            const int first = low + step * S::kStageKeys;
            auto copy = [&](int row, int unit) {
                const int key = first + row;
                const bool read = key < high && unit < units;
                cp_async16_or_zero(k_tile + tile_unit<WIDTH>(row, unit), keys + (read ? key * a.k_row + unit * 8 : 0), read);
                cp_async16_or_zero(v_tile + tile_unit<WIDTH>(row, unit), values + (read ? key * a.v_row + unit * 8 : 0), read);
            };
            if constexpr (KEY_WARPS > 1) {  // a warp copies its own keys
#pragma unroll
                for (int i = 0; i < KEYS * kUnits / 32; ++i) copy(key_warp * KEYS + (lane + 32 * i) / kUnits, (lane + 32 * i) % kUnits);
            } else {  // the block copies all, in whole 16s
                const int rows = min(KEYS, (high - first + 15) / 16 * 16);
                for (int at = threadIdx.x; at < rows * kUnits; at += blockDim.x) copy(at / kUnits, at % kUnits);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) load(s);

    // the queries' fragments: rows g and g + 8 of the warp's 16, columns 2t, 2t + 1 and 8 + 2t, 9 + 2t of each 16
    uint32_t q[WIDTH / 16][4];
    int limit[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = row_warp * 16 + g + 8 * half;
        const bool mine = live(r);
        limit[half] = mine ? min(high, b.limit(token_of(r), a.causal)) : high;
        const uint16_t* row = a.q + (mine ? (b.row + token_of(r)) * a.q_row + head_of(r) * a.q_head : 0);
#pragma unroll
        for (int s = 0; s < WIDTH / 16; ++s)
#pragma unroll
            for (int part = 0; part < 2; ++part)
                q[s][half + 2 * part] = mine && 2 * s + part < units ? *reinterpret_cast<const uint32_t*>(row + s * 16 + part * 8 + 2 * t) : 0u;
    }

    // where this lane's rows of the B fragments lie: units swap within 8 (or 16) rows alike, so 16 keys on is a fixed step
    const int key_row = key_warp * KEYS + (lane >> 4) * 8 + (lane & 7), value_row = key_warp * KEYS + ((lane >> 3) & 1) * 8 + (lane & 7);
    const uint32_t k_offset = tile_unit<WIDTH>(key_row, 0) & ~127u, v_offset = tile_unit<WIDTH>(value_row, 0) & ~127u;
    uint32_t k_units[WIDTH / 16], v_units[WIDTH / 16];
#pragma unroll
    for (int c = 0; c < WIDTH / 16; ++c) {
        k_units[c] = tile_unit<WIDTH>(key_row, 2 * c + ((lane >> 3) & 1)) - k_offset;
        v_units[c] = tile_unit<WIDTH>(value_row, 2 * c + (lane >> 4)) - v_offset;
    }

    float o[WIDTH / 8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    for (int step = 0; step < steps; ++step) {
        cp_async_wait<STAGES - 2>();
        if constexpr (KEY_WARPS > 1) __syncwarp();
        else __syncthreads();
        load(step + STAGES - 1);  // into the stage read in the step before, which every reader has left
        const uint32_t k_tile = smem_addr(smem + (step % STAGES) * 2 * S::kTileBytes), v_tile = k_tile + S::kTileBytes;
        const int first_key = low + step * S::kStageKeys + key_warp * KEYS, left = high - first_key;  // this warp's keys
        if (idle || left <= 0) continue;
        float s[KEYS / 8][4];
        const uint32_t k_lane = k_tile + k_offset, v_lane = v_tile + v_offset;
#pragma unroll
        for (int n = 0; n < KEYS / 16; ++n) {
            if (n * 16 >= left) break;  // 16 keys at a time, none behind the last
#pragma unroll
            for (int c = 0; c < WIDTH / 16; ++c) {
                uint32_t f[4];
                ldmatrix_x4(k_lane + n * 16 * WIDTH * 2 + k_units[c], f);
                if (c == 0)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[2 * n][e] = s[2 * n + 1][e] = 0.0f;
                mma16816<BF16>(s[2 * n], q[c], f[0], f[1]);
                mma16816<BF16>(s[2 * n + 1], q[c], f[2], f[3]);
            }
        }
        if (first_key + KEYS > min(limit[0], limit[1])) {
            const int seen_here[2] = {limit[0] - first_key - 2 * t, limit[1] - first_key - 2 * t};
#pragma unroll
            for (int n = 0; n < KEYS / 8; ++n) {
                if (n % 2 == 0 && n * 8 >= left) break;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n * 8 + (e & 1) >= seen_here[e >> 1]) s[n][e] = -INFINITY;
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float top = s[0][2 * half];
#pragma unroll
            for (int n = 0; n < KEYS / 8; ++n) {
                if (n % 2 == 0 && n * 8 >= left) break;
                top = max3(top, s[n][2 * half], s[n][2 * half + 1]);
            }
            top = fmaxf(m[half], __fmul_rn(quad_max(top), a.scale_log2));
            const float base = top == -INFINITY ? 0.0f : top, shrink = ex2_approx_ftz(m[half] - base);
            m[half] = top;
            l[half] *= shrink;
#pragma unroll
            for (int c = 0; c < WIDTH / 8; ++c) o[c][2 * half] *= shrink, o[c][2 * half + 1] *= shrink;
            const uint64_t scale2 = pair2(a.scale_log2, a.scale_log2), base2 = pair2(-base, -base);
            uint64_t total2 = pair2(0.0f, 0.0f);
#pragma unroll
            for (int n = 0; n < KEYS / 8; ++n) {
                if (n % 2 == 0 && n * 8 >= left) break;
                const float2 x = lanes(add2(product2(pair2(s[n][2 * half], s[n][2 * half + 1]), scale2), base2));
                s[n][2 * half] = ex2_approx_ftz(x.x), s[n][2 * half + 1] = ex2_approx_ftz(x.y);
                total2 = add2(total2, pair2(s[n][2 * half], s[n][2 * half + 1]));
            }
            const float2 total = lanes(total2);
            l[half] += total.x + total.y;
        }
#pragma unroll
        for (int n = 0; n < KEYS / 16; ++n) {
            if (n * 16 >= left) break;
            const uint32_t p[4] = {pack16<BF16>(s[2 * n][0], s[2 * n][1]), pack16<BF16>(s[2 * n][2], s[2 * n][3]),
                                   pack16<BF16>(s[2 * n + 1][0], s[2 * n + 1][1]), pack16<BF16>(s[2 * n + 1][2], s[2 * n + 1][3])};
#pragma unroll
            for (int c = 0; c < WIDTH / 16; ++c) {
                uint32_t f[4];
                ldmatrix_x4_trans(v_lane + n * 16 * WIDTH * 2 + v_units[c], f);
                mma16816<BF16>(o[2 * c], p, f[0], f[1]);
                mma16816<BF16>(o[2 * c + 1], p, f[2], f[3]);
            }
        }
    }
    cp_async_wait<0>();
    __syncthreads();  // the stages are free
#pragma unroll
    for (int half = 0; half < 2; ++half) l[half] = quad_sum(l[half]);

    if constexpr (KEY_WARPS > 1) {
        float* sums = reinterpret_cast<float*>(smem);             // [KEY_WARPS][16][2]: m, l
        float* tops = sums + KEY_WARPS * 16 * 2;                  // [KEY_WARPS][16][kSumsPitch]
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = g + 8 * half;
            if (t == 0) sums[(warp * 16 + r) * 2] = m[half], sums[(warp * 16 + r) * 2 + 1] = l[half];
#pragma unroll
            for (int c = 0; c < WIDTH / 8; ++c)
                *reinterpret_cast<float2*>(tops + (warp * 16 + r) * S::kSumsPitch + c * 8 + 2 * t) = make_float2(o[c][2 * half], o[c][2 * half + 1]);
        }
        __syncthreads();
        for (int r = warp; r < 16; r += KEY_WARPS) {  // a warp a row, lane i columns i, i + 32, ...
            if (!live(r)) continue;
            float top = -INFINITY, total = 0.0f, joined[WIDTH / 32] = {};
#pragma unroll
            for (int w = 0; w < KEY_WARPS; ++w) top = fmaxf(top, sums[(w * 16 + r) * 2]);
            const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < KEY_WARPS; ++w) {
                const float share = ex2_approx_ftz(sums[(w * 16 + r) * 2] - base);
                total = __fmaf_rn(share, sums[(w * 16 + r) * 2 + 1], total);
#pragma unroll
                for (int i = 0; i < WIDTH / 32; ++i) joined[i] = __fmaf_rn(share, tops[(w * 16 + r) * S::kSumsPitch + lane + 32 * i], joined[i]);
            }
            bool finite = true;
#pragma unroll
            for (int i = 0; i < WIDTH / 32; ++i) finite = finite && isfinite(joined[i]);
            const int token = token_of(r), head = head_of(r);
            const AttentionOut to = attention_out(a, split, b.row + token, head);
            const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int i = 0; i < WIDTH / 32; ++i) {
                const int c = lane + 32 * i;
                if (c >= a.width) continue;
                if (a.splits > 1) to.part_out[c] = joined[i];
                else to.out[c] = static_cast<uint16_t>(pack16<BF16>(joined[i] * inverse, 0.0f) & 0xffff);
            }
            if (a.splits > 1 && lane == 0) to.part_sums[0] = top, to.part_sums[1] = total;
            if (isfinite(total) && !__all_sync(0xffffffffu, finite))
                repair_rows<BF16, WIDTH>(a, b, 1, RowsAt{r, 0, first_head}, top, total, low, high, high, split);
        }
    } else {
        uint8_t* staged = smem + warp * 16 * WIDTH * 2;
        bool finite[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = row_warp * 16 + g + 8 * half;
            uint64_t zero2 = pair2(0.0f, 0.0f);  // 0 * o is 0 where o is finite, else NaN
#pragma unroll
            for (int c = 0; c < WIDTH / 8; ++c) zero2 = fma2(pair2(o[c][2 * half], o[c][2 * half + 1]), pair2(0.0f, 0.0f), zero2);
            const float2 zero = lanes(zero2);
            finite[half] = zero.x + zero.y == 0.0f || !isfinite(l[half]) || !live(r);
            const float inverse = l[half] == 0.0f ? 0.0f : 1.0f / l[half];
            if (a.splits > 1) {
                if (live(r)) {
                    const AttentionOut to = attention_out(a, split, b.row + token_of(r), head_of(r));
#pragma unroll
                    for (int c = 0; c < WIDTH / 8; ++c)
                        if (c < units) *reinterpret_cast<float2*>(to.part_out + c * 8 + 2 * t) = make_float2(o[c][2 * half], o[c][2 * half + 1]);
                    if (t == 0) to.part_sums[0] = m[half], to.part_sums[1] = l[half];
                }
            } else {
#pragma unroll
                for (int c = 0; c < WIDTH / 8; ++c)
                    *reinterpret_cast<uint32_t*>(staged + tile_unit<WIDTH>(g + 8 * half, c) + 4 * t) =
                        pack16<BF16>(o[c][2 * half] * inverse, o[c][2 * half + 1] * inverse);
            }
        }
        __syncwarp();
        if (a.splits == 1) {
#pragma unroll
            for (int i = 0; i < 16 * kUnits / 32; ++i) {
                const int at = lane + i * 32, r = at / kUnits, unit = at % kUnits;
                if (unit < units && live(row_warp * 16 + r))
                    *reinterpret_cast<uint4*>(attention_out(a, 0, b.row + token_of(row_warp * 16 + r), head_of(row_warp * 16 + r)).out + unit * 8) =
                        *reinterpret_cast<const uint4*>(staged + tile_unit<WIDTH>(r, unit));
            }
        }
        if (__all_sync(0xffffffffu, finite[0] && finite[1])) return;
        // rows whose output is not finite though their sum is, from the votes of their quads; a row's m and l to the row's lane
        const uint32_t votes[2] = {__ballot_sync(0xffffffffu, !finite[0]), __ballot_sync(0xffffffffu, !finite[1])};
        uint32_t again = 0;
        for (int i = 0; i < 16; ++i) again |= (((i < 8 ? votes[0] : votes[1]) >> (i % 8 * 4)) & 15u) != 0 ? 1u << i : 0u;
        const int from = lane % 8 * 4;
        const float tops[2] = {__shfl_sync(0xffffffffu, m[0], from), __shfl_sync(0xffffffffu, m[1], from)};
        const float sums[2] = {__shfl_sync(0xffffffffu, l[0], from), __shfl_sync(0xffffffffu, l[1], from)};
        const RowsAt at{row_warp * 16, 0, first_head};
        repair_rows<BF16, WIDTH>(a, b, again, at, lane < 8 ? tops[0] : tops[1], lane < 8 ? sums[0] : sums[1], low, high, high, split);
    }
}

// Joins the splits of a (row, head), a block each: with M the largest m, out = sum 2^(m - M) o / sum 2^(m - M) l. Warp w
// takes splits w, w + 4, ..., whose loads do not wait for one another; the warps' sums are added in order.
constexpr int kJoinWarps = 4;
template <bool BF16>
__global__ void __launch_bounds__(kJoinWarps * 32) attention_join_kernel(const __grid_constant__ AttentionArgs a) {
    __shared__ float4 sums[kJoinWarps][32];
    __shared__ float totals[kJoinWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_start();
    const int64_t count = static_cast<int64_t>(a.queries.rows) * a.heads, at = blockIdx.x;
    // lane i holds m and l of splits i and i + 32
    static_assert(kMaxAttentionSplits <= 64, "two splits a lane");
    float2 mine[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        mine[i] = lane + 32 * i < a.splits ? *reinterpret_cast<const float2*>(a.part_sums + ((lane + 32 * i) * count + at) * 2) : make_float2(-INFINITY, 0.0f);
    const float top = warp_max(fmaxf(mine[0].x, mine[1].x)), base = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int column = 4 * lane < a.width ? lane : 0;
#pragma unroll 8
    for (int s = warp; s < a.splits; s += kJoinWarps) {
        float4 part = reinterpret_cast<const float4*>(a.part_out + (s * count + at) * a.width)[column];
        const float2 sums = s < 32 ? mine[0] : mine[1];
        const float m = __shfl_sync(0xffffffffu, sums.x, s & 31), l = __shfl_sync(0xffffffffu, sums.y, s & 31);
        const float share = ex2_approx_ftz(m - base);
        if (l == 0.0f) part = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // a split without keys for this row may have written none
        total = __fmaf_rn(share, l, total);
        o.x = __fmaf_rn(share, part.x, o.x), o.y = __fmaf_rn(share, part.y, o.y), o.z = __fmaf_rn(share, part.z, o.z), o.w = __fmaf_rn(share, part.w, o.w);
    }
    sums[warp][lane] = o;
    if (lane == 0) totals[warp] = total;
    __syncthreads();
    if (warp != 0 || 4 * lane >= a.width) return;
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w) {
        const float4 other = sums[w][lane];
        o.x += other.x, o.y += other.y, o.z += other.z, o.w += other.w;
        total += totals[w];
    }
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    reinterpret_cast<uint2*>(a.out + at * a.width)[lane] = make_uint2(pack16<BF16>(o.x * inverse, o.y * inverse), pack16<BF16>(o.z * inverse, o.w * inverse));
}

// ---- host side ---------------------------------------------------------------------------------------------

namespace {

template <int WIDTH, int KEY_WARPS, int KEYS, int STAGES, bool BF16>
cudaError_t launch_rows(AttentionArgs a, int row_warps, cudaStream_t stream) {
    using S = RowsShape<WIDTH, KEY_WARPS, KEYS, STAGES>;
    a.set_tile(row_warps * 16);
    const int slots = a.lengths ? a.queries.count : packed_slots(a.queries.rows, a.slot_tokens.rows, a.queries.count);
    const int warps = row_warps * KEY_WARPS, smem = S::smem_bytes(warps);
    auto kernel = attention_rows_kernel<WIDTH, KEY_WARPS, KEYS, STAGES, BF16>;
    const cudaError_t status = ensure_smem(reinterpret_cast<const void*>(kernel), smem);
    if (status != cudaSuccess) return status;
    return launch_dependent(kernel, dim3(slots, a.kv_heads * a.head_tiles, a.splits), dim3(warps * 32), smem, stream, a);
}

// Width 32, whose blocks have 64 registers a thread: 48 keys a stage spill less than 64 and waste less of a last stage (256 x
// 70 tokens, 61.4 -> 58.2 us; 200 x 96, 64.9 -> 58.6; 700 x 24, 48.0 -> 44.5; of 70 tokens 80 keys 67.9 us, 96 73.0). Sequences
// that fill one stage of 64 lose 2% by it (256 x 64, 45.7 -> 46.5 us).
template <int WIDTH, bool BF16>
cudaError_t launch_width(const AttentionArgs& a, const AttentionPlan& plan, cudaStream_t stream) {
    return plan.form == AttentionForm::kFew ? launch_rows<WIDTH, 4, 16, 3, BF16>(a, 1, stream) : launch_rows<WIDTH, 1, WIDTH == 32 ? 48 : 64, 2, BF16>(a, plan.row_warps, stream);
}

template <bool BF16>
cudaError_t launch_type(const AttentionArgs& a, const AttentionPlan& plan, cudaStream_t stream, std::string* error) {
    cudaError_t status;
    if (plan.form == AttentionForm::kPrompt && a.width <= 64) status = launch_prompt<64, 1, BF16>(a, stream, error);
    else if (plan.form == AttentionForm::kPrompt && plan.long_keys) status = launch_prompt<128, 2, BF16>(a, stream, error);
    else if (plan.form == AttentionForm::kPrompt) status = launch_prompt<128, 1, BF16>(a, stream, error);
    else if (a.width <= 32) status = launch_width<32, BF16>(a, plan, stream);
    else if (a.width <= 64) status = launch_width<64, BF16>(a, plan, stream);
    else status = launch_width<128, BF16>(a, plan, stream);
    if (status != cudaSuccess || a.splits == 1) return status;
    const int64_t count = static_cast<int64_t>(a.queries.rows) * a.heads;
    return launch_dependent(attention_join_kernel<BF16>, dim3(static_cast<unsigned>(count)), dim3(kJoinWarps * 32), 0, stream, a);
}

}  // namespace

AttentionPlan attention_plan(const AttentionShape& s) {
    AttentionPlan plan;
    const int64_t sequences = s.sequences > 0 ? s.sequences : 1;
    const int64_t all_rows = static_cast<int64_t>(s.q_rows) * (s.heads / s.kv_heads) / sequences, mean_rows = all_rows > 0 ? all_rows : 1;
    const int64_t mean_keys = s.cached ? s.capacity : s.key_rows / sequences;
    // Few rows against enough keys: the key warps (64 x 2 tokens of 8 grouped heads, 2000 keys, 48 us against the row
    // warps' 171; but 256 x 8 tokens against 8 keys 34 against 21). More rows: the prompt kernel, where its tiles of 128
    // rows and keys are filled well enough (64 x 64 tokens, 512 keys, 41 us against 59; x 128, 128 keys, 28 against 43; x 4
    // of 8 grouped heads, 2000 keys, 56 against 84 of the key warps; but 64 x 32 tokens, 256 keys, 28 against 22, and 128 x
    // 70 of 2 grouped heads, 70 keys, 80 against 52).
    // One kernel takes the whole batch, the mean's: the host has no other length. A batch of like requests loses nothing, one
    // prompt of 2000 tokens beside 255 single tokens after 2000 keys little (32/8 heads of 128: 406 us, 54 and 328 as two
    // calls); one of 8192 beside 4000 sequences of one token and 3 keys takes 11.2 ms, 0.48 and 0.37 as two calls.
    const bool few = s.cached || (mean_rows <= 16 && mean_keys >= 128);
    const bool prompt = !few && mean_rows > 16 && mean_keys >= 128 && mean_rows * mean_keys >= 128 * 128;
    plan.form = few ? AttentionForm::kFew : prompt ? AttentionForm::kPrompt : AttentionForm::kRows;
    // blocks without a split, and how many fit a round of the SMs twice over; a split keeps 256 keys or more of a mean sequence
    const int64_t group = s.heads / s.kv_heads;
    if (!few && !prompt) {
        // a mean sequence's rows in as few blocks as take them, spread evenly
        const int64_t row_blocks = (mean_rows + kMaxRowWarps * 16 - 1) / (kMaxRowWarps * 16);
        plan.row_warps = static_cast<int>((mean_rows + row_blocks * 16 - 1) / (row_blocks * 16));
    }
    plan.long_keys = prompt && s.width > 64 && mean_keys >= 6144;  // two tiles a block (prompt_attention.cu)
    const int64_t rows = few ? 16 : prompt ? (plan.long_keys ? 256 : 128) : plan.row_warps * 16, tile = rows / (group < rows ? group : rows);
    const int64_t blocks = s.kv_heads * ((group + rows - 1) / rows) * (s.cached ? sequences : (s.q_rows + tile - 1) / tile + sequences / 2);
    // (a cache's: a block an SM where that splits every sequence, else sixteen, which even out their lengths)
    const int64_t wanted = (s.cached && blocks >= kSms ? 16 : few || plan.long_keys ? 1 : 2) * kSms / (blocks > 0 ? blocks : 1), most = mean_keys / 256;
    const int64_t splits = wanted < most ? wanted : most;
    plan.splits = static_cast<int>(splits < 1 ? 1 : splits > kMaxAttentionSplits ? kMaxAttentionSplits : splits);
    const size_t parts = static_cast<size_t>(plan.splits) * s.q_rows * s.heads;
    plan.workspace_bytes = plan.splits > 1 ? parts * (static_cast<size_t>(s.width) + 2) * sizeof(float) : 0;
    return plan;
}

cudaError_t packed_attention(const AttentionShape& shape, const AttentionTensors& x, float scale, void* workspace, cudaStream_t stream, std::string* error) {
    const AttentionPlan plan = attention_plan(shape);
    AttentionArgs a;
    a.q = x.q, a.k = x.k, a.v = x.v, a.out = x.out;
    a.q_row = x.q_row, a.q_head = x.q_head, a.k_row = x.k_row, a.k_head = x.k_head, a.v_row = x.v_row, a.v_head = x.v_head;
    a.k_sequence = x.k_sequence, a.v_sequence = x.v_sequence;
    a.heads = shape.heads, a.kv_heads = shape.kv_heads, a.width = shape.width, a.group = shape.heads / shape.kv_heads;
    a.queries = PackedRows{x.q_offsets, shape.sequences, shape.q_rows};
    a.k_offsets = x.k_offsets, a.k_rows = shape.key_rows;
    a.lengths = x.lengths, a.capacity = shape.capacity;
    a.causal = shape.causal;
    a.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
    a.splits = plan.splits;
    a.part_out = static_cast<float*>(workspace);  // first: it is read 16 bytes at a time
    a.part_sums = a.part_out + static_cast<size_t>(plan.splits) * shape.q_rows * shape.heads * shape.width;
    return shape.bf16 ? launch_type<true>(a, plan, stream, error) : launch_type<false>(a, plan, stream, error);
}

}  // namespace fry
