// Attention over packed sequences on the fifth-generation tensor cores, for sequences of many rows (packed_attention.cuh has
// the operator's definition, packed_attention.cu the other kernels and the choice between them).
//
// A block takes TILES tiles of 128 rows (a row is a token and one of the query heads that share its keys) against keys in
// tiles of 128, each of the products a tcgen05.mma of M = 128: scores S = Q K^T into TMEM, and O += P V with P read from
// TMEM. One warp streams the key and value tiles through a ring of stages with TMA, one issues the MMAs, and four warps a
// tile are its softmax, a thread a row. Two tiles are on an SM, so that while one's scores are on the softmax the tensor
// core works on the other's products: in two blocks of one, or in one block of two.
// Two blocks start and end on their own, one's beginning and end under the other's work; one block's tiles share its key
// and value stages, half the traffic from L2. Measured (five calls in a graph, device busy; two blocks / one): 8 x 512 tokens
// of 12 heads of 64 after ragged keys 54 / 61 us; of 32 heads of 128, 16 prompts of 1000 tokens 228 / 236 us, one of 4096 141 /
// 138, of 5000 198 / 201, of 6144 290 / 289, of 7000 399 / 373, of 8192 535 / 502 (the power cap moves these by 5%).
// What bounds it: a step of both tiles (2 x 128 rows by 128 keys) takes about 3400 clocks at width 128, of which the
// tensor core is busy for 2048 and the exponentials (16 a clock and SM) for 2048. A row tile's chain of loads from TMEM
// (250 clocks), exponentials (64 at a time 520 to 900, with the other tile at its own), hand-over and products (1100)
// does not fill either; splitting S in two steps of 64 keys so that the softmax never waits loses more to the narrower
// products (their operands' shared memory reads bound them), exponentials in part on the FMA pipe gained 1%, two warps a
// row or turns at the exponentials lost 10 to 25%.
//
// TMEM (512 columns of 32 bits an SM): a tile's S (128 columns), O (WIDTH) and P (64: two 16-bit values a column). At width
// 128 that is 64 columns too many: there P overwrites the first half of S, which the thread that writes it has read, and
// the next Q K^T into S follows P V; one thread issues both, and products of one shape are taken in the order they are
// issued in. At width 64 the two have different shapes, whose order is not defined, but P has columns of its own: the next
// Q K^T is issued as soon as the softmax has read S, and P waits for the P V before it.
//
// Softmax: a row's 128 scores are in its thread's registers, so maximum and sum need no exchange, and P V of the first 64
// starts while the thread is at the others. The running maximum m may lag behind: the first probabilities are taken
// against the m of the keys before, while the new maximum is still being found, and as long as no row of the warp has risen
// by more than 2^8 they stand (they stay below 2^8, in the same relative steps); only where one has, O and the sum are
// scaled to the new m. The first tile of keys always sets m, so the largest probability of a row is at least 1.
#include "common.cuh"
#include "kernels.h"
#include "packed_attention.cuh"

namespace fry {

constexpr int kPromptTile = 128;  // rows of a tile, and keys of a stage
constexpr float kLagLog2 = 8.0f;

template <int WIDTH, int TILES>
struct PromptShape {
    static constexpr int kBlocks = 2 / TILES;               // blocks an SM
    static constexpr int kBoxBytes = kPromptTile * 128;     // 128 rows of 64 columns, the 128-byte swizzle
    static constexpr int kTileBytes = WIDTH / 64 * kBoxBytes;
    static constexpr int kStages = TILES == 2 ? 5 : WIDTH == 128 ? 2 : 4;  // key and value tiles in turn
    static constexpr int kBarrierBytes = 512;
    static constexpr int kSmemBytes = (TILES + kStages) * kTileBytes + kBarrierBytes;
    // warps: the tiles' softmax, then a group of four of which the first loads and the second issues the MMAs
    static constexpr int kSoftmaxWarps = 4 * TILES, kLoadWarp = kSoftmaxWarps, kMmaWarp = kSoftmaxWarps + 1, kThreads = (kSoftmaxWarps + 4) * 32;
    // Registers a thread: the softmax's warps take 208, which hold a row's 128 scores, and leave the others what remains of
    // the launch's: 168 a thread of 384 (256 x 208 + 128 x 88 = 64512), 128 of 256 (128 x 208 + 128 x 48 = 32768).
    static constexpr int kSoftmaxRegisters = 208, kOtherRegisters = TILES == 2 ? 88 : 48;
    // TMEM columns
    static constexpr bool kShared = WIDTH == 128;           // P lies in S
    static constexpr int kOutAt = TILES * kPromptTile, kProbabilitiesAt = kShared ? 0 : kOutAt + TILES * WIDTH, kProbabilities = kShared ? kPromptTile : 64;
    static constexpr int kColumns = TILES * 256;
    static_assert(kBlocks * (kSmemBytes + 1024) <= 228 * 1024, "an SM holds the blocks");
    static_assert(TILES * (kPromptTile + WIDTH + (kShared ? 0 : 64)) <= kColumns, "TMEM holds the tiles");
};

// D[tmem] (+)= A[tmem] * B[smem], 16-bit A two values a column
FRY_DEVICE void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate));
}
// 32 32-bit TMEM columns of this thread's lane, written
FRY_DEVICE void tmem_store32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
FRY_DEVICE void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
FRY_DEVICE void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}
FRY_DEVICE void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}
// Descriptor of the value tile as a B operand whose rows are the MMA's K: boxes of 64 columns, 128 bytes a key in the
// 128-byte swizzle. Leading offset: from a box to the next 64 columns; stride offset: from 8 keys to the next 8.
FRY_DEVICE uint64_t value_desc(uint32_t smem_byte_addr) {
    return static_cast<uint64_t>((smem_byte_addr >> 4) & 0x3FFF) | static_cast<uint64_t>(kPromptTile * 128 >> 4) << 16 |
           static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
// instr_desc<1> with the operands' type and, for the values, B's rows as K (bit 16)
template <bool BF16>
__host__ __device__ constexpr uint32_t prompt_desc(int n, bool rows_are_k) {
    return instr_desc<1>(n) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (rows_are_k ? 1u << 16 : 0u);
}

template <int WIDTH, int TILES, bool BF16>
__global__ void __launch_bounds__((PromptShape<WIDTH, TILES>::kThreads), (PromptShape<WIDTH, TILES>::kBlocks))
    attention_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                            const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttentionArgs a) {
    using S = PromptShape<WIDTH, TILES>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_addr(smem) & 1023u) {  // uniform across the block
        if (threadIdx.x == 0) record_error(kMisaligned, 30);
        return;
    }
    uint8_t* queries = smem;                              // [2][boxes][128 rows][128 bytes]
    uint8_t* stages = smem + TILES * S::kTileBytes;           // [kStages][boxes][128 keys][128 bytes]
    uint64_t* q_full = reinterpret_cast<uint64_t*>(stages + S::kStages * S::kTileBytes);
    uint64_t* full = q_full + 1;                          // [kStages]
    uint64_t* empty = full + S::kStages;                  // [kStages]
    uint64_t* s_full = empty + S::kStages;                // [2]: a tile's scores are there
    uint64_t* s_read = s_full + 2;                        // [2]: they have been read (width 64)
    uint64_t* p_full = s_read + 2;                        // [2][2]: the first and second half of its probabilities are there
    uint64_t* pv_done = p_full + 4;                       // [2]: P V is done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int s = 0; s < S::kStages; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
        for (int t = 0; t < TILES; ++t) mbar_init(&s_full[t], 1), mbar_init(&s_read[t], 4), mbar_init(&pv_done[t], 1);
        for (int h = 0; h < 4; ++h) mbar_init(&p_full[h], 4);
        fence_barrier_init();
    }
    grid_dependency_start();
    check_offsets(a);
    const int tile = a.slot_tokens.rows / TILES;  // tokens a tile
    RowBlock b;
    const int at = blockIdx.x / (a.kv_heads * a.head_tiles), column = blockIdx.x % (a.kv_heads * a.head_tiles);
    if (!find_rows(a, a.slot_tokens, at, lane, b)) return;  // uniform across the block
    const int kv_head = column / a.head_tiles, head_tile = column % a.head_tiles;
    const int split = blockIdx.z;
    // keys of this split, in whole tiles; those a tile's last token sees
    const int seen = b.limit(b.tokens - 1, a.causal);
    const int key_tiles = (seen + kPromptTile - 1) / kPromptTile, per_split = (key_tiles + a.splits - 1) / a.splits;
    const int low = min(seen, split * per_split * kPromptTile), high = min(seen, (split + 1) * per_split * kPromptTile);
    auto tile_high = [&](int t) {
        const int tokens = min(b.tokens - t * tile, tile);
        return tokens <= 0 ? low : max(low, min(high, b.limit(t * tile + tokens - 1, a.causal)));
    };
    const int highs[2] = {tile_high(0), TILES > 1 ? tile_high(1) : low};
    auto count_of = [&](int t) { return (highs[t] - low + kPromptTile - 1) / kPromptTile; };
    const int counts[2] = {count_of(0), count_of(1)}, steps = max(counts[0], counts[1]);

    if (steps == 0) {  // no keys: zeros (or an empty split)
        for (int r = warp; r < TILES * kPromptTile; r += S::kThreads / 32) {
            const int row = r % kPromptTile, token = r / kPromptTile * tile + a.token_of(row), in_group = head_tile * a.tile_heads + a.head_in_tile(row);
            if (a.token_of(row) >= tile || token >= b.tokens || in_group >= a.group) continue;
            const AttentionOut to = attention_out(a, split, b.row + token, kv_head * a.group + in_group);
            if (a.splits > 1) {
                if (lane == 0) to.part_sums[0] = -INFINITY, to.part_sums[1] = 0.0f;
            } else if (lane < a.width / 8) {
                reinterpret_cast<uint4*>(to.out)[lane] = make_uint4(0, 0, 0, 0);
            }
        }
        return;
    }
    if (warp == S::kMmaWarp) {
        tmem_alloc(tmem_slot, S::kColumns);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp >= S::kSoftmaxWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kOtherRegisters));
        if (warp == S::kLoadWarp) {
            if (elect_one()) {
                const int tiles = counts[1] > 0 ? 2 : 1;
                // a box has whole tokens: tile * tile_heads rows of the 128
                mbar_arrive_expect_tx(q_full, tiles * (WIDTH / 64) * tile * a.tile_heads * 128);
                for (int t = 0; t < tiles; ++t)
                    for (int box = 0; box < WIDTH / 64; ++box)
                        tma_load_4d(queries + t * S::kTileBytes + box * S::kBoxBytes, &map_q, q_full, box * 64, head_tile * a.tile_heads, b.row + t * tile, kv_head);
                bool ok = true;
                for (int i = 0; i < 2 * steps && ok; ++i) {  // keys and values of a step in turn
                    const int s = i % S::kStages;
                    ok = mbar_wait(&empty[s], ((i / S::kStages) & 1) ^ 1, 31);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&full[s], S::kTileBytes);
                    for (int box = 0; box < WIDTH / 64; ++box)
                        tma_load_3d(stages + s * S::kTileBytes + box * S::kBoxBytes, i & 1 ? &map_v : &map_k, &full[s], box * 64,
                                    b.k_first + low + (i >> 1) * kPromptTile, kv_head);
                }
            }
        } else if (warp == S::kMmaWarp) {
            if (elect_one()) {
                constexpr uint32_t score_desc = prompt_desc<BF16>(kPromptTile, false), out_desc = prompt_desc<BF16>(WIDTH, true);
                auto stage = [&](int i) { return smem_addr(stages + (i % S::kStages) * S::kTileBytes); };
                auto wait_stage = [&](int i) { return mbar_wait(&full[i % S::kStages], (i / S::kStages) & 1, 32); };
                // an address's 16-byte units are a descriptor's low bits: steps are added to it
                auto scores = [&](int t, int j) {  // S_t = Q_t K_j^T
                    const uint64_t q = smem_desc_sw128(smem_addr(queries + t * S::kTileBytes)), k = smem_desc_sw128(stage(2 * j));
#pragma unroll
                    for (int c = 0; c < WIDTH / 16; ++c) {
                        const int units = ((c / 4) * S::kBoxBytes + (c % 4) * 32) / 16;
                        mma_ss<1>(tmem + t * kPromptTile, q + units, k + units, score_desc, c > 0 ? 1u : 0u);
                    }
                    mma_commit(&s_full[t]);
                };
                bool ok = mbar_wait(q_full, 0, 33) && wait_stage(0);
                tc_fence_after();
                if (ok) {
                    for (int t = 0; t < TILES; ++t)
                        if (counts[t] > 0) scores(t, 0);
                    mma_commit(&empty[0]);
                }
                for (int j = 0; j < steps && ok; ++j) {
                    const int v_stage = 2 * j + 1, k_next = 2 * j + 2;
                    if (j + 1 < steps) ok = wait_stage(k_next);
                    if constexpr (!S::kShared) {
                        for (int t = 0; t < TILES && ok; ++t) {
                            if (j + 1 >= counts[t]) continue;
                            ok = mbar_wait(&s_read[t], j & 1, 39);
                            tc_fence_after();
                            if (ok) scores(t, j + 1);
                        }
                        if (j + 1 < steps) mma_commit(&empty[k_next % S::kStages]);
                    }
                    ok = ok && wait_stage(v_stage);
                    const uint64_t v = value_desc(stage(v_stage));
                    for (int t = 0; t < TILES && ok; ++t) {
                        if (j >= counts[t]) continue;
                        // O_t += P_t V_j over the keys the tile sees, 16 an MMA, in the halves that P comes in
                        const int keys = min(kPromptTile, highs[t] - low - j * kPromptTile), chunks = (keys + 15) / 16;
                        const uint32_t o = tmem + S::kOutAt + t * WIDTH, p = tmem + S::kProbabilitiesAt + t * S::kProbabilities;
                        for (int half = 0; half < 2 && ok; ++half) {
                            ok = mbar_wait(&p_full[2 * t + half], j & 1, 34);
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int c = 4 * half + i;
                                if (c < chunks) mma_ts(o, p + c * 8, v + c * 16 * 128 / 16, out_desc, j > 0 || c > 0 ? 1u : 0u);
                            }
                        }
                        if (!ok) break;
                        mma_commit(&pv_done[t]);
                        if (S::kShared && j + 1 < counts[t]) scores(t, j + 1);
                    }
                    if (ok) {
                        mma_commit(&empty[v_stage % S::kStages]);
                        if (S::kShared && j + 1 < steps) mma_commit(&empty[k_next % S::kStages]);
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSoftmaxRegisters));
        const int t = TILES > 1 ? warp >> 2 : 0, row = (warp & 3) * 32 + lane;  // this thread's row of tile t
        const int count = counts[t];
        const int token = t * tile + a.token_of(row), in_group = head_tile * a.tile_heads + a.head_in_tile(row);
        const bool live = a.token_of(row) < tile && token < b.tokens && in_group < a.group;
        const int limit = min(b.nk, live ? b.limit(token, a.causal) : INT_MAX);
        // the fewest keys a row of the warp sees: from there on scores are masked
        const int warp_limit = __reduce_min_sync(0xffffffffu, limit);
        const uint32_t lanes_at = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_tmem = tmem + t * kPromptTile + lanes_at, o_tmem = tmem + S::kOutAt + t * WIDTH + lanes_at;
        const uint32_t p_tmem = tmem + S::kProbabilitiesAt + t * S::kProbabilities + lanes_at;
        float scale = a.scale_log2;  // 1 once scores are scaled apart
        bool apart = false;
        float m = -INFINITY;
        uint64_t totals[2] = {pair2(0.0f, 0.0f), pair2(0.0f, 0.0f)};
        bool alive = true;
        for (int j = 0; j < count; ++j) {
            alive = __all_sync(0xffffffffu, mbar_wait(&s_full[t], j & 1, 35));
            if (!alive) break;
            tc_fence_after();
            const int first_key = low + j * kPromptTile;
            uint32_t raw[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_load32(s_tmem + c * 32, raw[c]);
            tmem_load_wait();
            if constexpr (!S::kShared) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_read[t]);
                __syncwarp();
            }
            if (first_key + kPromptTile > warp_limit) {
                const int here = limit - first_key;
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (c * 32 + e >= here) raw[c][e] = __float_as_uint(-INFINITY);
            }
            // value rows behind the sequence's last key that the last MMA's 16 keys still take are another sequence's: zeros
            if (first_key + kPromptTile > b.nk && (highs[t] - first_key + 15) / 16 * 16 > b.nk - first_key) {
                const int i = 2 * j + 1;
                alive = __all_sync(0xffffffffu, mbar_wait(&full[i % S::kStages], (i / S::kStages) & 1, 36));
                uint8_t* values = stages + (i % S::kStages) * S::kTileBytes;
                const int from = b.nk - first_key, rows = 16 - b.nk % 16;
                for (int u = threadIdx.x & 127; u < rows * (WIDTH / 8) && alive; u += 128)
                    *reinterpret_cast<uint4*>(values + (u % (WIDTH / 8)) / 8 * S::kBoxBytes + (from + u / (WIDTH / 8)) * 128 + u % 8 * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_shared();
                __syncwarp();
            }
            auto highest = [&] {
                float top[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    top[c] = fmaxf(__uint_as_float(raw[c][0]), __uint_as_float(raw[c][1]));
#pragma unroll
                    for (int e = 2; e < 32; e += 2) top[c] = max3(top[c], __uint_as_float(raw[c][e]), __uint_as_float(raw[c][e + 1]));
                }
                return fmaxf(m, __fmul_rn(max3(top[0], top[1], fmaxf(top[2], top[3])), scale));
            };
            uint32_t packed[32];
            uint64_t sums[2];
            auto probabilities = [&](int half) {  // of 64 keys, and their sums
                const float base = m == -INFINITY ? 0.0f : -m;
                const uint64_t base2 = pair2(base, base), scale2 = pair2(scale, scale);
                sums[0] = sums[1] = pair2(0.0f, 0.0f);
#pragma unroll
                for (int e = 0; e < 64; e += 2) {
                    const uint32_t* from = &raw[half * 2 + e / 32][e % 32];
                    const float2 x = lanes(fma2(pair2(__uint_as_float(from[0]), __uint_as_float(from[1])), scale2, base2));
                    const float2 p = make_float2(ex2_approx_ftz(x.x), ex2_approx_ftz(x.y));
                    sums[e / 2 % 2] = add2(sums[e / 2 % 2], pair2(p.x, p.y));
                    packed[e / 2] = pack16<BF16>(p.x, p.y);
                }
            };
            auto hand_over = [&](int half) {  // to the MMAs
                totals[0] = add2(totals[0], sums[0]), totals[1] = add2(totals[1], sums[1]);
                tmem_store32(p_tmem + half * 32, packed);
                tmem_store_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[2 * t + half]);
                __syncwarp();  // together again before the next warp-wide TMEM access
            };
            auto scale_apart = [&] {
                scale = 1.0f;
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int e = 0; e < 32; ++e) raw[c][e] = __float_as_uint(__fmul_rn(__uint_as_float(raw[c][e]), a.scale_log2));
            };
            if (j == 0) m = highest(), apart = __any_sync(0xffffffffu, rounds_apart(m));
            if (apart) scale_apart();
            probabilities(0);
            const float risen = highest();
            // P V of the keys before is done: at width 128 the scores came after it
            if (!S::kShared && j > 0) alive = __all_sync(0xffffffffu, alive && mbar_wait(&pv_done[t], (j - 1) & 1, 38));
            if (__any_sync(0xffffffffu, risen > m + kLagLog2)) {
                const float shrink = risen == -INFINITY ? 0.0f : ex2_approx_ftz(m - risen);
                m = risen;
                if (!apart && __any_sync(0xffffffffu, rounds_apart(m))) apart = true, scale_apart();
                totals[0] = mul2(totals[0], pair2(shrink, shrink)), totals[1] = mul2(totals[1], pair2(shrink, shrink));
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < WIDTH; c += 32) {
                    uint32_t o[32];
                    tmem_load32(o_tmem + c, o);
                    tmem_load_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
                    tmem_store32(o_tmem + c, o);
                }
                probabilities(0);
            }
            hand_over(0);
            probabilities(1);
            hand_over(1);
        }
        if (count > 0 && alive) alive = __all_sync(0xffffffffu, mbar_wait(&pv_done[t], (count - 1) & 1, 37));
        tc_fence_after();
        const float2 both = lanes(add2(totals[0], totals[1]));
        const float total = both.x + both.y, inverse = total == 0.0f ? 0.0f : 1.0f / total;
        const int head = kv_head * a.group + in_group;
        const AttentionOut to = attention_out(a, split, b.row + token, head);
        bool finite = true;
        if (alive) {
#pragma unroll 1
            for (int c = 0; c < WIDTH; c += 32) {
                uint32_t o[32];
                if (count > 0) {
                    tmem_load32(o_tmem + c, o);
                    tmem_load_wait();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0;
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (!live || c + u * 8 >= a.width) continue;
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(o[u * 8 + e]), finite = finite && isfinite(v[e]);
                    if (a.splits > 1) {
                        reinterpret_cast<float4*>(to.part_out + c + u * 8)[0] = make_float4(v[0], v[1], v[2], v[3]);
                        reinterpret_cast<float4*>(to.part_out + c + u * 8)[1] = make_float4(v[4], v[5], v[6], v[7]);
                    } else {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = pack16<BF16>(v[2 * e] * inverse, v[2 * e + 1] * inverse);
                        *reinterpret_cast<uint4*>(to.out + c + u * 8) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            if (a.splits > 1 && live) to.part_sums[0] = m, to.part_sums[1] = total;
            // rows of finite sums whose outputs are not finite; the MMAs took the tile's keys in 16s
            const uint32_t again = __ballot_sync(0xffffffffu, live && !finite && isfinite(total));
            const RowsAt at{(warp & 3) * 32, t * tile, kv_head * a.group + head_tile * a.tile_heads};
            if (again) repair_rows<BF16, WIDTH>(a, b, again, at, m, total, low, high, min(b.nk, low + (highs[t] - low + 15) / 16 * 16), split);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == S::kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, S::kColumns);
    }
}

namespace {

bool make_attention_map(CUtensorMap* map, const void* base, bool bf16, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                        const cuuint32_t* box, std::string* error) {
    EncodeTiled encode = encoder(error);
    if (!encode) return false;
    const cuuint32_t element_strides[4] = {1, 1, 1, 1};
    const CUresult result = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base), dims,
                                   strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (result != CUDA_SUCCESS && error) *error = "cuTensorMapEncodeTiled failed with CUresult " + std::to_string(static_cast<int>(result));
    return result == CUDA_SUCCESS;
}

template <int WIDTH, int TILES, bool BF16>
cudaError_t launch_prompt(AttentionArgs a, cudaStream_t stream, std::string* error) {
    using S = PromptShape<WIDTH, TILES>;
    a.set_tile(kPromptTile, TILES);
    const cuuint32_t tile = a.slot_tokens.rows / TILES;
    using Dim = cuuint64_t;
    CUtensorMap map_q, map_k, map_v;
    const Dim q_dims[4] = {Dim(a.width), Dim(a.group), Dim(a.queries.rows), Dim(a.kv_heads)};
    const Dim q_strides[3] = {Dim(a.q_head) * 2, Dim(a.q_row) * 2, Dim(a.q_head) * a.group * 2};
    const cuuint32_t q_box[4] = {64, static_cast<cuuint32_t>(a.tile_heads), tile, 1}, k_box[3] = {64, kPromptTile, 1};
    const Dim k_dims[3] = {Dim(a.width), Dim(a.k_rows), Dim(a.kv_heads)};
    const Dim k_strides[2] = {Dim(a.k_row) * 2, Dim(a.k_head) * 2}, v_strides[2] = {Dim(a.v_row) * 2, Dim(a.v_head) * 2};
    if (!make_attention_map(&map_q, a.q, BF16, 4, q_dims, q_strides, q_box, error) || !make_attention_map(&map_k, a.k, BF16, 3, k_dims, k_strides, k_box, error) ||
        !make_attention_map(&map_v, a.v, BF16, 3, k_dims, v_strides, k_box, error))
        return cudaErrorInvalidValue;
    auto kernel = attention_prompt_kernel<WIDTH, TILES, BF16>;
    const cudaError_t status = ensure_smem(reinterpret_cast<const void*>(kernel), S::kSmemBytes);
    if (status != cudaSuccess) return status;
    const int64_t blocks = static_cast<int64_t>(packed_slots(a.queries.rows, a.slot_tokens.rows, a.queries.count)) * a.kv_heads * a.head_tiles;
    if (blocks > 0x7fffffff) {
        if (error) *error = "more row tiles of a head than a launch takes";
        return cudaErrorInvalidValue;
    }
    return launch_dependent(kernel, dim3(static_cast<unsigned>(blocks), 1, a.splits), dim3(S::kThreads), S::kSmemBytes, stream, map_q, map_k, map_v, a);
}

}  // namespace

}  // namespace fry
