// Packed rows: the rows of several requests one behind the other, request s at [offsets[s], offsets[s + 1]). Row kernels
// that take them in tiles give every request slots for its tiles without knowing the lengths on the host.
#pragma once

#include "common.cuh"

namespace fry {

// Rows [0, rows) as count + 2 segments: segment 0 is what lies before the first request, segment s + 1 request s, and
// segment count + 1 what lies behind the last. An offset outside [0, rows] counts as the nearest end.
struct PackedRows {
    const int32_t* offsets;  // [count + 1]
    int count;
    int rows;

    FRY_DEVICE int clamped(int32_t offset) const { return offset < 0 ? 0 : offset > rows ? rows : offset; }
    // where segment i starts, i in [0, count + 2]; the last is the end of the rows
    FRY_DEVICE int start(int i) const { return i == 0 ? 0 : i == count + 2 ? rows : clamped(offsets[i - 1]); }
    FRY_DEVICE bool bad(int i) const {  // request i - 1's offsets, as the caller gave them
        const int32_t first = offsets[i - 1], last = offsets[i];
        return first < 0 || last < first || last > rows;
    }
};

// A tile's rows, and their division: row / rows is the high word of row * ceil(2^32 / rows), exact for row * rows < 2^32
// (row * (ceil(2^32 / rows) * rows - 2^32) < 2^32), so up to kMaxPackedRows rows in tiles of up to 256.
constexpr int kMaxPackedRows = (1 << 24) - 1;
struct TileRows {
    int rows;
    uint32_t inverse;
    __host__ __device__ explicit TileRows(int rows) : rows(rows), inverse(rows > 1 ? static_cast<uint32_t>(((1ull << 32) + rows - 1) / rows) : 0) {}
    FRY_DEVICE int of(int row) const { return rows > 1 ? static_cast<int>(__umulhi(static_cast<uint32_t>(row), inverse)) : row; }
};

// Slots. Segment i has the slots from start(i) / tile + i up to the next segment's: at least as many as its tiles of
// `tile` rows, since start(i + 1) / tile - start(i) / tile + 1 >= ceil(length / tile), and at most one more. So a grid of
// packed_slots(rows, tile, count) blocks holds every tile, and a block finds its segment by a search over the starts
// alone, with no sum over the lengths before it.
__host__ __device__ inline int packed_slots(int rows, int tile, int count) { return rows / tile + count + 2; }

// The last segment i whose first slot is at most `slot`. The warp searches 32 ways at once: two steps up to 1024
// requests. Every lane returns the same segment; for offsets that do not ascend it is some segment.
FRY_DEVICE int find_segment(const PackedRows& packed, const TileRows& tile, int slot, int lane) {
    int low = 0, count = packed.count + 2;
    while (count > 1) {
        const int step = (count + 31) / 32, probe = lane * step;
        const bool reached = probe < count && tile.of(packed.start(low + probe)) + low + probe <= slot;
        const uint32_t votes = __ballot_sync(0xffffffffu, reached);
        const int last = votes == 0 ? 0 : 31 - __clz(votes);
        low += last * step;
        count = min(step, count - last * step);
    }
    return low;
}

}  // namespace fry
