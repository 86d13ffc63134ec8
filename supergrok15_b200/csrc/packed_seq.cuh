// Work items over packed sequences of different lengths, found on the device from the offsets alone: no host copy of the lengths, no
// table built by another launch, the same grid for every layout of one (rows, sequences) pair, so a captured launch follows new offsets.
//
// The rows [0, total) are cut into n + 2 segments by the n + 1 offsets: rows before the first sequence, the sequences, rows behind the
// last one (the first and the last segment belong to no sequence: their outputs are zero).  Segment s gets the slots
// [slot_base(s), slot_base(s + 1)) with slot_base(s) = begin(s) / TILE + s.  That is monotone, leaves every segment at least
// ceil(length / TILE) slots and wastes at most one slot per segment, and a slot finds its segment by a search over the offsets (32-ary,
// one warp) without a prefix sum over tile counts.
//
// The offsets come from the caller and are not read by the host: every one is clamped to [0, total], and a slot that finds no rows is
// empty, so that offsets which do not ascend give wrong rows but never an access out of range.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace sg {

struct PackedSeqs {
    const int* cu;      // n + 1 ascending offsets
    int n, total;
};

__host__ __device__ __forceinline__ int packed_slots(int n, int total, int tile) { return total / tile + n + 2; }

struct PackedTile {
    int lo, hi;         // rows of the segment
    int row0;           // first row of the tile (lo + k * TILE); rows [row0, min(row0 + TILE, hi)) belong to it
    bool live, pad;     // live: the tile has rows; pad: they belong to no sequence
};

#ifdef __CUDACC__
__device__ __forceinline__ int packed_begin(const PackedSeqs& ps, int s) {
    if (s <= 0) return 0;
    if (s > ps.n + 1) return ps.total;
    const int c = __ldg(ps.cu + (s - 1));
    return c < 0 ? 0 : (c > ps.total ? ps.total : c);
}

// The tile of one slot; called by a whole warp, every lane gets the answer.
template <int TILE> __device__ __forceinline__ PackedTile packed_tile(const PackedSeqs& ps, int slot) {
    const int lane = (int)(threadIdx.x & 31);
    int a = 0, b = ps.n + 2;                                              // the segment lies in [a, b)
    while (b - a > 1) {
        const int step = (b - a + 31) / 32, s = a + lane * step;
        const bool le = s < b && packed_begin(ps, s) / TILE + s <= slot;
        const unsigned m = __ballot_sync(0xffffffffu, le);
        const int last = m ? 31 - __clz(m) : 0;
        a += last * step;
        if (a + step < b) b = a + step;
    }
    PackedTile t;
    t.lo = packed_begin(ps, a);
    t.hi = packed_begin(ps, a + 1);
    const int k = slot - (t.lo / TILE + a);
    t.row0 = t.lo + k * TILE;
    t.live = k >= 0 && t.row0 < t.hi;
    t.pad = a == 0 || a == ps.n + 1;
    return t;
}
#endif

}  // namespace sg
