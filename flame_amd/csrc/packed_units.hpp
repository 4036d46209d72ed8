// Sequences of different lengths one behind the other in one tensor: which tile of which sequence and head a workgroup takes, and which
// part of its walk.
//
// Sequence i has the rows [cu[i], cu[i + 1]) (int32 on the device, n + 1 of them, cu[0] taken as 0).  The host knows the number of
// rows and of sequences, not the lengths, so it launches as many workgroups as there can be tiles, and every workgroup finds its own.
//   Up to 64 sequences: a lane holds one.  The tiles come in the order of falling walks, so that the longest start first and what
//   is left at the end is short: under the causal flag tile by tile over all sequences (training on six documents of 333 to 4608, us:
//   sequence by sequence 1543, tile by tile 1515), else sequence by sequence.  On grids that leave compute units idle the walks are cut
//   into parts (PackedCut) whose partial sums a second launch joins.
//   More: in their own order, whole (100 of 16 to 512 rows, 32 heads on 8, D = 128, forward and backward 231 and 736 us; with one of 4096 behind them 357
//   and 1208, before them 372 and 1164).  Every sequence gets the slots [slot(i), slot(i + 1)) with slot(i) = cu[i] / tile + i, at least as many as
//   it has tiles and at most one more, so that a search finds it without a sum over the lengths.
// The rows behind the last sequence are the last tiles of that numbering: their workgroups write zeros.
// Bounds that fall or lead out of the tensor are cut to it: the result is then of no use, but nothing outside is touched.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fattn {

struct PackedUnit {
    int tile = 0;                  // of the sequence
    int Sq = 0, Sk = 0;            // its queries and keys
    int past = 0;                  // Sk - Sq: query i attends to key j <= i + past
    int head = 0, kv_head = 0;     // dK/dV: the first head that shares kv_head
    int rep = 1;                   // heads that share a key head
    int q_row = 0, k_row = 0;      // first rows of the sequence
    int total_q = 0;               // step from head to head in a [heads, all rows] tensor of one float per query
    int unit = 0;                  // number of this unit, and which of up to `parts` parts of its tile's walk it is (steps per part: `share`;
    int part = 0, parts = 1;       // a tile with a shorter walk has fewer)
    int share = 1 << 30;

    // places of the sequence's first row
    __device__ __forceinline__ int64_t stat_row() const { return (int64_t)head * total_q + q_row; }
    template <class S>
    __device__ __forceinline__ int64_t q_at(const S& st) const { return q_row * st.n + head * st.h; }
    template <class S>
    __device__ __forceinline__ int64_t k_at(const S& st) const { return k_row * st.n + kv_head * st.h; }
};

// How walks are cut.  The walks of all `units` tiles together have `steps` steps; the parts are to fill the workgroups that the card holds at
// once, of which the last part of every tile takes half a place on average.  Parts of fewer than 16 steps are `scale` times as long as that
// gives: longer, to leave places for the workgroups of parts that a tile with a shorter walk does not have; shorter, where a compute unit takes a
// second workgroup and has little to do.  At least `least`: a part should not spend its time on loading its rows and leaving its sums.
// Nothing is cut where the longest walk is hardly longer than what each of the 256 compute units has to do anyway: joining the parts
// costs about `gain` steps.
struct PackedCut {
    int room_log2, least, gain;    // log2 of the workgroups that the card holds, 0: whole walks
    float scale;
    static constexpr int kUnits_log2 = 8, kWhole = 1 << 30;
    __host__ __device__ bool pays(int longest, int64_t steps) const { return longest - (int)(steps >> kUnits_log2) > gain; }
    __host__ __device__ int share(int64_t steps, int units) const {
        const int room = 1 << room_log2, places = room - units / 2 > room / 4 ? room - units / 2 : room / 4;
        const float n = (float)steps / (float)places;
        if (n < 16.f) return scale * n < (float)least ? least : scale * n > 16.f ? 16 : (int)(scale * n);
        return n > 1e9f ? 1000000000 : (int)n + 1;
    }
    // units per head, at most, of `slots` tiles: a sequence's longest walk is at most twice the mean that `steps` counts, a part at least half
    // as long as the places give (one more for the rounding of `n`)
    int64_t most(int64_t slots, int heads) const { return slots + (((scale < 1.f ? 4 : 2) << room_log2) + heads - 1) / heads + 1; }
};

struct PackedArgs {
    const int32_t* cu_q;
    const int32_t* cu_k;
    int n;                         // sequences
    int total_q, total_k;          // rows of the tensors
    int H, Hkv;
    int causal;
    PackedCut cut;
};

inline int64_t packed_slots(int total, int n, int tile) { return (int64_t)total / tile + n + 1; }

enum PackedWork : int { kPackedIdle = 0, kPackedTile = 1, kPackedBehind = 2 };

__device__ __forceinline__ int packed_bound(const int32_t* cu, int i, int total) { return i == 0 ? 0 : min(max(cu[i], 0), total); }
// the same value in every lane, which the compiler does not see (loads, divisions): into a scalar register
__device__ __forceinline__ int packed_uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The last i of 0 .. n with slot(i) <= r, which is true of 0, 64 candidates at a time.  Every lane calls this.
template <class F>
__device__ __forceinline__ int packed_find(int n, int r, F&& slot) {
    const int lane = threadIdx.x & 63;
    int lo = 0, count = n + 1;
    while (count > 1) {
        const int step = (count + 63) / 64, at = lo + lane * step;
        const bool ok = lane == 0 || (lane * step < count && slot(at) <= r);
        const int last = 63 - __clzll((long long)__ballot(ok));
        lo += last * step;
        count = min(step, count - last * step);
    }
    return packed_uniform(lo);
}

// Workgroup `block` of slots x heads: an XCD (the workgroups go to them in turn) keeps its own key heads where eight divides their
// number, or its own heads where eight divides that, so that the tiles that read the same keys share an L2.
__device__ __forceinline__ void packed_order(int block, int heads, int per_kv, int& slot, int& head) {
    if (heads % 8 == 0) {
        const int x = block % 8, j = block / 8, mine = heads / 8, i = j % mine;
        slot = j / mine;
        head = heads / per_kv % 8 == 0 ? (x + 8 * (i / per_kv)) * per_kv + i % per_kv : x * mine + i;
    } else {
        slot = block / heads;
        head = block % heads;
    }
}

// sum over the lanes below and including this one
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);      // from 1, 2, 4 and 8 lanes below within 16 lanes
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);     // the last lane of 16 to the next 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);     // lane 31 to lanes 32 .. 63
    return x;
}

// The unit of workgroup `block`: a tile of TILE queries (KEYS: keys, of a key head) of one sequence, and a part of its walk.
// The tiles of a sequence come from the longest walk under the causal flag to the shortest: of queries from the last to the first.
// MERGE: `block` counts tiles, not parts, and the unit is the first part of the tile; u.parts the most it can have.
template <int TILE, bool KEYS, bool MERGE = false>
__device__ __forceinline__ PackedWork packed_unit(const PackedArgs& a, int block, PackedUnit& u) {
    constexpr int STEP = 64;       // rows of a step of the walk
    const int32_t* cu = KEYS ? a.cu_k : a.cu_q;
    const int total = KEYS ? a.total_k : a.total_q;
    const int rep = packed_uniform(a.H / a.Hkv), heads = KEYS ? a.Hkv : a.H;
    int slot, head;
    packed_order(block, heads, KEYS ? 1 : rep, slot, head);
    slot = packed_uniform(slot);
    head = packed_uniform(head);
    u.rep = rep;
    u.head = KEYS ? head * rep : head;
    u.kv_head = KEYS ? head : packed_uniform(head / rep);
    u.total_q = a.total_q;
    int t, n_tiles;                // this unit's tile, counted as the tiles come, and the sequence's
    if (a.n <= 64) {
        const int lane = threadIdx.x & 63;
        int q0 = 0, k0 = 0, Sq = 0, Sk = 0;
        if (lane < a.n) {
            q0 = packed_bound(a.cu_q, lane, a.total_q);
            k0 = packed_bound(a.cu_k, lane, a.total_k);
            Sq = max(packed_bound(a.cu_q, lane + 1, a.total_q) - q0, 0);
            Sk = max(packed_bound(a.cu_k, lane + 1, a.total_k) - k0, 0);
        }
        const int end = packed_uniform(packed_bound(cu, a.n, total));
        const int tiles = ((KEYS ? Sk : Sq) + TILE - 1) / TILE;
        const int walk = ((KEYS ? Sq : Sk) + STEP - 1) / STEP * (KEYS ? rep : 1);
        int parts = 1, share = PackedCut::kWhole;
        if (a.cut.room_log2) {
            // steps of the batch, every sequence's by its mean walk (the causal flag leaves its first tiles little): at least half the longest
            const float cut = a.causal ? 0.5f * (float)min(Sq, Sk) / (float)max(max(Sq, Sk), 1) : 0.f;
            const int64_t mine = (int64_t)tiles * max((walk + 1) / 2, (int)((float)walk * (1.0f - cut)));
            const int low = __builtin_amdgcn_readlane(wave_scan((int)(mine & 0xffffff)), 63), high = __builtin_amdgcn_readlane(wave_scan((int)(mine >> 24)), 63);
            const int64_t steps = (((int64_t)high << 24) + low) * heads;
            int longest = 0;
            for (int j = 0; j < a.n; ++j) longest = max(longest, __builtin_amdgcn_readlane(walk, j));
            if (a.cut.pays(longest, steps)) share = packed_uniform(a.cut.share(steps, __builtin_amdgcn_readlane(wave_scan(tiles), 63) * heads));
            parts = max((walk + share - 1) / share, 1);
        }
        if (MERGE && share == PackedCut::kWhole) return kPackedIdle;
        const int units = tiles * parts;
        int i, at;                 // the lane that has the unit, and the slots before the lane's (whole walks under the causal flag: t itself)
        if (a.causal && share == PackedCut::kWhole) {
            // Every tile of a sequence walks one step of TILE rows less than the one before it, so the t-th of a sequence has the
            // level `longest` - t, and the tiles of all sequences come in the order of falling levels, those of one level by lanes.
            // The level of a slot is found by halving: fewer than slot + 1 tiles lie above it.
            const int longest = (max(Sq, Sk) + TILE - 1) / TILE;
            const auto above = [&](int level) { return __builtin_amdgcn_readlane(wave_scan(min(max(longest - level, 0), tiles)), 63); };
            int lo = -1, hi = (max(a.total_q, a.total_k) + TILE - 1) / TILE;        // above(hi) = 0; above(lo): all (levels start at 1 or, with fewer keys than queries, below)
            const int all = __builtin_amdgcn_readlane(wave_scan(tiles), 63);
            if (slot >= all) {
                i = -1;
                at = all;
            } else {
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (above(mid) > slot) lo = mid;
                    else hi = mid;
                }
                // above(lo) > slot >= above(hi), hi = lo + 1: the slot's tile has level hi
                uint64_t here = __ballot(longest >= hi && longest - hi < tiles);
                for (int k = slot - above(hi); k > 0; --k) here &= here - 1;
                i = __ffsll((unsigned long long)here) - 1;
                at = __builtin_amdgcn_readlane(longest, i) - hi;
            }
        } else {
            int first = 0, first_tile = 0;                                          // units and tiles of the sequences that come before
            for (int j = 0; j < a.n; ++j) {
                const int w = __builtin_amdgcn_readlane(walk, j);
                const bool before = w > walk || (w == walk && j < lane);
                const int units_j = __builtin_amdgcn_readlane(units, j), tiles_j = MERGE ? __builtin_amdgcn_readlane(tiles, j) : 0;
                first += before ? units_j : 0;
                first_tile += before ? tiles_j : 0;
            }
            const int from = MERGE ? first_tile : first, count = MERGE ? tiles : units;
            i = __ffsll((unsigned long long)__ballot(lane < a.n && slot >= from && slot < from + count)) - 1;
            at = i < 0 ? __builtin_amdgcn_readlane(wave_scan(count), 63) : slot - __builtin_amdgcn_readlane(from, i);
            u.unit = i < 0 ? 0 : __builtin_amdgcn_readlane(first, i);
        }
        if (i < 0) {
            u.q_row = u.k_row = end;
            u.Sq = u.Sk = total - end;
            u.tile = slot - at;
            return (int64_t)u.tile * TILE < total - end ? kPackedBehind : kPackedIdle;
        }
        u.Sq = __builtin_amdgcn_readlane(Sq, i);
        u.Sk = __builtin_amdgcn_readlane(Sk, i);
        u.q_row = __builtin_amdgcn_readlane(q0, i);
        u.k_row = __builtin_amdgcn_readlane(k0, i);
        n_tiles = __builtin_amdgcn_readlane(tiles, i);
        u.parts = __builtin_amdgcn_readlane(parts, i);
        u.share = share;
        t = MERGE || u.parts == 1 ? at : packed_uniform(at / u.parts);
        u.part = MERGE ? 0 : at - t * u.parts;
        u.unit = (u.unit + t * u.parts + u.part) * heads + head;
    } else {
        const int i = packed_find(a.n, slot, [&](int at) { return packed_bound(cu, at, total) / TILE + at; });
        const int first = packed_uniform(packed_bound(cu, i, total));
        t = slot - (first / TILE + i);
        if (i == a.n) {
            u.tile = t;
            u.q_row = u.k_row = first;
            u.Sq = u.Sk = total - first;
            return (int64_t)t * TILE < total - first ? kPackedBehind : kPackedIdle;
        }
        u.q_row = packed_uniform(packed_bound(a.cu_q, i, a.total_q));
        u.k_row = packed_uniform(packed_bound(a.cu_k, i, a.total_k));
        u.Sq = packed_uniform(max(packed_bound(a.cu_q, i + 1, a.total_q) - u.q_row, 0));
        u.Sk = packed_uniform(max(packed_bound(a.cu_k, i + 1, a.total_k) - u.k_row, 0));
        n_tiles = ((KEYS ? u.Sk : u.Sq) + TILE - 1) / TILE;
        if (t >= n_tiles) return kPackedIdle;
    }
    u.past = u.Sk - u.Sq;
    u.tile = KEYS ? t : n_tiles - 1 - t;
    return kPackedTile;
}

// The parts that a walk of `steps` steps has, and the steps [lo, hi) of part u.part; part 0 of a walk without steps has none.
__device__ __forceinline__ int packed_parts(const PackedUnit& u, int steps) { return u.parts == 1 ? 1 : max(packed_uniform((steps + u.share - 1) / u.share), 1); }

// Zeros in the rows of one tile behind the last sequence: `first` is row 0 of the unit's head there.
template <int TILE>
__device__ __forceinline__ void packed_zero_rows(uint16_t* first, int64_t row_stride, int tile, int rows, int d) {
    typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
    const int per_row = d / 8, n = min(TILE, rows - tile * TILE);
    for (int i = threadIdx.x; i < n * per_row; i += blockDim.x)
        *reinterpret_cast<u32x4_t*>(first + (int64_t)(tile * TILE + i / per_row) * row_stride + 8 * (i % per_row)) = u32x4_t{0u, 0u, 0u, 0u};
}

}  // namespace fattn
