// Rows to the pages of a cache in 8 bits and back (kv_codes.hpp).
//
// A block of T tokens of one head has a scale.  The largest magnitude a of the rows that a call brings to a block decides it:
//   rows from the block's first token on:  s = a / Q rounded up to four significant bits, at least 2^-100 (Q: the largest code)
//   rows behind older tokens:              s' = s 2^k with the least k >= 0 such that a <= Q s', and the older codes c become c 2^-k, rounded
//   a not finite, or s none that a store has left:  NaN, which every answer that attends to the block then is
// and a number x becomes x / s, rounded to the nearest code, the even one of two.
// Growing by powers of two, a block's codes are off by less than one of its last steps however often it grew: 1/2 + 1/4 + ...; by the ratio that
// a needs they would drift by half a step each time.  What a block holds behind the new rows counts as not stored: its codes stay and its scale does not.
// Four bits of s make the steps of int8 up to an eighth wider than a / Q would (4 % on average over the fractions of a), and give this: x has
// eight significant bits, so x / s either is a border between two codes or is 2^-15 away from it, and fp32 arithmetic finds the same codes as exact
// arithmetic.
#pragma once
#include "kv_codes.hpp"
#include "packed_units.hpp"

namespace fattn {

// Which sequence has a slot, its rows and its first place.  slot(row, i): of sequence i, whose first row is `row`; rising.  ONE: all lanes of the
// wavefront ask for the same slot.  Up to 64 sequences a lane holds the bound and the first place of one, so that all is known after one way to memory;
// more are searched.  Every lane calls this; b = n: behind the last one.
struct KvSequence {
    int b, row0, next;             // next: row behind its last one
    int start;
};
template <bool ONE, class F>
__device__ __forceinline__ KvSequence kv_sequence(const int32_t* cu, const int32_t* start, int n, int rows, int wanted, F&& slot) {
    const int lane = threadIdx.x & 63;
    KvSequence q;
    if (n <= 64) {
        const int held = min(lane, n - 1), mine = packed_bound(cu, held, rows), first = start[held], end = packed_bound(cu, n, rows), at = slot(mine, lane);
        if (ONE) {
            q.b = __popcll(__ballot(lane >= 1 && lane < n && at <= wanted));
        } else {
            q.b = 0;
            for (int i = 1; i < n; ++i) q.b += __builtin_amdgcn_readlane(at, i) <= wanted;
        }
        q.row0 = __shfl(mine, q.b, 64);
        q.next = q.b + 1 < n ? __shfl(mine, min(q.b + 1, n - 1), 64) : end;
        q.start = __shfl(first, q.b, 64);
        if (slot(end, n) <= wanted) q.b = n;
        return q;
    }
    const int lowest = packed_uniform(wanted);         // (the first lane has the lowest slot)
    q.b = packed_find(n, lowest, [&](int i) { return slot(packed_bound(cu, i, rows), i); });
    if (!ONE)
        while (q.b < n && slot(packed_bound(cu, q.b + 1, rows), q.b + 1) <= wanted) ++q.b;
    const int b = min(q.b, n - 1);
    q.row0 = packed_bound(cu, b, rows);
    q.next = packed_bound(cu, b + 1, rows);
    q.start = start[b];
    return q;
}

struct KvStore8Params {
    const uint16_t* x[2];          // K and V: [rows][Hkv][d] through xs (n: row, h: head)
    uint8_t* c[2];                 // [pages][Hkv][page][d] through cs (b: page, h: head, n: token; bytes)
    float* s[2];                   // [pages][Hkv][page / T] through ss (b: page, h: head, n: block)
    Strides xs[2], cs[2], ss[2];
    const int32_t* table;
    int64_t table_stride;
    int table_pages;
    const int32_t* cu;             // [n + 1]: rows of the sequences
    const int32_t* start;          // [n]: place of a sequence's first row in its pages
    int n, rows, Hkv, d, n_pages, page_shift, block_shift;
    int slot_groups;               // groups of threads per slot, at most 2 Hkv: group i has its units i, i + slot_groups, ...
    uint32_t groups;
};

// Slots for the blocks that sequences write to, at least as many as there can be: [slot(i), slot(i + 1)).  n rows touch at most n / T + 2 blocks of
// T > 1 tokens.
__host__ __device__ inline int64_t kv_store8_slot(int64_t first_row, int i, int block_shift) {
    return (first_row >> block_shift) + (block_shift ? 2 * (int64_t)i : 0);
}

// LANES threads per unit, which is a block of one head of K or of V, with E granules of 8 numbers each, one unit after the other where there are
// many (`per`): the search and the page are found once.  Neighbouring threads have neighbouring heads.
// Bound by memory and, for few rows, by the chain of bounds, table, old scale and rows.  (7759 rows, 8 heads, D = 128, blocks of 16: 11.7 us, of 1: 20.3 with one
// unit each.  32768 rows, blocks of 16: 41 us, 4.9 TB/s.)
template <int CODE, int LANES, int E>
static __global__ __launch_bounds__(256) void kv_store8_kernel(const KvStore8Params p) {
    constexpr float Q = kLargestCode<CODE>;
    const uint32_t group = (blockIdx.x * 256u + threadIdx.x) / LANES, group0 = __builtin_amdgcn_readfirstlane(group);
    const int lane = threadIdx.x & (LANES - 1);
    __shared__ uint32_t tops[4];
    if (LANES <= 64 && group0 >= p.groups) return;     // (a workgroup of one unit: always below)
    const uint32_t at = min(group, p.groups - 1u), slot_groups = (uint32_t)p.slot_groups;
    const int slot = (int)(at / slot_groups), first_unit = (int)(at - (uint32_t)slot * slot_groups);
    auto slot_of = [&](int row, int i) { return (int)kv_store8_slot(row, i, p.block_shift); };
    const KvSequence q = kv_sequence<(LANES >= 64)>(p.cu, p.start, p.n, p.rows, slot, slot_of);
    // the block of this group: tokens [lo, hi) of the sequence are new in it
    const int64_t start = q.start, end = start + max(q.next - q.row0, 0);
    const int64_t begin = ((start >> p.block_shift) + (slot - slot_of(q.row0, q.b))) * (int64_t(1) << p.block_shift);
    const int64_t lo = max(start, begin), hi = min(end, begin + (1 << p.block_shift));
    const bool rows = group < p.groups && q.b < p.n && lo < hi;
    int page = -1;
    if (rows && begin >= 0 && (begin >> p.page_shift) < p.table_pages) page = p.table[q.b * p.table_stride + (begin >> p.page_shift)];
    const int per_row = p.d / 8, n = rows ? (int)(hi - lo) * per_row : 0;
    // granule lane + i LANES of the rows: row and number in the row, from one to the next without a division
    const int row_step = LANES / per_row, column_step = LANES - row_step * per_row, row_first = lane / per_row, column_first = lane - row_first * per_row;
    auto advance = [&](int& row, int& column) {
        row += row_step;
        column += column_step;
        if (column >= per_row) {
            column -= per_row;
            ++row;
        }
    };
    const int token0 = (int)(begin & ((1 << p.page_shift) - 1)), old = (int)(lo - begin);
    for (int number = first_unit; number < 2 * p.Hkv; number += p.slot_groups) {
        const int which = number >= p.Hkv, head = number - (which ? p.Hkv : 0);
        // the rows are on their way before the page is known
        const uint16_t* const x = (which ? p.x[1] : p.x[0]) + head * (which ? p.xs[1].h : p.xs[0].h) + (q.row0 + (lo - start)) * (which ? p.xs[1].n : p.xs[0].n);
        const int64_t x_row = which ? p.xs[1].n : p.xs[0].n, c_row = which ? p.cs[1].n : p.cs[0].n;
        u32x4 w[E];
        uint32_t top = 0;                                  // two magnitudes, as whole numbers: what is not finite is larger than all others
#pragma unroll
        for (int i = 0, row = row_first, column = column_first; i < E; ++i, advance(row, column)) {
            w[i] = u32x4{0u, 0u, 0u, 0u};
            if (lane + i * LANES < n) w[i] = *reinterpret_cast<const u32x4*>(x + row * x_row + 8 * column);
        }
        const bool there = page >= 0 && page < p.n_pages;
        if (LANES <= 64 && !there) return;                 // (a group's lanes leave together)
        uint8_t* const c = (which ? p.c[1] : p.c[0]) + page * (which ? p.cs[1].b : p.cs[0].b) + head * (which ? p.cs[1].h : p.cs[0].h) + token0 * c_row;
        float* const scale = (which ? p.s[1] : p.s[0]) + page * (which ? p.ss[1].b : p.ss[0].b) + head * (which ? p.ss[1].h : p.ss[0].h) +
                             (token0 >> p.block_shift) * (which ? p.ss[1].n : p.ss[0].n);
        const float s_old = there && old ? *scale : 0.f;
        auto higher = [](uint32_t a, uint32_t b) {
            typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
            return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
        };
#pragma unroll
        for (int i = 0; i < E; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) top = higher(top, w[i][j] & 0x7fff7fffu);
#pragma unroll
        for (int m = 1; m < (LANES < 64 ? LANES : 64); m *= 2) top = higher(top, (uint32_t)__shfl_xor((int)top, m, 64));
        if constexpr (LANES > 64) {
            if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
            __syncthreads();
            top = higher(higher(tops[0], tops[1]), higher(tops[2], tops[3]));
            if (!there) return;                            // (the whole workgroup)
        }
        top = max(top & 0xffffu, top >> 16);
        const float a = __builtin_bit_cast(float, top << 16);
        float s;
        int grow = 0;
        bool lost = top >= 0x7f80u;
        if (old == 0) {
            s = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, a / Q) + 0xfffffu) & ~0xfffffu);
            s = fmaxf(s, kLeastScale);
        } else {
            lost |= !(s_old >= kLeastScale && s_old <= 3.4e38f);
            if (!lost && a > Q * s_old) {
                // a <= Q s_old 2^k, by fractions and exponents: their quotient may lie outside of fp32 (2^221 for a block of zeros)
                int e_new, e_old;
                const float m_new = __builtin_frexpf(a, &e_new), m_old = __builtin_frexpf(Q * s_old, &e_old);
                grow = e_new - e_old + (m_new > m_old);
            }
            s = __builtin_ldexpf(s_old, grow);
        }
        if (lost) s = 1.f;
        const float r = 1.0f / s;
        auto quotient = [&](float v) {                     // v / s, correctly rounded where that is a border of the codes
            const float q = v * r;
            return fmaf(fmaf(-q, s, v), r, q);
        };
#pragma unroll
        for (int i = 0, row = row_first, column = column_first; i < E; ++i, advance(row, column)) {
            if (lane + i * LANES >= n) continue;
            u32x2 out;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                out[j] = lost ? 0u : f32_to_codes<CODE>(quotient(bf16_lo(w[i][2 * j])), quotient(bf16_hi(w[i][2 * j])), quotient(bf16_lo(w[i][2 * j + 1])),
                                                        quotient(bf16_hi(w[i][2 * j + 1])));
            *reinterpret_cast<u32x2*>(c + (old + row) * c_row + 8 * column) = out;
        }
        if (grow > 0 && !lost) {                           // the older tokens' codes
            const float f = __builtin_ldexpf(1.0f, -grow);
            for (int g = lane; g < old * per_row; g += LANES) {
                const int row = g / per_row;
                u32x2* const place = reinterpret_cast<u32x2*>(c + row * c_row + 8 * (g - row * per_row));
                u32x2 v = *place;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const f32x4 y = codes_to_f32<CODE>(v[j]);
                    v[j] = f32_to_codes<CODE>(y[0] * f, y[1] * f, y[2] * f, y[3] * f);
                }
                *place = v;
            }
        }
        if (lane == 0) *scale = lost ? __builtin_nanf("") : s;
        if (LANES > 64) __syncthreads();               // (`tops` of the next unit)
    }
}

struct KvLoadParams {
    const void* c[2];              // K and V: [pages][Hkv][page][d] through cs (b: page, h: head, n: token)
    const float* s[2];             // scales of codes, or null: bf16
    uint16_t* y[2];                // [rows][Hkv][d] through ys (n: row, h: head)
    Strides cs[2], ss[2], ys[2];
    const int32_t* table;
    int64_t table_stride;
    int table_pages;
    const int32_t* cu;             // [n + 1]: rows of the sequences
    const int32_t* start;          // [n]: place of a sequence's first row in its pages
    int n, rows, Hkv, d, n_pages, page_shift, block_shift;
    int rows_per_wave;
};

// CODE < 0: bf16.  A wavefront takes one row, all heads of K and V, 16 bytes of the cache per lane and access, or as many rows as make 64 accesses.
// Rows behind the last sequence are zeros, a row without a place in the cache is NaN.
template <int CODE>
static __global__ __launch_bounds__(256) void kv_load_kernel(const KvLoadParams p) {
    constexpr int PER = CODE < 0 ? 8 : 16;             // numbers in 16 bytes
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r0 = ((int)blockIdx.x * 4 + wave) * p.rows_per_wave;
    if (r0 >= p.rows) return;
    const int per_row = p.d / PER, n = p.Hkv * per_row, together = min(n, 64), sub = lane / together, r = r0 + sub;
    auto slot_of = [](int row, int) { return row; };
    const KvSequence q = p.rows_per_wave == 1 ? kv_sequence<true>(p.cu, p.start, p.n, p.rows, r0, slot_of) : kv_sequence<false>(p.cu, p.start, p.n, p.rows, r, slot_of);
    if (sub >= p.rows_per_wave || r >= p.rows) return;
    const bool behind = q.b >= p.n;
    int page = -1;
    int64_t pos = 0;
    if (!behind) {
        pos = (int64_t)q.start + (r - q.row0);
        if (pos >= 0 && (pos >> p.page_shift) < p.table_pages) page = p.table[q.b * p.table_stride + (pos >> p.page_shift)];
    }
    const bool there = page >= 0 && page < p.n_pages;
    const int token = (int)(pos & ((1 << p.page_shift) - 1));
    const uint32_t other = behind ? 0u : 0x7fc07fc0u;
    for (int e = lane - sub * together; e < n; e += together) {
        const int h = e / per_row, col = PER * (e - h * per_row);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            uint16_t* const to = p.y[t] + r * p.ys[t].n + h * p.ys[t].h + col;
            u32x4 w = u32x4{other, other, other, other}, more = w;
            if (there) {
                const int64_t from = page * p.cs[t].b + h * p.cs[t].h + token * p.cs[t].n + col;
                if constexpr (CODE < 0) {
                    w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p.c[t]) + from);
                } else {
                    const u32x4 c = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(p.c[t]) + from);
                    const float s = p.s[t][page * p.ss[t].b + h * p.ss[t].h + (token >> p.block_shift) * p.ss[t].n];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4 v = codes_to_f32<CODE>(c[i]);
                        (i < 2 ? w : more)[2 * (i & 1)] = pack_bf16(v[0] * s, v[1] * s);
                        (i < 2 ? w : more)[2 * (i & 1) + 1] = pack_bf16(v[2] * s, v[3] * s);
                    }
                }
            }
            *reinterpret_cast<u32x4*>(to) = w;
            if constexpr (CODE >= 0) *reinterpret_cast<u32x4*>(to + 8) = more;
        }
    }
}

}  // namespace fattn
