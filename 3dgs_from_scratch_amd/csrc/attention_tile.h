// What the attention kernels share: sequences in packed rows, tiles of rows in LDS,
// and matrix products over them.
//
// A tile holds rows of one head, DIM elements each (the head's dimension rounded up,
// zeros behind it), in 16-byte chunks.  It is read two ways: along a row, 8 elements
// a lane, as an operand that contracts over the dimension; and down the rows, 4 rows
// a lane, by the LDS's transposed read, as one that contracts over the rows.  The
// chunks of a row are permuted by an exclusive or with a function of the row, so that
// eight lanes at a time meet different banks either way, no more than half of the 64.  Of
// sixteen some meet the same: conflicts are 0.21 to 0.29 of the large launches' cycles.
//
// Products are v_mfma_f32_32x32x16: lane l gives column l % 32 of an operand and 8 of
// its 16 contracted places (half l / 32); of the 32x32 result it holds column l % 32
// and the rows (r & 3) + 8 (r >> 2) + 4 (l / 32).  A result is used again as an operand
// without leaving its lane: registers 8 s to 8 s + 7 hold 8 of the rows 16 s to
// 16 s + 15, and the other operand is read in the same order of rows.
#pragma once

#include "element.h"

namespace gs {

using f32x16 = __attribute__((ext_vector_type(16))) float;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using i16x4 = __attribute__((ext_vector_type(4))) short;
template <typename T>
struct Vec {
    using x4 = __attribute__((ext_vector_type(4))) T;
    using x8 = __attribute__((ext_vector_type(8))) T;
};
typedef __attribute__((address_space(3))) char lds_char;

__device__ __forceinline__ f32x16 mfma(Vec<bf16>::x8 a, Vec<bf16>::x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(Vec<f16>::x8 a, Vec<f16>::x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Rounds to nearest even.
template <typename T>
__device__ __forceinline__ typename Vec<T>::x8 pack8(const float *v) {
    typename Vec<T>::x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)v[i];
    return r;
}

// The sum and the maximum of a column's two halves, in both.
__device__ __forceinline__ float half_sum(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (uint32_t)s[0]) + __builtin_bit_cast(float, (uint32_t)s[1]);
}
__device__ __forceinline__ float half_max(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)s[0]),
                 __builtin_bit_cast(float, (uint32_t)s[1]));
}

// Row of a 32x32 result that a lane of half h holds in register r.
__device__ __forceinline__ constexpr int result_row(int r, int h) {
    return (r & 3) + 8 * (r >> 2) + 4 * h;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ---------------------------------------------------------------- sequences
// Sequence s = 1 .. sequences; 0 and sequences + 1 hold the rows before the first
// offset and after the last, and have no keys, so that every row is in one.  Offsets
// are clamped to the tensors, whatever they say.
__device__ __forceinline__ int clamp_row(int64_t v, int64_t low, int64_t high) {
    return (int)(v < low ? low : v > high ? high : v);
}

__device__ __forceinline__ int2 rows_of(const int32_t *offsets, int sequences, int64_t rows, int s) {
    int2 r;
    r.x = s == 0 ? 0 : clamp_row(offsets[s - 1], 0, rows);
    r.y = s > sequences ? (int)rows : clamp_row(offsets[s], r.x, rows);
    return r;
}

// The keys that count of sequence s, whose key rows are `k`.
__device__ __forceinline__ int keys_of(const GsAttention &a, int s, int2 k) {
    if (s == 0 || s > a.sequences) return 0;
    return a.lengths_k ? clamp_row(a.lengths_k[s - 1], 0, k.y - k.x) : k.y - k.x;
}

struct Span {
    int q0, lq;  // first query row, number of queries
    int k0, lk;  // first key row, number of keys that count
    int k1;      // end of the key rows
};

__device__ __forceinline__ Span span_of(const GsAttention &a, int s) {
    const int2 q = rows_of(a.offsets_q, a.sequences, a.rows_q, s);
    const int2 k = rows_of(a.offsets_k, a.sequences, a.rows_k, s);
    Span p;
    p.q0 = uniform(q.x);
    p.lq = uniform(q.y - q.x);
    p.k0 = uniform(k.x);
    p.k1 = uniform(k.y);
    p.lk = uniform(keys_of(a, s, k));
    return p;
}

// The group (of `groups`) and the place in it of number `number`, where group g has count(g)
// places; numbers count up from the first group's first place or down from the last one's
// last.  Every lane of a wave calls it.  False: there are not so many places.
template <typename Count>
__device__ __forceinline__ bool find_place(int groups, Count count, int number, bool from_back,
                                           int *group, int *place) {
    const int lane = __lane_id();
    int total = 0, sum = 0;
    const auto running = [&](int first) {  // up to and with group first + lane
        sum = first + lane < groups ? count(first + lane) : 0;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const int t = __shfl_up(sum, o, kWave);
            if (lane >= o) sum += t;
        }
        // (uniform, also to the compiler: what is found here addresses whole waves' copies)
        return uniform(__shfl(sum, kWave - 1, kWave));
    };
    for (int first = 0; first < groups; first += kWave) total += running(first);
    if (number >= total) return false;
    int want = from_back ? total - 1 - number : number;
    for (int first = 0; first < groups; first += kWave) {
        const int here = groups > kWave ? running(first) : total;
        if (want < here) {
            const int l = __ffsll((unsigned long long)__ballot(sum > want)) - 1;
            const int before = l ? __shfl(sum, l - 1, kWave) : 0;
            *group = uniform(first + l);
            *place = uniform(want - before);
            return true;
        }
        want -= here;
    }
    return false;
}

// The sequence and the tile in it of a launch's tile number, tiles of `size` units,
// `units` units a row.  Counted from the back on request: under a causal mask the last
// queries see most, and should start first.
__device__ __forceinline__ bool find_tile(const int32_t *offsets, int sequences, int64_t rows,
                                          int units, int size, int number, bool from_back,
                                          int *sequence, int *tile) {
    const auto count = [&](int s) {
        const int2 r = rows_of(offsets, sequences, rows, s);
        return (int)(((int64_t)(r.y - r.x) * units + size - 1) / size);
    };
    return find_place(sequences + 2, count, number, from_back, sequence, tile);
}

// -------------------------------------------------------------------- tiles
// The workgroup's copies into LDS that were started before are done, and its reads of LDS
// too.  A barrier alone does not wait for copies: to the compiler they are loads whose
// results nobody has asked for.
__device__ __forceinline__ void copies_done() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Four rows of the column that this lane gets of its 16 lanes' 4 x 16 block.  Without the
// restrict the compiler takes any copy to LDS that is under way for one to this address,
// and waits for the next tile's before the first such read of this one; copies_done() at a
// tile's start is what orders them.
typedef __attribute__((address_space(3))) i16x4 lds_x4;
__device__ __forceinline__ i16x4 transposed(const lds_x4 *__restrict__ p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_x4 *)p);
}

constexpr int64_t kMaxStride = 1 << 23;  // of rows, elements

template <typename T, int DIM, int ROWS, int WAVES>
struct Tile {
    // byte offsets and the bound in start() stay in 31 bits, below copy_of()'s mark
    static_assert(((ROWS - 1) * kMaxStride + DIM) * 2 < (1LL << 31), "offsets of a copy");
    static constexpr int kChunks = DIM / 8;                      // of a row
    static constexpr int kBytes = ROWS * DIM * 2;
    static constexpr int kPieces = ROWS * kChunks / 64;  // of 1 KiB, which a wave copies at once
    static constexpr int kCopies = (kPieces + WAVES - 1) / WAVES;  // of a wave
    static_assert(ROWS * kChunks % 64 == 0, "whole waves of chunks");
    using x8 = typename Vec<T>::x8;

    // Row r's chunk c lies at chunk c ^ swizzle(r); the same for row r + 8.
    static __device__ __forceinline__ constexpr int swizzle(int r) {
        return DIM == 128 ? (r & 7) << 1
               : DIM == 64 ? ((r >> 1) & 3) << 1
                           : (r >> 2) & 1;
    }

    // Byte offsets, from the tile's first row in memory, of the chunks that this lane
    // copies; past every bound where the chunk lies behind the dimension.
    struct Copy {
        uint32_t from[kCopies];
    };
    static __device__ __forceinline__ Copy copy_of(int wave, int64_t stride, int dim) {
        Copy c;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int at = (i * WAVES + wave) * 64 + __lane_id();
            const int row = at / kChunks, chunk = (at % kChunks) ^ swizzle(row);
            c.from[i] = chunk * 8 < dim ? (uint32_t)(row * (int)stride + chunk * 8) * 2u
                                        : 0x80000000u;
        }
        return c;
    }

    // Starts this wave's part of the copy of `rows` rows (the rest become zeros) into
    // LDS.  The descriptor's bound ends behind the last row: what lies past it is
    // read as zeros, and not touched.
    static __device__ __forceinline__ void start(const Copy &c, int wave, const T *first,
                                                 int64_t stride, int rows, int dim,
                                                 lds_char *tile) {
        const int n = rows < ROWS ? rows : ROWS;
        const int bytes = n > 0 ? ((n - 1) * (int)stride + dim) * 2 : 0;
        const auto from = __builtin_amdgcn_make_buffer_rsrc((void *)first, 0, bytes, 0x00027000);
#pragma unroll
        for (int i = 0; i < kCopies; ++i)
            if (kPieces % WAVES == 0 || i * WAVES + wave < kPieces)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    from, (__attribute__((address_space(3))) void *)(tile + (i * WAVES + wave) * 1024),
                    16, c.from[i], 0, 0, 0);
    }

    // Starts the copy of one float a row (64 rows, `present` of them in memory, the rest
    // become zeros); one wave does it.
    static __device__ __forceinline__ void start_floats(const float *first, int present,
                                                        lds_char *to) {
        const int n = uniform(present < 0 ? 0 : present < 64 ? present : 64);
        const auto from = __builtin_amdgcn_make_buffer_rsrc((void *)first, 0, n * 4, 0x00027000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            from, (__attribute__((address_space(3))) void *)to, 4, __lane_id() * 4, 0, 0, 0);
    }

    // Operand that contracts over the dimension: row `base` + l % 32, places 16 s + 8 (l / 32).
    static __device__ __forceinline__ x8 along(const lds_char *tile, int base, int s) {
        const int l = __lane_id(), row = l & 31;
        const int chunk = (2 * s + (l >> 5)) ^ swizzle(row);
        return *(const __attribute__((address_space(3))) x8 *)(tile + base * DIM * 2 +
                                                                row * DIM * 2 + chunk * 16);
    }

    // Operand that contracts over rows base .. base + 15 in the order of a result's
    // registers: column 32 d + l % 32, rows base + 4 (l / 32) + 0..3 and + 8..11.
    static __device__ __forceinline__ x8 down(const lds_char *tile, int base, int d) {
        const int l = __lane_id();
        const int row = 4 * (l >> 5) + ((l & 15) >> 2);
        const int chunk = (4 * d + ((l >> 4) & 1) * 2 + ((l & 3) >> 1)) ^ swizzle(row);
        const lds_char *p = tile + base * DIM * 2 + row * DIM * 2 + chunk * 16 + (l & 1) * 8;
        const int next = 8 * DIM * 2;
        const i16x4 lo = transposed((const lds_x4 *)p), hi = transposed((const lds_x4 *)(p + next));
        const auto both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(x8, both);
    }
};

}  // namespace gs
