// The forward pass of attention, one pass over the keys with a running maximum and sum, for
// kernels whose keys and values lie in packed rows or in pages: a source of keys says how many a
// sequence has and copies tiles of them into LDS.
#pragma once

#include <cfloat>
#include <type_traits>

#include "attention_tile.h"

namespace gs {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kWaves = 4;
constexpr int kKeysWaves = 2;  // where the waves share the rows

// Factor of a raw score in the exponent of two.  A negative scale turns the queries'
// sign instead, so that a row's maximum is that of its raw scores; 0 becomes the
// smallest normal number, so that a masked -infinity stays one.
__host__ __device__ __forceinline__ float exponent_factor(float scale) {
    return fmaxf(fabsf(scale) * kLog2e, 1.17549435e-38f);
}

// Query (or output gradient) operand of one packed row, straight from memory.
template <typename T, int DIM>
struct RowOperand {
    typename Vec<T>::x8 x[DIM / 16];
    // row: the lane's row, or null for zeros
    __device__ __forceinline__ void load(const T *row, int dim, bool negate) {
        const int h = __lane_id() >> 5;
#pragma unroll
        for (int s = 0; s < DIM / 16; ++s) {
            u32x4 v = {0, 0, 0, 0};
            if (row && 16 * s + 8 * h < dim) v = *(const u32x4 *)(row + 16 * s + 8 * h);
            if (negate) v ^= 0x80008000u;
            x[s] = __builtin_bit_cast(typename Vec<T>::x8, v);
        }
    }
};

// 32x32 results of a wave's 32 columns, DIM rows in all, written as 16-bit rows of the
// columns' own addresses (none where that is null); with_rest: to `rest` what the rounding
// took away.  Every lane calls it, with the same with_rest.
template <typename T, int DIM>
__device__ __forceinline__ void store_columns(const f32x16 *acc, float factor, T *row, int dim,
                                              bool with_rest = false, T *rest = nullptr) {
    const int h = __lane_id() >> 5;
    // a half holds rows 4 h + 0..3 and 8 + 4 h + 0..3; after the exchange half h holds
    // 8 h + 0..7
    const auto put = [&](T *to, const float *v, int at) {
        const u32x4 w = __builtin_bit_cast(u32x4, pack8<T>(v));
        const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
        const auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
        const u32x4 o = {(uint32_t)a[0], (uint32_t)b[0], (uint32_t)a[1], (uint32_t)b[1]};
        if (to && at < dim) *(u32x4 *)(to + at) = o;
    };
#pragma unroll
    for (int d = 0; d < DIM / 32; ++d) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {  // registers 8 g to 8 g + 7: rows 16 g + ...
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = acc[d][8 * g + i] * factor;
            const int at = 32 * d + 16 * g + 8 * h;
            put(row, v, at);
            if (with_rest) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] -= to_float(from_float<T>(v[i]));
                put(rest, v, at);
            }
        }
    }
}

// Infinities and NaN in rows of a tile that some columns do not see: their weights there are
// 0, but 0 times them is no 0.  Tiles at a causal edge are looked through for such rows; where
// there are any, the product takes zeros for these values, and a second one counts which of
// them each sum has: 1 an infinity, 64 a negative one, 2048 a NaN, and 2048 times that where the
// weight is 0, among 16 rows.  The sum becomes what the product itself gives in other tiles: an
// infinity, or NaN for a NaN, a weight of 0 and infinities of both signs.
using u16x8 = __attribute__((ext_vector_type(8))) uint16_t;

template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t bits) {
    constexpr uint32_t kInfinity = std::is_same<T, bf16>::value ? 0x7f80 : 0x7c00;
    return (bits & 0x7fff) >= kInfinity;
}

// The rows from `base` on, ROWS of them, that hold such a value: a bit each, in every lane.
template <typename T, int DIM, int ROWS>
__device__ __forceinline__ uint64_t rows_not_finite(const lds_char *tile, int base) {
    constexpr int kChunks = DIM / 8;
    const int row = __lane_id() % ROWS;
    const lds_char *p = tile + (base + row) * DIM * 2;
    int chunk = row % kChunks;  // each lane begins elsewhere: other banks
    // (or the compiler would keep all the chunks' addresses from tile to tile, and registers that
    // the products need would lie in memory)
    asm volatile("" : "+v"(chunk));
    u16x8 most = {};
    for (int i = 0; i < kChunks; ++i) {
        const u16x8 x = *(const __attribute__((address_space(3))) u16x8 *)(p + chunk * 16);
        most = __builtin_elementwise_max(most, x & (uint16_t)0x7fff);
        chunk = chunk + 1 == kChunks ? 0 : chunk + 1;
    }
    uint16_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = most[i] > m ? most[i] : m;
    const uint64_t found = __ballot(not_finite<T>(m));
    return ROWS == 64 ? found : found & 0xffffffffull;
}

// acc += X^T P over 32 rows of a tile X from `base`, P in two operands of 16 rows.
template <typename T, int DIM, typename XTile>
__device__ __forceinline__ void add_product(f32x16 *acc, const lds_char *tile, int base,
                                            const typename Vec<T>::x8 *p,
                                            const typename Vec<T>::x8 *rest = nullptr) {
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d) {
            const typename Vec<T>::x8 x = XTile::down(tile, base + 16 * g, d);
            acc[d] = mfma(x, p[g], acc[d]);
            if (rest) acc[d] = mfma(x, rest[g], acc[d]);
        }
}

// Eight elements, told apart; what: 0 finite, 1 an infinity, more NaN.
template <typename T>
struct Told {
    using x8 = typename Vec<T>::x8;
    static constexpr bool kBf16 = std::is_same<T, bf16>::value;
    static constexpr uint16_t kExponent = kBf16 ? 0x80 : 0x400;  // the last bit of an exponent
    static constexpr uint16_t kOne = (kBf16 ? 127 : 15) * kExponent;          // 1.0
    static constexpr uint16_t kLast = (kBf16 ? 255 : 31) * kExponent - 1;  // the largest number
    u16x8 bits, what, bad;
    __device__ __forceinline__ Told(x8 x) {
        bits = __builtin_bit_cast(u16x8, x);
        const u16x8 last = kLast;
        what = __builtin_elementwise_max(bits & (uint16_t)0x7fff, last) - last;
        bad = __builtin_elementwise_min(what, (u16x8)(uint16_t)1);
    }
    __device__ __forceinline__ x8 finite() const {  // zeros for the others
        return __builtin_bit_cast(x8, bits & (bad - (uint16_t)1));
    }
    __device__ __forceinline__ bool any() const {  // of all lanes'
        const u32x4 b = __builtin_bit_cast(u32x4, bad);
        return __ballot((b[0] | b[1] | b[2] | b[3]) != 0) != 0;
    }
    __device__ __forceinline__ x8 ones() const { return __builtin_bit_cast(x8, bad * kOne); }
    __device__ __forceinline__ x8 kinds() const {  // 0, 1, 64 or 2048 each
        const u16x8 nan = __builtin_elementwise_min(what - bad, (u16x8)(uint16_t)1);
        return __builtin_bit_cast(x8, bad * kOne + (bits >> 15 & (bad - nan)) * (uint16_t)(6 * kExponent) +
                                          nan * (uint16_t)(11 * kExponent));
    }
};

__device__ __forceinline__ void add_infinities(f32x16 &acc, const f32x16 &count) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const float c = count[r];
        // what is left of c without its multiple of 64: the infinities that are positive
        const float up = c - 64.0f * floorf(c * (1.0f / 64.0f));
        acc[r] += up > 0.0f ? INFINITY : 0.0f;
        acc[r] -= c - up > 0.0f ? INFINITY : 0.0f;
        acc[r] = c < 2048.0f ? acc[r] : NAN;
    }
}

// add_product where the rows hold infinities or NaN; sees(i): whether the lane's column sees row
// base + i.  SCORES: the rows made the weights' scores, so that a value that is not finite has
// made its weight 0 or NaN, and the sum NaN.
template <typename T, int DIM, typename XTile, bool SCORES, typename Sees>
__device__ __forceinline__ void add_product_seen(f32x16 *acc, const lds_char *tile, int base,
                                                 const typename Vec<T>::x8 *p, Sees sees,
                                                 const typename Vec<T>::x8 *rest = nullptr) {
    using x8 = typename Vec<T>::x8;
    const int half = __lane_id() >> 5;
#pragma unroll 1
    for (int g = 0; g < 2; ++g) {
        const x8 weights = g ? p[1] : p[0];
        x8 more = weights;
        if (rest) more = g ? rest[1] : rest[0];
        x8 seen;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            seen[j] = (T)(!sees(16 * g + result_row(j, half))  ? 0.0f
                          : (T)weights[j] == (T)0.0f ? 2048.0f
                                                     : 1.0f);
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d) {
            const Told<T> x(XTile::down(tile, base + 16 * g, d));
            acc[d] = mfma(x.finite(), weights, acc[d]);
            if (rest) acc[d] = mfma(x.finite(), more, acc[d]);
            if (!x.any()) continue;
            if constexpr (SCORES) {
                const f32x16 count = mfma(x.ones(), seen, f32x16{});
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] = count[r] > 0.0f ? NAN : acc[d][r];
            } else {
                add_infinities(acc[d], mfma(x.kinds(), seen, f32x16{}));
            }
        }
    }
}

// What the infinities and NaN of ROWS rows of a tile add to a product, by itself; no weight is
// taken for 0.
template <typename T, int DIM, typename XTile, int ROWS, typename Sees>
__device__ __forceinline__ void add_infinities_seen(f32x16 *acc, const lds_char *tile, Sees sees) {
    const int half = __lane_id() >> 5;
#pragma unroll 1
    for (int base = 0; base < ROWS; base += 16) {
        typename Vec<T>::x8 seen;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            seen[j] = (T)(sees(base + result_row(j, half)) ? 1.0f : 0.0f);
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d) {
            const Told<T> x(XTile::down(tile, base, d));
            if (x.any()) add_infinities(acc[d], mfma(x.kinds(), seen, f32x16{}));
        }
    }
}

// sum + the 8 rounded weights.
template <typename T>
__device__ __forceinline__ float add_weights(const typename Vec<T>::x8 &w, float sum) {
    const u32x4 pairs = __builtin_bit_cast(u32x4, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t pair = pairs[i];
        if constexpr (std::is_same<T, f16>::value) {
            using Two = __attribute__((ext_vector_type(2))) f16;
            sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(Two, pair), Two{(f16)1.0f, (f16)1.0f},
                                         sum, false);
        } else {
            using Two = __attribute__((ext_vector_type(2))) short;
            sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(Two, pair),
                                                  Two{0x3f80, 0x3f80}, sum, false);
        }
    }
    return sum;
}

// The same, not rounded, for a sum that is joined later.
template <int DIM>
__device__ __forceinline__ void store_partial(const f32x16 *acc, float factor, float *row, int dim) {
    const int half = __lane_id() >> 5;
#pragma unroll
    for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int column = 32 * d + result_row(4 * g, half);
            if (row && column < dim)
                *(float4 *)(row + column) =
                    make_float4(acc[d][4 * g] * factor, acc[d][4 * g + 1] * factor,
                                acc[d][4 * g + 2] * factor, acc[d][4 * g + 3] * factor);
        }
}

// A workgroup's place in its launch: splits of a tile next to each other, so that the longest
// tiles start first, and key heads innermost: workgroups go to the eight XCDs in turn, and
// with 8 or a divisor of 8 key heads an XCD's L2 holds one of them.
struct Place {
    int kh, split, tile;
};
__device__ __forceinline__ Place place_of(int heads_k, int splits) {
    const int rest = blockIdx.x / heads_k;
    return {(int)blockIdx.x % heads_k, rest % splits, rest / splits};
}

// Forward.  A workgroup takes a tile of packed rows of one key head (row r of a
// sequence: query r / group, head r % group of the group) and walks the sequence's
// keys, or a split's part of them, once:
//   S^T = K Q^T,  P = exp2(c S - m),  O^T += V^T P^T
// with a row in a lane pair, so that the softmax needs one exchange and the factors
// that follow a new maximum none.  K and V go from memory into LDS beside the work on
// the tile before.  BY_KEYS: a few rows only; the waves share the rows and split the
// keys of a tile, and join at the end.
//
// Bound by the matrix units and by LDS at once: a wave's 32 rows read all of a tile of K and
// V, so LDS is busy 80 to 93% of the time, and under that load the clock falls to 1.7 to 1.9
// GHz.  128 rows a workgroup and two of them a CU are what 160 KB of LDS and 256 registers a
// lane hold at 128 dimensions.  16320 rows and keys, 16 heads on 4, dim 128, bfloat16: 2.05
// to 2.15 ms, 1.01 to 1.06 PFLOP/s; 7 causal sequences of 1 to 8160: 0.29 ms, 0.94.
//
// Weights are rounded to the inputs' type for their product with V: 2^-9 (2^-12 in float16)
// of a weight, unbiased.  Infinities and NaN in rows that nothing sees change nothing; a
// query that sees one in V gets it where its column holds it (NaN where the weight was rounded
// to 0 or infinities of both signs meet), a tile with both kinds of query is told apart key by
// key; what a seen K holds goes into its score.
template <typename T, int DIM, bool BY_KEYS>
struct Forward {
    // by keys: two waves, so that a CU's LDS holds two workgroups, and one's first tile and
    // join pass beside the other's reads
    static constexpr int kWaves = BY_KEYS ? kKeysWaves : gs::kWaves;
    static constexpr int kSub = BY_KEYS ? 1 : 2;                    // 32-key parts of a wave
    static constexpr int kKeys = BY_KEYS ? 32 * kWaves : 32 * kSub;  // of a tile
    static constexpr int kRows = BY_KEYS ? 32 : 32 * kWaves;
    using KTile = Tile<T, DIM, kKeys, kWaves>;
    static constexpr int kLds = 4 * KTile::kBytes;
    static_assert(!BY_KEYS || kLds >= kWaves * 64 * (DIM / 2 * 4 + 8), "the join");
};

// Parts of the keys of a row that other workgroups have: un-normalised sums, and their
// maximum and sum of weights.
struct Partial {
    float *sums;      // (split, row, head, dim)
    float2 *max_sum;  // (split, row, head)
    int32_t *count;   // (row, head): splits that there are, where that depends on the keys
    int splits;       // at most
};

// One tile of rows with one split of its keys; share: tiles of a split, or 0 for as many as
// there are over the splits.  LOG_SUM: the weights' sum is kept as it is beside that of the
// rounded weights, for the log-sum and for the shares of parts; it costs 16 of a step's
// additions, 4% of the time at 128 dimensions (2.05 -> 2.13 ms for 16320 rows and keys, 16
// heads on 4).
template <typename T, int DIM, bool BY_KEYS, bool LOG_SUM, typename Source>
__device__ __forceinline__ void forward_rows(
    const GsAttention &a, const Source &source, const T *q, T *out, T *out_rest, float *log_sum,
    const Partial &partial, lds_char *tiles, int kh, int sequence, int number, int split, int share) {
    using F = Forward<T, DIM, BY_KEYS>;
    using KTile = typename F::KTile;
    constexpr bool kHoles = Source::kHoles;
    const int group = a.heads_q / a.heads_k;
    const Span p = source.span(a, sequence);
    constexpr int kWaves = F::kWaves;
    const int lane = __lane_id(), half = lane >> 5, wave = uniform(threadIdx.x / kWave);
    const int rows = p.lq * group;
    const int row0 = number * F::kRows + (BY_KEYS ? 0 : 32 * wave);  // this wave's first
    const int row = row0 + (lane & 31);
    const bool real = row < rows;
    const int query = (real ? row : rows - 1) / group;
    const int head = kh * group + (real ? row - query * group : 0);
    const int64_t at = (int64_t)(p.q0 + query) * a.heads_q + head;

    // the last key each row sees, and the least and greatest of the wave and workgroup
    const int shift = a.causal ? p.lk - p.lq : p.lk;
    const int last = a.causal ? min(query + shift, p.lk - 1) : p.lk - 1;
    const int all_see = a.causal ? min(number * F::kRows / group + shift, p.lk - 1) : p.lk - 1;
    const int wave_last =
        a.causal ? min(min(row0 + 31, rows - 1) / group + shift, p.lk - 1) : p.lk - 1;
    const int block_end = min(number * F::kRows + F::kRows, rows) - 1;
    const int seen = a.causal ? min(block_end / group + shift, p.lk - 1) + 1 : p.lk;

    // this split's tiles
    const int tiles_all = seen > 0 ? (seen + F::kKeys - 1) / F::kKeys : 0;
    const int tiles_keys = (p.lk + F::kKeys - 1) / F::kKeys;
    if (!share) share = (tiles_all + partial.splits - 1) / partial.splits;
    const int first_tile = min(split * share, tiles_all);
    const int end_tile = min(first_tile + share, tiles_all);

    const bool negate = a.scale < 0.0f;
    const float c = exponent_factor(a.scale);
    RowOperand<T, DIM> qr;
    qr.load(real ? q + (int64_t)(p.q0 + query) * a.q_row + (int64_t)head * a.q_head : nullptr,
            a.dim, negate);

    typename Source::template Reader<KTile> keys(source, a, p, sequence, kh, wave, first_tile, end_tile);
    const auto fetch = [&](int t) { keys.fetch(t, tiles + (t & 1) * 2 * KTile::kBytes); };

    f32x16 acc[DIM / 32];
#pragma unroll
    for (int d = 0; d < DIM / 32; ++d) acc[d] = f32x16{};
    // the maximum of c S; the weights' sum over this half's keys, and that of the rounded ones
    float top = -INFINITY, sum = 0.0f, rounded = 0.0f;
    bool met = false;  // a key that the row sees and that is there

    const auto step = [&](int t, auto masks) {
        constexpr bool kMasks = decltype(masks)::value;
        copies_done();  // tile t is in LDS, and tile t - 1 has been read
        [[maybe_unused]] const uint64_t there = keys.there;
        if (t + 1 < end_tile) fetch(t + 1);
        if constexpr (kHoles) {
            if (!there) return;
            met = met || (kMasks ? t * F::kKeys + __builtin_ctzll(there) <= last : true);
        }
        const lds_char *kt = tiles + (t & 1) * 2 * KTile::kBytes, *vt = kt + KTile::kBytes;
        const int base = BY_KEYS ? 32 * wave : 0;  // of this wave's keys in the tile
        const int key0 = t * F::kKeys + base;
        if (kMasks && key0 > wave_last) return;

        f32x16 s[F::kSub];
#pragma unroll
        for (int n = 0; n < F::kSub; ++n) {
            s[n] = f32x16{};
#pragma unroll
            for (int i = 0; i < DIM / 16; ++i)
                s[n] = mfma(KTile::along(kt, base + 32 * n, i), qr.x[i], s[n]);
        }
        uint64_t found = 0;
        if constexpr (kMasks) {
            if (a.causal) found = rows_not_finite<T, DIM, 32 * F::kSub>(vt, base);
#pragma unroll
            for (int n = 0; n < F::kSub; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (key0 + 32 * n + result_row(r, half) > last) s[n][r] = -INFINITY;
            if constexpr (kHoles) {
                // (keys that are not there are zeros in LDS)
                if (~there) {
#pragma unroll
                    for (int n = 0; n < F::kSub; ++n) {
                        const uint32_t mine = (uint32_t)(there >> (base + 32 * n)) >> (4 * half);
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (!(mine >> result_row(r, 0) & 1)) s[n][r] = -INFINITY;
                    }
                }
            }
        }
        if constexpr (Source::kScores) {
            if (real) source.keep(at, key0 + 4 * half, s[0]);
        }
        float m = s[0][0];
#pragma unroll
        for (int n = 0; n < F::kSub; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) m = fmaxf(m, s[n][r]);
        m = half_max(m) * c;
        // a new reference only where the maximum has grown by 2^8: until then the weights
        // are at most 2^8, which loses nothing in either type
        if (__ballot(m > top + 8.0f)) {
            const float now = fmaxf(top, m);
            const float keep = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - now);
            top = now;
            sum *= keep;
            rounded *= keep;
#pragma unroll
            for (int d = 0; d < DIM / 32; ++d) acc[d] *= keep;
        }
        const float minus = top == -INFINITY ? 0.0f : -top;
        typename Vec<T>::x8 weights[2 * F::kSub];
#pragma unroll
        for (int n = 0; n < F::kSub; ++n) {
            float w[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                w[r] = __builtin_amdgcn_exp2f(fmaf(s[n][r], c, minus));
                if (LOG_SUM) sum += w[r];
            }
            weights[2 * n] = pack8<T>(w);
            weights[2 * n + 1] = pack8<T>(w + 8);
            rounded = add_weights<T>(weights[2 * n + 1], add_weights<T>(weights[2 * n], rounded));
        }
#pragma unroll
        for (int n = 0; n < F::kSub; ++n) {
            const uint32_t part = (uint32_t)(found >> (32 * n));
            if (kMasks && part)
                add_product_seen<T, DIM, KTile, false>(
                    acc, vt, base + 32 * n, weights + 2 * n,
                    [&](int i) { return key0 + 32 * n + i <= last; });
            else
                add_product<T, DIM, KTile>(acc, vt, base + 32 * n, weights + 2 * n);
        }
    };
    if (first_tile < end_tile) fetch(first_tile);
    int t = first_tile;
    // tiles that every row of the workgroup sees whole, then the others
    const int whole = min(end_tile, (all_see + 1) / F::kKeys);
    if constexpr (kHoles) {
        while (t < end_tile) {
            for (; t < whole && !~keys.there; ++t) step(t, std::false_type{});
            if (t < end_tile) step(t++, std::true_type{});
        }
    } else {
        for (; t < whole; ++t) step(t, std::false_type{});
        for (; t < end_tile; ++t) step(t, std::true_type{});
    }
    // The sums are over the rounded weights, and so is what they are divided by: a weight's error
    // then counts by its value's distance from the output, which for a weight that outdoes the
    // others is next to none.  The log-sum, and a part's share of the whole, are of the
    // weights as they were.
    rounded = half_sum(rounded);
    sum = LOG_SUM ? half_sum(sum) : rounded;
    // a row whose scores are all NaN has no maximum, but is not one that saw nothing
    if (sum != sum) top = fmaxf(top, 0.0f);
    if (LOG_SUM && (BY_KEYS || partial.splits > 1)) {
        const float share_up = rounded > 0.0f ? sum / rounded : 1.0f;
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d) acc[d] *= share_up;
        rounded = sum;
    }

    if constexpr (BY_KEYS) {
        // the waves' sums over their keys, joined in LDS by the first
        __syncthreads();  // the tiles have been read
        auto *sums = (__attribute__((address_space(3))) float *)tiles;  // (wave, register, lane)
        auto *stats = sums + kWaves * (DIM / 2) * 64;                  // (wave, lane) pairs
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) sums[(wave * (DIM / 2) + 16 * d + r) * 64 + lane] = acc[d][r];
        stats[2 * (wave * 64 + lane)] = top;
        stats[2 * (wave * 64 + lane) + 1] = sum;
        __syncthreads();
        if (wave) return;  // (a wave of no rows of its own)
        float all = top, weight[kWaves], total = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) all = fmaxf(all, stats[2 * (w * 64 + lane)]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float its = stats[2 * (w * 64 + lane)];
            weight[w] = its == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(its - all);
            total = fmaf(stats[2 * (w * 64 + lane) + 1], weight[w], total);
        }
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float x = acc[d][r] * weight[0];
#pragma unroll
                for (int w = 1; w < kWaves; ++w)
                    x = fmaf(sums[(w * (DIM / 2) + 16 * d + r) * 64 + lane], weight[w], x);
                acc[d][r] = x;
            }
        top = all;
        sum = rounded = total;
    }
    // a row whose scores are all minus infinity has seen keys: its weights are 0 / 0.  (Not so
    // low as a part that saw none, so that it counts where all of a row's parts are such.)
    if (top == -INFINITY && (kHoles ? met : last >= first_tile * F::kKeys)) top = -FLT_MAX;

    if (partial.splits > 1) {
        const int64_t slot = (int64_t)split * a.rows_q * a.heads_q + at;
        if (real && half == 0) {
            partial.max_sum[slot] = make_float2(top, sum);
            if (partial.count && split == 0)
                partial.count[at] = max((tiles_keys + share - 1) / share, 1);
        }
        store_partial<DIM>(acc, 1.0f,
                           real && top != -INFINITY ? partial.sums + slot * a.dim : nullptr, a.dim);
        return;
    }
    // a row that saw nothing: zeros, whatever met them
    const bool none = top == -INFINITY;
    if (__ballot(none)) {
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] = none ? 0.0f : acc[d][r];
    }
    store_columns<T, DIM>(acc, none ? 1.0f : 1.0f / rounded, real ? out + at * a.dim : nullptr, a.dim,
                          out_rest != nullptr, real && out_rest ? out_rest + at * a.dim : nullptr);
    if (LOG_SUM && log_sum && real && half == 0)
        log_sum[at] = none ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// A workgroup's tile of rows.
template <typename T, int DIM, bool LOG_SUM, typename Source>
__device__ __forceinline__ void forward_tile(const GsAttention &a, const Source &source, const T *q,
                                             T *out, T *out_rest, float *log_sum,
                                             const Partial &partial, lds_char *lds) {
    using F = Forward<T, DIM, false>;
    const Place at = place_of(a.heads_k, partial.splits);
    int sequence, number;
    if (!find_tile(a.offsets_q, a.sequences, a.rows_q, a.heads_q / a.heads_k, F::kRows, at.tile, true,
                   &sequence, &number))
        return;
    forward_rows<T, DIM, false, LOG_SUM>(a, source, q, out, out_rest, log_sum, partial, lds, at.kh,
                                         sequence, number, at.split, 0);
}

// Few rows a sequence.  Caches differ in length, and the host does not know them: a split is as
// many tiles of any of them as make about kSplits splits in all, as far as a row may have
// that many, and the workgroups take them in turn.  Bound by memory: a split costs a first
// tile and a join of its own, so there are no more than run at a time on 256 CUs, two a CU
// at 128 dimensions, less an eighth for the last splits of the sequences, which are shorter.
// 16 sequences of 2500 to 32640 keys, 16 heads on 4, dim 128, with the join: 85 us, 4.7
// TB/s; twice as many splits 99, four times 104; equal splits of each sequence 105.
constexpr int kSplits = 448;

template <typename T, int DIM, bool BY_KEYS, typename Source>
__device__ __forceinline__ void forward_shared(const GsAttention &a, const Source &source,
                                               const T *q, T *out, T *out_rest, float *log_sum,
                                               const Partial &partial, lds_char *lds) {
    using F = Forward<T, DIM, BY_KEYS>;
    const int group = a.heads_q / a.heads_k, all = a.sequences + 2;
    const auto tiles_of = [&](int s) {  // of keys
        return (source.keys(a, s) + F::kKeys - 1) / F::kKeys;
    };
    const auto rows_tiles_of = [&](int s) {
        const int2 r = rows_of(a.offsets_q, a.sequences, a.rows_q, s);
        return (int)(((int64_t)(r.y - r.x) * group + F::kRows - 1) / F::kRows);
    };
    // Of up to 128 sequences a lane keeps two and their tiles, so that offsets and lengths are read
    // once; more are looked through again for every split.
    constexpr int kHeld = 2;
    const bool few = all <= kHeld * kWave;
    int rows_held[kHeld], held[kHeld], upto[kHeld];
    float total = 0.0f;  // tiles of all (far below 2^24 where a split is more than one)
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int s = i * kWave + (int)__lane_id();
        rows_held[i] = few && s < all ? rows_tiles_of(s) : 0;
        held[i] = few && s < all ? tiles_of(s) : 0;
        total += (float)rows_held[i] * (float)held[i];
    }
    if (!few)
        for (int s = (int)__lane_id(); s < all; s += kWave)
            total += (float)rows_tiles_of(s) * (float)tiles_of(s);
    total = wave_sum(total);
    const int least = uniform(max(4, (int)(total * (float)a.heads_k / (float)kSplits) + 1));
    const auto share_of = [&](int t) { return max(least, (t + partial.splits - 1) / partial.splits); };
    const auto splits_of = [&](int t) {
        const int share = share_of(t);
        return max((t + share - 1) / share, 1);
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        upto[i] = (int)lanes_sum_upto((uint32_t)(rows_held[i] * splits_of(held[i]) * a.heads_k));
    const auto count = [&](int s) { return rows_tiles_of(s) * splits_of(tiles_of(s)) * a.heads_k; };
    // the sequence and the place in it of an item, and the sequence's tiles of keys
    int sequence, number, t;
    const auto find = [&](int item) {
        if (!few) {
            if (!find_place(all, count, item, false, &sequence, &number)) return false;
            t = uniform(tiles_of(sequence));
            return true;
        }
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const uint64_t past = __ballot(upto[i] > item);
            if (past) {
                const int l = __builtin_ctzll(past);
                sequence = i * kWave + l;
                number = item - (l ? __builtin_amdgcn_readlane(upto[i], l - 1) : 0);
                t = __builtin_amdgcn_readlane(held[i], l);
                return true;
            }
            item -= __builtin_amdgcn_readlane(upto[i], kWave - 1);
        }
        return false;
    };
    for (int item = blockIdx.x; find(item); item += gridDim.x) {
        const int splits = splits_of(t), rest = number / a.heads_k;
        forward_rows<T, DIM, BY_KEYS, true>(a, source, q, out, out_rest, log_sum, partial, lds,
                                            number % a.heads_k, sequence, rest / splits, rest % splits,
                                            share_of(t));
        __syncthreads();  // LDS has been read
    }
}

// Joins the splits of a row: a workgroup a row, four elements a thread, every eighth split
// in each of its eight parts.  Bound by latency: 256 rows of 28 splits 4.8 us.
template <typename T>
__device__ __forceinline__ void join_row(int64_t row, int64_t rows, int dim, const Partial &partial,
                                         T *out, T *out_rest, float *log_sum, f32x4 (*sums)[32]) {
    const int lane = __lane_id(), column = threadIdx.x % 32 * 4, part = threadIdx.x / 32;
    const int splits = partial.count ? min(partial.count[row], partial.splits) : partial.splits;
    const float2 mine = lane < splits ? partial.max_sum[lane * rows + row]
                                      : make_float2(-INFINITY, 0.0f);
    const float top = wave_max(mine.x);
    const float weight = mine.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mine.x - top);
    const float sum = wave_sum(mine.x == -INFINITY ? 0.0f : mine.y * weight);
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int first = 0; first < splits; first += 8) {  // (the same rounds in every lane)
        const int s = first + part;
        const float w = __shfl(weight, s, kWave);
        // (a split that saw nothing has written no sums, and those past the last are as it)
        const bool there = __shfl(mine.x, s, kWave) != -INFINITY && column < dim;
        if (there) x += *(const f32x4 *)(partial.sums + (s * rows + row) * dim + column) * w;
    }
    sums[part][threadIdx.x % 32] = x;
    __syncthreads();
    if (threadIdx.x >= 32) return;
#pragma unroll
    for (int p = 1; p < 8; ++p) x += sums[p][threadIdx.x];
    const bool none = top == -INFINITY;
    const float r = 1.0f / sum;
    if (column < dim) {
        float o[4], e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[i] = none ? 0.0f : x[i] * r;
            e[i] = o[i] - to_float(from_float<T>(o[i]));
        }
        store_floats<T, 4>(out + row * dim + column, o);
        if (out_rest) store_floats<T, 4>(out_rest + row * dim + column, e);
    }
    if (log_sum && threadIdx.x == 0)
        log_sum[row] = none ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// ------------------------------------------------------------------- launches
constexpr int64_t kMaxRows = 0x7fffffffLL - 65536;  // row numbers stay in 32 bits

// Rows that a tile can be copied from: byte offsets fit, and a row past the last one lies
// wholly behind the copy's bound.
inline bool tile_stride(int64_t stride, int dim) { return stride >= dim && stride <= kMaxStride; }

// How a forward is launched.
struct ForwardPlan {
    bool by_keys;
    int64_t groups;  // workgroups
    int splits;
};

// longest, average: at most and on average, keys of a sequence.
inline ForwardPlan plan_forward(const GsAttention &a, int64_t longest, int64_t average) {
    const int64_t group = a.heads_q / a.heads_k, packed = a.rows_q * group;
    const int64_t sequences = a.sequences > 0 ? a.sequences : 1;
    ForwardPlan f;
    // One tile of rows a sequence on average: the lengths themselves are not known here.  16
    // sequences over 16320 keys each, 16 heads on 4, dim 128: 1 query 113 us, otherwise 130; 8
    // queries (32 rows) 117 and 142; 12 (48) 143 and 133.  Where lengths are skewed the average
    // serves the long ones badly: a scene of 8000 tokens among 1199 of one takes 1042 us here,
    // 456 among 1099, which go the other way, and 275 alone.
    f.by_keys = packed <= 32 * sequences;
    if (f.by_keys) {
        // a row may have up to 64 splits of at least 256 keys, as far as the rows' sums stay few:
        // by the number of sequences, so that a cache of 32640 keys among 15, 63 and 255 of 64 (16
        // heads on 4, dim 128) takes 34, 89 and 321 us, and 28 alone
        int64_t splits = 2048 / (sequences * a.heads_k);
        const int64_t most = (longest + 255) / 256;
        if (splits > most) splits = most;
        f.splits = (int)(splits < 1 ? 1 : splits > 64 ? 64 : splits);
        const int64_t items = (packed / 32 + a.sequences + 2) * f.splits * a.heads_k;
        f.groups = items < 1024 ? items : 1024;
        // (items have numbers of 32 bits: past those, more workgroups than a launch takes, so that it is refused)
        const int64_t tiles = a.rows_q * ((group + 31) / 32);  // at most, however many sequences have none
        const int64_t numbers = (tiles < packed / 32 + a.sequences + 2 ? tiles : packed / 32 + a.sequences + 2) *
                                f.splits * a.heads_k;
        if (numbers > kMaxRows) f.groups = numbers;
        return f;
    }
    // Workgroups that will find rows, at least, and as many splits of the keys as run at a time
    // with them, 512 workgroups in all, two a CU.  More wait for a second turn and pay a join:
    // 2500 rows and keys, 16 heads on 4, dim 128, in 1 split of 316 workgroups 83 us, in 2 splits
    // 113; 300 rows over 16320 keys, 48 workgroups, in 10 splits 82 us, in 1 split 301.  A split of
    // fewer than four tiles costs more than it hides.
    const int64_t rows = 32 * kWaves;
    const int64_t busy = (packed + rows - 1) / rows * a.heads_k;
    const int64_t want = busy > 0 ? 512 / busy : 1;
    const int64_t most = average / 256;
    const int64_t splits = want < most ? want : most;
    f.splits = (int)(splits < 1 ? 1 : splits > 64 ? 64 : splits);
    f.groups = (packed / rows + a.sequences + 2) * a.heads_k * f.splits;
    return f;
}

inline size_t partial_bytes(const GsAttention &a, int splits) {
    if (splits == 1) return 0;
    const size_t rows = (size_t)a.rows_q * a.heads_q;
    return splits * rows * (a.dim * sizeof(float) + sizeof(float2)) + rows * sizeof(int32_t);
}

// The parts in a workspace of that size; counted: rows may have fewer of them.
inline Partial partial_of(const GsAttention &a, const ForwardPlan &f, bool counted, void *workspace) {
    Partial partial;
    const size_t rows = (size_t)a.rows_q * a.heads_q;
    partial.splits = f.splits;
    partial.sums = (float *)workspace;
    partial.max_sum = (float2 *)(partial.sums + f.splits * rows * a.dim);
    partial.count = counted ? (int32_t *)(partial.max_sum + f.splits * rows) : nullptr;
    return partial;
}

template <typename F>
inline int with_tile(int dim, F f) {
    if (dim <= 32) return f(std::integral_constant<int, 32>{});
    if (dim <= 64) return f(std::integral_constant<int, 64>{});
    if (dim <= 96) return f(std::integral_constant<int, 96>{});
    return f(std::integral_constant<int, 128>{});
}

}  // namespace gs
