// Attention over packed sequences with grouped heads, and its gradients:
//   S = scale q k^T over the keys a query sees,  P = exp(S - L),  L = log sum exp S
//   out = P v,  delta = sum_d dout out,  dS = P (dout v^T - delta)
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout
// with dk and dv summed over the query heads of a group.  Scores, softmax
// statistics and sums are in float.

#include <cfloat>
#include <initializer_list>
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
template <typename T, int DIM, bool BY_KEYS, bool LOG_SUM>
__device__ __forceinline__ void forward_rows(
    const GsAttention &a, const T *q, const T *k, const T *v, T *out, T *out_rest, float *log_sum,
    const Partial &partial, lds_char *tiles, int kh, int sequence, int number, int split, int share) {
    using F = Forward<T, DIM, BY_KEYS>;
    using KTile = typename F::KTile;
    const int group = a.heads_q / a.heads_k;
    const Span p = span_of(a, sequence);
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

    const auto copy_k = KTile::copy_of(wave, a.k_row, a.dim);
    const auto copy_v = KTile::copy_of(wave, a.v_row, a.dim);
    const auto fetch = [&](int t) {
        lds_char *to = tiles + (t & 1) * 2 * KTile::kBytes;
        const int64_t key = p.k0 + (int64_t)t * F::kKeys;
        KTile::start(copy_k, wave, k + key * a.k_row + kh * a.k_head, a.k_row,
                     p.lk - t * F::kKeys, a.dim, to);
        KTile::start(copy_v, wave, v + key * a.v_row + kh * a.v_head, a.v_row,
                     p.lk - t * F::kKeys, a.dim, to + KTile::kBytes);
    };

    f32x16 acc[DIM / 32];
#pragma unroll
    for (int d = 0; d < DIM / 32; ++d) acc[d] = f32x16{};
    // the maximum of c S; the weights' sum over this half's keys, and that of the rounded ones
    float top = -INFINITY, sum = 0.0f, rounded = 0.0f;

    const auto step = [&](int t, auto masks) {
        constexpr bool kMasks = decltype(masks)::value;
        copies_done();  // tile t is in LDS, and tile t - 1 has been read
        if (t + 1 < end_tile) fetch(t + 1);
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
    for (const int whole = min(end_tile, (all_see + 1) / F::kKeys); t < whole; ++t)
        step(t, std::false_type{});
    for (; t < end_tile; ++t) step(t, std::true_type{});
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
    if (top == -INFINITY && last >= first_tile * F::kKeys) top = -FLT_MAX;

    if (partial.splits > 1) {
        const int64_t slot = (int64_t)split * a.rows_q * a.heads_q + at;
        if (real && half == 0) {
            partial.max_sum[slot] = make_float2(top, sum);
            if (BY_KEYS && split == 0)
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

template <typename T, int DIM, bool LOG_SUM>
__global__ __launch_bounds__(64 * kWaves, 2) void attention_kernel(
    GsAttention a, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    T *__restrict__ out, T *__restrict__ out_rest, float *__restrict__ log_sum, Partial partial) {
    using F = Forward<T, DIM, false>;
    __shared__ __attribute__((aligned(1024))) char lds[F::kLds];
    const Place at = place_of(a.heads_k, partial.splits);
    int sequence, number;
    if (!find_tile(a.offsets_q, a.sequences, a.rows_q, a.heads_q / a.heads_k, F::kRows, at.tile, true,
                   &sequence, &number))
        return;
    forward_rows<T, DIM, false, LOG_SUM>(a, q, k, v, out, out_rest, log_sum, partial, (lds_char *)lds,
                                         at.kh, sequence, number, at.split, 0);
}

// Few rows a sequence.  Caches differ in length, and the host does not know them: a split is as
// many tiles of any of them as make about kSplits splits in all, as far as a row may have
// that many, and the workgroups take them in turn.  Bound by memory: a split costs a first
// tile and a join of its own, so there are no more than run at a time on 256 CUs, two a CU
// at 128 dimensions, less an eighth for the last splits of the sequences, which are shorter.
// 16 sequences of 2500 to 32640 keys, 16 heads on 4, dim 128, with the join: 85 us, 4.7
// TB/s; twice as many splits 99, four times 104; equal splits of each sequence 105.
constexpr int kSplits = 448;

template <typename T, int DIM>
__global__ __launch_bounds__(64 * kKeysWaves, DIM > 96 ? 1 : 2) void attention_keys_kernel(
    GsAttention a, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    T *__restrict__ out, T *__restrict__ out_rest, float *__restrict__ log_sum, Partial partial) {
    using F = Forward<T, DIM, true>;
    __shared__ __attribute__((aligned(1024))) char lds[F::kLds];
    const int group = a.heads_q / a.heads_k, all = a.sequences + 2;
    const auto tiles_of = [&](int s) {  // of keys
        const int n = keys_of(a, s, rows_of(a.offsets_k, a.sequences, a.rows_k, s));
        return (n + F::kKeys - 1) / F::kKeys;
    };
    const auto rows_tiles_of = [&](int s) {
        const int2 r = rows_of(a.offsets_q, a.sequences, a.rows_q, s);
        return (int)(((int64_t)(r.y - r.x) * group + F::kRows - 1) / F::kRows);
    };
    float total = 0.0f;  // tiles of all (far below 2^24 where a split is more than one)
    for (int first = 0; first < all; first += kWave) {
        const int s = first + (int)__lane_id();
        total += wave_sum(s < all ? (float)rows_tiles_of(s) * (float)tiles_of(s) : 0.0f);
    }
    const int least = uniform(max(4, (int)(total * (float)a.heads_k / (float)kSplits) + 1));
    const auto share_of = [&](int t) { return max(least, (t + partial.splits - 1) / partial.splits); };
    const auto splits_of = [&](int t) {
        const int share = share_of(t);
        return max((t + share - 1) / share, 1);
    };
    const auto count = [&](int s) { return rows_tiles_of(s) * splits_of(tiles_of(s)) * a.heads_k; };
    int sequence, number;
    for (int item = blockIdx.x; find_place(all, count, item, false, &sequence, &number);
         item += gridDim.x) {
        const int t = uniform(tiles_of(sequence)), splits = splits_of(t);
        const int rest = number / a.heads_k;
        forward_rows<T, DIM, true, true>(a, q, k, v, out, out_rest, log_sum, partial,
                                         (lds_char *)lds, number % a.heads_k, sequence,
                                         rest / splits, rest % splits, share_of(t));
        __syncthreads();  // LDS has been read
    }
}

// Joins the splits of a row: a workgroup a row, four elements a thread, every eighth split
// in each of its eight parts.  Bound by latency: 256 rows of 28 splits 4.8 us.
template <typename T>
__global__ __launch_bounds__(256) void attention_join_kernel(int64_t rows, int dim, Partial partial,
                                                             T *__restrict__ out,
                                                             T *__restrict__ out_rest,
                                                             float *__restrict__ log_sum) {
    __shared__ f32x4 sums[8][32];
    const int64_t row = blockIdx.x;
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

// ---------------------------------------------------------------- gradients
// Two launches, neither with atomics: the queries' gradients, a workgroup a tile of
// packed rows as in the forward, which also leaves each row's log-sum (in the exponent
// of two) and delta for the second (and only these where queries have no gradient); then
// the keys' and values', a workgroup a tile of keys, over all the queries of all heads of
// the group.  Scores are computed again in both: seven products in all where one launch
// with atomics needs five, whose sums' order would change from run to run.
//
// Bound as the forward is, the keys' launch more by its registers: two sums of a tile of keys
// and both operands leave one wave a SIMD above 96 dimensions.  16320 rows and keys, 16 heads
// on 4, dim 128, bfloat16: queries 2.75 ms, 1.19 PFLOP/s of its three products; keys and
// values 4.4 to 5.1 ms, 0.86 to 0.99 of its four.
//
// Score gradients are rounded to the inputs' type for their products, which adds as much
// again to the rounding of the result (1.41 times its error in all, and more with what delta
// has from the output's rounded weights: 1.55 for rows of a few keys).  A second product of the
// same tile with what was rounded off takes it back.  In tiles with a mask, and where a sequence
// has only one, of up to 64 keys (or queries, in the keys' launch), where delta's part is
// largest, both launches have it (1.3 times the error for rows of 1 to 7 keys in bfloat16; the
// training pass over scenes of 12566 and 16320 tokens 8.53 -> 8.65 ms).  In float16, which is chosen for its bits, the queries'
// gradients have it in every tile (1.02 to 1.08 times the error); that costs the launch 28%,
// 171 -> 217 us for 4 sequences of 2500, 12 heads of 72 (249 with the range below), and neither
// bfloat16 nor the keys' launch, longer by itself, pays it.
// In float16 they are first put into its range: weights times 2^10, so that those of long rows keep their
// bits, and score gradients times a power of two that follows the largest that the query, or
// the key, has met so far (Fit), and that the sums follow.
template <typename T>
struct Range {
    static constexpr bool kScaled = std::is_same<T, f16>::value;
    static constexpr float kWeight = kScaled ? 10.0f : 0.0f;  // exponents of two
};

// The power of two at or below v's magnitude; 1 for zero, infinities and NaN.
__device__ __forceinline__ float power_below(float v) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v) & 0x7f800000u;
    return bits == 0 || bits == 0x7f800000u ? 1.0f : __builtin_bit_cast(float, bits);
}

// A column's score gradients in float16: `scale` times themselves, at most 2^15.  The bound is
// on what is rounded, whatever sizes of queries, values and output gradients made it: a
// column's largest so far is brought to between 2^9 and 2^10 when it is first met and whenever
// a greater one passes 2^15, so that what is 2^23 times smaller still has all its bits, and
// what falls below float16's smallest number is 2^-33 of the largest.  Greater than 2^60 the
// scale does not become, so that no product with it overflows; what that leaves too small is
// below any gradient's last bit.  Forward and gradients with it, and with a factor from the
// output gradients alone, which values of 34 overflow: 8160 rows and keys, 16 heads on 4, dim
// 128, 2.80 ms and 2.78; 4 sequences of 2500, 12 heads of 72, 611 us and 624; of 64, causal,
// 354 and 341.
struct Fit {
    float scale = 1.0f, limit = 0.0f;
    template <int SUMS>
    __device__ __forceinline__ void follow(float *ds, f32x16 *acc) {
        float most = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(ds[r]));
        if (__ballot(most > limit)) {
            most = half_max(most);  // (an infinity or NaN leaves the scale: its sums are lost)
            const bool passes = most > limit && most < INFINITY;
            const float ratio = passes ? fminf(512.0f / power_below(most), 0x1p60f / scale) : 1.0f;
            limit = passes ? 32768.0f : limit;
            scale *= ratio;
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] *= ratio;
#pragma unroll
            for (int d = 0; d < SUMS; ++d) acc[d] *= ratio;
        }
    }
};

constexpr int kBackRows = 64;             // of a tile in LDS
constexpr int kBackOwn = 32 * kWaves;     // rows of a workgroup

template <typename T, int DIM>
__global__ __launch_bounds__(64 * kWaves, 2) void attention_dq_kernel(
    GsAttention a, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    const T *__restrict__ out, const T *__restrict__ out_rest, const float *__restrict__ log_sum,
    const T *__restrict__ go, int64_t go_row, int64_t go_head, T *__restrict__ dq, float *__restrict__ row_log,
    float *__restrict__ row_delta, float *__restrict__ partial, int splits) {
    using KTile = Tile<T, DIM, kBackRows, kWaves>;
    __shared__ __attribute__((aligned(1024))) char lds[4 * KTile::kBytes];
    lds_char *const tiles = (lds_char *)lds;

    const Place at_grid = place_of(a.heads_k, splits);
    const int kh = at_grid.kh, split = at_grid.split, group = a.heads_q / a.heads_k;
    int sequence, number;
    if (!find_tile(a.offsets_q, a.sequences, a.rows_q, group, kBackOwn, at_grid.tile,
                   true, &sequence, &number))
        return;
    const Span p = span_of(a, sequence);
    const int lane = __lane_id(), half = lane >> 5, wave = uniform(threadIdx.x / kWave);
    const int rows = p.lq * group;
    const int row0 = number * kBackOwn + 32 * wave, row = row0 + (lane & 31);
    const bool real = row < rows;
    const int query = (real ? row : rows - 1) / group;
    const int head = kh * group + (real ? row - query * group : 0);
    const int64_t at = (int64_t)(p.q0 + query) * a.heads_q + head;

    const int shift = a.causal ? p.lk - p.lq : p.lk;
    const int last = a.causal ? min(query + shift, p.lk - 1) : p.lk - 1;
    const int all_see = a.causal ? min(number * kBackOwn / group + shift, p.lk - 1) : p.lk - 1;
    const int wave_last =
        a.causal ? min(min(row0 + 31, rows - 1) / group + shift, p.lk - 1) : p.lk - 1;
    const int block_end = min(number * kBackOwn + kBackOwn, rows) - 1;
    const int seen = a.causal ? min(block_end / group + shift, p.lk - 1) + 1 : p.lk;
    const int tiles_all = seen > 0 ? (seen + kBackRows - 1) / kBackRows : 0;
    const int share = (tiles_all + splits - 1) / splits;  // this split's tiles
    const int first_tile = min(split * share, tiles_all);
    const int end_tile = dq ? min(first_tile + share, tiles_all) : first_tile;

    RowOperand<T, DIM> qr, gr;
    qr.load(real ? q + (int64_t)(p.q0 + query) * a.q_row + (int64_t)head * a.q_head : nullptr,
            a.dim, false);
    gr.load(real ? go + (int64_t)(p.q0 + query) * go_row + (int64_t)head * go_head : nullptr,
            a.dim, false);
    // delta of the output before it was rounded: the rounded one's error in delta is shared by
    // all of a row's score gradients, and where these nearly cancel it is most of theirs
    float delta = 0.0f;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const T *from = part ? out_rest : out;
        RowOperand<T, DIM> o;
        o.load(real ? from + at * a.dim : nullptr, a.dim, false);
#pragma unroll
        for (int s = 0; s < DIM / 16; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                delta = fmaf(to_float(gr.x[s][i]), to_float(o.x[s][i]), delta);
    }
    delta = half_sum(delta);
    // a row that saw nothing has no weights: exp2(x - infinity) = 0; one that saw keys, with scores
    // of minus infinity, has none that are numbers
    const float given = real ? log_sum[at] : -INFINITY;
    const float log2_sum =
        given == -INFINITY ? (real && last >= 0 ? NAN : INFINITY) : given * kLog2e;
    // a row that sees one key has no score gradient: its dout v^T and delta are the same sum in
    // two orders, whose difference would be all there is of it
    const float row_exponent = last == 0 ? INFINITY : log2_sum;
    if (real && half == 0 && split == 0) {  // as the keys' launch uses them
        const int64_t to = (int64_t)head * a.rows_q + p.q0 + query;
        row_log[to] = log2_sum - Range<T>::kWeight;
        row_delta[to] = -delta;
    }

    const float c = a.scale * kLog2e;
    const auto copy_k = KTile::copy_of(wave, a.k_row, a.dim);
    const auto copy_v = KTile::copy_of(wave, a.v_row, a.dim);
    const auto fetch = [&](int t) {
        lds_char *to = tiles + (t & 1) * 2 * KTile::kBytes;
        const int64_t key = p.k0 + (int64_t)t * kBackRows;
        KTile::start(copy_k, wave, k + key * a.k_row + kh * a.k_head, a.k_row,
                     p.lk - t * kBackRows, a.dim, to);
        KTile::start(copy_v, wave, v + key * a.v_row + kh * a.v_head, a.v_row,
                     p.lk - t * kBackRows, a.dim, to + KTile::kBytes);
    };

    f32x16 acc[DIM / 32];
#pragma unroll
    for (int d = 0; d < DIM / 32; ++d) acc[d] = f32x16{};
    Fit fit;

    const auto step = [&](int t, auto masks) {
        constexpr bool kMasks = decltype(masks)::value;
        copies_done();  // tile t is in LDS, and tile t - 1 has been read
        if (t + 1 < end_tile) fetch(t + 1);
        const lds_char *kt = tiles + (t & 1) * 2 * KTile::kBytes, *vt = kt + KTile::kBytes;
        const int key0 = t * kBackRows;
        if (kMasks && key0 > wave_last) return;
        uint64_t found = 0;
        if (kMasks && a.causal) found = rows_not_finite<T, DIM, kBackRows>(kt, 0);
#pragma unroll
        for (int n = 0; n < kBackRows / 32; ++n) {
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int i = 0; i < DIM / 16; ++i) {
                s = mfma(KTile::along(kt, 32 * n, i), qr.x[i], s);
                dp = mfma(KTile::along(vt, 32 * n, i), gr.x[i], dp);
            }
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float w = __builtin_amdgcn_exp2f(fmaf(s[r], c, -row_exponent));
                // (the scale is a power of two: the same as scaling the difference)
                ds[r] = w * (Range<T>::kScaled ? fmaf(dp[r], fit.scale, -delta * fit.scale)
                                               : dp[r] - delta);
                if (kMasks && key0 + 32 * n + result_row(r, half) > last) ds[r] = 0.0f;
            }
            if constexpr (Range<T>::kScaled) fit.follow<DIM / 32>(ds, acc);
            const typename Vec<T>::x8 x[2] = {pack8<T>(ds), pack8<T>(ds + 8)};
            typename Vec<T>::x8 rests[2], *rest = nullptr;
            if constexpr (Range<T>::kScaled || kMasks) {
#pragma unroll
                for (int r = 0; r < 16; ++r) ds[r] -= to_float((T)x[r / 8][r % 8]);
                rests[0] = pack8<T>(ds);
                rests[1] = pack8<T>(ds + 8);
                rest = rests;
            }
            const uint32_t part = (uint32_t)(found >> (32 * n));
            if (kMasks && part)
                add_product_seen<T, DIM, KTile, true>(
                    acc, kt, 32 * n, x, [&](int i) { return key0 + 32 * n + i <= last; }, rest);
            else
                add_product<T, DIM, KTile>(acc, kt, 32 * n, x, rest);
        }
    };
    if (first_tile < end_tile) fetch(first_tile);
    int t = first_tile;
    // (one tile of keys goes the way of masked ones, which keeps what rounding takes off)
    const int whole = p.lk <= kBackRows ? 0 : min(end_tile, (all_see + 1) / kBackRows);
    for (; t < whole; ++t) step(t, std::false_type{});
    for (; t < end_tile; ++t) step(t, std::true_type{});
    if (splits > 1)
        store_partial<DIM>(acc, 1.0f / fit.scale,
                           real ? partial + ((int64_t)split * a.rows_q * a.heads_q + at) * a.dim
                                : nullptr,
                           a.dim);
    else
        store_columns<T, DIM>(acc, a.scale / fit.scale, real && dq ? dq + at * a.dim : nullptr, a.dim);
}

// Up to 64 dimensions a wave holds its keys' K and V and both sums in half a SIMD's registers,
// and four waves make a workgroup, two a CU.  At 65 to 96 two waves' sums leave no room for V,
// which lies in LDS; that then has room for one workgroup of eight waves.  At 97 to 128 the
// sums alone would take half of what two waves a SIMD have: one wave has K, V and both sums
// in 369 of 512, and four waves make a workgroup.
template <int DIM>
struct KeysShape {
    static constexpr bool kValuesInLds = DIM == 96;
    static constexpr int kWaves = kValuesInLds ? 8 : 4;
    static constexpr int kOwn = 32 * kWaves;  // keys of a workgroup
};

template <typename T, int DIM>
__global__ __launch_bounds__(64 * KeysShape<DIM>::kWaves, DIM > 96 ? 1 : 2) void attention_dkv_kernel(
    GsAttention a, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    const T *__restrict__ go, int64_t go_row, int64_t go_head, const float *__restrict__ row_log,
    const float *__restrict__ row_delta, T *__restrict__ dk, T *__restrict__ dv, float *__restrict__ partial, int splits) {
    using Shape = KeysShape<DIM>;
    constexpr int kOwn = Shape::kOwn;
    using QTile = Tile<T, DIM, kBackRows, Shape::kWaves>;
    using VTile = Tile<T, DIM, kOwn / 2, Shape::kWaves>;  // two, one behind the other
    constexpr int kFloats = kBackRows * 4;                         // bytes of one float a row
    constexpr int kStage = 2 * QTile::kBytes + 2 * kFloats;  // Q, dout, log-sums, deltas
    __shared__ __attribute__((aligned(1024))) char lds[2 * kStage + (Shape::kValuesInLds ? 2 * VTile::kBytes : 0)];
    lds_char *const tiles = (lds_char *)lds, *const values = tiles + 2 * kStage;

    const Place at_grid = place_of(a.heads_k, splits);
    const int kh = at_grid.kh, split = at_grid.split, group = a.heads_q / a.heads_k;
    int sequence, number;
    if (!find_tile(a.offsets_k, a.sequences, a.rows_k, 1, kOwn, at_grid.tile, false,
                   &sequence, &number))
        return;
    const Span p = span_of(a, sequence);
    const int lane = __lane_id(), half = lane >> 5, wave = uniform(threadIdx.x / kWave);
    const int block_key = number * kOwn;
    const int key = block_key + 32 * wave + (lane & 31);  // in the sequence
    const bool real = key < p.k1 - p.k0, counts = key < p.lk;

    // queries from `first` on see some key of the workgroup, from `whole` on all of them
    const int shift = a.causal ? p.lk - p.lq : p.lk;
    const int end_key = min(block_key + kOwn, p.lk);
    const int first = a.causal ? max(block_key - shift, 0) : 0;
    const int whole = a.causal ? max(end_key - 1 - shift, 0) : 0;
    const int first_tile = first / kBackRows;
    const int end_tile = block_key < p.lk ? (p.lq + kBackRows - 1) / kBackRows : 0;
    // (one tile of queries goes the way of masked ones, which keeps what rounding takes off)
    const int whole_tile = end_tile == 1 ? 1 : min((whole + kBackRows - 1) / kBackRows, end_tile);
    const int own_first = a.causal ? key - shift : 0;  // the first query that sees this key
    // and the first that sees another one too, so that it has a score gradient (where the
    // sequence has other keys: only with a causal mask)
    const int own_shared = own_first + (a.causal && key == 0);

    const T *key_row = counts ? k + (int64_t)(p.k0 + key) * a.k_row + (int64_t)kh * a.k_head : nullptr;
    const T *value_row = counts ? v + (int64_t)(p.k0 + key) * a.v_row + (int64_t)kh * a.v_head : nullptr;
    RowOperand<T, DIM> kr, vr;
    kr.load(key_row, a.dim, false);
    if constexpr (!Shape::kValuesInLds) vr.load(value_row, a.dim, false);

    const float c = a.scale * kLog2e;
    const auto copy_q = QTile::copy_of(wave, a.q_row, a.dim);
    const auto copy_g = QTile::copy_of(wave, go_row, a.dim);
    // (chosen here: inside, the compiler would index what the function captures by it, and
    // keep all of that in memory)
    const float *row_floats = wave == 0 ? row_log : row_delta;
    const auto fetch = [&](int i) {
        lds_char *to = tiles + (i & 1) * kStage;
        const int t = end_tile - 1 - i / group, head = kh * group + i % group;
        const int64_t row = p.q0 + (int64_t)t * kBackRows;
        const int present = p.lq - t * kBackRows;
        QTile::start(copy_q, wave, q + row * a.q_row + head * a.q_head, a.q_row, present, a.dim, to);
        QTile::start(copy_g, wave, go + row * go_row + head * go_head, go_row, present, a.dim,
                     to + QTile::kBytes);
        const int64_t f = head * a.rows_q + row;
        if (wave < 2)
            QTile::start_floats(row_floats + f, present, to + 2 * QTile::kBytes + wave * kFloats);
    };

    f32x16 gk[DIM / 32], gv[DIM / 32];
#pragma unroll
    for (int d = 0; d < DIM / 32; ++d) gk[d] = gv[d] = f32x16{};
    Fit fit;             // of the key's score gradients, their weights' 2^10 included

    const auto step = [&](int i, auto masks) {
        constexpr bool kMasks = decltype(masks)::value;
        constexpr int kUnroll = kMasks || DIM > 64 ? 1 : 2;
        const lds_char *qt = tiles + (i & 1) * kStage, *gt = qt + QTile::kBytes;
        const lds_char *logs = gt + QTile::kBytes, *deltas = logs + kFloats;
        const int query0 = (end_tile - 1 - i / group) * kBackRows;
        if constexpr (kMasks) {
            // infinities and NaN become zeros, for they must not meet the weight 0 of a key that
            // their query does not see.  Those of an output gradient reach the value gradients, in
            // their columns, of the keys that it sees; its query's delta, or the log-sum of a
            // query that holds such a value, is no number either, and makes the rest of it.
            const uint64_t found_g = rows_not_finite<T, DIM, kBackRows>(gt, 0);
            if (found_g | rows_not_finite<T, DIM, kBackRows>(qt, 0)) {
                if (found_g)
                    add_infinities_seen<T, DIM, QTile, kBackRows>(
                        gv, gt, [&](int j) { return query0 + j >= own_first; });
                __syncthreads();  // all waves have looked
                for (int at = threadIdx.x * 16; at < 2 * QTile::kBytes; at += 64 * Shape::kWaves * 16) {
                    auto *x = (__attribute__((address_space(3))) typename Vec<T>::x8 *)(
                        tiles + (i & 1) * kStage + at);
                    *x = Told<T>(*x).finite();
                }
                __syncthreads();
            }
        }
#pragma unroll kUnroll
        for (int n = 0; n < kBackRows / 32; ++n) {
            using lds_f4 = const __attribute__((address_space(3))) f32x4;
            f32x16 s = {}, dp;  // dp - delta: the product's sum begins at -delta
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const f32x4 e = *(lds_f4 *)(deltas + (32 * n + result_row(r, half)) * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) dp[r + j] = e[j];
            }
#pragma unroll
            for (int j = 0; j < DIM / 16; ++j) {
                s = mfma(QTile::along(qt, 32 * n, j), kr.x[j], s);
                if constexpr (Shape::kValuesInLds)
                    dp = mfma(QTile::along(gt, 32 * n, j), VTile::along(values, 32 * wave, j), dp);
                else
                    dp = mfma(QTile::along(gt, 32 * n, j), vr.x[j], dp);
            }
            float w[16], ds[16];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 l = *(lds_f4 *)(logs + (32 * n + result_row(4 * g, half)) * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 4 * g + j;
                    w[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -l[j]));
                    ds[r] = (Range<T>::kScaled ? w[r] * fit.scale : w[r]) * dp[r];
                    if (kMasks) {
                        const int query = query0 + 32 * n + result_row(r, half);
                        if (query < own_first) w[r] = 0.0f;
                        if (query < own_shared) ds[r] = 0.0f;
                    }
                }
            }
            const typename Vec<T>::x8 pw[2] = {pack8<T>(w), pack8<T>(w + 8)};
            add_product<T, DIM, QTile>(gv, gt, 32 * n, pw);
            if constexpr (Range<T>::kScaled) fit.follow<DIM / 32>(ds, gk);
            const typename Vec<T>::x8 pd[2] = {pack8<T>(ds), pack8<T>(ds + 8)};
            if constexpr (kMasks) {
#pragma unroll
                for (int r = 0; r < 16; ++r) ds[r] -= to_float((T)pd[r / 8][r % 8]);
                const typename Vec<T>::x8 rest[2] = {pack8<T>(ds), pack8<T>(ds + 8)};
                add_product<T, DIM, QTile>(gk, qt, 32 * n, pd, rest);
            } else {
                add_product<T, DIM, QTile>(gk, qt, 32 * n, pd);
            }
        }
    };
    // from the last tile back, every head of the group in turn: workgroups that start together
    // read the same tiles at the same time, also where a causal mask gives them different
    // first ones; the tiles with queries that do not see all the keys come last
    const int whole_steps = max(end_tile - whole_tile, 0) * group;
    const int steps_all = max(end_tile - first_tile, 0) * group;
    const int share = (steps_all + splits - 1) / splits;  // this split's steps
    const int first_step = min(split * share, steps_all);
    const int steps = min(first_step + share, steps_all);
    int i = first_step;
    if (i < steps) {
        if constexpr (Shape::kValuesInLds) {
            const auto copy_v = VTile::copy_of(wave, a.v_row, a.dim);
            for (int at = 0; at < kOwn; at += kOwn / 2)
                VTile::start(copy_v, wave,
                             v + (int64_t)(p.k0 + block_key + at) * a.v_row + (int64_t)kh * a.v_head,
                             a.v_row, p.lk - block_key - at, a.dim, values + at * DIM * 2);
        }
        fetch(i);
    }
    for (; i < min(whole_steps, steps); ++i) {
        copies_done();  // tile i is in LDS, and tile i - 1 has been read
        if (i + 1 < steps) fetch(i + 1);
        step(i, std::false_type{});
    }
    for (; i < steps; ++i) {
        copies_done();
        if (i + 1 < steps) fetch(i + 1);
        step(i, std::true_type{});
    }
    if (p.lk == 1) {  // no query sees another key
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d) gk[d] *= 0.0f;
    }
    // keys past the length that counts have no gradient
    if (__ballot(!counts)) {
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                gk[d][r] = counts ? gk[d][r] : 0.0f;
                gv[d][r] = counts ? gv[d][r] : 0.0f;
            }
    }
    const int64_t at = ((int64_t)(p.k0 + key) * a.heads_k + kh) * a.dim;
    const float back_v = Range<T>::kScaled ? 1.0f / 1024.0f : 1.0f, back_k = back_v / fit.scale;
    if (splits > 1) {
        const int64_t size = a.rows_k * a.heads_k * a.dim;
        float *to = partial + split * size + at;
        store_partial<DIM>(gk, back_k, real ? to : nullptr, a.dim);
        store_partial<DIM>(gv, back_v, real ? to + splits * size : nullptr, a.dim);
        return;
    }
    store_columns<T, DIM>(gk, a.scale * back_k, real ? dk + at : nullptr, a.dim);
    store_columns<T, DIM>(gv, back_v, real ? dv + at : nullptr, a.dim);
}

// Sums of splits, rounded: the y-th of the launch's outputs, four elements a thread.  Bound by
// memory: two splits of 16320 rows of 4 heads of 128, twice, 26 us.
template <typename T>
__global__ __launch_bounds__(256) void attention_sum_kernel(const float *__restrict__ partial,
                                                            int64_t size, int splits, float scale0,
                                                            float scale1, T *__restrict__ out0,
                                                            T *__restrict__ out1) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= size) return;
    const float *p = partial + (int64_t)blockIdx.y * splits * size + i;
    f32x4 sum = *(const f32x4 *)p;
    for (int s = 1; s < splits; ++s) sum += *(const f32x4 *)(p + s * size);
    sum *= blockIdx.y ? scale1 : scale0;
    const typename Vec<T>::x4 o = {(T)sum[0], (T)sum[1], (T)sum[2], (T)sum[3]};
    *(typename Vec<T>::x4 *)((blockIdx.y ? out1 : out0) + i) = o;
}

constexpr int64_t kMaxRows = 0x7fffffffLL - 65536;  // row numbers stay in 32 bits

// Rows that a tile can be copied from: byte offsets fit, and a row past the last one lies
// wholly behind the copy's bound.
static bool tile_stride(int64_t stride, int dim) { return stride >= dim && stride <= kMaxStride; }

static int check_attention(const GsAttention *a) {
    if (!a || a->rows_q < 0 || a->rows_k < 0 || a->sequences < 0 || a->heads_q < 1 ||
        a->heads_k < 1 || a->heads_q % a->heads_k != 0 || a->dim < 1 || a->q_row < 0 ||
        a->q_head < 0 || a->k_row < 0 || a->k_head < 0 || a->v_row < 0 || a->v_head < 0 ||
        !(a->scale == a->scale))
        return GS_ERR_INVALID_ARGUMENT;
    if (!a->offsets_q || !a->offsets_k) return GS_ERR_INVALID_ARGUMENT;
    if (!element_type(a->type)) return GS_ERR_INVALID_ARGUMENT;
    if (a->type == GS_F32 || a->dim % 8 != 0 || a->dim > GS_MAX_HEAD_DIM ||
        a->rows_q > kMaxRows / (a->heads_q / a->heads_k) || a->rows_k > kMaxRows ||
        !tile_stride(a->q_row, a->dim) || !tile_stride(a->k_row, a->dim) ||
        !tile_stride(a->v_row, a->dim) ||
        (a->q_row | a->q_head | a->k_row | a->k_head | a->v_row | a->v_head) % 8 != 0)
        return GS_ERR_UNSUPPORTED;
    return GS_OK;
}

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// How a forward is launched.
struct ForwardPlan {
    bool by_keys;
    int64_t groups;  // workgroups
    int splits;
};

static ForwardPlan plan_forward(const GsAttention &a) {
    const int64_t group = a.heads_q / a.heads_k, packed = a.rows_q * group;
    const int64_t sequences = a.sequences > 0 ? a.sequences : 1;
    ForwardPlan f;
    // One tile of rows a sequence on average: the lengths themselves are not known here.  16
    // sequences over 16320 keys each, 16 heads on 4, dim 128: 1 query 113 us, otherwise 130; 8
    // queries (32 rows) 117 and 142; 12 (48) 143 and 133.  Where lengths are skewed the average
    // serves the long ones badly: a scene of 8000 tokens among 1199 of one takes 1154 us here,
    // 456 among 1099, which go the other way, and 275 alone.
    f.by_keys = packed <= 32 * sequences;
    if (f.by_keys) {
        // a row may have up to 64 splits of at least 256 keys, as far as the rows' sums stay few:
        // by the number of sequences, so that a cache of 32640 keys among 15, 63 and 255 of 64 (16
        // heads on 4, dim 128) takes 34, 89 and 321 us, and 28 alone
        int64_t splits = 2048 / (sequences * a.heads_k);
        const int64_t most = (a.rows_k + 255) / 256;
        if (splits > most) splits = most;
        f.splits = (int)(splits < 1 ? 1 : splits > 64 ? 64 : splits);
        const int64_t items = (packed / 32 + a.sequences + 2) * f.splits * a.heads_k;
        f.groups = items < 1024 ? items : 1024;
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
    const int64_t most = a.rows_k / sequences / 256;
    const int64_t splits = want < most ? want : most;
    f.splits = (int)(splits < 1 ? 1 : splits > 64 ? 64 : splits);
    f.groups = (packed / rows + a.sequences + 2) * a.heads_k * f.splits;
    return f;
}

// How a backward is launched: its sums in as many splits as run at a time, as the forward's,
// 512 workgroups in all, or 256 of the eight waves that the keys' launch has for 65 to 96
// dimensions.  Forward and gradients of 2500 rows and keys, 16 heads on 4, dim 128, 340 us,
// with splits for 512 and 768 workgroups or more 396, with none 514.
struct BackwardPlan {
    int64_t tiles_q, tiles_k;
    int splits_q, splits_k;
};

static int backward_splits(int64_t busy, int64_t slots, int64_t steps) {
    if (busy < 1 || busy >= slots) return 1;
    const int64_t want = slots / busy, most = steps / 8;
    const int64_t splits = want < most ? want : most;
    return (int)(splits < 1 ? 1 : splits > 8 ? 8 : splits);
}

static BackwardPlan plan_backward(const GsAttention &a) {
    const int64_t group = a.heads_q / a.heads_k, packed = a.rows_q * group;
    const int64_t sequences = a.sequences > 0 ? a.sequences : 1, see = a.causal ? 2 : 1;
    BackwardPlan b;
    b.tiles_q = packed / kBackOwn + a.sequences + 2;
    const int64_t own = a.dim > 96 ? KeysShape<128>::kOwn : a.dim > 64 ? KeysShape<96>::kOwn : KeysShape<64>::kOwn;
    b.tiles_k = a.rows_k / own + a.sequences + 2;
    b.splits_q = backward_splits((packed + kBackOwn - 1) / kBackOwn * a.heads_k, 512,
                                 a.rows_k / sequences / kBackRows / see);
    b.splits_k = backward_splits((a.rows_k + own - 1) / own * a.heads_k, own > kBackOwn ? 256 : 512,
                                 packed / sequences / kBackRows / see);
    return b;
}

static size_t backward_partials(const GsAttention &a, const BackwardPlan &b) {
    const size_t q = b.splits_q > 1 ? (size_t)b.splits_q * a.rows_q * a.heads_q * a.dim : 0;
    const size_t k = b.splits_k > 1 ? (size_t)b.splits_k * a.rows_k * a.heads_k * a.dim * 2 : 0;
    return (q > k ? q : k) * sizeof(float);
}

// Bytes of the rows' log-sums and deltas, a multiple of 16.
static size_t backward_rows(const GsAttention &a) {
    return ((size_t)a.rows_q * a.heads_q * 2 * sizeof(float) + 15) / 16 * 16;
}

static size_t partial_bytes(const GsAttention &a, int splits) {
    if (splits == 1) return 0;
    const size_t rows = (size_t)a.rows_q * a.heads_q;
    return splits * rows * (a.dim * sizeof(float) + sizeof(float2)) + rows * sizeof(int32_t);
}

template <typename T, int DIM>
static int launch_forward(const GsAttention &a, const ForwardPlan &f, const void *q, const void *k,
                          const void *v, void *out, void *out_rest, float *log_sum,
                          const Partial &partial, hipStream_t stream) {
    const dim3 grid((unsigned)f.groups);
    const T *tq = (const T *)q, *tk = (const T *)k, *tv = (const T *)v;
    if (f.by_keys)
        hipLaunchKernelGGL((attention_keys_kernel<T, DIM>), grid,
                           dim3(64 * kKeysWaves), 0, stream, a, tq, tk, tv,
                           (T *)out, (T *)out_rest, log_sum, partial);
    else if (log_sum || f.splits > 1)
        hipLaunchKernelGGL((attention_kernel<T, DIM, true>), grid, dim3(64 * kWaves), 0, stream, a,
                           tq, tk, tv, (T *)out, (T *)out_rest, log_sum, partial);
    else
        hipLaunchKernelGGL((attention_kernel<T, DIM, false>), grid, dim3(64 * kWaves), 0, stream, a,
                           tq, tk, tv, (T *)out, (T *)out_rest, log_sum, partial);
    int st = launch_status();
    if (st || f.splits == 1) return st;
    const int64_t rows = a.rows_q * a.heads_q;
    hipLaunchKernelGGL((attention_join_kernel<T>), dim3((unsigned)rows), dim3(256), 0, stream,
                       rows, a.dim, partial, (T *)out, (T *)out_rest, log_sum);
    return launch_status();
}

template <typename F>
static int with_tile(int dim, F f) {
    if (dim <= 32) return f(std::integral_constant<int, 32>{});
    if (dim <= 64) return f(std::integral_constant<int, 64>{});
    if (dim <= 96) return f(std::integral_constant<int, 96>{});
    return f(std::integral_constant<int, 128>{});
}

}  // namespace gs

using namespace gs;

extern "C" int gs_attention_forward_workspace_size(const GsAttention *a, size_t *bytes) {
    const int st = check_attention(a);
    if (st) return st;
    if (!bytes) return GS_ERR_INVALID_ARGUMENT;
    *bytes = partial_bytes(*a, plan_forward(*a).splits);
    return GS_OK;
}

extern "C" int gs_attention_forward(const GsAttention *a, const void *q, const void *k,
                                    const void *v, void *out, void *out_rest, float *log_sum,
                                    void *workspace, size_t workspace_bytes, hipStream_t stream) {
    const int st = check_attention(a);
    if (st) return st;
    if (a->rows_q == 0) return GS_OK;
    if (!q || !out || (a->rows_k > 0 && (!k || !v))) return GS_ERR_INVALID_ARGUMENT;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(out_rest))
        return GS_ERR_UNSUPPORTED;
    const ForwardPlan f = plan_forward(*a);
    if (f.groups > 0x7fffffffLL) return GS_ERR_UNSUPPORTED;
    const size_t need = partial_bytes(*a, f.splits);
    if (need && !workspace) return GS_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < need) return GS_ERR_WORKSPACE_TOO_SMALL;
    Partial partial;
    const size_t rows = (size_t)a->rows_q * a->heads_q;
    partial.splits = f.splits;
    partial.sums = (float *)workspace;
    partial.max_sum = (float2 *)(partial.sums + f.splits * rows * a->dim);
    partial.count = f.by_keys ? (int32_t *)(partial.max_sum + f.splits * rows) : nullptr;
    const auto launch = [&](auto t) {
        return with_tile(a->dim, [&](auto d) {
            return launch_forward<decltype(t), decltype(d)::value>(
                *a, f, q, k, v, out, out_rest, log_sum, partial, stream);
        });
    };
    return a->type == GS_F16 ? launch(f16{}) : launch(bf16{});
}

extern "C" int gs_attention_backward_workspace_size(const GsAttention *a, size_t *bytes) {
    const int st = check_attention(a);
    if (st) return st;
    if (!bytes) return GS_ERR_INVALID_ARGUMENT;
    *bytes = backward_rows(*a) + backward_partials(*a, plan_backward(*a));
    return GS_OK;
}

extern "C" int gs_attention_backward(const GsAttention *a, const void *q, const void *k,
                                     const void *v, const void *out, const void *out_rest,
                                     const float *log_sum, const void *grad_out,
                                     int64_t grad_out_row,
                                     int64_t grad_out_head, void *grad_q, void *grad_k,
                                     void *grad_v, void *workspace, size_t workspace_bytes,
                                     hipStream_t stream) {
    size_t need = 0;
    int st = gs_attention_backward_workspace_size(a, &need);
    if (st) return st;
    if (grad_out_row < 0 || grad_out_head < 0) return GS_ERR_INVALID_ARGUMENT;
    if (a->rows_q > 0 && (!q || !out || !out_rest || !log_sum || !grad_out || !workspace))
        return GS_ERR_INVALID_ARGUMENT;
    if (!grad_k != !grad_v || (a->rows_k > 0 && (!k || !v))) return GS_ERR_INVALID_ARGUMENT;
    for (const void *x : {q, k, v, out, out_rest, grad_out, (const void *)grad_q, (const void *)grad_k,
                          (const void *)grad_v})
        if (!aligned16(x)) return GS_ERR_UNSUPPORTED;
    if ((grad_out_row | grad_out_head) % 8 != 0 || !tile_stride(grad_out_row, a->dim))
        return GS_ERR_UNSUPPORTED;
    if (workspace_bytes < need) return GS_ERR_WORKSPACE_TOO_SMALL;
    BackwardPlan b = plan_backward(*a);
    if (!grad_q) b.splits_q = 1;
    const int64_t blocks_q = b.tiles_q * a->heads_k * b.splits_q;
    const int64_t blocks_k = b.tiles_k * a->heads_k * b.splits_k;
    if (blocks_q > 0x7fffffffLL || blocks_k > 0x7fffffffLL) return GS_ERR_UNSUPPORTED;
    float *row_log = (float *)workspace, *row_delta = row_log + a->rows_q * a->heads_q;
    float *partial = (float *)((char *)workspace + backward_rows(*a));
    const auto launch = [&](auto t, auto d) {
        using T = decltype(t);
        constexpr int kDim = decltype(d)::value;
        const dim3 block(64 * kWaves);
        const auto join = [&](int64_t size, int splits, int outputs, float scale0, T *out0, T *out1) {
            hipLaunchKernelGGL((attention_sum_kernel<T>), dim3((unsigned)((size / 4 + 255) / 256), outputs),
                               dim3(256), 0, stream, (const float *)partial, size, splits, scale0,
                               1.0f, out0, out1);
        };
        if (a->rows_q > 0 && (grad_q || grad_k)) {
            hipLaunchKernelGGL((attention_dq_kernel<T, kDim>), dim3((unsigned)blocks_q),
                               block, 0, stream, *a, (const T *)q, (const T *)k, (const T *)v,
                               (const T *)out, (const T *)out_rest, log_sum, (const T *)grad_out,
                               grad_out_row, grad_out_head, (T *)grad_q, row_log, row_delta,
                               partial, b.splits_q);
            if (b.splits_q > 1)
                join(a->rows_q * a->heads_q * a->dim, b.splits_q, 1, a->scale, (T *)grad_q,
                     (T *)nullptr);
            const int s = launch_status();
            if (s) return s;
        }
        if (a->rows_k > 0 && grad_k) {
            hipLaunchKernelGGL((attention_dkv_kernel<T, kDim>), dim3((unsigned)blocks_k),
                               dim3(64 * KeysShape<kDim>::kWaves), 0, stream, *a, (const T *)q,
                               (const T *)k, (const T *)v, (const T *)grad_out, grad_out_row, grad_out_head, row_log, row_delta,
                               (T *)grad_k, (T *)grad_v, partial, b.splits_k);
            if (b.splits_k > 1)
                join(a->rows_k * a->heads_k * a->dim, b.splits_k, 2, a->scale, (T *)grad_k,
                     (T *)grad_v);
        }
        return launch_status();
    };
    return a->type == GS_F16 ? with_tile(a->dim, [&](auto d) { return launch(f16{}, d); })
                             : with_tile(a->dim, [&](auto d) { return launch(bf16{}, d); });
}
