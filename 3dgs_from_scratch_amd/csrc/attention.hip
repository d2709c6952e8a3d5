// Attention over packed sequences with grouped heads, and its gradients:
//   S = scale q k^T over the keys a query sees,  P = exp(S - L),  L = log sum exp S
//   out = P v,  delta = sum_d dout out,  dS = P (dout v^T - delta)
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout
// with dk and dv summed over the query heads of a group.  Scores, softmax
// statistics and sums are in float.

#include <initializer_list>

#include "attention_forward.h"

namespace gs {

// Keys and values in packed rows.
template <typename T>
struct PackedKeys {
    static constexpr bool kHoles = false, kScores = false;
    const T *k, *v;
    __device__ __forceinline__ Span span(const GsAttention &a, int s) const { return span_of(a, s); }
    __device__ __forceinline__ int keys(const GsAttention &a, int s) const {
        return keys_of(a, s, rows_of(a.offsets_k, a.sequences, a.rows_k, s));
    }
    template <typename KTile>
    struct Reader {
        static constexpr uint64_t there = ~0ull;
        const GsAttention &a;
        const T *k, *v;
        int lk, wave;
        typename KTile::Copy copy_k, copy_v;
        __device__ __forceinline__ Reader(const PackedKeys &s, const GsAttention &a, const Span &p,
                                          int, int kh, int wave, int, int)
            : a(a), k(s.k + p.k0 * a.k_row + kh * a.k_head), v(s.v + p.k0 * a.v_row + kh * a.v_head),
              lk(p.lk), wave(wave), copy_k(KTile::copy_of(wave, a.k_row, a.dim)),
              copy_v(KTile::copy_of(wave, a.v_row, a.dim)) {}
        // Starts the copies of a tile of keys and, behind it, of values.
        __device__ __forceinline__ void fetch(int t, lds_char *to) {
            const int64_t key = (int64_t)t * KTile::kRows;
            const int rows = lk - t * KTile::kRows;
            KTile::start(copy_k, wave, k + key * a.k_row, a.k_row, rows, a.dim, to);
            KTile::start(copy_v, wave, v + key * a.v_row, a.v_row, rows, a.dim, to + KTile::kBytes);
        }
    };
};

template <typename T, int DIM, bool LOG_SUM>
__global__ __launch_bounds__(64 * kWaves, 2) void attention_kernel(
    GsAttention a, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    T *__restrict__ out, T *__restrict__ out_rest, float *__restrict__ log_sum, Partial partial) {
    __shared__ __attribute__((aligned(1024))) char lds[Forward<T, DIM, false>::kLds];
    forward_tile<T, DIM, LOG_SUM>(a, PackedKeys<T>{k, v}, q, out, out_rest, log_sum, partial,
                                  (lds_char *)lds);
}

template <typename T, int DIM>
__global__ __launch_bounds__(64 * kKeysWaves, DIM > 96 ? 1 : 2) void attention_keys_kernel(
    GsAttention a, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    T *__restrict__ out, T *__restrict__ out_rest, float *__restrict__ log_sum, Partial partial) {
    __shared__ __attribute__((aligned(1024))) char lds[Forward<T, DIM, true>::kLds];
    forward_shared<T, DIM, true>(a, PackedKeys<T>{k, v}, q, out, out_rest, log_sum, partial,
                                 (lds_char *)lds);
}

template <typename T>
__global__ __launch_bounds__(256) void attention_join_kernel(int64_t rows, int dim, Partial partial,
                                                             T *__restrict__ out,
                                                             T *__restrict__ out_rest,
                                                             float *__restrict__ log_sum) {
    __shared__ f32x4 sums[8][32];
    join_row<T>(blockIdx.x, rows, dim, partial, out, out_rest, log_sum, sums);
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

static ForwardPlan plan_forward(const GsAttention &a) {
    return plan_forward(a, a.rows_k, a.rows_k / (a.sequences > 0 ? a.sequences : 1));
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
    if (!launchable(f.groups, 64 * kWaves)) return GS_ERR_UNSUPPORTED;
    const size_t need = partial_bytes(*a, f.splits);
    if (need && !workspace) return GS_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < need) return GS_ERR_WORKSPACE_TOO_SMALL;
    const Partial partial = partial_of(*a, f, f.by_keys, workspace);
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
