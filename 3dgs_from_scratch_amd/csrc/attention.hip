// Attention over packed sequences with grouped heads, and its gradients:
//   S = scale q k^T over the keys a query sees,  P = exp(S - L),  L = log sum exp S
//   out = P v,  delta = sum_d dout out,  dS = P (dout v^T - delta)
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout
// with dk and dv summed over the query heads of a group.  Scores, softmax
// statistics and sums are in float.

#include <type_traits>

#include "attention_tile.h"

namespace gs {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kWaves = 4;

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

// One 32x32 result of a wave's 32 columns, DIM rows: written as 16-bit rows of the
// columns' own addresses.
template <typename T, int DIM>
__device__ __forceinline__ void store_columns(const f32x16 *acc, float factor, T *row, int dim) {
    const int h = __lane_id() >> 5;
#pragma unroll
    for (int d = 0; d < DIM / 32; ++d) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {  // registers 8 g to 8 g + 7: rows 16 g + ...
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = acc[d][8 * g + i] * factor;
            const u32x4 w = __builtin_bit_cast(u32x4, pack8<T>(v));
            // a half holds rows 4 h + 0..3 and 8 + 4 h + 0..3; after the exchange
            // half h holds 8 h + 0..7
            const auto lo = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
            const auto hi = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
            const u32x4 o = {(uint32_t)lo[0], (uint32_t)hi[0], (uint32_t)lo[1], (uint32_t)hi[1]};
            const int at = 32 * d + 16 * g + 8 * h;
            if (row && at < dim) *(u32x4 *)(row + at) = o;
        }
    }
}

// Whether `rows` rows of a tile hold an infinity or a NaN; the same in every lane.
template <typename T, int DIM>
__device__ __forceinline__ bool not_finite(const lds_char *tile, int base, int rows) {
    using u16x8 = __attribute__((ext_vector_type(8))) uint16_t;
    u16x8 most = {};
    for (int at = __lane_id() * 16; at < rows * DIM * 2; at += 1024) {
        const u16x8 x = *(const __attribute__((address_space(3))) u16x8 *)(tile + base * DIM * 2 + at);
        most = __builtin_elementwise_max(most, x & (uint16_t)0x7fff);
    }
    uint16_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = most[i] > m ? most[i] : m;
    return __ballot(m >= (std::is_same<T, bf16>::value ? 0x7f80 : 0x7c00)) != 0;
}

// acc += V^T P^T over `groups` groups of 16 keys where V holds infinities or NaN that some
// columns do not see: a key at a time, added to the columns that see it.  last: the last key
// a column sees, from `base`.
template <typename T, int DIM, typename VTile>
__device__ __forceinline__ void add_seen(f32x16 *acc, const lds_char *tile, int base,
                                         const typename Vec<T>::x8 *p, int groups, int last) {
    const int half = __lane_id() >> 5;
#pragma unroll 1
    for (int key = 0; key < 16 * groups; ++key) {
        const int g = key >> 4;
        const auto only = [&](typename Vec<T>::x8 x) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (result_row(j, half) != (key & 15)) x[j] = (T)0.0f;
            return x;
        };
        const auto weights = only(g == 0 ? p[0] : g == 1 ? p[1] : g == 2 ? p[2] : p[3]);
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d) {
            const f32x16 one = mfma(only(VTile::down(tile, base + 16 * g, d)), weights, f32x16{});
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] += key <= last ? one[r] : 0.0f;
        }
    }
}

// Forward.  A workgroup takes a tile of packed rows of one key head (row r of a
// sequence: query r / group, head r % group of the group) and walks the sequence's
// keys, or a split's part of them, once:
//   S^T = K Q^T,  P = exp2(c S - m),  O^T += V^T P^T
// with a row in a lane pair, so that the softmax needs one exchange and the factors
// that follow a new maximum none.  K and V go from memory into LDS beside the work on
// the tile before.  BY_KEYS: a few rows only; the waves share the rows and split the
// keys of a tile, and join at the end.
template <typename T, int DIM, bool BY_KEYS>
struct Forward {
    static constexpr int kSub = BY_KEYS ? 1 : 2;                    // 32-key parts of a wave
    static constexpr int kKeys = BY_KEYS ? 32 * kWaves : 32 * kSub;  // of a tile
    static constexpr int kRows = BY_KEYS ? 32 : 32 * kWaves;
    using KTile = Tile<T, DIM, kKeys, kWaves>;
    static constexpr int kLds = 4 * KTile::kBytes;
    static_assert(!BY_KEYS || kLds >= kWaves * 64 * DIM / 2 * 4 + kWaves * 64 * 8, "the join");
};

// Rows of a split: un-normalised sums, and their maximum and sum of weights.
struct Partial {
    float *sums;        // (split, row, head, dim)
    float2 *max_sum;    // (split, row, head)
    int splits;
};

template <typename T, int DIM, bool BY_KEYS>
__global__ __launch_bounds__(64 * kWaves, BY_KEYS ? 1 : 2) void attention_kernel(
    GsAttention a, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    T *__restrict__ out, float *__restrict__ log_sum, Partial partial) {
    using F = Forward<T, DIM, BY_KEYS>;
    using KTile = typename F::KTile;
    __shared__ __attribute__((aligned(1024))) char lds[F::kLds];
    lds_char *const tiles = (lds_char *)lds;

    // key heads next to each other: with 8 or a divisor of 8 of them, an XCD's L2 holds one
    const int kh = blockIdx.x % a.heads_k, group = a.heads_q / a.heads_k;
    int sequence, number;
    if (!find_tile(a.offsets_q, a.sequences, a.rows_q, group, F::kRows, blockIdx.x / a.heads_k,
                   &sequence, &number))
        return;
    const Span p = span_of(a, sequence);
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
    const int share = (tiles_all + partial.splits - 1) / partial.splits;
    const int first_tile = min((int)blockIdx.y * share, tiles_all);
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
    float top = -INFINITY, sum = 0.0f;  // of c S; the sum of this half's keys

    const auto step = [&](int t, auto masks) {
        constexpr bool kMasks = decltype(masks)::value;
        __syncthreads();  // tile t is in LDS, and tile t - 1 has been read
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
        bool split_keys = false;
        if constexpr (kMasks) {
            // 0 times an infinity is no 0: a value that some rows of the tile do not see
            // must not meet their weights
            if (a.causal) split_keys = not_finite<T, DIM>(vt, base, 32 * F::kSub);
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
#pragma unroll
            for (int d = 0; d < DIM / 32; ++d) acc[d] *= keep;
        }
        const float minus = top == -INFINITY ? 0.0f : -top;
        typename Vec<T>::x8 weights[4] = {};  // (2 kSub are used)
#pragma unroll
        for (int n = 0; n < F::kSub; ++n) {
            float w[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                w[r] = __builtin_amdgcn_exp2f(fmaf(s[n][r], c, minus));
                sum += w[r];
            }
            weights[2 * n] = pack8<T>(w);
            weights[2 * n + 1] = pack8<T>(w + 8);
        }
        if constexpr (kMasks)
            if (split_keys) {
                add_seen<T, DIM, KTile>(acc, vt, base, weights, 2 * F::kSub, last - key0);
                return;
            }
#pragma unroll
        for (int g = 0; g < 2 * F::kSub; ++g)
#pragma unroll
            for (int d = 0; d < DIM / 32; ++d)
                acc[d] = mfma(KTile::down(vt, base + 16 * g, d), weights[g], acc[d]);
    };
    if (first_tile < end_tile) fetch(first_tile);
    int t = first_tile;
    // tiles that every row of the workgroup sees whole, then the others
    for (const int whole = min(end_tile, (all_see + 1) / F::kKeys); t < whole; ++t)
        step(t, std::false_type{});
    for (; t < end_tile; ++t) step(t, std::true_type{});
    sum = half_sum(sum);

    if constexpr (BY_KEYS) {
        // the four waves' sums over their keys, in LDS: wave w adds up the w-th quarter
        // of the registers
        __syncthreads();  // the tiles have been read
        float *sums = (float *)lds;  // (wave, register, lane)
        float2 *stats = (float2 *)(sums + kWaves * (DIM / 2) * 64);
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) sums[(wave * (DIM / 2) + 16 * d + r) * 64 + lane] = acc[d][r];
        stats[wave * 64 + lane] = make_float2(top, sum);
        __syncthreads();
        if (wave) return;
        float all = top, weight[kWaves], total = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) all = fmaxf(all, stats[w * 64 + lane].x);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float2 o = stats[w * 64 + lane];
            weight[w] = o.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(o.x - all);
            total = fmaf(o.y, weight[w], total);
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
        sum = total;
    }

    if (partial.splits > 1) {
        const int64_t slot = (int64_t)blockIdx.y * a.rows_q * a.heads_q + at;
        if (real && half == 0) partial.max_sum[slot] = make_float2(top, sum);
        if (real && top != -INFINITY) {
#pragma unroll
            for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int column = 32 * d + result_row(4 * g, half);
                    if (column < a.dim)
                        *(float4 *)(partial.sums + slot * a.dim + column) =
                            make_float4(acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2],
                                        acc[d][4 * g + 3]);
                }
        }
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
    store_columns<T, DIM>(acc, none ? 1.0f : 1.0f / sum, real ? out + at * a.dim : nullptr, a.dim);
    if (log_sum && real && half == 0)
        log_sum[at] = none ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// Joins the splits of a row: a wave a row, two elements a lane.
template <typename T>
__global__ __launch_bounds__(256) void attention_join_kernel(int64_t rows, int dim, Partial partial,
                                                             T *__restrict__ out,
                                                             float *__restrict__ log_sum) {
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    if (row >= rows) return;
    const int lane = __lane_id();
    const float2 mine = lane < partial.splits ? partial.max_sum[lane * rows + row]
                                              : make_float2(-INFINITY, 0.0f);
    float top = mine.x;
#pragma unroll
    for (int o = kWave / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
    const float weight = mine.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mine.x - top);
    const float sum = wave_sum(mine.x == -INFINITY ? 0.0f : mine.y * weight);
    const bool in = 2 * lane < dim;
    float x = 0.0f, y = 0.0f;
    for (int s = 0; s < partial.splits; ++s) {
        const float w = __shfl(weight, s, kWave);
        if (__shfl(mine.x, s, kWave) == -INFINITY) continue;
        if (!in) continue;
        const float2 o = *(const float2 *)(partial.sums + (s * rows + row) * dim + 2 * lane);
        x = fmaf(o.x, w, x);
        y = fmaf(o.y, w, y);
    }
    const bool none = top == -INFINITY;
    const float r = none ? 0.0f : 1.0f / sum;
    if (in) {
        const typename Vec<T>::x2 o = {(T)(x * r), (T)(y * r)};
        *(typename Vec<T>::x2 *)(out + row * dim + 2 * lane) = o;
    }
    if (log_sum && lane == 0) log_sum[row] = none ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// ---------------------------------------------------------------- gradients
__device__ __forceinline__ int sequence_of(const int32_t *offsets, int sequences, int64_t row) {
    int s = 0;
    while (s <= sequences && row >= offsets[s]) ++s;
    return s;
}

template <typename T>
__global__ __launch_bounds__(64) void attention_dq_kernel(
    GsAttention a, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    const T *__restrict__ out, const float *__restrict__ log_sum, const T *__restrict__ go,
    int64_t go_row, int64_t go_head, T *__restrict__ dq, float *__restrict__ delta) {
    const int64_t row = blockIdx.x;
    const int head = blockIdx.y, kh = head / (a.heads_q / a.heads_k), lane = threadIdx.x;
    const int s = sequence_of(a.offsets_q, a.sequences, row);
    const Span p = span_of(a, s);
    const int64_t keys = p.lk, i = row - p.q0, lq = p.lq;
    const int64_t seen = a.causal ? clamp_row(i + keys - lq + 1, 0, keys) : keys;
    const bool one = lane < a.dim, two = lane + 64 < a.dim;
    const T *qr = q + row * a.q_row + head * a.q_head;
    const T *gr = go + row * go_row + head * go_head;
    const int64_t at = row * a.heads_q + head;
    const float q0 = one ? to_float(qr[lane]) * a.scale : 0.0f;
    const float q1 = two ? to_float(qr[lane + 64]) * a.scale : 0.0f;
    const float g0 = one ? to_float(gr[lane]) : 0.0f, g1 = two ? to_float(gr[lane + 64]) : 0.0f;
    const float d = wave_sum(fmaf(g0, one ? to_float(out[at * a.dim + lane]) : 0.0f,
                                  g1 * (two ? to_float(out[at * a.dim + lane + 64]) : 0.0f)));
    if (lane == 0) delta[at] = d;
    const float l = log_sum[at];
    float s0 = 0.0f, s1 = 0.0f;
    for (int64_t j = 0; j < seen && l != -INFINITY; ++j) {
        const T *kr = k + (p.k0 + j) * a.k_row + kh * a.k_head;
        const T *vr = v + (p.k0 + j) * a.v_row + kh * a.v_head;
        const float k0 = one ? to_float(kr[lane]) : 0.0f, k1 = two ? to_float(kr[lane + 64]) : 0.0f;
        const float w = expf(wave_sum(fmaf(k0, q0, k1 * q1)) - l);
        const float gp = wave_sum(fmaf(g0, one ? to_float(vr[lane]) : 0.0f,
                                       g1 * (two ? to_float(vr[lane + 64]) : 0.0f)));
        const float ds = w * (gp - d);
        s0 = fmaf(ds, k0, s0);
        s1 = fmaf(ds, k1, s1);
    }
    T *dst = dq + at * a.dim;
    if (one) dst[lane] = from_float<T>(s0 * a.scale);
    if (two) dst[lane + 64] = from_float<T>(s1 * a.scale);
}

template <typename T>
__global__ __launch_bounds__(64) void attention_dkv_kernel(
    GsAttention a, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    const float *__restrict__ log_sum, const T *__restrict__ go, int64_t go_row, int64_t go_head,
    const float *__restrict__ delta, T *__restrict__ dk, T *__restrict__ dv) {
    const int64_t row = blockIdx.x;
    const int kh = blockIdx.y, group = a.heads_q / a.heads_k, lane = threadIdx.x;
    const int s = sequence_of(a.offsets_k, a.sequences, row);
    const Span p = span_of(a, s);
    const int64_t keys = p.lk, j = row - p.k0, lq = p.lq;
    int64_t first = a.causal ? j + lq - keys : 0;
    if (first < 0) first = 0;
    if (j >= keys) first = lq;
    const bool one = lane < a.dim, two = lane + 64 < a.dim;
    const T *kr = k + row * a.k_row + kh * a.k_head, *vr = v + row * a.v_row + kh * a.v_head;
    const float k0 = one ? to_float(kr[lane]) * a.scale : 0.0f;
    const float k1 = two ? to_float(kr[lane + 64]) * a.scale : 0.0f;
    const float v0 = one ? to_float(vr[lane]) : 0.0f, v1 = two ? to_float(vr[lane + 64]) : 0.0f;
    float dk0 = 0.0f, dk1 = 0.0f, dv0 = 0.0f, dv1 = 0.0f;
    for (int64_t i = first; i < lq; ++i)
        for (int g = 0; g < group; ++g) {
            const int64_t r = p.q0 + i, head = kh * group + g, at = r * a.heads_q + head;
            const float l = log_sum[at];
            if (l == -INFINITY) continue;
            const T *qr = q + r * a.q_row + head * a.q_head;
            const T *gr = go + r * go_row + head * go_head;
            const float q0 = one ? to_float(qr[lane]) : 0.0f;
            const float q1 = two ? to_float(qr[lane + 64]) : 0.0f;
            const float g0 = one ? to_float(gr[lane]) : 0.0f;
            const float g1 = two ? to_float(gr[lane + 64]) : 0.0f;
            const float w = expf(wave_sum(fmaf(k0, q0, k1 * q1)) - l);
            const float ds = w * (wave_sum(fmaf(g0, v0, g1 * v1)) - delta[at]);
            dk0 = fmaf(ds, q0, dk0);
            dk1 = fmaf(ds, q1, dk1);
            dv0 = fmaf(w, g0, dv0);
            dv1 = fmaf(w, g1, dv1);
        }
    const int64_t at = (row * a.heads_k + kh) * a.dim;
    if (one) {
        dk[at + lane] = from_float<T>(dk0 * a.scale);
        dv[at + lane] = from_float<T>(dv0);
    }
    if (two) {
        dk[at + lane + 64] = from_float<T>(dk1 * a.scale);
        dv[at + lane + 64] = from_float<T>(dv1);
    }
}

constexpr int64_t kMaxRows = 0x7fffffffLL - 65536;  // row numbers stay in 32 bits
constexpr int64_t kMaxStride = 1 << 23;             // and byte offsets in a tile

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
        a->k_row > kMaxStride || a->v_row > kMaxStride ||
        (a->q_row | a->q_head | a->k_row | a->k_head | a->v_row | a->v_head) % 8 != 0)
        return GS_ERR_UNSUPPORTED;
    return GS_OK;
}

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// How a forward is launched.
struct ForwardPlan {
    bool by_keys;
    int64_t tiles;
    int splits;
};

static ForwardPlan plan_forward(const GsAttention &a) {
    const int64_t group = a.heads_q / a.heads_k, packed = a.rows_q * group;
    const int64_t sequences = a.sequences > 0 ? a.sequences : 1;
    ForwardPlan f;
    f.by_keys = packed <= 32 * sequences;
    const int rows = f.by_keys ? 32 : 32 * kWaves;
    f.tiles = packed / rows + a.sequences + 2;
    // Workgroups that will find rows, at least, and how many splits of the keys fill the
    // card with them; a split of fewer than four tiles costs more than it hides.
    int64_t busy = (packed + rows - 1) / rows;
    if (busy < sequences) busy = sequences < a.rows_q ? sequences : a.rows_q;
    busy = busy > 0 ? busy * a.heads_k : 1;
    const int64_t want = (512 + busy - 1) / busy;
    const int64_t most = a.rows_k / sequences / (f.by_keys ? 512 : 256);
    int64_t splits = want < most ? want : most;
    f.splits = (int)(splits < 1 ? 1 : splits > 64 ? 64 : splits);
    return f;
}

static size_t partial_bytes(const GsAttention &a, int splits) {
    if (splits == 1) return 0;
    return (size_t)splits * a.rows_q * a.heads_q * (a.dim * sizeof(float) + sizeof(float2));
}

template <typename T, int DIM>
static int launch_forward(const GsAttention &a, const ForwardPlan &f, const void *q, const void *k,
                          const void *v, void *out, float *log_sum, const Partial &partial,
                          hipStream_t stream) {
    const dim3 grid((unsigned)(f.tiles * a.heads_k), f.splits);
    if (f.by_keys)
        hipLaunchKernelGGL((attention_kernel<T, DIM, true>), grid, dim3(64 * kWaves), 0, stream, a,
                           (const T *)q, (const T *)k, (const T *)v, (T *)out, log_sum, partial);
    else
        hipLaunchKernelGGL((attention_kernel<T, DIM, false>), grid, dim3(64 * kWaves), 0, stream, a,
                           (const T *)q, (const T *)k, (const T *)v, (T *)out, log_sum, partial);
    int st = launch_status();
    if (st || f.splits == 1) return st;
    const int64_t rows = a.rows_q * a.heads_q;
    hipLaunchKernelGGL((attention_join_kernel<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0,
                       stream, rows, a.dim, partial, (T *)out, log_sum);
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
                                    const void *v, void *out, float *log_sum, void *workspace,
                                    size_t workspace_bytes, hipStream_t stream) {
    const int st = check_attention(a);
    if (st) return st;
    if (a->rows_q == 0) return GS_OK;
    if (!q || !out || (a->rows_k > 0 && (!k || !v))) return GS_ERR_INVALID_ARGUMENT;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
        return GS_ERR_UNSUPPORTED;
    const ForwardPlan f = plan_forward(*a);
    if (f.tiles * a->heads_k > 0x7fffffffLL) return GS_ERR_UNSUPPORTED;
    const size_t need = partial_bytes(*a, f.splits);
    if (need && !workspace) return GS_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < need) return GS_ERR_WORKSPACE_TOO_SMALL;
    Partial partial;
    partial.splits = f.splits;
    partial.sums = (float *)workspace;
    partial.max_sum = (float2 *)((float *)workspace + (size_t)f.splits * a->rows_q * a->heads_q * a->dim);
    const auto launch = [&](auto t) {
        return with_tile(a->dim, [&](auto d) {
            return launch_forward<decltype(t), decltype(d)::value>(*a, f, q, k, v, out, log_sum,
                                                                   partial, stream);
        });
    };
    return a->type == GS_F16 ? launch(f16{}) : launch(bf16{});
}

extern "C" int gs_attention_backward_workspace_size(const GsAttention *a, size_t *bytes) {
    const int st = check_attention(a);
    if (st) return st;
    if (!bytes) return GS_ERR_INVALID_ARGUMENT;
    *bytes = (size_t)a->rows_q * a->heads_q * sizeof(float);
    return GS_OK;
}

extern "C" int gs_attention_backward(const GsAttention *a, const void *q, const void *k,
                                     const void *v, const void *out, const float *log_sum,
                                     const void *grad_out, int64_t grad_out_row,
                                     int64_t grad_out_head, void *grad_q, void *grad_k,
                                     void *grad_v, void *workspace, size_t workspace_bytes,
                                     hipStream_t stream) {
    size_t need = 0;
    int st = gs_attention_backward_workspace_size(a, &need);
    if (st) return st;
    if (grad_out_row < 0 || grad_out_head < 0) return GS_ERR_INVALID_ARGUMENT;
    if (a->rows_q > 0 && (!q || !out || !log_sum || !grad_out || !grad_q || !workspace))
        return GS_ERR_INVALID_ARGUMENT;
    if (a->rows_k > 0 && (!k || !v || !grad_k || !grad_v)) return GS_ERR_INVALID_ARGUMENT;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(grad_out) ||
        (grad_out_row | grad_out_head) % 8 != 0)
        return GS_ERR_UNSUPPORTED;
    if (workspace_bytes < need) return GS_ERR_WORKSPACE_TOO_SMALL;
    const auto launch = [&](auto t) {
        using T = decltype(t);
        if (a->rows_q > 0) {
            hipLaunchKernelGGL((attention_dq_kernel<T>), dim3((unsigned)a->rows_q, a->heads_q),
                               dim3(64), 0, stream, *a, (const T *)q, (const T *)k, (const T *)v,
                               (const T *)out, log_sum, (const T *)grad_out, grad_out_row,
                               grad_out_head, (T *)grad_q, (float *)workspace);
            const int s = launch_status();
            if (s) return s;
        }
        if (a->rows_k > 0)
            hipLaunchKernelGGL((attention_dkv_kernel<T>), dim3((unsigned)a->rows_k, a->heads_k),
                               dim3(64), 0, stream, *a, (const T *)q, (const T *)k, (const T *)v,
                               log_sum, (const T *)grad_out, grad_out_row, grad_out_head,
                               (const float *)workspace, (T *)grad_k, (T *)grad_v);
        return launch_status();
    };
    return a->type == GS_F16 ? launch(f16{}) : launch(bf16{});
}
