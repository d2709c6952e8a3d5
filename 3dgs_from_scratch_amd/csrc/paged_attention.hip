// Attention of new tokens over a paged cache, and the attention that its keys get:
//   S = scale q k^T over the slots a query sees,  L = log sum exp S,  out = exp(S - L) v
//   weight of a slot and head += sum over queries and heads of the group of exp(S - L)
// Scores, softmax statistics and sums are in float.

#include <cmath>

#include "attention_forward.h"
#include "paged.h"

namespace gs {

// Sequence s = 1 .. sequences, as in GsAttention; 0 and sequences + 1 have no keys.
__device__ __forceinline__ int slots_of(const GsPages &p, int s) {
    return s == 0 || s > p.sequences ? 0 : filled_slots(p, s - 1);
}

__device__ const __attribute__((aligned(16))) uint32_t kZeros[4] = {0, 0, 0, 0};

// Keys and values in pages.  WHOLE: pages of a multiple of a tile's rows, so that a tile lies in
// one; else each row of a tile finds its own, and a wave copies the rows of its 64 chunks as they
// follow one another in a page, or chunk by chunk where a page ends between them.  A tile's pages
// are read from the table while the tile before it is copied; a bit tells each row that is there.
//
// 2 sequences, 8160 queries each over 28284 and 32640 slots, 16 heads on 4, dim 128: 3.32 ms in pages of
// 256, 3.28 in packed rows, 3.58 in pages of 16 (4.0 where every chunk's row is exchanged between
// lanes, and no copy takes rows together).  Finding a tile's rows at the end of the step before, or between its
// products, took 2 to 8% longer: the registers that hold what was found are the products'.
//
// SCORES: the scores of few rows are kept, for the slots' weights.  The stores are waited for with the
// next tile's copies: 16 single tokens over 2500 to 32640 slots, dim 128, 97 us instead of 81.
template <typename T, bool WHOLE, bool SCORES = false>
struct PagedKeys {
    static constexpr bool kHoles = true, kScores = SCORES;
    GsPages p;
    const T *k, *v;
    float *scores;        // (row and head, slot)
    int64_t score_slots;  // of a row, a multiple of 64
    // Scores of a row and head in a lane's registers, its first slot: four slots in every eight.
    __device__ __forceinline__ void keep(int64_t row, int slot, const f32x16 &s) const {
        float *to = scores + row * score_slots + slot;
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *(float4 *)(to + 8 * g) = make_float4(s[4 * g], s[4 * g + 1], s[4 * g + 2], s[4 * g + 3]);
    }
    __device__ __forceinline__ Span span(const GsAttention &a, int s) const {
        const int2 q = rows_of(a.offsets_q, a.sequences, a.rows_q, s);
        return {uniform(q.x), uniform(q.y - q.x), 0, uniform(slots_of(p, s)), 0};
    }
    __device__ __forceinline__ int keys(const GsAttention &, int s) const { return slots_of(p, s); }

    template <typename KTile>
    struct Reader {
        static_assert(KTile::kRows == 64, "a bit a row");
        const GsPages &p;
        const T *k, *v;
        const int32_t *table;
        int wave, lk, end;
        uint64_t there;  // of the tile that was fetched last
        // WHOLE: of the tile that is looked for next; else of the lane's row of it
        int index, place, page;
        int more_pages, more_places;  // of a tile's rows: whole pages, and places
        // byte offsets of the lane's chunks from the tile's (WHOLE) or the copy's first row; past
        // every bound where the chunk lies behind the dimension
        typename KTile::Copy copy;
        // the tile that is fetched next.  WHOLE: its first element; else of the lane's row: bytes from
        // the first element, below 0 where it is not there, and how many may be copied from it, -1
        // where a page ends among the rows of the copy that it begins
        uint64_t ready;
        int64_t from;
        int bytes;

        __device__ __forceinline__ Reader(const PagedKeys &s, const GsAttention &, const Span &span,
                                          int sequence, int kh, int wave, int first, int end)
            : p(s.p), k(s.k + kh * s.p.head_stride), v(s.v + kh * s.p.head_stride),
              table(s.p.tables + (int64_t)(sequence - 1) * s.p.table_stride), wave(wave), lk(span.lk),
              end(end), there(0) {
            const int slot = first * KTile::kRows + (WHOLE ? 0 : (int)__lane_id());
            index = slot / p.page_size;
            place = slot - index * p.page_size;
            more_pages = KTile::kRows / p.page_size;
            more_places = KTile::kRows - more_pages * p.page_size;
            copy = KTile::copy_of(wave, p.slot_stride, p.dim);
            if constexpr (!WHOLE) {
#pragma unroll
                for (int i = 0; i < KTile::kCopies; ++i)
                    copy.from[i] -= copy.from[i] >> 31 ? 0u : first_row(i) * (uint32_t)p.slot_stride * 2u;
            }
            look(first);
        }
        // The first row that the wave's copy i has chunks of.
        __device__ __forceinline__ int first_row(int i) const {
            return (i * KTile::kCopyWaves + wave) * 64 / KTile::kChunks;
        }
        __device__ __forceinline__ void look(int t) {
            const bool is = WHOLE ? t < end : t * KTile::kRows + (int)__lane_id() < lk;
            page = is ? table[index] : -1;
        }
        // Finds the tile that was looked for.
        __device__ __forceinline__ void prepare() {
            if constexpr (WHOLE) {
                const int32_t number = uniform(page);
                const bool is = (uint32_t)number < (uint64_t)p.pages;
                from = is ? row_at(p, number, place) : 0;
                ready = is ? ~0ull : 0;
                place += KTile::kRows;
                if (place == p.page_size) place = 0, ++index;
            } else {
                const bool is = (uint32_t)page < (uint64_t)p.pages;
                ready = __ballot(is);
                const uint64_t begins = __ballot(place == 0);  // rows that begin a page
                from = is ? row_at(p, page, place) * 2 : -1;
                // a copy that begins here: rows in one page, of which those that are there come first
                constexpr int rows = (64 + KTile::kChunks - 1) / KTile::kChunks;
                const int row = __lane_id();
                const int n = __popcll((ready >> row) & ((1ull << rows) - 1));
                const bool breaks = (begins >> row >> 1) & ((1ull << (rows - 1)) - 1);
                bytes = breaks ? -1 : n ? ((n - 1) * (int)p.slot_stride + p.dim) * 2 : 0;
                place += more_places;
                index += more_pages;
                if (place >= p.page_size) place -= p.page_size, ++index;
            }
        }
        // Starts the copies of a tile of keys and, behind it, of values.  Tiles come in order.
        __device__ __forceinline__ void fetch(int t, lds_char *to) {
            prepare();
            there = ready;
            look(t + 1);  // (before the copies, so that it is there before them)
            if constexpr (WHOLE) {
                const int rows = ready ? lk - t * KTile::kRows : 0;
                KTile::start(copy, wave, k + from, p.slot_stride, rows, p.dim, to);
                KTile::start(copy, wave, v + from, p.slot_stride, rows, p.dim, to + KTile::kBytes);
            } else {
                const int low = (int)from, high = (int)(from >> 32);
#pragma unroll
                for (int i = 0; i < KTile::kCopies; ++i) {
                    const int piece = i * KTile::kCopyWaves + wave;
                    if (KTile::kPieces % KTile::kCopyWaves != 0 && piece >= KTile::kPieces) break;
                    lds_char *const key_to = to + piece * 1024, *const value_to = key_to + KTile::kBytes;
                    const int row0 = first_row(i), many = __builtin_amdgcn_readlane(bytes, row0);
                    if (many >= 0) {
                        const int64_t at =
                            (int64_t)(uint32_t)__builtin_amdgcn_readlane(low, row0) |
                            (int64_t)__builtin_amdgcn_readlane(high, row0) << 32;
                        copy_rows((const char *)k + at, many, copy.from[i], key_to);
                        copy_rows((const char *)v + at, many, copy.from[i], value_to);
                        continue;
                    }
                    const int chunk_at = piece * 64 + (int)__lane_id(), row = chunk_at / KTile::kChunks;
                    const int chunk = (chunk_at % KTile::kChunks) ^ KTile::swizzle(row);
                    const int64_t mine = (int64_t)(uint32_t)__builtin_amdgcn_ds_bpermute(row * 4, low) |
                                         (int64_t)__builtin_amdgcn_ds_bpermute(row * 4, high) << 32;
                    const bool has = mine >= 0 && chunk * 8 < p.dim;
                    const int64_t byte = mine + chunk * 16;
                    copy_chunk(has ? (const char *)k + byte : (const char *)kZeros, key_to);
                    copy_chunk(has ? (const char *)v + byte : (const char *)kZeros, value_to);
                }
            }
        }
        // 16 bytes a lane to the wave's piece of LDS: from an offset, or zeros past the bound, or from
        // the lane's own address.
        static __device__ __forceinline__ void copy_rows(const char *first, int bytes, uint32_t from,
                                                         lds_char *to) {
            const auto all = __builtin_amdgcn_make_buffer_rsrc((void *)first, 0, bytes, 0x00027000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                all, (__attribute__((address_space(3))) void *)to, 16, from, 0, 0, 0);
        }
        static __device__ __forceinline__ void copy_chunk(const char *from, lds_char *to) {
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void *)from,
                (__attribute__((address_space(3))) void *)to, 16, 0, 0);
        }
    };
};

template <typename T, int DIM, bool LOG_SUM, bool WHOLE>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_attention_kernel(
    GsAttention a, GsPages p, const T *__restrict__ q, const T *__restrict__ k,
    const T *__restrict__ v, T *__restrict__ out, float *__restrict__ log_sum, Partial partial) {
    __shared__ __attribute__((aligned(1024))) char lds[Forward<T, DIM, false>::kLds];
    forward_tile<T, DIM, LOG_SUM>(a, PagedKeys<T, WHOLE>{p, k, v, nullptr, 0}, q, out, (T *)nullptr, log_sum,
                                  partial, (lds_char *)lds);
}

template <typename T, int DIM, bool WHOLE, bool SCORES>
__global__ __launch_bounds__(64 * kKeysWaves, DIM > 96 ? 1 : 2) void paged_attention_keys_kernel(
    GsAttention a, GsPages p, const T *__restrict__ q, const T *__restrict__ k,
    const T *__restrict__ v, T *__restrict__ out, float *__restrict__ log_sum, Partial partial,
    float *__restrict__ scores, int64_t score_slots) {
    __shared__ __attribute__((aligned(1024))) char lds[Forward<T, DIM, true>::kLds];
    forward_shared<T, DIM, true>(a, PagedKeys<T, WHOLE, SCORES>{p, k, v, scores, score_slots}, q, out,
                                 (T *)nullptr, log_sum, partial, (lds_char *)lds);
}

// Tiles of rows too few for the GPU: their keys in splits of equal length across sequences.
template <typename T, int DIM, bool WHOLE>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_attention_split_kernel(
    GsAttention a, GsPages p, const T *__restrict__ q, const T *__restrict__ k,
    const T *__restrict__ v, T *__restrict__ out, float *__restrict__ log_sum, Partial partial) {
    __shared__ __attribute__((aligned(1024))) char lds[Forward<T, DIM, false>::kLds];
    forward_shared<T, DIM, false>(a, PagedKeys<T, WHOLE>{p, k, v, nullptr, 0}, q, out, (T *)nullptr, log_sum,
                                  partial, (lds_char *)lds);
}

// Few rows with many splits: a workgroup a row.
template <typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(int64_t rows, int dim, Partial partial,
                                                         T *__restrict__ out,
                                                         float *__restrict__ log_sum) {
    __shared__ f32x4 sums[8][32];
    join_row<T>(blockIdx.x, rows, dim, partial, out, (T *)nullptr, log_sum, sums);
}

// Many rows with few splits: 32 threads a row, four elements each; a lane has the maximum and the
// sum of two splits.  6864 rows of up to 16 splits, dim 72: 5.9 us, and 9.0 in workgroups a row; 256
// rows of 28, dim 128: 6.9 and 4.8.
constexpr int kJoinRows = 8;  // of a workgroup

template <typename T>
__global__ __launch_bounds__(32 * kJoinRows) void paged_join_rows_kernel(
    int64_t rows, int dim, Partial partial, T *__restrict__ out, float *__restrict__ log_sum) {
    const int lane = threadIdx.x % 32, column = 4 * lane, half = __lane_id() & 32;
    const int64_t at = (int64_t)blockIdx.x * kJoinRows + threadIdx.x / 32;
    const int64_t row = at < rows ? at : rows - 1;  // (every lane takes part in the exchanges)
    const int splits = min(partial.count[row], partial.splits);
    float most[2], weight[2], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int s = lane + 32 * n;
        const float2 x = s < splits ? partial.max_sum[s * rows + row] : make_float2(-INFINITY, 0.0f);
        most[n] = x.x;
        weight[n] = x.y;
        top = fmaxf(top, x.x);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const float share = most[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(most[n] - top);
        sum += most[n] == -INFINITY ? 0.0f : weight[n] * share;
        weight[n] = share;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor(sum, o, kWave);
    const int all = max(splits, __shfl_xor(splits, 32, kWave));  // (the same rounds in every lane)
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kAhead = 4;
    for (int first = 0; first < all; first += kAhead) {
        f32x4 part[kAhead];
        float w[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int s = first + i, from = half + (s & 31);
            w[i] = s < 32 ? __shfl(weight[0], from, kWave) : __shfl(weight[1], from, kWave);
            // (a split that saw nothing has written no sums, and those past the last are as it)
            const float m = s < 32 ? __shfl(most[0], from, kWave) : __shfl(most[1], from, kWave);
            part[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (m != -INFINITY && s < splits && column < dim)
                part[i] = *(const f32x4 *)(partial.sums + (s * rows + row) * dim + column);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) x += part[i] * w[i];
    }
    if (at >= rows) return;
    const bool none = top == -INFINITY;
    const float r = 1.0f / sum;
    if (column < dim) {
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = none ? 0.0f : x[i] * r;
        store_floats<T, 4>(out + row * dim + column, o);
    }
    if (log_sum && lane == 0) log_sum[row] = none ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

// ---------------------------------------------------------------- slots' weights
// S = Q K^T once more, now that a row's log-sum L is known: a lane has a slot, and adds up
// exp2(c S - L) over the rows in its registers.  A slot and head is one wave's, and its sum is added
// to the weight at once: other sequences, or other places of the same, may have the page too.  Where
// none has, that is one addition, the same in every call.
// 16 rows of a tile are added in pairs, so that chains of additions grow by one for 32 rows.

// Sum over the 16 rows of a 32x32 result that a lane holds; minus: -L of each, minus infinity for
// rows that add nothing; sees(i): whether row i of the 32 counts for the lane's slot.
template <bool MASKS, typename Sees>
__device__ __forceinline__ float sum_of_weights(const f32x16 &s, float c, const float *minus, Sees sees) {
    const int half = __lane_id() >> 5;
    float w[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        w[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, minus[r]));
        if (MASKS) w[r] = sees(result_row(r, half)) ? w[r] : 0.0f;
    }
#pragma unroll
    for (int n = 8; n > 0; n >>= 1)
#pragma unroll
        for (int r = 0; r < n; ++r) w[r] += w[r + n];
    return w[0];
}

// -L in the exponent of two; a row that saw nothing adds nothing.
__device__ __forceinline__ float minus_log(float log_sum) {
    return log_sum == -INFINITY ? -INFINITY : -log_sum * kLog2e;
}

constexpr int kWeightSlots = 32 * kWaves;  // of a workgroup
constexpr int kScoreSlots = 256;           // and heads, of one where the scores are there

// The slots of a workgroup, and what its lanes have of them.
template <typename T, int DIM>
struct SlotOperand {
    RowOperand<T, DIM> k;
    float *weight;  // null: no such slot
    __device__ __forceinline__ SlotOperand(const GsPages &p, const T *keys, float *weights, int sequence,
                                           int slot, int filled, int kh, bool negate)
        : weight(nullptr) {
        const T *row = nullptr;
        if (slot < filled) {
            const int index = slot / p.page_size, place = slot - index * p.page_size;
            const int page = page_of(p, sequence - 1, index);
            if (page >= 0) {
                row = keys + row_at(p, page, place) + kh * p.head_stride;
                weight = weights + sum_at(p, page, place, kh);
            }
        }
        k.load(row, p.dim, negate);
    }
    // sum: of the lane's rows, half of all
    __device__ __forceinline__ void add(float sum) const {
        sum = half_sum(sum);
        if (__lane_id() < 32 && weight) unsafeAtomicAdd(weight, sum);
    }
};

// f(sequence, tile, part) for the tiles of so many slots of all sequences that have queries, each in
// `parts` parts (of key heads), from number `item` on every `every`th.  Most workgroups have one, and find
// it in one look through the sequences.
template <typename F>
__device__ __forceinline__ void for_slot_tiles(const GsAttention &a, const GsPages &p, int slots, int parts,
                                               int item, int every, F f) {
    const int lane = __lane_id();
    int upto = 0;  // places of 64 sequences up to and with the lane's
    const auto look = [&](int first) {  // all of them
        const int s = first + lane + 1;
        int n = 0;
        if (s <= a.sequences) {
            const int2 q = rows_of(a.offsets_q, a.sequences, a.rows_q, s);
            n = q.x == q.y ? 0 : (slots_of(p, s) + slots - 1) / slots * parts;
        }
        upto = (int)lanes_sum_upto((uint32_t)n);
        return __builtin_amdgcn_readlane(upto, kWave - 1);
    };
    int first = 0, before = 0, here = look(0);
    for (;;) {
        while (item - before >= here) {
            before += here;
            first += kWave;
            if (first >= a.sequences) return;
            here = look(first);
        }
        const int l = __builtin_ctzll(__ballot(before + upto > item));
        const int place = item - before - (l ? __builtin_amdgcn_readlane(upto, l - 1) : 0);
        f(first + l + 1, place / parts, place % parts);
        item += every;
    }
}

// Many rows: tiles of a head's queries go through LDS, which the workgroup's waves share.  No unit is
// full: of the busy time matrix instructions take 43%, the others 54%, an exponential, a multiplication
// and an addition a score, and LDS 54%, 22 of them for conflicts; they overlap in part only.  2 sequences,
// 8160 queries each over 28284 and 32640 slots, 16 heads on 4, dim 128: 2.0 to 2.1 ms, 0.83 to 0.88 PFLOP/s.
template <typename T, int DIM>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_weights_kernel(
    GsAttention a, GsPages p, const T *__restrict__ q, const T *__restrict__ k,
    const float *__restrict__ log_sum, float *__restrict__ weights) {
    constexpr int kRows = 64;
    using QTile = Tile<T, DIM, kRows, kWaves>;
    __shared__ __attribute__((aligned(1024))) char lds[2 * QTile::kBytes];
    __shared__ __attribute__((aligned(16))) float minus[2][kRows];
    const int group = a.heads_q / a.heads_k, lane = __lane_id(), half = lane >> 5;
    const int wave = uniform(threadIdx.x / kWave);
    const float c = exponent_factor(a.scale);
    const auto copy = QTile::copy_of(wave, a.q_row, a.dim);
    for_slot_tiles(a, p, kWeightSlots, a.heads_k, blockIdx.x, gridDim.x, [&](int sequence, int tile, int kh) {
        const int2 rows = rows_of(a.offsets_q, a.sequences, a.rows_q, sequence);
        const int q0 = uniform(rows.x), lq = uniform(rows.y - rows.x);
        const int filled = uniform(slots_of(p, sequence));
        const int slot0 = tile * kWeightSlots + 32 * wave, slot = slot0 + (lane & 31);
        // query i sees slots up to i + shift (a sum that may pass 32 bits: i and slot - shift do not)
        const int shift = a.causal ? filled - lq : filled;
        const int first = max(tile * kWeightSlots - shift, 0) / kRows;
        const int tiles = (lq + kRows - 1) / kRows - first, steps = tiles * group;
        int head = kh * group, at = first;  // of the tile that is fetched next
        float next = 0.0f;                  // its rows' -L, a lane each
        const auto fetch = [&](int buffer) {
            const int rows = lq - at * kRows;
            const int64_t row = q0 + at * kRows;
            QTile::start(copy, wave, q + row * a.q_row + head * a.q_head, a.q_row, rows, a.dim,
                         (lds_char *)lds + buffer * QTile::kBytes);
            if (wave == 0)
                next = lane < rows ? minus_log(log_sum[(row + lane) * a.heads_q + head]) : -INFINITY;
            if (++at == first + tiles) at = first, ++head;
        };
        float sum = 0.0f;
        int now = first;
        if (steps > 0) fetch(0);
        // (beside the first copy)
        const SlotOperand<T, DIM> mine(p, k, weights, sequence, slot, filled, kh, a.scale < 0.0f);
        if (steps > 0 && wave == 0) minus[0][lane] = next;
        for (int t = 0; t < steps; ++t) {
            copies_done();
            if (t + 1 < steps) fetch((t + 1) & 1);
            const lds_char *qt = (const lds_char *)lds + (t & 1) * QTile::kBytes;
            const auto minus_of = [&](int n, float *m) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 x = *(const f32x4 *)&minus[t & 1][32 * n + result_row(4 * g, half)];
#pragma unroll
                    for (int i = 0; i < 4; ++i) m[4 * g + i] = x[i];
                }
            };
            const int row0 = now * kRows;
            if (row0 >= slot0 + 31 - shift && row0 + kRows <= lq) {
                f32x16 s[2] = {};
#pragma unroll
                for (int i = 0; i < DIM / 16; ++i)
#pragma unroll
                    for (int n = 0; n < 2; ++n) s[n] = mfma(QTile::along(qt, 32 * n, i), mine.k.x[i], s[n]);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float m[16];
                    minus_of(n, m);
                    sum += sum_of_weights<false>(s[n], c, m, [](int) { return true; });
                }
            } else {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int row = row0 + 32 * n;
                    if (row >= lq || row + 31 < slot0 - shift) continue;
                    f32x16 s = {};
#pragma unroll
                    for (int i = 0; i < DIM / 16; ++i) s = mfma(QTile::along(qt, 32 * n, i), mine.k.x[i], s);
                    float m[16];
                    minus_of(n, m);
                    sum += sum_of_weights<true>(
                        s, c, m, [&](int i) { return row + i < lq && row + i >= slot - shift; });
                }
            }
            if (++now == first + tiles) now = first;
            if (wave == 0 && t + 1 < steps) minus[(t + 1) & 1][lane] = next;
        }
        mine.add(sum);
        __syncthreads();  // LDS has been read
    });
}

// Few rows: a wave takes them from memory.  (Where the attention could not keep their scores.)  64 single
// tokens over 12 to 2500 slots, 12 heads of 64: 24 us more than without weights, and 7 from kept scores.
template <typename T, int DIM>
__global__ __launch_bounds__(64 * kWaves) void paged_few_weights_kernel(
    GsAttention a, GsPages p, const T *__restrict__ q, const T *__restrict__ k,
    const float *__restrict__ log_sum, float *__restrict__ weights) {
    const int group = a.heads_q / a.heads_k, lane = __lane_id(), half = lane >> 5;
    const int wave = uniform(threadIdx.x / kWave);
    const float c = exponent_factor(a.scale);
    for_slot_tiles(a, p, kWeightSlots, a.heads_k, blockIdx.x, gridDim.x, [&](int sequence, int tile, int kh) {
        const int2 range = rows_of(a.offsets_q, a.sequences, a.rows_q, sequence);
        const int q0 = uniform(range.x), lq = uniform(range.y - range.x), rows = lq * group;
        const int filled = uniform(slots_of(p, sequence));
        const int slot0 = tile * kWeightSlots + 32 * wave, slot = slot0 + (lane & 31);
        if (slot0 >= filled) return;
        const SlotOperand<T, DIM> mine(p, k, weights, sequence, slot, filled, kh, a.scale < 0.0f);
        const int shift = a.causal ? filled - lq : filled;
        float sum = 0.0f;
        for (int row0 = max(slot0 - shift, 0) * group / 32 * 32; row0 < rows; row0 += 32) {
            const int row = row0 + (lane & 31);
            const bool real = row < rows;
            const int query = row / group, head = kh * group + row - query * group;
            RowOperand<T, DIM> x;
            x.load(real ? q + (int64_t)(q0 + query) * a.q_row + (int64_t)head * a.q_head : nullptr, a.dim,
                   false);
            const float l = real ? minus_log(log_sum[(int64_t)(q0 + query) * a.heads_q + head]) : -INFINITY;
            f32x16 s = {};
#pragma unroll
            for (int i = 0; i < DIM / 16; ++i) s = mfma(x.x[i], mine.k.x[i], s);
            float m[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) m[r] = __shfl(l, result_row(r, half), kWave);
            // the first row that sees the lane's slot
            const int least = max(slot - shift, 0) * group - row0;
            sum += sum_of_weights<true>(s, c, m, [&](int i) { return i >= least && row0 + i < rows; });
        }
        mine.add(sum);
    });
}

// Few rows whose scores the attention has kept: a thread a slot and head, `beside` heads a workgroup.
// Weights of neighbouring heads are neighbours in memory where heads are the last dimension, and a
// workgroup adds them slot by slot, since additions go to memory a line at a time.  Rows in parts are joined
// by the last `joins` workgroups of the same launch, a row each, and the slots' workgroups find a row's
// log-sum from its parts for themselves: a launch less.  Bound by latency: the sequence, the log-sums, the
// scores and the page.
template <typename T>
__global__ __launch_bounds__(kScoreSlots) void paged_score_weights_kernel(
    GsAttention a, GsPages p, const float *__restrict__ scores, int64_t score_slots, Partial partial,
    int joins, int beside, T *__restrict__ out, float *log_sum, float *__restrict__ weights) {
    __shared__ f32x4 sums[8][32];
    __shared__ float minus[kScoreSlots / kWave][kWave];  // -L of so many rows a head, in the exponent of two
    const int64_t all_rows = a.rows_q * a.heads_q;
    const int tiles = gridDim.x - joins;
    if ((int)blockIdx.x >= tiles) {
        join_row<T>(blockIdx.x - tiles, all_rows, a.dim, partial, out, (T *)nullptr, log_sum, sums);
        return;
    }
    float *const sum_of = (float *)sums;  // of each thread
    const int group = a.heads_q / a.heads_k, lane = __lane_id(), wave = uniform(threadIdx.x / kWave);
    // waves of the same head follow one another every `beside`
    const int slots = kScoreSlots / beside, wave_slots = wave / beside, wave_head = wave % beside;
    const float c = exponent_factor(a.scale);
    const auto minus_of = [&](int64_t row) {  // (every lane of a wave calls it)
        if (partial.splits == 1) return minus_log(log_sum[row]);
        const float2 part = lane < min(partial.count[row], partial.splits)
                                ? partial.max_sum[lane * all_rows + row]
                                : make_float2(-INFINITY, 0.0f);
        const float top = wave_max(part.x);
        const float share = part.x == -INFINITY ? 0.0f : part.y * __builtin_amdgcn_exp2f(part.x - top);
        const float l = top == -INFINITY ? -INFINITY : top + __builtin_amdgcn_logf(wave_sum(share));
        return l == -INFINITY ? -INFINITY : -l;
    };
    for_slot_tiles(a, p, slots, a.heads_k / beside, blockIdx.x, tiles, [&](int sequence, int tile, int part) {
        const int2 range = rows_of(a.offsets_q, a.sequences, a.rows_q, sequence);
        const int q0 = uniform(range.x), lq = uniform(range.y - range.x), rows = lq * group;
        const int filled = uniform(slots_of(p, sequence)), kh = part * beside + wave_head;
        const int slot = tile * slots + wave_slots * kWave + lane;
        // the first row that sees the slot
        const int least = slot >= filled ? rows : a.causal ? max(slot - (filled - lq), 0) * group : 0;
        const auto row_of = [&](int r) {
            const int i = r / group;
            return (int64_t)(q0 + i) * a.heads_q + kh * group + (r - i * group);
        };
        // the slot and head whose sum this thread adds to its weight
        const int to = (int)threadIdx.x / beside, to_head = (int)threadIdx.x % beside;
        const int to_slot = tile * slots + to, index = to_slot / p.page_size;
        const int page = to_slot < filled ? page_of(p, sequence - 1, index) : -1;
        float sum = 0.0f;
        for (int r0 = 0; r0 < rows; r0 += kWave) {
            const int end = min(r0 + kWave, rows);
            __syncthreads();  // the rows before have been read
            for (int r = r0 + wave_slots; r < end; r += kScoreSlots / kWave / beside) {
                const float m = minus_of(row_of(r));
                if (lane == 0) minus[wave_head][r - r0] = m;
            }
            __syncthreads();
            for (int r = max(r0, least); r < end; r += 4) {
                float s[4], w[4];
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    s[n] = r + n < end ? scores[row_of(r + n) * score_slots + slot] : 0.0f;
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    w[n] = r + n < end ? __builtin_amdgcn_exp2f(fmaf(s[n], c, minus[wave_head][r + n - r0]))
                                       : 0.0f;
                sum += (w[0] + w[1]) + (w[2] + w[3]);
            }
        }
        if (beside > 1) {
            sum_of[threadIdx.x] = sum;
            __syncthreads();
            sum = sum_of[(to / kWave * beside + to_head) * kWave + to % kWave];
            __syncthreads();  // before the next tile's
        }
        if (page >= 0)
            unsafeAtomicAdd(
                &weights[sum_at(p, page, to_slot - index * p.page_size, part * beside + to_head)], sum);
    });
}

static int check_queries(const GsPages *p, const GsPagedQueries *a, bool weights) {
    if (!a || a->rows_q < 0 || a->row_stride < 0 || a->head_stride < 0 || a->heads_q < 1 ||
        a->heads_q % p->heads != 0 || !a->offsets || !(a->scale == a->scale))
        return GS_ERR_INVALID_ARGUMENT;
    if ((a->row_stride | a->head_stride) % 8 != 0 || !tile_stride(a->row_stride, p->dim) ||
        a->rows_q > kMaxRows / (a->heads_q / p->heads))
        return GS_ERR_UNSUPPORTED;
    // the numbers of the slots' tiles stay in 32 bits (as they do where each lies in its own memory)
    const int64_t tiles = ((int64_t)p->page_size * p->table_width + kWeightSlots - 1) / kWeightSlots;
    if (weights && tiles > 0 && (int64_t)p->sequences * p->heads > kMaxRows / tiles)
        return GS_ERR_UNSUPPORTED;
    return GS_OK;
}

// The queries and sequences as the shared forward reads them.
static GsAttention problem_of(const GsPages &p, const GsPagedQueries &q) {
    GsAttention a = {};
    a.rows_q = q.rows_q;
    a.q_row = q.row_stride;
    a.q_head = q.head_stride;
    a.offsets_q = q.offsets;
    a.sequences = p.sequences;
    a.heads_q = q.heads_q;
    a.heads_k = p.heads;
    a.dim = p.dim;
    a.type = p.type;
    a.causal = q.causal;
    a.scale = q.scale;
    return a;
}

// As the packed kernels', but that a call's few tiles of rows take splits of equal length across
// sequences, as many as make kSplits items in all; a sequence longer than the others may have twice
// as many as the average.  5 sequences of up to 300 over 8044 to 16320 slots, 12 heads on 4, dim 72:
// 85 us in equal splits of each sequence, 77 in equal splits of all; 1200 rows over 20000, 16 heads
// on 4, dim 128: 393 in 1, 243.  Not over short tables (600 over 1000: 34 in 1, 44), and not where the
// tiles fill the GPU once (2500 over 10000: 260 in 1, 434): then there are more items than run at a time,
// and what the last ones and the join take is more than what the CUs without a second tile lose.
static ForwardPlan plan_of(const GsPages &p, const GsAttention &a) {
    const int64_t slots = (int64_t)p.page_size * p.table_width;
    ForwardPlan f = plan_forward(a, slots, slots);
    if (f.by_keys) return f;
    const int64_t packed = a.rows_q * (a.heads_q / a.heads_k), rows = 32 * kWaves;
    const int64_t busy = (packed + rows - 1) / rows * a.heads_k;
    f.splits = 1;
    f.groups = (packed / rows + a.sequences + 2) * a.heads_k;
    if (busy < 1 || busy > 256 || slots < 2048) return f;
    const int64_t want = 2 * ((kSplits + busy - 1) / busy), most = slots / 256;
    f.splits = (int)(want < most ? want : most);
    if (f.splits > 64) f.splits = 64;
    f.groups *= f.splits;
    if (f.groups > 1024) f.groups = 1024;
    return f;
}

// Floats a row and head where the scores of few rows are kept for the slots' weights, 0 where they
// are not: where they would take more than 256 MB (a table may be much wider than what is filled),
// the keys are read a second time.
static int64_t score_slots_of(const GsPages &p, const GsAttention &a, const ForwardPlan &f) {
    const int64_t slots = ((int64_t)p.page_size * p.table_width + 63) / 64 * 64;
    return f.by_keys && slots * a.rows_q * a.heads_q <= (64 << 20) ? slots : 0;
}

template <typename T, int DIM, bool WHOLE>
static int launch(const GsPages &p, const GsAttention &a, const ForwardPlan &f, const T *q, const T *k,
                  const T *v, T *out, float *log_sum, const Partial &partial, float *scores,
                  int64_t score_slots, hipStream_t stream) {
    const dim3 grid((unsigned)f.groups);
    if (f.by_keys && scores)
        hipLaunchKernelGGL((paged_attention_keys_kernel<T, DIM, WHOLE, true>), grid, dim3(64 * kKeysWaves),
                           0, stream, a, p, q, k, v, out, log_sum, partial, scores, score_slots);
    else if (f.by_keys)
        hipLaunchKernelGGL((paged_attention_keys_kernel<T, DIM, WHOLE, false>), grid, dim3(64 * kKeysWaves),
                           0, stream, a, p, q, k, v, out, log_sum, partial, scores, score_slots);
    else if (f.splits > 1)
        hipLaunchKernelGGL((paged_attention_split_kernel<T, DIM, WHOLE>), grid, dim3(64 * kWaves), 0,
                           stream, a, p, q, k, v, out, log_sum, partial);
    else if (log_sum)
        hipLaunchKernelGGL((paged_attention_kernel<T, DIM, true, WHOLE>), grid, dim3(64 * kWaves), 0,
                           stream, a, p, q, k, v, out, log_sum, partial);
    else
        hipLaunchKernelGGL((paged_attention_kernel<T, DIM, false, WHOLE>), grid, dim3(64 * kWaves), 0,
                           stream, a, p, q, k, v, out, log_sum, partial);
    const int st = launch_status();
    if (st || f.splits == 1 || scores) return st;  // (with scores the weights' launch joins)
    const int64_t rows = a.rows_q * a.heads_q;
    if (f.by_keys)
        hipLaunchKernelGGL((paged_join_kernel<T>), dim3((unsigned)rows), dim3(256), 0, stream, rows, a.dim,
                           partial, out, log_sum);
    else
        hipLaunchKernelGGL((paged_join_rows_kernel<T>),
                           dim3((unsigned)((rows + kJoinRows - 1) / kJoinRows)), dim3(32 * kJoinRows), 0,
                           stream, rows, a.dim, partial, out, log_sum);
    return launch_status();
}

}  // namespace gs

using namespace gs;

extern "C" int gs_paged_attention_workspace_size(const GsPages *p, const GsPagedQueries *q,
                                                 int32_t weights, size_t *bytes) {
    int st = check_pages(p, weights != 0);
    if (!st) st = check_queries(p, q, weights != 0);
    if (st) return st;
    if (!bytes) return GS_ERR_INVALID_ARGUMENT;
    const GsAttention a = problem_of(*p, *q);
    const ForwardPlan f = plan_of(*p, a);
    const size_t scores = weights ? score_slots_of(*p, a, f) * a.rows_q * a.heads_q * sizeof(float) : 0;
    *bytes = scores + partial_bytes(a, f.splits);
    return GS_OK;
}

extern "C" int gs_paged_attention(const GsPages *p, const GsPagedQueries *queries, const void *q,
                                  const void *k_pages, const void *v_pages, void *out,
                                  float *log_sum, float *weights, void *workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
    size_t need = 0;
    const int st = gs_paged_attention_workspace_size(p, queries, weights != nullptr, &need);
    if (st) return st;
    if (queries->rows_q == 0) return GS_OK;
    if (!q || !out || (p->pages > 0 && (!k_pages || !v_pages)) || (weights && !log_sum))
        return GS_ERR_INVALID_ARGUMENT;
    if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out))
        return GS_ERR_UNSUPPORTED;
    const GsAttention a = problem_of(*p, *queries);
    const ForwardPlan f = plan_of(*p, a);
    if (!launchable(f.groups, 64 * kWaves)) return GS_ERR_UNSUPPORTED;
    if (need && !workspace) return GS_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < need) return GS_ERR_WORKSPACE_TOO_SMALL;
    // the scores, whole lines, then the parts
    const int64_t score_slots = weights ? score_slots_of(*p, a, f) : 0;
    float *const scores = score_slots ? (float *)workspace : nullptr;
    const Partial partial =
        partial_of(a, f, true, (float *)workspace + score_slots * a.rows_q * a.heads_q);
    const auto all = [&](auto t, auto d) {
        using T = decltype(t);
        constexpr int kDim = decltype(d)::value;
        const T *tq = (const T *)q, *tk = (const T *)k_pages, *tv = (const T *)v_pages;
        const int s = p->page_size % 64 == 0
                          ? launch<T, kDim, true>(*p, a, f, tq, tk, tv, (T *)out, log_sum, partial,
                                                   scores, score_slots, stream)
                          : launch<T, kDim, false>(*p, a, f, tq, tk, tv, (T *)out, log_sum, partial,
                                                    scores, score_slots, stream);
        if (s || !weights || (!scores && (p->sequences == 0 || p->table_width == 0))) return s;
        // as many workgroups as there are tiles if no page is in two tables; the workgroups go on
        // while there are more
        const auto grid = [&](int64_t size, int parts) {
            const int64_t slots = (int64_t)p->page_size * p->table_width;
            const int64_t tables = (slots + size - 1) / size * p->sequences;
            const int64_t pool = p->pages * p->page_size / size + p->sequences;
            const int64_t groups = (tables < pool ? tables : pool) * parts;
            return dim3((unsigned)(groups < 8192 ? groups : 8192));
        };
        const float *log = log_sum;
        const int joins = scores && f.splits > 1 ? (int)(a.rows_q * a.heads_q) : 0;
        // heads beside each other take fewer lines, and each row's log-sum more often: where a sequence has
        // fewer rows on average than there are key heads.  Single tokens, a head by itself and beside others:
        // 64 over 12 to 2500 slots, 12 heads 52 and 41 us, 48 heads on 12 54 and 46; 16 over 2500 to 32640, 16
        // heads on 4, 118 and 122; 8 times 8 over 2500 to 8160 41 and 52
        const bool few = a.rows_q * (a.heads_q / a.heads_k) < (int64_t)a.sequences * a.heads_k;
        const int beside = !few ? 1 : p->heads % 4 == 0 ? 4 : p->heads % 2 == 0 ? 2 : 1;
        const unsigned both = joins + grid(kScoreSlots / beside, p->heads / beside).x;
        if (scores && both > 0)
            hipLaunchKernelGGL((paged_score_weights_kernel<T>), dim3(both), dim3(kScoreSlots), 0, stream, a,
                               *p, (const float *)scores, score_slots, partial, joins, beside, (T *)out,
                               log_sum, weights);
        else if (f.by_keys && !scores)
            hipLaunchKernelGGL((paged_few_weights_kernel<T, kDim>), grid(kWeightSlots, p->heads),
                               dim3(64 * kWaves), 0, stream, a, *p, tq, tk, log, weights);
        else if (!scores)
            hipLaunchKernelGGL((paged_weights_kernel<T, kDim>), grid(kWeightSlots, p->heads),
                               dim3(64 * kWaves), 0, stream, a, *p, tq, tk, log, weights);
        return launch_status();
    };
    return p->type == GS_F16 ? with_tile(p->dim, [&](auto d) { return all(f16{}, d); })
                             : with_tile(p->dim, [&](auto d) { return all(bf16{}, d); });
}
