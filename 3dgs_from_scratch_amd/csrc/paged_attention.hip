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
// one; else each row of a tile finds its own.  A tile's pages are read from the table while the
// tile before it is copied, and its rows that are there are told by bits.
template <typename T, bool WHOLE>
struct PagedKeys {
    static constexpr bool kHoles = true;
    GsPages p;
    const T *k, *v;
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
        // WHOLE: of the tile that is fetched next; else of the lane's row of it
        int index, place, page;
        int more_pages, more_places;  // of a tile's rows: whole pages, and places
        typename KTile::Copy copy;    // WHOLE: a tile's chunks

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
            if (WHOLE) copy = KTile::copy_of(wave, p.slot_stride, p.dim);
            look(first);
        }
        __device__ __forceinline__ void look(int t) {
            const bool is = WHOLE ? t < end : t * KTile::kRows + (int)__lane_id() < lk;
            page = is ? table[index] : -1;
        }
        // Starts the copies of a tile of keys and, behind it, of values.  Tiles come in order.
        __device__ __forceinline__ void fetch(int t, lds_char *to) {
            if constexpr (WHOLE) {
                const int32_t number = uniform(page);
                const bool is = (uint32_t)number < (uint64_t)p.pages;
                const int rows = is ? lk - t * KTile::kRows : 0;
                const int64_t from = is ? row_at(p, number, place) : 0;
                there = is ? ~0ull : 0;
                KTile::start(copy, wave, k + from, p.slot_stride, rows, p.dim, to);
                KTile::start(copy, wave, v + from, p.slot_stride, rows, p.dim, to + KTile::kBytes);
                place += KTile::kRows;
                if (place == p.page_size) place = 0, ++index;
            } else {
                const bool is = (uint32_t)page < (uint64_t)p.pages;
                there = __ballot(is);
                // bytes from the first element; below 0 where the row is not there
                const int64_t from = is ? row_at(p, page, place) * 2 : -1;
                const int low = (int)from, high = (int)(from >> 32);
#pragma unroll
                for (int i = 0; i < KTile::kCopies; ++i) {
                    const int piece = i * KTile::kCopyWaves + wave;
                    if (KTile::kPieces % KTile::kCopyWaves != 0 && piece >= KTile::kPieces) break;
                    const int at = piece * 64 + (int)__lane_id(), row = at / KTile::kChunks;
                    const int chunk = (at % KTile::kChunks) ^ KTile::swizzle(row);
                    const int64_t mine = (int64_t)(uint32_t)__builtin_amdgcn_ds_bpermute(row * 4, low) |
                                         (int64_t)__builtin_amdgcn_ds_bpermute(row * 4, high) << 32;
                    const bool has = mine >= 0 && chunk * 8 < p.dim;
                    const int64_t byte = mine + chunk * 16;
                    copy_chunk(has ? (const char *)k + byte : (const char *)kZeros, to + piece * 1024);
                    copy_chunk(has ? (const char *)v + byte : (const char *)kZeros,
                               to + KTile::kBytes + piece * 1024);
                }
                // the lane's row of the next tile
                place += more_places;
                index += more_pages;
                if (place >= p.page_size) place -= p.page_size, ++index;
            }
            look(t + 1);
        }
        // 16 bytes a lane, from the lane's address to the wave's piece of LDS.
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
    forward_tile<T, DIM, LOG_SUM>(a, PagedKeys<T, WHOLE>{p, k, v}, q, out, (T *)nullptr, log_sum, partial,
                                  (lds_char *)lds);
}

template <typename T, int DIM, bool WHOLE>
__global__ __launch_bounds__(64 * kKeysWaves, DIM > 96 ? 1 : 2) void paged_attention_keys_kernel(
    GsAttention a, GsPages p, const T *__restrict__ q, const T *__restrict__ k,
    const T *__restrict__ v, T *__restrict__ out, float *__restrict__ log_sum, Partial partial) {
    __shared__ __attribute__((aligned(1024))) char lds[Forward<T, DIM, true>::kLds];
    forward_by_keys<T, DIM>(a, PagedKeys<T, WHOLE>{p, k, v}, q, out, (T *)nullptr, log_sum, partial,
                            (lds_char *)lds);
}

template <typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(int64_t rows, int dim, Partial partial,
                                                         T *__restrict__ out,
                                                         float *__restrict__ log_sum) {
    __shared__ f32x4 sums[8][32];
    join_row<T>(rows, dim, partial, out, (T *)nullptr, log_sum, sums);
}

// A wave a slot and head; a lane takes every 64th of the rows that see it.
template <typename T>
__global__ __launch_bounds__(64) void paged_weights_kernel(GsPages p, GsPagedQueries a,
                                                           const T *__restrict__ q,
                                                           const T *__restrict__ k_pages,
                                                           const float *__restrict__ log_sum,
                                                           float *__restrict__ weights) {
    __shared__ float key[GS_MAX_HEAD_DIM];
    const int slot = blockIdx.x, b = blockIdx.y / p.heads, kh = blockIdx.y % p.heads;
    const int filled = filled_slots(p, b), lane = threadIdx.x, group = a.heads_q / p.heads;
    if (slot >= filled) return;
    const int page = page_of(p, b, slot / p.page_size), place = slot % p.page_size;
    if (page < 0) return;
    const int64_t from = row_at(p, page, place) + kh * p.head_stride;
    for (int d = lane; d < p.dim; d += 64) key[d] = to_float(k_pages[from + d]);
    __syncthreads();
    const int64_t first = a.offsets[b] < 0 ? 0 : a.offsets[b];
    const int64_t end = a.offsets[b + 1] < a.rows_q ? a.offsets[b + 1] : a.rows_q;
    // query i sees slots up to i + filled - Lq
    const int64_t least = a.causal ? slot - filled + (end - first) : 0;
    float sum = 0.0f;
    for (int64_t i = (least > 0 ? least : 0) * group + lane; i < (end - first) * group; i += 64) {
        const int64_t r = first + i / group;
        const int head = kh * group + (int)(i % group);
        const float l = log_sum[r * a.heads_q + head];
        float s = 0.0f;
        for (int d = 0; d < p.dim; ++d)
            s = fmaf(key[d], to_float(q[r * a.row_stride + head * a.head_stride + d]), s);
        if (l != -INFINITY) sum += expf(s * a.scale - l);
    }
    sum = wave_sum(sum);
    if (lane == 0) weights[sum_at(p, page, place, kh)] += sum;
}

static int check_queries(const GsPages *p, const GsPagedQueries *a) {
    if (!a || a->rows_q < 0 || a->row_stride < 0 || a->head_stride < 0 || a->heads_q < 1 ||
        a->heads_q % p->heads != 0 || !a->offsets || !(a->scale == a->scale))
        return GS_ERR_INVALID_ARGUMENT;
    if ((a->row_stride | a->head_stride) % 8 != 0 || !tile_stride(a->row_stride, p->dim) ||
        a->rows_q > kMaxRows / (a->heads_q / p->heads))
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

static ForwardPlan plan_of(const GsPages &p, const GsAttention &a) {
    const int64_t slots = (int64_t)p.page_size * p.table_width;
    return plan_forward(a, slots, slots);
}

template <typename T, int DIM, bool WHOLE>
static int launch(const GsPages &p, const GsAttention &a, const ForwardPlan &f, const T *q, const T *k,
                  const T *v, T *out, float *log_sum, const Partial &partial, hipStream_t stream) {
    const dim3 grid((unsigned)f.groups);
    if (f.by_keys)
        hipLaunchKernelGGL((paged_attention_keys_kernel<T, DIM, WHOLE>), grid, dim3(64 * kKeysWaves), 0,
                           stream, a, p, q, k, v, out, log_sum, partial);
    else if (log_sum || f.splits > 1)
        hipLaunchKernelGGL((paged_attention_kernel<T, DIM, true, WHOLE>), grid, dim3(64 * kWaves), 0,
                           stream, a, p, q, k, v, out, log_sum, partial);
    else
        hipLaunchKernelGGL((paged_attention_kernel<T, DIM, false, WHOLE>), grid, dim3(64 * kWaves), 0,
                           stream, a, p, q, k, v, out, log_sum, partial);
    const int st = launch_status();
    if (st || f.splits == 1) return st;
    const int64_t rows = a.rows_q * a.heads_q;
    hipLaunchKernelGGL((paged_join_kernel<T>), dim3((unsigned)rows), dim3(256), 0, stream, rows, a.dim,
                       partial, out, log_sum);
    return launch_status();
}

}  // namespace gs

using namespace gs;

extern "C" int gs_paged_attention_workspace_size(const GsPages *p, const GsPagedQueries *q,
                                                 int32_t weights, size_t *bytes) {
    int st = check_pages(p, weights != 0);
    if (!st) st = check_queries(p, q);
    if (st) return st;
    if (!bytes) return GS_ERR_INVALID_ARGUMENT;
    const GsAttention a = problem_of(*p, *q);
    *bytes = partial_bytes(a, plan_of(*p, a).splits);
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
    if (f.groups > 0x7fffffffLL) return GS_ERR_UNSUPPORTED;
    if (need && !workspace) return GS_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < need) return GS_ERR_WORKSPACE_TOO_SMALL;
    const Partial partial = partial_of(a, f, workspace);
    const auto all = [&](auto t, auto d) {
        using T = decltype(t);
        constexpr int kDim = decltype(d)::value;
        const T *tq = (const T *)q, *tk = (const T *)k_pages, *tv = (const T *)v_pages;
        const int s = p->page_size % 64 == 0
                          ? launch<T, kDim, true>(*p, a, f, tq, tk, tv, (T *)out, log_sum, partial, stream)
                          : launch<T, kDim, false>(*p, a, f, tq, tk, tv, (T *)out, log_sum, partial, stream);
        if (s) return s;
        const int64_t slots = (int64_t)p->page_size * p->table_width;
        if (weights && slots > 0 && p->sequences > 0)
            hipLaunchKernelGGL((paged_weights_kernel<T>),
                               dim3((unsigned)slots, (unsigned)(p->sequences * p->heads)), dim3(64),
                               0, stream, *p, *queries, tq, tk, (const float *)log_sum, weights);
        return launch_status();
    };
    return p->type == GS_F16 ? with_tile(p->dim, [&](auto d) { return all(f16{}, d); })
                             : with_tile(p->dim, [&](auto d) { return all(bf16{}, d); });
}
