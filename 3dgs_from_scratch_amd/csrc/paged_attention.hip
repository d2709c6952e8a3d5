// Attention of new tokens over a paged cache, and the attention that its keys get:
//   S = scale q k^T over the slots a query sees,  L = log sum exp S,  out = exp(S - L) v
//   weight of a slot and head += sum over queries and heads of the group of exp(S - L)
// Scores, softmax statistics and sums are in float.

#include <cmath>

#include "paged.h"

namespace gs {

// A wave a row and head; a lane scores a key at a time, and has two columns of the output.
template <typename T>
__global__ __launch_bounds__(64) void paged_rows_kernel(GsPages p, GsPagedQueries a,
                                                        const T *__restrict__ q,
                                                        const T *__restrict__ k_pages,
                                                        const T *__restrict__ v_pages,
                                                        T *__restrict__ out,
                                                        float *__restrict__ log_sum) {
    __shared__ float row[GS_MAX_HEAD_DIM];
    const int64_t at = blockIdx.x, r = at / a.heads_q;
    const int head = (int)(at - r * a.heads_q), kh = head / (a.heads_q / p.heads);
    const int lane = threadIdx.x;
    int b = 0, first = 0, last = 0;
    for (; b < p.sequences; ++b) {
        first = a.offsets[b];
        last = a.offsets[b + 1];
        if (r >= first && r < last) break;
    }
    const int filled = b < p.sequences ? filled_slots(p, b) : 0;
    if (last > a.rows_q) last = (int)a.rows_q;
    const int64_t seen64 = a.causal ? r - last + filled + 1 : filled;
    const int seen = (int)(seen64 < filled ? seen64 : filled);
    for (int d = lane; d < p.dim; d += 64) row[d] = to_float(q[r * a.row_stride + head * a.head_stride + d]);
    __syncthreads();
    float top = -INFINITY, sum = 0.0f, x0 = 0.0f, x1 = 0.0f;
    bool any = false;
    for (int j0 = 0; j0 < seen; j0 += 64) {
        const int j = j0 + lane, index = j / p.page_size;
        const int page = j < seen ? page_of(p, b, index) : -1;
        const int64_t from = page < 0 ? 0 : row_at(p, page, j - index * p.page_size) + kh * p.head_stride;
        float s = -INFINITY;
        if (page >= 0) {
            s = 0.0f;
            for (int d = 0; d < p.dim; ++d) s = fmaf(row[d], to_float(k_pages[from + d]), s);
            s *= a.scale;
        }
        any = any || __ballot(page >= 0) != 0;
        const float now = fmaxf(top, wave_max(s));
        const float keep = now == -INFINITY ? 1.0f : expf(top - now);
        const float w = page < 0 ? 0.0f : expf(s - (now == -INFINITY ? 0.0f : now));
        sum = sum * keep + wave_sum(w);
        x0 *= keep;
        x1 *= keep;
        top = now;
        for (int i = 0; i < 64; ++i) {
            if (__shfl(page, i, 64) < 0) continue;
            const float wi = __shfl(w, i, 64);
            const int64_t line = __shfl(from, i, 64);
            if (lane < p.dim) x0 = fmaf(wi, to_float(v_pages[line + lane]), x0);
            if (lane + 64 < p.dim) x1 = fmaf(wi, to_float(v_pages[line + lane + 64]), x1);
        }
    }
    T *to = out + at * p.dim;
    if (lane < p.dim) to[lane] = from_float<T>(any ? x0 / sum : 0.0f);
    if (lane + 64 < p.dim) to[lane + 64] = from_float<T>(any ? x1 / sum : 0.0f);
    if (log_sum && lane == 0) log_sum[at] = any ? top + logf(sum) : -INFINITY;
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
    if ((a->row_stride | a->head_stride) % 8 != 0 || a->row_stride < p->dim ||
        a->row_stride > (1 << 23) || a->rows_q > kMaxSlots / (a->heads_q / p->heads))
        return GS_ERR_UNSUPPORTED;
    return GS_OK;
}

}  // namespace gs

using namespace gs;

extern "C" int gs_paged_attention_workspace_size(const GsPages *p, const GsPagedQueries *a,
                                                 int32_t weights, size_t *bytes) {
    int st = check_pages(p, weights != 0);
    if (!st) st = check_queries(p, a);
    if (st) return st;
    if (!bytes) return GS_ERR_INVALID_ARGUMENT;
    *bytes = 0;
    return GS_OK;
}

extern "C" int gs_paged_attention(const GsPages *p, const GsPagedQueries *a, const void *q,
                                  const void *k_pages, const void *v_pages, void *out,
                                  float *log_sum, float *weights, void *workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
    size_t need = 0;
    const int st = gs_paged_attention_workspace_size(p, a, weights != nullptr, &need);
    if (st) return st;
    if (need && !workspace) return GS_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < need) return GS_ERR_WORKSPACE_TOO_SMALL;
    if (a->rows_q == 0) return GS_OK;
    if (!q || !out || (p->pages > 0 && (!k_pages || !v_pages)) || (weights && !log_sum))
        return GS_ERR_INVALID_ARGUMENT;
    if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out))
        return GS_ERR_UNSUPPORTED;
    const auto launch = [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((paged_rows_kernel<T>), dim3((unsigned)(a->rows_q * a->heads_q)), dim3(64),
                           0, stream, *p, *a, (const T *)q, (const T *)k_pages, (const T *)v_pages,
                           (T *)out, log_sum);
        const int64_t slots = (int64_t)p->page_size * p->table_width;
        if (weights && slots > 0 && p->sequences > 0)
            hipLaunchKernelGGL((paged_weights_kernel<T>),
                               dim3((unsigned)slots, (unsigned)(p->sequences * p->heads)), dim3(64),
                               0, stream, *p, *a, (const T *)q, (const T *)k_pages,
                               (const float *)log_sum, weights);
        return launch_status();
    };
    return p->type == GS_F16 ? launch(f16{}) : launch(bf16{});
}
