// Attention over packed sequences with grouped heads, and its gradients:
//   S = scale q k^T over the keys a query sees,  P = exp(S - L),  L = log sum exp S
//   out = P v,  delta = sum_d dout out,  dS = P (dout v^T - delta)
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout
// with dk and dv summed over the query heads of a group.  Scores, softmax
// statistics and sums are in float.

#include "element.h"

namespace gs {

// A sequence's queries and keys.  Two more sequences without keys hold the rows
// before the first offset and after the last, so that every row has one.
struct Span {
    int64_t q0, q1;  // query rows
    int64_t k0, k1;  // key rows
};

__device__ __forceinline__ int64_t clamp_row(int64_t v, int64_t low, int64_t high) {
    return v < low ? low : v > high ? high : v;
}

__device__ __forceinline__ Span span_of(const GsAttention &a, int s) {
    Span p;
    p.q0 = s == 0 ? 0 : clamp_row(a.offsets_q[s - 1], 0, a.rows_q);
    p.q1 = s > a.sequences ? a.rows_q : clamp_row(a.offsets_q[s], p.q0, a.rows_q);
    p.k0 = s == 0 ? 0 : clamp_row(a.offsets_k[s - 1], 0, a.rows_k);
    p.k1 = s > a.sequences ? a.rows_k : clamp_row(a.offsets_k[s], p.k0, a.rows_k);
    return p;
}

// The keys that count: none outside the sequences, else up to the given length.
__device__ __forceinline__ int64_t keys_of(const GsAttention &a, int s, const Span &p) {
    if (s == 0 || s > a.sequences) return 0;
    const int64_t n = p.k1 - p.k0;
    return a.lengths_k ? clamp_row(a.lengths_k[s - 1], 0, n) : n;
}

// The sequence (1 based, 0 and sequences + 1 for the rows of none) of a row.
__device__ __forceinline__ int sequence_of(const int32_t *offsets, int sequences, int64_t row) {
    int s = 0;
    while (s <= sequences && row >= offsets[s]) ++s;
    return s;
}

template <typename T>
__global__ __launch_bounds__(64) void attention_kernel(GsAttention a, const T *__restrict__ q,
                                                       const T *__restrict__ k,
                                                       const T *__restrict__ v,
                                                       T *__restrict__ out,
                                                       float *__restrict__ log_sum) {
    const int64_t row = blockIdx.x;
    const int head = blockIdx.y, kh = head / (a.heads_q / a.heads_k), lane = threadIdx.x;
    const int s = sequence_of(a.offsets_q, a.sequences, row);
    const Span p = span_of(a, s);
    const int64_t keys = keys_of(a, s, p);
    const int64_t i = row - p.q0, lq = p.q1 - p.q0;
    const int64_t seen = a.causal ? clamp_row(i + keys - lq + 1, 0, keys) : keys;
    const bool one = lane < a.dim, two = lane + 64 < a.dim;
    const T *qr = q + row * a.q_row + head * a.q_head;
    const float q0 = one ? to_float(qr[lane]) * a.scale : 0.0f;
    const float q1 = two ? to_float(qr[lane + 64]) * a.scale : 0.0f;
    float top = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int64_t j = 0; j < seen; ++j) {
        const T *kr = k + (p.k0 + j) * a.k_row + kh * a.k_head;
        const T *vr = v + (p.k0 + j) * a.v_row + kh * a.v_head;
        const float x =
            wave_sum(fmaf(one ? to_float(kr[lane]) : 0.0f, q0,
                          (two ? to_float(kr[lane + 64]) : 0.0f) * q1));
        const float now = fmaxf(top, x);
        const float keep = now == -INFINITY ? 1.0f : expf(top - now);
        const float w = now == -INFINITY ? 0.0f : expf(x - now);
        top = now;
        sum = fmaf(sum, keep, w);
        o0 = fmaf(o0, keep, w * (one ? to_float(vr[lane]) : 0.0f));
        o1 = fmaf(o1, keep, w * (two ? to_float(vr[lane + 64]) : 0.0f));
    }
    const float r = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : NAN;
    T *dst = out + (row * a.heads_q + head) * a.dim;
    if (one) dst[lane] = from_float<T>(o0 * r);
    if (two) dst[lane + 64] = from_float<T>(o1 * r);
    if (log_sum && lane == 0) log_sum[row * a.heads_q + head] = top + logf(sum);
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
    const int64_t keys = keys_of(a, s, p);
    const int64_t i = row - p.q0, lq = p.q1 - p.q0;
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
    const int64_t keys = keys_of(a, s, p);
    const int64_t j = row - p.k0, lq = p.q1 - p.q0;
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

constexpr int64_t kMaxRows = 0x7fffffffLL - 65536;  // row numbers stay in 32 bits in a tile

static int check_attention(const GsAttention *a) {
    if (!a || a->rows_q < 0 || a->rows_k < 0 || a->sequences < 0 || a->heads_q < 1 ||
        a->heads_k < 1 || a->heads_q % a->heads_k != 0 || a->dim < 1 || a->q_row < 0 ||
        a->q_head < 0 || a->k_row < 0 || a->k_head < 0 || a->v_row < 0 || a->v_head < 0 ||
        !(a->scale == a->scale))
        return GS_ERR_INVALID_ARGUMENT;
    if (!a->offsets_q || !a->offsets_k) return GS_ERR_INVALID_ARGUMENT;
    if (!element_type(a->type)) return GS_ERR_INVALID_ARGUMENT;
    if (a->type == GS_F32 || a->dim % 8 != 0 || a->dim > GS_MAX_HEAD_DIM ||
        a->heads_q > 65535 || a->rows_q > kMaxRows || a->rows_k > kMaxRows ||
        (a->q_row | a->q_head | a->k_row | a->k_head | a->v_row | a->v_head) % 8 != 0)
        return GS_ERR_UNSUPPORTED;
    return GS_OK;
}

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace gs

using namespace gs;

extern "C" int gs_attention_forward_workspace_size(const GsAttention *a, size_t *bytes) {
    const int st = check_attention(a);
    if (st) return st;
    if (!bytes) return GS_ERR_INVALID_ARGUMENT;
    *bytes = 0;
    return GS_OK;
}

extern "C" int gs_attention_forward(const GsAttention *a, const void *q, const void *k,
                                    const void *v, void *out, float *log_sum, void *workspace,
                                    size_t workspace_bytes, hipStream_t stream) {
    const int st = check_attention(a);
    if (st) return st;
    if (a->rows_q == 0) return GS_OK;
    if (!q || !out || (a->rows_k > 0 && (!k || !v))) return GS_ERR_INVALID_ARGUMENT;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v)) return GS_ERR_UNSUPPORTED;
    (void)workspace;
    (void)workspace_bytes;
    const auto launch = [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((attention_kernel<T>), dim3((unsigned)a->rows_q, a->heads_q), dim3(64),
                           0, stream, *a, (const T *)q, (const T *)k, (const T *)v, (T *)out,
                           log_sum);
        return launch_status();
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
