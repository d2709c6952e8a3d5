// Layer norm over the channels of a row and its gradients:
//   h = (x - mean) r,  r = 1 / sqrt(mean((x - mean)^2) + eps),  y = h w + b
//   dx = r (g - mean(g) - h mean(g h)) with g = dy w,  dw = sum dy h,  db = sum dy
// the means over a row's channels, the sums over the rows.  All arithmetic is in
// float; an output is rounded once.
//
// Bound by memory: forward reads x and writes y, backward reads x and dy and writes dx,
// each once.  A row is held in the registers of 16 lanes, a wave or a workgroup, so the
// variance is taken of differences to the mean without a second read; the backward
// keeps the weight's sums of its rows in registers too, joins its waves in LDS, and a
// second launch adds up the workgroups' sums in an order that the sizes alone give.

#include <type_traits>

#include "element.h"

namespace gs {

constexpr int kNormBlock = 256;
constexpr int kNormGroups = 1024;  // most workgroups of a backward

// How a row lies in registers: LANES lanes, SLOTS packs of VEC elements in each; pack i of
// lane l is number i * LANES + l of the row.  WHOLE: the row ends with a pack.
template <int LANES_, int SLOTS_, int VEC_, bool WHOLE_>
struct Shape {
    static constexpr int kLanes = LANES_, kSlots = SLOTS_, kVec = VEC_;
    static constexpr bool kWhole = WHOLE_;
    static constexpr int kRows = kNormBlock / kLanes;  // of a workgroup at a time
    static constexpr int kHeld = kSlots * kVec;
};

// The sums of two values over a row's lanes, in all of them.
template <int LANES>
__device__ __forceinline__ float2 row_sum(float a, float b) {
    if constexpr (LANES <= kWave) {
        return make_float2(lane_sum<LANES>(a), lane_sum<LANES>(b));
    } else {
        __shared__ float2 part[LANES / kWave];
        a = lane_sum<kWave>(a);
        b = lane_sum<kWave>(b);
        __syncthreads();  // an earlier call's values have been read
        if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = make_float2(a, b);
        __syncthreads();
        float2 s = part[0];
#pragma unroll
        for (int w = 1; w < LANES / kWave; ++w) {
            s.x += part[w].x;
            s.y += part[w].y;
        }
        return s;
    }
}

// A weight or bias vector of any of the types, or nothing.
struct Weights {
    const void *p;
    int32_t type;
};

template <bool WHOLE, int VEC>
__device__ __forceinline__ void load_weights(const Weights &w, int at, int n, float none, float *v) {
    if (!w.p) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = none;
    } else if (w.type == GS_F32) {
        load_first<WHOLE, float, VEC>((const float *)w.p + at, v, n, none);
    } else if (w.type == GS_F16) {
        load_first<WHOLE, f16, VEC>((const f16 *)w.p + at, v, n, none);
    } else {
        load_first<WHOLE, bf16, VEC>((const bf16 *)w.p + at, v, n, none);
    }
}

// The lane's packs of a row; zeros past its end.
template <typename S, typename T>
__device__ __forceinline__ void load_row(const T *row, int lane, int channels, float *v) {
#pragma unroll
    for (int i = 0; i < S::kSlots; ++i) {
        const int at = (i * S::kLanes + lane) * S::kVec;
        load_first<S::kWhole, T, S::kVec>(row + at, v + i * S::kVec, channels - at, 0.0f);
    }
}

// 65280 rows of 1024 channels in bfloat16 in 49 us, 5.4 TB/s; 8163 of 771 in float16 in 13.
// The variance is of differences to the mean, so that channels far from zero lose nothing.
template <typename T, typename S>
__global__ __launch_bounds__(kNormBlock) void layer_norm_kernel(
    const T *__restrict__ x, int64_t x_stride, Weights weight, Weights bias, int64_t rows,
    int channels, float eps, T *__restrict__ y, float2 *__restrict__ stats) {
    const int lane = threadIdx.x % S::kLanes;
    const int64_t first = (int64_t)blockIdx.x * S::kRows + threadIdx.x / S::kLanes;
    const float n = (float)channels;
    // (rows a workgroup long: all its threads leave the loop together)
    for (int64_t row = first; row < rows; row += (int64_t)gridDim.x * S::kRows) {
        float v[S::kHeld];
        load_row<S>(x + row * x_stride, lane, channels, v);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < S::kHeld; ++i) s += v[i];
        const float mean = row_sum<S::kLanes>(s, 0.0f).x / n;
        float q = 0.0f;
#pragma unroll
        for (int i = 0; i < S::kSlots; ++i) {
            const int at = (i * S::kLanes + lane) * S::kVec;
            if (at >= channels) continue;
#pragma unroll
            for (int j = 0; j < S::kVec; ++j) {
                float &d = v[i * S::kVec + j];
                d = S::kWhole || at + j < channels ? d - mean : 0.0f;
                q = fmaf(d, d, q);
            }
        }
        const float r = 1.0f / sqrtf(row_sum<S::kLanes>(q, 0.0f).x / n + eps);
#pragma unroll
        for (int i = 0; i < S::kSlots; ++i) {
            const int at = (i * S::kLanes + lane) * S::kVec;
            if (at >= channels) continue;
            float w[S::kVec], b[S::kVec];
            const int held = S::kWhole ? S::kVec : channels - at;
            load_weights<S::kWhole, S::kVec>(weight, at, held, 1.0f, w);
            load_weights<S::kWhole, S::kVec>(bias, at, held, 0.0f, b);
#pragma unroll
            for (int j = 0; j < S::kVec; ++j) w[j] = fmaf(v[i * S::kVec + j] * r, w[j], b[j]);
            store_first<S::kWhole, T, S::kVec>(y + row * channels + at, w, held);
        }
        if (stats && lane == 0) stats[row] = make_float2(mean, r);
    }
}

// partial[workgroup][0..1][channel]: the workgroup's sums of dy h and of dy.  At most 1024
// workgroups, four a CU: each leaves 2 floats a channel for the join to read.  65280 rows of
// 1024 channels in bfloat16 in 80 us, 5.0 TB/s; 8163 of 771 in float16 in 21.
template <typename T, typename S, bool SUMS>
__global__ __launch_bounds__(kNormBlock) void layer_norm_backward_kernel(
    const T *__restrict__ dy, int64_t dy_stride, const T *__restrict__ x, int64_t x_stride,
    Weights weight, const float2 *__restrict__ stats, int64_t rows, int channels,
    T *__restrict__ dx, float *__restrict__ partial) {
    const int lane = threadIdx.x % S::kLanes, group = threadIdx.x / S::kLanes;
    const float n = (float)channels;
    float w[S::kHeld], sum_w[SUMS ? S::kHeld : 1], sum_b[SUMS ? S::kHeld : 1];
#pragma unroll
    for (int i = 0; i < S::kSlots; ++i) {
        const int at = (i * S::kLanes + lane) * S::kVec;
        load_weights<S::kWhole, S::kVec>(weight, at, channels - at, 1.0f, w + i * S::kVec);
    }
    if constexpr (SUMS)
#pragma unroll
        for (int i = 0; i < S::kHeld; ++i) sum_w[i] = sum_b[i] = 0.0f;
    for (int64_t row = (int64_t)blockIdx.x * S::kRows + group; row < rows;
         row += (int64_t)gridDim.x * S::kRows) {
        float g[S::kHeld], h[S::kHeld];
        load_row<S>(dy + row * dy_stride, lane, channels, g);
        load_row<S>(x + row * x_stride, lane, channels, h);
        const float2 st = stats[row];
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int i = 0; i < S::kHeld; ++i) {
            h[i] = (h[i] - st.x) * st.y;
            if constexpr (SUMS) {
                sum_w[i] = fmaf(g[i], h[i], sum_w[i]);
                sum_b[i] += g[i];
            }
            g[i] *= w[i];
            a += g[i];  // (both are 0 past the row's end: g is)
            b = fmaf(g[i], h[i], b);
        }
        if (!dx) continue;
        const float2 m = row_sum<S::kLanes>(a, b);
        const float ma = m.x / n, mb = m.y / n;
#pragma unroll
        for (int i = 0; i < S::kSlots; ++i) {
            const int at = (i * S::kLanes + lane) * S::kVec;
            if (at >= channels) continue;
#pragma unroll
            for (int j = 0; j < S::kVec; ++j) {
                const int e = i * S::kVec + j;
                g[e] = st.y * (g[e] - ma - h[e] * mb);
            }
            store_first<S::kWhole, T, S::kVec>(dx + row * channels + at, g + i * S::kVec,
                                               channels - at);
        }
    }
    if constexpr (SUMS) {
        // the workgroup's rows of lanes, one pack after another
        __shared__ float joined[S::kRows > 1 ? 2 * kNormBlock * S::kVec : 1];
        float *to = partial + (int64_t)blockIdx.x * 2 * channels;
#pragma unroll
        for (int i = 0; i < S::kSlots; ++i) {
            const int at = (i * S::kLanes + lane) * S::kVec;
            if constexpr (S::kRows > 1) {
                __syncthreads();  // the pack before has been read
#pragma unroll
                for (int j = 0; j < S::kVec; ++j) {
                    joined[(2 * j) * kNormBlock + threadIdx.x] = sum_w[i * S::kVec + j];
                    joined[(2 * j + 1) * kNormBlock + threadIdx.x] = sum_b[i * S::kVec + j];
                }
                __syncthreads();
                if (group == 0 && at < channels) {
#pragma unroll
                    for (int j = 0; j < S::kVec; ++j) {
                        float a = 0.0f, b = 0.0f;
                        for (int r = 0; r < S::kRows; ++r) {
                            a += joined[(2 * j) * kNormBlock + r * S::kLanes + lane];
                            b += joined[(2 * j + 1) * kNormBlock + r * S::kLanes + lane];
                        }
                        if (S::kWhole || at + j < channels) {
                            to[at + j] = a;
                            to[channels + at + j] = b;
                        }
                    }
                }
            } else if (at < channels) {
#pragma unroll
                for (int j = 0; j < S::kVec; ++j)
                    if (S::kWhole || at + j < channels) {
                        to[at + j] = sum_w[i * S::kVec + j];
                        to[channels + at + j] = sum_b[i * S::kVec + j];
                    }
            }
        }
    }
}

// Rows too long for registers (more than 8192 channels of 16 bits): the row is read once for
// each of the mean, the variance and the output.
template <typename T>
__global__ __launch_bounds__(kNormBlock) void layer_norm_long_kernel(
    const T *__restrict__ x, int64_t x_stride, Weights weight, Weights bias, int64_t rows,
    int channels, float eps, T *__restrict__ y, float2 *__restrict__ stats) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * x_stride;
        float s = 0.0f;
        for (int c = threadIdx.x; c < channels; c += kNormBlock) s += to_float(xr[c]);
        const float mean = row_sum<kNormBlock>(s, 0.0f).x / (float)channels;
        float q = 0.0f;
        for (int c = threadIdx.x; c < channels; c += kNormBlock) {
            const float d = to_float(xr[c]) - mean;
            q = fmaf(d, d, q);
        }
        const float r = 1.0f / sqrtf(row_sum<kNormBlock>(q, 0.0f).x / (float)channels + eps);
        for (int c = threadIdx.x; c < channels; c += kNormBlock) {
            float w, b;
            load_weights<true, 1>(weight, c, 1, 1.0f, &w);
            load_weights<true, 1>(bias, c, 1, 0.0f, &b);
            y[row * channels + c] = from_float<T>(fmaf((to_float(xr[c]) - mean) * r, w, b));
        }
        if (stats && threadIdx.x == 0) stats[row] = make_float2(mean, r);
    }
}

template <typename T>
__global__ __launch_bounds__(kNormBlock) void layer_norm_long_dx_kernel(
    const T *__restrict__ dy, int64_t dy_stride, const T *__restrict__ x, int64_t x_stride,
    Weights weight, const float2 *__restrict__ stats, int64_t rows, int channels,
    T *__restrict__ dx) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * x_stride, *gr = dy + row * dy_stride;
        const float2 st = stats[row];
        float a = 0.0f, b = 0.0f, w;
        for (int c = threadIdx.x; c < channels; c += kNormBlock) {
            load_weights<true, 1>(weight, c, 1, 1.0f, &w);
            const float g = to_float(gr[c]) * w;
            a += g;
            b = fmaf(g, (to_float(xr[c]) - st.x) * st.y, b);
        }
        const float2 m = row_sum<kNormBlock>(a, b);
        const float ma = m.x / (float)channels, mb = m.y / (float)channels;
        for (int c = threadIdx.x; c < channels; c += kNormBlock) {
            load_weights<true, 1>(weight, c, 1, 1.0f, &w);
            const float g = to_float(gr[c]) * w;
            const float h = (to_float(xr[c]) - st.x) * st.y;
            dx[row * channels + c] = from_float<T>(st.y * (g - ma - h * mb));
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kNormBlock) void layer_norm_long_sums_kernel(
    const T *__restrict__ dy, int64_t dy_stride, const T *__restrict__ x, int64_t x_stride,
    const float2 *__restrict__ stats, int64_t rows, int channels, float *__restrict__ partial) {
    const int c = blockIdx.x * kNormBlock + threadIdx.x;
    if (c >= channels) return;
    float w = 0.0f, b = 0.0f;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float2 st = stats[row];
        const float g = to_float(dy[row * dy_stride + c]);
        w = fmaf(g, (to_float(x[row * x_stride + c]) - st.x) * st.y, w);
        b += g;
    }
    float *p = partial + (int64_t)blockIdx.y * 2 * channels + c;
    p[0] = w;
    p[channels] = b;
}

// The sums of the workgroups' sums: 16 columns of the 2 * channels a workgroup, in 64 groups
// of workgroups each.  Bound by latency, so the more groups the better: 1024 workgroups' of
// 1024 channels 4.6 us, in 16 groups 20.5.
constexpr int kJoinColumns = 16, kJoinRows = 64;

__global__ __launch_bounds__(kJoinColumns *kJoinRows) void layer_norm_join_kernel(
    const float *__restrict__ partial, int groups, int channels, int32_t type,
    void *__restrict__ dw, void *__restrict__ db) {
    __shared__ float part[kJoinRows][kJoinColumns + 1];
    const int across = threadIdx.x % kJoinColumns, down = threadIdx.x / kJoinColumns;
    const int c = blockIdx.x * kJoinColumns + across;
    float s = 0.0f;
    if (c < 2 * channels)
#pragma unroll 8
        for (int g = down; g < groups; g += kJoinRows) s += partial[(int64_t)g * 2 * channels + c];
    part[down][across] = s;
    __syncthreads();
    // a row of 16 lanes a column: 4 of its sums each, then across the lanes
    const int column = threadIdx.x / 16, lane = threadIdx.x % 16;
    if (column >= kJoinColumns) return;
    s = 0.0f;
#pragma unroll
    for (int g = 0; g < kJoinRows / 16; ++g) s += part[g * 16 + lane][column];
    s = lane_sum<16>(s);
    const int at = blockIdx.x * kJoinColumns + column;
    if (lane || at >= 2 * channels) return;
    void *out = at < channels ? dw : db;
    const int to = at < channels ? at : at - channels;
    if (!out) return;
    if (type == GS_F32)
        ((float *)out)[to] = s;
    else if (type == GS_F16)
        ((f16 *)out)[to] = from_float<f16>(s);
    else
        ((bf16 *)out)[to] = from_float<bf16>(s);
}

// Rows of lanes and packs of 16 bytes for a number of channels: a row of 16 lanes up to 2
// packs a lane, else a wave up to 3, else a workgroup; f gets the shape, or 0 if the row does
// not fit in registers.  Both sides, forward and backward of 65280 rows in bfloat16: 256
// channels on 16 lanes 75 us, on a wave 137; 512 on a wave 73, on 16 lanes of 4 packs 144;
// 1024 on a wave 138, on a workgroup 227; 1536 on a wave 267 (forward 83), on a workgroup 265
// (98); 2048 on a wave of 4 packs 350, on a workgroup 297.
template <typename T, bool WHOLE, typename F>
static int with_shape(int channels, F f) {
    constexpr int kVec = 16 / sizeof(T);
    const int packs = (channels + kVec - 1) / kVec;
    if (packs <= 16) return f(Shape<16, 1, kVec, WHOLE>{});
    if (packs <= 32) return f(Shape<16, 2, kVec, WHOLE>{});
    if (packs <= 64) return f(Shape<64, 1, kVec, WHOLE>{});
    if (packs <= 128) return f(Shape<64, 2, kVec, WHOLE>{});
    if (packs <= 192) return f(Shape<64, 3, kVec, WHOLE>{});
    if (packs <= 256) return f(Shape<256, 1, kVec, WHOLE>{});
    if (packs <= 512) return f(Shape<256, 2, kVec, WHOLE>{});
    if (packs <= 1024) return f(Shape<256, 4, kVec, WHOLE>{});
    return f(0);
}

template <typename T, typename F>
static int with_shape(int channels, F f) {
    return channels % (16 / (int)sizeof(T)) == 0 ? with_shape<T, true>(channels, f)
                                                 : with_shape<T, false>(channels, f);
}

// Workgroups of a backward: one for every 16 rows (four a wave, or one a row of 16 lanes), at
// most kNormGroups.
static int norm_groups(int64_t rows) {
    const int64_t g = (rows + 15) / 16;
    return (int)(g < kNormGroups ? g : kNormGroups);
}

static unsigned norm_grid(int64_t rows, int at_once) {
    const int64_t g = (rows + at_once - 1) / at_once;
    return (unsigned)(g < 65536 ? g : 65536);
}

}  // namespace gs

using namespace gs;

extern "C" int gs_layer_norm_forward(const void *x, int64_t x_stride, const void *weight,
                                     const void *bias, int64_t rows, int32_t channels, float eps,
                                     int32_t type, int32_t weight_type, void *y, float *stats,
                                     hipStream_t stream) {
    if (rows < 0 || channels <= 0 || x_stride < 0 || !(eps >= 0.0f) || !element_type(type) ||
        !element_type(weight_type))
        return GS_ERR_INVALID_ARGUMENT;
    if (channels > GS_MAX_CHANNELS) return GS_ERR_UNSUPPORTED;
    if (rows == 0) return GS_OK;
    if (!x || !y) return GS_ERR_INVALID_ARGUMENT;
    return with_element(type, [&](auto t) {
        using T = decltype(t);
        return with_shape<T>(channels, [&](auto shape) {
            using S = decltype(shape);
            const Weights w = {weight, weight_type}, b = {bias, weight_type};
            if constexpr (std::is_same<S, int>::value)
                hipLaunchKernelGGL((layer_norm_long_kernel<T>), dim3(norm_grid(rows, 1)),
                                   dim3(kNormBlock), 0, stream, (const T *)x, x_stride, w, b, rows,
                                   channels, eps, (T *)y, (float2 *)stats);
            else
                hipLaunchKernelGGL((layer_norm_kernel<T, S>), dim3(norm_grid(rows, S::kRows)),
                                   dim3(kNormBlock), 0, stream, (const T *)x, x_stride, w, b, rows,
                                   channels, eps, (T *)y, (float2 *)stats);
            return launch_status();
        });
    });
}

extern "C" int gs_layer_norm_backward_workspace_size(int64_t rows, int32_t channels,
                                                     size_t *bytes) {
    if (rows < 0 || channels <= 0 || !bytes) return GS_ERR_INVALID_ARGUMENT;
    if (channels > GS_MAX_CHANNELS) return GS_ERR_UNSUPPORTED;
    *bytes = (size_t)norm_groups(rows) * 2 * channels * sizeof(float);
    return GS_OK;
}

extern "C" int gs_layer_norm_backward(const void *grad_y, int64_t grad_y_stride, const void *x,
                                      int64_t x_stride, const void *weight, const float *stats,
                                      int64_t rows, int32_t channels, int32_t type,
                                      int32_t weight_type, void *grad_x, void *grad_weight,
                                      void *grad_bias, void *workspace, size_t workspace_bytes,
                                      hipStream_t stream) {
    if (rows < 0 || channels <= 0 || x_stride < 0 || grad_y_stride < 0 || !element_type(type) ||
        !element_type(weight_type))
        return GS_ERR_INVALID_ARGUMENT;
    if (channels > GS_MAX_CHANNELS) return GS_ERR_UNSUPPORTED;
    if (rows > 0 && (!grad_y || !x || !stats)) return GS_ERR_INVALID_ARGUMENT;
    const bool sums = grad_weight || grad_bias;
    const int groups = norm_groups(rows);
    if (sums && rows > 0) {
        if (!workspace) return GS_ERR_INVALID_ARGUMENT;
        if (workspace_bytes < (size_t)groups * 2 * channels * sizeof(float))
            return GS_ERR_WORKSPACE_TOO_SMALL;
    }
    if (rows > 0 && (sums || grad_x)) {
        const int st = with_element(type, [&](auto t) {
            using T = decltype(t);
            return with_shape<T>(channels, [&](auto shape) {
                using S = decltype(shape);
                const Weights w = {weight, weight_type};
                const dim3 block(kNormBlock);
                float *partial = (float *)workspace;
                if constexpr (std::is_same<S, int>::value) {
                    if (grad_x)
                        hipLaunchKernelGGL((layer_norm_long_dx_kernel<T>), dim3(norm_grid(rows, 1)),
                                           block, 0, stream, (const T *)grad_y, grad_y_stride,
                                           (const T *)x, x_stride, w, (const float2 *)stats, rows,
                                           channels, (T *)grad_x);
                    if (sums)
                        hipLaunchKernelGGL((layer_norm_long_sums_kernel<T>),
                                           dim3(ceil_div(channels, kNormBlock), groups), block, 0,
                                           stream, (const T *)grad_y, grad_y_stride, (const T *)x,
                                           x_stride, (const float2 *)stats, rows, channels, partial);
                } else if (sums) {
                    hipLaunchKernelGGL((layer_norm_backward_kernel<T, S, true>), dim3(groups), block,
                                       0, stream, (const T *)grad_y, grad_y_stride, (const T *)x,
                                       x_stride, w, (const float2 *)stats, rows, channels,
                                       (T *)grad_x, partial);
                } else {
                    hipLaunchKernelGGL((layer_norm_backward_kernel<T, S, false>),
                                       dim3(norm_grid(rows, S::kRows)), block, 0, stream,
                                       (const T *)grad_y, grad_y_stride, (const T *)x, x_stride, w,
                                       (const float2 *)stats, rows, channels, (T *)grad_x,
                                       (float *)nullptr);
                }
                return launch_status();
            });
        });
        if (st) return st;
    }
    if (!sums) return GS_OK;
    hipLaunchKernelGGL(layer_norm_join_kernel, dim3(ceil_div(2 * (int64_t)channels, kJoinColumns)),
                       dim3(kJoinColumns * kJoinRows), 0, stream, (const float *)workspace,
                       rows > 0 ? groups : 0, channels, weight_type, grad_weight, grad_bias);
    return launch_status();
}
