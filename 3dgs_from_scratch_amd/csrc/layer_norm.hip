// Layer norm over the channels of a row and its gradients:
//   h = (x - mean) r,  r = 1 / sqrt(mean((x - mean)^2) + eps),  y = h w + b
//   dx = r (g - mean(g) - h mean(g h)) with g = dy w,  dw = sum dy h,  db = sum dy
// the means over a row's channels, the sums over the rows.  All arithmetic is in
// float; an output is rounded once.

#include "element.h"

namespace gs {

constexpr int kNormBlock = 256;
constexpr int kNormSplits = 512;  // most row ranges of the weight's gradient

// The sums of a and b over the workgroup, in every thread.
__device__ __forceinline__ float2 block_sum2(float a, float b) {
    __shared__ float2 part[kNormBlock / kWave];
    a = wave_sum(a);
    b = wave_sum(b);
    __syncthreads();  // an earlier call's values have been read
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = make_float2(a, b);
    __syncthreads();
    float2 s = part[0];
#pragma unroll
    for (int w = 1; w < kNormBlock / kWave; ++w) {
        s.x += part[w].x;
        s.y += part[w].y;
    }
    return s;
}

template <typename T, typename W>
__global__ __launch_bounds__(kNormBlock) void layer_norm_kernel(
    const T *__restrict__ x, int64_t x_stride, const W *__restrict__ weight,
    const W *__restrict__ bias, int64_t rows, int channels, float eps, T *__restrict__ y,
    float2 *__restrict__ stats) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * x_stride;
        T *yr = y + row * channels;
        float s = 0.0f;
        for (int c = threadIdx.x; c < channels; c += kNormBlock) s += to_float(xr[c]);
        const float mean = block_sum2(s, 0.0f).x / (float)channels;
        float q = 0.0f;
        for (int c = threadIdx.x; c < channels; c += kNormBlock) {
            const float d = to_float(xr[c]) - mean;
            q = fmaf(d, d, q);
        }
        const float r = 1.0f / sqrtf(block_sum2(q, 0.0f).x / (float)channels + eps);
        for (int c = threadIdx.x; c < channels; c += kNormBlock) {
            const float h = (to_float(xr[c]) - mean) * r;
            yr[c] = from_float<T>(fmaf(h, weight ? to_float(weight[c]) : 1.0f,
                                       bias ? to_float(bias[c]) : 0.0f));
        }
        if (stats && threadIdx.x == 0) stats[row] = make_float2(mean, r);
    }
}

template <typename T, typename W>
__global__ __launch_bounds__(kNormBlock) void layer_norm_dx_kernel(
    const T *__restrict__ dy, int64_t dy_stride, const T *__restrict__ x, int64_t x_stride,
    const W *__restrict__ weight, const float2 *__restrict__ stats, int64_t rows, int channels,
    T *__restrict__ dx) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * x_stride, *gr = dy + row * dy_stride;
        const float2 st = stats[row];
        float a = 0.0f, b = 0.0f;
        for (int c = threadIdx.x; c < channels; c += kNormBlock) {
            const float g = to_float(gr[c]) * (weight ? to_float(weight[c]) : 1.0f);
            a += g;
            b = fmaf(g, (to_float(xr[c]) - st.x) * st.y, b);
        }
        const float2 m = block_sum2(a, b);
        const float ma = m.x / (float)channels, mb = m.y / (float)channels;
        for (int c = threadIdx.x; c < channels; c += kNormBlock) {
            const float g = to_float(gr[c]) * (weight ? to_float(weight[c]) : 1.0f);
            const float h = (to_float(xr[c]) - st.x) * st.y;
            dx[row * channels + c] = from_float<T>(st.y * (g - ma - h * mb));
        }
    }
}

// partial[split][0..1][channel]: sums of dy h and of dy over the split's rows.
template <typename T>
__global__ __launch_bounds__(kNormBlock) void layer_norm_dw_kernel(
    const T *__restrict__ dy, int64_t dy_stride, const T *__restrict__ x, int64_t x_stride,
    const float2 *__restrict__ stats, int64_t rows, int channels, int64_t split_rows,
    float *__restrict__ partial) {
    const int c = blockIdx.x * kNormBlock + threadIdx.x;
    if (c >= channels) return;
    const int64_t first = blockIdx.y * split_rows;
    const int64_t last = first + split_rows < rows ? first + split_rows : rows;
    float w = 0.0f, b = 0.0f;
    for (int64_t row = first; row < last; ++row) {
        const float2 st = stats[row];
        const float g = to_float(dy[row * dy_stride + c]);
        w = fmaf(g, (to_float(x[row * x_stride + c]) - st.x) * st.y, w);
        b += g;
    }
    float *p = partial + (int64_t)blockIdx.y * 2 * channels + c;
    p[0] = w;
    p[channels] = b;
}

template <typename W>
__global__ __launch_bounds__(kNormBlock) void layer_norm_join_kernel(
    const float *__restrict__ partial, int splits, int channels, W *__restrict__ dw,
    W *__restrict__ db) {
    const int c = blockIdx.x * kNormBlock + threadIdx.x;
    if (c >= channels) return;
    float w = 0.0f, b = 0.0f;
    for (int s = 0; s < splits; ++s) {
        w += partial[(int64_t)s * 2 * channels + c];
        b += partial[(int64_t)s * 2 * channels + channels + c];
    }
    if (dw) dw[c] = from_float<W>(w);
    if (db) db[c] = from_float<W>(b);
}

static int norm_splits(int64_t rows) {
    const int64_t s = (rows + 15) / 16;
    return (int)(s < kNormSplits ? s : kNormSplits);
}

static unsigned norm_grid(int64_t rows) { return (unsigned)(rows < 65536 ? rows : 65536); }

}  // namespace gs

using namespace gs;

extern "C" int gs_layer_norm_forward(const void *x, int64_t x_stride, const void *weight,
                                     const void *bias, int64_t rows, int32_t channels, float eps,
                                     int32_t type, int32_t weight_type, void *y, float *stats,
                                     hipStream_t stream) {
    if (rows < 0 || channels <= 0 || x_stride < 0 || !(eps >= 0.0f) || !element_type(type) ||
        !element_type(weight_type))
        return GS_ERR_INVALID_ARGUMENT;
    if (rows == 0) return GS_OK;
    if (!x || !y) return GS_ERR_INVALID_ARGUMENT;
    return with_element(type, [&](auto t) {
        return with_element(weight_type, [&](auto w) {
            using T = decltype(t);
            using W = decltype(w);
            hipLaunchKernelGGL((layer_norm_kernel<T, W>), dim3(norm_grid(rows)), dim3(kNormBlock),
                               0, stream, (const T *)x, x_stride, (const W *)weight,
                               (const W *)bias, rows, channels, eps, (T *)y, (float2 *)stats);
            return launch_status();
        });
    });
}

extern "C" int gs_layer_norm_backward_workspace_size(int64_t rows, int32_t channels,
                                                     size_t *bytes) {
    if (rows < 0 || channels <= 0 || !bytes) return GS_ERR_INVALID_ARGUMENT;
    *bytes = (size_t)norm_splits(rows) * 2 * channels * sizeof(float);
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
    if (rows > 0 && (!grad_y || !x || !stats)) return GS_ERR_INVALID_ARGUMENT;
    const bool sums = grad_weight || grad_bias;
    const int splits = norm_splits(rows);
    if (sums && rows > 0) {
        if (!workspace) return GS_ERR_INVALID_ARGUMENT;
        if (workspace_bytes < (size_t)splits * 2 * channels * sizeof(float))
            return GS_ERR_WORKSPACE_TOO_SMALL;
    }
    return with_element(type, [&](auto t) {
        return with_element(weight_type, [&](auto w) {
            using T = decltype(t);
            using W = decltype(w);
            const dim3 block(kNormBlock);
            int st = GS_OK;
            if (grad_x && rows > 0) {
                hipLaunchKernelGGL((layer_norm_dx_kernel<T, W>), dim3(norm_grid(rows)), block, 0,
                                   stream, (const T *)grad_y, grad_y_stride, (const T *)x,
                                   x_stride, (const W *)weight, (const float2 *)stats, rows,
                                   channels, (T *)grad_x);
                if ((st = launch_status())) return st;
            }
            if (!sums) return st;
            const int columns = ceil_div(channels, kNormBlock);
            if (splits > 0) {
                const int64_t split_rows = (rows + splits - 1) / splits;
                hipLaunchKernelGGL((layer_norm_dw_kernel<T>), dim3(columns, splits), block, 0,
                                   stream, (const T *)grad_y, grad_y_stride, (const T *)x,
                                   x_stride, (const float2 *)stats, rows, channels, split_rows,
                                   (float *)workspace);
                if ((st = launch_status())) return st;
            }
            hipLaunchKernelGGL((layer_norm_join_kernel<W>), dim3(columns), block, 0, stream,
                               (const float *)workspace, splits, channels, (W *)grad_weight,
                               (W *)grad_bias);
            return launch_status();
        });
    });
}
