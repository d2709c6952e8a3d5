// Rotary positions of several axes: pair p of every head of a token is turned by
// the angle position[axis(p)] * frequency[p]; the gradient is the turn back.

#include "element.h"

namespace gs {

constexpr int kRotaryBlock = 256;
constexpr int kRotaryTensors = 2;

struct RotaryBatch {
    GsRotaryTensor t[kRotaryTensors];
    int32_t ends[GS_MAX_AXES];  // one past each axis's last pair
    int32_t axes, pairs, n;
};

// sin and cos of position * frequency.  The product is reduced to a quarter turn
// in double: a float product of a position in the thousands is off by 1e-4 of a
// radian before any sine is taken.
__device__ __forceinline__ void turn_of(double position, float frequency, float *s, float *c) {
    const double angle = position * (double)frequency;
    sincosf((float)(angle - 6.283185307179586 * rint(angle * 0.15915494309189535)), s, c);
}

template <typename T, typename P>
__global__ __launch_bounds__(kRotaryBlock) void rotary_kernel(
    RotaryBatch batch, const P *__restrict__ positions, int64_t position_stride,
    const float *__restrict__ frequencies, int64_t tokens, int dim, bool interleaved,
    bool inverse) {
    const int pairs = batch.pairs, tail = dim - 2 * pairs, units = pairs + tail;
    const int64_t i = (int64_t)blockIdx.x * kRotaryBlock + threadIdx.x;
    const int64_t token = i / units;
    if (token >= tokens) return;
    const int p = (int)(i - token * units);
    float s = 0.0f, c = 1.0f;
    if (p < pairs) {
        int axis = 0;
        while (axis + 1 < batch.axes && p >= batch.ends[axis]) ++axis;
        turn_of((double)positions[token * position_stride + axis], frequencies[p], &s, &c);
        if (inverse) s = -s;
    }
    const int a = interleaved && p < pairs ? 2 * p : p < pairs ? p : pairs + p;
    const int b = interleaved ? 2 * p + 1 : p + pairs;
    for (int n = 0; n < batch.n; ++n) {
        const GsRotaryTensor &t = batch.t[n];
        const T *x = (const T *)t.x + token * t.x_token;
        T *y = (T *)t.y + token * t.y_token;
        for (int h = 0; h < t.heads; ++h) {
            if (p >= pairs) {
                y[h * t.y_head + a] = x[h * t.x_head + a];
                continue;
            }
            const float u = to_float(x[h * t.x_head + a]), v = to_float(x[h * t.x_head + b]);
            y[h * t.y_head + a] = from_float<T>(u * c - v * s);
            y[h * t.y_head + b] = from_float<T>(u * s + v * c);
        }
    }
}

}  // namespace gs

using namespace gs;

extern "C" int gs_axial_rotary(const GsRotaryTensor *tensors, int32_t n_tensors,
                               const void *positions, int64_t position_stride,
                               int32_t position_type, const float *frequencies,
                               const int32_t *sections, int32_t axes, int64_t tokens, int32_t dim,
                               int32_t type, int32_t interleaved, int32_t inverse,
                               hipStream_t stream) {
    if (!tensors || n_tensors < 1 || n_tensors > kRotaryTensors || !sections || axes < 1 ||
        axes > GS_MAX_AXES || tokens < 0 || dim < 1 || position_stride < 0 || !element_type(type) ||
        position_type < GS_POS_I32 || position_type > GS_POS_F32)
        return GS_ERR_INVALID_ARGUMENT;
    RotaryBatch batch{};
    batch.axes = axes;
    batch.n = n_tensors;
    int64_t pairs = 0;
    for (int a = 0; a < axes; ++a) {
        if (sections[a] < 0) return GS_ERR_INVALID_ARGUMENT;
        pairs += sections[a];
        if (2 * pairs > dim) return GS_ERR_INVALID_ARGUMENT;
        batch.ends[a] = (int32_t)pairs;
    }
    batch.pairs = (int32_t)pairs;
    for (int n = 0; n < n_tensors; ++n) {
        const GsRotaryTensor &t = tensors[n];
        if (t.heads < 0 || t.x_token < 0 || t.x_head < 0 || t.y_token < 0 || t.y_head < 0)
            return GS_ERR_INVALID_ARGUMENT;
        if (tokens > 0 && t.heads > 0 && (!t.x || !t.y)) return GS_ERR_INVALID_ARGUMENT;
        batch.t[n] = t;
    }
    if (tokens == 0) return GS_OK;
    if (pairs > 0 && (!positions || !frequencies)) return GS_ERR_INVALID_ARGUMENT;
    const int64_t blocks = (tokens * (dim - pairs) + kRotaryBlock - 1) / kRotaryBlock;
    if (blocks > 0x7fffffffLL) return GS_ERR_UNSUPPORTED;
    return with_element(type, [&](auto t) {
        using T = decltype(t);
        const auto launch = [&](auto p) {
            using P = decltype(p);
            hipLaunchKernelGGL((rotary_kernel<T, P>), dim3((unsigned)blocks), dim3(kRotaryBlock),
                               0, stream, batch, (const P *)positions, position_stride,
                               frequencies, tokens, dim, interleaved != 0, inverse != 0);
            return launch_status();
        };
        return position_type == GS_POS_I32   ? launch(int32_t{})
               : position_type == GS_POS_I64 ? launch(int64_t{})
                                             : launch(float{});
    });
}
