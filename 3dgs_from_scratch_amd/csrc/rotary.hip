// Rotary positions of several axes: pair p of every head of a token is turned by
// the angle position[axis(p)] * frequency[p]; the gradient is the turn back.
//
// Bound by memory: every element is read and written once.  A thread takes the same
// pairs of up to five heads of a token, so that an angle's sine and cosine are computed
// once for them, and reads and writes 16 (or 8) bytes at a time where the layout
// allows it.

#include <type_traits>

#include "element.h"

namespace gs {

constexpr int kRotaryBlock = 256;
constexpr int kRotaryTensors = 2;

struct RotaryBatch {
    GsRotaryTensor t[kRotaryTensors];
    int32_t ends[GS_MAX_AXES];  // one past each axis's last pair
    int32_t axes, pairs, dim, n;
    int32_t heads, groups;  // of all tensors; a thread has every groups-th head
    const void *positions;
    int64_t position_stride;
    const float *frequencies;
    float sign;  // of the angle
};

// sin and cos of position * frequency.  The product is reduced to an eighth of a turn
// to either side in double: a float product of a position in the thousands is off by
// 1e-4 of a radian before any sine is taken.  On what is left, at most pi / 4, Taylor's
// sums to x^9 and x^10 are within 2e-9.  FAR: also where the number of quarter turns is rounded,
// from 2^53 on by whole ones (a position may be a time in nanoseconds): what it is off by is
// reduced again.
template <bool FAR>
__device__ __forceinline__ void turn_of(double angle, float *s, float *c) {
    const double quarters = rint(angle * 0.63661977236758134308);
    // pi / 2 in two parts: quarters * the first is exact to 2^-53 of the angle
    double rest = fma(quarters, -6.123233995736766e-17, fma(quarters, -1.5707963267948966, angle));
    int quarter = (int)((int64_t)quarters & 3);
    if constexpr (FAR) {
        const double more = rint(rest * 0.63661977236758134308);
        rest = fma(more, -6.123233995736766e-17, fma(more, -1.5707963267948966, rest));
        quarter = (int)(quarters - 4.0 * floor(quarters * 0.25)) + (int)more;
    }
    const float x = (float)rest, x2 = x * x;
    float sine = fmaf(x2, 2.7557319e-6f, -1.9841270e-4f);
    sine = fmaf(x2, sine, 8.3333333e-3f);
    sine = fmaf(x2, sine, -1.6666667e-1f);
    sine = fmaf(x2 * sine, x, x);
    float cosine = fmaf(x2, -2.7557319e-7f, 2.4801587e-5f);
    cosine = fmaf(x2, cosine, -1.3888889e-3f);
    cosine = fmaf(x2, cosine, 4.1666667e-2f);
    cosine = fmaf(x2, cosine, -0.5f);
    cosine = fmaf(x2, cosine, 1.0f);
    const float a = quarter & 1 ? cosine : sine, b = quarter & 1 ? sine : cosine;
    *s = quarter & 2 ? -a : a;
    *c = (quarter + 1) & 2 ? -b : b;
}

// A thread's accesses are VEC elements; interleaved pairs that may not be read together
// are two of one.  Thread (token, unit) has the pairs from VEC * unit on (halves of a head
// apart), or the pairs of the elements from unit * kElements on (interleaved), or as many
// elements of the part that is copied.
template <bool INTERLEAVED, int VEC>
struct Unit {
    static constexpr int kElements = INTERLEAVED && VEC == 1 ? 2 : VEC;
    static constexpr int kPairs = INTERLEAVED ? kElements / 2 : VEC;
    __host__ __device__ static int64_t count(int dim, int pairs) {  // a head
        return INTERLEAVED ? (dim + kElements - 1) / kElements : (dim - pairs) / VEC;
    }
};

template <typename T, typename P, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(kRotaryBlock) void rotary_kernel(RotaryBatch b, int64_t tokens) {
    using U = Unit<INTERLEAVED, VEC>;
    const int units = (int)U::count(b.dim, b.pairs);
    const int64_t i = (int64_t)blockIdx.x * kRotaryBlock + threadIdx.x;
    const int64_t token = i / ((int64_t)units * b.groups);
    if (token >= tokens) return;
    const int64_t place = i - token * units * b.groups;
    const int head0 = (int)(place / units);
    const int unit = (int)(place - (int64_t)head0 * units), pair = unit * U::kPairs;
    const bool turned = pair < b.pairs;
    float s[U::kPairs], c[U::kPairs];
    if (turned) {
        const P *at = (const P *)b.positions + token * b.position_stride;
        const auto turns = [&](auto far) {
            bool near = true;
#pragma unroll
            for (int j = 0; j < U::kPairs; ++j) {
                int axis = 0;
                for (int a = 0; a + 1 < b.axes; ++a) axis += pair + j >= b.ends[a];
                const double angle = (double)at[axis] * (double)b.frequencies[pair + j];
                near = near && !(fabs(angle) > 0x1p40);
                turn_of<decltype(far)::value>(angle, &s[j], &c[j]);
                s[j] *= b.sign;
            }
            return near;
        };
        if (!turns(std::false_type{})) turns(std::true_type{});
    }
    const int first = INTERLEAVED ? unit * U::kElements : turned ? pair : pair + b.pairs;
    const bool odd_end = U::kElements > VEC && first + 1 >= b.dim;  // one element is left
#pragma unroll 2
    for (int head = head0; head < b.heads; head += b.groups) {
        const bool second = head >= b.t[0].heads;
        const GsRotaryTensor &t = b.t[second];
        const int h = second ? head - b.t[0].heads : head;
        const T *x = (const T *)t.x + token * t.x_token + h * t.x_head + first;
        T *y = (T *)t.y + token * t.y_token + h * t.y_head + first;
        float u[U::kElements];
#pragma unroll
        for (int j = 0; j < U::kElements; j += VEC)
            if (j == 0 || !odd_end) load_floats<T, VEC>(x + j, u + j);
        if (turned) {
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int j = 0; j < U::kPairs; ++j) {
                    const float p = u[2 * j], q = u[2 * j + 1];
                    u[2 * j] = p * c[j] - q * s[j];
                    u[2 * j + 1] = p * s[j] + q * c[j];
                }
            } else {
                float v[VEC];
                load_floats<T, VEC>(x + b.pairs, v);
#pragma unroll
                for (int j = 0; j < U::kPairs; ++j) {
                    const float p = u[j], q = v[j];
                    u[j] = p * c[j] - q * s[j];
                    v[j] = p * s[j] + q * c[j];
                }
                store_floats<T, VEC>(y + b.pairs, v);
            }
        }
#pragma unroll
        for (int j = 0; j < U::kElements; j += VEC)
            if (j == 0 || !odd_end) store_floats<T, VEC>(y + j, u + j);
    }
}

// The widest access that the layout allows, of 16 or 8 bytes (4 elements) or one element.
template <typename T>
static int rotary_vector(const RotaryBatch &b, bool interleaved) {
    int vec = 16 / sizeof(T);
    const auto fits = [&](int v) {
        if (b.dim % v || (interleaved ? 2 * b.pairs : b.pairs) % v) return false;
        for (int n = 0; n < b.n; ++n) {
            const GsRotaryTensor &t = b.t[n];
            if ((t.x_token | t.x_head | t.y_token | t.y_head) % v ||
                (((uintptr_t)t.x | (uintptr_t)t.y) % (v * sizeof(T))))
                return false;
        }
        return true;
    };
    while (vec >= 4 && !fits(vec)) vec /= 2;
    return vec >= 4 ? vec : 1;
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
    int64_t pairs = 0, heads = 0;
    for (int a = 0; a < axes; ++a) {
        if (sections[a] < 0) return GS_ERR_INVALID_ARGUMENT;
        pairs += sections[a];
        if (2 * pairs > dim) return GS_ERR_INVALID_ARGUMENT;
        batch.ends[a] = (int32_t)pairs;
    }
    for (int n = 0; n < n_tensors; ++n) {
        const GsRotaryTensor &t = tensors[n];
        if (t.heads < 0 || t.x_token < 0 || t.x_head < 0 || t.y_token < 0 || t.y_head < 0)
            return GS_ERR_INVALID_ARGUMENT;
        if (tokens > 0 && t.heads > 0 && (!t.x || !t.y)) return GS_ERR_INVALID_ARGUMENT;
        batch.t[n] = t;
        heads += t.heads;
    }
    if (tokens == 0 || heads == 0) return GS_OK;
    if (pairs > 0 && (!positions || !frequencies)) return GS_ERR_INVALID_ARGUMENT;
    if (heads > 0x7fffffffLL) return GS_ERR_UNSUPPORTED;
    batch.axes = axes;
    batch.n = n_tensors;
    batch.pairs = (int32_t)pairs;
    batch.dim = dim;
    batch.heads = (int32_t)heads;
    batch.positions = positions;
    batch.position_stride = position_stride;
    batch.frequencies = frequencies;
    batch.sign = inverse ? -1.0f : 1.0f;
    return with_element(type, [&](auto t) {
        using T = decltype(t);
        const auto launch = [&](auto p, auto vec, auto between) {
            using P = decltype(p);
            constexpr int kVec = decltype(vec)::value;
            constexpr bool kBetween = decltype(between)::value;
            const int64_t units = Unit<kBetween, kVec>::count(dim, (int)pairs);
            // Five heads a thread, so that an angle is computed a fifth as often, or fewer where
            // the card would have less than 512 workgroups; a token's threads lie next to each
            // other and take every groups-th head, so that a wave's accesses do too.  65280
            // tokens of 20 heads of 128, bfloat16, one way: 5 heads a thread 136 us (4.9 TB/s),
            // 10 151, 20 168, 1 173; 2500 tokens: 3 heads 9 us, 20 25; 12 tokens: 1 head 4, 20 13.
            int64_t each = 5;
            const auto threads = [&] { return tokens * units * ((heads + each - 1) / each); };
            while (each > 1 && threads() < 512 * kRotaryBlock) each = (each + 1) / 2;
            RotaryBatch b = batch;
            b.groups = (int32_t)((heads + each - 1) / each);
            const int64_t blocks = (threads() + kRotaryBlock - 1) / kRotaryBlock;
            if (blocks > 0x7fffffffLL) return (int)GS_ERR_UNSUPPORTED;
            hipLaunchKernelGGL((rotary_kernel<T, P, kVec, kBetween>), dim3((unsigned)blocks),
                               dim3(kRotaryBlock), 0, stream, b, tokens);
            return launch_status();
        };
        const auto with_position = [&](auto vec, auto between) {
            return position_type == GS_POS_I32   ? launch(int32_t{}, vec, between)
                   : position_type == GS_POS_I64 ? launch(int64_t{}, vec, between)
                                                 : launch(float{}, vec, between);
        };
        const int vec = rotary_vector<T>(batch, interleaved != 0);
        const auto with_vector = [&](auto between) {
            if constexpr (sizeof(T) == 2)
                if (vec == 8) return with_position(std::integral_constant<int, 8>{}, between);
            if (vec >= 4) return with_position(std::integral_constant<int, 4>{}, between);
            return with_position(std::integral_constant<int, 1>{}, between);
        };
        return interleaved ? with_vector(std::true_type{}) : with_vector(std::false_type{});
    });
}
