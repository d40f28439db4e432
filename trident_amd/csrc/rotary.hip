// Rotary positions: in every head, pairs of columns are turned by an angle that grows with the token's
// position,
//
//   (x0, x1) -> a (x0 cos t - x1 sin t, x0 sin t + x1 cos t),   t = position * frequency,
//
// the pairs being columns 2 i and 2 i + 1 (interleaved) or i and i + R / 2 (halves) of a head's first R; the
// rest is copied.  The inverse turns back, with the same factor a: the gradient.
//
// Bound by bytes: one read and one write (131,072 tokens of 24 heads of 64, bfloat16, 157 us, 5.1 TB/s; 16,385
// of 40 heads of 128, half of each turned, float32, 142 us, 4.7 TB/s).  A token's angles are the same for all
// of its heads, so a workgroup first makes those of its tokens, in LDS: the turns in float64, since a position
// of 1e6 leaves a float32 no digits of the angle, and sine and cosine of what is left of a whole turn in
// float32.
#include "encoder.hpp"

namespace trident {
namespace {

constexpr int kAngles = 1024;  // of a workgroup's tokens, at most

struct RotaryArgs {
    const void* x;
    void* out;
    const double* frequencies;
    const void* positions;
    int64_t x_row, x_head, out_row, out_head;  // elements
    int64_t tokens, period;
    int heads, D, pairs, tokens_each, wide, interleaved, copy;
    float amplitude, sign;
};

template <typename T, int V>
__device__ __forceinline__ void load_some(const T* p, float (&f)[V]) {
    typedef T tv __attribute__((ext_vector_type(V)));
    tv t;
    __builtin_memcpy(&t, p, sizeof(T) * V);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (float)t[i];
}

// V columns at a time: 16 bytes where what is turned is whole multiples of it.
template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kBlock) void rotary_kernel(RotaryArgs a) {
    __shared__ float2 angles[kAngles];  // sine and cosine, times the amplitude
    const int64_t t0 = (int64_t)blockIdx.x * a.tokens_each;
    const int n = (int)min((int64_t)a.tokens_each, a.tokens - t0);
    for (int i = threadIdx.x; i < n * a.pairs; i += kBlock) {
        const int t = i / a.pairs;
        const int64_t p = (t0 + t) % a.period;
        const double position =
            !a.positions ? (double)p
                         : a.wide ? (double)static_cast<const int64_t*>(a.positions)[p]
                                  : (double)static_cast<const int32_t*>(a.positions)[p];
        const double turns = position * a.frequencies[i - t * a.pairs] * 0.15915494309189535;  // 1 / 2 pi
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        angles[i] = make_float2(a.amplitude * a.sign * s, a.amplitude * c);
    }
    __syncthreads();
    constexpr int kOf = INTERLEAVED ? 2 : 1;  // columns of a vector's angle
    const int turned = a.pairs * (INTERLEAVED ? 2 : 1) / V, items = turned + (a.copy ? (a.D - 2 * a.pairs + V - 1) / V : 0);
    const int each = a.heads * items;
    for (int i = threadIdx.x; i < n * each; i += kBlock) {
        const int t = i / each, in = i - t * each, h = in / items, c = in - h * items;
        const T* x = static_cast<const T*>(a.x) + (t0 + t) * a.x_row + h * a.x_head;
        T* y = static_cast<T*>(a.out) + (t0 + t) * a.out_row + h * a.out_head;
        float f[V];
        if (c >= turned) {
            const int col = 2 * a.pairs + (c - turned) * V;
            if (col + V <= a.D) {
                load_some<T, V>(x + col, f);
                store_vec(y + col, f);
            } else {
                for (int e = col; e < a.D; ++e) y[e] = x[e];
            }
            continue;
        }
        const float2* w = angles + t * a.pairs + c * V / kOf;
        if constexpr (INTERLEAVED) {
            load_some<T, V>(x + c * V, f);
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const float2 r = w[e / 2];
                const float x0 = f[e], x1 = f[e + 1];
                f[e] = __builtin_fmaf(x0, r.y, -x1 * r.x);
                f[e + 1] = __builtin_fmaf(x0, r.x, x1 * r.y);
            }
            store_vec(y + c * V, f);
        } else {
            float g[V];
            load_some<T, V>(x + c * V, f);
            load_some<T, V>(x + a.pairs + c * V, g);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 r = w[e];
                const float x0 = f[e], x1 = g[e];
                f[e] = __builtin_fmaf(x0, r.y, -x1 * r.x);
                g[e] = __builtin_fmaf(x0, r.x, x1 * r.y);
            }
            store_vec(y + c * V, f);
            store_vec(y + a.pairs + c * V, g);
        }
    }
}

template <typename T, int V>
int launch(RotaryArgs a, hipStream_t st) {
    if constexpr (V > 1) {
        if ((a.interleaved ? 2 * a.pairs : a.pairs) % V) return launch<T, V / 2>(a, st);
    }
    const unsigned grid = (unsigned)((a.tokens + a.tokens_each - 1) / a.tokens_each);
    if (!a.interleaved) rotary_kernel<T, V, false><<<grid, kBlock, 0, st>>>(a);
    else if constexpr (V > 1) rotary_kernel<T, V, true><<<grid, kBlock, 0, st>>>(a);
    return capi_check_launch("rotary_kernel");
}

}  // namespace
}  // namespace trident

using namespace trident;

extern "C" int trident_rotary(const void* x, int32_t dtype, int64_t tokens, int64_t heads, int64_t head_dim,
                              int64_t x_row, int64_t x_head, const double* frequencies, int64_t pairs,
                              const void* positions, int32_t ids64, int64_t period, int32_t interleaved,
                              double amplitude, int32_t inverse, void* out, int64_t out_row, int64_t out_head,
                              void* stream) {
    if (!dtype_ok(dtype)) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "rotary: dtype=%d", dtype);
    if (tokens < 0 || tokens > (1 << 30) || heads < 0 || heads > (1 << 20) || head_dim < 1 || head_dim > (1 << 20) ||
        pairs < 0 || 2 * pairs > head_dim || period < 1 || heads * head_dim > (1 << 24))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT,
                         "rotary: bad sizes tokens=%lld heads=%lld head_dim=%lld pairs=%lld period=%lld",
                         (long long)tokens, (long long)heads, (long long)head_dim, (long long)pairs, (long long)period);
    if (pairs > kAngles) return capi_fail(TRIDENT_ERR_UNSUPPORTED, "rotary: %lld pairs", (long long)pairs);
    // as many tokens as leave every CU eight workgroups
    const int64_t most = std::min<int64_t>(kAngles / std::max<int64_t>(pairs, 1), 16);
    const int64_t tokens_each = std::max<int64_t>(1, std::min(most, tokens / 2048));
    if (tokens / tokens_each >= 0xffffff)  // a launch has fewer than 2^32 threads
        return capi_fail(TRIDENT_ERR_UNSUPPORTED, "rotary: %lld tokens of %lld pairs are too many", (long long)tokens,
                         (long long)pairs);
    if (!(amplitude > -1e30 && amplitude < 1e30))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "rotary: amplitude=%g", amplitude);
    if (tokens == 0 || heads == 0) return TRIDENT_OK;
    if (!x || !out || (pairs && !frequencies)) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "rotary: NULL pointer");
    RotaryArgs a{x, out, frequencies, positions, x_row, x_head, out_row, out_head, tokens, period, (int)heads,
                 (int)head_dim, (int)pairs, (int)tokens_each, ids64, interleaved != 0, x != out, (float)amplitude,
                 inverse ? -1.0f : 1.0f};
    int rc = TRIDENT_OK;
    with_dtype(dtype, [&](auto e) {
        using T = decltype(e);
        rc = launch<T, kVec<T>>(a, (hipStream_t)stream);
    });
    return rc;
}
