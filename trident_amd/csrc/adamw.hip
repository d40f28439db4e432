// One AdamW step over many tensors.
//
//   g = grad_scale G     m = b1 m + (1 - b1) g     v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// All arithmetic is float32 and each operation is rounded by itself (no fused multiply-add), so the
// states are the same bits as those of the formulas evaluated one operation at a time.
//
// The states of all tensors lie in one flat buffer each, a tensor's at a multiple of 256 elements.  In
// 8 bits, a block of 256 shares one float32 scale per moment:
//   m       = c |c| sm   c in [-127, 127]   sm = max |m| / 127^2
//   sqrt(v) = c^2 sv     c in [0, 255]      sv = max sqrt(v) / 255^2
// with c one of the two integers around the root of the value over the scale.  The square spaces the
// codes finely near zero: the smallest code is 6e-5 (m) and 1.5e-5 (sqrt v) of the block's largest value.
// A second moment that is not zero keeps a code of at least 1, which errs towards the shorter step: a
// zero there would divide by eps alone.  A block with a value that is not finite gets the scale NaN, so
// that every later step shows it; blocks whose largest value is below 2^-100 are stored as zeros.
//
// Which of the two: the upper one with the probability that makes the stored m, or v, its value in the
// mean, decided by a hash of the element's place, the step and the block's two largest values, so that equal
// calls give equal bits (and a graph, which replays its capture's step number, still goes on to other
// ones).  The nearest would not do:
// a step moves v by a thousandth, which is never half a code, and m below code 10 by less than half of one,
// so beside a larger value of its block a moment would stand still for good.  (These formulas evaluated on
// 256-element blocks, half with a gradient in every step and half with one at step 10: 5,000 steps move the
// second half 5.2 lr with states in 32 bits, 5.2 so, and 1,700, without end, by the nearest code.)
// The first 2 / (1 - b1) steps do take the nearest code: they are too few for that, and the rounding's
// noise counts most in them (10,240 parameters with noisy gradients of all magnitudes, distance to the
// 32-bit run after 100 steps, three seeds: 0.079, 0.077 and 0.078 so, 0.083, 0.084 and 0.085 without them,
// 0.15 by nearest codes throughout; the gradient at step 10 above then moves 8 lr).
#include <algorithm>
#include <cmath>

#include "encoder.hpp"

namespace trident {
namespace {

constexpr int kStateBlock = 256;                 // elements that share a scale: one wave, four a lane
constexpr int kPer = kStateBlock / kWave;
constexpr int kChunkElems = 4096;                // elements of one workgroup
constexpr int kMaxTensors = 88;                  // of one launch: the table travels as kernel argument
constexpr float kTiny = 0x1p-100f;

struct Entry {
    void* param;
    const void* grad;
    int64_t numel, offset;
    int32_t first_chunk;
    int16_t dtype, grad_dtype;
};

struct AdamArgs {
    Entry t[kMaxTensors];
    void *m, *v;
    float *m_scale, *v_scale;
    int32_t tensors;
    float b1, b1c, b2, b2c, eps, decay, rate, inv_root, grad_scale;
    uint32_t step_hash;
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");

template <bool PAST_L2, typename T>
__device__ __forceinline__ void load4(const T* p, float (&f)[kPer]) {
    typedef T tv __attribute__((ext_vector_type(kPer)));
    typedef uint32_t words __attribute__((ext_vector_type(sizeof(tv) / 4)));
    const tv v = __builtin_bit_cast(tv, load_words<PAST_L2, words>(p));
#pragma unroll
    for (int i = 0; i < kPer; ++i) f[i] = (float)v[i];
}

// Elements at .. at + 3 of a tensor of `left` more; zeros past its end.
template <bool PAST_L2>
__device__ __forceinline__ void load_any(const void* base, int dtype, int64_t at, int64_t left, float (&f)[kPer]) {
    const auto get = [&](auto t) {
        using T = decltype(t);
        const T* p = static_cast<const T*>(base) + at;
        if (left >= kPer) {
            load4<PAST_L2>(p, f);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) f[i] = i < left ? (float)p[i] : 0.0f;
        }
    };
    if (dtype == TRIDENT_F32) get(float{});
    else if (dtype == TRIDENT_BF16) get(bf16_t{});
    else get(f16_t{});
}

template <bool PAST_L2>
__device__ __forceinline__ void store_any(void* base, int dtype, int64_t at, int64_t left, const float (&f)[kPer]) {
    const auto put = [&](auto t) {
        using T = decltype(t);
        T* p = static_cast<T*>(base) + at;
        if (left >= kPer) {
            put_vec<PAST_L2>(p, f);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (i < left) p[i] = (T)f[i];
        }
    };
    if (dtype == TRIDENT_F32) put(float{});
    else if (dtype == TRIDENT_BF16) put(bf16_t{});
    else put(f16_t{});
}

// The largest of a block's values that are not negative, as bits (NaN above infinity above the rest).
__device__ __forceinline__ float block_top(const float (&x)[kPer]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) top = max(top, __float_as_uint(x[i]));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, kWave));
    return __uint_as_float(top);
}

// A round of a hash: a multiplication by an odd constant takes a key's low bits up, shifts take its high
// bits down.  Four elements of a lane share the first round and have a constant each in the second.
__device__ __forceinline__ uint32_t scatter(uint32_t key, uint32_t by) {
    key = (key ^ (key >> 16)) * by;
    return key ^ (key >> 15);
}
// the fractions of (1 + root 5) / 2 and of the roots of 2, 3, 7 and 11 in 32 bits, made odd
constexpr uint32_t kPhi = 0x9e3779b1u, kRoot2 = 0x6a09e667u, kRoot3 = 0xbb67ae85u, kRoot7 = 0xa54ff53bu,
                   kRoot11 = 0x510e527fu;

// Codes of the block's values x >= 0, the largest of them `top`, with `levels` = (largest code)^2; returns the
// scale.  POWER: what is stored in the mean is x (1) or x^2 (2).  dither: a random number in (0, 1) a value, or null: the nearest
// code.  The root finds the two codes only, so there the instruction's own will do: where it is an ulp off
// over an integer, that integer is the upper code with probability one, or the lower.
template <int POWER>
__device__ __forceinline__ float encode(const float (&x)[kPer], float top, float levels, float inv_levels,
                                        float most, const float* dither, float (&c)[kPer]) {
    const bool fine = top >= kTiny && __float_as_uint(top) < 0x7f800000u;
    const float factor = fine ? (1.0f / top) * levels : 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const float y = x[i] * factor;
        float code;
        if (dither) {
            const float lo = floorf(__builtin_amdgcn_sqrtf(y)), a = lo * lo, gap = lo + lo + 1.0f;
            float step = dither[i] * gap, past = y - a;  // over the scale; past the lower code's value
            if constexpr (POWER == 2) {
                step *= a + (a + gap);
                past *= y + a;
            }
            code = step < past || x[i] == top ? lo + 1.0f : lo;  // the largest value's is exact
        } else {
            code = rintf(sqrtf(y));
        }
        c[i] = fine ? fminf(code, most) : 0.0f;
    }
    return __float_as_uint(top) >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fine ? top * inv_levels : 0.0f;
}

constexpr float kLevelsM = 127.0f * 127.0f, kLevelsV = 255.0f * 255.0f;

// Bound by bytes: every operand is read and written once, a wave a block of 256 elements at a time, so that
// an 8-bit block's largest value is one wave's.  All tensors are one launch (26 small ones 6.8 us).  62
// million float32 elements: states in 32 bits and bfloat16 gradients 300 us, 5.4 TB/s; states in 8 bits and
// float32 gradients 192 us, 5.2 TB/s, and 182 in the first steps, whose codes are the nearest.
template <int BITS, bool DITHER, bool PAST_L2>
__global__ __launch_bounds__(kBlock) void adamw_kernel(AdamArgs a) {
    int lo = 0, hi = a.tensors - 1;  // the last tensor whose first chunk is not past this one
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.t[mid].first_chunk <= (int)blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    const Entry t = a.t[lo];
    const int64_t chunk = (int64_t)(blockIdx.x - t.first_chunk) * kChunkElems;
    const int lane = lane_id();
    for (int b = threadIdx.x / kWave; b < kChunkElems / kStateBlock; b += kWavesPerBlock) {
        const int64_t first = chunk + b * kStateBlock;
        if (first >= t.numel) return;
        const int64_t at = first + lane * kPer, left = t.numel - at, s = t.offset + at;
        const int64_t block = (t.offset + first) / kStateBlock;
        float p[kPer], g[kPer], m[kPer], v[kPer];
        load_any<PAST_L2>(t.param, t.dtype, at, left, p);
        load_any<PAST_L2>(t.grad, t.grad_dtype, at, left, g);
        if constexpr (BITS == 32) {
            load4<PAST_L2>(static_cast<const float*>(a.m) + s, m);
            load4<PAST_L2>(static_cast<const float*>(a.v) + s, v);
        } else {
            const uint32_t cm = *reinterpret_cast<const uint32_t*>(static_cast<const int8_t*>(a.m) + s);
            const uint32_t cv = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.v) + s);
            const float sm = a.m_scale[block], sv = a.v_scale[block];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const float c = (float)(int8_t)(cm >> (8 * i)), r = (float)((cv >> (8 * i)) & 255u);
                m[i] = c * fabsf(c) * sm;
                v[i] = r * r * sv;
                v[i] = v[i] * v[i];
            }
        }
        float root[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const float gi = g[i] * a.grad_scale;
            m[i] = m[i] * a.b1 + gi * a.b1c;
            v[i] = v[i] * a.b2 + (gi * gi) * a.b2c;
            root[i] = sqrtf(v[i]);
            p[i] = p[i] * a.decay - a.rate * (m[i] / (root[i] * a.inv_root + a.eps));
        }
        store_any<PAST_L2>(t.param, t.dtype, at, left, p);
        if constexpr (BITS == 32) {
            put_vec<PAST_L2>(static_cast<float*>(a.m) + s, m);
            put_vec<PAST_L2>(static_cast<float*>(a.v) + s, v);
        } else {
            float size[kPer], cm[kPer], cv[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                size[i] = i < left ? fabsf(m[i]) : 0.0f;
                root[i] = i < left ? root[i] : 0.0f;
            }
            const float top_m = block_top(size), top_v = block_top(root);
            float um[kPer], uv[kPer];  // 16 random bits each, centred
            if constexpr (DITHER) {
                constexpr uint32_t kBy[kPer] = {kPhi, kRoot2, kRoot7, kRoot11};
                const uint64_t quad = (uint64_t)s / kPer;
                const uint32_t tops = __float_as_uint(top_m) * kRoot7 + __float_as_uint(top_v) * kRoot2;
                const uint32_t key = scatter((uint32_t)quad * kPhi + (uint32_t)(quad >> 32) * kRoot11 + a.step_hash + tops,
                                             kRoot3);
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const uint32_t bits = scatter(key, kBy[i]);
                    um[i] = (float)(bits & 0xffffu) * 0x1p-16f + 0x1p-17f;
                    uv[i] = (float)(bits >> 16) * 0x1p-16f + 0x1p-17f;
                }
            }
            const float sm =
                encode<1>(size, top_m, kLevelsM, (float)(1.0 / 16129.0), 127.0f, DITHER ? um : nullptr, cm);
            const float sv =
                encode<2>(root, top_v, kLevelsV, (float)(1.0 / 65025.0), 255.0f, DITHER ? uv : nullptr, cv);
            uint32_t wm = 0, wv = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (root[i] > 0.0f && sv > 0.0f) cv[i] = fmaxf(cv[i], 1.0f);
                const int c = m[i] < 0.0f ? -(int)cm[i] : (int)cm[i];
                wm |= (uint32_t)(c & 255) << (8 * i);
                wv |= (uint32_t)cv[i] << (8 * i);
            }
            *reinterpret_cast<uint32_t*>(static_cast<int8_t*>(a.m) + s) = wm;
            *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.v) + s) = wv;
            if (lane == 0) {
                a.m_scale[block] = sm;
                a.v_scale[block] = sv;
            }
        }
    }
}

// The values that 8-bit states stand for.  Bound by bytes: 62 million 88 us, 7 TB/s, most of it written.
template <bool PAST_L2>
__global__ __launch_bounds__(kBlock) void adam_values_kernel(const uint32_t* __restrict__ cm,
                                                             const uint32_t* __restrict__ cv,
                                                             const float* __restrict__ sm,
                                                             const float* __restrict__ sv, int64_t quads,
                                                             float* __restrict__ m, float* __restrict__ v) {
    const int64_t q = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (q >= quads) return;
    const uint32_t wm = cm[q], wv = cv[q];
    const float fm = sm[q / kWave], fv = sv[q / kWave];
    float x[kPer], y[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const float c = (float)(int8_t)(wm >> (8 * i)), r = (float)((wv >> (8 * i)) & 255u);
        x[i] = c * fabsf(c) * fm;
        y[i] = r * r * fv;
        y[i] = y[i] * y[i];
    }
    put_vec<PAST_L2>(m + q * kPer, x);
    put_vec<PAST_L2>(v + q * kPer, y);
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

}  // namespace
}  // namespace trident

using namespace trident;

extern "C" {

int trident_adamw(const TridentAdamTensor* tensors, int32_t count, const TridentAdamState* state,
                  const TridentAdamParams* params, void* stream) {
    if (count < 0 || (count > 0 && !tensors) || !state || !params)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "adamw: NULL pointer or count=%d", count);
    const TridentAdamParams& h = *params;
    if (h.step < 1 || !(h.beta1 >= 0.0 && h.beta1 < 1.0) || !(h.beta2 >= 0.0 && h.beta2 < 1.0) || !(h.eps >= 0.0))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "adamw: step=%lld betas=%g, %g eps=%g", (long long)h.step,
                         h.beta1, h.beta2, h.eps);
    if (state->bits != 32 && state->bits != 8)
        return capi_fail(TRIDENT_ERR_UNSUPPORTED, "adamw: states of %d bits (32 or 8)", state->bits);
    if (count > 0 && (!state->m || !state->v || (state->bits == 8 && (!state->m_scale || !state->v_scale))))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "adamw: NULL state");
    if (!aligned4(state->m) || !aligned4(state->v))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "adamw: states must be 4-byte aligned");
    for (int i = 0; i < count; ++i) {
        const TridentAdamTensor& t = tensors[i];
        if (!dtype_ok(t.dtype) || !dtype_ok(t.grad_dtype) || t.numel < 0 || t.state_offset < 0 ||
            t.state_offset % kStateBlock || (t.numel > 0 && (!t.param || !t.grad)))
            return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT,
                             "adamw: tensor %d: dtype=%d, %d numel=%lld state_offset=%lld (a multiple of %d)", i,
                             t.dtype, t.grad_dtype, (long long)t.numel, (long long)t.state_offset, kStateBlock);
        // a block is written whole
        if (t.numel > state->len || t.state_offset > state->len - (t.numel + kStateBlock - 1) / kStateBlock * kStateBlock)
            return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "adamw: tensor %d ends past the state's %lld elements", i,
                             (long long)state->len);
        if ((t.numel + kChunkElems - 1) / kChunkElems > 0x3fffffff)
            return capi_fail(TRIDENT_ERR_UNSUPPORTED, "adamw: tensor %d has %lld elements", i, (long long)t.numel);
    }
    AdamArgs a{};
    a.m = state->m;
    a.v = state->v;
    a.m_scale = state->m_scale;
    a.v_scale = state->v_scale;
    a.b1 = (float)h.beta1;
    a.b1c = (float)(1.0 - h.beta1);
    a.b2 = (float)h.beta2;
    a.b2c = (float)(1.0 - h.beta2);
    a.eps = (float)h.eps;
    a.decay = (float)(1.0 - h.lr * h.weight_decay);
    a.rate = (float)(h.lr / (1.0 - std::pow(h.beta1, (double)h.step)));
    a.inv_root = (float)(1.0 / std::sqrt(1.0 - std::pow(h.beta2, (double)h.step)));
    a.grad_scale = (float)h.grad_scale;
    a.step_hash = (uint32_t)h.step * kRoot2 + (uint32_t)((uint64_t)h.step >> 32) * kRoot7;
    const bool dither = (double)h.step * (1.0 - h.beta1) > 2.0;
    hipStream_t st = static_cast<hipStream_t>(stream);
    for (int i = 0; i < count;) {
        int64_t chunks = 0;
        a.tensors = 0;
        for (; i < count && a.tensors < kMaxTensors; ++i) {
            const TridentAdamTensor& t = tensors[i];
            const int64_t c = (t.numel + kChunkElems - 1) / kChunkElems;
            if (c == 0) continue;
            if (chunks + c > 0x7fffffff) break;
            a.t[a.tensors++] = Entry{t.param, t.grad, t.numel, t.state_offset, (int32_t)chunks, (int16_t)t.dtype,
                                     (int16_t)t.grad_dtype};
            chunks += c;
        }
        if (chunks == 0) continue;
        with_bool(chunks * kChunkElems * 4 > kL2Bytes, [&](auto past) {
            constexpr bool P = decltype(past)::value;
            if (state->bits == 32) adamw_kernel<32, false, P><<<(unsigned)chunks, kBlock, 0, st>>>(a);
            else if (dither) adamw_kernel<8, true, P><<<(unsigned)chunks, kBlock, 0, st>>>(a);
            else adamw_kernel<8, false, P><<<(unsigned)chunks, kBlock, 0, st>>>(a);
        });
        const int rc = capi_check_launch("adamw_kernel");
        if (rc) return rc;
    }
    return TRIDENT_OK;
}

int trident_adamw_state_values(const TridentAdamState* state, float* m, float* v, void* stream) {
    if (!state || !m || !v || !state->m || !state->v || !state->m_scale || !state->v_scale)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "adamw_state_values: NULL pointer");
    if (state->bits != 8 || state->len < 0 || state->len % kStateBlock || !aligned4(state->m) || !aligned4(state->v))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "adamw_state_values: bits=%d len=%lld (whole blocks of %d)",
                         state->bits, (long long)state->len, kStateBlock);
    const int64_t quads = state->len / kPer, blocks = (quads + kBlock - 1) / kBlock;
    if (blocks > 0x7fffffff) return capi_fail(TRIDENT_ERR_UNSUPPORTED, "adamw_state_values: len=%lld", (long long)state->len);
    if (quads == 0) return TRIDENT_OK;
    with_bool(state->len * 8 > kL2Bytes, [&](auto past) {
        adam_values_kernel<decltype(past)::value><<<(unsigned)blocks, kBlock, 0, static_cast<hipStream_t>(stream)>>>(
            static_cast<const uint32_t*>(state->m), static_cast<const uint32_t*>(state->v), state->m_scale,
            state->v_scale, quads, m, v);
    });
    return capi_check_launch("adam_values_kernel");
}

}  // extern "C"
