// Products of matrices held in 8-bit floating point (e4m3), each row in blocks of 128 columns that
// share a scale:
//
//   x[r, k] ~ code[r, k] 2^(e[r, k / 128] - 127)       C = A B^T + bias,  A [M, K], B [N, K]
//
// The scale is a power of two, 2^s with the least s such that the block's largest value is at most
// 448 2^s (448: the largest e4m3 value), stored as e = s + 127 in one byte.  A power of two because
// the matrix core then applies it: v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 128 columns and takes
// one such byte per row and operand, so a block costs one instruction and no vector work.  e4m3 is
// itself a floating format, so against a scale of any value nothing is lost but the last part of the
// range of small codes.
//
// Sums: that instruction aligns each 8 neighbouring products to the largest of them and keeps 13 bits
// below it (measured with powers of two; between groups and onto the accumulator it adds in float32).
// A product is so off by 1.5e-5 of its size for normal inputs and 5e-5 for codes of all magnitudes,
// whatever K is: a hundredth of a bfloat16 rounding, but not a float32 sum.  So it is taken where the
// caller says so (fast_accum).  Otherwise the codes are turned into bfloat16 with the scale applied,
// which is exact, and multiplied by the bfloat16 instruction, which adds in float32, at half the rate.
#include <algorithm>

#include "encoder.hpp"

namespace trident {
namespace {

constexpr int kBlockK = 128;

inline int64_t blocks_of(int64_t K) { return (K + kBlockK - 1) / kBlockK; }
inline int64_t pitch_of(int64_t K) { return blocks_of(K) * kBlockK; }           // bytes of a row of codes
inline int64_t scale_pitch_of(int64_t K) { return (blocks_of(K) + 3) / 4 * 4; } // bytes of a row of scales

struct QuantArgs {
    const void* x;   // [rows, ld]
    uint8_t* codes;  // [rows, 128 kb]
    uint8_t* scales; // [rows, kbp]
    int64_t rows, ld;
    int K, kb, kbp;
};

constexpr int kQuantLanes = 16;  // lanes of a block of 128, eight values each

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
    if constexpr (sizeof(T) == 2) {
        load_vec(p, f);
    } else {
        float a[4], b[4];
        load_vec(p, a);
        load_vec(p + 4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = a[i];
            f[4 + i] = b[i];
        }
    }
}

// The scale byte of a block whose largest finite |value| is `top`.
__device__ __forceinline__ int scale_of(float top) {
    const uint32_t bits = __float_as_uint(top);
    const int e = (int)(bits >> 23) - 135 + ((bits & 0x7fffffu) > 0x600000u);  // 0x600000: 1.75 = 448 / 2^8
    return bits == 0 ? 127 : max(e, -126) + 127;
}

// Eight codes of x * 2^(127 - e); values that are not finite become NaN.
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], int e) {
    const float by = __uint_as_float((uint32_t)(254 - e) << 23);
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = fabsf(x[i]) < INFINITY ? x[i] * by : __uint_as_float(0x7fc00000u);
    uint2 w;
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    w.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], v, true);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
    w.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], v, true);
    return w;
}

// Bound by bytes: one read, one write, 16 lanes a block.
template <typename T>
__global__ __launch_bounds__(kBlock) void quantize_kernel(QuantArgs a) {
    const int64_t block = (int64_t)blockIdx.x * (kBlock / kQuantLanes) + threadIdx.x / kQuantLanes;
    if (block >= a.rows * a.kb) return;
    const int64_t row = block / a.kb;
    const int kb = (int)(block - row * a.kb), l = threadIdx.x % kQuantLanes;
    const int col = kb * kBlockK + l * 8;
    const T* x = static_cast<const T*>(a.x) + row * a.ld + col;
    float f[8];
    if (col + 8 <= a.K) {
        load8(x, f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = col + i < a.K ? (float)x[i] : 0.0f;
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[i]) < INFINITY ? fabsf(f[i]) : 0.0f);
#pragma unroll
    for (int o = kQuantLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
    const int e = scale_of(top);
    *reinterpret_cast<uint2*>(a.codes + row * ((int64_t)a.kb * kBlockK) + col) = codes_of(f, e);
    if (l == 0) {
        uint8_t* s = a.scales + row * a.kbp;
        s[kb] = (uint8_t)e;
        if (kb == a.kb - 1)
            for (int i = a.kb; i < a.kbp; ++i) s[i] = 127;
    }
}

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));

struct MatmulArgs {
    const uint8_t *a, *b;    // codes [M, pitch], [N, pitch]
    const uint8_t *sa, *sb;  // scales [M, spitch], [N, spitch]
    const void* bias;        // [N] or null
    void* out;               // [M, ldo]
    int64_t pitch, ldo;
    int M, N, kb, spitch, bias_f32;
};

__device__ __forceinline__ float scale_value(uint32_t e) {
    return __uint_as_float(e ? e << 23 : 0x00400000u);
}

// 32 codes as bfloat16, times the row's scale: exact, a code has four significant bits.
__device__ __forceinline__ void to_bf16(const i32x8& codes, float scale, bf16x8 (&out)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[2 * i + j], scale, false);
            const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[2 * i + j], scale, true);
            out[i][4 * j] = lo[0];
            out[i][4 * j + 1] = lo[1];
            out[i][4 * j + 2] = hi[0];
            out[i][4 * j + 3] = hi[1];
        }
}

constexpr int kTile = 128;

// A workgroup's 128 x 128 tile, 64 x 64 a wave.  The weight is the instruction's first operand, so a
// lane holds four neighbouring columns of a result row.
template <typename T, bool FAST>
__global__ __launch_bounds__(kBlock) void matmul_kernel(MatmulArgs g) {
    __shared__ __align__(16) uint8_t sA[kTile * kBlockK], sB[kTile * kBlockK];
    const int lane = lane_id(), wave = threadIdx.x / kWave, r = lane & 15, q = lane >> 4;
    const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    f32x4 acc[4][4] = {};
    for (int kb = 0; kb < g.kb; ++kb) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = i * kBlock + threadIdx.x, row = c / 8, slot = (c % 8) ^ (row & 7);
            const int64_t k = (int64_t)kb * kBlockK + slot * 16;
            const uint4 va = *reinterpret_cast<const uint4*>(g.a + min(m0 + row, g.M - 1) * g.pitch + k);
            const uint4 vb = *reinterpret_cast<const uint4*>(g.b + min(n0 + row, g.N - 1) * g.pitch + k);
            *reinterpret_cast<uint4*>(sA + c * 16) = va;
            *reinterpret_cast<uint4*>(sB + c * 16) = vb;
        }
        __syncthreads();
        i32x8 fa[4], fb[4];
        int ea[4], eb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int ra = wm + i * 16 + r, rb = wn + i * 16 + r;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x4 va = *reinterpret_cast<const u32x4*>(sA + ra * kBlockK + ((2 * q + h) ^ (ra & 7)) * 16);
                const u32x4 vb = *reinterpret_cast<const u32x4*>(sB + rb * kBlockK + ((2 * q + h) ^ (rb & 7)) * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    fa[i][4 * h + j] = (int)va[j];
                    fb[i][4 * h + j] = (int)vb[j];
                }
            }
            ea[i] = g.sa[(int64_t)min(m0 + ra, g.M - 1) * g.spitch + kb];
            eb[i] = g.sb[(int64_t)min(n0 + rb, g.N - 1) * g.spitch + kb];
        }
        if constexpr (!FAST) {
            bf16x8 ha[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                to_bf16(fa[i], scale_value(ea[i]), ha);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    bf16x8 hb[4];
                    to_bf16(fb[j], scale_value(eb[j]), hb);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hb[k], ha[k], acc[i][j], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa[i], acc[i][j], 0, 0, 0,
                                                                                 eb[j], 0, ea[i]);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = n0 + wn + j * 16 + q * 4;
        float bias[4] = {};
        if (g.bias)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < g.N)
                    bias[e] = g.bias_f32 ? static_cast<const float*>(g.bias)[n + e]
                                         : (float)static_cast<const T*>(g.bias)[n + e];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = m0 + wm + i * 16 + r;
            if (m >= g.M) continue;
            T* out = static_cast<T*>(g.out) + (int64_t)m * g.ldo + n;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < g.N) out[e] = (T)(acc[i][j][e] + bias[e]);
        }
    }
}

bool counts_ok(int64_t M, int64_t K) { return M >= 0 && M <= (1 << 30) && K >= 1 && K <= (1 << 30); }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

}  // namespace
}  // namespace trident

using namespace trident;

extern "C" {

int trident_fp8_quantize(const void* x, int32_t dtype, int64_t rows, int64_t K, int64_t ld_x, uint8_t* codes,
                         uint8_t* scales, void* stream) {
    if (!dtype_ok(dtype)) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "fp8_quantize: dtype=%d", dtype);
    if (!counts_ok(rows, K) || ld_x < K)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "fp8_quantize: bad sizes rows=%lld K=%lld ld=%lld",
                         (long long)rows, (long long)K, (long long)ld_x);
    if (rows == 0) return TRIDENT_OK;
    if (!x || !codes || !scales || !aligned16(codes))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "fp8_quantize: NULL pointer, or codes not 16-byte aligned");
    QuantArgs a{x, codes, scales, rows, ld_x, (int)K, (int)blocks_of(K), (int)scale_pitch_of(K)};
    constexpr int per = kBlock / kQuantLanes;
    const int64_t grid = (rows * a.kb + per - 1) / per;
    if (grid > 0x7fffffff)
        return capi_fail(TRIDENT_ERR_UNSUPPORTED, "fp8_quantize: rows * K = %lld is too large", (long long)(rows * K));
    with_dtype(dtype, [&](auto t) {
        quantize_kernel<decltype(t)><<<(unsigned)grid, kBlock, 0, static_cast<hipStream_t>(stream)>>>(a);
    });
    return capi_check_launch("quantize_kernel");
}

int trident_fp8_matmul(const uint8_t* a_codes, const uint8_t* a_scales, int64_t M, const uint8_t* b_codes,
                       const uint8_t* b_scales, int64_t N, int64_t K, const void* bias, int32_t bias_dtype, void* out,
                       int32_t dtype, int64_t ld_out, int32_t fast_accum, void* stream) {
    if (!dtype_ok(dtype) || (bias && bias_dtype != dtype && bias_dtype != TRIDENT_F32))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "fp8_matmul: dtype=%d bias_dtype=%d", dtype, bias_dtype);
    if (!counts_ok(M, K) || !counts_ok(N, K) || ld_out < N)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "fp8_matmul: bad sizes M=%lld N=%lld K=%lld ld=%lld",
                         (long long)M, (long long)N, (long long)K, (long long)ld_out);
    if (M == 0 || N == 0) return TRIDENT_OK;
    if (!a_codes || !a_scales || !b_codes || !b_scales || !out || !aligned16(a_codes) || !aligned16(b_codes))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "fp8_matmul: NULL pointer, or codes not 16-byte aligned");
    MatmulArgs g{a_codes, b_codes, a_scales, b_scales, bias, out, pitch_of(K), ld_out, (int)M, (int)N,
                 (int)blocks_of(K), (int)scale_pitch_of(K), bias_dtype == TRIDENT_F32};
    const int64_t gy = (M + kTile - 1) / kTile, gx = (N + kTile - 1) / kTile;
    if (gy > 65535) return capi_fail(TRIDENT_ERR_UNSUPPORTED, "fp8_matmul: M=%lld is too large", (long long)M);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const dim3 grid((unsigned)gx, (unsigned)gy);
        hipStream_t st = static_cast<hipStream_t>(stream);
        if (fast_accum) matmul_kernel<T, true><<<grid, kBlock, 0, st>>>(g);
        else matmul_kernel<T, false><<<grid, kBlock, 0, st>>>(g);
    });
    return capi_check_launch("matmul_kernel");
}

size_t trident_fp8_linear_workspace_bytes(int64_t M, int64_t K) {
    if (!counts_ok(M, K)) return 0;
    return up256((size_t)(M * pitch_of(K))) + up256((size_t)(M * scale_pitch_of(K)));
}

int trident_fp8_linear(const void* x, int32_t dtype, int64_t M, int64_t K, int64_t ld_x, const uint8_t* w_codes,
                       const uint8_t* w_scales, int64_t N, const void* bias, int32_t bias_dtype, void* out,
                       int64_t ld_out, int32_t fast_accum, void* workspace, size_t workspace_bytes, void* stream) {
    const size_t need = trident_fp8_linear_workspace_bytes(M, K);
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
        return capi_fail(TRIDENT_ERR_WORKSPACE_TOO_SMALL, "fp8_linear: workspace %zu < %zu bytes, or not 16-byte aligned",
                         workspace_bytes, need);
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    uint8_t* scales = codes + up256((size_t)(M * pitch_of(K)));
    const int rc = trident_fp8_quantize(x, dtype, M, K, ld_x, codes, scales, stream);
    if (rc) return rc;
    return trident_fp8_matmul(codes, scales, M, w_codes, w_scales, N, K, bias, bias_dtype, out, dtype, ld_out,
                              fast_accum, stream);
}

}  // extern "C"
