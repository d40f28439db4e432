// Layer norm of rows of D elements, and its backward pass.
//
//   m = mean(x)   r = 1 / sqrt(mean((x - m)^2) + eps)   h = (x - m) r   y = w h + b
//   a = w dy      dx = r (a - mean(a) - h mean(a h))    dw = sum_rows dy h   db = sum_rows dy
//
// The variance is that of the centred values (a second pass over registers, no further read), sums and
// statistics are float32.  The weight's gradient is summed without atomics: each workgroup keeps its
// rows' share in registers, and a second launch adds the workgroups' shares in order.
#include <algorithm>

#include "encoder.hpp"

namespace trident {
namespace {

struct NormArgs {
    const void* x;        // [rows, ldx]
    const void* dy;       // [rows, lddy]
    const void* weight;   // [D] or null: ones
    const void* bias;     // [D] or null: zeros
    void* y;              // [rows, ldy]
    void* dx;             // [rows, lddx]
    float* mean;          // [rows] or null
    float* rstd;
    float* part;          // [workgroups, 2, D]
    void *dw, *db;        // [D] or null: written by the only workgroup of a pass over few rows
    int64_t rows, ldx, lddy, ldy, lddx;
    int D, nv;            // nv: vectors of a row
    float eps, inv_D;
};

// The vectors of a row that this lane holds: G lanes share a row (a part of a wave, or whole waves), and
// lane l of them holds the vectors l + G c.  The last vector of a row ends with the row; its first `dup` elements are also the
// vector before's and count there.
template <int VEC, int NV, int G>
struct Columns {
    int col[NV], dup[NV];
    bool on[NV];
    __device__ __forceinline__ void init(const NormArgs& a, int l) {
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int v = l + G * c;
            on[c] = v < a.nv;
            col[c] = min(v * VEC, a.D - VEC);
            dup[c] = v * VEC - col[c];
        }
    }
};

template <typename T, int VEC, int NV>
struct Row {
    Vec<T, VEC> v[NV];
    template <int G>
    __device__ __forceinline__ void load(const T* __restrict__ p, const Columns<VEC, NV, G>& k) {
#pragma unroll
        for (int c = 0; c < NV; ++c)
            if (k.on[c]) v[c].load(p + k.col[c]);
    }
    // the values, zeros in a lane's vectors past the row
    template <int G>
    __device__ __forceinline__ void get(const Columns<VEC, NV, G>& k, float (&f)[NV][VEC]) const {
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            if (k.on[c]) v[c].get(f[c]);
            else
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[c][i] = 0.0f;
        }
    }
};

// Sum over the G lanes that share a row, the same in each; with more than a wave (G > 64) every thread of
// the workgroup calls it.
template <int G>
__device__ __forceinline__ float row_sum(float v, float* s_red) {
    if constexpr (G < kWave) {
        v = add_from<0xb1>(v);                        // the neighbour's
        v = add_from<0x4e>(v);                        // the other two's of four
        if constexpr (G >= 8) v = add_from<0x141>(v);  // eight lanes mirrored: the other four's
        if constexpr (G >= 16) v = add_from<0x140>(v);
        if constexpr (G >= 32) v += __shfl_xor(v, 16, kWave);
        return v;
    }
    v = wave_sum(v);
    if constexpr (G > kWave) {
        __syncthreads();
        if (lane_id() == 0) s_red[threadIdx.x / kWave] = v;
        __syncthreads();
        v = s_red[0];
#pragma unroll
        for (int i = 1; i < G / kWave; ++i) v += s_red[i];
    }
    return v;
}

// The row that this lane's group takes first, and the lane's number in it.
template <int G>
__device__ __forceinline__ int64_t first_row(int* lane) {
    *lane = threadIdx.x % G;
    if constexpr (G < kWave) return (int64_t)blockIdx.x * (kBlock / G) + threadIdx.x / G;
    return (int64_t)blockIdx.x * (kBlock / G) + __builtin_amdgcn_readfirstlane(threadIdx.x / G);
}

// Bound by bytes.  G lanes (a wave; a part of one for rows of up to 32 vectors; a workgroup of four for
// more than 256) take every so many rows and load the next one while they work on this one.  Narrow rows
// share a wave because its lanes are what it is fed by: 131,072 x 128 bfloat16 a wave a row 36.6 us, four
// rows a wave 13.8.  131,072 x 768 bfloat16 with the statistics: 75 us, 5.4 TB/s.
template <typename T, typename TW, int VEC, int NV, int G, bool PAST_L2>
__global__ __launch_bounds__(kBlock) void norm_kernel(NormArgs a) {
    __shared__ float s_red[kWavesPerBlock];
    const int64_t step = (int64_t)gridDim.x * (kBlock / G);
    int lane;
    int64_t row = first_row<G>(&lane);
    if (row >= a.rows) return;
    Columns<VEC, NV, G> k;
    k.init(a, lane);
    const T* X = static_cast<const T*>(a.x);
    Row<T, VEC, NV> now, next;
    Row<TW, VEC, NV> weight, bias;
    now.load(X + row * a.ldx, k);
    if (a.weight) weight.load(static_cast<const TW*>(a.weight), k);
    if (a.bias) bias.load(static_cast<const TW*>(a.bias), k);
    for (;;) {
        const bool more = row + step < a.rows;
        if (more) next.load(X + (row + step) * a.ldx, k);
        float x[NV][VEC];
        now.get(k, x);
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i >= k.dup[c]) s += x[c][i];
        const float mean = row_sum<G>(s, s_red) * a.inv_D;
        s = 0.0f;
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                x[c][i] -= mean;
                if (k.on[c] && i >= k.dup[c]) s += x[c][i] * x[c][i];
            }
        const float rstd = 1.0f / sqrtf(row_sum<G>(s, s_red) * a.inv_D + a.eps);
        T* y = static_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            if (!k.on[c]) continue;
            float w[VEC], b[VEC];
            if (a.weight) weight.v[c].get(w);
            if (a.bias) bias.v[c].get(b);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float v = x[c][i] * rstd;
                if (a.weight) v *= w[i];
                if (a.bias) v += b[i];
                x[c][i] = v;
            }
            put_vec<PAST_L2>(y + k.col[c], x[c]);
        }
        if (a.mean && lane == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        if (!more) return;
        now = next;
        row += step;
    }
}

// Rows too long for a workgroup's registers: the row is read three times (from L2 after the first).
template <typename T, typename TW>
__global__ __launch_bounds__(kBlock) void norm_long_kernel(NormArgs a) {
    __shared__ float s_red[kWavesPerBlock];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    T* y = static_cast<T*>(a.y) + row * a.ldy;
    float s = 0.0f;
    for (int d = threadIdx.x; d < a.D; d += kBlock) s += (float)x[d];
    const float mean = row_sum<kBlock>(s, s_red) * a.inv_D;
    s = 0.0f;
    for (int d = threadIdx.x; d < a.D; d += kBlock) s += ((float)x[d] - mean) * ((float)x[d] - mean);
    const float rstd = 1.0f / sqrtf(row_sum<kBlock>(s, s_red) * a.inv_D + a.eps);
    for (int d = threadIdx.x; d < a.D; d += kBlock) {
        float v = ((float)x[d] - mean) * rstd;
        if (a.weight) v *= (float)static_cast<const TW*>(a.weight)[d];
        if (a.bias) v += (float)static_cast<const TW*>(a.bias)[d];
        y[d] = (T)v;
    }
    if (a.mean && threadIdx.x == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
}

// Bound by bytes.  G lanes as above take every so many rows, the next one's loads ahead of this one's work:
// dx from the row's two means, and dy h and dy added to the columns' sums, which stay in registers until the
// last row.  131,072 x 768 bfloat16: 111 us, 5.4 TB/s.
template <typename T, typename TW, int VEC, int NV, int G, bool PAST_L2>
__global__ __launch_bounds__(kBlock) void norm_grad_kernel(NormArgs a) {
    extern __shared__ float s_part[];  // [kGroups][D], more groups than one only
    __shared__ float s_red[kWavesPerBlock];
    constexpr int kGroups = kBlock / G;
    const int64_t step = (int64_t)gridDim.x * kGroups;
    int lane;
    int64_t row = first_row<G>(&lane);
    Columns<VEC, NV, G> k;
    k.init(a, lane);
    float dw[NV][VEC] = {}, db[NV][VEC] = {};
    Row<TW, VEC, NV> weight;
    if (a.weight) weight.load(static_cast<const TW*>(a.weight), k);
    const T* X = static_cast<const T*>(a.x);
    const T* DY = static_cast<const T*>(a.dy);
    Row<T, VEC, NV> now_x, now_dy, next_x, next_dy;
    if (row < a.rows) {
        now_x.load(X + row * a.ldx, k);
        now_dy.load(DY + row * a.lddy, k);
    }
    for (; row < a.rows; row += step) {
        if (row + step < a.rows) {
            next_x.load(X + (row + step) * a.ldx, k);
            next_dy.load(DY + (row + step) * a.lddy, k);
        }
        const float mean = a.mean[row], rstd = a.rstd[row];
        float h[NV][VEC], g[NV][VEC];
        now_x.get(k, h);
        now_dy.get(k, g);
        float sa = 0.0f, sh = 0.0f;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            float w[VEC];
            if (a.weight) weight.v[c].get(w);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                h[c][i] = (h[c][i] - mean) * rstd;
                const float dy = g[c][i];
                dw[c][i] += dy * h[c][i];
                db[c][i] += dy;
                if (a.weight) g[c][i] = dy * w[i];
                if (k.on[c] && i >= k.dup[c]) {
                    sa += g[c][i];
                    sh += g[c][i] * h[c][i];
                }
            }
        }
        sa = row_sum<G>(sa, s_red) * a.inv_D;
        sh = row_sum<G>(sh, s_red) * a.inv_D;
        T* dx = static_cast<T*>(a.dx) + row * a.lddx;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            if (!k.on[c]) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) g[c][i] = rstd * (g[c][i] - sa - h[c][i] * sh);
            put_vec<PAST_L2>(dx + k.col[c], g[c]);
        }
        now_x = next_x;
        now_dy = next_dy;
    }
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.D;
    if constexpr (kGroups > 1) {
        const bool only = gridDim.x == 1;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            TW* out = static_cast<TW*>(which ? a.db : a.dw);
            __syncthreads();
#pragma unroll
            for (int c = 0; c < NV; ++c)
                if (k.on[c])
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        s_part[threadIdx.x / G * a.D + k.col[c] + i] = which ? db[c][i] : dw[c][i];
            __syncthreads();
            for (int d = threadIdx.x; d < a.D; d += kBlock) {
                float s = s_part[d];
#pragma unroll
                for (int i = 1; i < kGroups; ++i) s += s_part[i * a.D + d];
                if (!only) part[which * a.D + d] = s;
                else if (out) out[d] = (TW)s;
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < NV; ++c)
            if (k.on[c])
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    part[k.col[c] + i] = dw[c][i];
                    part[a.D + k.col[c] + i] = db[c][i];
                }
    }
}

template <typename T, typename TW>
__global__ __launch_bounds__(kBlock) void norm_grad_long_kernel(NormArgs a) {
    __shared__ float s_red[kWavesPerBlock];
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.D;
    if ((int64_t)blockIdx.x >= a.rows)  // no row: a share of zeros
        for (int d = threadIdx.x; d < 2 * a.D; d += kBlock) part[d] = 0.0f;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.ldx;
        const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
        T* dx = static_cast<T*>(a.dx) + row * a.lddx;
        const float mean = a.mean[row], rstd = a.rstd[row];
        const bool first = row == (int64_t)blockIdx.x;
        float sa = 0.0f, sh = 0.0f;
        for (int d = threadIdx.x; d < a.D; d += kBlock) {
            const float h = ((float)x[d] - mean) * rstd, g = (float)dy[d];
            const float v = a.weight ? g * (float)static_cast<const TW*>(a.weight)[d] : g;
            sa += v;
            sh += v * h;
            // a column is always this thread's: its sums need no lock
            part[d] = (first ? 0.0f : part[d]) + g * h;
            part[a.D + d] = (first ? 0.0f : part[a.D + d]) + g;
        }
        sa = row_sum<kBlock>(sa, s_red) * a.inv_D;
        sh = row_sum<kBlock>(sh, s_red) * a.inv_D;
        for (int d = threadIdx.x; d < a.D; d += kBlock) {
            const float h = ((float)x[d] - mean) * rstd, g = (float)dy[d];
            const float v = a.weight ? g * (float)static_cast<const TW*>(a.weight)[d] : g;
            dx[d] = (T)(rstd * (v - sa - h * sh));
        }
    }
}

constexpr int kJoinBlock = 1024;

// dw and db from the workgroups' shares: 64 columns a workgroup, its 16 waves each every 16th share,
// then the waves' sums in order.  512 shares of 768 columns: 4.7 us, a launch's time.
template <typename TW>
__global__ __launch_bounds__(kJoinBlock) void norm_join_kernel(const float* __restrict__ part, int parts, int D,
                                                               TW* __restrict__ dw, TW* __restrict__ db) {
    __shared__ float s_sum[kJoinBlock / kWave][kWave];
    const int wave = threadIdx.x / kWave;
    const int64_t col = (int64_t)blockIdx.x * kWave + lane_id();
    float s = 0.0f;
    if (col < 2 * (int64_t)D) {
#pragma unroll 8
        for (int p = wave; p < parts; p += kJoinBlock / kWave) s += part[(int64_t)p * 2 * D + col];
    }
    s_sum[wave][lane_id()] = s;
    __syncthreads();
    if (wave == 0 && col < 2 * (int64_t)D) {
        for (int i = 1; i < kJoinBlock / kWave; ++i) s += s_sum[i][lane_id()];
        if (col < D) {
            if (dw) dw[col] = (TW)s;
        } else if (db) {
            db[col - D] = (TW)s;
        }
    }
}

// Calls f<VEC, NV, G> for rows of D elements of type T; false if they are too long for registers.
template <typename T, typename F>
bool with_shape(int64_t D, F&& f) {
    constexpr int V = kVec<T>;
    const int64_t nv = D < V ? D : (D + V - 1) / V;
    const auto go = [&](auto vec, auto n, auto g) { f(vec, n, g); return true; };
    const std::integral_constant<int, 1> i1;
    const std::integral_constant<int, 2> i2;
    const std::integral_constant<int, 3> i3;
    const std::integral_constant<int, 4> i4;
    const std::integral_constant<int, 8> i8;
    const std::integral_constant<int, 16> i16;
    const std::integral_constant<int, 32> i32;
    const std::integral_constant<int, kWave> wave;
    const std::integral_constant<int, kBlock> block;
    const std::integral_constant<int, V> v;
    if (D < V) return go(i1, i1, i8);
    if (nv <= 4) return go(v, i1, i4);
    if (nv <= 16) return go(v, i1, i16);
    if (nv <= 32) return go(v, i1, i32);
    if (nv <= 64) return go(v, i1, wave);
    if (nv <= 128) return go(v, i2, wave);
    if (nv <= 192) return go(v, i3, wave);
    if (nv <= 256) return go(v, i4, wave);
    if (nv <= 512) return go(v, i2, block);
    if (nv <= 1024) return go(v, i4, block);
    return false;
}

// Workgroups of a forward pass, of which 256 CUs hold 2,048 at a time: more of them, with fewer rows each,
// end more evenly, until the next row's loads ahead are lost.  float32 rows are twice as long: 131,072 x 768,
// 2,048, 4,096, 8,192, 16,384 and 32,768 workgroups 147, 145, 139, 136, 134 us.  For 16 bits no number is the
// best: 2,048, 4,096 and 8,192, bfloat16, 131,072 x 768 77, 75.5, 74.5 us; x 960 81.6, 78, 73.5; x 256 23.9,
// 23.1, 21.5; x 128 13.1, 13.0, 13.9; 65,536 x 512 23.9, 23.0, 23.1; 32,768 x 1,024 23.2, 21.9, 23.2; float16
// 131,072 x 768 68.6, 69.0, 72.4; 32,768 x 1,024 23.1, 23.1, 25.5: 4,096 loses 7% at most, 8,192 11.
template <typename T>
constexpr int kNormBlocks = sizeof(T) == 4 ? 16384 : 4096;

// Workgroups of a backward pass, each of which leaves a share of the weight's gradient: enough waves to
// cover the loads' latency, and few shares.  131,072 x 768 bfloat16, 256, 512 and 1,024: 194, 117 and 134 us;
// 8,192 x 4,096 50, 48 and 58; float32 218, 221 and 236.
constexpr int kGradBlocks = 512;

// Few rows are one workgroup's, whose share is the gradient, so there is no second launch: 32 x 768
// bfloat16 13.7 us for 16.3, 64 x 768 18.8 for 16.2, 32 x 2,048 20.3 for 16.3.
constexpr int kFewRows = 32, kFewElements = 32 * 1024;

int64_t grad_parts(int64_t rows, int64_t D, int64_t per) {
    return rows <= kFewRows && rows * D <= kFewElements ? 1 : std::min<int64_t>(kGradBlocks, (rows + per - 1) / per);
}

bool sizes_ok(int64_t rows, int64_t D) { return rows >= 0 && rows <= 0x7fffffff && D >= 1 && D <= (1 << 29); }

}  // namespace
}  // namespace trident

using namespace trident;

extern "C" {

int trident_layer_norm(const void* x, int32_t dtype, int64_t rows, int64_t D, int64_t ld_x, const void* weight,
                       const void* bias, int32_t weight_dtype, double eps, void* y, int64_t ld_y, float* mean,
                       float* rstd, void* stream) {
    if (!dtype_ok(dtype) || (weight_dtype != dtype && weight_dtype != TRIDENT_F32))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "layer_norm: dtype=%d weight_dtype=%d", dtype, weight_dtype);
    if (!sizes_ok(rows, D) || ld_x < D || ld_y < D || !(eps >= 0.0))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "layer_norm: bad sizes rows=%lld D=%lld ld=%lld, %lld eps=%g",
                         (long long)rows, (long long)D, (long long)ld_x, (long long)ld_y, eps);
    if (rows == 0) return TRIDENT_OK;
    if (!x || !y || !mean != !rstd) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "layer_norm: NULL pointer");
    hipStream_t st = static_cast<hipStream_t>(stream);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        with_dtype(weight_dtype, [&](auto u) {
            using TW = decltype(u);
            if constexpr (std::is_same<T, TW>::value || std::is_same<TW, float>::value) {
                NormArgs a{x, nullptr, weight, bias, y, nullptr, mean, rstd, nullptr, nullptr, nullptr, rows, ld_x, 0, ld_y,
                           0, (int)D, 0, (float)eps, (float)(1.0 / (double)D)};
                const bool ok = with_shape<T>(D, [&](auto vec, auto nv, auto g) {
                    constexpr int VEC = decltype(vec)::value, NV = decltype(nv)::value, G = decltype(g)::value;
                    a.nv = (int)((D + VEC - 1) / VEC);
                    const int64_t per = kBlock / G;
                    const unsigned grid = (unsigned)std::min<int64_t>(kNormBlocks<T>, (rows + per - 1) / per);
                    with_bool(rows * D * (int64_t)sizeof(T) > kL2Bytes, [&](auto past) {
                        norm_kernel<T, TW, VEC, NV, G, decltype(past)::value><<<grid, kBlock, 0, st>>>(a);
                    });
                });
                if (!ok) norm_long_kernel<T, TW><<<(unsigned)rows, kBlock, 0, st>>>(a);
            }
        });
    });
    return capi_check_launch("norm_kernel");
}

size_t trident_layer_norm_grad_workspace_bytes(int64_t rows, int64_t D) {
    if (!sizes_ok(rows, D)) return 0;
    return (size_t)grad_parts(rows, D, kWavesPerBlock) * 2 * (size_t)D * sizeof(float);
}

int trident_layer_norm_grad(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int32_t dtype, int64_t rows,
                            int64_t D, const void* weight, int32_t weight_dtype, const float* mean, const float* rstd,
                            void* dx, int64_t ld_dx, void* dweight, void* dbias, void* workspace,
                            size_t workspace_bytes, void* stream) {
    if (!dtype_ok(dtype) || (weight_dtype != dtype && weight_dtype != TRIDENT_F32))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "layer_norm_grad: dtype=%d weight_dtype=%d", dtype,
                         weight_dtype);
    if (!sizes_ok(rows, D) || ld_x < D || ld_dy < D || ld_dx < D)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT,
                         "layer_norm_grad: bad sizes rows=%lld D=%lld ld=%lld, %lld, %lld", (long long)rows,
                         (long long)D, (long long)ld_dy, (long long)ld_x, (long long)ld_dx);
    if (rows > 0 && (!dy || !x || !mean || !rstd || !dx))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "layer_norm_grad: NULL pointer");
    const size_t need = trident_layer_norm_grad_workspace_bytes(rows, D);
    if (!workspace || workspace_bytes < need)
        return capi_fail(TRIDENT_ERR_WORKSPACE_TOO_SMALL, "layer_norm_grad: workspace %zu < %zu bytes",
                         workspace_bytes, need);
    hipStream_t st = static_cast<hipStream_t>(stream);
    int rc = TRIDENT_OK;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        with_dtype(weight_dtype, [&](auto u) {
            using TW = decltype(u);
            if constexpr (std::is_same<T, TW>::value || std::is_same<TW, float>::value) {
                NormArgs a{x, dy, weight, nullptr, nullptr, dx, const_cast<float*>(mean), const_cast<float*>(rstd),
                           static_cast<float*>(workspace), dweight, dbias, rows, ld_x, ld_dy, 0, ld_dx, (int)D, 0,
                           0.0f, (float)(1.0 / (double)D)};
                // with no rows every share is zero: the kernels' loops are empty
                bool joined = !dweight && !dbias;
                int64_t parts = grad_parts(rows, D, kWavesPerBlock);
                const bool ok = with_shape<T>(D, [&](auto vec, auto nv, auto g) {
                    constexpr int VEC = decltype(vec)::value, NV = decltype(nv)::value, G = decltype(g)::value;
                    a.nv = (int)((D + VEC - 1) / VEC);
                    constexpr int groups = kBlock / G;
                    const size_t lds = groups > 1 ? groups * (size_t)D * sizeof(float) : 0;
                    parts = grad_parts(rows, D, std::max(groups, kWavesPerBlock));
                    with_bool(rows * D * (int64_t)sizeof(T) > kL2Bytes, [&](auto past) {
                        norm_grad_kernel<T, TW, VEC, NV, G, decltype(past)::value>
                            <<<(unsigned)parts, kBlock, lds, st>>>(a);
                    });
                    joined = joined || (groups > 1 && parts == 1);
                });
                if (!ok) norm_grad_long_kernel<T, TW><<<(unsigned)parts, kBlock, 0, st>>>(a);
                if ((rc = capi_check_launch("norm_grad_kernel")) || joined) return;
                norm_join_kernel<TW><<<(unsigned)((2 * D + kWave - 1) / kWave), kJoinBlock, 0, st>>>(
                    static_cast<const float*>(workspace), (int)parts, (int)D, static_cast<TW*>(dweight),
                    static_cast<TW*>(dbias));
                rc = capi_check_launch("norm_join_kernel");
            }
        });
    });
    return rc;
}

}  // extern "C"
