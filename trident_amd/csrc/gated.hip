// The gated half of a feed-forward block and its backward pass,
//
//   g = x Wg^T,   u = x Wu^T,   h = act(g) u
//   dg = dh u act'(g),   du = dh act(g),   dx = dg Wg + du Wu,   dWg = dg^T x,   dWu = du^T x
//
// with x [M, K], Wg and Wu [N, K], all row-major.  One kernel of tiles computes every product: an operand's
// tile is read by rows where the summed axis is its columns (x, Wg, Wu in the forward pass; dg, du in dx) and
// by columns where it is its rows (Wg, Wu in dx; all of dWg, dWu).  Sums are float32, and g and u are kept so
// for the backward pass: rounded to 16 bits they would add as much error to dg and du as these two's own
// rounding for their products does, and as much again to the gradients (bfloat16: 3.1e-3 rms with them rounded,
// 2.4e-3 without, of which the results' own rounding is 1.7e-3).
//
// Many rows are bound by the matrix unit and by LDS, that feeds it, and by the start and end of a tile, which
// nothing covers where a CU holds one: 16,384 x 1,024 by 2 x 4,096, bfloat16, 298 to 309 us on three cards (890 to
// 922 TFLOP/s; 275 GFLOP at the rate of a large square product take 196, a library's product alone of this shape
// 272), 340 to 360 where gate and up are kept; its gradients 240 us of dx and 280 of both weights'.  Few rows are
// bound by the weights' bytes.
#include <algorithm>

#include "mfma.hpp"

namespace trident {
namespace {

enum Activation { kSilu = TRIDENT_SILU, kGelu = TRIDENT_GELU, kGeluTanh = TRIDENT_GELU_TANH };

// act(g), and act'(g) where SLOPE.  By the vector unit's own exp2 and reciprocal, off by 1 ulp each: a tile of
// a short sum is not much longer than its activations (expf, erfcf and divisions are several times as many
// instructions).
template <bool SLOPE>
__device__ __forceinline__ void activate(int kind, float g, float* value, float* slope) {
    constexpr float kLog2e = 1.4426950408889634f;
    const float g2 = g * g;
    if (kind == kGelu) {
        // g Phi(g), Phi(-x) = erfc(x / sqrt 2) / 2.  For x >= 0, erfc(x) = t q(t) exp(-x^2) with t = 1 / (1 + x
        // / 2) and q a polynomial fitted to exp(x^2) erfc(x) / t, off by 5e-8 relative up to x = 14, so small
        // values keep their digits.
        const float x = fabsf(g) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.5f, x, 1.0f));
        constexpr float q[] = {0.282084331f, 0.282412099f, 0.242835108f, 0.203752563f, -0.0291486356f, 0.281733461f, -0.490406549f, 0.286124062f, -0.0593864829f};
        float v = q[8];
#pragma unroll
        for (int i = 7; i >= 0; --i) v = __builtin_fmaf(v, t, q[i]);
        const float e = __builtin_amdgcn_exp2f(g2 * (-0.5f * kLog2e));
        const float tail = 0.5f * (v * t) * e, p = g < 0.0f ? tail : 1.0f - tail;
        *value = g * p;
        if constexpr (SLOPE) *slope = __builtin_fmaf(g * 0.39894228040143268f, e, p);
        return;
    }
    // both others are g times a logistic: of g, or of 2 sqrt(2 / pi) (g + 0.044715 g^3)
    const float z = kind == kSilu ? g : 1.5957691216057308f * g * __builtin_fmaf(0.044715f, g2, 1.0f);
    const float p = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
    *value = g * p;
    if constexpr (SLOPE) {
        // dz grows as g^2, and from g = 1e13 on g dz passes float32 where the logistic's own slope p (1 - p) is
        // zero: so that is multiplied first, and g^2 stops at 1e4, where it is zero for long.  1 - p is its own
        // quotient: no digits are lost where p is near 1.
        const float dz = kind == kSilu ? 1.0f : 1.5957691216057308f * __builtin_fmaf(3 * 0.044715f, fminf(g2, 1e4f), 1.0f);
        const float dp = p * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(kLog2e * z));
        *slope = __builtin_fmaf(g * dp, dz, p);
    }
}

// ------------------------------------------------------------------------------------------------
// products

// An operand: rows of `pitch` bytes.  By rows, its rows are the tile's and its columns are summed over; by
// columns the other way round.
struct Operand {
    const uint8_t* p;
    int64_t pitch;
};

struct ProductArgs {
    // out[m, n] = sum over k of second[m, k] first[n, k]; two sums one after another where there are second
    // operands of both (dx), or first ones whose sums are kept apart (gate and up)
    Operand first[2], second[2];
    void* out[3];
    int64_t ldo;       // elements
    int M, N, K;       // rows and columns of the result, length of a sum
    int parts;         // sums one after another
    int tiles_m, tiles_n, activation;
    int shares;        // SPLIT: workgroups that share a tile's sum
    float* part;       // [shares][sums of a place: gate and up, or the results][M, N]
    const float* back; // kScaled: what the sums are multiplied by
};

// The second operand of the backward products, dg and du, is held in float16 times a power of two (slope_kernel).
template <typename T>
constexpr bool kScaled = std::is_same<T, f16_t>::value;

// One of a grid's tiles in an order that keeps neighbours on one XCD: workgroups go to the eight XCDs, each
// with its own L2, in turn, so each takes a contiguous eighth, in bands of 8 tile rows.
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int* tm, int* tn) {
    constexpr int kBand = 8;
    const int total = tiles_m * tiles_n, each = total / 8, more = total % 8;
    const int xcd = id % 8, t = xcd * each + min(xcd, more) + id / 8;
    const int first = t / (kBand * tiles_n) * kBand, rows = min(kBand, tiles_m - first);
    const int in = t - first * tiles_n;
    *tm = first + in % rows;
    *tn = in / rows;
}

// How the first and the second operand are read.
enum Reading { kRowsRows, kColumnsRows, kColumnsColumns };

// Of the summed axis, bytes of a stage in LDS; and the stages there at a time.  Operands that are both read by
// rows come in whole lines of 128 bytes, two stages; else four of 64 (forward pass of 16,384 x 1,024 by 2 x
// 4,096 bfloat16 307 us, 315 by four of 64; its dx 252 by four, 268 by two).
constexpr int stage_row(int read) { return read == kRowsRows ? 128 : 64; }
constexpr int stages(int read) { return read == kRowsRows ? 2 : 4; }

// A stage of `ROWS` operand rows (by columns: columns) and ROW bytes of the summed axis, and its loads.
template <typename T, bool COLUMNS, int ROWS, int ROW, int WAVES>
struct OperandTile {
    static constexpr int kStep = ROW / (int)sizeof(T), kPitch = COLUMNS ? ROWS * (int)sizeof(T) : ROW;
    static constexpr int kBytes = ROWS * ROW, kLoads = kBytes / 1024 / WAVES;
    static_assert(kBytes % (1024 * WAVES) == 0, "whole loads");
    using L = Tile<T, kPitch>;
    const uint8_t* base;
    int64_t pitch;
    int length;          // of the summed axis
    uint32_t at[kLoads]; // of this lane's piece in the first step

    // rows `first` on of `limit`; those past it are zeros
    __device__ __forceinline__ void start(const Operand& o, int first, int limit, int K, int wave) {
        pitch = o.pitch;
        length = K;
        base = o.p + (COLUMNS ? (int64_t)first * sizeof(T) : first * o.pitch);
        const int lane = lane_id(), in = lane / L::kPieces, slot = lane % L::kPieces;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = (i * WAVES + wave) * L::kRowsAtOnce + in, piece = slot ^ L::exchange(r);
            const bool there = COLUMNS ? first + piece * (16 / (int)sizeof(T)) < limit : first + r < limit;
            at[i] = there ? (uint32_t)r * (uint32_t)pitch + piece * 16 : kPastBuffer;
        }
    }
    __device__ __forceinline__ void fetch(lds_bytes to, int step, int wave) const {
        const int k = step * kStep, left = length - k;
        if constexpr (COLUMNS) {
            const __amdgpu_buffer_rsrc_t buf =
                buffer_of(base + k * pitch, (uint32_t)min(left, kStep) * (uint32_t)pitch);
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (lds_ptr)(to + (i * WAVES + wave) * 1024), 16, at[i], 0, 0, 0);
        } else {
            const __amdgpu_buffer_rsrc_t buf = buffer_of(base + (int64_t)step * ROW, 0x7fffffffu);
            const int lane = lane_id(), slot = lane % L::kPieces;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                uint32_t from = at[i];
                if (left < kStep) {  // columns past the last one are zeros
                    const int r = (i * WAVES + wave) * L::kRowsAtOnce + lane / L::kPieces;
                    if ((slot ^ L::exchange(r)) * (16 / (int)sizeof(T)) >= left) from = kPastBuffer;
                }
                __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (lds_ptr)(to + (i * WAVES + wave) * 1024), 16, from, 0, 0, 0);
            }
        }
    }
    // eight steps 16 s + 8 half .. of this lane's row (column) `row`
    static __device__ __forceinline__ frag<T> read(lds_bytes tile, int row, int s) {
        if constexpr (COLUMNS) return L::col_frag_in_order(tile, 16 * s, row);
        else return L::row_frag(tile, row + (lane_id() & 31), s);
    }
};

// A workgroup of WM x WN waves computes WM MT x WN NT blocks of 32 x 32, a wave MT x NT.  Stages of both
// operands go straight from memory to LDS, ahead of the one that is multiplied.  The first operand gives the
// result's columns, so a lane holds four neighbours of a row.
//
// GATED: the first operand's tile is half gate, half up, and each wave's blocks too, so that a lane holds both
// sums of the same places: out[0] = act(g) u, and g and u themselves where KEEP.
//
// SPLIT: a workgroup takes a share of the stages and writes its sums as they are, for the join.
template <typename T, int READ, int WM, int WN, int MT, int NT, bool GATED, bool KEEP, bool SPLIT>
__device__ __forceinline__ void product(const ProductArgs& a) {
    constexpr int kWaves = WM * WN, BM = WM * MT * 32, BN = WN * NT * 32;
    constexpr int BR = GATED ? BN / 2 : BN;  // the result's columns
    constexpr int kRow = stage_row(READ), kStep = kRow / (int)sizeof(T), kStages = stages(READ);
    using First = OperandTile<T, READ != kRowsRows, BR, kRow, kWaves>;
    using Second = OperandTile<T, READ == kColumnsColumns, BM, kRow, kWaves>;
    constexpr int kFirst = BN * kRow, kStage = kFirst + Second::kBytes, G = kStep / 16;
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane >> 5;
    int tm, tn;
    tile_of(blockIdx.x, a.tiles_m, a.tiles_n, &tm, &tn);
    const int m0 = tm * BM, n0 = tn * BR, z = blockIdx.y;  // z: one of two results of their own (dWg, dWu)
    const int wm = wave / WN * MT * 32, wn = wave % WN * NT * 32;

    First first[GATED ? 2 : 1];
    Second second;
    const auto begin = [&](int part) {
        first[0].start(a.first[part], n0, a.N, a.K, wave);
        if constexpr (GATED) first[1].start(a.first[1], n0, a.N, a.K, wave);
        second.start(a.second[part + z], m0, a.M, a.K, wave);
    };
    const int each = (a.K + kStep - 1) / kStep, total = each * a.parts;
    const int from0 = SPLIT ? total * (int)blockIdx.z / a.shares : 0;
    const int steps = SPLIT ? total * ((int)blockIdx.z + 1) / a.shares - from0 : total;
    const lds_bytes base = (lds_bytes)(lds_ptr)lds;
    const auto fetch = [&](int n, lds_bytes to) {
        if (n >= steps) return;
        const int at = n + from0, step = at < each ? at : at - each;
        if (at == each && n > 0) begin(1);
        first[0].fetch(to, step, wave);
        if constexpr (GATED) first[1].fetch(to + kFirst / 2, step, wave);
        second.fetch(to + kFirst, step, wave);
    };
    begin(from0 >= each ? 1 : 0);
    constexpr int kAhead = READ == kRowsRows ? 2 : kStages - 1;  // stages loaded before the first is read
#pragma unroll
    for (int n = 0; n < kAhead; ++n) fetch(n, base + n * kStage);

    constexpr int kSets = READ == kRowsRows ? G : 2;  // groups held
    f32x16 acc[MT][NT] = {};
    frag<T> f1[kSets][NT], f2[kSets][MT];
    const auto read = [&](lds_bytes from, int g, int set) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            if constexpr (GATED) {  // the wave's first half of blocks from the gate's tile
                f1[set][j] = First::read(from + (j < NT / 2 ? 0 : kFirst / 2), wn / 2 + j % (NT / 2) * 32, g);
            } else {
                f1[set][j] = First::read(from, wn + j * 32, g);
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) f2[set][i] = Second::read(from + kFirst, wm + i * 32, g);
    };
    const auto multiply = [&](int set) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = mma<T>(f1[set][j], f2[set][i], acc[i][j]);
    };
    constexpr int kFlight = (GATED ? 2 : 1) * First::kLoads + Second::kLoads;  // a wave's loads of one stage
    if constexpr (READ == kRowsRows) {
        // A stage's next loads are issued as soon as every wave holds its part of it in registers, halfway
        // through its products, so that they have a stage and a half to arrive.
        for (int n = 0; n < steps; ++n) {
            if (n + 1 < steps) wait_and_meet<kFlight>();
            else wait_and_meet<0>();
            const lds_bytes from = base + n % 2 * kStage;
#pragma unroll
            for (int g = 0; g < G; ++g) read(from, g, g);
#pragma unroll
            for (int g = 0; g < G / 2; ++g) multiply(g);
            if constexpr (sizeof(T) == 2) {
                // the first half's reads, the second half's among the first half's products
                constexpr int kReads = G / 2 * (NT + MT), kProducts = G / 2 * MT * NT;
                constexpr int kEach = (kReads + kProducts - 1) / kProducts;
                __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
#pragma unroll
                for (int i = 0; i < kProducts; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);
                }
            }
            // the first half's products stay before the wait (the compiler would sink them past it)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) asm volatile("" : "+v"(acc[i][j]));
            meet();  // every wave has read the stage
            fetch(n + 2, from);
#pragma unroll
            for (int g = G / 2; g < G; ++g) multiply(g);
        }
    } else {
        // One barrier a stage, past which it has arrived and the one before is no longer read; a group's blocks
        // are read while the group before is multiplied.  What is loaded and what is read between two barriers
        // lie in different stages, which __restrict says: else the compiler waits for every load before a
        // transposing read.
        const auto body = [&](int n, lds_bytes __restrict from, lds_bytes __restrict to, int of, bool before) {
            fetch(n + kStages - 1, to);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int set = (of + g) % 2;
                read(from, g, set);
                if (g > 0 || before) multiply(1 - set);
            }
        };
        const auto arrive = [&](int n) {
            if (n + 2 < steps) wait_and_meet<2 * kFlight>();
            else if (n + 1 < steps) wait_and_meet<kFlight>();
            else wait_and_meet<0>();
        };
        const auto stage = [&](int n) { return base + n % kStages * kStage; };
        arrive(0);
        body(0, stage(0), stage(kStages - 1), 0, false);
        int n = 1;
        if constexpr (G == 2) {
            for (; n < steps; ++n) {
                arrive(n);
                body(n, stage(n), stage(n + kStages - 1), 0, true);
            }
            multiply(1);
        } else {
            static_assert(G == 1, "groups of a stage");
            for (; n + 1 < steps; n += 2) {
                arrive(n);
                body(n, stage(n), stage(n + kStages - 1), 1, true);
                arrive(n + 1);
                body(n + 1, stage(n + 1), stage(n + kStages), 0, true);
            }
            if (n < steps) {
                arrive(n);
                body(n, stage(n), stage(n + kStages - 1), 1, true);
                multiply(1);
            } else {
                multiply(0);
            }
        }
    }
    // Results go through LDS, 32 rows of a wave at a time, so that whole lines are written.
    wait_and_meet<0>();
    constexpr int kBlocks = GATED ? NT / 2 : NT, kCols = kBlocks * 32;
    constexpr int kRegion = 32 * (kCols * (KEEP || SPLIT ? 4 : (int)sizeof(T)) + 16);  // a wave's, for the widest results
    static_assert(kWaves * kRegion <= kStages * kStage, "the results fit where the operands were");
    uint8_t* mine = lds + wave * kRegion;
    const auto put = [&](int i, auto* out, auto&& value) {
        using O = std::remove_pointer_t<decltype(out)>;
        constexpr int kPitch = kCols * (int)sizeof(O) + 16;
        constexpr int kPer = 16 / (int)sizeof(O), kRowPieces = kCols / kPer, kRowsAtOnce = kWave / kRowPieces;
        const int col = n0 + (GATED ? wn / 2 : wn) + lane % kRowPieces * kPer, left = a.N - col;
        wave_sync();
#pragma unroll
        for (int j = 0; j < kBlocks; ++j)
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = value(j, 4 * p + e);
                store_vec(reinterpret_cast<O*>(mine + (lane & 31) * kPitch) + j * 32 + p * 8 + half * 4, v);
            }
        wave_sync();
#pragma unroll
        for (int k = 0; k < 32; k += kRowsAtOnce) {
            const int row = k + lane / kRowPieces, m = m0 + wm + i * 32 + row;
            if (m >= a.M || left <= 0) continue;
            const uint8_t* from = mine + row * kPitch + lane % kRowPieces * 16;
            O* to = out + m * a.ldo + col;
            if (left >= kPer) {
                __builtin_memcpy(to, from, 16);
            } else {
                for (int e = 0; e < left; ++e) to[e] = reinterpret_cast<const O*>(from)[e];
            }
        }
    };
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        if constexpr (SPLIT) {
            const int64_t plane = (int64_t)a.M * a.ldo;
            float* to = a.part + (blockIdx.z * (GATED ? 2 : gridDim.y) + z) * plane;
            put(i, to, [&](int j, int e) { return acc[i][j][e]; });
            if constexpr (GATED) put(i, to + plane, [&](int j, int e) { return acc[i][j + kBlocks][e]; });
        } else if constexpr (GATED) {
            put(i, static_cast<T*>(a.out[0]), [&](int j, int e) {
                float v;
                activate<false>(a.activation, acc[i][j][e], &v, nullptr);
                return v * acc[i][j + kBlocks][e];
            });
            if constexpr (KEEP) {
                put(i, static_cast<float*>(a.out[1]), [&](int j, int e) { return acc[i][j][e]; });
                put(i, static_cast<float*>(a.out[2]), [&](int j, int e) { return acc[i][j + kBlocks][e]; });
            }
        } else {
            const float by = kScaled<T> ? *a.back : 1.0f;
            put(i, static_cast<T*>(a.out[z]), [&](int j, int e) { return kScaled<T> ? acc[i][j][e] * by : acc[i][j][e]; });
        }
    }
}

// (A function of its own: with the body in the kernel template the compiler leaves out the host's half of some
// instantiations.)
template <typename T, int READ, int WM, int WN, int MT, int NT, bool GATED, bool KEEP, bool SPLIT>
__global__ __launch_bounds__(WM* WN* kWave) void product_kernel(ProductArgs a) {
    product<T, READ, WM, WN, MT, NT, GATED, KEEP, SPLIT>(a);
}

// The sums of SPLIT workgroups, in order: four places a thread, or one where rows do not hold whole fours.
template <typename T, int V, bool GATED, bool KEEP>
__global__ __launch_bounds__(kBlock) void join_product_kernel(ProductArgs a, int results) {
    const int64_t n = (int64_t)a.M * a.N, at = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * V;
    if (at >= n) return;
    constexpr int kSums = GATED ? 2 : 1;
    float sum[kSums][V] = {};
    for (int s = 0; s < a.shares; ++s)
#pragma unroll
        for (int k = 0; k < kSums; ++k) {
            float f[V];
            load_vec<float, V>(a.part + (s * (GATED ? 2 : results) + (GATED ? k : (int)blockIdx.y)) * n + at, f);
#pragma unroll
            for (int e = 0; e < V; ++e) sum[k][e] += f[e];
        }
    if constexpr (GATED) {
        float h[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            activate<false>(a.activation, sum[0][e], &h[e], nullptr);
            h[e] *= sum[1][e];
        }
        store_vec<T, V>(static_cast<T*>(a.out[0]) + at, h);
        if constexpr (KEEP) {
            store_vec<float, V>(static_cast<float*>(a.out[1]) + at, sum[0]);
            store_vec<float, V>(static_cast<float*>(a.out[2]) + at, sum[1]);
        }
    } else {
        if constexpr (kScaled<T>) {
            const float by = *a.back;
#pragma unroll
            for (int e = 0; e < V; ++e) sum[0][e] *= by;
        }
        store_vec<T, V>(static_cast<T*>(a.out[blockIdx.y]) + at, sum[0]);
    }
}

template <typename T, int READ, int WM, int WN, int MT, int NT, bool GATED, bool KEEP, bool SPLIT = false>
int launch_product(ProductArgs a, int results, hipStream_t st) {
    constexpr int BM = WM * MT * 32, BN = WN * NT * 32, BR = GATED ? BN / 2 : BN;
    constexpr size_t lds = stages(READ) * (size_t)(BM + BN) * stage_row(READ);
    static_assert(lds <= 163840, "LDS of a CU");
    const auto kernel = product_kernel<T, READ, WM, WN, MT, NT, GATED, KEEP, SPLIT>;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return capi_fail(TRIDENT_ERR_HIP, "hipFuncSetAttribute(product): %s", hipGetErrorString(e));
    }
    a.tiles_m = (a.M + BM - 1) / BM;
    a.tiles_n = (a.N + BR - 1) / BR;
    if ((int64_t)a.tiles_m * a.tiles_n > 0x7fffffff)
        return capi_fail(TRIDENT_ERR_UNSUPPORTED, "gated_linear: %d x %d is too large", a.M, a.N);
    kernel<<<dim3((unsigned)(a.tiles_m * a.tiles_n), (unsigned)results, (unsigned)(SPLIT ? a.shares : 1)), WM * WN * kWave, lds,
             st>>>(a);
    const int rc = capi_check_launch("product_kernel");
    if (!SPLIT || rc != TRIDENT_OK) return rc;
    const int64_t n = (int64_t)a.M * a.N;
    with_bool(a.N % 4 == 0, [&](auto fours) {
        constexpr int V = decltype(fours)::value ? 4 : 1;
        const dim3 grid((unsigned)((n / V + kBlock - 1) / kBlock), (unsigned)(GATED ? 1 : results));
        join_product_kernel<T, V, GATED, KEEP><<<grid, kBlock, 0, st>>>(a, results);
    });
    return capi_check_launch("join_product_kernel");
}

// Workgroups that share the sum of a tile of 64 x 64, where the tiles leave CUs idle and the sum is long: a
// stage takes 0.3 us (float32 1.2, or 0.6 of half the length) however few the tiles, the join another launch.
// bfloat16, whole and shared: the forward pass of 100 x 5,000 by 2 x 333 31 and 13 us, the backward pass of 16
// x 960 by 2 x 2,560 48 and 19; float32 176 and 26, 150 and 32.
inline int shares_for(int64_t M, int64_t N, int results, int64_t K, int parts, bool rows, int64_t es) {
    const int64_t tiles = (M + 63) / 64 * ((N + 63) / 64) * results, row = (rows ? 128 : 64) / es;
    const int64_t stages = (K + row - 1) / row * parts, length = stages * (es == 2 ? 1 : rows ? 4 : 2);
    if (tiles < 1 || tiles > 192 || length < 32) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>({512 / tiles, length / 12, stages, 16}));
}
// Bytes of their sums.
inline size_t part_bytes(int64_t M, int64_t N, int results, int64_t K, int parts, bool rows, int64_t es, int sums) {
    const int shares = shares_for(M, N, results, K, parts, rows, es);
    return shares > 1 ? (size_t)shares * sums * M * N * 4 : 0;
}

// The tile.  A larger one reads its operands less often (256 x 256: 64 bytes of LDS for 8,192 products), but
// takes a CU alone, so its tiles go in rounds of 256: it wins where the rounds are three quarters full
// (bfloat16, against 128 x 128: the forward pass of 16,384 x 1,024 by 2 x 4,096, 2,048 tiles, 336 and 378 us;
// dx, 256 tiles, 265 and 330; but dWg and dWu, 128 tiles, 445 and 315).  Where 128 x 128 leaves CUs idle, 64 x
// 64 (float32, 1,237 x 333 by 2 x 777: forward 39 to 32 us, dx 112 to 42, both weights 96 to 34).
//
// Few tiles of a long sum share it (shares_for), each with a join behind.
template <typename T, int READ, bool GATED = false, bool KEEP = false>
int product_of(ProductArgs a, int results, float* part, hipStream_t st) {
    const auto tiles = [&](int64_t bm, int64_t bn) { return (a.M + bm - 1) / bm * ((a.N + bn - 1) / bn) * results; };
    constexpr int kShare = GATED ? 2 : 1;  // of a tile's columns are one of two sums
    a.shares = shares_for(a.M, a.N, results, a.K, a.parts, READ == kRowsRows, sizeof(T));
    a.part = part;
    if (a.shares > 1) return launch_product<T, READ, 2, 2, 1, kShare, GATED, KEEP, true>(a, results, st);
    if constexpr (sizeof(T) == 2) {
        const int64_t large = tiles(256, 256 / kShare);
        if (large * 4 >= (large + 255) / 256 * 256 * 3)
            return launch_product<T, READ, 2, 4, 4, 2, GATED, KEEP>(a, results, st);
    }
    if (tiles(128, 128 / kShare) >= 256) return launch_product<T, READ, 2, 2, 2, 2, GATED, KEEP>(a, results, st);
    return launch_product<T, READ, 2, 2, 1, kShare, GATED, KEEP>(a, results, st);
}

// ------------------------------------------------------------------------------------------------
// the rest

struct SlopeArgs {
    const void *grad, *gate, *up;
    void *dgate, *dup;
    int64_t ld_grad, ld, pitch;  // of grad, of gate and up, of dgate and dup: elements
    int64_t M;
    int N, activation;
    float *tops, *back;          // kScaled: the largest values of workgroups, and one over the factor
    int groups;
};

// dg and du of eight columns, zeros from N on.
template <typename T>
__device__ __forceinline__ void slopes_at(const SlopeArgs& a, int64_t m, int col, float (&dg)[8], float (&du)[8]) {
    const T* dh = static_cast<const T*>(a.grad) + m * a.ld_grad + col;
    const float* g = static_cast<const float*>(a.gate) + m * a.ld + col;
    const float* u = static_cast<const float*>(a.up) + m * a.ld + col;
    float fh[8], fg[8], fu[8];
    if (col + 8 <= a.N) {
        load_vec<T, 8>(dh, fh);
        load_vec<float, 8>(g, fg);
        load_vec<float, 8>(u, fu);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = col + e < a.N;
            fh[e] = in ? (float)dh[e] : 0.0f;
            fg[e] = in ? g[e] : 0.0f;
            fu[e] = in ? u[e] : 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float v, s;
        activate<true>(a.activation, fg[e], &v, &s);
        dg[e] = fh[e] * fu[e] * s;
        du[e] = fh[e] * v;
    }
}

// The largest of a workgroup's values, in every thread.
__device__ __forceinline__ float block_max(float v) {
    __shared__ float s_top[kBlock / kWave];
#pragma unroll
    for (int by = 1; by < kWave; by *= 2) v = fmaxf(v, __shfl_xor(v, by, kWave));
    if (lane_id() == 0) s_top[threadIdx.x / kWave] = v;
    __syncthreads();
    v = s_top[0];
#pragma unroll
    for (int w = 1; w < kBlock / kWave; ++w) v = fmaxf(v, s_top[w]);
    return v;
}

// float16: a gradient of 1e-4 by an up of 1e-2 is below its normal numbers, one of 50 by 1e4 above them (errors of
// some per cent, or infinities, in results that are neither).  So dg and du are held times the power of two that
// brings the largest finite one of the call to 2^14 .. 2^15, and the products' sums are multiplied by its
// reciprocal: digits are lost only 2^28 below the largest.  To find that takes a pass of its own over what
// slope_kernel reads again (the gradients of 16,384 x 1,024 by 2 x 4,096 681 -> 799 us, of 64 x 512 by 2 x 1,024 25 -> 28).
// The other types have the exponents.
constexpr int kTops = 1024;
template <typename T>
__global__ __launch_bounds__(kBlock) void largest_slope_kernel(SlopeArgs a) {
    const int pieces = (int)((a.N + 7) / 8);
    float top = 0.0f;
    for (int64_t at = (int64_t)blockIdx.x * kBlock + threadIdx.x; at < a.M * pieces; at += (int64_t)gridDim.x * kBlock) {
        const int64_t m = at / pieces;
        float dg[8], du[8];
        slopes_at<T>(a, m, (int)(at - m * pieces) * 8, dg, du);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float g = fabsf(dg[e]), u = fabsf(du[e]);
            top = fmaxf(top, fmaxf(g < INFINITY ? g : 0.0f, u < INFINITY ? u : 0.0f));
        }
    }
    top = block_max(top);
    if (threadIdx.x == 0) a.tops[blockIdx.x] = top;
}

// dg and du.  Bound by bytes: three reads, two writes (16,384 x 4,096 bfloat16, 940 MB, 206 us, 4.6 TB/s).
template <typename T>
__global__ __launch_bounds__(kBlock) void slope_kernel(SlopeArgs a) {
    float by = 1.0f;
    if constexpr (kScaled<T>) {
        float top = 0.0f;
        for (int i = threadIdx.x; i < a.groups; i += kBlock) top = fmaxf(top, a.tops[i]);
        const int e = (int)(__float_as_uint(block_max(top)) >> 23);     // 2^(e - 127) <= top
        const uint32_t exponent = (uint32_t)min(268 - e, 227);          // 2^100 at most
        by = __uint_as_float(exponent << 23);
        if (blockIdx.x == 0 && threadIdx.x == 0) *a.back = __uint_as_float((254 - exponent) << 23);
    }
    const int pieces = (int)(a.pitch / 8);
    const int64_t at = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (at >= a.M * pieces) return;
    const int64_t m = at / pieces;
    const int col = (int)(at - m * pieces) * 8;
    float dg[8], du[8];
    slopes_at<T>(a, m, col, dg, du);
    if constexpr (kScaled<T>) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dg[e] *= by;
            du[e] *= by;
        }
    }
    store_vec<T, 8>(static_cast<T*>(a.dgate) + m * a.pitch + col, dg);
    store_vec<T, 8>(static_cast<T*>(a.dup) + m * a.pitch + col, du);
}

// Rows copied to a pitch of whole pieces of 16 bytes, zeros behind: for operands whose rows do not begin at
// such pieces, which LDS cannot take straight, or lie too far apart for a tile's offsets.  Those of a product in one
// launch (blockIdx.y): 1,237 x 333 and 2 x 777 in float32 take 3 us each, most of it a launch's own (forward and
// backward pass 102 us, 95 in one launch each way).
struct PackArgs {
    const void* from[3];
    void* to[3];
    int64_t ld[3], rows[3];
    int64_t pitch;
    int cols;
};

template <typename T>
__global__ __launch_bounds__(kBlock) void pack_kernel(PackArgs a) {
    constexpr int kPer = 16 / (int)sizeof(T);
    const int which = blockIdx.y, pieces = (int)(a.pitch / kPer);
    const int64_t at = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (at >= a.rows[which] * pieces) return;
    const int64_t r = at / pieces;
    const int col = (int)(at - r * pieces) * kPer;
    const T* from = static_cast<const T*>(a.from[which]) + r * a.ld[which] + col;
    float f[kPer];
    if (col + kPer <= a.cols) {
        load_vec<T, kPer>(from, f);
    } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) f[e] = col + e < a.cols ? (float)from[e] : 0.0f;
    }
    store_vec<T, kPer>(static_cast<T*>(a.to[which]) + r * a.pitch + col, f);
}

constexpr int kFewRows = 16;   // rows of x that one instruction takes
constexpr int kFewWaves = 8;

struct FewArgs {
    const void *x, *gate, *up;
    void* out[3];
    int64_t ld_x, ld_gate, ld_up, ldo;
    int M, N, K, activation;
};

typedef float f32x4v __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ f32x4v mma16(const frag<T>& a, const frag<T>& b, f32x4v c) {
    if constexpr (std::is_same<T, bf16_t>::value) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    else if constexpr (std::is_same<T, f16_t>::value) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else {
#pragma unroll
        for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
}

// Eight elements from p on, those past `left` zeros; any element's address.
template <typename T>
__device__ __forceinline__ frag<T> load_eight(const T* p, int left) {
    frag<T> f = {};
    if (left >= 8) {
        __builtin_memcpy(&f, p, sizeof(f));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) f[e] = p[e];
    }
    return f;
}

// Up to 16 rows, such as a query's: a workgroup takes 16 columns of gate and up, and its waves share K by
// blocks of 64. Bound by the bytes of the weights, each of which one wave reads once, straight to registers:
// rows of 16 lanes' pieces (bfloat16: one row of 960 by 2 x 2,560 4.7 us, 16 of 8,192 by 2 x 8,192 49, 5.4
// TB/s).
template <typename T, bool KEEP>
__global__ __launch_bounds__(kFewWaves* kWave) void few_kernel(FewArgs a) {
    __shared__ f32x4v s_acc[2][kFewWaves][kWave];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r = lane % 16, quarter = lane / 16;
    const int n0 = blockIdx.x * 16, n = min(n0 + r, a.N - 1), m = min(r, a.M - 1);
    const T* x = static_cast<const T*>(a.x) + m * a.ld_x;
    const T* wg = static_cast<const T*>(a.gate) + n * a.ld_gate;
    const T* wu = static_cast<const T*>(a.up) + n * a.ld_up;
    f32x4v g = {}, u = {};
    for (int k = wave * 64; k < a.K; k += kFewWaves * 64) {
        frag<T> fg[2], fu[2], fx[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = k + i * 32 + quarter * 8, left = a.K - at;
            fg[i] = load_eight(wg + at, left);
            fu[i] = load_eight(wu + at, left);
            fx[i] = load_eight(x + at, left);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            g = mma16<T>(fg[i], fx[i], g);
            u = mma16<T>(fu[i], fx[i], u);
        }
    }
    s_acc[0][wave][lane] = g;
    s_acc[1][wave][lane] = u;
    __syncthreads();
    if (wave != 0 || r >= a.M) return;
    for (int w = 1; w < kFewWaves; ++w) {
        g += s_acc[0][w][lane];
        u += s_acc[1][w][lane];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int col = n0 + quarter * 4 + e;
        if (col >= a.N) break;
        float v;
        activate<false>(a.activation, g[e], &v, nullptr);
        const int64_t at = r * a.ldo + col;
        static_cast<T*>(a.out[0])[at] = (T)(v * u[e]);
        if constexpr (KEEP) {
            static_cast<float*>(a.out[1])[at] = g[e];
            static_cast<float*>(a.out[2])[at] = u[e];
        }
    }
}

// ------------------------------------------------------------------------------------------------
// calls

inline int64_t size_of(int32_t dtype) { return dtype == TRIDENT_F32 ? 4 : 2; }
inline int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
// Elements of a packed row: whole pieces, no power of two apart.
inline int64_t pitch_of(int64_t cols, int64_t es) {
    const int64_t p = round_up(cols, 8);
    return p * es % 1024 == 0 ? p + 64 / es * 2 : p;
}
inline size_t bytes_of(int64_t rows, int64_t pitch, int64_t es) { return (size_t)round_up(rows * pitch * es, 256); }

constexpr int64_t kFarthest = 1 << 21;  // elements from row to row, so that a tile's rows are within 32-bit offsets

inline bool whole(const void* p, int64_t ld, int64_t es) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * es % 16 == 0 && ld <= kFarthest;
}

struct Scratch {
    uint8_t* p;
    size_t left;
    void* take(size_t n) {
        void* r = p;
        p += n;
        left -= n;
        return r;
    }
};

// Operands of K columns as they are, or packed into scratch by one launch.
template <typename T>
struct Operands {
    Scratch* s;
    PackArgs a{};
    int count = 0;
    int64_t most = 0;  // pieces of one

    Operands(Scratch* scratch, int64_t cols) : s(scratch) {
        a.pitch = pitch_of(cols, sizeof(T));
        a.cols = (int)cols;
    }
    Operand add(const void* p, int64_t ld, int64_t rows) {
        if (whole(p, ld, sizeof(T)) && a.cols % (16 / sizeof(T)) == 0)
            return {static_cast<const uint8_t*>(p), ld * (int64_t)sizeof(T)};
        void* to = s->take(bytes_of(rows, a.pitch, sizeof(T)));
        a.from[count] = p;
        a.to[count] = to;
        a.ld[count] = ld;
        a.rows[count++] = rows;
        most = std::max(most, rows * (a.pitch / (16 / (int64_t)sizeof(T))));
        return {static_cast<const uint8_t*>(to), a.pitch * (int64_t)sizeof(T)};
    }
    int pack(hipStream_t st) const {
        if (!count) return TRIDENT_OK;
        pack_kernel<T><<<dim3((unsigned)((most + kBlock - 1) / kBlock), (unsigned)count), kBlock, 0, st>>>(a);
        return capi_check_launch("pack_kernel");
    }
};

size_t packed_bytes(const void* p, int64_t ld, int64_t rows, int64_t cols, int64_t es) {
    return whole(p, ld, es) && cols % (16 / es) == 0 ? 0 : bytes_of(rows, pitch_of(cols, es), es);
}

constexpr size_t kTopsBytes = (kTops + 64) * sizeof(float);  // and the factor back

size_t forward_bytes(const TridentGated* t) {
    if (t->M <= kFewRows) return 0;
    const int64_t es = size_of(t->dtype);
    return packed_bytes(t->x, t->ld_x, t->M, t->K, es) + packed_bytes(t->gate_weight, t->ld_gate, t->N, t->K, es) +
           packed_bytes(t->up_weight, t->ld_up, t->N, t->K, es) + part_bytes(t->M, t->N, 1, t->K, 1, true, es, 2);
}

// Of dx and of the weights' gradients, which come one after the other.
size_t backward_part(const TridentGated* t) {
    const int64_t es = size_of(t->dtype);
    return round_up(std::max(part_bytes(t->M, t->K, 1, t->N, 2, false, es, 1), part_bytes(t->N, t->K, 2, t->M, 1, false, es, 2)),
                    256);
}

size_t backward_bytes(const TridentGated* t) {
    const int64_t es = size_of(t->dtype);
    return packed_bytes(t->x, t->ld_x, t->M, t->K, es) + packed_bytes(t->gate_weight, t->ld_gate, t->N, t->K, es) +
           packed_bytes(t->up_weight, t->ld_up, t->N, t->K, es) + 2 * bytes_of(t->M, pitch_of(t->N, es), es) + backward_part(t) +
           (t->dtype == TRIDENT_F16 ? kTopsBytes : 0);
}

int check(const TridentGated* t, bool backward) {
    const char* name = backward ? "gated_linear_grad" : "gated_linear";
    if (!t) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "%s: NULL arguments", name);
    if (!dtype_ok(t->dtype)) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "%s: dtype=%d", name, t->dtype);
    if (t->activation < TRIDENT_SILU || t->activation > TRIDENT_GELU_TANH)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "%s: activation=%d", name, t->activation);
    constexpr int64_t most = (int64_t)1 << 40;
    if (t->M < 0 || t->N < 0 || t->K < 1 || t->M > (1 << 30) || t->N > kFarthest || t->K > kFarthest || t->ld_x < t->K ||
        t->ld_gate < t->K || t->ld_up < t->K || t->ld_x > most || t->ld_gate > most || t->ld_up > most)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "%s: bad sizes M=%lld N=%lld K=%lld pitches %lld, %lld, %lld", name,
                         (long long)t->M, (long long)t->N, (long long)t->K, (long long)t->ld_x, (long long)t->ld_gate,
                         (long long)t->ld_up);
    return TRIDENT_OK;
}

template <typename T>
int forward(const TridentGated* t, Scratch s, hipStream_t st) {
    const bool keep = t->gate != nullptr;
    if (t->M <= kFewRows) {
        FewArgs a{t->x, t->gate_weight, t->up_weight, {t->h, t->gate, t->up}, t->ld_x, t->ld_gate, t->ld_up, t->N,
                  (int)t->M, (int)t->N, (int)t->K, t->activation};
        const unsigned grid = (unsigned)((t->N + 15) / 16);
        if (keep) few_kernel<T, true><<<grid, kFewWaves * kWave, 0, st>>>(a);
        else few_kernel<T, false><<<grid, kFewWaves * kWave, 0, st>>>(a);
        return capi_check_launch("few_kernel");
    }
    ProductArgs a{};
    Operands<T> operands(&s, t->K);
    a.second[0] = operands.add(t->x, t->ld_x, t->M);
    a.first[0] = operands.add(t->gate_weight, t->ld_gate, t->N);
    a.first[1] = operands.add(t->up_weight, t->ld_up, t->N);
    const int rc = operands.pack(st);
    if (rc != TRIDENT_OK) return rc;
    a.out[0] = t->h;
    a.out[1] = t->gate;
    a.out[2] = t->up;
    a.ldo = t->N;
    a.M = (int)t->M;
    a.N = (int)t->N;
    a.K = (int)t->K;
    a.parts = 1;
    a.activation = t->activation;
    float* part = reinterpret_cast<float*>(s.p);
    if (keep) return product_of<T, kRowsRows, true, true>(a, 1, part, st);
    return product_of<T, kRowsRows, true, false>(a, 1, part, st);
}

template <typename T>
int backward(const TridentGated* t, Scratch s, hipStream_t st) {
    const int64_t pitch = pitch_of(t->N, sizeof(T));
    float* part = static_cast<float*>(s.take(backward_part(t)));
    SlopeArgs d{t->grad, t->gate, t->up, s.take(bytes_of(t->M, pitch, sizeof(T))), s.take(bytes_of(t->M, pitch, sizeof(T))),
                t->ld_grad, t->N, pitch, t->M, (int)t->N, t->activation, nullptr, nullptr, 0};
    if constexpr (kScaled<T>) {
        d.tops = static_cast<float*>(s.take(kTopsBytes));
        d.back = d.tops + kTops;
        d.groups = (int)std::min<int64_t>(kTops, (t->M * ((t->N + 7) / 8) + kBlock - 1) / kBlock);
        largest_slope_kernel<T><<<(unsigned)d.groups, kBlock, 0, st>>>(d);
        const int rc = capi_check_launch("largest_slope_kernel");
        if (rc != TRIDENT_OK) return rc;
    }
    slope_kernel<T><<<(unsigned)((t->M * (pitch / 8) + kBlock - 1) / kBlock), kBlock, 0, st>>>(d);
    int rc = capi_check_launch("slope_kernel");
    const Operand dg{static_cast<const uint8_t*>(d.dgate), pitch * (int64_t)sizeof(T)},
        du{static_cast<const uint8_t*>(d.dup), pitch * (int64_t)sizeof(T)};
    if (rc != TRIDENT_OK) return rc;
    Operands<T> operands(&s, t->K);
    Operand x{}, gate{}, up{};
    if (t->dx) {
        gate = operands.add(t->gate_weight, t->ld_gate, t->N);
        up = operands.add(t->up_weight, t->ld_up, t->N);
    }
    if (t->dgate_weight) x = operands.add(t->x, t->ld_x, t->M);
    rc = operands.pack(st);
    if (rc == TRIDENT_OK && t->dx) {
        ProductArgs a{};
        a.first[0] = gate;
        a.first[1] = up;
        a.second[0] = dg;
        a.second[1] = du;
        a.out[0] = t->dx;
        a.ldo = t->K;
        a.M = (int)t->M;
        a.N = (int)t->K;
        a.K = (int)t->N;
        a.parts = 2;
        a.back = d.back;
        rc = product_of<T, kColumnsRows>(a, 1, part, st);
    }
    if (rc == TRIDENT_OK && t->dgate_weight) {
        ProductArgs a{};
        a.first[0] = x;
        a.second[0] = dg;
        a.second[1] = du;
        a.out[0] = t->dgate_weight;
        a.out[1] = t->dup_weight;
        a.ldo = t->K;
        a.M = (int)t->N;
        a.N = (int)t->K;
        a.K = (int)t->M;
        a.parts = 1;
        a.back = d.back;
        rc = product_of<T, kColumnsColumns>(a, 2, part, st);
    }
    return rc;
}

}  // namespace
}  // namespace trident

using namespace trident;

extern "C" {

size_t trident_gated_linear_workspace_bytes(const TridentGated* t) {
    return check(t, false) == TRIDENT_OK && t->M > 0 && t->N > 0 ? forward_bytes(t) : 0;
}

size_t trident_gated_linear_grad_workspace_bytes(const TridentGated* t) {
    return check(t, true) == TRIDENT_OK && t->M > 0 && t->N > 0 ? backward_bytes(t) : 0;
}

int trident_gated_linear(const TridentGated* t, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check(t, false);
    if (rc != TRIDENT_OK || t->M == 0 || t->N == 0) return rc;
    if (!t->x || !t->gate_weight || !t->up_weight || !t->h || (t->gate == nullptr) != (t->up == nullptr))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "gated_linear: NULL pointer, or one of gate and up without the other");
    const size_t need = forward_bytes(t);
    if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
        return capi_fail(TRIDENT_ERR_WORKSPACE_TOO_SMALL, "gated_linear needs %zu bytes, 16-byte aligned, got %zu", need,
                         workspace ? workspace_bytes : 0);
    with_dtype(t->dtype, [&](auto e) {
        rc = forward<decltype(e)>(t, {static_cast<uint8_t*>(workspace), workspace_bytes}, (hipStream_t)stream);
    });
    return rc;
}

int trident_gated_linear_grad(const TridentGated* t, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check(t, true);
    if (rc != TRIDENT_OK) return rc;
    if (t->ld_grad < t->N) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "gated_linear_grad: ld_grad=%lld", (long long)t->ld_grad);
    if (t->M == 0 || t->N == 0)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "gated_linear_grad: no rows or columns: the gradients are zeros");
    if (!t->x || !t->gate_weight || !t->up_weight || !t->grad || !t->gate || !t->up ||
        (t->dgate_weight == nullptr) != (t->dup_weight == nullptr))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT,
                         "gated_linear_grad: NULL pointer, or one of dgate_weight and dup_weight without the other");
    const size_t need = backward_bytes(t);
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return capi_fail(TRIDENT_ERR_WORKSPACE_TOO_SMALL, "gated_linear_grad needs %zu bytes, 16-byte aligned, got %zu", need,
                         workspace ? workspace_bytes : 0);
    with_dtype(t->dtype, [&](auto e) {
        rc = backward<decltype(e)>(t, {static_cast<uint8_t*>(workspace), workspace_bytes}, (hipStream_t)stream);
    });
    return rc;
}

}  // extern "C"
