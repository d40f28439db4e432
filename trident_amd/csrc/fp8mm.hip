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
    uint8_t* codes;  // [rows, pitch]
    uint8_t* scales; // [rows, kbp]
    int64_t rows, ld, pitch;
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

// Bound by bytes: one read, one write, 16 lanes a block, whose largest value they find among themselves.
// 8192 x 4096 bfloat16 19 us, 5.3 TB/s; 1237 x 1000 float32 3.6 us, a launch's time.
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
    *reinterpret_cast<uint2*>(a.codes + row * a.pitch + col) = codes_of(f, e);
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
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct MatmulArgs {
    const uint8_t *a, *b;    // codes [M, pitch], [N, pitch]
    const uint8_t *sa, *sb;  // scales [M, spitch], [N, spitch]
    const void* bias;        // [N] or null
    void* out;               // [M, ldo]
    int64_t pitch_a, pitch_b, ldo;
    int M, N, kb, spitch, bias_f32, tiles_m, tiles_n;
    int share;               // blocks of K of one workgroup, SPLIT only
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

// One of a grid of workgroups in an order that keeps neighbouring tiles on one XCD (workgroups go to the
// eight XCDs in turn, each with its own L2): each XCD takes a contiguous eighth, in bands of `band` tile
// rows, so that the tiles it works on at a time share their rows and columns.
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int band, int* tm, int* tn) {
    const int total = tiles_m * tiles_n, each = total / 8, more = total % 8;
    const int xcd = id % 8, k = id / 8;
    const int t = xcd * each + min(xcd, more) + k;
    const int first = t / (band * tiles_n) * band, rows = min(band, tiles_m - first);
    const int in = t - first * tiles_n;
    *tm = first + in % rows;
    *tn = in / rows;
}

typedef __attribute__((address_space(3))) void* lds_ptr;

// A buffer that begins at p.  Offsets are 32 bits; the caller keeps them inside.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0xffffffffu, 0x00027000);
}

// The bias of columns first .. first + N - 1; those past the last one repeat it.
template <typename T, int N>
__device__ __forceinline__ void load_bias(const void* bias, int f32, int first, int columns, float (&out)[N]) {
    if (!bias) {
#pragma unroll
        for (int e = 0; e < N; ++e) out[e] = 0.0f;
    } else if (f32) {
#pragma unroll
        for (int e = 0; e < N; ++e) out[e] = static_cast<const float*>(bias)[min(first + e, columns - 1)];
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) out[e] = (float)static_cast<const T*>(bias)[min(first + e, columns - 1)];
    }
}

// A workgroup of WM x WN waves computes a tile of WM MT x WN NT blocks of 32 x 32, a wave MT x NT of
// them.  128 columns of both operands at a time go straight from memory to LDS (no registers between),
// the next ones while these are multiplied.  The eight 16-byte pieces of a row are stored exchanged by
// bits 1 to 3 of its number: 16 lanes that read the same piece of as many rows then read from all of
// LDS's 64 banks (a row is half of them, so rows that differ in bit 0 never meet).  The
// weight is the instruction's first operand, so a lane holds four neighbouring columns of a result row.
// A block of 128 columns is two instructions of 64 each with the same scale; in both operands a lane
// passes the same columns, in whatever order the instruction takes them.  WK teams of such waves take
// WK blocks at a time, where a CU has one small tile and the length of K is what it waits for.  The rows'
// scales (a word a row, that of four blocks) go to LDS as well: no register waits for memory in the loop,
// and every stage is the same number of loads, so the wait for one leaves the next one's in flight.
//
// Bound by the matrix core and the power it is given.  8-bit products, 256 x 256: 8192 x 4096 x 4096 138 us,
// 2.0 PFLOP/s, x 8192 252 us, 2.2; as bfloat16, 128 x 128: 8192 x 4096 x 8192 470 us, 1.17 PFLOP/s, where
// the conversion shares the time.  A small product is bound by its few tiles' latency: 1237 x 777 x 1000
// in float32 10 us.
//
// With SPLIT a tile's K is shared by the workgroups of a column of the grid, each of which writes its sums to
// an array of its own.
template <typename T, bool FAST, int WM, int WN, int MT, int NT, int WK, bool SPLIT>
__global__ __launch_bounds__(WM* WN* WK* kWave) void matmul_kernel(MatmulArgs g) {
    constexpr int kTeam = WM * WN, kWaves = kTeam * WK, BM = WM * MT * 32, BN = WN * NT * 32, kRows = BM + BN;
    constexpr int kStage = WK * kRows * kBlockK;
    constexpr int kLoads = WK * kRows / 8 / kWaves;  // a wave's loads of eight rows each
    static_assert(WK * kRows / 8 % kWaves == 0 && kLoads % 2 == 0, "whole loads, of either parity by turns");
    static_assert(BM % kWave == 0 && BN % kWave == 0, "a load of scales is of one operand and block");
    constexpr int kScaleLoads = (WK * kRows + kWaves * kWave - 1) / (kWaves * kWave);
    constexpr int kScaleStage = kScaleLoads * kWaves * kWave * 4;
    constexpr int kFlight = kLoads + kScaleLoads;  // a wave's loads of one stage
    extern __shared__ __align__(16) uint8_t lds[];  // [2][WK][BM + BN][128], [2][WK][BM + BN] words of scales
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r = lane & 31, q = lane >> 5;
    int tm, tn;
    tile_of(blockIdx.x, g.tiles_m, g.tiles_n, 8, &tm, &tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int team = wave / kTeam, wm = wave % kTeam / WN * MT * 32, wn = wave % WN * NT * 32;

    const int kb0 = SPLIT ? (int)blockIdx.y * g.share : 0, kb1 = SPLIT ? min(g.kb, kb0 + g.share) : g.kb;

    // A stage is WK times BM rows of a and BN of b, kLoads loads of eight rows for each wave: of one
    // operand, so the wave's loads differ in a scalar only.  Rows past the operand's end repeat the last.
    constexpr int kWaveRows = kLoads * 8;
    static_assert(BM % kWaveRows == 0 && kRows % kWaveRows == 0, "a wave loads from one operand");
    const auto operand = [&](int first, auto&& of_a, auto&& of_b) { return first % kRows < BM ? of_a : of_b; };
    const int first = wave * kWaveRows, load_part = first / kRows;
    const int row0 = first % kRows < BM ? m0 + first % kRows : n0 + first % kRows - BM;
    const int limit = operand(first, g.M, g.N), start = min(row0, limit - 1), rows = min(kWaveRows, limit - start);
    const int64_t pitch = operand(first, g.pitch_a, g.pitch_b);
    const __amdgpu_buffer_rsrc_t buf = buffer_at(operand(first, g.a, g.b) + start * pitch);
    const uint32_t row_step = (uint32_t)pitch * 8;
    // row l / 8 of a load, piece l % 8, exchanged by bits 1 to 3 of the row, the last being the load's parity
    const uint32_t piece = (uint32_t)((lane % 8) ^ (lane / 16)) * 16;
    const uint32_t even = (uint32_t)(lane / 8) * (uint32_t)pitch + piece, odd = even ^ 64;
    // the scales: 64 rows a load
    __amdgpu_buffer_rsrc_t scale_buf[kScaleLoads];
    uint32_t scale_row[kScaleLoads];
    int scale_part[kScaleLoads];
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) {
        const int at = min((i * kWaves + wave) * kWave, WK * kRows - kWave), in = at % kRows;
        const int row = in < BM ? m0 + in : n0 + in - BM, last = operand(at, g.M, g.N) - 1;
        scale_part[i] = at / kRows;
        scale_buf[i] = buffer_at(operand(at, g.sa, g.sb) + (int64_t)min(row, last) * g.spitch);
        scale_row[i] = (uint32_t)(min(row + lane, last) - min(row, last)) * (uint32_t)g.spitch;
    }
    const auto fetch = [&](int step) {
        uint8_t* to = lds + step % 2 * kStage + wave * kLoads * 1024;
        const uint32_t k = (uint32_t)min(kb0 + step * WK + load_part, kb1 - 1) * kBlockK;
        if (rows == kWaveRows) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (lds_ptr)(to + i * 1024), 16, i % 2 ? odd : even,
                                                         k + i * row_step, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    buf, (lds_ptr)(to + i * 1024), 16,
                    (uint32_t)min(i * 8 + lane / 8, rows - 1) * (uint32_t)pitch + (piece ^ (i % 2 * 64)), k, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kScaleLoads; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                scale_buf[i],
                (lds_ptr)(lds + 2 * kStage + step % 2 * kScaleStage + (i * kWaves + wave) * kWave * 4), 4, scale_row[i],
                min(kb0 + step * WK + scale_part[i], kb1 - 1) & ~3, 0, 0);
    };
    // where this lane reads the four pieces of its first row of either operand; the other rows are 32
    // rows on, the other stage is the next bit
    static_assert((kStage & (kStage - 1)) == 0, "a stage is a bit of the address");
    uint32_t at_a[4], at_b[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t p = (uint32_t)((4 * (c / 2) + 2 * q + c % 2) ^ (r >> 1 & 7)) * 16;
        at_a[c] = (uint32_t)(team * kRows + wm + r) * kBlockK + p;
        at_b[c] = (uint32_t)(team * kRows + BM + wn + r) * kBlockK + p;
    }
    typedef const __attribute__((address_space(3))) uint8_t* lds_bytes;
    typedef const __attribute__((address_space(3))) u32x4* lds_piece;
    const lds_bytes stage0 = (lds_bytes)(lds_ptr)lds;
    const auto read = [&](const uint32_t (&at)[4], int half, int block) {
        const u32x4 lo = *(lds_piece)(stage0 + at[2 * half] + block * (32 * kBlockK));
        const u32x4 hi = *(lds_piece)(stage0 + at[2 * half + 1] + block * (32 * kBlockK));
        i32x8 f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = (int)lo[e];
            f[4 + e] = (int)hi[e];
        }
        return f;
    };

    // at the end this lane writes kPer columns of every kRowsAtOnce-th row: their bias, early where
    // registers are left
    constexpr bool kEarly = MT * NT < 8;
    constexpr int kCols = NT * 32, kPitch = kCols * 4 + 16, kPer = 16 / (int)sizeof(T);
    constexpr int kRowPieces = kCols / kPer, kRowsAtOnce = kWave / kRowPieces;
    static_assert(kTeam * 32 * kPitch <= 2 * kStage, "the results fit where the operands were");
    const int piece_col = n0 + wn + lane % kRowPieces * kPer, left = g.N - piece_col;
    float bias[kPer];
    if constexpr (kEarly) load_bias<T, kPer>(g.bias, g.bias_f32, piece_col, g.N, bias);

    f32x16 acc[MT][NT] = {};
    // Two stages.  A stage's next loads are issued as soon as every wave holds its part of it in
    // registers, halfway through its products, so they have a step and a half to arrive.
    const int steps = (kb1 - kb0 + WK - 1) / WK;
    fetch(0);
    if (steps > 1) fetch(1);
    for (int step = 0; step < steps; ++step) {
        // past the barrier this stage has arrived, every wave's part of it (loads arrive in order)
        if (step + 1 < steps) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(kFlight) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int kb = kb0 + step * WK + team;
        const bool live = WK == 1 || kb < kb1;  // not in the last step of the last team of an odd number
        const uint32_t* st = reinterpret_cast<const uint32_t*>(lds + 2 * kStage + step % 2 * kScaleStage) + team * kRows;
        uint32_t ea[MT], eb[NT];  // the scale of this block in the lowest byte
#pragma unroll
        for (int i = 0; i < MT; ++i) ea[i] = st[wm + i * 32 + r];
#pragma unroll
        for (int j = 0; j < NT; ++j) eb[j] = st[BM + wn + j * 32 + r];
        __builtin_amdgcn_sched_barrier(0);  // these reads first: every product needs them
#pragma unroll
        for (int i = 0; i < MT; ++i) ea[i] >>= kb % 4 * 8;
#pragma unroll
        for (int j = 0; j < NT; ++j) eb[j] >>= kb % 4 * 8;
        i32x8 fa[2][MT], fb[2][NT];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int j = 0; j < NT; ++j) fb[half][j] = read(at_b, half, j);
#pragma unroll
            for (int i = 0; i < MT; ++i) fa[half][i] = read(at_a, half, i);
        }
        const auto multiply = [&](int half) {
            if constexpr (FAST) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                            fb[half][j], fa[half][i], acc[i][j], 0, 0, 0, (int)eb[j], 0, (int)ea[i]);
            } else {
                bf16x8 hb[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j) to_bf16(fb[half][j], scale_value(eb[j] & 255u), hb[j]);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    bf16x8 ha[4];
                    to_bf16(fa[half][i], scale_value(ea[i] & 255u), ha);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int j = 0; j < NT; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hb[j][k], ha[k], acc[i][j], 0, 0, 0);
                }
            }
        };
        if (live) multiply(0);
        if constexpr (FAST) {
            // the first half's reads, the second half's among the first half's products
            constexpr int kReads = 2 * (MT + NT), kProducts = MT * NT, kEach = (kReads + kProducts - 1) / kProducts;
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
        // past this barrier every wave has read the stage
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (step + 2 < steps) fetch(step + 2);
        if (live) multiply(1);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            at_a[c] ^= kStage;
            at_b[c] ^= kStage;
        }
    }
    // The results go through this wave's part of LDS, 32 rows at a time, so that it writes whole lines: a
    // lane holds four columns, and rows a power of two apart would all meet in one channel of L2.
    if constexpr (!kEarly) load_bias<T, kPer>(g.bias, g.bias_f32, piece_col, g.N, bias);
    __syncthreads();
    if constexpr (WK > 1) {  // the other teams' sums first, added in order
        static_assert(WK == 2 && MT * NT * kTeam * kWave * 64 <= 2 * kStage, "one more team, whose sums fit");
        f32x16* sums = reinterpret_cast<f32x16*>(lds) + wave % kTeam * (MT * NT * kWave) + lane;
        if (team == 1) {
#pragma unroll
            for (int i = 0; i < MT * NT; ++i) sums[i * kWave] = acc[i / NT][i % NT];
        }
        __syncthreads();
        if (team == 0) {
#pragma unroll
            for (int i = 0; i < MT * NT; ++i) acc[i / NT][i % NT] += sums[i * kWave];
        }
        __syncthreads();
        if (team == 1) return;
    }
    float* mine = reinterpret_cast<float*>(lds + wave * 32 * kPitch);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * p + e];
                *reinterpret_cast<f32x4*>(mine + r * (kPitch / 4) + j * 32 + p * 8 + q * 4) = v;
            }
        wave_sync();
#pragma unroll
        for (int k = 0; k < 32; k += kRowsAtOnce) {
            const int row = k + lane / kRowPieces, m = m0 + wm + i * 32 + row;
            const f32x4* from = reinterpret_cast<const f32x4*>(mine + row * (kPitch / 4) + lane % kRowPieces * kPer);
            T v[kPer];
#pragma unroll
            for (int e = 0; e < kPer; ++e) v[e] = (T)(from[e / 4][e % 4] + bias[e]);
            if (m >= g.M) continue;
            T* out = static_cast<T*>(g.out) + ((SPLIT ? (int64_t)blockIdx.y * g.M : 0) + m) * g.ldo + piece_col;
            if (left >= kPer) {
                __builtin_memcpy(out, v, 16);
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e)
                    if (e < left) out[e] = v[e];
            }
        }
        wave_sync();
    }
}

// The sums of SPLIT workgroups, in order, with the bias: four columns a thread.  A launch's time, 3.3 us
// beside the others.
template <typename T>
__global__ __launch_bounds__(kBlock) void join_products_kernel(const float* __restrict__ part, int shares, int64_t M,
                                                               int N, int quads, const void* bias, int bias_f32,
                                                               T* __restrict__ out, int64_t ldo) {
    const int64_t at = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (at >= M * quads) return;
    const int64_t m = at / quads;
    const int col = (int)(at - m * quads) * 4;
    f32x4 sum = {};
    for (int s = 0; s < shares; ++s) sum += *reinterpret_cast<const f32x4*>(part + (s * M * quads + at) * 4);
    float b[4];
    load_bias<T, 4>(bias, bias_f32, col, N, b);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (col + e < N) out[m * ldo + col + e] = (T)(sum[e] + b[e]);
}

constexpr int kFewWaves = 8;
constexpr int kFewRows = 16;    // rows that one instruction takes
constexpr int kFewCost = 512;   // of quantising the rows in every workgroup: what a second launch costs

struct FewArgs {
    const void* x;           // [M, ldx], or null: the codes of a
    const uint8_t *a, *sa;
    const uint8_t *b, *sb;
    const void* bias;
    void* out;
    int64_t ldx, pitch_a, pitch_b, ldo;
    int M, N, K, kb, spitch, bias_f32;
};

// Up to 64 rows, bound by the weight's bytes or, for one query, by the latency of a launch.  A workgroup
// takes 16 NT columns; its eight waves take the blocks of 128 of K in turn, the weight straight from memory
// to registers, and their sums are added in order at the end.  The rows may be quantised on the way
// (QUANT): a lane holds the 32 columns of its row that the instruction wants from it, and a block's largest
// value is that of four lanes, so one launch does all and nothing is stored between.
//
// Each workgroup begins at another block: the rows of a weight are a power of two apart in most models, so
// all workgroups would else read the same few channels of memory at a time (one row by 8192 x 8192: 19.8
// us, 14.9 so: 4.5 TB/s).  One row of 960 columns by 1024 x 960: 4.9 us.
template <typename T, bool FAST, bool QUANT, int MT, int NT>
__global__ __launch_bounds__(kFewWaves* kWave) void matmul_few_kernel(FewArgs g) {
    constexpr int U = MT > 1 || NT > 2 ? 1 : NT > 1 || sizeof(T) == 4 ? 2 : 4;  // blocks of a wave in flight
    __shared__ f32x4 s_acc[kFewWaves][MT * NT][kWave];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r = lane & 15, q = lane >> 4, n0 = blockIdx.x * (16 * NT);
    const uint8_t *b[NT], *sb[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t n = min(n0 + j * 16 + r, g.N - 1);
        b[j] = g.b + n * g.pitch_b + q * 32;
        sb[j] = g.sb + n * g.spitch;
    }
    float bias[4];  // of the columns that this lane writes: wave w joins 16 rows and 16 columns
    const int m = wave % MT * 16 + r, c0 = n0 + wave / MT * 16 + q * 4;
    load_bias<T, 4>(g.bias, g.bias_f32, c0, g.N, bias);
    const int turn = (int)(blockIdx.x % (unsigned)g.kb);
    f32x4 acc[MT][NT] = {};
    for (int k0 = wave; k0 < g.kb; k0 += kFewWaves * U) {
        u32x4 wb[U][NT][2], wa[U][MT][2];
        Vec<T, 8> x[U][MT][4];
        int eb[U][NT], ea[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int kb = k0 + u * kFewWaves;
            if (kb >= g.kb) break;
            if ((kb += turn) >= g.kb) kb -= g.kb;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                __builtin_memcpy(wb[u][j], b[j] + (int64_t)kb * kBlockK, 32);
                eb[u][j] = sb[j][kb];
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int64_t m = min(i * kFewRows + r, g.M - 1);
                if constexpr (QUANT) {
                    const T* row = static_cast<const T*>(g.x) + m * g.ldx;
                    const int col = kb * kBlockK + q * 32;
                    if (col + 32 <= g.K) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[u][i][e].load(row + col + e * 8);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            T v[8];
#pragma unroll
                            for (int c = 0; c < 8; ++c)
                                v[c] = col + e * 8 + c < g.K ? row[col + e * 8 + c] : (T)0.0f;
                            x[u][i][e].load(v);
                        }
                    }
                } else {
                    __builtin_memcpy(wa[u][i], g.a + m * g.pitch_a + (int64_t)kb * kBlockK + q * 32, 32);
                    ea[u][i] = g.sa[m * g.spitch + kb];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k0 + u * kFewWaves >= g.kb) break;
            i32x8 fb[NT];
            bf16x8 hb[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int e = 0; e < 8; ++e) fb[j][e] = (int)wb[u][j][e / 4][e % 4];
                if constexpr (!FAST) to_bf16(fb[j], scale_value((uint32_t)eb[u][j]), hb[j]);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                i32x8 fa;
                if constexpr (QUANT) {
                    float v[4][8], top = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[u][i][e].get(v[e]);
#pragma unroll
                        for (int c = 0; c < 8; ++c) top = fmaxf(top, fabsf(v[e][c]) < INFINITY ? fabsf(v[e][c]) : 0.0f);
                    }
                    top = fmaxf(top, __shfl_xor(top, 16, kWave));
                    top = fmaxf(top, __shfl_xor(top, 32, kWave));
                    ea[u][i] = scale_of(top);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint2 c = codes_of(v[e], ea[u][i]);
                        fa[2 * e] = (int)c.x;
                        fa[2 * e + 1] = (int)c.y;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) fa[e] = (int)wa[u][i][e / 4][e % 4];
                }
                bf16x8 ha[4];
                if constexpr (!FAST) to_bf16(fa, scale_value((uint32_t)ea[u][i]), ha);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if constexpr (FAST) {
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, acc[i][j], 0, 0, 0,
                                                                                     eb[u][j], 0, ea[u][i]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hb[j][k], ha[k], acc[i][j], 0, 0, 0);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) s_acc[wave][j * MT + i][lane] = acc[i][j];
    __syncthreads();
    if (wave >= MT * NT || m >= g.M) return;
    f32x4 sum = s_acc[0][wave][lane];
    for (int w = 1; w < kFewWaves; ++w) sum += s_acc[w][wave][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (c0 + e >= g.N) break;
        static_cast<T*>(g.out)[(int64_t)m * g.ldo + c0 + e] = (T)(sum[e] + bias[e]);
    }
}

// Blocks of 16 columns that a workgroup takes: more than one, which reads the rows less often, where that
// still leaves every CU a workgroup (16 float32 rows by 16384 x 2048: one block 22.6 us, four 11.8).
inline int few_columns(int64_t M, int64_t N) { return M > kFewRows || N < 8192 ? 1 : N < 16384 ? 2 : 4; }

// Whether a projection is one launch, in which every workgroup quantises all rows: where that costs a CU
// less than a second launch.  It grows with the blocks, and for each with the bytes of the rows beside a
// fixed part.  Measured, one launch against two: float32, 1 row, K = 4096 9.3 and 12.6 us, K = 8192 13.5
// and 11.5; 8 rows, K = 4096 10.6 and 11.6; 16 rows, K = 2048 9.0 and 12.2, K = 4096 14.4 and 11.3; 64
// rows, K = 768 10.2 and 11.5, K = 2048 21 and 12.  bfloat16, 16 rows, K = 4096 10.9 and 11.2, K = 8192
// 17.1 and 16.0; 32 rows, K = 2048 8.5 and 11.9 (N = 4096, 64 rows 1024).
inline bool one_launch(int64_t M, int64_t N, int64_t K, int64_t bytes) {
    if (M > 4 * kFewRows) return false;
    const int64_t groups = (N + 16 * few_columns(M, N) - 1) / (16 * few_columns(M, N));
    return blocks_of(K) * (8 + M * bytes / 4) * ((groups + 255) / 256) <= kFewCost;
}

// Whether the kernel for few rows takes codes.  Against the tiles, which wait for the length of K where
// there are few of them: 16 rows by 4096 x 4096 8.7 and 15.6 us, 32 rows 10.6 and 15.7, but 64 rows 16.6
// and 15.9, 32 rows by 16384 x 2048 16.3 and 9.8.
inline bool few_codes(int64_t M, int64_t N) { return M <= kFewRows || (M <= 2 * kFewRows && N <= 4096); }

// Launches the kernel of one tile size.
template <typename T, bool FAST, int WM, int WN, int MT, int NT, int WK, bool SPLIT = false>
int launch_matmul(MatmulArgs g, hipStream_t st) {
    constexpr int BM = WM * MT * 32, BN = WN * NT * 32;
    constexpr size_t threads = WM * WN * WK * kWave, rows = WK * (size_t)(BM + BN);
    constexpr size_t lds = 2 * (rows * kBlockK + (rows + threads - 1) / threads * threads * 4);
    const auto kernel = matmul_kernel<T, FAST, WM, WN, MT, NT, WK, SPLIT>;
    static_assert(lds <= 163840, "LDS of a CU");
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return capi_fail(TRIDENT_ERR_HIP, "hipFuncSetAttribute(matmul): %s", hipGetErrorString(e));
    }
    g.tiles_m = (g.M + BM - 1) / BM;
    g.tiles_n = (g.N + BN - 1) / BN;
    if ((int64_t)g.tiles_m * g.tiles_n > 0x7fffffff)
        return capi_fail(TRIDENT_ERR_UNSUPPORTED, "fp8_matmul: %d x %d is too large", g.M, g.N);
    const unsigned shares = SPLIT ? (unsigned)((g.kb + g.share - 1) / g.share) : 1;
    kernel<<<dim3((unsigned)(g.tiles_m * g.tiles_n), shares), threads, lds, st>>>(g);
    return capi_check_launch("matmul_kernel");
}

// The tile.  A larger one reads its operands less often (256 x 256: 64 bytes of LDS for 8,192 products),
// but takes a CU alone, so its tiles are worked off in rounds of 256: it wins where the rounds are three
// quarters full (K = 4096, against 128 x 128: 4096 x 3328, 208 tiles, 67 and 76 us; 6144 x 4352, 408, 116
// and 128; 4352 x 4352, 289, 114 and 93; two rounds 70% full of 5000 x 4608 x 1024 43 and 40).  The
// smallest, whose two teams take K in half the steps, wins while a CU has two at most (1024 x 2048 x 4096,
// 512 tiles, 20.7 us and 24.2 with 128 x 128; 2048 x 1152, 576, 29.5 and 24.7; 4096 x 768 x 768, 768, 10.5
// and 9.4).  The exact products turn at the same sizes (25.7 and 35.9, 35.8 and 36.6, 12.2 and 11.5); their
// 256 x 256 tile does not fit the registers.
template <typename T, bool FAST>
int matmul(const MatmulArgs& g, hipStream_t st) {
    const auto tiles = [&](int64_t bm, int64_t bn) { return (g.M + bm - 1) / bm * ((g.N + bn - 1) / bn); };
    if constexpr (FAST) {
        const int64_t large = tiles(256, 256);
        if (large * 4 >= (large + 255) / 256 * 256 * 3) return launch_matmul<T, FAST, 2, 4, 4, 2, 1>(g, st);
    }
    if (tiles(64, 64) <= 512) return launch_matmul<T, FAST, 2, 2, 1, 1, 2>(g, st);
    return launch_matmul<T, FAST, 2, 2, 2, 2, 1>(g, st);
}

// Blocks of K of one workgroup where a product has so few tiles and so long a K that its tiles are split,
// else 0.  A tile takes 0.4 us a block of K, joining the shares another launch.  The whole projection, tiles
// whole and split: float32, exact sums, 64 x 1024 x 2048 12.2 and 16.0 us, x 4096 18.4 and 16.2, x 8192 30.7
// and 16.2; 512 x 1024 (128 tiles) x 4096 20.9 and 20.0, x 8192 34.5 and 26.5; bfloat16, fast sums, 64 x 1024
// x 4096 15.7 and 15.6, x 8192 25.3 and 15.6.
inline int split_share(int64_t M, int64_t N, int64_t K) {
    const int64_t tiles = (M + 63) / 64 * ((N + 63) / 64), kb = blocks_of(K);
    if (tiles < 1 || few_codes(M, N) || tiles > 128 || kb < 32) return 0;
    const int64_t shares = std::min(256 / tiles, kb / 8);
    return (int)((kb + shares - 1) / shares + 1) / 2 * 2;
}
inline int64_t shares_of(int64_t K, int share) { return (blocks_of(K) + share - 1) / share; }

bool counts_ok(int64_t M, int64_t K) { return M >= 0 && M <= (1 << 30) && K >= 1 && K <= (1 << 30); }

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// The pitch of codes that only this library reads: rows that are not a power of two apart, so that the
// same columns of neighbouring rows lie in different channels of L2.
inline int64_t own_pitch_of(int64_t K) { return pitch_of(K) + (pitch_of(K) % 1024 == 0 ? kBlockK : 0); }

int quantize(const void* x, int32_t dtype, int64_t rows, int64_t K, int64_t ld_x, uint8_t* codes, int64_t pitch,
             uint8_t* scales, void* stream) {
    if (!dtype_ok(dtype)) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "fp8_quantize: dtype=%d", dtype);
    if (!counts_ok(rows, K) || ld_x < K)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "fp8_quantize: bad sizes rows=%lld K=%lld ld=%lld",
                         (long long)rows, (long long)K, (long long)ld_x);
    if (rows == 0) return TRIDENT_OK;
    if (!x || !codes || !scales || !aligned16(codes))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "fp8_quantize: NULL pointer, or codes not 16-byte aligned");
    QuantArgs a{x, codes, scales, rows, ld_x, pitch, (int)K, (int)blocks_of(K), (int)scale_pitch_of(K)};
    constexpr int per = kBlock / kQuantLanes;
    const int64_t grid = (rows * a.kb + per - 1) / per;
    if (grid > 0x7fffffff)
        return capi_fail(TRIDENT_ERR_UNSUPPORTED, "fp8_quantize: rows * K = %lld is too large", (long long)(rows * K));
    with_dtype(dtype, [&](auto t) {
        quantize_kernel<decltype(t)><<<(unsigned)grid, kBlock, 0, static_cast<hipStream_t>(stream)>>>(a);
    });
    return capi_check_launch("quantize_kernel");
}

int check_product(int64_t M, int64_t N, int64_t K, const void* a, const void* b_codes, const void* b_scales,
                  const void* bias, int32_t bias_dtype, const void* out, int32_t dtype, int64_t ld_out) {
    if (!dtype_ok(dtype) || (bias && bias_dtype != dtype && bias_dtype != TRIDENT_F32))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "fp8_matmul: dtype=%d bias_dtype=%d", dtype, bias_dtype);
    if (K > (1 << 22)) return capi_fail(TRIDENT_ERR_UNSUPPORTED, "fp8_matmul: K=%lld is too large", (long long)K);
    if (!counts_ok(M, K) || !counts_ok(N, K) || ld_out < N)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "fp8_matmul: bad sizes M=%lld N=%lld K=%lld ld=%lld",
                         (long long)M, (long long)N, (long long)K, (long long)ld_out);
    if (M > 0 && N > 0 && (!a || !b_codes || !b_scales || !out || !aligned16(b_codes) || !aligned4(b_scales)))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT,
                         "fp8_matmul: NULL pointer, or codes not 16-byte, scales not 4-byte aligned");
    return TRIDENT_OK;
}

// Few rows: of codes and scales, or (QUANT) rows of out's type themselves.
template <bool QUANT>
int product_few(const void* x, int64_t ld_x, const uint8_t* a, int64_t pitch_a, const uint8_t* sa, int64_t M,
                const uint8_t* b, const uint8_t* sb, int64_t N, int64_t K, const void* bias, int32_t bias_dtype, void* out,
                int32_t dtype, int64_t ld_out, int32_t fast_accum, hipStream_t st) {
    const FewArgs g{x, a, sa, b, sb, bias, out, ld_x, pitch_a, pitch_of(K), ld_out, (int)M, (int)N, (int)K,
                    (int)blocks_of(K), (int)scale_pitch_of(K), bias_dtype == TRIDENT_F32};
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const auto go = [&](auto fast, auto mt, auto nt) {
            constexpr int MT = decltype(mt)::value, NT = decltype(nt)::value;
            matmul_few_kernel<T, decltype(fast)::value, QUANT, MT, NT>
                <<<(unsigned)((N + 16 * NT - 1) / (16 * NT)), kFewWaves * kWave, 0, st>>>(g);
        };
        using std::integral_constant;
        const auto rows = [&](auto fast) {
            const integral_constant<int, 1> one;
            const integral_constant<int, 2> two;
            const integral_constant<int, 4> four;
            const int nt = few_columns(M, N);
            if (nt == 4) go(fast, one, four);
            else if (nt == 2) go(fast, one, two);
            else if (M <= kFewRows) go(fast, one, one);
            else if (!QUANT || M <= 2 * kFewRows) go(fast, two, one);
            else if constexpr (QUANT) go(fast, four, one);
        };
        if (fast_accum) rows(std::true_type{});
        else rows(std::false_type{});
    });
    return capi_check_launch("matmul_few_kernel");
}

int product(const uint8_t* a, int64_t pitch_a, const uint8_t* sa, int64_t M, const uint8_t* b, const uint8_t* sb,
            int64_t N, int64_t K, const void* bias, int32_t bias_dtype, void* out, int32_t dtype, int64_t ld_out,
            int32_t fast_accum, hipStream_t st) {
    if (few_codes(M, N))
        return product_few<false>(nullptr, 0, a, pitch_a, sa, M, b, sb, N, K, bias, bias_dtype, out, dtype, ld_out,
                                  fast_accum, st);
    const MatmulArgs g{a, b, sa, sb, bias, out, pitch_a, pitch_of(K), ld_out, (int)M, (int)N,
                       (int)blocks_of(K), (int)scale_pitch_of(K), bias_dtype == TRIDENT_F32, 0, 0, 0};
    int rc = TRIDENT_OK;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        rc = fast_accum ? matmul<T, true>(g, st) : matmul<T, false>(g, st);
    });
    return rc;
}

// A product whose tiles' K is split: `part` holds the shares' sums, rows of N rounded up to four columns.
int product_split(const uint8_t* a, int64_t pitch_a, const uint8_t* sa, int64_t M, const uint8_t* b,
                  const uint8_t* sb, int64_t N, int64_t K, int share, float* part, const void* bias,
                  int32_t bias_dtype, void* out, int32_t dtype, int64_t ld_out, int32_t fast_accum, hipStream_t st) {
    const int quads = (int)((N + 3) / 4);
    const MatmulArgs g{a, b, sa, sb, nullptr, part, pitch_a, pitch_of(K), 4 * (int64_t)quads, (int)M, (int)N,
                       (int)blocks_of(K), (int)scale_pitch_of(K), 0, 0, 0, share};
    const int rc = fast_accum ? launch_matmul<float, true, 2, 2, 1, 1, 2, true>(g, st)
                              : launch_matmul<float, false, 2, 2, 1, 1, 2, true>(g, st);
    if (rc) return rc;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        join_products_kernel<T><<<(unsigned)((M * quads + kBlock - 1) / kBlock), kBlock, 0, st>>>(
            part, (int)shares_of(K, share), M, (int)N, quads, bias, bias_dtype == TRIDENT_F32, static_cast<T*>(out),
            ld_out);
    });
    return capi_check_launch("join_products_kernel");
}

}  // namespace
}  // namespace trident

using namespace trident;

extern "C" {

int trident_fp8_quantize(const void* x, int32_t dtype, int64_t rows, int64_t K, int64_t ld_x, uint8_t* codes,
                         uint8_t* scales, void* stream) {
    return quantize(x, dtype, rows, K, ld_x, codes, pitch_of(K), scales, stream);
}

int trident_fp8_matmul(const uint8_t* a_codes, const uint8_t* a_scales, int64_t M, const uint8_t* b_codes,
                       const uint8_t* b_scales, int64_t N, int64_t K, const void* bias, int32_t bias_dtype, void* out,
                       int32_t dtype, int64_t ld_out, int32_t fast_accum, void* stream) {
    const int rc = check_product(M, N, K, a_codes, b_codes, b_scales, bias, bias_dtype, out, dtype, ld_out);
    if (rc || M == 0 || N == 0) return rc;
    if (!a_scales || !aligned16(a_codes) || !aligned4(a_scales))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT,
                         "fp8_matmul: NULL pointer, or codes not 16-byte, scales not 4-byte aligned");
    hipStream_t st = static_cast<hipStream_t>(stream);
    return product(a_codes, pitch_of(K), a_scales, M, b_codes, b_scales, N, K, bias, bias_dtype, out, dtype, ld_out,
                   fast_accum, st);
}

size_t trident_fp8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (!counts_ok(M, K) || !counts_ok(N, K) || M == 0 || N == 0 || one_launch(M, N, K, 4)) return 0;
    const int share = split_share(M, N, K);
    return up256((size_t)(M * own_pitch_of(K))) + up256((size_t)(M * scale_pitch_of(K))) +
           (share ? (size_t)(shares_of(K, share) * M * ((N + 3) / 4)) * 16 : 0);
}

int trident_fp8_linear(const void* x, int32_t dtype, int64_t M, int64_t K, int64_t ld_x, const uint8_t* w_codes,
                       const uint8_t* w_scales, int64_t N, const void* bias, int32_t bias_dtype, void* out,
                       int64_t ld_out, int32_t fast_accum, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_product(M, N, K, x, w_codes, w_scales, bias, bias_dtype, out, dtype, ld_out);
    if (rc) return rc;
    if (ld_x < K)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "fp8_linear: ld=%lld < K=%lld", (long long)ld_x, (long long)K);
    if (M == 0 || N == 0) return TRIDENT_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (one_launch(M, N, K, dtype == TRIDENT_F32 ? 4 : 2))
        return product_few<true>(x, ld_x, nullptr, 0, nullptr, M, w_codes, w_scales, N, K, bias, bias_dtype, out, dtype,
                                 ld_out, fast_accum, st);
    const size_t need = trident_fp8_linear_workspace_bytes(M, N, K);
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
        return capi_fail(TRIDENT_ERR_WORKSPACE_TOO_SMALL, "fp8_linear: workspace %zu < %zu bytes, or not 16-byte aligned",
                         workspace_bytes, need);
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    uint8_t* scales = codes + up256((size_t)(M * own_pitch_of(K)));
    if ((rc = quantize(x, dtype, M, K, ld_x, codes, own_pitch_of(K), scales, stream))) return rc;
    if (const int share = split_share(M, N, K)) {
        float* part = reinterpret_cast<float*>(scales + up256((size_t)(M * scale_pitch_of(K))));
        return product_split(codes, own_pitch_of(K), scales, M, w_codes, w_scales, N, K, share, part, bias, bias_dtype,
                             out, dtype, ld_out, fast_accum, st);
    }
    return product(codes, own_pitch_of(K), scales, M, w_codes, w_scales, N, K, bias, bias_dtype, out, dtype, ld_out,
                   fast_accum, st);
}

}  // extern "C"
