// Shared by the transformer layer's kernels (attention.hip, attention_grad.hip, gated.hip): products of 32 x 32
// blocks in any of the three element types, and operand tiles in LDS that are read by rows or by columns.
//
// A block product takes 16 steps of the summed axis from both operands; a lane passes eight of them, lanes 0 to
// 31 one half and lanes 32 to 63 the other, for row (first operand) or column (second) lane % 32. Which eight
// is free as long as both operands agree.  float32 takes eight instructions of two steps, so all types share
// one layout.  The result's column is lane % 32, its rows 8 (i / 4) + 4 (lane / 32) + i % 4 for i < 16: the
// eight of registers 8 s to 8 s + 7 are 16 s + 4 half + {0..3, 8..11}.  So a result can be the second operand
// of the next product as it is, if the first one's columns are read in that order (col_frag): no lane exchanges
// anything.
#pragma once

#include "encoder.hpp"

namespace trident {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef __attribute__((address_space(3))) uint8_t* lds_bytes;

template <typename T>
struct FragOf {
    typedef T type __attribute__((ext_vector_type(8)));
};
template <typename T>
using frag = typename FragOf<T>::type;

template <typename T>
__device__ __forceinline__ f32x16 mma(const frag<T>& a, const frag<T>& b, f32x16 c) {
    if constexpr (std::is_same<T, bf16_t>::value) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    else if constexpr (std::is_same<T, f16_t>::value) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    else {
#pragma unroll
        for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
}

// A tile in LDS: rows of PITCH bytes (a power of two from 64 on), cut into pieces of 16 bytes.  A piece is
// stored exchanged by some bits of its row's number, so that the lanes of either kind of read meet all of LDS's
// 64 banks: 16 lanes that read one piece of as many rows, and 32 lanes that read four pieces of four rows each.
template <typename T, int PITCH>
struct Tile {
    static constexpr int kPieces = PITCH / 16, kPer = 16 / (int)sizeof(T);
    static constexpr int kRowsAtOnce = 1024 / PITCH;  // rows that one load of a wave fills
    static_assert(PITCH >= 64 && (PITCH & (PITCH - 1)) == 0, "pieces are exchanged by exclusive or");

    static __device__ __forceinline__ int exchange(int row) {
        constexpr int shared = PITCH >= 256 ? 0 : PITCH == 128 ? 1 : 2;  // bits of the row within 256 bytes
        return ((row & 3) >> shared) << 2 | (row >> 2 & 3);
    }

    // Eight steps of this lane's row `row`: those of columns 16 step + 8 half.
    static __device__ __forceinline__ frag<T> row_frag(lds_bytes tile, int row, int step) {
        const int half = lane_id() >> 5, by = exchange(row);
        if constexpr (sizeof(T) == 2) {
            typedef const __attribute__((address_space(3))) u32x4* words;
            return __builtin_bit_cast(frag<T>, *(words)(tile + row * PITCH + (((2 * step + half) ^ by) << 4)));
        } else {
            typedef const __attribute__((address_space(3))) f32x4* words;
            const f32x4 lo = *(words)(tile + row * PITCH + (((4 * step + 2 * half) ^ by) << 4));
            const f32x4 hi = *(words)(tile + row * PITCH + (((4 * step + 2 * half + 1) ^ by) << 4));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }

    // Eight rows of this lane's column col + lane % 32: rows row + 4 half + {0..3, 8..11} (a result's), or
    // row + 8 half + {0..7} (a row_frag's); row and col are multiples of 16 and 32.  16-bit types by the
    // transposing read: of 16 lanes that read 4 x 16 elements, each gets a column of four.
    template <bool ROW_ORDER>
    static __device__ __forceinline__ frag<T> read_columns(lds_bytes tile, int row, int col) {
        const int lane = lane_id(), first = (ROW_ORDER ? 8 : 4) * (lane >> 5);
        constexpr int kNext = ROW_ORDER ? 4 : 8;
        if constexpr (sizeof(T) == 2) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4* quads;
            const int in = first + (lane >> 2 & 3);  // of 16 rows
            const int piece = (lane >> 4 & 1) * 2 + (lane >> 1 & 1) + col / 8;
            const lds_bytes at = tile + (row + in) * PITCH + (lane & 1) * 8;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((quads)(at + ((piece ^ exchange(in)) << 4)));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (quads)(at + kNext * PITCH + ((piece ^ exchange(in + kNext)) << 4)));
            return __builtin_bit_cast(frag<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            typedef const __attribute__((address_space(3))) float* one;
            const int piece = (lane & 31) / 4 + col / 4;
            frag<T> f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int in = first + i % 4 + i / 4 * kNext;
                f[i] = *(one)(tile + (row + in) * PITCH + ((piece ^ exchange(in)) << 4) + (lane & 3) * 4);
            }
            return f;
        }
    }
    static __device__ __forceinline__ frag<T> col_frag(lds_bytes tile, int row, int col) {
        return read_columns<false>(tile, row, col);
    }
    static __device__ __forceinline__ frag<T> col_frag_in_order(lds_bytes tile, int row, int col) {
        return read_columns<true>(tile, row, col);
    }
};

// A barrier for waves that hold what they read from LDS.
__device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A lane's places in such tiles, made once: of its first row's DP / 16 steps, and of its first column of DP /
// 32 blocks, in a result's order.  A read is then one addition and a constant.
template <typename T, int PITCH, int DP>
struct TileReader {
    using L = Tile<T, PITCH>;
    static constexpr bool kPlaces = sizeof(T) == 2;
    uint32_t row_at[DP / 16], col_at[2][DP / 32];

    __device__ __forceinline__ TileReader() {
        if constexpr (kPlaces) {
            const int lane = lane_id(), row = lane & 31, half = lane >> 5;
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                row_at[i] = row * PITCH + (((2 * i + half) ^ L::exchange(row)) << 4);
                asm volatile("" : "+v"(row_at[i]));  // not made again for every read
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    const int in = 4 * half + (lane >> 2 & 3) + 8 * h;
                    const int piece = (lane >> 4 & 1) * 2 + (lane >> 1 & 1) + 4 * j;
                    col_at[h][j] = in * PITCH + (lane & 1) * 8 + ((piece ^ L::exchange(in)) << 4);
                    asm volatile("" : "+v"(col_at[h][j]));
                }
        }
    }
    // row_frag of row block * 32 + lane % 32
    __device__ __forceinline__ frag<T> rows(lds_bytes tile, int block, int step) const {
        if constexpr (kPlaces) {
            typedef const __attribute__((address_space(3))) u32x4* words;
            return __builtin_bit_cast(frag<T>, *(words)(tile + row_at[step] + block * 32 * PITCH));
        } else {
            return L::row_frag(tile, block * 32 + (lane_id() & 31), step);
        }
    }
    // col_frag of columns j * 32 ..
    __device__ __forceinline__ frag<T> columns(lds_bytes tile, int row, int j) const {
        if constexpr (kPlaces) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4* quads;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((quads)(tile + col_at[0][j] + row * PITCH));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((quads)(tile + col_at[1][j] + row * PITCH));
            return __builtin_bit_cast(frag<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            return L::col_frag(tile, row, j * 32);
        }
    }
};

// A buffer of `bytes` from p on: loads past it give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00027000);
}
constexpr uint32_t kPastBuffer = 0x80000000u;  // an offset past any buffer here

// Past this barrier every wave's loads to LDS have arrived but for the last N of each, and every wave has what
// it read from LDS.
template <int N>
__device__ __forceinline__ void wait_and_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The other half's value of the same row or column.
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, kWave); }

}  // namespace trident
