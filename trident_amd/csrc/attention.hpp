// Shared by attention's forward and backward kernels: the sequences, and tiles of tokens in LDS.
#pragma once

#include "mfma.hpp"

namespace trident {

constexpr int kMaxHeadDim = 128;
constexpr int64_t kMaxGroups = 0xffffff;  // workgroups of 256 threads: a launch has fewer than 2^32 threads

struct AttentionArgs {
    const void *q, *k, *v, *grad;
    void *out, *dq, *dk, *dv;
    float* lse;    // [Hq, rows], base 2
    float* delta;  // [Hq, rows]
    float* part;   // of several shares: [2][shares][rows, Hkv, D]
    const void *offsets, *lengths;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // bytes
    int64_t rows, count;
    int slots;     // rows of a padded sequence, 0 if packed
    int wide;      // offsets and lengths are int64
    int Hq, Hkv, D, causal;
    int shares;
    int tiles;     // of all sequences, at most
    float scale, scale2;  // scale2 = scale log2(e)
};

// A tile of `size` rows of one sequence: rows first .. of [start, start + extent), the first `length` of
// them tokens.
struct SequenceTile {
    int64_t start;
    int first, length, extent;
};

__device__ __forceinline__ int64_t sequence_value(const void* p, int wide, int64_t i) {
    return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// The tile with number `tile`; false where there is none.  Padded sequences have a fixed number of tiles.
// Packed ones begin at tile offset / size + index, which leaves each enough and at most one too many: so no
// kernel has to lay the tiles out first, and the sequence is found by a search in which a wave's lanes probe 64
// places at a time.  The rows before the first and after the last offset are sequences without tokens. Values
// outside [0, rows] are brought inside, so whatever the offsets are, no row outside the tensors is touched.
__device__ __forceinline__ bool find_tile(const AttentionArgs& a, int tile, int size, SequenceTile* t) {
    if (a.slots) {
        const int each = (a.slots + size - 1) / size, b = tile / each;
        t->first = (tile - b * each) * size;
        t->start = (int64_t)b * a.slots;
        t->extent = a.slots;
        t->length = a.slots;
        if (a.lengths) {
            const int64_t m = sequence_value(a.lengths, a.wide, b);
            t->length = (int)min(max(m, (int64_t)0), (int64_t)a.slots);
        }
        return true;
    }
    const auto bound = [&](int64_t j) -> int64_t {  // where sequence j begins, 0 .. count + 2
        if (j == 0) return 0;
        if (j > a.count + 1) return a.rows;
        return min(max(sequence_value(a.offsets, a.wide, j - 1), (int64_t)0), a.rows);
    };
    int64_t low = 0, left = a.count + 2;
    while (left > 1) {
        const int64_t step = (left + kWave - 1) / kWave, at = lane_id() * step;
        const bool before = at < left && bound(low + at) / size + low + at <= tile;
        const int k = max(__popcll(__ballot(before)) - 1, 0);
        low += k * step;
        left = min(step, left - k * step);
    }
    const int64_t start = bound(low), end = bound(low + 1);
    // one value in all lanes
    t->start = (int64_t)__builtin_amdgcn_readfirstlane((int)start);
    t->extent = __builtin_amdgcn_readfirstlane((int)max(end - start, (int64_t)0));
    const int64_t at = tile - (start / size + low);
    t->first = __builtin_amdgcn_readfirstlane((int)min(max(at, (int64_t)-1), (int64_t)(0x7fffffff / size)) * size);
    t->length = low >= 1 && low <= a.count ? t->extent : 0;
    return t->first >= 0 && t->first < t->extent;
}

// A workgroup's tile of queries and head.  Tiles in the order of their work where they differ (causal: a
// sequence's last ones first), so that the longest do not begin last; for each the heads, the key heads
// changing fastest: workgroups go to the eight XCDs in turn, so with eight key heads each XCD's L2 sees one.
__device__ __forceinline__ void tile_and_head(const AttentionArgs& a, int* tile, int* h, int* hk) {
    const int at = blockIdx.x / a.Hq, j = blockIdx.x % a.Hq;
    *tile = a.causal ? a.tiles - 1 - at : at;
    *hk = j % a.Hkv;
    *h = *hk * (a.Hq / a.Hkv) + j / a.Hkv;
}

template <typename T, int DP>
constexpr int kTilePitch = sizeof(T) == 2 ? (DP <= 32 ? 64 : DP <= 64 ? 128 : 256) : (DP <= 32 ? 128 : DP <= 64 ? 256 : 512);
// tokens of a tile in LDS
template <typename T>
constexpr int kTileRows = sizeof(T) == 2 ? 64 : 32;

// One wave's share of loading rows 0 .. ROWS - 1 at `p` (pitch `row` bytes, `live` of them there) to LDS.
// Rows past the live ones and columns past D bytes become zeros: what lies there is never multiplied.
template <typename T, int PITCH, int ROWS, int WAVES>
__device__ __forceinline__ void fetch_tile(lds_bytes to, const void* p, int64_t row, int live, int bytes, int wave) {
    using L = Tile<T, PITCH>;
    constexpr int kLoads = ROWS / L::kRowsAtOnce;
    // (read from one lane: of min and max the compiler makes a vector instruction, and of a descriptor in vector registers a
    // loop over the lanes for every load)
    const int there = __builtin_amdgcn_readfirstlane(max(min(live, ROWS), 0));
    const __amdgpu_buffer_rsrc_t buf = buffer_of(p, (uint32_t)(there * (int)row));
    const int lane = lane_id(), in = lane / L::kPieces, slot = lane % L::kPieces;
#pragma unroll
    for (int i = 0; i < (kLoads + WAVES - 1) / WAVES; ++i) {
        const int load = i * WAVES + wave;
        if (kLoads % WAVES != 0 && load >= kLoads) break;
        const int r = load * L::kRowsAtOnce + in, piece = slot ^ L::exchange(r);
        const uint32_t at = piece * 16 < bytes ? (uint32_t)r * (uint32_t)row + piece * 16 : kPastBuffer;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (lds_ptr)(to + load * 1024), 16, at, 0, 0, 0);
    }
}

// This lane's row as operand fragments, straight from memory; zeros past D.
template <typename T, int DP>
__device__ __forceinline__ void load_row(const void* p, int D, frag<T> (&f)[DP / 16]) {
    const int half = lane_id() >> 5;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int col = 16 * s + 8 * half;
        f[s] = frag<T>{};
        if (col < D) f[s] = *reinterpret_cast<const frag<T>*>(static_cast<const T*>(p) + col);
    }
}

// Waits for a row's fragments: else every pass of a loop that uses them would wait for all of its loads.
template <typename F, int N>
__device__ __forceinline__ void arrived(F (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// Magnitudes from infinity on carry into the sign's place.
template <typename T>
struct NotFinite {
    static constexpr uint32_t kMask = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
    static constexpr uint32_t kCarry = sizeof(T) == 4                          ? 0x00800000u
                                       : std::is_same<T, bf16_t>::value ? 0x00800080u
                                                                               : 0x04000400u;
    uint32_t seen = 0;
    __device__ __forceinline__ void look(u32x4 w) {
#pragma unroll
        for (int e = 0; e < 4; ++e) seen |= (w[e] & kMask) + kCarry;
    }
    __device__ __forceinline__ bool any() const { return __any((seen & ~kMask) != 0); }  // in the wave
};

// Whether 32 rows of a tile hold a value that is not finite.
template <typename T, int PITCH>
__device__ __forceinline__ bool any_not_finite(lds_bytes rows) {
    typedef const __attribute__((address_space(3))) u32x4* words;
    NotFinite<T> n;
#pragma unroll
    for (int i = 0; i < PITCH / 32; ++i) n.look(*(words)(rows + i * 1024 + lane_id() * 16));
    return n.any();
}

// Whether the wave's rows do.
template <typename T, int N>
__device__ __forceinline__ bool any_not_finite(const frag<T> (&f)[N]) {
    NotFinite<T> n;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        u32x4 w[sizeof(f[i]) / 16];
        __builtin_memcpy(w, &f[i], sizeof(f[i]));
#pragma unroll
        for (const u32x4& part : w) n.look(part);
    }
    return n.any();
}

// The block on the diagonal of causal attention is seen in part by each column, and its product would add zero
// times infinity where a row that is not finite is not seen.  So there such values are multiplied as zeros
// (finite_only), and after the loop added to the columns that do see them (add_not_finite), from memory: slow,
// and rarely taken.
template <typename T>
__device__ __forceinline__ frag<T> finite_only(const frag<T>& f) {
    if constexpr (sizeof(T) == 2) {
        constexpr uint32_t kCarry = std::is_same<T, bf16_t>::value ? 0x00800080u : 0x04000400u;
        u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t past = ((w[e] & 0x7fff7fffu) + kCarry) & 0x80008000u;  // the sign's place: not finite
            w[e] &= ~((past >> 15) * 0xffffu);
        }
        return __builtin_bit_cast(frag<T>, w);
    } else {
        frag<T> g;
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = fabsf(f[e]) < INFINITY ? f[e] : 0.0f;
        return g;
    }
}

// The values that are not finite in `rows` rows at p (NANS: a NaN for each) to the columns that `sees(row)`
// names.
template <typename T, int DP, bool NANS, typename F>
__device__ __forceinline__ void add_not_finite(const void* p, int64_t pitch, int rows, int D, f32x16 (&acc)[DP / 32],
                                               F&& sees) {
    const int half = lane_id() >> 5;
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
        const T* x = reinterpret_cast<const T*>(static_cast<const uint8_t*>(p) + r * pitch);
        const bool seen = sees(r);
#pragma unroll
        for (int j = 0; j < DP / 32; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int col = 32 * j + 8 * (i / 4) + 4 * half + i % 4;
                const float v = col < D ? (float)x[col] : 0.0f;
                if (seen && !(fabsf(v) < INFINITY)) acc[j][i] += NANS ? NAN : v;
            }
    }
}

// Four consecutive columns of a row.
template <typename T>
__device__ __forceinline__ void store_quad(T* p, float a, float b, float c, float d) {
    const float f[4] = {a, b, c, d};
    store_vec(p, f);
}

// acc, a block column per lane (rows 32 j + 8 p + 4 half + {0..3} of it), times `by`, to the row at p.
template <typename T, int DP>
__device__ __forceinline__ void store_column(T* p, int D, const f32x16 (&acc)[DP / 32], float by) {
    const int half = lane_id() >> 5;
#pragma unroll
    for (int j = 0; j < DP / 32; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = 32 * j + 8 * i + 4 * half;
            if (col < D)
                store_quad(p + col, acc[j][4 * i] * by, acc[j][4 * i + 1] * by, acc[j][4 * i + 2] * by,
                           acc[j][4 * i + 3] * by);
        }
}

// Rows first .. last - 1 of one head's result to zeros, by the whole workgroup.
template <typename T>
__device__ __forceinline__ void zero_rows(T* base, int64_t row, int first, int last, int D, int threads) {
    const int each = D / 8;
    for (int i = threadIdx.x; i < (last - first) * each; i += threads) {
        const float z[8] = {};
        store_vec(base + (first + i / each) * row + i % each * 8, z);
    }
}

int attention_check(const TridentAttention* t, bool backward, AttentionArgs* a);

}  // namespace trident
