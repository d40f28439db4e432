// Token embedding: rows of a table, scaled, and the table's gradient.
//
//   y[t, :] = s W[id_t, :]        id_t < 0: an empty slot of a padded batch, zeros; id_t >= V: NaN
//   dW[v, :] = s sum_{t : id_t = v} dY[t, :]
//
// The gradient is summed without float atomics, each row in the order of its tokens, so a call gives
// the same bits every time: the tokens are ordered by id (a stable counting sort), then every table
// row is summed over its tokens by one group of lanes and written once, rows without tokens as zeros.
#include <algorithm>

#include "encoder.hpp"

namespace trident {
namespace {

struct EmbedArgs {
    const void* weight;  // [V, ld]
    const void* ids;     // [n]
    void* out;           // [n, ldo]
    int64_t n, V, ld, ldo;
    int D, nv;           // nv: vectors of a row
    float scale;
};

constexpr int kEmbedUnroll = 4;

// Bound by bytes: the rows' vectors of all tokens, one after the other, are dealt to the lanes, so a
// row of any length leaves no lane idle; four independent gathers per lane cover the latency of the
// id and of the row behind it.
template <typename T, int VEC, typename ID>
__global__ __launch_bounds__(kBlock) void embed_kernel(EmbedArgs a) {
    const int64_t base = (int64_t)blockIdx.x * (kBlock * kEmbedUnroll);
    const int64_t row0 = base / a.nv;
    const uint32_t c0 = (uint32_t)(base - row0 * a.nv);
    const ID* ids = static_cast<const ID*>(a.ids);
    const T* W = static_cast<const T*>(a.weight);
    T* out = static_cast<T*>(a.out);
    int64_t row[kEmbedUnroll], id[kEmbedUnroll];
    int col[kEmbedUnroll];
    float f[kEmbedUnroll][VEC];
#pragma unroll
    for (int u = 0; u < kEmbedUnroll; ++u) {
        const uint32_t at = c0 + threadIdx.x + u * kBlock;
        const uint32_t r = at / (uint32_t)a.nv;
        row[u] = row0 + r;
        col[u] = min((int)(at - r * a.nv) * VEC, a.D - VEC);
        id[u] = row[u] < a.n ? (int64_t)ids[row[u]] : -1;
    }
#pragma unroll
    for (int u = 0; u < kEmbedUnroll; ++u) {
        if (id[u] >= 0 && id[u] < a.V) {
            load_vec(W + id[u] * a.ld + col[u], f[u]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[u][i] *= a.scale;
        } else {
            const float none = id[u] < 0 ? 0.0f : __uint_as_float(0x7fc00000u);
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[u][i] = none;
        }
    }
#pragma unroll
    for (int u = 0; u < kEmbedUnroll; ++u)
        if (row[u] < a.n) store_vec(out + row[u] * a.ldo + col[u], f[u]);
}

// ---------------------------------------------------------------------------------------------
// gradient

constexpr int kSortBlock = 1024;
constexpr int kSortWaves = kSortBlock / kWave;
constexpr int kSortAhead = 8;   // groups of 64 ids a wave loads at once
constexpr int kMaxOwned = 512;  // ids a sorting workgroup owns at most (32 KB of counters)
constexpr int kChunk = 64;      // tokens of a part of a long row; longer rows are split

// Orders the tokens by id.  A workgroup owns `w` consecutive ids and reads all n ids twice: first it
// counts the tokens of smaller ids and, per wave, those of each id it owns (each wave takes a
// contiguous part of the tokens), which gives every (id, wave) its first place; then it places its
// tokens in order.  row_off[v] .. row_off[v + 1] are the places of id v in pos.  One launch, no
// workgroup waits for another.
template <typename ID>
__global__ __launch_bounds__(kSortBlock) void sort_ids_kernel(const ID* __restrict__ ids, int n, int V, int w,
                                                              int64_t skip, int* __restrict__ row_off,
                                                              int* __restrict__ pos) {
    extern __shared__ int hist[];  // [kSortWaves][w]
    __shared__ int s_sum[kSortWaves];
    const int lane = lane_id(), wave = threadIdx.x / kWave;
    const int lo = blockIdx.x * w, owned = min(w, V - lo);
    const int seg = (n + kSortBlock - 1) / kSortBlock * kWave;
    const int beg = (int)min((int64_t)n, (int64_t)wave * seg), end = (int)min((int64_t)n, (int64_t)beg + seg);
    for (int i = threadIdx.x; i < kSortWaves * w; i += kSortBlock) hist[i] = 0;
    __syncthreads();
    int* mine = hist + wave * w;
    int lower = 0;
    for (int t0 = beg; t0 < end; t0 += kWave * kSortAhead) {
        int64_t id[kSortAhead];
#pragma unroll
        for (int u = 0; u < kSortAhead; ++u) {
            const int t = t0 + u * kWave + lane;
            id[u] = t < end ? (int64_t)ids[t] : -1;
        }
#pragma unroll
        for (int u = 0; u < kSortAhead; ++u) {
            if (id[u] < 0 || id[u] == skip) continue;
            const int64_t rel = id[u] - lo;
            if (rel < 0) ++lower;
            else if (rel < owned) atomicAdd(&mine[rel], 1);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) lower += __shfl_xor(lower, o, kWave);
    if (lane == 0) s_sum[wave] = lower;
    __syncthreads();
    int place = 0;
    for (int i = 0; i < kSortWaves; ++i) place += s_sum[i];
    __syncthreads();
    // thread j: the first place of id lo + j
    const int j = threadIdx.x;
    int count = 0;
    if (j < owned)
        for (int i = 0; i < kSortWaves; ++i) count += hist[i * w + j];
    int inc = count;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int t = __shfl_up(inc, o, kWave);
        if (lane >= o) inc += t;
    }
    if (lane == kWave - 1) s_sum[wave] = inc;
    __syncthreads();
    for (int i = 0; i < wave; ++i) place += s_sum[i];
    place += inc - count;
    if (j < owned) {
        row_off[lo + j] = place;
        if (lo + j == V - 1) row_off[V] = place + count;
        for (int i = 0; i < kSortWaves; ++i) {
            const int c = hist[i * w + j];
            hist[i * w + j] = place;
            place += c;
        }
    }
    __syncthreads();
    for (int t0 = beg; t0 < end; t0 += kWave * kSortAhead) {
        int rel[kSortAhead];
#pragma unroll
        for (int u = 0; u < kSortAhead; ++u) {
            const int t = t0 + u * kWave + lane;
            const int64_t id = t < end ? (int64_t)ids[t] : -1;
            const int64_t r = id - lo;
            rel[u] = id >= 0 && id != skip && r >= 0 && r < owned ? (int)r : -1;
        }
#pragma unroll
        for (int u = 0; u < kSortAhead; ++u) {
            const int t = t0 + u * kWave + lane;
            uint64_t left = __ballot(rel[u] >= 0);
            while (left) {  // one turn per id among these 64 tokens
                const int first = __ffsll((unsigned long long)left) - 1;
                const int r = __builtin_amdgcn_readlane(rel[u], first);
                const uint64_t same = __ballot(rel[u] == r);
                const int at = mine[r];
                if (rel[u] == r) pos[at + mask_rank(same)] = t;
                wave_sync();
                if (lane == first) mine[r] = at + __popcll((unsigned long long)same);
                wave_sync();
                left &= ~same;
            }
        }
    }
}

struct EmbedGradArgs {
    const void* grad;     // [n, ld]
    const void* ids;      // [n]
    const int* row_off;   // [V + 1]
    const int* pos;       // tokens by id
    float* part;          // [2 chunks, D]: sums of the parts of long rows
    void* out;            // [V, ldo]
    int64_t ld, ldo;
    int V, D, nv;
    int lanes;            // lanes of a row: a power of two, 64 where a row has more vectors
    int row_blocks;       // workgroups that take whole rows; the others take chunks
    float scale;
};

// Sums the gradient rows of the tokens pos[beg .. end), every `step`-th, into acc; four rows are in
// flight, added in order.
template <typename T, int VEC, int NVL>
__device__ __forceinline__ void sum_rows(const EmbedGradArgs& a, int beg, int end, int step, const int (&col)[NVL],
                                         const bool (&on)[NVL], float (&acc)[NVL][VEC]) {
    const T* g = static_cast<const T*>(a.grad);
    int k = beg;
    for (; k + 3 * step < end; k += 4 * step) {
        float f[4][NVL][VEC];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const T* row = g + (int64_t)a.pos[k + u * step] * a.ld;
#pragma unroll
            for (int c = 0; c < NVL; ++c)
                if (on[c]) load_vec(row + col[c], f[u][c]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int c = 0; c < NVL; ++c)
                if (on[c])
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[c][i] += f[u][c][i];
    }
    for (; k < end; k += step) {
        const T* row = g + (int64_t)a.pos[k] * a.ld;
#pragma unroll
        for (int c = 0; c < NVL; ++c)
            if (on[c]) {
                float f[VEC];
                load_vec(row + col[c], f);
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[c][i] += f[i];
            }
    }
}

// The two rows that a chunk of kChunk ordered tokens can hold a part of a long row of: the row of its
// first token and that of its last.
template <typename ID>
struct ChunkRows {
    int beg, end;       // the chunk's places
    int row[2], lo[2], hi[2];
    bool is_long[2];
    __device__ __forceinline__ bool init(const EmbedGradArgs& a, int chunk) {
        const int live = a.row_off[a.V];
        beg = chunk * kChunk;
        if (beg >= live) return false;
        end = min(live, beg + kChunk);
        const ID* ids = static_cast<const ID*>(a.ids);
        row[0] = (int)ids[a.pos[beg]];
        row[1] = (int)ids[a.pos[end - 1]];
        for (int i = 0; i < 2; ++i) {
            lo[i] = a.row_off[row[i]];
            hi[i] = a.row_off[row[i] + 1];
            is_long[i] = hi[i] - lo[i] > kChunk && (i == 0 || row[1] != row[0]);
        }
        return is_long[0] || is_long[1];
    }
};

// Bound by bytes.  Rows of up to kChunk tokens: a group of lanes per row, each lane the same columns
// of every token.  Longer rows (frequent tokens): the ordered tokens are cut into chunks of kChunk, a
// workgroup sums what its chunk holds of long rows into `part` (at most two: the row it begins in and
// the row it ends in), and join_long_kernel adds a row's parts in order.
template <typename T, int VEC, int NVL, typename ID>
__global__ __launch_bounds__(kBlock) void embed_grad_kernel(EmbedGradArgs a) {
    extern __shared__ float sums[];  // [groups][lanes * NVL * VEC]
    const int groups = kBlock / a.lanes;
    const int group = threadIdx.x / a.lanes, l = threadIdx.x % a.lanes;
    int col[NVL];
    bool on[NVL];
    float acc[NVL][VEC];
#pragma unroll
    for (int c = 0; c < NVL; ++c) {
        const int v = (blockIdx.y * NVL + c) * a.lanes + l;
        on[c] = v < a.nv;
        col[c] = min(v * VEC, a.D - VEC);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[c][i] = 0.0f;
    }
    if ((int)blockIdx.x < a.row_blocks) {
        const int row = blockIdx.x * groups + group;
        if (row >= a.V) return;
        const int beg = a.row_off[row], end = a.row_off[row + 1];
        if (end - beg > kChunk) return;
        sum_rows<T, VEC, NVL>(a, beg, end, 1, col, on, acc);
        T* out = static_cast<T*>(a.out) + (int64_t)row * a.ldo;
#pragma unroll
        for (int c = 0; c < NVL; ++c)
            if (on[c]) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[c][i] *= a.scale;
                store_vec(out + col[c], acc[c]);
            }
        return;
    }
    const int chunk = blockIdx.x - a.row_blocks;
    ChunkRows<ID> rows;
    if (!rows.init(a, chunk)) return;
    for (int i = 0; i < 2; ++i) {
        if (!rows.is_long[i]) continue;  // the same in every lane
        const int beg = max(rows.beg, rows.lo[i]), end = min(rows.end, rows.hi[i]);
#pragma unroll
        for (int c = 0; c < NVL; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[c][e] = 0.0f;
        sum_rows<T, VEC, NVL>(a, beg + group, end, groups, col, on, acc);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < NVL; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) sums[(c * VEC + e) * kBlock + threadIdx.x] = acc[c][e];
        __syncthreads();
        if (group == 0) {
#pragma unroll
            for (int c = 0; c < NVL; ++c) {
                if (!on[c]) continue;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    float s = 0.0f;
                    for (int g = 0; g < groups; ++g) s += sums[(c * VEC + e) * kBlock + g * a.lanes + l];
                    a.part[(int64_t)(2 * chunk + i) * a.D + col[c] + e] = s;
                }
            }
        }
    }
}

// Adds the parts of the long row that begins in this chunk (at most one does: a long row reaches into
// the next chunk).
template <typename T, typename ID>
__global__ __launch_bounds__(kBlock) void join_long_kernel(EmbedGradArgs a) {
    ChunkRows<ID> rows;
    const int chunk = blockIdx.x;
    if (!rows.init(a, chunk)) return;
    for (int i = 0; i < 2; ++i) {
        if (!rows.is_long[i] || rows.lo[i] < rows.beg) continue;
        const int last = (rows.hi[i] - 1) / kChunk;
        T* out = static_cast<T*>(a.out) + (int64_t)rows.row[i] * a.ldo;
        for (int d = blockIdx.y * kBlock + threadIdx.x; d < a.D; d += gridDim.y * kBlock) {
            float s = a.part[(int64_t)(2 * chunk + i) * a.D + d];
#pragma unroll 8
            for (int c = chunk + 1; c <= last; ++c) s += a.part[(int64_t)(2 * c) * a.D + d];
            out[d] = (T)(s * a.scale);
        }
    }
}

template <typename F>
void with_ids(int32_t ids64, F&& f) {
    if (ids64) f(int64_t{});
    else f(int32_t{});
}

struct GradSpace {
    int* row_off;
    int* pos;
    float* part;
    size_t bytes;
};

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

GradSpace grad_space(void* base, int64_t n, int64_t V, int64_t D) {
    GradSpace s;
    const size_t chunks = (size_t)((n + kChunk - 1) / kChunk);
    const size_t off = up256((size_t)(V + 1) * 4), pos = up256((size_t)n * 4);
    char* p = static_cast<char*>(base);
    s.row_off = reinterpret_cast<int*>(p);
    s.pos = reinterpret_cast<int*>(p + off);
    s.part = reinterpret_cast<float*>(p + off + pos);
    s.bytes = off + pos + up256(2 * chunks * (size_t)D * 4);
    return s;
}

constexpr int64_t kMaxCount = 0x7fffffff - 4 * kSortBlock;  // tokens, rows and columns count in 32 bits

}  // namespace
}  // namespace trident

using namespace trident;

extern "C" {

int trident_embedding(const void* weight, int32_t dtype, int64_t V, int64_t D, int64_t ld_weight, const void* ids,
                      int32_t ids64, int64_t n, double scale, void* out, int64_t ld_out, void* stream) {
    if (!dtype_ok(dtype)) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "embedding: dtype=%d", dtype);
    if (V < 1 || D < 1 || n < 0 || V > kMaxCount || D > kMaxCount || n > kMaxCount || ld_weight < D || ld_out < D)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "embedding: bad sizes V=%lld D=%lld n=%lld ld=%lld, %lld",
                         (long long)V, (long long)D, (long long)n, (long long)ld_weight, (long long)ld_out);
    if (n == 0) return TRIDENT_OK;
    if (!weight || !ids || !out) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "embedding: NULL pointer");
    int rc = TRIDENT_OK;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        with_ids(ids64, [&](auto i) {
            using ID = decltype(i);
            EmbedArgs a{weight, ids, out, n, V, ld_weight, ld_out, (int)D, 0, (float)scale};
            const int vec = D >= kVec<T> ? kVec<T> : 1;
            a.nv = (int)((D + vec - 1) / vec);
            const int64_t per = kBlock * kEmbedUnroll, blocks = (n * a.nv + per - 1) / per;
            if (blocks > 0x7fffffff) {
                rc = capi_fail(TRIDENT_ERR_UNSUPPORTED, "embedding: n * D = %lld is too large", (long long)(n * D));
                return;
            }
            hipStream_t st = static_cast<hipStream_t>(stream);
            if (vec > 1) embed_kernel<T, kVec<T>, ID><<<(unsigned)blocks, kBlock, 0, st>>>(a);
            else embed_kernel<T, 1, ID><<<(unsigned)blocks, kBlock, 0, st>>>(a);
            rc = capi_check_launch("embed_kernel");
        });
    });
    return rc;
}

size_t trident_embedding_grad_workspace_bytes(int64_t n, int64_t V, int64_t D) {
    if (n < 0 || V < 1 || D < 1 || n > kMaxCount || V > kMaxCount || D > kMaxCount) return 0;
    return grad_space(nullptr, n, V, D).bytes;
}

int trident_embedding_grad(const void* grad, int32_t dtype, int64_t ld_grad, const void* ids, int32_t ids64,
                           int64_t n, int64_t V, int64_t D, double scale, int64_t padding_idx, void* out,
                           int64_t ld_out, void* workspace, size_t workspace_bytes, void* stream) {
    if (!dtype_ok(dtype)) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "embedding_grad: dtype=%d", dtype);
    if (V < 1 || D < 1 || n < 0 || V > kMaxCount || D > kMaxCount || n > kMaxCount || ld_grad < D || ld_out < D)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "embedding_grad: bad sizes V=%lld D=%lld n=%lld ld=%lld, %lld",
                         (long long)V, (long long)D, (long long)n, (long long)ld_grad, (long long)ld_out);
    if (!out || (n > 0 && (!grad || !ids)))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "embedding_grad: NULL pointer");
    const GradSpace s = grad_space(workspace, n, V, D);
    if (!workspace || workspace_bytes < s.bytes)
        return capi_fail(TRIDENT_ERR_WORKSPACE_TOO_SMALL, "embedding_grad: workspace %zu < %zu bytes", workspace_bytes,
                         s.bytes);
    hipStream_t st = static_cast<hipStream_t>(stream);
    int rc = TRIDENT_OK;
    with_ids(ids64, [&](auto i) {
        using ID = decltype(i);
        // one workgroup per CU where the ids they own allow it
        const int w = (int)std::min<int64_t>(kMaxOwned, (V + 255) / 256);
        sort_ids_kernel<ID><<<(unsigned)((V + w - 1) / w), kSortBlock, sizeof(int) * kSortWaves * w, st>>>(
            static_cast<const ID*>(ids), (int)n, (int)V, w, padding_idx, s.row_off, s.pos);
        if ((rc = capi_check_launch("sort_ids_kernel"))) return;
        with_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            EmbedGradArgs a{grad, ids, s.row_off, s.pos, s.part, out, ld_grad, ld_out, (int)V, (int)D, 0, 0, 0,
                            (float)scale};
            const int vec = D >= kVec<T> ? kVec<T> : 1;
            a.nv = (int)((D + vec - 1) / vec);
            a.lanes = 1;
            while (a.lanes < a.nv && a.lanes < kWave) a.lanes *= 2;
            const int nvl = std::min(4, (a.nv + kWave - 1) / kWave);
            const int groups = kBlock / a.lanes;
            a.row_blocks = (int)((V + groups - 1) / groups);
            const int64_t chunks = (n + kChunk - 1) / kChunk;
            const unsigned tiles = (unsigned)((a.nv + nvl * a.lanes - 1) / (nvl * a.lanes));
            if (tiles > 65535) {
                rc = capi_fail(TRIDENT_ERR_UNSUPPORTED, "embedding_grad: D=%lld is too large", (long long)D);
                return;
            }
            const dim3 grid((unsigned)(a.row_blocks + chunks), tiles);
            const size_t lds = (size_t)kBlock * nvl * vec * sizeof(float);
            if (vec == 1) embed_grad_kernel<T, 1, 1, ID><<<grid, kBlock, lds, st>>>(a);
            else if (nvl == 1) embed_grad_kernel<T, kVec<T>, 1, ID><<<grid, kBlock, lds, st>>>(a);
            else if (nvl == 2) embed_grad_kernel<T, kVec<T>, 2, ID><<<grid, kBlock, lds, st>>>(a);
            else if (nvl == 3) embed_grad_kernel<T, kVec<T>, 3, ID><<<grid, kBlock, lds, st>>>(a);
            else embed_grad_kernel<T, kVec<T>, 4, ID><<<grid, kBlock, lds, st>>>(a);
            if ((rc = capi_check_launch("embed_grad_kernel")) || n <= kChunk) return;
            const dim3 join((unsigned)chunks, (unsigned)std::min<int64_t>(64, (D + kBlock - 1) / kBlock));
            join_long_kernel<T, ID><<<join, kBlock, 0, st>>>(a);
            rc = capi_check_launch("join_long_kernel");
        });
    });
    return rc;
}

}  // extern "C"
