// Token embedding: rows of a table, scaled, and the table's gradient.
//
//   y[t, :] = s W[id_t, :]        id_t < 0: an empty slot of a padded batch, zeros; id_t >= V: NaN
//   dW[v, :] = s sum_{t : id_t = v} dY[t, :]
//
// The gradient is summed without float atomics, so a call gives the same bits every time: the tokens are
// ordered by id (a stable counting sort), and every table row is summed over its tokens and written once,
// rows without tokens as zeros.  A row of few tokens is summed in their order by one group of lanes, a longer
// one in parts, which are then added in order; where the parts begin goes by the sizes and the other ids.
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
// id and of the row behind it.  131,072 tokens x 960 bfloat16 of 65,536 rows: 46 us, 5.5 TB/s written
// and as much read, mostly from the caches.
template <typename T, int VEC, typename ID, bool PAST_L2>
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
        if (row[u] < a.n) put_vec<PAST_L2>(out + row[u] * a.ldo + col[u], f[u]);
}

// ---------------------------------------------------------------------------------------------
// gradient

constexpr int kOwned = 512;      // ids of one sorting workgroup, of a table of up to kMaxBuckets of them;
constexpr int kMaxOwned = 2048;  // of a larger table

struct RowInfo {
    int beg, count;  // a row's places among the ordered tokens
};

// Where a table row's RowInfo lies: those of one sorting workgroup (ids equal modulo 2^shift) next to
// one another, so that it writes whole lines.
__device__ __forceinline__ int64_t info_at(int v, int shift, int owned) {
    return (int64_t)(v & ((1 << shift) - 1)) * owned + (v >> shift);
}

struct Token {
    int t, row;
};

// Tokens ordered in one launch, and not in two: four waves can keep all of them.  The whole gradient,
// 768 columns, one and two: 4,096 tokens 22.0 and 26.4 us, 8,192 25.8 and 26.5, 12,288 33.3 and 32.3,
// 16,384 38.5 and 34.7.
constexpr int kSmallTokens = 4 * 2048;
constexpr int kPartTokens = 1024;       // tokens that bucket_ids_kernel orders at a time
constexpr int kMaxBuckets = 1024;

struct SortArgs {
    const void* ids;
    int n, V, owned, shift, chunk, parts;
    uint32_t skip;     // an id without a gradient; 2^32 - 1: none
    RowInfo* row;      // [2^shift, owned], and one more: the number of all tokens
    Token* token;      // [n]
    int* long_count;   // [2^shift]
    int* long_rows;    // [2^shift, owned]
    Token* bucketed;   // [n]: each part's tokens by bucket (t, id)
    uint16_t* starts;  // [parts, 2^shift + 1]: the buckets' first places in their part
};

// An id if it is a row's that takes part, else 2^32 - 1.
template <bool SKIP>
__device__ __forceinline__ uint32_t row_id(int64_t id, uint32_t V, uint32_t skip) {
    return (uint64_t)id < V && !(SKIP && id == skip) ? (uint32_t)id : ~0u;
}
template <bool SKIP>
__device__ __forceinline__ uint32_t row_id(int32_t id, uint32_t V, uint32_t skip) {
    return (uint32_t)id < V && !(SKIP && (uint32_t)id == skip) ? (uint32_t)id : ~0u;
}

// The lanes whose key (of `bits` bits) equals this one's, among those with `in`: found bit by bit.
__device__ __forceinline__ uint64_t lanes_with(bool in, uint32_t key, int bits) {
    uint64_t same = __ballot(in);
    for (int i = 0; i < bits; ++i) {
        const bool set = (key >> i) & 1;
        const uint64_t m = __ballot(set);
        same &= set ? m : ~m;
    }
    return same;
}

// Inclusive sum over a workgroup of WAVES waves, and the total of all; two barriers.
template <int WAVES>
__device__ __forceinline__ int block_sum(int v, int* s_sum, int* total) {
    const int lane = lane_id(), wave = threadIdx.x / kWave;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int t = __shfl_up(v, o, kWave);
        if (lane >= o) v += t;
    }
    __syncthreads();
    if (lane == kWave - 1) s_sum[wave] = v;
    __syncthreads();
    int all = 0;
    for (int i = 0; i < WAVES; ++i) {
        if (i < wave) v += s_sum[i];
        all += s_sum[i];
    }
    *total = all;
    return v;
}

// Many tokens, first step: a part of kPartTokens of them is ordered by bucket, id modulo 2^shift, and
// the buckets' first places are written beside it.
template <typename ID, bool SKIP>
__global__ __launch_bounds__(kBlock) void bucket_ids_kernel(SortArgs a) {
    constexpr int G = kPartTokens / kBlock;
    __shared__ int hist[kWavesPerBlock * kMaxBuckets];
    __shared__ Token sorted[kPartTokens];
    __shared__ int s_sum[kWavesPerBlock];
    const int lane = lane_id(), wave = threadIdx.x / kWave, buckets = 1 << a.shift;
    const int t0 = blockIdx.x * kPartTokens + wave * (G * kWave) + lane;
    const ID* ids = static_cast<const ID*>(a.ids);
    uint32_t id[G];
#pragma unroll
    for (int u = 0; u < G; ++u) {
        const ID raw = ids[min(t0 + u * kWave, a.n - 1)];
        id[u] = t0 + u * kWave < a.n ? row_id<SKIP>(raw, (uint32_t)a.V, a.skip) : ~0u;
    }
    for (int i = threadIdx.x; i < kWavesPerBlock * buckets; i += kBlock) hist[i] = 0;
    __syncthreads();
    int* mine = hist + wave * buckets;
#pragma unroll
    for (int u = 0; u < G; ++u)
        if (id[u] != ~0u) atomicAdd(&mine[id[u] & (buckets - 1)], 1);
    __syncthreads();
    uint16_t* starts = a.starts + (int64_t)blockIdx.x * (buckets + 1);
    int place = 0;
    for (int j0 = 0; j0 < buckets; j0 += kBlock) {
        const int j = j0 + threadIdx.x;
        int count = 0, total;
        if (j < buckets)
            for (int i = 0; i < kWavesPerBlock; ++i) count += hist[i * buckets + j];
        int at = place + block_sum<kWavesPerBlock>(count, s_sum, &total) - count;
        place += total;
        if (j < buckets) {
            starts[j] = (uint16_t)at;
            for (int i = 0; i < kWavesPerBlock; ++i) {
                const int c = hist[i * buckets + j];
                hist[i * buckets + j] = at;
                at += c;
            }
        }
    }
    if (threadIdx.x == 0) starts[buckets] = (uint16_t)place;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < G; ++u) {
        const uint32_t key = id[u] & (buckets - 1);
        const uint64_t same = lanes_with(id[u] != ~0u, key, a.shift);
        if (id[u] != ~0u) {
            const int rank = mask_rank(same), at = mine[key];
            sorted[at + rank] = Token{t0 + u * kWave, (int)id[u]};
            wave_sync();
            if (rank == 0) mine[key] = at + __popcll((unsigned long long)same);
        }
        wave_sync();
    }
    __syncthreads();
    for (int i = threadIdx.x; i < place; i += kBlock) a.bucketed[(int64_t)blockIdx.x * kPartTokens + i] = sorted[i];
}

// What a sorting workgroup's waves read: all ids (FROM_PARTS false), or its bucket of every part.  A
// wave takes a contiguous share, and calls f(t, rel) for 64 tokens at a time in their order, rel < 0 in
// lanes without one; returns how many tokens of lower buckets its share has.
template <typename ID, int WAVES, bool SKIP, bool FROM_PARTS>
struct SortSource {
    template <typename F>
    static __device__ __forceinline__ int read(const SortArgs& a, F&& f) {
        const int lane = lane_id(), wave = threadIdx.x / kWave;
        const uint32_t b = blockIdx.x, mask = (1u << a.shift) - 1;
        int lower = 0;
        if constexpr (FROM_PARTS) {
            constexpr int A = 4;
            const int share = (a.parts + WAVES - 1) / WAVES, stride = (int)mask + 2;
            const int p0 = min(a.parts, wave * share), p1 = min(a.parts, p0 + share);
            for (int p = p0; p < p1; p += kWave) {
                const int mine = min(p + lane, p1 - 1);
                const int beg = a.starts[(int64_t)mine * stride + b];
                const int num = p + lane < p1 ? a.starts[(int64_t)mine * stride + b + 1] - beg : 0;
                lower += p + lane < p1 ? beg : 0;
                for (int q = 0; q < min(kWave, p1 - p); q += A) {
                    Token tok[A];
                    int n[A], s[A];
#pragma unroll
                    for (int u = 0; u < A; ++u) {
                        n[u] = __builtin_amdgcn_readlane(num, q + u);  // 0 past the share's end
                        s[u] = (p + q + u) * kPartTokens + __builtin_amdgcn_readlane(beg, q + u);
                        if (lane < n[u]) tok[u] = a.bucketed[s[u] + lane];
                    }
#pragma unroll
                    for (int u = 0; u < A; ++u) {
                        if (n[u] == 0) continue;
                        f(tok[u].t, lane < n[u] ? tok[u].row >> a.shift : -1);
                        for (int k = kWave; k < n[u]; k += kWave) {
                            const bool in = k + lane < n[u];
                            const Token more = in ? a.bucketed[s[u] + k + lane] : Token{0, 0};
                            f(more.t, in ? more.row >> a.shift : -1);
                        }
                    }
                }
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) lower += __shfl_xor(lower, o, kWave);
        } else {
            constexpr int A = 16;
            const int n = a.n, seg = (n + WAVES * kWave - 1) / (WAVES * kWave) * kWave;
            const int beg = (int)min((int64_t)n, (int64_t)wave * seg), end = (int)min((int64_t)n, (int64_t)beg + seg);
            const ID* ids = static_cast<const ID*>(a.ids);
            for (int t0 = beg; t0 < end; t0 += kWave * A) {
                ID raw[A];
#pragma unroll
                for (int u = 0; u < A; ++u) raw[u] = ids[min(t0 + u * kWave + lane, n - 1)];
#pragma unroll
                for (int u = 0; u < A; ++u) {
                    const int t = t0 + u * kWave + lane;
                    const uint32_t id = t < end ? row_id<SKIP>(raw[u], (uint32_t)a.V, a.skip) : ~0u;
                    const uint32_t owner = id == ~0u ? ~0u : id & mask;
                    lower += __popcll((unsigned long long)__ballot(owner < b));
                    if (__ballot(owner == b)) f(t, owner == b ? (int)(id >> a.shift) : -1);
                }
            }
        }
        return lower;
    }
};

template <int WAVES>
struct SortShape {
    static constexpr int kList = WAVES == 4 ? 2048 : 1024;  // tokens a wave keeps in LDS
    static constexpr size_t lds(int w) {
        return (size_t)WAVES * w * sizeof(int) + (size_t)WAVES * kList * (sizeof(int) + sizeof(uint16_t));
    }
};

// Orders the tokens by id: row[info_at(v)] says where in `token` the tokens of id v lie, in their own
// order; the last entry holds the number of all.  Workgroup b owns the ids = b modulo gridDim.x (a power
// of two): the most frequent ids of a vocabulary are neighbours, so a range of them would be one
// workgroup's work.  Each wave goes through its share of the tokens, keeps those its workgroup owns in a list in LDS, and
// counts them by id; the counts, and the number of tokens of lower workgroups, give every (id, wave)
// its first place, and the lists are placed in order.  A wave whose list overflows (an id with a large
// share of many tokens) goes through its share again instead.  No workgroup waits for another.
//
// Few tokens are read by every workgroup.  For many that is most of the time (131,072: 35 us), so they
// are bucketed first, which leaves each workgroup its own (5.4 + 13.4 us, most of it in the workgroups of
// the most frequent ids).
template <typename ID, int WAVES, bool SKIP, bool FROM_PARTS>
__global__ __launch_bounds__(WAVES* kWave) void sort_ids_kernel(SortArgs a) {
    using Source = SortSource<ID, WAVES, SKIP, FROM_PARTS>;
    constexpr int kList = SortShape<WAVES>::kList;
    extern __shared__ int lds[];
    __shared__ int s_sum[WAVES], s_long;
    const int w = a.owned, lane = lane_id(), wave = threadIdx.x / kWave;
    const uint32_t b = blockIdx.x;
    int* hist = lds;              // [WAVES][w]
    int* list = lds + WAVES * w;  // [WAVES][kList]
    uint16_t* list_id = reinterpret_cast<uint16_t*>(list + WAVES * kList);
    for (int i = threadIdx.x; i < WAVES * w; i += WAVES * kWave) hist[i] = 0;
    if (threadIdx.x == 0) s_long = 0;
    __syncthreads();
    int* mine = hist + wave * w;
    int* kept = list + wave * kList;
    uint16_t* kept_id = list_id + wave * kList;
    int found = 0;
    const int lower = Source::read(a, [&](int t, int rel) {
        const uint64_t m = __ballot(rel >= 0);
        if (!m) return;
        // the first token's id is counted at once: a frequent one would else be most lanes' atomic, one
        // after the other on one word, and all waves share the LDS unit (16.4 us where this takes 13.4)
        const int first = __ffsll((unsigned long long)m) - 1, id = __builtin_amdgcn_readlane(rel, first);
        const uint64_t same = __ballot(rel == id);
        if (lane == first) atomicAdd(&mine[id], __popcll((unsigned long long)same));
        if (rel >= 0) {
            const int at = found + mask_rank(m);
            if (rel != id) atomicAdd(&mine[rel], 1);
            if (at < kList) {
                kept[at] = t;
                kept_id[at] = (uint16_t)rel;
            }
        }
        found += __popcll((unsigned long long)m);
    });
    int place;
    block_sum<WAVES>(lane == 0 ? lower : 0, s_sum, &place);
    // the first place of each owned id, a workgroup's threads of them at a time
    for (int j0 = 0; j0 < w; j0 += WAVES * kWave) {
        const int j = j0 + threadIdx.x;
        const int64_t v = ((int64_t)j << a.shift) + b;
        const bool live = j < w && v < a.V;
        int count = 0, total;
        if (live)
            for (int i = 0; i < WAVES; ++i) count += hist[i * w + j];
        int at = place + block_sum<WAVES>(count, s_sum, &total) - count;
        place += total;
        if (live) {
            a.row[(int64_t)b * w + j] = RowInfo{at, count};
            if (count > a.chunk) a.long_rows[(int64_t)b * w + atomicAdd(&s_long, 1)] = (int)v;  // in any order
            for (int i = 0; i < WAVES; ++i) {
                const int c = hist[i * w + j];
                hist[i * w + j] = at;
                at += c;
            }
        }
    }
    if (b == gridDim.x - 1 && threadIdx.x == 0) a.row[(int64_t)gridDim.x * w] = RowInfo{place, 0};
    __syncthreads();
    if (threadIdx.x == 0) a.long_count[b] = s_long;
    int bits = 0;
    while ((1 << bits) < w) ++bits;
    const auto put = [&](int t, int rel) {
        const uint64_t same = lanes_with(rel >= 0, (uint32_t)rel, bits);
        if (rel >= 0) {
            const int rank = mask_rank(same), at = mine[rel];
            a.token[at + rank] = Token{t, (int)(((uint32_t)rel << a.shift) + b)};
            wave_sync();
            if (rank == 0) mine[rel] = at + __popcll((unsigned long long)same);
        }
        wave_sync();
    };
    if (found <= kList) {
        for (int k = lane; k - lane < found; k += kWave) put(k < found ? kept[k] : 0, k < found ? (int)kept_id[k] : -1);
    } else {
        Source::read(a, put);
    }
}

struct EmbedGradArgs {
    const void* grad;       // [n, ld]
    const RowInfo* row;     // at info_at
    const Token* token;     // tokens by id
    float* part;            // [2 chunks, D]: sums of the parts of long rows
    const int* long_count;  // [owners]: long rows of each sorting workgroup
    const int* long_rows;   // [owners, owned]
    void* out;              // [V, ldo]
    int64_t ld, ldo;
    int V, D, nv, owned, shift;
    int lanes;              // lanes of a row: a power of two, 64 where a row has more vectors
    int chunk;              // tokens of a group of lanes
    int chunk_blocks;       // workgroups that take tokens; the others clear the rows without any
    float scale;
};

constexpr int kClear = 16;  // rows of a wave that clears

// Bound by bytes.  The ordered tokens are cut into chunks, a group of lanes each, every lane the same
// columns of all of its tokens, kAhead of them in flight.  A row of up to a chunk's tokens belongs to
// the chunk that it begins in, which sums it to its end and writes it.  A longer row (a frequent token)
// is summed chunk by chunk into `part`, of which a chunk needs two: for the row it begins in and the
// row it ends in; join_long_kernel adds a row's parts in order.  So every group has between one and two
// chunks of work, whatever the frequencies.  131,072 x 768 bfloat16 into 65,536 rows: 41 us,
// about 6 TB/s.
template <typename T, int VEC, int NVL, bool PAST_L2>
__global__ __launch_bounds__(kBlock) void embed_grad_kernel(EmbedGradArgs a) {
    constexpr int kAhead = NVL > 2 ? 4 : 8;
    const int l = threadIdx.x % a.lanes;
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
    T* out = static_cast<T*>(a.out);
    if ((int)blockIdx.x >= a.chunk_blocks) {
        const int per = kClear * (kWave / a.lanes);  // of this wave's rows, its groups take turns
        const int64_t r0 = ((int64_t)(blockIdx.x - a.chunk_blocks) * kWavesPerBlock + threadIdx.x / kWave) * per;
        const int64_t rows = (int64_t)a.owned << a.shift;
        for (int i = lane_id() / a.lanes; i < per && r0 + i < rows; i += kWave / a.lanes) {
            const int64_t v = ((r0 + i) % a.owned << a.shift) + (r0 + i) / a.owned;
            if (v >= a.V || a.row[r0 + i].count) continue;
#pragma unroll
            for (int c = 0; c < NVL; ++c)
                if (on[c]) put_vec<PAST_L2>(out + v * a.ldo + col[c], acc[c]);
        }
        return;
    }
    const int chunk = blockIdx.x * (kBlock / a.lanes) + threadIdx.x / a.lanes;
    const int live = a.row[(int64_t)a.owned << a.shift].beg;
    const int64_t first = (int64_t)chunk * a.chunk;
    if (first >= live) return;
    int beg = (int)first, end = min(live, beg + a.chunk);
    const int row0 = a.token[beg].row, row1 = a.token[end - 1].row;
    const RowInfo i0 = a.row[info_at(row0, a.shift, a.owned)], i1 = a.row[info_at(row1, a.shift, a.owned)];
    const bool long0 = i0.count > a.chunk, long1 = i1.count > a.chunk;
    if (!long0 && i0.beg < beg) beg = i0.beg + i0.count;  // the chunk before has it
    if (!long1) end = i1.beg + i1.count;
    if (beg >= end) return;
    const T* g = static_cast<const T*>(a.grad);
    const auto flush = [&](int row) {
        const bool is0 = long0 && row == row0, is1 = long1 && row == row1;
        float* part = a.part + (int64_t)(2 * chunk + (is0 ? 0 : 1)) * a.D;
#pragma unroll
        for (int c = 0; c < NVL; ++c) {
            if (on[c]) {
                if (is0 || is1) {
                    __builtin_memcpy(part + col[c], acc[c], sizeof(acc[c]));
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[c][i] *= a.scale;
                    put_vec<PAST_L2>(out + (int64_t)row * a.ldo + col[c], acc[c]);
                }
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[c][i] = 0.0f;
        }
    };
    Token next[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) next[u] = beg + u < end ? a.token[beg + u] : Token{-1, -1};
    int row = next[0].row;
    for (int k = beg; k < end; k += kAhead) {
        Vec<T, VEC> f[kAhead][NVL];
        Token now[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            now[u] = next[u];
            if (now[u].t >= 0)
#pragma unroll
                for (int c = 0; c < NVL; ++c)
                    if (on[c]) f[u][c].load(g + (int64_t)now[u].t * a.ld + col[c]);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            next[u] = k + kAhead + u < end ? a.token[k + kAhead + u] : Token{-1, -1};
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (now[u].t < 0) break;
            if (now[u].row != row) {
                flush(row);
                row = now[u].row;
            }
#pragma unroll
            for (int c = 0; c < NVL; ++c) {
                float x[VEC];
                f[u][c].get(x);
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[c][i] += x[i];
            }
        }
    }
    flush(row);
}

// Adds the parts of the long rows, those of one sorting workgroup's ids here: 64 VEC columns a workgroup,
// each of its waves a quarter of a row's parts, then the waves' sums in order.  Bound by the longest row:
// 9.6 us for the same; eight or sixteen waves take as long.
template <typename T, int VEC>
__global__ __launch_bounds__(kBlock) void join_long_kernel(EmbedGradArgs a) {
    __shared__ float s_sum[kWavesPerBlock][VEC][kWave];
    const int lane = lane_id(), wave = threadIdx.x / kWave, d = (blockIdx.y * kWave + lane) * VEC;
    const int count = a.long_count[blockIdx.x], col = min(d, a.D - VEC);
    for (int i0 = 0; i0 < count; i0 += kWave) {
        // 64 rows' places at once, a row a lane
        const int v_of = a.long_rows[(int64_t)blockIdx.x * a.owned + min(i0 + lane, count - 1)];
        const RowInfo info = a.row[info_at(v_of, a.shift, a.owned)];
        for (int i = 0; i < min(kWave, count - i0); ++i) {
            const int v = __builtin_amdgcn_readlane(v_of, i), beg = __builtin_amdgcn_readlane(info.beg, i);
            const int first = beg / a.chunk;
            const int parts = (beg + __builtin_amdgcn_readlane(info.count, i) - 1) / a.chunk - first + 1;
            const int per = (parts + kWavesPerBlock - 1) / kWavesPerBlock;
            float s[VEC] = {};
#pragma unroll 8
            for (int c = wave * per; c < min(parts, (wave + 1) * per); ++c) {
                // in its first chunk a row is the last one, unless it begins it
                const int64_t at = 2 * (first + c) + (c == 0 && beg % a.chunk);
                float x[VEC];
                load_vec(a.part + at * a.D + col, x);
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[e] += x[e];
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < VEC; ++e) s_sum[wave][e][lane] = s[e];
            __syncthreads();
            if (wave == 0 && d < a.D) {
                T* out = static_cast<T*>(a.out) + (int64_t)v * a.ldo + col;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    for (int k = 1; k < kWavesPerBlock; ++k) s[e] += s_sum[k][e][lane];
                    out[e] = (T)(s[e] * a.scale);
                }
            }
        }
    }
}

// Few tokens, in one launch: the time is that of launches, not of bytes.  Workgroup b owns the ids = b
// modulo gridDim.x as in sort_ids_kernel, orders its tokens in LDS, and sums and writes its own rows, so
// nothing passes between workgroups: groups of lanes clear the rows without tokens, take those with up to
// kShared of them in turn, and sum the others together.  2,368 tokens x 128 float32 into
// 32,768 rows: 11.3 us, of which uniform ids leave 9; the zeros take 3.
constexpr int kFewThreads = 512;
constexpr int kFewTokens = 8192;           // 16 a thread, held in registers
constexpr int kFewElements = 1024 * 1024;  // tokens * columns: past it one workgroup may have too much to sum
constexpr int kShared = 8;

struct FewArgs {
    const void *grad, *ids;
    void* out;
    int64_t ld, ldo;
    int n, V, D, nv, owned, shift, lanes;
    uint32_t skip;
    float scale;
};

inline size_t few_lds(int owned, int nvl, int vec) {
    const size_t sums = (size_t)kFewThreads * nvl * vec * sizeof(float);
    return ((size_t)kFewThreads / kWave * owned + 2 * owned + 1) * sizeof(int) + kFewTokens * sizeof(uint16_t) + sums;
}

template <typename T, int VEC, int NVL, typename ID>
__global__ __launch_bounds__(kFewThreads) void embed_grad_few_kernel(FewArgs a) {
    constexpr int WAVES = kFewThreads / kWave, A = kFewTokens / kFewThreads;
    extern __shared__ __align__(16) float sums[];  // [NVL * VEC][kFewThreads]
    __shared__ int s_sum[WAVES], s_shared, s_single;
    const int w = a.owned, lane = lane_id(), wave = threadIdx.x / kWave;
    int* hist = reinterpret_cast<int*>(sums + kFewThreads * NVL * VEC);    // [WAVES][w]
    int* start = hist + WAVES * w;                                         // [w + 1]
    int* busy = start + w + 1;  // [w]: rows with tokens, those of all groups from the front, of one from the back
    uint16_t* order = reinterpret_cast<uint16_t*>(busy + w);  // tokens by id
    const uint32_t b = blockIdx.x, mask = (1u << a.shift) - 1;
    const ID* ids = static_cast<const ID*>(a.ids);
    for (int i = threadIdx.x; i < WAVES * w; i += kFewThreads) hist[i] = 0;
    if (threadIdx.x == 0) s_shared = s_single = 0;
    const int per = (a.n + kFewThreads - 1) / kFewThreads;  // groups of 64 tokens of a wave
    const int first = wave * per * kWave + lane;
    uint32_t rel[A];
#pragma unroll
    for (int u = 0; u < A; ++u) {
        const int t = first + u * kWave;
        const bool in = u < per && t < a.n;
        const ID raw = u < per ? ids[min(t, a.n - 1)] : (ID)-1;
        const uint32_t id = in ? row_id<true>(raw, (uint32_t)a.V, a.skip) : ~0u;
        rel[u] = id != ~0u && (id & mask) == b ? id >> a.shift : ~0u;
    }
    __syncthreads();
    int* mine = hist + wave * w;
#pragma unroll
    for (int u = 0; u < A; ++u)
        if (rel[u] != ~0u) atomicAdd(&mine[rel[u]], 1);
    __syncthreads();
    int place = 0;
    for (int j0 = 0; j0 < w; j0 += kFewThreads) {
        const int j = j0 + threadIdx.x;
        int count = 0, total;
        if (j < w)
            for (int i = 0; i < WAVES; ++i) count += hist[i * w + j];
        int at = place + block_sum<WAVES>(count, s_sum, &total) - count;
        place += total;
        if (j < w) {
            start[j] = at;
            if (count > kShared) busy[atomicAdd(&s_shared, 1)] = j;  // in any order
            else if (count > 0) busy[w - 1 - atomicAdd(&s_single, 1)] = j;
            for (int i = 0; i < WAVES; ++i) {
                const int c = hist[i * w + j];
                hist[i * w + j] = at;
                at += c;
            }
        }
    }
    if (threadIdx.x == 0) start[w] = place;
    __syncthreads();
    int bits = 0;
    while ((1 << bits) < w) ++bits;
#pragma unroll
    for (int u = 0; u < A; ++u) {
        if (!__ballot(rel[u] != ~0u)) continue;
        const uint64_t same = lanes_with(rel[u] != ~0u, rel[u], bits);
        if (rel[u] != ~0u) {
            const int rank = mask_rank(same), at = mine[rel[u]];
            order[at + rank] = (uint16_t)(first + u * kWave);
            wave_sync();
            if (rank == 0) mine[rel[u]] = at + __popcll((unsigned long long)same);
        }
        wave_sync();
    }
    __syncthreads();

    const int groups = kFewThreads / a.lanes, group = threadIdx.x / a.lanes, l = threadIdx.x % a.lanes;
    const T* g = static_cast<const T*>(a.grad);
    int col[NVL];
    bool on[NVL];
    float acc[NVL][VEC];
#pragma unroll
    for (int c = 0; c < NVL; ++c) {
        const int v = c * a.lanes + l;
        on[c] = v < a.nv;
        col[c] = min(v * VEC, a.D - VEC);
    }
    const auto clear = [&] {
#pragma unroll
        for (int c = 0; c < NVL; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[c][i] = 0.0f;
    };
    // adds the tokens order[beg], order[beg + step] .. below end, kAhead in flight
    constexpr int kAhead = NVL > 1 ? 4 : 8;
    const auto add = [&](int beg, int end, int step) {
        for (int k = beg; k < end; k += kAhead * step) {
            Vec<T, VEC> f[kAhead][NVL];
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (k + u * step < end) {
                    const T* row = g + (int64_t)order[k + u * step] * a.ld;
#pragma unroll
                    for (int c = 0; c < NVL; ++c)
                        if (on[c]) f[u][c].load(row + col[c]);
                }
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (k + u * step < end)
#pragma unroll
                    for (int c = 0; c < NVL; ++c) {
                        float x[VEC];
                        f[u][c].get(x);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) acc[c][i] += x[i];
                    }
        }
    };
    const auto write = [&](int j) {
        T* out = static_cast<T*>(a.out) + (((int64_t)j << a.shift) + b) * a.ldo;
#pragma unroll
        for (int c = 0; c < NVL; ++c)
            if (on[c]) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[c][i] *= a.scale;
                store_vec(out + col[c], acc[c]);
            }
    };
    const int rows = (int)(((int64_t)a.V - b + mask) >> a.shift);  // owned ids below V
    clear();
    for (int j = group; j < rows; j += groups)
        if (start[j] == start[j + 1]) write(j);
    for (int i = group; i < s_single; i += groups) {
        const int j = busy[w - 1 - i];
        clear();
        add(start[j], start[j + 1], 1);
        write(j);
    }
    for (int i = 0; i < s_shared; ++i) {  // the same in every thread
        const int j = busy[i], beg = start[j], end = start[j + 1];
        clear();
        add(beg + group, end, groups);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < NVL; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) sums[(c * VEC + i) * kFewThreads + threadIdx.x] = acc[c][i];
        __syncthreads();
        if (group == 0) {
            const int used = min(groups, end - beg);
#pragma unroll 4
            for (int k = 1; k < used; ++k)
#pragma unroll
                for (int c = 0; c < NVL; ++c)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[c][i] += sums[(c * VEC + i) * kFewThreads + k * a.lanes + l];
            write(j);
        }
    }
}

template <typename F>
void with_ids(int32_t ids64, F&& f) {
    if (ids64) f(int64_t{});
    else f(int32_t{});
}

struct GradSpace {
    RowInfo* row;
    Token* token;
    float* part;
    int *long_count, *long_rows;
    Token* bucketed;
    uint16_t* starts;
    int shift, owned;  // sorting workgroups: 2^shift, of `owned` ids each
    int parts;         // of the bucketing step; 0: none
    int64_t chunk, chunks;
    size_t bytes;
};

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

GradSpace grad_space(void* base, int64_t n, int64_t V, int64_t D) {
    GradSpace s;
    // Short chunks leave waves for every CU, long ones fewer parts, each a write and a read of four bytes
    // a column.  Chunks of 8, 16 and 32 tokens, ids by a 1 / rank law, us: 16,384 x 768 34.3, 38.2, 37.3;
    // 16,384 x 2,048 61.9, 53.8, 62.2; 32,768 x 768 45.9, 41.4, 43.6; 49,152 x 768 58.1, 48.9, 49.8;
    // 65,536 x 768 69, 58, 52; 131,072 x 64 59.3, 46.8, 47.9; 131,072 x 768 114, 92, 79.
    s.chunk = n > 49152 ? 32 : n > 24576 || n * D > (16 << 20) ? 16 : 8;
    s.chunks = (n + s.chunk - 1) / s.chunk;
    s.shift = 8;  // one sorting workgroup per CU, more where they would own too many ids
    while (((int64_t)((1 << s.shift) < kMaxBuckets ? kOwned : kMaxOwned) << s.shift) < V) ++s.shift;
    s.parts = n > kSmallTokens && (1 << s.shift) <= kMaxBuckets ? (int)((n + kPartTokens - 1) / kPartTokens) : 0;
    s.owned = (int)((V + ((int64_t)1 << s.shift) - 1) >> s.shift);
    char* p = static_cast<char*>(base);
    size_t off = 0;
    const auto take = [&](size_t bytes) {
        char* at = p ? p + off : nullptr;
        off += up256(bytes);
        return at;
    };
    s.row = reinterpret_cast<RowInfo*>(take((((size_t)s.owned << s.shift) + 1) * sizeof(RowInfo)));
    s.token = reinterpret_cast<Token*>(take((size_t)n * sizeof(Token)));
    s.part = reinterpret_cast<float*>(take(2 * (size_t)s.chunks * (size_t)D * sizeof(float)));
    s.long_count = reinterpret_cast<int*>(take(sizeof(int) << s.shift));
    s.long_rows = reinterpret_cast<int*>(take(((size_t)s.owned << s.shift) * sizeof(int)));
    s.bucketed = reinterpret_cast<Token*>(take(s.parts ? (size_t)n * sizeof(Token) : 0));
    s.starts = reinterpret_cast<uint16_t*>(take((size_t)s.parts * ((1 << s.shift) + 1) * sizeof(uint16_t)));
    s.bytes = off;
    return s;
}

template <typename ID, int WAVES, bool SKIP, bool FROM_PARTS>
int sort_ids(const SortArgs& a, hipStream_t st) {
    const auto kernel = sort_ids_kernel<ID, WAVES, SKIP, FROM_PARTS>;
    const size_t lds = SortShape<WAVES>::lds(a.owned);
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess)
            return capi_fail(TRIDENT_ERR_HIP, "hipFuncSetAttribute(sort_ids): %s", hipGetErrorString(e));
    }
    kernel<<<1u << a.shift, WAVES * kWave, lds, st>>>(a);
    return capi_check_launch("sort_ids_kernel");
}

template <typename ID, bool SKIP>
int order_tokens(const SortArgs& a, hipStream_t st) {
    if (a.n <= kSmallTokens) return sort_ids<ID, 4, SKIP, false>(a, st);
    if (a.parts == 0) return sort_ids<ID, 8, SKIP, false>(a, st);  // a table of more than 2^21 rows
    bucket_ids_kernel<ID, SKIP><<<(unsigned)a.parts, kBlock, 0, st>>>(a);
    const int rc = capi_check_launch("bucket_ids_kernel");
    if (rc) return rc;
    // the waves' counters of more ids leave room for fewer waves
    return a.owned <= kOwned ? sort_ids<ID, 16, SKIP, true>(a, st) : sort_ids<ID, 8, SKIP, true>(a, st);
}

// Which calls take one launch instead of three: at most kFewTokens and kFewElements, rows within one
// group's registers, and ids within the 256 workgroups' counters.  One and three, ids uniform and by a
// 1 / rank law: 64 x 768 11.8 and 15.8 us; 1,024 x 768 12.6 and 16.9, 15.6 and 19.0; 8,192 x 128 10.9 and
// 17.8, 16.7 and 23.5; but 4,096 x 768 by the law 26.3 and 22.0.  With one id for all tokens, the worst that
// one workgroup can be given, 1,024 x 768 takes 43 and 22.
bool few_ok(int64_t n, int64_t V, int64_t D) {
    return n > 0 && n <= kFewTokens && n * D <= kFewElements && D <= 1024 && V <= (int64_t)kOwned << 8;
}

template <typename T, typename ID>
int embed_grad_few(const void* grad, int64_t ld, const void* ids, int64_t n, int64_t V, int64_t D, double scale,
                   int64_t padding_idx, void* out, int64_t ldo, hipStream_t st) {
    FewArgs a{grad, ids, out, ld, ldo, (int)n, (int)V, (int)D, 0, (int)((V + 255) >> 8), 8, 1,
              padding_idx >= 0 && padding_idx < V ? (uint32_t)padding_idx : ~0u, (float)scale};
    const int vec = D >= kVec<T> ? kVec<T> : 1;
    a.nv = (int)((D + vec - 1) / vec);
    while (a.lanes < a.nv && a.lanes < kWave) a.lanes *= 2;
    const int nvl = vec == 1 ? 1 : (a.nv + kWave - 1) / kWave;
    const unsigned grid = (unsigned)std::min<int64_t>(256, V);
    const auto go = [&](auto v, auto c) {
        constexpr int VEC = decltype(v)::value, NVL = decltype(c)::value;
        const auto kernel = embed_grad_few_kernel<T, VEC, NVL, ID>;
        const size_t lds = few_lds(a.owned, NVL, VEC);
        if (lds > 65536) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess)
                return capi_fail(TRIDENT_ERR_HIP, "hipFuncSetAttribute(embed_grad): %s", hipGetErrorString(e));
        }
        kernel<<<grid, kFewThreads, lds, st>>>(a);
        return capi_check_launch("embed_grad_few_kernel");
    };
    using std::integral_constant;
    integral_constant<int, kVec<T>> v;
    if (vec == 1) return go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    if (nvl == 1) return go(v, integral_constant<int, 1>{});
    if (nvl == 2) return go(v, integral_constant<int, 2>{});
    return go(v, integral_constant<int, 4>{});
}

constexpr int64_t kMaxCount = 0x7fffffff - 4096;  // tokens, rows and columns count in 32 bits

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
            if (vec == 1) embed_kernel<T, 1, ID, false><<<(unsigned)blocks, kBlock, 0, st>>>(a);
            else if (n * D * (int64_t)sizeof(T) <= kL2Bytes)
                embed_kernel<T, kVec<T>, ID, false><<<(unsigned)blocks, kBlock, 0, st>>>(a);
            else embed_kernel<T, kVec<T>, ID, true><<<(unsigned)blocks, kBlock, 0, st>>>(a);
            rc = capi_check_launch("embed_kernel");
        });
    });
    return rc;
}

size_t trident_embedding_grad_workspace_bytes(int64_t n, int64_t V, int64_t D) {
    if (n < 0 || V < 1 || D < 1 || n > kMaxCount || V > kMaxCount || D > kMaxCount) return 0;
    return few_ok(n, V, D) ? 0 : grad_space(nullptr, n, V, D).bytes;
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
    if (D > 65535 * (int64_t)kWave)
        return capi_fail(TRIDENT_ERR_UNSUPPORTED, "embedding_grad: D=%lld is too large", (long long)D);
    hipStream_t st = static_cast<hipStream_t>(stream);
    int rc = TRIDENT_OK;
    if (few_ok(n, V, D)) {
        with_ids(ids64, [&](auto i) {
            using ID = decltype(i);
            with_dtype(dtype, [&](auto t) {
                rc = embed_grad_few<decltype(t), ID>(grad, ld_grad, ids, n, V, D, scale, padding_idx, out, ld_out, st);
            });
        });
        return rc;
    }
    const GradSpace s = grad_space(workspace, n, V, D);
    if (!workspace || workspace_bytes < s.bytes)
        return capi_fail(TRIDENT_ERR_WORKSPACE_TOO_SMALL, "embedding_grad: workspace %zu < %zu bytes", workspace_bytes,
                         s.bytes);
    with_ids(ids64, [&](auto i) {
        using ID = decltype(i);
        const SortArgs order{ids, (int)n, (int)V, s.owned, s.shift, (int)s.chunk, s.parts,
                             padding_idx >= 0 && padding_idx < V ? (uint32_t)padding_idx : ~0u, s.row, s.token,
                             s.long_count, s.long_rows, s.bucketed, s.starts};
        rc = order.skip == ~0u ? order_tokens<ID, false>(order, st) : order_tokens<ID, true>(order, st);
    });
    if (rc) return rc;
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        EmbedGradArgs a{grad,   s.row,  s.token, s.part, s.long_count, s.long_rows, out, ld_grad,       ld_out,
                        (int)V, (int)D, 0,       s.owned, s.shift,     0,           (int)s.chunk, 0, (float)scale};
        const int vec = D >= kVec<T> ? kVec<T> : 1;
        a.nv = (int)((D + vec - 1) / vec);
        a.lanes = 1;
        while (a.lanes < a.nv && a.lanes < kWave) a.lanes *= 2;
        const int nvl = std::min(4, (a.nv + kWave - 1) / kWave);
        const int groups = kBlock / a.lanes;
        const int64_t clear = kClear * (int64_t)groups;
        a.chunk_blocks = (int)((s.chunks + groups - 1) / groups);
        const dim3 grid((unsigned)(a.chunk_blocks + (((int64_t)s.owned << s.shift) + clear - 1) / clear),
                        (unsigned)((a.nv + nvl * a.lanes - 1) / (nvl * a.lanes)));
        with_bool(V * D * (int64_t)sizeof(T) > kL2Bytes, [&](auto past) {
            constexpr bool P = decltype(past)::value;
            if (vec == 1) embed_grad_kernel<T, 1, 1, P><<<grid, kBlock, 0, st>>>(a);
            else if (nvl == 1) embed_grad_kernel<T, kVec<T>, 1, P><<<grid, kBlock, 0, st>>>(a);
            else if (nvl == 2) embed_grad_kernel<T, kVec<T>, 2, P><<<grid, kBlock, 0, st>>>(a);
            else if (nvl == 3) embed_grad_kernel<T, kVec<T>, 3, P><<<grid, kBlock, 0, st>>>(a);
            else embed_grad_kernel<T, kVec<T>, 4, P><<<grid, kBlock, 0, st>>>(a);
        });
        if ((rc = capi_check_launch("embed_grad_kernel")) || n <= s.chunk) return;
        const auto tiles = [&](int v) { return dim3(1u << s.shift, (unsigned)((D + kWave * v - 1) / (kWave * v))); };
        if (D >= 4) join_long_kernel<T, 4><<<tiles(4), kBlock, 0, st>>>(a);
        else join_long_kernel<T, 1><<<tiles(1), kBlock, 0, st>>>(a);
        rc = capi_check_launch("join_long_kernel");
    });
    return rc;
}

}  // extern "C"
