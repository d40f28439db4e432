// The backward pass of attention.  With P = softmax(scale q k^T) made again from the kept lse,
//
//   dv = P^T do,   dP = do v^T,   dS = P (dP - delta),  delta = rowsum(do out),   dq = scale dS k,   dk = scale dS^T q,
//
// dk and dv summed over the query heads of a group.  Two kernels, both without atomics, so results are the
// same bits every time: one holds a tile of queries and passes over the keys (dq, and delta on the way), the other
// holds a tile of keys and passes over the queries of every head of the group.  Each makes S and dP for itself: seven
// products where five are the least, but no sum crosses workgroups.
#include "attention.hpp"

namespace trident {
namespace {

// dS can be far smaller than float16's least normal number (a gradient of 1e-3 on a row of 10,000 keys), so
// in float16 it is held times a power of two of its column's own, which follows the largest magnitude so far; the
// accumulators are scaled along.  bfloat16 and float32 have the exponents and skip all this.
template <typename T>
constexpr bool kFollow = std::is_same<T, f16_t>::value;
// P <= 1 (up to the rounding of lse) in float16 times 2^15: held in full down to 2^-29.
template <typename T>
constexpr float kShift = kFollow<T> ? 15.0f : 0.0f;

template <int N>
struct Power {
    float by = 0x1p100f;
    // ds *= by for |ds| <= top in this lane, after by was lowered so that the products are at most 2^15.
    __device__ __forceinline__ void follow(float top, f32x16 (&acc)[N]) {
        top = fmaxf(top, other_half(top));
        if (!__any(top * by > 0x1p15f)) return;
        const int e = (int)(__float_as_uint(top) >> 23);  // 2^(e - 127) <= top
        const float next = top * by > 0x1p15f ? __uint_as_float((uint32_t)max(268 - e, 1) << 23) : by;
        const float ratio = next / by;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[j][i] *= ratio;
        by = next;
    }
};

// dq: as the forward pass, with the values' rows for dP and the keys' columns for dq.
template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void attention_dq_kernel(AttentionArgs a) {
    constexpr int BM = WAVES * 32, BN = kTileRows<T>, kPitch = kTilePitch<T, DP>, kTile = BN * kPitch;
    constexpr int KB = BN / 32;
    extern __shared__ __align__(16) uint8_t lds[];  // [2][keys, values]
    int tile, h, hk;
    tile_and_head(a, &tile, &h, &hk);
    SequenceTile t;
    if (!find_tile(a, tile, BM, &t)) return;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane >> 5;
    const int64_t out_row = (int64_t)a.Hq * a.D;
    T* dq = static_cast<T*>(a.dq) + t.start * out_row + (int64_t)h * a.D;
    const int live = min(t.first + BM, t.length);
    if (live < t.first + BM) zero_rows(dq, out_row, max(live, t.first), min(t.first + BM, t.extent), a.D, WAVES * kWave);
    if (live <= t.first) return;

    const uint8_t* k = static_cast<const uint8_t*>(a.k) + t.start * a.k_row + hk * a.k_head;
    const uint8_t* v = static_cast<const uint8_t*>(a.v) + t.start * a.v_row + hk * a.v_head;
    const int bytes = a.D * (int)sizeof(T);
    const int tiles = ((a.causal ? live : t.length) + BN - 1) / BN;
    const lds_bytes base = (lds_bytes)(lds_ptr)lds;
    const auto fetch = [&](int n, lds_bytes to) {
        if (n >= tiles) return;
        fetch_tile<T, kPitch, BN, WAVES>(to, k + (int64_t)n * BN * a.k_row, a.k_row, t.length - n * BN, bytes, wave);
        fetch_tile<T, kPitch, BN, WAVES>(to + kTile, v + (int64_t)n * BN * a.v_row, a.v_row, t.length - n * BN, bytes,
                                         wave);
    };
    fetch(0, base);

    const int first = t.first + wave * 32, row = first + (lane & 31);
    const int64_t at = t.start + min(row, t.length - 1);
    frag<T> q[DP / 16], go[DP / 16];
    load_row<T, DP>(static_cast<const uint8_t*>(a.q) + at * a.q_row + h * a.q_head, a.D, q);
    load_row<T, DP>(static_cast<const T*>(a.grad) + at * out_row + (int64_t)h * a.D, a.D, go);
    float delta = 0.0f;
    {
        frag<T> o[DP / 16];
        load_row<T, DP>(static_cast<const T*>(a.out) + at * out_row + (int64_t)h * a.D, a.D, o);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf((float)go[i][e], (float)o[i][e], delta);
        delta += other_half(delta);
    }
    const float lse = a.lse[h * a.rows + at];
    if (row < live && half == 0) a.delta[h * a.rows + at] = delta;
    arrived(q);
    arrived(go);
    f32x16 acc[DP / 32] = {};
    Power<DP / 32> power;
    const int last = first + 31, end = a.causal ? min(row + 1, t.length) : t.length;
    const TileReader<T, kPitch, DP> reader;
    // One tile of keys; EDGE: with keys that some row of the wave does not see.  What is loaded meanwhile lies elsewhere
    // than what is read, which __restrict says: else the compiler waits for every load before a transposing read.
    const auto pass = [&](int n, lds_bytes __restrict from, lds_bytes __restrict to, bool work, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        fetch(n + 1, to);
        if (!work) return;
        const lds_bytes keys = from, values = from + kTile;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const int key = n * BN + kb * 32;
            if (EDGE && a.causal && key > last) continue;
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                s = mma<T>(reader.rows(keys, kb, i), q[i], s);
                dp = mma<T>(reader.rows(values, kb, i), go[i], dp);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale2, -lse)) * (dp[i] - delta);
            if constexpr (EDGE) {
                const int seen_here = end - key - 4 * half;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (8 * (i / 4) + i % 4 >= seen_here) s[i] = 0.0f;
            }
            if constexpr (kFollow<T>) {
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(s[i]));
                power.follow(top, acc);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] *= power.by;
            }
            frag<T> ds[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) ds[i / 8][i % 8] = (T)s[i];
            const bool apart = EDGE && a.causal && key >= first && any_not_finite<T, kPitch>(keys + kb * 32 * kPitch);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (EDGE && apart) {
                    add_seen_rows<T, kPitch, DP>(keys, kb * 32 + i * 16, ds[i], acc,
                                                 [&](int r) { return key + i * 16 + r <= row; });
                    continue;
                }
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) acc[j] = mma<T>(reader.columns(keys, kb * 32 + i * 16, j), ds[i], acc[j]);
            }
        }
    };
    const int whole = first >= live ? 0 : (a.causal ? min(first + 1, t.length) : t.length) / BN;
    const int seen = first >= live ? 0 : a.causal ? min(last / BN + 1, tiles) : tiles;
    const auto place = [&](int n) { return base + n % 2 * 2 * kTile; };
    int n = 0;
    for (; n < whole; ++n) {
        wait_and_meet<0>();
        pass(n, place(n), place(n + 1), true, std::false_type{});
    }
    for (; n < tiles; ++n) {
        wait_and_meet<0>();
        pass(n, place(n), place(n + 1), n < seen, std::true_type{});
    }
    if (row < live) store_column<T, DP>(dq + (int64_t)row * out_row, a.D, acc, kFollow<T> ? a.scale / power.by : a.scale);
}

// dk and dv: a wave holds 32 keys and their values; tiles of queries and of their gradients pass through
// LDS with the rows' lse and delta.  S is queries by keys, so a lane holds one key.  Rows past the
// sequence's end are zeros in LDS, lse and delta among them, and add nothing.
template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void attention_dkv_kernel(AttentionArgs a) {
    constexpr int BM = WAVES * 32, BN = kTileRows<T>, kPitch = kTilePitch<T, DP>, kTile = BN * kPitch;
    constexpr int KB = BN / 32;
    constexpr int kStage = 2 * kTile + 2 * kWave * 4;  // queries, gradients, 64 words of lse and of delta
    extern __shared__ __align__(16) uint8_t lds[];
    const int tile = blockIdx.x / a.Hkv, hk = blockIdx.x % a.Hkv, group = a.Hq / a.Hkv;
    SequenceTile t;
    if (!find_tile(a, tile, BM, &t)) return;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane >> 5;
    const int64_t kv_row = (int64_t)a.Hkv * a.D, out_row = (int64_t)a.Hq * a.D;
    T* dk = static_cast<T*>(a.dk) + t.start * kv_row + (int64_t)hk * a.D;
    T* dv = static_cast<T*>(a.dv) + t.start * kv_row + (int64_t)hk * a.D;
    const int live = min(t.first + BM, t.length);
    if (live < t.first + BM) {
        const int from = max(live, t.first), to = min(t.first + BM, t.extent);
        zero_rows(dk, kv_row, from, to, a.D, WAVES * kWave);
        zero_rows(dv, kv_row, from, to, a.D, WAVES * kWave);
    }
    if (live <= t.first) return;

    const int bytes = a.D * (int)sizeof(T);
    const int n0 = a.causal ? t.first / BN : 0, each = (t.length + BN - 1) / BN - n0, tiles = each * group;
    const lds_bytes base = (lds_bytes)(lds_ptr)lds;
    const auto fetch = [&](int n, lds_bytes to) {
        if (n >= tiles) return;
        const int g = n / each, r = (n0 + n - g * each) * BN, h = hk * group + g;
        const int64_t at = t.start + r;
        fetch_tile<T, kPitch, BN, WAVES>(to, static_cast<const uint8_t*>(a.q) + at * a.q_row + h * a.q_head, a.q_row,
                                         t.length - r, bytes, wave);
        fetch_tile<T, kPitch, BN, WAVES>(to + kTile, static_cast<const T*>(a.grad) + at * out_row + (int64_t)h * a.D,
                                         out_row * (int)sizeof(T), t.length - r, bytes, wave);
        const uint32_t words = (uint32_t)min(t.length - r, BN) * 4;
        const uint32_t mine = lane < BN ? (uint32_t)lane * 4 : kPastBuffer;
        if (wave == 0)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer_of(a.lse + h * a.rows + at, words), (lds_ptr)(to + 2 * kTile),
                                                     4, mine, 0, 0, 0);
        if (wave == WAVES - 1)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer_of(a.delta + h * a.rows + at, words),
                                                     (lds_ptr)(to + 2 * kTile + kWave * 4), 4, mine, 0, 0, 0);
    };
    fetch(0, base);

    const int first = t.first + wave * 32, row = first + (lane & 31);
    const int64_t at = t.start + min(row, t.length - 1);
    const uint8_t* k_at = static_cast<const uint8_t*>(a.k) + at * a.k_row + hk * a.k_head;
    const uint8_t* v_at = static_cast<const uint8_t*>(a.v) + at * a.v_row + hk * a.v_head;
    // Wide float32 rows do not fit the registers beside the accumulators: they are read again for every block,
    // from L2, which a float32 product of their size hides.
    constexpr bool kHold = sizeof(T) == 2 || DP <= 64;
    frag<T> k[DP / 16], v[DP / 16];
    if constexpr (kHold) {
        load_row<T, DP>(k_at, a.D, k);
        load_row<T, DP>(v_at, a.D, v);
        arrived(k);
        arrived(v);
    }
    f32x16 ak[DP / 32] = {}, av[DP / 32] = {};
    Power<DP / 32> power;
    const TileReader<T, kPitch, DP> reader;
    // One tile of queries from row r on; EDGE: causal, with queries before some key of the wave.  For __restrict see above.
    const auto pass = [&](int n, int r, lds_bytes __restrict from, lds_bytes __restrict to, bool work, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        fetch(n + 1, to);
        if (!work) return;
        const lds_bytes queries = from, grads = from + kTile;
        typedef const __attribute__((address_space(3))) f32x4* quads;
        const quads lse = (quads)(grads + kTile), delta = (quads)(grads + kTile + kWave * 4);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const int query = r + kb * 32;
            if (EDGE && query < first) continue;
            f32x16 s = {}, dp = {};
            if constexpr (!kHold) {
                asm volatile("" : "+v"(k_at), "+v"(v_at));  // not before the loop
                load_row<T, DP>(k_at, a.D, k);
                load_row<T, DP>(v_at, a.D, v);
            }
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                s = mma<T>(reader.rows(queries, kb, i), k[i], s);
                dp = mma<T>(reader.rows(grads, kb, i), v[i], dp);
            }
            const int hidden = EDGE ? row - query - 4 * half : 0;  // of this half's rows are before the key
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 le = lse[kb * 8 + 2 * i + half], de = delta[kb * 8 + 2 * i + half];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool masked = EDGE && 8 * i + e < hidden;
                    const float x =
                        masked ? 0.0f
                               : __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * i + e], a.scale2, kShift<T> - le[e]));
                    s[4 * i + e] = x;
                    dp[4 * i + e] = masked ? 0.0f : x * (dp[4 * i + e] - de[e]);
                }
            }
            if constexpr (kFollow<T>) {
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(dp[i]));
                power.follow(top, ak);
#pragma unroll
                for (int i = 0; i < 16; ++i) dp[i] *= power.by;
            }
            frag<T> p[2], ds[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                p[i / 8][i % 8] = (T)s[i];
                ds[i / 8][i % 8] = (T)dp[i];
            }
            const bool apart = EDGE && query < first + 32 && (any_not_finite<T, kPitch>(queries + kb * 32 * kPitch) ||
                                                              any_not_finite<T, kPitch>(grads + kb * 32 * kPitch));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (EDGE && apart) {
                    const auto sees = [&](int r) { return query + i * 16 + r >= row; };
                    add_seen_rows<T, kPitch, DP>(grads, kb * 32 + i * 16, p[i], av, sees);
                    add_seen_rows<T, kPitch, DP>(queries, kb * 32 + i * 16, ds[i], ak, sees);
                    continue;
                }
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    av[j] = mma<T>(reader.columns(grads, kb * 32 + i * 16, j), p[i], av[j]);
                    ak[j] = mma<T>(reader.columns(queries, kb * 32 + i * 16, j), ds[i], ak[j]);
                }
            }
        }
    };
    const auto place = [&](int n) { return base + n % 2 * kStage; };
    // of each head's tiles, those before this wave's last key come first
    const int edges = a.causal ? min((first + 32 + BN - 1) / BN - n0, each) : 0;
    for (int n = 0, g = 0; g < group; ++g) {
        int m = 0;
        for (; m < edges; ++m, ++n) {
            const int r = (n0 + m) * BN;
            wait_and_meet<0>();
            pass(n, r, place(n), place(n + 1), first < live && r + BN > first, std::true_type{});
        }
        for (; m < each; ++m, ++n) {
            wait_and_meet<0>();
            pass(n, (n0 + m) * BN, place(n), place(n + 1), first < live, std::false_type{});
        }
    }
    if (row >= live) return;
    constexpr float kUnshift = kFollow<T> ? 0x1p-15f : 1.0f;
    store_column<T, DP>(dk + (int64_t)row * kv_row, a.D, ak, kFollow<T> ? a.scale * kUnshift / power.by : a.scale);
    store_column<T, DP>(dv + (int64_t)row * kv_row, a.D, av, kUnshift);
}

template <typename T, int DP, int WAVES>
int launch(AttentionArgs a, hipStream_t st) {
    constexpr int BM = WAVES * 32;
    constexpr size_t lds = 4 * (size_t)kTileRows<T> * kTilePitch<T, DP> + 4 * kWave * 4;
    static_assert(lds <= 163840, "LDS of a CU");
    const auto dq = attention_dq_kernel<T, DP, WAVES>, dkv = attention_dkv_kernel<T, DP, WAVES>;
    if (lds > 65536)
        for (const void* f : {reinterpret_cast<const void*>(dq), reinterpret_cast<const void*>(dkv)}) {
            const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess)
                return capi_fail(TRIDENT_ERR_HIP, "hipFuncSetAttribute(attention_grad): %s", hipGetErrorString(e));
        }
    const int64_t tiles = a.slots ? a.count * ((a.slots + BM - 1) / BM) : a.rows / BM + a.count + 2;
    if (tiles * a.Hq > 0x7fffffff) return capi_fail(TRIDENT_ERR_UNSUPPORTED, "attention_grad: too many tiles");
    a.tiles = (int)tiles;
    dq<<<(unsigned)(tiles * a.Hq), WAVES * kWave, lds, st>>>(a);
    const int rc = capi_check_launch("attention_dq_kernel");
    if (rc != TRIDENT_OK) return rc;
    dkv<<<(unsigned)(tiles * a.Hkv), WAVES * kWave, lds, st>>>(a);
    return capi_check_launch("attention_dkv_kernel");
}

template <typename T, int DP>
int by_length(const AttentionArgs& a, hipStream_t st) {
    const int64_t mean = a.slots ? a.slots : a.rows / std::max<int64_t>(a.count, 1);
    if (mean <= 32) return launch<T, DP, 1>(a, st);
    return launch<T, DP, 4>(a, st);
}

}  // namespace
}  // namespace trident

using namespace trident;

extern "C" {

size_t trident_attention_grad_workspace_bytes(const TridentAttention* t) {
    if (!t || t->rows < 0 || t->rows > (1 << 30) || t->q_heads < 1 || t->q_heads > (1 << 15)) return 0;
    return (size_t)t->rows * t->q_heads * 4;
}

int trident_attention_grad(const TridentAttention* t, void* workspace, size_t workspace_bytes, void* stream) {
    AttentionArgs a;
    const int rc = attention_check(t, true, &a);
    if (rc != TRIDENT_OK || t->rows == 0) return rc;
    const size_t need = trident_attention_grad_workspace_bytes(t);
    if (!workspace || workspace_bytes < need)
        return capi_fail(TRIDENT_ERR_WORKSPACE_TOO_SMALL, "attention_grad needs %zu bytes, got %zu", need,
                         workspace ? workspace_bytes : 0);
    a.delta = static_cast<float*>(workspace);
    int out = TRIDENT_OK;
    with_dtype(t->dtype, [&](auto e) {
        using T = decltype(e);
        const hipStream_t st = (hipStream_t)stream;
        if (a.D <= 32) out = by_length<T, 32>(a, st);
        else if (a.D <= 64) out = by_length<T, 64>(a, st);
        else if (a.D <= 96) out = by_length<T, 96>(a, st);
        else out = by_length<T, 128>(a, st);
    });
    return out;
}

}  // extern "C"
