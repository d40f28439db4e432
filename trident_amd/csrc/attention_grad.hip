// The backward pass of attention.  With P = softmax(scale q k^T) made again from the kept lse,
//
//   dv = P^T do,   dP = do v^T,   dS = P (dP - delta),  delta = rowsum(do out),   dq = scale dS k,   dk = scale dS^T q,
//
// dk and dv summed over the query heads of a group.  Two kernels, both without atomics, so results are the same
// bits every time: one holds a tile of queries and passes over the keys (dq, and delta on the way), the other
// holds a tile of keys and passes over the queries of every head of the group.  Each makes S and dP for itself:
// seven products (eight in 16 bits, kMendDelta below) where five are the least, but no sum crosses workgroups.
//
// Bound as the forward pass is, by matrix and vector unit in turns, and by what is held: q, do and dq (or k, v,
// dk and dv) leave one to four waves a SIMD.  Measured: 12 heads of 64 over 4, float16, 64 sequences of up to
// 2,048 tokens: dq 708 us, dk and dv 851; 6 heads of 80 over 2, causal, float32, 17 sequences of up to 777
// tokens: 179 and 266 us, and 9 for the join; 32 heads of 128 over 8, causal, bfloat16, four sequences of up to 16,384: 23.4
// ms in all, 890 TFLOP/s of the eight products (the five that are the least would take 9.3 ms at the rate of a large one).
#include "attention.hpp"

namespace trident {
namespace {

// dS can be far smaller than float16's least normal number (a gradient of 1e-3 on a row of 10,000 keys), so in
// float16 it is held times a power of two of its column's own, which follows the largest magnitude so far; the
// accumulators are scaled along.  bfloat16 and float32 have the exponents and skip all this.
template <typename T>
constexpr bool kFollow = std::is_same<T, f16_t>::value;
// delta made of an out of 16 bits is off by out's rounding, which can be as large as dP - delta is (values that
// share a part).  But the rows of P sum to one, so those of dS, made with a delta that is off by e, sum to -e
// instead of zero: the dq kernel adds them up in float32, takes their sum times that of P k from dq, and keeps the
// mended delta for dk and dv.  Error of dq in 1e-3, rms, bfloat16, without and with (dk alike): 2.40 and 2.37 of
// 2,000 rows with flat scores, 3.1 and 2.4 of 4 rows, 4.6 and 2.4 of scores six times as large, 14.4 and 2.4 of 500
// rows whose values share 4, 73 and 2.4 of 20,000.  It costs a product more, of keys that are in registers
// already, and its accumulators: of the whole backward pass 8 to 11 % at heads of 64 (sequences of up to 2,048), 1
// to 4 % at short ones, 18 to 23 % at heads of 128, where one wave of a SIMD is left of two.  float32 does without:
// there out's rounding is no more than the sums' own.
template <typename T>
constexpr bool kMendDelta = sizeof(T) == 2;
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
template <typename T, int DP, int WAVES, bool CAUSAL>
__global__ __launch_bounds__(WAVES* kWave, WAVES > 2 && sizeof(T) == 2 && DP <= 96 ? 2 : 1) void attention_dq_kernel(AttentionArgs a) {
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
    const int tiles = ((CAUSAL ? live : t.length) + BN - 1) / BN;
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
    const bool keeps = row < live && half == 0;
    if (!kMendDelta<T> && keeps) a.delta[h * a.rows + at] = delta;
    arrived(q);
    arrived(go);
    f32x16 acc[DP / 32] = {}, pk[kMendDelta<T> ? DP / 32 : 1] = {};
    float off = 0.0f;  // this half's part of the sum of dS
    Power<DP / 32> power;
    const int last = first + 31, end = CAUSAL ? min(row + 1, t.length) : t.length;
    const TileReader<T, kPitch, DP> reader;
    bool not_finite = false;
    // One tile of keys; EDGE: with keys that some row of the wave does not see.  What is loaded meanwhile lies
    // elsewhere than what is read, which __restrict says: else the compiler waits for every load before a
    // transposing read.
    const auto pass = [&](int n, lds_bytes __restrict from, lds_bytes __restrict to, bool work, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        fetch(n + 1, to);
        if (!work) return;
        const lds_bytes keys = from, values = from + kTile;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const int key = n * BN + kb * 32;
            if (EDGE && CAUSAL && key > last) continue;
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                s = mma<T>(reader.rows(keys, kb, i), q[i], s);
                dp = mma<T>(reader.rows(values, kb, i), go[i], dp);
            }
            frag<T> p[2], ds[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale2, -lse));
                s[i] = x * (dp[i] - delta);
                if constexpr (kMendDelta<T>) p[i / 8][i % 8] = (T)x;
            }
            if constexpr (EDGE) {
                const int seen_here = end - key - 4 * half;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (8 * (i / 4) + i % 4 >= seen_here) {
                        s[i] = 0.0f;
                        if constexpr (kMendDelta<T>) p[i / 8][i % 8] = (T)0.0f;
                    }
            }
            if constexpr (kMendDelta<T>) {
#pragma unroll
                for (int i = 0; i < 16; ++i) off += s[i];
            }
            if constexpr (kFollow<T>) {
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(s[i]));
                power.follow(top, acc);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] *= power.by;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) ds[i / 8][i % 8] = (T)s[i];
            const bool apart = EDGE && CAUSAL && key >= first && any_not_finite<T, kPitch>(keys + kb * 32 * kPitch);
            not_finite |= apart;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    frag<T> f = reader.columns(keys, kb * 32 + i * 16, j);
                    if constexpr (EDGE && CAUSAL) {
                        if (apart) f = finite_only<T>(f);
                    }
                    acc[j] = mma<T>(f, ds[i], acc[j]);
                    if constexpr (kMendDelta<T>) pk[j] = mma<T>(f, p[i], pk[j]);
                }
        }
    };
    const int whole = first >= live ? 0 : (CAUSAL ? min(first + 1, t.length) : t.length) / BN;
    const int seen = first >= live ? 0 : CAUSAL ? min(last / BN + 1, tiles) : tiles;
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
    if constexpr (kMendDelta<T>) {
        off += other_half(off);
        if (keeps) a.delta[h * a.rows + at] = delta + off;
        const float by = kFollow<T> ? off * power.by : off;
#pragma unroll
        for (int j = 0; j < DP / 32; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[j][i] = __builtin_fmaf(-by, pk[j][i], acc[j][i]);
    }
    if constexpr (CAUSAL) {
        if (not_finite)
            add_not_finite<T, DP, true>(k + first * a.k_row, a.k_row, min(32, t.length - first), a.D, acc,
                                        [&](int r) { return first + r <= row; });
    }
    if (row < live) store_column<T, DP>(dq + (int64_t)row * out_row, a.D, acc, kFollow<T> ? a.scale / power.by : a.scale);
}

// dk and dv: a wave holds 32 keys and their values; tiles of queries and of their gradients pass through
// LDS with the rows' lse and delta.  S is queries by keys, so a lane holds one key.  Rows past the
// sequence's end have gradients and delta of zero in LDS and add nothing.
template <typename T, int DP, int WAVES, bool CAUSAL>
__global__ __launch_bounds__(WAVES* kWave, WAVES > 2 && sizeof(T) == 2 && DP <= 96 ? 2 : 1) void attention_dkv_kernel(AttentionArgs a) {
    constexpr int BM = WAVES * 32, BN = kTileRows<T>, kPitch = kTilePitch<T, DP>, kTile = BN * kPitch;
    constexpr int KB = BN / 32;
    constexpr int kStage = 2 * kTile + 2 * kWave * 4;  // queries, gradients, 64 words of lse and of delta
    extern __shared__ __align__(16) uint8_t lds[];     // two of them, and a word a wave
    const int hk = blockIdx.x % a.Hkv, share = blockIdx.x / a.Hkv % a.shares, tile = blockIdx.x / a.Hkv / a.shares;
    const int group = a.Hq / a.Hkv;
    SequenceTile t;
    if (!find_tile(a, tile, BM, &t)) return;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane >> 5;
    const int64_t kv_row = (int64_t)a.Hkv * a.D, out_row = (int64_t)a.Hq * a.D;
    T* dk = static_cast<T*>(a.dk) + t.start * kv_row + (int64_t)hk * a.D;
    T* dv = static_cast<T*>(a.dv) + t.start * kv_row + (int64_t)hk * a.D;
    float* part = a.part + (share * a.rows + t.start) * kv_row + (int64_t)hk * a.D;  // of several shares, dk and then dv
    const int64_t next = a.shares * a.rows * kv_row;
    const int live = min(t.first + BM, t.length);
    if (live < t.first + BM) {
        const int from = max(live, t.first), to = min(t.first + BM, t.extent);
        if (a.shares > 1) {
            zero_rows(part, kv_row, from, to, a.D, WAVES * kWave);
            zero_rows(part + next, kv_row, from, to, a.D, WAVES * kWave);
        } else {
            zero_rows(dk, kv_row, from, to, a.D, WAVES * kWave);
            zero_rows(dv, kv_row, from, to, a.D, WAVES * kWave);
        }
    }
    if (live <= t.first) return;

    const int bytes = a.D * (int)sizeof(T);
    const int n0 = CAUSAL ? t.first / BN : 0, each = (t.length + BN - 1) / BN - n0;
    const int begin = (int)((int64_t)each * group * share / a.shares);
    const int tiles = (int)((int64_t)each * group * (share + 1) / a.shares);  // up to this one
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
    fetch(begin, base + begin % 2 * kStage);

    const int first = t.first + wave * 32, row = first + (lane & 31);
    const int64_t at = t.start + min(row, t.length - 1);
    const uint8_t* k_at = static_cast<const uint8_t*>(a.k) + at * a.k_row + hk * a.k_head;
    const uint8_t* v_at = static_cast<const uint8_t*>(a.v) + at * a.v_row + hk * a.v_head;
    // Wide float32 rows do not fit the registers beside the accumulators: they are read again for every block,
    // from L2, which a float32 product of their size hides.
    constexpr bool kHold = sizeof(T) == 2 || DP <= 64;
    frag<T> k[DP / 16], v[DP / 16];
    load_row<T, DP>(k_at, a.D, k);
    if constexpr (kHold) {
        load_row<T, DP>(v_at, a.D, v);
        arrived(v);
    }
    arrived(k);
    typedef __attribute__((address_space(3))) uint32_t* words;
    const words not_finite_keys = (words)(base + 2 * kStage);  // of each wave
    not_finite_keys[wave] = any_not_finite<T, DP / 16>(k);
    meet();
    const bool infinite = __any(not_finite_keys[lane % WAVES]);
    f32x16 ak[DP / 32] = {}, av[DP / 32] = {};
    Power<DP / 32> power;
    const TileReader<T, kPitch, DP> reader;
    bool not_finite = false;
    // One tile of queries from row r on; EDGE: causal, with queries before some key of the wave.  For
    // __restrict see above.
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
            not_finite |= apart;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    frag<T> fv = reader.columns(grads, kb * 32 + i * 16, j), fk = reader.columns(queries, kb * 32 + i * 16, j);
                    if constexpr (EDGE) {
                        if (apart) {
                            fv = finite_only<T>(fv);
                            fk = finite_only<T>(fk);
                        }
                    }
                    av[j] = mma<T>(fv, p[i], av[j]);
                    ak[j] = mma<T>(fk, ds[i], ak[j]);
                }
        }
    };
    const auto place = [&](int n) { return base + n % 2 * kStage; };
    // Past this barrier the tile of rows r on is there.  With an infinity among the keys, rows past the sequence's end
    // get the last one's query and lse: zeros would make a NaN of a key to which every row gives a P of zero.
    const auto arrive = [&](int r, lds_bytes at) {
        wait_and_meet<0>();
        const int rows = t.length - r;
        if (__builtin_expect(!infinite || rows >= BN, 1)) return;
        using L = Tile<T, kPitch>;
        typedef __attribute__((address_space(3))) u32x4* pieces;
        int id = threadIdx.x;
        asm volatile("" : "+v"(id));  // nothing of it is made, and held, before the loop
#pragma unroll 1
        for (int i = id; i < (BN - rows) * L::kPieces; i += WAVES * kWave) {
            const int to = rows + i / L::kPieces, piece = i % L::kPieces;
            *(pieces)(at + to * kPitch + ((piece ^ L::exchange(to)) << 4)) =
                *(pieces)(at + (rows - 1) * kPitch + ((piece ^ L::exchange(rows - 1)) << 4));
        }
        const words lse = (words)(at + 2 * kTile);
        if (id < BN - rows) lse[rows + id] = lse[rows - 1];
        meet();
    };
    // of each head's tiles, those before this wave's last key come first
    const int edges = CAUSAL ? min((first + 32 + BN - 1) / BN - n0, each) : 0;
    for (int n = begin; n < tiles;) {
        const int g = n / each;
        int m = n - g * each;
        const int stop = min(tiles - g * each, each);
        for (; m < min(edges, stop); ++m, ++n) {
            const int r = (n0 + m) * BN;
            arrive(r, place(n));
            pass(n, r, place(n), place(n + 1), first < live && r + BN > first, std::true_type{});
        }
        for (; m < stop; ++m, ++n) {
            const int r = (n0 + m) * BN;
            arrive(r, place(n));
            pass(n, r, place(n), place(n + 1), first < live, std::false_type{});
        }
    }
    if constexpr (CAUSAL) {
        for (int g = begin / each; not_finite && g * each < tiles; ++g) {
            const int h = hk * group + g, rows = min(32, t.length - first);
            const int64_t from = t.start + first;
            const auto sees = [&](int r) { return first + r >= row; };
            add_not_finite<T, DP, false>(static_cast<const T*>(a.grad) + from * out_row + (int64_t)h * a.D,
                                         out_row * (int)sizeof(T), rows, a.D, av, sees);
            add_not_finite<T, DP, true>(static_cast<const uint8_t*>(a.q) + from * a.q_row + h * a.q_head, a.q_row, rows, a.D,
                                        ak, sees);
        }
    }
    if (row >= live) return;
    constexpr float kUnshift = kFollow<T> ? 0x1p-15f : 1.0f;
    const float by = kFollow<T> ? a.scale * kUnshift / power.by : a.scale;
    if (a.shares > 1) {
        store_column<float, DP>(part + (int64_t)row * kv_row, a.D, ak, by);
        store_column<float, DP>(part + next + (int64_t)row * kv_row, a.D, av, kUnshift);
    } else {
        store_column<T, DP>(dk + (int64_t)row * kv_row, a.D, ak, by);
        store_column<T, DP>(dv + (int64_t)row * kv_row, a.D, av, kUnshift);
    }
}

// dk (blockIdx.y 0) and dv of several shares: their sums, in order, eight elements a thread.
template <typename T>
__global__ __launch_bounds__(kBlock) void attention_join_kernel(const float* part, int shares, int64_t n, T* dk, T* dv) {
    const int64_t at = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * 8;
    if (at >= n) return;
    const float* p = part + blockIdx.y * shares * n + at;
    float sum[8], f[8];
    load_vec<float, 8>(p, sum);
    for (int s = 1; s < shares; ++s) {
        load_vec<float, 8>(p + s * n, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += f[e];
    }
    store_vec<T, 8>((blockIdx.y ? dv : dk) + at, sum);
}

size_t delta_bytes(const TridentAttention* t) { return ((size_t)t->rows * t->q_heads * 4 + 255) & ~(size_t)255; }

// Shares of the queries that a tile of keys is cut into, each to a workgroup of its own, where the tiles alone
// leave CUs idle: then the longest sequence's tile is what the others wait for (17 sequences of up to 777, 2
// key heads, float32: the whole backward pass 847 us, with three shares and the join 456).
int shares_of(const TridentAttention* t) {
    const int64_t sequences = std::max<int64_t>(t->sequences, 1), length = t->rows / sequences;
    const int64_t tiles = std::max<int64_t>((t->rows + 127) / 128, sequences) * t->kv_heads;
    const int64_t most = std::min<int64_t>(8, length / 64 * (t->q_heads / t->kv_heads) / 2);  // two tiles of queries each
    return (int)std::max<int64_t>(1, std::min(most, 512 / tiles));
}

size_t workspace_of(const TridentAttention* t) {
    const int shares = shares_of(t);
    return delta_bytes(t) + (shares > 1 ? (size_t)2 * shares * t->rows * t->kv_heads * t->head_dim * 4 : 0);
}

template <typename T, int DP, int WAVES, bool CAUSAL>
int launch(AttentionArgs a, hipStream_t st) {
    constexpr int BM = WAVES * 32;
    constexpr size_t lds = 4 * (size_t)kTileRows<T> * kTilePitch<T, DP> + 4 * kWave * 4 + WAVES * 4;
    static_assert(lds <= 163840, "LDS of a CU");
    const auto dq = attention_dq_kernel<T, DP, WAVES, CAUSAL>, dkv = attention_dkv_kernel<T, DP, WAVES, CAUSAL>;
    if (lds > 65536)
        for (const void* f : {reinterpret_cast<const void*>(dq), reinterpret_cast<const void*>(dkv)}) {
            const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess)
                return capi_fail(TRIDENT_ERR_HIP, "hipFuncSetAttribute(attention_grad): %s", hipGetErrorString(e));
        }
    const int64_t tiles = a.slots ? a.count * ((a.slots + BM - 1) / BM) : a.rows / BM + a.count + 2;
    if (tiles * std::max(a.Hq, a.Hkv * a.shares) > kMaxGroups) return capi_fail(TRIDENT_ERR_UNSUPPORTED, "attention_grad: too many tiles");
    a.tiles = (int)tiles;
    dq<<<(unsigned)(tiles * a.Hq), WAVES * kWave, lds, st>>>(a);
    int rc = capi_check_launch("attention_dq_kernel");
    if (rc != TRIDENT_OK) return rc;
    dkv<<<(unsigned)(tiles * a.Hkv * a.shares), WAVES * kWave, lds, st>>>(a);
    rc = capi_check_launch("attention_dkv_kernel");
    if (rc != TRIDENT_OK || a.shares == 1) return rc;
    const int64_t n = a.rows * a.Hkv * a.D;
    attention_join_kernel<T><<<dim3((unsigned)((n / 8 + kBlock - 1) / kBlock), 2), kBlock, 0, st>>>(
        a.part, a.shares, n, static_cast<T*>(a.dk), static_cast<T*>(a.dv));
    return capi_check_launch("attention_join_kernel");
}

// Two waves where sequences are short (1,000 of 16 tokens, 12 heads of 64, bfloat16: 124 us, 172 by four; of
// 50: 268 and 309).
template <typename T, int DP, bool CAUSAL>
int by_length(const AttentionArgs& a, hipStream_t st) {
    const int64_t mean = a.slots ? a.slots : a.rows / std::max<int64_t>(a.count, 1);
    if (mean <= 64) return launch<T, DP, 2, CAUSAL>(a, st);
    return launch<T, DP, 4, CAUSAL>(a, st);
}

}  // namespace
}  // namespace trident

using namespace trident;

extern "C" {

size_t trident_attention_grad_workspace_bytes(const TridentAttention* t) {
    AttentionArgs a;
    if (attention_check(t, true, &a) != TRIDENT_OK || t->rows == 0) return 0;
    return workspace_of(t);
}

int trident_attention_grad(const TridentAttention* t, void* workspace, size_t workspace_bytes, void* stream) {
    AttentionArgs a;
    const int rc = attention_check(t, true, &a);
    if (rc != TRIDENT_OK || t->rows == 0) return rc;
    const size_t need = workspace_of(t);
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return capi_fail(TRIDENT_ERR_WORKSPACE_TOO_SMALL, "attention_grad needs %zu bytes, 16-byte aligned, got %zu", need,
                         workspace ? workspace_bytes : 0);
    a.delta = static_cast<float*>(workspace);
    a.shares = shares_of(t);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + delta_bytes(t));
    int out = TRIDENT_OK;
    with_dtype(t->dtype, [&](auto e) {
        using T = decltype(e);
        const hipStream_t st = (hipStream_t)stream;
        with_bool(a.causal, [&](auto causal) {
            constexpr bool CAUSAL = decltype(causal)::value;
            if (a.D <= 32) out = by_length<T, 32, CAUSAL>(a, st);
            else if (a.D <= 64) out = by_length<T, 64, CAUSAL>(a, st);
            else if (a.D <= 96) out = by_length<T, 96, CAUSAL>(a, st);
            else out = by_length<T, 128, CAUSAL>(a, st);
        });
    });
    return out;
}

}  // extern "C"
