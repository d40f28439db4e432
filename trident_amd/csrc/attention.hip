// Attention of every token over its own sequence,
//
//   S = scale q k^T,   P = softmax over the row's keys (causal: those up to the row),   out = P v,
//
// with sequences packed one after another or padded to one length, and query heads in groups that share a key
// and value head.  A workgroup takes a tile of queries of one head and passes over the keys once: tiles of keys
// and values go straight from memory to LDS, the next one while this one is multiplied, and each row keeps a
// running reference value and sum.
//
// Bound by the vector unit with heads of 64, by both it and the matrix unit with wider ones: 32 x 32 scores of
// a head of 64 are 8 matrix instructions, 256 cycles, and about 475 of exponentials, multiply-adds, maxima, sums and
// roundings, and the waves of a SIMD take turns at both.  Measured: causal, 32 heads of 128 over 8, bfloat16,
// four sequences of up to 16,384 tokens (5.2 TFLOP) 4.8 ms, 1.09 PFLOP/s; 12 heads of 64, bfloat16, 512 passages
// padded to 256 tokens 177 us (its bytes take 115); 12 heads of 64 over 4, float16, 64 sequences of up to 2,048
// tokens 371 us; one query of 16 tokens 3.8 us, a launch and three loads one after another (cards differ by up
// to 7 %).  A causal kernel is
// apart from the full one: without the diagonal the full one is small enough for four waves of a SIMD in place
// of three (217 us with it, 185 without).
#include "attention.hpp"

namespace trident {
namespace {

// The scores are computed transposed, keys by queries, so a lane holds one query: its maximum and sum are of
// its own registers and one other lane's, and exp(S) is the second operand of the product with the values as it
// is (mfma.hpp).  P is rounded to the elements' type for that product, relative to a reference that the row's
// largest score exceeds by at most 2^kSlack: the accumulators are only scaled when it would be more.  float16's
// small exponents are used by holding P times 2^kShift, so that probabilities of 2^-21 are still held in full.
template <typename T>
constexpr float kShift = std::is_same<T, f16_t>::value ? 7.0f : 0.0f;
constexpr float kSlack = 8.0f;

// Waves of a workgroup, 32 queries each.  Short sequences leave some without a row, and still four load their
// keys sooner: 12 heads of 64, bfloat16, one sequence of 16 tokens 3.8 us (one wave 4.4), 1,000 of them 44
// (49).
constexpr int kWaves = 4;

template <typename T, int DP, bool CAUSAL>
__global__ __launch_bounds__(kWaves* kWave, sizeof(T) == 2 || DP <= 64 ? 2 : 1) void attention_kernel(AttentionArgs a) {
    constexpr int BM = kWaves * 32, BN = kTileRows<T>, kPitch = kTilePitch<T, DP>, kTile = BN * kPitch;
    constexpr int KB = BN / 32;
    extern __shared__ __align__(16) uint8_t lds[];  // [2][keys, values]
    int tile, h, hk;
    tile_and_head(a, &tile, &h, &hk);
    SequenceTile t;
    if (!find_tile(a, tile, BM, &t)) return;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane >> 5;
    const int64_t out_row = (int64_t)a.Hq * a.D;
    T* out = static_cast<T*>(a.out) + t.start * out_row + (int64_t)h * a.D;
    const int live = min(t.first + BM, t.length);  // rows past it are slots without a token
    if (live < t.first + BM) zero_rows(out, out_row, max(live, t.first), min(t.first + BM, t.extent), a.D, kWaves * kWave);
    if (live <= t.first) return;

    const uint8_t* k = static_cast<const uint8_t*>(a.k) + t.start * a.k_row + hk * a.k_head;
    const uint8_t* v = static_cast<const uint8_t*>(a.v) + t.start * a.v_row + hk * a.v_head;
    const int bytes = a.D * (int)sizeof(T);
    const int tiles = ((CAUSAL ? live : t.length) + BN - 1) / BN;
    const lds_bytes base = (lds_bytes)(lds_ptr)lds;
    const auto fetch = [&](int n, lds_bytes to) {
        if (n >= tiles) return;
        fetch_tile<T, kPitch, BN, kWaves>(to, k + (int64_t)n * BN * a.k_row, a.k_row, t.length - n * BN, bytes, wave);
        fetch_tile<T, kPitch, BN, kWaves>(to + kTile, v + (int64_t)n * BN * a.v_row, a.v_row, t.length - n * BN, bytes,
                                         wave);
    };
    fetch(0, base);

    const int first = t.first + wave * 32, last = first + 31, row = first + (lane & 31);
    frag<T> q[DP / 16];
    load_row<T, DP>(static_cast<const uint8_t*>(a.q) + (t.start + min(row, t.length - 1)) * a.q_row + h * a.q_head, a.D, q);
    arrived(q);
    f32x16 acc[DP / 32] = {};
    float top = -INFINITY, sum = 0.0f;  // the reference, times scale2, and this half's part of the sum
    const int end = CAUSAL ? min(row + 1, t.length) : t.length;  // the keys that this row sees

    const TileReader<T, kPitch, DP> reader;
    f32x16 s[KB];
    frag<T> p[KB][2];
    const auto scores = [&](lds_bytes keys) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) s[kb] = f32x16{};
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) s[kb] = mma<T>(reader.rows(keys, kb, i), q[i], s[kb]);
    };
    // EDGE: with keys that some row of the wave does not see.
    const auto exponentials = [&](int n, auto edge) {
        if constexpr (decltype(edge)::value) {
            const int seen_here = end - n * BN - 4 * half;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (kb * 32 + 8 * (i / 4) + i % 4 >= seen_here) s[kb][i] = -INFINITY;
        }
        float m = s[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) m = fmaxf(m, s[kb][i]);
        m = fmaxf(m, other_half(m)) * a.scale2;
        if (__any(m > top + kSlack)) {
            const float by = m > top ? __builtin_amdgcn_exp2f(top - m) : 1.0f;
            top = fmaxf(m, top);
            sum *= by;
#pragma unroll
            for (int j = 0; j < DP / 32; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[j][i] *= by;
        }
        const float from = top == -INFINITY ? 0.0f : kShift<T> - top;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], a.scale2, from));
                p[kb][i / 8][i % 8] = (T)e;
                sum += e;
            }
    };
    bool not_finite = false;
    const auto add_values = [&](int n, lds_bytes values, auto edge) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const int key = n * BN + kb * 32;
            bool apart = false;  // on the diagonal and not finite
            if constexpr (CAUSAL && decltype(edge)::value) {
                if (key > last) continue;
                apart = key >= first && any_not_finite<T, kPitch>(values + kb * 32 * kPitch);
                not_finite |= apart;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    frag<T> f = reader.columns(values, kb * 32 + i * 16, j);
                    if constexpr (CAUSAL && decltype(edge)::value) {
                        if (apart) f = finite_only<T>(f);
                    }
                    acc[j] = mma<T>(f, p[kb][i], acc[j]);
                }
        }
    };
    // Tiles that every row of the wave sees whole, those that some see in part, and (in step with the other
    // waves) the rest, for which this wave only loads.
    const int whole = first >= live ? 0 : (CAUSAL ? min(first + 1, t.length) : t.length) / BN;
    const int seen = first >= live ? 0 : CAUSAL ? min(last / BN + 1, tiles) : tiles;
    constexpr std::false_type kWhole{};
    constexpr std::true_type kEdge{};
    // Past a barrier tile n is there, and every wave is done with the one before, in whose place the next one
    // goes.  That lies elsewhere than what is read, which __restrict says: else the compiler waits for every
    // load before a transposing read.
    const auto pass = [&](int n, lds_bytes __restrict from, lds_bytes __restrict to, bool work, auto edge) {
        fetch(n + 1, to);
        if (!work) return;
        scores(from);
        exponentials(n, edge);
        add_values(n, from + kTile, edge);
    };
    const auto place = [&](int n) { return base + n % 2 * 2 * kTile; };
    int n = 0;
    for (; n < whole; ++n) {
        wait_and_meet<0>();
        pass(n, place(n), place(n + 1), true, kWhole);
    }
    for (; n < tiles; ++n) {
        wait_and_meet<0>();
        pass(n, place(n), place(n + 1), n < seen, kEdge);
    }
    if constexpr (CAUSAL) {
        if (not_finite)
            add_not_finite<T, DP, false>(v + first * a.v_row, a.v_row, min(32, t.length - first), a.D, acc,
                                         [&](int r) { return first + r <= row; });
    }
    const float all = sum + other_half(sum);
    if (row >= live) return;
    store_column<T, DP>(out + (int64_t)row * out_row, a.D, acc, 1.0f / all);
    if (a.lse && half == 0) a.lse[h * a.rows + t.start + row] = top - kShift<T> + __builtin_amdgcn_logf(all);
}

template <typename T, int DP, bool CAUSAL>
int launch(AttentionArgs a, hipStream_t st) {
    constexpr int BM = kWaves * 32;
    constexpr size_t lds = 4 * (size_t)kTileRows<T> * kTilePitch<T, DP>;
    const auto kernel = attention_kernel<T, DP, CAUSAL>;
    static_assert(lds <= 163840, "LDS of a CU");
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return capi_fail(TRIDENT_ERR_HIP, "hipFuncSetAttribute(attention): %s", hipGetErrorString(e));
    }
    const int64_t tiles = a.slots ? a.count * ((a.slots + BM - 1) / BM) : a.rows / BM + a.count + 2;
    if (tiles * a.Hq > kMaxGroups) return capi_fail(TRIDENT_ERR_UNSUPPORTED, "attention: too many tiles");
    a.tiles = (int)tiles;
    kernel<<<(unsigned)(tiles * a.Hq), kWaves * kWave, lds, st>>>(a);
    return capi_check_launch("attention_kernel");
}

}  // namespace

// Strides are those of 16-byte pieces, so that rows go to LDS whole.
int attention_check(const TridentAttention* t, bool backward, AttentionArgs* a) {
    const char* name = backward ? "attention_grad" : "attention";
    if (!t) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "%s: NULL arguments", name);
    if (!dtype_ok(t->dtype)) return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "%s: dtype=%d", name, t->dtype);
    if (t->rows < 0 || t->rows > (1 << 30) || t->sequences < 0 || t->sequences > (1 << 30) || t->slots < 0 ||
        t->slots > (1 << 30) || t->q_heads < 1 || t->kv_heads < 1 || t->q_heads > (1 << 15) ||
        t->q_heads % t->kv_heads || t->head_dim < 1)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT,
                         "%s: bad sizes rows=%lld sequences=%lld slots=%lld q_heads=%lld kv_heads=%lld head_dim=%lld", name,
                         (long long)t->rows, (long long)t->sequences, (long long)t->slots, (long long)t->q_heads,
                         (long long)t->kv_heads, (long long)t->head_dim);
    if (t->head_dim > kMaxHeadDim || t->head_dim % 8)
        return capi_fail(TRIDENT_ERR_UNSUPPORTED, "%s: head_dim=%lld is not a multiple of 8 up to %d", name,
                         (long long)t->head_dim, kMaxHeadDim);
    if (t->slots ? t->sequences * t->slots != t->rows || t->offsets : t->lengths != nullptr)
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT,
                         "%s: %lld rows are not %lld sequences of %lld slots, or offsets and lengths do not go with them",
                         name, (long long)t->rows, (long long)t->sequences, (long long)t->slots);
    // float32 holds it: a scale that became zero would make NaN of the scores that are not seen
    if (!(t->scale >= 0x1p-149) || !(t->scale < 1e30))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "%s: scale=%g", name, t->scale);
    const int64_t es = t->dtype == TRIDENT_F32 ? 4 : 2;
    const int64_t strides[6] = {t->q_row, t->q_head, t->k_row, t->k_head, t->v_row, t->v_head};
    for (int i = 0; i < 6; ++i)
        if (strides[i] < (i % 2 ? 0 : t->head_dim) || strides[i] * es % 16 || strides[i] > (i % 2 ? (int64_t)1 << 40 : (1 << 24) / es))
            return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "%s: stride %lld", name, (long long)strides[i]);
    *a = {};
    if (t->rows == 0) return TRIDENT_OK;
    if (!t->q || !t->k || !t->v || !t->out || (!t->slots && !t->offsets) ||
        (backward && (!t->lse || !t->grad || !t->dq || !t->dk || !t->dv)))
        return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "%s: NULL pointer", name);
    const void* all[] = {t->q, t->k, t->v, t->out, t->grad, t->dq, t->dk, t->dv};
    for (const void* p : all)
        if (reinterpret_cast<uintptr_t>(p) & 15)
            return capi_fail(TRIDENT_ERR_INVALID_ARGUMENT, "%s: tensors must be 16-byte aligned", name);
    a->q = t->q;
    a->k = t->k;
    a->v = t->v;
    a->grad = t->grad;
    a->out = t->out;
    a->dq = t->dq;
    a->dk = t->dk;
    a->dv = t->dv;
    a->lse = t->lse;
    a->offsets = t->offsets;
    a->lengths = t->lengths;
    a->q_row = t->q_row * es;
    a->q_head = t->q_head * es;
    a->k_row = t->k_row * es;
    a->k_head = t->k_head * es;
    a->v_row = t->v_row * es;
    a->v_head = t->v_head * es;
    a->rows = t->rows;
    a->count = t->sequences;
    a->slots = (int)t->slots;
    a->wide = t->ids64;
    a->Hq = (int)t->q_heads;
    a->Hkv = (int)t->kv_heads;
    a->D = (int)t->head_dim;
    a->causal = t->causal != 0;
    a->scale = (float)t->scale;
    a->scale2 = (float)(t->scale * 1.4426950408889634);
    return TRIDENT_OK;
}

}  // namespace trident

using namespace trident;

extern "C" int trident_attention(const TridentAttention* t, void* stream) {
    AttentionArgs a;
    const int rc = attention_check(t, false, &a);
    if (rc != TRIDENT_OK || t->rows == 0) return rc;
    int out = TRIDENT_OK;
    with_dtype(t->dtype, [&](auto e) {
        using T = decltype(e);
        const hipStream_t st = (hipStream_t)stream;
        with_bool(a.causal, [&](auto causal) {
            constexpr bool CAUSAL = decltype(causal)::value;
            if (a.D <= 32) out = launch<T, 32, CAUSAL>(a, st);
            else if (a.D <= 64) out = launch<T, 64, CAUSAL>(a, st);
            else if (a.D <= 96) out = launch<T, 96, CAUSAL>(a, st);
            else out = launch<T, 128, CAUSAL>(a, st);
        });
    });
    return out;
}
