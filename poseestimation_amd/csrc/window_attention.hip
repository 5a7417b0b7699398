// Attention with a sliding window and first tokens that stay visible, forward.
//
//   key j is seen by query i iff j <= i + right and (j >= i - left or j < sinks), j < length, visible[j]
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j - lse_i) over the seen keys; a row that sees none is zero
//
// A wave takes 32 queries of one head; a workgroup of 4 waves (or of one, for short windows, whose keys two waves may share) walks
// the tiles of 64 (32) keys that any of its queries sees: first those of the sinks, then the window.  Scores come out
// transposed (keys in registers, queries in lanes), so the softmax of a query runs inside a lane and its partner 32 lanes on,
// with a running maximum and sum, and the weighted sum of the values takes the scores where they lie.  A tile is held in LDS
// for all waves and the next one travels from memory meanwhile; tiles that every query sees whole skip the mask, and a wave
// skips a tile that none of its queries sees.
// Scores and sums are float32; the weights (at most 2^kSlack) are rounded to the element type for the second product.  The sum
// that divides the result is that of the rounded weights: the result is a mean of the values whose weights are off by relative
// errors alone, so a row that one key dominates is as exact as that key's value, which the backward's differences need.  What
// the backward takes the weights from, the logarithm of the sum, is that of the weights before rounding.
//
// Bound by the matrix and vector units taking turns: the softmax of a block takes about as long as its products, and two waves
// per SIMD, all that the registers hold, do not hide one behind the other (counters of 8192 tokens x 16 heads of 128, 1040 keys:
// matrix units busy 31 % of the time, vector units 39 %).  bfloat16, each with the flops of the pairs that are seen: that prompt
// 98 to 115 us with the clocks (670 to 570 Tflop/s), all keys of 2 x 4096 x 16: heads of 64 228 us (605), of 128 332 us (830);
// 4 x 4096 x 8 x 64 with 256 keys and 4 sinks 36 us (240; blocks cut by the window's edges and the sinks' add a third to the
// products, and a workgroup's eight tiles leave its first loads exposed).  A large product reaches 1100.  float32 in its three
// parts: 4 x 4096 x 8 x 64, 1024 keys, 206 us.
#include "attention_tiles.h"

namespace mvx {

namespace {

constexpr float kSlack = 8.0f;  // in powers of 2; float16 holds weights up to 2^15

// The registers are cut for two waves per SIMD where they suffice: with one, a long prompt of heads of 128 took 1.8 times as long.
// kWaves: waves with queries of their own, which share tiles; kSplit: waves that share the queries of one, each with every
// kSplit-th tile, kept to itself.
template <typename T, int DP, int kWaves, int kSplit>
__global__ __launch_bounds__(64 * kWaves * kSplit, kWaves > 1 && sizeof(T) * DP <= 256 ? 2 : 1) void window_attention(
    TokenTensor q, TokenTensor k, TokenTensor v, AttentionShape a, int q_blocks, T* __restrict__ out, float* __restrict__ lse,
    T* __restrict__ rest) {
    using Tl = Tiles<T, DP>;
    constexpr int DT = DP / 32, kBQ = 32 * kWaves, kBK = kWaves == 1 ? 32 : kTileRows<T>;  // queries of the workgroup, keys of a tile
    // Copies of the loop over blocks of 32 keys: of longer heads two need more registers than two waves per SIMD have (4 x 4096 x
    // 8 x 64 bfloat16, 255 keys: 37 us with one, 35 with two).
    constexpr int kBlocks = DP <= 64 ? kBK / 32 : 1;
    __shared__ __attribute__((aligned(16))) typename Tl::Cell k_tile[kSplit][2][kBK * Tl::LD];
    __shared__ __attribute__((aligned(16))) typename Tl::Cell v_tile[kSplit][2][kBK * Tl::LD];
    // heads that share keys, then blocks of queries, are neighbours on one XCD
    unsigned id = xcd_contiguous(blockIdx.x, gridDim.x);
    const int share = a.heads / a.kv_heads;
    const int in_group = id % share;
    id /= share;
    const int block = id % q_blocks;
    id /= q_blocks;
    const int kv_head = id % a.kv_heads;
    const int64_t seq = id / a.kv_heads;
    const int head = kv_head * share + in_group;
    const int half = lane_id() >> 5, wave = kSplit == 1 ? wave_id() : 0, part = kSplit == 1 ? 0 : wave_id();
    const int length = seq_length(a, seq);
    const int q0 = block * kBQ, w0 = q0 + wave * 32;  // the workgroup's and the wave's first query

    const T* kb = static_cast<const T*>(k.p) + seq * k.seq + kv_head * k.head;
    const T* vb = static_cast<const T*>(v.p) + seq * v.seq + kv_head * v.head;
    const T* qb = static_cast<const T*>(q.p) + seq * q.seq + head * q.head;
    const int mine = w0 + (lane_id() & 31);  // this lane's query, and the keys it sees: j <= hi and (j >= lo or j < sinks)
    const int hi = mine < length ? min(mine + a.right, length - 1) : -1, lo = mine - a.left;
    typename Tl::Frag qf;
    Tl::load_column(qf, qb + static_cast<int64_t>(mine) * q.token, a.dim, mine < length);
    v16f acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = v16f{};
    float top = -kInf, sum = 0.0f, divisor = 0.0f;

    const KeyTiles tiles = key_tiles(a, q0, kBQ, length, kBK);
    const int n_tiles = (tiles.count - part + kSplit - 1) / kSplit;  // of this wave: part, part + kSplit, ...
    TileInFlight<T, DP, kBK, 64 * kWaves> k_next, v_next;
    k_next.place(k.token, a.dim);
    v_next.place(v.token, a.dim);
    bool kept_next = false;
    const auto fetch = [&](int t) {
        const int k0 = tiles.key0(part + t * kSplit, kBK);
        k_next.load(kb, k.token, k0, length);
        v_next.load(vb, v.token, k0, length);
        kept_next = token_kept(a, seq, k0, length);
    };
    const auto put = [&](int t) {
        const uint64_t keep = __ballot(kept_next);
        if (a.visible != nullptr && keep != ~0ull) {
            k_next.hide(keep);
            v_next.hide(keep);
        }
        k_next.store(k_tile[part][t & 1]);
        v_next.store(v_tile[part][t & 1]);
        return keep;
    };
    uint64_t keep = 0, keep_next = 0;
    if (n_tiles > 0) {
        fetch(0);
        keep_next = put(0);
    }
    if (n_tiles > 1) fetch(1);
    for (int t = 0; t < n_tiles; ++t) {
        keep = keep_next;
        // tile t is in LDS, and nobody reads tile t - 1 any more
        if constexpr (kSplit == 1)
            __syncthreads();
        else
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (t + 1 < n_tiles) keep_next = put(t + 1);
        if (t + 2 < n_tiles) fetch(t + 2);
        const int k0 = tiles.key0(part + t * kSplit, kBK);
        const typename Tl::Cell *kt = k_tile[part][t & 1], *vt = v_tile[part][t & 1];
#pragma unroll kBlocks
        for (int b = 0; b < kBK; b += 32) {
            if (!sees_any(a, w0, k0 + b, 32, length)) continue;
            typename Tl::Pool pool;
            Tl::rows(pool, kt + b * Tl::LD);
            v16f s = Tl::rows_times(pool, qf);
            Tl::cols(pool, vt + b * Tl::LD);
            const unsigned kept = static_cast<unsigned>(keep >> b);
            if (kept != ~0u || !sees_all(a, w0, k0 + b, 32, length)) {
                const int at = k0 + b + 4 * half;  // register i is key at + 8 (i / 4) + i % 4
                const int hi_r = hi - at, lo_r = lo - at, sink_r = a.sinks - at;
                if (a.visible == nullptr && k0 + b >= a.sinks) {  // one range of keys, lo <= key <= hi
                    const int from = hi < lo ? 1 << 30 : lo_r;  // a query at or behind the length sees none
                    const unsigned span = hi < lo ? 0 : hi - lo;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        s[i] = static_cast<unsigned>(8 * (i / 4) + i % 4 - from) <= span ? s[i] : -kInf;
                } else {
                    const unsigned bits = kept >> (4 * half);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int r = 8 * (i / 4) + i % 4;
                        const bool seen = (r <= hi_r) & ((r >= lo_r) | (r < sink_r)) & ((bits >> r) & 1);
                        s[i] = seen ? s[i] : -kInf;
                    }
                }
            }
            float most = s[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) most = fmaxf(most, s[i]);
            most = both_halves_max(most) * a.scale_log2;
            // The reference of the exponents moves only when a score passes it by 2^kSlack: weights stay below that, and what
            // they lose in the rounding to 16 bits is relative.
            if (__any(most > top + kSlack)) {
                const float next = fmaxf(top, most), f = __builtin_amdgcn_exp2f(top - (next == -kInf ? 0.0f : next));
                sum *= f;
                divisor *= f;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;  // top = -inf: 0
                top = next;
            }
            const float ref = top == -kInf ? 0.0f : top;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale_log2, -ref));
            Tl::cols_times(pool, s, acc);
            if constexpr (sizeof(T) == 2) divisor = Tl::rounded_sum(s, divisor);
            if (sizeof(T) == 4 || lse != nullptr) {
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += s[i];
            }
        }
    }
    if constexpr (kSplit > 1) {  // the waves' lanes hold the same queries: the first adds up what the others leave, in order
        __shared__ float left_by[kSplit - 1][DT * 16 + 3][64];
        if (part > 0) {
            float(*mine)[64] = left_by[part - 1];
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) mine[dt * 16 + i][lane_id()] = acc[dt][i];
            mine[DT * 16][lane_id()] = top;
            mine[DT * 16 + 1][lane_id()] = sum;
            mine[DT * 16 + 2][lane_id()] = divisor;
        }
        __syncthreads();
        if (part > 0) return;
#pragma unroll
        for (int n = 0; n < kSplit - 1; ++n) {
            const float top2 = left_by[n][DT * 16][lane_id()], next = fmaxf(top, top2), ref = next == -kInf ? 0.0f : next;
            const float f = __builtin_amdgcn_exp2f(top - ref), f2 = __builtin_amdgcn_exp2f(top2 - ref);
            top = next;
            sum = sum * f + left_by[n][DT * 16 + 1][lane_id()] * f2;
            divisor = divisor * f + left_by[n][DT * 16 + 2][lane_id()] * f2;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[dt][i] = acc[dt][i] * f + left_by[n][dt * 16 + i][lane_id()] * f2;
        }
    }
    sum = both_halves_sum(sum);
    divisor = sizeof(T) == 2 ? both_halves_sum(divisor) : sum;
    if (in_either_half(mine < length && !(all_finite(acc) && divisor < kInf))) {
        const T* qr = qb + static_cast<int64_t>(mine) * q.token;
        top = -kInf;
        sum = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] = v16f{};
        bool nan = false;
        for_seen_keys(a, seq, lo, hi, [&](int j) {
            const float x = dot_rows(qr, kb + j * k.token, a.dim) * a.scale_log2;
            nan |= x != x;
            top = fmaxf(top, x);
        });
        // Scores of minus infinity alone leave an empty row, as if no key were seen; NaN among them do not.
        if (nan && top == -kInf) top = 0.0f;
        for_seen_keys(a, seq, lo, top == -kInf ? -1 : hi, [&](int j) {
            const float p = __builtin_amdgcn_exp2f(dot_rows(qr, kb + j * k.token, a.dim) * a.scale_log2 - top);
            sum += p;
            add_row<T, DP>(acc, p, vb + j * v.token, a.dim);
        });
        divisor = sum;
    }
    if (mine >= a.n_tokens) return;
    const bool none = top == -kInf;
    if (lse != nullptr && half == 0)  // log2; an empty row's makes its weights zero
        lse[(seq * a.heads + head) * a.n_tokens + mine] = none ? kInf : top + __builtin_amdgcn_logf(sum);
    const float factor = none ? 0.0f : 1.0f / divisor;
    const int64_t row = ((seq * a.n_tokens + mine) * a.heads + head) * a.dim;
    store_columns<T, DP>(acc, factor, out + row, a.dim, sizeof(T) == 2 && lse != nullptr ? rest + row : nullptr);
}

}  // namespace

// Checks that the forward and the backward share; fills `s`.
int attention_shape(const char* name, int dtype, int64_t n_seqs, int64_t n_tokens, int heads, int kv_heads, int dim,
                    int64_t left, int64_t right, int64_t sinks, float scale, const int64_t* lengths, const uint8_t* visible,
                    AttentionShape* s) {
    MVX_REQUIRE(dtype == MVX_F32 || dtype == MVX_BF16 || dtype == MVX_F16, MVX_ERR_INVALID_ARGUMENT, "%s: unknown element type %d",
                name, dtype);
    MVX_REQUIRE(n_seqs >= 0 && n_tokens >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0, MVX_ERR_INVALID_ARGUMENT,
                "%s: bad shape n_seqs=%lld n_tokens=%lld heads=%d kv_heads=%d", name, (long long)n_seqs, (long long)n_tokens,
                heads, kv_heads);
    MVX_REQUIRE(dim > 0 && dim % 8 == 0, MVX_ERR_INVALID_ARGUMENT, "%s: head dimension %d is not a multiple of 8", name, dim);
    MVX_REQUIRE(dim <= 128, MVX_ERR_UNSUPPORTED, "%s: head dimension %d above 128", name, dim);
    MVX_REQUIRE(n_tokens <= (1 << 30), MVX_ERR_UNSUPPORTED, "%s: more than 2^30 tokens", name);
    MVX_REQUIRE(left >= 0 && right >= 0 && sinks >= 0, MVX_ERR_INVALID_ARGUMENT, "%s: bad window (%lld, %lld) or sinks %lld", name,
                (long long)left, (long long)right, (long long)sinks);
    MVX_REQUIRE(scale > 0.0f && scale < kInf, MVX_ERR_INVALID_ARGUMENT, "%s: scale must be positive and finite", name);
    const auto within = [&](int64_t x) { return static_cast<int>(x < n_tokens ? x : n_tokens); };
    *s = {n_seqs, static_cast<int>(n_tokens), heads, kv_heads, dim, within(left), within(right), within(sinks), scale * kLog2e,
          lengths, visible};
    return MVX_OK;
}

int attention_tensor(const char* name, const char* what, const void* p, const int64_t* strides, int dtype, int64_t n_seqs,
                     int64_t n_tokens, int heads, int dim, TokenTensor* t) {
    MVX_REQUIRE(p != nullptr && strides != nullptr, MVX_ERR_INVALID_ARGUMENT, "%s: null pointer (%s)", name, what);
    // the stride of an axis of length 1 is never used, whatever it says
    *t = {p, n_seqs > 1 ? strides[0] : 0, n_tokens > 1 ? strides[1] : dim, heads > 1 ? strides[2] : 0};
    const int64_t vec = 16 / element_bytes(dtype);
    MVX_REQUIRE(aligned16(p) && t->seq % vec == 0 && t->token % vec == 0 && t->head % vec == 0, MVX_ERR_INVALID_ARGUMENT,
                "%s: %s must be 16-byte aligned in its base and strides", name, what);
    // a tile of 64 tokens is addressed with 31 bits, and bounded by its last token
    MVX_REQUIRE(t->token >= dim && t->token < (1LL << 31) / 64 / element_bytes(dtype), MVX_ERR_INVALID_ARGUMENT,
                "%s: tokens of %s must be at least a head (%d values) and less than 2^25 bytes apart, got %lld values", name, what,
                dim, (long long)t->token);
    return MVX_OK;
}

}  // namespace mvx

extern "C" size_t mvx_window_attention_saved_bytes(int dtype, int64_t n_seqs, int64_t n_tokens, int heads, int dim) {
    if (n_seqs <= 0 || n_tokens <= 0 || heads <= 0 || dim <= 0) return 0;
    const int64_t rows = n_seqs * n_tokens * heads;
    return static_cast<size_t>(mvx::padded_rows(rows)) * sizeof(float) + (dtype == MVX_F32 ? 0 : static_cast<size_t>(rows) * dim * 2);
}

extern "C" int mvx_window_attention(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                    const void* v, const int64_t* v_strides, int dtype, int64_t n_seqs, int64_t n_tokens,
                                    int heads, int kv_heads, int dim, int64_t left, int64_t right, int64_t sinks, float scale,
                                    const int64_t* lengths, const uint8_t* visible, void* out, void* saved, void* stream) {
    using namespace mvx;
    const char* name = "mvx_window_attention";
    AttentionShape s;
    int rc = attention_shape(name, dtype, n_seqs, n_tokens, heads, kv_heads, dim, left, right, sinks, scale, lengths, visible, &s);
    if (rc != MVX_OK) return rc;
    if (n_seqs == 0 || n_tokens == 0) return MVX_OK;
    TokenTensor qt, kt, vt;
    if ((rc = attention_tensor(name, "q", q, q_strides, dtype, n_seqs, n_tokens, heads, dim, &qt)) != MVX_OK) return rc;
    if ((rc = attention_tensor(name, "k", k, k_strides, dtype, n_seqs, n_tokens, kv_heads, dim, &kt)) != MVX_OK) return rc;
    if ((rc = attention_tensor(name, "v", v, v_strides, dtype, n_seqs, n_tokens, kv_heads, dim, &vt)) != MVX_OK) return rc;
    MVX_REQUIRE(out != nullptr && aligned16(out), MVX_ERR_INVALID_ARGUMENT, "%s: out is null or not 16-byte aligned", name);
    MVX_REQUIRE(aligned16(saved), MVX_ERR_INVALID_ARGUMENT, "%s: saved is not 16-byte aligned", name);
    float* lse = static_cast<float*>(saved);
    // Four waves share their tiles, and wait for each other's: of a window of w keys a wave sees 32 + w, the workgroup 128 + w.
    // Short windows are therefore walked by single waves where their tiles leave room for enough of them: always with 16-bit
    // types (4 x 4096 tokens x 8 heads x 64, 33 keys: 22.8 -> 20.7 us; from 255 keys on four waves are faster), with float32, whose
    // tiles are three times as large, up to one round of them (257 tokens x 4 heads x 64, 33 keys: 15.9 -> 12.7 us; 4 x 2000 x 4 x
    // 32, 127 keys: 14.9 -> 12.8, but 4 x 4096 x 8 x 32, 33 keys: 27.4 -> 31.8).
    const int64_t all_waves = n_seqs * heads * ((n_tokens + 31) / 32);
    const bool room = dtype != MVX_F32 || all_waves <= (dim <= 32 ? 1536 : 768);
    const int waves = dim <= 64 && static_cast<int64_t>(s.left) + s.right < 128 && room ? 1 : 4;
    // Float32, where a tile's chain of products is three times as long: two waves share the queries of one where that still leaves
    // every SIMD one wave at most (257 tokens x 4 heads x 64, 33 keys, some hidden: 15.3 -> 12.7 us; 512 x 8 x 64, 127 keys: 18.7 ->
    // 14.0; 752 waves of 2 x 1500 x 8 x 32, 101 keys: 14.7 -> 21).
    const bool split = dtype == MVX_F32 && waves == 1 && all_waves <= 512;
    const int q_blocks = static_cast<int>((n_tokens + 32 * waves - 1) / (32 * waves));
    // 2^31 threads in one launch
    MVX_REQUIRE(n_seqs <= (1 << 25) / waves / q_blocks / heads, MVX_ERR_UNSUPPORTED,
                "%s: too many sequences, heads and tokens for one launch", name);
    const unsigned blocks = static_cast<unsigned>(n_seqs * heads * q_blocks);
    return with_element(dtype, name, [&](auto zero) -> int {
        using T = decltype(zero);
        T* rest = reinterpret_cast<T*>(lse != nullptr ? lse + padded_rows(n_seqs * heads * n_tokens) : nullptr);
        const auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * waves * (split ? 2 : 1)), 0, static_cast<hipStream_t>(stream), qt, kt,
                               vt, s, q_blocks, static_cast<T*>(out), lse, rest);
        };
        if constexpr (sizeof(T) == 4) {
            if (split) {
                dim <= 32 ? launch(window_attention<T, 32, 1, 2>) : launch(window_attention<T, 64, 1, 2>);
                MVX_CHECK_LAUNCH(name);
                return MVX_OK;
            }
        }
        if (dim <= 32)
            waves == 1 ? launch(window_attention<T, 32, 1, 1>) : launch(window_attention<T, 32, 4, 1>);
        else if (dim <= 64)
            waves == 1 ? launch(window_attention<T, 64, 1, 1>) : launch(window_attention<T, 64, 4, 1>);
        else if (dim <= 96)
            launch(window_attention<T, 96, 4, 1>);
        else
            launch(window_attention<T, 128, 4, 1>);
        MVX_CHECK_LAUNCH(name);
        return MVX_OK;
    });
}
