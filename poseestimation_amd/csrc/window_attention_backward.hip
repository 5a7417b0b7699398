// Backward of the windowed attention.  With p_ij = exp(scale q_i . k_j - lse_i) over the seen pairs and g = dL/do:
//
//   dv_j = sum_i p_ij g_i          dp_ij = g_i . v_j         delta_i = g_i . o_i = sum_j p_ij dp_ij
//   ds_ij = p_ij (dp_ij - delta_i)  dq_i = scale sum_j ds_ij k_j   dk_j = scale sum_i ds_ij q_i
//
// Two kernels, each recomputing p from the scores and the forward's lse, so that every gradient is summed in registers in a
// fixed order and no atomics are needed (two more products of five; the result is the same in every run):
//   1. queries in lanes, walking the tiles of keys as the forward does: delta and dq;
//   2. keys in lanes, walking the tiles of queries that see them, over all heads that share the keys: dk and dv.
// In the second a block of sink keys is seen by the whole rest of the sequence.  The queries behind the block's own window
// are therefore cut into chunks that a third kernel takes, between the two: a workgroup per chunk and 32 sinks, its waves
// on queries of their own, its sum left in float32.  A fourth adds the chunks in order, and the block of keys adds that to its own
// (but for many sinks, whose blocks fill the GPU and walk all queries).
// delta is taken from the output together with what its rounding left: a row that one key dominates has dp - delta near zero
// there, and the output rounded to bfloat16 alone would be off by as much as the difference (three keys of unit spread: dq and dk
// off by 0.0033 of their size instead of 0.0025, of twice that spread 0.0066 instead of 0.0024).
// p and ds are rounded to the element type for the products they enter; scores, dp, delta and all sums are float32.  In
// bfloat16 dq and dk are so off by 0.0024 of their size (one rounding of the exact ones: 0.0017); ds in two parts of 16 bits would
// give 0.0018, at 10 to 20 % more time.
// A query that sees a single key weighs it with 1 whatever its score: dp - delta is zero there, but rounding would leave noise,
// which is all there is where every query sees one key.  The first kernel counts the keys a query sees, gives such a query no
// gradient, and leaves a mark in the place of its delta.  A query whose scores are all minus infinity is an empty row like one
// that sees no key: its lse is plus infinity, so its weights are zero.
//
// bfloat16, 4 x 4096 x 8 x 64 with 256 keys and 4 sinks: dq 47 us, far queries 12, their sums 5, dk and dv 48; what these have to
// read and write takes 23, 7, 1 and 20 us at a large copy's rate, the rest is the latency of a few tiles per workgroup.  All keys
// of 2 x 4096 x 8 x 64: 295 us together (580 Tflop/s of the five products that are counted; two more are computed), of
// 4096 x 16 x 128, causal: 424 us (405), one wave per SIMD.
#include "attention_tiles.h"

namespace mvx {

namespace {

constexpr int kBlock = 128;  // queries and keys of a workgroup of four waves; where the far queries of sinks begin

// In the place of a query's delta: it sees a single key.  A NaN of its own, which no arithmetic makes.
constexpr unsigned kAlone = 0x7fe5a10eu;
__device__ __forceinline__ bool is_alone(float delta) { return __builtin_bit_cast(unsigned, delta) == kAlone; }

// Both kernels run two blocks of 32 rows of a tile of 64 in one piece of code, and the registers are cut for two waves per SIMD up
// to heads of 64; longer ones gain more from two blocks in flight in one wave than from a second wave (4096 x 16 x 128 bfloat16,
// causal: dq 337 us with two waves, 283 with one, 246 with one and two blocks; dk and dv 234 and 219; 2 x 2000 x 8 x 96 float16:
// 75 and 67 us together.  4 x 4096 x 8 x 64 bfloat16, 255 keys, one block: dq 50 instead of 47, dk and dv 49 instead of 48).
template <typename T, int DP, int kWaves>
constexpr int kPerSimd = sizeof(T) * DP <= 128 || (kWaves == 4 && DP <= 64) ? 2 : 1;

// float16 is exact to its half step from 2^-14 to 2^16 only, and score gradients may lie anywhere: as small as the weights of a
// long window times what the loss left, as large as its scaling made them.  Every column (a query for dq, a key for dk) therefore
// carries its sums times a power of two: the first block of score gradients above 2^(15 - kFirstPower) brings its largest to
// 2^5 .. 2^6, which leaves 19 binades below it, and one that passes 2^15 later lowers the power again, with the sums so far.
// Weights are at most 1 and enter dv times 2^kWeightPower.  The other types have float32's range and no power.
// Without it (4096 causal tokens, gradients of 1e-3 and 1e-4) dq and dk are off by 0.0016 and 0.016 of their size instead of 0.0004
// and 0.0028, of which one rounding of the exact ones is 0.0003 and 0.0028, and score gradients beyond 65504 are infinite.  It costs
// the largest of 16 values and, for dk, a product each: 4 x 4096 x 8 x 64 with 255 keys 113 -> 119 us, all keys of 2 x 4096 x 8 x 64
// 299 -> 317, 4096 x 16 x 128 causal 423 -> 482.
template <typename T>
constexpr bool kScaled = std::is_same_v<T, f16>;
template <typename T>
constexpr int kFirstPower = kScaled<T> ? 60 : 0;
template <typename T>
constexpr int kWeightPower = kScaled<T> ? 14 : 0;

// Lowers the powers where the block `ds`, already times 2^power, needs it; whether any lane's has moved.
template <int N>
__device__ __forceinline__ bool fit(v16f& ds, int& power, v16f (&acc)[N]) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) most = fmaxf(fmaxf(most, fabsf(ds[i])), fabsf(ds[i + 1]));
    if (__builtin_expect(!__any(most > 0x1p15f), 1)) return false;
    most = both_halves_max(most);
    const int by = most > 0x1p15f && most < kInf ? 6 - __builtin_amdgcn_frexp_expf(most) : 0;
    const float f = __builtin_amdgcn_ldexpf(1.0f, by);
    power += by;
    ds *= f;
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] *= f;
    return true;
}
template <int N>
__device__ __forceinline__ void unscale(v16f (&acc)[N], int power) {
    const float f = __builtin_amdgcn_ldexpf(1.0f, -power);
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] *= f;
}

// The lowest n bits.
__device__ __forceinline__ uint64_t below(int n) { return n <= 0 ? 0 : (n >= 64 ? ~0ull : (1ull << n) - 1); }

template <typename T, int DP, int kWaves>
__global__ __launch_bounds__(64 * kWaves, (kPerSimd<T, DP, kWaves>)) void window_attention_dq(
    TokenTensor q, TokenTensor k, TokenTensor v, TokenTensor o, const T* __restrict__ rest, TokenTensor g, AttentionShape a,
    float scale, int q_blocks, const float* __restrict__ lse, float* __restrict__ delta, T* __restrict__ dq) {
    using Tl = Tiles<T, DP>;
    constexpr int kThreads = 64 * kWaves, kMine = 32 * kWaves, kTile = kTileRows<T>, kBlocks = kTile / 32;
    __shared__ __attribute__((aligned(16))) typename Tl::Cell k_tile[2][kTile * Tl::LD];
    __shared__ __attribute__((aligned(16))) typename Tl::Cell v_tile[2][kTile * Tl::LD];
    unsigned id = xcd_contiguous(blockIdx.x, gridDim.x);
    const int share = a.heads / a.kv_heads;
    const int in_group = id % share;
    id /= share;
    const int block = id % q_blocks;
    id /= q_blocks;
    const int kv_head = id % a.kv_heads;
    const int64_t seq = id / a.kv_heads;
    const int head = kv_head * share + in_group;
    const int half = lane_id() >> 5, wave = wave_id();
    const int length = seq_length(a, seq);
    const int q0 = block * kMine, w0 = q0 + wave * 32, mine = w0 + (lane_id() & 31);

    const T* kb = static_cast<const T*>(k.p) + seq * k.seq + kv_head * k.head;
    const T* vb = static_cast<const T*>(v.p) + seq * v.seq + kv_head * v.head;
    const bool live = mine < length;
    const T* q_row = static_cast<const T*>(q.p) + seq * q.seq + static_cast<int64_t>(mine) * q.token + head * q.head;
    const T* g_row = static_cast<const T*>(g.p) + seq * g.seq + static_cast<int64_t>(mine) * g.token + head * g.head;
    typename Tl::Frag qf, gf;
    Tl::load_column(qf, q_row, a.dim, live);
    Tl::load_column(gf, g_row, a.dim, live);
    float my_lse = 0.0f;
    const T* o_row = static_cast<const T*>(o.p) + seq * o.seq + static_cast<int64_t>(mine) * o.token + head * o.head;
    float my_delta;
    if constexpr (sizeof(T) == 2) {
        typename Tl::Frag of, rf;
        Tl::load_column(of, o_row, a.dim, live);
        Tl::load_column(rf, rest + ((seq * a.n_tokens + mine) * a.heads + head) * a.dim, a.dim, live);
        my_delta = both_halves_sum(Tl::dot(gf, of, rf));
    } else {
        my_delta = both_halves_sum(half_dot(g_row, o_row, a.dim, live));
    }
    const int64_t at_row = (seq * a.heads + head) * a.n_tokens + mine;
    if (live) my_lse = lse[at_row];

    const int hi = live ? min(mine + a.right, length - 1) : -1, lo = mine - a.left;
    const KeyTiles tiles = key_tiles(a, q0, kMine, length, kTile);
    // Counted ahead of the products, which have no registers left (counting along with them took 3 to 6 % more time).
    int n_seen = max(0, hi + 1 - max(lo, 0)) + max(0, min(min(a.sinks, hi + 1), lo));
    if (a.visible != nullptr) {
        n_seen = 0;
        for (int t = 0; t < tiles.count && __any(live && n_seen < 2); ++t) {
            const int k0 = tiles.key0(t, kTile);
            const uint64_t keep = __ballot(token_kept(a, seq, k0, length)) & below(kTile);
            n_seen += __popcll(keep & below(hi + 1 - k0) & (~below(lo - k0) | below(a.sinks - k0)));
        }
    }
    // not where the key or what it gave is infinite or NaN: 0 times that is NaN
    const bool alone = n_seen == 1 && __builtin_isfinite(my_lse) && __builtin_isfinite(my_delta);
    if (mine < a.n_tokens && half == 0) delta[at_row] = alone ? __builtin_bit_cast(float, kAlone) : my_delta;
    if (alone) my_lse = kInf;  // weights of zero: no gradient
    v16f acc[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = v16f{};
    int power = kFirstPower<T>;
    float shift = kScaled<T> ? static_cast<float>(power) - my_lse : -my_lse;

    TileInFlight<T, DP, kTile, kThreads> k_next, v_next;
    k_next.place(k.token, a.dim);
    v_next.place(v.token, a.dim);
    bool kept_next = false;
    const auto fetch = [&](int t) {
        const int k0 = tiles.key0(t, kTile);
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
        k_next.store(k_tile[t & 1]);
        v_next.store(v_tile[t & 1]);
        return keep;
    };
    uint64_t keep = 0, keep_next = 0;
    if (tiles.count > 0) {
        fetch(0);
        keep_next = put(0);
    }
    if (tiles.count > 1) fetch(1);
    for (int t = 0; t < tiles.count; ++t) {
        keep = keep_next;
        __syncthreads();
        if (t + 1 < tiles.count) keep_next = put(t + 1);
        if (t + 2 < tiles.count) fetch(t + 2);
        const int k0 = tiles.key0(t, kTile);
        const typename Tl::Cell *kt = k_tile[t & 1], *vt = v_tile[t & 1];
        const int at = k0 + 4 * half;
        const int hi_r = hi - at, lo_r = lo - at, sink_r = a.sinks - at;
        const uint64_t bits = keep >> (4 * half);
#pragma unroll kBlocks
        for (int b = 0; b < kTile / 32; ++b) {
            if (!sees_any(a, w0, k0 + 32 * b, 32, length)) continue;
            const bool whole = static_cast<unsigned>(keep >> (32 * b)) == ~0u && sees_all(a, w0, k0 + 32 * b, 32, length);
            typename Tl::Pool pool;
            Tl::rows(pool, kt + 32 * b * Tl::LD);
            v16f s = Tl::rows_times(pool, qf);
            Tl::rows(pool, vt + 32 * b * Tl::LD);
            const v16f dp = Tl::rows_times(pool, gf);
            Tl::cols(pool, kt + 32 * b * Tl::LD);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale_log2, shift)) * (dp[i] - my_delta);
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = 32 * b + 8 * (i / 4) + i % 4;
                    s[i] = (r <= hi_r) & ((r >= lo_r) | (r < sink_r)) & ((bits >> r) & 1) ? s[i] : 0.0f;
                }
            }
            if constexpr (kScaled<T>)
                if (fit(s, power, acc)) shift = static_cast<float>(power) - my_lse;
            Tl::cols_times(pool, s, acc);
        }
    }
    if constexpr (kScaled<T>) unscale(acc, power);
    if (in_either_half(live && !all_finite(acc))) {
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = v16f{};
        // not of an empty row, or one without a gradient: its weights are zero, and zero times an infinite key is a NaN
        for_seen_keys(a, seq, lo, my_lse == kInf ? -1 : hi, [&](int j) {
            const float p = __builtin_amdgcn_exp2f(fmaf(dot_rows(q_row, kb + j * k.token, a.dim), a.scale_log2, -my_lse));
            add_row<T, DP>(acc, p * (dot_rows(g_row, vb + j * v.token, a.dim) - my_delta), kb + j * k.token, a.dim);
        });
    }
    if (mine < a.n_tokens) store_columns<T, DP>(acc, scale, dq + ((seq * a.n_tokens + mine) * a.heads + head) * a.dim, a.dim);
}

// First query behind the window of the 128 keys from k0 on: those from here on see its sinks alone.
__device__ __forceinline__ int window_end(const AttentionShape& a, int k0, int length) {
    return min(length, k0 + kBlock + a.left);
}
// Sums of 32 sinks over one chunk of queries, in the order of the registers: [4 registers][dk, dv][lane][4].
template <int DP>
constexpr int64_t kSinkSums = static_cast<int64_t>(DP) * 32 * 2;
template <int DP>
__device__ __forceinline__ v4f* sink_vec(float* sums, int dt, int i4, int which) {
    return reinterpret_cast<v4f*>(sums) + ((dt * 4 + i4) * 2 + which) * 64 + lane_id();
}
template <int DP>
__device__ __forceinline__ int64_t sink_sums(const AttentionShape& a, int64_t seq, int kv_head, int sink_block, int chunks) {
    return ((seq * a.kv_heads + kv_head) * ((a.sinks + 31) / 32) + sink_block) * chunks * kSinkSums<DP>;
}

// One chunk of the queries behind the window of 32 sinks.  Every wave takes 32 queries of one head at a time through tiles of
// its own (no barrier in the loop); the waves' sums are added in order at the end.
template <typename T, int DP>
constexpr int kSinkWaves = sizeof(T) * DP > 384 ? 2 : 4;  // float32 heads of 128: 49 KB of tiles per wave
template <typename T, int DP>
__global__ __launch_bounds__(64 * (kSinkWaves<T, DP>), sizeof(T) * DP <= 192 ? 2 : 1) void window_attention_sinks(
    TokenTensor q, TokenTensor k, TokenTensor v, TokenTensor g, AttentionShape a, int chunk, int chunks,
    const float* __restrict__ lse, const float* __restrict__ delta, float* __restrict__ partial) {
    using Tl = Tiles<T, DP>;
    constexpr int kOwn = kSinkWaves<T, DP>;
    struct WaveTiles {
        __attribute__((aligned(16))) typename Tl::Cell q[32 * Tl::LD];
        __attribute__((aligned(16))) typename Tl::Cell g[32 * Tl::LD];
        __attribute__((aligned(16))) float stats[2][32];  // lse, delta
    };
    __shared__ union Shared {
        WaveTiles wave[kOwn];
        __attribute__((aligned(16))) float sums[kSinkSums<DP>];
    } shared;
    unsigned id = xcd_contiguous(blockIdx.x, gridDim.x);
    const int c = id % chunks;
    id /= chunks;
    const int sink_blocks = (a.sinks + 31) / 32, block = id % sink_blocks;
    id /= sink_blocks;
    const int kv_head = id % a.kv_heads;
    const int64_t seq = id / a.kv_heads;
    const int share = a.heads / a.kv_heads;
    const int lane = lane_id(), half = lane >> 5, wave = wave_id();
    const int length = seq_length(a, seq), mine = block * 32 + (lane & 31);
    const int begin = window_end(a, block * 32 / kBlock * kBlock, length) + c * chunk, end = min(length, begin + chunk);
    if (begin >= end) return;  // the block of keys reads the chunks that its length leaves, no others
    const int per_head = (end - begin + 31) / 32, items = per_head * share;

    const bool kept = mine < min(a.sinks, length) && (a.visible == nullptr || a.visible[seq * a.n_tokens + mine] != 0);
    typename Tl::Frag kf, vf;
    Tl::load_column(kf, static_cast<const T*>(k.p) + seq * k.seq + static_cast<int64_t>(mine) * k.token + kv_head * k.head, a.dim, kept);
    Tl::load_column(vf, static_cast<const T*>(v.p) + seq * v.seq + static_cast<int64_t>(mine) * v.token + kv_head * v.head, a.dim, kept);
    v16f dk_acc[DP / 32], dv_acc[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) dk_acc[dt] = dv_acc[dt] = v16f{};
    int power = kFirstPower<T> - kWeightPower<T>;
    float gain = __builtin_amdgcn_ldexpf(1.0f, power);

    WaveTiles& tile = shared.wave[wave];
    TileInFlight<T, DP, 32, 64> q_next, g_next;
    q_next.place(q.token, a.dim);
    g_next.place(g.token, a.dim);
    for (int t = wave; t < items; t += kOwn) {
        const int head = kv_head * share + t / per_head, i0 = begin + t % per_head * 32;
        q_next.load(static_cast<const T*>(q.p) + seq * q.seq + head * q.head, q.token, i0, end);
        g_next.load(static_cast<const T*>(g.p) + seq * g.seq + head * g.head, g.token, i0, end);
        const int row = i0 + (lane & 31);
        const float stat = row < end ? (half == 0 ? lse : delta)[(seq * a.heads + head) * a.n_tokens + row] : 0.0f;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's reads of the last tile come before these writes
        q_next.store(tile.q);
        g_next.store(tile.g);
        tile.stats[half][lane & 31] = half == 0 ? stat - kWeightPower<T> : stat;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        typename Tl::Pool pool;
        Tl::rows(pool, tile.q);
        v16f s = Tl::rows_times(pool, kf);
        Tl::rows(pool, tile.g);
        v16f dp = Tl::rows_times(pool, vf);
        Tl::cols(pool, tile.g);
        const int rows = end - i0 - 4 * half;
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
            const v4f l4 = *reinterpret_cast<const v4f*>(&tile.stats[0][8 * i4 + 4 * half]);
            const v4f d4 = *reinterpret_cast<const v4f*>(&tile.stats[1][8 * i4 + 4 * half]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 4 * i4 + e;
                const float p = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale_log2, -l4[e]));
                const float ds = (kScaled<T> ? p * gain : p) * (dp[i] - d4[e]);
                const bool seen = kept && 8 * i4 + e < rows;
                s[i] = seen ? p : 0.0f;
                dp[i] = seen && !is_alone(d4[e]) ? ds : 0.0f;
            }
        }
        Tl::cols_times(pool, s, dv_acc);
        Tl::cols(pool, tile.q);
        if constexpr (kScaled<T>)
            if (fit(dp, power, dk_acc)) gain = __builtin_amdgcn_ldexpf(1.0f, power);
        Tl::cols_times(pool, dp, dk_acc);
    }
    if constexpr (kScaled<T>) {
        unscale(dk_acc, power + kWeightPower<T>);
        unscale(dv_acc, kWeightPower<T>);
    }
    __syncthreads();
    for (int w = 0; w < kOwn; ++w) {
        if (w == wave) {
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    v4f k4, v4;
#pragma unroll
                    for (int e = 0; e < 4; ++e) k4[e] = dk_acc[dt][4 * i4 + e], v4[e] = dv_acc[dt][4 * i4 + e];
                    v4f *pk = sink_vec<DP>(shared.sums, dt, i4, 0), *pv = sink_vec<DP>(shared.sums, dt, i4, 1);
                    *pk = w == 0 ? k4 : *pk + k4;
                    *pv = w == 0 ? v4 : *pv + v4;
                }
        }
        __syncthreads();
    }
    float* out = partial + sink_sums<DP>(a, seq, kv_head, block, chunks) + c * kSinkSums<DP>;
    for (int i = threadIdx.x; i < kSinkSums<DP>; i += 64 * kOwn) out[i] = shared.sums[i];
}

// Adds the chunks of one block of 32 sinks (blockIdx.x) into the first of them, in order.
template <int DP>
__global__ __launch_bounds__(256) void window_attention_sinks_join(AttentionShape a, int chunk, int chunks, float* __restrict__ partial) {
    const int sink_blocks = (a.sinks + 31) / 32, block = blockIdx.x % sink_blocks;
    const int64_t seq = blockIdx.x / sink_blocks / a.kv_heads;
    const int length = seq_length(a, seq), left = length - window_end(a, block * 32 / kBlock * kBlock, length);
    v4f* p = reinterpret_cast<v4f*>(partial + static_cast<int64_t>(blockIdx.x) * chunks * kSinkSums<DP>) + blockIdx.y * 256 + threadIdx.x;
    const int filled = (left + chunk - 1) / chunk;
    if (filled <= 1) return;
    v4f sum = *p;
#pragma unroll 8
    for (int n = 1; n < filled; ++n) sum += p[n * (kSinkSums<DP> / 4)];
    *p = sum;
}

// Keys [k0, k0 + 32 kWaves) of one key/value head and the queries of the block's window.
template <typename T, int DP, int kWaves>
__global__ __launch_bounds__(64 * kWaves, (kPerSimd<T, DP, kWaves>)) void window_attention_dkv(
    TokenTensor q, TokenTensor k, TokenTensor v, TokenTensor g, AttentionShape a, float scale, int k_blocks, int chunks,
    const float* __restrict__ lse, const float* __restrict__ delta, float* __restrict__ partial, T* __restrict__ dk,
    T* __restrict__ dv) {
    using Tl = Tiles<T, DP>;
    constexpr int kThreads = 64 * kWaves, kMine = 32 * kWaves, kTile = kTileRows<T>, kBlocks = kTile / 32;
    __shared__ __attribute__((aligned(16))) typename Tl::Cell q_tile[2][kTile * Tl::LD];
    __shared__ __attribute__((aligned(16))) typename Tl::Cell g_tile[2][kTile * Tl::LD];
    __shared__ __attribute__((aligned(16))) float stats[2][2][kTile];  // of a tile: lse - kWeightPower, delta
    unsigned id = xcd_contiguous(blockIdx.x, gridDim.x);
    const int block = id % k_blocks;
    id /= k_blocks;
    const int kv_head = id % a.kv_heads;
    const int64_t seq = id / a.kv_heads;
    const int share = a.heads / a.kv_heads;
    const int half = lane_id() >> 5, wave = wave_id();
    const int length = seq_length(a, seq);
    const int k0 = block * kMine, w0 = k0 + wave * 32, mine = w0 + (lane_id() & 31);
    const int begin = max(0, k0 - a.right);
    // without chunks the sinks' block walks their far queries itself
    const int end = k0 >= a.sinks ? min(length, k0 + kMine + a.left) : chunks > 0 ? window_end(a, k0 / kBlock * kBlock, length) : length;
    const int per_head = begin < end && k0 < length ? (end - begin + kTile - 1) / kTile : 0, tiles = per_head * share;

    const bool kept = mine < length && (a.visible == nullptr || a.visible[seq * a.n_tokens + mine] != 0);
    typename Tl::Frag kf, vf;
    Tl::load_column(kf, static_cast<const T*>(k.p) + seq * k.seq + static_cast<int64_t>(mine) * k.token + kv_head * k.head, a.dim, kept);
    Tl::load_column(vf, static_cast<const T*>(v.p) + seq * v.seq + static_cast<int64_t>(mine) * v.token + kv_head * v.head, a.dim, kept);
    // the queries that see this lane's key: lo <= i <= hi
    const int lo = mine - a.right, hi = !kept ? -1 : (mine < a.sinks ? length - 1 : min(mine + a.left, length - 1));
    const bool all_kept = __all(kept);
    // last query that sees any key of the wave
    const int wave_last = w0 < a.sinks ? length - 1 : min(w0 + 31 + a.left, length - 1);

    v16f dk_acc[DP / 32], dv_acc[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) dk_acc[dt] = dv_acc[dt] = v16f{};
    const auto add_far_queries = [&] {  // what the queries behind the window give the sinks
        if (w0 >= a.sinks || end >= length) return;
        float* sums = partial + sink_sums<DP>(a, seq, kv_head, w0 / 32, chunks);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const v4f k4 = *sink_vec<DP>(sums, dt, i4, 0), v4 = *sink_vec<DP>(sums, dt, i4, 1);
#pragma unroll
                for (int e = 0; e < 4; ++e) dk_acc[dt][4 * i4 + e] += k4[e], dv_acc[dt][4 * i4 + e] += v4[e];
            }
    };
    if constexpr (!kScaled<T>) add_far_queries();
    int power = kFirstPower<T> - kWeightPower<T>;
    float gain = __builtin_amdgcn_ldexpf(1.0f, power);

    TileInFlight<T, DP, kTile, kThreads> q_next, g_next;
    q_next.place(q.token, a.dim);
    g_next.place(g.token, a.dim);
    float stat_next = 0.0f;
    const auto fetch = [&](int t) {
        const int head = kv_head * share + t / per_head, i0 = begin + t % per_head * kTile;
        q_next.load(static_cast<const T*>(q.p) + seq * q.seq + head * q.head, q.token, i0, end);
        g_next.load(static_cast<const T*>(g.p) + seq * g.seq + head * g.head, g.token, i0, end);
        const int r = i0 + (threadIdx.x & (kTile - 1));
        if (threadIdx.x < 2 * kTile)
            stat_next = r < end ? (threadIdx.x < kTile ? lse : delta)[(seq * a.heads + head) * a.n_tokens + r] : 0.0f;
        if (kScaled<T> && threadIdx.x < kTile) stat_next -= kWeightPower<T>;
    };
    const auto put = [&](int t) {
        q_next.store(q_tile[t & 1]);
        g_next.store(g_tile[t & 1]);
        if (threadIdx.x < 2 * kTile) stats[t & 1][threadIdx.x / kTile][threadIdx.x % kTile] = stat_next;
    };
    if (tiles > 0) {
        fetch(0);
        put(0);
    }
    if (tiles > 1) fetch(1);
    for (int t = 0; t < tiles; ++t) {
        const int i0 = begin + t % per_head * kTile;
        __syncthreads();
        if (t + 1 < tiles) put(t + 1);
        if (t + 2 < tiles) fetch(t + 2);
        if (w0 >= length) continue;
        const typename Tl::Cell *qt = q_tile[t & 1], *gt = g_tile[t & 1];
        const int at = i0 + 4 * half, lo_r = lo - at, hi_r = min(hi, end - 1) - at;
#pragma unroll kBlocks
        for (int b = 0; b < kTile / 32; ++b) {
            const int r0 = i0 + 32 * b;  // the block's first query
            if (r0 >= end || r0 + 32 <= w0 - a.right || r0 > wave_last) continue;
            const bool whole = all_kept && r0 + 32 <= end && r0 >= w0 + 31 - a.right && (r0 + 31 <= w0 + a.left || w0 + 32 <= a.sinks);
            typename Tl::Pool pool;
            Tl::rows(pool, qt + 32 * b * Tl::LD);
            v16f s = Tl::rows_times(pool, kf);
            Tl::rows(pool, gt + 32 * b * Tl::LD);
            v16f dp = Tl::rows_times(pool, vf);
            Tl::cols(pool, gt + 32 * b * Tl::LD);
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const v4f l4 = *reinterpret_cast<const v4f*>(&stats[t & 1][0][32 * b + 8 * i4 + 4 * half]);
                const v4f d4 = *reinterpret_cast<const v4f*>(&stats[t & 1][1][32 * b + 8 * i4 + 4 * half]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 4 * i4 + e;
                    s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale_log2, -l4[e]));
                    dp[i] = (kScaled<T> ? s[i] * gain : s[i]) * (dp[i] - d4[e]);
                }
            }
            if (!whole) {
                const unsigned alone = static_cast<unsigned>(__ballot(is_alone(stats[t & 1][1][32 * b + (lane_id() & 31)]))) >> (4 * half);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int e = 8 * (i / 4) + i % 4, r = 32 * b + e;
                    const bool seen = r >= lo_r && r <= hi_r;
                    s[i] = seen ? s[i] : 0.0f;
                    dp[i] = seen && !((alone >> e) & 1) ? dp[i] : 0.0f;
                }
            }
            Tl::cols_times(pool, s, dv_acc);
            Tl::cols(pool, qt + 32 * b * Tl::LD);
            if constexpr (kScaled<T>)
                if (fit(dp, power, dk_acc)) gain = __builtin_amdgcn_ldexpf(1.0f, power);
            Tl::cols_times(pool, dp, dk_acc);
        }
    }
    if constexpr (kScaled<T>) {
        unscale(dk_acc, power + kWeightPower<T>);
        unscale(dv_acc, kWeightPower<T>);
        add_far_queries();
    }
    if (in_either_half(kept && !(all_finite(dk_acc) && all_finite(dv_acc)))) {
        const T* kr = static_cast<const T*>(k.p) + seq * k.seq + static_cast<int64_t>(mine) * k.token + kv_head * k.head;
        const T* vr = static_cast<const T*>(v.p) + seq * v.seq + static_cast<int64_t>(mine) * v.token + kv_head * v.head;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) dk_acc[dt] = dv_acc[dt] = v16f{};
        for (int h = kv_head * share; h < (kv_head + 1) * share; ++h)
            for (int i = max(lo, 0); i <= hi; ++i) {
                const T* qr = static_cast<const T*>(q.p) + seq * q.seq + static_cast<int64_t>(i) * q.token + h * q.head;
                const T* gr = static_cast<const T*>(g.p) + seq * g.seq + static_cast<int64_t>(i) * g.token + h * g.head;
                const int64_t at = (seq * a.heads + h) * a.n_tokens + i;
                if (lse[at] == kInf) continue;  // an empty row
                const float p = __builtin_amdgcn_exp2f(fmaf(dot_rows(qr, kr, a.dim), a.scale_log2, -lse[at]));
                if (!is_alone(delta[at])) add_row<T, DP>(dk_acc, p * (dot_rows(gr, vr, a.dim) - delta[at]), qr, a.dim);
                add_row<T, DP>(dv_acc, p, gr, a.dim);
            }
    }
    if (mine < a.n_tokens) {
        const int64_t row = ((seq * a.n_tokens + mine) * a.kv_heads + kv_head) * a.dim;
        store_columns<T, DP>(dk_acc, scale, dk + row, a.dim);
        store_columns<T, DP>(dv_acc, 1.0f, dv + row, a.dim);
    }
}

// How the queries behind the windows of the sinks are cut: chunks of 128, one round of a workgroup's waves, where all of them
// run at once (two workgroups per CU), else of 256 (4 x 4096 x 8 x 64 bfloat16: 11.7 against 16.5 us; 4 x 2000 x 2 x 32 float32:
// 14.4 against 9.6 us with chunks of 128); at most 32 chunks.  A chunk of 32 sinks leaves 8 KB (heads of 32) to 32 KB (of 128):
// together no more than what 2048 of them take or a quarter of the gradients of 16-bit keys and values, whichever is more, but one
// chunk in any case (8192 tokens x 8 x 64 bfloat16, 127 keys, 1000 sinks: backward 211 -> 142 us for it).
// Where many sinks fill the GPU with their blocks alone there are no chunks, and the kernel of the keys walks all queries (8192 x 8
// x 128 bfloat16, all of them sinks: 1227 us with two chunks, 724 with none; few sinks leave three of its four waves without work,
// 128 x 2048 x 8 x 64 with four of them: 1150 and 1593).
struct FarPlan {
    int sink_blocks, chunk, chunks;
};
FarPlan far_plan(int64_t rows, int64_t n_tokens, int64_t left, int64_t sinks) {  // rows: key/value heads of all sequences
    FarPlan f = {0, 1, 0};
    if (left > n_tokens) left = n_tokens;
    if (sinks > n_tokens) sinks = n_tokens;
    const int64_t far = n_tokens - kBlock - left;
    if (sinks <= 0 || far <= 0) return f;
    f.sink_blocks = static_cast<int>((sinks + 31) / 32);
    const int64_t blocks = rows * f.sink_blocks;
    if (f.sink_blocks >= kBlock / 32 && blocks > 1024) return f;
    int64_t most = 2048 / blocks, share = n_tokens / (256 * f.sink_blocks);
    if (most < share) most = share;
    most = most < 1 ? 1 : (most > 32 ? 32 : most);
    int64_t chunk = blocks * ((far + 127) / 128) <= 512 ? 128 : 256;
    if (chunk * most < far) chunk = ((far + most - 1) / most + 127) / 128 * 128;
    f.chunk = static_cast<int>(chunk);
    f.chunks = static_cast<int>((far + chunk - 1) / chunk);
    return f;
}
// Waves of a workgroup of the first and the last kernel, each with 32 queries or keys.  Four share their tiles; where that leaves
// CUs without work, two take their place if the window is short (4 x 2000 x 2 x 32 float32, 127 keys: 128 workgroups of four 41 us,
// twice as many of two 34 us; 257 tokens x 4 heads x 64, 33 keys: 24 -> 18 us) or the heads longer than 64 (2048 x 4 x 128
// bfloat16, all keys: 87 -> 84 us for dk and dv, 70 -> 68 for dq).  Long windows of shorter heads gain from the sharing
// (2048 x 4 x 64 float32, all keys: 147 and 167 us).
int waves_of_block(int64_t rows, const AttentionShape& s) {  // rows: sequences times heads
    const bool idle = rows * ((s.n_tokens + kBlock - 1) / kBlock) < 256;
    return idle && (static_cast<int64_t>(s.left) + s.right < 256 || s.dim > 64) ? 2 : 4;
}
int padded_dim(int dim) { return (dim + 31) / 32 * 32; }

}  // namespace

int attention_shape(const char* name, int dtype, int64_t n_seqs, int64_t n_tokens, int heads, int kv_heads, int dim,
                    int64_t left, int64_t right, int64_t sinks, float scale, const int64_t* lengths, const uint8_t* visible,
                    AttentionShape* s);
int attention_tensor(const char* name, const char* what, const void* p, const int64_t* strides, int dtype, int64_t n_seqs,
                     int64_t n_tokens, int heads, int dim, TokenTensor* t);

}  // namespace mvx

extern "C" size_t mvx_window_attention_backward_workspace_bytes(int64_t n_seqs, int64_t n_tokens, int heads, int kv_heads, int dim,
                                                                int64_t left, int64_t sinks) {
    if (n_seqs <= 0 || n_tokens <= 0 || heads <= 0 || kv_heads <= 0 || dim <= 0 || left < 0) return 0;
    const mvx::FarPlan f = mvx::far_plan(n_seqs * kv_heads, n_tokens, left, sinks);
    const size_t rows = mvx::padded_rows(n_seqs * heads * n_tokens);  // delta
    return (rows + static_cast<size_t>(n_seqs) * kv_heads * f.sink_blocks * f.chunks * mvx::padded_dim(dim) * 64) *
           sizeof(float);
}

extern "C" int mvx_window_attention_backward(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                             const void* v, const int64_t* v_strides, const void* out, const void* saved,
                                             const void* grad_out, const int64_t* grad_strides, int dtype, int64_t n_seqs,
                                             int64_t n_tokens, int heads, int kv_heads, int dim, int64_t left, int64_t right,
                                             int64_t sinks, float scale, const int64_t* lengths, const uint8_t* visible,
                                             void* grad_q, void* grad_k, void* grad_v, void* workspace, size_t workspace_bytes,
                                             void* stream) {
    using namespace mvx;
    const char* name = "mvx_window_attention_backward";
    AttentionShape s;
    int rc = attention_shape(name, dtype, n_seqs, n_tokens, heads, kv_heads, dim, left, right, sinks, scale, lengths, visible, &s);
    if (rc != MVX_OK) return rc;
    if (n_seqs == 0 || n_tokens == 0) return MVX_OK;
    TokenTensor qt, kt, vt, gt;
    if ((rc = attention_tensor(name, "q", q, q_strides, dtype, n_seqs, n_tokens, heads, dim, &qt)) != MVX_OK) return rc;
    if ((rc = attention_tensor(name, "k", k, k_strides, dtype, n_seqs, n_tokens, kv_heads, dim, &kt)) != MVX_OK) return rc;
    if ((rc = attention_tensor(name, "v", v, v_strides, dtype, n_seqs, n_tokens, kv_heads, dim, &vt)) != MVX_OK) return rc;
    if ((rc = attention_tensor(name, "grad_out", grad_out, grad_strides, dtype, n_seqs, n_tokens, heads, dim, &gt)) != MVX_OK) return rc;
    MVX_REQUIRE(out != nullptr && saved != nullptr && grad_q != nullptr && grad_k != nullptr && grad_v != nullptr,
                MVX_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    MVX_REQUIRE(aligned16(out) && aligned16(saved) && aligned16(grad_q) && aligned16(grad_k) && aligned16(grad_v) && aligned16(workspace),
                MVX_ERR_INVALID_ARGUMENT, "%s: out, saved, the gradients and the workspace must be 16-byte aligned", name);
    const size_t need = mvx_window_attention_backward_workspace_bytes(n_seqs, n_tokens, heads, kv_heads, dim, left, sinks);
    MVX_REQUIRE(workspace != nullptr && workspace_bytes >= need, MVX_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu",
                name, need, workspace_bytes);
    const int64_t row = static_cast<int64_t>(heads) * dim;
    const TokenTensor ot = {out, n_tokens * row, row, dim};
    const int q_waves = waves_of_block(n_seqs * heads, s), q_blocks = (s.n_tokens + 32 * q_waves - 1) / (32 * q_waves);
    const int k_waves = waves_of_block(n_seqs * kv_heads, s), k_blocks = (s.n_tokens + 32 * k_waves - 1) / (32 * k_waves);
    const FarPlan f = far_plan(n_seqs * kv_heads, n_tokens, left, sinks);
    MVX_REQUIRE(n_seqs <= (1 << 23) / q_blocks / heads && n_seqs * kv_heads * f.sink_blocks * f.chunks <= (1 << 23),
                MVX_ERR_UNSUPPORTED, "%s: too many sequences, heads and tokens for one launch", name);
    float* delta = static_cast<float*>(workspace);
    float* partial = delta + padded_rows(n_seqs * heads * n_tokens);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return with_element(dtype, name, [&](auto zero) -> int {
        using T = decltype(zero);
        const float *d = delta, *lse = static_cast<const float*>(saved);
        const T* rest = reinterpret_cast<const T*>(lse + padded_rows(n_seqs * heads * n_tokens));
        const auto launch = [&](auto dq_kernel, auto sinks_kernel, int sink_waves, auto join_kernel, auto dkv_kernel) {
            hipLaunchKernelGGL(dq_kernel, dim3(static_cast<unsigned>(n_seqs * heads * q_blocks)), dim3(64 * q_waves), 0, st, qt, kt, vt,
                               ot, rest, gt, s, scale, q_blocks, lse, delta, static_cast<T*>(grad_q));
            const unsigned sinks_of_all = static_cast<unsigned>(n_seqs * kv_heads * f.sink_blocks);
            if (f.chunks > 0)
                hipLaunchKernelGGL(sinks_kernel, dim3(sinks_of_all * f.chunks), dim3(64 * sink_waves), 0, st, qt, kt, vt, gt, s, f.chunk,
                                   f.chunks, lse, d, partial);
            if (f.chunks > 1)
                hipLaunchKernelGGL(join_kernel, dim3(sinks_of_all, padded_dim(dim) * 64 / 4 / 256), dim3(256), 0, st, s, f.chunk, f.chunks,
                                   partial);
            hipLaunchKernelGGL(dkv_kernel, dim3(static_cast<unsigned>(n_seqs * kv_heads * k_blocks)), dim3(64 * k_waves), 0, st, qt, kt,
                               vt, gt, s, scale, k_blocks, f.chunks, lse, d, partial, static_cast<T*>(grad_k), static_cast<T*>(grad_v));
        };
#define MVX_LAUNCH(DP)                                                                                                        \
    launch(q_waves == 2 ? window_attention_dq<T, DP, 2> : window_attention_dq<T, DP, 4>, window_attention_sinks<T, DP>,      \
           kSinkWaves<T, DP>, window_attention_sinks_join<DP>,                                                                \
           k_waves == 2 ? window_attention_dkv<T, DP, 2> : window_attention_dkv<T, DP, 4>)
        if (dim <= 32)
            MVX_LAUNCH(32);
        else if (dim <= 64)
            MVX_LAUNCH(64);
        else if (dim <= 96)
            MVX_LAUNCH(96);
        else
            MVX_LAUNCH(128);
#undef MVX_LAUNCH
        MVX_CHECK_LAUNCH(name);
        return MVX_OK;
    });
}
