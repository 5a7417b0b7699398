// The one-token form of the windowed attention over a ring of cached tokens, and the filling of that ring from a recorded
// sequence.
//
// A stream keeps sinks + window slots of keys and values.  Token t lies in slot t for t < sinks, else in slot
// sinks + (t - sinks) % window, so the slots hold exactly what token t sees with left = window - 1, right = 0: the first
// tokens and the last `window` ones.  The order of the slots does not matter to a softmax, so nothing is ever moved.
//
// One step is bound by reading the held keys and values: once for up to 32 heads that share them with 16-bit types, for four with
// float32, for two in a short ring (the caches may hold them from then on).  Three kernels share the work:
//   window_step_tiles   16-bit types: a wave takes 32 slots at a time through tiles of its own and multiplies them with all
//                       heads that share them on the matrix units (up to 32 heads cost what one costs)
//   window_step_lanes   float32, and short rings of any type: 4, 8 or 16 lanes hold one key (8 values per lane), so a wave
//                       reads whole rows; every such group keeps its own running maximum and sum and they are merged at the end
//   window_step_join    the slots of a long ring are cut into shares, a workgroup each, which leave their sums in float32; this
//                       adds them and advances the lengths (all readers of the old length are done by then)
// A short ring is one workgroup's work for all heads of its stream: window_step_lanes then finishes the step in one launch.
// 64 streams x 4112 slots x 4 heads of 128 bfloat16, 16 heads reading them: 99 us (5.4 TB/s) and 5 us for the join; 32 x 4112 x 4 x
// 128 float32, 8 heads: 101 us together (5.3 TB/s), 32 heads 160 us; one stream x 68 slots x 8 heads of 64 float32: 6.9 us.  The
// filling copies; 32 x 4112 slots x 4 heads of 128 bfloat16: 97 us (5.5 TB/s).
#include "attention_tiles.h"

namespace mvx {

namespace {

constexpr int kThreads = 256, kUnroll = 4, kStreamWaves = 16, kMaxShares = 1024;

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&out)[8]) {
    if constexpr (sizeof(T) == 4) {
        const v4f a = *reinterpret_cast<const v4f*>(p), b = *reinterpret_cast<const v4f*>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = a[e], out[4 + e] = b[e];
    } else {
        load_vec<T>(p, out);
    }
}

// sum over the LPK lanes of a group (every lane gets it)
template <int LPK>
__device__ __forceinline__ float group_sum(float v) {
    v += dpp_mov<0xB1>(v);
    v += dpp_mov<0x4E>(v);
    if constexpr (LPK >= 8) v += dpp_mov<0x141>(v);
    if constexpr (LPK >= 16) v += dpp_mov<0x140>(v);
    return v;
}

// merges (m2, l2, o2) into (m, l, o): two disjoint sets of keys
template <int N>
__device__ __forceinline__ void merge(float& m, float& l, float (&o)[N], float m2, float l2, const float (&o2)[N]) {
    const float top = fmaxf(m, m2), ref = top == -kInf ? 0.0f : top;
    const float f = __builtin_amdgcn_exp2f(m - ref), f2 = __builtin_amdgcn_exp2f(m2 - ref);
    m = top;
    l = l * f + l2 * f2;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = o[e] * f + o2[e] * f2;
}

struct StepShape {
    int heads, kv_heads, dim, slots, sinks;
    int per_share;  // slots of a share, at blockIdx.x
    float scale_log2;
    __device__ __forceinline__ int held(int64_t length) const { return static_cast<int>(length + 1 < slots ? length + 1 : slots); }
    __device__ __forceinline__ int slot(int64_t length) const {
        return static_cast<int>(length < sinks ? length : sinks + (length - sinks) % (slots - sinks));
    }
};
// The sums of the shares: [stream][head][share][dim] values, then [stream][head][share] (maximum, sum).
struct Shares {
    float* values;
    float2* stats;
};

// Stores `count` values of the new token's heads, from `first` on, in its slot.
template <typename T>
__device__ __forceinline__ void store_token(const T* k, const T* v, T* k_cache, T* v_cache, int64_t seq, int slot, int first, int count,
                                            const StepShape& s) {
    const int64_t row = static_cast<int64_t>(s.kv_heads) * s.dim, from = seq * row + first, to = (seq * s.slots + slot) * row + first;
    for (int e = threadIdx.x; e < count; e += blockDim.x) {
        k_cache[to + e] = k[from + e];
        v_cache[to + e] = v[from + e];
    }
}

// WHOLE: a workgroup takes all heads of a stream and writes the result; otherwise one key/value head (and GQ of the heads that
// share it) and one share of the slots, and leaves its sums.
template <typename T, int LPK, int GQ, bool WHOLE>
__global__ __launch_bounds__(WHOLE ? 64 * kStreamWaves : kThreads) void window_step_lanes(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, T* __restrict__ k_cache, T* __restrict__ v_cache,
    int64_t* __restrict__ lengths, StepShape s, Shares shares, T* __restrict__ out) {
    constexpr int KPW = 64 / LPK, kWaves = WHOLE ? kStreamWaves : kThreads / 64;  // KPW: keys of a wave's access
    __shared__ float joined[kWaves][GQ][LPK * 8 + 2];
    const int group_heads = s.heads / s.kv_heads, parts = (group_heads + GQ - 1) / GQ, all_units = s.kv_heads * parts;
    const int64_t seq = WHOLE ? blockIdx.x : blockIdx.z;
    const int64_t length = lengths[seq];
    if (length < 0) {
        if (WHOLE)
            for (int i = threadIdx.x; i < s.heads * s.dim; i += 64 * kWaves) out[seq * s.heads * s.dim + i] = static_cast<T>(0.0f);
        return;
    }
    const int held = s.held(length), slot = s.slot(length);
    const int s0 = WHOLE ? 0 : blockIdx.x * s.per_share, s1 = WHOLE ? held : min(s0 + s.per_share, held);
    const int lane = lane_id(), in_key = lane % LPK, wave = wave_id(), d = in_key * 8;
    const bool active = d < s.dim;
    const int64_t row = static_cast<int64_t>(s.kv_heads) * s.dim;
    // a unit is GQ heads that share a key/value head; several waves share a unit's slots
    const int units = WHOLE ? all_units : 1, per_unit = kWaves / units;
    const int unit = WHOLE ? wave / per_unit : blockIdx.y, first_slot = wave % per_unit;
    const int kv_head = unit / parts, first = (unit % parts) * GQ;
    if (WHOLE) {
        store_token(k, v, k_cache, v_cache, seq, slot, 0, static_cast<int>(row), s);
        __syncthreads();
    } else if (slot >= s0 && slot < s1) {
        store_token(k, v, k_cache, v_cache, seq, slot, kv_head * s.dim, s.dim, s);
        __syncthreads();
    }
    if (unit < all_units) {
        const T* kc = k_cache + seq * s.slots * row + static_cast<int64_t>(kv_head) * s.dim;
        const T* vc = v_cache + seq * s.slots * row + static_cast<int64_t>(kv_head) * s.dim;
        float qv[GQ][8], m[GQ], l[GQ], o[GQ][8];
#pragma unroll
        for (int g = 0; g < GQ; ++g) {
            const bool there = active && first + g < group_heads;
            if (there) load8<T>(q + (seq * s.heads + kv_head * group_heads + first + g) * s.dim + d, qv[g]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                qv[g][e] = there ? qv[g][e] * s.scale_log2 : 0.0f;
                o[g][e] = 0.0f;
            }
            m[g] = -kInf;
            l[g] = 0.0f;
        }
        for (int base = s0 + first_slot * KPW * kUnroll; base < s1; base += per_unit * KPW * kUnroll) {
            float kv[kUnroll][8], vv[kUnroll][8];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int at = base + u * KPW + lane / LPK;
                if (at < s1 && active) {
                    load8<T>(kc + at * row + d, kv[u]);
                    load8<T>(vc + at * row + d, vv[u]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) kv[u][e] = vv[u][e] = 0.0f;
                }
            }
#pragma unroll
            for (int g = 0; g < GQ; ++g) {
                float sc[kUnroll], most = m[g];
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    float x = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) x = fmaf(qv[g][e], kv[u][e], x);
                    x = group_sum<LPK>(x);
                    sc[u] = base + u * KPW + lane / LPK < s1 ? x : -kInf;
                    most = fmaxf(most, sc[u]);
                }
                const float ref = most == -kInf ? 0.0f : most, f = __builtin_amdgcn_exp2f(m[g] - ref);
                m[g] = most;
                l[g] *= f;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[g][e] *= f;
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    const float p = __builtin_amdgcn_exp2f(sc[u] - ref);
                    l[g] += p;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[g][e] = fmaf(p, vv[u][e], o[g][e]);
                }
            }
        }
#pragma unroll
        for (int g = 0; g < GQ; ++g) {
#pragma unroll
            for (int step = LPK; step < 64; step *= 2) {
                float o2[8];
                const float m2 = __shfl_xor(m[g], step), l2 = __shfl_xor(l[g], step);
#pragma unroll
                for (int e = 0; e < 8; ++e) o2[e] = __shfl_xor(o[g][e], step);
                merge(m[g], l[g], o[g], m2, l2, o2);
            }
            if (lane < LPK) {
#pragma unroll
                for (int e = 0; e < 8; ++e) joined[wave][g][d + e] = o[g][e];
                if (lane == 0) {
                    joined[wave][g][LPK * 8] = m[g];
                    joined[wave][g][LPK * 8 + 1] = l[g];
                }
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < units * GQ * s.dim; i += 64 * kWaves) {
        const int e = i % s.dim, g = i / s.dim % GQ, u = i / s.dim / GQ;
        const int which = WHOLE ? u : unit, in_group = which % parts * GQ + g;
        if (in_group >= group_heads) continue;
        float top = -kInf, value = 0.0f, sum = 0.0f;
        for (int w = u * per_unit; w < (u + 1) * per_unit; ++w) top = fmaxf(top, joined[w][g][LPK * 8]);
        const float ref = top == -kInf ? 0.0f : top;
        for (int w = u * per_unit; w < (u + 1) * per_unit; ++w) {
            const float f = __builtin_amdgcn_exp2f(joined[w][g][LPK * 8] - ref);
            value = fmaf(joined[w][g][e], f, value);
            sum = fmaf(joined[w][g][LPK * 8 + 1], f, sum);
        }
        const int64_t head = seq * s.heads + which / parts * group_heads + in_group;
        if (WHOLE) {
            out[head * s.dim + e] = static_cast<T>(sum == 0.0f ? 0.0f : value / sum);  // 0: scores of minus infinity alone
        } else {
            shares.values[(head * gridDim.x + blockIdx.x) * s.dim + e] = value;
            if (e == 0) shares.stats[head * gridDim.x + blockIdx.x] = make_float2(top, sum);
        }
    }
    if (WHOLE && threadIdx.x == 0) lengths[seq] = length + 1;  // every wave has read it
}

// One key/value head, up to 32 of the heads that share it (the columns), one share of the slots.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads, 2) void window_step_tiles(const T* __restrict__ q, const T* __restrict__ k,
                                                                 const T* __restrict__ v, T* __restrict__ k_cache,
                                                                 T* __restrict__ v_cache, const int64_t* __restrict__ lengths,
                                                                 StepShape s, Shares shares) {
    using Tl = Tiles<T, DP>;
    constexpr int kWaves = kThreads / 64, DT = DP / 32;
    struct WaveTiles {
        __attribute__((aligned(16))) T k[32 * Tl::LD];
        __attribute__((aligned(16))) T v[32 * Tl::LD];
    };
    __shared__ union Shared {
        WaveTiles tiles[kWaves];
        float sums[kWaves][32][DP];  // [wave][head][value]
    } shared;
    __shared__ float2 stats[kWaves][32];  // maximum, sum
    const int group_heads = s.heads / s.kv_heads, parts = (group_heads + 31) / 32;
    const int kv_head = blockIdx.y / parts, first = blockIdx.y % parts * 32, here = min(32, group_heads - first);
    const int64_t seq = blockIdx.z;
    const int64_t length = lengths[seq];
    if (length < 0) return;
    const int s0 = blockIdx.x * s.per_share, s1 = same_in_all(min(s0 + s.per_share, s.held(length))), slot = s.slot(length);
    const int lane = lane_id(), half = lane >> 5, col = lane & 31, wave = wave_id();
    const int64_t row = static_cast<int64_t>(s.kv_heads) * s.dim;
    if (slot >= s0 && slot < s1) {
        store_token(k, v, k_cache, v_cache, seq, slot, kv_head * s.dim, s.dim, s);
        __syncthreads();
    }
    const T* kc = k_cache + seq * s.slots * row + static_cast<int64_t>(kv_head) * s.dim;
    const T* vc = v_cache + seq * s.slots * row + static_cast<int64_t>(kv_head) * s.dim;
    typename Tl::Frag qf;
    Tl::load_column(qf, q + (seq * s.heads + kv_head * group_heads + first + col) * s.dim, s.dim, col < here);
    v16f acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = v16f{};
    float top = -kInf, sum = 0.0f;

    WaveTiles& tile = shared.tiles[wave];
    TileInFlight<T, DP, 32, 64> k_next, v_next;
    k_next.place(row, s.dim);
    v_next.place(row, s.dim);
    const int begin = s0 + 32 * wave;
    if (begin < s1) {
        k_next.load(kc, row, begin, s1);
        v_next.load(vc, row, begin, s1);
    }
    for (int base = begin; base < s1; base += 32 * kWaves) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's reads of the last tile come before these writes
        k_next.store(tile.k);
        v_next.store(tile.v);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (base + 32 * kWaves < s1) {
            k_next.load(kc, row, base + 32 * kWaves, s1);
            v_next.load(vc, row, base + 32 * kWaves, s1);
        }
        typename Tl::Pool pool;
        Tl::rows(pool, tile.k);
        v16f x = Tl::rows_times(pool, qf);
        Tl::cols(pool, tile.v);
        if (base + 32 > s1) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = base + 4 * half + 8 * (i / 4) + i % 4 < s1 ? x[i] : -kInf;
        }
        float most = x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) most = fmaxf(most, x[i]);
        most = both_halves_max(most) * s.scale_log2;
        if (__any(most > top)) {
            const float next = fmaxf(top, most), f = __builtin_amdgcn_exp2f(top - (next == -kInf ? 0.0f : next));
            sum *= f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
            top = next;
        }
        const float ref = top == -kInf ? 0.0f : top;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], s.scale_log2, -ref));
        Tl::cols_times(pool, x, acc);
        sum = Tl::rounded_sum(x, sum);  // of the weights as the product takes them: the result stays a mean of the values
    }
    sum = both_halves_sum(sum);
    __syncthreads();  // the tiles are read: their memory takes the sums
    if (col < here) {
        if (half == 0) stats[wave][col] = make_float2(top, sum);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const v4f w = {acc[dt][4 * b], acc[dt][4 * b + 1], acc[dt][4 * b + 2], acc[dt][4 * b + 3]};
                *reinterpret_cast<v4f*>(&shared.sums[wave][col][32 * dt + 8 * b + 4 * half]) = w;
            }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < here * s.dim; i += kThreads) {
        const int e = i % s.dim, g = i / s.dim;
        float most = -kInf, value = 0.0f, total = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) most = fmaxf(most, stats[w][g].x);
        const float ref = most == -kInf ? 0.0f : most;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(stats[w][g].x - ref);
            value = fmaf(shared.sums[w][g][e], f, value);
            total = fmaf(stats[w][g].y, f, total);
        }
        const int64_t head = seq * s.heads + kv_head * group_heads + first + g;
        shares.values[(head * gridDim.x + blockIdx.x) * s.dim + e] = value;
        if (e == 0) shares.stats[head * gridDim.x + blockIdx.x] = make_float2(most, total);
    }
}

// Joins the shares of one head of one stream; the first head's workgroup advances the stream's length (only its sign is
// read by the others).
template <typename T>
__global__ __launch_bounds__(256) void window_step_join(Shares shares, int n_shares, int heads, int dim, T* __restrict__ out,
                                                        int64_t* __restrict__ lengths) {
    __shared__ v4f sums[256];
    __shared__ float factor[kMaxShares], of_wave[2][4];
    const int64_t head = static_cast<int64_t>(blockIdx.y) * heads + blockIdx.x;
    const int64_t length = lengths[blockIdx.y];
    const int vecs = dim / 4, rows = 256 / vecs, vec = threadIdx.x % vecs, r = threadIdx.x / vecs;
    const float2* stats = shares.stats + head * n_shares;
    const v4f* values = reinterpret_cast<const v4f*>(shares.values + head * n_shares * dim);
    float total = 0.0f;
    v4f value = {};
    if (length >= 0) {  // the same in all threads
        float2 mine[kMaxShares / 256];
        float top = -kInf;
#pragma unroll
        for (int n = 0; n < kMaxShares / 256; ++n) {
            const int i = threadIdx.x + 256 * n;
            mine[n] = i < n_shares ? stats[i] : make_float2(-kInf, 0.0f);
            top = fmaxf(top, mine[n].x);
        }
        of_wave[0][wave_id()] = wave_max(top);
        __syncthreads();
        top = fmaxf(fmaxf(of_wave[0][0], of_wave[0][1]), fmaxf(of_wave[0][2], of_wave[0][3]));
        const float ref = top == -kInf ? 0.0f : top;
#pragma unroll
        for (int n = 0; n < kMaxShares / 256; ++n) {
            const int i = threadIdx.x + 256 * n;
            const float f = __builtin_amdgcn_exp2f(mine[n].x - ref);
            if (i < n_shares) factor[i] = f;
            total = fmaf(mine[n].y, f, total);
        }
        of_wave[1][wave_id()] = wave_sum(total);
        __syncthreads();
        total = (of_wave[1][0] + of_wave[1][1]) + (of_wave[1][2] + of_wave[1][3]);
        if (r < rows)
#pragma unroll 4
            for (int i = r; i < n_shares; i += rows) value += values[i * vecs + vec] * factor[i];
    }
    sums[threadIdx.x] = value;
    __syncthreads();
    if (r == 0) {
        for (int i = 1; i < rows; ++i) value += sums[i * vecs + vec];
        const bool none = length < 0 || total == 0.0f;  // an idle stream, or scores of minus infinity alone
        const float inv = none ? 0.0f : 1.0f / total;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[head * dim + vec * 4 + e] = static_cast<T>(none ? 0.0f : value[e] * inv);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0 && length >= 0) lengths[blockIdx.y] = length + 1;
}

// One thread per 16 bytes of a slot, key and value: looks up the token that belongs there, if the sequence holds one.
template <typename T>
__global__ __launch_bounds__(256) void window_fill(TokenTensor k, TokenTensor v, const int64_t* __restrict__ lengths,
                                                   int64_t n_tokens, int kv_heads, int dim, int slots, int sinks,
                                                   T* __restrict__ k_cache, T* __restrict__ v_cache) {
    constexpr int VEC = Element<T>::vec;
    typedef typename Element<T>::vec_t vec_t;
    const int per_head = dim / VEC, per_slot = kv_heads * per_head;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= static_cast<int64_t>(slots) * per_slot) return;
    const int64_t seq = blockIdx.y;
    const int slot = static_cast<int>(i / per_slot), rest = static_cast<int>(i % per_slot);
    const int head = rest / per_head, d = rest % per_head * VEC;
    int64_t length = lengths[seq];
    if (length > n_tokens) length = n_tokens;
    int64_t token = slot;
    if (slot >= sinks) {  // the last token t >= sinks below length with (t - sinks) % window == slot - sinks
        const int64_t window = slots - sinks, last = length - 1 - sinks, r = slot - sinks;
        if (last < r) return;
        token = sinks + last - (last - r) % window;
    } else if (slot >= length) {
        return;
    }
    const int64_t to = ((seq * slots + slot) * kv_heads + head) * dim + d;
    *reinterpret_cast<vec_t*>(k_cache + to) =
        *reinterpret_cast<const vec_t*>(static_cast<const T*>(k.p) + seq * k.seq + token * k.token + head * k.head + d);
    *reinterpret_cast<vec_t*>(v_cache + to) =
        *reinterpret_cast<const vec_t*>(static_cast<const T*>(v.p) + seq * v.seq + token * v.token + head * v.head + d);
}

// How a step is spread over workgroups: shares of a stream's slots, 0 where one workgroup takes the whole stream.
//   Whole streams: up to 1024 slots of (pairs of) heads, where one launch instead of two counts (68 slots x 8 heads: 6.9 against
//   7.2 us on the GPU, and a launch less on the host; at 260 slots 12.0 against 7.3), and up to 2048 where many streams hide each
//   other's latency (256 streams x 132 slots x 8 heads: 15.9 against 24.9 us).
//   Shares: as many workgroups as are resident at once, two per CU (64 streams x 4112 slots x 4 heads of 128: 110 us with 512,
//   117 with 1024, 134 with 2048); float32, whose workgroups are smaller, twice that.
int step_shares(int64_t n_seqs, int heads, int kv_heads, int slots, int dtype) {
    const int group = heads / kv_heads, pairs = kv_heads * ((group + 1) / 2);
    if (pairs <= kStreamWaves && static_cast<int64_t>(slots) * pairs <= (n_seqs >= 128 ? 2048 : 1024)) return 0;
    const int64_t rows = n_seqs * kv_heads * (dtype == MVX_F32 ? (group + 3) / 4 : (group + 31) / 32);
    const int64_t want = dtype == MVX_F32 ? 1024 : 512, least = dtype == MVX_F32 ? 64 : 128;  // workgroups; slots of a share
    int64_t shares = (want + rows - 1) / rows;
    const int64_t most = (slots + least - 1) / least;
    if (shares > most) shares = most;
    return static_cast<int>(shares < 1 ? 1 : shares);  // at most `want`, which is at most kMaxShares
}

int check_cache(const char* name, int dtype, int64_t n_seqs, int kv_heads, int dim, int64_t window, int64_t sinks) {
    MVX_REQUIRE(dtype == MVX_F32 || dtype == MVX_BF16 || dtype == MVX_F16, MVX_ERR_INVALID_ARGUMENT, "%s: unknown element type %d",
                name, dtype);
    MVX_REQUIRE(n_seqs >= 0 && kv_heads > 0 && window > 0 && sinks >= 0, MVX_ERR_INVALID_ARGUMENT,
                "%s: bad shape n_seqs=%lld kv_heads=%d window=%lld sinks=%lld", name, (long long)n_seqs, kv_heads,
                (long long)window, (long long)sinks);
    MVX_REQUIRE(dim > 0 && dim % 8 == 0, MVX_ERR_INVALID_ARGUMENT, "%s: head dimension %d is not a multiple of 8", name, dim);
    MVX_REQUIRE(dim <= 128, MVX_ERR_UNSUPPORTED, "%s: head dimension %d above 128", name, dim);
    MVX_REQUIRE(n_seqs <= 65535 && kv_heads <= 4096 && window <= (1 << 30) && sinks <= (1 << 30) - window, MVX_ERR_UNSUPPORTED,
                "%s: more than 65535 streams, 4096 heads or 2^30 slots", name);
    return MVX_OK;
}

}  // namespace

int attention_tensor(const char* name, const char* what, const void* p, const int64_t* strides, int dtype, int64_t n_seqs,
                     int64_t n_tokens, int heads, int dim, TokenTensor* t);

}  // namespace mvx

extern "C" size_t mvx_window_attention_step_workspace_bytes(int dtype, int64_t n_seqs, int heads, int kv_heads, int dim,
                                                            int64_t window, int64_t sinks) {
    if (n_seqs <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || dim <= 0 || window <= 0 || sinks < 0 ||
        window > (1 << 30) || sinks > (1 << 30) - window)
        return 0;
    return static_cast<size_t>(n_seqs) * heads *
           mvx::step_shares(n_seqs, heads, kv_heads, static_cast<int>(window + sinks), dtype) * (dim + 2) * sizeof(float);
}

extern "C" int mvx_window_attention_step(const void* q, const void* k, const void* v, int dtype, int64_t n_seqs, int heads,
                                         int kv_heads, int dim, int64_t window, int64_t sinks, float scale, void* k_cache,
                                         void* v_cache, int64_t* lengths, void* out, void* workspace, size_t workspace_bytes,
                                         void* stream) {
    using namespace mvx;
    const char* name = "mvx_window_attention_step";
    const int rc = check_cache(name, dtype, n_seqs, kv_heads, dim, window, sinks);
    if (rc != MVX_OK) return rc;
    MVX_REQUIRE(heads > 0 && heads % kv_heads == 0 && heads <= 65535, MVX_ERR_INVALID_ARGUMENT, "%s: bad head counts %d, %d", name,
                heads, kv_heads);
    MVX_REQUIRE(scale > 0.0f && scale < kInf, MVX_ERR_INVALID_ARGUMENT, "%s: scale must be positive and finite", name);
    if (n_seqs == 0) return MVX_OK;
    MVX_REQUIRE(q != nullptr && k != nullptr && v != nullptr && k_cache != nullptr && v_cache != nullptr && lengths != nullptr &&
                    out != nullptr,
                MVX_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    MVX_REQUIRE(aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(workspace), MVX_ERR_INVALID_ARGUMENT,
                "%s: q, the caches and the workspace must be 16-byte aligned", name);
    const int slots = static_cast<int>(window + sinks);
    const size_t need = mvx_window_attention_step_workspace_bytes(dtype, n_seqs, heads, kv_heads, dim, window, sinks);
    MVX_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), MVX_ERR_WORKSPACE,
                "%s: workspace of %zu bytes needed, got %zu", name, need, workspace_bytes);
    const int group = heads / kv_heads, gq = group >= 4 ? 4 : (group >= 2 ? 2 : 1);
    const int shares = step_shares(n_seqs, heads, kv_heads, slots, dtype);
    const StepShape s = {heads, kv_heads, dim, slots, static_cast<int>(sinks), shares > 0 ? (slots + shares - 1) / shares : slots,
                         scale * kLog2e};
    float* values = static_cast<float*>(workspace);
    const Shares sums = {values, reinterpret_cast<float2*>(values + static_cast<size_t>(n_seqs) * heads * shares * dim)};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return with_element(dtype, name, [&](auto zero) -> int {
        using T = decltype(zero);
        const T *qt = static_cast<const T*>(q), *kt = static_cast<const T*>(k), *vt = static_cast<const T*>(v);
        T *kc = static_cast<T*>(k_cache), *vc = static_cast<T*>(v_cache), *o = static_cast<T*>(out);
        const unsigned streams = static_cast<unsigned>(n_seqs);
        const auto lanes = [&](auto one, auto two, auto four, dim3 grid, int threads) {
            hipLaunchKernelGGL(gq == 1 ? one : gq == 2 ? two : four, grid, dim3(threads), 0, st, qt, kt, vt, kc, vc, lengths, s, sums, o);
        };
        if (shares == 0) {
            // heads that share keys go in pairs: four of them spill the registers of a workgroup of 16 waves
            const dim3 grid(streams);
            constexpr int kAll = 64 * kStreamWaves;
            if (dim <= 32)
                lanes(window_step_lanes<T, 4, 1, true>, window_step_lanes<T, 4, 2, true>, window_step_lanes<T, 4, 2, true>, grid, kAll);
            else if (dim <= 64)
                lanes(window_step_lanes<T, 8, 1, true>, window_step_lanes<T, 8, 2, true>, window_step_lanes<T, 8, 2, true>, grid, kAll);
            else
                lanes(window_step_lanes<T, 16, 1, true>, window_step_lanes<T, 16, 2, true>, window_step_lanes<T, 16, 2, true>, grid, kAll);
            MVX_CHECK_LAUNCH(name);
            return MVX_OK;
        }
        if constexpr (sizeof(T) == 4) {
            const dim3 grid(shares, kv_heads * ((group + gq - 1) / gq), streams);
            if (dim <= 32)
                lanes(window_step_lanes<T, 4, 1, false>, window_step_lanes<T, 4, 2, false>, window_step_lanes<T, 4, 4, false>, grid,
                      kThreads);
            else if (dim <= 64)
                lanes(window_step_lanes<T, 8, 1, false>, window_step_lanes<T, 8, 2, false>, window_step_lanes<T, 8, 4, false>, grid,
                      kThreads);
            else
                lanes(window_step_lanes<T, 16, 1, false>, window_step_lanes<T, 16, 2, false>, window_step_lanes<T, 16, 4, false>, grid,
                      kThreads);
        } else {
            const dim3 grid(shares, kv_heads * ((group + 31) / 32), streams);
            const auto tiles = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, qt, kt, vt, kc, vc, lengths, s, sums);
            };
            if (dim <= 32)
                tiles(window_step_tiles<T, 32>);
            else if (dim <= 64)
                tiles(window_step_tiles<T, 64>);
            else if (dim <= 96)
                tiles(window_step_tiles<T, 96>);
            else
                tiles(window_step_tiles<T, 128>);
        }
        hipLaunchKernelGGL((window_step_join<T>), dim3(heads, streams), dim3(256), 0, st, sums, shares, heads, dim, o, lengths);
        MVX_CHECK_LAUNCH(name);
        return MVX_OK;
    });
}

extern "C" int mvx_window_cache_fill(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, int dtype,
                                     const int64_t* lengths, int64_t n_seqs, int64_t n_tokens, int kv_heads, int dim,
                                     int64_t window, int64_t sinks, void* k_cache, void* v_cache, void* stream) {
    using namespace mvx;
    const char* name = "mvx_window_cache_fill";
    int rc = check_cache(name, dtype, n_seqs, kv_heads, dim, window, sinks);
    if (rc != MVX_OK) return rc;
    MVX_REQUIRE(n_tokens >= 0, MVX_ERR_INVALID_ARGUMENT, "%s: bad n_tokens=%lld", name, (long long)n_tokens);
    if (n_seqs == 0 || n_tokens == 0) return MVX_OK;
    TokenTensor kt, vt;
    if ((rc = attention_tensor(name, "k", k, k_strides, dtype, n_seqs, n_tokens, kv_heads, dim, &kt)) != MVX_OK) return rc;
    if ((rc = attention_tensor(name, "v", v, v_strides, dtype, n_seqs, n_tokens, kv_heads, dim, &vt)) != MVX_OK) return rc;
    MVX_REQUIRE(lengths != nullptr && k_cache != nullptr && v_cache != nullptr && aligned16(k_cache) && aligned16(v_cache),
                MVX_ERR_INVALID_ARGUMENT, "%s: lengths or a cache is null, or a cache is not 16-byte aligned", name);
    const int slots = static_cast<int>(window + sinks);
    const int64_t vecs = static_cast<int64_t>(slots) * kv_heads * (dim * element_bytes(dtype) / 16);
    MVX_REQUIRE(vecs < (1LL << 32) - 256, MVX_ERR_UNSUPPORTED, "%s: a stream's cache is too large for one launch", name);
    return with_element(dtype, name, [&](auto zero) -> int {
        using T = decltype(zero);
        hipLaunchKernelGGL((window_fill<T>), dim3(static_cast<unsigned>((vecs + 255) / 256), static_cast<unsigned>(n_seqs)),
                           dim3(256), 0, static_cast<hipStream_t>(stream), kt, vt, lengths, n_tokens, kv_heads, dim, slots,
                           static_cast<int>(sinks), static_cast<T*>(k_cache), static_cast<T*>(v_cache));
        MVX_CHECK_LAUNCH(name);
        return MVX_OK;
    });
}
