// The one-token form of the windowed attention over a ring of cached tokens, and the filling of that ring from a recorded
// sequence.
//
// A stream keeps sinks + window slots of keys and values.  Token t lies in slot t for t < sinks, else in slot
// sinks + (t - sinks) % window, so the slots hold exactly what token t sees with left = window - 1, right = 0: the first
// tokens and the last `window` ones.  The order of the slots does not matter to a softmax, so nothing is ever moved.
//
// One step reads every held key and value once and is bound by that (4 * heads / kv_heads operations per value are far below
// the vector rate).  A workgroup takes one key/value head of one stream and a share of its slots; 4, 8 or 16 lanes hold one
// key (8 values per lane), so a wave reads whole rows, and each such group keeps its own running maximum and sum and merges
// them at the end: within the wave, over the waves through LDS, over the shares by a second launch that also advances the
// lengths (it runs when every reader of the old length is done).
#include "attention_tiles.h"

namespace mvx {

namespace {

constexpr int kThreads = 256, kUnroll = 4;

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

// partial: [stream][head][share][dim + 2]: the weighted sum of the share's values, its maximum and its sum
template <typename T, int LPK, int GQ>
__global__ __launch_bounds__(kThreads) void window_step(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                        T* __restrict__ k_cache, T* __restrict__ v_cache,
                                                        const int64_t* __restrict__ lengths, int heads, int kv_heads, int dim,
                                                        int slots, int sinks, float scale_log2, int per_share,
                                                        float* __restrict__ partial) {
    constexpr int KPW = 64 / LPK;  // keys of a wave's access
    __shared__ float joined[kThreads / 64][GQ][LPK * 8 + 2];
    const int group_heads = heads / kv_heads, parts = (group_heads + GQ - 1) / GQ;
    const int kv_head = blockIdx.y / parts, first = (blockIdx.y % parts) * GQ;
    const int64_t seq = blockIdx.z;
    const int64_t length = lengths[seq];
    if (length < 0) return;
    const int held = static_cast<int>(length + 1 < slots ? length + 1 : slots);
    const int s0 = blockIdx.x * per_share, s1 = min(s0 + per_share, held);
    const int lane = lane_id(), in_key = lane % LPK, wave = threadIdx.x >> 6, d = in_key * 8;
    const bool active = d < dim;
    const int64_t row = static_cast<int64_t>(kv_heads) * dim;
    T* kc = k_cache + seq * slots * row + static_cast<int64_t>(kv_head) * dim;
    T* vc = v_cache + seq * slots * row + static_cast<int64_t>(kv_head) * dim;
    // the new token enters its slot in the workgroup(s) whose share holds it
    const int slot = static_cast<int>(length < sinks ? length : sinks + (length - sinks) % (slots - sinks));
    if (slot >= s0 && slot < s1) {
        for (int e = threadIdx.x; e < dim; e += kThreads) {
            kc[slot * row + e] = k[(seq * kv_heads + kv_head) * dim + e];
            vc[slot * row + e] = v[(seq * kv_heads + kv_head) * dim + e];
        }
        __syncthreads();
    }
    float qv[GQ][8], m[GQ], l[GQ], o[GQ][8];
#pragma unroll
    for (int g = 0; g < GQ; ++g) {
        const bool there = active && first + g < group_heads;
        if (there) load8<T>(q + (seq * heads + kv_head * group_heads + first + g) * dim + d, qv[g]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            qv[g][e] = there ? qv[g][e] * scale_log2 : 0.0f;
            o[g][e] = 0.0f;
        }
        m[g] = -kInf;
        l[g] = 0.0f;
    }
    for (int base = s0 + wave * KPW * kUnroll; base < s1; base += kThreads / 64 * KPW * kUnroll) {
        float kv[kUnroll][8], vv[kUnroll][8];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int s = base + u * KPW + lane / LPK;
            if (s < s1 && active) {
                load8<T>(kc + s * row + d, kv[u]);
                load8<T>(vc + s * row + d, vv[u]);
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
    __syncthreads();
    for (int i = threadIdx.x; i < GQ * (dim + 2); i += kThreads) {
        const int g = i / (dim + 2), e = i % (dim + 2);
        if (first + g >= group_heads) break;
        float top = -kInf;
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, joined[w][g][LPK * 8]);
        const float ref = top == -kInf ? 0.0f : top;
        float r = 0.0f;
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w)
            r += joined[w][g][e < dim ? e : LPK * 8 + 1] * __builtin_amdgcn_exp2f(joined[w][g][LPK * 8] - ref);
        if (e == dim) r = top;
        partial[((seq * heads + kv_head * group_heads + first + g) * gridDim.x + blockIdx.x) * (dim + 2) + e] = r;
    }
}

// Joins the shares of one head of one stream; the first head's workgroup advances the stream's length (only its sign is
// read by the others).
template <typename T>
__global__ __launch_bounds__(128) void window_step_join(const float* __restrict__ partial, int shares, int heads, int dim,
                                                        T* __restrict__ out, int64_t* __restrict__ lengths) {
    const int64_t seq = blockIdx.y;
    const int head = blockIdx.x;
    const int64_t length = lengths[seq];
    T* o = out + (seq * heads + head) * dim;
    const float* p = partial + (seq * heads + head) * shares * (dim + 2);
    float top = -kInf;
    if (length >= 0)
        for (int s = 0; s < shares; ++s) top = fmaxf(top, p[s * (dim + 2) + dim]);
    const float ref = top == -kInf ? 0.0f : top;
    for (int d = threadIdx.x; d < dim; d += 128) {
        float r = 0.0f, total = 0.0f;
        if (length >= 0)
            for (int s = 0; s < shares; ++s) {
                const float f = __builtin_amdgcn_exp2f(p[s * (dim + 2) + dim] - ref);
                r = fmaf(p[s * (dim + 2) + d], f, r);
                total = fmaf(p[s * (dim + 2) + dim + 1], f, total);
            }
        o[d] = static_cast<T>(length >= 0 ? r / total : 0.0f);
    }
    __syncthreads();
    if (head == 0 && threadIdx.x == 0 && length >= 0) lengths[seq] = length + 1;
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

// Shares a stream's slots are cut into: enough workgroups to fill the GPU, at least 64 slots each.
int step_shares(int64_t n_seqs, int heads, int kv_heads, int slots) {
    const int group = heads / kv_heads, gq = group >= 4 ? 4 : (group >= 2 ? 2 : 1);
    const int64_t rows = n_seqs * kv_heads * ((group + gq - 1) / gq);
    int64_t shares = (1024 + rows - 1) / rows;
    const int64_t most = (slots + 63) / 64;
    if (shares > most) shares = most;
    return static_cast<int>(shares < 1 ? 1 : shares);
}

int check_cache(const char* name, int dtype, int64_t n_seqs, int kv_heads, int dim, int64_t window, int64_t sinks) {
    MVX_REQUIRE(dtype == MVX_F32 || dtype == MVX_BF16 || dtype == MVX_F16, MVX_ERR_INVALID_ARGUMENT, "%s: unknown element type %d",
                name, dtype);
    MVX_REQUIRE(n_seqs >= 0 && kv_heads > 0 && window > 0 && sinks >= 0, MVX_ERR_INVALID_ARGUMENT,
                "%s: bad shape n_seqs=%lld kv_heads=%d window=%lld sinks=%lld", name, (long long)n_seqs, kv_heads,
                (long long)window, (long long)sinks);
    MVX_REQUIRE(dim > 0 && dim % 8 == 0, MVX_ERR_INVALID_ARGUMENT, "%s: head dimension %d is not a multiple of 8", name, dim);
    MVX_REQUIRE(dim <= 128, MVX_ERR_UNSUPPORTED, "%s: head dimension %d above 128", name, dim);
    MVX_REQUIRE(n_seqs <= 65535 && kv_heads <= 4096 && window + sinks <= (1 << 30), MVX_ERR_UNSUPPORTED,
                "%s: more than 65535 streams, 4096 heads or 2^30 slots", name);
    return MVX_OK;
}

}  // namespace

int attention_tensor(const char* name, const char* what, const void* p, const int64_t* strides, int dtype, int64_t n_seqs,
                     int64_t n_tokens, int heads, int dim, TokenTensor* t);

}  // namespace mvx

extern "C" size_t mvx_window_attention_step_workspace_bytes(int64_t n_seqs, int heads, int kv_heads, int dim, int64_t window,
                                                            int64_t sinks) {
    if (n_seqs <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || dim <= 0 || window <= 0 || sinks < 0 ||
        window + sinks > (1 << 30))
        return 0;
    return static_cast<size_t>(n_seqs) * heads * mvx::step_shares(n_seqs, heads, kv_heads, static_cast<int>(window + sinks)) *
           (dim + 2) * sizeof(float);
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
    MVX_REQUIRE(aligned16(q) && aligned16(k_cache) && aligned16(v_cache), MVX_ERR_INVALID_ARGUMENT,
                "%s: q and the caches must be 16-byte aligned", name);
    const int slots = static_cast<int>(window + sinks);
    const size_t need = mvx_window_attention_step_workspace_bytes(n_seqs, heads, kv_heads, dim, window, sinks);
    MVX_REQUIRE(workspace != nullptr && workspace_bytes >= need, MVX_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, got %zu",
                name, need, workspace_bytes);
    const int group = heads / kv_heads, gq = group >= 4 ? 4 : (group >= 2 ? 2 : 1);
    const int shares = step_shares(n_seqs, heads, kv_heads, slots), per_share = (slots + shares - 1) / shares;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return with_element(dtype, name, [&](auto zero) -> int {
        using T = decltype(zero);
        const dim3 grid(shares, kv_heads * ((group + gq - 1) / gq), static_cast<unsigned>(n_seqs));
        const auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, static_cast<const T*>(q), static_cast<const T*>(k),
                               static_cast<const T*>(v), static_cast<T*>(k_cache), static_cast<T*>(v_cache), lengths, heads,
                               kv_heads, dim, slots, static_cast<int>(sinks), scale * kLog2e, per_share,
                               static_cast<float*>(workspace));
        };
        const auto by_heads = [&](auto one, auto two, auto four) { gq == 1 ? launch(one) : gq == 2 ? launch(two) : launch(four); };
        if (dim <= 32)
            by_heads(window_step<T, 4, 1>, window_step<T, 4, 2>, window_step<T, 4, 4>);
        else if (dim <= 64)
            by_heads(window_step<T, 8, 1>, window_step<T, 8, 2>, window_step<T, 8, 4>);
        else
            by_heads(window_step<T, 16, 1>, window_step<T, 16, 2>, window_step<T, 16, 4>);
        hipLaunchKernelGGL((window_step_join<T>), dim3(heads, static_cast<unsigned>(n_seqs)), dim3(128), 0, st,
                           static_cast<const float*>(workspace), shares, heads, dim, static_cast<T*>(out), lengths);
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
