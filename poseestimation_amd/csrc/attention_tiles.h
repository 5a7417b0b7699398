// Building blocks of the windowed attention kernels: 32 x 32 products on the matrix units whose results stay in registers
// in the layout the next product needs, and the mask of a sliding window with first tokens that stay visible.
//
// A wave works on 32 columns (c = lane & 31, one query or one key each; half = lane >> 5) against rows of a tile in LDS:
//   rows_times:  S[row][col]  += sum_d tile[row][d] * column[d]     (columns in registers as fragments)
//   cols_times:  A[d][col]    += sum_row tile[row][d] * S[row][col] (S as rows_times left it)
// rows_times leaves register i of a lane at row 8 (i / 4) + 4 half + i % 4.  The second product sums over rows, whose order
// is free as long as both operands agree, so it takes the registers as they lie: its other operand is read from the same
// row-major tile, for 16-bit types by the transposing LDS read (4 rows x 16 columns per 16 lanes), for float32 one row per
// instruction.  Nothing is shuffled between lanes and no tile is stored twice.
#pragma once

#include "element.h"

namespace mvx {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_inff();

__device__ __forceinline__ int lane_id() { return __lane_id(); }

// max / sum over the two lanes (l, l ^ 32) that share a column: the upper half of one copy and the lower half of the other
// are exchanged, after which the copies hold both halves' values.  (The results are copied to scalars first: a bit cast of a
// vector's element in place reads element 0 whichever is named.)
__device__ __forceinline__ void both_halves(float v, float* lower, float* upper) {
    const unsigned bits = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    const unsigned a = r[0], b = r[1];
    *lower = __builtin_bit_cast(float, a);
    *upper = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float both_halves_max(float v) {
    float a, b;
    both_halves(v, &a, &b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float both_halves_sum(float v) {
    float a, b;
    both_halves(v, &a, &b);
    return a + b;
}

// DP: head dimension rounded up to a multiple of 32 (columns behind the real dimension are zero in fragments and tiles).
template <typename T, int DP>
struct Tiles;

template <typename T, int DP>
struct Tiles16 {
    typedef typename Element<T>::vec_t v8;
    static constexpr int VEC = 8;
    static constexpr int LD = DP + 8;  // row pitch: 16-byte row reads of 8 lanes fall into different banks
    struct Frag {
        v8 step[DP / 16];
    };
    // the lane's column: `row` points at its dim contiguous values (valid == false: zeros)
    static __device__ __forceinline__ void load_column(Frag& f, const T* row, int dim, bool valid) {
        const int half = lane_id() >> 5;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const int d = 16 * s + 8 * half;
            f.step[s] = valid && d < dim ? *reinterpret_cast<const v8*>(row + d) : v8{};
        }
    }
    static __device__ __forceinline__ float dot(const Frag& a, const Frag& b) {  // this half's share
        float r = 0.0f;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) r = fmaf(static_cast<float>(a.step[s][e]), static_cast<float>(b.step[s][e]), r);
        return r;
    }
    static __device__ __forceinline__ v16f mfma(v8 a, v8 b, v16f c) {
        if constexpr (__is_same(T, bf16))
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ v16f rows_times(const T* tile, const Frag& f, v16f acc) {
        const T* p = tile + (lane_id() & 31) * LD + 8 * (lane_id() >> 5);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) acc = mfma(*reinterpret_cast<const v8*>(p + 16 * s), f.step[s], acc);
        return acc;
    }
    static __device__ __forceinline__ void cols_times(const T* tile, const v16f& w, v16f (&acc)[DP / 32]) {
        typedef __attribute__((address_space(3))) v4s lds_v4s;
        const int l = lane_id(), j = l & 15;
        const T* p = tile + (4 * (l >> 5) + (j >> 2)) * LD + 16 * ((l >> 4) & 1) + 4 * (j & 3);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            v8 b;
#pragma unroll
            for (int e = 0; e < 8; ++e) b[e] = static_cast<T>(w[8 * s + e]);
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) {
                const T* q = p + 16 * s * LD + 32 * dt;
                const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(q));
                const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(q + 8 * LD));
                const auto both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                acc[dt] = mfma(__builtin_bit_cast(v8, both), b, acc[dt]);
            }
        }
    }
};
template <int DP>
struct Tiles<bf16, DP> : Tiles16<bf16, DP> {};
template <int DP>
struct Tiles<f16, DP> : Tiles16<f16, DP> {};

template <int DP>
struct Tiles<float, DP> {
    static constexpr int VEC = 4;
    static constexpr int LD = DP + 4;
    struct Frag {
        v4f step[DP / 8];  // d = 8 t + 4 half + e: the order the row reads of 16 bytes give
    };
    static __device__ __forceinline__ void load_column(Frag& f, const float* row, int dim, bool valid) {
        const int half = lane_id() >> 5;
#pragma unroll
        for (int t = 0; t < DP / 8; ++t) {
            const int d = 8 * t + 4 * half;
            f.step[t] = valid && d < dim ? *reinterpret_cast<const v4f*>(row + d) : v4f{};
        }
    }
    static __device__ __forceinline__ float dot(const Frag& a, const Frag& b) {
        float r = 0.0f;
#pragma unroll
        for (int t = 0; t < DP / 8; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) r = fmaf(a.step[t][e], b.step[t][e], r);
        return r;
    }
    static __device__ __forceinline__ v16f rows_times(const float* tile, const Frag& f, v16f acc) {
        const float* p = tile + (lane_id() & 31) * LD + 4 * (lane_id() >> 5);
#pragma unroll
        for (int t = 0; t < DP / 8; ++t) {
            const v4f a = *reinterpret_cast<const v4f*>(p + 8 * t);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], f.step[t][e], acc, 0, 0, 0);
        }
        return acc;
    }
    static __device__ __forceinline__ void cols_times(const float* tile, const v16f& w, v16f (&acc)[DP / 32]) {
        const float* p = tile + 4 * (lane_id() >> 5) * LD + (lane_id() & 31);
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
                acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(p[(8 * (i / 4) + i % 4) * LD + 32 * dt], w[i], acc[dt], 0, 0, 0);
    }
};

// ROWS x DP tile on its way from global memory to LDS, carried by THREADS neighbouring threads (the workgroup, or a wave): held
// in registers while the previous tile is worked on.
template <typename T, int DP, int ROWS, int THREADS>
struct TileInFlight {
    static constexpr int VEC = Tiles<T, DP>::VEC, LD = Tiles<T, DP>::LD;
    static constexpr int PER_ROW = DP / VEC, N = ROWS * PER_ROW / THREADS;
    static_assert(ROWS * PER_ROW % THREADS == 0, "tile must spread evenly");
    typename Element<T>::vec_t v[N];
    // rows row0 .. row0 + ROWS - 1 of `base` (row_stride elements apart); rows from `limit` on and columns from `dim` on are
    // zero
    __device__ __forceinline__ void load(const T* base, int64_t row_stride, int row0, int limit, int dim) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = threadIdx.x % THREADS + n * THREADS, r = row0 + i / PER_ROW, c = i % PER_ROW * VEC;
            v[n] = r < limit && c < dim
                       ? *reinterpret_cast<const typename Element<T>::vec_t*>(base + static_cast<int64_t>(r) * row_stride + c)
                       : typename Element<T>::vec_t{};
        }
    }
    // rows whose bit is clear in `keep` are stored as zeros: what a hidden token holds never enters a product
    __device__ __forceinline__ void store(T* tile, uint64_t keep) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = threadIdx.x % THREADS + n * THREADS, r = i / PER_ROW, c = i % PER_ROW * VEC;
            *reinterpret_cast<typename Element<T>::vec_t*>(tile + r * LD + c) =
                (keep >> r) & 1 ? v[n] : typename Element<T>::vec_t{};
        }
    }
};

// What the attention entry points share.
struct TokenTensor {
    const void* p;
    int64_t seq, token, head;  // strides in elements
};
struct AttentionShape {
    int64_t n_seqs;
    int n_tokens, heads, kv_heads, dim;
    int left, right, sinks;  // key j is seen by query i iff j <= i + right and (j >= i - left or j < sinks)
    float scale_log2;        // scale * log2(e)
    const int64_t* lengths;  // [n_seqs] or NULL
    const uint8_t* visible;  // [n_seqs][n_tokens] or NULL
};

__device__ __forceinline__ int seq_length(const AttentionShape& s, int64_t seq) {
    if (s.lengths == nullptr) return s.n_tokens;
    const int64_t n = s.lengths[seq];
    return static_cast<int>(n < 0 ? 0 : (n < s.n_tokens ? n : s.n_tokens));
}
// Bit r: token first + r exists (below `length`) and is visible.  Every lane of the wave takes part.
__device__ __forceinline__ uint64_t tokens_kept(const AttentionShape& s, int64_t seq, int first, int length) {
    const int j = first + lane_id();
    bool keep = j < length;
    if (s.visible != nullptr && keep) keep = s.visible[seq * s.n_tokens + j] != 0;
    return __ballot(keep);
}

// ---- pairs one by one -------------------------------------------------------------------------------------------------
// A product over a tile multiplies what the window hides from a query with a weight of zero, and zero times an infinity or a
// NaN is a NaN: a value that is not finite would reach queries (or keys) of its tile that do not see it.  Where a wave ends
// with sums that are not finite it therefore computes its columns again, over the seen pairs alone, with the functions below;
// the columns that do see such a value then hold what the formula gives, the others their ordinary result.

// Whether the lane's sums are all finite.
template <int N>
__device__ __forceinline__ bool all_finite(const v16f (&acc)[N]) {
    float t = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) t = fmaf(acc[n][i], 0.0f, t);
    return t == 0.0f;
}
template <typename T>
__device__ __forceinline__ float dot_rows(const T* a, const T* b, int dim) {
    float s = 0.0f;
    for (int d = 0; d < dim; ++d) s = fmaf(static_cast<float>(a[d]), static_cast<float>(b[d]), s);
    return s;
}
// acc += weight * row, in the register layout of cols_times
template <typename T, int DP>
__device__ __forceinline__ void add_row(v16f (&acc)[DP / 32], float weight, const T* row, int dim) {
    const int half = lane_id() >> 5;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int d = 32 * dt + 8 * (i / 4) + 4 * half + i % 4;
            if (d < dim) acc[dt][i] = fmaf(weight, static_cast<float>(row[d]), acc[dt][i]);
        }
}
// calls f(j) for every key that the query with these bounds sees
template <typename F>
__device__ __forceinline__ void for_seen_keys(const AttentionShape& s, int64_t seq, int lo, int hi, F&& f) {
    const int sinks = min(s.sinks, hi + 1), from = max(max(lo, 0), sinks);
    for (int n = 0; n < sinks + max(0, hi + 1 - from); ++n) {
        const int j = n < sinks ? n : from + n - sinks;
        if (s.visible == nullptr || s.visible[seq * s.n_tokens + j] != 0) f(j);
    }
}

}  // namespace mvx
