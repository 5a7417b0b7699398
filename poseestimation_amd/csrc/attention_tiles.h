// Building blocks of the windowed attention kernels: 32 x 32 products on the matrix units whose results stay in registers
// in the layout the next product needs, and the mask of a sliding window with first tokens that stay visible.
//
// A wave works on 32 columns (c = lane & 31, one query or one key each; half = lane >> 5) against rows of a tile in LDS:
//   rows_times:  S[row][col]  += sum_d tile[row][d] * column[d]     (columns in registers as fragments)
//   cols_times:  A[d][col]    += sum_row tile[row][d] * S[row][col] (S as rows_times left it)
// rows_times leaves register i of a lane at row 8 (i / 4) + 4 half + i % 4.  The second product sums over rows, whose order
// is free as long as both operands agree, so it takes the registers as they lie: its other operand is read from the same
// row-major tile by the transposing LDS read (4 rows x 16 columns per 16 lanes).  Nothing is shuffled between lanes and no tile
// is stored twice.
#pragma once

#include "element.h"

namespace mvx {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_inff();

__device__ __forceinline__ int lane_id() { return __lane_id(); }
// The wave's number in its workgroup, known to be the same in all lanes: what depends on it stays in scalar registers.
__device__ __forceinline__ int same_in_all(int v) { return __builtin_amdgcn_readfirstlane(v); }
template <typename T>
__device__ __forceinline__ T* same_in_all(T* p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const uint64_t lo = static_cast<unsigned>(same_in_all(static_cast<int>(a))), hi = static_cast<unsigned>(same_in_all(static_cast<int>(a >> 32)));
    return reinterpret_cast<T*>(hi << 32 | lo);
}
__device__ __forceinline__ int wave_id() { return same_in_all(threadIdx.x >> 6); }

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

// A fragment pool holds the LDS side of 32 rows' products: filled by rows() for rows_times (16 bytes of a row per lane and
// step) or by cols() for cols_times, and used up by the matrix instructions.  Filling and using are separate so that the reads
// of the next product can be in flight behind the matrix instructions of this one.
template <typename T, int DP>
struct Tiles16 {
    typedef typename Element<T>::vec_t v8;
    typedef T Cell;  // what a tile holds
    static constexpr int VEC = 8;
    static constexpr int STEPS = DP / 16;
    // Tiles of 32, 64 and 128 columns are stored without padding; 16-byte chunk c of row r lies at chunk c ^ twist(r).  The
    // twist takes 16 rows in a row (row reads: the same chunk of 16 rows) to different banks, and 4 rows in a row to different
    // groups of 4 chunks (transposing reads: the same 4 chunks of 4 rows).  96 columns are padded by 8.
    static constexpr bool kTwisted = (DP & (DP - 1)) == 0;
    static constexpr int LD = kTwisted ? DP : DP + 8;
    static __device__ __forceinline__ int twist(int r) {
        if constexpr (DP == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
        if constexpr (DP == 64) return ((r & 2) << 1) | ((r >> 2) & 3);
        if constexpr (DP == 32) return (r >> 2) & 3;
        return 0;
    }
    // index of column `col` (a multiple of 4) of row r
    static __device__ __forceinline__ int at(int r, int col) { return r * LD + (col ^ (twist(r) << 3)); }

    struct Frag {
        v8 step[STEPS];
    };
    struct Pool {
        v8 a[STEPS];
    };
    // the lane's column: `row` points at its dim contiguous values (valid == false: zeros)
    static __device__ __forceinline__ void load_column(Frag& f, const T* row, int dim, bool valid) {
        const int half = lane_id() >> 5;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int d = 16 * s + 8 * half;
            f.step[s] = valid && d < dim ? *reinterpret_cast<const v8*>(row + d) : v8{};
        }
    }
    static __device__ __forceinline__ v16f mfma(v8 a, v8 b, v16f c) {
        if constexpr (__is_same(T, bf16))
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    // `tile` points at a row that is a multiple of 32
    static __device__ __forceinline__ void rows(Pool& p, const T* tile) {
        const int r = lane_id() & 31, half = lane_id() >> 5;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) p.a[s] = *reinterpret_cast<const v8*>(tile + at(r, 16 * s + 8 * half));
    }
    // two transposing reads: 4 values each from 4 rows
    static __device__ __forceinline__ v8 turned(const T* lower, const T* upper) {
        typedef __attribute__((address_space(3))) v4s lds_v4s;
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(lower));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(upper));
        const auto both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(v8, both);
    }
    static __device__ __forceinline__ void cols(Pool& p, const T* tile) {
        const int l = lane_id(), j = l & 15, r = 4 * (l >> 5) + (j >> 2), c = 16 * ((l >> 4) & 1) + 4 * (j & 3);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) {
                // bit 2 of c selects the half of a chunk and is not twisted
                p.a[s * (DP / 32) + dt] = turned(tile + at(16 * s + r, 32 * dt + c), tile + at(16 * s + r + 8, 32 * dt + c));
            }
    }
    static __device__ __forceinline__ v16f rows_times(const Pool& p, const Frag& f) {
        v16f acc = {};
#pragma unroll
        for (int s = 0; s < STEPS; ++s) acc = mfma(p.a[s], f.step[s], acc);
        return acc;
    }
    static __device__ __forceinline__ void cols_times(const Pool& p, const v16f& w, v16f (&acc)[DP / 32]) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            v8 b;
#pragma unroll
            for (int e = 0; e < 8; ++e) b[e] = static_cast<T>(w[8 * s + e]);
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = mfma(p.a[s * (DP / 32) + dt], b, acc[dt]);
        }
    }
    // start + the sum of the weights as cols_times rounds them
    static __device__ __forceinline__ float rounded_sum(const v16f& w, float start) {
        typedef T v2 __attribute__((ext_vector_type(2)));
        const v2 one = {static_cast<T>(1.0f), static_cast<T>(1.0f)};
        float sum[2] = {start, 0.0f};
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const v2 b = {static_cast<T>(w[i]), static_cast<T>(w[i + 1])};
            float& s = sum[i / 2 % 2];
            if constexpr (std::is_same_v<T, bf16>)
                s = __builtin_amdgcn_fdot2_f32_bf16(b, one, s, false);
            else
                s = __builtin_amdgcn_fdot2(b, one, s, false);
        }
        return sum[0] + sum[1];
    }
    // this half's share of the product of a column and the sum of two
    static __device__ __forceinline__ float dot(const Frag& f, const Frag& g, const Frag& rest) {
        float r = 0.0f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                r = fmaf(static_cast<float>(f.step[s][i]), static_cast<float>(g.step[s][i]) + static_cast<float>(rest.step[s][i]), r);
        return r;
    }
};
template <int DP>
struct Tiles<bf16, DP> : Tiles16<bf16, DP> {};
template <int DP>
struct Tiles<f16, DP> : Tiles16<f16, DP> {};

// float32 on the bfloat16 matrix units, which are sixteen times as fast as the float32 ones: a value is the sum of three
// bfloat16 parts, x = a + b + c, each the rounding of what the parts before it leave (8 bits of significand each, together all
// 24), and a product of two values is the sum of the six products of parts that matter,
//
//   x y = a a' + (a b' + b a') + (a c' + b b' + c a'),
//
// added smallest first in the float32 accumulators.  |b| <= 2^-9 |x| and |c| <= 2^-18 |x| (1 + 2^-9), so the three products left
// out are below 2^-26 |x y| together: less than the rounding of one float32 product.  A value that is not finite has parts that
// are NaN; columns that see one are computed again pair by pair.  Tiles hold the three parts of a row one behind the other.
template <int DP>
struct Tiles<float, DP> {
    typedef Tiles16<bf16, DP> Part;
    typedef typename Part::v8 v8;
    typedef bf16 Cell;
    static constexpr int VEC = 4;
    static constexpr int STEPS = Part::STEPS;
    static constexpr int LD = 3 * Part::LD;
    static __device__ __forceinline__ int at(int r, int col) { return r * LD + (col ^ (Part::twist(r) << 3)); }
    struct Frag {
        v8 step[3][STEPS];
    };
    struct Pool {  // three parts are too many registers to fill ahead of their use
        const Cell* tile;
    };
    static __device__ __forceinline__ void split(float x, bf16& a, bf16& b, bf16& c) {
        a = static_cast<bf16>(x);
        const float rest = x - static_cast<float>(a);
        b = static_cast<bf16>(rest);
        c = static_cast<bf16>(rest - static_cast<float>(b));
    }
    static __device__ __forceinline__ void load_column(Frag& f, const float* row, int dim, bool valid) {
        const int half = lane_id() >> 5;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int d = 16 * s + 8 * half;
            const bool there = valid && d < dim;
            const v4f lo = there ? *reinterpret_cast<const v4f*>(row + d) : v4f{}, hi = there ? *reinterpret_cast<const v4f*>(row + d + 4) : v4f{};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                bf16 a, b, c;
                split(e < 4 ? lo[e % 4] : hi[e % 4], a, b, c);
                f.step[0][s][e] = a, f.step[1][s][e] = b, f.step[2][s][e] = c;
            }
        }
    }
    static __device__ __forceinline__ void rows(Pool& p, const Cell* tile) { p.tile = tile; }
    static __device__ __forceinline__ void cols(Pool& p, const Cell* tile) { p.tile = tile; }
    static __device__ __forceinline__ v16f six(const v8 (&x)[3], const v8 (&y)[3], v16f acc) {
        acc = Part::mfma(x[0], y[2], acc);
        acc = Part::mfma(x[2], y[0], acc);
        acc = Part::mfma(x[1], y[1], acc);
        acc = Part::mfma(x[0], y[1], acc);
        acc = Part::mfma(x[1], y[0], acc);
        return Part::mfma(x[0], y[0], acc);
    }
    static __device__ __forceinline__ v16f rows_times(const Pool& p, const Frag& f) {
        const int r = lane_id() & 31, half = lane_id() >> 5;
        v16f acc = {};
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            v8 x[3], y[3];
#pragma unroll
            for (int n = 0; n < 3; ++n) {
                x[n] = *reinterpret_cast<const v8*>(p.tile + n * Part::LD + at(r, 16 * s + 8 * half));
                y[n] = f.step[n][s];
            }
            acc = six(x, y, acc);
        }
        return acc;
    }
    static __device__ __forceinline__ void cols_times(const Pool& p, const v16f& w, v16f (&acc)[DP / 32]) {
        const int l = lane_id(), j = l & 15, r = 4 * (l >> 5) + (j >> 2), col = 16 * ((l >> 4) & 1) + 4 * (j & 3);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            v8 y[3];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                bf16 a, b, c;
                split(w[8 * s + e], a, b, c);
                y[0][e] = a, y[1][e] = b, y[2][e] = c;
            }
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) {
                v8 x[3];
#pragma unroll
                for (int n = 0; n < 3; ++n)
                    x[n] = Part::turned(p.tile + n * Part::LD + at(16 * s + r, 32 * dt + col),
                                        p.tile + n * Part::LD + at(16 * s + r + 8, 32 * dt + col));
                acc[dt] = six(x, y, acc[dt]);
            }
        }
    }
};

// Keys (or queries) of a tile that a workgroup shares.
template <typename T>
constexpr int kTileRows = sizeof(T) == 4 ? 32 : 64;

// This half's share of the product of two float32 rows, in the columns that load_column gives it.
__device__ __forceinline__ float half_dot(const float* a, const float* b, int dim, bool valid) {
    float r = 0.0f;
    if (valid)
        for (int d = 8 * (lane_id() >> 5); d < dim; d += 16)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const v4f x = *reinterpret_cast<const v4f*>(a + d + e), y = *reinterpret_cast<const v4f*>(b + d + e);
#pragma unroll
                for (int i = 0; i < 4; ++i) r = fmaf(x[i], y[i], r);
            }
    return r;
}

// ROWS x DP tile on its way from global memory to LDS, carried by THREADS neighbouring threads (the workgroup, or a wave): held
// in registers while the previous tile is worked on.
template <typename T, int DP, int ROWS, int THREADS>
struct TileInFlight {
    static constexpr int VEC = Tiles<T, DP>::VEC;
    static constexpr int PER_ROW = DP / VEC, ALL = ROWS * PER_ROW, N = (ALL + THREADS - 1) / THREADS;
    typename Element<T>::vec_t v[N];
    // What a thread loads of a tile, in bytes from the tile's first value: the same in every tile.  Columns from `dim` on point
    // behind any tile.
    int offset[N];
    __device__ __forceinline__ void place(int64_t row_stride, int dim) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = threadIdx.x % THREADS + n * THREADS, r = i / PER_ROW, c = i % PER_ROW * VEC;
            offset[n] = c < dim && i < ALL ? static_cast<int>((r * row_stride + c) * sizeof(T)) : 0x7ffffff0;
        }
    }
    // rows row0 .. row0 + ROWS - 1 of `base` (row_stride elements apart, at least dim; ROWS rows span less than 2^31 bytes).  A
    // buffer that ends with row `limit` - 1 takes the bounds check: the loads behind it, and those of columns from `dim` on,
    // give zeros.
    __device__ __forceinline__ void load(const T* base, int64_t row_stride, int row0, int limit) {
        const int rows = max(0, min(limit - row0, ROWS));
        const auto buffer = __builtin_amdgcn_make_buffer_rsrc(same_in_all(const_cast<T*>(base + row0 * row_stride)), 0,
                                                              same_in_all(static_cast<int>(rows * row_stride * sizeof(T))), 0x00020000);
#pragma unroll
        for (int n = 0; n < N; ++n)
            v[n] = __builtin_bit_cast(typename Element<T>::vec_t, __builtin_amdgcn_raw_buffer_load_b128(buffer, offset[n], 0, 0));
    }
    __device__ __forceinline__ void store(typename Tiles<T, DP>::Cell* tile) const {
        using Tl = Tiles<T, DP>;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = threadIdx.x % THREADS + n * THREADS, r = i / PER_ROW, c = i % PER_ROW * VEC;
            if (ALL % THREADS != 0 && i >= ALL) continue;
            if constexpr (sizeof(T) == 4) {
                typedef bf16 v4b __attribute__((ext_vector_type(4)));
                v4b part[3];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    bf16 x, y, z;
                    Tl::split(v[n][e], x, y, z);
                    part[0][e] = x, part[1][e] = y, part[2][e] = z;
                }
#pragma unroll
                for (int m = 0; m < 3; ++m) *reinterpret_cast<v4b*>(tile + m * Tl::Part::LD + Tl::at(r, c)) = part[m];
            } else {
                *reinterpret_cast<typename Element<T>::vec_t*>(tile + Tl::at(r, c)) = v[n];
            }
        }
    }
    // zeros in the rows whose bit is clear in `keep`: what a hidden token holds never enters a product
    __device__ __forceinline__ void hide(uint64_t keep) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int r = (threadIdx.x % THREADS + n * THREADS) / PER_ROW;
            if (!((keep >> r) & 1)) v[n] = typename Element<T>::vec_t{};
        }
    }
};

// Stores the lane's column of a 32 x DP block of sums: times `factor`, the first `dim` values of `row`.  `rest`, where
// given, takes what this rounding to T left of them.
template <typename T, int DP>
__device__ __forceinline__ void store_columns(const v16f (&acc)[DP / 32], float factor, T* row, int dim, T* rest = nullptr) {
    typedef T vec4 __attribute__((ext_vector_type(4)));
    const int half = lane_id() >> 5;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int d = 32 * dt + 8 * b + 4 * half;
            if (d >= dim) continue;
            float x[4];
            vec4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = static_cast<T>(x[e] = acc[dt][4 * b + e] * factor);
            // one rounding for both: made twice, by a conversion and inside a product, near ties fell to either side
            unsigned pair[sizeof(w) / 4];
            __builtin_memcpy(pair, &w, sizeof(w));
#pragma unroll
            for (unsigned& p : pair) asm("" : "+v"(p));
            __builtin_memcpy(&w, pair, sizeof(w));
            *reinterpret_cast<vec4*>(row + d) = w;
            if (rest == nullptr) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float left = x[e] - static_cast<float>(w[e]);
                w[e] = static_cast<T>(__builtin_isfinite(left) ? left : 0.0f);
            }
            *reinterpret_cast<vec4*>(rest + d) = w;
        }
}

// What the attention entry points share.
inline int64_t padded_rows(int64_t rows) { return (rows + 3) / 4 * 4; }  // a float per row, and what follows aligned to 16 bytes
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
    return same_in_all(static_cast<int>(n < 0 ? 0 : (n < s.n_tokens ? n : s.n_tokens)));
}
// Whether token first + lane exists (below `length`) and is visible; its ballot has a bit per token of a tile.
__device__ __forceinline__ bool token_kept(const AttentionShape& s, int64_t seq, int first, int length) {
    const int j = first + lane_id();
    return j < length && (s.visible == nullptr || s.visible[seq * s.n_tokens + j] != 0);
}

// The tiles of `step` keys that the queries [q0, q0 + n) see: first those of the sinks, then the window.
struct KeyTiles {
    int count, sinks, first;
    __device__ __forceinline__ int key0(int t, int step) const { return (t < sinks ? t : first + t - sinks) * step; }
};
__device__ __forceinline__ KeyTiles key_tiles(const AttentionShape& s, int q0, int n, int length, int step) {
    KeyTiles k = {0, 0, 0};
    if (q0 >= length) return k;
    k.first = max(0, q0 - s.left) / step;
    k.sinks = min((min(s.sinks, length) + step - 1) / step, k.first);
    k.count = min(q0 + n - 1 + s.right, length - 1) / step + 1 - k.first + k.sinks;
    return k;
}
// Whether any / each of the queries [w0, w0 + 32) sees any / each of the keys [k0, k0 + n), hidden ones aside.
__device__ __forceinline__ bool sees_any(const AttentionShape& s, int w0, int k0, int n, int length) {
    return (w0 < length) & (k0 <= min(w0 + 31 + s.right, length - 1)) & ((k0 + n > w0 - s.left) | (k0 < s.sinks));
}
__device__ __forceinline__ bool sees_all(const AttentionShape& s, int w0, int k0, int n, int length) {
    return (w0 + 32 <= length) & (k0 + n <= min(w0 + s.right + 1, length)) & ((k0 >= w0 + 31 - s.left) | (k0 + n <= s.sinks));
}

// ---- pairs one by one -------------------------------------------------------------------------------------------------
// A product over a tile multiplies what the window hides from a query with a weight of zero, and zero times an infinity or a
// NaN is a NaN: a value that is not finite would reach queries (or keys) of its tile that do not see it.  A column (a query, a
// key) whose sums end up not finite is therefore computed again, over the pairs it sees alone, with the functions below: if it
// does see such a value it then holds what the formula gives, otherwise the ordinary result, to rounding.  Columns whose sums
// are finite met no such value and stay as they are.
// This walk reads rows lane by lane and is slow: one infinite upstream gradient makes the backward of 4 x 4096 x 8 x 64, 255 keys
// and 4 sinks, take 59 ms instead of 0.11 (each sink's lane walks all queries), one NaN among the values the forward 8 ms.

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
// Whether either of the two lanes that share this lane's column says so (called by whole waves).
__device__ __forceinline__ bool in_either_half(bool v) {
    const uint64_t b = __ballot(v);
    return (static_cast<unsigned>(b | b >> 32) >> (lane_id() & 31)) & 1;
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
