// Rotary positions with several axes (time, height, width; x, y, z; ...): the first 2 * pairs values of every head are turned
// pair by pair, pair i by the angle position[axis(i)] * base^-e(i), where axis(i) is the section pair i lies in and e(i) is
// i_in_section / pairs_of_section (each axis has the whole spectrum) or i / pairs (the axes share one spectrum):
//
//   (x1, x2) -> (x1 c - x2 s, x1 s + x2 c),   c = cos(angle), s = sin(angle)
//
// The backward is the rotation by the opposite angle.  Angles are formed in float64 as revolutions and reduced there
// (position 10^6 at frequency 1 would keep four digits in float32); cos and sin of the reduced angle are float32.
//
// Bound by memory: q and k are read once and written once in one launch (8 x 4608 tokens x 20 heads of 128 bfloat16: 68 us,
// 5.5 TB/s; a large copy runs at 5.0).  A workgroup takes a few tokens, computes their cos / sin once into LDS and applies them to
// all heads of q and k, 16 bytes per access.  Vectors are placed at element alignment with the last one of a stretch moved back
// to its end (its first values are then written twice, with the same result), so any number of pairs runs at the vector rate;
// stretches shorter than a vector go element by element.
#include <math.h>

#include "element.h"

namespace mvx {

namespace {

constexpr int kMaxPairs = 128, kMaxAxes = 4;

// Passed by value as a kernel argument: no device table to keep, nothing to upload during a capture.
struct RotaryTable {
    double turns[kMaxPairs];  // revolutions per unit of position
    int end[kMaxAxes];        // first pair after the section of each axis
};
struct RotaryTensor {
    const void* in;
    void* out;
    int64_t batch, token, head;  // strides of `in` in elements; `out` is contiguous
    int heads;
};

enum { POS_I32 = 0, POS_I64 = 1, POS_F32 = 2, POS_F64 = 3 };

__device__ __forceinline__ double position_at(const void* p, int type, int64_t at) {
    switch (type) {
        case POS_I32: return static_cast<double>(static_cast<const int32_t*>(p)[at]);
        case POS_I64: return static_cast<double>(static_cast<const int64_t*>(p)[at]);
        case POS_F32: return static_cast<double>(static_cast<const float*>(p)[at]);
        default: return static_cast<const double*>(p)[at];
    }
}

template <typename T, bool PAIRS>
__global__ __launch_bounds__(256) void rotate_tokens(RotaryTensor q, RotaryTensor k, const void* __restrict__ positions,
                                                     int pos_type, int64_t pos_batch, int n_axes, RotaryTable table, int n_pairs,
                                                     float sign, int64_t n_rows, FastDiv tokens, int dim, int per_block,
                                                     FastDiv units_per_head, FastDiv units_per_token) {
    constexpr int VEC = Element<T>::vec;
    extern __shared__ float2 turned[];  // [per_block][n_pairs] cos, sin
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * per_block;
    const int here = static_cast<int>(n_rows - row0 < per_block ? n_rows - row0 : per_block);
    for (int i = threadIdx.x; i < here * n_pairs; i += 256) {
        const int r = i / n_pairs, pair = i - r * n_pairs;
        int axis = 0;
        while (axis < n_axes - 1 && pair >= table.end[axis]) ++axis;
        const unsigned row = static_cast<unsigned>(row0 + r);
        const unsigned b = fast_div(row, tokens), t = row - b * tokens.divisor;
        const double p = position_at(positions, pos_type, static_cast<int64_t>(b) * pos_batch + static_cast<int64_t>(t) * n_axes + axis);
        const double turns = p * table.turns[pair];
        const float part = static_cast<float>(turns - rint(turns));  // exact reduction; |part| <= 1/2 revolution
        float s, c;
        sincospif(2.0f * part, &s, &c);
        turned[i] = make_float2(c, sign * s);
    }
    __syncthreads();
    const int rotated = 2 * n_pairs;
    // units of a head: vectors of pairs, then vectors of the values behind them, which are copied
    const int pair_span = PAIRS ? rotated : n_pairs;
    const int pair_units = (pair_span + VEC - 1) / VEC;
    const unsigned total = static_cast<unsigned>(here) * units_per_token.divisor;
    for (unsigned u = threadIdx.x; u < total; u += 256) {
        const unsigned r = fast_div(u, units_per_token);
        unsigned rest = u - r * units_per_token.divisor;
        unsigned head = fast_div(rest, units_per_head);
        const int unit = static_cast<int>(rest - head * units_per_head.divisor);
        const unsigned row = static_cast<unsigned>(row0 + r);
        const unsigned b = fast_div(row, tokens), t = row - b * tokens.divisor;
        const bool is_k = head >= static_cast<unsigned>(q.heads);
        if (is_k) head -= q.heads;
        const T* in = static_cast<const T*>(is_k ? k.in : q.in) + static_cast<int64_t>(b) * (is_k ? k.batch : q.batch) +
                      static_cast<int64_t>(t) * (is_k ? k.token : q.token) + static_cast<int64_t>(head) * (is_k ? k.head : q.head);
        T* out = static_cast<T*>(is_k ? k.out : q.out) + (static_cast<int64_t>(row) * (is_k ? k.heads : q.heads) + head) * dim;
        const float2* cs = turned + r * n_pairs;
        if (unit < pair_units) {
            if (pair_span >= VEC) {
                const int at = unit * VEC + VEC <= pair_span ? unit * VEC : pair_span - VEC;
                float a[VEC], y[VEC];
                load_vec<T>(in + at, a);
                if constexpr (PAIRS) {
#pragma unroll
                    for (int e = 0; e < VEC; e += 2) {
                        const float2 f = cs[(at + e) / 2];
                        y[e] = fmaf(a[e], f.x, -a[e + 1] * f.y);
                        y[e + 1] = fmaf(a[e], f.y, a[e + 1] * f.x);
                    }
                    store_vec<T>(out + at, y);
                } else {
                    float b2[VEC], z[VEC];
                    load_vec<T>(in + n_pairs + at, b2);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float2 f = cs[at + e];
                        y[e] = fmaf(a[e], f.x, -b2[e] * f.y);
                        z[e] = fmaf(a[e], f.y, b2[e] * f.x);
                    }
                    store_vec<T>(out + at, y);
                    store_vec<T>(out + n_pairs + at, z);
                }
            } else {
                for (int p = 0; p < n_pairs; ++p) {
                    const int one = PAIRS ? 2 * p : p, two = PAIRS ? 2 * p + 1 : n_pairs + p;
                    const float x1 = static_cast<float>(in[one]), x2 = static_cast<float>(in[two]);
                    out[one] = static_cast<T>(fmaf(x1, cs[p].x, -x2 * cs[p].y));
                    out[two] = static_cast<T>(fmaf(x1, cs[p].y, x2 * cs[p].x));
                }
            }
        } else {
            const int span = dim - rotated, c = unit - pair_units;
            if (span >= VEC) {
                const int at = rotated + (c * VEC + VEC <= span ? c * VEC : span - VEC);
                *reinterpret_cast<typename Element<T>::loose_t*>(out + at) =
                    *reinterpret_cast<const typename Element<T>::loose_t*>(in + at);
            } else {
                for (int i = rotated; i < dim; ++i) out[i] = in[i];
            }
        }
    }
}

}  // namespace

}  // namespace mvx

extern "C" int mvx_rotate_positions(const void* q, const int64_t* q_strides, int q_heads, const void* k,
                                    const int64_t* k_strides, int k_heads, int dtype, int64_t n_seqs, int64_t n_tokens, int dim,
                                    const void* positions, int position_type, int64_t position_seq_stride, int n_axes,
                                    const int32_t* sections, double base, int shared_spectrum, int adjacent_pairs, int inverse,
                                    void* q_out, void* k_out, void* stream) {
    using namespace mvx;
    const char* name = "mvx_rotate_positions";
    MVX_REQUIRE(n_seqs >= 0 && n_tokens >= 0 && dim > 0 && q_heads > 0 && k_heads >= 0, MVX_ERR_INVALID_ARGUMENT,
                "%s: bad shape n_seqs=%lld n_tokens=%lld q_heads=%d k_heads=%d dim=%d", name, (long long)n_seqs,
                (long long)n_tokens, q_heads, k_heads, dim);
    MVX_REQUIRE(n_axes >= 1 && n_axes <= kMaxAxes && sections != nullptr, MVX_ERR_INVALID_ARGUMENT, "%s: 1 to %d axes, got %d",
                name, kMaxAxes, n_axes);
    MVX_REQUIRE(position_type >= POS_I32 && position_type <= POS_F64, MVX_ERR_INVALID_ARGUMENT, "%s: unknown position type %d",
                name, position_type);
    MVX_REQUIRE(base > 0.0 && base <= 1.7976931348623157e308, MVX_ERR_INVALID_ARGUMENT, "%s: base must be positive and finite", name);
    RotaryTable table;
    int64_t pairs = 0;
    for (int a = 0; a < n_axes; ++a) {
        MVX_REQUIRE(sections[a] >= 0 && sections[a] <= kMaxPairs, MVX_ERR_INVALID_ARGUMENT, "%s: bad section %d", name, sections[a]);
        pairs += sections[a];
        table.end[a] = static_cast<int>(pairs);
    }
    MVX_REQUIRE(pairs >= 1 && 2 * pairs <= dim, MVX_ERR_INVALID_ARGUMENT, "%s: the sections hold %lld pairs, a head of %d values has %d",
                name, (long long)pairs, dim, dim / 2);
    MVX_REQUIRE(pairs <= kMaxPairs, MVX_ERR_UNSUPPORTED, "%s: at most %d pairs, got %lld", name, kMaxPairs, (long long)pairs);
    if (n_seqs == 0 || n_tokens == 0) return MVX_OK;
    MVX_REQUIRE(q != nullptr && q_strides != nullptr && q_out != nullptr && positions != nullptr &&
                    (k_heads == 0 || (k != nullptr && k_strides != nullptr && k_out != nullptr)),
                MVX_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
    const int64_t rows = n_seqs * n_tokens;
    MVX_REQUIRE(n_seqs <= 0x7fffffffLL && n_tokens <= 0x7fffffffLL && rows <= 0x7fffffffLL, MVX_ERR_UNSUPPORTED,
                "%s: more than 2^31 - 1 tokens", name);
    // The powers cost more host time than the launch: a thread keeps those of its last sections and base.
    thread_local struct {
        double base = 0.0;
        int n_axes = 0, shared = 0, end[kMaxAxes] = {};
        double turns[kMaxPairs];
    } last;
    bool same = last.base == base && last.n_axes == n_axes && last.shared == (shared_spectrum != 0);
    for (int a = 0; a < n_axes; ++a) same = same && last.end[a] == table.end[a];
    if (!same) {
        for (int a = 0, i = 0; a < n_axes; ++a)
            for (int j = 0; j < sections[a]; ++j, ++i) {
                const double e = shared_spectrum ? static_cast<double>(i) / static_cast<double>(pairs)
                                                 : static_cast<double>(j) / static_cast<double>(sections[a]);
                last.turns[i] = pow(base, -e) / 6.283185307179586476925286766559;
            }
        last.base = base, last.n_axes = n_axes, last.shared = shared_spectrum != 0;
        for (int a = 0; a < n_axes; ++a) last.end[a] = table.end[a];
    }
    for (int i = 0; i < pairs; ++i) table.turns[i] = last.turns[i];
    return with_element(dtype, name, [&](auto zero) -> int {
        using T = decltype(zero);
        constexpr int VEC = Element<T>::vec;
        const int p = static_cast<int>(pairs), span = adjacent_pairs ? 2 * p : p;
        const int units = (span + VEC - 1) / VEC + (dim - 2 * p + VEC - 1) / VEC;
        const int64_t per_token = static_cast<int64_t>(units) * (q_heads + k_heads);
        MVX_REQUIRE(per_token <= (1 << 24), MVX_ERR_UNSUPPORTED, "%s: too many heads", name);
        // Tokens of a workgroup: about 16 KB of values (two vectors per unit of halves, one of neighbours; 8 x 4608 tokens x 20
        // heads of 128 bfloat16: halves 68 us with 512 units, 73 with 1024; neighbours 87 and 71), at most 16 KB of cos and sin.
        // A short call takes one token per workgroup, so that its few tokens run side by side.
        int64_t per_block = (adjacent_pairs ? 1024 : 512) / per_token;
        if (per_block > 2048 / p) per_block = 2048 / p;
        if (per_block < 1 || rows < 1024) per_block = 1;
        const int64_t blocks = (rows + per_block - 1) / per_block;
        MVX_REQUIRE(blocks < (1LL << 24), MVX_ERR_UNSUPPORTED, "%s: too many tokens for one launch", name);
        const RotaryTensor qt = {q, q_out, q_strides[0], q_strides[1], q_strides[2], q_heads};
        RotaryTensor kt = {k, k_out, 0, 0, 0, k_heads};
        if (k_heads > 0) kt.batch = k_strides[0], kt.token = k_strides[1], kt.head = k_strides[2];
        const auto kernel = adjacent_pairs ? rotate_tokens<T, true> : rotate_tokens<T, false>;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), per_block * p * sizeof(float2),
                           static_cast<hipStream_t>(stream), qt, kt, positions, position_type, position_seq_stride, n_axes, table,
                           p, inverse ? -1.0f : 1.0f, rows, fast_divisor(static_cast<unsigned>(n_tokens)), dim,
                           static_cast<int>(per_block), fast_divisor(static_cast<unsigned>(units)),
                           fast_divisor(static_cast<unsigned>(per_token)));
        MVX_CHECK_LAUNCH(name);
        return MVX_OK;
    });
}
