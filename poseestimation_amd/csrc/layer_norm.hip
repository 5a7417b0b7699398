// Layer norm over the last axis, forward and backward, with the reduction of the weight's and the bias's gradient.
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), h = (x - m) r, y = h w + b
//   g = dL/dy, a = g w:  dx = r (a - mean(a) - h mean(a h)),  dw = sum over rows of g h,  db = sum over rows of g
//
// All arithmetic is float32 (the variance as the mean square of the centred values, so an offset of the row costs nothing);
// results are rounded once.  Both directions are bound by memory down to rows of 512 16-bit or 256 float32 values: a row is read
// once into registers (x; x and g), reduced there and written once.  A row is held by one wave (up to 4 vectors of 16 bytes per lane), by 256 or by 1024 threads; its
// vectors are loaded at element alignment, and the last one is moved back to end with the row (its first elements then
// repeat another lane's and are left out of the sums), so odd widths run at the same rate as even ones.  Narrower rows leave lanes
// without work and are bound by instructions, the same number for every row (2^26 bfloat16 values in rows of 256, 128, 64 and 33:
// forward 66, 123, 237 and 453 us).
// Both directions load the next row while they work on one; the forward keeps the weights of the lane's columns in registers.
// The backward keeps dw and db of the lane's columns there, over all rows its workgroup visits, and writes one row of partial sums
// per workgroup; a second launch adds those up in a fixed order (no atomics: the result is the same in every run).
// 65536 x 1024 bfloat16: forward 44 us (6.1 TB/s; torch's copy of 1 GiB runs at 5.0), backward 86 us (4.7 TB/s); 32768 x 1024
// float32: 42 and 84 us.
#include "element.h"

namespace mvx {

namespace {

constexpr int kMaxRegWidth = 16384;  // widest row that 1024 threads hold in registers

// Sum over the ROW_T threads that share a row (ROW_T = 64: one wave; otherwise the whole workgroup).
template <int ROW_T, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* scratch) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = wave_sum(v[n]);
    if constexpr (ROW_T > 64) {
        constexpr int W = ROW_T / 64;
        __syncthreads();  // the previous use of scratch is over
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) scratch[n * W + threadIdx.x / 64] = v[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += scratch[n * W + w];
            v[n] = s;
        }
    }
}

// Vector v of a row: where it begins, and the first of its elements that no earlier vector holds (vec: none).
__device__ __forceinline__ void place_vec(int v, int vec, int width, int* start, int* fresh) {
    const int at = v * vec;
    *start = at + vec <= width ? at : width - vec;
    *fresh = at >= width ? vec : at - *start;
}

// weight and bias may be float32 beside 16-bit x
template <typename T>
__device__ __forceinline__ void load_param(const void* p, int f32, int at, float (&out)[Element<T>::vec]) {
    if (f32) {
        const float* q = static_cast<const float*>(p) + at;
        if constexpr (Element<T>::vec == 4) {
            load_vec<float>(q, out);
        } else {
            float a[4], b[4];
            load_vec<float>(q, a);
            load_vec<float>(q + 4, b);
#pragma unroll
            for (int e = 0; e < 4; ++e) out[e] = a[e], out[4 + e] = b[e];
        }
    } else {
        load_vec<T>(static_cast<const T*>(p) + at, out);
    }
}
template <typename T>
__device__ __forceinline__ float load_param1(const void* p, int f32, int at) {
    return f32 ? static_cast<const float*>(p)[at] : static_cast<float>(static_cast<const T*>(p)[at]);
}

// The vectors of one row that a thread holds, as they lie in memory.
template <typename T, int NV>
struct RowVecs {
    static constexpr int VEC = Element<T>::vec;
    typedef typename Element<T>::loose_t vec_t;
    vec_t v[NV];
    __device__ __forceinline__ void load(const T* row, const int (&start)[NV], const int (&fresh)[NV]) {
#pragma unroll
        for (int n = 0; n < NV; ++n) v[n] = fresh[n] < VEC ? *reinterpret_cast<const vec_t*>(row + start[n]) : vec_t{};
    }
};

template <typename T, int ROW_T, int BLOCK, int NV>
__global__ __launch_bounds__(BLOCK) void layer_norm_rows(const T* __restrict__ x, const void* __restrict__ weight,
                                                         const void* __restrict__ bias, int param_f32, int64_t rows, int width,
                                                         float eps, T* __restrict__ y, float* __restrict__ stats) {
    constexpr int VEC = Element<T>::vec;
    __shared__ float scratch[ROW_T > 64 ? ROW_T / 64 : 1];
    const int t = threadIdx.x % ROW_T;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * (BLOCK / ROW_T);
    int start[NV], fresh[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) place_vec(t + n * ROW_T, VEC, width, &start[n], &fresh[n]);
    const float inv_width = 1.0f / static_cast<float>(width);
    int64_t row = static_cast<int64_t>(blockIdx.x) * (BLOCK / ROW_T) + threadIdx.x / ROW_T;
    float w[NV][VEC], b[NV][VEC];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) w[n][e] = 1.0f, b[n][e] = 0.0f;
        if (fresh[n] >= VEC) continue;
        if (weight != nullptr) load_param<T>(weight, param_f32, start[n], w[n]);
        if (bias != nullptr) load_param<T>(bias, param_f32, start[n], b[n]);
    }
    RowVecs<T, NV> x_next;
    if (row < rows) x_next.load(x + row * width, start, fresh);
    for (; row < rows; row += stride) {
        RowVecs<T, NV> xv = x_next;
        if (row + stride < rows) x_next.load(x + (row + stride) * width, start, fresh);  // travels while this row is worked on
        float v[NV][VEC];
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[n][e] = static_cast<float>(xv.v[n][e]);
        float sum[1] = {0.0f};
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[0] += e >= fresh[n] ? v[n][e] : 0.0f;
        row_sum<ROW_T>(sum, scratch);
        const float mean = sum[0] * inv_width;
        float sq[1] = {0.0f};
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[n][e] -= mean;
                sq[0] = e >= fresh[n] ? fmaf(v[n][e], v[n][e], sq[0]) : sq[0];
            }
        row_sum<ROW_T>(sq, scratch);
        const float rstd = 1.0f / sqrtf(sq[0] * inv_width + eps);
        if (stats != nullptr && t == 0) {
            stats[2 * row] = mean;
            stats[2 * row + 1] = rstd;
        }
        T* yr = y + row * width;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            if (fresh[n] >= VEC) continue;
            float out[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) out[e] = fmaf(v[n][e] * rstd, w[n][e], b[n][e]);
            store_vec<T>(yr + start[n], out);
        }
    }
}

// Any width (rows shorter than a vector, or longer than the registers of a workgroup): element by element, the row read
// three times, from the caches after the first.
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_any(const T* __restrict__ x, const void* __restrict__ weight,
                                                      const void* __restrict__ bias, int param_f32, int64_t rows, int64_t width,
                                                      float eps, T* __restrict__ y, float* __restrict__ stats) {
    __shared__ float scratch[4];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * width;
        float s[1] = {0.0f};
        for (int64_t i = threadIdx.x; i < width; i += 256) s[0] += static_cast<float>(xr[i]);
        row_sum<256>(s, scratch);
        const float mean = s[0] / static_cast<float>(width);
        float sq[1] = {0.0f};
        for (int64_t i = threadIdx.x; i < width; i += 256) {
            const float c = static_cast<float>(xr[i]) - mean;
            sq[0] = fmaf(c, c, sq[0]);
        }
        row_sum<256>(sq, scratch);
        const float rstd = 1.0f / sqrtf(sq[0] / static_cast<float>(width) + eps);
        if (stats != nullptr && threadIdx.x == 0) {
            stats[2 * row] = mean;
            stats[2 * row + 1] = rstd;
        }
        for (int64_t i = threadIdx.x; i < width; i += 256) {
            const float h = (static_cast<float>(xr[i]) - mean) * rstd;
            y[row * width + i] =
                static_cast<T>(fmaf(h, weight != nullptr ? load_param1<T>(weight, param_f32, i) : 1.0f,
                                    bias != nullptr ? load_param1<T>(bias, param_f32, i) : 0.0f));
        }
    }
}

// One pass of the backward: dx of every row of the workgroup's share, and its partial sums of dw and db.
template <typename T, int ROW_T, int BLOCK, int NV>
__global__ __launch_bounds__(BLOCK) void layer_norm_backward_rows(
    const T* __restrict__ grad, const T* __restrict__ x, const void* __restrict__ weight, int param_f32,
    const float* __restrict__ stats, int64_t rows, int width, T* __restrict__ dx, float* __restrict__ partial) {
    constexpr int VEC = Element<T>::vec, RPB = BLOCK / ROW_T;
    __shared__ float scratch[ROW_T > 64 ? 2 * ROW_T / 64 : 1];
    extern __shared__ __attribute__((aligned(16))) float shared_floats[];  // the weight; then the columns' sums, [2][width]
    const int t = threadIdx.x % ROW_T, sub = threadIdx.x / ROW_T;
    const float inv_width = 1.0f / static_cast<float>(width);
    int start[NV], fresh[NV];
    float dw[NV][VEC], db[NV][VEC];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        place_vec(t + n * ROW_T, VEC, width, &start[n], &fresh[n]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[n][e] = db[n][e] = 0.0f;
    }
    const int64_t stride = static_cast<int64_t>(gridDim.x) * RPB;
    int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + sub;
    RowVecs<T, NV> x_next, g_next;
    float2 stat_next = {};
    const auto fetch = [&](int64_t r) {
        x_next.load(x + r * width, start, fresh);
        g_next.load(grad + r * width, start, fresh);
        stat_next = make_float2(stats[2 * r], stats[2 * r + 1]);
    };
    // The weight waits in LDS, in the order its threads read it: loaded from memory with every row, it would be waited for
    // behind the row that is on its way (loads return in order).
    typedef float v4f __attribute__((ext_vector_type(4)));
    v4f* own_weight = reinterpret_cast<v4f*>(shared_floats) + t;  // [vector][4 values][thread of the row]
    if (weight != nullptr && sub == 0) {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            float w[VEC];
            if (fresh[n] < VEC) load_param<T>(weight, param_f32, start[n], w);
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
                const v4f four = {w[e], w[e + 1], w[e + 2], w[e + 3]};
                own_weight[(n * VEC + e) / 4 * ROW_T] = four;
            }
        }
    }
    if (RPB > 1) __syncthreads();
    const auto load_weight = [&](int n, float (&w)[VEC]) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
            const v4f four = weight != nullptr ? own_weight[(n * VEC + e) / 4 * ROW_T] : v4f{1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
            for (int i = 0; i < 4; ++i) w[e + i] = four[i];
        }
    };
    if (row < rows) fetch(row);
    for (; row < rows; row += stride) {
        RowVecs<T, NV> xv = x_next, gv = g_next;
        const float mean = stat_next.x, rstd = stat_next.y;
        if (row + stride < rows) fetch(row + stride);  // travels while this row is worked on
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            float w[VEC];
            load_weight(n, w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float h = (static_cast<float>(xv.v[n][e]) - mean) * rstd, g = static_cast<float>(gv.v[n][e]);
                dw[n][e] = fmaf(g, h, dw[n][e]);
                db[n][e] += g;
                const float a = e >= fresh[n] ? g * w[e] : 0.0f;
                s[0] += a;
                s[1] = fmaf(a, h, s[1]);
            }
        }
        row_sum<ROW_T>(s, scratch);
        const float a = s[0] * inv_width, b = s[1] * inv_width;
        if (dx != nullptr) {
            T* dr = dx + row * width;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                if (fresh[n] >= VEC) continue;
                float w[VEC], out[VEC];
                load_weight(n, w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float h = (static_cast<float>(xv.v[n][e]) - mean) * rstd;
                    out[e] = rstd * (static_cast<float>(gv.v[n][e]) * w[e] - a - h * b);
                }
                store_vec<T>(dr + start[n], out);
            }
        }
    }
    if (partial == nullptr) return;
    float* mine = partial + static_cast<int64_t>(blockIdx.x) * 2 * width;
    if constexpr (RPB == 1) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (e >= fresh[n]) {
                    mine[start[n] + e] = dw[n][e];
                    mine[width + start[n] + e] = db[n][e];
                }
    } else {  // the waves of the workgroup hold the same columns: added up one after the other
        float* columns = shared_floats;
        __syncthreads();
        for (int w = 0; w < RPB; ++w) {
            if (w == sub) {
#pragma unroll
                for (int n = 0; n < NV; ++n)
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (e >= fresh[n]) {
                            const int c = start[n] + e;
                            columns[c] = w == 0 ? dw[n][e] : columns[c] + dw[n][e];
                            columns[width + c] = w == 0 ? db[n][e] : columns[width + c] + db[n][e];
                        }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < 2 * width; c += BLOCK) mine[c] = columns[c];
    }
}

template <typename T>
__global__ __launch_bounds__(256) void layer_norm_backward_any(const T* __restrict__ grad, const T* __restrict__ x,
                                                               const void* __restrict__ weight, int param_f32,
                                                               const float* __restrict__ stats, int64_t rows, int64_t width,
                                                               T* __restrict__ dx) {
    __shared__ float scratch[8];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * width, *gr = grad + row * width;
        const float mean = stats[2 * row], rstd = stats[2 * row + 1];
        float s[2] = {0.0f, 0.0f};
        for (int64_t i = threadIdx.x; i < width; i += 256) {
            const float a = static_cast<float>(gr[i]) * (weight != nullptr ? load_param1<T>(weight, param_f32, i) : 1.0f);
            s[0] += a;
            s[1] = fmaf(a, (static_cast<float>(xr[i]) - mean) * rstd, s[1]);
        }
        row_sum<256>(s, scratch);
        const float a0 = s[0] / static_cast<float>(width), b0 = s[1] / static_cast<float>(width);
        for (int64_t i = threadIdx.x; i < width; i += 256) {
            const float a = static_cast<float>(gr[i]) * (weight != nullptr ? load_param1<T>(weight, param_f32, i) : 1.0f);
            const float h = (static_cast<float>(xr[i]) - mean) * rstd;
            dx[row * width + i] = static_cast<T>(rstd * (a - a0 - h * b0));
        }
    }
}

// Partial sums of dw and db for any width: one thread per column, a share of the rows per workgroup row.
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_columns_any(const T* __restrict__ grad, const T* __restrict__ x,
                                                              const float* __restrict__ stats, int64_t rows, int64_t width,
                                                              float* __restrict__ partial) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= width) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float g = static_cast<float>(grad[row * width + c]);
        dw = fmaf(g, (static_cast<float>(x[row * width + c]) - stats[2 * row]) * stats[2 * row + 1], dw);
        db += g;
    }
    partial[static_cast<int64_t>(blockIdx.y) * 2 * width + c] = dw;
    partial[(static_cast<int64_t>(blockIdx.y) * 2 + 1) * width + c] = db;
}

// Adds the workgroups' partial sums: 32 columns x 32 shares of the partial rows per workgroup, then the shares, in order.
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_join(const float* __restrict__ partial, int groups, int64_t width,
                                                        int param_f32, void* __restrict__ dweight, void* __restrict__ dbias) {
    __shared__ float share[32][33];
    const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float s = 0.0f;
    if (c < 2 * width)
#pragma unroll 8
        for (int g = part; g < groups; g += 32) s += partial[static_cast<int64_t>(g) * 2 * width + c];
    share[part][lane] = s;
    __syncthreads();
    if (part != 0 || c >= 2 * width) return;
#pragma unroll
    for (int p = 1; p < 32; ++p) s += share[p][lane];
    void* out = c < width ? dweight : dbias;
    const int64_t at = c < width ? c : c - width;
    if (out == nullptr) return;
    if (param_f32)
        static_cast<float*>(out)[at] = s;
    else
        static_cast<T*>(out)[at] = static_cast<T>(s);
}

// How a width is spread over threads: ROW_T, and vectors per thread; {0, 0} for the element-by-element kernels.
struct RowPlan {
    int row_t, nv;
};
RowPlan row_plan(int64_t width, int vec) {
    if (width < vec || width > kMaxRegWidth) return {0, 0};
    const int64_t vecs = (width + vec - 1) / vec;
    for (int row_t : {64, 256, 1024})
        for (int nv : {1, 2, 4}) {
            if (row_t > 64 && nv == 1) continue;             // the smaller row_t's nv = 4 holds as much
            if (row_t == 1024 && nv == 4 && vec == 8) break;  // 32 elements per thread leave no registers for 1024 threads
            if (vecs <= static_cast<int64_t>(row_t) * nv) return {row_t, nv};
        }
    return {0, 0};
}
// Workgroups of the backward: as many as are resident at once or half of that, so that none waits for another to end and the
// partial sums stay small (65536 x 1024 bfloat16: 85 us with 512, 88 with 768, 89 with 1024).
int backward_groups(int64_t rows, int64_t width, int vec) {
    const RowPlan p = row_plan(width, vec);
    int64_t per = 1, most = 0;
    if (p.row_t == 64) per = 4;  // rows of a workgroup
    if (p.row_t == 64) most = p.nv == 1 ? 1024 : 512;
    if (p.row_t == 256) most = p.nv == 2 ? 512 : 256;
    if (p.row_t == 1024) most = 256;
    if (p.row_t == 0) most = 64;
    const int64_t need = (rows + per - 1) / per;
    return static_cast<int>(need < most ? (need > 0 ? need : 1) : most);
}

// Workgroups of the forward: few enough that each takes several rows, with its weights in registers and the next row on its way
// (65536 x 1024 bfloat16: 43 us with 1024 of four rows, 47 with 8192, 49 with one row per wave and nothing in flight; 8192 x 8192
// float16: 47 us with 2048 of one row, 50 with 1024, 54 with one row each).
unsigned forward_groups(int64_t rows, int block, int row_t) {
    const int64_t groups = (rows + block / row_t - 1) / (block / row_t), most = row_t == 64 ? 1024 : 2048;
    return static_cast<unsigned>(groups < most ? groups : most);
}

// Dynamic LDS of the backward: the weight, and where rows share a workgroup the columns' sums in the same place.
size_t norm_lds(int64_t width, int row_t, int nv, int vec, bool sums) {
    const size_t weight = static_cast<size_t>(row_t) * nv * vec, columns = sums ? 2 * static_cast<size_t>(width) : 0;
    return (weight > columns ? weight : columns) * sizeof(float);
}

int check_norm(const char* name, int dtype, int64_t rows, int64_t width) {
    MVX_REQUIRE(dtype == MVX_F32 || dtype == MVX_BF16 || dtype == MVX_F16, MVX_ERR_INVALID_ARGUMENT, "%s: unknown element type %d",
                name, dtype);
    MVX_REQUIRE(rows >= 0 && width > 0, MVX_ERR_INVALID_ARGUMENT, "%s: bad shape rows=%lld width=%lld", name, (long long)rows,
                (long long)width);
    MVX_REQUIRE(width <= 0x7fffffffLL && rows <= 0x7fffffffLL, MVX_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows or columns", name);
    return MVX_OK;
}

}  // namespace

}  // namespace mvx

extern "C" int mvx_layer_norm(const void* x, const void* weight, const void* bias, int dtype, int param_f32, int64_t rows,
                              int64_t width, float eps, void* y, float* stats, void* stream) {
    using namespace mvx;
    const int rc = check_norm("mvx_layer_norm", dtype, rows, width);
    if (rc != MVX_OK) return rc;
    if (rows == 0) return MVX_OK;
    MVX_REQUIRE(x != nullptr && y != nullptr, MVX_ERR_INVALID_ARGUMENT, "mvx_layer_norm: null pointer");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return with_element(dtype, "mvx_layer_norm", [&](auto zero) -> int {
        using T = decltype(zero);
        const T* xt = static_cast<const T*>(x);
        T* yt = static_cast<T*>(y);
        const RowPlan p = row_plan(width, Element<T>::vec);
        const int w = static_cast<int>(width);
#define MVX_NORM(ROW_T, BLOCK, NV)                                                                                             \
    if (p.row_t == ROW_T && p.nv == NV)                                                                                        \
        hipLaunchKernelGGL((layer_norm_rows<T, ROW_T, BLOCK, NV>), dim3(forward_groups(rows, BLOCK, ROW_T)), dim3(BLOCK), 0,     \
                           st, xt, weight, bias, param_f32, rows, w, eps, yt, stats)
        MVX_NORM(64, 256, 1);
        MVX_NORM(64, 256, 2);
        MVX_NORM(64, 256, 4);
        MVX_NORM(256, 256, 2);
        MVX_NORM(256, 256, 4);
        MVX_NORM(1024, 1024, 2);
        if constexpr (Element<T>::vec == 4) MVX_NORM(1024, 1024, 4);
#undef MVX_NORM
        if (p.row_t == 0)
            hipLaunchKernelGGL((layer_norm_any<T>), dim3(rows < 4096 ? rows : 4096), dim3(256), 0, st, xt, weight, bias, param_f32,
                               rows, width, eps, yt, stats);
        MVX_CHECK_LAUNCH("mvx_layer_norm");
        return MVX_OK;
    });
}

extern "C" size_t mvx_layer_norm_backward_workspace_bytes(int dtype, int64_t rows, int64_t width) {
    if (rows <= 0 || width <= 0) return 0;
    return static_cast<size_t>(mvx::backward_groups(rows, width, dtype == MVX_F32 ? 4 : 8)) * 2 * width * sizeof(float);
}

extern "C" int mvx_layer_norm_backward(const void* grad_y, const void* x, const void* weight, const float* stats, int dtype,
                                       int param_f32, int64_t rows, int64_t width, void* grad_x, void* grad_weight,
                                       void* grad_bias, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace mvx;
    const int rc = check_norm("mvx_layer_norm_backward", dtype, rows, width);
    if (rc != MVX_OK) return rc;
    const bool columns = grad_weight != nullptr || grad_bias != nullptr;
    MVX_REQUIRE(rows == 0 || (grad_y != nullptr && x != nullptr && stats != nullptr), MVX_ERR_INVALID_ARGUMENT,
                "mvx_layer_norm_backward: null pointer");
    if (!columns && (grad_x == nullptr || rows == 0)) return MVX_OK;
    const size_t need = mvx_layer_norm_backward_workspace_bytes(dtype, rows, width);
    MVX_REQUIRE(!columns || rows == 0 || (workspace != nullptr && workspace_bytes >= need), MVX_ERR_WORKSPACE,
                "mvx_layer_norm_backward: workspace of %zu bytes needed, got %zu", need, workspace_bytes);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return with_element(dtype, "mvx_layer_norm_backward", [&](auto zero) -> int {
        using T = decltype(zero);
        const T *gt = static_cast<const T*>(grad_y), *xt = static_cast<const T*>(x);
        T* dxt = static_cast<T*>(grad_x);
        float* partial = columns ? static_cast<float*>(workspace) : nullptr;
        const RowPlan p = row_plan(width, Element<T>::vec);
        const int w = static_cast<int>(width);
        const int groups = rows == 0 ? 0 : backward_groups(rows, width, Element<T>::vec);
        if (rows > 0) {
#define MVX_NORM(ROW_T, BLOCK, NV)                                                                                              \
    if (p.row_t == ROW_T && p.nv == NV)                                                                                         \
        hipLaunchKernelGGL((layer_norm_backward_rows<T, ROW_T, BLOCK, NV>), dim3(groups), dim3(BLOCK),                          \
                           norm_lds(width, ROW_T, NV, Element<T>::vec, BLOCK != ROW_T), st, gt, xt, weight, param_f32, stats, rows, w, dxt,  \
                           partial)
            MVX_NORM(64, 256, 1);
            MVX_NORM(64, 256, 2);
            MVX_NORM(64, 256, 4);
            MVX_NORM(256, 256, 2);
            MVX_NORM(256, 256, 4);
            MVX_NORM(1024, 1024, 2);
            if constexpr (Element<T>::vec == 4) MVX_NORM(1024, 1024, 4);
#undef MVX_NORM
            if (p.row_t == 0) {
                if (dxt != nullptr)
                    hipLaunchKernelGGL((layer_norm_backward_any<T>), dim3(rows < 4096 ? rows : 4096), dim3(256), 0, st, gt, xt,
                                       weight, param_f32, stats, rows, width, dxt);
                if (columns)
                    hipLaunchKernelGGL((layer_norm_columns_any<T>), dim3((width + 255) / 256, groups), dim3(256), 0, st, gt, xt,
                                       stats, rows, width, partial);
            }
        }
        if (columns)  // no rows: zeros
            hipLaunchKernelGGL((layer_norm_join<T>), dim3((2 * width + 31) / 32), dim3(1024), 0, st, partial, groups, width,
                               param_f32, grad_weight, grad_bias);
        MVX_CHECK_LAUNCH("mvx_layer_norm_backward");
        return MVX_OK;
    });
}
