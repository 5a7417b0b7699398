// Element types of the sequence operators (float32, bfloat16, float16): 16-byte vectors and their conversions.
// Arithmetic is float32 throughout; values are rounded to the element type once, when they are stored (to nearest, ties to
// even).
#pragma once

#include "mvx_common.h"

namespace mvx {

using bf16 = __bf16;
using f16 = _Float16;

template <typename T>
struct Element;
template <>
struct Element<float> {
    static constexpr int vec = 4;  // elements of 16 bytes
    typedef float vec_t __attribute__((ext_vector_type(4)));
    typedef float loose_t __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct Element<bf16> {
    static constexpr int vec = 8;
    typedef bf16 vec_t __attribute__((ext_vector_type(8)));
    typedef bf16 loose_t __attribute__((ext_vector_type(8), aligned(2)));
};
template <>
struct Element<f16> {
    static constexpr int vec = 8;
    typedef f16 vec_t __attribute__((ext_vector_type(8)));
    typedef f16 loose_t __attribute__((ext_vector_type(8), aligned(2)));
};

// 16 bytes of elements from any element-aligned address (global memory takes unaligned vector accesses; a vector that
// crosses a 128-byte line costs a second line, nothing else), and back.
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[Element<T>::vec]) {
    const typename Element<T>::loose_t v = *reinterpret_cast<const typename Element<T>::loose_t*>(p);
#pragma unroll
    for (int e = 0; e < Element<T>::vec; ++e) out[e] = static_cast<float>(v[e]);
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[Element<T>::vec]) {
    typename Element<T>::loose_t v;
#pragma unroll
    for (int e = 0; e < Element<T>::vec; ++e) v[e] = static_cast<T>(in[e]);
    *reinterpret_cast<typename Element<T>::loose_t*>(p) = v;
}

__device__ __forceinline__ float wave_sum(float v) {
    v += dpp_mov<0xB1>(v);
    v += dpp_mov<0x4E>(v);
    v += dpp_mov<0x141>(v);
    v += dpp_mov<0x140>(v);
    return (read_lane(v, 0) + read_lane(v, 16)) + (read_lane(v, 32) + read_lane(v, 48));
}

// One switch over the element types of the C ABI: `call` is invoked with a value of the type.
template <typename F>
inline int with_element(int dtype, const char* name, F&& call) {
    switch (dtype) {
        case MVX_F32: return call(float{});
        case MVX_BF16: return call(bf16{});
        case MVX_F16: return call(f16{});
    }
    set_error("%s: unknown element type %d", name, dtype);
    return MVX_ERR_INVALID_ARGUMENT;
}
inline int64_t element_bytes(int dtype) { return dtype == MVX_F32 ? 4 : 2; }

}  // namespace mvx
