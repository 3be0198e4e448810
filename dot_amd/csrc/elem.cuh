// Elements of 16 or 32 bits as floats: loads, stores and the dispatch on a
// type tag of the C ABI.  bf16 is the upper half of a float, so reading it is
// a shift; writing rounds to nearest even (the hardware conversion of gfx950).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/dot_amd.h"

namespace dot_amd {

struct F16 {
    uint16_t bits;
};
struct BF16 {
    uint16_t bits;
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(F16 x) { return float(__builtin_bit_cast(_Float16, x.bits)); }
__device__ __forceinline__ float to_float(BF16 x) { return __builtin_bit_cast(float, uint32_t(x.bits) << 16); }

template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ F16 from_float<F16>(float x) {
    return F16{__builtin_bit_cast(uint16_t, _Float16(x))};
}
template <>
__device__ __forceinline__ BF16 from_float<BF16>(float x) {
    return BF16{__builtin_bit_cast(uint16_t, __bf16(x))};
}

// 16 bytes of elements.
template <class T>
struct Pack {
    static constexpr int N = 16 / int(sizeof(T));
    T v[N];
};

// 16-byte load of a pack; the address is 16-byte aligned.
template <class T>
__device__ __forceinline__ Pack<T> load_pack(const T* p) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(Pack<T>, *reinterpret_cast<const u4*>(p));
}
// As load_pack, for inputs that nothing reads again soon.
template <class T>
__device__ __forceinline__ Pack<T> load_pack_stream(const T* p) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(Pack<T>, __builtin_nontemporal_load(reinterpret_cast<const u4*>(p)));
}
// 16-byte store of a pack that nothing reads back soon.
template <class T>
__device__ __forceinline__ void store_pack_stream(T* p, const Pack<T>& x) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(__builtin_bit_cast(u4, x), reinterpret_cast<u4*>(p));
}

// Element i of an array of 32- or 64-bit integers.
__device__ __forceinline__ int64_t int_at(const void* p, int is64, int64_t i) {
    return is64 ? static_cast<const int64_t*>(p)[i] : int64_t(static_cast<const int32_t*>(p)[i]);
}

inline bool known_dtype(int dtype) { return dtype == DOT_F32 || dtype == DOT_F16 || dtype == DOT_BF16; }
inline int dtype_bytes(int dtype) { return dtype == DOT_F32 ? 4 : 2; }

// f(T{}) with the element type of a tag that known_dtype() accepts.
template <class F>
void dispatch_dtype(int dtype, F&& f) {
    if (dtype == DOT_F32) f(float{});
    else if (dtype == DOT_F16) f(F16{});
    else f(BF16{});
}

}  // namespace dot_amd
