// Rows of f32, f16 or bf16 values at any element-aligned address, and reductions over the 64 lanes of a wave.
#pragma once

#include "cml_device.hpp"
#include "cml_host.hpp"

#pragma clang fp contract(off)

namespace cml {

typedef uint32_t v4u_row __attribute__((ext_vector_type(4)));

// Element types by GGUF type id.  bits16: the 16-bit types are carried as bit patterns.
struct TypeF32 {
    typedef float Bits;
};
struct TypeF16 {
    typedef uint16_t Bits;
    static __device__ __forceinline__ float widen(uint32_t b) { return f16_bits_to_f32(b & 0xffffu); }
    static __device__ __forceinline__ uint32_t narrow(float v) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v)); }  // to nearest, ties to even
};
struct TypeBF16 {
    typedef uint16_t Bits;
    static __device__ __forceinline__ float widen(uint32_t b) { return __builtin_bit_cast(float, b << 16); }
    static __device__ __forceinline__ uint32_t narrow(float v) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }  // to nearest, ties to even
};

// Calls f with the tag of a known type id.
template <class F>
int with_type(int dtype, F f) {
    switch (dtype) {
        case CML_F32: return f(TypeF32{});
        case CML_F16: return f(TypeF16{});
        default: return f(TypeBF16{});
    }
}

template <class T>
__device__ __forceinline__ float load_value(const typename T::Bits *p) {
    if constexpr (sizeof(typename T::Bits) == 4) return *p;
    else return T::widen(*p);
}
template <class T>
__device__ __forceinline__ void store_value(typename T::Bits *p, float v) {
    if constexpr (sizeof(typename T::Bits) == 4) *p = v;
    else *p = static_cast<uint16_t>(T::narrow(v));
}
// The value as the type holds it.
template <class T>
__device__ __forceinline__ float rounded(float v) {
    if constexpr (sizeof(typename T::Bits) == 4) return v;
    else return T::widen(T::narrow(v));
}

// Eight neighbouring values.  The address only has to be aligned to the element: global loads and stores of 16 bytes take any
// address on this chip (rows of an odd number of values start anywhere).
// ONCE: with the non-temporal hint.
template <class T, bool ONCE = false>
__device__ __forceinline__ void load8(const typename T::Bits *p, float (&v)[8]) {
    if constexpr (sizeof(typename T::Bits) == 4) {
        typedef float v4f __attribute__((ext_vector_type(4), aligned(4)));
        const v4f *q = reinterpret_cast<const v4f *>(p);
        const v4f a = ONCE ? __builtin_nontemporal_load(q) : q[0], b = ONCE ? __builtin_nontemporal_load(q + 1) : q[1];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    } else {
        typedef uint32_t v4u __attribute__((ext_vector_type(4), aligned(2)));
        const v4u *q = reinterpret_cast<const v4u *>(p);
        const v4u a = ONCE ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = T::widen(a[i] & 0xffffu);
            v[2 * i + 1] = T::widen(a[i] >> 16);
        }
    }
}
template <class T>
__device__ __forceinline__ void store8(typename T::Bits *p, const float (&v)[8]) {
    if constexpr (sizeof(typename T::Bits) == 4) {
        typedef float v4f __attribute__((ext_vector_type(4), aligned(4)));
        reinterpret_cast<v4f *>(p)[0] = v4f{v[0], v[1], v[2], v[3]};
        reinterpret_cast<v4f *>(p)[1] = v4f{v[4], v[5], v[6], v[7]};
    } else {
        typedef uint32_t v4u __attribute__((ext_vector_type(4), aligned(2)));
        v4u a;
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] = T::narrow(v[2 * i]) | T::narrow(v[2 * i + 1]) << 16;
        *reinterpret_cast<v4u *>(p) = a;
    }
}

// ---- over the 16 lanes of a row and the 64 of a wave, the same result in every lane; the association is fixed ----
__device__ __forceinline__ float row_allsum(float v) {
    v = v + dpp_f32<0xB1>(v);   // quad_perm [1,0,3,2]
    v = v + dpp_f32<0x4E>(v);   // quad_perm [2,3,0,1]
    v = v + dpp_f32<0x141>(v);  // row_half_mirror: the other quad
    return v + dpp_f32<0x140>(v);  // row_mirror: the other eight (both sides add the same two numbers every time)
}
__device__ __forceinline__ int row_allmax_i32(int v) {
    v = max(v, row_ror_i32<1>(v));
    v = max(v, row_ror_i32<2>(v));
    v = max(v, row_ror_i32<4>(v));
    return max(v, row_ror_i32<8>(v));
}
__device__ __forceinline__ int row_allmin_i32(int v) {
    v = min(v, row_ror_i32<1>(v));
    v = min(v, row_ror_i32<2>(v));
    v = min(v, row_ror_i32<4>(v));
    return min(v, row_ror_i32<8>(v));
}
__device__ __forceinline__ float lane_of(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }
__device__ __forceinline__ float rows_allsum(float v) {  // rows of 16 like row_allsum, then the four of them
    v = row_allsum(v);
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
__device__ __forceinline__ float wave_allsum(float v) {
    v = v + dpp_f32<0x121>(v);  // row_ror 1, 2, 4, 8: the sum of the row of 16 in all its lanes (each with its own association: one lane is read)
    v = v + dpp_f32<0x122>(v);
    v = v + dpp_f32<0x124>(v);
    v = v + dpp_f32<0x128>(v);
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
// f32 values as integers that order like them (-0 and 0 alike where 0 has been added), and back.
__device__ __forceinline__ float from_total_key(int key) { return __builtin_bit_cast(float, key ^ static_cast<int>(static_cast<unsigned>(key >> 31) >> 1)); }

}  // namespace cml
