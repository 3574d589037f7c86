// vec_io.hpp -- loads and stores of 4 or 8 neighbouring values of fp32, bf16
// or fp16, as fp32 in registers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "codec_kernels.hpp"

namespace coset {

typedef float f32x2_io __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_io __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_io __attribute__((ext_vector_type(2)));

// Two values rounded to nearest even, low half first.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
    const f32x2_io v = {a, b};
    if constexpr (DT == DT_BF16)
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_io));
    else
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_io));
}

template <int DT>
__device__ __forceinline__ void unpack2(uint32_t u, float& a, float& b)
{
    if constexpr (DT == DT_BF16) {
        a = __uint_as_float(u << 16);
        b = __uint_as_float(u & 0xffff0000u);
    } else {
        const f16x2_io h = __builtin_bit_cast(f16x2_io, u);
        a = (float)h.x;
        b = (float)h.y;
    }
}

template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i)
{
    if constexpr (DT == DT_F32)
        return reinterpret_cast<const float*>(p)[i];
    else if constexpr (DT == DT_BF16)
        return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
    else
        return (float)reinterpret_cast<const _Float16*>(p)[i];
}

template <int DT>
__device__ __forceinline__ void store1(void* p, int64_t i, float v)
{
    if constexpr (DT == DT_F32)
        reinterpret_cast<float*>(p)[i] = v;
    else
        reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)pack2<DT>(v, 0.f);
}

// N = 4 or 8 values from element i on; vec: the address is a multiple of the
// load's width (at most 16 bytes).
template <int DT, int N>
__device__ __forceinline__ void load_n(const void* p, int64_t i, bool vec, float* x)
{
    if (!vec) {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = load1<DT>(p, i + j);
        return;
    }
    if constexpr (DT == DT_F32) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i + j);
            x[j] = v.x;
            x[j + 1] = v.y;
            x[j + 2] = v.z;
            x[j + 3] = v.w;
        }
    } else {
        uint32_t u[N / 2];
        if constexpr (N == 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
            u[0] = v.x;
            u[1] = v.y;
            u[2] = v.z;
            u[3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i);
            u[0] = v.x;
            u[1] = v.y;
        }
#pragma unroll
        for (int j = 0; j < N / 2; ++j) unpack2<DT>(u[j], x[2 * j], x[2 * j + 1]);
    }
}

template <int DT, int N>
__device__ __forceinline__ void store_n(void* p, int64_t i, const float* x)
{
    if constexpr (DT == DT_F32) {
#pragma unroll
        for (int j = 0; j < N; j += 4)
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i + j) =
                make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
    } else if constexpr (N == 8) {
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i) =
            make_uint4(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]), pack2<DT>(x[4], x[5]), pack2<DT>(x[6], x[7]));
    } else {
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + i) =
            make_uint2(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]));
    }
}

}  // namespace coset
