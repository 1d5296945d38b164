// mx_device.h -- what the MXFP4 kernels share on the device.
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <tuple>
#include <utility>

#include "../../include/yolo2_hip.h"
#include "activations.h"

namespace yl {

// A launch and its own status.  (hipGetLastError behind it would also report what an earlier call of the thread, another library's
// included, left there.)  A launch counts its threads in 32 bits.
template <typename... P, size_t... I>
inline int mx_launch_with(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t s, std::tuple<P...> values, std::index_sequence<I...>)
{
    if ((uint64_t)grid.x * block.x > 0xFFFFFFFFull) return (int)hipErrorInvalidConfiguration;
    void *args[] = {&std::get<I>(values)...};
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, args, 0, s);
    if (e != hipSuccess) (void)hipGetLastError();          // it is this call's answer, not one for the thread's next question
    return (int)e;
}
template <typename... P, typename... A>
inline int mx_launch(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t s, A... args)
{
    return mx_launch_with(kernel, grid, block, s, std::tuple<P...>(args...), std::index_sequence_for<P...>{});
}

typedef int mx_v4i __attribute__((ext_vector_type(4)));
typedef int mx_v8i __attribute__((ext_vector_type(8)));
typedef float mx_f32x2 __attribute__((ext_vector_type(2)));
typedef float mx_f32x4 __attribute__((ext_vector_type(4)));
typedef float mx_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 mx_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 mx_f16x8 __attribute__((ext_vector_type(8)));

// one value of an ordinary tensor <-> FP32.  To FP16 / BF16: nearest even, half a step (2^-11 / 2^-8 of the value) at most.
template <int TYPE>
__device__ __forceinline__ float mx_load(const void *p, int64_t i)
{
    if constexpr (TYPE == YL_F32) return reinterpret_cast<const float *>(p)[i];
    else if constexpr (TYPE == YL_F16) return (float)reinterpret_cast<const _Float16 *>(p)[i];
    else return __builtin_bit_cast(float, (unsigned)reinterpret_cast<const unsigned short *>(p)[i] << 16);
}
template <int TYPE>
__device__ __forceinline__ void mx_store(void *p, int64_t i, float v)
{
    if constexpr (TYPE == YL_F32) reinterpret_cast<float *>(p)[i] = v;
    else if constexpr (TYPE == YL_F16) reinterpret_cast<_Float16 *>(p)[i] = (_Float16)v;
    else reinterpret_cast<__bf16 *>(p)[i] = (__bf16)v;
}

// 16 bytes of neighbouring values, the first on a whole vector: 4 of FP32, 8 of the others
template <int TYPE>
constexpr int MX_VEC = TYPE == YL_F32 ? 4 : 8;
typedef unsigned mx_u32x4 __attribute__((ext_vector_type(4)));
template <int TYPE>
__device__ __forceinline__ mx_u32x4 mx_pack(const float *v)
{
    if constexpr (TYPE == YL_F32) return __builtin_bit_cast(mx_u32x4, mx_f32x4{v[0], v[1], v[2], v[3]});
    else if constexpr (TYPE == YL_F16) return __builtin_bit_cast(mx_u32x4, mx_f16x8{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3], (_Float16)v[4], (_Float16)v[5], (_Float16)v[6], (_Float16)v[7]});
    else return __builtin_bit_cast(mx_u32x4, mx_bf16x8{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3], (__bf16)v[4], (__bf16)v[5], (__bf16)v[6], (__bf16)v[7]});
}
template <int TYPE>
__device__ __forceinline__ void mx_unpack(mx_u32x4 x, float *v)
{
    if constexpr (TYPE == YL_F32) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const unsigned w = x[q];                       // a copy: the cast of the element itself gives element 0
            v[q] = __builtin_bit_cast(float, w);
        }
    } else if constexpr (TYPE == YL_F16) {
        const mx_f16x8 h = __builtin_bit_cast(mx_f16x8, x);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = (float)h[q];
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            v[2 * q] = __builtin_bit_cast(float, x[q] << 16);
            v[2 * q + 1] = __builtin_bit_cast(float, x[q] & 0xffff0000u);
        }
    }
}
// vectors where memory has no more than the type's alignment: the hardware takes them
typedef mx_u32x4 mx_u32x4_any __attribute__((aligned(2)));
template <int TYPE>
__device__ __forceinline__ mx_u32x4 mx_load_vec(const void *p, int64_t i) { return *reinterpret_cast<const mx_u32x4_any *>(reinterpret_cast<const char *>(p) + i * (16 / MX_VEC<TYPE>)); }
template <int TYPE>
__device__ __forceinline__ void mx_store_vec(void *p, int64_t i, mx_u32x4 v) { *reinterpret_cast<mx_u32x4_any *>(reinterpret_cast<char *>(p) + i * (16 / MX_VEC<TYPE>)) = v; }

// activate(): LINEAR, LEAKY and RELU (x * (x > 0): NaN of -Inf) by one slope below zero, in 32 bits; the others only where RARE says so.
// LEAKY's product by 0.1f is off by 2^-24 (the rounding) + 2^-26 (0.1f) of the value at most; (float)(.1 * (double)x), the other
// convolutions' LEAKY, by 2^-24, for three conversions and multiplies in 64 bits an element.
template <bool RARE>
__device__ __forceinline__ float mx_activate(float v, int act)
{
    if (RARE && act != YL_LINEAR && act != YL_LEAKY && act != YL_RELU) return yl_activate(v, act);
    const float slope = act == YL_LINEAR ? 1.f : act == YL_LEAKY ? .1f : 0.f;
    return v > 0.f ? v : __fmul_rn(v, slope);
}

// The scale byte of a block whose largest magnitude has the FP32 bits `top` (exponent field f): floor(log2) is f - 127, the largest
// E2M1 exponent is 2, so the byte is f - 2, not below 0 (2^-127; subnormals and zero have f = 0).  f = 255 is an Inf or a NaN.
__device__ __forceinline__ unsigned mx_scale_byte(unsigned top)
{
    const unsigned f = top >> 23;
    return f == 255 ? 255u : (f > 2 ? f - 2 : 0u);
}
// eight values / 2^(byte - 127) -> eight codes: nearest even, saturated at 6 (v_cvt_scalef32_pk_fp4_f32 reads the scale's exponent
// field alone, byte 0 included).  Dividing by a power of two is exact here: |value| < 8 * scale.
__device__ __forceinline__ unsigned mx_codes8(const float *v, unsigned byte)
{
    const float s = __builtin_bit_cast(float, byte << 23);
    unsigned q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], s, 3);
    return q;
}
// eight codes -> the values they stand for; NaN under scale byte 255
__device__ __forceinline__ void mx_values8(unsigned codes, unsigned byte, float *v)
{
    const float s = __builtin_bit_cast(float, byte << 23);
    const mx_f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 1);
    const mx_f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
    if (byte == 255)
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = __builtin_nanf("");
}
__device__ __forceinline__ unsigned mx_abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

__device__ __forceinline__ mx_v8i mx_operand(mx_v4i c) { return mx_v8i{c[0], c[1], c[2], c[3], 0, 0, 0, 0}; }

// eight values from x[i], the first `n` of them; 16 bytes at a time where all eight are there
template <int TYPE>
__device__ __forceinline__ void mx_read8(const void *x, int64_t i, int n, float *v)
{
    if (n >= 8) {
        const char *p = reinterpret_cast<const char *>(x) + i * (16 / MX_VEC<TYPE>);
        if constexpr (TYPE == YL_F32) {
            mx_unpack<TYPE>(*reinterpret_cast<const mx_u32x4_any *>(p), v);
            mx_unpack<TYPE>(*reinterpret_cast<const mx_u32x4_any *>(p + 16), v + 4);
        } else mx_unpack<TYPE>(*reinterpret_cast<const mx_u32x4_any *>(p), v);
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = q < n ? mx_load<TYPE>(x, i + q) : 0.f;
    }
}
}  // namespace yl
