// mx_quant.hip -- K14: ordinary tensors <-> MXFP4 (yl_mx_quantize, yl_mx_dequantize; formats in include/yolo2_hip.h).
//
// A block of 32 values along k: m = max |x|, S = 2^(floor(log2 m) - 2), codes = RNE_E2M1(x / S) saturated at 6.  Pure data movement:
// bound by the bytes of the ordinary tensor (4 or 2 a value) and of the codes (17/32).
#include "mx_device.h"
#include "mx.h"

namespace yl {

// one thread a block
template <int TYPE>
__global__ __launch_bounds__(256) void mx_quantize_kernel(MxDense s, uint4 *__restrict__ codes, unsigned char *__restrict__ scales, int64_t ld, int64_t kb)
{
    const int64_t n = s.batch * s.rows * kb;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (int64_t)gridDim.x * 256) {
        const int64_t row = t / kb, j = t - row * kb;
        const int64_t b = row / s.rows, r = row - b * s.rows;
        const int64_t at = b * s.batch_stride + r * s.row_stride + j * MX_BLOCK * s.k_stride;
        float v[MX_BLOCK];
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < MX_BLOCK; ++i) {
            v[i] = j * MX_BLOCK + i < s.k ? mx_load<TYPE>(s.data, at + i * s.k_stride) : 0.f;
            top = max(top, mx_abs_bits(v[i]));
        }
        const unsigned byte = mx_scale_byte(top);
        uint4 q = make_uint4(0, 0, 0, 0);
        if (byte != 255) q = make_uint4(mx_codes8(v, byte), mx_codes8(v + 8, byte), mx_codes8(v + 16, byte), mx_codes8(v + 24, byte));
        codes[row * ld + j] = q;
        scales[row * ld + j] = (unsigned char)byte;
    }
}

template <int TYPE>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint4 *__restrict__ codes, const unsigned char *__restrict__ scales, int64_t ld, MxDense d, int64_t kb)
{
    const int64_t n = d.batch * d.rows * kb;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (int64_t)gridDim.x * 256) {
        const int64_t row = t / kb, j = t - row * kb;
        const int64_t b = row / d.rows, r = row - b * d.rows;
        const int64_t at = b * d.batch_stride + r * d.row_stride + j * MX_BLOCK * d.k_stride;
        const uint4 q = codes[row * ld + j];
        const unsigned byte = scales[row * ld + j];
        const float s = __builtin_bit_cast(float, byte << 23);
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < MX_BLOCK; i += 2) {
            const mx_f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i / 8] >> (4 * (i % 8)), s, 0);
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (j * MX_BLOCK + i + e < d.k)
                    mx_store<TYPE>(const_cast<void *>(d.data), at + (i + e) * d.k_stride, byte == 255 ? __builtin_nanf("") : v[e]);
        }
    }
}

static unsigned mx_blocks_for(int64_t n)
{
    const int64_t g = (n + 255) / 256;
    return (unsigned)(g < 1 ? 1 : (g > 256 * 64 ? 256 * 64 : g));
}

int launch_mx_quantize(const MxDense &src, void *codes, void *scales, int64_t ld, void *stream)
{
    const int64_t kb = (src.k + MX_BLOCK - 1) / MX_BLOCK, n = src.batch * src.rows * kb;
    if (n == 0) return 0;
    const dim3 grid(mx_blocks_for(n)), block(256);
    hipStream_t s = (hipStream_t)stream;
    uint4 *c = (uint4 *)codes;
    unsigned char *e = (unsigned char *)scales;
    switch (src.type) {
    case YL_F32: hipLaunchKernelGGL(mx_quantize_kernel<YL_F32>, grid, block, 0, s, src, c, e, ld, kb); break;
    case YL_F16: hipLaunchKernelGGL(mx_quantize_kernel<YL_F16>, grid, block, 0, s, src, c, e, ld, kb); break;
    default: hipLaunchKernelGGL(mx_quantize_kernel<YL_BF16>, grid, block, 0, s, src, c, e, ld, kb); break;
    }
    return (int)hipGetLastError();
}

int launch_mx_dequantize(const void *codes, const void *scales, int64_t ld, const MxDense &dst, void *stream)
{
    const int64_t kb = (dst.k + MX_BLOCK - 1) / MX_BLOCK, n = dst.batch * dst.rows * kb;
    if (n == 0) return 0;
    const dim3 grid(mx_blocks_for(n)), block(256);
    hipStream_t s = (hipStream_t)stream;
    const uint4 *c = (const uint4 *)codes;
    const unsigned char *e = (const unsigned char *)scales;
    switch (dst.type) {
    case YL_F32: hipLaunchKernelGGL(mx_dequantize_kernel<YL_F32>, grid, block, 0, s, c, e, ld, dst, kb); break;
    case YL_F16: hipLaunchKernelGGL(mx_dequantize_kernel<YL_F16>, grid, block, 0, s, c, e, ld, dst, kb); break;
    default: hipLaunchKernelGGL(mx_dequantize_kernel<YL_BF16>, grid, block, 0, s, c, e, ld, dst, kb); break;
    }
    return (int)hipGetLastError();
}

}  // namespace yl
