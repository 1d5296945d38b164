// mx_product.hip -- K15: products of MXFP4 matrices on v_mfma_scale_f32_32x32x64_f8f6f4 (yl_mx_matmul, yl_mx_linear, yl_mx_conv2d).
//
//   D[i][j] = sum over blocks b of Sa[i][b] Sb[j][b] sum_{t < 32} ca[i][32 b + t] cb[j][32 b + t], summed in FP32
//
// The instruction takes 64 summed elements: lanes 0-31 hold one block (16 bytes) of rows 0-31 of an operand, lanes 32-63 the next block
// of the same rows, each with its own scale byte -- exactly the format's block, so no code is ever unpacked.  Products of codes are
// exact; the sum is FP32.  D's layout: lane l holds column l & 31, rows 8 (e / 4) + 4 (l >> 5) + e % 4.
#include <cstdio>

#include "activations.h"
#include "mx_device.h"
#include "mx.h"

namespace yl {

// one wave a 32 x 32 tile of D, operands straight from memory; the right answer for every case
template <int TYPE, bool CONV>
__global__ __launch_bounds__(256) void mx_product_plain_kernel(MxProductArgs p)
{
    const int lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5;
    const int64_t tiles_j = (p.J + 31) / 32, tiles = (p.I + 31) / 32 * tiles_j;
    const int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int64_t i0 = tile / tiles_j * 32, j0 = tile % tiles_j * 32;
    const int64_t i = i0 + l31, j = j0 + l31;
    const bool i_ok = i < p.I, j_ok = j < p.J;
    const uint4 *a_codes = (const uint4 *)p.a_codes + (i_ok ? i : 0) * p.a_ld;
    const unsigned char *a_scales = (const unsigned char *)p.a_scales + (i_ok ? i : 0) * p.a_ld;
    const uint4 *b_codes = (const uint4 *)p.b_codes;
    const unsigned char *b_scales = (const unsigned char *)p.b_scales;
    int64_t image = 0, pix = 0;
    int y0 = 0, x0 = 0;
    if (CONV) {
        const int64_t area = (int64_t)p.OH * p.OW;
        image = j / area;
        pix = j - image * area;
        y0 = (int)(pix / p.OW) * p.stride - p.pad;
        x0 = (int)(pix % p.OW) * p.stride - p.pad;
    } else {
        b_codes += (j_ok ? j : 0) * p.b_ld;
        b_scales += (j_ok ? j : 0) * p.b_ld;
    }
    mx_f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    for (int64_t b = 0; b < p.kb; b += 2) {
        const int64_t u = b + half;
        uint4 av = make_uint4(0, 0, 0, 0), bv = av;
        int as = 0, bs = 0;
        if (u < p.kb) {
            if (i_ok) { av = a_codes[u]; as = a_scales[u]; }
            if (CONV) {
                const int tap = (int)(u / p.G), g = (int)(u - (int64_t)tap * p.G);
                const int y = y0 + tap / p.size, x = x0 + tap % p.size;
                if (j_ok && y >= 0 && y < p.H && x >= 0 && x < p.W) {
                    const int64_t at = ((image * p.H + y) * p.W + x) * p.b_ld + g;
                    bv = b_codes[at];
                    bs = b_scales[at];
                }
            } else if (j_ok) { bv = b_codes[u]; bs = b_scales[u]; }
        }
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(__builtin_bit_cast(mx_v4i, av)), mx_operand(__builtin_bit_cast(mx_v4i, bv)),
                                                              acc, 4, 4, 0, as, 0, bs);
    }
    float y[16];
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int64_t r = i0 + 8 * (e / 4) + 4 * half + e % 4;
        const bool ok = r < p.I && j_ok;
        float v = acc[e];
        if (p.bias && ok) v += p.bias[CONV ? r : j];
        v = yl_act_epilogue(v, p.act);
        const int64_t at = CONV ? (image * p.I + r) * p.OH * p.OW + pix : r * p.out_stride + j;
        if (p.residual && ok) v += mx_load<TYPE>(p.residual, CONV ? at : r * p.residual_stride + j);
        if (p.out && ok) mx_store<TYPE>(p.out, at, v);
        y[e] = ok ? v : 0.f;
        top = max(top, mx_abs_bits(y[e]));
    }
    if (CONV && p.q_codes) {
        // the tile's 32 rows of column j are one block of the result: rows 0-3, 8-11, ... here, the others in lane l ^ 32
        top = max(top, (unsigned)__shfl_xor((int)top, 32));
        const unsigned byte = mx_scale_byte(top);
        float o[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = __shfl_xor(y[e], 32);
        if (j_ok && half == 0) {
            uint4 q = make_uint4(0, 0, 0, 0);
            if (byte != 255) {
                unsigned w[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float v[8] = {y[4 * g], y[4 * g + 1], y[4 * g + 2], y[4 * g + 3], o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]};
                    w[g] = mx_codes8(v, byte);
                }
                q = make_uint4(w[0], w[1], w[2], w[3]);
            }
            reinterpret_cast<uint4 *>(p.q_codes)[j * p.q_ld + i0 / 32] = q;
            reinterpret_cast<unsigned char *>(p.q_scales)[j * p.q_ld + i0 / 32] = (unsigned char)byte;
        }
    }
}

template <int TYPE, bool CONV>
static int launch_plain(const MxProductArgs &a, hipStream_t s)
{
    const int64_t tiles = (a.I + 31) / 32 * ((a.J + 31) / 32), grid = (tiles + 3) / 4;
    if (grid > 0x7fffffffLL) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((mx_product_plain_kernel<TYPE, CONV>), dim3((unsigned)grid), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

int launch_mx_product(const MxProductArgs &a, void *stream, char *name, size_t name_len)
{
    if (a.I == 0 || a.J == 0) return 0;
    hipStream_t s = (hipStream_t)stream;
    if (name) snprintf(name, name_len, "mx_product_plain");
    if (a.conv) return launch_plain<YL_F32, true>(a, s);
    switch (a.type) {
    case YL_F32: return launch_plain<YL_F32, false>(a, s);
    case YL_F16: return launch_plain<YL_F16, false>(a, s);
    default: return launch_plain<YL_BF16, false>(a, s);
    }
}

bool mx_linear_fused(int64_t, int64_t) { return false; }
int launch_mx_linear(const MxProductArgs &, const MxDense &, void *) { return (int)hipErrorInvalidValue; }

}  // namespace yl
