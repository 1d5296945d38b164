// mx.h -- launch interfaces of the MXFP4 kernels (mx_quant.hip, mx_product.hip) and what they share.
#pragma once
#include <cstdint>
#include <cstddef>

namespace yl {

constexpr int MX_BLOCK = 32;       // values a scale covers; 16 bytes of codes
constexpr int MX_MAX_SIZE = 5;     // filter edge: the taps' validity is a 25-bit mask

struct MxDense {                   // see yl_dense
    const void *data;
    int type;
    int64_t batch, rows, k, batch_stride, row_stride, k_stride;
};

// codes / scales with a row stride of ld blocks; kb = ceil(k / 32) blocks a row are used
int launch_mx_quantize(const MxDense &src, void *codes, void *scales, int64_t ld, void *stream);
int launch_mx_dequantize(const void *codes, const void *scales, int64_t ld, const MxDense &dst, void *stream);

// D[i][j] = sum_k A[i][k] * B[j][k]: i are the matrix instruction's rows, j its columns -- neighbouring lanes, so the memory a row of D
// is written to is contiguous along j.  A linear layer has A = x, B = w; a convolution writes NCHW planes and has A = filters, B = pixels.
struct MxProductArgs {
    const void *a_codes, *a_scales, *b_codes, *b_scales;
    int64_t a_ld, b_ld;
    int64_t I, J;
    int64_t k = 0;                 // the summed axis (linear)
    int64_t kb;                    // ... in blocks
    const float *bias;             // along j (linear) or along i (conv)
    int act;
    const void *residual;
    int64_t residual_stride;
    void *out;
    int64_t out_stride;            // elements from i to i + 1
    int type;                      // YL_F32 / YL_F16 / YL_BF16 of out and residual
    // convolution: B is a map [batch][H][W][G blocks], j = (image, oy, ox); out[image][i][oy][ox] float
    bool conv = false;
    int H = 0, W = 0, OH = 0, OW = 0, G = 0, size = 1, stride = 1, pad = 0, batch = 1;
    void *q_codes = nullptr, *q_scales = nullptr;     // optional: D rounded to MXFP4, one row a j
    int64_t q_ld = 0;
};
int launch_mx_product(const MxProductArgs &a, void *stream, char *name = nullptr, size_t name_len = 0);

// few rows (mx_few.hip)
bool mx_few_takes(int64_t rows);
int launch_mx_few(const MxProductArgs &a, void *stream);
// the linear layer on an ordinary x (launch_mx_product's a_codes / a_scales / a_ld unused), where mx_linear_fused(rows, k)
bool mx_linear_fused(int64_t rows, int64_t k);
int launch_mx_linear(const MxProductArgs &a, const MxDense &x, void *stream);

}  // namespace yl
