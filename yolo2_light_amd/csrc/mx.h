// mx.h -- launch interfaces of the MXFP4 kernels (mx_quant.hip, mx_product.hip) and what they share.
#pragma once
#include <cstdint>
#include <cstddef>

#include "../../include/yolo2_hip.h"

namespace yl {

constexpr int MX_BLOCK = 32;       // values a scale covers; 16 bytes of codes
constexpr int MX_MAX_SIZE = 5;     // filter edge: the taps' validity is a 25-bit mask

constexpr int64_t MX_MAX_ELEMENTS = (int64_t)1 << 46;     // what a stride or a size may address: products of two stay in 64 bits
constexpr int64_t MX_MAX_ROWS = 0x7fffffff - 256;         // rows of a product's side: the end of a tile of 256 is still a 32-bit number

// Why the kernel's 32-bit counts and offsets do not hold a convolution (of a map of `c` channels, x_ld blocks from pixel to pixel, with n
// filters), or nullptr.  0 <= pad < size, 1 <= h, w, c, stride, and the filter is no larger than the padded map.
inline const char *mx_conv_beyond(int64_t batch, int64_t h, int64_t w, int64_t c, int64_t x_ld, int64_t n, int size, int64_t stride, int pad)
{
    if (h > 1 << 20 || w > 1 << 20 || stride > 1 << 20) return "a map edge or stride above 2^20";
    if (c > 1 << 18) return "more than 2^18 channels";
    if (n > MX_MAX_ROWS || batch > MX_MAX_ROWS / (h * w)) return "map or result is too large";
    const int64_t oh = (h + 2 * pad - size) / stride + 1, ow = (w + 2 * pad - size) / stride + 1, area = oh * ow;
    if (batch > MX_MAX_ROWS / area || (batch > 0 && n > MX_MAX_ELEMENTS / (batch * area))) return "map or result is too large";
    // the rows of the map under 256 neighbouring positions of the result
    const int64_t rows = batch * h * w, under = (size + 1) * (w + 1), part = 256 % area;
    const int64_t reach = (256 / area + 1) * h * w + ((part + ow - 1) / ow + 1) * stride * w + under;
    if ((reach < rows ? reach : rows) + under > 0xFFFFFFFFLL / 16 / x_ld) return "rows of the map are too far apart";
    // the planes of the images that 256 neighbouring positions lie in
    if ((256 / area + 2) > 0xFFFFFFFFLL / 4 / (area * (n > 0 ? n : 1))) return "an image's result is too large";
    return nullptr;
}

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
// an activation other than LINEAR, LEAKY and RELU
inline bool mx_rare(int act) { return act != YL_LINEAR && act != YL_LEAKY && act != YL_RELU; }
// the linear layer on an ordinary x (launch_mx_product's a_codes / a_scales / a_ld unused), where mx_linear_fused(rows, k)
bool mx_linear_fused(int64_t rows, int64_t k);
int launch_mx_linear(const MxProductArgs &a, const MxDense &x, void *stream);

// Whether a launch's threads are counted in 32 bits, for the form that a call of such a size takes (above 2^20 workgroups none depends on
// the number of CUs any more).  Rounding: only tensors whose k is not contiguous have a workgroup for every 64 rows.
constexpr int64_t MX_MAX_THREADS = 0xFFFFFFFFLL;
inline bool mx_rounding_fits(const MxDense &t)
{
    const int64_t kb = (t.k + MX_BLOCK - 1) / MX_BLOCK;
    return t.k_stride == 1 || t.k <= 1 || t.batch * t.rows <= 0 || (t.batch * t.rows + 63) / 64 <= MX_MAX_THREADS / 256 / ((kb + 7) / 8);
}
inline bool mx_product_fits(const MxProductArgs &a)
{
    auto tiles = [&](int64_t ti, int64_t tj) { return ((a.I + ti - 1) / ti) * ((a.J + tj - 1) / tj); };
    if (!a.conv && mx_few_takes(a.I)) return tiles(32, a.I <= 16 && mx_linear_fused(a.I, a.k) ? 16 : 32) <= MX_MAX_THREADS / 512;
    const int64_t n = mx_rare(a.act) ? tiles(64, 64) : a.conv ? tiles(64, 128) : a.kb >= 64 ? tiles(256, 256) : tiles(128, 128);
    return n <= MX_MAX_THREADS / 256;
}

}  // namespace yl
