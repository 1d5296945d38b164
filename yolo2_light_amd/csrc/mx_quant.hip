// mx_quant.hip -- K14: ordinary tensors <-> MXFP4 (yl_mx_quantize, yl_mx_dequantize; formats in include/yolo2_hip.h).
//
// A block of 32 values along k: m = max |x|, S = 2^(floor(log2 m) - 2), codes = RNE_E2M1(x / S) saturated at 6.  Pure data movement:
// bound by the bytes of the ordinary tensor (4 or 2 a value) and of the codes (17/32).  Two forms of each direction:
//   rows     k is contiguous: four neighbouring lanes hold a block, eight values each, read as 16-byte vectors; the block's maximum is
//            taken across the four, each makes the 32 bits of its own codes, so a wave reads and writes contiguous memory
//   columns  any other strides, in practice NCHW maps, where rows (pixels) are contiguous: a lane holds a whole block of one row, so a
//            wave reads 64 neighbouring pixels of a channel at a time; codes go through LDS, so that a row's blocks leave together
// MI355X: 16 x 256 x 76 x 76 FP32 to MXFP4 and back 20.0 + 20.3 us, 6.0 TB/s (out of the 256 MB cache; 51 us from HBM, where a large copy
// makes 5.1 TB/s); 4096 x 4096 BF16 rows 10.1 us; one row of 4096 2.3 us, which is a launch.  One thread a block with scalar loads, the
// first form, took 52 us for the map's pair and 27 instead of 7.1 us (both out of a graph; 4.4 + 4.1 each by itself) for the pair on
// 3001 x 1005 FP16 values in rows of 1016.
#include "mx_device.h"
#include "mx.h"
#include "kernels.h"

namespace yl {

template <int TYPE>
__device__ __forceinline__ void mx_write8(void *x, int64_t i, int n, const float *v)
{
    if (n >= 8) {
        char *p = reinterpret_cast<char *>(x) + i * (16 / MX_VEC<TYPE>);
        *reinterpret_cast<mx_u32x4_any *>(p) = mx_pack<TYPE>(v);
        if constexpr (TYPE == YL_F32) *reinterpret_cast<mx_u32x4_any *>(p + 16) = mx_pack<TYPE>(v + 4);
    } else {
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (q < n) mx_store<TYPE>(x, i + q, v[q]);
    }
}

// INDEX: 32 bits while all blocks can be counted in them (a division of 64 bits costs more than the block)
template <int TYPE, typename INDEX>
__global__ __launch_bounds__(256) void mx_quantize_rows_kernel(MxDense s, unsigned *__restrict__ codes, unsigned char *__restrict__ scales, int64_t ld, INDEX kb, INDEX n)
{
    const int part = threadIdx.x & 3;
    for (INDEX t = (INDEX)blockIdx.x * 64 + threadIdx.x / 4; t < n; t += (INDEX)gridDim.x * 64) {
        const INDEX row = t / kb, j = t - row * kb;
        int64_t at = (int64_t)row * s.row_stride;
        if (s.batch > 1) {
            const INDEX b = row / (INDEX)s.rows;
            at = (int64_t)b * s.batch_stride + (int64_t)(row - b * (INDEX)s.rows) * s.row_stride;
        }
        const int64_t first = (int64_t)j * MX_BLOCK + part * 8, left = s.k - first;
        float v[8];
        mx_read8<TYPE>(s.data, at + first, left > 8 ? 8 : (int)left, v);
        unsigned top = 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) top = max(top, mx_abs_bits(v[q]));
        top = max(top, (unsigned)__shfl_xor((int)top, 1));
        top = max(top, (unsigned)__shfl_xor((int)top, 2));
        const unsigned byte = mx_scale_byte(top);
        codes[((int64_t)row * ld + j) * 4 + part] = byte == 255 ? 0u : mx_codes8(v, byte);
        if (part == 0) scales[(int64_t)row * ld + j] = (unsigned char)byte;
    }
}

template <int TYPE, typename INDEX>
__global__ __launch_bounds__(256) void mx_dequantize_rows_kernel(const unsigned *__restrict__ codes, const unsigned char *__restrict__ scales, int64_t ld, MxDense d, INDEX kb, INDEX n)
{
    const int part = threadIdx.x & 3;
    for (INDEX t = (INDEX)blockIdx.x * 64 + threadIdx.x / 4; t < n; t += (INDEX)gridDim.x * 64) {
        const INDEX row = t / kb, j = t - row * kb;
        int64_t at = (int64_t)row * d.row_stride;
        if (d.batch > 1) {
            const INDEX b = row / (INDEX)d.rows;
            at = (int64_t)b * d.batch_stride + (int64_t)(row - b * (INDEX)d.rows) * d.row_stride;
        }
        const int64_t first = (int64_t)j * MX_BLOCK + part * 8, left = d.k - first;
        if (left <= 0) continue;
        const unsigned byte = scales[(int64_t)row * ld + j];
        float v[8];
        mx_values8(codes[((int64_t)row * ld + j) * 4 + part], byte, v);
        mx_write8<TYPE>(const_cast<void *>(d.data), at + first, left > 8 ? 8 : (int)left, v);
    }
}

// A workgroup takes 64 rows by BLOCKS blocks: 8, two a wave, or 4 where 8 would leave CUs without work.
constexpr int MX_COLS_ROWS = 64;

template <int TYPE, int BLOCKS>
__global__ __launch_bounds__(256) void mx_quantize_columns_kernel(MxDense s, uint4 *__restrict__ codes, unsigned char *__restrict__ scales, int64_t ld, int64_t kb, int64_t groups)
{
    __shared__ uint4 lc[MX_COLS_ROWS * BLOCKS];
    __shared__ unsigned char ls[MX_COLS_ROWS * BLOCKS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tile = blockIdx.x / groups, j0 = (blockIdx.x - tile * groups) * BLOCKS;
    const int64_t row0 = tile * MX_COLS_ROWS, rows = s.batch * s.rows, row = row0 + lane;
    const int blocks = (int)min((int64_t)BLOCKS, kb - j0), count = (int)min((int64_t)MX_COLS_ROWS, rows - row0);
    if (lane < count) {
        const int64_t b = s.batch > 1 ? row / s.rows : 0;
        const int64_t at = b * s.batch_stride + (row - b * s.rows) * s.row_stride;
#pragma unroll
        for (int h = 0; h < BLOCKS / 4; ++h) {
            const int j = wave + 4 * h;
            if (j >= blocks) break;
            const int64_t k0 = (j0 + j) * MX_BLOCK;
            float v[MX_BLOCK];
            if (k0 + MX_BLOCK <= s.k) {
#pragma unroll
                for (int i = 0; i < MX_BLOCK; ++i) v[i] = mx_load<TYPE>(s.data, at + (k0 + i) * s.k_stride);
            } else {
#pragma unroll
                for (int i = 0; i < MX_BLOCK; ++i) v[i] = k0 + i < s.k ? mx_load<TYPE>(s.data, at + (k0 + i) * s.k_stride) : 0.f;
            }
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < MX_BLOCK; ++i) top = max(top, mx_abs_bits(v[i]));
            const unsigned byte = mx_scale_byte(top);
            uint4 q = make_uint4(0, 0, 0, 0);
            if (byte != 255) q = make_uint4(mx_codes8(v, byte), mx_codes8(v + 8, byte), mx_codes8(v + 16, byte), mx_codes8(v + 24, byte));
            lc[lane * blocks + j] = q;
            ls[lane * blocks + j] = (unsigned char)byte;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < count * blocks; i += 256) {
        const int r = i / blocks;
        const int64_t to = (row0 + r) * ld + j0 + (i - r * blocks);
        codes[to] = lc[i];
        scales[to] = ls[i];
    }
}

template <int TYPE, int BLOCKS>
__global__ __launch_bounds__(256) void mx_dequantize_columns_kernel(const uint4 *__restrict__ codes, const unsigned char *__restrict__ scales, int64_t ld, MxDense d, int64_t kb, int64_t groups)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tile = blockIdx.x / groups, j0 = (blockIdx.x - tile * groups) * BLOCKS;
    const int64_t row = tile * MX_COLS_ROWS + lane;
    if (row >= d.batch * d.rows) return;
    const int64_t b = d.batch > 1 ? row / d.rows : 0;
    const int64_t at = b * d.batch_stride + (row - b * d.rows) * d.row_stride;
    for (int64_t j = j0 + wave; j < kb && j < j0 + BLOCKS; j += 4) {
        const uint4 q = codes[row * ld + j];
        const unsigned byte = scales[row * ld + j];
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float v[8];
            mx_values8(w[g], byte, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t k = j * MX_BLOCK + 8 * g + i;
                if (k < d.k) mx_store<TYPE>(const_cast<void *>(d.data), at + k * d.k_stride, v[i]);
            }
        }
    }
}

static int columns_blocks(int64_t tiles, int64_t kb) { return tiles * ((kb + 7) / 8) >= 2 * (int64_t)device_cu_count() ? 8 : 4; }

template <int TYPE>
static int launch_quantize(const MxDense &src, void *codes, void *scales, int64_t ld, hipStream_t s)
{
    const int64_t kb = (src.k + MX_BLOCK - 1) / MX_BLOCK, rows = src.batch * src.rows, n = rows * kb;
    if (src.k_stride == 1 || src.k == 1) {
        const int64_t g = (n + 63) / 64;
        const dim3 grid((unsigned)(g > 1 << 20 ? 1 << 20 : g));
        if (n < 0x60000000) return mx_launch(mx_quantize_rows_kernel<TYPE, unsigned>, grid, dim3(256), s, src, (unsigned *)codes, (unsigned char *)scales, ld, (unsigned)kb, (unsigned)n);
        return mx_launch(mx_quantize_rows_kernel<TYPE, int64_t>, grid, dim3(256), s, src, (unsigned *)codes, (unsigned char *)scales, ld, kb, n);
    } else {
        const int64_t tiles = (rows + MX_COLS_ROWS - 1) / MX_COLS_ROWS;
        const int blocks = columns_blocks(tiles, kb);
        const int64_t groups = (kb + blocks - 1) / blocks, g = tiles * groups;
        if (g > 0x7fffffff) return (int)hipErrorInvalidValue;
        if (blocks == 8) return mx_launch(mx_quantize_columns_kernel<TYPE, 8>, dim3((unsigned)g), dim3(256), s, src, (uint4 *)codes, (unsigned char *)scales, ld, kb, groups);
        return mx_launch(mx_quantize_columns_kernel<TYPE, 4>, dim3((unsigned)g), dim3(256), s, src, (uint4 *)codes, (unsigned char *)scales, ld, kb, groups);
    }
}

template <int TYPE>
static int launch_dequantize(const void *codes, const void *scales, int64_t ld, const MxDense &dst, hipStream_t s)
{
    const int64_t kb = (dst.k + MX_BLOCK - 1) / MX_BLOCK, rows = dst.batch * dst.rows, n = rows * kb;
    if (dst.k_stride == 1 || dst.k == 1) {
        const int64_t g = (n + 63) / 64;
        const dim3 grid((unsigned)(g > 1 << 20 ? 1 << 20 : g));
        if (n < 0x60000000) return mx_launch(mx_dequantize_rows_kernel<TYPE, unsigned>, grid, dim3(256), s, (const unsigned *)codes, (const unsigned char *)scales, ld, dst, (unsigned)kb, (unsigned)n);
        return mx_launch(mx_dequantize_rows_kernel<TYPE, int64_t>, grid, dim3(256), s, (const unsigned *)codes, (const unsigned char *)scales, ld, dst, kb, n);
    } else {
        const int64_t tiles = (rows + MX_COLS_ROWS - 1) / MX_COLS_ROWS;
        const int blocks = columns_blocks(tiles, kb);
        const int64_t groups = (kb + blocks - 1) / blocks, g = tiles * groups;
        if (g > 0x7fffffff) return (int)hipErrorInvalidValue;
        if (blocks == 8) return mx_launch(mx_dequantize_columns_kernel<TYPE, 8>, dim3((unsigned)g), dim3(256), s, (const uint4 *)codes, (const unsigned char *)scales, ld, dst, kb, groups);
        return mx_launch(mx_dequantize_columns_kernel<TYPE, 4>, dim3((unsigned)g), dim3(256), s, (const uint4 *)codes, (const unsigned char *)scales, ld, dst, kb, groups);
    }
}

int launch_mx_quantize(const MxDense &src, void *codes, void *scales, int64_t ld, void *stream)
{
    if (src.batch == 0 || src.rows == 0 || src.k == 0) return 0;
    hipStream_t s = (hipStream_t)stream;
    return src.type == YL_F32 ? launch_quantize<YL_F32>(src, codes, scales, ld, s)
         : src.type == YL_F16 ? launch_quantize<YL_F16>(src, codes, scales, ld, s) : launch_quantize<YL_BF16>(src, codes, scales, ld, s);
}

int launch_mx_dequantize(const void *codes, const void *scales, int64_t ld, const MxDense &dst, void *stream)
{
    if (dst.batch == 0 || dst.rows == 0 || dst.k == 0) return 0;
    hipStream_t s = (hipStream_t)stream;
    return dst.type == YL_F32 ? launch_dequantize<YL_F32>(codes, scales, ld, dst, s)
         : dst.type == YL_F16 ? launch_dequantize<YL_F16>(codes, scales, ld, dst, s) : launch_dequantize<YL_BF16>(codes, scales, ld, dst, s);
}

}  // namespace yl
