// mx_few.hip -- K15f: products of MXFP4 matrices with few rows on one side (yl_mx_matmul and yl_mx_linear up to 32 rows of x; the single
// token of a decoding step).
//
// With few rows the product is a reading of w: 17/32 bytes a weight, once.  What counts is that every CU has enough of w in flight, so
// columns go C = 16 or 32 to a workgroup and the summed axis to its eight waves, chunk by chunk in turn; each lane loads the 16-byte
// blocks that it feeds to the matrix instruction straight into its registers, one chunk ahead.  The waves' sums are added in LDS in the
// order of the waves (the same bits every time), then bias, activation, residual, store.
// FUSED (up to 16 rows): x is an ordinary tensor and every workgroup rounds all of it into its LDS while its first weights travel: no
// launch and no workspace for the rounding, and the same codes and the same sums as rounding first.
// MI355X: 1 x 4096 x 4096 from BF16 3.9 to 4.4 us (w alone at 5.1 TB/s: 1.7 us, the rest is the launch and one round trip to memory; three waits of
// four cycles), 1 x 8192 x 8192 8.7 us (7.0), 32 x 8192 x 8192 12.6.  More rows lie with the tiles of mx_product.hip: every workgroup
// here reads all of x, and at 64 rows that cost more than w (8192 x 8192, in a form for 64 rows: 18.3 us against 14.6).  At the border
// 32 x 8192 x 8192 12.6 us against 13.6 with the tiles, 32 x 4096 x 4096 7.6 against 8.2, but 32 x 16384 x 4096 12.7 against 9.5.
#include "activations.h"
#include "mx_device.h"
#include "mx.h"
#include "kernels.h"

namespace yl {

constexpr int MX_FEW_WAVES = 8, MX_FEW_THREADS = 64 * MX_FEW_WAVES;
constexpr int MX_FEW_LDS = 40960;      // bytes for the rounded x of the fused form

// bytes of LDS that rows x k take: rows of whole chunks of 16 blocks, one unit apart from a power of two, then the scales
static inline int64_t mx_few_lds(int64_t rows, int64_t k)
{
    const int64_t kbp = ((k + MX_BLOCK - 1) / MX_BLOCK + 15) / 16 * 16;
    return rows * ((kbp + 1) * 16 + kbp);
}

// Rounding x in every workgroup pays while it is little against the weights that travel meanwhile, and saves the host a launch of 3 us; one row always.
// MI355X, GPU time in us with it / with a launch of its own, k = 4096 (16 rows: k = 2048), by the rows of w:
//   rows    1024         4096         16384         65536
//   1       4.3 / 6.1    4.4 / 6.2    9.6 / 11.7    30.8 / 31.5     (k = 16384: 9.1 / 10.3, 10.1 / 11.2, 29.2 / 32.4, 117 / 129)
//   2       4.8 / 6.2    4.9 / 6.4    10.9 / 11.5   36.4 / 31.4
//   4       5.7 / 6.3    5.9 / 6.5    12.8 / 11.8   44.9 / 32.6
//   8       7.7 / 6.6    8.0 / 6.7    19.0 / 12.2   63.9 / 32.3
//   16      7.1 / 5.9    7.3 / 5.9    15.8 / 8.4    52.7 / 21.6
//   16 rows of k = 4096, above the border: 11.6 / 7.1, 12.1 / 7.2, 29.9 / 13.1, 101 / 35
// The rule sees rows and k alone (so does the workspace that a caller asks for): with up to 4096 rows of w the launch that it saves the
// host is worth more than what it costs the GPU; with a w of many more rows and 8 to 16 rows of x it costs up to 2.5 times the time.
bool mx_linear_fused(int64_t rows, int64_t k)
{
    return rows <= 16 && k <= (int64_t)1 << 20 && (rows <= 1 || rows * k <= 32768) && mx_few_lds(rows, k) <= MX_FEW_LDS;
}
bool mx_few_takes(int64_t rows) { return rows <= 32; }

typedef unsigned mx_u32_any __attribute__((aligned(1)));

template <int TYPE>
__device__ __forceinline__ void mx_few_round(const MxDense &x, char *lds, int kb, int kbp)
{
    uint4 *codes = reinterpret_cast<uint4 *>(lds);
    unsigned char *scales = reinterpret_cast<unsigned char *>(lds) + x.rows * (kbp + 1) * 16;
    const int part = threadIdx.x & 3, n = (int)x.rows * kbp;
    for (int t = threadIdx.x / 4; t < n; t += MX_FEW_THREADS / 4) {
        const int row = t / kbp, j = t - row * kbp;
        const int left = (int)x.k - j * MX_BLOCK - part * 8;
        float v[8];
        const int64_t at = row * x.row_stride + ((int64_t)j * MX_BLOCK + part * 8) * x.k_stride;
        if (x.k_stride == 1) mx_read8<TYPE>(x.data, at, left > 8 ? 8 : left, v);
        else
            for (int q = 0; q < 8; ++q) v[q] = q < left ? mx_load<TYPE>(x.data, at + q * x.k_stride) : 0.f;
        unsigned top = 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) top = max(top, mx_abs_bits(v[q]));
        top = max(top, (unsigned)__shfl_xor((int)top, 1));
        top = max(top, (unsigned)__shfl_xor((int)top, 2));
        const unsigned byte = mx_scale_byte(top);
        reinterpret_cast<unsigned *>(codes + row * (kbp + 1) + j)[part] = byte == 255 ? 0u : mx_codes8(v, byte);
        if (part == 0) scales[row * kbp + j] = (unsigned char)byte;
    }
}

// four steps of one side: the lane's blocks, and the scales of the chunk's blocks of its row
template <int C>
struct MxFewChunk {
    mx_v4i codes[4];
    unsigned scales[C == 16 ? 4 : 2];
};

template <int C>
__device__ __forceinline__ void mx_few_load(MxFewChunk<C> &f, const uint4 *codes, const unsigned char *scales, int chunk, int kb, int group)
{
    constexpr int G = 64 / C, U = 4 * G;
    const int first = chunk * U;
    if (first + U <= kb) {
#pragma unroll
        for (int s = 0; s < 4; ++s) f.codes[s] = *reinterpret_cast<const mx_v4i *>(codes + first + s * G + group);
#pragma unroll
        for (int w = 0; w < U / 4; ++w) f.scales[w] = reinterpret_cast<const mx_u32_any *>(scales + first)[w];
    } else {                                               // blocks from kb on are not read: zeros
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int u = first + s * G + group;
            f.codes[s] = mx_v4i{0, 0, 0, 0};
            if (u < kb) f.codes[s] = *reinterpret_cast<const mx_v4i *>(codes + u);
        }
#pragma unroll
        for (int w = 0; w < U / 4; ++w) {
            f.scales[w] = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (first + 4 * w + b < kb) f.scales[w] |= (unsigned)scales[first + 4 * w + b] << (8 * b);
        }
    }
}

// C rows by C columns; group: the lane's block of a step
template <int C, int S>
__device__ __forceinline__ auto mx_few_mfma(const MxFewChunk<C> &a, const MxFewChunk<C> &b, int group, decltype(mx_f32x4{}) acc)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(a.codes[S]), mx_operand(b.codes[S]), acc, 4, 4, 0, (int)(a.scales[S] >> (8 * group)),
                                                            0, (int)(b.scales[S] >> (8 * group)));
}
template <int C, int S>
__device__ __forceinline__ auto mx_few_mfma(const MxFewChunk<C> &a, const MxFewChunk<C> &b, int group, mx_f32x16 acc)
{
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(a.codes[S]), mx_operand(b.codes[S]), acc, 4, 4, 2 * (S & 1), (int)(a.scales[S / 2] >> (8 * group)),
                                                           2 * (S & 1), (int)(b.scales[S / 2] >> (8 * group)));
}

template <int C> struct MxFewAcc { typedef mx_f32x16 type; };
template <> struct MxFewAcc<16> { typedef mx_f32x4 type; };

template <int TYPE, int C, bool FUSED>
__global__ __launch_bounds__(MX_FEW_THREADS) void mx_product_few_kernel(MxProductArgs p, MxDense x)
{
    constexpr int G = 64 / C, U = 4 * G, E = C * C / 64, SUMS = MX_FEW_WAVES * C * C * 4;
    __shared__ __attribute__((aligned(16))) char lds[FUSED && MX_FEW_LDS > SUMS ? MX_FEW_LDS : SUMS];
    const int lane = threadIdx.x & 63, l = lane % C, group = lane / C;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int I = (int)p.I, J = (int)p.J, kb = (int)p.kb, chunks = (kb + U - 1) / U;
    const int j0 = blockIdx.x * C;
    const int64_t j = min(j0 + l, J - 1);
    const uint4 *b_codes = (const uint4 *)p.b_codes + j * p.b_ld;
    const unsigned char *b_scales = (const unsigned char *)p.b_scales + j * p.b_ld;
    MxFewChunk<C> b, b_next, a;
    if (wave < chunks) mx_few_load<C>(b, b_codes, b_scales, wave, kb, group);
    const int kbp = (kb + 15) / 16 * 16;
    const uint4 *a_codes;
    const unsigned char *a_scales;
    if constexpr (FUSED) {
        if (x.type == YL_F32) mx_few_round<YL_F32>(x, lds, kb, kbp);
        else if (x.type == YL_F16) mx_few_round<YL_F16>(x, lds, kb, kbp);
        else mx_few_round<YL_BF16>(x, lds, kb, kbp);
        __syncthreads();
        const int row = min(l, I - 1);
        a_codes = reinterpret_cast<const uint4 *>(lds) + row * (kbp + 1);
        a_scales = reinterpret_cast<const unsigned char *>(lds) + I * (kbp + 1) * 16 + row * kbp;
    } else {
        const int64_t row = min(l, I - 1);
        a_codes = (const uint4 *)p.a_codes + row * p.a_ld;
        a_scales = (const unsigned char *)p.a_scales + row * p.a_ld;
    }
    typename MxFewAcc<C>::type acc;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int c = wave; c < chunks; c += MX_FEW_WAVES) {
        if (c + MX_FEW_WAVES < chunks) mx_few_load<C>(b_next, b_codes, b_scales, c + MX_FEW_WAVES, kb, group);
        mx_few_load<C>(a, a_codes, a_scales, c, FUSED ? kbp : kb, group);      // LDS holds zeros up to kbp
        acc = mx_few_mfma<C, 0>(a, b, group, acc);
        acc = mx_few_mfma<C, 1>(a, b, group, acc);
        acc = mx_few_mfma<C, 2>(a, b, group, acc);
        acc = mx_few_mfma<C, 3>(a, b, group, acc);
        b = b_next;
    }
    float *sums = reinterpret_cast<float *>(lds);
    if constexpr (FUSED) __syncthreads();                  // every wave has read x
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int row = C == 16 ? 4 * group + e : 8 * (e / 4) + 4 * group + e % 4;
        sums[(wave * C + row) * C + l] = acc[e];
    }
    __syncthreads();
    for (int t = threadIdx.x; t < C * C; t += MX_FEW_THREADS) {
        const int i = t / C, jj = j0 + t % C;
        if (i >= I || jj >= J) continue;
        float v = sums[t];
#pragma unroll
        for (int w = 1; w < MX_FEW_WAVES; ++w) v += sums[w * C * C + t];
        if (p.bias) v += p.bias[jj];
        v = mx_activate<true>(v, p.act);
        if (p.residual) v += mx_load<TYPE>(p.residual, (int64_t)i * p.residual_stride + jj);
        mx_store<TYPE>(p.out, (int64_t)i * p.out_stride + jj, v);
    }
}

template <int C, bool FUSED>
static int launch_few(const MxProductArgs &a, const MxDense &x, hipStream_t s)
{
    const dim3 grid((unsigned)((a.J + C - 1) / C)), block(MX_FEW_THREADS);
    switch (a.type) {
    case YL_F32: return mx_launch(mx_product_few_kernel<YL_F32, C, FUSED>, grid, block, s, a, x);
    case YL_F16: return mx_launch(mx_product_few_kernel<YL_F16, C, FUSED>, grid, block, s, a, x);
    default: return mx_launch(mx_product_few_kernel<YL_BF16, C, FUSED>, grid, block, s, a, x);
    }
}

int launch_mx_few(const MxProductArgs &a, void *stream)
{
    hipStream_t s = (hipStream_t)stream;
    // 16 columns a workgroup where 32 would leave CUs without one (16 x 4096 x 4096 5.0 us against 6.5; 16 x 16384 x 4096 12.5 against
    // 10.6), and where the fused form, which has no other, would run: its sums are these
    if (a.I <= 16 && (a.J < 32 * (int64_t)device_cu_count() || mx_linear_fused(a.I, a.k))) return launch_few<16, false>(a, MxDense{}, s);
    return launch_few<32, false>(a, MxDense{}, s);
}

int launch_mx_linear(const MxProductArgs &a, const MxDense &x, void *stream)
{
    if (a.I == 0 || a.J == 0) return 0;
    return launch_few<16, true>(a, x, (hipStream_t)stream);
}

}  // namespace yl
