// mx_product.hip -- K15: products of MXFP4 matrices on v_mfma_scale_f32_32x32x64_f8f6f4 (yl_mx_matmul, yl_mx_linear, yl_mx_conv2d).
//
//   D[i][j] = sum over blocks b of Sa[i][b] Sb[j][b] sum_{t < 32} ca[i][32 b + t] cb[j][32 b + t], summed in FP32
//
// The instruction takes 64 summed elements: lanes 0-31 hold one block (16 bytes) of rows 0-31 of an operand, lanes 32-63 the next block
// of the same rows, each with its own scale byte -- exactly the format's block, so no code is ever unpacked.  Products of codes are
// exact; the sum is FP32.  D's layout: lane l holds column l & 31, rows 8 (e / 4) + 4 (l >> 5) + e % 4.
//
// MI355X: 8192^3 285 to 300 us, by card = 3.7 to 3.9 PFLOP/s, 4.7 on the slope from k = 8192 to 16384, where the ends of the tiles no longer count; a loop of nothing
// but these instructions makes 9.2, four times the BF16 rate of a large library product 4.8.  At 256 x 256 the instructions are half of a
// wave's cycles, a quarter are waits for panels out of L2 and at barriers.  One wave a tile with operands straight from memory, the
// first form: 3.72 ms.
#include <cstdio>

#include "activations.h"
#include "mx_device.h"
#include "mx.h"
#include "kernels.h"

namespace yl {

// ------------------------------------------------------------------ tiles staged through LDS
// A workgroup of four waves owns BI x BJ of D, a wave TI x TJ tiles of 32 x 32 of it.  The summed axis goes by panels of eight blocks (256
// values): the panel's codes lie in LDS as [row][8 units of 16 bytes], unit u at place u ^ (row / 2 & 7), so that one unit of sixteen
// neighbouring rows lies in all 64 banks once (u ^ (row & 7) puts rows r and r + 8 together: 580 cycles of conflicts a panel of 256 x 256); its scales as [row][8 bytes].  Lanes 0-31 feed the matrix instruction units
// 0-3, lanes 32-63 units 4-7: a row's four scales of a panel are then one word a lane, and the instruction picks the byte of the step.
// Two panels in LDS and one in registers: while the instructions of panel p run, panel p + 1 is written to the other half of LDS and
// panel p + 2 is requested from memory; operands of the next step are read one step ahead, across panels too, so the barrier of a panel
// falls in front of its last step's instructions.
constexpr int MX_PANEL = 8;        // blocks a panel
constexpr int MX_THREADS = 256;

// four scale bytes of the step-wise operands: byte S of each word
template <int S>
__device__ __forceinline__ mx_f32x16 mx_mfma(mx_v4i a, mx_v4i b, mx_f32x16 c, int sa, int sb)
{
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(a), mx_operand(b), c, 4, 4, S, sa, S, sb);
}

// A strip of D, 32 rows from ib by COLS columns from jb, in LDS: + bias, activation, + residual, to rows of memory.  WIDE: in 16-byte vectors,
// wherever they begin (3420 x 15311 x 149 to BF16: 51 us by single values, which the rare activations are left with, 36 to 41 so), the
// last of a row by its values; INSIDE: no column is behind a row's end; AHEAD rows' addends are requested before the first is used.
template <int TYPE, bool RARE, bool WIDE, bool INSIDE, int COLS, int PITCH>
__device__ __forceinline__ void mx_finish_rows(const MxProductArgs &p, const float *strip, int ib, int jb, int lane)
{
    constexpr int VEC = WIDE ? MX_VEC<TYPE> : 1;
    constexpr int LANES = COLS / VEC < 64 ? COLS / VEC : 64;   // lanes a row
    constexpr int ROWS = 64 / LANES, STEPS = 32 / ROWS, AHEAD = STEPS < 4 ? STEPS : 4;
    const int rows = min(32, (int)p.I - ib), act = p.act;
    const int64_t out_step = (int64_t)p.out_stride * ROWS, res_step = (int64_t)p.residual_stride * ROWS;
    const bool add = p.residual != nullptr;
    for (int c = lane % LANES * VEC; c < COLS; c += LANES * VEC) {
        const int j = jb + c;
        if (j >= (int)p.J) return;
        float bias[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) bias[q] = p.bias && (INSIDE || j + q < (int)p.J) ? p.bias[j + q] : 0.f;
        const int n = INSIDE ? VEC : min(VEC, (int)p.J - j);
        const int r0 = lane / LANES;
        if (r0 >= rows) return;                            // and below: the first row of a step is always one of the matrix
        int64_t at = (int64_t)(ib + r0) * p.out_stride + j, res = (int64_t)(ib + r0) * p.residual_stride + j;
#pragma unroll 1
        for (int step = 0; step < STEPS; step += AHEAD) {
            float v[AHEAD][VEC];
            mx_u32x4 rv[AHEAD];
            float rs[AHEAD];
            if (add) {
#pragma unroll
                for (int s = 0; s < AHEAD; ++s) {
                    const bool ok = r0 + (step + s) * ROWS < rows;
                    if constexpr (WIDE) {
                        if (n == VEC) rv[s] = mx_load_vec<TYPE>(p.residual, ok ? res + s * res_step : res);
                    } else rs[s] = mx_load<TYPE>(p.residual, ok ? res + s * res_step : res);
                }
            }
#pragma unroll
            for (int s = 0; s < AHEAD; ++s) {
                const float *from = strip + (r0 + (step + s) * ROWS) * PITCH + c;
                if constexpr (WIDE) {
#pragma unroll
                    for (int q = 0; q < VEC; q += 4) {
                        const mx_f32x4 x = *reinterpret_cast<const mx_f32x4 *>(from + q);
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[s][q + k] = x[k];
                    }
                } else v[s][0] = *from;
            }
#pragma unroll
            for (int s = 0; s < AHEAD; ++s) {
#pragma unroll
                for (int q = 0; q < VEC; ++q) v[s][q] = mx_activate<RARE>(v[s][q] + bias[q], act);
                if (WIDE && n < VEC) {
                    if (r0 + (step + s) * ROWS < rows) {
#pragma unroll
                        for (int q = 0; q < VEC; ++q)
                            if (q < n) mx_store<TYPE>(p.out, at + s * out_step + q, add ? v[s][q] + mx_load<TYPE>(p.residual, res + s * res_step + q) : v[s][q]);
                    }
                    continue;
                }
                if (add) {
                    float r[8];
                    if constexpr (WIDE) mx_unpack<TYPE>(rv[s], r);
                    else r[0] = rs[s];
#pragma unroll
                    for (int q = 0; q < VEC; ++q) v[s][q] += r[q];
                }
                if (r0 + (step + s) * ROWS < rows) {
                    if constexpr (WIDE) mx_store_vec<TYPE>(p.out, at + s * out_step, mx_pack<TYPE>(v[s]));
                    else mx_store<TYPE>(p.out, at + s * out_step, v[s][0]);
                }
            }
            at += AHEAD * out_step; res += AHEAD * res_step;
            if (r0 + (step + AHEAD) * ROWS >= rows) break;
        }
    }
}

// The 32 rows from ib of a position's result as one block of it.  y: this lane's 16 of them (rows 8 (e / 4) + 4 half + e % 4, zero where
// there is none), the others are in lane l ^ 32.
__device__ __forceinline__ void mx_side_block(const MxProductArgs &p, int64_t j, bool ok, int ib, int half, const float *y)
{
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = max(top, mx_abs_bits(y[e]));
    auto both = __builtin_amdgcn_permlane32_swap(top, top, false, false);      // {low half's, high half's} in every lane
    const unsigned byte = mx_scale_byte(max(both[0], both[1]));
    // four of a word's eight codes are this lane's: 16 bits each of the words 0-3
    unsigned h0 = 0, h1 = 0;
    if (byte != 255) { h0 = mx_codes8(y, byte); h1 = mx_codes8(y + 8, byte); }
    auto w0 = __builtin_amdgcn_permlane32_swap(h0, h0, false, false);
    auto w1 = __builtin_amdgcn_permlane32_swap(h1, h1, false, false);
    if (!ok || half != 0) return;
    const uint4 q = make_uint4((w0[0] & 0xffffu) | w0[1] << 16, w0[0] >> 16 | (w0[1] & 0xffff0000u),
                               (w1[0] & 0xffffu) | w1[1] << 16, w1[0] >> 16 | (w1[1] & 0xffff0000u));
    reinterpret_cast<uint4 *>(p.q_codes)[j * p.q_ld + ib / 32] = q;
    reinterpret_cast<unsigned char *>(p.q_scales)[j * p.q_ld + ib / 32] = (unsigned char)byte;
}

// A convolution's 32 x 32 tile of D from registers to planes of memory.  `at`: byte offset of (this lane's position, row 0 of the image's
// planes) in `out`; WHOLE: all 32 rows are filters.  This and the index arithmetic in front of the panels are most of a layer with few
// channels: the bias comes as four vectors, rows are offsets of the instruction (76 x 76 256 -> 128 1x1 of 8 images 16.4 -> 9.9 us, with the MXFP4 output alone 7.9).
template <bool RARE, bool WHOLE>
__device__ __forceinline__ void mx_finish_planes(const MxProductArgs &p, const mx_f32x16 &acc, int ib, int64_t j, bool ok, int half, __amdgpu_buffer_rsrc_t bias,
                                                 __amdgpu_buffer_rsrc_t out, __amdgpu_buffer_rsrc_t residual, int at)
{
    const int I = (int)p.I;
    const unsigned plane = (unsigned)p.OH * (unsigned)p.OW * 4u;      // bytes; a whole image's planes are below 2^32
    const int lane_off = ok ? (int)((unsigned)at + 4u * half * plane) : -1;
    auto off = [&](int e) { return WHOLE || ib + 8 * (e / 4) + e % 4 + 4 * half < I ? lane_off : -1; };
    auto row = [&](int e) { return (int)((ib + 8 * (e / 4) + e % 4) * plane); };
    float y[16], add[16];
    mx_u32x4 b[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) b[q] = __builtin_amdgcn_raw_buffer_load_b128(bias, (ib + 8 * q + 4 * half) * 4, 0, 0);   // zeros where there is none
    if (p.residual) {
#pragma unroll
        for (int e = 0; e < 16; ++e) add[e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(residual, off(e), row(e), 0));
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const unsigned w = b[e / 4][e % 4];
        y[e] = mx_activate<RARE>(acc[e] + __builtin_bit_cast(float, w), p.act);
        if (p.residual) y[e] += add[e];
    }
    if (p.out) {
#pragma unroll
        for (int e = 0; e < 16; ++e) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, y[e]), out, off(e), row(e), 0);
    }
    if (p.q_codes) {
        if (!WHOLE) {
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = ib + 8 * (e / 4) + e % 4 + 4 * half < I ? y[e] : 0.f;
        }
        mx_side_block(p, j, ok, ib, half, y);
    }
}

// n / d for 0 <= n < 2^31 by a multiplication: with l = ceil(log2 d), m = ceil(2^(31 + l) / d) fits 32 bits and n m / 2^(31 + l) is at most
// n / 2^(31 + l) < 1 / d above n / d
struct MxDiv {
    unsigned m = 0;
    int shift = 0, d = 1;
    MxDiv() = default;
    explicit MxDiv(int64_t by) : d((int)by)
    {
        if (by <= 1) return;
        int l = 0;
        while (((int64_t)1 << l) < by) ++l;
        m = (unsigned)((((uint64_t)1 << (31 + l)) + by - 1) / by);
        shift = l - 1;
    }
    __device__ __forceinline__ int operator()(int n) const { return d == 1 ? n : (int)(__umulhi((unsigned)n, m) >> shift); }
};

struct MxTileDev {
    MxProductArgs p;
    int tiles_i, tiles_j;
    MxDiv area, width, blocks;     // conv: positions of an image, positions of a line, blocks of a pixel
    int size_magic;                // conv: tap / size = tap * size_magic >> 8 for taps below 32
};

// logical tile of a workgroup: every XCD (blockIdx % 8) gets one contiguous run of tiles, walked in bands of 8 tiles along i so that the
// workgroups an XCD runs at a time share few rows of either operand in its L2
__device__ __forceinline__ void mx_tile_of(int bid, int nwg, int tiles_i, int tiles_j, int &ti, int &tj)
{
    const int q = nwg >> 3, r = nwg & 7, xcd = bid & 7;
    const int t = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (bid >> 3);
    const int band = t / (8 * tiles_j), in = t - band * 8 * tiles_j;
    const int high = min(8, tiles_i - band * 8);
    tj = in / high;
    ti = band * 8 + in - tj * high;
}

template <int TYPE, bool CONV, bool BYTES, bool RARE, int TI, int TJ>
__global__ __launch_bounds__(MX_THREADS, TI + TJ > 4 ? 1 : CONV && TI == TJ && !BYTES ? 3 : 6 - TI - TJ) void mx_product_tile_kernel(MxTileDev d)
{
    constexpr int BI = 64 * TI, BJ = 64 * TJ;
    constexpr int APT = BI / 32, BPT = BJ / 32, SPT = (BI + BJ + 127) / 128;
    constexpr int STAGE = (BI + BJ) * (MX_PANEL * 16 + MX_PANEL);
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
    const MxProductArgs &p = d.p;
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wi0 = (wave >> 1) * TI * 32, wj0 = (wave & 1) * TJ * 32;
    int tile_i, tile_j;
    mx_tile_of(blockIdx.x, gridDim.x, d.tiles_i, d.tiles_j, tile_i, tile_j);
    const int i0 = tile_i * BI, j0 = tile_j * BJ;
    const int I = (int)p.I, J = (int)p.J, kb = (int)p.kb;
    const int panels = (kb + MX_PANEL - 1) / MX_PANEL;

    // ---- what this thread brings: units (row t / 8 + 32 e, unit t % 8) and scale words (row t / 2 + 128 e, word t % 2)
    const int unit = tid & 7, word = tid & 1;
    auto resource = [](const void *base, int64_t off, int64_t bytes) {
        const int64_t n = bytes > 0xFFFFFFFELL ? 0xFFFFFFFELL : bytes < 0 ? 0 : bytes;
        return __builtin_amdgcn_make_buffer_rsrc((void *)((const char *)base + off), 0, (int)(unsigned)n, 0x00020000);
    };
    const int64_t a_row0 = i0, a_rows = p.I - i0;
    int64_t b_row0 = j0, b_rows = p.J - j0;            // the row that offset 0 of B's descriptors means, and rows from it to the end
    int cj_image = 0, cj_y = 0;                        // conv: image and first input line of the tile's first position
    if (CONV) {
        cj_image = d.area(j0);
        cj_y = d.width(j0 - cj_image * d.area.d) * p.stride;
        b_row0 = ((int64_t)cj_image * p.H + min(cj_y, p.H - 1)) * p.W - (int64_t)p.pad * p.W - p.pad;
        cj_y = min(cj_y, p.H - 1);
        b_rows = (int64_t)p.batch * p.H * p.W - b_row0;
    }
    const __amdgpu_buffer_rsrc_t ra = resource(p.a_codes, a_row0 * p.a_ld * 16, a_rows * p.a_ld * 16);
    const __amdgpu_buffer_rsrc_t ras = resource(p.a_scales, a_row0 * p.a_ld, a_rows * p.a_ld);
    const __amdgpu_buffer_rsrc_t rb = resource(p.b_codes, b_row0 * p.b_ld * 16, b_rows * p.b_ld * 16);
    const __amdgpu_buffer_rsrc_t rbs = resource(p.b_scales, b_row0 * p.b_ld, b_rows * p.b_ld);
    const int a_ld = (int)p.a_ld, b_ld = (int)p.b_ld;

    // row (relative to the descriptors) and, for a convolution, the taps outside the image (bit t = tap t) of tile row j
    auto b_row = [&](int jl, unsigned &outside) {
        const int j = min(j0 + jl, J - 1);
        outside = 0;
        if (!CONV) return j - j0;
        const int image = d.area(j), pix = j - image * d.area.d, oy = d.width(pix), ox = pix - oy * p.OW;
        const int y = oy * p.stride - p.pad, x = ox * p.stride - p.pad;
        if (p.size == 1) return ((image - cj_image) * p.H + y - cj_y) * p.W + x;      // pad < size: no tap is outside
        // columns of the filter from -x to W - x are inside, lines likewise
        const unsigned columns = ((1u << min(max(p.W - x, 0), p.size)) - 1u) & (~0u << max(-x, 0));
        unsigned in = 0;
        for (int ky = 0; ky < p.size; ++ky)
            if ((unsigned)(y + ky) < (unsigned)p.H) in |= columns << (ky * p.size);
        outside = ~in;
        return ((image - cj_image) * p.H + y + p.pad - cj_y) * p.W + x + p.pad;
    };
    int aoff[APT], boff[BPT], soff[SPT];
    unsigned bout[BPT], sout[SPT];
#pragma unroll
    for (int e = 0; e < APT; ++e) aoff[e] = (int)((unsigned)min(tid / 8 + 32 * e, I - 1 - i0) * (unsigned)a_ld * 16u) + unit * 16;
#pragma unroll
    for (int e = 0; e < BPT; ++e) boff[e] = (int)((unsigned)b_row(tid / 8 + 32 * e, bout[e]) * (unsigned)b_ld * 16u) + (CONV ? 0 : unit * 16);
#pragma unroll
    for (int e = 0; e < SPT; ++e) {
        const int row = tid / 2 + 128 * e;
        sout[e] = 0;
        if (32 * wave + 128 * e < BI) soff[e] = min(row, I - 1 - i0) * a_ld;
        else soff[e] = (int)((unsigned)b_row(min(row - BI, BJ - 1), sout[e]) * (unsigned)b_ld);
    }
    const int code_at = (tid / 8) * 128 + ((unit ^ ((tid / 16) & 7)) * 16);

    // ---- a convolution's blocks in the order (tap, channel block): of this thread's unit, stepped by a panel at a time
    auto tap_of = [&](int block) { return d.blocks(block); };
    int tap = 0, g = 0, step_tap = 0, step_g = 0;
    if (CONV) {
        tap = tap_of(unit); g = unit - tap * p.G;
        step_tap = tap_of(MX_PANEL); step_g = MX_PANEL - step_tap * p.G;
    }
    auto tap_row = [&](int t) {                        // tap -> rows of the map from the first tap
        const int ky = t * d.size_magic >> 8;
        return ky * p.W + t - ky * p.size;
    };
    auto outside_bit = [](unsigned m, int t) { return __builtin_amdgcn_sbfe((int)m, t, 1); };

    // the panel's ITEMS requests and, in the same order, the stores of what they brought: one or two between two matrix instructions
    constexpr int ITEMS = APT + BPT + SPT;
    constexpr int SETS = TI + TJ > 4 || TI != TJ || BYTES ? 1 : 2;          // panels in registers: small tiles are over too soon for one to hide memory
    mx_v4i areg[SETS][APT], breg[SETS][BPT];
    int sreg[SETS][SPT][BYTES ? 4 : 1];
    int here = 0, here_out[BPT];                       // conv: this thread's unit of the panel being requested, rows outside the image as -1
    auto begin_load = [&](int pn) {                    // the panels in order, each once
        const int end = pn * MX_PANEL + unit >= kb ? -1 : 0;
        here = end;
        if (CONV) {
            here = tap_row(tap) * b_ld * 16 + g * 16;
#pragma unroll
            for (int e = 0; e < BPT; ++e) here_out[e] = outside_bit(bout[e], tap) | end;
            tap += step_tap; g += step_g;
            if (g >= p.G) { g -= p.G; ++tap; }
        }
    };
    auto load = [&](int pn, int set, int k) {
        const int at = pn * MX_PANEL * 16, end = pn * MX_PANEL + unit >= kb ? -1 : 0;
        if (k < APT) areg[set][k] = __builtin_bit_cast(mx_v4i, __builtin_amdgcn_raw_buffer_load_b128(ra, aoff[k] | end, at, 0));
        else if (k < APT + BPT) {
            const int e = k - APT;
            breg[set][e] = __builtin_bit_cast(mx_v4i, CONV ? __builtin_amdgcn_raw_buffer_load_b128(rb, (boff[e] + here) | here_out[e], 0, 0)
                                                      : __builtin_amdgcn_raw_buffer_load_b128(rb, boff[e] | end, at, 0));
        } else {
            const int e = k - APT - BPT, block0 = pn * MX_PANEL + 4 * word;            // the word's first block
            const bool of_a = 32 * wave + 128 * e < BI;                                // a wave brings 32 rows' words
            // the word, or its bytes one by one
#pragma unroll
            for (int i = 0; i < (BYTES ? 4 : 1); ++i) {
                const int block = block0 + i, off_end = block >= kb ? -1 : 0;
                int off = (soff[e] + block) | off_end;
                if (CONV && !of_a) {
                    const int t = tap_of(block);
                    off = (soff[e] + tap_row(t) * b_ld + block - t * p.G) | outside_bit(sout[e], min(t, 31)) | off_end;
                }
                if constexpr (BYTES) sreg[set][e][i] = of_a ? __builtin_amdgcn_raw_buffer_load_b8(ras, off, 0, 0) : __builtin_amdgcn_raw_buffer_load_b8(rbs, off, 0, 0);
                else sreg[set][e][i] = of_a ? __builtin_amdgcn_raw_buffer_load_b32(ras, off, 0, 0) : __builtin_amdgcn_raw_buffer_load_b32(rbs, off, 0, 0);
            }
        }
    };
    auto store = [&](int pn, int set, int k) {                  // registers -> the panel's half of LDS
        char *st = smem + (pn & 1) * STAGE;
        if (k < APT) *reinterpret_cast<mx_v4i *>(st + code_at + k * 4096) = areg[set][k];
        else if (k < APT + BPT) *reinterpret_cast<mx_v4i *>(st + BI * 128 + code_at + (k - APT) * 4096) = breg[set][k - APT];
        else {
            const int e = k - APT - BPT, left = kb - (pn * MX_PANEL + 4 * word);
            const unsigned keep = left >= 4 ? 0xFFFFFFFFu : (left <= 0 ? 0u : (1u << (8 * left)) - 1u);     // scales behind the last block are not read
            unsigned w = (unsigned)sreg[set][e][0];
            if constexpr (BYTES) w = (w & 255u) | ((unsigned)sreg[set][e][1] & 255u) << 8 | ((unsigned)sreg[set][e][2] & 255u) << 16 | ((unsigned)sreg[set][e][3] & 255u) << 24;
            if ((BI + BJ) % 128 == 0 || tid + 256 * e < 2 * (BI + BJ)) *reinterpret_cast<unsigned *>(st + (BI + BJ) * 128 + (tid + 256 * e) * 4) = w & keep;
        }
    };

    mx_f32x16 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    const int ar = (wi0 + l31) * 128, br = BI * 128 + (wj0 + l31) * 128, x7 = (l31 >> 1) & 7;
    mx_v4i af[2][TI], bf[2][TJ];
    int sa[TI], sb[TJ], sa_next[TI], sb_next[TJ];
    constexpr int READS = TI + TJ;
    auto fetch = [&](int pn, int s, int into, int k) { // operands of step s of panel pn
        const char *st = smem + (pn & 1) * STAGE;
        const int at = ((4 * half + s) ^ x7) * 16;
        if (k < TI) af[into][k] = *reinterpret_cast<const mx_v4i *>(st + ar + at + k * 4096);
        else bf[into][k - TI] = *reinterpret_cast<const mx_v4i *>(st + br + at + (k - TI) * 4096);
    };
    auto fetch_scale = [&](int pn, int k) {
        const char *st = smem + (pn & 1) * STAGE + (BI + BJ) * 128;
        if (k < TI) sa_next[k] = *reinterpret_cast<const int *>(st + (wi0 + k * 32 + l31) * 8 + half * 4);
        else sb_next[k - TI] = *reinterpret_cast<const int *>(st + (BI + wj0 + (k - TI) * 32 + l31) * 8 + half * 4);
    };
    auto take_scales = [&]() {
#pragma unroll
        for (int i = 0; i < TI; ++i) sa[i] = sa_next[i];
#pragma unroll
        for (int j = 0; j < TJ; ++j) sb[j] = sb_next[j];
    };
    // step S of a panel: its matrix instructions, and between them the N calls of `other`, spread over the first WITHIN of them
    auto spread = [](int m, int n, int within) { return m >= within ? n : m * n / within; };
#define MX_STEP(S, CUR, N, WITHIN, OTHER)                                                                                        \
    _Pragma("unroll") for (int m = 0; m < TI * TJ; ++m) {                                                                        \
        acc[m / TJ][m % TJ] = mx_mfma<S>(af[CUR][m / TJ], bf[CUR][m % TJ], acc[m / TJ][m % TJ], sa[m / TJ], sb[m % TJ]);         \
        _Pragma("unroll") for (int k = spread(m, N, WITHIN); k < spread(m + 1, N, WITHIN); ++k) { OTHER }                        \
        __builtin_amdgcn_sched_barrier(0);                                                                                       \
    }

    constexpr int MM = TI * TJ, HALF = ITEMS / 2, EARLY = MM / 2 > 0 ? MM / 2 : 1;
    if (panels == 1) {                                     // nothing to overlap
        begin_load(0);
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) load(0, 0, k);
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) store(0, 0, k);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < READS; ++k) { fetch_scale(0, k); fetch(0, 0, 0, k); }
        take_scales();
        MX_STEP(0, 0, READS, EARLY, fetch(0, 1, 1, k);)
        MX_STEP(1, 1, READS, EARLY, fetch(0, 2, 0, k);)
        MX_STEP(2, 0, READS, EARLY, fetch(0, 3, 1, k);)
        MX_STEP(3, 1, 0, EARLY, )
    } else if (panels > 1) {
        begin_load(0);
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) load(0, 0, k);
#pragma unroll
        for (int set = 1; set < SETS; ++set) {
            begin_load(set);
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) load(set, set, k);
        }
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) store(0, 0, k);
        begin_load(SETS);
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) load(SETS, 0, k);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < READS; ++k) { fetch(0, 0, 0, k); fetch_scale(0, k); }
        take_scales();
        // Panel PN while panel PN + 1 lies in set SET of the registers: it is stored, and panel PN + 1 + SETS requested in its place.  Panels
        // behind the last one read as zeros and nothing of memory (every offset is out of its descriptor's range), so the loop needs no
        // case for its end.
#define MX_PANEL_BODY(PN, SET)                                                                                                   \
    {                                                                                                                            \
        MX_STEP(0, 0, READS, EARLY, fetch(PN, 1, 1, k);)                                                                         \
        begin_load((PN) + 1 + SETS);                                                                                             \
        MX_STEP(1, 1, READS + HALF, MM,                                                                                          \
                if (k < READS) fetch(PN, 2, 0, k); else { store((PN) + 1, SET, k - READS); load((PN) + 1 + SETS, SET, k - READS); }) \
        MX_STEP(2, 0, READS + ITEMS - HALF, MM,                                                                                  \
                if (k < READS) fetch(PN, 3, 1, k);                                                                               \
                else { store((PN) + 1, SET, k - READS + HALF); load((PN) + 1 + SETS, SET, k - READS + HALF); })                  \
        __syncthreads();                                                                                                         \
        MX_STEP(3, 1, 2 * READS, EARLY, if (k < READS) fetch_scale((PN) + 1, k); else fetch((PN) + 1, 0, 0, k - READS);)         \
        take_scales();                                                                                                           \
    }
        if constexpr (SETS == 1) {
            for (int pn = 0; pn < panels; ++pn) MX_PANEL_BODY(pn, 0)
        } else {
            int pn = 0;
            for (; pn + 1 < panels; pn += 2) {
                MX_PANEL_BODY(pn, 1)
                MX_PANEL_BODY(pn + 1, 0)
            }
            if (pn < panels) MX_PANEL_BODY(pn, 1)
        }
#undef MX_PANEL_BODY
    }
#undef MX_STEP

    if constexpr (CONV) {
        // ---- epilogue in D's layout: neighbouring lanes hold neighbouring positions of a plane
        const int area = d.area.d, image0 = d.area(j0 + wj0);
        const int64_t planes = (int64_t)I * area * 4;
        const __amdgpu_buffer_rsrc_t out = resource(p.out ? p.out : p.a_codes, p.out ? image0 * planes : 0, p.out ? (p.batch - image0) * planes : 0);
        const __amdgpu_buffer_rsrc_t bias = resource(p.bias ? (const void *)p.bias : p.a_codes, 0, p.bias ? (int64_t)I * 4 : 0);
        const __amdgpu_buffer_rsrc_t residual = resource(p.residual ? p.residual : p.a_codes, p.residual ? image0 * planes : 0, p.residual ? (p.batch - image0) * planes : 0);
#pragma unroll
        for (int tj = 0; tj < TJ; ++tj) {
            const int j = j0 + wj0 + tj * 32 + l31, image = d.area(j);
            const int at = (int)((unsigned)(image - image0) * (unsigned)planes + (unsigned)(j - image * area) * 4u);
#pragma unroll
            for (int ti = 0; ti < TI; ++ti) {
                const int ib = i0 + wi0 + ti * 32;
                if (ib + 32 <= I) mx_finish_planes<RARE, true>(p, acc[ti][tj], ib, j, j < J, half, bias, out, residual, at);
                else if (ib < I) mx_finish_planes<RARE, false>(p, acc[ti][tj], ib, j, j < J, half, bias, out, residual, at);
                __builtin_amdgcn_sched_barrier(0);         // one tile's addresses and addends at a time
            }
        }
    } else {
        // ---- epilogue: strips of 32 rows go through the wave's own part of LDS, so that the result leaves in whole vectors along its rows
        constexpr int COLS = TJ * 32, PITCH = COLS + 8;              // rows r and r + 4, written at once, are half the banks apart
        static_assert(4 * 32 * PITCH * 4 <= 2 * STAGE, "strips fit in the panels' LDS");
        __syncthreads();
        float *strip = reinterpret_cast<float *>(smem) + wave * 32 * PITCH;
        // A strip passes between the lanes of its wave alone.  The wave's LDS operations end in the order they were issued in; that the
        // compiler issues a lane's reads behind the other lanes' stores, and the next strip's stores behind the reads, is said here.
        auto wave_order = [] {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        };
#pragma unroll 1
        for (int t = 0; t < TI; ++t) {
#pragma unroll
            for (int ti = 0; ti < TI; ++ti)
                if (t == ti) {
#pragma unroll
                    for (int tj = 0; tj < TJ; ++tj)
#pragma unroll
                        for (int e = 0; e < 16; ++e) strip[(8 * (e / 4) + 4 * half + e % 4) * PITCH + tj * 32 + l31] = acc[ti][tj][e];
                }
            wave_order();
            const int ib = i0 + wi0 + t * 32;
            if (ib < I && j0 + wj0 + COLS <= J) mx_finish_rows<TYPE, RARE, !RARE, true, COLS, PITCH>(p, strip, ib, j0 + wj0, lane);
            else if (ib < I) mx_finish_rows<TYPE, RARE, !RARE, false, COLS, PITCH>(p, strip, ib, j0 + wj0, lane);
            wave_order();
        }
    }
}

template <int TYPE, bool CONV, bool BYTES, bool RARE, int TI, int TJ>
static int launch_tile(const MxProductArgs &a, hipStream_t s)
{
    MxTileDev d{a, (int)((a.I + 64 * TI - 1) / (64 * TI)), (int)((a.J + 64 * TJ - 1) / (64 * TJ)), MxDiv(), MxDiv(), MxDiv(), 0};
    if (CONV) {
        d.area = MxDiv((int64_t)a.OH * a.OW);
        d.width = MxDiv(a.OW);
        d.blocks = MxDiv(a.G);
        d.size_magic = (256 + a.size - 1) / a.size;
    }
    const int64_t grid = (int64_t)d.tiles_i * d.tiles_j;
    if (grid > 0x7fffffffLL) return (int)hipErrorInvalidValue;
    return mx_launch(mx_product_tile_kernel<TYPE, CONV, BYTES, RARE, TI, TJ>, dim3((unsigned)grid), dim3(MX_THREADS), s, d);
}

// The tile, measured on MI355X (GPU time, both sides of each border):
//   (BF16, replayed from a graph; both sides of a border from one build of this source with the tile forced, in turn)
//   rows    256 x 256 from k = 2048 on where it gives every CU a workgroup: 4096 x 16384 x 4096 171 us against 206 with 128 x 128 tiles,
//           4096 x 4096 x 2048 31.2 against 33.5, but 4096 x 4096 x 1024 24.3 against 22.9 (one workgroup a CU hides neither end of a tile behind another)
//           128 x 128 where it gives every CU two workgroups, or one from k = 2048 on: 512 x 8192 x 8192 29.6 us against 38.7 with 64 x 128
//           tiles, 2048 x 4096 x 512 11.5 against 12.3, but 1024 x 4096 x 512 8.2 against 7.8
//           64 x 128 where it gives every CU one (512 x 4096 x 4096 13.2 us against 14.7 with 128 x 128 and 13.5 with 64 x 64)
//           else 64 x 64 (1024^3 5.5 us against 6.8 with 64 x 128, 256 x 4096 x 4096 9.1 against 12.7)
//   planes  64 x 128 where it gives every CU two workgroups, else 64 x 64: bound by the map's and the result's bytes and by the latency of
//           gathering, they want waves (76 x 76 128 -> 256 3x3 of 64 images: 190 us against 230 with 64 x 64, 240 with 128 x 128 and 1350 with
//           256 x 256; 19 x 19 512 -> 1024 3x3 of 8 images 22.4 us with 64 x 64, 24.3 with 64 x 128; of 16 images 39.5 and 33.9)
//   The activations other than LINEAR, LEAKY and RELU have 64 x 64 tiles and single stores only: 4096 x 16384 x 4096 with LOGISTIC 369 us,
//   512 x 4096 x 4096 19.2, 3420 x 15311 x 149 123 (36 without).
template <int TYPE, bool CONV, bool BYTES>
static int launch_by_size(const MxProductArgs &a, hipStream_t s, char *name, size_t name_len)
{
    auto grid = [&](int64_t ti, int64_t tj) { return (a.I + 64 * ti - 1) / (64 * ti) * ((a.J + 64 * tj - 1) / (64 * tj)); };
    const int64_t cus = device_cu_count();
    const bool rare = mx_rare(a.act);
    int t = 11;
    if (!rare) {
        if (CONV) t = grid(1, 2) >= 2 * cus ? 12 : 11;
        else if (grid(4, 4) >= cus && a.kb >= 64) t = 44;
        else if (grid(2, 2) >= (a.kb >= 64 ? cus : 2 * cus)) t = 22;
        else if (grid(1, 2) >= cus) t = 12;
    }
    if (name) snprintf(name, name_len, "mx_product<%dx%d>", t / 10 * 64, t % 10 * 64);
    if (rare) return launch_tile<TYPE, CONV, BYTES, true, 1, 1>(a, s);
    if constexpr (!CONV) {
        if (t == 44) return launch_tile<TYPE, CONV, BYTES, false, 4, 4>(a, s);
        if (t == 22) return launch_tile<TYPE, CONV, BYTES, false, 2, 2>(a, s);
    }
    if (t == 12) return launch_tile<TYPE, CONV, BYTES, false, 1, 2>(a, s);
    return launch_tile<TYPE, CONV, BYTES, false, 1, 1>(a, s);
}

template <int TYPE, bool CONV>
static int launch_typed(const MxProductArgs &a, hipStream_t s, char *name, size_t name_len)
{
    // scales go by words of four where every row's begin on one: else by bytes
    const bool words = a.a_ld % 4 == 0 && a.b_ld % 4 == 0 && (uintptr_t)a.a_scales % 4 == 0 && (uintptr_t)a.b_scales % 4 == 0 && (!CONV || a.G % 4 == 0);
    return words ? launch_by_size<TYPE, CONV, false>(a, s, name, name_len) : launch_by_size<TYPE, CONV, true>(a, s, name, name_len);
}

int launch_mx_product(const MxProductArgs &a, void *stream, char *name, size_t name_len)
{
    if (a.I == 0 || a.J == 0) return 0;
    hipStream_t s = (hipStream_t)stream;
    if (a.conv) return launch_typed<YL_F32, true>(a, s, name, name_len);
    if (mx_few_takes(a.I)) return launch_mx_few(a, stream);
    switch (a.type) {
    case YL_F32: return launch_typed<YL_F32, false>(a, s, name, name_len);
    case YL_F16: return launch_typed<YL_F16, false>(a, s, name, name_len);
    default: return launch_typed<YL_BF16, false>(a, s, name, name_len);
    }
}

}  // namespace yl
