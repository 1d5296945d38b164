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
#include "kernels.h"

namespace yl {

// ------------------------------------------------------------------ tiles staged through LDS
// A workgroup of four waves owns BI x BJ of D, a wave TI x TJ tiles of 32 x 32 of it.  The summed axis goes by panels of eight blocks (256
// values): the panel's codes lie in LDS as [row][8 units of 16 bytes], unit u at place u ^ (row & 7), so the eight rows that a read
// of one unit touches per cycle fall into different banks; its scales as [row][8 bytes].  Lanes 0-31 feed the matrix instruction units
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

// A strip of D, 32 rows from ib by COLS columns from jb, in LDS: + bias, activation, + residual, to rows of memory.  A lane takes four
// neighbouring columns.
template <int TYPE, int COLS, int PITCH>
__device__ __forceinline__ void mx_finish_rows(const MxProductArgs &p, const float *strip, int ib, int jb, int lane)
{
    constexpr int LANES = COLS / 4, ROWS = 64 / LANES;     // lanes a row, rows a step
    const int c = lane % LANES * 4, j = jb + c, J = (int)p.J;
    const int rows = min(32, (int)p.I - ib);
    const int n = min(4, J - j);
    if (n <= 0) return;
    constexpr int BYTES = TYPE == YL_F32 ? 4 : 2;
    // four values at once where every row's begin on a whole vector
    const bool wide = n == 4 && p.out_stride % 4 == 0 && (uintptr_t)p.out % (4 * BYTES) == 0 &&
                      (!p.residual || (p.residual_stride % 4 == 0 && (uintptr_t)p.residual % (4 * BYTES) == 0));
    float bias[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.bias)
        for (int q = 0; q < 4; ++q) bias[q] = q < n ? p.bias[j + q] : 0.f;
    for (int r = lane / LANES; r < rows; r += ROWS) {
        const mx_f32x4 s = *reinterpret_cast<const mx_f32x4 *>(strip + r * PITCH + c);
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = s[q] + bias[q];
        if (p.act != YL_LINEAR) {
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {                  // one copy of the activations' code
                const float y = yl_act_epilogue(q == 0 ? v[0] : q == 1 ? v[1] : q == 2 ? v[2] : v[3], p.act);
                v[0] = q == 0 ? y : v[0]; v[1] = q == 1 ? y : v[1]; v[2] = q == 2 ? y : v[2]; v[3] = q == 3 ? y : v[3];
            }
        }
        const int64_t at = (int64_t)(ib + r) * p.out_stride + j, res = (int64_t)(ib + r) * p.residual_stride + j;
        if (wide) {
            if (p.residual) mx_add4<TYPE>(p.residual, res, v);
            mx_store4<TYPE>(p.out, at, v);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (q < n) {
                    if (p.residual) v[q] += mx_load<TYPE>(p.residual, res + q);
                    mx_store<TYPE>(p.out, at + q, v[q]);
                }
        }
    }
}

// The same for a convolution: rows are filters, columns positions; memory is planes of float, a lane takes a column.  With a side
// output the strip's rows are one block of every column's result.
template <int COLS, int PITCH>
__device__ __forceinline__ void mx_finish_planes(const MxProductArgs &p, float *strip, int ib, int jb, int lane)
{
    const int rows = min(32, (int)p.I - ib), area = p.OH * p.OW;
    for (int c = lane; c < COLS; c += 64) {
        const int j = jb + c;
        if (j >= (int)p.J) continue;
        const int image = j / area;
        int64_t at = ((int64_t)image * p.I + ib) * area + (j - image * area);
        const float *residual = reinterpret_cast<const float *>(p.residual);
        float *out = reinterpret_cast<float *>(p.out);
        unsigned top = 0;
#pragma unroll 4
        for (int r = 0; r < rows; ++r, at += area) {
            float v = strip[r * PITCH + c];
            if (p.bias) v += p.bias[ib + r];
            v = yl_act_epilogue(v, p.act);
            if (residual) v += residual[at];
            if (out) out[at] = v;
            if (p.q_codes) strip[r * PITCH + c] = v;
            top = max(top, mx_abs_bits(v));
        }
        if (!p.q_codes) continue;
        const unsigned byte = mx_scale_byte(top);
        unsigned w[4] = {0, 0, 0, 0};
        if (byte != 255) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float v[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = 8 * g + q < rows ? strip[(8 * g + q) * PITCH + c] : 0.f;
                w[g] = mx_codes8(v, byte);
            }
        }
        reinterpret_cast<uint4 *>(p.q_codes)[j * p.q_ld + ib / 32] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<unsigned char *>(p.q_scales)[j * p.q_ld + ib / 32] = (unsigned char)byte;
    }
}

struct MxTileDev {
    MxProductArgs p;
    int tiles_i, tiles_j;
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

template <int TYPE, bool CONV, bool BYTES, int TI, int TJ>
__global__ __launch_bounds__(MX_THREADS, TI * TJ > 4 ? 1 : 2) void mx_product_tile_kernel(MxTileDev d)
{
    constexpr int BI = 64 * TI, BJ = 64 * TJ;
    constexpr int APT = BI / 32, BPT = BJ / 32, SPT = (BI + BJ) / 128;
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
        const int64_t n = bytes > 0xFFFFFFFELL ? 0xFFFFFFFELL : bytes;
        return __builtin_amdgcn_make_buffer_rsrc((void *)((const char *)base + off), 0, (int)(unsigned)n, 0x00020000);
    };
    const int64_t a_row0 = i0, a_rows = p.I - i0;
    int64_t b_row0 = j0, b_rows = p.J - j0;            // the row that offset 0 of B's descriptors means, and rows from it to the end
    int cj_image = 0, cj_y = 0;                        // conv: image and first input line of the tile's first position
    if (CONV) {
        const int area = p.OH * p.OW;
        cj_image = j0 / area;
        cj_y = (j0 - cj_image * area) / p.OW * p.stride;
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
        const int area = p.OH * p.OW, image = j / area, pix = j - image * area, oy = pix / p.OW, ox = pix - oy * p.OW;
        const int y = oy * p.stride - p.pad, x = ox * p.stride - p.pad;
        unsigned in = 0;
        for (int ky = 0; ky < p.size; ++ky)
            for (int kx = 0; kx < p.size; ++kx)
                if (y + ky >= 0 && y + ky < p.H && x + kx >= 0 && x + kx < p.W) in |= 1u << (ky * p.size + kx);
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
        if (row < BI) soff[e] = min(row, I - 1 - i0) * a_ld;
        else soff[e] = (int)((unsigned)b_row(row - BI, sout[e]) * (unsigned)b_ld);
    }
    const int code_at = (tid / 8) * 128 + ((unit ^ ((tid / 8) & 7)) * 16);

    // ---- a convolution's blocks in the order (tap, channel block): of this thread's unit, stepped by a panel at a time
    int tap = 0, g = 0, step_tap = 0, step_g = 0;
    if (CONV) {
        tap = unit / p.G; g = unit - tap * p.G;
        step_tap = MX_PANEL / p.G; step_g = MX_PANEL - step_tap * p.G;
    }
    auto tap_row = [&](int t) {                        // tap -> rows of the map from the first tap
        const int ky = p.size == 3 ? (t * 11) >> 5 : (p.size == 1 ? 0 : t / p.size);
        return ky * p.W + t - ky * p.size;
    };
    auto outside_bit = [](unsigned m, int t) { return __builtin_amdgcn_sbfe((int)m, t, 1); };

    mx_v4i areg[APT], breg[BPT];
    int sreg[SPT][BYTES ? 4 : 1];
    auto load = [&](int pn) {                          // request panel pn (the panels in order, each once)
        const int end = pn * MX_PANEL + unit >= kb ? -1 : 0;
        const int at = pn * MX_PANEL * 16;
#pragma unroll
        for (int e = 0; e < APT; ++e) areg[e] = __builtin_bit_cast(mx_v4i, __builtin_amdgcn_raw_buffer_load_b128(ra, aoff[e] | end, at, 0));
        if (CONV) {
            const int here = tap_row(tap) * b_ld * 16 + g * 16;
#pragma unroll
            for (int e = 0; e < BPT; ++e)
                breg[e] = __builtin_bit_cast(mx_v4i, __builtin_amdgcn_raw_buffer_load_b128(rb, (boff[e] + here) | outside_bit(bout[e], tap) | end, 0, 0));
            tap += step_tap; g += step_g;
            if (g >= p.G) { g -= p.G; ++tap; }
        } else {
#pragma unroll
            for (int e = 0; e < BPT; ++e) breg[e] = __builtin_bit_cast(mx_v4i, __builtin_amdgcn_raw_buffer_load_b128(rb, boff[e] | end, at, 0));
        }
        const int block0 = pn * MX_PANEL + 4 * word;   // the word's first block
#pragma unroll
        for (int e = 0; e < SPT; ++e) {
            const bool of_a = BI % 128 == 0 ? 128 * e < BI : tid / 2 + 128 * e < BI;
            if constexpr (BYTES) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int block = block0 + i, off_end = block >= kb ? -1 : 0;
                    if (of_a) sreg[e][i] = __builtin_amdgcn_raw_buffer_load_b8(ras, (soff[e] + block) | off_end, 0, 0);
                    else if (CONV) {
                        const int t = block / p.G;
                        sreg[e][i] = __builtin_amdgcn_raw_buffer_load_b8(rbs, (soff[e] + tap_row(t) * b_ld + block - t * p.G) | outside_bit(sout[e], min(t, 31)) | off_end, 0, 0);
                    } else sreg[e][i] = __builtin_amdgcn_raw_buffer_load_b8(rbs, (soff[e] + block) | off_end, 0, 0);
                }
            } else {
                const int off_end = block0 >= kb ? -1 : 0;
                if (of_a) sreg[e][0] = __builtin_amdgcn_raw_buffer_load_b32(ras, (soff[e] + block0) | off_end, 0, 0);
                else if (CONV) {
                    const int t = block0 / p.G;
                    sreg[e][0] = __builtin_amdgcn_raw_buffer_load_b32(rbs, (soff[e] + tap_row(t) * b_ld + block0 - t * p.G) | outside_bit(sout[e], min(t, 31)) | off_end, 0, 0);
                } else sreg[e][0] = __builtin_amdgcn_raw_buffer_load_b32(rbs, (soff[e] + block0) | off_end, 0, 0);
            }
        }
    };
    auto store = [&](int pn) {                         // panel pn: registers -> its half of LDS
        char *st = smem + (pn & 1) * STAGE;
#pragma unroll
        for (int e = 0; e < APT; ++e) *reinterpret_cast<mx_v4i *>(st + code_at + e * 4096) = areg[e];
#pragma unroll
        for (int e = 0; e < BPT; ++e) *reinterpret_cast<mx_v4i *>(st + BI * 128 + code_at + e * 4096) = breg[e];
        const int left = kb - (pn * MX_PANEL + 4 * word);
        const unsigned keep = left >= 4 ? 0xFFFFFFFFu : (left <= 0 ? 0u : (1u << (8 * left)) - 1u);     // scales behind the last block are not read
#pragma unroll
        for (int e = 0; e < SPT; ++e) {
            unsigned w = (unsigned)sreg[e][0];
            if constexpr (BYTES) w = (w & 255u) | ((unsigned)sreg[e][1] & 255u) << 8 | ((unsigned)sreg[e][2] & 255u) << 16 | ((unsigned)sreg[e][3] & 255u) << 24;
            *reinterpret_cast<unsigned *>(st + (BI + BJ) * 128 + (tid + 256 * e) * 4) = w & keep;
        }
    };

    mx_f32x16 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    const int ar = (wi0 + l31) * 128, br = BI * 128 + (wj0 + l31) * 128, x7 = l31 & 7;
    mx_v4i af[2][TI], bf[2][TJ];
    int sa[TI], sb[TJ], sa_next[TI], sb_next[TJ];
    auto fetch = [&](int pn, int s, int into) {        // operands of step s of panel pn
        const char *st = smem + (pn & 1) * STAGE;
        const int at = ((4 * half + s) ^ x7) * 16;
#pragma unroll
        for (int i = 0; i < TI; ++i) af[into][i] = *reinterpret_cast<const mx_v4i *>(st + ar + at + i * 4096);
#pragma unroll
        for (int j = 0; j < TJ; ++j) bf[into][j] = *reinterpret_cast<const mx_v4i *>(st + br + at + j * 4096);
    };
    auto fetch_scales = [&](int pn) {
        const char *st = smem + (pn & 1) * STAGE + (BI + BJ) * 128;
#pragma unroll
        for (int i = 0; i < TI; ++i) sa_next[i] = *reinterpret_cast<const int *>(st + (wi0 + i * 32 + l31) * 8 + half * 4);
#pragma unroll
        for (int j = 0; j < TJ; ++j) sb_next[j] = *reinterpret_cast<const int *>(st + (BI + wj0 + j * 32 + l31) * 8 + half * 4);
    };
    auto take_scales = [&]() {
#pragma unroll
        for (int i = 0; i < TI; ++i) sa[i] = sa_next[i];
#pragma unroll
        for (int j = 0; j < TJ; ++j) sb[j] = sb_next[j];
    };
#define MX_STEP(S, CUR)                                                                                                          \
    _Pragma("unroll") for (int i = 0; i < TI; ++i)                                                                               \
        _Pragma("unroll") for (int j = 0; j < TJ; ++j) acc[i][j] = mx_mfma<S>(af[CUR][i], bf[CUR][j], acc[i][j], sa[i], sb[j]);  \
    __builtin_amdgcn_sched_barrier(0);

    if (panels > 0) {
        load(0);
        store(0);
        load(1);
        __syncthreads();
        fetch(0, 0, 0);
        fetch_scales(0);
        take_scales();
        // panels behind the last one read as zeros and nothing of memory (every offset is out of its descriptor's range), so the loop
        // needs no case for its end
        for (int pn = 0; pn < panels; ++pn) {
            fetch(pn, 1, 1);
            MX_STEP(0, 0)
            fetch(pn, 2, 0);
            store(pn + 1);
            MX_STEP(1, 1)
            fetch(pn, 3, 1);
            load(pn + 2);
            MX_STEP(2, 0)
            __syncthreads();
            fetch(pn + 1, 0, 0);
            fetch_scales(pn + 1);
            MX_STEP(3, 1)
            take_scales();
        }
    }
#undef MX_STEP

    // ---- epilogue: strips of 32 rows go through the wave's own part of LDS, so that bias, activation and residual are one loop over
    //      rows and the result leaves in runs along its rows
    constexpr int COLS = TJ * 32, PITCH = COLS + 4;
    static_assert(4 * 32 * PITCH * 4 <= 2 * STAGE, "strips fit in the panels' LDS");
    __syncthreads();
    float *strip = reinterpret_cast<float *>(smem) + wave * 32 * PITCH;
    for (int t = 0; t < TI; ++t) {
#pragma unroll
        for (int ti = 0; ti < TI; ++ti)
            if (t == ti) {
#pragma unroll
                for (int tj = 0; tj < TJ; ++tj)
#pragma unroll
                    for (int e = 0; e < 16; ++e) strip[(8 * (e / 4) + 4 * half + e % 4) * PITCH + tj * 32 + l31] = acc[ti][tj][e];
            }
        const int ib = i0 + wi0 + t * 32;
        if (ib < I) {
            if constexpr (CONV) mx_finish_planes<COLS, PITCH>(p, strip, ib, j0 + wj0, lane);
            else mx_finish_rows<TYPE, COLS, PITCH>(p, strip, ib, j0 + wj0, lane);
        }
    }
}

template <int TYPE, bool CONV, bool BYTES, int TI, int TJ>
static int launch_tile(const MxProductArgs &a, hipStream_t s)
{
    MxTileDev d{a, (int)((a.I + 64 * TI - 1) / (64 * TI)), (int)((a.J + 64 * TJ - 1) / (64 * TJ))};
    const int64_t grid = (int64_t)d.tiles_i * d.tiles_j;
    if (grid > 0x7fffffffLL) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL((mx_product_tile_kernel<TYPE, CONV, BYTES, TI, TJ>), dim3((unsigned)grid), dim3(MX_THREADS), 0, s, d);
    return (int)hipGetLastError();
}

// The tile by the size of D: the largest whose grid still gives every CU a workgroup.
template <int TYPE, bool CONV, bool BYTES>
static int launch_by_size(const MxProductArgs &a, hipStream_t s, char *name, size_t name_len)
{
    auto grid = [&](int64_t t) { return (a.I + t - 1) / t * ((a.J + t - 1) / t); };
    const int cus = device_cu_count();
    const int t = grid(256) >= cus ? 256 : grid(128) >= cus ? 128 : 64;
    if (name) snprintf(name, name_len, "mx_product<%dx%d>", t, t);
    if (t == 256) return launch_tile<TYPE, CONV, BYTES, 4, 4>(a, s);
    if (t == 128) return launch_tile<TYPE, CONV, BYTES, 2, 2>(a, s);
    return launch_tile<TYPE, CONV, BYTES, 1, 1>(a, s);
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
    switch (a.type) {
    case YL_F32: return launch_typed<YL_F32, false>(a, s, name, name_len);
    case YL_F16: return launch_typed<YL_F16, false>(a, s, name, name_len);
    default: return launch_typed<YL_BF16, false>(a, s, name, name_len);
    }
}

bool mx_linear_fused(int64_t, int64_t) { return false; }
int launch_mx_linear(const MxProductArgs &, const MxDense &, void *) { return (int)hipErrorInvalidValue; }

}  // namespace yl
