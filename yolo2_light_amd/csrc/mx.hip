// mx.hip -- the C entries of the MXFP4 operators (include/yolo2_hip.h): checks of the arguments, device and stream, launches.
#include <hip/hip_runtime.h>
#include <cstring>
#include <string>

#include "mx.h"
#include "yl_internal.h"

namespace yl {
namespace {

constexpr const char *MX_TOO_MANY = "more than 2^32 threads in a launch";
constexpr int64_t MX_MAX_LD = (int64_t)1 << 19;           // blocks a row: 32-bit offsets inside a tile of 256 rows

// nothing may be thrown through a C entry: an error text that finds no memory is left out
int refuse(const char *entry, const char *what, int rc = YL_ERR_ARG) noexcept
{
    try {
        set_error(std::string(entry) + ": " + what);
    } catch (...) {
    }
    return rc;
}

// the caller's current device is the same after the call
struct DeviceScope {
    int before = -1;
    bool changed = false;
    int enter(const char *entry, int device)
    {
        if (hipGetDevice(&before) == hipSuccess && before == device) return YL_OK;
        int count = 0;
        if (hipGetDeviceCount(&count) != hipSuccess || count <= 0) {
            return refuse(entry, "no HIP device visible (libyolo2hip has no CPU fallback)", YL_ERR_DEVICE);
        }
        if (device < 0 || device >= count) return refuse(entry, "no such device");
        const hipError_t e = hipSetDevice(device);
        changed = e == hipSuccess;
        return e == hipSuccess ? YL_OK : refuse(entry, hipGetErrorString(e), YL_ERR_DEVICE);
    }
    ~DeviceScope() { if (changed) (void)hipSetDevice(before); }
};

int launched(const char *entry, int e)
{
    return e == 0 ? YL_OK : refuse(entry, hipGetErrorString((hipError_t)e), YL_ERR_DEVICE);
}

int64_t blocks_of(int64_t k) { return (k + MX_BLOCK - 1) / MX_BLOCK; }
int type_bytes(int type) { return type == YL_F32 ? 4 : 2; }

struct Range {
    uintptr_t from, to;      // [from, to)
    bool meets(const Range &o) const { return from < o.to && o.from < to; }
};
Range range_of(const void *p, int64_t bytes) { return {(uintptr_t)p, (uintptr_t)p + (uintptr_t)(bytes > 0 ? bytes : 0)}; }

// Two sets of rows of one buffer side by side: the same row stride, and the column windows of `n` and `m` bytes do not meet.
bool beside(const void *a, int64_t n, const void *b, int64_t m, int64_t stride)
{
    if (stride <= 0) return false;
    int64_t d = (int64_t)((uintptr_t)b - (uintptr_t)a) % stride;
    if (d < 0) d += stride;
    return d >= n && d + m <= stride;
}

const char *check_matrix(const yl_mx_matrix *m)
{
    if (!m) return "matrix is NULL";
    if (m->rows < 0 || m->k < 0) return "negative size of a matrix";
    if (m->ld < blocks_of(m->k) || m->ld > MX_MAX_LD) return "ld of a matrix is smaller than its blocks, or above 2^19";
    if (m->rows > MX_MAX_ELEMENTS / (m->ld > 0 ? m->ld : 1)) return "matrix is too large";
    if (m->rows == 0 || m->k == 0) return nullptr;
    if (!m->codes || !m->scales) return "codes or scales of a matrix are NULL";
    if ((uintptr_t)m->codes % 16) return "codes of a matrix are not 16-byte aligned";
    return nullptr;
}
Range codes_range(const yl_mx_matrix *m) { return range_of(m->codes, m->rows && m->k ? ((m->rows - 1) * m->ld + blocks_of(m->k)) * 16 : 0); }
Range scales_range(const yl_mx_matrix *m) { return range_of(m->scales, m->rows && m->k ? (m->rows - 1) * m->ld + blocks_of(m->k) : 0); }

bool empty(const yl_dense *t) { return t->batch == 0 || t->rows == 0 || t->k == 0; }
const char *check_dense(const yl_dense *t)
{
    if (!t) return "tensor is NULL";
    if (t->type != YL_F32 && t->type != YL_F16 && t->type != YL_BF16) return "type of a tensor is not YL_F32, YL_F16 or YL_BF16";
    const int64_t n[3] = {t->batch, t->rows, t->k}, s[3] = {t->batch_stride, t->row_stride, t->k_stride};
    int64_t reach = 0;
    for (int i = 0; i < 3; ++i) {
        if (n[i] < 0 || s[i] < 0) return "negative size or stride of a tensor";
        if (n[i] > MX_MAX_ELEMENTS || s[i] > MX_MAX_ELEMENTS) return "tensor is too large";
        if (n[i] > 1 && s[i] > MX_MAX_ELEMENTS / (n[i] - 1)) return "tensor is too large";
        reach += n[i] > 1 ? (n[i] - 1) * s[i] : 0;
    }
    if (reach > MX_MAX_ELEMENTS || (t->batch && t->rows > MX_MAX_ELEMENTS / t->batch)) return "tensor is too large";
    if (empty(t)) return nullptr;
    if (!t->data) return "data of a tensor is NULL";
    if ((uintptr_t)t->data % type_bytes(t->type)) return "data of a tensor is not aligned to its type";
    return nullptr;
}
Range dense_range(const yl_dense *t)
{
    if (empty(t)) return range_of(t->data, 0);
    return range_of(t->data, ((t->batch - 1) * t->batch_stride + (t->rows - 1) * t->row_stride + (t->k - 1) * t->k_stride + 1) * type_bytes(t->type));
}
// where a result is written, no two of its elements may share a place
const char *check_written(const yl_dense *t)
{
    int64_t n[3] = {t->batch, t->rows, t->k}, s[3] = {t->batch_stride, t->row_stride, t->k_stride};
    for (int a = 0; a < 2; ++a)                       // by stride, smallest first
        for (int b = 0; b < 2 - a; ++b)
            if (s[b] > s[b + 1]) { std::swap(s[b], s[b + 1]); std::swap(n[b], n[b + 1]); }
    int64_t reach = 0;                                // the largest offset of the axes so far
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1) {
            if (s[i] <= reach) return "elements of a written tensor overlap";
            reach += (n[i] - 1) * s[i];
        }
    return nullptr;
}
MxDense dense_of(const yl_dense *t) { return MxDense{t->data, t->type, t->batch, t->rows, t->k, t->batch_stride, t->row_stride, t->k_stride}; }

const char *check_epilogue(const yl_mx_epilogue *e)
{
    if (!e) return nullptr;
    if (e->activation < YL_LOGISTIC || e->activation > YL_LHTAN) return "unknown activation";
    if ((uintptr_t)e->bias % 4) return "bias is not aligned to its type";
    return nullptr;
}

// the linear product's checks that matmul and linear share; `x_rows`, `x_k`: the left operand's
const char *check_product(int64_t x_rows, int64_t x_k, const yl_mx_matrix *w, const yl_mx_epilogue *e, const yl_dense *y, MxProductArgs *a)
{
    if (const char *m = check_matrix(w)) return m;
    if (const char *m = check_dense(y)) return m;
    if (const char *m = check_epilogue(e)) return m;
    if (x_k != w->k) return "the operands' k differ";
    if (y->batch != 1 || y->rows != x_rows || y->k != w->rows) return "y is not one batch of x's rows by w's rows";
    if (y->k > 1 && y->k_stride != 1) return "y's k_stride is not 1";
    if (y->rows > 1 && y->row_stride < y->k) return "rows of y overlap";
    if (x_rows > MX_MAX_ROWS || w->rows > MX_MAX_ROWS) return "more than 2^31 - 257 rows";
    const Range out = dense_range(y);
    if (out.meets(codes_range(w)) || out.meets(scales_range(w))) return "y overlaps w";
    if (e && e->bias && out.meets(range_of(e->bias, w->rows * 4))) return "y overlaps the bias";
    if (e && e->residual && !empty(y)) {
        if ((uintptr_t)e->residual % type_bytes(y->type)) return "residual is not aligned to its type";
        if (e->residual_stride < 0 || e->residual_stride > MX_MAX_ELEMENTS || (y->rows > 1 && e->residual_stride > MX_MAX_ELEMENTS / (y->rows - 1))) return "residual_stride is negative or too large";
        const Range r = range_of(e->residual, ((y->rows - 1) * e->residual_stride + y->k) * type_bytes(y->type));
        const bool same = e->residual == y->data && (y->rows <= 1 || e->residual_stride == y->row_stride);
        const int64_t el = type_bytes(y->type);
        const bool apart = e->residual_stride == y->row_stride && beside(y->data, y->k * el, e->residual, y->k * el, y->row_stride * el);
        if (!same && !apart && out.meets(r)) return "y overlaps the residual";
    }
    a->b_codes = w->codes; a->b_scales = w->scales; a->b_ld = w->ld;
    a->I = x_rows; a->J = w->rows; a->k = w->k; a->kb = blocks_of(w->k);
    a->bias = e ? e->bias : nullptr; a->act = e ? e->activation : YL_LINEAR;
    a->residual = e ? e->residual : nullptr; a->residual_stride = e ? e->residual_stride : 0;
    a->out = y->data; a->out_stride = y->row_stride; a->type = y->type;
    return mx_product_fits(*a) ? nullptr : MX_TOO_MANY;
}

}  // namespace
}  // namespace yl

using namespace yl;

extern "C" {

int64_t yl_mx_blocks(int64_t k)
{
    if (k < 0 || k > MX_MAX_LD * MX_BLOCK) return 0;
    return (blocks_of(k) + 3) / 4 * 4;
}

int yl_mx_quantize(int device, void *stream, const yl_dense *src, const yl_mx_matrix *dst)
{
    const char *entry = "yl_mx_quantize";
    if (const char *m = check_dense(src)) return refuse(entry, m);
    if (const char *m = check_matrix(dst)) return refuse(entry, m);
    if (dst->k != src->k || dst->rows != src->batch * src->rows) return refuse(entry, "dst is not batch * rows by k of src");
    const Range r = dense_range(src), c = codes_range(dst), s = scales_range(dst);
    if (r.meets(c) || r.meets(s)) return refuse(entry, "dst overlaps src");
    if (c.meets(s)) return refuse(entry, "codes and scales overlap");
    if (!mx_rounding_fits(dense_of(src))) return refuse(entry, MX_TOO_MANY);
    DeviceScope scope;
    if (int rc = scope.enter(entry, device)) return rc;
    return launched(entry, launch_mx_quantize(dense_of(src), dst->codes, dst->scales, dst->ld, stream));
}

int yl_mx_dequantize(int device, void *stream, const yl_mx_matrix *src, const yl_dense *dst)
{
    const char *entry = "yl_mx_dequantize";
    if (const char *m = check_matrix(src)) return refuse(entry, m);
    if (const char *m = check_dense(dst)) return refuse(entry, m);
    if (const char *m = check_written(dst)) return refuse(entry, m);
    if (src->k != dst->k || src->rows != dst->batch * dst->rows) return refuse(entry, "dst is not src's rows by k");
    const Range r = dense_range(dst);
    if (r.meets(codes_range(src)) || r.meets(scales_range(src))) return refuse(entry, "dst overlaps src");
    if (!mx_rounding_fits(dense_of(dst))) return refuse(entry, MX_TOO_MANY);
    DeviceScope scope;
    if (int rc = scope.enter(entry, device)) return rc;
    return launched(entry, launch_mx_dequantize(src->codes, src->scales, src->ld, dense_of(dst), stream));
}

int yl_mx_matmul(int device, void *stream, const yl_mx_matrix *x, const yl_mx_matrix *w, const yl_mx_epilogue *epilogue, const yl_dense *y)
{
    const char *entry = "yl_mx_matmul";
    MxProductArgs a{};
    if (const char *m = check_matrix(x)) return refuse(entry, m);
    if (const char *m = check_product(x->rows, x->k, w, epilogue, y, &a)) return refuse(entry, m);
    const Range out = dense_range(y);
    if (out.meets(codes_range(x)) || out.meets(scales_range(x))) return refuse(entry, "y overlaps x");
    a.a_codes = x->codes; a.a_scales = x->scales; a.a_ld = x->ld;
    DeviceScope scope;
    if (int rc = scope.enter(entry, device)) return rc;
    return launched(entry, launch_mx_product(a, stream));
}

int64_t yl_mx_linear_workspace(int64_t rows, int64_t k)
{
    if (rows <= 0 || k <= 0 || k > MX_MAX_LD * MX_BLOCK || rows > MX_MAX_ELEMENTS / yl_mx_blocks(k)) return 0;
    if (mx_linear_fused(rows, k)) return 0;
    return rows * yl_mx_blocks(k) * 17;
}

int yl_mx_linear(int device, void *stream, const yl_dense *x, const yl_mx_matrix *w, const yl_mx_epilogue *epilogue, const yl_dense *y,
                 void *workspace, int64_t workspace_bytes)
{
    const char *entry = "yl_mx_linear";
    MxProductArgs a{};
    if (const char *m = check_dense(x)) return refuse(entry, m);
    if (x->batch != 1) return refuse(entry, "x has more than one batch");
    if (const char *m = check_product(x->rows, x->k, w, epilogue, y, &a)) return refuse(entry, m);
    const Range in = dense_range(x), out = dense_range(y);
    const int64_t xe = type_bytes(x->type), ye = type_bytes(y->type);
    const bool apart = x->k_stride == 1 && x->row_stride * xe == y->row_stride * ye && beside(x->data, x->k * xe, y->data, y->k * ye, y->row_stride * ye);
    if (!apart && out.meets(in)) return refuse(entry, "y overlaps x");
    const bool fused = mx_linear_fused(x->rows, x->k), some = x->rows > 0 && x->k > 0;
    const int64_t need = yl_mx_linear_workspace(x->rows, x->k);
    if (some && !fused && need == 0) return refuse(entry, "x is too large for a workspace");
    if (need > 0 && !mx_rounding_fits(dense_of(x))) return refuse(entry, MX_TOO_MANY);
    if (need > 0) {
        if (!workspace || workspace_bytes < need) return refuse(entry, "workspace is smaller than yl_mx_linear_workspace(x->rows, x->k)");
        if ((uintptr_t)workspace % 16) return refuse(entry, "workspace is not 16-byte aligned");
        const Range ws = range_of(workspace, need);
        if (ws.meets(in) || ws.meets(out) || ws.meets(codes_range(w)) || ws.meets(scales_range(w)) ||
            (epilogue && epilogue->bias && ws.meets(range_of(epilogue->bias, w->rows * 4))) ||
            (epilogue && epilogue->residual && !empty(y) &&
             ws.meets(range_of(epilogue->residual, ((y->rows - 1) * epilogue->residual_stride + y->k) * type_bytes(y->type)))))
            return refuse(entry, "workspace overlaps a tensor");
    }
    DeviceScope scope;
    if (int rc = scope.enter(entry, device)) return rc;
    if (x->rows == 0 || w->rows == 0) return YL_OK;
    if (some && fused) return launched(entry, launch_mx_linear(a, dense_of(x), stream));
    const int64_t ld = yl_mx_blocks(x->k);
    a.a_codes = workspace; a.a_scales = (char *)workspace + x->rows * ld * 16; a.a_ld = ld;
    if (int rc = launched(entry, launch_mx_quantize(dense_of(x), workspace, (char *)workspace + x->rows * ld * 16, ld, stream))) return rc;
    return launched(entry, launch_mx_product(a, stream));
}

int yl_mx_conv2d(int device, void *stream, const yl_mx_matrix *x, const yl_mx_matrix *filters, const yl_mx_conv *shape,
                 const yl_mx_epilogue *epilogue, float *out, const yl_mx_matrix *q_out)
{
    const char *entry = "yl_mx_conv2d";
    if (const char *m = check_matrix(x)) return refuse(entry, m);
    if (const char *m = check_matrix(filters)) return refuse(entry, m);
    if (const char *m = check_epilogue(epilogue)) return refuse(entry, m);
    if (!shape) return refuse(entry, "shape is NULL");
    const yl_mx_conv c = *shape;
    if (c.batch < 0 || c.h < 1 || c.w < 1 || c.size < 1 || c.size > MX_MAX_SIZE || c.stride < 1 || c.pad < 0 || c.pad >= c.size)
        return refuse(entry, "shape: batch >= 0, h, w >= 1, 1 <= size <= 5, stride >= 1, 0 <= pad < size");
    if (x->k < 1 || c.h > 1 << 20 || c.w > 1 << 20 || c.stride > 1 << 20) return refuse(entry, "no channels, or a map edge or stride above 2^20");
    const int64_t pixels = (int64_t)c.h * c.w;
    if (c.batch > MX_MAX_ELEMENTS / pixels) return refuse(entry, "map or result is too large");
    if (x->rows != c.batch * pixels) return refuse(entry, "x is not batch * h * w rows");
    if (filters->k != (int64_t)c.size * c.size * blocks_of(x->k) * MX_BLOCK) return refuse(entry, "filters' k is not size * size * whole blocks of x's channels");
    const int oh_num = c.h + 2 * c.pad - c.size, ow_num = c.w + 2 * c.pad - c.size;
    if (oh_num < 0 || ow_num < 0) return refuse(entry, "the filter is larger than the padded map");
    if (const char *m = mx_conv_beyond(c.batch, c.h, c.w, x->k, x->ld, filters->rows, c.size, c.stride, c.pad)) return refuse(entry, m);
    const int oh = oh_num / c.stride + 1, ow = ow_num / c.stride + 1;
    const int64_t J = (int64_t)c.batch * oh * ow, I = filters->rows;
    const float *bias = epilogue ? epilogue->bias : nullptr;
    const float *residual = epilogue ? (const float *)epilogue->residual : nullptr;
    if ((uintptr_t)out % 4 || (uintptr_t)residual % 4) return refuse(entry, "out or residual is not aligned to its type");
    const Range xr[2] = {codes_range(x), scales_range(x)}, fr[2] = {codes_range(filters), scales_range(filters)};
    const Range br = range_of(bias, bias ? I * 4 : 0), rr = range_of(residual, residual ? I * J * 4 : 0), o = range_of(out, out ? I * J * 4 : 0);
    for (int i = 0; i < 2; ++i)
        if (o.meets(xr[i]) || o.meets(fr[i])) return refuse(entry, "out overlaps an operand");
    if (o.meets(br)) return refuse(entry, "out overlaps the bias");
    if (residual != out && o.meets(rr)) return refuse(entry, "out overlaps the residual");
    MxProductArgs a{};
    if (q_out) {
        if (const char *m = check_matrix(q_out)) return refuse(entry, m);
        if (q_out->rows != J || q_out->k != I) return refuse(entry, "q_out is not batch * oh * ow rows by filters");
        const Range qr[2] = {codes_range(q_out), scales_range(q_out)};
        for (int i = 0; i < 2; ++i)
            if (qr[i].meets(o) || qr[i].meets(br) || qr[i].meets(rr) || qr[i].meets(xr[0]) || qr[i].meets(xr[1]) || qr[i].meets(fr[0]) || qr[i].meets(fr[1]))
                return refuse(entry, "q_out overlaps another tensor");
        if (qr[0].meets(qr[1])) return refuse(entry, "codes and scales overlap");
        a.q_codes = q_out->codes; a.q_scales = q_out->scales; a.q_ld = q_out->ld;
    }
    a.a_codes = filters->codes; a.a_scales = filters->scales; a.a_ld = filters->ld;
    a.b_codes = x->codes; a.b_scales = x->scales; a.b_ld = x->ld;
    a.I = I; a.J = J; a.kb = blocks_of(filters->k);
    a.bias = bias; a.act = epilogue ? epilogue->activation : YL_LINEAR; a.residual = residual;
    a.out = out; a.type = YL_F32;
    a.conv = true;
    a.H = c.h; a.W = c.w; a.OH = oh; a.OW = ow; a.G = (int)blocks_of(x->k); a.size = c.size; a.stride = c.stride; a.pad = c.pad; a.batch = c.batch;
    if (!mx_product_fits(a)) return refuse(entry, MX_TOO_MANY);
    DeviceScope scope;
    if (int rc = scope.enter(entry, device)) return rc;
    if (!out && !q_out) return YL_OK;
    return launched(entry, launch_mx_product(a, stream));
}

}  // extern "C"
