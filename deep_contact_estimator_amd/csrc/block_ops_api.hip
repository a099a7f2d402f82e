// block_ops_api.hip -- the C entries of the matrix products as operators of their own (include/dce.h).  They hold no state: device and stream come
// with the call, there is no workspace inside, any number of threads may call, and a call may be captured into a graph.
#include "dce_ctx.h"
#include "block_ops.h"

using namespace dce;

namespace {

constexpr int64_t ROWS_MAX = 1ll << 30, DIM_MAX = 1ll << 24;

// `rows` rows of `width` bytes, `stride` apart (one row: its stride says nothing)
struct Rows {
    uintptr_t at; int64_t rows, stride, width;
    Rows(const void* p, int64_t rows_, int64_t ld, int64_t n, int64_t size)
        : at(reinterpret_cast<uintptr_t>(p)), rows(rows_), stride(rows_ > 1 ? ld * size : n * size), width(n * size) {}
    bool whole() const { return stride == width; }
    uintptr_t end() const { return at + (uintptr_t)(rows - 1) * stride + width; }
    bool meets(uintptr_t lo, uintptr_t hi) const
    {
        const uintptr_t first = at + width > lo ? 0 : (lo - at - width) / stride + 1;    // the first row that ends behind lo
        return first < (uintptr_t)rows && at + first * stride < hi;
    }
};
// no two rows in the same place?  Rows with gaps of different strides are taken to be apart.
bool apart(const Rows& a, const Rows& b)
{
    if (a.rows < 1 || b.rows < 1 || a.width < 1 || b.width < 1 || a.end() <= b.at || b.end() <= a.at) return true;
    if (a.whole()) return !b.meets(a.at, a.end());
    if (b.whole()) return !a.meets(b.at, b.end());
    if (a.stride != b.stride) return true;
    const int64_t d = a.at <= b.at ? (int64_t)((b.at - a.at) % a.stride) : (a.stride - (int64_t)((a.at - b.at) % a.stride)) % a.stride;
    return d >= a.width && d + b.width <= a.stride;
}
// rows that no address space holds (so that no offset below passes 64 bits)
bool endless(int64_t rows, int64_t ld, int size) { return rows > 1 && ld > (1ll << 47) / size / (rows - 1); }

bool off(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

int device_count()
{
    static const int n = [] { int c = 0; return hipGetDeviceCount(&c) == hipSuccess ? c : 0; }();
    return n;
}

#define OP_DEVICE(id)                                                                                                        \
    if (device_count() <= 0)                                                                                                 \
        return fail(nullptr, DCE_ERR_HIP, "no HIP device available: the HIP path is mandatory, there is no CPU fallback");   \
    if ((id) < 0 || (id) >= device_count()) return fail(nullptr, DCE_ERR_ARG, "device %d out of range (%d devices)", (id), device_count()); \
    DeviceGuard dev_guard_(id);                                                                                              \
    if (dev_guard_.err != hipSuccess) return fail(nullptr, DCE_ERR_HIP, "hipSetDevice(%d) failed: %s", (id), hipGetErrorString(dev_guard_.err))

}  // namespace

extern "C" {

int dce_quantize(int device_id, void* hip_stream, const dce_quantize_desc* d)
{
    if (!d) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: NULL descriptor");
    if (d->x_type != DCE_TYPE_F32 && d->x_type != DCE_TYPE_BF16) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: x must be fp32 or bf16 (type %d)", d->x_type);
    if (d->scale_type != DCE_SCALE_E8M0 && d->scale_type != DCE_SCALE_F32) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: unknown scale type %d", d->scale_type);
    if (d->block_rows != 1 && d->block_rows != BLK) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: a block has 1 row or %d, not %d", BLK, d->block_rows);
    if (d->batch < 0 || d->batch > 65535 || d->rows < 0 || d->rows > (d->block_rows == 1 ? ROWS_MAX : 65535ll * BLK) || d->k < 0 || d->k > DIM_MAX)
        return fail(nullptr, DCE_ERR_ARG, "dce_quantize: sizes out of range (batch %lld, rows %lld, k %lld)", (long long)d->batch, (long long)d->rows, (long long)d->k);
    if (d->block_rows == 1 && d->batch != 1) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: 1 x 128 blocks take one matrix (batch %lld)", (long long)d->batch);
    if (d->ldx < d->k || d->ldq < d->k) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: a row stride is below k = %lld (x %lld, q %lld)", (long long)d->k, (long long)d->ldx, (long long)d->ldq);
    if (endless(d->rows, d->ldx, 4) || endless(d->rows, d->ldq, 4)) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: a row stride is out of range (x %lld, q %lld)", (long long)d->ldx, (long long)d->ldq);
    if (d->batch > 1 && (d->x_batch < 0 || d->q_batch < d->rows * d->ldq)) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: the matrices of q overlap");
    if (d->batch == 0 || d->rows == 0 || d->k == 0) return DCE_OK;
    if (!d->x || !d->q || !d->scale) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: NULL argument");
    const int es = d->x_type == DCE_TYPE_F32 ? 4 : 2;
    if (off(d->x, es) || (d->scale_type == DCE_SCALE_F32 && off(d->scale, 4))) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: a pointer is not aligned to its type");
    if (d->block_rows == 1 && d->ld_scale < d->rows) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: ld_scale %lld is below the rows (%lld)", (long long)d->ld_scale, (long long)d->rows);
    const Rows x(d->x, d->rows, d->ldx, d->k, es), q(d->q, d->rows, d->ldq, d->k, 1);
    if (d->batch == 1 && !apart(x, q)) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: x and q overlap");
    OP_DEVICE(device_id);
    QuantArgs a{};
    a.x = static_cast<const char*>(d->x); a.x_row = x.stride; a.x_batch = d->x_batch * es;
    a.q = d->q; a.q_row = q.stride; a.q_batch = d->q_batch;
    a.k = (int)d->k; a.kblocks = (int)((d->k + BLK - 1) / BLK);
    a.rows = d->rows; a.units = d->rows * a.kblocks;
    a.s = d->scale; a.s_block = d->block_rows == 1 ? d->ld_scale : a.kblocks;
    HIP_TRY(nullptr, launch_quantize(a, d->x_type == DCE_TYPE_BF16, (int)d->batch, d->block_rows, d->scale_type == DCE_SCALE_E8M0, (hipStream_t)hip_stream));
    return DCE_OK;
}

int dce_matmul(int device_id, void* hip_stream, const dce_matmul_desc* d)
{
    if (!d) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: NULL descriptor");
    const bool f8 = d->in_type == DCE_TYPE_E4M3;
    if (!f8 && d->in_type != DCE_TYPE_BF16) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: operands must be bf16 or e4m3 (type %d)", d->in_type);
    if (d->out_type != DCE_TYPE_F32 && d->out_type != DCE_TYPE_BF16 && d->out_type != DCE_TYPE_E4M3) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: unknown result type %d", d->out_type);
    if (!f8 && d->out_type == DCE_TYPE_E4M3) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: e4m3 results need e4m3 operands");
    if (f8 && d->scale_type != DCE_SCALE_E8M0 && d->scale_type != DCE_SCALE_F32) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: unknown scale type %d", d->scale_type);
    if (d->m < 0 || d->m > ROWS_MAX || d->a_rows < 0 || d->a_rows > ROWS_MAX || d->n < 0 || d->n > DIM_MAX || d->k < 0 || d->k > DIM_MAX)
        return fail(nullptr, DCE_ERR_ARG, "dce_matmul: sizes out of range (m %lld, a_rows %lld, n %lld, k %lld)", (long long)d->m, (long long)d->a_rows, (long long)d->n, (long long)d->k);
    if (d->groups < 1 || d->groups > GROUPS_MAX) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: 1 .. %d groups, not %d", GROUPS_MAX, d->groups);
    if (d->groups > 1 && !d->offsets) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: %d groups need offsets", d->groups);
    if (!d->index && d->a_rows < d->m) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: a has %lld rows, the result %lld", (long long)d->a_rows, (long long)d->m);
    if (d->lda < d->k || d->ldb < d->k || d->ldy < d->n)
        return fail(nullptr, DCE_ERR_ARG, "dce_matmul: a row stride is below the row's length (a %lld, b %lld, y %lld)", (long long)d->lda, (long long)d->ldb, (long long)d->ldy);
    if (endless(d->a_rows, d->lda, 4) || endless(d->n, d->ldb, 4) || endless(d->m, d->ldy, 4))
        return fail(nullptr, DCE_ERR_ARG, "dce_matmul: a row stride is out of range (a %lld, b %lld, y %lld)", (long long)d->lda, (long long)d->ldb, (long long)d->ldy);
    if (d->groups > 1 && (d->b_group < 0 || d->bias_group < 0 || d->b_scale_group < 0)) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: a group stride is negative");
    if (endless(d->groups, d->b_group, 4)) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: a group stride is out of range");
    if (d->m == 0 || d->n == 0) return DCE_OK;
    if (!d->y || (d->k && (!d->b || (!d->a && d->a_rows)))) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: NULL argument");
    const int es = f8 ? 1 : 2, os = d->out_type == DCE_TYPE_F32 ? 4 : d->out_type == DCE_TYPE_BF16 ? 2 : 1;
    const int64_t kb = (d->k + BLK - 1) / BLK, nb = (d->n + BLK - 1) / BLK;
    if (f8 && d->k) {
        if (!d->a_scale && d->a_rows) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: e4m3 operands need a_scale and b_scale");
        if (!d->b_scale) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: e4m3 operands need a_scale and b_scale");
        if (d->ld_a_scale < d->a_rows || d->ld_b_scale < kb) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: a scale's stride is below its row's length");
        if (d->scale_type == DCE_SCALE_F32 && (off(d->a_scale, 4) || off(d->b_scale, 4))) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: a pointer is not aligned to its type");
    }
    if (d->out_type == DCE_TYPE_E4M3) {
        if (!d->y_scale || d->ld_y_scale < d->m) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: e4m3 results need y_scale (%lld, %lld)", (long long)nb, (long long)d->m);
        if (d->scale_type == DCE_SCALE_F32 && off(d->y_scale, 4)) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: a pointer is not aligned to its type");
    }
    if (off(d->a, es) || off(d->b, es) || off(d->y, os) || off(d->bias, 4) || off(d->offsets, 4) || off(d->index, 4)) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: a pointer is not aligned to its type");
    const Rows a(d->a, d->a_rows, d->lda, d->k, es), b(d->b, d->n, d->ldb, d->k, es), y(d->y, d->m, d->ldy, d->n, os);
    bool clear = apart(a, y);
    if (clear && d->k && y.at < b.end() + (d->groups - 1) * d->b_group * es && b.at < y.end())
        for (int g = 0; clear && g < d->groups; ++g) { Rows w = b; w.at += (uintptr_t)(g * d->b_group * es); clear = apart(w, y); }
    if (!clear) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: y overlaps an operand");
    OP_DEVICE(device_id);
    ProductArgs p{};
    p.a = static_cast<const char*>(d->a); p.a_row = a.stride;
    p.b = static_cast<const char*>(d->b); p.b_row = b.stride; p.b_group = d->b_group * es;
    p.sa = d->a_scale; p.sa_block = d->ld_a_scale;
    p.sb = d->b_scale; p.sb_row = d->ld_b_scale; p.sb_group = d->b_scale_group;
    p.bias = d->bias; p.bias_group = d->bias_group;
    p.y = static_cast<char*>(d->y); p.y_row = y.stride;
    p.ys = d->y_scale; p.ys_block = d->ld_y_scale;
    p.offsets = d->offsets; p.index = d->index;
    p.a_rows = d->a_rows;
    p.m = (int)d->m; p.n = (int)d->n; p.kbytes = (int)(d->k * es); p.groups = d->groups; p.relu = d->relu != 0;
    const int in = !f8 ? IN_BF16 : d->scale_type == DCE_SCALE_F32 ? IN_F8_F32 : IN_F8_E8;
    const hipError_t e = launch_product(p, in, d->out_type == DCE_TYPE_F32 ? OUT_F32 : d->out_type == DCE_TYPE_BF16 ? OUT_BF16 : OUT_E4M3, (hipStream_t)hip_stream);
    if (e == hipErrorInvalidConfiguration) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: m %lld x n %lld is more tiles than a launch has", (long long)d->m, (long long)d->n);
    HIP_TRY(nullptr, e);
    return DCE_OK;
}

int64_t dce_group_rows_work(int64_t n, int groups)
{
    if (n < 0 || n > ROWS_MAX || groups < 1 || groups > GROUPS_MAX) return fail(nullptr, DCE_ERR_ARG, "dce_group_rows: n %lld or groups %d out of range", (long long)n, groups);
    return group_rows_work(n, groups);
}

int dce_group_rows(int device_id, void* hip_stream, const void* ids, int id_bytes, int64_t n, int groups,
                   int32_t* offsets, int32_t* order, int32_t* place, int32_t* work)
{
    if (n < 0 || n > ROWS_MAX || groups < 1 || groups > GROUPS_MAX) return fail(nullptr, DCE_ERR_ARG, "dce_group_rows: n %lld or groups %d out of range", (long long)n, groups);
    if (id_bytes != 4 && id_bytes != 8) return fail(nullptr, DCE_ERR_ARG, "dce_group_rows: ids are int32 or int64 (%d bytes)", id_bytes);
    if (!offsets || (n && (!ids || !order || !place))) return fail(nullptr, DCE_ERR_ARG, "dce_group_rows: NULL argument");
    if (!work && group_rows_work(n, groups)) return fail(nullptr, DCE_ERR_ARG, "dce_group_rows: %lld rows need dce_group_rows_work's workspace", (long long)n);
    if (off(ids, id_bytes) || off(offsets, 4) || off(order, 4) || off(place, 4) || off(work, 4)) return fail(nullptr, DCE_ERR_ARG, "dce_group_rows: a pointer is not aligned to its type");
    OP_DEVICE(device_id);
    HIP_TRY(nullptr, launch_group_rows(ids, id_bytes, (int)n, groups, offsets, order, place, work, (hipStream_t)hip_stream));
    return DCE_OK;
}

int dce_decide(int device_id, void* hip_stream, const float* logits, int64_t rows, const int32_t* index, int64_t n,
               float* logits_out, int32_t* pred, uint8_t* contacts)
{
    if (n < 0 || n > ROWS_MAX || rows < 0 || (!index && rows < n)) return fail(nullptr, DCE_ERR_ARG, "dce_decide: %lld of %lld rows", (long long)n, (long long)rows);
    if (n == 0) return DCE_OK;
    if (!logits && rows) return fail(nullptr, DCE_ERR_ARG, "dce_decide: NULL argument");
    if (off(logits, 4) || off(index, 4) || off(logits_out, 4) || off(pred, 4)) return fail(nullptr, DCE_ERR_ARG, "dce_decide: a pointer is not aligned to its type");
    OP_DEVICE(device_id);
    HIP_TRY(nullptr, launch_decide(logits, n, rows, index, logits_out, pred, contacts, (hipStream_t)hip_stream));
    return DCE_OK;
}

}  // extern "C"
