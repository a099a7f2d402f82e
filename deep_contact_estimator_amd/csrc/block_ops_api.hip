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
// `count` matrices of the same rows, `step` bytes apart (0: one), and one that is written: none of them in its place?
bool apart(const Rows& r, int64_t count, int64_t step, const Rows& w)
{
    if (step == 0) count = 1;
    if (r.rows < 1 || r.width < 1 || w.rows < 1 || w.width < 1 || w.end() <= r.at || r.end() + (uintptr_t)((count - 1) * step) <= w.at) return true;
    const int64_t first = r.end() > w.at || count == 1 ? 0 : (int64_t)((w.at - r.end()) / step) + 1;          // (the matrices that reach w at all)
    const int64_t behind = count == 1 ? 1 : (int64_t)((w.end() - 1 - r.at) / step) + 1;
    for (int64_t g = first; g < count && g < behind; ++g) { Rows m = r; m.at += (uintptr_t)(g * step); if (!apart(m, w)) return false; }
    return true;
}
// one run of n values
Rows run(const void* p, int64_t n, int64_t size) { return Rows(p, p && n > 0 ? 1 : 0, n, n, size); }
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
    if (endless(d->batch, d->x_batch, 4) || endless(d->batch, d->q_batch, 4) || endless((d->k + BLK - 1) / BLK, d->block_rows == 1 ? d->ld_scale : 0, 4))
        return fail(nullptr, DCE_ERR_ARG, "dce_quantize: a stride is out of range (x_batch %lld, q_batch %lld, ld_scale %lld)", (long long)d->x_batch, (long long)d->q_batch, (long long)d->ld_scale);
    const Rows x(d->x, d->rows, d->ldx, d->k, es), q(d->q, d->rows, d->ldq, d->k, 1);
    const int64_t kb = (d->k + BLK - 1) / BLK, ss = d->scale_type == DCE_SCALE_F32 ? 4 : 1;
    const Rows scale = d->block_rows == 1 ? Rows(d->scale, kb, d->ld_scale, d->rows, ss) : run(d->scale, d->batch * ((d->rows + BLK - 1) / BLK) * kb, ss);
    bool clear = apart(x, d->batch, d->x_batch * es, scale) && apart(q, d->batch, d->q_batch, scale);
    const bool far = q.end() + (uintptr_t)((d->batch - 1) * d->q_batch) <= x.at || x.end() + (uintptr_t)((d->batch - 1) * d->x_batch * es) <= q.at;
    for (int64_t g = 0; clear && !far && g < d->batch; ++g) { Rows w = q; w.at += (uintptr_t)(g * d->q_batch); clear = apart(x, d->batch, d->x_batch * es, w); }
    if (!clear) return fail(nullptr, DCE_ERR_ARG, "dce_quantize: x, q and scale overlap");
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
    const int64_t kb = (d->k + BLK - 1) / BLK, nb = (d->n + BLK - 1) / BLK;
    if (endless(kb, d->ld_a_scale, 4) || endless(nb, d->ld_b_scale, 4) || (d->out_type == DCE_TYPE_E4M3 && endless(nb, d->ld_y_scale, 4)))
        return fail(nullptr, DCE_ERR_ARG, "dce_matmul: a scale's stride is out of range (a %lld, b %lld, y %lld)", (long long)d->ld_a_scale, (long long)d->ld_b_scale, (long long)d->ld_y_scale);
    if (endless(d->groups, d->b_group, 4) || endless(d->groups, d->bias_group, 4) || endless(d->groups, d->b_scale_group, 4)) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: a group stride is out of range");
    if (d->m == 0 || d->n == 0) return DCE_OK;
    if (!d->y || (d->k && (!d->b || (!d->a && d->a_rows)))) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: NULL argument");
    const int es = f8 ? 1 : 2, os = d->out_type == DCE_TYPE_F32 ? 4 : d->out_type == DCE_TYPE_BF16 ? 2 : 1;
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
    // workgroups run in any order: nothing that one may still read is written by another
    const int ss = d->scale_type == DCE_SCALE_F32 ? 4 : 1;
    const Rows sa(d->a_scale, f8 && d->a_scale ? kb : 0, d->ld_a_scale, d->a_rows, ss), sb(d->b_scale, f8 && d->b_scale ? nb : 0, d->ld_b_scale, kb, ss);
    const Rows ys(d->y_scale, d->out_type == DCE_TYPE_E4M3 ? nb : 0, d->ld_y_scale, d->m, ss);
    const Rows offsets = run(d->offsets, d->groups + 1, 4), index = run(d->index, d->m, 4), bias = run(d->bias, d->n, 4);
    auto clear_of_reads = [&](const Rows& w) {
        return (!d->k || (apart(a, w) && apart(b, d->groups, d->b_group * es, w) && apart(sa, w) && apart(sb, d->groups, d->b_scale_group * ss, w))) &&
               apart(bias, d->groups, d->bias_group * 4, w) && apart(offsets, w) && apart(index, w);
    };
    if (!clear_of_reads(y) || !clear_of_reads(ys) || !apart(y, ys)) return fail(nullptr, DCE_ERR_ARG, "dce_matmul: y or y_scale overlaps an operand, a scale, the bias, offsets or index, or one the other");
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
    const Rows in = run(ids, n, id_bytes), out[4] = {run(offsets, groups + 1, 4), run(order, n, 4), run(place, n, 4), run(work, group_rows_work(n, groups), 4)};
    for (int i = 0; i < 4; ++i) {
        bool clear = apart(in, out[i]);
        for (int j = 0; clear && j < i; ++j) clear = apart(out[j], out[i]);
        if (!clear) return fail(nullptr, DCE_ERR_ARG, "dce_group_rows: ids, offsets, order, place and work overlap");
    }
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
    if (rows > (1ll << 42)) return fail(nullptr, DCE_ERR_ARG, "dce_decide: %lld rows", (long long)rows);
    const Rows in = run(logits, rows * 16, 4), at = run(index, n, 4), out[3] = {run(logits_out, n * 16, 4), run(pred, n, 4), run(contacts, n * 4, 1)};
    for (int i = 0; i < 3; ++i) {
        const bool in_place = i == 0 && logits_out == logits && !index;      // (a row's lanes read it and then write it)
        bool clear = (in_place || apart(in, out[i])) && apart(at, out[i]);
        for (int j = 0; clear && j < i; ++j) clear = apart(out[j], out[i]);
        if (!clear) return fail(nullptr, DCE_ERR_ARG, "dce_decide: logits, index and the results overlap");
    }
    OP_DEVICE(device_id);
    HIP_TRY(nullptr, launch_decide(logits, n, rows, index, logits_out, pred, contacts, (hipStream_t)hip_stream));
    return DCE_OK;
}

}  // extern "C"
