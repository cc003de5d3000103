// C ABI of the norms with rotation (include/hy_rotary.h, hy_paged_kv_write_rotated
// of include/hy_paged.h): checks of arguments, launches.
#include <algorithm>
#include <cmath>

#include "hy_call.cuh"
#include "hy_paged_launch.cuh"
#include "hy_rotary.cuh"

using namespace hy;

namespace {

int check_rotation(const hy_rotation* t)
{
    if (!t) return fail(HY_ERR_INVALID_ARGUMENT, "rotation is null");
    if (!t->q_weight_dev || !t->k_weight_dev || (t->table_rows != 0 && (!t->cos_dev || !t->sin_dev)))
        return fail(HY_ERR_INVALID_ARGUMENT, "norm weights or angles are null");
    if (!aligned16(t->q_weight_dev) || !aligned16(t->k_weight_dev) || !aligned16(t->cos_dev) || !aligned16(t->sin_dev) ||
        off16(t->table_stride, 4, t->table_rows))
        return fail(HY_ERR_INVALID_ARGUMENT, "norm weights and rows of angles must start on 16 bytes");
    if (t->table_rows < 0 || t->table_stride < 0)
        return fail(HY_ERR_INVALID_ARGUMENT, "table_rows and table_stride must not be negative");
    if (!(t->eps >= 0.f) || !std::isfinite(t->eps)) return fail(HY_ERR_INVALID_ARGUMENT, "eps must be finite and not negative");
    return HY_OK;
}

// Row tensors of one type and as many rows.
struct RowTensor {
    const char* name;
    const void* p;
    int heads;
    long long row, head;   // strides
};

// Whether two of them share elements. Interleaved ones, views of one projection, are told apart exactly; only those whose
// ranges meet and whose rows lie differently far apart (in one buffer, that is) are not looked into.
bool rows_meet(const RowTensor& a, const RowTensor& b, int rows, int dim, int elem)
{
    using Wide = __int128;   // (strides may be anything)
    const Wide apart = (static_cast<Wide>(reinterpret_cast<uintptr_t>(b.p)) - static_cast<Wide>(reinterpret_cast<uintptr_t>(a.p))) / elem;
    auto extent = [&](const RowTensor& t) { return static_cast<Wide>(rows - 1) * t.row + static_cast<Wide>(t.heads - 1) * t.head + dim; };
    if (apart >= extent(a) || -apart >= extent(b)) return false;
    if (rows > 1 && a.row != b.row) return false;
    // Head i of a and j of b, rows d apart: |apart + j b.head - i a.head - d row| < dim for a d of at most rows - 1.
    auto heads_meet = [&](Wide i, Wide j) {
        const Wide x = apart + j * b.head - i * a.head;
        if (rows == 1 || a.row == 0) return x < dim && -x < dim;
        const Wide r = a.row, y = x < 0 ? -x : x;
        const Wide low = y / r, d = low < rows - 1 ? low : rows - 1;   // the nearest rows
        return y - d * r < dim || (d + 1 < rows && (d + 1) * r - y < dim);
    };
    if (a.head == b.head || a.heads == 1 || b.heads == 1)   // the heads' distance alone counts
    {
        for (int j = 0; j < b.heads; ++j)
            if (heads_meet(0, j)) return true;
        for (int i = 1; i < a.heads; ++i)
            if (heads_meet(i, 0)) return true;
        return false;
    }
    for (int i = 0; i < a.heads; ++i)
        for (int j = 0; j < b.heads; ++j)
            if (heads_meet(i, j)) return true;
    return false;
}

// An output is the input itself or lies elsewhere.
int check_output(const RowTensor& out, const RowTensor& in, int rows, int dim, int dtype)
{
    char msg[96];
    if (out.p == in.p && (rows < 2 || out.row == in.row) && (in.heads < 2 || out.head == in.head)) return HY_OK;
    if (out.p == in.p) snprintf(msg, sizeof msg, "%s in place of its input needs the input's strides", out.name);
    else if (rows_meet(out, in, rows, dim, elem_size(dtype))) snprintf(msg, sizeof msg, "%s must be its input or not overlap it", out.name);
    else return HY_OK;
    return fail(HY_ERR_INVALID_ARGUMENT, msg);
}

// Two that lie apart.
int check_elsewhere(const RowTensor& out, const RowTensor& other, int rows, int dim, int dtype)
{
    if (out.p != other.p && !rows_meet(out, other, rows, dim, elem_size(dtype))) return HY_OK;
    char msg[96];
    snprintf(msg, sizeof msg, "%s must not overlap %s", out.name, other.name);
    return fail(HY_ERR_INVALID_ARGUMENT, msg);
}

int check_heads(int rows, int q_heads, int kv_heads)
{
    if (q_heads < 1 || kv_heads < 1) return fail(HY_ERR_INVALID_ARGUMENT, "q_heads and kv_heads must be positive");
    if (q_heads > 1024 || kv_heads > 1024) return fail(HY_ERR_UNSUPPORTED, "q_heads and kv_heads must be at most 1024");
    if (static_cast<long long>(rows) * std::max(q_heads, kv_heads) > INT_MAX)
        return fail(HY_ERR_CAPACITY, "rows * heads must be below 2^31");
    return HY_OK;
}

RotateArgs rotate_args(const hy_rotation* t, int rows, int q_heads, int kv_heads, int head_dim)
{
    RotateArgs a{};
    a.q_weight = t->q_weight_dev;
    a.k_weight = t->k_weight_dev;
    a.cos = t->cos_dev;
    a.sin = t->sin_dev;
    a.positions = t->positions_dev;
    a.table_stride = t->table_stride;
    a.table_rows = t->table_rows;
    a.eps = t->eps;
    a.inv_dim = 1.f / static_cast<float>(head_dim);
    a.rows = rows;
    a.q_heads = q_heads;
    a.kv_heads = kv_heads;
    return a;
}

template <typename RT, typename CT, int D, bool CACHE>
cudaError_t launch_rotate(RotateArgs a, bool first, cudaStream_t s)
{
    constexpr int VPW = 32 / (D / (2 * (16 / static_cast<int>(sizeof(RT)))));
    const int heads = a.q_heads + (CACHE ? 2 : 1) * a.kv_heads;
    a.whole = a.rows >= 4 * 148;
    int parts = 1;
    if (a.whole)
        a.per_cta = std::min(kRowsPerCta, std::max(8, a.rows / (8 * 148) / 4 * 4));
    else
    {
        a.per_cta = 1;
        parts = std::min((heads + kRowWarps * VPW - 1) / (kRowWarps * VPW), std::max(1, 4 * 148 / a.rows));
    }
    return launch_pdl(first ? rotate_kernel<RT, CT, D, CACHE, true> : rotate_kernel<RT, CT, D, CACHE, false>, dim3((a.rows + a.per_cta - 1) / a.per_cta, parts), kRowWarps * 32, 0, s, a);
}

}  // namespace

extern "C" {

int hy_norm_rotate(const hy_rotation* rotation, int rows, int q_heads, int kv_heads, int head_dim, int dtype,
                   int device, const void* q_dev, int64_t q_row_stride, int64_t q_head_stride, const void* k_dev,
                   int64_t k_row_stride, int64_t k_head_stride, void* q_out_dev, int64_t q_out_row_stride,
                   int64_t q_out_head_stride, void* k_out_dev, int64_t k_out_row_stride, int64_t k_out_head_stride,
                   int* status_dev, void* stream)
{
    int rc = check_rotation(rotation);
    if (!rc) rc = check_dtype(rows, dtype);
    if (rc) return rc;
    if (head_dim != 64 && head_dim != 128) return fail(HY_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
    if (device < 0) return fail(HY_ERR_INVALID_ARGUMENT, "device must not be negative");
    rc = check_heads(rows, q_heads, kv_heads);
    if (rc || rows == 0) return rc;
    rc = check_rows("q", q_dev, rows, q_heads, q_row_stride, q_head_stride, dtype);
    if (!rc) rc = check_rows("k", k_dev, rows, kv_heads, k_row_stride, k_head_stride, dtype);
    if (!rc) rc = check_rows("q_out", q_out_dev, rows, q_heads, q_out_row_stride, q_out_head_stride, dtype);
    if (!rc) rc = check_rows("k_out", k_out_dev, rows, kv_heads, k_out_row_stride, k_out_head_stride, dtype);
    if (!rc) rc = check_apart("q_out", rows, q_heads, head_dim, q_out_row_stride, q_out_head_stride);
    if (!rc) rc = check_apart("k_out", rows, kv_heads, head_dim, k_out_row_stride, k_out_head_stride);
    const RowTensor q{"q", q_dev, q_heads, q_row_stride, q_head_stride}, k{"k", k_dev, kv_heads, k_row_stride, k_head_stride},
        q_out{"q_out", q_out_dev, q_heads, q_out_row_stride, q_out_head_stride}, k_out{"k_out", k_out_dev, kv_heads, k_out_row_stride, k_out_head_stride};
    if (!rc) rc = check_output(q_out, q, rows, head_dim, dtype);
    if (!rc) rc = check_output(k_out, k, rows, head_dim, dtype);
    if (!rc) rc = check_elsewhere(q_out, k_out, rows, head_dim, dtype);
    if (!rc) rc = check_elsewhere(q_out, k, rows, head_dim, dtype);
    if (!rc) rc = check_elsewhere(k_out, q, rows, head_dim, dtype);
    if (rc) return rc;
    DeviceGuard guard(device);
    if (guard.error() != cudaSuccess) return cuda_fail("device", guard.error());
    RotateArgs a = rotate_args(rotation, rows, q_heads, kv_heads, head_dim);
    a.q = q_dev; a.q_row = q_row_stride; a.q_head = q_head_stride;
    a.k = k_dev; a.k_row = k_row_stride; a.k_head = k_head_stride;
    a.q_out = q_out_dev; a.qo_row = q_out_row_stride; a.qo_head = q_out_head_stride;
    a.k_out = k_out_dev; a.ko_row = k_out_row_stride; a.ko_head = k_out_head_stride;
    a.status = status_dev;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool first = rotation->rotate_first != 0;
    const cudaError_t e =
        dtype == HY_DTYPE_F32
            ? (head_dim == 64 ? launch_rotate<float, float, 64, false>(a, first, s) : launch_rotate<float, float, 128, false>(a, first, s))
            : (head_dim == 64 ? launch_rotate<__nv_bfloat16, __nv_bfloat16, 64, false>(a, first, s)
                              : launch_rotate<__nv_bfloat16, __nv_bfloat16, 128, false>(a, first, s));
    return e == cudaSuccess ? HY_OK : cuda_fail("norm and rotation", e);
}

int hy_paged_kv_write_rotated(const hy_paged_cache* cache, const hy_paged_batch* batch, const hy_rotation* rotation,
                              int rows, int q_heads, int dtype, const void* q_dev, int64_t q_row_stride,
                              int64_t q_head_stride, const void* k_dev, int64_t k_row_stride, int64_t k_head_stride,
                              const void* v_dev, int64_t v_row_stride, int64_t v_head_stride, void* q_out_dev,
                              int64_t q_out_row_stride, int64_t q_out_head_stride, void* stream)
{
    int rc = check_cache(cache);
    if (!rc) rc = check_batch(batch, cache);
    if (!rc) rc = check_rotation(rotation);
    if (!rc) rc = check_dtype(rows, dtype);
    if (!rc) rc = check_heads(rows, q_heads, cache->num_kv_heads);
    if (rc) return rc;
    if (rows == 0 || batch->num_seqs == 0) return HY_OK;
    const int kv_heads = cache->num_kv_heads;
    rc = check_rows("q", q_dev, rows, q_heads, q_row_stride, q_head_stride, dtype);
    if (!rc) rc = check_rows("k", k_dev, rows, kv_heads, k_row_stride, k_head_stride, dtype);
    if (!rc) rc = check_rows("v", v_dev, rows, kv_heads, v_row_stride, v_head_stride, dtype);
    if (!rc) rc = check_rows("q_out", q_out_dev, rows, q_heads, q_out_row_stride, q_out_head_stride, dtype);
    if (!rc) rc = check_apart("q_out", rows, q_heads, cache->head_dim, q_out_row_stride, q_out_head_stride);
    const RowTensor q{"q", q_dev, q_heads, q_row_stride, q_head_stride}, k{"k", k_dev, kv_heads, k_row_stride, k_head_stride},
        v{"v", v_dev, kv_heads, v_row_stride, v_head_stride}, q_out{"q_out", q_out_dev, q_heads, q_out_row_stride, q_out_head_stride};
    if (!rc) rc = check_output(q_out, q, rows, cache->head_dim, dtype);
    if (!rc) rc = check_elsewhere(q_out, k, rows, cache->head_dim, dtype);
    if (!rc) rc = check_elsewhere(q_out, v, rows, cache->head_dim, dtype);
    if (rc) return rc;
    DeviceGuard guard(cache->device);
    if (guard.error() != cudaSuccess) return cuda_fail("device", guard.error());
    RotateArgs a = rotate_args(rotation, rows, q_heads, kv_heads, cache->head_dim);
    a.q = q_dev; a.q_row = q_row_stride; a.q_head = q_head_stride;
    a.k = k_dev; a.k_row = k_row_stride; a.k_head = k_head_stride;
    a.v = v_dev; a.v_row = v_row_stride; a.v_head = v_head_stride;
    a.q_out = q_out_dev; a.qo_row = q_out_row_stride; a.qo_head = q_out_head_stride;
    a.status = cache->status_dev;
    a.c = device_cache(cache);
    a.b = device_batch(batch, rows);
    const cudaError_t e = with_row_type(dtype, cache->dtype, cache->head_dim, [&](auto rt, auto ct, auto d) {
        return launch_rotate<typename decltype(rt)::type, typename decltype(ct)::type, decltype(d)::value, true>(
            a, rotation->rotate_first != 0, static_cast<cudaStream_t>(stream));
    });
    return e == cudaSuccess ? HY_OK : cuda_fail("rotated paged write", e);
}

}  // extern "C"
