// C ABI of the dense operators (see include/qkan_b200.h): argument validation and scratch carving.
#include <cmath>
#include <initializer_list>

#include "qk_linear.cuh"

namespace {

using qk::check_buffer;
using qk::cuda_fail;
using qk::fail;

bool is_dtype(int t) { return t == QK_F32 || t == QK_BF16; }
constexpr int kMost = 0x7fffff00;  // of a dimension: indices are rounded up to whole tiles (and steps) in 32 bits

int check_linear(const QkLinearDesc* d) {
    if (!d) return fail(QK_ERR_BAD_ARGUMENT, "desc is NULL");
    if (d->rows < 0 || d->in_features < 0 || d->out_features < 0)
        return fail(QK_ERR_BAD_ARGUMENT, "negative dimension (rows=%d in=%d out=%d)", d->rows, d->in_features,
                    d->out_features);
    if (d->rows > kMost || d->in_features > kMost || d->out_features > kMost)
        return fail(QK_ERR_UNSUPPORTED, "a dimension exceeds %d (rows=%d in=%d out=%d)", kMost, d->rows, d->in_features,
                    d->out_features);
    if (!is_dtype(d->io_dtype)) return fail(QK_ERR_BAD_ARGUMENT, "io_dtype %d is neither QK_F32 nor QK_BF16", d->io_dtype);
    if (d->activation < QK_ACT_NONE || d->activation > QK_ACT_SIGMOID)
        return fail(QK_ERR_BAD_ARGUMENT, "activation %d is not a QkActivation value", d->activation);
    if (d->flags & ~(uint32_t)QK_LINEAR_ROUND_GRADS) return fail(QK_ERR_BAD_ARGUMENT, "unknown flag bits 0x%x", d->flags);
    return QK_OK;
}

int check_norm(const QkNormDesc* d) {
    if (!d) return fail(QK_ERR_BAD_ARGUMENT, "desc is NULL");
    if (d->rows < 0 || d->dim < 1) return fail(QK_ERR_BAD_ARGUMENT, "rows=%d dim=%d: rows >= 0 and dim >= 1 are wanted", d->rows, d->dim);
    if (d->dim > kMost) return fail(QK_ERR_UNSUPPORTED, "dim=%d exceeds %d", d->dim, kMost);
    if (!is_dtype(d->io_dtype) || !is_dtype(d->param_dtype))
        return fail(QK_ERR_BAD_ARGUMENT, "io_dtype %d / param_dtype %d is neither QK_F32 nor QK_BF16", d->io_dtype, d->param_dtype);
    if (!(d->eps >= 0.f) || std::isinf(d->eps)) return fail(QK_ERR_BAD_ARGUMENT, "eps must be >= 0 and finite");
    if (d->flags) return fail(QK_ERR_BAD_ARGUMENT, "unknown flag bits 0x%x", d->flags);
    return QK_OK;
}

// The products read bfloat16 rows of whole 16-byte words where they lie, by TMA, which wants them aligned.
int check_aligned(const void* p, int width, int io_dtype, const char* what) {
    if (qk::reads_in_place(width, io_dtype) && (uintptr_t)p % 16)
        return fail(QK_ERR_BAD_ARGUMENT, "%s must be 16-byte aligned (its rows are whole 16-byte words)", what);
    return QK_OK;
}

// every pointer on a boundary of its element; a pointer that is not wanted is NULL, which is one
int check_elements(std::initializer_list<const void*> all, size_t bytes, const char* what) {
    uintptr_t bits = 0;
    for (const void* p : all) bits |= (uintptr_t)p;
    return bits % bytes ? fail(QK_ERR_BAD_ARGUMENT, "%s must be %zu-byte aligned", what, bytes) : QK_OK;
}

size_t norm_scratch(const QkNormDesc& d) {
    return qk::align256((size_t)2 * qk::norm_slices(d.rows, d.dim, d.io_dtype, d.param_dtype) * d.dim * sizeof(float));
}

// a size of 0 says that the descriptor was refused, so "none" is 1
size_t at_least_one(size_t n) { return n ? n : 1; }
int check_scratch(const void* p, size_t have, size_t need) {
    return need ? check_buffer(p, have, need, "workspace") : QK_OK;
}

// zeros for a gradient that sums over nothing
cudaError_t zero(void* p, size_t n, int dtype, cudaStream_t st) {
    return p && n ? cudaMemsetAsync(p, 0, n * qk::dtype_bytes(dtype), st) : cudaSuccess;
}

}  // namespace

extern "C" {

size_t qk_linear_forward_workspace_bytes(const QkLinearDesc* desc) {
    return check_linear(desc) ? 0 : at_least_one(qk::linear_forward_scratch(*desc));
}

int qk_linear_forward(const QkLinearDesc* desc, const void* x, const void* weight, const void* bias,
                      const void* residual, void* y, void* tape, void* ws, size_t ws_bytes, void* stream) {
    int rc = check_linear(desc);
    if (rc) return rc;
    const QkLinearDesc& d = *desc;
    if (d.rows == 0 || d.out_features == 0) return QK_OK;
    if (!y) return fail(QK_ERR_BAD_ARGUMENT, "y is NULL");
    if (d.in_features && (!x || !weight)) return fail(QK_ERR_BAD_ARGUMENT, "x or weight is NULL");
    // the tape's half is as wide as bfloat16
    if ((rc = check_elements({x, weight, bias, residual, y, tape}, qk::dtype_bytes(d.io_dtype), "every tensor"))) return rc;
    if ((rc = check_aligned(x, d.in_features, d.io_dtype, "x"))) return rc;
    if ((rc = check_aligned(weight, d.in_features, d.io_dtype, "weight"))) return rc;
    rc = check_scratch(ws, ws_bytes, qk::linear_forward_scratch(d));
    if (rc) return rc;
    qk::LinearArgs a{};
    a.rows = d.rows, a.in = d.in_features, a.out = d.out_features, a.act = d.activation, a.io_dtype = d.io_dtype;
    a.x = x, a.w = weight, a.bias = bias, a.residual = residual, a.y = y;
    a.tape = d.activation == QK_ACT_NONE ? nullptr : tape;
    a.scratch = ws;
    const cudaError_t e = qk::launch_linear_forward(a, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? QK_OK : cuda_fail(e, "linear forward launch");
}

size_t qk_linear_backward_workspace_bytes(const QkLinearDesc* desc) {
    return check_linear(desc) ? 0 : at_least_one(qk::linear_backward_scratch(*desc));
}

int qk_linear_backward(const QkLinearDesc* desc, const void* x, const void* weight, const void* tape, const void* gy,
                       void* gx, void* gw, void* gb, void* ws, size_t ws_bytes, void* stream) {
    int rc = check_linear(desc);
    if (rc) return rc;
    const QkLinearDesc& d = *desc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d.in_features == 0) gx = gw = nullptr;  // empty tensors
    if (d.rows == 0 || d.out_features == 0) {  // sums over nothing
        cudaError_t e = zero(gx, (size_t)d.rows * d.in_features, d.io_dtype, st);
        if (e == cudaSuccess) e = zero(gw, (size_t)d.out_features * d.in_features, d.io_dtype, st);
        if (e == cudaSuccess) e = zero(gb, d.out_features, d.io_dtype, st);
        return e == cudaSuccess ? QK_OK : cuda_fail(e, "memset gradients");
    }
    if (!gx && !gw && !gb) return QK_OK;
    if (!gy) return fail(QK_ERR_BAD_ARGUMENT, "grad_y is NULL");
    if (d.activation != QK_ACT_NONE && !tape) return fail(QK_ERR_BAD_ARGUMENT, "tape is NULL");
    if ((gx && !weight) || (gw && !x)) return fail(QK_ERR_BAD_ARGUMENT, "x or weight is NULL");
    if ((rc = check_elements({x, weight, tape, gy, gx, gw, gb}, qk::dtype_bytes(d.io_dtype), "every tensor"))) return rc;
    if (gw && (rc = check_aligned(x, d.in_features, d.io_dtype, "x"))) return rc;
    if (gx && (rc = check_aligned(weight, d.in_features, d.io_dtype, "weight"))) return rc;
    if ((gx || gw) && (rc = check_aligned(gy, d.out_features, d.io_dtype, "grad_y"))) return rc;
    rc = check_scratch(ws, ws_bytes, qk::linear_backward_scratch(d));
    if (rc) return rc;
    qk::LinearArgs a{};
    a.rows = d.rows, a.in = d.in_features, a.out = d.out_features, a.act = d.activation, a.io_dtype = d.io_dtype;
    a.flags = d.flags;
    a.x = x, a.w = weight, a.tape = const_cast<void*>(tape), a.gy = gy;
    a.gx = gx, a.gw = gw, a.gb = gb, a.scratch = ws;
    const cudaError_t e = qk::launch_linear_backward(a, st);
    return e == cudaSuccess ? QK_OK : cuda_fail(e, "linear backward launch");
}

int qk_linear_plan(const QkLinearDesc* desc, int product, QkLinearPlan* plan) {
    const int rc = check_linear(desc);
    if (rc) return rc;
    if (product < 0 || product > 2 || !plan) return fail(QK_ERR_BAD_ARGUMENT, "product %d is none of 0, 1, 2, or plan is NULL", product);
    *plan = qk::linear_plan(*desc, product);
    return QK_OK;
}

int qk_dense_status(void* stream) {
    unsigned n = 0;
    const cudaError_t e = qk::gemm_gave_up(&n, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(e, "dense status");
    return n ? fail(QK_ERR_LAUNCH, "%u waits of the linear map's kernels ran out; their results are not valid", n) : QK_OK;
}

int qk_layer_norm_forward(const QkNormDesc* desc, const void* x, const void* weight, const void* bias, void* y,
                          float* stats, void* stream) {
    int rc = check_norm(desc);
    if (rc) return rc;
    const QkNormDesc& d = *desc;
    if (d.rows == 0) return QK_OK;
    if (!x || !y) return fail(QK_ERR_BAD_ARGUMENT, "x or y is NULL");
    if ((rc = check_elements({x, y}, qk::dtype_bytes(d.io_dtype), "x and y"))) return rc;
    if ((rc = check_elements({weight, bias}, qk::dtype_bytes(d.param_dtype), "weight and bias"))) return rc;
    if ((rc = check_elements({stats}, 8, "stats"))) return rc;
    qk::NormArgs a{};
    a.rows = d.rows, a.dim = d.dim, a.io_dtype = d.io_dtype, a.param_dtype = d.param_dtype, a.eps = d.eps;
    a.x = x, a.w = weight, a.b = bias, a.y = y;
    a.stats_out = reinterpret_cast<float2*>(stats);
    const cudaError_t e = qk::launch_norm_forward(a, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? QK_OK : cuda_fail(e, "layer norm forward launch");
}

size_t qk_layer_norm_backward_workspace_bytes(const QkNormDesc* desc) {
    if (check_norm(desc)) return 0;
    return desc->rows == 0 ? 1 : norm_scratch(*desc);
}

int qk_layer_norm_backward(const QkNormDesc* desc, const void* x, const void* weight, const float* stats,
                           const void* gy, void* gx, void* gw, void* gb, void* ws, size_t ws_bytes, void* stream) {
    int rc = check_norm(desc);
    if (rc) return rc;
    const QkNormDesc& d = *desc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d.rows == 0) {
        cudaError_t e = zero(gw, d.dim, d.param_dtype, st);
        if (e == cudaSuccess) e = zero(gb, d.dim, d.param_dtype, st);
        return e == cudaSuccess ? QK_OK : cuda_fail(e, "memset gradients");
    }
    if (!gx && !gw && !gb) return QK_OK;
    if (!x || !stats || !gy) return fail(QK_ERR_BAD_ARGUMENT, "x, stats or grad_y is NULL");
    if ((rc = check_elements({x, gy, gx}, qk::dtype_bytes(d.io_dtype), "x, grad_y and grad_x"))) return rc;
    if ((rc = check_elements({weight, gw, gb}, qk::dtype_bytes(d.param_dtype), "weight and its gradients"))) return rc;
    if ((rc = check_elements({stats}, 8, "stats"))) return rc;
    qk::NormArgs a{};
    a.rows = d.rows, a.dim = d.dim, a.io_dtype = d.io_dtype, a.param_dtype = d.param_dtype, a.eps = d.eps;
    a.x = x, a.w = weight, a.gy = gy, a.gx = gx, a.gw = gw, a.gb = gb;
    a.stats = reinterpret_cast<const float2*>(stats);
    if (gw || gb) {
        rc = check_buffer(ws, ws_bytes, norm_scratch(d), "workspace");
        if (rc) return rc;
        a.part = static_cast<float*>(ws);
    }
    const cudaError_t e = qk::launch_norm_backward(a, st);
    return e == cudaSuccess ? QK_OK : cuda_fail(e, "layer norm backward launch");
}

}  // extern "C"
