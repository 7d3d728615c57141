// C ABI: the training operators (layer norm, gated feed-forward block, dropout).
#include "../../include/kfold_hip.h"

#include <cmath>

#include "api_util.hpp"
#include "train.hpp"

using namespace kfh;

static bool misaligned(const void* p, size_t a = 16) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// most rows / elements one call takes: grids and 64-bit offsets stay far from their ends
static constexpr long long kMaxRows = 1LL << 29;
static constexpr long long kMaxElems = 1LL << 34;

extern "C" {

int kfh_layer_norm_forward(const void* x, const float* weight, const float* bias, void* y, float* mean, float* rstd,
                           long long rows, int C, float eps, int io_dtype, void* stream) {
    if (rows < 0) return fail(KFH_EINVAL, "layer_norm_forward: rows=%lld", rows);
    if (C < 1 || C > 65536) return fail(KFH_EUNSUPPORTED, "layer_norm_forward: C=%d, built for 1..65536", C);
    if (rows > kMaxRows) return fail(KFH_EUNSUPPORTED, "layer_norm_forward: rows=%lld, at most %lld", rows, kMaxRows);
    if (!dtype_ok(io_dtype)) return fail(KFH_EINVAL, "layer_norm_forward: bad io_dtype %d", io_dtype);
    if (rows == 0) return KFH_OK;
    if (!x || !y) return fail(KFH_EINVAL, "layer_norm_forward: null pointer argument");
    if ((mean == nullptr) != (rstd == nullptr)) return fail(KFH_EINVAL, "layer_norm_forward: mean and rstd come together");
    launch_ln_forward(x, io_dtype, weight, bias, y, mean, rstd, rows, C, eps, static_cast<hipStream_t>(stream));
    return check_launch("layer_norm_forward");
}

size_t kfh_layer_norm_backward_workspace_bytes(long long rows, int C) {
    if (rows < 0 || rows > kMaxRows || C < 1 || C > 65536) return 0;
    return align_up((size_t)ln_bwd_blocks(rows) * 2 * C * sizeof(float));
}

int kfh_layer_norm_backward(const void* dy, const void* x, const float* mean, const float* rstd, const float* weight,
                            void* dx, float* dweight, float* dbias, void* workspace, size_t workspace_bytes,
                            long long rows, int C, int io_dtype, void* stream) {
    if (rows < 0) return fail(KFH_EINVAL, "layer_norm_backward: rows=%lld", rows);
    if (C < 1 || C > 65536) return fail(KFH_EUNSUPPORTED, "layer_norm_backward: C=%d, built for 1..65536", C);
    if (rows > kMaxRows) return fail(KFH_EUNSUPPORTED, "layer_norm_backward: rows=%lld, at most %lld", rows, kMaxRows);
    if (!dtype_ok(io_dtype)) return fail(KFH_EINVAL, "layer_norm_backward: bad io_dtype %d", io_dtype);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (rows == 0) {                       // sums over no rows
        launch_ln_backward(nullptr, nullptr, io_dtype, nullptr, nullptr, nullptr, nullptr, dweight, dbias, nullptr, 0, C, s);
        return check_launch("layer_norm_backward");
    }
    if (!dy || !x || !mean || !rstd) return fail(KFH_EINVAL, "layer_norm_backward: null pointer argument");
    if (dx && dx == x) return fail(KFH_EINVAL, "layer_norm_backward: dx may alias dy, not x");
    const size_t need = dweight || dbias ? kfh_layer_norm_backward_workspace_bytes(rows, C) : 0;
    if (need && (!workspace || workspace_bytes < need || misaligned(workspace, 256)))
        return fail(KFH_EINVAL, "layer_norm_backward: workspace %zu bytes, need %zu aligned to 256", workspace ? workspace_bytes : 0, need);
    launch_ln_backward(dy, x, io_dtype, mean, rstd, weight, dx, dweight, dbias, static_cast<float*>(workspace), rows, C, s);
    return check_launch("layer_norm_backward");
}

static int ffn_shape(const char* what, long long rows, int C, int F, int io_dtype) {
    if (rows < 0) return fail(KFH_EINVAL, "%s: rows=%lld", what, rows);
    if (!dtype_ok(io_dtype)) return fail(KFH_EINVAL, "%s: bad io_dtype %d", what, io_dtype);
    if (C < 8 || F < 8 || C % 8 || F % 8 || C > 16384 || F > 65536)
        return fail(KFH_EUNSUPPORTED, "%s: C=%d F=%d, built for multiples of 8 with C <= 16384, F <= 65536", what, C, F);
    if (rows > kMaxRows) return fail(KFH_EUNSUPPORTED, "%s: rows=%lld, at most %lld", what, rows, kMaxRows);
    return KFH_OK;
}

size_t kfh_gated_ffn_workspace_bytes(long long rows, int C, int F, int backward, int io_dtype) {
    if (ffn_shape("gated_ffn_workspace_bytes", rows, C, F, io_dtype) != KFH_OK) return 0;
    return align_up(gated_ffn_ws_bytes(rows, C, F, backward, io_dtype));
}

int kfh_gated_ffn_forward(const void* x, const void* w_in, const void* w_out, void* y, void* workspace,
                          size_t workspace_bytes, long long rows, int C, int F, int io_dtype, void* stream) {
    if (int rc = ffn_shape("gated_ffn_forward", rows, C, F, io_dtype)) return rc;
    if (rows == 0) return KFH_OK;
    if (!x || !w_in || !w_out || !y) return fail(KFH_EINVAL, "gated_ffn_forward: null pointer argument");
    if (misaligned(x) || misaligned(w_in) || misaligned(w_out) || misaligned(y))
        return fail(KFH_EINVAL, "gated_ffn_forward: tensors must be aligned to 16 bytes");
    if (y == x) return fail(KFH_EINVAL, "gated_ffn_forward: y must not alias x");
    const size_t need = kfh_gated_ffn_workspace_bytes(rows, C, F, 0, io_dtype);
    if (need && (!workspace || workspace_bytes < need || misaligned(workspace, 256)))
        return fail(KFH_EINVAL, "gated_ffn_forward: workspace %zu bytes, need %zu aligned to 256",
                    workspace ? workspace_bytes : 0, need);
    launch_gated_ffn_forward(x, w_in, w_out, y, static_cast<char*>(workspace), rows, C, F, io_dtype,
                             static_cast<hipStream_t>(stream));
    return check_launch("gated_ffn_forward");
}

int kfh_gated_ffn_backward(const void* dy, const void* x, const void* w_in, const void* w_out, void* dx, void* dw_in,
                           void* dw_out, int dw_dtype, void* workspace, size_t workspace_bytes, long long rows, int C,
                           int F, int io_dtype, void* stream) {
    if (int rc = ffn_shape("gated_ffn_backward", rows, C, F, io_dtype)) return rc;
    if (!dtype_ok(dw_dtype)) return fail(KFH_EINVAL, "gated_ffn_backward: bad dw_dtype %d", dw_dtype);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (misaligned(dw_in) || misaligned(dw_out))
        return fail(KFH_EINVAL, "gated_ffn_backward: tensors must be aligned to 16 bytes");
    if (rows == 0) {                       // sums over no rows
        const size_t e = dw_dtype == KFH_F32 ? 4 : 2;
        if (dw_in) launch_fill_zero(dw_in, (size_t)2 * F * C * e, s);
        if (dw_out) launch_fill_zero(dw_out, (size_t)F * C * e, s);
        return check_launch("gated_ffn_backward");
    }
    if (!dy || !x || !w_in || !w_out) return fail(KFH_EINVAL, "gated_ffn_backward: null pointer argument");
    if (misaligned(dy) || misaligned(x) || misaligned(w_in) || misaligned(w_out) || misaligned(dx))
        return fail(KFH_EINVAL, "gated_ffn_backward: tensors must be aligned to 16 bytes");
    if (dx && (dx == x || dx == dy)) return fail(KFH_EINVAL, "gated_ffn_backward: dx must not alias x or dy");
    const size_t need = kfh_gated_ffn_workspace_bytes(rows, C, F, 1, io_dtype);
    if (!workspace || workspace_bytes < need || misaligned(workspace, 256))
        return fail(KFH_EINVAL, "gated_ffn_backward: workspace %zu bytes, need %zu aligned to 256",
                    workspace ? workspace_bytes : 0, need);
    launch_gated_ffn_backward(dy, x, w_in, w_out, dx, dw_in, dw_out, dw_dtype, static_cast<char*>(workspace), rows, C, F,
                              io_dtype, s);
    return check_launch("gated_ffn_backward");
}

int kfh_dropout(const void* x, const void* residual, void* y, long long outer, long long shared, long long inner,
                double p, const unsigned long long* seed_dev, unsigned long long seed, unsigned long long offset,
                int io_dtype, void* stream) {
    if (outer < 0 || shared < 0 || inner < 0)
        return fail(KFH_EINVAL, "dropout: shape [%lld, %lld, %lld]", outer, shared, inner);
    if (!(p >= 0.0 && p <= 1.0)) return fail(KFH_EINVAL, "dropout: p=%g is no probability", p);
    if (!dtype_ok(io_dtype)) return fail(KFH_EINVAL, "dropout: bad io_dtype %d", io_dtype);
    if (outer == 0 || shared == 0 || inner == 0) return KFH_OK;
    if (outer > kMaxElems / shared || outer * shared > kMaxElems / inner)
        return fail(KFH_EUNSUPPORTED, "dropout: more than %lld elements", kMaxElems);
    if (!x || !y) return fail(KFH_EINVAL, "dropout: null pointer argument");
    DropArgs a;
    a.x = x; a.residual = residual; a.y = y;
    a.outer = outer; a.shared = shared; a.inner = inner;
    a.t = (uint32_t)std::floor(p * 65536.0 + 0.5);
    a.scale = a.t < 65536u ? (float)(65536.0 / (65536.0 - a.t)) : 0.f;
    a.seed_dev = seed_dev; a.seed = seed; a.offset = offset;
    launch_dropout(a, io_dtype, static_cast<hipStream_t>(stream));
    return check_launch("dropout");
}

}  // extern "C"
