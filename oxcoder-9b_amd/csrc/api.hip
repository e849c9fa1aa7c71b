// extern "C" entry points of libkq.so (declared in include/kq.h): argument checks, then launches.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include "kq_internal.h"

namespace kq {

// Compute units of the current device (cached per device).
int device_cus() {
    static int cus[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if (!cus[dev]) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
        cus[dev] = n;
    }
    return cus[dev];
}

static thread_local char g_err[512];

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof g_err, fmt, ap);
    va_end(ap);
    return code;
}

int check_ptr(const void* p, size_t align, const char* what, const char* fn) {
    if (!p) return fail(KQ_ERR_ARG, "%s: %s is NULL", fn, what);
    if (reinterpret_cast<uintptr_t>(p) % align)
        return fail(KQ_ERR_ARG, "%s: %s must be %zu-byte aligned", fn, what, align);
    return KQ_OK;
}

// Shape rules of the packed tensor (q4pack.py:97-103: rows % 8, ne0 % 256; type in {12, 14}).
int check_matrix(const void* w, int R, int C, int type, const char* fn) {
    if (type != KQ_TYPE_Q4_K && type != KQ_TYPE_Q6_K)
        return fail(KQ_ERR_ARG, "%s: type %d is not Q4_K (12) or Q6_K (14)", fn, type);
    if (R <= 0 || R % 8) return fail(KQ_ERR_ARG, "%s: R=%d must be a positive multiple of 8", fn, R);
    if (C <= 0 || C % 256) return fail(KQ_ERR_ARG, "%s: C=%d must be a positive multiple of 256", fn, C);
    if (C > 61440) return fail(KQ_ERR_ARG, "%s: C=%d exceeds the supported maximum 61440", fn, C);
    return check_ptr(w, 16, "w", fn);
}

int check_launch(const char* fn) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(KQ_ERR_HIP, "%s: launch failed: %s", fn, hipGetErrorString(e));
    g_err[0] = 0;
    return KQ_OK;
}

}  // namespace kq

using namespace kq;

#define KQ_TRY(expr)            \
    do {                        \
        const int _rc = (expr); \
        if (_rc) return _rc;    \
    } while (0)

extern "C" {

const char* kq_last_error(void) { return g_err; }

int kq_version(void) { return (1 << 16) | 0; }

#ifndef KQ_SOURCE_HASH
#define KQ_SOURCE_HASH "unknown"
#endif
const char* kq_source_hash(void) { return KQ_SOURCE_HASH; }

int kq_gemv(const void* w, int R, int C, int type, const float* x, float* y, void* stream) {
    static const char* fn = "kq_gemv";
    KQ_TRY(check_matrix(w, R, C, type, fn));
    KQ_TRY(check_ptr(x, 4, "x", fn));
    KQ_TRY(check_ptr(y, 4, "y", fn));
    if (R / 8 > (1 << 27)) return fail(KQ_ERR_ARG, "%s: R=%d too large for one call", fn, R);
    const uint8_t* wb = static_cast<const uint8_t*>(w);
    launch_gemv_f32_group(1, &wb, &R, C, type, x, &y, as_stream(stream));
    return check_launch(fn);
}

int kq_gemv_multi(int n, const void* const* w, const int* R, int C, const int* type,
                  const float* x, float* const* y, void* stream) {
    static const char* fn = "kq_gemv_multi";
    if (n < 1 || n > 3) return fail(KQ_ERR_ARG, "%s: n=%d must be 1..3", fn, n);
    if (!w || !R || !type || !y) return fail(KQ_ERR_ARG, "%s: NULL array argument", fn);
    int64_t tiles = 0;
    for (int i = 0; i < n; i++) {
        KQ_TRY(check_matrix(w[i], R[i], C, type[i], fn));
        KQ_TRY(check_ptr(y[i], 4, "y[i]", fn));
        tiles += R[i] / 8;
    }
    if (tiles > (1 << 27)) return fail(KQ_ERR_ARG, "%s: too many rows in one call", fn);
    KQ_TRY(check_ptr(x, 4, "x", fn));
    // both weight types (a Q4_K_M layer's q, k and Q6_K v): one launch where possible
    {
        const uint8_t* wa[3];
        for (int i = 0; i < n; i++) wa[i] = static_cast<const uint8_t*>(w[i]);
        if (launch_gemv_f32_mixed(n, wa, R, type, C, x, y, as_stream(stream))) return check_launch(fn);
    }
    // matrices of the same type share a launch
    for (int ty : {KQ_TYPE_Q4_K, KQ_TYPE_Q6_K}) {
        const uint8_t* ws[3];
        int rs[3];
        float* ys[3];
        int k = 0;
        for (int i = 0; i < n; i++)
            if (type[i] == ty) { ws[k] = static_cast<const uint8_t*>(w[i]); rs[k] = R[i]; ys[k] = y[i]; k++; }
        if (k) launch_gemv_f32_group(k, ws, rs, C, ty, x, ys, as_stream(stream));
    }
    return check_launch(fn);
}

int kq_gemv_rows(int n, const void* const* w, const int* R, int C, const int* type, const float* x, int64_t ldx,
                 int N, float* const* y, const int64_t* ldy, void* stream) {
    static const char* fn = "kq_gemv_rows";
    if (n < 1 || n > 3) return fail(KQ_ERR_ARG, "%s: n=%d must be 1..3", fn, n);
    if (!w || !R || !type || !y || !ldy) return fail(KQ_ERR_ARG, "%s: NULL array argument", fn);
    if (N < 1) return fail(KQ_ERR_ARG, "%s: N=%d must be positive", fn, N);
    if (N == 1) return kq_gemv_multi(n, w, R, C, type, x, y, stream);
    int64_t tiles = 0;
    for (int i = 0; i < n; i++) {
        KQ_TRY(check_matrix(w[i], R[i], C, type[i], fn));
        KQ_TRY(check_ptr(y[i], 4, "y[i]", fn));
        if (ldy[i] < R[i]) return fail(KQ_ERR_ARG, "%s: ldy[%d] is smaller than R", fn, i);
        tiles += R[i] / 8;
    }
    if (tiles > (1 << 27)) return fail(KQ_ERR_ARG, "%s: too many rows in one call", fn);
    if (ldx < 0) return fail(KQ_ERR_ARG, "%s: ldx=%lld is negative", fn, (long long)ldx);
    KQ_TRY(check_ptr(x, 4, "x", fn));
    for (int ty : {KQ_TYPE_Q4_K, KQ_TYPE_Q6_K}) {
        const uint8_t* ws[3];
        int rs[3];
        float* ys[3];
        int64_t ls[3];
        int k = 0;
        for (int i = 0; i < n; i++)
            if (type[i] == ty) {
                ws[k] = static_cast<const uint8_t*>(w[i]); rs[k] = R[i]; ys[k] = y[i]; ls[k] = ldy[i];
                k++;
            }
        if (k) launch_gemv_f32_rows(k, ws, rs, C, ty, x, ldx, N, ys, ls, as_stream(stream));
    }
    return check_launch(fn);
}

int kq_q8k_quantize(const float* x, int64_t ldx, int C, int N, void* xq, void* stream) {
    static const char* fn = "kq_q8k_quantize";
    if (C <= 0 || C % 256) return fail(KQ_ERR_ARG, "%s: C=%d must be a positive multiple of 256", fn, C);
    if (N <= 0) return fail(KQ_ERR_ARG, "%s: N=%d must be positive", fn, N);
    if (ldx < C) return fail(KQ_ERR_ARG, "%s: ldx=%lld is smaller than C=%d", fn, (long long)ldx, C);
    if ((int64_t)N * (C / 256) > 0x7fffffffLL)
        return fail(KQ_ERR_ARG, "%s: N*C/256 exceeds 2^31-1 blocks", fn);
    KQ_TRY(check_ptr(x, 4, "x", fn));
    KQ_TRY(check_ptr(xq, 4, "xq", fn));
    launch_q8k_quantize(x, ldx, C, N, static_cast<uint8_t*>(xq), as_stream(stream));
    return check_launch(fn);
}

int kq_rms_q8k(float* h, const float* residual, int add, const float* w, int D, int N, int64_t ld, float* xn,
               void* xq, void* stream) {
    static const char* fn = "kq_rms_q8k";
    if (D <= 0 || D % 256 || D > 16384)   // the kernel's per-thread row share (RMS_DMAX)
        return fail(KQ_ERR_ARG, "%s: D=%d must be a positive multiple of 256, at most 16384", fn, D);
    if (N <= 0 || N > 65535) return fail(KQ_ERR_ARG, "%s: N=%d must be 1..65535", fn, N);
    if (ld < D) return fail(KQ_ERR_ARG, "%s: ld=%lld is smaller than D=%d", fn, (long long)ld, D);
    KQ_TRY(check_ptr(h, 4, "h", fn));
    KQ_TRY(check_ptr(w, 4, "w", fn));
    KQ_TRY(check_ptr(xq, 4, "xq", fn));
    if (add) KQ_TRY(check_ptr(residual, 4, "residual", fn));
    if (xn) KQ_TRY(check_ptr(xn, 4, "xn", fn));
    launch_rms_q8k(h, add ? residual : nullptr, add ? 1 : 0, w, D, N, ld, xn, static_cast<uint8_t*>(xq),
                   as_stream(stream));
    return check_launch(fn);
}

int kq_swiglu_q8k(const float* gate, const float* up, int n, int N, int64_t ld, float* y, void* xq,
                  void* stream) {
    static const char* fn = "kq_swiglu_q8k";
    if (n <= 0 || n % 256) return fail(KQ_ERR_ARG, "%s: n=%d must be a positive multiple of 256", fn, n);
    if (N <= 0) return fail(KQ_ERR_ARG, "%s: N=%d must be positive", fn, N);
    if (ld < n) return fail(KQ_ERR_ARG, "%s: ld=%lld is smaller than n=%d", fn, (long long)ld, n);
    if ((int64_t)N * (n / 256) > 0x7fffffffLL) return fail(KQ_ERR_ARG, "%s: N*n/256 exceeds 2^31-1 blocks", fn);
    KQ_TRY(check_ptr(gate, 4, "gate", fn));
    KQ_TRY(check_ptr(up, 4, "up", fn));
    KQ_TRY(check_ptr(xq, 4, "xq", fn));
    if (y) KQ_TRY(check_ptr(y, 4, "y", fn));
    launch_swiglu_q8k(gate, up, n, N, ld, y, static_cast<uint8_t*>(xq), as_stream(stream));
    return check_launch(fn);
}

size_t kq_argmax_workspace(void) { return argmax_workspace_bytes(); }

static int check_argmax_ws(const void* ws, const int* out, const char* fn) {
    KQ_TRY(check_ptr(ws, 256, "ws", fn));
    return check_ptr(out, 4, "out", fn);
}

int kq_argmax(const float* y, int n, void* ws, int* out, void* stream) {
    static const char* fn = "kq_argmax";
    if (n <= 0) return fail(KQ_ERR_ARG, "%s: n=%d must be positive", fn, n);
    KQ_TRY(check_ptr(y, 4, "y", fn));
    KQ_TRY(check_argmax_ws(ws, out, fn));
    launch_argmax(y, n, static_cast<uint8_t*>(ws), out, as_stream(stream));
    return check_launch(fn);
}

int kq_gemv_q8k_argmax(const void* w, int R, int C, int type, const void* xq, float* y, void* ws, int* out,
                       void* stream) {
    static const char* fn = "kq_gemv_q8k_argmax";
    KQ_TRY(check_matrix(w, R, C, type, fn));
    KQ_TRY(check_ptr(xq, 4, "xq", fn));
    KQ_TRY(check_ptr(y, 4, "y", fn));
    KQ_TRY(check_argmax_ws(ws, out, fn));
    launch_gemv_q8k_argmax(static_cast<const uint8_t*>(w), R, C, type, static_cast<const uint8_t*>(xq), y,
                           static_cast<uint8_t*>(ws), out, as_stream(stream));
    return check_launch(fn);
}

int kq_gemv_q8k(const void* w, int R, int C, int type, const void* xq, int N, float* y,
                int64_t ldy, void* stream) {
    static const char* fn = "kq_gemv_q8k";
    KQ_TRY(check_matrix(w, R, C, type, fn));
    if (N < 1 || N > KQ_MAX_BATCH) return fail(KQ_ERR_ARG, "%s: N=%d must be 1..%d", fn, N, KQ_MAX_BATCH);
    if (N > 1 && ldy < R) return fail(KQ_ERR_ARG, "%s: ldy=%lld is smaller than R=%d", fn, (long long)ldy, R);
    if (R / 8 > (1 << 27)) return fail(KQ_ERR_ARG, "%s: R=%d too large for one call", fn, R);
    KQ_TRY(check_ptr(xq, 4, "xq", fn));
    KQ_TRY(check_ptr(y, 4, "y", fn));
    launch_gemv_q8k(static_cast<const uint8_t*>(w), R, C, type, static_cast<const uint8_t*>(xq), N, y,
                    ldy, as_stream(stream));
    return check_launch(fn);
}

int kq_gemv_q8k_x(int n, const void* const* w, const int* R, int C, const int* type, const float* x,
                  float* const* y, void* xq, void* stream) {
    static const char* fn = "kq_gemv_q8k_x";
    if (n < 1 || n > 3) return fail(KQ_ERR_ARG, "%s: n=%d must be 1..3", fn, n);
    if (!w || !R || !type || !y) return fail(KQ_ERR_ARG, "%s: NULL array argument", fn);
    int64_t tiles = 0;
    for (int i = 0; i < n; i++) {
        KQ_TRY(check_matrix(w[i], R[i], C, type[i], fn));
        KQ_TRY(check_ptr(y[i], 4, "y[i]", fn));
        tiles += R[i] / 8;
    }
    if (tiles > (1 << 27)) return fail(KQ_ERR_ARG, "%s: too many rows in one call", fn);
    KQ_TRY(check_ptr(x, 16, "x", fn));
    if (xq) KQ_TRY(check_ptr(xq, 4, "xq", fn));
    uint8_t* xq8 = static_cast<uint8_t*>(xq);
    if (C > 4096) {   // more than one column pass: the quantizer's own launch, then the grouped GEMV
        if (!xq8) return fail(KQ_ERR_ARG, "%s: C=%d > 4096 needs the xq buffer", fn, C);
        launch_q8k_quantize(x, C, C, 1, xq8, as_stream(stream));
        const int64_t ld[3] = {R[0], n > 1 ? R[1] : 0, n > 2 ? R[2] : 0};
        return kq_gemv_q8k_multi(n, w, R, C, type, xq8, 1, y, ld, stream);
    }
    {   // both weight types: one launch where possible
        const uint8_t* wa[3];
        for (int i = 0; i < n; i++) wa[i] = static_cast<const uint8_t*>(w[i]);
        if (launch_gemv_q8k_x_mixed(n, wa, R, type, C, x, y, xq8, as_stream(stream))) return check_launch(fn);
    }
    bool first = true;
    for (int ty : {KQ_TYPE_Q4_K, KQ_TYPE_Q6_K}) {
        const uint8_t* ws[3];
        int rs[3];
        float* ys[3];
        int k = 0;
        for (int i = 0; i < n; i++)
            if (type[i] == ty) { ws[k] = static_cast<const uint8_t*>(w[i]); rs[k] = R[i]; ys[k] = y[i]; k++; }
        if (!k) continue;
        launch_gemv_q8k_x_group(k, ws, rs, C, ty, x, ys, first ? xq8 : nullptr, as_stream(stream));
        first = false;
    }
    return check_launch(fn);
}

int kq_gemv_q8k_multi(int n, const void* const* w, const int* R, int C, const int* type, const void* xq,
                      int N, float* const* y, const int64_t* ldy, void* stream) {
    static const char* fn = "kq_gemv_q8k_multi";
    if (n < 1 || n > 3) return fail(KQ_ERR_ARG, "%s: n=%d must be 1..3", fn, n);
    if (!w || !R || !type || !y || !ldy) return fail(KQ_ERR_ARG, "%s: NULL array argument", fn);
    if (N < 1 || N > KQ_MAX_BATCH) return fail(KQ_ERR_ARG, "%s: N=%d must be 1..%d", fn, N, KQ_MAX_BATCH);
    int64_t tiles = 0;
    for (int i = 0; i < n; i++) {
        KQ_TRY(check_matrix(w[i], R[i], C, type[i], fn));
        KQ_TRY(check_ptr(y[i], 4, "y[i]", fn));
        if (N > 1 && ldy[i] < R[i]) return fail(KQ_ERR_ARG, "%s: ldy[%d] is smaller than R", fn, i);
        tiles += R[i] / 8;
    }
    if (tiles > (1 << 27)) return fail(KQ_ERR_ARG, "%s: too many rows in one call", fn);
    KQ_TRY(check_ptr(xq, 4, "xq", fn));
    // both weight types (a Q4_K_M layer's q, k and Q6_K v): one launch where possible
    {
        const uint8_t* wa[3];
        for (int i = 0; i < n; i++) wa[i] = static_cast<const uint8_t*>(w[i]);
        const uint8_t* x8 = static_cast<const uint8_t*>(xq);
        if (N == 1 ? launch_gemv_q8k_mixed(n, wa, R, type, C, x8, y, as_stream(stream))
                   : launch_gemv_mfma_mixed(n, wa, R, type, C, x8, N, y, ldy, as_stream(stream)))
            return check_launch(fn);
    }
    // matrices of the same type share a launch
    for (int ty : {KQ_TYPE_Q4_K, KQ_TYPE_Q6_K}) {
        const uint8_t* ws[3];
        int rs[3];
        float* ys[3];
        int64_t ls[3];
        int k = 0;
        for (int i = 0; i < n; i++)
            if (type[i] == ty) {
                ws[k] = static_cast<const uint8_t*>(w[i]); rs[k] = R[i]; ys[k] = y[i]; ls[k] = N > 1 ? ldy[i] : R[i];
                k++;
            }
        if (k) launch_gemv_q8k_group(k, ws, rs, C, ty, static_cast<const uint8_t*>(xq), N, ys, ls, as_stream(stream));
    }
    return check_launch(fn);
}

// A GEMM's matrix, M and output (the activations are checked by the caller).
static int check_gemm_out(const void* w, int R, int C, int type, int M, const float* y, int64_t ldy, const char* fn) {
    KQ_TRY(check_matrix(w, R, C, type, fn));
    if (M < 1) return fail(KQ_ERR_ARG, "%s: M=%d must be positive", fn, M);
    if (M > 1 && ldy < R) return fail(KQ_ERR_ARG, "%s: ldy=%lld is smaller than R=%d", fn, (long long)ldy, R);
    KQ_TRY(check_ptr(y, 4, "y", fn));
    if ((int64_t)M * (C / 256) > 0x7fffffffLL) return fail(KQ_ERR_ARG, "%s: M*C/256 too large", fn);
    return KQ_OK;
}

static int check_gemm(const void* w, int R, int C, int type, const void* xq, int M, const float* y, int64_t ldy,
                      const char* fn) {
    KQ_TRY(check_gemm_out(w, R, C, type, M, y, ldy, fn));
    return check_ptr(xq, 4, "xq", fn);
}

int kq_gemm_q8k(const void* w, int R, int C, int type, const void* xq, int M, float* y,
                int64_t ldy, void* stream) {
    static const char* fn = "kq_gemm_q8k";
    KQ_TRY(check_gemm(w, R, C, type, xq, M, y, ldy, fn));
    launch_gemm_q8k(static_cast<const uint8_t*>(w), R, C, type, static_cast<const uint8_t*>(xq), M, y, ldy,
                    nullptr, as_stream(stream));
    return check_launch(fn);
}

size_t kq_gemm_q8k_workspace(int R, int C, int M) {
    if (R < 8 || R % 8 || C < 256 || C % 256 || M < 1) return 0;
    return gemm_q8k_workspace(R, C, M);
}

int kq_gemm_q8k_ws(const void* w, int R, int C, int type, const void* xq, int M, float* y,
                   int64_t ldy, void* ws, size_t ws_bytes, void* stream) {
    static const char* fn = "kq_gemm_q8k_ws";
    KQ_TRY(check_gemm(w, R, C, type, xq, M, y, ldy, fn));
    KQ_TRY(check_ptr(ws, 256, "ws", fn));
    const size_t need = gemm_q8k_workspace(R, C, M);
    if (ws_bytes < need) return fail(KQ_ERR_ARG, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, need);
    launch_gemm_q8k(static_cast<const uint8_t*>(w), R, C, type, static_cast<const uint8_t*>(xq), M, y, ldy,
                    static_cast<uint8_t*>(ws), as_stream(stream));
    return check_launch(fn);
}

size_t kq_gemm_q8k_multi_workspace(int n, const int* R, int C, int M) {
    if (n < 1 || n > 3 || !R || C < 256 || C % 256 || M < 1) return 0;
    for (int i = 0; i < n; i++)
        if (R[i] < 8 || R[i] % 8) return 0;
    return gemm_q8k_group_workspace(n, R, C, M);
}

int kq_gemm_q8k_multi_ws(int n, const void* const* w, const int* R, int C, const int* type, const void* xq, int M,
                         float* const* y, const int64_t* ldy, void* ws, size_t ws_bytes, void* stream) {
    static const char* fn = "kq_gemm_q8k_multi_ws";
    if (n < 1 || n > 3) return fail(KQ_ERR_ARG, "%s: n=%d must be 1..3", fn, n);
    if (!w || !R || !type || !y || !ldy) return fail(KQ_ERR_ARG, "%s: NULL array argument", fn);
    for (int i = 0; i < n; i++) KQ_TRY(check_gemm(w[i], R[i], C, type[i], xq, M, y[i], ldy[i], fn));
    KQ_TRY(check_ptr(ws, 256, "ws", fn));
    const size_t need = gemm_q8k_group_workspace(n, R, C, M);
    if (ws_bytes < need) return fail(KQ_ERR_ARG, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, need);
    const uint8_t* wb[3];
    for (int i = 0; i < n; i++) wb[i] = static_cast<const uint8_t*>(w[i]);
    launch_gemm_q8k_group(n, wb, R, C, type, static_cast<const uint8_t*>(xq), M, y, ldy, static_cast<uint8_t*>(ws),
                          as_stream(stream));
    return check_launch(fn);
}

size_t kq_gemm_f32_multi_workspace(int n, const int* R, int C, int M) {
    if (!kq_gemm_q8k_multi_workspace(n, R, C, M)) return 0;
    return gemm_f32_group_workspace(n, R, C, M);
}

int kq_gemm_f32_multi(int n, const void* const* w, const int* R, int C, const int* type, const float* x, int64_t ldx,
                      int M, float* const* y, const int64_t* ldy, void* ws, size_t ws_bytes, void* stream) {
    static const char* fn = "kq_gemm_f32_multi";
    if (n < 1 || n > 3) return fail(KQ_ERR_ARG, "%s: n=%d must be 1..3", fn, n);
    if (!w || !R || !type || !y || !ldy) return fail(KQ_ERR_ARG, "%s: NULL array argument", fn);
    KQ_TRY(check_ptr(x, 4, "x", fn));
    if (M > 1 && ldx < C) return fail(KQ_ERR_ARG, "%s: ldx=%lld is smaller than C=%d", fn, (long long)ldx, C);
    for (int i = 0; i < n; i++) KQ_TRY(check_gemm_out(w[i], R[i], C, type[i], M, y[i], ldy[i], fn));
    KQ_TRY(check_ptr(ws, 256, "ws", fn));
    const size_t need = gemm_f32_group_workspace(n, R, C, M);
    if (ws_bytes < need) return fail(KQ_ERR_ARG, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, need);
    const uint8_t* wb[3];
    for (int i = 0; i < n; i++) wb[i] = static_cast<const uint8_t*>(w[i]);
    launch_gemm_f32_group(n, wb, R, C, type, x, ldx, M, y, ldy, static_cast<uint8_t*>(ws), as_stream(stream));
    return check_launch(fn);
}

int kq_gemm_q8k_static(const void* w, int R, int C, int type, const void* xq, int M, float* y,
                       int64_t ldy, void* stream) {
    static const char* fn = "kq_gemm_q8k_static";
    KQ_TRY(check_gemm(w, R, C, type, xq, M, y, ldy, fn));
    const size_t need = gemm_q8k_workspace(R, C, M);
    if (need > KQ_GEMM_STATIC_SCRATCH_BYTES)
        return fail(KQ_ERR_ARG,
                    "%s: R=%d C=%d M=%d needs %zu bytes of workspace, more than the %u-byte static scratch "
                    "(split M into chunks, or use kq_gemm_q8k_ws)", fn, R, C, M, need,
                    (unsigned)KQ_GEMM_STATIC_SCRATCH_BYTES);
    uint8_t* ws = nullptr;
    KQ_TRY(gemm_static_scratch(&ws, fn));
    launch_gemm_q8k(static_cast<const uint8_t*>(w), R, C, type, static_cast<const uint8_t*>(xq), M, y, ldy, ws,
                    as_stream(stream));
    return check_launch(fn);
}

int kq_subblock_sums(const void* w, int R, int C, int type, const void* xq, int N, int32_t* sums,
                     void* stream) {
    static const char* fn = "kq_subblock_sums";
    KQ_TRY(check_matrix(w, R, C, type, fn));
    if (N < 1) return fail(KQ_ERR_ARG, "%s: N=%d must be positive", fn, N);
    KQ_TRY(check_ptr(xq, 4, "xq", fn));
    KQ_TRY(check_ptr(sums, 4, "sums", fn));
    launch_subblock_sums(static_cast<const uint8_t*>(w), R, C, type, static_cast<const uint8_t*>(xq), N,
                         sums, as_stream(stream));
    return check_launch(fn);
}

int kq_dequant_rows(const void* w, int R, int C, int type, int row0, int nrows, float* y,
                    int64_t ldy, void* stream) {
    static const char* fn = "kq_dequant_rows";
    KQ_TRY(check_matrix(w, R, C, type, fn));
    if (nrows < 1 || nrows > 65535) return fail(KQ_ERR_ARG, "%s: nrows=%d must be 1..65535", fn, nrows);
    if (row0 < 0 || row0 > R - nrows)
        return fail(KQ_ERR_ARG, "%s: rows [%d, %d) outside [0, %d)", fn, row0, row0 + nrows, R);
    if (nrows > 1 && ldy < C) return fail(KQ_ERR_ARG, "%s: ldy=%lld is smaller than C=%d", fn, (long long)ldy, C);
    KQ_TRY(check_ptr(y, 4, "y", fn));
    launch_dequant_rows(static_cast<const uint8_t*>(w), R, C, type, row0, nrows, y, ldy, as_stream(stream));
    return check_launch(fn);
}

// A cache's own rules (include/kq.h, kq_kv).
static int check_kv(const kq_kv* kv, const char* fn) {
    if (!kv) return fail(KQ_ERR_ARG, "%s: kv is NULL", fn);
    if (kv->type != KQ_KV_F16 && kv->type != KQ_KV_BF16 && kv->type != KQ_KV_I8)
        return fail(KQ_ERR_ARG, "%s: cache type %d is not f16 (1), i8 (24) or bf16 (30)", fn, kv->type);
    if (kv->heads < 1 || kv->heads > 4096) return fail(KQ_ERR_ARG, "%s: heads=%d must be 1..4096", fn, kv->heads);
    if (kv->dim < 16 || kv->dim > 256 || kv->dim % 16)
        return fail(KQ_ERR_ARG, "%s: dim=%d must be a multiple of 16 up to 256", fn, kv->dim);
    if (kv->page_size < 1 || kv->page_size > (1 << 20) || (kv->page_size & (kv->page_size - 1)))
        return fail(KQ_ERR_ARG, "%s: page_size=%d must be a power of two up to 2^20", fn, kv->page_size);
    if (kv->pages < 1) return fail(KQ_ERR_ARG, "%s: pages=%d must be positive", fn, kv->pages);
    KQ_TRY(check_ptr(kv->k, 16, "k of the cache", fn));
    KQ_TRY(check_ptr(kv->v, 16, "v of the cache", fn));
    const int64_t unit = kv->type == KQ_KV_I8 ? 16 : 8;
    for (int64_t st : {kv->page_stride, kv->head_stride, kv->pos_stride})
        if (st < kv->dim || st % unit || st > (INT64_MAX >> 33))
            return fail(KQ_ERR_ARG, "%s: stride %lld of the cache must be a multiple of %lld, at least dim=%d", fn,
                        (long long)st, (long long)unit, kv->dim);
    if (kv->type == KQ_KV_I8) {
        KQ_TRY(check_ptr(kv->k_scale, 4, "k_scale of the cache", fn));
        KQ_TRY(check_ptr(kv->v_scale, 4, "v_scale of the cache", fn));
        for (int64_t st : {kv->scale_page_stride, kv->scale_head_stride, kv->scale_pos_stride})
            if (st < 1 || st > (INT64_MAX >> 33))
                return fail(KQ_ERR_ARG, "%s: scale stride %lld of the cache must be positive", fn, (long long)st);
    }
    return KQ_OK;
}

static int check_table(const kq_kv* kv, const int32_t* table, int64_t ldt, int seqs, int width, const char* fn,
                       PageTable* out) {
    KQ_TRY(check_ptr(table, 4, "table", fn));
    if (seqs < 1 || seqs > 65535) return fail(KQ_ERR_ARG, "%s: seqs=%d must be 1..65535", fn, seqs);
    if (width < 1 || (int64_t)width * kv->page_size > (1 << 30))
        return fail(KQ_ERR_ARG, "%s: width=%d pages of %d positions must be 1..2^30 positions", fn, width, kv->page_size);
    if (ldt < width) return fail(KQ_ERR_ARG, "%s: ldt=%lld is smaller than width=%d", fn, (long long)ldt, width);
    *out = PageTable{table, ldt, seqs, width * kv->page_size};
    return KQ_OK;
}

static int check_rows(const void* p, int64_t ld, int64_t n, int64_t row, const char* what, const char* fn) {
    KQ_TRY(check_ptr(p, 4, what, fn));
    if (n > 1 && ld < row)
        return fail(KQ_ERR_ARG, "%s: row stride %lld of %s is smaller than %lld", fn, (long long)ld, what, (long long)row);
    return KQ_OK;
}

static int check_q_heads(const kq_kv* kv, int q_heads, const char* fn) {
    if (q_heads < 1 || q_heads > 4096 || q_heads % kv->heads)
        return fail(KQ_ERR_ARG, "%s: q_heads=%d must be a multiple of the cache's %d heads, up to 4096", fn, q_heads,
                    kv->heads);
    return KQ_OK;
}

static int append(const char* fn, const kq_kv* kv, const int32_t* table, int64_t ldt, int seqs, int width, int N,
                  const int32_t* seq, const int32_t* pos, const int32_t* slot, const float* q, int64_t ldq, int q_heads,
                  float* q_out, int64_t ldqo, const float* k, int64_t ldk, const float* v, int64_t ldv, const float* rope,
                  int rope_rows, int rot, int interleaved, const float* q_norm, const float* k_norm, float eps, void* stream) {
    AppendArgs a = {};
    KQ_TRY(check_kv(kv, fn));
    KQ_TRY(check_table(kv, table, ldt, seqs, width, fn, &a.table));
    if (N < 0) return fail(KQ_ERR_ARG, "%s: N=%d is negative", fn, N);
    if (N && (q != nullptr) != (q_out != nullptr)) return fail(KQ_ERR_ARG, "%s: q and q_out go together", fn);
    if (q) KQ_TRY(check_q_heads(kv, q_heads, fn));
    if (rope) {
        KQ_TRY(check_ptr(rope, 4, "rope", fn));
        if (rot < 8 || rot % 8 || rot > kv->dim)
            return fail(KQ_ERR_ARG, "%s: rot=%d must be a multiple of 8 up to dim=%d", fn, rot, kv->dim);
        if (rope_rows < 1) return fail(KQ_ERR_ARG, "%s: rope_rows=%d must be positive", fn, rope_rows);
    }
    if (q_norm) KQ_TRY(check_ptr(q_norm, 4, "q_norm", fn));
    if (k_norm) KQ_TRY(check_ptr(k_norm, 4, "k_norm", fn));
    if ((q_norm || k_norm) && !(eps >= 0 && eps - eps == 0)) return fail(KQ_ERR_ARG, "%s: eps must be finite, at least 0", fn);
    if (N == 0) return KQ_OK;
    if (slot) KQ_TRY(check_ptr(slot, 4, "slot", fn));
    KQ_TRY(check_ptr(seq, 4, "seq", fn));
    KQ_TRY(check_ptr(pos, 4, "pos", fn));
    const int64_t kw = (int64_t)kv->heads * kv->dim, qw = (int64_t)q_heads * kv->dim;
    KQ_TRY(check_rows(k, ldk, N, kw, "k", fn));
    KQ_TRY(check_rows(v, ldv, N, kw, "v", fn));
    if (q) {
        KQ_TRY(check_rows(q, ldq, N, qw, "q", fn));
        KQ_TRY(check_rows(q_out, ldqo, N, qw, "q_out", fn));
    }
    a.kv = *kv;
    a.N = N;
    a.q_heads = q ? q_heads : 0;
    if ((int64_t)N * (a.q_heads + 2 * kv->heads) > (1 << 30))
        return fail(KQ_ERR_ARG, "%s: N=%d tokens are too many for one call", fn, N);
    a.rope_rows = rope_rows;
    a.rot = rope ? rot : 0;
    a.interleaved = interleaved;
    a.seq = seq, a.pos = pos, a.slot = slot, a.q = q, a.k = k, a.v = v, a.rope = rope, a.q_out = q_out;
    a.ldq = ldq, a.ldqo = ldqo, a.ldk = ldk, a.ldv = ldv;
    a.q_norm = q ? q_norm : nullptr, a.k_norm = k_norm, a.eps = eps;
    launch_kv_append(a, as_stream(stream));
    return check_launch(fn);
}

int kq_kv_append(const kq_kv* kv, const int32_t* table, int64_t ldt, int seqs, int width, int N, const int32_t* seq,
                 const int32_t* pos, const float* q, int64_t ldq, int q_heads, float* q_out, int64_t ldqo, const float* k,
                 int64_t ldk, const float* v, int64_t ldv, const float* rope, int rope_rows, int rot, int interleaved,
                 void* stream) {
    return append("kq_kv_append", kv, table, ldt, seqs, width, N, seq, pos, nullptr, q, ldq, q_heads, q_out, ldqo, k, ldk, v, ldv,
                  rope, rope_rows, rot, interleaved, nullptr, nullptr, 0.0f, stream);
}

int kq_kv_append_norm(const kq_kv* kv, const int32_t* table, int64_t ldt, int seqs, int width, int N, const int32_t* seq,
                      const int32_t* pos, const int32_t* slot, const float* q, int64_t ldq, int q_heads, float* q_out,
                      int64_t ldqo, const float* k, int64_t ldk, const float* v, int64_t ldv, const float* rope, int rope_rows,
                      int rot, int interleaved, const float* q_norm, const float* k_norm, float eps, void* stream) {
    return append("kq_kv_append_norm", kv, table, ldt, seqs, width, N, seq, pos, slot, q, ldq, q_heads, q_out, ldqo, k, ldk, v,
                  ldv, rope, rope_rows, rot, interleaved, q_norm, k_norm, eps, stream);
}

static int check_tree(int seqs, int T, const char* fn) {
    if (seqs < 1 || seqs > 65535) return fail(KQ_ERR_ARG, "%s: seqs=%d must be 1..65535", fn, seqs);
    if (T < 1 || T > KQ_MAX_TREE) return fail(KQ_ERR_ARG, "%s: T=%d must be 1..%d", fn, T, KQ_MAX_TREE);
    return KQ_OK;
}

// Row strides of parents: 0 is one row for all.
static int check_parents(const int32_t* parents, int64_t ldp, int T, const char* fn) {
    KQ_TRY(check_ptr(parents, 4, "parents", fn));
    if (ldp < 0 || (ldp > 0 && ldp < T)) return fail(KQ_ERR_ARG, "%s: ldp=%lld must be 0 or at least T=%d", fn, (long long)ldp, T);
    return KQ_OK;
}

int kq_tree_plan(const int32_t* parents, int64_t ldp, const int32_t* base, int seqs, int T, uint64_t* seen, int32_t* seq,
                 int32_t* pos, int32_t* slot, void* stream) {
    static const char* fn = "kq_tree_plan";
    KQ_TRY(check_tree(seqs, T, fn));
    KQ_TRY(check_parents(parents, ldp, T, fn));
    KQ_TRY(check_ptr(base, 4, "base", fn));
    KQ_TRY(check_ptr(seen, 8, "seen", fn));
    KQ_TRY(check_ptr(seq, 4, "seq", fn));
    KQ_TRY(check_ptr(pos, 4, "pos", fn));
    KQ_TRY(check_ptr(slot, 4, "slot", fn));
    launch_tree_plan(TreeArgs{parents, base, ldp, T, seen, seq, pos, slot}, seqs, as_stream(stream));
    return check_launch(fn);
}

int kq_kv_keep(const kq_kv* const* kv, int layers, const int32_t* table, int64_t ldt, int seqs, int width, const int32_t* base,
               const int32_t* path, int64_t ldp, int T, void* stream) {
    static const char* fn = "kq_kv_keep";
    if (!kv || layers < 1) return fail(KQ_ERR_ARG, "%s: no layer", fn);
    KeepArgs a = {};
    for (int i = 0; i < layers; i++) {
        KQ_TRY(check_kv(kv[i], fn));
        if (kv[i]->heads != kv[0]->heads || kv[i]->dim != kv[0]->dim || kv[i]->pages != kv[0]->pages ||
            kv[i]->page_size != kv[0]->page_size)
            return fail(KQ_ERR_ARG, "%s: the layers' caches must have the same heads, dim, pages and page_size", fn);
        for (int j = 0; j < i; j++)
            if ((kv[j]->k == kv[i]->k) != (kv[j]->v == kv[i]->v))
                return fail(KQ_ERR_ARG, "%s: layers %d and %d share one of k and v", fn, j, i);
    }
    KQ_TRY(check_table(kv[0], table, ldt, seqs, width, fn, &a.table));
    KQ_TRY(check_tree(seqs, T, fn));
    KQ_TRY(check_ptr(base, 4, "base", fn));
    KQ_TRY(check_rows(path, ldp, seqs, T, "path", fn));
    a.base = base, a.path = path, a.ldp = ldp, a.T = T;
    a.pages = kv[0]->pages, a.page_size = kv[0]->page_size;
    int n = 0;
    for (int i = 0; i < layers; i++) {
        const kq_kv* c = kv[i];
        bool again = false;                                    // layers that share a cache: its entries move once
        for (int j = 0; j < i && !again; j++) again = kv[j]->k == c->k;
        const bool i8 = c->type == KQ_KV_I8;
        const int64_t e = i8 ? 1 : 2;
        if (!again)
            a.layer[n++] = KeepLayer{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), i8 ? c->k_scale : nullptr,
                                     i8 ? c->v_scale : nullptr, c->page_stride * e, c->head_stride * e, c->pos_stride * e,
                                     c->scale_page_stride, c->scale_head_stride, c->scale_pos_stride, (int)(c->dim * e), c->heads};
        if ((n < KEEP_LAYERS && i + 1 < layers) || !n) continue;
        launch_kv_keep(a, n, seqs, as_stream(stream));
        KQ_TRY(check_launch(fn));
        n = 0;
    }
    return KQ_OK;
}

size_t kq_attn_paged_workspace(int seqs, int q_heads, int dim, int T, int max_len) {
    if (seqs < 1 || seqs > 65535 || q_heads < 1 || q_heads > 4096 || dim < 16 || dim > 256 || dim % 16 || T < 1 ||
        T > KQ_MAX_BATCH || max_len < 1 || max_len > (1 << 30))
        return 0;
    return attn_paged_workspace(seqs, q_heads, dim, T, max_len);
}

// lens: of trees (seen given) their bases.
static int attention(const char* fn, const kq_kv* kv, const int32_t* table, int64_t ldt, int seqs, int width,
                     const int32_t* lens, const uint64_t* seen, int max_len, int T, const float* q, int64_t ldq, int q_heads,
                     float scale, float* out, int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
    AttnArgs a = {};
    KQ_TRY(check_kv(kv, fn));
    KQ_TRY(check_table(kv, table, ldt, seqs, width, fn, &a.table));
    KQ_TRY(check_q_heads(kv, q_heads, fn));
    KQ_TRY(check_ptr(lens, 4, seen ? "base" : "lens", fn));
    if (!seen && (T < 1 || T > KQ_MAX_BATCH)) return fail(KQ_ERR_ARG, "%s: T=%d must be 1..%d", fn, T, KQ_MAX_BATCH);
    if (max_len < 1 || max_len > (1 << 30)) return fail(KQ_ERR_ARG, "%s: max_len=%d must be 1..2^30", fn, max_len);
    const int64_t rows = (int64_t)seqs * T, qw = (int64_t)q_heads * kv->dim;
    KQ_TRY(check_rows(q, ldq, rows, qw, "q", fn));
    KQ_TRY(check_rows(out, ldo, rows, qw, "out", fn));
    if (!(scale - scale == 0)) return fail(KQ_ERR_ARG, "%s: scale must be finite", fn);
    KQ_TRY(check_ptr(ws, 256, "ws", fn));
    const size_t need = seen ? attn_tree_bytes(seqs, kv->heads, q_heads / kv->heads, kv->dim, T, max_len)
                             : attn_paged_workspace(seqs, q_heads, kv->dim, T, max_len);
    if (ws_bytes < need)
        return fail(KQ_ERR_ARG, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, need);
    a.kv = *kv;
    a.lens = lens;
    a.seen = seen;
    a.bound = max_len;
    a.max_len = max_len < a.table.cap ? max_len : a.table.cap;
    a.T = T;
    a.q_heads = q_heads;
    a.q = q, a.ldq = ldq, a.out = out, a.ldo = ldo;
    a.scale = scale;
    a.ws = static_cast<uint8_t*>(ws);
    seen ? launch_attn_tree(a, as_stream(stream)) : launch_attn_paged(a, as_stream(stream));
    return check_launch(fn);
}

int kq_attn_paged(const kq_kv* kv, const int32_t* table, int64_t ldt, int seqs, int width, const int32_t* lens,
                  int max_len, int T, const float* q, int64_t ldq, int q_heads, float scale, float* out, int64_t ldo,
                  void* ws, size_t ws_bytes, void* stream) {
    return attention("kq_attn_paged", kv, table, ldt, seqs, width, lens, nullptr, max_len, T, q, ldq, q_heads, scale, out, ldo, ws,
                     ws_bytes, stream);
}

size_t kq_attn_tree_workspace(int seqs, int q_heads, int dim, int T, int max_len) {
    if (seqs < 1 || seqs > 65535 || q_heads < 1 || q_heads > 4096 || dim < 16 || dim > 256 || dim % 16 || T < 1 ||
        T > KQ_MAX_TREE || max_len < 1 || max_len > (1 << 30))
        return 0;
    return attn_tree_workspace(seqs, q_heads, dim, T, max_len);
}

int kq_attn_tree(const kq_kv* kv, const int32_t* table, int64_t ldt, int seqs, int width, const int32_t* base,
                 const uint64_t* seen, int max_len, int T, const float* q, int64_t ldq, int q_heads, float scale, float* out,
                 int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
    static const char* fn = "kq_attn_tree";
    KQ_TRY(check_tree(seqs, T, fn));
    KQ_TRY(check_ptr(base, 4, "base", fn));
    KQ_TRY(check_ptr(seen, 8, "seen", fn));
    return attention(fn, kv, table, ldt, seqs, width, base, seen, max_len, T, q, ldq, q_heads, scale, out, ldo, ws, ws_bytes, stream);
}

size_t kq_verify_workspace(int B, int T, int V) {
    if (B < 1 || T < 1 || T > KQ_MAX_TREE || V < 1 || V > (1 << 30) || (int64_t)B * T > 65535) return 0;
    return verify_workspace(B, T, V);
}

int kq_verify(const float* x, int64_t ldx, int B, int T, int V, const int32_t* tokens, int64_t ldt, const int32_t* parents,
              int64_t ldp, const float* uniform, int64_t ldu, const float* temperature, const float* draft, int64_t ldd,
              int32_t* accepted, int32_t* path, int32_t* token, void* ws, size_t ws_bytes, void* stream) {
    static const char* fn = "kq_verify";
    KQ_TRY(check_tree(B, T, fn));
    if ((int64_t)B * T > 65535) return fail(KQ_ERR_ARG, "%s: %d trees of %d nodes must be up to 65535 rows", fn, B, T);
    if (V < 1 || V > (1 << 30)) return fail(KQ_ERR_ARG, "%s: V=%d must be 1..2^30", fn, V);
    KQ_TRY(check_rows(x, ldx, (int64_t)B * T, V, "x", fn));
    KQ_TRY(check_rows(tokens, ldt, B, T, "tokens", fn));
    KQ_TRY(check_parents(parents, ldp, T, fn));
    KQ_TRY(check_rows(uniform, ldu, B, T, "uniform", fn));
    if (temperature) KQ_TRY(check_ptr(temperature, 4, "temperature", fn));
    if (draft) KQ_TRY(check_rows(draft, ldd, (int64_t)B * T, V, "draft", fn));
    KQ_TRY(check_ptr(accepted, 4, "accepted", fn));
    KQ_TRY(check_ptr(path, 4, "path", fn));
    KQ_TRY(check_ptr(token, 4, "token", fn));
    KQ_TRY(check_ptr(ws, 256, "ws", fn));
    const size_t need = verify_workspace(B, T, V);
    if (ws_bytes < need) return fail(KQ_ERR_ARG, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, need);
    VerifyArgs a = {};
    a.x = x, a.ldx = ldx, a.B = B, a.T = T, a.V = V;
    a.tokens = tokens, a.ldt = ldt, a.parents = parents, a.ldp = ldp, a.uniform = uniform, a.ldu = ldu;
    a.temperature = temperature, a.draft = draft, a.ldd = ldd;
    a.accepted = accepted, a.path = path, a.token = token, a.ws = static_cast<uint8_t*>(ws);
    launch_verify(a, as_stream(stream));
    return check_launch(fn);
}

size_t kq_logits_workspace(int B) { return B < 1 || B > 65535 ? 0 : logits_workspace(B); }

int kq_logits_penalize(const float* x, int64_t ldx, int B, int V, const int32_t* hist, int64_t ldh, int max_hist,
                       const int32_t* hist_len, const int32_t* prompt_len, const float* rep, const float* freq,
                       const float* pres, const int32_t* bias_id, const float* bias_val, int64_t ldb, int nb,
                       const uint32_t* allowed, int64_t ldm, float* y, int64_t ldy, void* ws, size_t ws_bytes,
                       int32_t* picked, void* stream) {
    static const char* fn = "kq_logits_penalize";
    if (B < 1 || B > 65535) return fail(KQ_ERR_ARG, "%s: B=%d must be 1..65535", fn, B);
    if (V < 1 || V > (1 << 30)) return fail(KQ_ERR_ARG, "%s: V=%d must be 1..2^30", fn, V);
    KQ_TRY(check_rows(x, ldx, B, V, "x", fn));
    if (hist) {
        if (max_hist < 0) return fail(KQ_ERR_ARG, "%s: max_hist=%d is negative", fn, max_hist);
        KQ_TRY(check_rows(hist, ldh, B, max_hist, "hist", fn));
        KQ_TRY(check_ptr(hist_len, 4, "hist_len", fn));
    }
    if (bias_id) {
        if (nb < 0) return fail(KQ_ERR_ARG, "%s: nb=%d is negative", fn, nb);
        KQ_TRY(check_rows(bias_id, ldb, B, nb, "bias_id", fn));
        KQ_TRY(check_ptr(bias_val, 4, "bias_val", fn));
    }
    if (allowed) {
        KQ_TRY(check_ptr(allowed, 4, "allowed", fn));
        if (ldm < 0 || (ldm > 0 && ldm < (V + 31) / 32))
            return fail(KQ_ERR_ARG, "%s: ldm=%lld words must be 0 or at least %d", fn, (long long)ldm, (V + 31) / 32);
    }
    for (const void* p : {(const void*)prompt_len, (const void*)rep, (const void*)freq, (const void*)pres})
        if (p) KQ_TRY(check_ptr(p, 4, "a per-row array", fn));
    if (!y && !picked) return fail(KQ_ERR_ARG, "%s: neither y nor picked is given", fn);
    if (y) KQ_TRY(check_rows(y, ldy, B, V, "y", fn));
    if (picked) {
        KQ_TRY(check_ptr(picked, 4, "picked", fn));
        KQ_TRY(check_ptr(ws, 256, "ws", fn));
        if (ws_bytes < logits_workspace(B))
            return fail(KQ_ERR_ARG, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes, logits_workspace(B));
    }
    LogitsArgs a = {};
    a.x = x, a.ldx = ldx, a.B = B, a.V = V;
    a.hist = hist, a.ldh = ldh, a.max_hist = max_hist, a.hist_len = hist_len, a.prompt_len = prompt_len;
    a.rep = rep, a.freq = freq, a.pres = pres;
    a.bias_id = bias_id, a.bias_val = bias_val, a.ldb = ldb, a.nb = nb;
    a.allowed = allowed, a.ldm = ldm;
    a.y = y, a.ldy = ldy, a.ws = static_cast<uint8_t*>(ws), a.picked = picked;
    launch_logits(a, as_stream(stream));
    return check_launch(fn);
}

}  // extern "C"
