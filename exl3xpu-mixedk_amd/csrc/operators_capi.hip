// operators_capi.hip -- C entries of the operators on trellis weights (declared
// in include/exl3_vit.h): arguments are checked on the host against everything
// the kernels assume, then the kernels are enqueued.  No state is kept between
// calls and nothing is locked.
#include <stdio.h>
#include <string.h>

#include "moe_device.h"
#include "operators.h"

namespace {

// Code of a trellis weight's name, or -1: the products take values that fp16
// holds, which "1mad"'s are not.
int parse_code(const char* code) {
    if (!strncmp(code, "exl3_", 5)) code += 5;
    if (!strcmp(code, "mul1")) return xtq::kCodeMul1;
    if (!strcmp(code, "3inst")) return xtq::kCode3Inst;
    if (!strcmp(code, "mcg")) return xtq::kCodeMcg;
    return -1;
}

bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

constexpr int kMaxRows = 1048560;       // 65,535 groups of 16 rows (a grid's second dimension)

int check_weight(const xtq_weight* w, xtq::Weight* out) {
    if (!w || !w->trellis || !w->suh || !w->svh || !w->code) return 12;
    if (!aligned(w->trellis, 2) || !aligned(w->suh, 2) || !aligned(w->svh, 2)) return 12;
    if (w->K < 2 || w->K > 7) return 9;
    const int code = parse_code(w->code);
    if (code < 0) return 8;
    if (w->k <= 0 || w->n <= 0 || w->k % 128 || w->n % 128 || w->k > (1 << 22) || w->n > (1 << 22))
        return 6;
    *out = xtq::Weight{w->trellis, w->suh, w->svh, w->scale, w->k, w->n, w->K, code};
    return 0;
}

// A matrix of 16-bit elements.
int check_rows(const void* p, int64_t stride, int cols) {
    if (!p || !aligned(p, 2)) return 12;
    return stride < cols ? 6 : 0;
}

int status(hipError_t e, const char* what) {
    if (e == hipSuccess) return 0;
    fprintf(stderr, "xtq_vit %s: %s\n", what, hipGetErrorString(e));
    return 4;
}

int check_ws(const void* ws, int64_t have, int64_t want) {
    if (want > 0 && (!ws || !aligned(ws, 16))) return 12;
    return have < want ? 14 : 0;
}

bool moe_sizes(int rows, int experts, int top, int d, int f) {
    return rows >= 0 && rows <= xtq::kMoeRows && experts >= 1 && experts <= xtq::kMoeExperts && top >= 1 &&
           top <= xtq::kMoeTop && top <= experts && d > 0 && f > 0 && d % 128 == 0 && f % 128 == 0 &&
           d <= (1 << 20) && f <= (1 << 20) &&
           (rows == 0 || xtq::moe_counters(rows, experts, top, d, f) <= XTQ_OP_COUNTERS);
}

}  // namespace

extern "C" {

int64_t xtq_linear_ws_bytes(const xtq_weight* w, int rows, int what) {
    if (what < XTQ_LINEAR_FORWARD || what > XTQ_LINEAR_TRAIN) return -15;
    if (!w || w->k <= 0 || w->n <= 0 || w->k % 128 || w->n % 128 || rows < 0 || rows > kMaxRows)
        return -6;
    if (!rows) return 0;
    // (the type and the activation decide which of the two it is)
    const size_t one = xtq::linear_ws_bytes(rows, w->k, w->n, what == XTQ_LINEAR_GRADIENT, false),
                 two = xtq::linear_ws_bytes(rows, w->k, w->n, what == XTQ_LINEAR_GRADIENT, true);
    return (int64_t)(one > two ? one : two);
}

int xtq_linear_dev(const xtq_weight* w, int type, const void* x, int64_t x_stride, int rows,
                   const void* bias, int bias_f32, int act, const void* res, int64_t res_stride,
                   void* z, void* y, int64_t y_stride, void* ws, int64_t ws_bytes,
                   uint32_t* counters, void* stream) {
    xtq::Weight wt;
    int rc = check_weight(w, &wt);
    if (rc) return rc;
    const bool fast = type & XTQ_FAST;
    type &= ~XTQ_FAST;
    if ((type != XTQ_BF16 && type != XTQ_F16) || act < XTQ_ACT_NONE || act > XTQ_ACT_GELU) return 15;
    if (rows < 0 || rows > kMaxRows) return 6;
    if (rows == 0) return 0;
    if ((rc = check_rows(x, x_stride, wt.k))) return rc;
    if ((rc = check_rows(y, y_stride, wt.n))) return rc;
    if (res && (rc = check_rows(res, res_stride, wt.n))) return rc;
    if (!aligned(z, 2) || !aligned(bias, bias_f32 ? 4 : 2)) return 12;
    if (!counters || !aligned(counters, 4)) return 12;
    const bool two = xtq::two_terms(type, act, fast);
    if ((rc = check_ws(ws, ws_bytes, xtq::linear_ws_bytes(rows, wt.k, wt.n, false, two)))) return rc;
    xtq::Epilogue ep{};
    ep.colscale = wt.svh;
    ep.scale = wt.scale;
    ep.bias = bias;
    ep.bias_f32 = bias_f32;
    ep.act = act;
    ep.res = res;
    ep.res_stride = res_stride;
    ep.z = z;
    ep.y = y;
    ep.y_stride = y_stride;
    ep.rows = rows;
    ep.cols = wt.n;
    return status(xtq::launch_linear(wt, type, x, x_stride, rows, ep, two, ws, counters,
                                     (hipStream_t)stream), "linear");
}

int xtq_linear_bwd_dev(const xtq_weight* w, int type, const void* dy, int64_t dy_stride,
                       const void* z, int act, int rows, void* dx, int64_t dx_stride, void* dbias,
                       int bias_f32, void* ws, int64_t ws_bytes, uint32_t* counters, void* stream) {
    xtq::Weight wt;
    int rc = check_weight(w, &wt);
    if (rc) return rc;
    const bool fast = type & XTQ_FAST;
    type &= ~XTQ_FAST;
    if ((type != XTQ_BF16 && type != XTQ_F16) || act < XTQ_ACT_NONE || act > XTQ_ACT_GELU) return 15;
    if (rows <= 0 || rows > kMaxRows) return 6;
    if ((rc = check_rows(dy, dy_stride, wt.n))) return rc;
    if (!dx && !dbias) return 12;
    if (dx && (rc = check_rows(dx, dx_stride, wt.k))) return rc;
    if (act != XTQ_ACT_NONE && (!z || !aligned(z, 2))) return 12;
    if (!aligned(dbias, bias_f32 ? 4 : 2)) return 12;
    if (!counters || !aligned(counters, 4)) return 12;
    const bool two = xtq::two_terms_gradient(type, fast);
    if ((rc = check_ws(ws, ws_bytes, xtq::linear_ws_bytes(rows, wt.k, wt.n, true, two)))) return rc;
    return status(xtq::launch_linear_bwd(wt, type, dy, dy_stride, z, act, rows, dx, dx_stride, dbias,
                                         bias_f32, two, ws, counters, (hipStream_t)stream), "linear_bwd");
}

int xtq_moe_table(const xtq_weight* weights, int experts, xtq_moe_weight* table) {
    if (!weights || !table) return 12;
    if (experts < 1 || experts > xtq::kMoeExperts) return 6;
    xtq::Weight first{};
    for (int i = 0; i < 3 * experts; ++i) {
        xtq::Weight w;
        const int rc = check_weight(weights + i, &w);
        if (rc) return rc;
        if (i == 0) first = w;
        if (w.code != first.code) return 8;
        const bool down = i % 3 == 2;
        if (w.k != (down ? first.n : first.k) || w.n != (down ? first.k : first.n)) return 6;
        table[i] = xtq_moe_weight{w.trellis, w.suh, w.svh, w.scale, w.K};
    }
    return 0;
}

int64_t xtq_moe_ws_bytes(int rows, int experts, int top, int d, int f) {
    if (!moe_sizes(rows, experts, top, d, f)) return -6;
    return rows ? (int64_t)xtq::moe_ws_bytes(rows, experts, top, d, f) : 0;
}

int xtq_moe_dev(const xtq_moe_weight* table, int experts, int d, int f, const char* code, int type,
                const void* x, int64_t x_stride, int rows, const void* router, int router_f32, int top,
                int act, int renorm, const uint8_t* valid, const void* res, int64_t res_stride, void* y,
                int64_t y_stride, int32_t* ids, float* weights, void* ws, int64_t ws_bytes,
                uint32_t* counters, void* stream) {
    if (!table || !aligned(table, 8) || !code) return 12;
    const int c = parse_code(code);
    if (c < 0) return 8;
    if ((type != XTQ_BF16 && type != XTQ_F16) || act < XTQ_ACT_NONE || act > XTQ_ACT_GELU) return 15;
    if (!moe_sizes(rows, experts, top, d, f)) return 6;
    if (rows == 0) return 0;
    int rc;
    if ((rc = check_rows(x, x_stride, d))) return rc;
    if ((rc = check_rows(y, y_stride, d))) return rc;
    if (res && (rc = check_rows(res, res_stride, d))) return rc;
    if (!router || !aligned(router, router_f32 ? 4 : 2)) return 12;
    if (!ids || !weights || !aligned(ids, 4) || !aligned(weights, 4)) return 12;
    if (!counters || !aligned(counters, 4)) return 12;
    if ((rc = check_ws(ws, ws_bytes, xtq::moe_ws_bytes(rows, experts, top, d, f)))) return rc;
    xtq::MoeArgs a{};
    a.table = table;
    a.experts = experts;
    a.d = d;
    a.f = f;
    a.code = c;
    a.type = type;
    a.rows = rows;
    a.top = top;
    a.act = act;
    a.renorm = renorm;
    a.x = (const uint16_t*)x;
    a.x_stride = x_stride;
    a.router = router;
    a.router_f32 = router_f32;
    a.valid = valid;
    a.res = (const uint16_t*)res;
    a.res_stride = res_stride;
    a.y = (uint16_t*)y;
    a.y_stride = y_stride;
    a.ids = ids;
    a.weights = weights;
    a.counters = counters;
    return status(xtq::launch_moe(a, ws, (hipStream_t)stream), "moe");
}

int64_t xtq_gram_ws_bytes(int rows, int k) {
    if (k <= 0 || k % 128 || k > (1 << 22) || rows < 0 || rows > (1 << 30)) return -6;
    return (int64_t)xtq::gram_ws_bytes(rows, k);
}

int xtq_gram_dev(int type, const void* x, int64_t x_stride, int rows, int k, const uint8_t* valid,
                 const float* prev, float* out, void* ws, int64_t ws_bytes, void* stream) {
    if (type != XTQ_BF16 && type != XTQ_F16) return 15;
    if (k <= 0 || k % 128 || k > (1 << 22) || rows < 0 || rows > (1 << 30)) return 6;
    int rc;
    if (rows && (rc = check_rows(x, x_stride, k))) return rc;
    if (!out || !aligned(out, 4) || !aligned(prev, 4)) return 12;
    if (prev && prev != out) {          // an element would be read after another's place was written over it
        const uintptr_t a = (uintptr_t)prev, b = (uintptr_t)out;
        if ((a < b ? b - a : a - b) < (uintptr_t)k * k * 4) return 12;
    }
    if ((rc = check_ws(ws, ws_bytes, xtq::gram_ws_bytes(rows, k)))) return rc;
    return status(xtq::launch_gram(type, x, x_stride, rows, k, valid, prev, out, ws,
                                   (hipStream_t)stream), "gram");
}

}  // extern "C"
