// operators.h -- internal launch interface of the operators on trellis-coded
// weights (linear layer, mixture layer, input Gram).  The exported entry points
// live in operators_capi.hip and are declared in include/exl3_vit.h.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/exl3_vit.h"
#include "trellis_math.h"

namespace xtq {

// The MI355X's compute units: launches are split to fill them (any number is
// right).
constexpr int kCUs = 256;

// A trellis weight as the kernels take it.
struct Weight {
    const int16_t* trellis;
    const uint16_t* suh;
    const uint16_t* svh;
    float scale;
    int k, n, K, code;
};

// Arguments of a product's epilogue, see finish_unit.
struct Epilogue {
    const uint16_t* colscale;   // fp16, per output column
    float scale;                // for all of them
    const int32_t* rowexp;      // per row: products are 2^rowexp too small; NULL: 0
    const void* bias;           // per output column or NULL
    int bias_f32;               // bias is fp32, else of the activations' type
    int act;
    const void* res;            // residual or NULL
    long long res_stride;
    void* z;                    // [M][n] values before the activation, or NULL
    void* y;
    long long y_stride;
    int rows, cols;
};

// Whether a forward product's rows enter with 22 bits, as two fp16 terms, and not with
// the 11 of one.  fp16: one rounding of the rows is as large as the result's own
// (together 1.4 times the error of that alone), so only the result's is left.
// bf16 results are rounded to 8 bits, beside which the rows' 11 do not show
// (0.0017 of a result's norm with one term and with two); but relu's slope jumps
// at zero: results that near to it take the wrong side, e of them for an error
// e, and the gradient is off by the root of that, so relu's rows have 22 bits in
// either type.  It does not go by whether z is kept: a call's results are the
// same with a gradient and without.  fast: the caller's choice of one term, which
// halves the work of the matrix cores (us with one and with two: 17408 by 5120, 1
// row 24.2 : 27.2, 48 rows 43.8 : 50.4; 5120 by 17408, 333 rows 130 : 170, 4096
// rows 722 : 1236).
inline bool two_terms(int type, int act, bool fast) { return !fast && (type == kF16 || act == kActRelu); }

// The same for a gradient's product: no slope is taken at what it gives.
inline bool two_terms_gradient(int type, bool fast) { return !fast && type == kF16; }

size_t linear_ws_bytes(int rows, int k, int n, bool backward, bool two);
hipError_t launch_linear(const Weight& w, int type, const void* x, long long x_stride, int rows,
                         const Epilogue& ep, bool two, void* ws, uint32_t* counters, hipStream_t s);
hipError_t launch_linear_bwd(const Weight& w, int type, const void* dy, long long dy_stride,
                             const void* z, int act, int rows, void* dx, long long dx_stride,
                             void* dbias, int dbias_f32, bool two, void* ws, uint32_t* counters,
                             hipStream_t s);

// Products of up to kFewRows rows (few_kernels.hip), one function per K.  The
// kernel transforms up to kFusedRows rows of x itself, or takes them transformed
// (transform_few_kernel): fragments frag [groups of 16 rows][k/32][64] and their
// shifts [groups][k/128][16], 1, 2 or 4 groups, all of whose places it reads.
constexpr int kFewRows = 64;
constexpr int kFusedRows = 16;
// Waves of a workgroup: 8, which with their registers make four a SIMD, or 4
// where 16 G rows' sums take the registers of two.
constexpr int few_waves(int G) { return G == 1 ? 8 : 4; }
struct FewArgs {
    int type;
    int two;                            // two terms
    const uint16_t* x;
    long long x_stride;
    const u4 *frag, *frag_lo;           // NULL: x is transformed by the kernel; lo: the second terms
    const int32_t* shift;
    int groups;
    int splits, steps, more;            // 32-row steps of a split; splits with one more
    uint32_t rinv;                      // item / rows is item * rinv >> 16
    float* part;
    uint32_t* counters;
};
#define XTQ_FEW(K) \
    hipError_t launch_few_k##K(const Weight& w, const FewArgs& a, const Epilogue& ep, hipStream_t s); \
    hipError_t launch_few2_k##K(const Weight& w, const FewArgs& a, const Epilogue& ep, hipStream_t s);
XTQ_FEW(2) XTQ_FEW(3) XTQ_FEW(4) XTQ_FEW(5) XTQ_FEW(6) XTQ_FEW(7)
#undef XTQ_FEW

struct MoeArgs;
size_t moe_ws_bytes(int rows, int experts, int top, int d, int f);
size_t moe_counters(int rows, int experts, int top, int d, int f);
hipError_t launch_moe(MoeArgs a, void* ws, hipStream_t s);

size_t gram_ws_bytes(int rows, int k);
hipError_t launch_gram(int type, const void* x, long long x_stride, int rows, int k,
                       const uint8_t* valid, const float* prev, float* out, void* ws,
                       hipStream_t s);
}  // namespace xtq
