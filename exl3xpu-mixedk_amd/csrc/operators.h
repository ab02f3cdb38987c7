// operators.h -- internal launch interface of the operators on trellis-coded
// weights (linear layer, mixture layer, input Gram) and of the norms around them.
// The exported entry points live in operators_capi.hip and are declared in
// include/exl3_vit.h.
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
// bf16 results are rounded to 8 bits, beside which the rows' 11 add little: 0.8% to
// the error of the rounded exact result in a linear layer, 1.4 to 1.6% in a gated
// projection, which takes two factors', and 1.8% in its gradient (48 and 500 rows of
// 5120 by 1280 and the other way round, 0.00166 of the norm); a second term would take
// that away for up to twice the matrix work.  But relu's slope jumps
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

struct Tiling {
    int nb, tiles, splits;
};

Tiling gemm_tiling(int rows, int n, int steps, bool two);

// Column sums' last step: out[c] = sum of part[g][c] over the groups, in an
// order that their number fixes: four threads a column take every fourth group.
struct ColSum {
    const float* part;
    int groups, cols, type, f32;
    void* out;
    int first, more_f32;                // columns from `first` on are another sum's
    void* more;
};

// A product of fragments.
struct Gemm {
    const uint16_t *A, *B, *B2;         // B2: B's second terms (TERMS 2)
    int ga, gb;                         // 16-wide groups of columns, rows
    int steps;                          // 32-wide steps of the summed dimension
    int tiles, splits;                  // splits of the summed dimension
    float* part;                        // partial: [splits][blocks of 128][gb][8][64][4]
    const float* prev;                  // Gram
    float* out;
    int dim;
};
// The product's parts, in g.splits runs of the summed dimension, by tiles of nb, and
// beside them `adders` workgroups of column sums.
hipError_t launch_parts(const Gemm& g, int type, int nb, bool two, const ColSum& sums, int adders, hipStream_t s);

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

// Workgroups per 128 columns and groups of 16 rows of those products, and their rows'
// way to fragments (suh2: for a second weight too, behind the first's).
int few_splits(int rows, int k, int n, int waves);
constexpr int few_groups(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }
void transform_few(bool two, const void* x, long long x_stride, int type, int rows, int k, int groups,
                   const uint16_t* suh, const uint16_t* suh2, u4* frag, u4* rest, int32_t* shift, hipStream_t s);

// The gated projection act(x Wg + bg) (x Wu + bu) (gated_kernels.hip; of few rows
// gated_few.hip).  Role 0 is the gate, 1 the up weight.
struct GatedArgs {
    Weight w[2];                        // one k, n and code
    int type, rows, act;
    const uint16_t* x;
    long long x_stride;
    const void* bias[2];                // [n] or NULL
    int bias_f32[2];
    float* z;                           // [2][rows][n] values before the activation and the product, or NULL
    uint16_t* y;
    long long y_stride;
    bool two;
};
struct GatedGradArgs {
    Weight w[2];
    int type, rows, act;
    const uint16_t* dy;
    long long dy_stride;
    const float* z;
    uint16_t* dx;                       // or NULL
    long long dx_stride;
    void* dbias[2];                     // or NULL
    int bias_f32[2];
    bool two;
};
size_t gated_ws_bytes(int rows, int k, int n, bool two);
size_t gated_bwd_ws_bytes(int rows, int k, int n, bool two);
hipError_t launch_gated(const GatedArgs& a, void* ws, uint32_t* counters, hipStream_t s);
hipError_t launch_gated_bwd(const GatedGradArgs& a, void* ws, hipStream_t s);

// Few rows, one function per codebook: frag [role][groups of 16 rows][k/32][64] and
// shifts as in FewArgs, or NULL (one group: the kernel transforms x).  1, 2 or 4
// groups, or fours of them: chunks of 64 rows.  workers: workgroups of a chunk, each a
// run of the steps of all blocks of 128 columns of both weights: per_block of every
// block's steps, or (per_block 0) of all.
struct GatedFew {
    const u4 *frag, *frag_lo;
    const int32_t* shift;
    int groups, workers, per_block;
    int each, more;                     // steps of a run; runs with one more
    float* part;                        // [chunk][worker + block][row][128], chunks 64 rows apart
    uint32_t* counters;                 // [n/128], up to 16 rows
};
#define XTQ_GATED(C) \
    hipError_t launch_gated_few_code##C(const GatedArgs& a, const GatedFew& f, hipStream_t s);
XTQ_GATED(0) XTQ_GATED(1) XTQ_GATED(2)
#undef XTQ_GATED

struct MoeArgs;
size_t moe_ws_bytes(int rows, int experts, int top, int d, int f);
size_t moe_counters(int rows, int experts, int top, int d, int f);
hipError_t launch_moe(MoeArgs a, void* ws, hipStream_t s);

// Norms of rows and the residual sum between blocks (norm_kernels.hip; the C-ABI's
// numbers).  kind and post: the norm of y and of x before it, or none.
enum NormKind { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };
enum GateAct { kGateNone = 0, kGateSigmoid = 1, kGateSilu = 2 };
struct NormParam {
    const void* p;                      // [d] or NULL
    int f32;                            // fp32, else of the rows' type
};
struct NormArgs {
    int rows, d, kind, post, gate_act;
    float eps, post_eps, scale_number;  // the number scales where there is no tensor
    NormParam weight, bias, scale, post_weight, post_bias;
    const uint16_t *x, *res, *gate;     // res NULL: y is x, and not written
    long long x_stride, res_stride, gate_stride;
    uint16_t *y, *h;
    long long y_stride, h_stride;
    float* stats;                       // [rows][4] or NULL: mean and factor of x's norm, of y's
};
enum NormSumOf { kSumWeight, kSumBias, kSumScale, kSumPostWeight, kSumPostBias, kNormSums };
struct NormSum {
    void* p;                            // [d] or NULL
    int f32;
};
struct NormGradArgs {
    NormArgs f;
    const uint16_t *dy, *dh;            // NULL: zero
    long long dy_stride, dh_stride;
    uint16_t *dx, *dres, *dgate;        // [rows][d] or NULL
    NormSum dparam[kNormSums];
    int place[kNormSums];               // of the sums in part
    float* part;                        // [place][workgroup][d]
    float* means;                       // [rows][4] what wide rows' gradients take of the whole row
};
constexpr int kNormMaxD = 32768;        // within 12 waves of six eights a lane
hipError_t launch_norm(const NormArgs& a, int type, hipStream_t s);
size_t norm_bwd_ws_bytes(int rows, int d, int sums);
hipError_t launch_norm_bwd(NormGradArgs a, int type, void* ws, hipStream_t s);

size_t gram_ws_bytes(int rows, int k);
hipError_t launch_gram(int type, const void* x, long long x_stride, int rows, int k,
                       const uint8_t* valid, const float* prev, float* out, void* ws,
                       hipStream_t s);
}  // namespace xtq
