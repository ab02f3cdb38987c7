// gated_few.hip -- the gated projection of few rows, 64 at a time: both weights are
// decoded on their way to the matrix cores, in one launch.
//
// Built once per codebook (XTQ_GATED_CODE); the weights' widths are chosen in the
// kernels, per workgroup.
#include "epilogue.h"
#include "few_device.h"

#pragma clang fp contract(off)

namespace xtq {
namespace {

constexpr int kCode = XTQ_GATED_CODE;

constexpr int most(int a, int b) { return a > b ? a : b; }
template <int G, bool FUSED, bool LO>
constexpr int gated_lds() {
    int n = 0;
    for (int K = 2; K <= 7; ++K) n = most(n, few_lds(K, few_waves(G), FUSED, LO));
    return n;
}

template <int G, bool FUSED, bool LO>
__device__ __forceinline__ void role_sums(int K, const FewSource& src, int s0, int s1, u4* lds, int32_t* shifts,
                                          f4 (&total)[G][8 / few_waves(G)], int lane) {
    constexpr int W = few_waves(G);
    switch (K) {
        case 2: return few_sums<2, kCode, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total, lane);
        case 3: return few_sums<3, kCode, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total, lane);
        case 4: return few_sums<4, kCode, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total, lane);
        case 5: return few_sums<5, kCode, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total, lane);
        case 6: return few_sums<6, kCode, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total, lane);
        default: return few_sums<7, kCode, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total, lane);
    }
}

// Scale and bias of a role's two columns of a lane.
__device__ __forceinline__ Columns<2> role_columns(const GatedArgs& a, int role, int col) {
    Epilogue ep{};
    ep.colscale = a.w[role].svh;
    ep.scale = a.w[role].scale;
    ep.bias = a.bias[role];
    ep.bias_f32 = a.bias_f32[role];
    return a.type == kBf16 ? load_columns<kBf16, 2>(ep, col) : load_columns<kF16, 2>(ep, col);
}

// The blocks are 128 columns of a weight, gate's and up's side by side (a gate's are
// even), and a workgroup multiplies a run of the steps of all blocks one behind the
// other.  EVEN: `each` steps and `more` times one more of every block's.  Else of all
// steps, so that a run may go over blocks' ends.  Run i's part of block q has place
// i + q: along the steps one of them or both grow.
struct Runs {
    int steps, each, more, per_block;
    template <bool EVEN>
    __device__ __forceinline__ int at(int i) const {
        const int q = EVEN ? i / per_block : 0, j = i - q * per_block;
        return q * steps + j * each + (j < more ? j : more);
    }
    // The run that holds a step (not EVEN).
    __device__ __forceinline__ int of(int step) const {
        const int big = more * (each + 1);
        return step < big ? step / (each + 1) : more + (step - big) / each;
    }
};

// First part and number of parts of both weights' columns of block blk.
template <bool EVEN>
__device__ __forceinline__ void parts_of(const GatedFew& f, const Runs& runs, int blk, int (&first)[2], int (&parts)[2]) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int b = 2 * blk + r;
        first[r] = EVEN ? b * f.per_block : runs.of(b * runs.steps);
        parts[r] = EVEN ? f.per_block : runs.of((b + 1) * runs.steps - 1) - first[r] + 1;
        first[r] += b;
    }
}

// R rows of a chunk (row0 + n step) of 128 columns: both weights' parts added in order
// and transformed, scales and biases, and act(gate) * up, with the values between in
// registers.
template <int U, int R>
__device__ __forceinline__ void finish_rows_of(const GatedArgs& a, const Columns<2>& cg, const Columns<2>& cu,
                                               const float* part, const int (&first)[2], const int (&parts)[2], int blk,
                                               int row_base, int rows, int row0, int step, int lane) {
    const size_t run = (size_t)rows * 128;
    const int col = blk * 128 + 2 * lane;
    float v[R][2], u[R][2];
    sum_rows<U, R>(v, part + first[0] * run, row0, step, rows, run, parts[0], lane);
    sum_rows<U, R>(u, part + first[1] * run, row0, step, rows, run, parts[1], lane);
#pragma unroll
    for (int n = 0; n < R; ++n) {
        transform_row(v[n][0], v[n][1], lane);
        transform_row(u[n][0], u[n][1], lane);
    }
#pragma unroll
    for (int n = 0; n < R; ++n) {
        if (row0 + n * step >= rows) break;
        const size_t row = row_base + row0 + n * step;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            v[n][c] = v[n][c] * cg.scale[c] + cg.bias[c];
            u[n][c] = u[n][c] * cu.scale[c] + cu.bias[c];
        }
        if (a.z) {
            float* z = a.z + row * a.w[0].n + col;
            z[0] = v[n][0];
            z[1] = v[n][1];
            z += (size_t)a.rows * a.w[0].n;
            z[0] = u[n][0];
            z[1] = u[n][1];
        }
        activate<2>(v[n], a.act);
        v[n][0] *= u[n][0];
        v[n][1] *= u[n][1];
        uint16_t* y = a.y + row * a.y_stride + col;
        if (a.type == kBf16) store16<kBf16, 2>(y, v[n]);
        else store16<kF16, 2>(y, v[n]);
    }
}

// Up to 16 rows the last run to arrive of two blocks' finishes them; more are left to
// gated_few_join_kernel, since the last runs' rows would be all that still works: 64
// rows of 4096 by 6144 45.9 us in all, and 34.7 with the other launch (31.8 since).
//
// EVEN where that fills the places, two workgroups a compute unit.  272 blocks of 17408
// columns do not, and two compute units of three then wait for the third: 48 rows of
// 5120 take 82.3 us in 272 runs and 62.8 in 512, one row 53.3 and 43 (calls one behind
// the other, bf16; few_workers has more).  (Going over a block's end is a loop, which
// costs registers: where runs are short, EVEN is faster.)
//
// One kernel holds all six widths, and the widest of them says how many registers it
// keeps in scratch: of four groups and two terms (33 rows of float16 and more) 43 to 70
// by the codebook, 109 to 126 over blocks' ends, some of them read again in the steps
// (48 rows of 5120 by 17408, K = 4: 78 us, 63 with one term), and of one term over
// blocks' ends 2 to 4; of one group 12 to 31 over blocks' ends, and 3 in one block where
// the rows are transformed here for two terms.
template <int G, bool FUSED, bool LO, bool EVEN>
__global__ __launch_bounds__(64 * few_waves(G), G == 1 ? 4 : 2) void gated_few_kernel(GatedArgs a, GatedFew f) {
    constexpr int W = few_waves(G), N = 8 / W;
    __shared__ __align__(16) u4 lds[gated_lds<G, FUSED, LO>() / 16];
    __shared__ int32_t shifts[FUSED ? kFewMaxSlice * 16 : 1];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nb = a.w[0].n / 128, steps = a.w[0].k / 32, nk = a.w[0].k / 128, chunk = blockIdx.y;
    const int row_base = chunk * kFewRows, rows = a.rows - row_base < 16 * G ? a.rows - row_base : 16 * G;
    const Runs runs{steps, f.each, f.more, f.per_block};
    // (EVEN: neighbours are blocks of the same steps, whose trellis lies side by side:
    // 64 rows of 4096 by 6144 44.7 us, 50.1 with a block's runs as neighbours)
    const int i = EVEN ? blockIdx.x % (2 * nb) * f.per_block + blockIdx.x / (2 * nb) : blockIdx.x;
    const size_t run = (size_t)rows * 128;
    float* const part = f.part + (size_t)chunk * (f.workers + 2 * nb) * 128 * kFewRows;
    // Steps s0 .. s1 of block q.
    auto multiply = [&](int q, int s0, int s1, int own) {
        const int blk = q >> 1, role = q & 1;
        const Weight& w = a.w[role];
        const size_t group = (size_t)role * f.groups + (FUSED ? 0 : chunk * (kFewRows / 16));
        const FewSource src{(const uint8_t*)w.trellis + (size_t)blk * 256 * w.K, (size_t)nb * 256 * w.K, rows, steps,
                            a.x, a.x_stride, w.suh, a.type, 65536u / rows + 1,
                            FUSED ? nullptr : f.frag + group * nk * 256,
                            FUSED || !LO ? nullptr : f.frag_lo + group * nk * 256,
                            FUSED ? nullptr : f.shift + group * nk * 16};
        f4 total[G][N];
        role_sums<G, FUSED, LO>(w.K, src, s0, s1, lds, shifts, total, own);
        float* const mine = part + (size_t)(i + q) * run + 4 * (lane >> 4);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int row = 16 * g + (lane & 15);
            if (row < rows)
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    float* const p = mine + row * 128 + 16 * (n * W + wv);
                    if constexpr (G == 1) store_shared(p, total[g][n]);
                    else *(f4*)p = total[g][n];
                }
        }
        if constexpr (G == 1) {
            // (on their way while the workgroups meet)
            const Columns<2> cg = role_columns(a, 0, blk * 128 + 2 * lane), cu = role_columns(a, 1, blk * 128 + 2 * lane);
            int first[2], parts[2];
            parts_of<EVEN>(f, runs, blk, first, parts);
            if (!arrive(f.counters + blk, parts[0] + parts[1], threadIdx.x)) return;
#pragma unroll 1
            for (int r0 = wv; r0 < rows; r0 += 2 * W)
                finish_rows_of<8, 2>(a, cg, cu, part, first, parts, blk, 0, rows, r0, W, lane);
        }
    };
    const int end = runs.at<EVEN>(i + 1);
    int at = runs.at<EVEN>(i);
    if constexpr (EVEN) {
        const int q = i / f.per_block;
        multiply(q, at - q * steps, end - q * steps, lane);
    } else {
#pragma unroll 1
        while (at < end) {
            const int q = at / steps, s0 = at - q * steps, s1 = end - at < steps - s0 ? s0 + end - at : steps;
            // (unknown to the compiler, which would keep every width's windows in
            // registers for the next block)
            int own = lane;
            asm volatile("" : "+v"(own));
            multiply(q, s0, s1, own);
            at += s1 - s0;
        }
    }
}

// Finishes 128 columns of eight rows, a wave two of them.
template <bool EVEN>
__global__ __launch_bounds__(256) void gated_few_join_kernel(GatedArgs a, GatedFew f) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, blk = blockIdx.x, nb = gridDim.x;
    const int row = blockIdx.y * 8 + wv, chunk = row / kFewRows, row_base = chunk * kFewRows;
    const int rows = a.rows - row_base < kFewRows ? a.rows - row_base : kFewRows;
    if (row - row_base >= rows) return;
    const Runs runs{a.w[0].k / 32, f.each, f.more, f.per_block};
    int first[2], parts[2];
    parts_of<EVEN>(f, runs, blk, first, parts);
    const Columns<2> cg = role_columns(a, 0, blk * 128 + 2 * lane), cu = role_columns(a, 1, blk * 128 + 2 * lane);
    finish_rows_of<4, 2>(a, cg, cu, f.part + (size_t)chunk * (f.workers + 2 * nb) * 128 * kFewRows, first, parts, blk,
                         row_base, rows, row - row_base, 4, lane);
}

template <int G, bool FUSED, bool LO>
hipError_t launch(const GatedArgs& a, const GatedFew& f, hipStream_t s) {
    const dim3 grid(f.workers, (a.rows + kFewRows - 1) / kFewRows), block(64 * few_waves(G));
    if (f.per_block) hipLaunchKernelGGL((gated_few_kernel<G, FUSED, LO, true>), grid, block, 0, s, a, f);
    else hipLaunchKernelGGL((gated_few_kernel<G, FUSED, LO, false>), grid, block, 0, s, a, f);
    if (G > 1) {
        const dim3 rest(a.w[0].n / 128, (a.rows + 7) / 8);
        if (f.per_block) hipLaunchKernelGGL(gated_few_join_kernel<true>, rest, dim3(256), 0, s, a, f);
        else hipLaunchKernelGGL(gated_few_join_kernel<false>, rest, dim3(256), 0, s, a, f);
    }
    return hipGetLastError();
}

}  // namespace

#define XTQ_CAT2(a, b) a##b
#define XTQ_CAT(a, b) XTQ_CAT2(a, b)

// (Rows, fragments and runs are held against each other here: the kernels take them
// as they come.)
hipError_t XTQ_CAT(launch_gated_few_code, XTQ_GATED_CODE)(const GatedArgs& a, const GatedFew& f, hipStream_t s) {
    const int groups = f.groups;
    if (a.rows > (f.frag ? 16 * groups : kFusedRows) || (groups > 4 && groups % 4) ||
        (a.two && f.frag && !f.frag_lo) || f.each < 1)
        return hipErrorInvalidValue;
    if (!f.frag) return a.two ? launch<1, true, true>(a, f, s) : launch<1, true, false>(a, f, s);
    if (groups == 1) return a.two ? launch<1, false, true>(a, f, s) : launch<1, false, false>(a, f, s);
    if (groups == 2) return a.two ? launch<2, false, true>(a, f, s) : launch<2, false, false>(a, f, s);
    return a.two ? launch<4, false, true>(a, f, s) : launch<4, false, false>(a, f, s);
}

}  // namespace xtq
