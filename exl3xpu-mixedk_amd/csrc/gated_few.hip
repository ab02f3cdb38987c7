// gated_few.hip -- the gated projection of few rows (up to 64): both weights are
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
                                          f4 (&total)[G][8 / few_waves(G)]) {
    constexpr int W = few_waves(G);
    switch (K) {
        case 2: return few_sums<2, kCode, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total);
        case 3: return few_sums<3, kCode, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total);
        case 4: return few_sums<4, kCode, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total);
        case 5: return few_sums<5, kCode, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total);
        case 6: return few_sums<6, kCode, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total);
        default: return few_sums<7, kCode, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total);
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

// A workgroup multiplies one weight's 128 columns over a run of the summed dimension
// (few_sums).  The last one of the two weights' runs adds them in order, transforms
// both and writes act(gate) * up: the values between stay in registers.
template <int G, bool FUSED, bool LO>
__global__ __launch_bounds__(64 * few_waves(G), G == 1 ? 4 : 2) void gated_few_kernel(GatedArgs a, GatedFew f) {
    constexpr int W = few_waves(G), N = 8 / W;
    __shared__ __align__(16) u4 lds[gated_lds<G, FUSED, LO>() / 16];
    __shared__ int32_t shifts[FUSED ? kFewMaxSlice * 16 : 1];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nb = a.w[0].n / 128, blk = blockIdx.x >> 1, role = blockIdx.x & 1, split = blockIdx.y;
    const Weight& w = a.w[role];
    const int steps = w.k / 32, nk = w.k / 128;
    const int s0 = (int)((long long)steps * split / f.splits), s1 = (int)((long long)steps * (split + 1) / f.splits);
    const FewSource src{(const uint8_t*)w.trellis + (size_t)blk * 256 * w.K, (size_t)nb * 256 * w.K, a.rows, steps,
                        a.x, a.x_stride, w.suh, a.type, 65536u / a.rows + 1,
                        FUSED ? nullptr : f.frag + (size_t)role * f.groups * nk * 256,
                        FUSED || !LO ? nullptr : f.frag_lo + (size_t)role * f.groups * nk * 256,
                        FUSED ? nullptr : f.shift + (size_t)role * f.groups * nk * 16};
    f4 total[G][N];
    role_sums<G, FUSED, LO>(w.K, src, s0, s1, lds, shifts, total);
    const size_t run = (size_t)a.rows * 128;
    float* const part = f.part + (size_t)blk * 2 * f.splits * run;
    float* const mine = part + (size_t)(role * f.splits + split) * run + 4 * (lane >> 4);
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const int row = 16 * g + (lane & 15);
        if (row < a.rows)
#pragma unroll
            for (int i = 0; i < N; ++i) store_shared(mine + row * 128 + 16 * (i * W + wv), total[g][i]);
    }
    // (on their way while the workgroups meet)
    const int col = blk * 128 + 2 * lane;
    const Columns<2> cg = role_columns(a, 0, col), cu = role_columns(a, 1, col);
    if (!arrive(f.counters + blk, 2 * f.splits, threadIdx.x)) return;
    constexpr int R = G == 1 ? 2 : 4, U = G == 1 ? 8 : 4;
#pragma unroll 1
    for (int r0 = wv; r0 < a.rows; r0 += R * W) {
        float v[R][2], u[R][2];
        sum_rows<U, R>(v, part, r0, W, a.rows, run, f.splits, lane);
        sum_rows<U, R>(u, part + f.splits * run, r0, W, a.rows, run, f.splits, lane);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            transform_row(v[i][0], v[i][1], lane);
            transform_row(u[i][0], u[i][1], lane);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int row = r0 + i * W;
            if (row >= a.rows) break;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                v[i][c] = v[i][c] * cg.scale[c] + cg.bias[c];
                u[i][c] = u[i][c] * cu.scale[c] + cu.bias[c];
            }
            if (a.z) {
                float* z = a.z + (size_t)row * a.w[0].n + col;
                z[0] = v[i][0];
                z[1] = v[i][1];
                z += (size_t)a.rows * a.w[0].n;
                z[0] = u[i][0];
                z[1] = u[i][1];
            }
            activate<2>(v[i], a.act);
            v[i][0] *= u[i][0];
            v[i][1] *= u[i][1];
            uint16_t* y = a.y + (size_t)row * a.y_stride + col;
            if (a.type == kBf16) store16<kBf16, 2>(y, v[i]);
            else store16<kF16, 2>(y, v[i]);
        }
    }
}

template <int G, bool FUSED, bool LO>
hipError_t launch(const GatedArgs& a, const GatedFew& f, hipStream_t s) {
    hipLaunchKernelGGL((gated_few_kernel<G, FUSED, LO>), dim3(2 * (a.w[0].n / 128), f.splits), dim3(64 * few_waves(G)),
                       0, s, a, f);
    return hipGetLastError();
}

}  // namespace

#define XTQ_CAT2(a, b) a##b
#define XTQ_CAT(a, b) XTQ_CAT2(a, b)

// (Rows and fragments are held against each other here: the kernels take them as
// they come.)
hipError_t XTQ_CAT(launch_gated_few_code, XTQ_GATED_CODE)(const GatedArgs& a, const GatedFew& f, hipStream_t s) {
    if (a.rows > (f.frag ? 16 * f.groups : kFusedRows) || (a.two && f.frag && !f.frag_lo)) return hipErrorInvalidValue;
    if (!f.frag) return a.two ? launch<1, true, true>(a, f, s) : launch<1, true, false>(a, f, s);
    if (f.groups == 1) return a.two ? launch<1, false, true>(a, f, s) : launch<1, false, false>(a, f, s);
    if (f.groups == 2) return a.two ? launch<2, false, true>(a, f, s) : launch<2, false, false>(a, f, s);
    if (f.groups == 4) return a.two ? launch<4, false, true>(a, f, s) : launch<4, false, false>(a, f, s);
    return hipErrorInvalidValue;
}

}  // namespace xtq
