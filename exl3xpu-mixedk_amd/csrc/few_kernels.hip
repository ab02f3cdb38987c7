// few_kernels.hip -- linear layers of few rows (up to 64): the weight is decoded
// on its way to the matrix cores.
//
// Built once per width K (XTQ_FEW_K), so that the widths compile side by side,
// and once more (XTQ_FEW_TWO) for two terms of rows that come transformed.
#include "epilogue.h"
#include "few_device.h"

#pragma clang fp contract(off)

namespace xtq {
namespace {

// A workgroup makes 128 columns (one transform block) of up to 16 G rows over a
// run of the summed dimension, its waves each a part of that.  FUSED (up to
// kFusedRows rows): it transforms the rows' part itself, a wave one row's block
// at a time, into LDS.  The waves' sums meet in LDS, the workgroups' in scratch,
// where the last one to arrive adds them in order and finishes the columns.
// LO: with two terms.
//
// The decoding bounds it.  One row of 17408 by 5120 at K = 4 (22.9 us; 44.6 MB that
// a copy would move in 9.0) is 7.0 M wave instructions, 5.0 a weight, 3.85 of which
// issue at 33-37 T lane-operations/s: 27,400 cycles of every SIMD, 12.3 us.  By
// clocks of all waves, 51,000 cycles from a wave's start: 7,600 until the row is
// transformed and the first weights lie in LDS (12,100 for the last wave), 31,000
// more until the last wave has multiplied, 2,100 for the waves' sums, 1,000 to
// store them, 1,800 to arrive, 3,100 to read the other workgroups' parts and
// finish.  In the 31,000 the two workgroups of a compute unit
// go one after the other more than side by side: the first is through its 8 blocks
// at 14,300, the second at 32,400, and each then transforms the row's 4 further
// blocks (few_slice) and starts its loads anew, 5,900 cycles that only the
// neighbour's decoding can hide, and the last of them nothing.
// 5120 by 5120 takes 12.6 us: 6,300 cycles (9,000) until the loop, 8,100 in it, 2,500,
// 1,000 and 2,300 for sums, parts and arrival, 2,200 to finish.
template <int K, int CODE, int G, bool FUSED, bool LO>
__global__ __launch_bounds__(64 * few_waves(G), G == 1 ? 4 : 2) void few_kernel(Weight w, FewArgs a, Epilogue ep) {
    constexpr int W = few_waves(G), N = 8 / W;
    __shared__ __align__(16) u4 lds[few_lds(K, W, FUSED, LO) / 16];
    __shared__ int32_t shifts[FUSED ? kFewMaxSlice * 16 : 1];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nb = gridDim.x, blk = blockIdx.x, split = blockIdx.y;
    // this workgroup's 32-row steps
    const int s0 = split * a.steps + (split < a.more ? split : a.more), s1 = s0 + a.steps + (split < a.more ? 1 : 0);
    const FewSource src{(const uint8_t*)w.trellis + (size_t)blk * 256 * K, (size_t)nb * 256 * K, ep.rows, w.k / 32,
                        a.x, a.x_stride, w.suh, a.type, a.rinv, a.frag, a.frag_lo, a.shift};
    f4 total[G][N];
    few_sums<K, CODE, G, W, FUSED, LO>(src, s0, s1, lds, shifts, total);
    // (on their way while the workgroups meet)
    const Columns<2> cols = a.type == kBf16 ? load_columns<kBf16, 2>(ep, blk * 128 + 2 * lane)
                                            : load_columns<kF16, 2>(ep, blk * 128 + 2 * lane);
    if (a.splits > 1) {
        // [split][blk][row][128]
        float* mine = a.part + ((size_t)split * nb + blk) * ep.rows * 128 + 4 * (lane >> 4);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int row = 16 * g + (lane & 15);
            if (row < ep.rows) {
#pragma unroll
                for (int i = 0; i < N; ++i) store_shared(mine + row * 128 + 16 * (i * W + wv), total[g][i]);
            }
        }
        if (!arrive(a.counters + blk, a.splits, threadIdx.x)) return;
        constexpr int R = G == 1 ? 2 : 4, U = G == 1 ? 16 : 4;
#pragma unroll 1
        for (int r0 = wv; r0 < ep.rows; r0 += R * W) {
            float v[R][2];
            sum_rows<U, R>(v, a.part + (size_t)blk * ep.rows * 128, r0, W, ep.rows, (size_t)nb * ep.rows * 128,
                           a.splits, lane);
            finish_rows<R>(v, cols, ep, a.type, blk, r0, W, lane);
        }
        return;
    }
    f4* const sums = (f4*)lds;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < N; ++i) sums[(g * 8 + i * W + wv) * 64 + lane] = total[g][i];
    __syncthreads();
#pragma unroll 1
    for (int r0 = wv; r0 < ep.rows; r0 += 4 * W) {
        float v[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = r0 + i * W < ep.rows ? r0 + i * W : r0;
            unit_row(sums + (row >> 4) * 512, row & 15, lane, v[i][0], v[i][1]);
        }
        finish_rows<4>(v, cols, ep, a.type, blk, r0, W, lane);
    }
}

template <int K, int CODE, int G, bool FUSED, bool LO>
hipError_t few_launch(const Weight& w, const FewArgs& a, const Epilogue& ep, hipStream_t s) {
    hipLaunchKernelGGL((few_kernel<K, CODE, G, FUSED, LO>), dim3(w.n / 128, a.splits), dim3(64 * few_waves(G)), 0, s,
                       w, a, ep);
    return hipGetLastError();
}

// (Rows and fragments are held against each other here once more: the kernels
// themselves take them as they come.)
template <int K, int CODE>
hipError_t few_kc(const Weight& w, const FewArgs& a, const Epilogue& ep, hipStream_t s) {
    if (ep.rows > (a.frag ? 16 * a.groups : kFusedRows)) return hipErrorInvalidValue;
#ifdef XTQ_FEW_TWO
    if (!a.frag || !a.frag_lo) return hipErrorInvalidValue;
    if (a.groups == 1) return few_launch<K, CODE, 1, false, true>(w, a, ep, s);
    if (a.groups == 2) return few_launch<K, CODE, 2, false, true>(w, a, ep, s);
    return few_launch<K, CODE, 4, false, true>(w, a, ep, s);
#else
    if (a.two) return few_launch<K, CODE, 1, true, true>(w, a, ep, s);
    if (!a.frag) return few_launch<K, CODE, 1, true, false>(w, a, ep, s);
    if (a.groups == 1) return few_launch<K, CODE, 1, false, false>(w, a, ep, s);
    if (a.groups == 2) return few_launch<K, CODE, 2, false, false>(w, a, ep, s);
    return few_launch<K, CODE, 4, false, false>(w, a, ep, s);
#endif
}

}  // namespace

#define XTQ_CAT2(a, b) a##b
#define XTQ_CAT(a, b) XTQ_CAT2(a, b)
#ifdef XTQ_FEW_TWO
#define XTQ_FEW_NAME launch_few2_k
#else
#define XTQ_FEW_NAME launch_few_k
#endif

hipError_t XTQ_CAT(XTQ_FEW_NAME, XTQ_FEW_K)(const Weight& w, const FewArgs& a, const Epilogue& ep,
                                            hipStream_t s) {
    if (w.code == kCodeMul1) return few_kc<XTQ_FEW_K, kCodeMul1>(w, a, ep, s);
    if (w.code == kCodeMcg) return few_kc<XTQ_FEW_K, kCodeMcg>(w, a, ep, s);
    return few_kc<XTQ_FEW_K, kCode3Inst>(w, a, ep, s);
}

}  // namespace xtq
