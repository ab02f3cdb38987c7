// few_kernels.hip -- linear layers of few rows (up to 64): the weight is decoded
// on its way to the matrix cores.
//
// Built once per width K (XTQ_FEW_K), so that the widths compile side by side.
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
template <int K, int CODE, int G, bool FUSED>
__global__ __launch_bounds__(64 * kFewWaves, 2) void few_kernel(Weight w, FewArgs a, Epilogue ep) {
    __shared__ __align__(16) u4 lds[kFewLds];
    __shared__ __align__(16) uint8_t bufs[kFewWaves][2][kPairBytes<K>];
    __shared__ int32_t shifts[FUSED ? kSlice<false> * 16 : 1];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nb = gridDim.x, blk = blockIdx.x, split = blockIdx.y;
    // this workgroup's 32-row steps
    const int s0 = split * a.steps + (split < a.more ? split : a.more), s1 = s0 + a.steps + (split < a.more ? 1 : 0);
    const FewSource src{(const uint8_t*)w.trellis + (size_t)blk * 256 * K, (size_t)nb * 256 * K, ep.rows, w.k / 32,
                        a.x, a.x_stride, nullptr, w.suh, a.type, a.rinv, a.frag, nullptr, a.shift};
    f4 total[G][kFewTotals];
    few_sums<K, CODE, G, FUSED, false>(src, s0, s1, lds, bufs[wv][0], shifts, total);
    if (a.splits > 1) {
        float* mine = a.part + ((size_t)split * nb + blk) * G * 2048 + wv * 256 + lane * 4;
#pragma unroll
        for (int g = 0; g < G; ++g)
            if (16 * g + (lane & 15) < ep.rows) {
#pragma unroll
                for (int i = 0; i < kFewTotals; ++i)
                    store_shared(mine + g * 2048 + i * kFewWaves * 256, total[g][i]);
            }
        if (!arrive(a.counters + blk, a.splits, threadIdx.x)) return;
#pragma unroll
        for (int g = 0; g < G; ++g)
            if (16 * g + (lane & 15) < ep.rows)
                sum_shared<16 / G>(total[g], a.part + ((size_t)blk * G + g) * 2048 + wv * 256 + lane * 4,
                                   kFewWaves * 256, (size_t)nb * G * 2048, a.splits);
    }
    f4* const sums = (f4*)lds;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < kFewTotals; ++i) sums[(g * 8 + i * kFewWaves + wv) * 64 + lane] = total[g][i];
    __syncthreads();
    if (a.type == kBf16) finish_rows<kBf16>(sums, ep, blk, wv, kFewWaves, lane);
    else finish_rows<kF16>(sums, ep, blk, wv, kFewWaves, lane);
}

template <int K, int CODE>
hipError_t few_kc(const Weight& w, const FewArgs& a, const Epilogue& ep, hipStream_t s) {
    const dim3 grid(w.n / 128, a.splits), block(64 * kFewWaves);
    if (!a.frag) hipLaunchKernelGGL((few_kernel<K, CODE, 1, true>), grid, block, 0, s, w, a, ep);
    else if (ep.rows <= 32) hipLaunchKernelGGL((few_kernel<K, CODE, 2, false>), grid, block, 0, s, w, a, ep);
    else hipLaunchKernelGGL((few_kernel<K, CODE, 4, false>), grid, block, 0, s, w, a, ep);
    return hipGetLastError();
}

}  // namespace

#define XTQ_CAT2(a, b) a##b
#define XTQ_CAT(a, b) XTQ_CAT2(a, b)

hipError_t XTQ_CAT(launch_few_k, XTQ_FEW_K)(const Weight& w, const FewArgs& a, const Epilogue& ep,
                                            hipStream_t s) {
    if (w.code == kCodeMul1) return few_kc<XTQ_FEW_K, kCodeMul1>(w, a, ep, s);
    if (w.code == kCodeMcg) return few_kc<XTQ_FEW_K, kCodeMcg>(w, a, ep, s);
    return few_kc<XTQ_FEW_K, kCode3Inst>(w, a, ep, s);
}

}  // namespace xtq
