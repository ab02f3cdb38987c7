// few_kernels.hip -- linear layers of few rows (up to 64): the weight is decoded
// on its way to the matrix cores.
//
// Built once per width K (XTQ_FEW_K), so that the widths compile side by side.
#include "epilogue.h"
#include "few_device.h"

#pragma clang fp contract(off)

namespace xtq {
namespace {

constexpr int kSlice = 8;               // 128-row blocks transformed at a time (FUSED)

// A workgroup makes 128 columns (one transform block) of up to 16 G rows over a
// run of the summed dimension, its waves each a part of that.  FUSED (up to
// kFusedRows rows): it transforms the rows' part itself, a wave one row's block
// at a time, into LDS.  The waves' sums meet in LDS, the workgroups'
// in scratch, where the last one to arrive adds them in order and finishes the
// columns.
template <int K, int CODE, int G, bool FUSED>
__global__ __launch_bounds__(64 * kFewWaves, 2) void few_kernel(Weight w, FewArgs a, Epilogue ep) {
    // the rows' fragments, later the waves' sums
    __shared__ __align__(16) u4 lds[FUSED && kSlice * 256 > kFewWaves * 512 ? kSlice * 256 : kFewWaves * 512];
    __shared__ __align__(16) uint8_t bufs[kFewWaves][2][kPairBytes<K>];
    __shared__ int32_t shifts[FUSED ? kSlice * 16 : 1];
    u4* const frag = lds;
    f4* const sums = (f4*)lds;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4;
    const int nb = gridDim.x, blk = blockIdx.x, split = blockIdx.y, pairs = w.k / 32;
    // this workgroup's 32-row steps
    const int s0 = split * a.steps + (split < a.more ? split : a.more), s1 = s0 + a.steps + (split < a.more ? 1 : 0);
    const size_t row_bytes = (size_t)nb * 256 * K;
    const uint8_t* tiles = (const uint8_t*)w.trellis + (size_t)blk * 256 * K;
    const Window win = lane_window<K>(lane);
    uint8_t* const buf = bufs[wv][0];

    f4 acc[G][8];
    int shift[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        shift[g] = kNoShift;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[g][j] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int chunk = FUSED ? 4 * kSlice : pairs;
    for (int c0 = s0; c0 < s1;) {
        const int kb0 = c0 >> 2, c1 = FUSED && (kb0 << 2) + chunk < s1 ? (kb0 << 2) + chunk : s1;
        const int p0 = c0 + (c1 - c0) * wv / kFewWaves, p1 = c0 + (c1 - c0) * (wv + 1) / kFewWaves;
        PairRegs<K> r[2];
        auto load = [&](PairRegs<K>& t, int p) {
            p = p < p1 ? p : p1 - 1;
            load_pair<K>(t, tiles + (size_t)p * 2 * row_bytes, row_bytes, lane);
        };
        if constexpr (FUSED) {
            const int nk = ((c1 + 3) >> 2) - kb0, items = ep.rows * nk;
            if (c0 > s0) __syncthreads();
            for (int t = wv; t < items || t == wv; t += 4 * kFewWaves) {
                uint32_t xw[4], sw[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int item = t + i * kFewWaves;
                    if (item >= items) break;
                    const int kbi = item * a.rinv >> 16, row = item - kbi * ep.rows;
                    xw[i] = load_two(a.x + (size_t)row * a.x_stride + 128 * (kb0 + kbi), lane);
                    sw[i] = load_two(w.suh + 128 * (kb0 + kbi), lane);
                }
                if (t == wv && p0 < p1) {               // behind the first rows' loads
                    load(r[0], p0);
                    load(r[1], p0 + 1);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int item = t + i * kFewWaves;
                    if (item >= items) break;
                    const int kbi = item * a.rinv >> 16, row = item - kbi * ep.rows;
                    float u, v, su, sv;
                    unpack_two(xw[i], a.type, u, v);
                    unpack_two(sw[i], kF16, su, sv);
                    const int sh = row_to_frags<false>(u * su, v * sv, lane, row, (uint32_t*)(frag + kbi * 256),
                                                       nullptr);
                    if (lane == 0) shifts[kbi * 16 + row] = sh;
                }
            }
            __syncthreads();
        } else if (p0 < p1) {
            load(r[0], p0);
            load(r[1], p0 + 1);
        }
        u4 x[G], nx[G];
        float f[G];
        const u4 zero = {0u, 0u, 0u, 0u};
        auto fetch = [&](u4 (&t)[G], int p) {
            if constexpr (FUSED) {
                t[0] = (lane & 15) < ep.rows ? frag[(p - 4 * kb0) * 64 + lane] : zero;
            } else {
                p = p < p1 ? p : p1 - 1;
#pragma unroll
                for (int g = 0; g < G; ++g) t[g] = a.frag[((size_t)g * pairs + p) * 64 + lane];
            }
        };
        // pair p lies in its buffer, p + 1 is on its way in r[odd ^ 1], p + 2 in r[odd]
        auto step = [&](int p, int odd) {
            pair_to_lds<K>(r[odd ^ 1], buf + (odd ^ 1) * kPairBytes<K>, lane);
            load(r[odd ^ 1], p + 3);
            if (p == p0 || (p & 3) == 0) {
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    int own;
                    if constexpr (FUSED) own = (lane & 15) < ep.rows ? shifts[((p >> 2) - kb0) * 16 + (lane & 15)] : kNoShift;
                    else own = a.shift[((size_t)g * (pairs >> 2) + (p >> 2)) * 16 + (lane & 15)];
                    meet(acc[g], shift[g], own, f[g]);
                }
            }
            if constexpr (FUSED) {
                fetch(x, p);
            } else {
#pragma unroll
                for (int g = 0; g < G; ++g) x[g] = nx[g];
                fetch(nx, p + 1);
            }
#pragma unroll
            for (int g = 0; g < G; ++g) x[g] = scaled(x[g], f[g]);
            pair_product<K, CODE, G>(acc, buf + odd * kPairBytes<K>, win, x);
            wave_sync();
        };
        if (p0 < p1) {
            if constexpr (!FUSED) fetch(nx, p0);
            pair_to_lds<K>(r[0], buf, lane);
            load(r[0], p0 + 2);
            wave_sync();
            for (int p = p0; p < p1; p += 2) {
                step(p, 0);
                if (p + 1 < p1) step(p + 1, 1);
            }
        }
        c0 = c1;
    }

    // the waves' sums, wave w adding tile columns w, w + kFewWaves, .. in the
    // order of the waves
    constexpr int NJ = 8 / kFewWaves;
    f4 total[G][NJ];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float s = shift[g] == kNoShift ? 0.0f : ldexpf(1.0f, -shift[g] - 7);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[(wv * 8 + j) * 64 + lane] = acc[g][j] * s;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NJ; ++i) {
            total[g][i] = sums[(i * kFewWaves + wv) * 64 + lane];
#pragma unroll
            for (int o = 1; o < kFewWaves; ++o) total[g][i] += sums[(o * 8 + i * kFewWaves + wv) * 64 + lane];
        }
    }
    if (a.splits > 1) {
        float* mine = a.part + ((size_t)split * nb + blk) * G * 2048 + wv * 256 + lane * 4;
#pragma unroll
        for (int g = 0; g < G; ++g)
            if (16 * g + (lane & 15) < ep.rows) {
#pragma unroll
                for (int i = 0; i < NJ; ++i) store_shared(mine + g * 2048 + i * kFewWaves * 256, total[g][i]);
            }
        if (!arrive(a.counters + blk, a.splits, threadIdx.x)) return;
#pragma unroll
        for (int g = 0; g < G; ++g)
            if (16 * g + (lane & 15) < ep.rows)
                sum_shared<16 / G>(total[g], a.part + ((size_t)blk * G + g) * 2048 + wv * 256 + lane * 4,
                                   kFewWaves * 256, (size_t)nb * G * 2048, a.splits);
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < NJ; ++i) sums[(g * 8 + i * kFewWaves + wv) * 64 + lane] = total[g][i];
    __syncthreads();
    if (a.type == kBf16) finish_rows<kBf16>(sums, ep, blk, wv, kFewWaves, lane);
    else finish_rows<kF16>(sums, ep, blk, wv, kFewWaves, lane);
}

template <int K, int CODE>
hipError_t few_kc(const Weight& w, const FewArgs& a, const Epilogue& ep, hipStream_t s) {
    const dim3 grid(w.n / 128, a.splits), block(64 * kFewWaves);
    if (!a.frag) hipLaunchKernelGGL((few_kernel<K, CODE, 1, true>), grid, block, 0, s, w, a, ep);
    else if (ep.rows <= 16) hipLaunchKernelGGL((few_kernel<K, CODE, 1, false>), grid, block, 0, s, w, a, ep);
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
