// moe_kernels.hip -- the mixture layer's products with its experts' trellis
// weights, for a few rows: gate and up, then down.
//
// Built once per codebook (XTQ_MOE_CODE); the experts' widths are chosen in the
// kernels, per workgroup.
#include "epilogue.h"
#include "moe_device.h"

#pragma clang fp contract(off)

namespace xtq {
namespace {

constexpr int kCode = XTQ_MOE_CODE;
constexpr int W = 8;                    // waves of a workgroup
constexpr int kLds = few_lds(7, W, true, true), kLdsApart = few_lds(7, W, false, true);
static_assert(kLds >= few_lds(2, W, true, true) && kLds >= few_lds(4, W, true, true) &&
              kLds >= few_lds(6, W, true, true), "LDS of every width");

// few_sums of an expert's width (one of 2..7: checked when the table was made).
template <bool FUSED>
__device__ __forceinline__ void expert_sums(int K, const FewSource& src, int s0, int s1, u4* lds, int32_t* shifts,
                                            f4 (&total)[1][1]) {
    switch (K) {
        case 2: return few_sums<2, kCode, 1, W, FUSED, true>(src, s0, s1, lds, shifts, total);
        case 3: return few_sums<3, kCode, 1, W, FUSED, true>(src, s0, s1, lds, shifts, total);
        case 4: return few_sums<4, kCode, 1, W, FUSED, true>(src, s0, s1, lds, shifts, total);
        case 5: return few_sums<5, kCode, 1, W, FUSED, true>(src, s0, s1, lds, shifts, total);
        case 6: return few_sums<6, kCode, 1, W, FUSED, true>(src, s0, s1, lds, shifts, total);
        default: return few_sums<7, kCode, 1, W, FUSED, true>(src, s0, s1, lds, shifts, total);
    }
}

__device__ __forceinline__ void split_range(int pairs, int splits, int split, int& s0, int& s1) {
    const int each = pairs / splits, more = pairs - each * splits;
    s0 = split * each + (split < more ? split : more);
    s1 = s0 + each + (split < more ? 1 : 0);
}

// Rows of x for the first product, as fragments and what their rounding left,
// one wave per chunk, weight (gate, up) and 128-column block.  (For one row the
// product's workgroups do this themselves, each again: one launch less; us of
// whole layers in replayed graphs with and without it, 2048 by 1024 and 4096 by 2048: one row 46 : 41 and 52 : 51, two 53 :
// 52 and 67 : 73, four 72 : 73 and 96 : 107.)  Latency bounds it: 8.9 us for 37 rows of 4096 and 4 of 32
// experts.
__global__ __launch_bounds__(256) void moe_x_kernel(MoeArgs a) {
    const int lane = threadIdx.x & 63, nk = a.d / 128, role = blockIdx.y, ch = blockIdx.z;
    const int kb = blockIdx.x * 4 + (threadIdx.x >> 6);
    const MoeChunk& c = a.chunks[ch];
    const xtq_moe_weight w = c.w[role];
    if (ch >= *a.nchunks || kb >= nk) return;
    float su, sv;
    unpack_two(load_two(w.suh + 128 * kb, lane), kF16, su, sv);
    u4* hi = a.xf + ((size_t)(ch * 2 + role) * 2 * nk + kb) * 256;
    int32_t* sh = a.xs + ((size_t)(ch * 2 + role) * nk + kb) * 16;
#pragma unroll 4
    for (int r = 0; r < c.rows; ++r) {
        const size_t row = c.slots[r] / a.top;
        float u, v;
        unpack_two(load_two(a.x + row * a.x_stride + 128 * kb, lane), a.type, u, v);
        const int s = row_to_frags<true>(u * su, v * sv, lane, r, (uint32_t*)hi, (uint32_t*)(hi + (size_t)nk * 256));
        if (lane == 0) sh[r] = s;
    }
}

// One weight's (gate's or up's) 128 columns for a chunk over a part of the summed
// dimension (FUSED: of the only row, transformed here); the last workgroup of the two weights' parts adds them, applies the
// activation and leaves the product's rows as fragments for the second product.
// The decoding bounds it: 32 experts' gate and up of 4096 by 2048 are 537 M
// weights, 57 us of vector instructions, of 102 us in all; the compute units
// decode for 117,000 of a launch's 201,000 cycles, two workgroups a unit, the rest
// are joins while one decodes alone.  (Four waves a workgroup and four workgroups:
// 105 us.)  One token and 8 experts of 2048 by 1024: 16 us, latency.
template <bool FUSED>
__global__ __launch_bounds__(64 * W, 4) void moe_up_kernel(MoeArgs a) {
    __shared__ __align__(16) u4 lds[(FUSED ? kLds : kLdsApart) / 16];
    __shared__ int32_t shifts[kFewMaxSlice * 16];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nf = a.f / 128, nk = a.d / 128, ch = blockIdx.z, split = blockIdx.y;
    const int fb = blockIdx.x >> 1, role = blockIdx.x & 1;
    const MoeChunk& c = a.chunks[ch];   // (read before its number is known to be one)
    const int rows = c.rows;
    const xtq_moe_weight w = c.w[role];
    if (ch >= *a.nchunks) return;
    int s0, s1;
    split_range(a.d / 32, a.up_splits, split, s0, s1);
    const u4* hi = FUSED ? nullptr : a.xf + (size_t)(ch * 2 + role) * 2 * nk * 256;
    const FewSource src{(const uint8_t*)w.trellis + (size_t)fb * 256 * w.K, (size_t)nf * 256 * w.K, rows, a.d / 32,
                        a.x, a.x_stride, w.suh, a.type, 65536u / rows + 1, hi,
                        FUSED ? nullptr : hi + (size_t)nk * 256,
                        FUSED ? nullptr : a.xs + (size_t)(ch * 2 + role) * nk * 16};
    f4 total[1][1];
    expert_sums<FUSED>(w.K, src, s0, s1, lds, shifts, total);
    // [chunk][fb][role][split][row][128]
    float* part = a.up_part + ((size_t)ch * nf + fb) * 2 * a.up_splits * 2048;
    if ((lane & 15) < rows)
        store_shared(part + (size_t)(role * a.up_splits + split) * 2048 + (lane & 15) * 128 + 16 * wv + 4 * (lane >> 4),
                     total[0][0]);
    const xtq_moe_weight wg = c.w[0], wu = c.w[1], wd = c.w[2];
    float g0, g1, u0, u1, d0, d1;       // (on their way while the workgroups meet)
    unpack_two(load_two(wg.svh + 128 * fb, lane), kF16, g0, g1);
    unpack_two(load_two(wu.svh + 128 * fb, lane), kF16, u0, u1);
    unpack_two(load_two(wd.suh + 128 * fb, lane), kF16, d0, d1);
    if (!arrive(a.counters + kMoeRouterCounters + a.d / 128 + ch * nf + fb, 2 * a.up_splits, threadIdx.x)) return;
    u4* out = a.hf + ((size_t)ch * 2 * nf + fb) * 256;
#pragma unroll 1
    for (int r0 = wv; r0 < rows; r0 += 2 * W) {
        float v[2][2], u[2][2];
        sum_rows<4, 2>(v, part, r0, W, rows, 2048, a.up_splits, lane);
        sum_rows<4, 2>(u, part + (size_t)a.up_splits * 2048, r0, W, rows, 2048, a.up_splits, lane);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + i * W;
            if (r >= rows) break;
            transform_row(v[i][0], v[i][1], lane);
            transform_row(u[i][0], u[i][1], lane);
            v[i][0] *= g0 * wg.scale;
            v[i][1] *= g1 * wg.scale;
            activate<2>(v[i], a.act);
            v[i][0] *= u[i][0] * (u0 * wu.scale);
            v[i][1] *= u[i][1] * (u1 * wu.scale);
            const int sh = row_to_frags<true>(v[i][0] * d0, v[i][1] * d1, lane, r, (uint32_t*)out,
                                              (uint32_t*)(out + (size_t)nf * 256));
            if (lane == 0) a.hs[((size_t)ch * nf + fb) * 16 + r] = sh;
        }
    }
}

// The last step for 128 columns: each row's residual and the weighted results
// of its slots, four rows and eight parts of each in flight by a wave.
__device__ __forceinline__ void moe_finish(const MoeArgs& a, int db, int first, int step, int lane) {
    const int col = 128 * db + 2 * lane;
    const size_t slots = (size_t)a.rows * a.top;
    for (int r0 = first; r0 < a.rows; r0 += 4 * step) {
        float o[4][2];
        bool in[4], any = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = r0 + i * step;
            in[i] = row < a.rows && !(a.valid && !a.valid[row]);
            any |= in[i];
            o[i][0] = o[i][1] = 0.0f;
        }
        const int parts = a.top * a.down_splits;
        if (any)
            for (int p0 = 0; p0 < parts; p0 += 8) {
                u64 t[8][4];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int p = p0 + u < parts ? p0 + u : p0, place = p / a.down_splits;
                    const float* at = a.out + (size_t)(p - place * a.down_splits) * slots * a.d + col;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        t[u][i] = in[i] ? __hip_atomic_load((const u64*)(at + ((size_t)(r0 + i * step) * a.top + place) * a.d),
                                                            __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                                        : 0;
                }
#pragma unroll
                for (int u = 0; u < 8; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (p0 + u < parts) {
                            o[i][0] += __uint_as_float((uint32_t)t[u][i]);
                            o[i][1] += __uint_as_float((uint32_t)(t[u][i] >> 32));
                        }
            }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = r0 + i * step;
            if (row >= a.rows) break;
            if (a.res) {
                float u, v;
                unpack_two(*(const u1_a2*)(a.res + (size_t)row * a.res_stride + col), a.type, u, v);
                o[i][0] += u;
                o[i][1] += v;
            }
            uint16_t* y = a.y + (size_t)row * a.y_stride + col;
            if (a.type == kBf16) store16<kBf16, 2>(y, o[i]);
            else store16<kF16, 2>(y, o[i]);
        }
    }
}

// down's 128 columns for a chunk over a part of the summed dimension, weighted,
// by slot; the last workgroup of the columns adds each row's slots in order.
// Bound as up is: 64 us for the 268 M weights of 32 experts of 2048 by 4096, 28 of
// them instructions of the decoding; 13 us for one token and 8 experts.
__global__ __launch_bounds__(64 * W, 4) void moe_down_kernel(MoeArgs a) {
    __shared__ __align__(16) u4 lds[kLdsApart / 16];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nf = a.f / 128, db = blockIdx.x, split = blockIdx.y, ch = blockIdx.z, nchunks = *a.nchunks;
    const MoeChunk& c = a.chunks[ch];
    const xtq_moe_weight w = c.w[2];
    if (ch >= nchunks) {
        // no row has an expert: residuals and zeros
        if (nchunks == 0 && ch == 0 && split == 0) moe_finish(a, db, wv, W, lane);
        return;
    }
    int s0, s1;
    split_range(a.f / 32, a.down_splits, split, s0, s1);
    const u4* hi = a.hf + (size_t)ch * 2 * nf * 256;
    const FewSource src{(const uint8_t*)w.trellis + (size_t)db * 256 * w.K, (size_t)(a.d / 128) * 256 * w.K, c.rows,
                        a.f / 32, nullptr, 0, nullptr, 0, 0, hi, hi + (size_t)nf * 256,
                        a.hs + (size_t)ch * nf * 16};
    f4 total[1][1];
    expert_sums<false>(w.K, src, s0, s1, lds, nullptr, total);
    f4* const sums = (f4*)lds;
    sums[wv * 64 + lane] = total[0][0];
    float v0, v1;
    unpack_two(load_two(w.svh + 128 * db, lane), kF16, v0, v1);
    __syncthreads();
    for (int r = wv; r < c.rows; r += W) {
        float v[2];
        unit_row(sums, r, lane, v[0], v[1]);
        transform_row(v[0], v[1], lane);
        const int slot = c.slots[r];
        const float by = a.weights[slot] * w.scale;
        float* at = a.out + ((size_t)split * a.rows * a.top + slot) * a.d + 128 * db + 2 * lane;
        __hip_atomic_store((u64*)at, (u64)__float_as_uint(v[0] * (v0 * by)) | (u64)__float_as_uint(v[1] * (v1 * by)) << 32,
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (!arrive(a.counters + kMoeRouterCounters + db, nchunks * a.down_splits, threadIdx.x)) return;
    moe_finish(a, db, wv, W, lane);
}

}  // namespace

#define XTQ_CAT2(a, b) a##b
#define XTQ_CAT(a, b) XTQ_CAT2(a, b)

hipError_t XTQ_CAT(launch_moe_code, XTQ_MOE_CODE)(const MoeArgs& a, hipStream_t s) {
    const dim3 block(64 * W), up(2 * (a.f / 128), a.up_splits, a.max_chunks),
        down(a.d / 128, a.down_splits, a.max_chunks);
    if (a.rows == 1) {
        hipLaunchKernelGGL((moe_up_kernel<true>), up, block, 0, s, a);
    } else {
        hipLaunchKernelGGL(moe_x_kernel, dim3((a.d / 128 + 3) / 4, 2, a.max_chunks), dim3(256), 0, s, a);
        hipLaunchKernelGGL((moe_up_kernel<false>), up, block, 0, s, a);
    }
    hipLaunchKernelGGL(moe_down_kernel, down, block, 0, s, a);
    return hipGetLastError();
}

}  // namespace xtq
