// moe_router.hip -- the mixture layer's router: logits, top-k with softmax
// weights, and the experts' work lists, in one launch; and the layer's launch.
#include "moe_device.h"

#pragma clang fp contract(off)

namespace xtq {
namespace {

constexpr int kGroup = 4;               // rows of a workgroup

__device__ __forceinline__ float wave_sum(float v) {
    v += lane_xor<1>(v);
    v += lane_xor<2>(v);
    v += lane_xor<4>(v);
    v += lane_xor<8>(v);
    const uint32_t a = __float_as_uint(v);
    auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const uint32_t b = __float_as_uint(v);
    r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto most = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
    auto move = [](uint32_t x, auto c) {
        return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, decltype(c)::value, 0xf, 0xf, true);
    };
    v = most(v, move(v, std::integral_constant<int, 0xB1>()));     // pairs, fours, eights, sixteens
    v = most(v, move(v, std::integral_constant<int, 0x4E>()));
    v = most(v, move(v, std::integral_constant<int, 0x141>()));
    v = most(v, move(v, std::integral_constant<int, 0x140>()));
    auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = most(r[0], r[1]);
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return most(r[0], r[1]);
}

// Order of the logits as unsigned numbers: -0 is 0, NaN is above infinity.
__device__ __forceinline__ uint32_t order_key(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// The logit of a key (NaN for NaN's).
__device__ __forceinline__ float order_value(uint32_t key) {
    return __uint_as_float(key == 0xFFFFFFFFu ? key : (key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// A row's top-k by a wave: the largest logits, ties to the lowest expert, and
// their softmax weights over all experts (renorm: over the chosen ones).  N: 64
// N experts at most.
template <int N>
__device__ void choose(const MoeArgs& a, int row, int lane) {
    if (a.valid && !a.valid[row]) {
        if (lane < a.top) {
            a.ids[row * a.top + lane] = -1;
            a.weights[row * a.top + lane] = 0.0f;
        }
        return;
    }
    float v[N];
    uint32_t key[N];
    float top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = lane + 64 * i;
        v[i] = -INFINITY;
        key[i] = 0u;                                    // below every logit's
        if (e < a.experts) {
            const uint32_t b = __hip_atomic_load((const uint32_t*)a.logits + (size_t)row * a.experts + e,
                                                 __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            v[i] = __uint_as_float(b);
            key[i] = order_key(v[i]);
            nan |= v[i] != v[i];
        }
        top = fmaxf(top, v[i]);
    }
    top = wave_max(top);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (lane + 64 * i < a.experts) sum += expf(v[i] - top);
    sum = wave_sum(sum);
    if (__any(nan)) sum = __builtin_nanf("");
    uint32_t mine = 0u;
    int id = 0;
    for (int j = 0; j < a.top; ++j) {
        uint32_t best = 0u;
#pragma unroll
        for (int i = 0; i < N; ++i) best = key[i] > best ? key[i] : best;
        best = wave_max_u32(best);
        bool found = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const unsigned long long at = __ballot(key[i] == best && lane + 64 * i < a.experts);
            if (at && !found) {
                const int l = __builtin_ctzll(at);
                found = true;
                if (lane == j) {
                    mine = best;
                    id = l + 64 * i;
                }
                if (lane == l) key[i] = 0u;
            }
        }
    }
    // (the choice is a chain of maxima; what it weighs is found for all at once)
    const float p = lane < a.top ? expf(order_value(mine) - top) / sum : 0.0f;
    const float chosen = wave_sum(p);
    if (lane < a.top) {
        const float w = a.renorm ? p / chosen : p;
        __hip_atomic_store(a.ids + row * a.top + lane, id, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        a.weights[row * a.top + lane] = w;
    }
}

// The experts' chunks from all rows' choices, in the order of the experts and of
// the rows.  A row chooses an expert once at most, so 64 bits hold an expert's
// rows, and a slot's place among them is the number of lower bits.
__device__ void make_chunks(const MoeArgs& a) {
    __shared__ unsigned long long mask[kMoeExperts];
    __shared__ int32_t first[kMoeExperts];
    const int t = threadIdx.x, slots = a.rows * a.top;
    for (int e = t; e < a.experts; e += blockDim.x) mask[e] = 0;
    __syncthreads();
    int own[kMoeRows * kMoeTop / 256];
#pragma unroll
    for (int i = 0; i < kMoeRows * kMoeTop / 256; ++i) {
        const int s = t + 256 * i, row = s / a.top;
        own[i] = -1;
        if (s < slots && !(a.valid && !a.valid[row])) {
            own[i] = __hip_atomic_load(a.ids + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            atomicOr(&mask[own[i]], 1ull << row);
        }
    }
    __syncthreads();
    if (t < 64) {                                       // exclusive sums of the experts' chunks
        constexpr int N = kMoeExperts / 64;
        int n[N], mine = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            n[i] = t * N + i < a.experts ? (__popcll(mask[t * N + i]) + 15) / 16 : 0;
            mine += n[i];
        }
        int upto = mine;
        for (int m = 1; m < 64; m <<= 1) {
            const int o = __shfl_up(upto, m);
            if (t >= m) upto += o;
        }
        int at = upto - mine;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (t * N + i < a.experts) first[t * N + i] = at;
            at += n[i];
        }
        if (t == 63) *a.nchunks = upto;
    }
    __syncthreads();
    for (int e = t; e < a.experts; e += blockDim.x) {
        const int rows = __popcll(mask[e]);
        for (int c = 0; 16 * c < rows; ++c) {
            MoeChunk& k = a.chunks[first[e] + c];
            for (int i = 0; i < 3; ++i) k.w[i] = a.table[3 * e + i];
            k.rows = rows - 16 * c < 16 ? rows - 16 * c : 16;
        }
    }
#pragma unroll
    for (int i = 0; i < kMoeRows * kMoeTop / 256; ++i) {
        const int s = t + 256 * i;
        if (own[i] < 0) continue;
        const int place = __popcll(mask[own[i]] & ((1ull << (s / a.top)) - 1));
        a.chunks[first[own[i]] + place / 16].slots[place % 16] = s;
    }
}

// A workgroup makes one expert's logits of 4 rows, in fp32, its waves a quarter
// of the products each.  The one that finishes the last logits of its rows
// chooses for them, the one that finishes the last rows makes the lists.
// Latency bounds it: loads, sums, two arrivals and the choice in turn, 8.3 us for one
// token and 64 experts of 2048, 14 for 37 tokens and 32 experts of 4096.
__global__ __launch_bounds__(256) void moe_router_kernel(MoeArgs a) {
    __shared__ float sums[4][kGroup];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, e = blockIdx.x, r0 = blockIdx.y * kGroup;
    const int n = a.rows - r0 < kGroup ? a.rows - r0 : kGroup;
    float acc[kGroup];
#pragma unroll
    for (int i = 0; i < kGroup; ++i) acc[i] = 0.0f;
#pragma unroll 2
    for (int c = 8 * (int)threadIdx.x; c < a.d; c += 2048) {
        float w[8];
        if (a.router_f32) {
            const float* p = (const float*)a.router + (size_t)e * a.d + c;
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = p[i];
        } else {
            const u4 t = *(const u4_a2*)((const uint16_t*)a.router + (size_t)e * a.d + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) unpack_two(t[i], a.type, w[2 * i], w[2 * i + 1]);
        }
        u4 t[kGroup];
#pragma unroll
        for (int r = 0; r < kGroup; ++r)
            t[r] = *(const u4_a2*)(a.x + (size_t)(r0 + (r < n ? r : 0)) * a.x_stride + c);
#pragma unroll
        for (int r = 0; r < kGroup; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float u, v;
                unpack_two(t[r][i], a.type, u, v);
                acc[r] = __builtin_fmaf(u, w[2 * i], acc[r]);
                acc[r] = __builtin_fmaf(v, w[2 * i + 1], acc[r]);
            }
    }
#pragma unroll
    for (int r = 0; r < kGroup; ++r) {
        const float s = wave_sum(acc[r]);
        if (lane == 0) sums[wv][r] = s;
    }
    __syncthreads();
    if ((int)threadIdx.x < n) {
        const float s = (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
        __hip_atomic_store(a.logits + (size_t)(r0 + threadIdx.x) * a.experts + e, s, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    }
    if (!arrive(a.counters + blockIdx.y, gridDim.x, threadIdx.x)) return;
    if (wv < n) {
        if (a.experts <= 64) choose<1>(a, r0 + wv, lane);
        else if (a.experts <= 128) choose<2>(a, r0 + wv, lane);
        else choose<kMoeExperts / 64>(a, r0 + wv, lane);
    }
    if (gridDim.y > 1) {
        if (!arrive(a.counters + kMoeRouterCounters - 1, gridDim.y, threadIdx.x)) return;
    } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // the choices are read below
        __syncthreads();
    }
    make_chunks(a);
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

int most_chunks(int rows, int experts, int top) {
    const int slots = rows * top, used = slots < experts ? slots : experts;
    const int by = used + slots / 16;
    return by < slots ? by : slots;
}

// Parts of a product's summed dimension that make `most` workgroups when the
// slots fall on different experts; each wave has a 32-row step at least.  Up's
// fill the compute units twice; down's once, since the last of its workgroups
// reads every part of every slot (one token, 8 experts of 2048 by 1024: 15 us,
// 20 with twice the parts; up 17, 19 with half).
int moe_splits(int dim, int wgs, int most) {
    int s = most / wgs;
    if (s > dim / 256) s = dim / 256;
    return s < 1 ? 1 : s;
}

struct MoePlan {
    int chunks, up_splits, down_splits;
    size_t logits, nchunks, list, xf, xs, part, hf, hs, out, total;
};

MoePlan moe_plan(int rows, int experts, int top, int d, int f) {
    MoePlan p;
    p.chunks = most_chunks(rows, experts, top);
    const int slots = rows * top, likely = slots < experts ? slots : experts;
    p.up_splits = moe_splits(d, likely * 2 * (f / 128), 2 * kCUs);
    p.down_splits = moe_splits(f, likely * (d / 128), kCUs);
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t a = at; at += align256(bytes); return a; };
    const size_t n = p.chunks;
    p.logits = take((size_t)rows * experts * 4);
    p.nchunks = take(4);
    p.list = take(n * sizeof(MoeChunk));
    const bool apart = rows > 1;
    p.xf = take(apart ? n * 4 * d * 32 : 0);
    p.xs = take(apart ? n * 2 * (d / 128) * 64 : 0);
    p.part = take(n * (f / 128) * 2 * p.up_splits * 8192);
    p.hf = take(n * 2 * f * 32);
    p.hs = take(n * (f / 128) * 64);
    p.out = take((size_t)p.down_splits * slots * d * 4);
    p.total = at;
    return p;
}

}  // namespace

size_t moe_ws_bytes(int rows, int experts, int top, int d, int f) { return moe_plan(rows, experts, top, d, f).total; }

size_t moe_counters(int rows, int experts, int top, int d, int f) {
    return kMoeRouterCounters + d / 128 + (size_t)most_chunks(rows, experts, top) * (f / 128);
}

hipError_t launch_moe(MoeArgs a, void* ws, hipStream_t s) {
    const MoePlan p = moe_plan(a.rows, a.experts, a.top, a.d, a.f);
    uint8_t* b = (uint8_t*)ws;
    a.logits = (float*)(b + p.logits);
    a.nchunks = (int32_t*)(b + p.nchunks);
    a.chunks = (MoeChunk*)(b + p.list);
    a.xf = (u4*)(b + p.xf);
    a.xs = (int32_t*)(b + p.xs);
    a.up_part = (float*)(b + p.part);
    a.hf = (u4*)(b + p.hf);
    a.hs = (int32_t*)(b + p.hs);
    a.out = (float*)(b + p.out);
    a.max_chunks = p.chunks;
    a.up_splits = p.up_splits;
    a.down_splits = p.down_splits;
    hipLaunchKernelGGL(moe_router_kernel, dim3(a.experts, (a.rows + kGroup - 1) / kGroup), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.code == kCodeMul1) return launch_moe_code0(a, s);
    if (a.code == kCode3Inst) return launch_moe_code1(a, s);
    return launch_moe_code2(a, s);
}

}  // namespace xtq
