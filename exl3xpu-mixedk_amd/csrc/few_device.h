// few_device.h -- the inner loop of products with trellis weights for few rows.
//
// A wave multiplies 16-row groups of activations with "units" of 128 by 128
// weights (8 by 8 tiles), decoding the trellis in its own registers, straight
// into the matrix cores' operand layout.  In a tile's symbol order
// (tensor_core_perm, quantize.py:101-118) the four symbols 32 (c % 8) + 8 q +
// 4 (c / 8) .. + 3 are column c, rows 2q, 2q + 1, 2q + 8, 2q + 9: lane 16 q + c
// takes them from one window of 16 + 3 K bits, and two tiles one below the other
// give the 8 summed elements of its operand of v_mfma_f32_16x16x32_f16.  The
// activations' fragments follow the same order of the summed dimension, in
// which the lanes of a row differ in bits 1 and 2 only: of the block-128
// transform's seven stages, five are inside a lane and two between lanes.
#pragma once
#include "operators.h"

#pragma clang fp contract(off)

namespace xtq {
namespace {

// Where a lane's window lies in every tile: byte offsets of its last words and
// the shift.  (Words before the first are the stream's last: it is circular.)
struct Window {
    uint32_t o[3], sh;
};

template <int K>
__device__ __forceinline__ Window lane_window(int lane) {
    const int c = lane & 15, q = lane >> 4, t0 = 32 * (c & 7) + 8 * q + 4 * (c >> 3);
    const int e = (t0 + 4) * K - 1, lo = e >> 5;        // the window's last bit
    Window w;
#pragma unroll
    for (int i = 0; i < 3; ++i) w.o[i] = 4u * (uint32_t)((lo - i + 8 * K) % (8 * K));
    w.sh = 31u - ((uint32_t)e & 31u);
    return w;
}

// Words of a window: 16 + 3 K bits ending at a multiple of 4 K.  At K = 7 they
// can begin one bit before the second last word.
template <int K>
constexpr int kWinWords = K == 7 ? 3 : 2;

// Two tile rows by eight tiles on their way from memory: 16 consecutive bytes a
// lane (a lane loading its own windows' words took 16 cycles of the address
// unit per load, four times its share of the decoding).  They pass through a
// buffer of the wave's own in LDS, from which each lane reads its windows.
template <int K>
constexpr int kPairBytes = 512 * K;

template <int K>
struct PairRegs {
    u4 r[(K + 1) / 2];
};

// Lane's i-th 16-byte piece of a pair (odd K: the upper lanes' last is their first
// once more).
template <int K>
__device__ __forceinline__ int pair_piece(int i, int lane) {
    const int c = 64 * i + lane;
    return !(K & 1) || c < 32 * K ? c : lane;
}

template <int K>
__device__ __forceinline__ void load_pair(PairRegs<K>& t, const uint8_t* tiles, size_t row_bytes, int lane) {
#pragma unroll
    for (int i = 0; i < (K + 1) / 2; ++i) {
        const int c = pair_piece<K>(i, lane);
        const bool low = c >= 16 * K;
        t.r[i] = *(const u4_a2*)(tiles + (low ? row_bytes : 0) + 16 * (low ? c - 16 * K : c));
    }
}

template <int K>
__device__ __forceinline__ void pair_to_lds(const PairRegs<K>& t, uint8_t* buf, int lane) {
#pragma unroll
    for (int i = 0; i < (K + 1) / 2; ++i) *(u4*)(buf + 16 * pair_piece<K>(i, lane)) = t.r[i];
}

// Orders a wave's own LDS accesses across its lanes (they execute in order; the
// compiler must keep them so).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Four values of a window, as two pairs of halves.
template <int K, int CODE>
__device__ __forceinline__ u2 decode4(const uint32_t* d, uint32_t sh) {
    const uint32_t w = __builtin_amdgcn_alignbit(d[1], d[0], sh);
    const uint32_t s3 = w & 0xFFFFu, s2 = __builtin_amdgcn_ubfe(w, K, 16),
                   s1 = __builtin_amdgcn_ubfe(w, 2 * K, 16);
    uint32_t s0;
    if constexpr (3 * K + 16 <= 32) {
        s0 = __builtin_amdgcn_ubfe(w, 3 * K, 16);
    } else {
        const uint32_t hi = K == 7 ? __builtin_amdgcn_alignbit(d[kWinWords<K> - 1], d[1], sh) : d[1] >> sh;
        s0 = __builtin_amdgcn_alignbit(hi, w, 3 * K) & 0xFFFFu;
    }
    return (u2){code_pair<CODE>(s0, s1), code_pair<CODE>(s2, s3)};
}

__device__ __forceinline__ f4 mfma16(u4 a, u4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b),
                                                  c, 0, 0, 0);
}

// acc[g][j] += (tiles j of one pair of tile rows, in LDS) x (fragment g, and with
// LO what its rounding left).
template <int K, int CODE, int G, bool LO>
__device__ __forceinline__ void pair_product(f4 (&acc)[G][8], const uint8_t* buf, const Window& win,
                                             const u4 (&x)[G], const u4 (&lo)[G]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        uint32_t d[2][kWinWords<K>];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < kWinWords<K>; ++i)
                d[h][i] = *(const uint32_t*)(buf + win.o[i] + 256 * K * h + 32 * K * j);
        const u2 a = decode4<K, CODE>(d[0], win.sh), b = decode4<K, CODE>(d[1], win.sh);
        const u4 m = {a[0], a[1], b[0], b[1]};
#pragma unroll
        for (int g = 0; g < G; ++g) {
            acc[g][j] = mfma16(m, x[g], acc[g][j]);
            if constexpr (LO) acc[g][j] = mfma16(m, lo[g], acc[g][j]);
        }
    }
}

// A block's values are multiplied with 2^shift, which brings the largest to
// [2^14, 2^15), before they are rounded to fp16.  A wave's sums go by the
// smallest shift of its blocks so far: a block of a larger shift is brought down
// (its fp16 values then lose nothing that counts beside the row's largest), and
// the sums are when the smallest falls.
constexpr int kNoShift = 1000;          // a block of zeros

// One row's 128-column block, times its column scales, transformed and rounded,
// by a wave whose lane l has columns 2 l and 2 l + 1 in x.  Returns the block's
// shift.  frag: the block's fragments; lo (LO): what the rounding left, so that
// products with both have 22 bits of the values.
template <bool LO>
__device__ __forceinline__ int row_to_frags(float a, float b, int lane, int row, uint32_t* frag, uint32_t* lo) {
    transform_row(a, b, lane);
    const float top = wave_max(fmaxf(fabsf(a), fabsf(b)));
    const int sh = top == 0.0f ? kNoShift : shift_to(top, 14);
    const int by = sh == kNoShift ? 0 : sh;
    const float u = ldexpf(a, by), v = ldexpf(b, by);
    const h2 r = {(_Float16)u, (_Float16)v};
    // columns 16 i + 2 q + 8 e, + 1: words 2 (i & 1) + e of lane 16 q + row of fragment i / 2
    const int i = lane >> 3, q = lane & 3, e = (lane >> 2) & 1;
    const int at = ((i >> 1) * 64 + q * 16 + row) * 4 + 2 * (i & 1) + e;
    frag[at] = __builtin_bit_cast(uint32_t, r);
    if constexpr (LO) {
        const h2 l = {(_Float16)(u - (float)r[0]), (_Float16)(v - (float)r[1])};
        lo[at] = __builtin_bit_cast(uint32_t, l);
    }
    return sh;
}

// Lane l's two columns of a 128-column block of 16-bit values.
__device__ __forceinline__ uint32_t load_two(const void* row, int lane) { return ((const u1_a2*)row)[lane]; }

__device__ __forceinline__ void unpack_two(uint32_t w, int type, float& a, float& b) {
    if (type == kBf16) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xFFFF0000u);
    } else {
        a = half_bits(w & 0xFFFFu);
        b = half_bits(w >> 16);
    }
}

// Brings a wave's sums and a block's fragments to one scale; `own`: the block's
// shift, `shift`: the sums', f: what the fragments are multiplied with.
__device__ __forceinline__ void meet(f4 (&acc)[8], int& shift, int own, float& f) {
    const int now = own < shift ? own : shift;
    if (__any(now < shift && shift != kNoShift)) {
        const float d = shift == kNoShift ? 1.0f : ldexpf(1.0f, now - shift);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] *= d;
    }
    shift = now;
    f = own == kNoShift ? 1.0f : ldexpf(1.0f, now - own);
}

__device__ __forceinline__ u4 scaled(u4 x, float f) {
    const _Float16 h = (_Float16)f;
    return __builtin_bit_cast(u4, __builtin_bit_cast(h8, x) * (h8){h, h, h, h, h, h, h, h});
}

// Joining workgroups.  store_shared and load_shared pass what workgroups of other
// XCDs, whose L2 is another, have to see: agent-scope accesses go through to
// memory.  arrive is called by all threads once their stores are issued: each
// wave waits for its own, then one thread counts the workgroup; true for the
// last of `parts`, which has cleared the count for the next call and may read
// all parts with load_shared.  (Release and acquire fences would write back and
// drop whole L2 caches for these few lines.)
typedef unsigned long long u64;
__device__ __forceinline__ void store_shared(float* p, f4 v) {
    const u4 b = __builtin_bit_cast(u4, v);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        __hip_atomic_store((u64*)p + i, (u64)b[2 * i] | (u64)b[2 * i + 1] << 32, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ u64 load_shared(const float* p) {
    return __hip_atomic_load((const u64*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ bool arrive(uint32_t* counter, uint32_t parts, int thread) {
    __shared__ uint32_t before;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (thread == 0) {
        before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (before == parts - 1)
            __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return before == parts - 1;
}

// Lane l's columns 2 l and 2 l + 1 of R rows (row0 + i step, up to rows), each the
// sum of `parts` parts `stride` floats apart, in order; R U loads in flight.  A
// wave's load is one row's 512 bytes: such loads pass no cache, and four lanes'
// 8 bytes of as many lines took four times as long.
template <int U, int R>
__device__ __forceinline__ void sum_rows(float (&v)[R][2], const float* part, int row0, int step, int rows,
                                         size_t stride, int parts, int lane) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i][0] = v[i][1] = 0.0f;
    for (int s = 0; s < parts; s += U) {
        u64 t[U][R];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float* p = part + (s + u < parts ? s + u : s) * stride + 2 * lane;
#pragma unroll
            for (int i = 0; i < R; ++i) t[u][i] = load_shared(p + (row0 + i * step < rows ? row0 + i * step : row0) * 128);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s + u < parts) {
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    v[i][0] += __uint_as_float((uint32_t)t[u][i]);
                    v[i][1] += __uint_as_float((uint32_t)(t[u][i] >> 32));
                }
            }
    }
}

// What a workgroup multiplies: 128 columns of a weight, from `tiles` (row_bytes
// from one tile row to the next), by up to 16 G rows.
struct FewSource {
    const uint8_t* tiles;
    size_t row_bytes;
    int rows, pairs;                    // pairs: 32-row steps of the weight
    // FUSED: the rows, transformed here
    const uint16_t* x;
    long long x_stride;
    const uint16_t* suh;
    int type;
    uint32_t rinv;                      // item / rows is item * rinv >> 16
    // else the rows' fragments [g][pair][64] and shifts [g][block][16]
    const u4 *hi, *lo;
    const int32_t* shift;
};

// LDS of a workgroup of W waves: the waves' trellis buffers, and FUSED the rows'
// fragments (4 KiB a block, 8 with LO), of as many blocks as leave room for a
// second workgroup on the compute unit; at the end the waves' sums lie there.
constexpr int few_slice(int K, int W, bool LO) {
    const int n = (76 * 1024 - W * 2 * 512 * K) / (LO ? 8192 : 4096);
    return n > 8 ? 8 : n;
}
constexpr int few_lds(int K, int W, bool fused, bool LO) {
    const int need = W * 2 * 512 * K + (fused ? few_slice(K, W, LO) * (LO ? 8192 : 4096) : 0);
    return need > 32768 ? need : 32768;
}
constexpr int kFewMaxSlice = 8;

// Sums of steps s0 .. s1 of the summed dimension by W waves: total[g][i] of a
// wave's lane is tile column i W + wave of row group g, in the matrix cores'
// layout.
template <int K, int CODE, int G, int W, bool FUSED, bool LO>
__device__ __forceinline__ void few_sums(const FewSource& a, int s0, int s1, u4* lds, int32_t* shifts,
                                         f4 (&total)[G][8 / W]) {
    constexpr int SL = few_slice(K, W, LO);
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Window win = lane_window<K>(lane);
    uint8_t* const buf = (uint8_t*)lds + wv * 2 * kPairBytes<K>;
    u4 *const frag = lds + W * 64 * K, *const frag_lo = frag + SL * 256;
    f4* const sums = (f4*)lds;
    f4 acc[G][8];
    int shift[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        shift[g] = kNoShift;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[g][j] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (int c0 = s0; c0 < s1;) {
        const int kb0 = c0 >> 2, cut = (kb0 + SL) << 2, c1 = FUSED && cut < s1 ? cut : s1;
        const int p0 = c0 + (c1 - c0) * wv / W, p1 = c0 + (c1 - c0) * (wv + 1) / W;
        PairRegs<K> r[2];
        auto load = [&](PairRegs<K>& t, int p) {
            p = p < p1 ? p : p1 - 1;
            load_pair<K>(t, a.tiles + (size_t)p * 2 * a.row_bytes, a.row_bytes, lane);
        };
        if constexpr (FUSED) {
            const int nk = ((c1 + 3) >> 2) - kb0, items = a.rows * nk;
            if (c0 > s0) __syncthreads();
            for (int t = wv; t < items || t == wv; t += 4 * W) {
                uint32_t xw[4], sw[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int item = t + i * W;
                    if (item >= items) break;
                    const int kbi = item * a.rinv >> 16, row = item - kbi * a.rows;
                    xw[i] = load_two(a.x + (size_t)row * a.x_stride + 128 * (kb0 + kbi), lane);
                    sw[i] = load_two(a.suh + 128 * (kb0 + kbi), lane);
                }
                if (t == wv && p0 < p1) {               // behind the first rows' loads
                    load(r[0], p0);
                    load(r[1], p0 + 1);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int item = t + i * W;
                    if (item >= items) break;
                    const int kbi = item * a.rinv >> 16, row = item - kbi * a.rows;
                    float u, v, su, sv;
                    unpack_two(xw[i], a.type, u, v);
                    unpack_two(sw[i], kF16, su, sv);
                    const int sh = row_to_frags<LO>(u * su, v * sv, lane, row, (uint32_t*)(frag + kbi * 256),
                                                    (uint32_t*)(frag_lo + kbi * 256));
                    if (lane == 0) shifts[kbi * 16 + row] = sh;
                }
            }
            __syncthreads();
        } else if (p0 < p1) {
            load(r[0], p0);
            load(r[1], p0 + 1);
        }
        u4 x[G], lo[G], nx[G], nlo[G];
        int own[G];
        float f[G];
        // A pair's fragments and its block's shifts.  (What lies in the places of
        // rows past the end reaches only such rows' sums, which nobody reads.)  From
        // memory they come a step ahead, and before the trellis words of a later
        // step: loads arrive in order, so a wait for these behind those would be one
        // for both; and all of them unconditionally, so that the waits can count.
        auto fetch = [&](u4 (&t)[G], u4 (&u)[G], int p) {
            if constexpr (FUSED) {
                t[0] = frag[(p - 4 * kb0) * 64 + lane];
                if constexpr (LO) u[0] = frag_lo[(p - 4 * kb0) * 64 + lane];
                own[0] = shifts[((p >> 2) - kb0) * 16 + (lane & 15)];
            } else {
                p = p < p1 ? p : p1 - 1;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    t[g] = a.hi[((size_t)g * a.pairs + p) * 64 + lane];
                    if constexpr (LO) u[g] = a.lo[((size_t)g * a.pairs + p) * 64 + lane];
                    own[g] = a.shift[((size_t)g * (a.pairs >> 2) + (p >> 2)) * 16 + (lane & 15)];
                }
            }
        };
        // pair p lies in its buffer, p + 1 is on its way in r[odd ^ 1], p + 2 in r[odd]
        auto step = [&](int p, int odd) {
            if constexpr (FUSED) {
                fetch(x, lo, p);
            } else {
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    x[g] = nx[g];
                    if constexpr (LO) lo[g] = nlo[g];
                }
            }
            if (p == p0 || (p & 3) == 0) {
#pragma unroll
                for (int g = 0; g < G; ++g)
                    meet(acc[g], shift[g], 16 * g + (lane & 15) < a.rows ? own[g] : kNoShift, f[g]);
            }
            pair_to_lds<K>(r[odd ^ 1], buf + (odd ^ 1) * kPairBytes<K>, lane);
            if constexpr (!FUSED) fetch(nx, nlo, p + 1);
            load(r[odd ^ 1], p + 3);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                x[g] = scaled(x[g], f[g]);
                if constexpr (LO) lo[g] = scaled(lo[g], f[g]);
            }
            pair_product<K, CODE, G, LO>(acc, buf + odd * kPairBytes<K>, win, x, lo);
            wave_sync();
        };
        if (p0 < p1) {
            if constexpr (!FUSED) fetch(nx, nlo, p0);
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
    // the waves' sums, wave w + 4 added to wave w's first where there are eight
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float s = shift[g] == kNoShift ? 0.0f : ldexpf(1.0f, -shift[g] - 7);
        f4* const mine = sums + (wv & 3) * 512 + lane;
        __syncthreads();
        if (W == 8) {
            if (wv >= 4) {
#pragma unroll
                for (int j = 0; j < 8; ++j) mine[j * 64] = acc[g][j] * s;
            }
            __syncthreads();
        }
        if (wv < 4) {
#pragma unroll
            for (int j = 0; j < 8; ++j) mine[j * 64] = W == 8 ? acc[g][j] * s + mine[j * 64] : acc[g][j] * s;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8 / W; ++i) {
            const f4* p = sums + (i * W + wv) * 64 + lane;
            total[g][i] = (p[0] + p[512]) + (p[1024] + p[1536]);
        }
    }
    __syncthreads();
}

}  // namespace
}  // namespace xtq
