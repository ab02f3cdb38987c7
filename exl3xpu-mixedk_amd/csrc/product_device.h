// product_device.h -- what the matrix products of many rows share: their operands'
// layout, the rows' way into it, the joining of parts.
//
// Operands are laid out beforehand in the order in which the products' waves load
// them ("fragments"): 16 rows by 32 of the summed dimension are 1 KiB, lane 16 q + r
// holding elements 8 q .. 8 q + 7 of row r, the operand of one v_mfma_f32_16x16x32.
#pragma once
#include "epilogue.h"
#include "operators.h"

#pragma clang fp contract(off)

namespace xtq {
namespace {

constexpr int kFragBytes = 1024;

// Where fragment `step` of group `grp` starts, in elements.  Groups come in
// sixteens; scratch is sized for whole ones, and what is not written there
// reaches no result.
__host__ __device__ __forceinline__ size_t frag_at(size_t grp, size_t step, size_t steps) {
    return (((grp >> 4) * steps + step) * 16 + (grp & 15)) * 512;
}

// Bytes of `groups` groups' fragments.
size_t frag_bytes(size_t groups, size_t steps) { return (groups + 15) / 16 * 16 * steps * kFragBytes; }

__device__ __forceinline__ void unpack8(u4 w, int type, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (type == kBf16) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            v[2 * i] = half_bits(w[i] & 0xFFFFu);
            v[2 * i + 1] = half_bits(w[i] >> 16);
        }
    }
}

// Where a weight's fragments lie among another's: half: of groups of 128 columns, its
// half of 256, or -1; step: its first of `steps` of the summed dimension.
struct FragPlace {
    int half, step, steps;
};

// Trellis to fragments of the inner weight.  BWD = 0: fragment (ng, p) holds
// columns 16 ng + r, summed rows 32 p + 8 q + j (operand of x Wi); BWD = 1:
// rows 16 kg + r, summed columns (operand of dz Wi^T).  Element (r, c) of a tile
// is symbol 32 (c % 8) + 8 ((r % 8) / 2) + 4 (c / 8) + 2 (r / 8) + r % 2, its state
// the 16-bit circular window ending with the symbol's K bits.  A workgroup
// (`block`) takes 8 by 4 tiles (along the summed dimension by the other), the trellis
// words staged in LDS, 256 K of them.
template <int K, int CODE, int BWD>
__device__ __forceinline__ void decode_tiles(uint32_t* words, int block, const int16_t* __restrict__ trellis, int tn,
                                             uint16_t* __restrict__ frags, const FragPlace& place) {
    constexpr int TW = 8 * K;                           // words of a tile
    constexpr int NJ = BWD ? 8 : 4;
    const int nj = tn / NJ, bi = block / nj, i0 = bi * (32 / NJ), j0 = (block - bi * nj) * NJ;   // first tile
    for (int t = threadIdx.x; t < 32 * TW; t += 256) {
        const int tile = t / TW, w = t - tile * TW;
        const int i = i0 + tile / NJ, j = j0 + tile % NJ;
        words[t] = *(const u1_a2*)(trellis + ((size_t)i * tn + j) * 16 * K + 2 * w);
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        // tile of this lane's elements: summed-dimension tile 2 p + q / 2
        const int tile = BWD ? wv * NJ + 2 * p + (q >> 1) : (2 * p + (q >> 1)) * NJ + wv;
        const uint32_t* tw = words + tile * TW;
        uint32_t st[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int row = BWD ? r : 8 * (q & 1) + j, col = BWD ? 8 * (q & 1) + j : r;
            const int t = 32 * (col & 7) + 8 * ((row & 7) >> 1) + 4 * (col >> 3) + 2 * (row >> 3) +
                          (row & 1);
            const int e = t * K + K - 1, lo = e >> 5, hi = lo > 0 ? lo - 1 : TW - 1;
            st[j] = __builtin_amdgcn_alignbit(tw[hi], tw[lo], 31 - (e & 31)) & 0xFFFFu;
        }
        u4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = code_pair<CODE>(st[2 * j], st[2 * j + 1]);
        size_t g = BWD ? i0 + wv : j0 + wv;
        if (place.half >= 0) g = (g >> 3) * 16 + 8 * place.half + (g & 7);
        const size_t f = place.step + (BWD ? j0 : i0) / 2 + p;
        *(u4*)(frags + frag_at(g, f, place.steps) + lane * 8) = o;
    }
}

// A wave's 16 rows of one 128-column block to fragments, `step` the block's first:
// block-128 transform, times 2^shift, rounded to fp16.  Lane 16 q + r holds columns
// 32 p + 8 q + j of row r in v[8 p + j], so five of the transform's seven stages are
// between its own registers.  rest: or NULL, the fragments of what the rounding left.
__device__ __forceinline__ void rows_to_frags(float (&v)[32], int sh, int lane, size_t grp, size_t step, size_t steps,
                                              uint16_t* __restrict__ frags, uint16_t* __restrict__ rest) {
#pragma unroll
    for (int b = 1; b < 32; b <<= 1)
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (!(i & b)) {
                const float a = v[i], c = v[i | b];
                v[i] = a + c;
                v[i | b] = a - c;
            }
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        cross_pair<16>(v[i], v[i + 1]);
        cross_pair<32>(v[i], v[i + 1]);
        v[i] = ldexpf(v[i], sh);
        v[i + 1] = ldexpf(v[i + 1], sh);
    }
    uint16_t* const out = frags + lane * 8;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        h8 o;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (_Float16)v[8 * p + i];
        *(h8*)(out + frag_at(grp, step + p, steps)) = o;
        if (rest) {
            h8 l;
#pragma unroll
            for (int i = 0; i < 8; ++i) l[i] = (_Float16)(v[8 * p + i] - (float)o[i]);
            *(h8*)(rest + lane * 8 + frag_at(grp, step + p, steps)) = l;
        }
    }
}

// Sums of a wave's 16 rows by columns, laid out as above, to one row of partial sums.
__device__ __forceinline__ void rows_sum(const float (&v)[32], int lane, float* __restrict__ out) {
    const int q = lane >> 4;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        float t = v[i];
        t += dpp<0xB1>(t);              // lanes 1 0 3 2
        t += dpp<0x4E>(t);              // lanes 2 3 0 1
        t += dpp<0x141>(t);             // mirrored in eights, then in sixteens
        t += dpp<0x140>(t);
        if ((lane & 15) == 0) out[32 * (i >> 3) + 8 * q + (i & 7)] = t;
    }
}

__device__ void column_sums(const ColSum& a, int block, float* part) {
    const int c = block * 64 + (threadIdx.x & 63), wv = threadIdx.x >> 6;
    float t = 0.0f;
    if (c < a.cols)
#pragma unroll 8
        for (int g = wv; g < a.groups; g += 4) t += a.part[(size_t)g * a.cols + c];
    part[threadIdx.x] = t;
    __syncthreads();
    if (wv || c >= a.cols) return;
    t = (part[c & 63] + part[64 + (c & 63)]) + (part[128 + (c & 63)] + part[192 + (c & 63)]);
    void* const out = c < a.first ? a.out : a.more;
    const int at = c < a.first ? c : c - a.first;
    if (!out) return;
    if (c < a.first ? a.f32 : a.more_f32) ((float*)out)[at] = t;
    else ((uint16_t*)out)[at] = (uint16_t)(a.type == kBf16 ? to16<kBf16>(t) : to16<kF16>(t));
}

// A product's workgroup makes 256 columns: two transform blocks.
constexpr int kTileN = 256;

// Workgroups go round robin over the 8 XCDs, each with an L2 of its own: an XCD
// gets a run of tiles that lie side by side, in bands of kBand rows of tiles.
constexpr int kXcds = 8;
constexpr int kBand = 8;

__device__ __forceinline__ int xcd_order(int id, int all) {
    const int x = id % kXcds, each = all / kXcds, more = all % kXcds;
    return x * each + (x < more ? x : more) + id / kXcds;
}

template <bool BF>
__device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a),
                                                                    __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a),
                                                       __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) void lds_void;

// The sum over the splits from `first` to before `last` of a unit (128 columns by 16
// rows), in order, U of them in flight for each register.
template <int U>
__device__ __forceinline__ void sum_splits(f4 (&v)[8], const Gemm& g, int grp, int blk, int lane, int first,
                                           int last) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    const f4* p = (const f4*)g.part + ((size_t)blk * g.gb + grp) * 512 + lane;
    const size_t stride = (size_t)(g.ga / 8) * g.gb * 512;
    for (int s = first; s < last; s += U) {
        f4 t[U][8];
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) t[i][j] = p[(s + i < last ? s + i : s) * stride + j * 64];
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (s + i < last) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += t[i][j];
            }
    }
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

}  // namespace
}  // namespace xtq
