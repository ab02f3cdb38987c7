// linear_kernels.hip -- products of activations with trellis-coded weights
// (linear layer, forward and gradient) and the Gram matrix of activations,
// for many rows.
//
// With B the block-128 transform without its 1/sqrt(128), a weight is
//   W = scale/128 diag(suh) B Wi B diag(svh),
// so a product is x W = scale/128 svh * B((B(x * suh)) Wi): the transforms act
// on the rows of activations and results, and the matrix product reads the
// codebook values Wi themselves, which fp16 holds exactly.
//
// The matrix product's operands are laid out beforehand in the order in which
// its waves load them ("fragments"): 16 rows by 32 of the summed dimension are
// 1 KiB, lane 16 q + r holding elements 8 q .. 8 q + 7 of row r, the operand of
// one v_mfma_f32_16x16x32.  A fragment moves from memory to LDS and from LDS to
// registers as 64 consecutive 16-byte pieces: no bank conflict, no address
// arithmetic.  16 fragments of a step lie side by side (frag_at), the rows or
// columns of a workgroup's tile: it reads two streams of 16 KiB pieces, and not
// 32 of 1 KiB from as many pages.
#include "epilogue.h"
#include "few_device.h"
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

// Input of a product: activations, or (z set) a gradient dy times the
// activation's slope at the saved z.
struct Source {
    const uint16_t* x;
    long long stride;
    const uint16_t* z;          // [rows][cols] or NULL
    int act;
    const uint16_t* colscale;   // fp16 per column
    int type, rows, cols;
};

// Eight consecutive values of a row before its column scales.
__device__ __forceinline__ void load8(const Source& s, size_t row, int col, float* v) {
    unpack8(*(const u4_a2*)(s.x + row * (size_t)s.stride + col), s.type, v);
    if (s.z) {
        float z[8];
        unpack8(*(const u4_a2*)(s.z + row * (size_t)s.cols + col), s.type, z);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= act_slope(z[i], s.act);
    }
}

__device__ __forceinline__ void scale8(const uint16_t* colscale, int col, float* v) {
    float c[8];
    unpack8(*(const u4_a2*)(colscale + col), kF16, c);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= c[i];
}

// Rows to fragments: values times column scales, block-128 transform, times
// 2^shift, rounded to fp16 (the one rounding of the activations: 2^-11
// relative, as fp16 activations have themselves).  A wave takes 16 rows of one
// 128-column block; lane 16 q + r holds columns 32 p + 8 q + j of row r, so five
// of the transform's seven stages are between its own registers.  Rows past the
// end are zeros.  rest: or NULL, the fragments of what the rounding left.
// colsum: sums over the 16 rows of the unscaled values, one row of partial sums
// per 16 rows (for the bias' gradient).  4096 rows of 5120 take 18.8 us, 4.5 TB/s:
// as fast as a copy.  The exponents come before, a workgroup a row beside the
// decoding: a workgroup of this kernel that looks for its rows' largest values
// itself, in one launch with the decoding, has too little company (27 us for the
// decoding, the exponents and 2047 rows apart, 150 together).
__global__ __launch_bounds__(256) void transform_kernel(Source s, const int32_t* __restrict__ shift,
                                                        uint16_t* __restrict__ frags,
                                                        uint16_t* __restrict__ rest,
                                                        float* __restrict__ colsum) {
    const int lane = threadIdx.x & 63, nblk = s.cols / 128;
    const int blk = blockIdx.x * 4 + (threadIdx.x >> 6), grp = blockIdx.y;
    if (blk >= nblk) return;
    const int q = lane >> 4, row = grp * 16 + (lane & 15);
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = 0.0f;
    if (row < s.rows) {
#pragma unroll
        for (int p = 0; p < 4; ++p) load8(s, row, 128 * blk + 32 * p + 8 * q, v + 8 * p);
    }
    if (colsum) {
        float* out = colsum + (size_t)grp * s.cols + 128 * blk;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            float t = v[i];
            t += dpp<0xB1>(t);          // lanes 1 0 3 2
            t += dpp<0x4E>(t);          // lanes 2 3 0 1
            t += dpp<0x141>(t);         // mirrored in eights, then in sixteens
            t += dpp<0x140>(t);
            if ((lane & 15) == 0) out[32 * (i >> 3) + 8 * q + (i & 7)] = t;
        }
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) scale8(s.colscale, 128 * blk + 32 * p + 8 * q, v + 8 * p);
#pragma unroll
    for (int b = 1; b < 32; b <<= 1)
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (!(i & b)) {
                const float a = v[i], c = v[i | b];
                v[i] = a + c;
                v[i | b] = a - c;
            }
    const int sh = row < s.rows ? shift[row] : 0;
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        cross_pair<16>(v[i], v[i + 1]);
        cross_pair<32>(v[i], v[i + 1]);
        v[i] = ldexpf(v[i], sh);
        v[i + 1] = ldexpf(v[i + 1], sh);
    }
    uint16_t* out = frags + lane * 8;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        h8 o;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (_Float16)v[8 * p + i];
        *(h8*)(out + frag_at(grp, 4 * blk + p, 4 * nblk)) = o;
        if (rest) {
            h8 l;
#pragma unroll
            for (int i = 0; i < 8; ++i) l[i] = (_Float16)(v[8 * p + i] - (float)o[i]);
            *(h8*)(rest + lane * 8 + frag_at(grp, 4 * blk + p, 4 * nblk)) = l;
        }
    }
}

// Column sums' last step: out[c] = sum of part[g][c] over the groups, in an
// order that their number fixes: four threads a column take every fourth group.
struct ColSum {
    const float* part;
    int groups, cols, type, f32;
    void* out;
};

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
    if (a.f32) ((float*)a.out)[c] = t;
    else ((uint16_t*)a.out)[c] = (uint16_t)(a.type == kBf16 ? to16<kBf16>(t) : to16<kF16>(t));
}

__global__ __launch_bounds__(256) void column_sums_kernel(ColSum a) {
    __shared__ float part[256];
    column_sums(a, blockIdx.x, part);
}

// Per row, the power of two that brings its transformed values into fp16's
// range: the largest |x * colscale| goes to [2^7, 2^8), the transform's sums of
// 128 stay below 2^15.  rowexp[m]: what the product has to be multiplied with
// (as a power of two), with the two transforms' 1/128.
__device__ void row_exponents(const Source& s, int row, int32_t* __restrict__ shift,
                              int32_t* __restrict__ rowexp) {
    __shared__ float part[4];
    float top = 0.0f;
    for (int c = threadIdx.x * 8; c < s.cols; c += 2048) {
        float v[8];
        load8(s, row, c, v);
        scale8(s.colscale, c, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
    }
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
        const int sh = shift_to(top, 7);
        shift[row] = sh;
        rowexp[row] = -sh - 7;
    }
}

// Trellis to fragments of the inner weight.  BWD = 0: fragment (ng, p) holds
// columns 16 ng + r, summed rows 32 p + 8 q + j (operand of x Wi); BWD = 1:
// rows 16 kg + r, summed columns (operand of dz Wi^T).  Element (r, c) of a tile
// is symbol 32 (c % 8) + 8 ((r % 8) / 2) + 4 (c / 8) + 2 (r / 8) + r % 2, its state
// the 16-bit circular window ending with the symbol's K bits.  A workgroup
// takes 8 by 4 tiles (along the summed dimension by the other), the trellis
// words staged in LDS.  Memory bounds it: 5120 by 17408 at K = 4 reads 45 MB and
// writes 178 in 50 us, 4.5 TB/s (a copy moves 4.97).  The workgroups past `decoders` find the exponents of the
// source's rows, which nothing here waits for.
template <int K, int CODE, int BWD>
__global__ __launch_bounds__(256) void prepare_kernel(const int16_t* __restrict__ trellis, int tk, int tn,
                                                      uint16_t* __restrict__ frags, int decoders, Source src,
                                                      int32_t* __restrict__ shift,
                                                      int32_t* __restrict__ rowexp) {
    if ((int)blockIdx.x >= decoders) return row_exponents(src, blockIdx.x - decoders, shift, rowexp);
    constexpr int TW = 8 * K;                           // words of a tile
    __shared__ uint32_t words[32 * TW];
    constexpr int NJ = BWD ? 8 : 4;
    const int nj = tn / NJ, bi = blockIdx.x / nj, i0 = bi * (32 / NJ), j0 = (blockIdx.x - bi * nj) * NJ;   // first tile
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
        const size_t g = BWD ? i0 + wv : j0 + wv;
        const size_t np = (BWD ? tn : tk) / 2, f = (BWD ? j0 : i0) / 2 + p;
        *(u4*)(frags + frag_at(g, f, np) + lane * 8) = o;
    }
}

// -------------------------------------------------------------------- matrix
// product of fragments: columns (fragments A) by rows (fragments B).  A
// workgroup's tile is 256 columns by 32 NB rows, 4 waves of 128 columns (a whole
// transform block, so the epilogue's transform stays in registers) by 16 NB
// rows.  The summed dimension goes by in steps of 32; while the matrix cores
// work on one step, the next two move from memory into the other two of three
// LDS buffers.  Two workgroups share a compute unit, so one's epilogue and waits
// overlap with the other's products.  (One workgroup of 8 waves and 256 by 256,
// its fragments fetched a step ahead: the epilogue, 17 us a tile, stood alone.)
// 4096 rows by 5120 by 17408 with the epilogue: 666 us, 1.10 PFLOP/s; the library's
// product of the same size alone takes 594, 8192 cubed runs at 1.29.
constexpr int kTileN = 256;

// Workgroups go round robin over the 8 XCDs, each with an L2 of its own: an XCD
// gets a run of tiles that lie side by side, in bands of kBand rows of tiles.
constexpr int kXcds = 8;
constexpr int kBand = 8;

__device__ __forceinline__ int xcd_order(int id, int all) {
    const int x = id % kXcds, each = all / kXcds, more = all % kXcds;
    return x * each + (x < more ? x : more) + id / kXcds;
}

enum GemmOut { kOutEpilogue, kOutPartial, kOutGram };

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

template <bool BF>
__device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a),
                                                                    __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a),
                                                       __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

// out = prev + sums of 32 rows by 128 columns of the Gram, at and below the
// diagonal and mirrored.  They go through t, 32 lines in LDS that only this wave
// uses, and come out as whole lines of memory: 512 bytes of a row, 128 of a
// mirrored one.  (From the registers, 64 bytes of a row at a time and in a launch
// of its own, 8192 rows of 5120 channels took 282 us in all, not 259.)
constexpr int kGramLine = 132;

__device__ __forceinline__ void finish_gram(const f4 (&v)[2][8], float* t, const Gemm& g, int grp, int blk,
                                            int lane) {
    const int row0 = grp * 16, col0 = blk * 128, r = lane & 15, q = lane >> 4;
    const size_t dim = g.dim;
    const bool below = col0 + 127 < row0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j) *(f4*)(t + (16 * h + r) * kGramLine + 16 * j + 4 * q) = v[h][j];
    wave_sync();
    auto put = [&](const f4* s, const size_t* at, auto keep) {
        f4 p[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            p[n] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
            if (g.prev && below) p[n] = *(const f4_a4*)(g.prev + at[n]);
            else if (g.prev)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (keep(n, i)) p[n][i] = g.prev[at[n] + i];
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            if (below) *(f4_a4*)(g.out + at[n]) = p[n] + s[n];
            else
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (keep(n, i)) g.out[at[n] + i] = p[n][i] + s[n][i];
        }
    };
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
        f4 s[8];
        size_t at[8];
        const int row = 16 * half + (lane >> 5), col = 4 * (lane & 31);     // row + 2 n
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            s[n] = *(const f4*)(t + (row + 2 * n) * kGramLine + col);
            at[n] = (size_t)(row0 + row + 2 * n) * dim + col0 + col;
        }
        put(s, at, [&](int n, int i) { return col0 + col + i <= row0 + row + 2 * n; });
    }
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
        f4 s[8];
        size_t at[8];
        const int row = 4 * (lane & 7), col = 64 * half + (lane >> 3);      // col + 8 n
#pragma unroll
        for (int n = 0; n < 8; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = t[(row + i) * kGramLine + col + 8 * n];
            at[n] = (size_t)(col0 + col + 8 * n) * dim + row0 + row;
        }
        put(s, at, [&](int n, int i) { return col0 + col + 8 * n < row0 + row + i; });
    }
    wave_sync();
}

template <int T, int OUT, bool BF, int NB, int TERMS>
__global__ __launch_bounds__(256, 2) void gemm_kernel(Gemm g, Epilogue ep, ColSum sums) {
    // of a step: the workgroup's fragments, a wave's to move
    constexpr int kFrags = 16 + 2 * NB * TERMS, kOwn = 4 + NB / 2 * TERMS;
    // (One LDS object: beside another, the compiler takes every read of this one
    // for a possible read of what a load to LDS still has to write, and waits.)
    __shared__ __align__(1024) uint8_t lds[3][kFrags * kFragBytes];
    // workgroups past the tiles: column sums that the launch before left parts of
    if ((int)blockIdx.x >= g.tiles) {
        if (blockIdx.y == 0) column_sums(sums, blockIdx.x - g.tiles, (float*)lds[0]);
        return;
    }
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wv & 1, wm = wv >> 1;
    const int tile = xcd_order(blockIdx.x, g.tiles);
    int tn, tm;
    if constexpr (OUT == kOutGram) {
        // tiles that reach the diagonal or lie below: columns tn, rows tm >= R tn
        constexpr int R = kTileN / (32 * NB);
        const int mt = (g.gb + 2 * NB - 1) / (2 * NB);
        int at = tile;
        for (tn = 0; at >= mt - R * tn; ++tn) at -= mt - R * tn;
        tm = R * tn + at;
    } else {                            // bands of kBand tiles of rows
        const int nt = (g.ga + 15) / 16, mt = (g.gb + 2 * NB - 1) / (2 * NB), band = tile / (nt * kBand);
        const int high = mt - band * kBand < kBand ? mt - band * kBand : kBand, in = tile - band * nt * kBand;
        tn = in / high;
        tm = band * kBand + in - tn * high;
    }
    const int split = blockIdx.y;
    const int s0 = (int)((long long)g.steps * split / g.splits);
    const int s1 = (int)((long long)g.steps * (split + 1) / g.splits);

    // this wave's fragments of a step: a quarter of A's 16 and of B's 2 NB
    const uint16_t* fa = g.A + (size_t)tn * g.steps * 8192 + wv * 2048 + lane * 8;
    const int gb0 = tm * 2 * NB;        // first group of rows
    const size_t at_b = ((size_t)(gb0 >> 4) * g.steps * 16 + (gb0 & 15) + wv * (NB / 2)) * 512 + lane * 8;
    const uint16_t *fb = g.B + at_b, *fb2 = TERMS == 2 ? g.B2 + at_b : nullptr;
    int to = 0;                         // buffer of the next step to load
    auto load = [&](int s) {
        uint8_t* l = lds[to];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            __builtin_amdgcn_global_load_lds((global_void*)(fa + (size_t)s * 8192 + i * 512),
                                             (lds_void*)(l + (wv * 4 + i) * kFragBytes), 16, 0, 0);
#pragma unroll
        for (int i = 0; i < NB / 2; ++i)
            __builtin_amdgcn_global_load_lds((global_void*)(fb + (size_t)s * 8192 + i * 512),
                                             (lds_void*)(l + (16 + wv * (NB / 2) + i) * kFragBytes), 16, 0, 0);
        if constexpr (TERMS == 2) {
#pragma unroll
            for (int i = 0; i < NB / 2; ++i)
                __builtin_amdgcn_global_load_lds((global_void*)(fb2 + (size_t)s * 8192 + i * 512),
                                                 (lds_void*)(l + (16 + 2 * NB + wv * (NB / 2) + i) * kFragBytes), 16, 0, 0);
        }
        to = to == 2 ? 0 : to + 1;
    };
    // All waves' pieces of the next step are in LDS, and all waves have read this
    // one (their reads were waited for before they came here).
    auto meet_up = [&](bool more) {
        if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kOwn) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    f4 acc[8][NB];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[j][b] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    if (s0 < s1) {
        load(s0);
        if (s0 + 1 < s1) load(s0 + 1);
        meet_up(s0 + 1 < s1);
        int from = 0;
        for (int s = s0; s < s1; ++s) {
            if (s + 2 < s1) load(s + 2);
            u4 a[8], b[TERMS][NB];
            const uint8_t* l = lds[from] + lane * 16;
#pragma unroll
            for (int t = 0; t < TERMS; ++t)
#pragma unroll
                for (int i = 0; i < NB; ++i) b[t][i] = *(const u4*)(l + (16 + 2 * NB * t + wm * NB + i) * kFragBytes);
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] = *(const u4*)(l + (wn * 8 + j) * kFragBytes);
            __builtin_amdgcn_sched_barrier(0);          // all reads under way before the first product
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int t = 0; t < TERMS; ++t)
#pragma unroll
                    for (int i = 0; i < NB; ++i) acc[j][i] = mfma<BF>(a[j], b[t][i], acc[j][i]);
            __builtin_amdgcn_sched_barrier(0);          // none after the others have met
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            meet_up(s + 2 < s1);
            from = from == 2 ? 0 : from + 1;
        }
    }
    const int blk = tn * 2 + wn;
    if (blk * 8 >= g.ga) return;
    if constexpr (OUT == kOutGram) {
        if (g.splits == 1) {
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
                const int grp = gb0 + wm * NB + b;
                if (grp >= g.gb || blk * 128 > grp * 16 + 31) continue;     // (above the diagonal)
                f4 v[2][8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[0][j] = acc[j][b];
                    v[1][j] = acc[j][b + 1];
                }
                finish_gram(v, (float*)lds + wv * 32 * kGramLine, g, grp, blk, lane);
            }
            return;
        }
    }
    Columns<4> cols[8];
    if constexpr (OUT == kOutEpilogue) unit_columns<T>(cols, ep, blk, lane);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int grp = gb0 + wm * NB + b;
        if (grp >= g.gb) continue;
        __builtin_amdgcn_sched_barrier(0);
        f4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = acc[j][b];
        if constexpr (OUT == kOutEpilogue) {
            finish_unit<T>(v, cols, ep, grp, blk, lane);
        } else {
            f4* o = (f4*)g.part + (((size_t)split * (g.ga / 8) + blk) * g.gb + grp) * 512 + lane;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j * 64] = v[j];
        }
    }
}

// The sum over the splits of a unit (128 columns by 16 rows), in order, U of
// them in flight for each register.
template <int U>
__device__ __forceinline__ void sum_splits(f4 (&v)[8], const Gemm& g, int grp, int blk, int lane) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    const f4* p = (const f4*)g.part + ((size_t)blk * g.gb + grp) * 512 + lane;
    const size_t stride = (size_t)(g.ga / 8) * g.gb * 512;
    for (int s = 0; s < g.splits; s += U) {
        f4 t[U][8];
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) t[i][j] = p[(s + i < g.splits ? s + i : s) * stride + j * 64];
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (s + i < g.splits) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += t[i][j];
            }
    }
}

// Joins the splits' partial products and finishes them, a workgroup of one wave
// one unit: units are few, so each may land where there is room (four waves a
// workgroup: 15.9 us, not 14.6, for 333 rows by 6144 columns in three parts, whose
// 25 MB take 5 us to copy; the rest is the latency of loads, transform and
// stores one after the other).
template <int T>
__global__ __launch_bounds__(64) void join_kernel(Gemm g, Epilogue ep) {
    const int lane = threadIdx.x, grp = blockIdx.x, blk = blockIdx.y;
    f4 v[8];
    sum_splits<4>(v, g, grp, blk, lane);
    Columns<4> cols[8];
    unit_columns<T>(cols, ep, blk, lane);
    finish_unit<T>(v, cols, ep, grp, blk, lane);
}

// The same for the Gram, a wave two units.
__global__ __launch_bounds__(256) void join_gram_kernel(Gemm g) {
    __shared__ __align__(16) float t[4][32 * kGramLine];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, grp = (blockIdx.x * 4 + wv) * 2, blk = blockIdx.y;
    if (grp >= g.gb || blk * 128 > grp * 16 + 31) return;       // (above the diagonal)
    f4 v[2][8];
    sum_splits<2>(v[0], g, grp, blk, lane);
    sum_splits<2>(v[1], g, grp + 1, blk, lane);
    finish_gram(v, t[wv], g, grp, blk, lane);
}

// ---------------------------------------------------------------------- Gram
// Rows of activations to fragments of their transpose: 16 channels by 32 rows.
// Rows that are not valid, or past the end, are zeros whatever they hold.  A
// workgroup takes 32 rows by 128 channels.  Memory bounds it: 8192 by 5120 moves
// its 168 MB in 29 us, 5.8 TB/s.
__global__ __launch_bounds__(256) void transpose_kernel(const uint16_t* __restrict__ x,
                                                        long long stride, int rows, int steps,
                                                        const uint8_t* __restrict__ valid,
                                                        uint16_t* __restrict__ frags) {
    __shared__ uint16_t t[32][136];
    const int p = blockIdx.x, c0 = blockIdx.y * 128;
    for (int i = threadIdx.x; i < 512; i += 256) {
        const int r = i >> 4, c = (i & 15) * 8, row = p * 32 + r;
        u4 w = {0u, 0u, 0u, 0u};
        if (row < rows && (!valid || valid[row])) w = *(const u4_a2*)(x + (size_t)row * stride + c0 + c);
        *(u4*)&t[r][c] = w;
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, q = lane >> 4;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int c = (wv * 2 + g) * 16 + (lane & 15);
        u4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = t[8 * q + 2 * i][c] | (uint32_t)t[8 * q + 2 * i + 1][c] << 16;
        *(u4*)(frags + frag_at(c0 / 16 + wv * 2 + g, p, steps) + lane * 8) = o;
    }
}

// The Gram of few rows in one launch.  A workgroup makes 64 by 64 of it (at or
// below the diagonal) from x as it lies: lane 16 q + r loads four channels,
// 4 r .. + 3, of the eight rows 8 q .. 8 q + 7 of a 32-row step, and what it then
// holds of channel 4 r + j is its part of an MFMA operand whose index r stands
// for that channel: the transpose is 16 byte permutes between a lane's own
// registers.  Its W waves take a step each in turn and meet in LDS, in an order
// that the number of rows fixes.  Eight waves, 64 KiB of LDS and 125 registers
// let two workgroups share a compute unit: one loads while the other multiplies
// (with a wave's next step fetched ahead, 160 registers and one workgroup, 5120
// channels took 129 us at 1021 rows and not 92, and 65 at one row, not the 40
// that its 210 MB take to copy).  Where there is a compute unit for every tile,
// sixteen waves halve the loads that wait for each other (1024 channels by 1021
// rows that no cache holds: under 10.5 us, of eight waves 18).
constexpr int kGramTile = 64;

template <bool BF, int W>
__global__ __launch_bounds__(64 * W, 4) void gram_few_kernel(const uint16_t* __restrict__ x, long long stride,
                                                              int rows, int dim,
                                                              const uint8_t* __restrict__ valid,
                                                              const float* prev, float* out) {
    __shared__ __align__(16) f4 lds[W / 2][16][64];
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tm = 0, tn = xcd_order(blockIdx.x, gridDim.x);
    // rows of tiles of 1, 2, 3 .. tiles
    tm = (int)((sqrtf(8.0f * tn + 1.0f) - 1.0f) * 0.5f);
    while (tm * (tm + 1) / 2 > tn) --tm;
    while ((tm + 1) * (tm + 2) / 2 <= tn) ++tm;
    tn -= tm * (tm + 1) / 2;
    const uint16_t *xa = x + tn * kGramTile + 4 * r, *xb = x + tm * kGramTile + 4 * r;
    const int steps = (int)(((long long)rows + 31) / 32);
    u2 a[8], b[8];
    auto load = [&](int s) {
        u2 mask = {~0u, ~0u};           // a byte for each of the lane's rows
        if (valid) {
            const int row = s * 32 + 8 * q;
            if (row + 8 <= rows) mask = *(const u2_a1*)(valid + row);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (row + e >= rows || !valid[row + e]) mask[e >> 2] &= ~(0xFFu << (8 * (e & 3)));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int row = s * 32 + 8 * q + e, at = row < rows ? row : rows - 1;
            const bool keep = row < rows && (mask[e >> 2] >> (8 * (e & 3)) & 0xFFu);
            a[e] = *(const u2_a2*)(xa + at * (size_t)stride);
            b[e] = *(const u2_a2*)(xb + at * (size_t)stride);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[e][i] = keep ? a[e][i] : 0u;
                b[e][i] = keep ? b[e][i] : 0u;
            }
        }
    };
    f4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i >> 2][i & 3] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = wv; s < steps; s += W) {
        load(s);
        u4 fa[4], fb[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
                fa[j][i] = __builtin_amdgcn_perm(a[2 * i + 1][j >> 1], a[2 * i][j >> 1], sel);
                fb[j][i] = __builtin_amdgcn_perm(b[2 * i + 1][j >> 1], b[2 * i][j >> 1], sel);
            }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] = mfma<BF>(fa[j], fb[i], acc[j][i]);
    }
    // the upper waves to the lower, these to all
    if (wv >= W / 2)
#pragma unroll
        for (int i = 0; i < 16; ++i) lds[wv - W / 2][i][lane] = acc[i >> 2][i & 3];
    __syncthreads();
    if (wv < W / 2)
#pragma unroll
        for (int i = 0; i < 16; ++i) lds[wv][i][lane] = acc[i >> 2][i & 3] + lds[wv][i][lane];
    __syncthreads();
    constexpr int N = 16 / W;
    f4 sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        sum[i] = lds[0][N * wv + i][lane];
#pragma unroll
        for (int w = 1; w < W / 2; ++w) sum[i] += lds[w][N * wv + i][lane];
    }
    __syncthreads();
    // operand indices 4 q + i and r of products (j, i2) are channels
    // 16 q + 4 i + j and 4 r + i2
    constexpr int kRow = kGramTile + 4;
    float* const t = (float*)lds;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = N * wv + n, col = 16 * q + 4 * i + (at >> 2), row = 4 * r + (at & 3);
            if (tm != tn || col <= row) t[row * kRow + col] = sum[n][i];
            if (tm == tn && col < row) t[col * kRow + row] = sum[n][i];
        }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int line = 4 * (N * wv + n) + q;
        const size_t at = (size_t)(tm * kGramTile + line) * dim + tn * kGramTile + 4 * r;
        const f4 v = *(const f4*)(t + line * kRow + 4 * r);
        *(f4_a4*)(out + at) = prev ? *(const f4_a4*)(prev + at) + v : v;
        if (tm == tn) continue;
        const size_t to = (size_t)(tn * kGramTile + line) * dim + tm * kGramTile + 4 * r;
        f4 m;
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = t[(4 * r + i) * kRow + line];
        *(f4_a4*)(out + to) = prev ? *(const f4_a4*)(prev + to) + m : m;
    }
}

struct Prepare {
    uint16_t* frags;
    int decoders;
    Source src;
    int32_t *shift, *rowexp;
};

template <int K, int CODE>
void prepare_kc(const Weight& w, int bwd, const Prepare& p, hipStream_t s) {
    const int tk = w.k / 16, tn = w.n / 16;
    const dim3 grid(p.decoders + p.src.rows);
    if (bwd) hipLaunchKernelGGL((prepare_kernel<K, CODE, 1>), grid, dim3(256), 0, s, w.trellis, tk, tn, p.frags,
                                p.decoders, p.src, p.shift, p.rowexp);
    else hipLaunchKernelGGL((prepare_kernel<K, CODE, 0>), grid, dim3(256), 0, s, w.trellis, tk, tn, p.frags,
                            p.decoders, p.src, p.shift, p.rowexp);
}

template <int K>
void prepare_k(const Weight& w, int bwd, const Prepare& p, hipStream_t s) {
    if (w.code == kCodeMul1) prepare_kc<K, kCodeMul1>(w, bwd, p, s);
    else if (w.code == kCodeMcg) prepare_kc<K, kCodeMcg>(w, bwd, p, s);
    else prepare_kc<K, kCode3Inst>(w, bwd, p, s);
}

void prepare(const Weight& w, int bwd, const Prepare& p, hipStream_t s) {
    switch (w.K) {
        case 2: return prepare_k<2>(w, bwd, p, s);
        case 3: return prepare_k<3>(w, bwd, p, s);
        case 4: return prepare_k<4>(w, bwd, p, s);
        case 5: return prepare_k<5>(w, bwd, p, s);
        case 6: return prepare_k<6>(w, bwd, p, s);
        default: return prepare_k<7>(w, bwd, p, s);
    }
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// How a product of `steps` steps is cut: nb groups of 16 rows to a wave's tile,
// splits of the summed dimension.  The choice is the shortest estimate, from what
// the kernels measured: a workgroup's step takes 0.62 us (nb 4) or 0.38 (nb 2)
// alone on a compute unit, two at once 0.72 and 0.46, and where a unit has more to
// do than those, every two 0.84 and 0.64; parts are written and read at 4 TB/s.  (us of
// whole calls in replayed graphs with nb 4, nb 2: 5120 by 5120, 333 rows 67 : 56, 1000
// rows 92 : 107, 2047 rows 150 : 182; 5120 by 17408, 96 rows 101 : 84, 600 rows 176 :
// 205.)
struct Tiling {
    int nb, tiles, splits;
};

Tiling gemm_tiling(int rows, int n, int steps, bool two) {
    Tiling best{};
    double least = 0.0;
    for (int nb = two ? 2 : 4; nb >= 2; nb -= 2) {      // (two terms: the LDS of two workgroups)
        const int tiles = (n + kTileN - 1) / kTileN * ((rows + 32 * nb - 1) / (32 * nb));
        const double alone = nb == 4 ? 0.62 : 0.38, pair = nb == 4 ? 0.72 : 0.46, more = nb == 4 ? 0.42 : 0.32;
        for (int s = 1; s == 1 || (s <= steps / 8 && (s - 1) * tiles < 2 * kCUs); ++s) {
            const int each = (int)(((long long)tiles * s + kCUs - 1) / kCUs);
            const double step = each == 1 ? alone : each == 2 ? pair : more * (each % 2 ? each + 0.4 : each);
            const double us = step * (two ? 2 : 1) * ((steps + s - 1) / s) +
                              (s > 1 ? 3.0 + 2e-6 * s * rows * n : 0.0);
            if (!best.nb || us < least) {
                least = us;
                best = Tiling{nb, tiles, s};
            }
        }
    }
    return best;
}

struct ManyPlan {
    int groups, nb, tiles, splits;
    size_t shift, rowexp, xf, x2, wf, part, colsum, total;
};

// Scratch of a product of `rows` rows: summed dimension k, columns n.
ManyPlan many_plan(int rows, int k, int n, bool colsum, bool two) {
    ManyPlan p;
    p.groups = (rows + 15) / 16;
    const Tiling t = gemm_tiling(rows, n, k / 32, two);
    p.nb = t.nb;
    p.tiles = t.tiles;
    p.splits = t.splits;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t a = at; at += align256(bytes); return a; };
    p.shift = take((size_t)p.groups * 64);
    p.rowexp = take((size_t)p.groups * 64);
    p.xf = take(frag_bytes(p.groups, k / 32));
    p.x2 = take(two ? frag_bytes(p.groups, k / 32) : 0);
    p.wf = take(frag_bytes(n / 16, k / 32));
    p.part = take(p.splits > 1 ? (size_t)p.splits * p.groups * 64 * n : 0);
    p.colsum = take(colsum ? (size_t)p.groups * k * 4 : 0);
    p.total = at;
    return p;
}

// The product of a source's rows with a weight (bwd: its transpose).
template <int T>
hipError_t many(const Weight& w, int bwd, const Source& src, Epilogue ep, void* dbias, int dbias_f32,
                bool two, void* ws, hipStream_t s) {
    const int k = src.cols, n = ep.cols, rows = src.rows;
    const ManyPlan p = many_plan(rows, k, n, dbias != nullptr, two);
    uint8_t* base = (uint8_t*)ws;
    int32_t *shift = (int32_t*)(base + p.shift), *rowexp = (int32_t*)(base + p.rowexp);
    uint16_t *xf = (uint16_t*)(base + p.xf), *x2 = two ? (uint16_t*)(base + p.x2) : nullptr, *wf = (uint16_t*)(base + p.wf);
    float* colsum = dbias ? (float*)(base + p.colsum) : nullptr;
    const int decoders = ep.y ? (w.k / 16) * (w.n / 16) / 32 : 0;
    prepare(w, bwd, Prepare{wf, decoders, src, shift, rowexp}, s);
    hipLaunchKernelGGL(transform_kernel, dim3((k / 128 + 3) / 4, p.groups), dim3(256), 0, s, src,
                       (const int32_t*)shift, xf, x2, colsum);
    const ColSum sums{colsum, p.groups, k, T, dbias_f32, dbias};
    const int adders = dbias ? (k + 63) / 64 : 0;
    if (!ep.y) {
        hipLaunchKernelGGL(column_sums_kernel, dim3(adders), dim3(256), 0, s, sums);
        return hipGetLastError();
    }
    ep.rowexp = rowexp;
    const Gemm g{wf, xf, x2, n / 16, p.groups, k / 32, p.tiles, p.splits, (float*)(base + p.part), nullptr, nullptr, 0};
    const dim3 grid(p.tiles + adders, p.splits), block(256);
    if (p.splits == 1) {
        if (two) hipLaunchKernelGGL((gemm_kernel<T, kOutEpilogue, false, 2, 2>), grid, block, 0, s, g, ep, sums);
        else if (p.nb == 4) hipLaunchKernelGGL((gemm_kernel<T, kOutEpilogue, false, 4, 1>), grid, block, 0, s, g, ep, sums);
        else hipLaunchKernelGGL((gemm_kernel<T, kOutEpilogue, false, 2, 1>), grid, block, 0, s, g, ep, sums);
    } else {
        if (two) hipLaunchKernelGGL((gemm_kernel<T, kOutPartial, false, 2, 2>), grid, block, 0, s, g, ep, sums);
        else if (p.nb == 4) hipLaunchKernelGGL((gemm_kernel<T, kOutPartial, false, 4, 1>), grid, block, 0, s, g, ep, sums);
        else hipLaunchKernelGGL((gemm_kernel<T, kOutPartial, false, 2, 1>), grid, block, 0, s, g, ep, sums);
        hipLaunchKernelGGL((join_kernel<T>), dim3(p.groups, n / 128), dim3(64), 0, s, g, ep);
    }
    return hipGetLastError();
}

// Rows to fragments for the products of few rows, a wave for one row's
// 128-column block.  Rows past the end are zeros.  rest (LO): the second terms.
// Latency alone: 2.3 us for 48 rows of 5120.
template <bool LO>
__global__ __launch_bounds__(256) void transform_few_kernel(const uint16_t* __restrict__ x, long long stride,
                                                            int type, int rows, int k,
                                                            const uint16_t* __restrict__ suh,
                                                            u4* __restrict__ frag, u4* __restrict__ rest,
                                                            int32_t* __restrict__ shift) {
    const int lane = threadIdx.x & 63, nk = k / 128;
    const int kb = blockIdx.x * 4 + (threadIdx.x >> 6), row = blockIdx.y;
    if (kb >= nk) return;
    float a = 0.0f, b = 0.0f, sa, sb;
    if (row < rows) unpack_two(load_two(x + (size_t)row * stride + 128 * kb, lane), type, a, b);
    unpack_two(load_two(suh + 128 * kb, lane), kF16, sa, sb);
    const size_t at = (size_t)(row >> 4) * nk + kb;
    const int sh = row_to_frags<LO>(a * sa, b * sb, lane, row & 15, (uint32_t*)(frag + at * 256),
                                    LO ? (uint32_t*)(rest + at * 256) : nullptr);
    if (lane == 0) shift[at * 16 + (row & 15)] = sh;
}

// Workgroups per 128 columns of a product of few rows: two for each compute
// unit, each wave with a 32-row step at least, and no more than balances what
// they share, k / 32 steps, with what the last of them adds alone, their parts of
// every row, 0.01 us each (5120 by 1024: 17 rows 20.0 us, 27.2 with 40 parts; 64
// rows 27.3, 47.7).  (One workgroup for each: one row of 5120 by 17408 33.2 us, not
// 27.5; three: 64 rows of 17408 by 5120 61.5, not 51.7.)  Above 16 rows one is
// better where that fills them and no wave has more than 16 steps: the joins weigh
// more (4096 by 4096, 17 rows 17.4 us, 20.2 with two; 48 rows 24.6, 29.2; 17408 by
// 5120, 23 steps, 36.4, 34.4).
int few_splits(int rows, int k, int n, int waves) {
    const int most = k / 32 / waves;
    int s = 2 * kCUs / (n / 128);
    if (s > most) s = most;
    while (s > 1 && (long long)s * s * waves * rows > 4 * k) --s;
    const int one = kCUs / (n / 128);
    if (rows > 16 && s > one && 5 * one * (n / 128) > 4 * kCUs && k / 32 <= 16 * waves * one) s = one;
    return s < 1 ? 1 : s;
}

// (5120 by 5120, one launch or two against decoding apart: 17 rows 20 : 42 us, 64
// rows 31 : 44; 5120 by 1024 20 : 30 and 27 : 32; with two terms 24 : 43, 35 : 43, 23 :
// 34 and, at K = 7, whose 64 rows of two terms spill, 38 : 37.)
bool takes_few(int rows, int n) { return rows <= kFewRows && n / 128 <= XTQ_OP_COUNTERS; }

// Blocks of rows that a workgroup transforms itself at most, two a wave (us where
// the product's workgroups transform, and in a launch before it: 5120 by 5120, one
// row 14.0 : 15.4, four 15.4 : 16.0, six 17.6 : 16.5, sixteen 21.4 : 17.2; 5120 by
// 17408, one row 27.6 : 27.2, sixteen 45.2 : 29.5; with two terms 5120 by 5120, one
// row 15.3 : 16.8, six 17.7 : 17.8, sixteen 22.0 : 19.2; 5120 by 17408 29.4 : 28.4,
// 48.3 : 30.5.  These, few_splits' and takes_few's with two terms are graphs
// replayed, which clear the counters before each product; the kernel of one row of
// 5120 by 5120 alone takes 12.6).
constexpr int kFewItems = 16;

constexpr int few_groups(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

// The kernels read every place of their groups, so there is one for each row, in a
// number that has a kernel; one group where the kernel transforms the rows.
constexpr bool groups_fit() {
    for (int r = 1; r <= kFewRows; ++r) {
        const int g = few_groups(r);
        if (16 * g < r || (g != 1 && g != 2 && g != 4) || (r <= kFusedRows && g != 1)) return false;
    }
    return true;
}
static_assert(groups_fit(), "groups of fragments that the kernels of few rows read");

struct FewPlan {
    int splits, groups;
    bool apart;
    size_t part, frag, rest, shift, total;
};

FewPlan few_plan(int rows, int k, int n, bool two) {
    FewPlan p;
    p.groups = few_groups(rows);
    p.splits = few_splits(rows, k, n, few_waves(p.groups));
    p.apart = rows > kFusedRows || rows * (k / 128) > kFewItems * p.splits;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t a = at; at += align256(bytes); return a; };
    p.part = take(p.splits > 1 ? (size_t)p.splits * n * rows * 4 : 0);
    p.frag = take(p.apart ? (size_t)p.groups * k * 32 : 0);
    p.rest = take(p.apart && two ? (size_t)p.groups * k * 32 : 0);
    p.shift = take(p.apart ? (size_t)p.groups * k / 2 : 0);
    p.total = at;
    return p;
}

}  // namespace

size_t linear_ws_bytes(int rows, int k, int n, bool backward, bool two) {
    if (backward) return many_plan(rows, n, k, true, two).total;
    return takes_few(rows, n) ? few_plan(rows, k, n, two).total : many_plan(rows, k, n, false, two).total;
}

hipError_t launch_linear(const Weight& w, int type, const void* x, long long x_stride, int rows,
                         const Epilogue& ep, bool two, void* ws, uint32_t* counters, hipStream_t s) {
    if (takes_few(rows, w.n)) {
        static decltype(&launch_few_k2) const few[] = {launch_few_k2, launch_few_k3, launch_few_k4,
                                                       launch_few_k5, launch_few_k6, launch_few_k7},
                                              few2[] = {launch_few2_k2, launch_few2_k3, launch_few2_k4,
                                                        launch_few2_k5, launch_few2_k6, launch_few2_k7};
        const FewPlan p = few_plan(rows, w.k, w.n, two);
        uint8_t* base = (uint8_t*)ws;
        FewArgs a{type, two, (const uint16_t*)x, x_stride, nullptr, nullptr, nullptr, p.groups, p.splits,
                  w.k / 32 / p.splits, w.k / 32 % p.splits, 65536u / rows + 1, (float*)(base + p.part), counters};
        if (!p.apart) return few[w.K - 2](w, a, ep, s);
        u4 *frag = (u4*)(base + p.frag), *rest = two ? (u4*)(base + p.rest) : nullptr;
        int32_t* shift = (int32_t*)(base + p.shift);
        hipLaunchKernelGGL(two ? transform_few_kernel<true> : transform_few_kernel<false>,
                           dim3((w.k / 128 + 3) / 4, 16 * p.groups), dim3(256), 0, s, a.x, x_stride, type, rows, w.k,
                           w.suh, frag, rest, shift);
        a.frag = frag;
        a.frag_lo = rest;
        a.shift = shift;
        return (two ? few2 : few)[w.K - 2](w, a, ep, s);
    }
    const Source src{(const uint16_t*)x, x_stride, nullptr, 0, w.suh, type, rows, w.k};
    return type == kBf16 ? many<kBf16>(w, 0, src, ep, nullptr, 0, two, ws, s)
                         : many<kF16>(w, 0, src, ep, nullptr, 0, two, ws, s);
}

hipError_t launch_linear_bwd(const Weight& w, int type, const void* dy, long long dy_stride,
                             const void* z, int act, int rows, void* dx, long long dx_stride,
                             void* dbias, int dbias_f32, bool two, void* ws, uint32_t* counters,
                             hipStream_t s) {
    (void)counters;
    const Source src{(const uint16_t*)dy, dy_stride, act == kActNone ? nullptr : (const uint16_t*)z, act,
                     w.svh, type, rows, w.n};
    Epilogue ep{};
    ep.colscale = w.suh;
    ep.scale = w.scale;
    ep.y = dx;
    ep.y_stride = dx_stride;
    ep.rows = rows;
    ep.cols = w.k;
    return type == kBf16 ? many<kBf16>(w, 1, src, ep, dbias, dbias_f32, two, ws, s)
                         : many<kF16>(w, 1, src, ep, dbias, dbias_f32, two, ws, s);
}

namespace {

struct GramPlan {
    int steps, tiles, splits;
    size_t xf, part, total;
};

// Whether the Gram comes in one launch, from x itself.  Its time grows with every
// tile's 256 bytes a row, the transpose's and the product's with a large constant
// (us, both with prev, one launch against several: 1024 channels 10 : 41 at 1021
// rows, 46 : 67 at 8192; 2048 57 : 65 at 4096, 103 : 85 at 8192; 5120 51 : 76 at
// 256, 92 : 91 at 1021, 152 : 112 at 2048; 17408 594 : 541 at one row).
bool takes_gram_few(int rows, int k) {
    return rows <= 8192 && k <= 8192 && (long long)rows * k * k <= 24LL << 30;
}

// Parts of the summed dimension, each of 8 steps at least, so that the tiles fill
// the compute units' two places.
int gemm_splits(int tiles, int steps) {
    const int most = steps / 8;
    int s = tiles >= 2 * kCUs ? 1 : 2 * kCUs / tiles;
    if (s > most) s = most;
    return s < 1 ? 1 : s;
}

GramPlan gram_plan(int rows, int k) {
    GramPlan p{};
    if (takes_gram_few(rows, k)) return p;
    p.steps = (int)(((long long)rows + 31) / 32);
    const int nt = (k + kTileN - 1) / kTileN, mt = (k + 127) / 128;
    p.tiles = 0;
    for (int t = 0; t < nt; ++t) p.tiles += mt - 2 * t;
    p.splits = gemm_splits(p.tiles, p.steps);
    p.xf = 0;
    p.part = align256(frag_bytes(k / 16, p.steps));
    p.total = p.part + (p.splits > 1 ? (size_t)p.splits * k * k * 4 : 0);
    return p;
}

template <int T, bool BF>
hipError_t gram(const GramPlan& p, Gemm g, hipStream_t s) {
    const Epilogue ep{};
    const dim3 grid(p.tiles, p.splits), block(256);
    hipLaunchKernelGGL((gemm_kernel<T, kOutGram, BF, 4, 1>), grid, block, 0, s, g, ep, ColSum{});
    if (p.splits > 1) hipLaunchKernelGGL(join_gram_kernel, dim3((g.gb + 7) / 8, g.ga / 8), block, 0, s, g);
    return hipGetLastError();
}

}  // namespace

size_t gram_ws_bytes(int rows, int k) { return gram_plan(rows, k).total; }

hipError_t launch_gram(int type, const void* x, long long x_stride, int rows, int k,
                       const uint8_t* valid, const float* prev, float* out, void* ws,
                       hipStream_t s) {
    if (takes_gram_few(rows, k)) {
        const int nt = k / kGramTile;
        const int tiles = nt * (nt + 1) / 2, waves = tiles > kCUs ? 8 : 16;
        auto launch = [&](auto* kernel) {
            hipLaunchKernelGGL(kernel, dim3(tiles), dim3(64 * waves), 0, s, (const uint16_t*)x, x_stride, rows, k,
                               valid, prev, out);
        };
        if (type == kBf16) launch(waves == 8 ? gram_few_kernel<true, 8> : gram_few_kernel<true, 16>);
        else launch(waves == 8 ? gram_few_kernel<false, 8> : gram_few_kernel<false, 16>);
        return hipGetLastError();
    }
    const GramPlan p = gram_plan(rows, k);
    uint16_t* xf = (uint16_t*)ws;
    if (p.steps) hipLaunchKernelGGL(transpose_kernel, dim3(p.steps, k / 128), dim3(256), 0, s, (const uint16_t*)x,
                                    x_stride, rows, p.steps, valid, xf);
    const Gemm g{xf, xf, nullptr, k / 16, k / 16, p.steps, p.tiles, p.splits, (float*)((uint8_t*)ws + p.part), prev, out, k};
    return type == kBf16 ? gram<kBf16, true>(p, g, s) : gram<kF16, false>(p, g, s);
}

}  // namespace xtq
