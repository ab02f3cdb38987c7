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
// arithmetic.
#include "epilogue.h"
#include "few_device.h"
#include "operators.h"

#pragma clang fp contract(off)

namespace xtq {
namespace {

constexpr int kFragBytes = 1024;

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

// Per row, the power of two that brings its transformed values into fp16's
// range: the largest |x * colscale| goes to [2^7, 2^8), the transform's sums of
// 128 stay below 2^15.  rowexp[m]: what the product has to be multiplied with
// (as a power of two), with the two transforms' 1/128.
__global__ __launch_bounds__(256) void row_exp_kernel(Source s, int32_t* __restrict__ shift,
                                                      int32_t* __restrict__ rowexp) {
    __shared__ float part[4];
    const int row = blockIdx.x;
    float top = 0.0f;
    for (int c = threadIdx.x * 8; c < s.cols; c += 2048) {
        float v[8];
        load8(s, row, c, v);
        scale8(s.colscale, c, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
        const int sh = shift_to(top, 7);
        shift[row] = sh;
        rowexp[row] = -sh - 7;
    }
}

// Rows to fragments: values times column scales, block-128 transform, times
// 2^shift, rounded to fp16 (the one rounding of the activations: 2^-11
// relative, as fp16 activations have themselves).  A wave takes 16 rows of one
// 128-column block; lane 16 q + r holds columns 32 p + 8 q + j of row r, so five
// of the transform's seven stages are between its own registers.  Rows past the
// end are zeros.  colsum: sums over the 16 rows of the unscaled values, one row
// of partial sums per 16 rows (for the bias' gradient).
__global__ __launch_bounds__(256) void transform_kernel(Source s, const int32_t* __restrict__ shift,
                                                        uint16_t* __restrict__ frags,
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
#pragma unroll
            for (int m = 1; m < 16; m <<= 1) t += __shfl_xor(t, m);
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
    uint16_t* out = frags + ((size_t)grp * nblk + blk) * 2048 + lane * 8;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        h8 o;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (_Float16)v[8 * p + i];
        *(h8*)(out + p * 512) = o;
    }
}

// Column sums' last step: out[c] = sum of part[g][c] over the groups, in order.
__global__ __launch_bounds__(256) void colsum_kernel(const float* __restrict__ part, int groups,
                                                     int cols, int type, int f32, void* out) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float t = 0.0f;
    for (int g = 0; g < groups; ++g) t += part[(size_t)g * cols + c];
    if (f32) ((float*)out)[c] = t;
    else ((uint16_t*)out)[c] = (uint16_t)(type == kBf16 ? to16<kBf16>(t) : to16<kF16>(t));
}

// Trellis to fragments of the inner weight.  BWD = 0: fragment (ng, p) holds
// columns 16 ng + r, summed rows 32 p + 8 q + j (operand of x Wi); BWD = 1:
// rows 16 kg + r, summed columns (operand of dz Wi^T).  Element (r, c) of a tile
// is symbol 32 (c % 8) + 8 ((r % 8) / 2) + 4 (c / 8) + 2 (r / 8) + r % 2, its state
// the 16-bit circular window ending with the symbol's K bits.  A workgroup
// takes 8 by 4 tiles (along the summed dimension by the other), the trellis
// words staged in LDS.
template <int K, int CODE, int BWD>
__global__ __launch_bounds__(256) void decode_frag_kernel(const int16_t* __restrict__ trellis,
                                                          int tk, int tn,
                                                          uint16_t* __restrict__ frags) {
    constexpr int TW = 8 * K;                           // words of a tile
    __shared__ uint32_t words[32 * TW];
    const int i0 = blockIdx.y * (BWD ? 4 : 8), j0 = blockIdx.x * (BWD ? 8 : 4);   // first tile
    constexpr int NJ = BWD ? 8 : 4;
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
        *(u4*)(frags + (g * np + f) * 512 + lane * 8) = o;
    }
}

// -------------------------------------------------------------------- matrix
// product of fragments: columns (fragments A) by rows (fragments B).  A
// workgroup's tile is 256 columns by 256 rows, 8 waves of 128 columns (a whole
// transform block, so the epilogue's transform stays in registers) by 64 rows.
constexpr int kTile = 256;              // rows and columns of a workgroup's tile
constexpr int kStage = 2;               // 32-wide steps of the summed dimension per stage

enum GemmOut { kOutEpilogue, kOutPartial, kOutGram };

struct Gemm {
    const uint16_t *A, *B;
    int ga, gb;                         // 16-wide groups of columns, rows
    int steps;                          // 32-wide steps of the summed dimension (even)
    int splits;                         // of the summed dimension
    float* part;                        // kOutPartial: [splits][blocks of 128][gb][8][64][4]
    const float* prev;                  // kOutGram
    float* out;
    int dim;
};

template <int T, bool BF>
__device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a),
                                                                    __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a),
                                                       __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

template <int T, int OUT, bool BF>
__global__ __launch_bounds__(512, 2) void gemm_kernel(Gemm g, Epilogue ep) {
    __shared__ __align__(1024) uint8_t lds[2][2 * 16 * kStage * kFragBytes];
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wv & 1, wm = wv >> 1;
    int tn, tm;
    if constexpr (OUT == kOutGram) {    // tiles on and below the diagonal, tn <= tm
        tm = (int)((sqrtf(8.0f * blockIdx.x + 1.0f) - 1.0f) * 0.5f);
        while ((tm + 1) * (tm + 2) / 2 <= (int)blockIdx.x) ++tm;
        while (tm * (tm + 1) / 2 > (int)blockIdx.x) --tm;
        tn = blockIdx.x - tm * (tm + 1) / 2;
    } else {
        const int nt = (g.ga + 15) / 16;
        tn = blockIdx.x % nt;
        tm = blockIdx.x / nt;
    }
    const int nst = g.steps / kStage, split = blockIdx.y;
    const int s0 = (int)((long long)nst * split / g.splits);
    const int s1 = (int)((long long)nst * (split + 1) / g.splits);

    // this wave's eight fragments of a stage: 4 groups of A or B by 2 steps
    const bool isb = wv >= 4;
    const uint16_t* base = isb ? g.B : g.A;
    const int lim = (isb ? g.gb : g.ga) - 1, first = (isb ? tm : tn) * 16 + (wv & 3) * 4;
    auto load = [&](int s, int buf) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int grp = first + (i >> 1);
            grp = grp < lim ? grp : lim;
            const uint16_t* p = base + ((size_t)grp * g.steps + (size_t)s * kStage + (i & 1)) * 512 +
                                lane * 8;
            __builtin_amdgcn_global_load_lds((global_void*)p,
                                             (lds_void*)(lds[buf] + (wv * 8 + i) * kFragBytes), 16, 0, 0);
        }
    };
    f4 acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[j][b] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    if (s0 < s1) load(s0, 0);
    for (int s = s0; s < s1; ++s) {
        const int buf = (s - s0) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        u4 a[2][8], b[2][4];
        const uint8_t* l = lds[buf] + lane * 16;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int j = 0; j < 8; ++j) a[p][j] = *(const u4*)(l + ((wn * 8 + j) * 2 + p) * kFragBytes);
#pragma unroll
            for (int i = 0; i < 4; ++i) b[p][i] = *(const u4*)(l + (32 + (wm * 4 + i) * 2 + p) * kFragBytes);
        }
        if (s + 1 < s1) load(s + 1, buf ^ 1);
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[j][i] = mfma<T, BF>(a[p][j], b[p][i], acc[j][i]);
    }
    const int blk = tn * 2 + wn;
    if (blk * 8 >= g.ga) return;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int grp = tm * 16 + wm * 4 + b;
        if (grp >= g.gb) continue;
        f4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = acc[j][b];
        if constexpr (OUT == kOutEpilogue) {
            finish_unit<T>(v, ep, grp, blk, lane);
        } else if constexpr (OUT == kOutPartial) {
            f4* o = (f4*)g.part + (((size_t)split * (g.ga / 8) + blk) * g.gb + grp) * 512 + lane;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j * 64] = v[j];
        } else {
            const size_t row = (size_t)grp * 16 + (lane & 15);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const size_t col = (size_t)blk * 128 + 16 * j + 4 * (lane >> 4);
                f4 o = v[j];
                if (g.prev) {
                    const f4 p = *(const f4_a4*)(g.prev + row * g.dim + col);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = p[i] + v[j][i];
                }
                *(f4_a4*)(g.out + row * g.dim + col) = o;
                if (tn != tm) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const size_t at = (col + i) * g.dim + row;
                        g.out[at] = g.prev ? g.prev[at] + v[j][i] : v[j][i];
                    }
                }
            }
        }
    }
}

// Sums the splits' partial products of a unit (128 columns by 16 rows), in
// order, and finishes it.
template <int T>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, int splits,
                                                   int blocks, int groups, Epilogue ep) {
    const int lane = threadIdx.x & 63, grp = blockIdx.x * 4 + (threadIdx.x >> 6), blk = blockIdx.y;
    if (grp >= groups) return;
    f4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < splits; ++s) {
        const f4* p = (const f4*)part + (((size_t)s * blocks + blk) * groups + grp) * 512 + lane;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const f4 t = p[j * 64];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[j][i] += t[i];
        }
    }
    finish_unit<T>(v, ep, grp, blk, lane);
}

// ---------------------------------------------------------------------- Gram
// Rows of activations to fragments of their transpose: 16 channels by 32 rows.
// Rows that are not valid, or past the end, are zeros whatever they hold.  A
// workgroup takes 32 rows by 128 channels.
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
        *(u4*)(frags + ((size_t)(c0 / 16 + wv * 2 + g) * steps + p) * 512 + lane * 8) = o;
    }
}

template <int K, int CODE>
void decode_kc(const Weight& w, int bwd, uint16_t* frags, hipStream_t s) {
    const int tk = w.k / 16, tn = w.n / 16;
    if (bwd) hipLaunchKernelGGL((decode_frag_kernel<K, CODE, 1>), dim3(tn / 8, tk / 4), dim3(256), 0, s,
                                w.trellis, tk, tn, frags);
    else hipLaunchKernelGGL((decode_frag_kernel<K, CODE, 0>), dim3(tn / 4, tk / 8), dim3(256), 0, s,
                            w.trellis, tk, tn, frags);
}

template <int K>
void decode_k(const Weight& w, int bwd, uint16_t* frags, hipStream_t s) {
    if (w.code == kCodeMul1) decode_kc<K, kCodeMul1>(w, bwd, frags, s);
    else if (w.code == kCodeMcg) decode_kc<K, kCodeMcg>(w, bwd, frags, s);
    else decode_kc<K, kCode3Inst>(w, bwd, frags, s);
}

void decode_frags(const Weight& w, int bwd, uint16_t* frags, hipStream_t s) {
    switch (w.K) {
        case 2: return decode_k<2>(w, bwd, frags, s);
        case 3: return decode_k<3>(w, bwd, frags, s);
        case 4: return decode_k<4>(w, bwd, frags, s);
        case 5: return decode_k<5>(w, bwd, frags, s);
        case 6: return decode_k<6>(w, bwd, frags, s);
        default: return decode_k<7>(w, bwd, frags, s);
    }
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// Splits of the summed dimension: as many as fill the compute units, each with
// at least 8 stages.
int gemm_splits(int tiles, int steps) {
    const int most = steps / kStage / 8;
    int s = tiles >= kCUs ? 1 : kCUs / tiles;
    if (s > most) s = most;
    return s < 1 ? 1 : s;
}

struct ManyPlan {
    int groups, tiles, splits;
    size_t shift, rowexp, xf, wf, part, colsum, total;
};

// Scratch of a product of `rows` rows: summed dimension k, columns n.
ManyPlan many_plan(int rows, int k, int n, bool colsum) {
    ManyPlan p;
    p.groups = (rows + 15) / 16;
    p.tiles = ((n + kTile - 1) / kTile) * ((rows + kTile - 1) / kTile);
    p.splits = gemm_splits(p.tiles, k / 32);
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t a = at; at += align256(bytes); return a; };
    p.shift = take((size_t)p.groups * 64);
    p.rowexp = take((size_t)p.groups * 64);
    p.xf = take((size_t)p.groups * 32 * k);
    p.wf = take((size_t)n * k * 2);
    p.part = take(p.splits > 1 ? (size_t)p.splits * p.groups * 64 * n : 0);
    p.colsum = take(colsum ? (size_t)p.groups * k * 4 : 0);
    p.total = at;
    return p;
}

// The product of a source's rows with a weight (bwd: its transpose).
template <int T>
hipError_t many(const Weight& w, int bwd, const Source& src, Epilogue ep, void* dbias, int dbias_f32,
                void* ws, hipStream_t s) {
    const int k = src.cols, n = ep.cols, rows = src.rows;
    const ManyPlan p = many_plan(rows, k, n, dbias != nullptr);
    uint8_t* base = (uint8_t*)ws;
    int32_t *shift = (int32_t*)(base + p.shift), *rowexp = (int32_t*)(base + p.rowexp);
    uint16_t *xf = (uint16_t*)(base + p.xf), *wf = (uint16_t*)(base + p.wf);
    float* colsum = dbias ? (float*)(base + p.colsum) : nullptr;
    hipLaunchKernelGGL(row_exp_kernel, dim3(rows), dim3(256), 0, s, src, shift, rowexp);
    hipLaunchKernelGGL(transform_kernel, dim3((k / 128 + 3) / 4, p.groups), dim3(256), 0, s, src,
                       (const int32_t*)shift, xf, colsum);
    if (dbias) hipLaunchKernelGGL(colsum_kernel, dim3((k + 255) / 256), dim3(256), 0, s, colsum, p.groups,
                                  k, T, dbias_f32, dbias);
    if (!ep.y) return hipGetLastError();
    decode_frags(w, bwd, wf, s);
    ep.rowexp = rowexp;
    Gemm g{wf, xf, n / 16, p.groups, k / 32, p.splits, (float*)(base + p.part), nullptr, nullptr, 0};
    if (p.splits == 1) {
        hipLaunchKernelGGL((gemm_kernel<T, kOutEpilogue, false>), dim3(p.tiles), dim3(512), 0, s, g, ep);
    } else {
        hipLaunchKernelGGL((gemm_kernel<T, kOutPartial, false>), dim3(p.tiles, p.splits), dim3(512), 0, s,
                           g, ep);
        hipLaunchKernelGGL((join_kernel<T>), dim3((p.groups + 3) / 4, n / 128), dim3(256), 0, s, g.part,
                           p.splits, n / 128, p.groups, ep);
    }
    return hipGetLastError();
}

// Rows to fragments for the products of few rows, a wave for one row's
// 128-column block.  Rows past the end are zeros.
__global__ __launch_bounds__(256) void transform_few_kernel(const uint16_t* __restrict__ x, long long stride,
                                                            int type, int rows, int k,
                                                            const uint16_t* __restrict__ suh,
                                                            u4* __restrict__ frag, int32_t* __restrict__ shift) {
    const int lane = threadIdx.x & 63, nk = k / 128;
    const int kb = blockIdx.x * 4 + (threadIdx.x >> 6), row = blockIdx.y;
    if (kb >= nk) return;
    float a = 0.0f, b = 0.0f, sa, sb;
    if (row < rows) unpack_two(load_two(x + (size_t)row * stride + 128 * kb, lane), type, a, b);
    unpack_two(load_two(suh + 128 * kb, lane), kF16, sa, sb);
    const size_t at = (size_t)(row >> 4) * nk + kb;
    const int sh = row_to_frags<false>(a * sa, b * sb, lane, row & 15, (uint32_t*)(frag + at * 256), nullptr);
    if (lane == 0) shift[at * 16 + (row & 15)] = sh;
}

// Workgroups per 128 columns of a product of few rows: two for each compute
// unit, each wave with two 32-row steps at least.
int few_splits(int k, int n) {
    const int most = k / 256;
    int s = 2 * kCUs / (n / 128);
    if (s > most) s = most;
    return s < 1 ? 1 : s;
}

bool takes_few(int rows, int n) { return rows <= kFewRows && n / 128 <= XTQ_OP_COUNTERS; }

int few_groups(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

struct FewPlan {
    int splits;
    size_t part, frag, shift, total;
};

FewPlan few_plan(int rows, int k, int n) {
    FewPlan p;
    p.splits = few_splits(k, n);
    const int g = few_groups(rows);
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t a = at; at += align256(bytes); return a; };
    p.part = take(p.splits > 1 ? (size_t)p.splits * n * g * 64 : 0);
    const bool apart = rows > kFusedRows;
    p.frag = take(apart ? (size_t)g * k * 32 : 0);
    p.shift = take(apart ? (size_t)g * k / 2 : 0);
    p.total = at;
    return p;
}

}  // namespace

size_t linear_ws_bytes(int rows, int k, int n, int backward) {
    if (!backward && takes_few(rows, n)) return few_plan(rows, k, n).total;
    return backward ? many_plan(rows, n, k, true).total : many_plan(rows, k, n, false).total;
}

hipError_t launch_linear(const Weight& w, int type, const void* x, long long x_stride, int rows,
                         const Epilogue& ep, void* ws, uint32_t* counters, hipStream_t s) {
    if (takes_few(rows, w.n)) {
        static decltype(&launch_few_k2) const few[] = {launch_few_k2, launch_few_k3, launch_few_k4,
                                                       launch_few_k5, launch_few_k6, launch_few_k7};
        const FewPlan p = few_plan(rows, w.k, w.n);
        uint8_t* base = (uint8_t*)ws;
        FewArgs a{type, (const uint16_t*)x, x_stride, nullptr, nullptr, p.splits, w.k / 32 / p.splits,
                  w.k / 32 % p.splits, 65536u / rows + 1, (float*)(base + p.part), counters};
        if (rows > kFusedRows) {
            u4* frag = (u4*)(base + p.frag);
            int32_t* shift = (int32_t*)(base + p.shift);
            hipLaunchKernelGGL(transform_few_kernel, dim3((w.k / 128 + 3) / 4, 16 * few_groups(rows)),
                               dim3(256), 0, s, a.x, x_stride, type, rows, w.k, w.suh, frag, shift);
            a.frag = frag;
            a.shift = shift;
        }
        return few[w.K - 2](w, a, ep, s);
    }
    const Source src{(const uint16_t*)x, x_stride, nullptr, 0, w.suh, type, rows, w.k};
    return type == kBf16 ? many<kBf16>(w, 0, src, ep, nullptr, 0, ws, s)
                         : many<kF16>(w, 0, src, ep, nullptr, 0, ws, s);
}

hipError_t launch_linear_bwd(const Weight& w, int type, const void* dy, long long dy_stride,
                             const void* z, int act, int rows, void* dx, long long dx_stride,
                             void* dbias, int dbias_f32, void* ws, uint32_t* counters,
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
    return type == kBf16 ? many<kBf16>(w, 1, src, ep, dbias, dbias_f32, ws, s)
                         : many<kF16>(w, 1, src, ep, dbias, dbias_f32, ws, s);
}

size_t gram_ws_bytes(int rows, int k) {
    const size_t steps = ((size_t)rows + 63) / 64 * 2;
    return steps * (k / 16) * kFragBytes;
}

hipError_t launch_gram(int type, const void* x, long long x_stride, int rows, int k,
                       const uint8_t* valid, const float* prev, float* out, void* ws,
                       hipStream_t s) {
    const int steps = (rows + 63) / 64 * 2, nt = (k + kTile - 1) / kTile;
    uint16_t* xf = (uint16_t*)ws;
    if (steps) hipLaunchKernelGGL(transpose_kernel, dim3(steps, k / 128), dim3(256), 0, s, (const uint16_t*)x, x_stride,
                       rows, steps, valid, xf);
    Gemm g{xf, xf, k / 16, k / 16, steps, 1, nullptr, prev, out, k};
    const Epilogue ep{};
    if (type == kBf16) hipLaunchKernelGGL((gemm_kernel<kBf16, kOutGram, true>), dim3(nt * (nt + 1) / 2),
                                          dim3(512), 0, s, g, ep);
    else hipLaunchKernelGGL((gemm_kernel<kF16, kOutGram, false>), dim3(nt * (nt + 1) / 2), dim3(512), 0, s, g,
                            ep);
    return hipGetLastError();
}

}  // namespace xtq
