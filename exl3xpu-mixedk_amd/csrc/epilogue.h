// epilogue.h -- what follows a product with a trellis weight, in the registers of
// the wave that holds its sums.
#pragma once
#include "operators.h"

#pragma clang fp contract(off)

namespace xtq {
namespace {

// Block-128 transform (without its 1/sqrt(128)) of the columns of a unit:
// results of 128 columns by 16 rows in a wave's registers, v[j][i] of lane
// 16 q + r column 16 j + 4 q + i of row r, as the matrix cores leave them.
__device__ __forceinline__ void transform_unit(f4* v) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const f4 a = v[j];
        const float s0 = a[0] + a[1], d0 = a[0] - a[1], s1 = a[2] + a[3], d1 = a[2] - a[3];
        v[j] = (f4){s0 + s1, d0 + d1, s0 - s1, d0 - d1};
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            float a0 = v[j][i], a1 = v[j][i + 1];
            cross_pair<16>(a0, a1);
            cross_pair<32>(a0, a1);
            v[j][i] = a0;
            v[j][i + 1] = a1;
        }
    }
#pragma unroll
    for (int b = 1; b < 8; b <<= 1)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (!(j & b)) {
                const f4 a = v[j], c = v[j | b];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[j][i] = a[i] + c[i];
                    v[j | b][i] = a[i] - c[i];
                }
            }
}

// N (2 or 4) columns' scales and bias.
template <int N>
struct Columns {
    float scale[N], bias[N];
};

template <int N>
__device__ __forceinline__ void load16(const uint16_t* p, uint32_t* w) {
    if constexpr (N == 4) {
        const u2 t = *(const u2_a2*)p;
        w[0] = t[0];
        w[1] = t[1];
    } else {
        w[0] = *(const u1_a2*)p;
    }
}

template <int T, int N>
__device__ __forceinline__ void store16(uint16_t* p, const float* o) {
    if constexpr (N == 4)
        *(u2_a2*)p = (u2){to16<T>(o[0]) | to16<T>(o[1]) << 16, to16<T>(o[2]) | to16<T>(o[3]) << 16};
    else
        *(u1_a2*)p = to16<T>(o[0]) | to16<T>(o[1]) << 16;
}

template <int T, int N>
__device__ __forceinline__ Columns<N> load_columns(const Epilogue& ep, int col) {
    Columns<N> c;
    uint32_t w[N / 2];
    load16<N>(ep.colscale + col, w);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        c.scale[i] = half_bits((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu) * ep.scale;
        c.bias[i] = 0.0f;
    }
    if (ep.bias) {
        if (ep.bias_f32) {
#pragma unroll
            for (int i = 0; i < N; ++i) c.bias[i] = ((const float*)ep.bias)[col + i];
        } else {
            load16<N>((const uint16_t*)ep.bias + col, w);
#pragma unroll
            for (int i = 0; i < N; ++i) c.bias[i] = from16<T>((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
        }
    }
    return c;
}

// Scales, bias, activation and residual of N columns of a row, and their store
// (v: transformed sums).  y comes of the unrounded z; the z that is kept for the
// gradient has the activations' type, as they are kept themselves: a slope taken
// at it is off by |z act''(z)| <= 0.32 times z's relative rounding, which adds 6 %
// at most to the error that the gradient's own rounding leaves.
template <int T, int N>
__device__ __forceinline__ void finish_cols(const float* v, const Columns<N>& c, const Epilogue& ep, int row,
                                            int col) {
    const int e = ep.rowexp ? ep.rowexp[row] : 0;
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = ldexpf(v[i], e) * c.scale[i] + c.bias[i];
    if (ep.z) store16<T, N>((uint16_t*)ep.z + (size_t)row * ep.cols + col, o);
    activate<N>(o, ep.act);
    if (ep.res) {
        uint32_t w[N / 2];
        load16<N>((const uint16_t*)ep.res + (size_t)row * ep.res_stride + col, w);
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] += from16<T>((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
    }
    store16<T, N>((uint16_t*)ep.y + (size_t)row * ep.y_stride + col, o);
}

// Columns of a unit's lanes.
template <int T>
__device__ __forceinline__ void unit_columns(Columns<4> (&c)[8], const Epilogue& ep, int blk, int lane) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = load_columns<T, 4>(ep, blk * 128 + 16 * j + 4 * (lane >> 4));
}

// A whole unit.
template <int T>
__device__ __forceinline__ void finish_unit(f4* v, const Columns<4> (&c)[8], const Epilogue& ep, int grp, int blk,
                                            int lane) {
    transform_unit(v);
    const int row = grp * 16 + (lane & 15);
    if (row >= ep.rows) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float t[4] = {v[j][0], v[j][1], v[j][2], v[j][3]};
        finish_cols<T, 4>(t, c[j], ep, row, blk * 128 + 16 * j + 4 * (lane >> 4));
    }
}

// Two columns, 2 l and 2 l + 1, of a row of a unit that lies in LDS as the
// matrix cores left it.
__device__ __forceinline__ void unit_row(const f4* unit, int row, int lane, float& a, float& b) {
    const float* p = (const float*)(unit + (lane >> 3) * 64 + ((lane >> 1) & 3) * 16 + row) + 2 * (lane & 1);
    a = p[0];
    b = p[1];
}

// R rows (row0 + i step, up to ep.rows) of the columns whose sums the wave's
// lanes hold, 2 l and 2 l + 1 of block blk: transform, scales, bias, activation,
// residual, store.
template <int R>
__device__ __forceinline__ void finish_rows(float (&v)[R][2], const Columns<2>& c, const Epilogue& ep, int type,
                                            int blk, int row0, int step, int lane) {
    const int col = blk * 128 + 2 * lane;
#pragma unroll
    for (int i = 0; i < R; ++i) transform_row(v[i][0], v[i][1], lane);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int row = row0 + i * step;
        if (row >= ep.rows) break;
        if (type == kBf16) finish_cols<kBf16, 2>(v[i], c, ep, row, col);
        else finish_cols<kF16, 2>(v[i], c, ep, row, col);
    }
}

}  // namespace
}  // namespace xtq
