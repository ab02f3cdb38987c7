// norm_kernels.hip -- norms of rows, and the residual sum between two blocks with
// the norms before and after it, its gate and its scale; with their gradients.
//
// Of a block's result x, its residual r, gate g and scale s,
//   p = post norm of x (or x),  q = p ga(g),  y = r + s q,  h = norm of y,
// the norm of t being (t - mean) / sqrt(mean (t - mean)^2 + eps) w + b, without its
// mean for "rms".  The plain norm is h of y = x.  h comes of y before it is rounded.
//
// A row's group of lanes (16, a wave or a workgroup, by the width alone, so that a
// row's result does not depend on how many there are) holds the row in registers:
// every input is read once, deviations are squared around the mean itself.
#include "operators.h"

#pragma clang fp contract(off)

namespace xtq {
namespace {

// Rows of 16 lanes (four a wave), of a wave, of a workgroup.
enum Mode { kSub, kWave, kBlock };

template <int T>
__device__ __forceinline__ void unpack(u4 w, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = from16<T>(w[i] & 0xFFFFu);
        v[2 * i + 1] = from16<T>(w[i] >> 16);
    }
}

// Eight values of a row, `n` of which (at most 8) lie inside it; the others are 0.
__device__ __forceinline__ u4 load8(const uint16_t* p, int n) {
    if (n >= 8) return *(const u4_a2*)p;
    u4 w = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) w[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    return w;
}

template <int T>
__device__ __forceinline__ void store8(uint16_t* p, int n, const float* v) {
    u4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = to16<T>(v[2 * i]) | to16<T>(v[2 * i + 1]) << 16;
    if (n >= 8) {
        *(u4_a2*)p = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
}

// Eight channels of a parameter (of the rows' type or fp32), `missing` where there is none.
template <int T>
__device__ __forceinline__ void param8(const NormParam& p, int col, int n, float missing, float* v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = missing;
    if (!p.p || n <= 0) return;
    if (p.f32) {
        const float* f = (const float*)p.p + col;
        if (n >= 8) {
            const f4 a = *(const f4_a4*)f, b = *(const f4_a4*)(f + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = a[i];
                v[4 + i] = b[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) v[i] = f[i];
        }
    } else {
        unpack<T>(load8((const uint16_t*)p.p + col, n), v);
    }
}

// Gate's factor and its slope.
__device__ __forceinline__ float gate_value(float g, int act) {
    if (act == kGateNone) return g;
    const float s = fast_rcp(1.0f + fast_exp(-g));
    return act == kGateSigmoid ? s : g * s;
}
__device__ __forceinline__ float gate_slope(float g, int act) {
    if (act == kGateNone) return 1.0f;
    if (act == kGateSilu) return act_slope(g, kActSilu);
    // s (1 - s) without the difference, which loses s's neighbourhood of 1
    const float e = fast_exp(-fabsf(g)), r = fast_rcp(1.0f + e);
    return e * r * r;
}

// Sum over the lanes of 16, of the wave.
__device__ __forceinline__ float sum16(float v) {
    v += lane_xor<1>(v);
    v += lane_xor<2>(v);
    v += dpp<0x141>(v);
    v += dpp<0x140>(v);
    return v;
}

__device__ __forceinline__ float sum64(float v) {
    v = sum16(v);
    uint32_t b = __float_as_uint(v);
    auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    b = __float_as_uint(v);
    r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sums over a row's lanes.  A workgroup's waves meet in LDS, one barrier a sum: two
// places in turn, and who comes to write a place again has met, in between, all
// who read it.
template <int MODE>
struct Group {
    int lane, width, turn = 0;          // the row's lane and lanes
    __device__ Group() {
        lane = MODE == kSub ? threadIdx.x & 15 : MODE == kWave ? threadIdx.x & 63 : threadIdx.x;
        width = MODE == kSub ? 16 : MODE == kWave ? 64 : blockDim.x;
    }
    template <int N>
    __device__ __forceinline__ void sum(float (&v)[N]) {
        if constexpr (MODE == kSub) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = sum16(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = sum64(v[i]);
        }
        if constexpr (MODE == kBlock) {
            __shared__ float part[2][2][16];
            const int wv = threadIdx.x >> 6, waves = blockDim.x >> 6, l = threadIdx.x & 15;
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int i = 0; i < N; ++i) part[turn][i][wv] = v[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = sum16(l < waves ? part[turn][i][l] : 0.0f);
            turn ^= 1;
        }
    }
    __device__ __forceinline__ float sum(float t) {
        float v[1] = {t};
        sum(v);
        return v[0];
    }
};

// Mean (0 for "rms") and 1 / sqrt(mean square of the deviations + eps) of a row.
template <int MODE, int V>
__device__ __forceinline__ void row_stats(Group<MODE>& g, const float (&t)[V][8], int d, int kind, float eps,
                                          float& mean, float& rstd) {
    mean = 0.0f;
    float s = 0.0f;
    if (kind == kNormLayer) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) s += t[v][i];
        mean = g.sum(s) / (float)d;
    }
    s = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = (v * g.width + g.lane) * 8 + i < d ? t[v][i] - mean : 0.0f;
            s = __builtin_fmaf(c, c, s);
        }
    rstd = 1.0f / sqrtf(g.sum(s) / (float)d + eps);
}

template <int T, int MODE, int V>
__global__ __launch_bounds__(MODE == kBlock ? 1024 : 256) void norm_kernel(NormArgs a) {
    Group<MODE> g;
    const int row = MODE == kSub ? blockIdx.x * 16 + (threadIdx.x >> 4)
                                 : MODE == kWave ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    const bool in = row < a.rows;
    const size_t at = in ? row : 0;
    int col[V], n[V];
    u4 wx[V], wr[V], wg[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        col[v] = (v * g.width + g.lane) * 8;
        n[v] = in ? a.d - col[v] : 0;
        wx[v] = load8(a.x + at * a.x_stride + col[v], n[v]);
        wr[v] = a.res ? load8(a.res + at * a.res_stride + col[v], n[v]) : (u4){0u, 0u, 0u, 0u};
        if (a.gate) wg[v] = load8(a.gate + at * a.gate_stride + col[v], n[v]);
    }
    float t[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) unpack<T>(wx[v], t[v]);
    float mean, rstd;
    f4 stats = {0.0f, 0.0f, 0.0f, 0.0f};
    if (a.post) {
        row_stats<MODE, V>(g, t, a.d, a.post, a.post_eps, mean, rstd);
        stats[0] = mean;
        stats[1] = rstd;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float w[8], b[8];
            param8<T>(a.post_weight, col[v], n[v], 1.0f, w);
            param8<T>(a.post_bias, col[v], n[v], 0.0f, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) t[v][i] = (t[v][i] - mean) * rstd * w[i] + b[i];
        }
    }
    if (a.res) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float s[8], r[8], y[8];
            param8<T>(a.scale, col[v], n[v], a.scale_number, s);
            unpack<T>(wr[v], r);
            if (a.gate) {
                float e[8];
                unpack<T>(wg[v], e);
#pragma unroll
                for (int i = 0; i < 8; ++i) t[v][i] *= gate_value(e[i], a.gate_act);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) t[v][i] = r[i] + s[i] * t[v][i];
            if (n[v] > 0) store8<T>(a.y + at * a.y_stride + col[v], n[v], t[v]);
        }
    }
    if (a.kind) {
        row_stats<MODE, V>(g, t, a.d, a.kind, a.eps, mean, rstd);
        stats[2] = mean;
        stats[3] = rstd;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float w[8], b[8];
            param8<T>(a.weight, col[v], n[v], 1.0f, w);
            param8<T>(a.bias, col[v], n[v], 0.0f, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) t[v][i] = (t[v][i] - mean) * rstd * w[i] + b[i];
            if (n[v] > 0) store8<T>(a.h + at * a.h_stride + col[v], n[v], t[v]);
        }
    }
    if (a.stats && in && g.lane == 0) *(f4*)(a.stats + 4 * at) = stats;
}

// Gradients.  With c = dh w, t^ = (y - mean) rstd,
//   dy' = dy + rstd (c - t^ mean(c t^) - mean(c))       (the last for "layer"),
//   dres = dy',  ds = sum of dy' q,  dgate = dy' s p ga'(g),  dp = dy' s ga(g),
// and dx from dp as dy' from dh.  y and the norms are computed anew from the inputs
// and the rows' saved means and factors, so nothing of y's rounding enters.  A
// group goes through its rows with the channels' sums in registers; a workgroup
// leaves one row of partial sums, which norm_sums_kernel adds in order.
template <int T, int MODE, int V, bool SUMS>
__global__ __launch_bounds__(MODE == kBlock ? 1024 : 256) void norm_bwd_kernel(NormGradArgs a) {
    Group<MODE> g;
    constexpr int R = MODE == kSub ? 16 : MODE == kWave ? 4 : 1;        // rows of a workgroup at a time
    const int sub = MODE == kSub ? threadIdx.x >> 4 : MODE == kWave ? threadIdx.x >> 6 : 0;
    float sums[SUMS ? kNormSums : 1][V][8];
    if constexpr (SUMS)
#pragma unroll
        for (int k = 0; k < kNormSums; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) sums[k][v][i] = 0.0f;
    const float inv = 1.0f / (float)a.f.d;
    for (int base = blockIdx.x * R; base < a.f.rows; base += gridDim.x * R) {
        const int row = base + sub;
        const bool in = row < a.f.rows;
        const size_t at = in ? row : 0;
        const f4 stats = *(const f4*)(a.f.stats + 4 * at);
        int n[V];
        u4 wx[V], wr[V], wg[V], wy[V], wh[V];
        const u4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int col = (v * g.width + g.lane) * 8;
            n[v] = in ? a.f.d - col : 0;
            wx[v] = load8(a.f.x + at * a.f.x_stride + col, n[v]);
            wr[v] = a.f.res ? load8(a.f.res + at * a.f.res_stride + col, n[v]) : zero;
            wg[v] = a.f.gate ? load8(a.f.gate + at * a.f.gate_stride + col, n[v]) : zero;
            wy[v] = a.dy ? load8(a.dy + at * a.dy_stride + col, n[v]) : zero;
            wh[v] = a.dh ? load8(a.dh + at * a.dh_stride + col, n[v]) : zero;
        }
        float hat[V][8], that[V][8], p[V][8], q[V][8], dt[V][8], c[V][8];
        float two[2] = {0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int col = (v * g.width + g.lane) * 8;
            float w[8], b[8], s[8];
            unpack<T>(wx[v], hat[v]);
            if (a.f.post) {
                param8<T>(a.f.post_weight, col, n[v], 1.0f, w);
                param8<T>(a.f.post_bias, col, n[v], 0.0f, b);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    hat[v][i] = i < n[v] ? (hat[v][i] - stats[0]) * stats[1] : 0.0f;
                    p[v][i] = hat[v][i] * w[i] + b[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) p[v][i] = hat[v][i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) q[v][i] = p[v][i];
            if (a.f.gate) {
                float e[8];
                unpack<T>(wg[v], e);
#pragma unroll
                for (int i = 0; i < 8; ++i) q[v][i] *= gate_value(e[i], a.f.gate_act);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) that[v][i] = q[v][i];
            if (a.f.res) {
                float r[8];
                unpack<T>(wr[v], r);
                param8<T>(a.f.scale, col, n[v], a.f.scale_number, s);
#pragma unroll
                for (int i = 0; i < 8; ++i) that[v][i] = r[i] + s[i] * q[v][i];
            }
            unpack<T>(wy[v], dt[v]);
            if (a.dh) {
                float dh[8];
                unpack<T>(wh[v], dh);
                param8<T>(a.f.weight, col, n[v], 1.0f, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    that[v][i] = i < n[v] ? (that[v][i] - stats[2]) * stats[3] : 0.0f;
                    c[v][i] = dh[i] * w[i];
                    two[0] = __builtin_fmaf(c[v][i], that[v][i], two[0]);
                    two[1] += c[v][i];
                    if constexpr (SUMS) {
                        sums[kSumWeight][v][i] = __builtin_fmaf(dh[i], that[v][i], sums[kSumWeight][v][i]);
                        sums[kSumBias][v][i] += dh[i];
                    }
                }
            }
        }
        if (a.dh) {
            g.sum(two);
            const float c1 = two[0] * inv, c2 = a.f.kind == kNormLayer ? two[1] * inv : 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) dt[v][i] += stats[3] * (c[v][i] - that[v][i] * c1 - c2);
        }
        two[0] = two[1] = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int col = (v * g.width + g.lane) * 8;
            if (a.dres && n[v] > 0) store8<T>(a.dres + at * a.f.d + col, n[v], dt[v]);
            if (a.f.res) {
                float s[8];
                param8<T>(a.f.scale, col, n[v], a.f.scale_number, s);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (SUMS)
                        sums[kSumScale][v][i] = __builtin_fmaf(i < n[v] ? dt[v][i] : 0.0f, q[v][i], sums[kSumScale][v][i]);
                    dt[v][i] *= s[i];
                }
            }
            if (a.f.gate) {
                float e[8], o[8];
                unpack<T>(wg[v], e);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    o[i] = dt[v][i] * p[v][i] * gate_slope(e[i], a.f.gate_act);
                    dt[v][i] *= gate_value(e[i], a.f.gate_act);
                }
                if (a.dgate && n[v] > 0) store8<T>(a.dgate + at * a.f.d + col, n[v], o);
            }
            if (a.f.post) {
                float w[8];
                param8<T>(a.f.post_weight, col, n[v], 1.0f, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float dp = i < n[v] ? dt[v][i] : 0.0f;
                    c[v][i] = dp * w[i];
                    two[0] = __builtin_fmaf(c[v][i], hat[v][i], two[0]);
                    two[1] += c[v][i];
                    if constexpr (SUMS) {
                        sums[kSumPostWeight][v][i] = __builtin_fmaf(dp, hat[v][i], sums[kSumPostWeight][v][i]);
                        sums[kSumPostBias][v][i] += dp;
                    }
                }
            }
        }
        if (a.f.post) {
            g.sum(two);
            const float c1 = two[0] * inv, c2 = a.f.post == kNormLayer ? two[1] * inv : 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) dt[v][i] = stats[1] * (c[v][i] - hat[v][i] * c1 - c2);
        }
        if (a.dx)
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (n[v] > 0) store8<T>(a.dx + at * a.f.d + (v * g.width + g.lane) * 8, n[v], dt[v]);
    }
    if constexpr (SUMS) {
        // [sum][workgroup][d]
        __shared__ float join[MODE == kBlock ? 1 : 256 * 8];
#pragma unroll
        for (int k = 0; k < kNormSums; ++k) {
            if (!a.dparam[k].p) continue;
            float* out = a.part + ((size_t)a.place[k] * gridDim.x + blockIdx.x) * a.f.d;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int col = (v * g.width + g.lane) * 8;
                if constexpr (MODE != kBlock) {
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < 8; ++i) join[threadIdx.x * 8 + i] = sums[k][v][i];
                    __syncthreads();
                    if (sub == 0)
                        for (int o = 1; o < R; ++o)
#pragma unroll
                            for (int i = 0; i < 8; ++i) sums[k][v][i] += join[(threadIdx.x + o * g.width) * 8 + i];
                    if (sub != 0) continue;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (col + i < a.f.d) out[col + i] = sums[k][v][i];
            }
        }
    }
}

// The channels' sums: 16 waves take every 16th part of 64 channels and meet in LDS.
__global__ __launch_bounds__(1024) void norm_sums_kernel(NormGradArgs a, int parts, int type) {
    __shared__ float t[16][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    int k = 0;
    for (; k < kNormSums; ++k)
        if (a.dparam[k].p && a.place[k] == (int)blockIdx.y) break;
    float s = 0.0f;
    if (c < a.f.d) {
        const float* p = a.part + (size_t)blockIdx.y * parts * a.f.d + c;
#pragma unroll 8
        for (int i = wv; i < parts; i += 16) s += p[(size_t)i * a.f.d];
    }
    t[wv][lane] = s;
    __syncthreads();
    if (wv || c >= a.f.d) return;
    for (int w = 1; w < 16; ++w) s += t[w][lane];
    const NormSum& o = a.dparam[k];
    if (o.f32) ((float*)o.p)[c] = s;
    else ((uint16_t*)o.p)[c] = (uint16_t)(type == kBf16 ? to16<kBf16>(s) : to16<kF16>(s));
}

// Lanes of a row and eights of a lane, by the width.
struct Shape {
    int mode, v, threads, rows;         // rows of a workgroup
};

Shape norm_shape(int d) {
    if (d <= 128) return {kSub, 1, 256, 16};
    if (d <= 512) return {kWave, 1, 256, 4};
    if (d <= 1024) return {kWave, 2, 256, 4};
    const int v = d <= 8192 ? 1 : d <= 16384 ? 2 : 4;
    return {kBlock, v, (d + 512 * v - 1) / (512 * v) * 64, 1};
}

template <int T, typename F>
void with_shape(const Shape& s, F f) {
    using std::integral_constant;
    if (s.mode == kSub) f(integral_constant<int, kSub>(), integral_constant<int, 1>());
    else if (s.mode == kWave && s.v == 1) f(integral_constant<int, kWave>(), integral_constant<int, 1>());
    else if (s.mode == kWave) f(integral_constant<int, kWave>(), integral_constant<int, 2>());
    else if (s.v == 1) f(integral_constant<int, kBlock>(), integral_constant<int, 1>());
    else if (s.v == 2) f(integral_constant<int, kBlock>(), integral_constant<int, 2>());
    else f(integral_constant<int, kBlock>(), integral_constant<int, 4>());
}

template <int T>
void forward(const NormArgs& a, hipStream_t s) {
    const Shape sh = norm_shape(a.d);
    const dim3 grid((a.rows + sh.rows - 1) / sh.rows), block(sh.threads);
    with_shape<T>(sh, [&](auto mode, auto v) {
        hipLaunchKernelGGL((norm_kernel<T, decltype(mode)::value, decltype(v)::value>), grid, block, 0, s, a);
    });
}

// Workgroups of a gradient, each of which leaves a part of the channels' sums.
int norm_parts(int rows, int d) {
    const int r = norm_shape(d).rows, all = (rows + r - 1) / r;
    return all < 2 * kCUs ? all : 2 * kCUs;
}

template <int T>
void backward(const NormGradArgs& a, int sums, hipStream_t s) {
    const Shape sh = norm_shape(a.f.d);
    const int parts = norm_parts(a.f.rows, a.f.d);
    with_shape<T>(sh, [&](auto mode, auto v) {
        constexpr int M = decltype(mode)::value, V = decltype(v)::value;
        if (sums) hipLaunchKernelGGL((norm_bwd_kernel<T, M, V, true>), dim3(parts), dim3(sh.threads), 0, s, a);
        else hipLaunchKernelGGL((norm_bwd_kernel<T, M, V, false>), dim3(parts), dim3(sh.threads), 0, s, a);
    });
    if (sums)
        hipLaunchKernelGGL(norm_sums_kernel, dim3((a.f.d + 63) / 64, sums), dim3(1024), 0, s, a, parts, T);
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, int type, hipStream_t s) {
    if (type == kBf16) forward<kBf16>(a, s);
    else forward<kF16>(a, s);
    return hipGetLastError();
}

size_t norm_bwd_ws_bytes(int rows, int d, int sums) {
    return rows ? (size_t)norm_parts(rows, d) * d * 4 * sums : 0;
}

hipError_t launch_norm_bwd(NormGradArgs a, int type, void* ws, hipStream_t s) {
    a.part = (float*)ws;
    int sums = 0;
    for (int k = 0; k < kNormSums; ++k)
        if (a.dparam[k].p) a.place[k] = sums++;
    if (type == kBf16) backward<kBf16>(a, sums, s);
    else backward<kF16>(a, sums, s);
    return hipGetLastError();
}

}  // namespace xtq
