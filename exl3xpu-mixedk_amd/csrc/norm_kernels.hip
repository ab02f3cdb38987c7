// norm_kernels.hip -- norms of rows, and the residual sum between two blocks with
// the norms before and after it, its gate and its scale; with their gradients.
//
// Of a block's result x, its residual r, gate g and scale s,
//   p = post norm of x (or x),  q = p ga(g),  y = r + s q,  h = norm of y,
// the norm of t being (t - mean) / sqrt(mean (t - mean)^2 + eps) w + b, without its
// mean for "rms".  The plain norm is h of y = x.  h comes of y before it is rounded.
//
// A row's group of lanes (16, 32, a wave or a workgroup, by the width alone, so that a
// row's result does not depend on how many there are) holds the row in registers:
// every input is read once, deviations are squared around the mean itself.
#include "operators.h"

#pragma clang fp contract(off)

namespace xtq {
namespace {

// Rows of 16 lanes (four a wave), of 32, of a wave, of a workgroup.
enum Mode { kSub, kHalf, kWave, kBlock };
constexpr int lanes_of(int mode) { return mode == kSub ? 16 : mode == kHalf ? 32 : 64; }
// Rows that a workgroup has at a time.
constexpr int rows_of(int mode) { return mode == kBlock ? 1 : 256 / lanes_of(mode); }

// Waves that share a row at most: three a SIMD, whose 168 registers hold, of a
// gradient, most of eight channels' parameters and sums and two rows' inputs.  With the
// channels' sums a workgroup's gradient keeps 6 registers a lane in scratch where there
// is a gate, 48 where there are means or biases too (8191 rows of 5120 with everything,
// forward and back: 270 us without biases, 438 with), and 6 to 14 with those alone; the
// forward pass of rows wider than 24576, six eights a lane, 64 or 65 (2000 rows with
// everything: of 24576 144 us, of 32768 334; the plain norm 47 and 70).
constexpr int kRowWaves = 12;

template <int T>
__device__ __forceinline__ void unpack(u4 w, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = from16<T>(w[i] & 0xFFFFu);
        v[2 * i + 1] = from16<T>(w[i] >> 16);
    }
}

// Eight values of a row from column `col` on, on their way: every lane loads 16 bytes
// inside the row, those at its end where its own reach past it, and in_place brings
// them home once they are there.  (A load under a condition is waited for where the
// branches meet: a residual's norm of 8191 rows of 5120 and its gradient took 316 us so,
// and 302 without.)
template <int MODE>
__device__ __forceinline__ u4 load8(const uint16_t* row, int col, int d) {
    if (MODE != kSub || d >= 8) return *(const u4_a2*)(row + (col < d - 8 ? col : d - 8));
    u4 w = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 1; i < 8; ++i)
        if (8 - i <= d) w[i >> 1] |= (uint32_t)row[d - 8 + i] << (16 * (i & 1));
    return w;
}

// The `n` last of eight values (all for 8 and more, none for less than 1) to the
// front, zeros behind them.
__device__ __forceinline__ void in_place(u4& w, int n) {
    if (n >= 8) return;
    const int by = 16 * (8 - (n > 0 ? n : 0));
    uint64_t lo = (uint64_t)w[0] | (uint64_t)w[1] << 32, hi = (uint64_t)w[2] | (uint64_t)w[3] << 32;
    lo = by >= 128 ? 0 : by >= 64 ? hi >> (by - 64) : lo >> by | hi << (64 - by);
    hi = by >= 64 ? 0 : hi >> by;
    w = (u4){(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
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

// Eight channels of a parameter (of the rows' type or fp32) from `col` on, `missing`
// where there is none.  Those past the end are any numbers.
template <int T, int MODE>
__device__ __forceinline__ void param8(const NormParam& p, int col, int d, float missing, float* v) {
    if (!p.p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = missing;
    } else if (!p.f32) {
        u4 w = load8<MODE>((const uint16_t*)p.p, col, d);
        in_place(w, d - col);
        unpack<T>(w, v);
    } else if (d & 7) {
        const float* f = (const float*)p.p;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = f[col + i < d ? col + i : d - 1];
    } else {
        const float* f = (const float*)p.p + (col < d ? col : 0);
        const f4 a = *(const f4_a4*)f, b = *(const f4_a4*)(f + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    }
}

// Gate's factor, and its slope.  s (1 - s) comes without the difference, which loses
// s's neighbourhood of 1.
__device__ __forceinline__ void gate_at(float g, int act, float& value, float& slope) {
    value = g;
    slope = 1.0f;
    if (act == kGateNone) return;
    const float e = fast_exp(-fabsf(g)), r = fast_rcp(1.0f + e), s = g < 0.0f ? e * r : r, t = e * r * r;
    value = act == kGateSigmoid ? s : g * s;
    slope = act == kGateSigmoid ? t : __builtin_fmaf(g, t, s);
}

// Sum over 16 lanes, over 32 and over the wave.
__device__ __forceinline__ float sum16(float v) {
    v += lane_xor<1>(v);
    v += lane_xor<2>(v);
    v += dpp<0x141>(v);
    v += dpp<0x140>(v);
    return v;
}

__device__ __forceinline__ float sum32(float v) {
    const uint32_t b = __float_as_uint(sum16(v));
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float sum64(float v) {
    const uint32_t b = __float_as_uint(sum32(v));
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sums over a row's lanes.  A workgroup's waves meet in LDS, one barrier a sum: two
// places in turn, and who comes to write a place again has met, in between, all
// who read it.
template <int MODE>
struct Group {
    int lane, width, turn = 0;          // the row's lane and lanes
    __device__ Group() {
        lane = MODE == kBlock ? threadIdx.x : threadIdx.x & (lanes_of(MODE) - 1);
        width = MODE == kBlock ? blockDim.x : lanes_of(MODE);
    }
    template <int N>
    __device__ __forceinline__ void sum(float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] = MODE == kSub ? sum16(v[i]) : MODE == kHalf ? sum32(v[i]) : sum64(v[i]);
        if constexpr (MODE == kBlock) {
            __shared__ float part[2][N][16];
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
            for (int i = 0; i < 8; ++i) s += (v * g.width + g.lane) * 8 + i < d ? t[v][i] : 0.0f;
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
__global__ __launch_bounds__(MODE == kBlock ? 64 * kRowWaves : 256) void norm_kernel(NormArgs a) {
    Group<MODE> g;
    const int row = blockIdx.x * rows_of(MODE) + (MODE == kBlock ? 0 : threadIdx.x / lanes_of(MODE));
    const bool in = row < a.rows;
    const size_t at = in ? row : 0;
    int col[V], n[V];
    u4 wx[V], wr[V], wg[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        col[v] = (v * g.width + g.lane) * 8;
        n[v] = in ? a.d - col[v] : 0;
        wx[v] = load8<MODE>(a.x + at * a.x_stride, col[v], a.d);
        if (a.res) wr[v] = load8<MODE>(a.res + at * a.res_stride, col[v], a.d);
        if (a.gate) wg[v] = load8<MODE>(a.gate + at * a.gate_stride, col[v], a.d);
    }
    float t[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        in_place(wx[v], n[v]);
        unpack<T>(wx[v], t[v]);
    }
    float mean, rstd;
    f4 stats = {0.0f, 1.0f, 0.0f, 1.0f};
    if (a.post) {
        row_stats<MODE, V>(g, t, a.d, a.post, a.post_eps, mean, rstd);
        stats[0] = mean;
        stats[1] = rstd;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float w[8], b[8];
            param8<T, MODE>(a.post_weight, col[v], a.d, 1.0f, w);
            param8<T, MODE>(a.post_bias, col[v], a.d, 0.0f, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) t[v][i] = (t[v][i] - mean) * rstd * w[i] + b[i];
        }
    }
    if (a.res) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float s[8], r[8];
            param8<T, MODE>(a.scale, col[v], a.d, a.scale_number, s);
            in_place(wr[v], n[v]);
            unpack<T>(wr[v], r);
            if (a.gate) {
                float e[8], slope;
                in_place(wg[v], n[v]);
                unpack<T>(wg[v], e);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    gate_at(e[i], a.gate_act, e[i], slope);
                    t[v][i] *= e[i];
                }
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
            param8<T, MODE>(a.weight, col[v], a.d, 1.0f, w);
            param8<T, MODE>(a.bias, col[v], a.d, 0.0f, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) t[v][i] = (t[v][i] - mean) * rstd * w[i] + b[i];
            if (n[v] > 0) store8<T>(a.h + at * a.h_stride + col[v], n[v], t[v]);
        }
    }
    if (a.stats && in && g.lane == 0) *(f4*)(a.stats + 4 * at) = stats;
}

// Parameters of eight channels, as a gradient's rows use them.
struct Channels {
    float w[8], s[8], pw[8], pb[8];
};

// What a gradient is of: the plain norm, a residual sum, one with a gate.
enum GradOf { kPlain, kResidual, kWithGate };

template <int T, int MODE, int OF>
__device__ __forceinline__ void load_channels(Channels& c, const NormArgs& a, int col) {
    param8<T, MODE>(a.weight, col, a.d, 1.0f, c.w);
    if constexpr (OF != kPlain) {
        param8<T, MODE>(a.scale, col, a.d, a.scale_number, c.s);
        param8<T, MODE>(a.post_weight, col, a.d, 1.0f, c.pw);
        param8<T, MODE>(a.post_bias, col, a.d, 0.0f, c.pb);
    }
    // (past the row's end zeros: an infinite one would make NaN of the zeros there)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (col + i < a.d) continue;
        c.w[i] = 0.0f;
        if constexpr (OF != kPlain) c.s[i] = c.pw[i] = c.pb[i] = 0.0f;
    }
}

// Eight channels of a row's inputs.
struct Raw {
    u4 x, r, g, y, h;
};

template <int MODE, int OF>
__device__ __forceinline__ void load_raw(Raw& t, const NormGradArgs& a, size_t at, int col) {
    const u4 zero = {0u, 0u, 0u, 0u};
    t.x = load8<MODE>(a.f.x + at * a.f.x_stride, col, a.f.d);
    t.h = a.dh ? load8<MODE>(a.dh + at * a.dh_stride, col, a.f.d) : zero;
    if constexpr (OF != kPlain) {
        t.r = load8<MODE>(a.f.res + at * a.f.res_stride, col, a.f.d);
        t.y = a.dy ? load8<MODE>(a.dy + at * a.dy_stride, col, a.f.d) : zero;
    }
    if constexpr (OF == kWithGate) t.g = load8<MODE>(a.f.gate + at * a.f.gate_stride, col, a.f.d);
}

template <int OF>
__device__ __forceinline__ void raw_in_place(Raw& t, int n) {
    in_place(t.x, n);
    in_place(t.h, n);
    if constexpr (OF != kPlain) {
        in_place(t.r, n);
        in_place(t.y, n);
    }
    if constexpr (OF == kWithGate) in_place(t.g, n);
}

// Tells the compiler nothing of what the inputs are, so that what was computed of
// them before is not kept in registers until it is needed once more.
template <int OF>
__device__ __forceinline__ void forget(Raw& t) {
    asm volatile("" : "+v"(t.x), "+v"(t.h));
    if constexpr (OF != kPlain) asm volatile("" : "+v"(t.r), "+v"(t.y));
    if constexpr (OF == kWithGate) asm volatile("" : "+v"(t.g));
}

// i-th of eight values.
template <int T>
__device__ __forceinline__ float pick(const u4& w, int i) {
    return from16<T>(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xFFFFu);
}

// Eight gates' factors and slopes.
struct Gate {
    float ga[8], slope[8];
};

template <int T, int OF>
__device__ __forceinline__ void gates(Gate& e, const Raw& t, int act) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        e.ga[i] = e.slope[i] = 1.0f;
        if constexpr (OF == kWithGate) gate_at(pick<T>(t.g, i), act, e.ga[i], e.slope[i]);
    }
}

// What a row's i-th channel is forward: x^, p, q, t^, and c = dh w.  (A norm that is
// not there has mean 0 and factor 1.)  FULL: with means and biases.  Without them, "rms"
// alone, a gradient has a tenth less to work out (the same call without biases, 8191 rows
// of 5120, forward and back: with gate, scale and two norms 287 us with their code, 274
// without; two norms 199 and 182.  A call that has them takes 438 and 295).
struct Forward {
    float hat, p, q, that, dh, c;
};

template <int T, int OF, bool FULL>
__device__ __forceinline__ Forward again(const Raw& t, int i, const Gate& e, const Channels& ch, const f4& stats) {
    Forward f;
    f.p = pick<T>(t.x, i);
    f.that = f.p;
    if constexpr (OF != kPlain) {
        f.hat = (FULL ? f.p - stats[0] : f.p) * stats[1];
        f.p = FULL ? __builtin_fmaf(f.hat, ch.pw[i], ch.pb[i]) : f.hat * ch.pw[i];
        f.q = OF == kWithGate ? f.p * e.ga[i] : f.p;
        f.that = __builtin_fmaf(ch.s[i], f.q, pick<T>(t.r, i));
    }
    f.that = (FULL ? f.that - stats[2] : f.that) * stats[3];
    f.dh = pick<T>(t.h, i);
    f.c = f.dh * ch.w[i];
    return f;
}

// Sums of eight channels over rows, of the norm and of the rest.
template <int OF, bool FULL>
struct Sums {
    static constexpr int N = OF == kPlain ? 2 : kNormSums;
    static constexpr bool has(int k) { return k < N && (FULL || (k != kSumBias && k != kSumPostBias)); }
    float of[N][8];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) of[k][i] = 0.0f;
    }
    __device__ __forceinline__ void norm(int i, const Forward& f, bool dh) {
        of[kSumWeight][i] = __builtin_fmaf(f.dh, dh ? f.that : 0.0f, of[kSumWeight][i]);
        if constexpr (FULL) of[kSumBias][i] += f.dh;
    }
    __device__ __forceinline__ void rest(int i, const Forward& f, float dt, float dp) {
        of[kSumScale][i] = __builtin_fmaf(dt, f.q, of[kSumScale][i]);
        of[kSumPostWeight][i] = __builtin_fmaf(dp, f.hat, of[kSumPostWeight][i]);
        if constexpr (FULL) of[kSumPostBias][i] += dp;
    }
};

// dy' of a channel; `in`: of h's gradient too.
template <int T, int OF, bool FULL>
__device__ __forceinline__ float total(const Forward& f, const Raw& t, int i, const f4& stats, float c1, float c2,
                                       bool in) {
    const float dy = OF == kPlain ? 0.0f : pick<T>(t.y, i), part = __builtin_fmaf(-c1, f.that, f.c);
    return in ? __builtin_fmaf(stats[3], FULL ? part - c2 : part, dy) : dy;
}

// Gradients.  With c = dh w, t^ = (y - mean) rstd,
//   dy' = dy + rstd (c - t^ mean(c t^) - mean(c))       (the last for "layer"),
//   dres = dy',  ds = sum of dy' q,  dgate = dy' s p ga'(g),  dp = dy' s ga(g),
// and dx from dp as dy' from dh.  y and the norms are computed anew from the inputs
// and the rows' saved means and factors, so nothing of y's rounding enters.
//
// Rows of one eight a lane: a group goes through its rows with the parameters and
// (SUMS) the channels' sums in registers, a row's inputs on their way while the row
// before is worked on, and a workgroup leaves one row of partial sums, which
// norm_sums_kernel adds in order.  What a sum over the row needs again after it is
// computed anew, which costs less than registers for it.
template <int T, int MODE, int OF, bool SUMS, bool FULL>
__global__ __launch_bounds__(MODE == kBlock ? 64 * kRowWaves : 256) void norm_bwd_kernel(NormGradArgs a) {
    Group<MODE> g;
    constexpr int R = rows_of(MODE);
    const int sub = MODE == kBlock ? 0 : threadIdx.x / lanes_of(MODE);
    const int d = a.f.d, step = gridDim.x * R, col = g.lane * 8;
    const float inv = 1.0f / (float)d;
    struct Row {
        Raw raw;
        f4 stats;
    };
    auto load = [&](Row& t, int row) {
        const size_t at = row < a.f.rows ? row : 0;
        t.stats = *(const f4*)(a.f.stats + 4 * at);
        if (row >= a.f.rows) t.stats = (f4){0.0f, 0.0f, 0.0f, 0.0f};     // (the first row's may be infinite)
        load_raw<MODE, OF>(t.raw, a, at, col);
    };
    Sums<OF, FULL> sums;
    if constexpr (SUMS) sums.clear();
    Channels ch;
    Row next;
    load(next, blockIdx.x * R + sub);
    load_channels<T, MODE, OF>(ch, a.f, col);
    for (int base = blockIdx.x * R; base < a.f.rows; base += step) {
        const int row = base + sub, n = row < a.f.rows ? d - col : 0, nh = a.dh ? n : 0;
        const size_t at = row < a.f.rows ? row : 0;
        Row now = next;
        if (base + step < a.f.rows) load(next, row + step);
        Gate gate;
        float two[2] = {0.0f, 0.0f};
        raw_in_place<OF>(now.raw, n);
        gates<T, OF>(gate, now.raw, a.f.gate_act);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const Forward f = again<T, OF, FULL>(now.raw, i, gate, ch, now.stats);
            two[0] = __builtin_fmaf(f.c, f.that, two[0]);
            if constexpr (FULL) two[1] += f.c;
            if constexpr (SUMS) sums.norm(i, f, a.dh);
        }
        float c1 = 0.0f, c2 = 0.0f;
        if (a.dh) {
            g.sum(two);
            c1 = two[0] * inv;
            if (a.f.kind == kNormLayer) c2 = two[1] * inv;
        }
        two[0] = two[1] = 0.0f;
        forget<OF>(now.raw);
        float dt[8], dg[8], dp[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            Forward f = again<T, OF, FULL>(now.raw, i, gate, ch, now.stats);
            dt[i] = total<T, OF, FULL>(f, now.raw, i, now.stats, c1, c2, i < nh);
            dp[i] = dt[i];
            if constexpr (OF != kPlain) {
                const float ds = dt[i] * ch.s[i];
                float to = OF == kWithGate ? ds * gate.ga[i] : ds;
                // (where there is no row an infinite parameter makes NaN of its zeros)
                if (MODE != kBlock && row >= a.f.rows) f.q = to = 0.0f;
                dg[i] = ds * f.p * gate.slope[i];
                if constexpr (SUMS) sums.rest(i, f, dt[i], to);
                dp[i] = to * ch.pw[i];
                two[0] = __builtin_fmaf(dp[i], f.hat, two[0]);
                if constexpr (FULL) two[1] += dp[i];
            }
        }
        if constexpr (OF != kPlain)
            if (a.dres && n > 0) store8<T>(a.dres + at * d + col, n, dt);
        if constexpr (OF == kWithGate)
            if (a.dgate && n > 0) store8<T>(a.dgate + at * d + col, n, dg);
        if (OF != kPlain && a.f.post) {
            g.sum(two);
            const float e1 = two[0] * inv, e2 = a.f.post == kNormLayer ? two[1] * inv : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = pick<T>(now.raw.x, i), hat = (FULL ? x - now.stats[0] : x) * now.stats[1];
                const float part = __builtin_fmaf(-e1, hat, dp[i]);
                dp[i] = now.stats[1] * (FULL ? part - e2 : part);
            }
        }
        if (a.dx && n > 0) store8<T>(a.dx + at * d + col, n, dp);
    }
    if constexpr (SUMS) {
        // [sum][workgroup][d]
        __shared__ float join[MODE == kBlock ? 1 : 256 * 8];
#pragma unroll
        for (int k = 0; k < Sums<OF, FULL>::N; ++k) {
            if (!Sums<OF, FULL>::has(k) || !a.dparam[k].p) continue;
            float* out = a.part + ((size_t)a.place[k] * gridDim.x + blockIdx.x) * d;
            if constexpr (MODE != kBlock) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; ++i) join[i * 256 + threadIdx.x] = sums.of[k][i];
                __syncthreads();
                if (sub != 0) continue;
                for (int o = 1; o < R; ++o)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sums.of[k][i] += join[i * 256 + threadIdx.x + o * g.width];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (col + i < d) out[col + i] = sums.of[k][i];
        }
    }
}

// Wider rows do not stay in registers, and are read twice.  First all that a row's
// gradients take of the whole row: with u = s ga(g) w' (w' the post norm's weight) and
// x^ the post norm before it, dp = u dy', so that dx's sums over the row of u x^ dy' and
// u dy' are, dy' being linear in them, combinations of sums that need no other first.
// (2000 rows with everything, forward and back: of 17408 313 us, 483 with a lane's three
// eights kept in registers, of 32768 685 and 1953; of 6144, a lane's one, 95.)
constexpr int kWideWaves = 8;

template <int T, int OF, bool FULL>
__global__ __launch_bounds__(64 * kWideWaves) void norm_rows_kernel(NormGradArgs a) {
    constexpr int N = OF == kPlain ? 2 : 10;
    Group<kBlock> g;
    const int d = a.f.d;
    const float inv = 1.0f / (float)d;
    for (int row = blockIdx.x; row < a.f.rows; row += gridDim.x) {
        const f4 stats = *(const f4*)(a.f.stats + 4 * (size_t)row);
        float v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = 0.0f;
        Raw next;
        load_raw<kBlock, OF>(next, a, row, g.lane * 8);
        for (int col = g.lane * 8; col < d; col += 512 * kWideWaves) {
            Raw now = next;
            load_raw<kBlock, OF>(next, a, row, col + 512 * kWideWaves);
            Channels ch;
            load_channels<T, kBlock, OF>(ch, a.f, col);
            raw_in_place<OF>(now, d - col);
            Gate gate;
            gates<T, OF>(gate, now, a.f.gate_act);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const Forward f = again<T, OF, FULL>(now, i, gate, ch, stats);
                v[0] = __builtin_fmaf(f.c, f.that, v[0]);
                if constexpr (FULL) v[1] += f.c;
                if constexpr (OF != kPlain) {
                    const float dy = pick<T>(now.y, i), u = ch.s[i] * gate.ga[i] * ch.pw[i], uh = u * f.hat;
                    v[2] = __builtin_fmaf(uh, dy, v[2]);
                    v[3] = __builtin_fmaf(uh, f.c, v[3]);
                    v[4] = __builtin_fmaf(uh, f.that, v[4]);
                    if constexpr (FULL) {
                        v[5] += uh;
                        v[6] = __builtin_fmaf(u, dy, v[6]);
                        v[7] = __builtin_fmaf(u, f.c, v[7]);
                        v[8] = __builtin_fmaf(u, f.that, v[8]);
                        v[9] += u;
                    }
                }
            }
        }
        g.sum(v);
        f4 m = {0.0f, 0.0f, 0.0f, 0.0f};
        if (a.dh) {
            m[0] = v[0] * inv;
            if (a.f.kind == kNormLayer) m[1] = v[1] * inv;
        }
        if constexpr (OF != kPlain) {
            if (a.f.post) m[2] = (v[2] + (a.dh ? stats[3] * (v[3] - m[0] * v[4] - m[1] * v[5]) : 0.0f)) * inv;
            if (a.f.post == kNormLayer) m[3] = (v[6] + (a.dh ? stats[3] * (v[7] - m[0] * v[8] - m[1] * v[9]) : 0.0f)) * inv;
        }
        if (threadIdx.x == 0) *(f4*)(a.means + 4 * (size_t)row) = m;
    }
}

// Then the gradients, with the channels' sums beside: a workgroup takes 2048 channels
// of every gridDim.y-th row and leaves a part of the sums.
template <int T, int OF, bool FULL>
__global__ __launch_bounds__(256) void norm_wide_kernel(NormGradArgs a) {
    const int d = a.f.d, col = (blockIdx.x * 256 + threadIdx.x) * 8, n = d - col;
    if (n <= 0) return;
    Channels ch;
    load_channels<T, kBlock, OF>(ch, a.f, col);
    Sums<OF, FULL> sums;
    sums.clear();
    Raw next;
    load_raw<kBlock, OF>(next, a, blockIdx.y, col);
    for (int row = blockIdx.y; row < a.f.rows; row += gridDim.y) {
        Raw now = next;
        const f4 stats = *(const f4*)(a.f.stats + 4 * (size_t)row), m = *(const f4*)(a.means + 4 * (size_t)row);
        if (row + (int)gridDim.y < a.f.rows) load_raw<kBlock, OF>(next, a, row + gridDim.y, col);
        raw_in_place<OF>(now, n);
        Gate gate;
        gates<T, OF>(gate, now, a.f.gate_act);
        float dt[8], dg[8], dp[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const Forward f = again<T, OF, FULL>(now, i, gate, ch, stats);
            sums.norm(i, f, a.dh);
            dt[i] = total<T, OF, FULL>(f, now, i, stats, m[0], m[1], a.dh && i < n);
            dp[i] = dt[i];
            if constexpr (OF != kPlain) {
                const float ds = dt[i] * ch.s[i], to = OF == kWithGate ? ds * gate.ga[i] : ds;
                dg[i] = ds * f.p * gate.slope[i];
                sums.rest(i, f, dt[i], to);
                dp[i] = to * ch.pw[i];
                if (a.f.post) dp[i] = stats[1] * (dp[i] - f.hat * m[2] - m[3]);
            }
        }
        const size_t at = (size_t)row * d + col;
        if constexpr (OF != kPlain)
            if (a.dres) store8<T>(a.dres + at, n, dt);
        if constexpr (OF == kWithGate)
            if (a.dgate) store8<T>(a.dgate + at, n, dg);
        if (a.dx) store8<T>(a.dx + at, n, dp);
    }
#pragma unroll
    for (int k = 0; k < Sums<OF, FULL>::N; ++k) {
        if (!Sums<OF, FULL>::has(k) || !a.dparam[k].p) continue;
        float* out = a.part + ((size_t)a.place[k] * gridDim.y + blockIdx.y) * d;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) out[col + i] = sums.of[k][i];
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

// Lanes of a row and eights of a lane, by the width.  A workgroup's lanes have two
// eights each forward, whose loads are then half as many workgroups' (8191 rows of 5120
// with everything 94 us, 108 with one; one row 0.8 us more), and one for a gradient.
struct Shape {
    int mode, v, threads;
};

constexpr int kWide = 512 * kRowWaves;          // rows wider than this have no one eight a lane

Shape norm_shape(int d, bool gradient) {
    if (d <= 512) return {d <= 128 ? kSub : d <= 256 ? kHalf : kWave, 1, 256};
    int v = d <= 4 * kWide ? (d + kWide - 1) / kWide : 6;
    if (!gradient && v == 1) v = 2;
    return {kBlock, v, (d + 512 * v - 1) / (512 * v) * 64};
}

template <typename F>
void with_shape(const Shape& s, F f) {
    using std::integral_constant;
    if (s.mode == kSub) f(integral_constant<int, kSub>(), integral_constant<int, 1>());
    else if (s.mode == kHalf) f(integral_constant<int, kHalf>(), integral_constant<int, 1>());
    else if (s.mode == kWave) f(integral_constant<int, kWave>(), integral_constant<int, 1>());
    else if (s.v == 1) f(integral_constant<int, kBlock>(), integral_constant<int, 1>());
    else if (s.v == 2) f(integral_constant<int, kBlock>(), integral_constant<int, 2>());
    else if (s.v == 3) f(integral_constant<int, kBlock>(), integral_constant<int, 3>());
    else if (s.v == 4) f(integral_constant<int, kBlock>(), integral_constant<int, 4>());
    else f(integral_constant<int, kBlock>(), integral_constant<int, 6>());
}

// A grid has less than 2^32 lanes: so many workgroups, of kRowWaves waves at most, a launch.
constexpr int kMostGroups = 1 << 22;

template <int T>
void forward(NormArgs a, hipStream_t s) {
    const Shape sh = norm_shape(a.d, false);
    const int all = (a.rows + rows_of(sh.mode) - 1) / rows_of(sh.mode), rows = kMostGroups * rows_of(sh.mode);
    for (int at = 0; at < all; at += kMostGroups) {
        const dim3 grid(all - at < kMostGroups ? all - at : kMostGroups), block(sh.threads);
        with_shape(sh, [&](auto mode, auto v) {
            constexpr int M = decltype(mode)::value, V = decltype(v)::value;
            if constexpr (M != kBlock || V > 1) hipLaunchKernelGGL((norm_kernel<T, M, V>), grid, block, 0, s, a);
        });
        a.rows -= rows;
        a.x += rows * a.x_stride;
        a.res += a.res ? rows * a.res_stride : 0;
        a.gate += a.gate ? rows * a.gate_stride : 0;
        a.y += a.y ? rows * a.y_stride : 0;
        a.h += a.h ? rows * a.h_stride : 0;
        a.stats += a.stats ? 4 * (size_t)rows : 0;
    }
}

// A gradient's workgroups, and the parts of the channels' sums: as many of either as
// are on the compute units at once, by their waves.
struct NormPlan {
    int groups, parts;
    size_t means, total;
};

NormPlan norm_plan(int rows, int d, int sums) {
    const Shape sh = norm_shape(d, true);
    NormPlan p;
    const int all = (rows + rows_of(sh.mode) - 1) / rows_of(sh.mode);
    const int most = d > kWide ? kMostGroups : kRowWaves / (sh.threads / 64) * kCUs;
    p.groups = all < most ? all : most;
    p.parts = p.groups;
    if (d > kWide) {
        const int fill = kRowWaves / 4 * kCUs / ((d + 2047) / 2048);
        p.parts = rows < fill ? rows : fill;
    }
    p.means = ((size_t)sums * p.parts * d * 4 + 255) & ~(size_t)255;
    p.total = p.means + (d > kWide ? (size_t)rows * 16 : 0);
    return p;
}

template <int T, int OF, bool FULL>
void backward_of(const NormGradArgs& a, const NormPlan& p, bool sums, hipStream_t s) {
    const Shape sh = norm_shape(a.f.d, true);
    if (a.f.d > kWide) {
        hipLaunchKernelGGL((norm_rows_kernel<T, OF, FULL>), dim3(p.groups), dim3(64 * kWideWaves), 0, s, a);
        hipLaunchKernelGGL((norm_wide_kernel<T, OF, FULL>), dim3((a.f.d + 2047) / 2048, p.parts), dim3(256), 0, s, a);
        return;
    }
    auto launch = [&](auto mode) {
        constexpr int M = decltype(mode)::value;
        auto* kernel = sums ? norm_bwd_kernel<T, M, OF, true, FULL> : norm_bwd_kernel<T, M, OF, false, FULL>;
        hipLaunchKernelGGL(kernel, dim3(p.groups), dim3(sh.threads), 0, s, a);
    };
    if (sh.mode == kSub) launch(std::integral_constant<int, kSub>());
    else if (sh.mode == kHalf) launch(std::integral_constant<int, kHalf>());
    else if (sh.mode == kWave) launch(std::integral_constant<int, kWave>());
    else launch(std::integral_constant<int, kBlock>());
}

template <int T>
void backward(const NormGradArgs& a, const NormPlan& p, int sums, hipStream_t s) {
    const bool full = a.f.post_bias.p || a.dparam[kSumBias].p || a.dparam[kSumPostBias].p || a.f.kind == kNormLayer ||
                      a.f.post == kNormLayer;
    auto of = [&](auto what) {
        constexpr int OF = decltype(what)::value;
        if (full) backward_of<T, OF, true>(a, p, sums > 0, s);
        else backward_of<T, OF, false>(a, p, sums > 0, s);
    };
    if (!a.f.res) of(std::integral_constant<int, kPlain>());
    else if (!a.f.gate) of(std::integral_constant<int, kResidual>());
    else of(std::integral_constant<int, kWithGate>());
    if (sums)
        hipLaunchKernelGGL(norm_sums_kernel, dim3((a.f.d + 63) / 64, sums), dim3(1024), 0, s, a, p.parts, T);
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, int type, hipStream_t s) {
    if (type == kBf16) forward<kBf16>(a, s);
    else forward<kF16>(a, s);
    return hipGetLastError();
}

size_t norm_bwd_ws_bytes(int rows, int d, int sums) { return rows ? norm_plan(rows, d, sums).total : 0; }

hipError_t launch_norm_bwd(NormGradArgs a, int type, void* ws, hipStream_t s) {
    int sums = 0;
    for (int k = 0; k < kNormSums; ++k)
        if (a.dparam[k].p) a.place[k] = sums++;
    const NormPlan p = norm_plan(a.f.rows, a.f.d, sums);
    a.part = (float*)ws;
    a.means = (float*)((uint8_t*)ws + p.means);
    if (type == kBf16) backward<kBf16>(a, p, sums, s);
    else backward<kF16>(a, p, sums, s);
    return hipGetLastError();
}

}  // namespace xtq
