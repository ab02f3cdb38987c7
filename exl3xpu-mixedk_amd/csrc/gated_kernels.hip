// gated_kernels.hip -- the gated projection act(x Wg + bg) (x Wu + bu) on two trellis
// weights for many rows, and its gradient.
//
// Forward: the columns of both weights lie in one operand, 128 of gate beside 128 of
// up, so that a tile of 256 columns holds both factors of 128 results: its waves hand
// each other what they need in LDS, and only the product leaves.  Each weight has its
// own row signs and scales, so the rows come in two transforms, and a wave reads that
// of its own weight.
//
// Gradient: with dg = dy zu act'(zg), du = dy act(zg), dx = dg Wg^T + du Wu^T is one
// product over both weights' columns one after the other, in parts that lie in one
// weight each: the parts are transformed apart and added.
#include "few_device.h"
#include "product_device.h"

#pragma clang fp contract(off)

namespace xtq {
namespace {

// ------------------------------------------------------------------ operands
// Rows for both weights: x times each one's row signs, or (GRAD) dg and du, of dy and
// z, times each one's column scales.
struct PairRows {
    const uint16_t* v;                  // x or dy
    long long stride;
    const float* z;                     // [2][rows][cols] (GRAD)
    const uint16_t* scale[2];           // fp16 per column
    int type, act, rows, cols;
};

// Eight values of a row for each weight, before the scales.
template <bool GRAD>
__device__ __forceinline__ void load_pair8(const PairRows& s, size_t row, int col, float* a, float* b) {
    unpack8(*(const u4_a2*)(s.v + row * (size_t)s.stride + col), s.type, a);
    if constexpr (GRAD) {
        const float* zg = s.z + row * (size_t)s.cols + col;
        const float* zu = zg + (size_t)s.rows * s.cols;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f4 g = *(const f4_a4*)(zg + 4 * h), u = *(const f4_a4*)(zu + 4 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float value, slope;
                act_and_slope(g[i], s.act, value, slope);
                b[4 * h + i] = a[4 * h + i] * value;
                a[4 * h + i] *= u[i] * slope;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = a[i];
    }
}

__device__ __forceinline__ void scale_pair8(const uint16_t* scale, int col, float* v) {
    float c[8];
    unpack8(*(const u4_a2*)(scale + col), kF16, c);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= c[i];
}

// As row_exponents of linear_kernels.hip, for both weights at once: to [weight][places].
// (2048 rows of 17408 read 356 MB in 115 us; other orders of the columns, more loads in
// flight and z in the matrix cores' layout took as long.)
template <bool GRAD>
__device__ __forceinline__ void pair_exponents(const PairRows& s, int row, int32_t* __restrict__ shift,
                                               int32_t* __restrict__ rowexp, int places) {
    __shared__ float part[2][4];
    float top[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x * 8; c < s.cols; c += 2048) {
        float v[2][8];
        load_pair8<GRAD>(s, row, c, v[0], v[1]);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            scale_pair8(s.scale[n], c, v[n]);
#pragma unroll
            for (int i = 0; i < 8; ++i) top[n] = fmaxf(top[n], fabsf(v[n][i]));
        }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        top[n] = wave_max(top[n]);
        if ((threadIdx.x & 63) == 0) part[n][threadIdx.x >> 6] = top[n];
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        const float* p = part[threadIdx.x];
        const int sh = shift_to(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), 7);
        shift[threadIdx.x * places + row] = sh;
        rowexp[threadIdx.x * places + row] = -sh - 7;
    }
}

// Both weights to fragments, and their rows' exponents beside, in one launch.
struct PairWeights {
    const int16_t* trellis[2];
    int K[2], tn, decoders;             // workgroups of either weight
    uint16_t* frags;
    FragPlace place[2];
};

template <int CODE, int GRAD>
__global__ __launch_bounds__(256) void pair_prepare_kernel(PairWeights w, PairRows s, int32_t* __restrict__ shift,
                                                           int32_t* __restrict__ rowexp, int places) {
    __shared__ uint32_t words[256 * 7];
    int block = blockIdx.x;
    if (block >= 2 * w.decoders) return pair_exponents<GRAD>(s, block - 2 * w.decoders, shift, rowexp, places);
    const int role = block >= w.decoders;
    if (role) block -= w.decoders;
    auto decode = [&](auto K) {
        decode_tiles<decltype(K)::value, CODE, GRAD>(words, block, w.trellis[role], w.tn, w.frags, w.place[role]);
    };
    switch (w.K[role]) {
        case 2: return decode(std::integral_constant<int, 2>());
        case 3: return decode(std::integral_constant<int, 3>());
        case 4: return decode(std::integral_constant<int, 4>());
        case 5: return decode(std::integral_constant<int, 5>());
        case 6: return decode(std::integral_constant<int, 6>());
        default: return decode(std::integral_constant<int, 7>());
    }
}

// Rows to fragments for both weights, a wave 16 rows of one 128-column block: apart, or
// (GRAD) one weight's behind the other's in the summed dimension, with the sums of 16
// rows for the biases' gradients.
template <bool GRAD>
__global__ __launch_bounds__(256) void pair_transform_kernel(PairRows s, const int32_t* __restrict__ shift, int places,
                                                             uint16_t* __restrict__ f0, uint16_t* __restrict__ f1,
                                                             uint16_t* __restrict__ r0, uint16_t* __restrict__ r1,
                                                             float* __restrict__ colsum) {
    const int lane = threadIdx.x & 63, nblk = s.cols / 128;
    const int blk = blockIdx.x * 4 + (threadIdx.x >> 6), grp = blockIdx.y;
    if (blk >= nblk) return;
    const int q = lane >> 4, row = grp * 16 + (lane & 15);
    float v[2][32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[0][i] = v[1][i] = 0.0f;
    if (row < s.rows) {
#pragma unroll
        for (int p = 0; p < 4; ++p) load_pair8<GRAD>(s, row, 128 * blk + 32 * p + 8 * q, v[0] + 8 * p, v[1] + 8 * p);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        if (GRAD && colsum) rows_sum(v[n], lane, colsum + ((size_t)grp * 2 + n) * s.cols + 128 * blk);
        if (GRAD && !f0) continue;
#pragma unroll
        for (int p = 0; p < 4; ++p) scale_pair8(s.scale[n], 128 * blk + 32 * p + 8 * q, v[n] + 8 * p);
        rows_to_frags(v[n], row < s.rows ? shift[n * places + row] : 0, lane, grp, 4 * (GRAD * n * nblk + blk),
                      (GRAD ? 8 : 4) * nblk, n ? f1 : f0, n ? r1 : r0);
    }
}

// ------------------------------------------------------------------- product
// Fused epilogue or parts for gated_join_kernel.
enum GatedOut { kGatedFinish, kGatedParts };

struct GatedGemm {
    const uint16_t* A;                  // both weights, 8 groups of one, 8 of the other
    const uint16_t *B[2], *B2[2];       // the rows transformed for each; second terms
    const int32_t* rowexp[2];
    int nb, gb;                         // blocks of 128 columns, groups of 16 rows
    int steps, tiles, splits;
    float* part;                        // [splits][2 nb][gb][8][64][4]
};

template <int T>
__device__ __forceinline__ void role_columns(Columns<4> (&c)[8], const GatedArgs& a, int role, int blk, int lane) {
    Epilogue ep{};
    ep.colscale = a.w[role].svh;
    ep.scale = a.w[role].scale;
    ep.bias = a.bias[role];
    ep.bias_f32 = a.bias_f32[role];
    unit_columns<T>(c, ep, blk, lane);
}

// Transform, scales and bias of a unit of one weight, in place, and its z's store.
__device__ __forceinline__ void finish_role(f4* v, const Columns<4> (&c)[8], const GatedArgs& a, const GatedGemm& g,
                                            int role, int grp, int blk, int lane) {
    transform_unit(v);
    const int row = grp * 16 + (lane & 15), e = g.rowexp[role][row];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j][i] = ldexpf(v[j][i], e) * c[j].scale[i] + c[j].bias[i];
    if (a.z && row < a.rows) {
        float* z = a.z + ((size_t)role * a.rows + row) * a.w[0].n + blk * 128 + 4 * (lane >> 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) *(f4_a4*)(z + 16 * j) = v[j];
    }
}

// act(gate) up of a unit, and its store.
template <int T>
__device__ __forceinline__ void store_gated(const f4* gate, const f4* up, const GatedArgs& a, int grp, int blk,
                                            int lane) {
    const int row = grp * 16 + (lane & 15);
    if (row >= a.rows) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float o[4] = {gate[j][0], gate[j][1], gate[j][2], gate[j][3]};
        activate<4>(o, a.act);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= up[j][i];
        store16<T, 4>(a.y + (size_t)row * a.y_stride + blk * 128 + 16 * j + 4 * (lane >> 4), o);
    }
}

// The product of fragments.  A workgroup's tile is 256 columns by 8 W NB rows, a wave of
// its W one weight's 128 columns by 16 NB rows, in steps of 32 of the summed dimension.
// The columns' fragments are read by W / 2 waves each and come through three LDS buffers,
// two steps ahead, as in gemm_kernel of linear_kernels.hip, but by buffer loads: behind
// one of those, unlike behind a global load to LDS, the compiler counts what is still
// under way, and waits for what it needs alone.  A wave's rows are its own weight's and
// its own part, so they come straight into its registers.
// Eight waves read 48 KiB for as many products as twice four waves 64, which is what the
// compute unit's vector memory takes as long for as the matrix cores for the products:
// 4096 rows of 5120 by 17408 1386 us in all, 1527 with four waves, whose two workgroups
// share a compute unit.  (Rows through LDS too 1597; two terms 2395, 2365 with four.)
// Tiles go by XCD as gemm_kernel's, in bands of kRowBand.
constexpr int kRowBand = 4;             // (4096 rows 1386 us in all; of 2 and 8: 1391, 1394)

template <int T, int OUT, int NB, int TERMS, int W>
__global__ __launch_bounds__(64 * W, 2) void gated_gemm_kernel(GatedGemm g, GatedArgs a) {
    constexpr int kGroups = NB * W / 2, kA = 16 / W;
    constexpr int kOwn = kA + NB * TERMS;        // a wave's loads of a step
    constexpr int kExchange = OUT == kGatedFinish ? W * (NB / 2) * 8192 : 0, kLoop = 3 * 16 * kFragBytes;
    __shared__ __align__(1024) uint8_t lds[kLoop > kExchange ? kLoop : kExchange];
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), role = wv & 1, wm = wv >> 1;
    const int tile = xcd_order(blockIdx.x, g.tiles);
    const int mt = (g.gb + kGroups - 1) / kGroups, band = tile / (g.nb * kRowBand);
    const int high = mt - band * kRowBand < kRowBand ? mt - band * kRowBand : kRowBand, in = tile - band * g.nb * kRowBand;
    const int tn = in / high, tm = band * kRowBand + in - tn * high;
    const int split = blockIdx.y;
    const int s0 = (int)((long long)g.steps * split / g.splits);
    const int s1 = (int)((long long)g.steps * (split + 1) / g.splits);

    const int gb0 = tm * kGroups;        // first group of rows
    const auto fa = __builtin_amdgcn_make_buffer_rsrc((void*)(g.A + (size_t)tn * g.steps * 8192), 0, 0xFFFFFFFF, 0x00027000);
    const int at_a = wv * kA * kFragBytes + lane * 16;
    const size_t at_b = ((size_t)(gb0 >> 4) * g.steps * 16 + (gb0 & 15) + wm * NB) * 512 + lane * 8;
    const uint16_t* const fb[2] = {g.B[role] + at_b, TERMS == 2 ? g.B2[role] + at_b : nullptr};
    // Stages of the rows' registers: a step's come two steps ahead, or one where four
    // groups of two terms leave no room for more.
    constexpr int kStages = NB * TERMS > 4 ? 2 : 3;
    u4 b[kStages][TERMS][NB];
    // (Past the end the last step comes once more, so that the waits can count.)
    int to = 0;
    auto load_a = [&](int s) {
        const uint32_t at = (uint32_t)(s < s1 ? s : s1 - 1) * (16 * kFragBytes);
#pragma unroll
        for (int i = 0; i < kA; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(fa, (lds_void*)(lds + (to * 16 + wv * kA + i) * kFragBytes), 16, at_a,
                                                     at + i * kFragBytes, 0, 0);
        to = to == 2 ? 0 : to + 1;
    };
    auto load_b = [&](int s, auto stage) {
        const size_t at = (size_t)(s < s1 ? s : s1 - 1) * 8192;
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
#pragma unroll
            for (int i = 0; i < NB; ++i) b[decltype(stage)::value][t][i] = *(const u4*)(fb[t] + at + i * 512);
    };
    f4 acc[8][NB];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[j][i] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    // All waves' pieces of the next step are in LDS, and all waves have read this one
    // (their reads were waited for before they came here).
    auto meet_up = [&] {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kOwn) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    int from = 0;
    auto step = [&](int s, auto stage) {
        constexpr int I = decltype(stage)::value;
        load_a(s + 2);
        load_b(s + kStages - 1, std::integral_constant<int, (I + kStages - 1) % kStages>());
        u4 fr[8];
        const uint8_t* l = lds + from * 16 * kFragBytes + lane * 16;
#pragma unroll
        for (int j = 0; j < 8; ++j) fr[j] = *(const u4*)(l + (role * 8 + j) * kFragBytes);
        __builtin_amdgcn_sched_barrier(0);      // all reads under way before the first product
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int t = 0; t < TERMS; ++t)
#pragma unroll
                for (int i = 0; i < NB; ++i) acc[j][i] = mfma<false>(fr[j], b[I][t][i], acc[j][i]);
        __builtin_amdgcn_sched_barrier(0);      // none after the others have met
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        meet_up();
        from = from == 2 ? 0 : from + 1;
    };
    const std::integral_constant<int, 0> c0;
    const std::integral_constant<int, 1> c1;
    // (The first step's pieces before all else: the wait below leaves under way the last
    // loads to be issued, and these may not be among them.  Loads to registers could
    // otherwise be moved ahead of loads to LDS.)
    load_a(s0);
    asm volatile("" ::: "memory");
    load_b(s0, c0);
    load_a(s0 + 1);
    if constexpr (kStages == 3) load_b(s0 + 1, c1);
    meet_up();
    // (Whole turns of the stages, and the rest: were a turn cut short in the loop, the
    // compiler would take a stage's loads for still under way where the next are issued.)
    int s = s0;
    for (; s + kStages <= s1; s += kStages) {
        step(s, c0);
        step(s + 1, c1);
        if constexpr (kStages == 3) step(s + 2, std::integral_constant<int, 2>());
    }
    if (s < s1) step(s, c0);
    if constexpr (kStages == 3)
        if (s + 1 < s1) step(s + 1, c1);
    if constexpr (OUT == kGatedParts) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int grp = gb0 + wm * NB + b;
            if (grp >= g.gb) continue;
            f4* o = (f4*)g.part + (((size_t)split * 2 * g.nb + 2 * tn + role) * g.gb + grp) * 512 + lane;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j * 64] = acc[j][b];
        }
        return;
    }
    // Of each two units a wave keeps one and gives the other's factor to the wave of
    // the other weight.  (Rows past the last group are finished like others, from what
    // their places hold, and not stored; the exponents' places are there for all of
    // a tile's groups.)
    Columns<4> cols[8];
    role_columns<T>(cols, a, role, tn, lane);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // (the steps past the end lie where the factors go)
    __syncthreads();
    f4* const give = (f4*)lds + (size_t)wv * (NB / 2) * 512 + lane;
    const f4* const take = (const f4*)lds + (size_t)(wv ^ 1) * (NB / 2) * 512 + lane;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        f4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = acc[j][b];
        finish_role(v, cols, a, g, role, gb0 + wm * NB + b, tn, lane);
        // wave `role` keeps units b with b % 2 == role
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if ((b & 1) != role) give[(b >> 1) * 512 + j * 64] = v[j];
            else acc[j][b & ~1] = v[j];
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; b += 2) {
        f4 mine[8], other[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            mine[j] = acc[j][b];
            other[j] = take[(b >> 1) * 512 + j * 64];
        }
        const int grp = gb0 + wm * NB + b + role;
        if (role == 0) store_gated<T>(mine, other, a, grp, tn, lane);
        else store_gated<T>(other, mine, a, grp, tn, lane);
    }
}

// Joins the splits' parts of both weights, a workgroup of one wave one unit.
template <int T>
__global__ __launch_bounds__(64) void gated_join_kernel(GatedGemm g, GatedArgs a) {
    const int lane = threadIdx.x, grp = blockIdx.x, blk = blockIdx.y;
    const Gemm parts{nullptr, nullptr, nullptr, 16 * g.nb, g.gb, g.steps, g.tiles, g.splits, g.part, nullptr, nullptr, 0};
    f4 v[2][8];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        sum_splits<4>(v[r], parts, grp, 2 * blk + r, lane, 0, g.splits);
        Columns<4> cols[8];
        role_columns<T>(cols, a, r, blk, lane);
        finish_role(v[r], cols, a, g, r, grp, blk, lane);
    }
    store_gated<T>(v[0], v[1], a, grp, blk, lane);
}

// ------------------------------------------------------------------ gradient
__global__ __launch_bounds__(256) void gated_column_sums_kernel(ColSum a) {
    __shared__ float part[256];
    column_sums(a, blockIdx.x, part);
}

// dx's units: each weight's parts added and transformed, times its scales, and both added.
template <int T>
__global__ __launch_bounds__(64) void gated_dx_kernel(Gemm g, GatedGradArgs a, const int32_t* __restrict__ rowexp,
                                                      int places) {
    const int lane = threadIdx.x, grp = blockIdx.x, blk = blockIdx.y, row = grp * 16 + (lane & 15);
    f4 v[2][8];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        sum_splits<4>(v[r], g, grp, blk, lane, r * (g.splits / 2), (r + 1) * (g.splits / 2));
        transform_unit(v[r]);
        Epilogue ep{};
        ep.colscale = a.w[r].suh;
        ep.scale = a.w[r].scale;
        Columns<4> cols[8];
        unit_columns<T>(cols, ep, blk, lane);
        const int e = row < a.rows ? rowexp[r * places + row] : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[r][j][i] = ldexpf(v[r][j][i], e) * cols[j].scale[i];
    }
    if (row >= a.rows) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const f4 t = v[0][j] + v[1][j];
        const float o[4] = {t[0], t[1], t[2], t[3]};
        store16<T, 4>(a.dx + (size_t)row * a.dx_stride + blk * 128 + 16 * j + 4 * (lane >> 4), o);
    }
}

// ---------------------------------------------------------------- host side
struct Taker {
    size_t at = 0;
    size_t operator()(size_t bytes) {
        const size_t a = at;
        at += align256(bytes);
        return a;
    }
};

struct FewPlan {
    int groups, workers, per_block;
    bool apart;
    size_t part, frag, rest, shift, total;
};

// Rows that go through the kernel of few rows, 64 at a time.
constexpr int kGatedFew = 256;

int few_chunks(int rows) { return (rows + kFewRows - 1) / kFewRows; }

bool takes_few(int rows, int k, int n) {
    return rows <= kGatedFew && n / 128 <= XTQ_OP_COUNTERS &&
           (long long)(n / 64) * (k / 32) < 1LL << 30;
}

// A chunk's workgroups: as few_splits cuts the blocks, with 16 steps each at least where
// there are several chunks (100 rows of 1024 by 4096 21 us, 24 with 8).  Where that
// leaves a fifth of the places empty, blocks that come twice into them in four parts
// each, others evenly over all steps if a run still has 32 of them.
//
// us a call, called one behind the other, bf16, K = 4, weights that no cache holds:
//   blocks, steps       rows   whole   in 2   in 3   in 4   in 5   over all   taken
//   172 of 4096            1    28.9   29.1   31.8   25.1   28.8       33.0   4
//                         64    51.7   45.4   50.8   44.4   49.1       46.4
//   172 of 2048            1    20.1   18.1   20.6   18.3   20.9       23.6   2
//   272 of 5120            1    53.3   43.1   47.2   45.0   42.5       42.9   over all
//                         64    84.2   74.7   71.4   72.3   74.7       65.6
//   96 of 4096             1    28.5   20.5   23.1   18.2   17.6       22.7   5
//   144 of 16384          24   132.5  103.6   76.7   77.0   67.0       71.6   3
// In 268 cases (19 sizes of 1024 to 17408 by 4096 to 17408, 1 to 200 rows, one term and
// two) what is taken is 1.4% slower in the mean than the fastest of these, 6 and 8 parts.
// It is furthest off in the table's last row (14%) and at one row of two terms of 8192 by
// 11008 (52.7 in four parts, 46.7 over all) and 2048 by 11008 (20.7 in two, 18.2 in four).
void few_workers(FewPlan& p, int rows, int k, int n, int waves) {
    const int blocks = n / 64, chunks = few_chunks(rows), steps = k / 32, places = 2 * kCUs;
    int s = few_splits(rows < kFewRows ? rows : kFewRows, k, 2 * n, waves);
    if (chunks > 1 && s > steps / 16) s = steps / 16 > 1 ? steps / 16 : 1;
    while (s > 1 && blocks * s * chunks > places) --s;
    const int all = blocks * s * chunks, rounds = (all + places - 1) / places;
    p.per_block = s;
    if (2 * all > places && 5LL * all < 4LL * rounds * places && (long long)blocks * steps * chunks / places >= 32)
        p.per_block = chunks == 1 && s == 2 && steps >= 4 * waves ? 4 : 0;
    p.workers = p.per_block ? blocks * p.per_block : places / chunks;
}

FewPlan few_plan(int rows, int k, int n, bool two) {
    FewPlan p;
    const int chunks = few_chunks(rows), blocks = n / 64;
    p.groups = chunks > 1 ? 4 * chunks : few_groups(rows);
    few_workers(p, rows, k, n, few_waves(chunks > 1 ? 4 : p.groups));
    // (16: as few_plan of linear_kernels.hip, by the blocks of rows of a run)
    p.apart = rows > kFusedRows || (long long)rows * blocks * (k / 128) > 16LL * p.workers;
    Taker take;
    p.part = take((size_t)chunks * (p.workers + blocks) * 128 * (chunks > 1 ? kFewRows : rows) * 4);
    p.frag = take(p.apart ? (size_t)2 * p.groups * k * 32 : 0);
    p.rest = take(p.apart && two ? (size_t)2 * p.groups * k * 32 : 0);
    p.shift = take(p.apart ? (size_t)2 * p.groups * k / 2 : 0);
    p.total = take.at;
    return p;
}

// How the product of many rows is cut, as gemm_tiling of linear_kernels.hip does: by the
// shortest estimate.  Tiles have 32 nb rows; nb 8, of one term, those of eight waves.  us
// of a workgroup's step alone on a compute unit, of two at once, and of each where there
// are more, by terms and rows, fitted to 90 sizes' times under every cut (257 to 4096
// rows): the chosen one was 1.3% off the fastest in the mean when timed anew, 9% at most.
Tiling gated_tiling(int rows, int n, int steps, bool two) {
    static const double cost[2][3][3] = {{{0.30, 0.51, 0.26}, {0.53, 0.59, 0.30}, {0.57, 1.00, 0.45}},
                                         {{0.89, 0.93, 0.58}, {0.97, 1.40, 0.63}}};
    Tiling best{};
    double least = 0.0;
    for (int nb = two ? 4 : 8; nb >= 2; nb /= 2) {
        const double* c = cost[two][nb / 4];
        const int tiles = n / 128 * ((rows + 32 * nb - 1) / (32 * nb));
        for (int s = 1; s == 1 || (s <= steps / 8 && (s - 1) * tiles < 2 * kCUs); ++s) {
            const int each = (int)(((long long)tiles * s + kCUs - 1) / kCUs);
            const double step = each == 1 ? c[0] : each == 2 ? c[1] : c[2] * (nb < 8 && each % 2 ? each + 0.2 : each);
            const double us = step * ((steps + s - 1) / s) + (s > 1 ? 3.0 + 3.8e-6 * s * rows * n : 0.0);
            if (!best.nb || us < least) {
                least = us;
                best = Tiling{nb, tiles, s};
            }
        }
    }
    return best;
}

struct ManyPlan {
    int groups, places, nb, tiles, splits;
    size_t shift, rowexp, xf[2], x2[2], wf, part, total;
};

ManyPlan many_plan(int rows, int k, int n, bool two) {
    ManyPlan p;
    p.groups = (rows + 15) / 16;
    p.places = (p.groups + 15) / 16 * 256;      // whole tiles' rows
    const Tiling t = gated_tiling(rows, n, k / 32, two);
    p.nb = t.nb;
    p.tiles = t.tiles;
    p.splits = t.splits;
    Taker take;
    p.shift = take((size_t)2 * p.places * 4);
    p.rowexp = take((size_t)2 * p.places * 4);
    for (int r = 0; r < 2; ++r) {
        p.xf[r] = take(frag_bytes(p.groups, k / 32));
        p.x2[r] = take(two ? frag_bytes(p.groups, k / 32) : 0);
    }
    p.wf = take(frag_bytes(2 * n / 16, k / 32));
    p.part = take(p.splits > 1 ? (size_t)p.splits * p.groups * 64 * 2 * n : 0);
    p.total = take.at;
    return p;
}

template <int GRAD>
void pair_prepare(const Weight* w, uint16_t* frags, FragPlace p0, FragPlace p1, const PairRows& src, int32_t* shift,
                  int32_t* rowexp, int places, hipStream_t s) {
    const int decoders = (w[0].k / 16) * (w[0].n / 16) / 32;
    const PairWeights pw{{w[0].trellis, w[1].trellis}, {w[0].K, w[1].K}, w[0].n / 16, decoders, frags, {p0, p1}};
    auto launch = [&](auto* kernel) {
        hipLaunchKernelGGL(kernel, dim3(2 * decoders + src.rows), dim3(256), 0, s, pw, src, shift, rowexp, places);
    };
    if (w[0].code == kCodeMul1) launch(pair_prepare_kernel<kCodeMul1, GRAD>);
    else if (w[0].code == kCodeMcg) launch(pair_prepare_kernel<kCodeMcg, GRAD>);
    else launch(pair_prepare_kernel<kCode3Inst, GRAD>);
}

template <int T, int OUT>
void gemm(const GatedGemm& g, const GatedArgs& a, int nb, hipStream_t s) {
    auto launch = [&](auto* kernel, int waves) {
        hipLaunchKernelGGL(kernel, dim3(g.tiles, g.splits), dim3(64 * waves), 0, s, g, a);
    };
    if (a.two && nb == 4) launch(gated_gemm_kernel<T, OUT, 4, 2, 4>, 4);
    else if (a.two) launch(gated_gemm_kernel<T, OUT, 2, 2, 4>, 4);
    else if (nb == 8) launch(gated_gemm_kernel<T, OUT, 4, 1, 8>, 8);
    else if (nb == 4) launch(gated_gemm_kernel<T, OUT, 4, 1, 4>, 4);
    else launch(gated_gemm_kernel<T, OUT, 2, 1, 4>, 4);
}

template <int T>
hipError_t many(const GatedArgs& a, void* ws, hipStream_t s) {
    const int k = a.w[0].k, n = a.w[0].n;
    const ManyPlan p = many_plan(a.rows, k, n, a.two);
    uint8_t* base = (uint8_t*)ws;
    GatedGemm g{};
    g.A = (uint16_t*)(base + p.wf);
    g.nb = n / 128;
    g.gb = p.groups;
    g.steps = k / 32;
    g.tiles = p.tiles;
    g.splits = p.splits;
    g.part = (float*)(base + p.part);
    int32_t *shift = (int32_t*)(base + p.shift), *rowexp = (int32_t*)(base + p.rowexp);
    uint16_t *xf[2], *x2[2];
    for (int r = 0; r < 2; ++r) {
        g.B[r] = xf[r] = (uint16_t*)(base + p.xf[r]);
        g.B2[r] = x2[r] = a.two ? (uint16_t*)(base + p.x2[r]) : nullptr;
        g.rowexp[r] = rowexp + r * p.places;
    }
    const PairRows src{a.x, a.x_stride, nullptr, {a.w[0].suh, a.w[1].suh}, T, 0, a.rows, k};
    pair_prepare<0>(a.w, (uint16_t*)(base + p.wf), FragPlace{0, 0, k / 32}, FragPlace{1, 0, k / 32}, src, shift, rowexp,
                    p.places, s);
    hipLaunchKernelGGL(pair_transform_kernel<false>, dim3((k / 128 + 3) / 4, p.groups), dim3(256), 0, s, src,
                       (const int32_t*)shift, p.places, xf[0], xf[1], x2[0], x2[1], (float*)nullptr);
    if (p.splits == 1) {
        gemm<T, kGatedFinish>(g, a, p.nb, s);
    } else {
        gemm<T, kGatedParts>(g, a, p.nb, s);
        hipLaunchKernelGGL((gated_join_kernel<T>), dim3(p.groups, n / 128), dim3(64), 0, s, g, a);
    }
    return hipGetLastError();
}

struct GradPlan {
    int groups, places, nb, tiles, splits;      // splits: of both weights together
    size_t shift, rowexp, zf, z2, wf, part, colsum, total;
};

GradPlan grad_plan(int rows, int k, int n, bool two) {
    GradPlan p;
    p.groups = (rows + 15) / 16;
    p.places = p.groups * 16;
    const Tiling t = gemm_tiling(rows, k, n / 32, two);
    p.nb = t.nb;
    p.tiles = t.tiles;
    p.splits = 2 * t.splits;
    Taker take;
    p.shift = take((size_t)2 * p.places * 4);
    p.rowexp = take((size_t)2 * p.places * 4);
    p.zf = take(frag_bytes(p.groups, n / 16));
    p.z2 = take(two ? frag_bytes(p.groups, n / 16) : 0);
    p.wf = take(frag_bytes(k / 16, n / 16));
    p.part = take((size_t)p.splits * p.groups * 64 * k);
    p.colsum = take((size_t)p.groups * 2 * n * 4);
    p.total = take.at;
    return p;
}

template <int T>
hipError_t gradient(const GatedGradArgs& a, void* ws, hipStream_t s) {
    const int k = a.w[0].k, n = a.w[0].n;
    const GradPlan p = grad_plan(a.rows, k, n, a.two);
    uint8_t* base = (uint8_t*)ws;
    int32_t *shift = (int32_t*)(base + p.shift), *rowexp = (int32_t*)(base + p.rowexp);
    uint16_t *wf = (uint16_t*)(base + p.wf), *zf = (uint16_t*)(base + p.zf), *z2 = a.two ? (uint16_t*)(base + p.z2) : nullptr;
    const bool sum = a.dbias[0] || a.dbias[1];
    float* colsum = sum ? (float*)(base + p.colsum) : nullptr;
    const PairRows src{a.dy, a.dy_stride, a.z, {a.w[0].svh, a.w[1].svh}, T, a.act, a.rows, n};
    const ColSum sums{colsum, p.groups, 2 * n, T, a.bias_f32[0], a.dbias[0], n, a.bias_f32[1], a.dbias[1]};
    const int adders = sum ? 2 * n / 64 : 0;
    auto transform = [&](const int32_t* sh, uint16_t* f, uint16_t* rest) {
        hipLaunchKernelGGL(pair_transform_kernel<true>, dim3((n / 128 + 3) / 4, p.groups), dim3(256), 0, s, src, sh,
                           p.places, f, f, rest, rest, colsum);
    };
    if (!a.dx) {
        transform(nullptr, nullptr, nullptr);
        hipLaunchKernelGGL(gated_column_sums_kernel, dim3(adders), dim3(256), 0, s, sums);
        return hipGetLastError();
    }
    pair_prepare<1>(a.w, wf, FragPlace{-1, 0, n / 16}, FragPlace{-1, n / 32, n / 16}, src, shift, rowexp, p.places, s);
    transform(shift, zf, z2);
    const Gemm g{wf, zf, z2, k / 16, p.groups, n / 16, p.tiles, p.splits, (float*)(base + p.part), nullptr, nullptr, 0};
    const hipError_t e = launch_parts(g, T, p.nb, a.two, sums, adders, s);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((gated_dx_kernel<T>), dim3(p.groups, k / 128), dim3(64), 0, s, g, a, (const int32_t*)rowexp, p.places);
    return hipGetLastError();
}

}  // namespace

size_t gated_ws_bytes(int rows, int k, int n, bool two) {
    return takes_few(rows, k, n) ? few_plan(rows, k, n, two).total : many_plan(rows, k, n, two).total;
}

size_t gated_bwd_ws_bytes(int rows, int k, int n, bool two) { return grad_plan(rows, k, n, two).total; }

hipError_t launch_gated(const GatedArgs& a, void* ws, uint32_t* counters, hipStream_t s) {
    const int k = a.w[0].k, n = a.w[0].n;
    if (!takes_few(a.rows, k, n)) return a.type == kBf16 ? many<kBf16>(a, ws, s) : many<kF16>(a, ws, s);
    const FewPlan p = few_plan(a.rows, k, n, a.two);
    uint8_t* base = (uint8_t*)ws;
    const int steps = p.per_block ? k / 32 : n / 64 * (k / 32), of = p.per_block ? p.per_block : p.workers;
    GatedFew f{nullptr, nullptr, nullptr, p.groups, p.workers, p.per_block, steps / of, steps % of,
               (float*)(base + p.part), counters};
    if (p.apart) {
        u4 *frag = (u4*)(base + p.frag), *rest = a.two ? (u4*)(base + p.rest) : nullptr;
        int32_t* shift = (int32_t*)(base + p.shift);
        transform_few(a.two, a.x, a.x_stride, a.type, a.rows, k, p.groups, a.w[0].suh, a.w[1].suh, frag, rest, shift, s);
        f.frag = frag;
        f.frag_lo = rest;
        f.shift = shift;
    }
    static decltype(&launch_gated_few_code0) const few[] = {launch_gated_few_code0, launch_gated_few_code1,
                                                            launch_gated_few_code2};
    return few[a.w[0].code](a, f, s);
}

hipError_t launch_gated_bwd(const GatedGradArgs& a, void* ws, hipStream_t s) {
    return a.type == kBf16 ? gradient<kBf16>(a, ws, s) : gradient<kF16>(a, ws, s);
}

}  // namespace xtq
