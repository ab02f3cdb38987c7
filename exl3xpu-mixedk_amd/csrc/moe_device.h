// moe_device.h -- what the kernels of the mixture layer share.
#pragma once
#include "few_device.h"

namespace xtq {

// Work of the experts: up to 16 of an expert's rows, in the order of the experts,
// with the expert's weights (gate, up, down), so that a workgroup finds all it
// needs in one load.
struct MoeChunk {
    xtq_moe_weight w[3];
    int32_t rows, pad[3];
    int32_t slots[16];                  // token * top + place
};

// One call's arguments and scratch.  A token's choices are its slots.
struct MoeArgs {
    const xtq_moe_weight* table;        // [experts][3]: gate, up, down
    int experts, d, f, code, type, rows, top, act, renorm;
    const uint16_t* x;
    long long x_stride;
    const void* router;
    int router_f32;
    const uint8_t* valid;
    const uint16_t* res;
    long long res_stride;
    uint16_t* y;
    long long y_stride;
    int32_t* ids;                       // [rows][top]
    float* weights;                     // [rows][top]
    float* logits;                      // [rows][experts]
    int32_t* nchunks;
    MoeChunk* chunks;
    u4* xf;                             // not fused: [chunk][role][hi, lo][d/32][64]
    int32_t* xs;                        // [chunk][role][d/128][16]
    float* up_part;                     // [chunk][f/128][role][splits][512][4]
    u4* hf;                             // [chunk][hi, lo][f/32][64]
    int32_t* hs;                        // [chunk][f/128][16]
    float* out;                         // [splits][slot][d]
    int max_chunks, up_splits, down_splits;
    uint32_t* counters;                 // router, then d/128, then [chunk][f/128]
};

constexpr int kMoeRows = 64;            // rows of a call
constexpr int kMoeTop = 16;
constexpr int kMoeExperts = 512;
constexpr int kMoeRouterCounters = 32;  // one for each 4 rows, one for all

#define XTQ_MOE(C) \
    hipError_t launch_moe_code##C(const MoeArgs& a, hipStream_t s);
XTQ_MOE(0) XTQ_MOE(1) XTQ_MOE(2)
#undef XTQ_MOE

}  // namespace xtq
