// gated_delta.h -- linear attention by the gated delta rule: S <- e^g S, u = beta (v - S^T k), S <- S + k u^T, o = scale S^T q,
// the state carried from pass to pass in 32-bit floats, one slot per sequence.
#pragma once

#include "nvllm_internal.h"

namespace nvllm {

constexpr int DELTA_SPANS = 32;   // portions that travel with a launch's arguments
constexpr int DELTA_MAX_DIM = 256;

struct Delta {
    const void *q, *k, *v;      // rows of [Q][dim], [Q][dim], [H][vdim], `ld` elements apart
    const float *g, *beta;      // [T][H]
    float* state;               // [slot][H][dim][vdim]
    void* out;                  // [T][H][vdim]
    long q_ld, k_ld, v_ld;
    float scale, eps;           // eps 0: queries and keys as they are
    int Q, H, dim, vdim;
    const int4* spans;          // (first token, count, first position, slot); null: the ones here
    int n_spans;
    int4 here[DELTA_SPANS];
};

}  // namespace nvllm
