// gated_delta.h -- linear attention by the gated delta rule: S <- e^g S, u = beta (v - S^T k), S <- S + k u^T, o = scale S^T q,
// the state carried from pass to pass in 32-bit floats, one slot per sequence.
#pragma once

#include "nvllm_internal.h"

namespace nvllm {

constexpr int DELTA_SPANS = 96;   // portions that travel with a launch's arguments
constexpr int DELTA_MAX_DIM = 256;

struct Delta {
    const void *q, *k, *v;      // rows of [Q][dim], [Q][dim], [H][vdim], `ld` elements apart
    const float *g, *beta;      // [T][H]
    float* state;               // [slot][H][dim][vdim]
    void* out;                  // [T][H][vdim]
    long q_ld, k_ld, v_ld;
    float scale, eps;           // eps 0: queries and keys as they are
    int Q, H, dim, vdim;
    int dim_kept;               // of the state: dim without padding
    int v_cols;                 // of v's rows: vdim with padding
    const int4* spans;          // (first token, count, first position, slot); null: the ones here
    int n_spans;
    int4 here[DELTA_SPANS];
};

// Portions of several tokens in chunks of DELTA_CHUNK tokens.
constexpr int DELTA_CHUNK = 64;
// What a chunk's tokens need of each other, per (chunk, head): the operands of T' and P (six 16 x 32 tiles on and below the diagonal
// each, three parts), then per token the factors a, b and c, then what is left of the state.
constexpr int DELTA_PART = 1024, DELTA_TILE = 3 * DELTA_PART, DELTA_OPS = 12 * DELTA_TILE, DELTA_RECORD = DELTA_OPS + 1024;
struct DeltaChunks {           // (what every workgroup asks for first lies together)
    char* mem;                  // [chunk of the launch][H] records
    const int* first;           // [n_spans] the launch's first chunk of each span; null: the ones here
    int from, most;             // chunks [from, from + most) of every span
    int step_waves;             // of portions behind the first n_spans, which go token by token beside the first chunks
    int segs, per_seg;          // segments of a portion's chunks of the launch at most, chunks of one
    int out_four;               // out can be stored four elements at a time
    float* starts;              // [span][segs][H][dims][columns] states that segments start from, both padded ...
    float* trans;               // [span][segs][H][dims][dims] ... and what becomes of a state over a segment
    double bytes, flops;        // kernel timing
    Delta a;                    // queries and keys: dims padded with zeros to a multiple of 8, rows 16-byte aligned
    int first_here[DELTA_SPANS];
};

}  // namespace nvllm
