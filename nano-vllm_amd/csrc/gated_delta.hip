// gated_delta.hip -- the gated delta rule (gated_delta.h).
//
// k_delta_step: token by token.  With the state S of before, a = S^T k, b = S^T q and c = k . q, the token's correction and result are
//   u = beta (v - e^g a),   o = scale (e^g b + c u),   S <- e^g S + k u^T,
// so one pass over S and one sum over its rows serve both.  A wave holds 32 value columns of a head's state in registers (a lane: 4
// columns x NR rows: 8 lanes read 128 bytes of a row), reads it once, goes through the portion's tokens and writes it once.  Bound by
// memory: 64 sequences, 32 heads of 128 x 128: 270 MB in 52.5 us, 5.1 TB/s as a copy of 1 GiB; the smallest calls by the launch and
// their trips to memory (4 heads of 64 x 64: 5.8 us).
//
// Portions of several tokens go in chunks of 64.  With G_t the sum of g up to token t of the chunk, k and q normed, S the state in front:
//   A_ts = beta_t e^(G_t - G_s) k_t . k_s  for s < t,   T' = (I + A)^-1 diag(beta),   P_ts = scale e^(G_t - G_s) q_t . k_s  for s <= t,
//   X_t = v_t - e^(G_t) S^T k_t,   U = T' X,   o_t = scale e^(G_t) S^T q_t + sum_s P_ts u_s,   S <- e^(G_n) S + sum_s e^(G_n - G_s) k_s u_s^T
// k_delta_prepare forms T' and P of all chunks and heads side by side, k_delta_chunks walks a portion's chunks.  What norms keys and
// queries is a factor per token, so the rows themselves enter the matrix cores as they are: bf16 values exactly.  All other
// factors (S, X, U, T', P, and fp32 rows) enter as three bf16 parts, 26 bits together: a product of two of them is the six products
// of parts above 2^-26.
#include "gated_delta.h"

#include <algorithm>
#include <new>
#include <vector>

#include "gemm_common.h"
#include "sequence_memory.h"

namespace nvllm {

typedef unsigned int u2_t __attribute__((ext_vector_type(2)));

// Memory by descriptors: what lies behind `bytes` (and every offset of NOWHERE) reads as zeros and is not written, so that a chunk's
// loads have no branch around them and all of them are in flight together.
constexpr unsigned NOWHERE = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t memory(const void* base, long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ u4_t load16(__amdgpu_buffer_rsrc_t m, unsigned at, int base = 0) { return __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(m, (int)at, base, 0)); }
__device__ __forceinline__ float load4(__amdgpu_buffer_rsrc_t m, unsigned at) { return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(m, (int)at, 0, 0)); }
__device__ __forceinline__ unsigned two_b16(float lo, float hi) {
    typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, b2_t{(__bf16)lo, (__bf16)hi});
}
// Four neighbouring elements as they lie in memory, of which the first `left` are there; one by one where the addresses are no multiples of
// four elements.
template <bool B16, bool VEC>
struct Four {
    u4_t w;
    template <int AUX = 0>
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t m, unsigned at, int left) {
        if (VEC) {
            const int from = (int)(left > 0 ? at : NOWHERE);
            if (B16) {
                const u2_t p = __builtin_amdgcn_raw_buffer_load_b64(m, from, 0, AUX);
                w = u4_t{p[0], p[1], 0, 0};
            } else w = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(m, from, 0, AUX));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (B16) w[i] = (unsigned)(unsigned short)__builtin_amdgcn_raw_buffer_load_b16(m, (int)(i < left ? at + 2 * i : NOWHERE), 0, AUX) << 16;
                else w[i] = __builtin_amdgcn_raw_buffer_load_b32(m, (int)(i < left ? at + 4 * i : NOWHERE), 0, AUX);
            }
        }
    }
    __device__ __forceinline__ f4_t get() const {
        if (VEC && B16)
            return f4_t{__builtin_bit_cast(float, w[0] << 16), __builtin_bit_cast(float, w[0] & 0xffff0000u), __builtin_bit_cast(float, w[1] << 16),
                        __builtin_bit_cast(float, w[1] & 0xffff0000u)};
        return __builtin_bit_cast(f4_t, w);
    }
};
template <bool B16, bool VEC, int AUX = 0>
__device__ __forceinline__ void store_four(__amdgpu_buffer_rsrc_t m, unsigned at, const f4_t& v, int left) {
    if (VEC) {
        const int to = (int)(left > 0 ? at : NOWHERE);
        if (B16) __builtin_amdgcn_raw_buffer_store_b64(u2_t{two_b16(v[0], v[1]), two_b16(v[2], v[3])}, m, to, 0, AUX);
        else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, v), m, to, 0, AUX);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float z = v[i];
            if (B16) __builtin_amdgcn_raw_buffer_store_b16((unsigned short)two_b16(z, z), m, (int)(i < left ? at + 2 * i : NOWHERE), 0, AUX);
            else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, z), m, (int)(i < left ? at + 4 * i : NOWHERE), 0, AUX);
        }
    }
}
// e^g, the product with log2(e) in 64 bits: its rounding would count for large |g|
__device__ __forceinline__ float decay_f(float g) { return __builtin_amdgcn_exp2f((float)((double)g * 1.4426950408889634)); }
// the sum over the eight lanes that are a multiple of eight apart, in all of them
__device__ __forceinline__ float sum_over_rows(float x) {
    x += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x128 /* row_ror:8 */, 0xf, 0xf, true));
    const unsigned a = __builtin_bit_cast(unsigned, x);
    const auto p = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    x = __builtin_bit_cast(float, (unsigned)p[0]) + __builtin_bit_cast(float, (unsigned)p[1]);
    const unsigned b = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}

constexpr int STEP_COLS = 32;   // of a wave

// A kernel's arguments come from memory, and each is asked for where it is first used: one trip behind the other before the first load of
// data.  Named together in front they take one trip.
#define ASKED_FOR_AT_ONCE(A)                                                                                                                            \
    asm volatile("" ::"s"((A).q), "s"((A).k), "s"((A).v), "s"((A).g), "s"((A).beta), "s"((A).state), "s"((A).q_ld), "s"((A).k_ld), "s"((A).v_ld), "s"((A).H), "s"((A).Q), \
                 "s"((A).dim), "s"((A).vdim), "s"((A).spans), "s"((A).eps), "s"((A).scale))
__device__ __forceinline__ int4 scalars(const int4& v) {
    return int4{__builtin_amdgcn_readfirstlane(v.x), __builtin_amdgcn_readfirstlane(v.y), __builtin_amdgcn_readfirstlane(v.z), __builtin_amdgcn_readfirstlane(v.w)};
}
// a portion of the launch, in scalar registers
__device__ __forceinline__ int4 span_of(const Delta& a, int s) {
    int4 v = a.here[min(s, DELTA_SPANS - 1)];
    ASKED_FOR_AT_ONCE(a);
    asm volatile("" ::"s"(v.x), "s"(v.y), "s"(v.z), "s"(v.w));
    if (a.spans) v = a.spans[s];
    return scalars(v);
}

template <bool B16, int NR, bool VEC>
__device__ __forceinline__ void delta_step(const Delta& a, const int4& span, int h, int slice, int lane) {   // portion, head and slice of the wave
    constexpr int R4 = NR / 4;
    typedef Four<B16, VEC> F;
    const int col = slice * STEP_COLS + (lane & 7) * 4, row0 = (lane >> 3) * NR, hq = h / (a.H / a.Q);
    constexpr int ELEM = B16 ? 2 : 4;
    const int cols = a.vdim - col;   // that this lane has at most
    // Rows behind the last one lie behind the descriptors' ends.  States are read once and written once, past the caches, which other layers'
    // states pass through before they are back: twelve layers in turn, 64 sequences, 32 heads of 128 x 128: 59.1 us through the caches, 53.5
    // past them; of 64 x 64: 17.5, 14.1.  (Three layers that fit the caches: 32 sequences of 128 x 128 22.6, 27.8.)
    constexpr int PAST = 2;
    float* st = a.state + ((size_t)span.w * a.H + h) * a.dim * a.vdim;
    const long st_bytes = (long)a.dim * a.vdim * 4;
    const unsigned st_at = ((unsigned)row0 * a.vdim + col) * 4, st_row = 4u * a.vdim;
    f4_t S[NR];
    {
        const auto m = memory(st, span.z > 0 ? st_bytes : 0);
        Four<false, VEC> in[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) in[r].template load<PAST>(m, st_at + r * st_row, cols);
#pragma unroll
        for (int r = 0; r < NR; r++) S[r] = in[r].get();
    }
    F kn[R4], qn[R4], vn;
    float gn, bn;
    auto fetch = [&](int t) {
        const auto mk = memory((const char*)a.k + ((size_t)t * a.k_ld + hq * a.dim) * ELEM, a.dim * ELEM), mq = memory((const char*)a.q + ((size_t)t * a.q_ld + hq * a.dim) * ELEM, a.dim * ELEM);
#pragma unroll
        for (int r = 0; r < R4; r++) {
            kn[r].load(mk, (row0 + 4 * r) * ELEM, a.dim - row0 - 4 * r);
            qn[r].load(mq, (row0 + 4 * r) * ELEM, a.dim - row0 - 4 * r);
        }
        vn.load(memory((const char*)a.v + ((size_t)t * a.v_ld + h * a.vdim) * ELEM, a.vdim * ELEM), col * ELEM, cols);
        gn = a.g[(size_t)t * a.H + h];
        bn = a.beta[(size_t)t * a.H + h];
    };
    fetch(span.x);
    for (int i = 0; i < span.y; i++) {
        const int t = span.x + i;
        f4_t k[R4], q[R4];
#pragma unroll
        for (int r = 0; r < R4; r++) {
            k[r] = kn[r].get();
            q[r] = qn[r].get();
        }
        const f4_t v = vn.get();
        const float decay = decay_f(gn), beta = bn;
        fetch(min(t + 1, span.x + span.y - 1));
        f4_t sk = {0.f, 0.f, 0.f, 0.f}, sq = {0.f, 0.f, 0.f, 0.f};
        float kq = 0.f, kk = 0.f, qq = 0.f;
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const float kr = k[r / 4][r % 4], qr = q[r / 4][r % 4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                sk[e] = fmaf(kr, S[r][e], sk[e]);
                sq[e] = fmaf(qr, S[r][e], sq[e]);
            }
            kq = fmaf(kr, qr, kq);
            kk = fmaf(kr, kr, kk);
            qq = fmaf(qr, qr, qq);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            sk[e] = sum_over_rows(sk[e]);
            sq[e] = sum_over_rows(sq[e]);
        }
        kq = sum_over_rows(kq);
        float rk = 1.f, rq = 1.f;   // what norms queries and keys
        if (a.eps > 0.f) {
            rk = 1.f / sqrtf(sum_over_rows(kk) + a.eps);
            rq = 1.f / sqrtf(sum_over_rows(qq) + a.eps);
        }
        const float of = a.scale * rq;
        f4_t u, o;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            u[e] = rk * beta * fmaf(-rk * decay, sk[e], v[e]);
            o[e] = of * fmaf(kq, u[e], decay * sq[e]);
        }
#pragma unroll
        for (int r = 0; r < NR; r++)
#pragma unroll
            for (int e = 0; e < 4; e++) S[r][e] = fmaf(k[r / 4][r % 4], u[e], decay * S[r][e]);
        store_four<B16, VEC>(memory((const char*)a.out + ((size_t)t * a.H + h) * a.vdim * ELEM, a.vdim * ELEM), col * ELEM, o, lane < 8 ? cols : 0);
    }
#pragma unroll
    for (int r = 0; r < NR; r++) store_four<false, VEC, PAST>(memory(st, st_bytes), st_at + r * st_row, S[r], cols);
}

template <bool B16, int NR, bool VEC>
__global__ __launch_bounds__(64) void k_delta_step(Delta a) {
    const int4 span = span_of(a, blockIdx.y);
    const int slices = (a.vdim + STEP_COLS - 1) / STEP_COLS, h = blockIdx.x / slices;
    delta_step<B16, NR, VEC>(a, span, h, blockIdx.x - h * slices, threadIdx.x);
}

template <bool B16, bool VEC>
static void launch_step(const Delta& a) {
    const dim3 grid((unsigned)(cdiv(a.vdim, STEP_COLS) * a.H), a.n_spans);
    const int nr = cdiv(a.dim, 8);
    if (nr <= 4) NVLLM_LAUNCH((k_delta_step<B16, 4, VEC>), grid, dim3(64), 0, a);
    else if (nr <= 8) NVLLM_LAUNCH((k_delta_step<B16, 8, VEC>), grid, dim3(64), 0, a);
    else if (nr <= 12) NVLLM_LAUNCH((k_delta_step<B16, 12, VEC>), grid, dim3(64), 0, a);
    else if (nr <= 16) NVLLM_LAUNCH((k_delta_step<B16, 16, VEC>), grid, dim3(64), 0, a);
    else if (nr <= 24) NVLLM_LAUNCH((k_delta_step<B16, 24, VEC>), grid, dim3(64), 0, a);
    else NVLLM_LAUNCH((k_delta_step<B16, 32, VEC>), grid, dim3(64), 0, a);
}

// ------------------------------------------------------------------ chunks
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4_t lds_s4;
constexpr int CH = DELTA_CHUNK;
constexpr float MIN_G = -1e4f;   // e^MIN_G is zero, and differences of sums of it are numbers

// x = a + b + c, each rounded to the nearest bf16 of what is left: exact but for the 26th bit, and what a product of two leaves out has no
// sign of its own.  (Truncations, of the factors' own signs, left a bias: sums of 64 corrections to one key were off by 520 halves
// of a step.)
__device__ __forceinline__ u2_t next_part(f4_t& v) {   // the part of four values, and what it leaves of them
    u2_t p = {two_b16(v[0], v[1]), two_b16(v[2], v[3])};
    asm("" : "+v"(p));   // (the upper halves come from these registers, not from roundings of their own)
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const unsigned two = p[i];
        v[2 * i] -= __builtin_bit_cast(float, two << 16);
        v[2 * i + 1] -= __builtin_bit_cast(float, two & 0xffff0000u);
    }
    return p;
}
__device__ __forceinline__ void parts_of_four(f4_t v, u2_t (&out)[3]) {
#pragma unroll
    for (int k = 0; k < 3; k++) out[k] = next_part(v);
}
__device__ __forceinline__ void parts_of_eight(const f4_t& lo, const f4_t& hi, b8_t (&out)[3]) {
    u2_t l[3], h[3];
    parts_of_four(lo, l);
    parts_of_four(hi, h);
#pragma unroll
    for (int k = 0; k < 3; k++) out[k] = __builtin_bit_cast(b8_t, u4_t{l[k][0], l[k][1], h[k][0], h[k][1]});
}
__device__ __forceinline__ f4_t mfma(const b8_t& a, const b8_t& b, const f4_t& c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
// the six products of 32-bit values' parts, small ones first
__device__ __forceinline__ f4_t mfma6(const b8_t (&a)[3], const b8_t (&b)[3], f4_t c) {
    c = mfma(a[1], b[1], c);
    c = mfma(a[2], b[0], c);
    c = mfma(a[0], b[2], c);
    c = mfma(a[1], b[0], c);
    c = mfma(a[0], b[1], c);
    return mfma(a[0], b[0], c);
}
__device__ __forceinline__ f4_t mfma4(float a, float b, const f4_t& c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
// Sums of g in units of log2(e): two floats, so that differences of neighbouring tokens' keep 32 bits however far the sums have come.
struct Sum2 {
    float hi, lo;
};
__device__ __forceinline__ float exp_of(const Sum2& a, const Sum2& b) { return __builtin_amdgcn_exp2f((a.hi - b.hi) + (a.lo - b.lo)); }
template <int CTRL>
__device__ __forceinline__ double from_lane(double x) {   // zeros from outside the row of lanes
    const long v = __builtin_bit_cast(long, x);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, (long)(unsigned)lo | (long)hi << 32);
}
__device__ __forceinline__ double scalar_of(double x, int lane) {
    const long v = __builtin_bit_cast(long, x);
    return __builtin_bit_cast(double, (long)(unsigned)__builtin_amdgcn_readlane((int)v, lane) | (long)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32);
}
// the sum over the wave's lanes up to this one
__device__ __forceinline__ double sum_up_to(double x, int lane) {
    x += from_lane<0x111>(x);   // row_shr:1, 2, 4, 8
    x += from_lane<0x112>(x);
    x += from_lane<0x114>(x);
    x += from_lane<0x118>(x);
    const double r0 = scalar_of(x, 15), r1 = r0 + scalar_of(x, 31), r2 = r1 + scalar_of(x, 47);
    return x + (lane < 16 ? 0.0 : lane < 32 ? r0 : lane < 48 ? r1 : r2);
}

// A token's row of queries or keys as operands: lane (x, g) has dims 32 cc + 8 g .. + 7 of the tile's row x.
template <int DC, bool B16>
struct Rows {
    static constexpr int W = B16 ? 1 : 2;
    u4_t w[DC][W];
    // row: the offset of a token's row in bytes
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t m, unsigned row, int dim, int g) {
#pragma unroll
        for (int cc = 0; cc < DC; cc++) {
            const unsigned d = 32 * cc + 8 * g, at = (int)d < dim ? row + d * (B16 ? 2 : 4) : NOWHERE;
#pragma unroll
            for (int i = 0; i < W; i++) w[cc][i] = load16(m, at + 16 * i);
        }
    }
    __device__ __forceinline__ void operand(int cc, b8_t (&p)[B16 ? 1 : 3]) const {
        if constexpr (B16) p[0] = __builtin_bit_cast(b8_t, w[cc][0]);
        else parts_of_eight(__builtin_bit_cast(f4_t, w[cc][0]), __builtin_bit_cast(f4_t, w[cc][1]), p);
    }
    __device__ __forceinline__ float squares() const {   // of this lane's values
        float s = 0.f;
#pragma unroll
        for (int cc = 0; cc < DC; cc++)
#pragma unroll
            for (int i = 0; i < W; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const unsigned bits = w[cc][i][e];   // (a value: the cast of a vector's element in place takes the first one)
                    if (B16) {
                        const float lo = __builtin_bit_cast(float, bits << 16), hi = __builtin_bit_cast(float, bits & 0xffff0000u);
                        s = fmaf(lo, lo, fmaf(hi, hi, s));
                    } else {
                        const float v = __builtin_bit_cast(float, bits);
                        s = fmaf(v, v, s);
                    }
                }
        return s;
    }
};
// products over all dims: rows of a, columns of b
template <bool B16>
__device__ __forceinline__ f4_t mfma_rows(const b8_t (&a)[B16 ? 1 : 3], const b8_t (&b)[B16 ? 1 : 3], f4_t c) {
    if constexpr (B16) return mfma(a[0], b[0], c);
    else return mfma6(a, b, c);
}

// ... and its first record
struct Portion {
    int4 span;
    int first;
};
__device__ __forceinline__ Portion portion_of(const DeltaChunks& c, int s) {
    const int at = min(s, DELTA_SPANS - 1);
    Portion p = {c.a.here[at], c.first_here[at]};
    ASKED_FOR_AT_ONCE(c.a);
    asm volatile("" ::"s"(p.span.x), "s"(p.span.y), "s"(p.span.z), "s"(p.span.w), "s"(p.first), "s"(c.mem), "s"(c.first), "s"(c.from), "s"(c.most), "s"(c.segs), "s"(c.per_seg), "s"(c.out_four),
                 "s"(c.a.out), "s"(c.a.v_cols), "s"(c.a.dim_kept), "s"(c.a.n_spans));
    if (c.a.spans) {   // (s may be a segment's number: those go further than portions, whose own is looked up then)
        const int own = min(s, c.a.n_spans - 1);
        p = {c.a.spans[own], c.first[own]};
    }
    return {scalars(p.span), __builtin_amdgcn_readfirstlane(p.first)};
}
struct ChunkAt {
    int4 span;
    int first, n;   // token of the batch, tokens
    char* record;
};
__device__ __forceinline__ ChunkAt chunk_at(const DeltaChunks& c, int s, int h, int i) {
    ChunkAt at;
    const Portion p = portion_of(c, s);
    at.span = p.span;
    at.first = at.span.x + (c.from + i) * CH;
    at.n = min(CH, at.span.y - (c.from + i) * CH);
    at.record = c.mem + ((size_t)(p.first + i) * c.a.H + h) * DELTA_RECORD;
    return at;
}
// T' and P: tile (token tile w, 32 tokens p) of the six that are not empty
__device__ __forceinline__ int op_tile(int w, int p) { return w < 2 ? w : 2 * w - 2 + p; }

constexpr int LD = CH + 4;   // floats of a row of A or T in LDS
// keys as operands, in whose place T comes later; A; sums of g, what norms a key, beta
template <int DC, bool B16>
constexpr int prepare_keys() { return std::max(4 * DC * (B16 ? 1 : 3) * 1024, CH * LD * 4); }
template <int DC, bool B16>
constexpr int prepare_lds() { return prepare_keys<DC, B16>() + CH * LD * 4 + CH * (8 + 4 + 4); }

// A workgroup = (portion, chunk, head), four waves of 16 tokens each.  A and P by the matrix cores, A in LDS for the inverse, whose sums are of
// 32-bit products.  Bound by memory where chunks are many: 4,096 of 128 dims in bf16 move 230 MB in 50 us; few take 7 to 8 us, the
// inverse's substitutions, one behind the other.
template <int DC, bool B16, bool STEPS>
__global__ __launch_bounds__(256) void k_delta_prepare(DeltaChunks c) {
    constexpr int PARTS = B16 ? 1 : 3;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds_d[];
    u4_t* s_k = reinterpret_cast<u4_t*>(lds_d);                            // [token tile][DC][part][64]
    float* s_T = reinterpret_cast<float*>(lds_d);                          // [t][LD]
    float* s_A = reinterpret_cast<float*>(lds_d + prepare_keys<DC, B16>());
    Sum2* s_G = reinterpret_cast<Sum2*>(s_A + CH * LD);
    float* s_r = reinterpret_cast<float*>(s_G + CH);                       // what norms a key
    float* s_b = s_r + CH;
    const Delta& a = c.a;
    if (STEPS && (int)blockIdx.z >= a.n_spans) {   // portions that go token by token, behind the others
        const int wave = (((blockIdx.z - a.n_spans) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (wave < c.step_waves) {
            const int slices = (a.vdim + STEP_COLS - 1) / STEP_COLS, i = wave / slices, s = i / a.H;
            delta_step<B16, 4 * DC, true>(a, span_of(a, a.n_spans + s), i - s * a.H, wave - i * slices, threadIdx.x & 63);
        }
        return;
    }
    const int h = blockIdx.x;
    const ChunkAt at = chunk_at(c, blockIdx.z, h, blockIdx.y);
    const int hq = h / (a.H / a.Q);
    if (at.n <= 0) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), x = lane & 15, g = lane >> 4;
    const int t = 16 * w + x;
    constexpr int ELEM = B16 ? 2 : 4;
    Rows<DC, B16> k, q;
    auto rows_of = [&](const void* base, long ld) { return memory((const char*)base + ((size_t)at.first * ld + hq * a.dim) * ELEM, ((at.n - 1) * ld + a.dim) * ELEM); };
    const auto gates = [&](const float* base) { return load4(memory(base + (size_t)at.first * a.H + h, ((long)(at.n - 1) * a.H + 1) * 4), (unsigned)lane * a.H * 4); };
    const float gl = gates(a.g), bl = gates(a.beta);   // (zeros behind the last token)
    k.load(rows_of(a.k, a.k_ld), (unsigned)t * (unsigned)a.k_ld * ELEM, a.dim, g);
    q.load(rows_of(a.q, a.q_ld), (unsigned)t * (unsigned)a.q_ld * ELEM, a.dim, g);
    if (w == 0) {
        const double G = sum_up_to((double)(gl < MIN_G ? MIN_G : gl) * 1.4426950408889634, lane);
        const float hi = (float)G;
        s_G[lane] = Sum2{hi, (float)(G - (double)hi)};
        s_b[lane] = bl;
    }
    float rk = 1.f, rq = 1.f;
    if (a.eps > 0.f) {
        float kk = k.squares(), qq = q.squares();
        kk += __shfl_xor(kk, 16, 64);
        qq += __shfl_xor(qq, 16, 64);
        kk += __shfl_xor(kk, 32, 64);
        qq += __shfl_xor(qq, 32, 64);
        rk = 1.f / sqrtf(kk + a.eps);
        rq = 1.f / sqrtf(qq + a.eps);
    }
    if (g == 0) s_r[t] = rk;
    b8_t ko[DC][PARTS], qo[DC][PARTS];
#pragma unroll
    for (int cc = 0; cc < DC; cc++) {
        k.operand(cc, ko[cc]);
        q.operand(cc, qo[cc]);
#pragma unroll
        for (int p = 0; p < PARTS; p++) s_k[((w * DC + cc) * PARTS + p) * 64 + lane] = __builtin_bit_cast(u4_t, ko[cc][p]);
    }
    __syncthreads();
    // rows s of tile i, columns t of tile w
    const Sum2 Gt = s_G[t], none = {0.f, 0.f};
    const float bt = s_b[t] * rk, qt = a.scale * rq;
    f4_t kq[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f4_t kk = {0.f, 0.f, 0.f, 0.f};
        kq[i] = f4_t{0.f, 0.f, 0.f, 0.f};
        if (i <= w) {
#pragma unroll
            for (int cc = 0; cc < DC; cc++) {
                b8_t r[PARTS];
#pragma unroll
                for (int p = 0; p < PARTS; p++) r[p] = __builtin_bit_cast(b8_t, s_k[((i * DC + cc) * PARTS + p) * 64 + lane]);
                kk = mfma_rows<B16>(r, ko[cc], kk);
                kq[i] = mfma_rows<B16>(r, qo[cc], kq[i]);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int s = 16 * i + 4 * g + r;
                const float f = exp_of(Gt, s_G[s]) * s_r[s];   // (not used where s lies behind t)
                kk[r] = s < t ? bt * f * kk[r] : 0.f;
                kq[i][r] = s <= t ? qt * f * kq[i][r] : 0.f;
            }
        }
        *reinterpret_cast<f4_t*>(s_A + t * LD + 16 * i + 4 * g) = kk;
    }
    u4_t* ops = reinterpret_cast<u4_t*>(at.record) + lane;
#pragma unroll
    for (int p = 0; p < 2; p++)
        if (p <= w >> 1) {
            b8_t parts[3];
            parts_of_eight(kq[2 * p], kq[2 * p + 1], parts);
#pragma unroll
            for (int j = 0; j < 3; j++) ops[((6 + op_tile(w, p)) * 3 + j) * 64] = __builtin_bit_cast(u4_t, parts[j]);
        }
    if (threadIdx.x < CH) {   // (wave 0: t is not this thread's token)
        float* f = reinterpret_cast<float*>(at.record + DELTA_OPS);
        const int tok = threadIdx.x;
        f[tok] = exp_of(s_G[tok], none) * s_r[tok];
        f[2 * CH + tok] = exp_of(s_G[CH - 1], s_G[tok]) * s_r[tok];
        if (tok == 0) f[3 * CH] = exp_of(s_G[CH - 1], none);
    }
    if (g == 0) reinterpret_cast<float*>(at.record + DELTA_OPS)[CH + t] = qt * exp_of(Gt, none);
    __syncthreads();
    // (I + A)^-1: first the four blocks on the diagonal, by one wave: lane (x, g) has column x of block g, and row x of its A, whose
    // values the row of lanes shares (by a fused move; one LDS read after the other took 7,000 clocks, scalars 2,800).
    if (w == 0) {
        f4_t A[4];
        float col[16];
#pragma unroll
        for (int i = 0; i < 4; i++) A[i] = *reinterpret_cast<const f4_t*>(s_A + (16 * g + x) * LD + 16 * g + 4 * i);
#pragma unroll
        for (int i = 0; i < 16; i++) col[i] = i == x ? 1.f : 0.f;
        // (row_newbcast: the value of lane i of each row of lanes)
#define COLUMN_STEP(S, I) \
    if (I > S) col[I] = fmaf(-__builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, as), 0x150 + I, 0xf, 0xf, true)), col[S], col[I]);
#define COLUMN(S)                                                                                                                                       \
    {                                                                                                                                                   \
        const float as = A[S / 4][S % 4];                                                                                                               \
        COLUMN_STEP(S, 1) COLUMN_STEP(S, 2) COLUMN_STEP(S, 3) COLUMN_STEP(S, 4) COLUMN_STEP(S, 5) COLUMN_STEP(S, 6) COLUMN_STEP(S, 7) COLUMN_STEP(S, 8) \
        COLUMN_STEP(S, 9) COLUMN_STEP(S, 10) COLUMN_STEP(S, 11) COLUMN_STEP(S, 12) COLUMN_STEP(S, 13) COLUMN_STEP(S, 14) COLUMN_STEP(S, 15)             \
    }
        COLUMN(0) COLUMN(1) COLUMN(2) COLUMN(3) COLUMN(4) COLUMN(5) COLUMN(6) COLUMN(7) COLUMN(8) COLUMN(9) COLUMN(10) COLUMN(11) COLUMN(12) COLUMN(13) COLUMN(14)
#undef COLUMN
#undef COLUMN_STEP
#pragma unroll
        for (int i = 0; i < 16; i++) s_T[(16 * g + i) * LD + 16 * g + x] = col[i];
    }
    __syncthreads();
    // ... then the blocks under it, block column w by wave w, from the top: T_iw = -T_ii sum_j A_ij T_jw, every T_jw added to all sums
    // below as soon as it is there.  (k of these products runs 4 g + step, as results lie)
    {
        f4_t T, sum[4] = {};
#pragma unroll
        for (int r = 0; r < 4; r++) T[r] = s_T[(16 * w + 4 * g + r) * LD + 16 * w + x];
#pragma unroll
        for (int j = 0; j < 3; j++) {
            if (w + j >= 3) break;
#pragma unroll
            for (int i = j + 1; i < 4; i++) {
                if (w + i >= 4) break;
                const f4_t A = *reinterpret_cast<const f4_t*>(s_A + (16 * (w + i) + x) * LD + 16 * (w + j) + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; e++) sum[i] = mfma4(A[e], T[e], sum[i]);
            }
            asm volatile("s_nop 15" : "+v"(sum[j + 1]));   // (it has come over a branch)
            const int row = 16 * (w + j + 1);
            const f4_t D = *reinterpret_cast<const f4_t*>(s_T + (row + x) * LD + row + 4 * g);
            T = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; e++) T = mfma4(-D[e], sum[j + 1][e], T);
#pragma unroll
            for (int r = 0; r < 4; r++) s_T[(row + 4 * g + r) * LD + 16 * w + x] = T[r];
        }
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 2; p++)
        if (p <= w >> 1) {
            f4_t v[2];
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int s0 = 32 * p + 16 * half + 4 * g;
                v[half] = f4_t{0.f, 0.f, 0.f, 0.f};
                if (2 * p + half <= w) v[half] = *reinterpret_cast<const f4_t*>(s_T + t * LD + s0);
#pragma unroll
                for (int r = 0; r < 4; r++) v[half][r] = v[half][r] * s_b[s0 + r];
            }
            b8_t parts[3];
            parts_of_eight(v[0], v[1], parts);
#pragma unroll
            for (int j = 0; j < 3; j++) ops[(op_tile(w, p) * 3 + j) * 64] = __builtin_bit_cast(u4_t, parts[j]);
        }
}

// A workgroup = (portion, head, 16 value columns), eight waves.
//   0 .. 3, the chain, in which every chunk waits for the last one: wave w keeps the state's 32 dims w (and w + 4) in registers and
//     forms their share of S^T k for all 64 tokens; the shares meet in LDS, wave w goes on with tokens 16 w .. + 15 up to U, which all
//     of them take for their dims.  A state's two tiles of 16 dims have dim 8 g + 4 half + r of the 32 in row 4 g + r, so that a lane's
//     eight values are the k of one operand and 16 bytes of a row of keys are the other.
//   4, 5, the results of 32 tokens each, from the state and U as the chain leaves them in LDS.
//   6, 7 bring keys, values, T' and factors of coming chunks from memory, one or two chunks ahead, and lay them out in LDS: the chain
//     itself asks memory for nothing.
// Three barriers a chunk (a fourth where LDS holds one chunk's keys only).  Bound by the chain: a chunk of 128 x 128 in bf16 takes 1.6 us,
// 3,300 clocks, in which LDS is busy for 1,750 (400 of them conflicts) and a SIMD's matrix core for 960; the exchanges and their barriers
// cost the rest.  The results' waves add a fifth to what the chain would take alone, the loaders' work 4 %.  Sixteen columns are
// the fewest that the products take: more workgroups for the same heads, each as long.
//
// A portion's chunks may be cut into segments that are walked side by side: scouts (RESULTS false) find out what a segment makes of an empty
// state (the first one: of the portion's) and, for columns of the unit matrix, what becomes of a state over it, k_delta_join forms the
// states that segments start from, and they are walked from there.
template <int DC, bool B16>
struct Walk {
    static constexpr int PARTS = B16 ? 1 : 3;
    static constexpr int STATE = DC * DELTA_TILE, SHARES = (DC < 4 ? DC : 4) * 4096, EX = 2 * DELTA_TILE, KEYS = DC * PARTS * 4096, OPS = 7 * DELTA_TILE, VALUES = 4096, FACTORS = 1024;
    static constexpr int REST = STATE + SHARES + 3 * EX + VALUES + FACTORS, MOST = 160 * 1024;
    static constexpr bool STAGED = REST + KEYS + OPS <= MOST;                          // T' goes through LDS
    static constexpr int BUFFERS = REST + EX + 2 * KEYS + OPS <= MOST ? 2 : 1;         // of keys and of U
    static constexpr int LDS = REST + (BUFFERS - 1) * EX + BUFFERS * KEYS + (STAGED ? OPS : 0);
    static constexpr bool PAIR = B16 && 2 * LDS <= MOST;   // two workgroups on a CU
};

template <int DC, bool B16, bool RESULTS>
__global__ __launch_bounds__(512, (Walk<DC, B16>::PAIR ? 4 : 2)) void k_delta_chunks(DeltaChunks c) {
    typedef Walk<DC, B16> L;
    constexpr int PARTS = L::PARTS, OWN = (DC + 3) / 4, SHARES = DC < 4 ? DC : 4, ELEM = B16 ? 2 : 4;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds_d[];
    u4_t* s_S = reinterpret_cast<u4_t*>(lds_d);            // [DC][part][64] the state as operand
    f4_t* s_D = reinterpret_cast<f4_t*>(s_S + DC * 192);   // [wave][token tile][64] shares of S^T k
    u4_t* s_X = reinterpret_cast<u4_t*>(s_D + SHARES * 256);    // [32 tokens][part][64]
    u4_t* s_U = s_X + 6 * 64;                              // [buffer]
    u4_t* s_V = s_U + L::BUFFERS * 6 * 64;                 // U as the state takes it
    u4_t* s_v = s_V + 6 * 64;                              // [token][16] values
    float* s_f = reinterpret_cast<float*>(s_v + 4 * 64);   // factors a, c, what is left of the state
    u4_t* s_k = reinterpret_cast<u4_t*>(s_f + 256);        // [buffer][DC][part][token][4] keys, 32 dims together
    u4_t* s_t = s_k + L::BUFFERS * DC * PARTS * 256;       // T', and a tile of zeros
    const Delta& a = c.a;
    int of = blockIdx.z;
    Portion portion = portion_of(c, of);
    if (c.segs > 1) {
        of = blockIdx.z / c.segs;
        portion = portion_of(c, of);
    }
    const int h = blockIdx.x, hq = h / (a.H / a.Q), seg = blockIdx.z - of * c.segs;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), x = lane & 15, g = lane >> 4;
    const int4 span = portion.span;
    const int all = min(c.most, (span.y + CH - 1) / CH - c.from), c0 = seg * c.per_seg, chunks = min(c.per_seg, all - c0);
    const int slices = (a.vdim + 15) / 16;
    const bool unit = !RESULTS && (int)blockIdx.y >= slices;   // columns of the unit matrix
    if (chunks <= 0 || (!RESULTS && (c0 + chunks >= all || (unit && seg == 0)))) return;
    const int slice = unit ? blockIdx.y - slices : blockIdx.y;
    const int first = span.x + (c.from + c0) * CH, tokens = min(span.y - (c.from + c0) * CH, chunks * CH);
    const char* record = c.mem + ((size_t)(portion.first + c0) * a.H + h) * DELTA_RECORD;
    auto rows_of = [&](const void* base, long ld, int at, int i, int width) {   // of chunk i's tokens; behind the last chunk: the last one's
        const int ci = min(i, chunks - 1), n = min(CH, tokens - ci * CH);
        return memory((const char*)base + ((size_t)(first + ci * CH) * ld + at) * ELEM, ((n - 1) * ld + width) * ELEM);
    };
    auto record_of = [&](int i) { return memory(record + (size_t)min(i, chunks - 1) * a.H * DELTA_RECORD, DELTA_RECORD); };
    auto get = [&](const u4_t* from, b8_t (&p)[3]) {
#pragma unroll
        for (int j = 0; j < 3; j++) p[j] = __builtin_bit_cast(b8_t, from[j * 64 + lane]);
    };
    const f4_t zero = {0.f, 0.f, 0.f, 0.f};

    if (wave < 4) {
        // ================================================================ the chain
        const int w = wave, col = slice * 16 + x, columns = slices * 16;   // columns: of a start
        float* start = c.starts + ((size_t)(of * c.segs + seg) * a.H + h) * (32 * DC) * columns;
        float* st = a.state + ((size_t)span.w * a.H + h) * a.dim_kept * a.vdim;
        // (a portion of one segment has no scouts)
        const bool from_start = RESULTS && chunks < all, from_slot = RESULTS ? !from_start : !unit && seg == 0, keeps = from_slot && span.z + c.from > 0;
        f4_t S[OWN][2];
#pragma unroll
        for (int j = 0; j < OWN; j++)
#pragma unroll
            for (int half = 0; half < 2; half++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int d = 32 * (w + 4 * j) + 8 * g + 4 * half + r;
                    float v = unit && d == col ? 1.f : 0.f;
                    if (d < 32 * DC) {
                        if (keeps && col < a.vdim && d < a.dim_kept) v = st[(size_t)d * a.vdim + col];
                        if (from_start) v = start[(size_t)d * columns + col];
                        if (!RESULTS && seg == 0) start[(size_t)d * columns + col] = v;   // (another workgroup writes the slot later on)
                    }
                    S[j][half][r] = v;
                }
        auto put = [&](u4_t* to, const f4_t& val) {   // [part][64] operands: this tile's half of a lane's eight values
            u2_t parts[3];
            parts_of_four(val, parts);
#pragma unroll
            for (int p = 0; p < 3; p++) reinterpret_cast<u2_t*>(to + p * 64 + lane)[w & 1] = parts[p];
        };
        const unsigned op0 = op_tile(w, 0) * DELTA_TILE + lane * 16, op1 = w >= 2 ? op0 + DELTA_TILE : NOWHERE;   // (no tokens behind the wave's own)
        b8_t to[2][3];
        auto fetch_ops = [&](int i) {
            const auto m = record_of(i);
#pragma unroll
            for (int j = 0; j < 3; j++) {
                to[0][j] = __builtin_bit_cast(b8_t, load16(m, op0 + j * DELTA_PART));
                to[1][j] = __builtin_bit_cast(b8_t, load16(m, op1 + j * DELTA_PART));
            }
        };
        b8_t k[OWN][4][PARTS];
        auto keys_of = [&](int i) { return s_k + (L::BUFFERS == 2 ? i & 1 : 0) * DC * PARTS * 256; };
        auto read_keys = [&](int i, int j) {
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int p = 0; p < PARTS; p++) k[j][t][p] = __builtin_bit_cast(b8_t, keys_of(i)[(((w + 4 * j) * PARTS + p) * CH + 16 * t + x) * 4 + g]);
        };
        if (!L::STAGED) fetch_ops(0);
        __syncthreads();
        if (L::BUFFERS == 2)
#pragma unroll
            for (int j = 0; j < OWN; j++)
                if (DC % 4 == 0 || w + 4 * j < DC) read_keys(0, j);
        for (int i = 0; i < chunks; i++) {
            // ---- shares of S^T k, each part of the state as soon as it is there
            f4_t D[4] = {zero, zero, zero, zero};
#pragma unroll
            for (int j = 0; j < OWN; j++) {
                const int cc = w + 4 * j;
                if (DC % 4 != 0 && cc >= DC) break;
                if (L::BUFFERS == 1) read_keys(i, j);
                b8_t s[3];
                if constexpr (B16) {
                    f4_t lo = S[j][0], hi = S[j][1];
#pragma unroll
                    for (int p = 0; p < 3; p++) {
                        const u2_t l = next_part(lo), u = next_part(hi);
                        s[p] = __builtin_bit_cast(b8_t, u4_t{l[0], l[1], u[0], u[1]});
#pragma unroll
                        for (int t = 0; t < 4; t++) D[t] = mfma(k[j][t][0], s[p], D[t]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else {
                    parts_of_eight(S[j][0], S[j][1], s);
#pragma unroll
                    for (int t = 0; t < 4; t++) D[t] = mfma6(k[j][t], s, D[t]);
                }
#pragma unroll
                for (int p = 0; p < 3; p++)
                    if (RESULTS) s_S[(cc * 3 + p) * 64 + lane] = __builtin_bit_cast(u4_t, s[p]);
            }
            if (DC % 4 != 0) asm volatile("s_nop 15" : "+v"(D[0]), "+v"(D[1]), "+v"(D[2]), "+v"(D[3]));   // (they have come over a branch)
            if (SHARES == 4 || w < SHARES)
#pragma unroll
                for (int t = 0; t < 4; t++) s_D[(w * 4 + t) * 64 + lane] = D[t];
            __syncthreads();
            // ---- X of the wave's tokens; T' and factors are read behind the shares, in front of their sums
            f4_t d[SHARES];
#pragma unroll
            for (int j = 0; j < SHARES; j++) d[j] = s_D[(j * 4 + w) * 64 + lane];
            const f4_t fa = *reinterpret_cast<const f4_t*>(s_f + 16 * w + 4 * g);
            f4_t v;   // tokens 4 g .. + 3 of column x
            if constexpr (B16) {
                const u2_t two = __builtin_bit_cast(u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(reinterpret_cast<unsigned short*>(s_v) + (16 * w + 4 * g + (x >> 2)) * 16 + 4 * (x & 3))));
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const unsigned bits = r & 1 ? two[r >> 1] & 0xffff0000u : two[r >> 1] << 16;
                    v[r] = __builtin_bit_cast(float, bits);
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++) v[r] = reinterpret_cast<const float*>(s_v)[(16 * w + 4 * g + r) * 16 + x];
            }
            if (L::STAGED) {
                get(s_t + op_tile(w, 0) * 192, to[0]);
                get(s_t + (w >= 2 ? op_tile(w, 1) : 6) * 192, to[1]);   // (no tokens behind the wave's own)
            }
            const f4_t fc = *reinterpret_cast<const f4_t*>(s_f + 64 + 16 * w + 4 * g);
            const float left = s_f[128];
            __builtin_amdgcn_sched_barrier(0);
            f4_t X = d[0];
#pragma unroll
            for (int j = 1; j < SHARES; j++) X += d[j];
#pragma unroll
            for (int r = 0; r < 4; r++) X[r] = fmaf(-fa[r], X[r], v[r]);
            put(s_X + (w >> 1) * 192, X);
            __syncthreads();
            // ---- U = T' X
            // (without a branch for waves 0 and 1: results of the matrix cores that come to their first reader over a branch are not
            // waited for by the compiler, which left tokens of these waves without their first columns' sums)
            b8_t e[2][3];
            get(s_X, e[0]);
            get(s_X + 192, e[1]);
            // Keys as columns (16 lanes bring 4 tokens x 16 dims, lane x receives dim x of the four), and the next chunk's.  Where they are
            // many and of one part they are asked for behind U's products, which need not wait for them (LDS gives 128 bytes a clock to
            // all waves: 16 heads of 128 x 128 over 8,192 tokens 230 -> 222 us; in 32 bits and for 64 dims it costs 1 %).
            constexpr bool LATE = B16 && DC % 4 == 0;
            b8_t kt[OWN][2][2][PARTS];
            auto read_columns = [&] {
#pragma unroll
                for (int j = 0; j < OWN; j++) {
                    const int cc = w + 4 * j;
                    if (DC % 4 != 0 && cc >= DC) break;
#pragma unroll
                    for (int half = 0; half < 2; half++)
#pragma unroll
                        for (int p = 0; p < 2; p++)
#pragma unroll
                            for (int part = 0; part < PARTS; part++) {
                                const u2_t* at = reinterpret_cast<const u2_t*>(keys_of(i) + ((cc * PARTS + part) * CH + 32 * p + 4 * g + (x >> 2)) * 4 + (x & 3)) + half;
                                const u2_t lo = __builtin_bit_cast(u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)at));
                                const u2_t hi = __builtin_bit_cast(u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + 16 * 8)));
                                kt[j][half][p][part] = __builtin_bit_cast(b8_t, u4_t{lo[0], lo[1], hi[0], hi[1]});
                            }
                    if (!LATE && L::BUFFERS == 2) read_keys(i + 1, j);
                }
            };
            if (!LATE) read_columns();
            __builtin_amdgcn_sched_barrier(0);
            f4_t U0 = mfma(to[0][1], e[0][1], zero), U1 = mfma(to[0][1], e[0][0], zero), U2 = mfma(to[1][1], e[1][1], zero), U3 = mfma(to[1][1], e[1][0], zero);
            U0 = mfma(to[0][2], e[0][0], U0);
            U1 = mfma(to[0][0], e[0][1], U1);
            U2 = mfma(to[1][2], e[1][0], U2);
            U3 = mfma(to[1][0], e[1][1], U3);
            U0 = mfma(to[0][0], e[0][2], U0);
            U1 = mfma(to[0][0], e[0][0], U1);
            U2 = mfma(to[1][0], e[1][2], U2);
            U3 = mfma(to[1][0], e[1][0], U3);
            if (LATE) {
                __builtin_amdgcn_sched_barrier(0);
                read_columns();
                __builtin_amdgcn_sched_barrier(0);
            }
            const f4_t U = (U0 + U2) + (U1 + U3);
            put(s_V + (w >> 1) * 192, U * fc);
#pragma unroll
            for (int j = 0; j < OWN; j++) {
                S[j][0] *= left;
                S[j][1] *= left;
            }
            if (!L::STAGED) fetch_ops(i + 1);
            __syncthreads();
            // ---- the state
            get(s_V, e[0]);
            get(s_V + 192, e[1]);
            if (LATE && L::BUFFERS == 2) {
#pragma unroll
                for (int j = 0; j < OWN; j++) read_keys(i + 1, j);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int j = 0; j < OWN; j++) {
                const int cc = w + 4 * j;
                if (DC % 4 != 0 && cc >= DC) break;
                if constexpr (B16) {
                    f4_t more[2] = {zero, zero};
#pragma unroll
                    for (int part = 0; part < 3; part++)
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            S[j][half] = mfma(kt[j][half][0][0], e[0][part], S[j][half]);
                            more[half] = mfma(kt[j][half][1][0], e[1][part], more[half]);
                        }
                    S[j][0] += more[0];
                    S[j][1] += more[1];
                } else {
#pragma unroll
                    for (int half = 0; half < 2; half++) S[j][half] = mfma6(kt[j][half][1], e[1], mfma6(kt[j][half][0], e[0], S[j][half]));
                    asm volatile("s_nop 15" : "+v"(S[j][0]), "+v"(S[j][1]));   // (the way round the loop is a branch)
                }
            }
            if (RESULTS) put(s_U + (L::BUFFERS == 2 ? i & 1 : 0) * 384 + (w >> 1) * 192, U);   // (for the results: nobody here waits for it)
            if (L::BUFFERS == 1) __syncthreads();
        }
        __syncthreads();   // U is there
        if (RESULTS && c0 + chunks < all) return;
        float* out = RESULTS ? st : unit ? c.trans + ((size_t)(of * c.segs + seg) * a.H + h) * (32 * DC) * (32 * DC) : start + (size_t)a.H * (32 * DC) * columns;
        const int ld = RESULTS ? a.vdim : unit ? 32 * DC : columns;
#pragma unroll
        for (int j = 0; j < OWN; j++)
#pragma unroll
            for (int half = 0; half < 2; half++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int d = 32 * (w + 4 * j) + 8 * g + 4 * half + r;
                    if (RESULTS ? col < a.vdim && d < a.dim_kept : d < 32 * DC) out[(size_t)d * ld + col] = S[j][half][r];
                }
    } else if (!RESULTS && wave < 6) {
        for (int i = 0; i < (L::BUFFERS == 1 ? 4 : 3) * chunks + 2; i++) __syncthreads();   // (nothing to do but to be counted)
    } else if (wave < 6) {
        // ================================================================ results: lane (x, g) has tokens 16 t + x, columns 4 g .. + 3
        const int t0 = 2 * (wave - 4);   // token tiles t0, t0 + 1
        const unsigned o_row = ((16 * t0 + x) * (unsigned)(a.H * a.vdim) + 4 * g) * ELEM, o_tile = 16 * (unsigned)(a.H * a.vdim) * ELEM;
        bool has_out[4];
#pragma unroll
        for (int e = 0; e < 4; e++) has_out[e] = slice * 16 + 4 * g + e < a.vdim;
        struct Set {
            Rows<DC, B16> q[2];
            float fb[2];
            b8_t po[2][2][3];
        };
        constexpr int SETS = !L::PAIR && sizeof(Set) / 4 <= 84 ? 2 : 1;   // (chunks in flight: what fits the registers)
        Set set[SETS];
        auto fetch_queries = [&](Set& s, int i) {
            const auto m = record_of(i);
            const auto mq = rows_of(a.q, a.q_ld, hq * a.dim, i, a.dim);
#pragma unroll
            for (int t = 0; t < 2; t++) {
                s.fb[t] = load4(m, DELTA_OPS + (CH + 16 * (t0 + t) + x) * 4);
                s.q[t].load(mq, (16 * (t0 + t) + x) * (unsigned)a.q_ld * ELEM, a.dim, g);
            }
        };
        auto fetch_ops = [&](Set& s, int i) {
            const auto m = record_of(i);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int p = 0; p < 2; p++)
#pragma unroll
                    for (int j = 0; j < 3; j++)
                        s.po[t][p][j] = __builtin_bit_cast(b8_t, load16(m, p == 0 || t0 > 0 ? lane * 16 : NOWHERE, (6 + op_tile(t0 + t, p)) * DELTA_TILE + j * DELTA_PART));
        };
        f4_t o[2];
        auto finish = [&](const Set& s, int i) {   // chunk i's results: U has come
            b8_t e[2][3];
            const u4_t* U = s_U + (L::BUFFERS == 2 ? i & 1 : 0) * 384;
            get(U, e[0]);
            f4_t first[2];
            if (L::PAIR) {   // (one after the other: registers)
#pragma unroll
                for (int t = 0; t < 2; t++) first[t] = mfma6(e[0], s.po[t][0], o[t]);
                __builtin_amdgcn_sched_barrier(0);
            }
            get(U + 192, e[1]);
            const auto m = rows_of(a.out, (long)a.H * a.vdim, h * a.vdim + slice * 16, i, min(16, a.vdim - slice * 16));
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const f4_t y = L::PAIR ? mfma6(e[1], s.po[t][1], first[t]) : mfma6(e[0], s.po[t][0], o[t]) + mfma6(e[1], s.po[t][1], zero);
                const unsigned at = o_row + t * o_tile;
                if (c.out_four) {
                    if (B16) __builtin_amdgcn_raw_buffer_store_b64(u2_t{two_b16(y[0], y[1]), two_b16(y[2], y[3])}, m, (int)(has_out[0] ? at : NOWHERE), 0, 0);
                    else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, y), m, (int)(has_out[0] ? at : NOWHERE), 0, 0);
                } else {
#pragma unroll
                    for (int e1 = 0; e1 < 4; e1++) {
                        const float z = y[e1];
                        if (B16) __builtin_amdgcn_raw_buffer_store_b16((unsigned short)two_b16(z, z), m, (int)(has_out[e1] ? at + 2 * e1 : NOWHERE), 0, 0);
                        else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, z), m, (int)(has_out[e1] ? at + 4 * e1 : NOWHERE), 0, 0);
                    }
                }
            }
        };
#pragma unroll
        for (int n = 0; n < SETS; n++) {
            fetch_queries(set[n], n);
            fetch_ops(set[n], n);
        }
        __syncthreads();
        // (each piece where the chain has as much to do: nobody waits for results)
        auto step = [&](Set& mine, Set& before, int i) {
            f4_t O[2][2] = {{zero, zero}, {zero, zero}};
            auto meet = [&](int c0, int c1) {
#pragma unroll
                for (int cc = 0; cc < DC; cc++) {
                    if (cc < c0 || cc >= c1) continue;
                    b8_t s[3];
                    get(s_S + cc * 192, s);
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        b8_t qp[PARTS];
                        mine.q[t].operand(cc, qp);
                        if constexpr (B16) {
#pragma unroll
                            for (int p = 2; p >= 0; p--) O[t][p & 1] = mfma(s[p], qp[0], O[t][p & 1]);
                        } else O[t][cc & 1] = mfma6(s, qp, O[t][cc & 1]);
                    }
                }
            };
            __syncthreads();   // the state is there, and U of the chunk before
            meet(0, DC / 2);
            __syncthreads();
            meet(DC / 2, DC);
            f4_t now[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                now[t] = (O[t][0] + O[t][1]) * mine.fb[t];
                asm volatile("" : "+v"(now[t]));   // (here, not behind the branch below)
            }
            fetch_queries(mine, i + SETS);
            __syncthreads();
            if (L::BUFFERS == 1) __syncthreads();   // U is there
            if (L::BUFFERS == 2 && i > 0) {
                finish(before, i - 1);
                fetch_ops(before, i - 1 + SETS);
            }
            o[0] = now[0];
            o[1] = now[1];
            if (L::BUFFERS == 1) {
                finish(mine, i);
                fetch_ops(mine, i + SETS);
            }
        };
        for (int i = 0; i < chunks; i += SETS) {
            step(set[0], set[SETS - 1], i);
            if (SETS == 2 && i + 1 < chunks) step(set[SETS - 1], set[0], i + 1);
        }
        __syncthreads();
        if (L::BUFFERS == 2) {
            if (SETS == 2 && chunks % 2 == 0) finish(set[SETS - 1], chunks - 1);
            else finish(set[0], chunks - 1);
        }
    } else {
        // ================================================================ keys, values, T' and factors on their way to LDS
        const int tid = threadIdx.x - 384;   // of 128
        constexpr int ROW = DC <= 1 ? 4 : DC <= 2 ? 8 : DC <= 4 ? 16 : 32, ITEMS = CH * ROW / 128, W = B16 ? 1 : 2;   // a row's pieces of 8 dims, rounded up
        const int piece = tid % ROW, row = tid / ROW;   // items: tokens row + i * (128 / ROW)
        const bool has_piece = piece < 4 * DC;
        const unsigned k_at = 8 * piece < a.dim ? ((unsigned)row * (unsigned)a.k_ld + 8 * piece) * ELEM : NOWHERE, k_step = (128 / ROW) * (unsigned)a.k_ld * ELEM;
        // 16 bytes of a token's 16 values: thread 2 t (+ 1) of token t, in 32 bits 4 t' .. + 3 of tokens t' and 32 + t'
        const int v_col = slice * 16 + (B16 ? 8 * (tid & 1) : 4 * (tid & 3));
        const unsigned v_ld = (unsigned)a.v_ld * ELEM, v_at = v_col < a.v_cols && !unit ? (B16 ? (tid >> 1) * v_ld + 16 * (tid & 1) : (tid >> 2) * v_ld + 16 * (tid & 3)) : NOWHERE;
        const unsigned f_at = tid < 16 ? DELTA_OPS + tid * 16 : tid < 32 ? DELTA_OPS + 2 * CH * 4 + (tid - 16) * 16 : tid == 32 ? DELTA_OPS + 3 * CH * 4 : NOWHERE;
        struct Set {
            u4_t k[ITEMS][W], t[L::STAGED ? 9 : 1], f, v[W];
        };
        constexpr int SETS = !L::PAIR && sizeof(Set) / 4 <= 88 ? 2 : 1;   // (chunks in flight: what fits the registers)
        Set set[SETS];
        auto fetch_keys = [&](Set& s, int i) {
            const auto m = rows_of(a.k, a.k_ld, hq * a.dim, i, a.dim);
#pragma unroll
            for (int n = 0; n < ITEMS; n++)
#pragma unroll
                for (int e = 0; e < W; e++) s.k[n][e] = load16(m, k_at + n * k_step + 16 * e);
        };
        auto fetch_values = [&](Set& s, int i) {
            const auto m = rows_of(a.v, a.v_ld, h * a.v_cols + slice * 16, i, unit ? 0 : min(16, a.v_cols - slice * 16));
#pragma unroll
            for (int e = 0; e < W; e++) s.v[e] = load16(m, v_at + 32 * e * v_ld);
        };
        auto fetch_ops = [&](Set& s, int i) {
            const auto m = record_of(i);
            if (L::STAGED)
#pragma unroll
                for (int n = 0; n < 9; n++) s.t[n] = load16(m, (n * 128 + tid) * 16);
            s.f = load16(m, f_at);
        };
        auto lay_keys = [&](const Set& s, int i) {
            u4_t* keys = s_k + (L::BUFFERS == 2 ? i & 1 : 0) * DC * PARTS * 256 + (piece >> 2) * PARTS * 256 + row * 4 + (piece & 3);
#pragma unroll
            for (int n = 0; n < ITEMS; n++) {
                b8_t p[PARTS];
                if constexpr (B16) p[0] = __builtin_bit_cast(b8_t, s.k[n][0]);
                else parts_of_eight(__builtin_bit_cast(f4_t, s.k[n][0]), __builtin_bit_cast(f4_t, s.k[n][1]), p);
                if (has_piece)
#pragma unroll
                    for (int j = 0; j < PARTS; j++) keys[j * 256 + n * (128 / ROW) * 4] = __builtin_bit_cast(u4_t, p[j]);
            }
        };
        auto lay_values = [&](const Set& s) {
#pragma unroll
            for (int e = 0; e < W; e++) s_v[tid + 128 * e] = s.v[e];
            if (tid < 16) reinterpret_cast<u4_t*>(s_f)[tid] = s.f;
        };
        auto lay_ops = [&](const Set& s) {
            if (L::STAGED)
#pragma unroll
                for (int n = 0; n < 9; n++) s_t[n * 128 + tid] = s.t[n];
            if (tid >= 16 && tid <= 32) reinterpret_cast<u4_t*>(s_f)[tid] = s.f;
        };
        auto fetch = [&](Set& s, int i) {
            fetch_keys(s, i);
            fetch_values(s, i);
            fetch_ops(s, i);
        };
        fetch(set[0], 0);
        if (SETS == 2) fetch(set[1], 1);
        lay_keys(set[0], 0);
        lay_values(set[0]);
        lay_ops(set[0]);
        if (L::STAGED) {
            s_t[6 * 192 + tid] = u4_t{0, 0, 0, 0};
            if (tid < 64) s_t[6 * 192 + 128 + tid] = u4_t{0, 0, 0, 0};
        }
        fetch(set[0], SETS);
        __syncthreads();
        auto step = [&](Set& s, int i) {   // while chunk i is computed: chunk i + 1 to LDS, the one that is SETS behind it is asked for
            const int then = i + 1 + SETS;
            __syncthreads();
            if (L::BUFFERS == 2) {
                lay_keys(s, i + 1);
                fetch_keys(s, then);
            }
            __syncthreads();
            lay_values(s);
            fetch_values(s, then);
            __syncthreads();
            if (L::BUFFERS == 1) {
                lay_keys(s, i + 1);
                fetch_keys(s, then);
            }
            lay_ops(s);
            fetch_ops(s, then);
            if (L::BUFFERS == 1) __syncthreads();
        };
        for (int i = 0; i < chunks; i += SETS) {
            step(set[SETS - 1], i);
            if (SETS == 2 && i + 1 < chunks) step(set[0], i + 1);
        }
        __syncthreads();
    }
}

// The states that a portion's segments start from: start[e + 1] += trans[e] start[e], e = 1 .. (start[1] is complete).  A workgroup =
// (portion, head, 16 columns), wave w has dim tiles w, w + WAVES; rows of a tile as in k_delta_chunks.  Every step waits for the last one,
// so the next step's operands travel meanwhile.
template <int DC>
constexpr int join_waves() { return DC <= 6 ? 2 * DC : DC; }

template <int DC>
__global__ __launch_bounds__(64 * join_waves<DC>()) void k_delta_join(DeltaChunks c) {
    constexpr int WAVES = join_waves<DC>(), TILES = 2 * DC / WAVES;
    __shared__ u4_t s_S[DC * 192];
    const Delta& a = c.a;
    const int h = blockIdx.x, s = blockIdx.z, columns = (a.vdim + 15) & ~15, col0 = blockIdx.y * 16;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), x = lane & 15, g = lane >> 4;
    const int4 span = span_of(a, s);
    const int all = min(c.most, (span.y + CH - 1) / CH - c.from), segs = (all + c.per_seg - 1) / c.per_seg;
    if (segs < 3) return;
    const size_t step = (size_t)a.H * (32 * DC) * columns, t_step = (size_t)a.H * (32 * DC) * (32 * DC);
    float* start = c.starts + ((size_t)(s * c.segs) * a.H + h) * (32 * DC) * columns + col0 + x;
    const float* trans = c.trans + ((size_t)(s * c.segs) * a.H + h) * (32 * DC) * (32 * DC) + 8 * g;
    int tile[TILES];
#pragma unroll
    for (int j = 0; j < TILES; j++) tile[j] = w + WAVES * j;
    auto at = [&](int j, int r) { return (size_t)(32 * (tile[j] >> 1) + 8 * g + 4 * (tile[j] & 1) + r) * columns; };
    f4_t S[TILES], next[TILES], m[TILES][DC][2];
    auto fetch = [&](int e) {   // of the step from start e to start e + 1; behind the last step: its own again
        const int i = min(e, segs - 2);
#pragma unroll
        for (int j = 0; j < TILES; j++) {
#pragma unroll
            for (int r = 0; r < 4; r++) next[j][r] = start[(i + 1) * step + at(j, r)];
            const float* row = trans + i * t_step + (size_t)(32 * (tile[j] >> 1) + 8 * (x >> 2) + 4 * (tile[j] & 1) + (x & 3)) * (32 * DC);
#pragma unroll
            for (int cc = 0; cc < DC; cc++)
#pragma unroll
                for (int i2 = 0; i2 < 2; i2++) m[j][cc][i2] = *reinterpret_cast<const f4_t*>(row + 32 * cc + 4 * i2);
        }
    };
#pragma unroll
    for (int j = 0; j < TILES; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) S[j][r] = start[step + at(j, r)];
    fetch(1);
    for (int e = 1; e + 1 < segs; e++) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < TILES; j++) {
            u2_t parts[3];
            parts_of_four(S[j], parts);
#pragma unroll
            for (int p = 0; p < 3; p++) reinterpret_cast<u2_t*>(s_S + ((tile[j] >> 1) * 3 + p) * 64 + lane)[tile[j] & 1] = parts[p];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < TILES; j++) {
            f4_t sum[2] = {next[j], {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int cc = 0; cc < DC; cc++) {
                b8_t mp[3], sp[3];
                parts_of_eight(m[j][cc][0], m[j][cc][1], mp);
#pragma unroll
                for (int p = 0; p < 3; p++) sp[p] = __builtin_bit_cast(b8_t, s_S[(cc * 3 + p) * 64 + lane]);
                sum[cc & 1] = mfma6(mp, sp, sum[cc & 1]);
            }
            S[j] = sum[0] + sum[1];
        }
        fetch(e + 1);
#pragma unroll
        for (int j = 0; j < TILES; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) start[(e + 1) * step + at(j, r)] = S[j][r];
    }
}

// Rows of queries and keys whose dims or addresses the chunk kernels' loads do not fit: dims padded to a multiple of 8 with zeros.
// (The same for values.)
template <typename E>
__global__ __launch_bounds__(256) void k_delta_rows(E* __restrict__ dst, const E* __restrict__ src, int T, int Q, int dim, int dim_ld, long ld) {
    for (long row = blockIdx.x; row < T; row += gridDim.x)
        for (int i = threadIdx.x; i < Q * dim_ld; i += 256) {
            const int hq = i / dim_ld, d = i - hq * dim_ld;
            dst[row * Q * dim_ld + i] = d < dim ? src[row * ld + hq * dim + d] : (E)0;
        }
}
constexpr int ROWS_GRID = 1 << 20;   // its workgroups at most (a grid has fewer than 2^32 threads)

template <typename F>
static void more_lds(F* kernel, int bytes) {
    HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
}
template <int DC, bool B16>
static void launch_chunks_of(const DeltaChunks& c) {
    const Delta& a = c.a;
    constexpr int prep = prepare_lds<DC, B16>(), walk = Walk<DC, B16>::LDS;
    static bool enabled = false;
    if (!enabled) {
        more_lds(&k_delta_prepare<DC, B16, false>, prep);
        more_lds(&k_delta_prepare<DC, B16, true>, prep);
        more_lds(&k_delta_chunks<DC, B16, true>, walk);
        more_lds(&k_delta_chunks<DC, B16, false>, walk);
        enabled = true;
    }
    const int slices = cdiv(a.vdim, 16), launches = c.segs == 1 ? 2 : 4;
    const double bytes = c.bytes / launches, flops = c.flops / launches;
    {
        ProfScope ps(PC_DELTA, bytes, flops);
        if (c.step_waves > 0) NVLLM_LAUNCH((k_delta_prepare<DC, B16, true>), dim3(a.H, c.most, a.n_spans + cdiv(c.step_waves, 4 * a.H * c.most)), dim3(256), prep, c);
        else NVLLM_LAUNCH((k_delta_prepare<DC, B16, false>), dim3(a.H, c.most, a.n_spans), dim3(256), prep, c);
    }
    if (c.segs > 1) {
        ProfScope ps(PC_DELTA, bytes, flops);
        NVLLM_LAUNCH((k_delta_chunks<DC, B16, false>), dim3(a.H, slices + 2 * DC, a.n_spans * c.segs), dim3(512), walk, c);
    }
    if (c.segs > 1) {
        ProfScope ps(PC_DELTA, bytes, flops);
        NVLLM_LAUNCH((k_delta_join<DC>), dim3(a.H, slices, a.n_spans), dim3(64 * join_waves<DC>()), 0, c);
    }
    ProfScope ps(PC_DELTA, bytes, flops);
    NVLLM_LAUNCH((k_delta_chunks<DC, B16, true>), dim3(a.H, slices, a.n_spans * c.segs), dim3(512), walk, c);
}
template <bool B16>
static void launch_chunks(const DeltaChunks& c) {
    const int steps = cdiv(c.a.dim, 32);
    if (steps == 1) launch_chunks_of<1, B16>(c);
    else if (steps == 2) launch_chunks_of<2, B16>(c);
    else if (steps == 3) launch_chunks_of<3, B16>(c);
    else if (steps == 4) launch_chunks_of<4, B16>(c);
    else if (steps <= 6) launch_chunks_of<6, B16>(c);
    else launch_chunks_of<8, B16>(c);
}

// Portions of a batch; a refusal if its sequences do not fit.
static int delta_spans(std::vector<int4>& spans, const int* seq_ids, const int* pos, int T, int n_slots) {
    for (int t = 0; t < T;) {
        if (seq_ids[t] < 0 || seq_ids[t] >= n_slots || pos[t] < 0) return NVLLM_BAD_INDEX;
        int n = 1;
        while (t + n < T && seq_ids[t + n] == seq_ids[t]) {
            if (pos[t + n] != pos[t] + n) return NVLLM_BAD_INDEX;
            n++;
        }
        spans.push_back(int4{t, n, pos[t], seq_ids[t]});
        t += n;
    }
    std::vector<int> ids;
    for (const int4& s : spans) ids.push_back(s.w);
    std::sort(ids.begin(), ids.end());
    return std::adjacent_find(ids.begin(), ids.end()) == ids.end() ? 0 : NVLLM_BAD_INDEX;
}

constexpr size_t CHUNK_MEMORY = (size_t)192 << 20;   // of the chunks' records at a time

// Tokens from which a portion goes by chunks.  A token of a portion costs 1 us on the way token by token (128 dims), 3.3 us where states by
// the hundred fill the chip; a chunk costs 13 us (18 us in 32 bits) whatever its tokens, and 5 us (8 us) more for every 256 workgroups
// behind the first.  Measured, token by token and by chunks, heads of 128 x 128 in bf16: 32 heads, 8 tokens 11.3 and 12.9 us, 12 tokens 15.5
// and 13.1; eight sequences (2,048 workgroups), 32 tokens: 40 and 46, 48: 58 and 48; 32 sequences, 32 tokens: 105 and 162, 48: 156
// and 167; beyond that both grow with the batch.
constexpr int CHUNK_LEAST = 10;
static int chunk_min(const Delta& a, const std::vector<int4>& spans, bool b16) {
    double wgs = 0;
    for (const int4& s : spans) wgs += s.y >= CHUNK_LEAST ? (double)a.H * cdiv(a.vdim, 16) : 0.0;
    return (int)((b16 ? 1.0 : 1.5) * CHUNK_LEAST * std::min(5.0, sqrt(std::max(1.0, wgs / 256))));
}

// Segments of the portions' chunks, walked side by side, where heads and columns alone leave most of the chip empty.  They cost another walk
// for what a segment does to a state (its scouts), of which as many run at a time as there are CUs, and a join in which one start waits for
// the other; n segments of m chunks take about m / n + DC n / 2.5 of a chunk's time, least at sqrt(2.5 m / DC).  Measured, in one segment and
// in this many: 8,192 tokens, one head of 128 x 128: 194 us, 83 in 8; four: 195, 105 in 5; eight: 201, 146 in 3 (161 in 4, which no longer
// fit side by side); one of 64 x 64: 174, 58 in 12; 4,096 tokens, two of 256 x 256: 157, 117 in 4; 1,024 tokens, one of 128 x 128: 35, 39 in 3.
static void delta_segments(const Delta& a, int n_spans, int DC, int most, int& segs, int& per_seg) {
    const long walks = (long)a.H * cdiv(a.vdim, 16) * n_spans, unit = (long)a.H * 2 * DC * n_spans, cus = rt().num_cus;
    segs = 1;
    per_seg = most;
    if (most < 6 * DC || walks + unit > cus) return;
    const long fit = std::min(2 + (cus - walks) / (walks + unit), cus / walks), best = (long)sqrt(2.5 * most / DC);
    const int n = (int)std::min(fit, best);
    if (n < 3) return;
    per_seg = cdiv(most, n);
    segs = cdiv(most, per_seg);
}

// Portions whose chunks are prepared and walked together, `most` chunks of each per launch: as many portions as have room for the records of one
// chunk each, and then as many chunks.
struct DeltaGroup {
    int at, n, most, longest, segs, per_seg;
    long tokens;
    double states;                         // bytes
    size_t records, start_floats, bytes;   // of a launch
};
static std::vector<DeltaGroup> delta_groups(const Delta& a, const std::vector<int4>& spans, int n_chunked, std::vector<int>& first) {
    const size_t room = std::max((size_t)1, CHUNK_MEMORY / ((size_t)a.H * DELTA_RECORD));
    const int steps = cdiv(a.dim, 32), DC = steps <= 4 ? steps : steps <= 6 ? 6 : 8;
    const int n_groups = (int)((n_chunked + room - 1) / room), portions = n_groups ? cdiv(n_chunked, n_groups) : 0;   // of one size, or about
    std::vector<DeltaGroup> groups;
    for (int at = 0; at < n_chunked;) {
        DeltaGroup g{};
        g.at = at;
        g.n = std::min(n_chunked - at, portions);
        for (int i = at; i < at + g.n; i++) {
            g.tokens += spans[i].y;
            g.states += (spans[i].z > 0 ? 8.0 : 4.0) * a.H * a.dim * (double)a.vdim;
            g.longest = std::max(g.longest, cdiv(spans[i].y, CH));
        }
        auto records = [&](int per) {
            size_t n = 0;
            for (int i = at; i < at + g.n; i++) {
                first[i] = (int)n;
                n += (size_t)std::min(per, cdiv(spans[i].y, CH));
            }
            return n;
        };
        g.most = g.longest;
        while (g.most > 1 && records(g.most) > room) g.most = (g.most + 1) / 2;
        g.records = records(g.most);
        delta_segments(a, g.n, DC, g.most, g.segs, g.per_seg);
        const size_t columns = (size_t)((a.vdim + 15) & ~15), places = g.segs > 1 ? (size_t)g.n * g.segs * a.H * (32 * DC) : 0;
        g.start_floats = places * columns;
        g.bytes = g.records * a.H * DELTA_RECORD + places * (columns + 32 * DC) * sizeof(float);
        groups.push_back(g);
        at += g.n;
    }
    return groups;
}

static int gated_delta(Delta& a, const int* seq_ids, const int* pos, int T, int n_slots, int elem) {
    std::vector<int4> spans;
    if (const int e = delta_spans(spans, seq_ids, pos, T, n_slots)) return e;
    if ((double)cdiv(a.vdim, STEP_COLS) * a.H * (double)spans.size() > 2e9) return NVLLM_BAD_SIZE;
    const bool b16 = elem == 2;
    const int least = chunk_min(a, spans, b16);   // portions that go by chunks come first
    std::stable_sort(spans.begin(), spans.end(), [&](const int4& l, const int4& r) { return (l.y >= least) > (r.y >= least); });
    int n_chunked = 0;
    double tok_states = 0;
    for (const int4& s : spans) {
        if (s.y >= least) n_chunked++;
        else tok_states += (s.z > 0 ? 8.0 : 4.0) * a.H * a.dim * (double)a.vdim;
    }
    const size_t ints = spans.size() * 5 + 4;
    if (ints > staging_ints()) return NVLLM_BAD_SIZE;
    ensure_init();
    if (stream_is_captured()) return NVLLM_CAPTURED;
    std::vector<int> first(spans.size(), 0);
    const std::vector<DeltaGroup> groups = delta_groups(a, spans, n_chunked, first);
    const size_t four = 4 * (size_t)elem;
    const bool vec = a.dim % 4 == 0 && a.vdim % 4 == 0 && a.q_ld % 4 == 0 && a.k_ld % 4 == 0 && a.v_ld % 4 == 0 && (size_t)a.q % four == 0 && (size_t)a.k % four == 0 &&
                     (size_t)a.v % four == 0 && (size_t)a.out % four == 0 && (size_t)a.state % 16 == 0;
    a.n_spans = (int)spans.size() - n_chunked;
    const double token_bytes = elem * (2.0 * a.Q * a.dim + 2.0 * a.H * a.vdim) + 8.0 * a.H, token_flops = 6.0 * a.H * a.dim * (double)a.vdim;
    long tokens = 0;
    for (const DeltaGroup& gr : groups) tokens += gr.tokens;
    const int per16 = 16 / elem, dim_ld = (a.dim + 7) & ~7, vdim_ld = (a.vdim + 7) & ~7;
    const bool fits = a.dim % 8 == 0 && a.q_ld % per16 == 0 && a.k_ld % per16 == 0 && ((size_t)a.q | (size_t)a.k) % 16 == 0;
    const bool v_fits = a.vdim % per16 == 0 && a.v_ld % per16 == 0 && (size_t)a.v % 16 == 0;
    auto room = [&](bool needed, int heads, int ld) { return needed ? ((size_t)T * heads * ld * elem + 255) & ~(size_t)255 : 0; };
    const size_t qk_room = room(!fits, a.Q, dim_ld), v_room = room(!v_fits, a.H, vdim_ld);
    size_t most_bytes = 0;
    for (const DeltaGroup& gr : groups) most_bytes = std::max(most_bytes, gr.bytes);
    // (all of the memory before the first launch)
    const size_t rows_bytes = n_chunked > 0 ? 2 * qk_room + v_room + most_bytes : 0, step_bytes = spans.size() > DELTA_SPANS ? ints * sizeof(int) : 0;
    char* mem = (char*)ws_try(WS_DELTA, rows_bytes);
    int* dev = (int*)ws_try(WS_STEP, step_bytes);
    if ((rows_bytes > 0 && !mem) || (step_bytes > 0 && !dev)) return NVLLM_NO_MEMORY;
    const int4* d_spans = nullptr;
    const int* d_first = nullptr;
    if (spans.size() > DELTA_SPANS) {
        int* host = pinned_ints(ints);
        std::copy(spans.begin(), spans.end(), (int4*)host);
        std::copy(first.begin(), first.end(), host + 4 * spans.size());
        launch_copy_ints(dev, host, spans.size() * 5);
        d_spans = (const int4*)dev;
        d_first = dev + 4 * spans.size();
    }
    if (n_chunked > 0) {
        DeltaChunks c{};
        c.a = a;
        c.out_four = a.vdim % 4 == 0 && (size_t)a.out % (4 * elem) == 0;
        auto pack = [&](const void*& src, long& ld, int heads, int dim, int wide) {
            const dim3 grid(std::min(T, ROWS_GRID));
            if (b16) NVLLM_LAUNCH((k_delta_rows<unsigned short>), grid, dim3(256), 0, (unsigned short*)mem, (const unsigned short*)src, T, heads, dim, wide, ld);
            else NVLLM_LAUNCH((k_delta_rows<float>), grid, dim3(256), 0, (float*)mem, (const float*)src, T, heads, dim, wide, ld);
            src = mem;
            ld = (long)heads * wide;
        };
        c.a.v_cols = a.vdim;
        if (!fits) {
            pack(c.a.q, c.a.q_ld, a.Q, a.dim, dim_ld);
            mem += qk_room;
            pack(c.a.k, c.a.k_ld, a.Q, a.dim, dim_ld);
            mem += qk_room;
            c.a.dim = dim_ld;
        }
        if (!v_fits) {
            pack(c.a.v, c.a.v_ld, a.H, a.vdim, vdim_ld);
            mem += v_room;
            c.a.v_cols = vdim_ld;
        }
        c.mem = mem;
        for (const DeltaGroup& gr : groups) {
            c.a.n_spans = gr.n;
            c.a.spans = d_spans ? d_spans + gr.at : nullptr;
            c.first = d_first ? d_first + gr.at : nullptr;
            if (!d_spans) {
                std::copy(spans.begin() + gr.at, spans.end(), c.a.here);
                std::copy(first.begin() + gr.at, first.begin() + gr.at + gr.n, c.first_here);
            }
            c.segs = gr.segs;
            c.per_seg = gr.per_seg;
            c.starts = (float*)(mem + gr.records * a.H * DELTA_RECORD);
            c.trans = c.starts + gr.start_floats;
            // the algorithm's bytes and flops, split over the launches
            const int rounds = cdiv(gr.longest, gr.most);
            c.bytes = (gr.states + (double)gr.tokens * token_bytes) / rounds;
            c.flops = (double)gr.tokens * token_flops / rounds;
            // The others' steps go with the last group's first launch where rows are aligned for both.  Apart and together: three portions of 512 tokens
            // and eleven of one, 32 heads of 64 x 64: 36.5 us, 32.0; one of 512 and 64, 128 x 128: 83, 72 (in 32 bits 101, 89); four of 1,024
            // and 64: 207, 199 (350, 340).
            const long waves = (long)cdiv(a.vdim, STEP_COLS) * a.H * a.n_spans;
            if (gr.at + gr.n == n_chunked && fits && v_fits && vec && gr.n + waves / (4L * a.H * gr.most) < 65535) {
                c.step_waves = (int)waves;
                c.bytes += (tok_states + (double)(T - tokens) * token_bytes) / rounds;
                c.flops += (double)(T - tokens) * token_flops / rounds;
                a.n_spans = 0;
            }
            for (c.from = 0; c.from < gr.longest; c.from += gr.most) {
                c.most = std::min(gr.most, gr.longest - c.from);
                if (b16) launch_chunks<true>(c);
                else launch_chunks<false>(c);
                c.step_waves = 0;
            }
        }
    }
    if (a.n_spans == 0) return 0;
    a.spans = d_spans ? d_spans + n_chunked : nullptr;
    if (!d_spans) std::copy(spans.begin() + n_chunked, spans.end(), a.here);
    ProfScope ps(PC_DELTA_TOK, tok_states + (double)(T - tokens) * token_bytes, (double)(T - tokens) * token_flops);
    for (int left = a.n_spans; left > 0; left -= a.n_spans, a.spans += a.n_spans) {   // (what a grid takes)
        a.n_spans = std::min(left, 65535);
        if (b16 && vec) launch_step<true, true>(a);
        else if (b16) launch_step<true, false>(a);
        else if (vec) launch_step<false, true>(a);
        else launch_step<false, false>(a);
    }
    return 0;
}

}  // namespace nvllm

using namespace nvllm;

extern "C" int nvllm_gated_delta(void* out, const void* q, const void* k, const void* v, const float* g, const float* beta, float* state, const int* seq_ids,
                                 const int* pos_arr, int n_slots, float scale, float norm_eps, int qk_heads, int heads, int dim, int vdim, int q_ld, int k_ld, int v_ld,
                                 int elem_bytes, int num_tokens) {
    if (num_tokens < 0) return NVLLM_BAD_ARGUMENT;
    if (num_tokens == 0) return 0;
    if (!out || !q || !k || !v || !g || !beta || !state || !seq_ids || !pos_arr || n_slots <= 0 || qk_heads <= 0 || heads <= 0 || dim <= 0 || vdim <= 0 || !(norm_eps >= 0.f))
        return NVLLM_BAD_ARGUMENT;
    if (std::max(std::max(q_ld, k_ld), v_ld) > 1 << 23 || (long)heads * vdim > 1 << 23) return NVLLM_BAD_SIZE;   // (offsets inside a chunk are 31 bits)
    if ((elem_bytes != 2 && elem_bytes != 4) || dim > DELTA_MAX_DIM || heads % qk_heads || heads > 65535 || vdim > 65535) return NVLLM_BAD_SIZE;
    if (q_ld < (long)qk_heads * dim || k_ld < (long)qk_heads * dim || v_ld < (long)heads * vdim) return NVLLM_BAD_ARGUMENT;
    if (((size_t)q | (size_t)k | (size_t)v | (size_t)out) % elem_bytes || ((size_t)g | (size_t)beta | (size_t)state) % 4) return NVLLM_BAD_ARGUMENT;
    Delta a{};
    a.q = q; a.k = k; a.v = v; a.g = g; a.beta = beta; a.state = state; a.out = out;
    a.q_ld = q_ld; a.k_ld = k_ld; a.v_ld = v_ld;
    a.scale = scale; a.eps = norm_eps;
    a.Q = qk_heads; a.H = heads; a.dim = a.dim_kept = dim; a.vdim = vdim;
    try {
        return gated_delta(a, seq_ids, pos_arr, num_tokens, n_slots, elem_bytes);
    } catch (const std::bad_alloc&) {
        return NVLLM_NO_MEMORY;
    }
}
