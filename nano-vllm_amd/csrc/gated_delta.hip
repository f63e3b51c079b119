// gated_delta.hip -- the gated delta rule (gated_delta.h).
//
// k_delta_step: token by token.  With the state S of before, a = S^T k, b = S^T q and c = k . q, the token's correction and result are
//   u = beta (v - e^g a),   o = scale (e^g b + c u),   S <- e^g S + k u^T,
// so one pass over S and one sum over its rows serve both.  A wave holds 32 value columns of a head's state in registers (a lane: 4
// columns x NR rows), reads it once, goes through the portion's tokens and writes it once.
#include "gated_delta.h"

#include <algorithm>
#include <new>
#include <vector>

#include "gemm_common.h"
#include "sequence_memory.h"

namespace nvllm {

typedef unsigned int u2_t __attribute__((ext_vector_type(2)));

// Four neighbouring elements as they lie in memory; in 32 bits each where the addresses are no multiples of four elements.
template <bool B16, bool VEC>
struct Four {
    u4_t w;
    __device__ __forceinline__ void load(const void* base, size_t at, int left) {
        if (VEC) {
            if (left <= 0) w = u4_t{0, 0, 0, 0};
            else if (B16) {
                const u2_t p = *reinterpret_cast<const u2_t*>((const unsigned short*)base + at);
                w = u4_t{p[0], p[1], 0, 0};
            } else w = *reinterpret_cast<const u4_t*>((const float*)base + at);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (i >= left) w[i] = 0;
                else if (B16) w[i] = (unsigned)((const unsigned short*)base)[at + i] << 16;
                else w[i] = ((const unsigned*)base)[at + i];
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
template <bool B16, bool VEC>
__device__ __forceinline__ void store_four(void* base, size_t at, const f4_t& v, int left) {
    if (VEC) {
        if (left <= 0) return;
        if (B16) {
            typedef __bf16 b4_t __attribute__((ext_vector_type(4)));
            *reinterpret_cast<b4_t*>((__bf16*)base + at) = b4_t{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        } else *reinterpret_cast<f4_t*>((float*)base + at) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < left) {
                if (B16) ((__bf16*)base)[at + i] = (__bf16)v[i];
                else ((float*)base)[at + i] = v[i];
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

template <bool B16, int NR, bool VEC>
__global__ __launch_bounds__(64) void k_delta_step(Delta a) {
    constexpr int R4 = NR / 4;
    typedef Four<B16, VEC> F;
    const int slices = (a.vdim + STEP_COLS - 1) / STEP_COLS;
    int idx = blockIdx.x;
    const int slice = idx % slices;
    idx /= slices;
    const int h = idx % a.H;
    const int4 span = (a.spans ? a.spans : a.here)[idx / a.H];
    const int lane = threadIdx.x, col = slice * STEP_COLS + (lane & 7) * 4, row0 = (lane >> 3) * NR, hq = h / (a.H / a.Q);
    const int cols = a.vdim - col, rows = a.dim - row0;   // that this lane has at most
    float* st = a.state + ((size_t)span.w * a.H + h) * a.dim * a.vdim;
    f4_t S[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) {
        S[r] = f4_t{0.f, 0.f, 0.f, 0.f};
        if (span.z > 0 && r < rows) {
            Four<false, VEC> w;
            w.load(st, (size_t)(row0 + r) * a.vdim + col, cols);
            S[r] = w.get();
        }
    }
    F kn[R4], qn[R4], vn;
    float gn, bn;
    auto fetch = [&](int t) {
#pragma unroll
        for (int r = 0; r < R4; r++) {
            kn[r].load(a.k, (size_t)t * a.k_ld + hq * a.dim + row0 + 4 * r, rows - 4 * r);
            qn[r].load(a.q, (size_t)t * a.q_ld + hq * a.dim + row0 + 4 * r, rows - 4 * r);
        }
        vn.load(a.v, (size_t)t * a.v_ld + h * a.vdim + col, cols);
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
        if (lane < 8) store_four<B16, VEC>(a.out, ((size_t)t * a.H + h) * a.vdim + col, o, cols);
    }
#pragma unroll
    for (int r = 0; r < NR; r++)
        if (r < rows) store_four<false, VEC>(st, (size_t)(row0 + r) * a.vdim + col, S[r], cols);
}

template <bool B16, bool VEC>
static void launch_step(const Delta& a) {
    const dim3 grid((unsigned)(cdiv(a.vdim, STEP_COLS) * a.H * a.n_spans));
    const int nr = cdiv(a.dim, 8);
    if (nr <= 4) NVLLM_LAUNCH((k_delta_step<B16, 4, VEC>), grid, dim3(64), 0, a);
    else if (nr <= 8) NVLLM_LAUNCH((k_delta_step<B16, 8, VEC>), grid, dim3(64), 0, a);
    else if (nr <= 12) NVLLM_LAUNCH((k_delta_step<B16, 12, VEC>), grid, dim3(64), 0, a);
    else if (nr <= 16) NVLLM_LAUNCH((k_delta_step<B16, 16, VEC>), grid, dim3(64), 0, a);
    else if (nr <= 24) NVLLM_LAUNCH((k_delta_step<B16, 24, VEC>), grid, dim3(64), 0, a);
    else NVLLM_LAUNCH((k_delta_step<B16, 32, VEC>), grid, dim3(64), 0, a);
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

static int gated_delta(Delta& a, const int* seq_ids, const int* pos, int T, int n_slots, int elem) {
    std::vector<int4> spans;
    if (const int e = delta_spans(spans, seq_ids, pos, T, n_slots)) return e;
    if ((double)cdiv(a.vdim, STEP_COLS) * a.H * (double)spans.size() > 2e9 || spans.size() * 4 > staging_ints()) return NVLLM_BAD_SIZE;
    ensure_init();
    if (stream_is_captured()) return NVLLM_CAPTURED;
    double state_floats = 0;
    for (const int4& s : spans) state_floats += (s.z > 0 ? 2.0 : 1.0) * a.H * a.dim * (double)a.vdim;
    a.n_spans = (int)spans.size();
    a.spans = nullptr;
    if (a.n_spans <= DELTA_SPANS) {
        std::copy(spans.begin(), spans.end(), a.here);
    } else {
        int* host = pinned_ints(spans.size() * 4);
        std::copy(spans.begin(), spans.end(), (int4*)host);
        int* dev = (int*)ws_get(WS_STEP, spans.size() * 16);
        launch_copy_ints(dev, host, spans.size() * 4);
        a.spans = (const int4*)dev;
    }
    const bool b16 = elem == 2;
    const size_t four = 4 * (size_t)elem;
    const bool vec = a.dim % 4 == 0 && a.vdim % 4 == 0 && a.q_ld % 4 == 0 && a.k_ld % 4 == 0 && a.v_ld % 4 == 0 && (size_t)a.q % four == 0 && (size_t)a.k % four == 0 &&
                     (size_t)a.v % four == 0 && (size_t)a.out % four == 0 && (size_t)a.state % 16 == 0;
    ProfScope ps(PC_DELTA_TOK, state_floats * 4 + (double)T * (elem * (2.0 * a.Q * a.dim + 2.0 * a.H * a.vdim) + 8.0 * a.H), 6.0 * T * a.H * a.dim * (double)a.vdim);
    if (b16 && vec) launch_step<true, true>(a);
    else if (b16) launch_step<true, false>(a);
    else if (vec) launch_step<false, true>(a);
    else launch_step<false, false>(a);
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
    if ((elem_bytes != 2 && elem_bytes != 4) || dim > DELTA_MAX_DIM || heads % qk_heads || heads > 65535 || vdim > 65535) return NVLLM_BAD_SIZE;
    if (q_ld < (long)qk_heads * dim || k_ld < (long)qk_heads * dim || v_ld < (long)heads * vdim) return NVLLM_BAD_ARGUMENT;
    if (((size_t)q | (size_t)k | (size_t)v | (size_t)out) % elem_bytes || ((size_t)g | (size_t)beta | (size_t)state) % 4) return NVLLM_BAD_ARGUMENT;
    Delta a{};
    a.q = q; a.k = k; a.v = v; a.g = g; a.beta = beta; a.state = state; a.out = out;
    a.q_ld = q_ld; a.k_ld = k_ld; a.v_ld = v_ld;
    a.scale = scale; a.eps = norm_eps;
    a.Q = qk_heads; a.H = heads; a.dim = dim; a.vdim = vdim;
    try {
        return gated_delta(a, seq_ids, pos_arr, num_tokens, n_slots, elem_bytes);
    } catch (const std::bad_alloc&) {
        return NVLLM_NO_MEMORY;
    }
}
