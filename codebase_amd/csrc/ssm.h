// Shared pieces of the state space sequence operators (ssm_scan.hip, ssm_conv.hip): element types, argument checks, wave helpers.
//
// Sequences are [agent][step][row][channel], channels contiguous, any stride elsewhere (marlhip_ssm_seq).  Consecutive lanes own
// consecutive channels, so every access along the sequence is a coalesced row; the carried state is [agent][row][state][channel] and the
// weights are [network][..][channel] for the same reason.
#pragma once
#include "common.h"

namespace marl {

constexpr int SSM_MAX_STATE = 32;  // states per channel the scan keeps in registers
constexpr int SSM_MAX_WIDTH = 8;   // taps of the short convolution

template <class T>
__device__ __forceinline__ float up(T v) { return static_cast<float>(v); }
// one rounding to the nearest value of T, ties to even (the conversion instructions' own mode)
template <class T>
__device__ __forceinline__ T down(float v) { return static_cast<T>(v); }

struct SsmSeq {
    const void* data;
    int64_t sp, st, sb;  // elements between agents, steps, rows
};

inline SsmSeq ssm_seq(const marlhip_ssm_seq& s) { return SsmSeq{s.data, s.agent_stride, s.step_stride, s.row_stride}; }

template <class T>
__device__ __forceinline__ const T* seq_at(const SsmSeq& s, int p, int b) {
    return static_cast<const T*>(s.data) + p * s.sp + b * s.sb;
}

constexpr int ROW_MAX = 0x7fffffff;    // bytes of a row descriptor that does not bound its row
constexpr int OOB = (int)0x80000000;   // an offset behind any row

// One row of a wave through a buffer descriptor: the base is uniform, `bytes` of it exist.  Lanes behind them load 0 and store nothing, and
// with bytes = 0 a whole row is skipped - no predicate registers, no per-lane 64-bit addresses.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const void* base, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
}
// (soff: a uniform offset that the bound does not count)
template <class T>
__device__ __forceinline__ float row_load(const T* base, int bytes, int voff, int soff = 0) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(row_rsrc(base, bytes), voff, soff, 0));
    else return up(__builtin_bit_cast(T, (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(row_rsrc(base, bytes), voff, soff, 0)));
}
template <class T>
__device__ __forceinline__ void row_store(float v, T* base, int bytes, int voff, int soff = 0) {
    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), row_rsrc(base, bytes), voff, soff, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, down<T>(v)), row_rsrc(base, bytes), voff, soff, 0);
}

struct SsmDims {
    int P, S, B, C, N, G;
    int8_t net[16];  // agent -> network
    int M;           // networks
};

inline SsmDims ssm_dims(const marlhip_ssm_shape* s) {
    SsmDims d;
    d.P = s->n_agents; d.S = s->steps; d.B = s->batch; d.C = s->channels; d.N = s->state; d.G = s->groups;
    d.M = s->n_networks > 0 ? s->n_networks : s->n_agents;
    for (int i = 0; i < 16; ++i) d.net[i] = (int8_t)(s->n_networks > 0 ? (i < s->n_agents ? s->net_of[i] : 0) : i);
    return d;
}

inline int ssm_validate(const marlhip_ssm_shape* s, const char* what) {
    MARL_REQUIRE(s != nullptr, "%s: shape is NULL", what);
    MARL_REQUIRE(s->n_agents >= 1 && s->n_agents <= 16, "%s: %d agents (1..16 supported)", what, s->n_agents);
    MARL_REQUIRE(s->steps >= 0 && s->batch >= 0 && s->channels >= 1, "%s: steps %d, batch %d, channels %d", what, s->steps, s->batch, s->channels);
    MARL_REQUIRE(s->steps <= (1 << 30) && s->batch <= (1 << 26) && s->channels <= (1 << 20), "%s: steps %d, batch %d, channels %d are too many", what,
                 s->steps, s->batch, s->channels);
    MARL_REQUIRE(s->dtype >= 0 && s->dtype <= 2, "%s: dtype %d (0 f32, 1 bf16, 2 f16)", what, s->dtype);
    if (s->n_networks > 0) {
        MARL_REQUIRE(s->n_networks <= s->n_agents, "%s: %d networks for %d agents", what, s->n_networks, s->n_agents);
        for (int i = 0; i < s->n_agents; ++i)
            MARL_REQUIRE(s->net_of[i] >= 0 && s->net_of[i] < s->n_networks, "%s: net_of[%d] = %d out of range", what, i, s->net_of[i]);
    }
    return 0;
}

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// rows of a padded batch: steps of row b that belong to its sequence
__device__ __forceinline__ int seq_len(const int32_t* lengths, int b, int S) {
    if (lengths == nullptr) return S;
    const int l = lengths[b];
    return l < 0 ? 0 : (l > S ? S : l);
}

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// 2^v on the transcendental unit (results below 2^-126 become 0: a decay that small has emptied the state either way)
__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(-LOG2E * v)); }
// log(1 + e^v) = max(v, 0) + log(1 + e), e = e^-|v| <= 1.  What rounding u = 1 + e lost of e, c = e - (u - 1), is added to log u.  The exact term is
// c / u: with |c| <= 2^-24 u the difference |c - c / u| = |c| e / u is at most 2^-24 e, a step and a half of log(1 + e) >= e log 2.
__device__ __forceinline__ float softplus(float v) {
    const float e = exp2_fast(-LOG2E * fabsf(v)), u = 1.f + e;
    return fmaxf(v, 0.f) + fmaf(LN2, __builtin_amdgcn_logf(u), e - (u - 1.f));
}

// ---- sums over a wave's lanes ----------------------------------------------------------------------------------------------------
__device__ __forceinline__ float dpp_mirror(float v) {  // lane ^ 15
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, true));
}
__device__ __forceinline__ float dpp_half_mirror(float v) {  // lane ^ 7
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, true));
}
__device__ __forceinline__ float dpp_xor3(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x1b, 0xf, 0xf, true)); }
__device__ __forceinline__ float dpp_xor1(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xb1, 0xf, 0xf, true)); }

template <int I> struct Idx { static constexpr int v = I; };

// keeps one of two sums in either half of a lane group: lanes with `bit` clear return lo, the others hi, each with its partner's share
template <int BIT>
__device__ __forceinline__ float half_sum(float lo, float hi, int lane) {
    if constexpr (BIT == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(lo), __float_as_uint(hi), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    } else if constexpr (BIT == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(lo), __float_as_uint(hi), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    } else {
        const float keep = (lane & BIT) ? hi : lo, give = (lane & BIT) ? lo : hi;
        if constexpr (BIT == 8) return keep + dpp_mirror(give);
        if constexpr (BIT == 4) return keep + dpp_half_mirror(give);
        if constexpr (BIT == 2) return keep + dpp_xor3(give);
        return keep + dpp_xor1(give);
    }
}

// Sums of NL pairs over the TOP * 2 lanes of a group, formed as the pairs appear: f(n, b, c) gives (b_n, c_n).  The pairs merge as soon as two
// exist - 2 to 3 instructions a value, where a butterfly each would take 2 log2(lanes) - and need a handful of registers.  gfx950's lane
// swaps exchange halves of two registers in one instruction, so that a merge takes 2; inside a row of 16 lanes the partners are mirrors (DPP),
// and it takes 3, two selects and an addition (every merge where four lanes share a channel: TOP = 8).  Lane bit TOP tells b
// from c, the log2(NL) below it are n; lanes that differ in lower bits only hold the same sum.
template <int NL, int TOP, int LVL, int I, class F>
__device__ __forceinline__ float pair_tree(F& f, int lane) {
    if constexpr (LVL == 0) {
        float b, c;
        f(Idx<I>{}, b, c);
        return half_sum<TOP>(b, c, lane);
    } else {
        const float lo = pair_tree<NL, TOP, LVL - 1, I>(f, lane), hi = pair_tree<NL, TOP, LVL - 1, I + (NL >> LVL)>(f, lane);
        return half_sum<(TOP >> LVL)>(lo, hi, lane);
    }
}
template <int NL, int TOP, class F>
__device__ __forceinline__ float pair_sums(F& f, int lane) {
    static_assert(NL == 4 || NL == 8, "4 or 8 pairs");
    float v = pair_tree<NL, TOP, NL == 8 ? 3 : 2, 0>(f, lane);
    if constexpr (TOP / NL > 4) v += dpp_half_mirror(v);
    if constexpr (TOP / NL > 2) v += dpp_xor3(v);
    if constexpr (TOP / NL > 1) v += dpp_xor1(v);
    return v;
}

// The gradients of one network's weights: the partial sums [agent][slot][rows + extra][C] of its agents, in order.  The first `rows` rows go
// to d0, the next to d1, the one after that to d2 (NULL: not wanted).
// A workgroup takes 64 columns, its 16 waves every 16th slot with eight requests in flight each (bound by latency: the sums are small).
static __global__ __launch_bounds__(1024) void ssm_weights_sum_kernel(SsmDims d, int slots, int rows, int extra, const float* __restrict__ part,
                                                                      float* __restrict__ d0, float* __restrict__ d1, float* __restrict__ d2) {
    const int m = blockIdx.y;
    const int64_t n = (int64_t)(rows + extra) * d.C;
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
    const int64_t i = (int64_t)blockIdx.x * 64 + lane;
    float s = 0.f;
    if (i < n)
        for (int p = 0; p < d.P; ++p)
            if (d.net[p] == m) {
                const float* src = part + (int64_t)p * slots * n + i;
#pragma unroll 8
                for (int k = q; k < slots; k += 16) s += src[k * n];
            }
    red[q][lane] = s;
    __syncthreads();
    if (q != 0 || i >= n) return;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += red[k][lane];
    const int64_t r = i / d.C, c = i % d.C;
    if (r < rows) d0[((int64_t)m * rows + r) * d.C + c] = s;
    else if (r == rows) { if (d1 != nullptr) d1[(int64_t)m * d.C + c] = s; }
    else if (d2 != nullptr) d2[(int64_t)m * d.C + c] = s;
}

// order LDS traffic between the lanes of ONE wave (the queue itself is in order; this holds the compiler to it)
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

}  // namespace marl
