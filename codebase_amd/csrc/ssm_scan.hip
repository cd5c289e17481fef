// Selective state space scan: marlhip_ssm_scan (forward, any number of steps, one included) and marlhip_ssm_scan_grad.
//
//   h_t[n] = exp(dt_t A[n]) h_{t-1}[n] + dt_t B_t[n] x_t,   y_t = sum_n C_t[n] h_t[n] + D x_t        for every channel
//
// Layout of a wave.  A lane keeps NL = 8 or 4 states of one channel in registers, NS = 1, 2 or 4 lanes share a channel (N <= NL NS): lane =
// group * CL + channel, CL = 64 / NS channels a wave.  The work of a step that does not depend on the state (loads, softplus, gate, store) is
// done for NS steps at once, group g taking step s + g; a lane swap then hands every group the step it needs, and another one adds the groups'
// shares of y.  So more lanes a channel cost swaps, but take fewer registers and give more waves, which is what small batches need (scan_plan).
// B and C of a step are the same for a group's channels and come as LDS broadcasts, K steps at a time.
#include <cfloat>

#include "ssm.h"

using namespace marl;

namespace {

constexpr int K = 8;     // steps of a block: between two recorded states
constexpr int WMAX = 8;  // waves of a backward workgroup
constexpr int STEP_WAVES = 8192;  // waves of an acting step

struct ScanArgs {
    SsmDims d;
    SsmSeq x, delta, Bm, Cm, z, dy;
    const float *A, *D, *bias, *h_in, *dh_out;
    const uint8_t* reset;
    const int32_t* lengths;
    void *y, *dx, *ddelta, *dB, *dC, *dz;
    float *h_out, *record, *dh_in;
    float* carry;    // [row][chunk][N][C] states (forward) or gradients (backward) a chunk starts from; first its own contribution
    float* sums;     // [row][chunk][C] sum of dt over a chunk, NaN with a reset inside
    float *pB, *pC;  // [wgs][P][S][B][G][N] partial sums of dB / dC, NULL: one workgroup a row, which writes dB / dC
    float* part;     // [P][slots][N + 2][C] partial sums of dA, dD, ddelta_bias
    int softplus, nblk, slots, nck, chunk, nchunk, wpb, wgs;
    int items;
};

// ---- a wave's place ------------------------------------------------------------------------------------------------------------------
template <int NL, int NS>
struct Lane {
    static constexpr int CL = 64 / NS;
    int lane, g, cl;      // group, channel within the block
    int grp, kblk, first; // channel group, block within it, first channel
    bool act;
    int n0;               // first state
    __device__ __forceinline__ Lane(const ScanArgs& a, int cb, int ln) {
        const int Cg = a.d.C / a.d.G;
        lane = ln;
        g = ln / CL;
        cl = ln % CL;
        grp = uni(cb / a.nblk);
        kblk = cb - grp * a.nblk;
        first = grp * Cg + kblk * CL;
        act = first + cl < (grp + 1) * Cg;
        n0 = g * NL;
    }
    // this lane's element of an [N][C] array: its offset from state n of the first channel, for every n; states from N on are not there
    __device__ __forceinline__ int state_off(const ScanArgs& a) const { return act ? (n0 * a.d.C + cl) * 4 : OOB; }
    __device__ __forceinline__ int no_state(const ScanArgs& a, int n) const { return (a.d.N - 1 - n - n0) & OOB; }
    __device__ __forceinline__ int chan_off(int bytes) const { return act ? cl * bytes : OOB; }
};

template <int NL, int NS>
__device__ __forceinline__ void load_state(const ScanArgs& a, const Lane<NL, NS>& q, const float* p, float (&r)[NL]) {
    const int off = q.state_off(a), bytes = p != nullptr ? ROW_MAX : 0;
#pragma unroll
    for (int n = 0; n < NL; ++n) r[n] = row_load(p + q.first, bytes, off | q.no_state(a, n), n * a.d.C * 4);
}
// A log2 e of the states.  A rate of -inf empties a state at every step that is there; where a block or chunk has steps that are not, with dt = 0,
// their product would be NaN, so it becomes the lowest finite value (which empties a state unless dt is below 2^-120).
__device__ __forceinline__ float rate(float A) {
    const float r = A * LOG2E;
    return r < -FLT_MAX ? -FLT_MAX : r;
}
template <int NL, int NS>
__device__ __forceinline__ void load_rates(const ScanArgs& a, const Lane<NL, NS>& q, int net, float (&A)[NL]) {
    load_state(a, q, a.A + (int64_t)net * a.d.N * a.d.C, A);
#pragma unroll
    for (int n = 0; n < NL; ++n) A[n] = rate(A[n]);
}
template <int NL, int NS>
__device__ __forceinline__ void store_state(const ScanArgs& a, const Lane<NL, NS>& q, float* p, const float (&r)[NL]) {
    const int off = q.state_off(a);
#pragma unroll
    for (int n = 0; n < NL; ++n) row_store(r[n], p + q.first, ROW_MAX, off | q.no_state(a, n), n * a.d.C * 4);
}

// value of group i of a register that holds one value a group, in every group
template <int NS>
__device__ __forceinline__ void to_groups(float v, float (&r)[NS]) {
    if constexpr (NS == 1) {
        r[0] = v;
    } else {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        if constexpr (NS == 2) {
            r[0] = __uint_as_float(s[0]);
            r[1] = __uint_as_float(s[1]);
        } else {
            const auto t = __builtin_amdgcn_permlane16_swap(s[0], s[0], false, false), u = __builtin_amdgcn_permlane16_swap(s[1], s[1], false, false);
            r[0] = __uint_as_float(t[0]);
            r[1] = __uint_as_float(t[1]);
            r[2] = __uint_as_float(u[0]);
            r[3] = __uint_as_float(u[1]);
        }
    }
}
// r[i]: every group's share for step i -> the sum for step g in group g
template <int NS>
__device__ __forceinline__ float from_groups(const float (&r)[NS]) {
    if constexpr (NS == 1) return r[0];
    if constexpr (NS == 2) return half_sum<32>(r[0], r[1], 0);
    if constexpr (NS == 4) return half_sum<16>(half_sum<32>(r[0], r[2], 0), half_sum<32>(r[1], r[3], 0), 0);
}

// waits for loads here: the ones a loop needs from before it are not waited for inside it, where stores would be waited for with them
template <int N>
__device__ __forceinline__ void wait_for(float (&r)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) asm volatile("" : "+v"(r[n]));
}

// ---- K steps of inputs, requested ahead of their use ----------------------------------------------------------------------------------------
template <class T>
struct Raw;  // an element as it comes, widened at its use
template <>
struct Raw<float> {
    float v;
    __device__ __forceinline__ float get() const { return v; }
    __device__ __forceinline__ void load(const float* p, int voff) { v = row_load(p, ROW_MAX, voff); }
};
template <class T>
struct Raw {
    unsigned short v;
    __device__ __forceinline__ float get() const { return up(__builtin_bit_cast(T, v)); }
    __device__ __forceinline__ void load(const T* p, int voff) { v = __builtin_amdgcn_raw_buffer_load_b16(row_rsrc(p, ROW_MAX), voff, 0, 0); }
};

// A sequence's steps for a wave: a uniform pointer to step t (moved by adding, no product a load) and this lane's offset to its own step t + g
template <class T, int NS>
struct SeqPtr {
    const char* p;
    int64_t st;  // bytes between steps
    int voff;
    template <int NL>
    __device__ __forceinline__ SeqPtr(const SsmSeq& s, const Lane<NL, NS>& q, int pa, int b, int t)
        : p(reinterpret_cast<const char*>(seq_at<T>(s, pa, b) + q.first + t * s.st)), st(s.st * (int64_t)sizeof(T)),
          voff(q.act ? q.g * (int)(s.st * (int64_t)sizeof(T)) + q.cl * (int)sizeof(T) : OOB) {}
    __device__ __forceinline__ void load(Raw<T>& r, int steps, int out) const { r.load(reinterpret_cast<const T*>(p + steps * st), voff | out); }
    __device__ __forceinline__ void move(int steps) { p += steps * st; }
};
// the sign bit where step t + g is behind the end: OR-ed into an offset it points behind any row
constexpr int NO_END = -1;
__device__ __forceinline__ int behind(int t, int g, int end) { return end == NO_END ? 0 : (end - 1 - t - g) & OOB; }

// B / C of K steps: what this thread of NT carries to LDS
template <class T, int NP, int NT>
struct Maps {
    static constexpr int M = (K * NP + NT - 1) / NT;
    Raw<T> b[M], c[M];
};
template <class T, int NP, int NT>
struct MapsPtr {
    static constexpr int M = (K * NP + NT - 1) / NT;
    const char *pb, *pc;  // step t
    int64_t sb, sc;
    int vb[M], vc[M];
    __device__ __forceinline__ MapsPtr(const ScanArgs& a, int pa, int b, int grp, int t, int tid)
        : pb(reinterpret_cast<const char*>(seq_at<T>(a.Bm, pa, b) + grp * a.d.N + t * a.Bm.st)),
          pc(reinterpret_cast<const char*>(seq_at<T>(a.Cm, pa, b) + grp * a.d.N + t * a.Cm.st)), sb(a.Bm.st * (int64_t)sizeof(T)), sc(a.Cm.st * (int64_t)sizeof(T)) {
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int e = tid + NT * i, s = e / NP, n = e % NP;
            const bool ok = e < K * NP && n < a.d.N;
            vb[i] = ok ? s * (int)sb + n * (int)sizeof(T) : OOB;
            vc[i] = ok ? s * (int)sc + n * (int)sizeof(T) : OOB;
        }
    }
    __device__ __forceinline__ void load(Maps<T, NP, NT>& m, int t, int end, int tid) const {  // t: where the pointers are
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int out = behind(t, (tid + NT * i) / NP, end);
            m.b[i].load(reinterpret_cast<const T*>(pb), vb[i] | out);
            m.c[i].load(reinterpret_cast<const T*>(pc), vc[i] | out);
        }
    }
    __device__ __forceinline__ void move(int steps) {
        pb += steps * sb;
        pc += steps * sc;
    }
};
template <class T, int NP, int NT>
__device__ __forceinline__ void store_maps(const Maps<T, NP, NT>& m, float* lb, float* lc, int tid) {
#pragma unroll
    for (int i = 0; i < Maps<T, NP, NT>::M; ++i) {
        const int e = tid + NT * i;
        if (NT * Maps<T, NP, NT>::M == K * NP || e < K * NP) {
            lb[e] = m.b[i].get();
            lc[e] = m.c[i].get();
        }
    }
}

// bit s: an episode starts at step t0 + s.  Two forms of the load: through a descriptor, without a branch, so that the waits around it stay counted
// (forwards), and under one, where scalar registers are short (backwards: 261 us, with a descriptor 292)
__device__ __forceinline__ int load_reset_row(const ScanArgs& a, int b, int t0, int end, int lane) {
    const auto row = row_rsrc(a.reset + (int64_t)t0 * a.d.B + b, a.reset != nullptr ? ROW_MAX : 0);
    return __builtin_amdgcn_raw_buffer_load_b8(row, lane % K * a.d.B | behind(t0, lane % K, end), 0, 0);
}
__device__ __forceinline__ int load_reset(const ScanArgs& a, int b, int t0, int end, int lane) {
    if (a.reset == nullptr) return 0;
    const int t = t0 + (lane % K);
    return t < end ? a.reset[(int64_t)t * a.d.B + b] : 0;
}
__device__ __forceinline__ unsigned reset_bits(int v) { return (unsigned)__builtin_amdgcn_ballot_w64(v != 0) & ((1u << K) - 1); }

// Resets are rare and the same for a whole wave: a branch, which the empty asm keeps the compiler from turning into a select a state
template <int NL>
__device__ __forceinline__ void clear(float (&h)[NL]) {
    asm volatile("");
#pragma unroll
    for (int n = 0; n < NL; ++n) h[n] = 0.f;
}

__device__ __forceinline__ float step_size(const ScanArgs& a, float d, float bias) {
    const float r = d + bias;
    return a.softplus ? softplus(r) : r;
}

// ---- forward ---------------------------------------------------------------------------------------------------------------------------
// Bound by the vector ALUs: a state of a step is a product, an exponential (two issue slots), a product and two fused multiply-adds, and with the
// softplus, the gate and the loads a step of 32 channels x 16 states takes 58 instructions.  128 steps x 1024 rows x 128 channels f32: 79 us,
// 3.8 TB/s; the bytes alone would take 64 us.  The inputs of a block are requested a block ahead.
// CARRY: only the state a chunk contributes and its sum of dt are formed (sequences split over their length, first pass: 29 us of the 77 us that
// 16384 steps x 512 channels bf16 take).
//
// The stores of a whole block come together at its end, outside all branches, and the record has a kernel of its own: loads and stores are counted
// by one counter, and where the number of stores behind the loads for the next block is not known the wait for those loads is one for all stores as
// well (501 steps x 128 rows x 256 channels bf16 with the record: 120 us, with every wait a counted one 105).
enum Pass { CARRY_PASS, STEPS_PASS, RECORD_PASS };
template <class T, int NL, int NS, int PASS>
__global__ __launch_bounds__(256) void ssm_scan_fwd_kernel(ScanArgs a) {
    constexpr int NP = NS * NL, KG = K / NS;
    constexpr bool CARRY = PASS == CARRY_PASS;
    __shared__ float lds[4][2][K * NP];
    const int wv = uni(threadIdx.x >> 6);
    const int item = blockIdx.x * 4 + wv;
    if (item >= a.items) return;
    const int ncb = a.d.G * a.nblk, rc = uni(item / ncb), cb = item - rc * ncb;  // rc: (row, chunk)
    const int row = uni(rc / a.nchunk), ch = rc - row * a.nchunk, p = uni(row / a.d.B), b = row - p * a.d.B;
    const Lane<NL, NS> q(a, cb, threadIdx.x & 63);
    const int N = a.d.N, C = a.d.C, net = a.d.net[p], len = uni(seq_len(a.lengths, b, a.d.S));
    const int first = ch * a.chunk, last = first + a.chunk < a.d.S ? first + a.chunk : a.d.S, end = len < last ? len : last;
    SeqPtr<T, NS> xs(a.x, q, p, b, first), ds(a.delta, q, p, b, first), zs(a.z, q, p, b, first);
    MapsPtr<T, NP, 64> ms(a, p, b, q.grp, first, threadIdx.x & 63);
    const bool gated = !CARRY && a.z.data != nullptr;
    const int lane = q.lane, no_gate = gated ? 0 : OOB;

    Raw<T> x[KG], dr[KG], z[KG];
    Maps<T, NP, 64> maps;
    int rs;
    auto request = [&](int t0) __attribute__((always_inline)) {  // the pointers are at t0
        auto load = [&](int last) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                const int out = behind(t0 + i * NS, q.g, last);
                xs.load(x[i], i * NS, out);
                ds.load(dr[i], i * NS, out);
                if (!CARRY) zs.load(z[i], i * NS, out | no_gate);
            }
            ms.load(maps, t0, last, lane);
        };
        if (t0 + K <= end) load(NO_END);  // a whole block: no offset has to be masked
        else load(end);
        rs = load_reset_row(a, b, t0, end, lane);
        xs.move(K);
        ds.move(K);
        zs.move(K);
        ms.move(K);
    };
    if (first < end) request(first);
    float A[NL], h[NL];
    load_rates(a, q, net, A);
    if (CARRY) load_state(a, q, (const float*)nullptr, h);
    else load_state(a, q, a.nchunk > 1 ? a.carry + ((int64_t)row * a.nchunk + ch) * N * C : (a.h_in != nullptr ? a.h_in + (int64_t)row * N * C : nullptr), h);
    const int co = q.chan_off(4);
    const float D = row_load(a.D + (int64_t)net * C + q.first, a.D != nullptr ? ROW_MAX : 0, co);
    const float bias = row_load(a.bias + (int64_t)net * C + q.first, a.bias != nullptr ? ROW_MAX : 0, co);
    const int64_t yst = (int64_t)a.d.B * C;
    T* yp = static_cast<T*>(a.y) + ((int64_t)p * a.d.S * a.d.B + b) * C + q.first + first * yst;  // at step t0
    const int yoff = q.act ? q.g * (int)(yst * (int64_t)sizeof(T)) + q.cl * (int)sizeof(T) : OOB;
    float *lb = lds[wv][0], *lc = lds[wv][1];
    float total = 0.f;  // CARRY: sum of dt
    wait_for(h);
    float db[2] = {D, bias};
    wait_for(db);
    int t0 = first;
    auto block = [&](auto whole) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole)::v;
        wave_lds_sync();
        store_maps(maps, lb, lc, lane);
        const unsigned fresh = reset_bits(rs);
        float xv[KG], dt[KG], gate[KG], yv[KG];  // yv: stored behind both forms of the steps
#pragma unroll
        for (int i = 0; i < KG; ++i) {
            xv[i] = x[i].get();
            dt[i] = step_size(a, dr[i].get(), bias);
            gate[i] = gated ? z[i].get() : 0.f;
        }
        wave_lds_sync();
        if (WHOLE && t0 + K < end) request(t0 + K);
        if (PASS == RECORD_PASS) store_state(a, q, a.record + ((int64_t)row * a.nck + t0 / K) * N * C, h);
        auto steps = [&](auto plain) __attribute__((always_inline)) {
            constexpr bool PLAIN = decltype(plain)::v;
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                if (!WHOLE) {
                    if (t0 + i * NS >= end) break;
                    if (behind(t0 + i * NS, q.g, end)) dt[i] = 0.f;  // a step behind the end changes nothing: dt = 0, x = 0
                }
                float dts[NS], us[NS], ys[NS];
                to_groups<NS>(dt[i], dts);
                to_groups<NS>(dt[i] * xv[i], us);
                if (CARRY) total += !PLAIN && (fresh >> (i * NS + q.g) & 1) ? __builtin_nanf("") : dt[i];
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    const int s = i * NS + j;
                    const bool re = !PLAIN && (fresh >> s & 1);
                    float y = 0.f;
#pragma unroll
                    for (int n = 0; n < NL; ++n) {
                        h[n] = fmaf(exp2_fast(dts[j] * A[n]), re ? 0.f : h[n], us[j] * lb[s * NP + q.n0 + n]);
                        if (!CARRY) y = fmaf(h[n], lc[s * NP + q.n0 + n], y);
                    }
                    ys[j] = y;
                }
                if (!CARRY) {
                    yv[i] = fmaf(D, xv[i], from_groups<NS>(ys));
                    if (gated) yv[i] *= gate[i] * sigmoid(gate[i]);
                    if (!WHOLE) row_store(yv[i], yp + i * NS * yst, ROW_MAX, yoff | behind(t0 + i * NS, q.g, end));
                }
            }
        };
        if (WHOLE && fresh == 0) steps(Idx<1>{});
        else steps(Idx<0>{});
        if (!CARRY && WHOLE)
#pragma unroll
            for (int i = 0; i < KG; ++i) row_store(yv[i], yp + i * NS * yst, ROW_MAX, yoff);
        yp += K * yst;
    };
    // three forms of a block: without resets it is straight-line code, so that the maps' LDS reads run ahead of their use; resets are a select a state;
    // and the last block of a sequence may end inside
    for (; t0 + K <= end; t0 += K) block(Idx<1>{});
    if (t0 < end) block(Idx<0>{});
    if (CARRY) {
        store_state(a, q, a.carry + ((int64_t)row * a.nchunk + ch) * N * C, h);
        float r[NS];
        to_groups<NS>(total, r);
        total = r[0];
#pragma unroll
        for (int j = 1; j < NS; ++j) total += r[j];
        row_store(total, a.sums + ((int64_t)row * a.nchunk + ch) * C + q.first, ROW_MAX, q.g == 0 ? co : OOB);
        return;
    }
    yp = static_cast<T*>(a.y) + ((int64_t)p * a.d.S * a.d.B + b) * C + q.first;
    for (int t = end > first ? end : first; t < last; ++t) row_store(0.f, yp + t * yst, ROW_MAX, q.g == 0 ? q.chan_off(sizeof(T)) : OOB);
    if (a.h_out != nullptr && ch == a.nchunk - 1) store_state(a, q, a.h_out + (int64_t)row * N * C, h);
}

// One step a row (acting).  All there is to do is to read a row's state, to move it on and to write it back: a lane keeps one channel with all
// its states, so that nothing crosses lanes, a wave takes rows b = slot, slot + slots, .. of one agent with its decay rates in registers, and the
// next row is requested before the current one is worked on.  Bound by HBM: 16384 rows x 256 channels x 16 states take 103 us, 5.5 TB/s.
template <class T, int NP>
__global__ __launch_bounds__(256) void ssm_scan_step_kernel(ScanArgs a) {
    __shared__ float lds[4][2][NP];
    const int wv = uni(threadIdx.x >> 6);
    const int item = blockIdx.x * 4 + wv;
    if (item >= a.items) return;
    const int ncb = a.d.G * a.nblk, ps = uni(item / ncb), cb = item - ps * ncb, p = uni(ps / a.slots), slot = ps - p * a.slots;
    const Lane<NP, 1> q(a, cb, threadIdx.x & 63);
    const int N = a.d.N, C = a.d.C, NB = a.d.B, net = a.d.net[p], lane = q.lane;
    const int ct = q.chan_off(sizeof(T)), cf = q.chan_off(4);
    float A[NP], h[NP], nh[NP];
    Raw<T> x, d, z, m;
    int rs, ln;
    const bool gated = a.z.data != nullptr;
    // lanes 0 .. N-1 fetch B, lanes NP .. NP+N-1 (of 2 NP <= 64) C
    const bool isC = lane >= NP;
    const int n_of = isC ? lane - NP : lane;
    const bool fetch = n_of < N;
    const int hbytes = a.h_in != nullptr ? ROW_MAX : 0;
    auto request = [&](int b) __attribute__((always_inline)) {
        x.load(seq_at<T>(a.x, p, b) + q.first, ct);
        d.load(seq_at<T>(a.delta, p, b) + q.first, ct);
        if (gated) z.load(seq_at<T>(a.z, p, b) + q.first, ct);
        const T* mp = (isC ? seq_at<T>(a.Cm, p, b) : seq_at<T>(a.Bm, p, b)) + q.grp * N + (fetch ? n_of : 0);
        m.v = *reinterpret_cast<const decltype(m.v)*>(mp);
        rs = a.reset != nullptr ? a.reset[b] : 0;
        ln = a.lengths != nullptr ? a.lengths[b] : 1;
        const float* hp = a.h_in + ((int64_t)p * NB + b) * N * C + q.first;
#pragma unroll
        for (int n = 0; n < NP; ++n) nh[n] = row_load(hp, hbytes, n < N ? cf : OOB, n * C * 4);
    };
    request(slot);
    const float* Ap = a.A + (int64_t)net * N * C + q.first;
#pragma unroll
    for (int n = 0; n < NP; ++n) A[n] = row_load(Ap, ROW_MAX, n < N ? cf : OOB, n * C * 4);
    const float D = row_load(a.D + (int64_t)net * C + q.first, a.D != nullptr ? ROW_MAX : 0, cf);
    const float bias = row_load(a.bias + (int64_t)net * C + q.first, a.bias != nullptr ? ROW_MAX : 0, cf);
#pragma unroll
    for (int n = 0; n < NP; ++n) A[n] = rate(A[n]);
    float* lm = lds[wv][0];
    for (int b = slot; b < NB; b += a.slots) {
        const bool fresh = uni(rs) != 0, live = uni(ln) > 0;
        wave_lds_sync();
        if (lane < 2 * NP) lm[lane] = fetch ? m.get() : 0.f;
        wave_lds_sync();
        const float xv = x.get(), dv = d.get(), zv = gated ? z.get() : 0.f;
#pragma unroll
        for (int n = 0; n < NP; ++n) h[n] = fresh && live ? 0.f : nh[n];
        if (b + a.slots < NB) request(b + a.slots);
        float y = 0.f;
        if (live) {
            const float dt = step_size(a, dv, bias), u = dt * xv;
            y = D * xv;
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                h[n] = fmaf(exp2_fast(dt * A[n]), h[n], u * lm[n]);
                y = fmaf(h[n], lm[NP + n], y);
            }
            if (gated) y *= zv * sigmoid(zv);
        }
        const int64_t row = (int64_t)p * NB + b;
        row_store(y, static_cast<T*>(a.y) + row * C + q.first, ROW_MAX, ct);
        if (a.h_out != nullptr) {
            float* hp = a.h_out + row * N * C + q.first;
#pragma unroll
            for (int n = 0; n < NP; ++n) row_store(h[n], hp, ROW_MAX, n < N ? cf : OOB, n * C * 4);
        }
    }
}

// What follows a chunk that starts from h and gives `own` by itself: the decay exp(a sum dt), a = A log2 e, is put on in two factors, since over a
// whole chunk, or a run of them, it may leave the range of a float where its product with the state does not (A > 0 or steps below 0).  A state of 0
// stays 0 even where the decay is infinite.
__device__ __forceinline__ float join_chunk(float a, float sum, float own, float h) {
    const float r = a * sum, k = fminf(fmaxf(rintf(r), -1000.f), 1000.f);
    return sum == sum && h != 0.f ? ldexpf(exp2_fast(r - k) * h, (int)k) + own : own;
}

// Joins the chunks of a sequence: carry[j] (what chunk j contributes) becomes what chunk j starts from.  A chunk multiplies what it is given by
// exp(A sum dt), or drops it at a reset (sum = NaN).  A workgroup takes 64 channels of one state, its 16 waves a run of chunks each; the runs
// are joined through LDS, so the serial part is nchunk / 16 steps twice and 16 once.  reverse: from the last chunk to the first.
// Bound by latency: 12.6 us for 256 chunks of 512 channels x 16 states, 128 workgroups on half of the compute units.
__global__ __launch_bounds__(1024) void ssm_scan_join_kernel(ScanArgs a, const float* __restrict__ start, int reverse) {
    __shared__ float ls[16][64], lh[16][64];
    const int cbs = (a.d.C + 63) / 64, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n = (blockIdx.x / cbs) % a.d.N, row = blockIdx.x / cbs / a.d.N, c0 = (blockIdx.x % cbs) * 64 + lane;
    const bool act = c0 < a.d.C;
    const int c = act ? c0 : a.d.C - 1;
    const float A = rate(a.A[((int64_t)a.d.net[row / a.d.B] * a.d.N + n) * a.d.C + c]);
    const int per = (a.nchunk + 15) / 16, lo = w * per, hi = lo + per < a.nchunk ? lo + per : a.nchunk;
    auto at = [&](int k) { return (int64_t)row * a.nchunk + (reverse ? a.nchunk - 1 - k : k); };
    float s = 0.f, h = 0.f;
#pragma unroll 4
    for (int k = lo; k < hi; ++k) {
        const float sk = a.sums[at(k) * a.d.C + c], own = a.carry[(at(k) * a.d.N + n) * a.d.C + c];
        h = join_chunk(A, sk, own, h);
        s += sk;
    }
    ls[w][lane] = s;
    lh[w][lane] = h;
    __syncthreads();
    h = start != nullptr ? start[((int64_t)row * a.d.N + n) * a.d.C + c] : 0.f;
    for (int k = 0; k < w; ++k) h = join_chunk(A, ls[k][lane], lh[k][lane], h);
#pragma unroll 4
    for (int k = lo; k < hi; ++k) {
        float* q = a.carry + (at(k) * a.d.N + n) * a.d.C + c;
        const float sk = a.sums[at(k) * a.d.C + c], own = *q;
        if (act) *q = h;
        h = join_chunk(A, sk, own, h);
    }
}

// The same for few chunks: a thread takes a state of a channel through all of them.
__global__ __launch_bounds__(256) void ssm_scan_join_few_kernel(ScanArgs a, const float* __restrict__ start, int reverse) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, nc = (int64_t)a.d.N * a.d.C;
    if (i >= (int64_t)a.d.P * a.d.B * nc) return;
    const int row = (int)(i / nc), e = (int)(i % nc), c = e % a.d.C;
    const float A = rate(a.A[a.d.net[row / a.d.B] * nc + e]);
    float h = start != nullptr ? start[i] : 0.f;
#pragma unroll 4
    for (int k = 0; k < a.nchunk; ++k) {
        const int64_t at = (int64_t)row * a.nchunk + (reverse ? a.nchunk - 1 - k : k);
        const float s = a.sums[at * a.d.C + c], own = a.carry[at * nc + e];
        a.carry[at * nc + e] = h;
        h = join_chunk(A, s, own, h);
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------------------
// G_t = C_t dys_t + exp(dt_{t+1} A) G_{t+1} (dys: dy through the gate); a chunk leaves exp(dt_t A) G_t of its first step.
// CARRY pass of a split sequence: what a chunk leaves by itself, and its sum of dt.
template <class T, int NL, int NS>
__global__ __launch_bounds__(256) void ssm_scan_bwd_carry_kernel(ScanArgs a) {
    constexpr int NP = NS * NL, KG = K / NS;
    __shared__ float lds[4][2][K * NP];
    const int wv = uni(threadIdx.x >> 6);
    const int item = blockIdx.x * 4 + wv;
    if (item >= a.items) return;
    const int ncb = a.d.G * a.nblk, rc = uni(item / ncb), cb = item - rc * ncb;
    const int row = uni(rc / a.nchunk), ch = rc - row * a.nchunk, p = uni(row / a.d.B), b = row - p * a.d.B;
    const Lane<NL, NS> q(a, cb, threadIdx.x & 63);
    const int N = a.d.N, C = a.d.C, net = a.d.net[p], len = uni(seq_len(a.lengths, b, a.d.S)), lane = q.lane;
    const int first = ch * a.chunk, last = first + a.chunk < a.d.S ? first + a.chunk : a.d.S, end = len < last ? len : last;
    const int tl = first + (end - 1 - first) / K * K;  // the last block
    SeqPtr<T, NS> ds(a.delta, q, p, b, tl), zs(a.z, q, p, b, tl), gs(a.dy, q, p, b, tl);
    MapsPtr<T, NP, 64> ms(a, p, b, q.grp, tl, threadIdx.x & 63);
    const bool gated = a.z.data != nullptr;
    float A[NL], dh[NL];
    load_rates(a, q, net, A);
    load_state(a, q, (const float*)nullptr, dh);
    const int co = q.chan_off(4);
    const float bias = row_load(a.bias + (int64_t)net * C + q.first, a.bias != nullptr ? ROW_MAX : 0, co);
    float *lb = lds[wv][0], *lc = lds[wv][1];
    float total = 0.f;
    Raw<T> dr[KG], z[KG], gy[KG];
    Maps<T, NP, 64> maps;
    int rs;
    auto request = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KG; ++i) {
            const int out = behind(t0 + i * NS, q.g, end);
            ds.load(dr[i], i * NS, out);
            gs.load(gy[i], i * NS, out);
            if (gated) zs.load(z[i], i * NS, out);
        }
        ms.load(maps, t0, end, lane);
        rs = load_reset(a, b, t0, end, lane);
        ds.move(-K);
        zs.move(-K);
        gs.move(-K);
        ms.move(-K);
    };
    if (first < end) request(tl);
    for (int t0 = tl; t0 >= first && first < end; t0 -= K) {
        wave_lds_sync();
        store_maps(maps, lb, lc, lane);
        const unsigned fresh = reset_bits(rs);
        float dt[KG], dys[KG];
#pragma unroll
        for (int i = 0; i < KG; ++i) {
            dt[i] = behind(t0 + i * NS, q.g, end) ? 0.f : step_size(a, dr[i].get(), bias);
            dys[i] = gy[i].get();
            if (gated) {
                const float v = z[i].get();
                dys[i] *= v * sigmoid(v);
            }
        }
        wave_lds_sync();
        if (t0 > first) request(t0 - K);
#pragma unroll
        for (int i = KG - 1; i >= 0; --i) {
            float dts[NS], gys[NS];
            to_groups<NS>(dt[i], dts);
            to_groups<NS>(dys[i], gys);
            total += fresh >> (i * NS + q.g) & 1 ? __builtin_nanf("") : dt[i];
#pragma unroll
            for (int j = NS - 1; j >= 0; --j) {
                const int s = i * NS + j;
#pragma unroll
                for (int n = 0; n < NL; ++n) dh[n] = fmaf(gys[j], lc[s * NP + q.n0 + n], dh[n]) * exp2_fast(dts[j] * A[n]);
                if (fresh >> s & 1) clear(dh);
            }
        }
    }
    store_state(a, q, a.carry + ((int64_t)row * a.nchunk + ch) * N * C, dh);
    float r[NS];
    to_groups<NS>(total, r);
    total = r[0];
#pragma unroll
    for (int j = 1; j < NS; ++j) total += r[j];
    row_store(total, a.sums + ((int64_t)row * a.nchunk + ch) * C + q.first, ROW_MAX, q.g == 0 ? co : OOB);
}

// value i of a step's row of maps (i < NP: dB, else dC)
template <class T, int NP>
__device__ __forceinline__ void put_map(const ScanArgs& a, float v, int64_t om, int64_t pm, int64_t at, int i) {
    const int n = i % NP;
    if (n >= a.d.N) return;
    if (a.pB != nullptr) (i < NP ? a.pB : a.pC)[pm + at + n] = v;
    else static_cast<T*>(i < NP ? a.dB : a.dC)[om + at + n] = down<T>(v);
}

// the waves' shares of a block's dB and dC, in order
template <class T, int NP>
__device__ __forceinline__ void sum_maps(const ScanArgs& a, const float (&red)[WMAX][K * 2 * NP], int64_t om, int64_t pm, int t0, int end, int64_t mst, int nthr) {
    for (int e = threadIdx.x; e < K * 2 * NP; e += nthr) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WMAX; ++w) v += red[w][e];
        const int t = t0 + e / (2 * NP);
        if (t < end) put_map<T, NP>(a, v, om, pm, t * mst, e % (2 * NP));
    }
}

// Blocks of K steps from the last to the first: a block's states are recomputed from its record into registers, then its steps run backwards.
// A workgroup's waves own neighbouring channels of the same rows: they share B and C in LDS and add up their shares of dB and dC there (sums over
// channels are sums over lanes: pair_sums).  Sums over rows stay in registers until the end.  Bound by the vector ALUs: 501 steps x 128 rows x 256
// channels bf16 take 260 us with 29 instructions a state of a step (counted), the ALUs busy 86 % of the time that the compute units are (two waves a
// SIMD: a block's states fill the registers).  About 7 of the 29 recompute the states, 15 walk back over them - a third of those merge lanes for dB
// and dC - and the rest are inputs, sums over waves, stores and scalars that spill.  26 steps x 1024 rows x 128 channels f32: 73 us; its last block
// of 8 steps has 2 that are there, and all 8 are worked on.
template <class T, int NL, int NS>
__global__ __launch_bounds__(64 * WMAX, 2) void ssm_scan_bwd_kernel(ScanArgs a) {
    constexpr int NP = NS * NL, KG = K / NS, TOP = 32 / NS;
    constexpr bool KEEP = NL == 4;  // decays stay in registers between the two walks over a block: with 8 states a lane there is no room for them
    // two of each: a block's shares are added up while the next block is worked on, so that one barrier a block does
    __shared__ float maps_lds[2][2][K * NP], red[2][WMAX][K * 2 * NP];
    const int wv = uni(threadIdx.x >> 6), nthr = a.wpb * 64;
    for (int i = threadIdx.x; i < 2 * WMAX * K * 2 * NP; i += nthr) (&red[0][0][0])[i] = 0.f;  // waves that this workgroup does not have
    int buf = 0;
    // workgroup -> (agent, slot, channel group, run of blocks)
    const int gw = a.d.G * a.wgs, ps = uni((int)blockIdx.x / gw), wg = (int)blockIdx.x - ps * gw, p = uni(ps / a.slots), slot = ps - p * a.slots;
    const int grp = uni(wg / a.wgs), run = wg - grp * a.wgs;
    const int kblk = run * a.wpb + wv;  // may lie behind the last block: such a wave has no channels and only helps along
    Lane<NL, NS> q(a, grp * a.nblk + (kblk < a.nblk ? kblk : a.nblk - 1), threadIdx.x & 63);
    if (kblk >= a.nblk) q.act = false;
    const int N = a.d.N, C = a.d.C, S = a.d.S, NB = a.d.B, net = a.d.net[p], lane = q.lane;
    float A[NL], dA[NL];
    load_rates(a, q, net, A);
#pragma unroll
    for (int n = 0; n < NL; ++n) dA[n] = 0.f;
    const int co = q.chan_off(4);
    const float D = row_load(a.D + (int64_t)net * C + q.first, a.D != nullptr ? ROW_MAX : 0, co);
    const float bias = row_load(a.bias + (int64_t)net * C + q.first, a.bias != nullptr ? ROW_MAX : 0, co);
    float dD = 0.f, dbias = 0.f;
    const int64_t yst = (int64_t)NB * C, mst = (int64_t)NB * a.d.G * N;
    const int yoff = q.act ? q.g * (int)(yst * (int64_t)sizeof(T)) + q.cl * (int)sizeof(T) : OOB;
    const bool gated = a.z.data != nullptr;
    for (int it = slot; it < NB * a.nchunk; it += a.slots) {
        const int b = uni(it / a.nchunk), ch = it - b * a.nchunk;
        const int row = p * NB + b, len = uni(seq_len(a.lengths, b, S));
        const int first = ch * a.chunk, last = first + a.chunk < S ? first + a.chunk : S, end = len < last ? len : last;
        const int tl = first + (end - 1 - first) / K * K;  // the last block
        SeqPtr<T, NS> xs(a.x, q, p, b, tl), ds(a.delta, q, p, b, tl), zs(a.z, q, p, b, tl), gs(a.dy, q, p, b, tl);
        MapsPtr<T, NP, 64> ms(a, p, b, grp, tl, lane);
        const int64_t o = ((int64_t)p * S * NB + b) * C + q.first, om = (((int64_t)p * S * NB + b) * a.d.G + grp) * N;
        const int64_t pm = om + (int64_t)run * a.d.P * S * NB * a.d.G * N;
        T *dxp = static_cast<T*>(a.dx) + o, *ddp = static_cast<T*>(a.ddelta) + o, *dzp = static_cast<T*>(a.dz) + o;
        float dh[NL];
        load_state(a, q, a.nchunk > 1 ? a.carry + ((int64_t)row * a.nchunk + ch) * N * C : (a.dh_out != nullptr ? a.dh_out + (int64_t)row * N * C : nullptr), dh);
        for (int t = last - 1; t >= end && t >= first; --t) {  // behind the end
            const int off = q.g == 0 ? q.chan_off(sizeof(T)) : OOB;
            row_store(0.f, dxp + t * yst, ROW_MAX, off);
            row_store(0.f, ddp + t * yst, ROW_MAX, off);
            if (gated) row_store(0.f, dzp + t * yst, ROW_MAX, off);
            for (int i = threadIdx.x; i < 2 * NP; i += nthr) put_map<T, NP>(a, 0.f, om, pm, t * mst, i);
        }
        Raw<T> xr[KG], dr[KG], zr[KG], gr[KG];
        Maps<T, NP, 64> maps;
        int rs;
        float hb[NL];  // the state the block starts from
        auto request = [&](int t0) __attribute__((always_inline)) {  // the pointers are at t0
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                const int out = behind(t0 + i * NS, q.g, end);
                xs.load(xr[i], i * NS, out);
                ds.load(dr[i], i * NS, out);
                gs.load(gr[i], i * NS, out);
                if (gated) zs.load(zr[i], i * NS, out);
            }
            rs = load_reset(a, b, t0, end, lane);
            load_state(a, q, a.record + ((int64_t)row * a.nck + t0 / K) * N * C, hb);
            if (wv == 0) ms.load(maps, t0, end, lane);
            xs.move(-K);
            ds.move(-K);
            zs.move(-K);
            gs.move(-K);
            ms.move(-K);
        };
        if (first < end) request(tl);
        for (int t0 = tl; t0 >= first && first < end; t0 -= K) {
            float hs[K + 1][NL];                       // hs[s]: the state before step s; hs[K]: after the block
            float x[KG], dt[KG], dys[KG], sd[KG], zv[KG];  // sd: the step size's slope
            float *lb = maps_lds[buf][0], *lc = maps_lds[buf][1];
            if (wv == 0) store_maps(maps, lb, lc, lane);
            const unsigned fresh = reset_bits(rs);
#pragma unroll
            for (int n = 0; n < NL; ++n) hs[0][n] = hb[n];
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                const float raw = dr[i].get() + bias;
                x[i] = xr[i].get();
                dys[i] = gr[i].get();
                zv[i] = gated ? zr[i].get() : 0.f;
                // a step behind the end changes nothing: dt = 0, x = 0, dy = 0
                dt[i] = behind(t0 + i * NS, q.g, end) ? 0.f : (a.softplus ? softplus(raw) : raw);
                sd[i] = a.softplus ? sigmoid(raw) : 1.f;
            }
            __syncthreads();
            if (t0 > first) request(t0 - K);
            if (t0 < tl) sum_maps<T, NP>(a, red[buf ^ 1], om, pm, t0 + K, end, mst, nthr);
            int t1 = uni(t0);
            // two forms of the block's steps, as forwards: without resets no step has a branch or a select
            auto steps = [&](auto plain) __attribute__((always_inline)) {
                constexpr bool PLAIN = decltype(plain)::v;
                float ea[KEEP ? K : 1][NL], keep_dt[KEEP ? KG : 1][NS], keep_u[KEEP ? KG : 1][NS];
#pragma unroll
                for (int i = 0; i < KG; ++i) {
                    const int out = behind(t0 + i * NS, q.g, end);
                    float dts[NS], us[NS], ys[NS];
                    to_groups<NS>(dt[i], dts);
                    to_groups<NS>(dt[i] * x[i], us);
                    if (KEEP) {
#pragma unroll
                        for (int j = 0; j < NS; ++j) {
                            keep_dt[KEEP ? i : 0][j] = dts[j];
                            keep_u[KEEP ? i : 0][j] = us[j];
                        }
                    }
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        const int s = i * NS + j;
                        // a reset: the step starts from 0.  hs[s] stays what it is, the state after the step before, whose dC is made of it
                        int lre = !PLAIN && (fresh >> s & 1);
                        if (!PLAIN) asm volatile("" : "+v"(lre));  // a lane's own flag: a select a state, where the compiler would branch for each
                        float y = 0.f;
#pragma unroll
                        for (int n = 0; n < NL; ++n) {
                            const float ex = exp2_fast(dts[j] * A[n]);
                            if (KEEP) ea[KEEP ? s : 0][n] = ex;
                            const float ub = us[j] * lb[s * NP + q.n0 + n], hn = fmaf(ex, hs[s][n], ub);
                            hs[s + 1][n] = lre == 0 ? hn : ub;
                            y = fmaf(hs[s + 1][n], lc[s * NP + q.n0 + n], y);
                        }
                        ys[j] = y;
                    }
                    if (gated) {
                        const float y = fmaf(D, x[i], from_groups<NS>(ys)), z = zv[i], sg = sigmoid(z);
                        row_store(dys[i] * y * sg * fmaf(z, 1.f - sg, 1.f), dzp + (t0 + i * NS) * yst, ROW_MAX, yoff | out);
                        dys[i] *= z * sg;
                    }
                }
                // below, addresses, maps and (8 states a lane) decays are formed anew: kept from above they would take the registers of a wave
                asm volatile("" : "+s"(t1)::"memory");
#pragma unroll
                for (int i = KG - 1; i >= 0; --i) {
                    if (!KEEP) asm volatile("" : "+v"(dt[i]));
                    float dts[NS], us[NS], gys[NS], gb[NS], ga[NS];
                    if (KEEP) {
#pragma unroll
                        for (int j = 0; j < NS; ++j) {
                            dts[j] = keep_dt[KEEP ? i : 0][j];
                            us[j] = keep_u[KEEP ? i : 0][j];
                        }
                    } else {
                        to_groups<NS>(dt[i], dts);
                        to_groups<NS>(dt[i] * x[i], us);
                    }
                    to_groups<NS>(dys[i], gys);
#pragma unroll
                    for (int j = NS - 1; j >= 0; --j) {
                        const int s = i * NS + j;
                        const bool re = !PLAIN && (fresh >> s & 1);  // nothing goes from the step to the state before it
                        float sb = 0.f, sa = 0.f;
                        auto state = [&](auto idx, float& vb, float& vc) __attribute__((always_inline)) {
                            constexpr int n = decltype(idx)::v;
                            vc = gys[j] * hs[s + 1][n];  // dC
                            const float gn = fmaf(gys[j], lc[s * NP + q.n0 + n], dh[n]);
                            vb = gn * us[j];             // dB
                            sb = fmaf(gn, lb[s * NP + q.n0 + n], sb);
                            dh[n] = gn * (KEEP ? ea[KEEP ? s : 0][n] : exp2_fast(dts[j] * A[n]));
                            float w = dh[n] * hs[s][n];
                            if (!PLAIN) {
                                w = re ? 0.f : w;
                                dh[n] = re ? 0.f : dh[n];
                            }
                            sa = fmaf(w, A[n], sa);
                            dA[n] = fmaf(w, dts[j], dA[n]);
                        };
                        const float sum = pair_sums<NL, TOP>(state, lane);
                        gb[j] = sb;
                        ga[j] = sa;
                        red[buf][wv][s * 2 * NP + (lane / TOP & 1) * NP + q.n0 + (lane / (TOP / NL) & (NL - 1))] = sum;
                    }
                    const int out = behind(t1 + i * NS, q.g, end);
                    const float b_ = from_groups<NS>(gb), a_ = from_groups<NS>(ga);
                    dD = fmaf(dys[i], x[i], dD);
                    const float dd = out ? 0.f : fmaf(LN2, a_, b_ * x[i]) * sd[i];
                    dbias += dd;
                    row_store(fmaf(dys[i], D, b_ * dt[i]), dxp + (t1 + i * NS) * yst, ROW_MAX, yoff | out);
                    row_store(dd, ddp + (t1 + i * NS) * yst, ROW_MAX, yoff | out);
                }
            };
            if (fresh == 0) steps(Idx<1>{});
            else steps(Idx<0>{});
            buf ^= 1;
        }
        if (first < end) {
            __syncthreads();
            sum_maps<T, NP>(a, red[buf ^ 1], om, pm, first, end, mst, nthr);
        }
        if (a.dh_in != nullptr && ch == 0) store_state(a, q, a.dh_in + (int64_t)row * N * C, dh);
    }
    float* part = a.part + ((int64_t)(p * a.slots + slot) * (N + 2)) * C;
    store_state(a, q, part, dA);
    float r[NS];
    to_groups<NS>(dD, r);
    dD = r[0];
#pragma unroll
    for (int j = 1; j < NS; ++j) dD += r[j];
    to_groups<NS>(dbias, r);
    dbias = r[0];
#pragma unroll
    for (int j = 1; j < NS; ++j) dbias += r[j];
    const int po = q.g == 0 ? co : OOB;
    row_store(dD, part + (int64_t)N * C + q.first, ROW_MAX, po);
    row_store(dbias, part + (int64_t)(N + 1) * C + q.first, ROW_MAX, po);
}

// dB / dC: the workgroups' partial sums, in order
template <class T>
__global__ __launch_bounds__(256) void ssm_maps_sum_kernel(const float* __restrict__ pB, const float* __restrict__ pC, T* __restrict__ dB, T* __restrict__ dC,
                                                           int nblk, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float sb = 0.f, sc = 0.f;
        for (int k = 0; k < nblk; ++k) {
            sb += pB[k * n + i];
            sc += pC[k * n + i];
        }
        dB[i] = down<T>(sb);
        dC[i] = down<T>(sc);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------------
int scan_validate(const marlhip_ssm_shape* s) {
    if (ssm_validate(s, "ssm_scan") != 0) return -1;
    MARL_REQUIRE(s->state >= 1 && s->state <= SSM_MAX_STATE, "ssm_scan: %d states a channel (1..%d supported)", s->state, SSM_MAX_STATE);
    MARL_REQUIRE(s->groups >= 1 && s->channels % s->groups == 0, "ssm_scan: %d groups of %d channels", s->groups, s->channels);
    return 0;
}

struct ScanPlan {
    int NL, NS, nblk, chunk, nchunk, nck, wpb, wgs, slots;
};

// How a call is split.  A row of N states a channel takes N / 8 x C / 64 waves with 8 states a lane; the chip has 1024 SIMDs and wants about
// four waves on each.
//   <= 512 waves and long enough: the sequences are cut into chunks of at least 64 steps for 4096 waves.  That costs a first pass of about 0.8
//     of the second (16384 steps x 512 channels bf16: 12300 us in one piece, 29 + 13 + 36 us in 256 chunks).
//   <= 1024 waves otherwise: 4 states a lane, twice the waves for a sixth more instructions (501 steps x 128 rows x 256 channels bf16: forwards
//     113 -> 97 us; cut into 4 chunks 141.  Backwards 486 -> 262; cut 330.  With 2048 waves 8 a lane are better: 128 steps x 256 rows x 256
//     channels, forwards with the record 51 against 57 us, backwards 144 against 147).
ScanPlan scan_plan(const marlhip_ssm_shape* s) {
    constexpr int64_t CUT_WAVES = 512, FEW_WAVES = 1024, WANT_WAVES = 4096;
    constexpr int CUT_STEPS = 64;
    ScanPlan q;
    const int Cg = s->channels / s->groups;
    auto lanes = [&](int nl, int ns) {
        q.NL = nl;
        q.NS = ns;
        q.nblk = (Cg + 64 / ns - 1) / (64 / ns);
        return (int64_t)s->n_agents * s->batch * s->groups * q.nblk;
    };
    const bool cuts = s->steps >= 2 * CUT_STEPS;
    auto choose = [&](int nl, int ns) {
        const int64_t w = lanes(nl, ns);
        return w > FEW_WAVES || (cuts && w <= CUT_WAVES) ? w : lanes(nl / 2, ns * 2);
    };
    const int64_t waves = s->state <= 4 ? lanes(4, 1) : (s->state <= 8 ? choose(8, 1) : (s->state <= 16 ? choose(8, 2) : lanes(8, 4)));
    q.nck = (s->steps + K - 1) / K;
    q.nchunk = 1;
    q.chunk = q.nck > 0 ? q.nck * K : K;
    if (waves > 0 && waves <= CUT_WAVES && cuts) {
        const int64_t want = WANT_WAVES / waves, most = s->steps / CUT_STEPS;
        const int64_t n = want < most ? want : most;
        if (n > 1) {
            q.chunk = (int)((q.nck + n - 1) / n) * K;
            q.nchunk = (s->steps + q.chunk - 1) / q.chunk;
        }
    }
    q.wpb = q.nblk < WMAX ? q.nblk : WMAX;
    q.wgs = (q.nblk + q.wpb - 1) / q.wpb;
    // items of one agent that a backward workgroup takes one after the other (its sums over them stay in registers): 4096 waves for them all
    const int64_t items = (int64_t)s->batch * q.nchunk, k = WANT_WAVES / ((int64_t)s->n_agents * s->groups * q.wgs * q.wpb);
    q.slots = (int)(items < 1 ? 1 : (items < k ? items : (k < 1 ? 1 : k)));
    return q;
}

int64_t scan_items(const marlhip_ssm_shape* s, const ScanPlan& pl) { return (int64_t)s->n_agents * s->batch * pl.nchunk * s->groups * pl.nblk; }

int seq_check(const char* what, const char* name, const marlhip_ssm_seq& q, int esize, int64_t steps, int log_bytes) {
    MARL_REQUIRE(q.data == nullptr || steps <= 1 || (q.step_stride >= 0 && q.step_stride <= (1ll << log_bytes) / esize),
                 "%s: %s has %lld elements between steps (0..2^%d bytes supported)", what, name, (long long)q.step_stride, log_bytes);
    return 0;
}
int scan_seqs(const char* what, const marlhip_ssm_shape* s, const marlhip_ssm_scan_args* q, bool grad) {
    const int e = s->dtype == 0 ? 4 : 2;
    // 32-bit offsets run over up to 4 steps of a sequence, over 8 of a map
    if (seq_check(what, "x", q->x, e, s->steps, 29) || seq_check(what, "delta", q->delta, e, s->steps, 29) || seq_check(what, "z", q->z, e, s->steps, 29)) return -1;
    if (grad && seq_check(what, "dy", q->dy, e, s->steps, 29)) return -1;
    if (seq_check(what, "B", q->B, e, s->steps, 28) || seq_check(what, "C", q->C, e, s->steps, 28)) return -1;
    MARL_REQUIRE(scan_items(s, scan_plan(s)) < (1ll << 31) - 8, "%s: batch %d x channels %d is too large", what, s->batch, s->channels);
    MARL_REQUIRE(s->steps <= 1 || (int64_t)s->batch * s->channels * e <= (1ll << 29), "%s: batch %d x channels %d: a step is over 2^29 bytes", what, s->batch,
                 s->channels);
    return 0;
}

ScanArgs scan_args(const marlhip_ssm_shape* s, const marlhip_ssm_scan_args* q, const ScanPlan& pl) {
    ScanArgs a = {};
    a.d = ssm_dims(s);
    a.x = ssm_seq(q->x); a.delta = ssm_seq(q->delta); a.Bm = ssm_seq(q->B); a.Cm = ssm_seq(q->C); a.z = ssm_seq(q->z); a.dy = ssm_seq(q->dy);
    a.A = q->A; a.D = q->D; a.bias = q->delta_bias; a.h_in = q->h_in; a.dh_out = q->dh_out;
    a.reset = q->reset; a.lengths = q->lengths;
    a.y = q->y; a.dx = q->dx; a.ddelta = q->ddelta; a.dB = q->dB; a.dC = q->dC; a.dz = q->dz;
    a.h_out = q->h_out; a.record = q->record; a.dh_in = q->dh_in;
    a.softplus = q->softplus != 0;
    a.nblk = pl.nblk; a.nck = pl.nck; a.chunk = pl.chunk; a.nchunk = pl.nchunk; a.wpb = pl.wpb; a.wgs = pl.wgs; a.slots = pl.slots;
    return a;
}

int64_t round256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// f(type, states a lane, lanes a channel)
template <class F>
void by_type_and_lanes(const marlhip_ssm_shape* s, const ScanPlan& pl, F f) {
    auto by_lanes = [&](auto t) {
        if (pl.NL == 8) {
            if (pl.NS == 1) f(t, Idx<8>{}, Idx<1>{});
            else if (pl.NS == 2) f(t, Idx<8>{}, Idx<2>{});
            else f(t, Idx<8>{}, Idx<4>{});
        } else {
            if (pl.NS == 1) f(t, Idx<4>{}, Idx<1>{});
            else if (pl.NS == 2) f(t, Idx<4>{}, Idx<2>{});
            else f(t, Idx<4>{}, Idx<4>{});
        }
    };
    if (s->dtype == 0) by_lanes(float{});
    else if (s->dtype == 1) by_lanes(__bf16{});
    else by_lanes(_Float16{});
}

struct CarryWs {
    int64_t carry, sums, total;
};
CarryWs carry_ws(const marlhip_ssm_shape* s, const ScanPlan& pl) {
    CarryWs w = {0, 0, 0};
    if (pl.nchunk <= 1) return w;
    const int64_t rows = (int64_t)s->n_agents * s->batch * pl.nchunk;
    w.sums = round256(rows * s->state * s->channels * 4);
    w.total = w.sums + round256(rows * s->channels * 4);
    return w;
}

int join(const ScanArgs& a, const float* start, int reverse, hipStream_t st) {
    if (a.nchunk <= 16) {
        const int64_t wgs = ((int64_t)a.d.P * a.d.B * a.d.N * a.d.C + 255) / 256;
        MARL_REQUIRE(wgs < (1ll << 31), "ssm_scan: too many rows");
        hipLaunchKernelGGL(ssm_scan_join_few_kernel, dim3((unsigned)wgs), dim3(256), 0, st, a, start, reverse);
        MARL_CHECK_LAUNCH("ssm_scan_join_few_kernel");
        return 0;
    }
    const int64_t wgs = (int64_t)a.d.P * a.d.B * a.d.N * ((a.d.C + 63) / 64);
    MARL_REQUIRE(wgs < (1ll << 31), "ssm_scan: too many rows");
    hipLaunchKernelGGL(ssm_scan_join_kernel, dim3((unsigned)wgs), dim3(1024), 0, st, a, start, reverse);
    MARL_CHECK_LAUNCH("ssm_scan_join_kernel");
    return 0;
}

int scan_step(const marlhip_ssm_shape* s, ScanArgs a, hipStream_t st) {
    a.nblk = (s->channels / s->groups + 63) / 64;
    const int64_t per = (int64_t)s->n_agents * s->groups * a.nblk;  // waves that one row of every agent takes
    const int64_t slots = STEP_WAVES / per;
    a.slots = (int)(slots < 1 ? 1 : (slots < s->batch ? slots : s->batch));
    a.items = (int)(per * a.slots);
    const dim3 grid((unsigned)((a.items + 3) / 4));
    auto by_state = [&](auto t) {
        using T = decltype(t);
        if (s->state <= 8) hipLaunchKernelGGL((ssm_scan_step_kernel<T, 8>), grid, dim3(256), 0, st, a);
        else if (s->state <= 16) hipLaunchKernelGGL((ssm_scan_step_kernel<T, 16>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((ssm_scan_step_kernel<T, 32>), grid, dim3(256), 0, st, a);
    };
    if (s->dtype == 0) by_state(float{});
    else if (s->dtype == 1) by_state(__bf16{});
    else by_state(_Float16{});
    MARL_CHECK_LAUNCH("ssm_scan_step_kernel");
    return 0;
}

}  // namespace

extern "C" int64_t marlhip_ssm_scan_record_floats(const marlhip_ssm_shape* s) {
    if (scan_validate(s) != 0) return -1;
    return (int64_t)s->n_agents * s->batch * ((s->steps + K - 1) / K) * s->state * s->channels;
}

extern "C" int64_t marlhip_ssm_scan_workspace_bytes(const marlhip_ssm_shape* s) {
    if (scan_validate(s) != 0) return -1;
    return carry_ws(s, scan_plan(s)).total;
}

extern "C" int marlhip_ssm_scan(const marlhip_ssm_shape* s, const marlhip_ssm_scan_args* q, void* workspace, int64_t workspace_bytes, void* stream) {
    if (scan_validate(s) != 0) return -1;
    MARL_REQUIRE(q != nullptr && q->A != nullptr, "ssm_scan: NULL argument");
    const bool any = s->steps > 0 && s->batch > 0;
    MARL_REQUIRE(!any || (q->x.data && q->delta.data && q->B.data && q->C.data && q->y), "ssm_scan: NULL pointer");
    if (scan_seqs("ssm_scan", s, q, false) != 0) return -1;
    const ScanPlan pl = scan_plan(s);
    const CarryWs w = carry_ws(s, pl);
    MARL_REQUIRE(w.total == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= w.total),
                 "ssm_scan: aligned workspace of %lld bytes needed, %lld given", (long long)w.total, (long long)workspace_bytes);
    if (s->batch == 0) return 0;
    ScanArgs a = scan_args(s, q, pl);
    if (s->steps == 1 && a.record == nullptr) return scan_step(s, a, (hipStream_t)stream);
    a.items = (int)scan_items(s, pl);
    const dim3 grid((unsigned)((a.items + 3) / 4));
    hipStream_t st = (hipStream_t)stream;
    if (pl.nchunk > 1) {
        a.carry = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.carry);
        a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.sums);
        by_type_and_lanes(s, pl, [&](auto t, auto nl, auto ns) {
            hipLaunchKernelGGL((ssm_scan_fwd_kernel<decltype(t), decltype(nl)::v, decltype(ns)::v, CARRY_PASS>), grid, dim3(256), 0, st, a);
        });
        MARL_CHECK_LAUNCH("ssm_scan_fwd_kernel");
        if (join(a, a.h_in, 0, st) != 0) return -2;
    }
    by_type_and_lanes(s, pl, [&](auto t, auto nl, auto ns) {
        constexpr int NL = decltype(nl)::v, NS = decltype(ns)::v;
        if (a.record != nullptr) hipLaunchKernelGGL((ssm_scan_fwd_kernel<decltype(t), NL, NS, RECORD_PASS>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((ssm_scan_fwd_kernel<decltype(t), NL, NS, STEPS_PASS>), grid, dim3(256), 0, st, a);
    });
    MARL_CHECK_LAUNCH("ssm_scan_fwd_kernel");
    return 0;
}

namespace {
struct GradWs {
    int64_t pB, pC, part, total;
    CarryWs carry;
};
GradWs grad_ws(const marlhip_ssm_shape* s, const ScanPlan& pl) {
    GradWs w;
    w.carry = carry_ws(s, pl);
    int64_t off = w.carry.total;
    auto take = [&](int64_t floats) { const int64_t o = off; off += round256(floats * 4); return o; };
    const int64_t maps = pl.wgs > 1 ? (int64_t)pl.wgs * s->n_agents * s->steps * s->batch * s->groups * s->state : 0;
    w.pB = take(maps);
    w.pC = take(maps);
    w.part = take((int64_t)s->n_agents * pl.slots * (s->state + 2) * s->channels);
    w.total = off;
    return w;
}
}  // namespace

extern "C" int64_t marlhip_ssm_scan_grad_workspace_bytes(const marlhip_ssm_shape* s) {
    if (scan_validate(s) != 0) return -1;
    return grad_ws(s, scan_plan(s)).total;
}

extern "C" int marlhip_ssm_scan_grad(const marlhip_ssm_shape* s, const marlhip_ssm_scan_args* q, void* workspace, int64_t workspace_bytes, void* stream) {
    if (scan_validate(s) != 0) return -1;
    MARL_REQUIRE(q != nullptr && q->A != nullptr && q->dA != nullptr, "ssm_scan_grad: NULL argument");
    const bool any = s->steps > 0 && s->batch > 0;
    MARL_REQUIRE(!any || (q->x.data && q->delta.data && q->B.data && q->C.data && q->dy.data && q->record && q->dx && q->ddelta && q->dB && q->dC),
                 "ssm_scan_grad: NULL pointer");
    MARL_REQUIRE(!any || (q->z.data == nullptr) == (q->dz == nullptr), "ssm_scan_grad: dz goes with z");
    if (scan_seqs("ssm_scan_grad", s, q, true) != 0) return -1;
    const ScanPlan pl = scan_plan(s);
    const GradWs w = grad_ws(s, pl);
    MARL_REQUIRE(workspace != nullptr && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= w.total,
                 "ssm_scan_grad: aligned workspace of %lld bytes needed, %lld given", (long long)w.total, (long long)workspace_bytes);
    ScanArgs a = scan_args(s, q, pl);
    char* ws = static_cast<char*>(workspace);
    hipStream_t st = (hipStream_t)stream;
    a.part = reinterpret_cast<float*>(ws + w.part);
    if (pl.wgs > 1) {
        a.pB = reinterpret_cast<float*>(ws + w.pB);
        a.pC = reinterpret_cast<float*>(ws + w.pC);
    }
    if (pl.nchunk > 1) {
        a.carry = reinterpret_cast<float*>(ws + w.carry.carry);
        a.sums = reinterpret_cast<float*>(ws + w.carry.sums);
        a.items = (int)scan_items(s, pl);
        const dim3 grid((unsigned)((a.items + 3) / 4));
        by_type_and_lanes(s, pl, [&](auto t, auto nl, auto ns) {
            hipLaunchKernelGGL((ssm_scan_bwd_carry_kernel<decltype(t), decltype(nl)::v, decltype(ns)::v>), grid, dim3(256), 0, st, a);
        });
        MARL_CHECK_LAUNCH("ssm_scan_bwd_carry_kernel");
        if (join(a, a.dh_out, 1, st) != 0) return -2;
    }
    const dim3 grid((unsigned)(s->n_agents * pl.slots * s->groups * pl.wgs)), block(64 * pl.wpb);
    by_type_and_lanes(s, pl, [&](auto t, auto nl, auto ns) { hipLaunchKernelGGL((ssm_scan_bwd_kernel<decltype(t), decltype(nl)::v, decltype(ns)::v>), grid, block, 0, st, a); });
    MARL_CHECK_LAUNCH("ssm_scan_bwd_kernel");
    const int64_t maps = (int64_t)s->n_agents * s->steps * s->batch * s->groups * s->state;
    if (pl.wgs > 1 && maps > 0) {
        const unsigned blocks = (unsigned)((maps + 255) / 256 < 4096 ? (maps + 255) / 256 : 4096);
#define MAPS_SUM(T) hipLaunchKernelGGL((ssm_maps_sum_kernel<T>), dim3(blocks), dim3(256), 0, st, a.pB, a.pC, (T*)q->dB, (T*)q->dC, pl.wgs, maps)
        if (s->dtype == 0) MAPS_SUM(float);
        else if (s->dtype == 1) MAPS_SUM(__bf16);
        else MAPS_SUM(_Float16);
#undef MAPS_SUM
        MARL_CHECK_LAUNCH("ssm_maps_sum_kernel");
    }
    const int64_t cols = (int64_t)(s->state + 2) * s->channels;
    hipLaunchKernelGGL(ssm_weights_sum_kernel, dim3((unsigned)((cols + 63) / 64), a.d.M), dim3(1024), 0, st, a.d, pl.slots, s->state, 2, a.part, q->dA, q->dD,
                       q->ddelta_bias);
    MARL_CHECK_LAUNCH("ssm_weights_sum_kernel");
    return 0;
}
