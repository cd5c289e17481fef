// Selective state space scan: marlhip_ssm_scan (forward, any number of steps, one included) and marlhip_ssm_scan_grad.
//
//   h_t[n] = exp(dt_t A[n]) h_{t-1}[n] + dt_t B_t[n] x_t,   y_t = sum_n C_t[n] h_t[n] + D x_t        for every channel
//
// A wave owns 64 channels of one row and walks its steps with the state in registers; B and C of a step are the same for all of them and
// come as LDS broadcasts.
#include "ssm.h"

using namespace marl;

namespace {

struct ScanArgs {
    SsmDims d;
    SsmSeq x, delta, Bm, Cm, z, dy;
    const float *A, *D, *bias, *h_in, *dh_out;
    const uint8_t* reset;
    const int32_t* lengths;
    void *y, *dx, *ddelta, *dB, *dC, *dz;
    float *h_out, *record, *dh_in;
    float *pB, *pC;  // [nblk][P][S][B][G][N] partial sums of dB / dC, NULL: one block a group, written to dB / dC directly
    float* part;     // [P][slots][N + 2][C] partial sums of dA, dD, ddelta_bias
    int softplus, nblk, slots, nck;
    int64_t items;
};

// steps between two recorded states: their states of a block stay in registers in the backward pass (K * N of them)
template <int NP>
constexpr int scan_k() { return 128 / NP < 8 ? 4 : (NP == 8 ? 16 : 8); }
inline int scan_np(int N) { return N <= 8 ? 8 : (N <= 16 ? 16 : 32); }
inline int scan_k_of(int N) { return scan_np(N) == 8 ? scan_k<8>() : (scan_np(N) == 16 ? scan_k<16>() : scan_k<32>()); }

// what a wave works on: 64 channels of one group, `bytes`-wise through row descriptors
template <class T>
struct ScanCols {
    int g, kblk, first, nt, nf, vt, vf;  // group, block, first channel; bytes of a row of T / float; this lane's offsets
    __device__ __forceinline__ ScanCols(const ScanArgs& a, int cb, int lane) {
        const int Cg = a.d.C / a.d.G;
        g = cb / a.nblk;
        kblk = cb % a.nblk;
        first = g * Cg + kblk * 64;
        const int left = (g + 1) * Cg - first, valid = left < 64 ? left : 64;
        nt = valid * (int)sizeof(T);
        nf = valid * 4;
        vt = lane * (int)sizeof(T);
        vf = lane * 4;
    }
};

// B and C of K steps from t0 on (zeros behind the end and in the padding up to NP) to the wave's LDS, f32
template <class T, int NP, int K>
__device__ __forceinline__ void stage_maps(const ScanArgs& a, const T* Bp, const T* Cp, int t0, int len, float* lb, float* lc, int lane) {
#pragma unroll
    for (int i = 0; i < (K * NP + 63) / 64; ++i) {
        const int e = lane + 64 * i, s = e / NP, n = e % NP, t = t0 + s;
        if (K * NP >= 64 || e < K * NP) {
            const bool ok = n < a.d.N && t < len;
            lb[e] = ok ? up(Bp[t * a.Bm.st + n]) : 0.f;
            lc[e] = ok ? up(Cp[t * a.Cm.st + n]) : 0.f;
        }
    }
}

template <class T, int NP>
__global__ __launch_bounds__(256) void ssm_scan_fwd_kernel(ScanArgs a) {
    constexpr int K = scan_k<NP>();
    __shared__ float lds[4][2][K * NP];
    const int lane = threadIdx.x & 63, wv = uni(threadIdx.x >> 6);
    const int64_t item = (int64_t)blockIdx.x * 4 + wv;
    if (item >= a.items) return;
    const int N = a.d.N, C = a.d.C, S = a.d.S, ncb = a.d.G * a.nblk;
    const int cb = (int)(item % ncb), row = (int)(item / ncb), p = row / a.d.B, b = row % a.d.B;
    const ScanCols<T> q(a, cb, lane);
    const int net = a.d.net[p], len = uni(seq_len(a.lengths, b, S));
    float A[NP], h[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        A[n] = n < N ? row_load(a.A + ((int64_t)net * N + n) * C + q.first, q.nf, q.vf) * LOG2E : 0.f;
        h[n] = n < N && a.h_in != nullptr ? row_load(a.h_in + ((int64_t)row * N + n) * C + q.first, q.nf, q.vf) : 0.f;
    }
    const float D = a.D != nullptr ? row_load(a.D + (int64_t)net * C + q.first, q.nf, q.vf) : 0.f;
    const float bias = a.bias != nullptr ? row_load(a.bias + (int64_t)net * C + q.first, q.nf, q.vf) : 0.f;
    const T *xp = seq_at<T>(a.x, p, b) + q.first, *dp = seq_at<T>(a.delta, p, b) + q.first, *zp = seq_at<T>(a.z, p, b) + q.first;
    const T *Bp = seq_at<T>(a.Bm, p, b) + q.g * N, *Cp = seq_at<T>(a.Cm, p, b) + q.g * N;
    T* yp = static_cast<T*>(a.y) + ((int64_t)p * S * a.d.B + b) * C + q.first;
    const int64_t yst = (int64_t)a.d.B * C;
    const bool gated = a.z.data != nullptr;
    float *lb = lds[wv][0], *lc = lds[wv][1];
    for (int t0 = 0; t0 < len; t0 += K) {
        wave_lds_sync();
        stage_maps<T, NP, K>(a, Bp, Cp, t0, len, lb, lc, lane);
        if (a.record != nullptr)
#pragma unroll
            for (int n = 0; n < NP; ++n)
                if (n < N) row_store(h[n], a.record + (((int64_t)row * a.nck + t0 / K) * N + n) * C + q.first, q.nf, q.vf);
        wave_lds_sync();
        const int m = len - t0 < K ? len - t0 : K;
        for (int s = 0; s < m; ++s) {
            const int64_t t = t0 + s;
            const float x = row_load(xp + t * a.x.st, q.nt, q.vt), dr = row_load(dp + t * a.delta.st, q.nt, q.vt) + bias;
            const float z = gated ? row_load(zp + t * a.z.st, q.nt, q.vt) : 0.f;
            const float dt = a.softplus ? softplus(dr) : dr, u = dt * x;
            if (a.reset != nullptr && a.reset[t * a.d.B + b] != 0)
#pragma unroll
                for (int n = 0; n < NP; ++n) h[n] = 0.f;
            float y = D * x;
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                h[n] = fmaf(exp2_fast(dt * A[n]), h[n], u * lb[s * NP + n]);
                y = fmaf(h[n], lc[s * NP + n], y);
            }
            if (gated) y *= z * sigmoid(z);
            row_store(y, yp + t * yst, q.nt, q.vt);
        }
    }
    for (int t = len; t < S; ++t) row_store(0.f, yp + t * yst, q.nt, q.vt);
    if (a.h_out != nullptr)
#pragma unroll
        for (int n = 0; n < NP; ++n)
            if (n < N) row_store(h[n], a.h_out + ((int64_t)row * N + n) * C + q.first, q.nf, q.vf);
}

// Backward: blocks of K steps from the last to the first; a block's states are recomputed from its record into registers, then the steps
// run backwards with G_t = C_t dys_t + exp(dt_{t+1} A) G_{t+1} (dys: dy through the gate).
template <class T, int NP>
__global__ __launch_bounds__(256, NP == 32 ? 1 : 2) void ssm_scan_bwd_kernel(ScanArgs a) {
    constexpr int K = scan_k<NP>();
    __shared__ float lds[4][2][K * NP];
    const int lane = threadIdx.x & 63, wv = uni(threadIdx.x >> 6);
    const int64_t item = (int64_t)blockIdx.x * 4 + wv;
    if (item >= a.items) return;
    const int N = a.d.N, C = a.d.C, S = a.d.S, NB = a.d.B, ncb = a.d.G * a.nblk;
    const int cb = (int)(item % ncb), ps = (int)(item / ncb), p = ps / a.slots, slot = ps % a.slots;
    const ScanCols<T> q(a, cb, lane);
    const int net = a.d.net[p];
    float A[NP], dA[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        A[n] = n < N ? row_load(a.A + ((int64_t)net * N + n) * C + q.first, q.nf, q.vf) * LOG2E : 0.f;
        dA[n] = 0.f;
    }
    const float D = a.D != nullptr ? row_load(a.D + (int64_t)net * C + q.first, q.nf, q.vf) : 0.f;
    const float bias = a.bias != nullptr ? row_load(a.bias + (int64_t)net * C + q.first, q.nf, q.vf) : 0.f;
    float dD = 0.f, dbias = 0.f;
    float *lb = lds[wv][0], *lc = lds[wv][1];
    const int64_t yst = (int64_t)NB * C;
    const int64_t mst = (int64_t)NB * a.d.G * N;  // between steps of dB / dC
    // the lane's place in a row of dB or dC (lanes with nothing to store point behind the row): pair_sums leaves b_n at lane n R, c_n behind
    constexpr int R = 32 / NP;
    const int mi = lane / R, mn = mi % NP;
    const bool mine = lane % R == 0 && mn < N;
    const int me = a.pB != nullptr ? 4 : (int)sizeof(T);
    const int vB = mine && mi < NP ? mn * me : 1 << 30, vC = mine && mi >= NP ? mn * me : 1 << 30;
    const bool gated = a.z.data != nullptr;
    for (int b = slot; b < NB; b += a.slots) {
        const int row = p * NB + b, len = uni(seq_len(a.lengths, b, S));
        const T *xp = seq_at<T>(a.x, p, b) + q.first, *dp = seq_at<T>(a.delta, p, b) + q.first, *zp = seq_at<T>(a.z, p, b) + q.first;
        const T *Bp = seq_at<T>(a.Bm, p, b) + q.g * N, *Cp = seq_at<T>(a.Cm, p, b) + q.g * N, *gp = seq_at<T>(a.dy, p, b) + q.first;
        const int64_t o = ((int64_t)p * S * NB + b) * C + q.first, om = (((int64_t)p * S * NB + b) * a.d.G + q.g) * N;
        const int64_t pm = om + (int64_t)q.kblk * a.d.P * S * NB * a.d.G * N;
        T *dxp = static_cast<T*>(a.dx) + o, *ddp = static_cast<T*>(a.ddelta) + o, *dzp = static_cast<T*>(a.dz) + o;
        auto put_maps = [&](float v, int64_t t, bool in) {
            const int n = in ? N * me : 0;
            if (a.pB != nullptr) {
                row_store(v, a.pB + pm + t * mst, n, vB);
                row_store(v, a.pC + pm + t * mst, n, vC);
            } else {
                row_store(v, static_cast<T*>(a.dB) + om + t * mst, n, vB);
                row_store(v, static_cast<T*>(a.dC) + om + t * mst, n, vC);
            }
        };
        float dh[NP];
#pragma unroll
        for (int n = 0; n < NP; ++n)
            dh[n] = n < N && a.dh_out != nullptr ? row_load(a.dh_out + ((int64_t)row * N + n) * C + q.first, q.nf, q.vf) : 0.f;
        for (int t = S - 1; t >= len; --t) {  // behind the end
            row_store(0.f, dxp + t * yst, q.nt, q.vt);
            row_store(0.f, ddp + t * yst, q.nt, q.vt);
            if (gated) row_store(0.f, dzp + t * yst, q.nt, q.vt);
            put_maps(0.f, t, true);
        }
        for (int t0 = (len - 1) / K * K; t0 >= 0 && len > 0; t0 -= K) {
            wave_lds_sync();
            stage_maps<T, NP, K>(a, Bp, Cp, t0, len, lb, lc, lane);
            wave_lds_sync();
            float hs[K + 1][NP];  // hs[s]: the state before step s; hs[K]: after the block
#pragma unroll
            for (int n = 0; n < NP; ++n)
                hs[0][n] = n < N ? row_load(a.record + (((int64_t)row * a.nck + t0 / K) * N + n) * C + q.first, q.nf, q.vf) : 0.f;
            float x[K], dr[K], dt[K], dys[K], zv[K];
            unsigned fresh = 0;
#pragma unroll
            for (int s = 0; s < K; ++s) {
                const int64_t t = t0 + s;
                const bool in = t < len;  // a step behind the end changes nothing: dt = 0, x = 0, dy = 0
                const int nt = in ? q.nt : 0;
                x[s] = row_load(xp + t * a.x.st, nt, q.vt);
                dr[s] = row_load(dp + t * a.delta.st, nt, q.vt) + bias;
                dys[s] = row_load(gp + t * a.dy.st, nt, q.vt);
                zv[s] = gated ? row_load(zp + t * a.z.st, nt, q.vt) : 0.f;
                if (in && a.reset != nullptr && a.reset[t * NB + b] != 0) fresh |= 1u << s;
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int s = 0; s < K; ++s) {
                const int64_t t = t0 + s;
                const bool in = t < len;
                dt[s] = in ? (a.softplus ? softplus(dr[s]) : dr[s]) : 0.f;
                const float u = dt[s] * x[s];
                // a reset empties the state through the decay, e^-inf = 0; what is not finite has to go by hand
                const bool re = fresh >> s & 1;
                const float fr = re ? -INFINITY : 0.f;
                if (re)
#pragma unroll
                    for (int n = 0; n < NP; ++n) hs[s][n] = fabsf(hs[s][n]) < INFINITY ? hs[s][n] : 0.f;
                float y = D * x[s];
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    hs[s + 1][n] = fmaf(exp2_fast(fmaf(dt[s], A[n], fr)), hs[s][n], u * lb[s * NP + n]);
                    y = fmaf(hs[s + 1][n], lc[s * NP + n], y);
                }
                if (gated) {
                    const float sg = sigmoid(zv[s]);
                    row_store(dys[s] * y * sg * fmaf(zv[s], 1.f - sg, 1.f), dzp + t * yst, in ? q.nt : 0, q.vt);
                    dys[s] *= zv[s] * sg;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            // below, addresses, maps and decays are formed anew: kept from above they would cost more registers than they save time
            int t1 = t0;
            asm volatile("" : "+s"(t1)::"memory");
#pragma unroll
            for (int s = K - 1; s >= 0; --s) {
                asm volatile("" : "+v"(dt[s])::"memory");
                const int64_t t = t1 + s;
                const bool in = t < len;
                const bool re = fresh >> s & 1;
                const float fr = re ? -INFINITY : 0.f, u = dt[s] * x[s];
                float gb = 0.f, ga = 0.f;
                auto state = [&](auto idx, float& vb, float& vc) {
                    constexpr int n = decltype(idx)::v;
                    vc = dys[s] * hs[s + 1][n];  // dC
                    const float gn = fmaf(dys[s], lc[s * NP + n], dh[n]);
                    vb = gn * u;                 // dB
                    gb = fmaf(gn, lb[s * NP + n], gb);
                    dh[n] = gn * exp2_fast(fmaf(dt[s], A[n], fr));
                    const float w = dh[n] * hs[s][n];
                    ga = fmaf(w, A[n], ga);
                    dA[n] = fmaf(w, dt[s], dA[n]);
                };
                const float sum = pair_sums<NP>(state, lane);
                if (re)
#pragma unroll
                    for (int n = 0; n < NP; ++n) dh[n] = 0.f;
                dD = fmaf(dys[s], x[s], dD);
                float dd = fmaf(LN2, ga, gb * x[s]);
                if (a.softplus) dd *= sigmoid(dr[s]);
                if (!in) dd = 0.f;
                dbias += dd;
                row_store(fmaf(dys[s], D, gb * dt[s]), dxp + t * yst, in ? q.nt : 0, q.vt);
                row_store(dd, ddp + t * yst, in ? q.nt : 0, q.vt);
                put_maps(sum, t, in);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (a.dh_in != nullptr)
#pragma unroll
            for (int n = 0; n < NP; ++n)
                if (n < N) row_store(dh[n], a.dh_in + ((int64_t)row * N + n) * C + q.first, q.nf, q.vf);
    }
    float* part = a.part + ((int64_t)(p * a.slots + slot) * (N + 2)) * C + q.first;
#pragma unroll
    for (int n = 0; n < NP; ++n)
        if (n < N) row_store(dA[n], part + (int64_t)n * C, q.nf, q.vf);
    row_store(dD, part + (int64_t)N * C, q.nf, q.vf);
    row_store(dbias, part + (int64_t)(N + 1) * C, q.nf, q.vf);
}

// dB / dC: the channel blocks' partial sums, in order
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

int scan_validate(const marlhip_ssm_shape* s) {
    if (ssm_validate(s, "ssm_scan") != 0) return -1;
    MARL_REQUIRE(s->state >= 1 && s->state <= SSM_MAX_STATE, "ssm_scan: %d states a channel (1..%d supported)", s->state, SSM_MAX_STATE);
    MARL_REQUIRE(s->groups >= 1 && s->channels % s->groups == 0, "ssm_scan: %d groups of %d channels", s->groups, s->channels);
    return 0;
}

int scan_blocks(const marlhip_ssm_shape* s) { return (s->channels / s->groups + 63) / 64; }

// rows of one agent that a wave takes one after the other (its sums over rows stay in registers)
int scan_slots(const marlhip_ssm_shape* s) {
    const int64_t waves = 4096 / ((int64_t)s->n_agents * s->groups * scan_blocks(s));
    const int64_t k = waves < 1 ? 1 : waves;
    return (int)(s->batch < k ? s->batch : k);
}

ScanArgs scan_args(const marlhip_ssm_shape* s, const marlhip_ssm_scan_args* q) {
    ScanArgs a = {};
    a.d = ssm_dims(s);
    a.x = ssm_seq(q->x); a.delta = ssm_seq(q->delta); a.Bm = ssm_seq(q->B); a.Cm = ssm_seq(q->C); a.z = ssm_seq(q->z); a.dy = ssm_seq(q->dy);
    a.A = q->A; a.D = q->D; a.bias = q->delta_bias; a.h_in = q->h_in; a.dh_out = q->dh_out;
    a.reset = q->reset; a.lengths = q->lengths;
    a.y = q->y; a.dx = q->dx; a.ddelta = q->ddelta; a.dB = q->dB; a.dC = q->dC; a.dz = q->dz;
    a.h_out = q->h_out; a.record = q->record; a.dh_in = q->dh_in;
    a.softplus = q->softplus != 0;
    a.nblk = scan_blocks(s);
    const int K = scan_k_of(s->state);
    a.nck = (s->steps + K - 1) / K;
    return a;
}

#define SSM_FOR_TYPE_AND_STATE(call)                                             \
    do {                                                                         \
        const int np_ = scan_np(s->state);                                       \
        if (s->dtype == 0) { if (np_ == 8) { call(float, 8); } else if (np_ == 16) { call(float, 16); } else { call(float, 32); } }            \
        else if (s->dtype == 1) { if (np_ == 8) { call(__bf16, 8); } else if (np_ == 16) { call(__bf16, 16); } else { call(__bf16, 32); } }    \
        else { if (np_ == 8) { call(_Float16, 8); } else if (np_ == 16) { call(_Float16, 16); } else { call(_Float16, 32); } }                 \
    } while (0)

}  // namespace

extern "C" int64_t marlhip_ssm_scan_record_floats(const marlhip_ssm_shape* s) {
    if (scan_validate(s) != 0) return -1;
    const int K = scan_k_of(s->state);
    return (int64_t)s->n_agents * s->batch * ((s->steps + K - 1) / K) * s->state * s->channels;
}

extern "C" int64_t marlhip_ssm_scan_workspace_bytes(const marlhip_ssm_shape* s) {
    if (scan_validate(s) != 0) return -1;
    return 0;
}

extern "C" int marlhip_ssm_scan(const marlhip_ssm_shape* s, const marlhip_ssm_scan_args* q, void* workspace, int64_t workspace_bytes, void* stream) {
    if (scan_validate(s) != 0) return -1;
    MARL_REQUIRE(q != nullptr && q->A != nullptr, "ssm_scan: NULL argument");
    const bool any = s->steps > 0 && s->batch > 0;
    MARL_REQUIRE(!any || (q->x.data && q->delta.data && q->B.data && q->C.data && q->y), "ssm_scan: NULL pointer");
    const int64_t need = marlhip_ssm_scan_workspace_bytes(s);
    MARL_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), "ssm_scan: workspace of %lld bytes needed, %lld given", (long long)need,
                 (long long)workspace_bytes);
    if (s->batch == 0) return 0;
    ScanArgs a = scan_args(s, q);
    a.items = (int64_t)s->n_agents * s->batch * s->groups * a.nblk;
    MARL_REQUIRE((a.items + 3) / 4 < (1ll << 31), "ssm_scan: too many rows");
#define SCAN_FWD(T, NP) hipLaunchKernelGGL((ssm_scan_fwd_kernel<T, NP>), dim3((unsigned)((a.items + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a)
    SSM_FOR_TYPE_AND_STATE(SCAN_FWD);
#undef SCAN_FWD
    MARL_CHECK_LAUNCH("ssm_scan_fwd_kernel");
    return 0;
}

namespace {
struct GradWs {
    int64_t pB, pC, part, total;
    int slots;
};
GradWs grad_ws(const marlhip_ssm_shape* s) {
    GradWs w;
    int64_t off = 0;
    auto take = [&](int64_t floats) { const int64_t o = off; off += (floats * 4 + 255) / 256 * 256; return o; };
    const int64_t maps = scan_blocks(s) > 1 ? (int64_t)scan_blocks(s) * s->n_agents * s->steps * s->batch * s->groups * s->state : 0;
    w.pB = take(maps);
    w.pC = take(maps);
    w.slots = scan_slots(s);
    w.part = take((int64_t)s->n_agents * w.slots * (s->state + 2) * s->channels);
    w.total = off;
    return w;
}
}  // namespace

extern "C" int64_t marlhip_ssm_scan_grad_workspace_bytes(const marlhip_ssm_shape* s) {
    if (scan_validate(s) != 0) return -1;
    return grad_ws(s).total;
}

extern "C" int marlhip_ssm_scan_grad(const marlhip_ssm_shape* s, const marlhip_ssm_scan_args* q, void* workspace, int64_t workspace_bytes, void* stream) {
    if (scan_validate(s) != 0) return -1;
    MARL_REQUIRE(q != nullptr && q->A != nullptr && q->dA != nullptr, "ssm_scan_grad: NULL argument");
    const bool any = s->steps > 0 && s->batch > 0;
    MARL_REQUIRE(!any || (q->x.data && q->delta.data && q->B.data && q->C.data && q->dy.data && q->record && q->dx && q->ddelta && q->dB && q->dC),
                 "ssm_scan_grad: NULL pointer");
    MARL_REQUIRE(!any || (q->z.data == nullptr) == (q->dz == nullptr), "ssm_scan_grad: dz goes with z");
    const GradWs w = grad_ws(s);
    MARL_REQUIRE(w.total == 0 || (workspace != nullptr && workspace_bytes >= w.total), "ssm_scan_grad: workspace of %lld bytes needed, %lld given",
                 (long long)w.total, (long long)workspace_bytes);
    ScanArgs a = scan_args(s, q);
    char* ws = static_cast<char*>(workspace);
    const int64_t maps = (int64_t)s->n_agents * s->steps * s->batch * s->groups * s->state;
    a.slots = w.slots;
    a.part = reinterpret_cast<float*>(ws + w.part);
    if (a.nblk > 1) {
        a.pB = reinterpret_cast<float*>(ws + w.pB);
        a.pC = reinterpret_cast<float*>(ws + w.pC);
    }
    a.items = (int64_t)s->n_agents * w.slots * s->groups * a.nblk;
    hipStream_t st = (hipStream_t)stream;
    if (a.items > 0) {
#define SCAN_BWD(T, NP) hipLaunchKernelGGL((ssm_scan_bwd_kernel<T, NP>), dim3((unsigned)((a.items + 3) / 4)), dim3(256), 0, st, a)
        SSM_FOR_TYPE_AND_STATE(SCAN_BWD);
#undef SCAN_BWD
        MARL_CHECK_LAUNCH("ssm_scan_bwd_kernel");
        if (a.nblk > 1 && maps > 0) {
            const unsigned blocks = (unsigned)((maps + 255) / 256 < 4096 ? (maps + 255) / 256 : 4096);
#define MAPS_SUM(T) hipLaunchKernelGGL((ssm_maps_sum_kernel<T>), dim3(blocks), dim3(256), 0, st, a.pB, a.pC, (T*)q->dB, (T*)q->dC, a.nblk, maps)
            if (s->dtype == 0) MAPS_SUM(float);
            else if (s->dtype == 1) MAPS_SUM(__bf16);
            else MAPS_SUM(_Float16);
#undef MAPS_SUM
            MARL_CHECK_LAUNCH("ssm_maps_sum_kernel");
        }
    }
    const int64_t cols = (int64_t)(s->state + 2) * s->channels;
    hipLaunchKernelGGL(ssm_weights_sum_kernel, dim3((unsigned)((cols + 63) / 64), a.d.M), dim3(256), 0, st, a.d, w.slots, s->state, 2, a.part, q->dA, q->dD,
                       q->ddelta_bias);
    MARL_CHECK_LAUNCH("ssm_weights_sum_kernel");
    return 0;
}
