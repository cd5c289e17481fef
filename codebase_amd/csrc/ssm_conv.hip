// Short causal depthwise convolution with its SiLU: marlhip_ssm_conv (any number of steps, one included) and marlhip_ssm_conv_grad.
//
//   pre_t = bias + sum_j w_j x_{t-j},  y_t = silu(pre_t);   lags j = 0..W-1, none beyond the last reset
//
// A thread owns V neighbouring channels of one row and a stretch of steps; the window slides through its registers.  Bound by HBM, so the loads
// are 16 bytes wide and four steps are in flight: 65536 steps x 1024 channels bf16 take 48 us out of warm caches, 66 us (4.1 TB/s) out of cold ones.
// Stretches in place of one walk through a row give the threads: a stretch reads W - 1 steps again, which the caches hold.
#include "ssm.h"

using namespace marl;

namespace {

struct ConvArgs {
    SsmDims d;
    SsmSeq x, dy;
    const float *weight, *bias;
    const void *state, *dstate_out;
    const uint8_t* reset;
    const int32_t* lengths;
    void *y, *state_out, *dx, *dstate;
    float* part;  // [P][slots][W + 1][C]
    int W, silu, chunk, nchunk, slots;
};

constexpr int U = 4;  // steps requested together

// Kernels for 2, 3, 4 and up to 8 taps (WM); a tap that is not there is left out, not multiplied by 0, which an infinity would show
#define HAS_TAP(j) (WM < 8 || (j) < a.W)

template <class T, int V>
struct alignas(V * sizeof(T)) Vec {
    T v[V];
};
template <class T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&r)[V]) {
    const Vec<T, V> q = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = up(q.v[i]);
}
template <class T, int V>
__device__ __forceinline__ void widen(const Vec<T, V>& q, float (&r)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = up(q.v[i]);
}
template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&r)[V]) {
    Vec<T, V> q;
#pragma unroll
    for (int i = 0; i < V; ++i) q.v[i] = down<T>(r[i]);
    *reinterpret_cast<Vec<T, V>*>(p) = q;
}

// input at position t of row (p, b): the carried window before step 0, zeros before that and without one
template <class T, int V>
__device__ __forceinline__ void input_at(const ConvArgs& a, const T* xp, int p, int b, int c, int t, float (&r)[V]) {
    if (t >= 0) {
        load_vec<T, V>(xp + t * a.x.st, r);
    } else if (a.state != nullptr && t >= -(a.W - 1)) {
        load_vec<T, V>(static_cast<const T*>(a.state) + (((int64_t)p * a.d.B + b) * (a.W - 1) + a.W - 1 + t) * a.d.C + c, r);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = 0.f;
    }
}

// weights by lag, zero beyond the W - 1st; the bias
template <int WM, int V>
__device__ __forceinline__ void load_taps(const ConvArgs& a, int net, int c, float (&w)[WM][V], float (&bias)[V]) {
#pragma unroll
    for (int j = 0; j < WM; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) w[j][i] = j < a.W ? a.weight[((int64_t)net * a.W + a.W - 1 - j) * a.d.C + c + i] : 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = a.bias != nullptr ? a.bias[(int64_t)net * a.d.C + c + i] : 0.f;
}

// the last W - 1 inputs of the row's sequence; those before its last reset as zeros
template <class T, int V, int WM>
__device__ __forceinline__ void window_out(const ConvArgs& a, const T* xp, int p, int b, int c, int len) {
    float r[WM - 1][V];
    int start = -WM;
    for (int t = len - 1; a.reset != nullptr && t >= 0 && t > len - a.W; --t)
        if (a.reset[(int64_t)t * a.d.B + b] != 0) {
            start = t;
            break;
        }
#pragma unroll
    for (int k = 0; k < WM - 1; ++k) {
        const int t = len - (a.W - 1) + k;
        if (k < a.W - 1 && t >= start) input_at<T, V>(a, xp, p, b, c, t, r[k]);
        else
#pragma unroll
            for (int i = 0; i < V; ++i) r[k][i] = 0.f;
    }
    T* o = static_cast<T*>(a.state_out) + ((int64_t)p * a.d.B + b) * (a.W - 1) * a.d.C + c;
#pragma unroll
    for (int k = 0; k < WM - 1; ++k)
        if (k < a.W - 1) store_vec<T, V>(o + (int64_t)k * a.d.C, r[k]);
}

// thread -> (row, channels) within a stretch of steps
template <class T, int V, int WM, bool RESET>
__global__ __launch_bounds__(256) void ssm_conv_fwd_kernel(ConvArgs a) {
    const int CV = a.d.C / V;
    const unsigned nb = gridDim.x / a.nchunk;  // workgroups of a stretch
    const int64_t i = (int64_t)(blockIdx.x % nb) * 256 + threadIdx.x;
    if (i >= (int64_t)a.d.P * a.d.B * CV) return;
    const int row = (int)(i / CV), c = (int)(i % CV) * V, p = row / a.d.B, b = row % a.d.B;
    const int len = seq_len(a.lengths, b, a.d.S), t0 = (int)(blockIdx.x / nb) * a.chunk, t1 = t0 + a.chunk < a.d.S ? t0 + a.chunk : a.d.S;
    const T* xp = seq_at<T>(a.x, p, b) + c;
    float w[WM][V], bias[V], win[WM][V];  // win[j]: the input j steps ago
    load_taps<WM, V>(a, a.d.net[p], c, w, bias);
    int start = -WM;  // the last reset
#pragma unroll
    for (int j = 1; j < WM; ++j) {
        if (j < a.W) input_at<T, V>(a, xp, p, b, c, t0 - j, win[j]);
        else
#pragma unroll
            for (int e = 0; e < V; ++e) win[j][e] = 0.f;
        if (RESET && start < 0 && t0 - j >= 0 && j < a.W && a.reset[(int64_t)(t0 - j) * a.d.B + b] != 0) start = t0 - j;
    }
    T* yp = static_cast<T*>(a.y) + ((int64_t)p * a.d.S * a.d.B + b) * a.d.C + c;
    const int64_t yst = (int64_t)a.d.B * a.d.C;
    for (int t = t0; t < t1; t += U) {
        Vec<T, V> raw[U];
        uint8_t fresh[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {  // U steps requested together; those behind the end are there, but not used
            const int64_t tu = t + u < t1 ? t + u : t1 - 1;
            raw[u] = *reinterpret_cast<const Vec<T, V>*>(xp + tu * a.x.st);
            fresh[u] = RESET ? a.reset[tu * a.d.B + b] : 0;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (t + u >= t1) break;
            float y[V];
            widen<T, V>(raw[u], win[0]);
            if (RESET && fresh[u] != 0) start = t + u;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float s = bias[e];
#pragma unroll
                for (int j = 0; j < WM; ++j) {
                    if (!HAS_TAP(j)) continue;
                    if (!RESET || j == 0) s = fmaf(w[j][e], win[j][e], s);
                    else s = t + u - j >= start ? fmaf(w[j][e], win[j][e], s) : s;
                }
                y[e] = t + u < len ? (a.silu ? s * sigmoid(s) : s) : 0.f;
            }
#pragma unroll
            for (int j = WM - 1; j > 0; --j)
#pragma unroll
                for (int e = 0; e < V; ++e) win[j][e] = win[j - 1][e];
            store_vec<T, V>(yp + (t + u) * yst, y);
        }
    }
    // the stretch with the row's last step leaves the window; updated in place it has to wait for the first stretch's reads (ssm_conv_window_kernel)
    if (a.state_out != nullptr && (a.nchunk == 1 || a.state_out != a.state) && t0 == (len > 0 ? (len - 1) / a.chunk * a.chunk : 0))
        window_out<T, V, WM>(a, xp, p, b, c, len);
}

template <class T, int V, int WM>
__global__ __launch_bounds__(256) void ssm_conv_window_kernel(ConvArgs a) {
    const int CV = a.d.C / V;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.d.P * a.d.B * CV) return;
    const int row = (int)(i / CV), c = (int)(i % CV) * V, p = row / a.d.B, b = row % a.d.B;
    window_out<T, V, WM>(a, seq_at<T>(a.x, p, b) + c, p, b, c, seq_len(a.lengths, b, a.d.S));
}

// Backward.  A workgroup owns a tile of channels and walks (row, stretch) items of one agent, its sums of dweight / dbias in registers.
// Not bound by its bytes yet: 26 steps x 1024 rows x 128 channels f32 take 15 us, 2.7 TB/s out of the last-level cache, where a copy would take 9.
// The ALUs are busy 47 % of the time (62 instructions an element: with 4 taps and stretches of 8 steps a stretch works on 11, the window is moved by
// hand, bounds are decided a step at a time), and two or three waves a SIMD, whose registers hold window, gradients and sums, do not hide the loads.
// Within a stretch [t0, t1) the steps run forwards to t1 + W - 2: what a step gives to an input j steps ago is collected in de[j], and an
// input's gradient is complete when it leaves the window.
template <class T, int V, int WM, bool RESET>
__global__ __launch_bounds__(256) void ssm_conv_bwd_kernel(ConvArgs a, int tile) {
    const int CV = a.d.C / V, tiles = (CV + tile - 1) / tile, per = 256 / tile;
    const int p = blockIdx.x / tiles, cv = (blockIdx.x % tiles) * tile + threadIdx.x % tile, lane_row = threadIdx.x / tile;
    const bool act = cv < CV;
    const int c = (act ? cv : 0) * V;
    float w[WM][V], bias[V], dw[WM][V], db[V];
    load_taps<WM, V>(a, a.d.net[p], c, w, bias);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        db[e] = 0.f;
#pragma unroll
        for (int j = 0; j < WM; ++j) dw[j][e] = 0.f;
    }
    const int64_t items = (int64_t)a.d.B * a.nchunk, yst = (int64_t)a.d.B * a.d.C;
    for (int64_t it = (int64_t)blockIdx.y * per + lane_row; it < items && act; it += (int64_t)a.slots * per) {
        const int b = (int)(it % a.d.B), t0 = (int)(it / a.d.B) * a.chunk, t1 = t0 + a.chunk < a.d.S ? t0 + a.chunk : a.d.S;
        const int len = seq_len(a.lengths, b, a.d.S);
        const T *xp = seq_at<T>(a.x, p, b) + c, *gp = seq_at<T>(a.dy, p, b) + c;
        const int64_t row = (int64_t)p * a.d.B + b;
        T* dxp = static_cast<T*>(a.dx) + ((int64_t)p * a.d.S * a.d.B + b) * a.d.C + c;
        float win[WM][V], de[WM][V];
        int start = -WM;
#pragma unroll
        for (int j = 1; j < WM; ++j) {
            if (j < a.W && t0 - j < len) input_at<T, V>(a, xp, p, b, c, t0 - j, win[j]);
            else
#pragma unroll
                for (int e = 0; e < V; ++e) win[j][e] = 0.f;
            if (RESET && start < 0 && t0 - j >= 0 && t0 - j < len && j < a.W && a.reset[(int64_t)(t0 - j) * a.d.B + b] != 0) start = t0 - j;
        }
#pragma unroll
        for (int j = 0; j < WM; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) de[j][e] = 0.f;
        const int tl = len < t1 + a.W - 1 ? len : t1 + a.W - 1;  // steps from tl on give nothing to this stretch
        for (int tb = t0; tb < t1 + WM - 1; tb += U) {
            Vec<T, V> rx[U], rg[U];
            uint8_t fresh[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t tu = tb + u < a.d.S ? tb + u : a.d.S - 1;
                if (tb < tl) {
                    rx[u] = *reinterpret_cast<const Vec<T, V>*>(xp + tu * a.x.st);
                    rg[u] = *reinterpret_cast<const Vec<T, V>*>(gp + tu * a.dy.st);
                    fresh[u] = RESET ? a.reset[tu * a.d.B + b] : 0;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int t = tb + u;
                if (t >= t1 + WM - 1) break;
                if (t < tl) {
                    float g[V];
                    widen<T, V>(rx[u], win[0]);
                    widen<T, V>(rg[u], g);
                    if (RESET && fresh[u] != 0) start = t;
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        float s = bias[e], xw[WM];
#pragma unroll
                        for (int j = 0; j < WM; ++j) {
                            xw[j] = !RESET || t - j >= start ? win[j][e] : 0.f;
                            if (HAS_TAP(j)) s = fmaf(w[j][e], xw[j], s);
                        }
                        if (a.silu) {
                            const float sg = sigmoid(s);
                            g[e] *= sg * fmaf(s, 1.f - sg, 1.f);
                        }
#pragma unroll
                        for (int j = 0; j < WM; ++j)
                            if (HAS_TAP(j) && (!RESET || t - j >= start)) de[j][e] = fmaf(w[j][e], g[e], de[j][e]);
                        if (t < t1) {
                            db[e] += g[e];
#pragma unroll
                            for (int j = 0; j < WM; ++j) dw[j][e] = fmaf(xw[j], g[e], dw[j][e]);
                        }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) win[0][e] = 0.f;
                }
                const int q = t - (WM - 1);  // this input has met its last step
                if ((q >= t0 || (t0 == 0 && q >= -(a.W - 1))) && q < t1) {
                    const int k = q - (len - (a.W - 1));  // its place in the window after the last step
                    if (a.dstate_out != nullptr && k >= 0 && k < a.W - 1 && q >= start) {
                        float r[V];
                        load_vec<T, V>(static_cast<const T*>(a.dstate_out) + (row * (a.W - 1) + k) * a.d.C + c, r);
#pragma unroll
                        for (int e = 0; e < V; ++e) de[WM - 1][e] += r[e];
                    }
                    if (q >= 0) store_vec<T, V>(dxp + q * yst, de[WM - 1]);
                    else if (a.dstate != nullptr) store_vec<T, V>(static_cast<T*>(a.dstate) + (row * (a.W - 1) + a.W - 1 + q) * a.d.C + c, de[WM - 1]);
                }
#pragma unroll
                for (int j = WM - 1; j > 0; --j)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        win[j][e] = win[j - 1][e];
                        de[j][e] = de[j - 1][e];
                    }
#pragma unroll
                for (int e = 0; e < V; ++e) de[0][e] = 0.f;
            }
        }
    }
    // the workgroup's rows, in order
    __shared__ float red[V][256];
#pragma unroll
    for (int j = 0; j <= WM; ++j) {
        if (j != WM && !HAS_TAP(j)) continue;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) red[e][threadIdx.x] = j < WM ? dw[j < WM ? j : 0][e] : db[e];
        __syncthreads();
        for (int i = threadIdx.x; i < tile * V; i += 256) {
            const int cl = i / V, e = i % V, cw = (blockIdx.x % tiles) * tile + cl;
            if (cw >= CV) continue;
            float s = 0.f;
            for (int k = 0; k < per; ++k) s += red[e][k * tile + cl];
            const int r = j < WM ? a.W - 1 - j : a.W;
            a.part[(((int64_t)p * a.slots + blockIdx.y) * (a.W + 1) + r) * a.d.C + cw * V + e] = s;
        }
    }
}

int conv_validate(const marlhip_ssm_shape* s) {
    if (ssm_validate(s, "ssm_conv") != 0) return -1;
    MARL_REQUIRE(s->state >= 1 && s->state <= SSM_MAX_WIDTH, "ssm_conv: %d taps (1..%d supported)", s->state, SSM_MAX_WIDTH);
    MARL_REQUIRE(s->groups == 1, "ssm_conv: %d groups (one: the convolution is depthwise)", s->groups);
    return 0;
}

// Steps of a stretch.  A stretch reads W - 1 inputs (backward: steps) beyond its own, so longer ones cost less, shorter ones give more threads:
// the longest of 32, 16 and 8 that makes 2048 waves of 8 channels a thread, or 8.  Measured: 65536 steps x 1024 channels bf16 forwards 66 us with
// 32, 69 with 16, 77 with 8; 26 x 1024 rows x 128 channels f32 both ways 30.8 us with 8, 35.3 with 16, 43 with 32.
int conv_chunk(const marlhip_ssm_shape* s) {
    const int64_t work = (int64_t)s->n_agents * s->batch * s->steps * s->channels;
    constexpr int64_t WAVES = 8ll * 64 * 2048;
    return work >= 32 * WAVES ? 32 : (work >= 16 * WAVES ? 16 : 8);
}

ConvArgs conv_args(const marlhip_ssm_shape* s, const marlhip_ssm_conv_args* q) {
    ConvArgs a = {};
    a.d = ssm_dims(s);
    a.W = s->state;
    a.x = ssm_seq(q->x); a.dy = ssm_seq(q->dy);
    a.weight = q->weight; a.bias = q->bias; a.silu = q->silu != 0;
    a.state = q->state; a.dstate_out = q->dstate_out; a.reset = q->reset; a.lengths = q->lengths;
    a.y = q->y; a.state_out = q->state_out; a.dx = q->dx; a.dstate = q->dstate;
    a.chunk = conv_chunk(s);
    a.nchunk = s->steps > 0 ? (s->steps + a.chunk - 1) / a.chunk : 1;
    return a;
}

// channels a thread takes at once where every pointer and stride allows it: 16 bytes of them forwards, 4 of them backwards (its window, its
// gradients and its sums are kept for each: with 8 they take the whole register file)
bool aligned(const SsmSeq& q, int v, int e) {
    return q.data == nullptr || ((uintptr_t)q.data % (v * e) == 0 && q.sp % v == 0 && q.st % v == 0 && q.sb % v == 0);
}
bool aligned(const void* p, int v, int e) { return (uintptr_t)p % (v * e) == 0; }
int conv_vec(const ConvArgs& a, int dtype, bool grad) {
    const int e = dtype == 0 ? 4 : 2, v = grad ? 4 : 16 / e;
    const bool ok = a.d.C % v == 0 && aligned(a.x, v, e) && aligned(a.dy, v, e) && aligned(a.state, v, e) && aligned(a.dstate_out, v, e) && aligned(a.y, v, e) &&
                    aligned(a.state_out, v, e) && aligned(a.dx, v, e) && aligned(a.dstate, v, e);
    return ok ? v : 1;
}

int conv_tile(int CV) {  // threads along the channels of a backward workgroup
    int t = 1;
    while (t < CV && t < 64) t *= 2;
    return t;
}
// workgroups that share the rows and stretches of one agent and channel tile
int conv_slots(const marlhip_ssm_shape* s, int V) {
    const int chunk = conv_chunk(s), CV = (s->channels + V - 1) / V, tile = conv_tile(CV), tiles = (CV + tile - 1) / tile, per = 256 / tile;
    const int64_t items = ((int64_t)s->batch * (s->steps > 0 ? (s->steps + chunk - 1) / chunk : 1) + per - 1) / per;
    const int64_t cap = 2048 / ((int64_t)s->n_agents * tiles) > 1 ? 2048 / ((int64_t)s->n_agents * tiles) : 1;
    return (int)(items < 1 ? 1 : (items < cap ? items : cap));
}
int conv_slots_max(const marlhip_ssm_shape* s) {  // whatever the alignment
    const int a = conv_slots(s, 1), b = conv_slots(s, 4);
    return a > b ? a : b;
}

template <class T, int V, int WM, bool RESET>
int conv_fwd(const ConvArgs& a, hipStream_t st) {
    const int64_t n = (int64_t)a.d.P * a.d.B * (a.d.C / V), blocks = (n + 255) / 256;
    MARL_REQUIRE(blocks * a.nchunk < (1ll << 31), "ssm_conv: too many rows");
    hipLaunchKernelGGL((ssm_conv_fwd_kernel<T, V, WM, RESET>), dim3((unsigned)(blocks * a.nchunk)), dim3(256), 0, st, a);
    MARL_CHECK_LAUNCH("ssm_conv_fwd_kernel");
    if (a.nchunk > 1 && a.state_out != nullptr && a.state_out == a.state) {
        hipLaunchKernelGGL((ssm_conv_window_kernel<T, V, WM>), dim3((unsigned)blocks), dim3(256), 0, st, a);
        MARL_CHECK_LAUNCH("ssm_conv_window_kernel");
    }
    return 0;
}

template <class T, int V, int WM, bool RESET>
int conv_bwd(const ConvArgs& a, hipStream_t st) {
    const int CV = a.d.C / V, tile = conv_tile(CV), tiles = (CV + tile - 1) / tile;
    hipLaunchKernelGGL((ssm_conv_bwd_kernel<T, V, WM, RESET>), dim3((unsigned)(a.d.P * tiles), (unsigned)a.slots), dim3(256), 0, st, a, tile);
    MARL_CHECK_LAUNCH("ssm_conv_bwd_kernel");
    return 0;
}

template <class F>
int conv_dispatch(const marlhip_ssm_shape* s, const ConvArgs& a, int vec, F f) {  // f(type, channels a thread, taps, resets)
    auto by_reset = [&](auto t, auto v, auto wm) { return a.reset != nullptr ? f(t, v, wm, Idx<1>{}) : f(t, v, wm, Idx<0>{}); };
    auto by_width = [&](auto t, auto v) {
        if (a.W == 4) return by_reset(t, v, Idx<4>{});
        if (a.W == 3) return by_reset(t, v, Idx<3>{});
        if (a.W == 2) return by_reset(t, v, Idx<2>{});
        return by_reset(t, v, Idx<8>{});
    };
    auto by_vec = [&](auto t) {
        if (vec == 1) return by_width(t, Idx<1>{});
        if constexpr (sizeof(t) == 2)
            if (vec == 8) return by_width(t, Idx<8>{});
        return by_width(t, Idx<4>{});
    };
    if (s->dtype == 0) return by_vec(float{});
    if (s->dtype == 1) return by_vec(__bf16{});
    return by_vec(_Float16{});
}

int conv_fwd_any(const marlhip_ssm_shape* s, const ConvArgs& a, hipStream_t st) {
    return conv_dispatch(s, a, conv_vec(a, s->dtype, false), [&](auto t, auto v, auto wm, auto re) {
        constexpr int V = decltype(v)::v;
        if constexpr (V == 4 && sizeof(t) == 2) return -1;  // 16-bit types take 8 forwards
        else return conv_fwd<decltype(t), V, decltype(wm)::v, decltype(re)::v != 0>(a, st);
    });
}
int conv_bwd_any(const marlhip_ssm_shape* s, const ConvArgs& a, hipStream_t st) {
    return conv_dispatch(s, a, conv_vec(a, s->dtype, true), [&](auto t, auto v, auto wm, auto re) {
        constexpr int V = decltype(v)::v;
        if constexpr (V == 8) return -1;
        else return conv_bwd<decltype(t), V, decltype(wm)::v, decltype(re)::v != 0>(a, st);
    });
}

}  // namespace

extern "C" int marlhip_ssm_conv(const marlhip_ssm_shape* s, const marlhip_ssm_conv_args* q, void* stream) {
    if (conv_validate(s) != 0) return -1;
    MARL_REQUIRE(q != nullptr && q->weight != nullptr, "ssm_conv: NULL argument");
    MARL_REQUIRE(s->steps == 0 || s->batch == 0 || (q->x.data && q->y), "ssm_conv: NULL pointer");
    if (s->batch == 0) return 0;
    ConvArgs a = conv_args(s, q);
    if (a.W == 1) a.state_out = nullptr;  // a window of no inputs
    if (s->steps == 0 && a.state_out == nullptr) return 0;
    return conv_fwd_any(s, a, (hipStream_t)stream);
}

extern "C" int64_t marlhip_ssm_conv_grad_workspace_bytes(const marlhip_ssm_shape* s) {
    if (conv_validate(s) != 0) return -1;
    return (int64_t)s->n_agents * conv_slots_max(s) * (s->state + 1) * s->channels * 4;
}

extern "C" int marlhip_ssm_conv_grad(const marlhip_ssm_shape* s, const marlhip_ssm_conv_args* q, void* workspace, int64_t workspace_bytes, void* stream) {
    if (conv_validate(s) != 0) return -1;
    MARL_REQUIRE(q != nullptr && q->weight != nullptr && q->dweight != nullptr, "ssm_conv_grad: NULL argument");
    MARL_REQUIRE(s->steps == 0 || s->batch == 0 || (q->x.data && q->dy.data && q->dx), "ssm_conv_grad: NULL pointer");
    const int64_t need = marlhip_ssm_conv_grad_workspace_bytes(s);
    MARL_REQUIRE(workspace != nullptr && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need, "ssm_conv_grad: aligned workspace of %lld bytes needed, %lld given", (long long)need,
                 (long long)workspace_bytes);
    ConvArgs a = conv_args(s, q);
    if (a.W == 1) a.dstate_out = nullptr, a.dstate = nullptr;
    a.slots = conv_slots(s, conv_vec(a, s->dtype, true));
    a.part = static_cast<float*>(workspace);
    if (conv_bwd_any(s, a, (hipStream_t)stream) != 0) return -1;
    const int64_t cols = (int64_t)(a.W + 1) * a.d.C;
    hipLaunchKernelGGL(ssm_weights_sum_kernel, dim3((unsigned)((cols + 63) / 64), a.d.M), dim3(1024), 0, (hipStream_t)stream, a.d, a.slots, a.W, 1, a.part,
                       q->dweight, q->dbias, (float*)nullptr);
    MARL_CHECK_LAUNCH("ssm_weights_sum_kernel");
    return 0;
}
