// Global 2-norm over many tensors and the clip: marlhip_grad_norm, marlhip_clip_grad_norm.
//
// The tensors' pointers travel in the kernel's own arguments, up to 160 a launch: no table has to be copied to the device, and a captured
// graph holds them.  A first pass leaves one 64-bit sum of squares a workgroup, a second one adds them up in every workgroup (the same order
// everywhere) and scales, in the opposite direction: what the first pass read last is still in the caches.  Bound by HBM: the gradients are
// read twice, less what the caches keep, and written once.  320 tensors, 112 M elements of bf16 and f32: 60 us + 130 us, 5.3 TB/s of what the two
// passes touch; 12 tensors of two small networks: 3.6 us + 3.9 us, launch latency.
#include <algorithm>
#include <vector>

#include "common.h"

using namespace marl;

namespace {

constexpr int64_t NORM_PIECE = 1ll << 30;  // elements of an entry (larger tensors take several)
constexpr int64_t NORM_WGS = 4096;         // workgroups of a pass, about
constexpr int FEW = 16, MANY = 160;        // entries of a launch (the small table saves the host's copy of the large one)

struct NormEntry {
    const void* p;
    void* o;
    uint32_t n;
    uint32_t first;  // first workgroup of the launch that works on it, type in the top two bits
};
template <int E>
struct NormTable {
    NormEntry e[E];
    int count;
    uint32_t chunk;    // elements a workgroup takes
    int part0, parts;  // first partial sum of the launch; all of the call's
    float max_norm;
    int stream;  // stores past the caches
};
static_assert(sizeof(NormTable<MANY>) <= 4000, "kernel arguments");

template <int W>
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < W; ++w) v += red[w];
    __syncthreads();
    return v;
}

__device__ __forceinline__ float clip_coef(float max_norm, float norm) {
    const float ratio = max_norm / (norm + 1e-6f);
    return ratio > 1.f ? 1.f : ratio;  // NaN stays NaN
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <class T>
struct Pack {  // 16 bytes of elements
    static constexpr int V = 16 / sizeof(T);
    u32x4 w;
    __device__ __forceinline__ T get(int j) const {
        const uint32_t x = w[sizeof(T) == 4 ? j : j / 2];
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, x);
        else return __builtin_bit_cast(T, (unsigned short)(x >> (j % 2 * 16)));
    }
    __device__ __forceinline__ void scale(float coef) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                w[i] = __builtin_bit_cast(uint32_t, get(i) * coef);
            } else {
                const T lo = static_cast<T>(static_cast<float>(get(2 * i)) * coef), hi = static_cast<T>(static_cast<float>(get(2 * i + 1)) * coef);
                w[i] = (uint32_t)__builtin_bit_cast(unsigned short, lo) | ((uint32_t)__builtin_bit_cast(unsigned short, hi) << 16);
            }
        }
    }
    __device__ __forceinline__ double squares() const {
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const double g = static_cast<float>(get(j));
            s = fma(g, g, s);
        }
        return s;
    }
};

// the entry of this workgroup, and its elements [i0, i1)
template <int E>
__device__ __forceinline__ const NormEntry& find_entry(const NormTable<E>& t, uint32_t blk, uint32_t& i0, uint32_t& i1) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {  // the last entry whose first workgroup is not behind this one
        const int mid = (lo + hi + 1) >> 1;
        if ((t.e[mid].first & 0x3fffffffu) <= blk) lo = mid;
        else hi = mid - 1;
    }
    const NormEntry& e = t.e[lo];
    i0 = (blk - (e.first & 0x3fffffffu)) * t.chunk;
    i1 = i0 + t.chunk < e.n ? i0 + t.chunk : e.n;
    return e;
}

constexpr int U = 4;  // 16-byte requests of a thread in flight

template <class T>
__device__ __forceinline__ double square_sum(const T* p, uint32_t i0, uint32_t i1) {
    constexpr int V = Pack<T>::V;
    double s[U] = {};
    uint32_t i = i0;
    if ((uintptr_t)p % 16 == 0) {
        const Pack<T>* v = reinterpret_cast<const Pack<T>*>(p + i0);
        const uint32_t nv = (i1 - i0) / V;
        uint32_t k = threadIdx.x;
        for (; k + (U - 1) * 256 < nv; k += U * 256) {
            Pack<T> q[U];
#pragma unroll
            for (int u = 0; u < U; ++u) q[u] = v[k + u * 256];
#pragma unroll
            for (int u = 0; u < U; ++u) s[u] += q[u].squares();
        }
        for (; k < nv; k += 256) s[0] += v[k].squares();
        i = i0 + nv * V;
    }
    for (uint32_t k = i + threadIdx.x; k < i1; k += 256) {
        const double g = static_cast<float>(p[k]);
        s[0] = fma(g, g, s[0]);
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

template <class T, bool STREAM>
__device__ __forceinline__ void scale_all(const T* p, T* o, float coef, uint32_t i0, uint32_t i1) {
    constexpr int V = Pack<T>::V;
    uint32_t i = i0;
    if (((uintptr_t)p | (uintptr_t)o) % 16 == 0) {
        const Pack<T>* v = reinterpret_cast<const Pack<T>*>(p + i0);
        u32x4* w = reinterpret_cast<u32x4*>(o + i0);
        const uint32_t nv = (i1 - i0) / V;
        uint32_t k = threadIdx.x;
        for (; k + (U - 1) * 256 < nv; k += U * 256) {
            Pack<T> q[U];
#pragma unroll
            for (int u = 0; u < U; ++u) q[u] = v[k + u * 256];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                q[u].scale(coef);
                if (STREAM) __builtin_nontemporal_store(q[u].w, w + k + u * 256);
                else w[k + u * 256] = q[u].w;
            }
        }
        for (; k < nv; k += 256) {
            Pack<T> q = v[k];
            q.scale(coef);
            w[k] = q.w;
        }
        i = i0 + nv * V;
    }
    for (uint32_t k = i + threadIdx.x; k < i1; k += 256) o[k] = static_cast<T>(static_cast<float>(p[k]) * coef);
}

template <int E>
__global__ __launch_bounds__(256) void grad_square_kernel(NormTable<E> t, double* __restrict__ part) {
    __shared__ double red[4];
    uint32_t i0, i1;
    const NormEntry& e = find_entry(t, blockIdx.x, i0, i1);
    const int dt = e.first >> 30;
    const double s = dt == 0 ? square_sum(static_cast<const float*>(e.p), i0, i1)
                             : (dt == 1 ? square_sum(static_cast<const __bf16*>(e.p), i0, i1) : square_sum(static_cast<const _Float16*>(e.p), i0, i1));
    const double sum = block_sum<4>(s, red);
    if (threadIdx.x == 0) part[t.part0 + blockIdx.x] = sum;
}

__device__ __forceinline__ float total_norm(const double* part, int parts, double* red) {
    double s = 0.0;
#pragma unroll 4
    for (int k = threadIdx.x; k < parts; k += 256) s += part[k];
    return (float)sqrt(block_sum<4>(s, red));
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const double* __restrict__ part, int parts, float* __restrict__ norm_out) {
    __shared__ double red[4];
    const float norm = total_norm(part, parts, red);
    if (threadIdx.x == 0) norm_out[0] = norm;
}

template <bool STREAM>
__device__ __forceinline__ void scale_entry(const NormEntry& e, float coef, uint32_t i0, uint32_t i1) {
    const int dt = e.first >> 30;
    if (dt == 0) scale_all<float, STREAM>(static_cast<const float*>(e.p), static_cast<float*>(e.o), coef, i0, i1);
    else if (dt == 1) scale_all<__bf16, STREAM>(static_cast<const __bf16*>(e.p), static_cast<__bf16*>(e.o), coef, i0, i1);
    else scale_all<_Float16, STREAM>(static_cast<const _Float16*>(e.p), static_cast<_Float16*>(e.o), coef, i0, i1);
}

template <int E>
__global__ __launch_bounds__(256) void grad_clip_kernel(NormTable<E> t, const double* __restrict__ part, float* __restrict__ norm_out) {
    __shared__ double red[4];
    const float norm = total_norm(part, t.parts, red);
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = norm;
    const float coef = clip_coef(t.max_norm, norm);
    uint32_t i0, i1;
    const NormEntry& e = find_entry(t, blockIdx.x, i0, i1);
    if (t.stream) scale_entry<true>(e, coef, i0, i1);
    else scale_entry<false>(e, coef, i0, i1);
}

struct NormPlan {
    int64_t chunk, parts;
    bool stream;  // more bytes than half of the last-level cache: what is written does not push out what is still to be read
};

int norm_plan(const marlhip_tensor* t, int32_t count, NormPlan& plan, bool clip) {
    MARL_REQUIRE(count >= 0 && (count == 0 || t != nullptr), "grad_norm: %d tensors", count);
    int64_t total = 0, bytes = 0;
    for (int i = 0; i < count; ++i) {
        MARL_REQUIRE(t[i].n >= 0 && t[i].n < (1ll << 40) && (t[i].n == 0 || t[i].data != nullptr), "grad_norm: tensor %d", i);
        MARL_REQUIRE(t[i].dtype >= 0 && t[i].dtype <= 2, "grad_norm: tensor %d: dtype %d (0 f32, 1 bf16, 2 f16)", i, t[i].dtype);
        const int e = t[i].dtype == 0 ? 4 : 2;
        MARL_REQUIRE((uintptr_t)t[i].data % e == 0 && (!clip || (uintptr_t)t[i].out % e == 0), "grad_norm: tensor %d is not aligned to its type", i);
        total += t[i].n;
        bytes += t[i].n * e;
    }
    // about 4096 workgroups: enough to fill the chip evenly (2048 took 15 % longer on 112 M elements), few enough sums for every one to add up
    const int64_t c = (total / NORM_WGS + 4095) / 4096 * 4096;
    plan.chunk = c < 4096 ? 4096 : c;
    plan.stream = bytes > (1ll << 27);
    plan.parts = 0;
    for (int i = 0; i < count; ++i)
        for (int64_t o = 0; o < t[i].n; o += NORM_PIECE) {
            const int64_t n = t[i].n - o < NORM_PIECE ? t[i].n - o : NORM_PIECE;
            plan.parts += (n + plan.chunk - 1) / plan.chunk;
        }
    MARL_REQUIRE(plan.parts < (1 << 30), "grad_norm: too many tensors");
    return 0;
}

// launch(table, workgroups) for every E pieces, from the last tensor to the first if reverse
template <int E, class F>
int norm_tables(const marlhip_tensor* t, int32_t count, const NormPlan& plan, float max_norm, bool reverse, F launch) {
    NormTable<E> tab;
    tab.count = 0;
    tab.chunk = (uint32_t)plan.chunk;
    tab.part0 = 0;
    tab.parts = (int)plan.parts;
    tab.max_norm = max_norm;
    tab.stream = plan.stream;
    uint32_t blocks = 0;
    auto flush = [&]() {
        if (tab.count == 0) return 0;
        const int rc = launch(tab, blocks);
        tab.part0 += (int)blocks;
        tab.count = 0;
        blocks = 0;
        return rc;
    };
    for (int j = 0; j < count; ++j) {
        const int i = reverse ? count - 1 - j : j, es = t[i].dtype == 0 ? 4 : 2;
        for (int64_t o = 0; o < t[i].n; o += NORM_PIECE) {
            if (tab.count == E && flush() != 0) return -2;
            const int64_t n = t[i].n - o < NORM_PIECE ? t[i].n - o : NORM_PIECE;
            NormEntry& e = tab.e[tab.count++];
            e.p = static_cast<const char*>(t[i].data) + o * es;
            e.o = static_cast<char*>(t[i].out != nullptr ? t[i].out : const_cast<void*>(t[i].data)) + o * es;
            e.n = (uint32_t)n;
            e.first = blocks | ((uint32_t)t[i].dtype << 30);
            blocks += (uint32_t)((n + plan.chunk - 1) / plan.chunk);
        }
    }
    return flush();
}

template <int E>
int square_pass(const marlhip_tensor* t, int32_t count, const NormPlan& plan, double* part, hipStream_t st) {
    return norm_tables<E>(t, count, plan, 0.f, false, [&](const NormTable<E>& tab, uint32_t blocks) {
        hipLaunchKernelGGL(grad_square_kernel<E>, dim3(blocks), dim3(256), 0, st, tab, part);
        MARL_CHECK_LAUNCH("grad_square_kernel");
        return 0;
    });
}

template <int E>
int clip_passes(const marlhip_tensor* t, int32_t count, const NormPlan& plan, float max_norm, double* part, float* norm_out, hipStream_t st) {
    if (square_pass<E>(t, count, plan, part, st) != 0) return -2;
    return norm_tables<E>(t, count, plan, max_norm, true, [&](const NormTable<E>& tab, uint32_t blocks) {
        hipLaunchKernelGGL(grad_clip_kernel<E>, dim3(blocks), dim3(256), 0, st, tab, part, norm_out);
        MARL_CHECK_LAUNCH("grad_clip_kernel");
        return 0;
    });
}

int norm_check(const marlhip_tensor* t, int32_t count, NormPlan& plan, void* workspace, int64_t workspace_bytes, bool clip) {
    if (norm_plan(t, count, plan, clip) != 0) return -1;
    MARL_REQUIRE(plan.parts == 0 || (workspace != nullptr && (uintptr_t)workspace % 8 == 0 && workspace_bytes >= plan.parts * 8),
                 "grad_norm: aligned workspace of %lld bytes needed, %lld given", (long long)(plan.parts * 8), (long long)workspace_bytes);
    return 0;
}

}  // namespace

extern "C" int marlhip_tensors_apart(const marlhip_tensor* t, int32_t count) {
    MARL_REQUIRE(count >= 0 && (count == 0 || t != nullptr), "tensors_apart: %d tensors", count);
    struct Span {
        uintptr_t lo, hi;
        int i;
    };
    // caught here: no exception may leave a C entry point
    try {
        std::vector<Span> v;
        v.reserve(2 * (size_t)count);
        for (int i = 0; i < count; ++i) {
            const uintptr_t n = (uintptr_t)t[i].n * (t[i].dtype == 0 ? 4 : 2), p = (uintptr_t)t[i].data, o = t[i].out != nullptr ? (uintptr_t)t[i].out : p;
            if (n == 0) continue;
            v.push_back({p, p + n, i});
            if (o != p) v.push_back({o, o + n, i});
        }
        std::sort(v.begin(), v.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
        for (size_t k = 1; k < v.size(); ++k)
            MARL_REQUIRE(v[k - 1].hi <= v[k].lo, "tensors %d and %d overlap", v[k - 1].i, v[k].i);
    } catch (...) {
        set_error("tensors_apart: out of memory");
        return -1;
    }
    return 0;
}

extern "C" int64_t marlhip_grad_norm_workspace_bytes(const marlhip_tensor* tensors, int32_t count) {
    NormPlan plan;
    if (norm_plan(tensors, count, plan, false) != 0) return -1;
    return plan.parts * 8;
}

extern "C" int marlhip_grad_norm(const marlhip_tensor* tensors, int32_t count, float* norm_out, void* workspace, int64_t workspace_bytes, void* stream) {
    NormPlan plan;
    if (norm_check(tensors, count, plan, workspace, workspace_bytes, false) != 0) return -1;
    MARL_REQUIRE(norm_out != nullptr, "grad_norm: NULL pointer");
    double* part = static_cast<double*>(workspace);
    hipStream_t st = (hipStream_t)stream;
    if ((count <= FEW ? square_pass<FEW>(tensors, count, plan, part, st) : square_pass<MANY>(tensors, count, plan, part, st)) != 0) return -2;
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, st, part, (int)plan.parts, norm_out);
    MARL_CHECK_LAUNCH("grad_norm_kernel");
    return 0;
}

extern "C" int marlhip_clip_grad_norm(const marlhip_tensor* tensors, int32_t count, float max_norm, float* norm_out, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
    NormPlan plan;
    if (norm_check(tensors, count, plan, workspace, workspace_bytes, true) != 0) return -1;
    MARL_REQUIRE(max_norm >= 0.f, "clip_grad_norm: max_norm %g", (double)max_norm);
    MARL_REQUIRE(norm_out != nullptr, "clip_grad_norm: NULL pointer");
    double* part = static_cast<double*>(workspace);
    hipStream_t st = (hipStream_t)stream;
    if (plan.parts == 0) {
        hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, st, part, 0, norm_out);
        MARL_CHECK_LAUNCH("grad_norm_kernel");
        return 0;
    }
    return count <= FEW ? clip_passes<FEW>(tensors, count, plan, max_norm, part, norm_out, st)
                        : clip_passes<MANY>(tensors, count, plan, max_norm, part, norm_out, st);
}
