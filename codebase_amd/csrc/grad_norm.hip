// Global 2-norm over many tensors and the clip: marlhip_grad_norm, marlhip_clip_grad_norm.
//
// The tensors' pointers travel in the kernel's own arguments, up to NORM_ENTRIES a launch: no table has to be copied to the device, and a
// captured graph holds them.  A first pass leaves one 64-bit sum of squares a workgroup, a second one adds them up in every workgroup (the
// same order everywhere) and scales.  Bound by HBM: the gradients are read once or twice and written once.
#include <algorithm>
#include <vector>

#include "common.h"

using namespace marl;

namespace {

constexpr int NORM_ENTRIES = 160;
constexpr int64_t NORM_PIECE = 1ll << 30;  // elements of an entry (larger tensors take several)

struct NormEntry {
    const void* p;
    void* o;
    uint32_t n;
    uint32_t first;  // first workgroup of the launch that works on it, type in the top two bits
};
struct NormTable {
    NormEntry e[NORM_ENTRIES];
    int count;
    uint32_t chunk;    // elements a workgroup takes
    int part0, parts;  // first partial sum of the launch; all of the call's
    float max_norm;
};
static_assert(sizeof(NormTable) <= 4000, "kernel arguments");

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
    __syncthreads();
    return v;
}

template <class T, int V>
struct alignas(V * sizeof(T)) NVec {
    T v[V];
};

// the entry of this workgroup, and its elements [i0, i1)
__device__ __forceinline__ const NormEntry& find_entry(const NormTable& t, uint32_t blk, uint32_t& i0, uint32_t& i1) {
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

template <class T>
__device__ __forceinline__ double square_sum(const T* p, uint32_t i0, uint32_t i1) {
    constexpr int V = 16 / sizeof(T);
    double s = 0.0;
    uint32_t i = i0;
    if ((uintptr_t)p % 16 == 0) {
        const uint32_t nv = (i1 - i0) / V;
        for (uint32_t k = threadIdx.x; k < nv; k += 256) {
            const NVec<T, V> q = *reinterpret_cast<const NVec<T, V>*>(p + i0 + k * V);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const double g = static_cast<float>(q.v[j]);
                s = fma(g, g, s);
            }
        }
        i = i0 + nv * V;
    }
    for (uint32_t k = i + threadIdx.x; k < i1; k += 256) {
        const double g = static_cast<float>(p[k]);
        s = fma(g, g, s);
    }
    return s;
}

template <class T>
__device__ __forceinline__ void scale_all(const T* p, T* o, float coef, uint32_t i0, uint32_t i1) {
    constexpr int V = 16 / sizeof(T);
    uint32_t i = i0;
    if (((uintptr_t)p | (uintptr_t)o) % 16 == 0) {
        const uint32_t nv = (i1 - i0) / V;
        for (uint32_t k = threadIdx.x; k < nv; k += 256) {
            NVec<T, V> q = *reinterpret_cast<const NVec<T, V>*>(p + i0 + k * V);
#pragma unroll
            for (int j = 0; j < V; ++j) q.v[j] = static_cast<T>(static_cast<float>(q.v[j]) * coef);
            *reinterpret_cast<NVec<T, V>*>(o + i0 + k * V) = q;
        }
        i = i0 + nv * V;
    }
    for (uint32_t k = i + threadIdx.x; k < i1; k += 256) o[k] = static_cast<T>(static_cast<float>(p[k]) * coef);
}

__global__ __launch_bounds__(256) void grad_square_kernel(NormTable t, double* __restrict__ part) {
    __shared__ double red[4];
    uint32_t i0, i1;
    const NormEntry& e = find_entry(t, blockIdx.x, i0, i1);
    const int dt = e.first >> 30;
    const double s = dt == 0 ? square_sum(static_cast<const float*>(e.p), i0, i1)
                             : (dt == 1 ? square_sum(static_cast<const __bf16*>(e.p), i0, i1) : square_sum(static_cast<const _Float16*>(e.p), i0, i1));
    const double sum = block_sum(s, red);
    if (threadIdx.x == 0) part[t.part0 + blockIdx.x] = sum;
}

__device__ __forceinline__ float total_norm(const double* part, int parts, double* red) {
    double s = 0.0;
    for (int k = threadIdx.x; k < parts; k += 256) s += part[k];
    return (float)sqrt(block_sum(s, red));
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const double* __restrict__ part, int parts, float* __restrict__ norm_out) {
    __shared__ double red[4];
    const float norm = total_norm(part, parts, red);
    if (threadIdx.x == 0) norm_out[0] = norm;
}

__global__ __launch_bounds__(256) void grad_clip_kernel(NormTable t, const double* __restrict__ part, float* __restrict__ norm_out) {
    __shared__ double red[4];
    const float norm = total_norm(part, t.parts, red);
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = norm;
    const float ratio = t.max_norm / (norm + 1e-6f), coef = ratio > 1.f ? 1.f : ratio;  // NaN stays NaN
    uint32_t i0, i1;
    const NormEntry& e = find_entry(t, blockIdx.x, i0, i1);
    const int dt = e.first >> 30;
    if (dt == 0) scale_all(static_cast<const float*>(e.p), static_cast<float*>(e.o), coef, i0, i1);
    else if (dt == 1) scale_all(static_cast<const __bf16*>(e.p), static_cast<__bf16*>(e.o), coef, i0, i1);
    else scale_all(static_cast<const _Float16*>(e.p), static_cast<_Float16*>(e.o), coef, i0, i1);
}

struct NormPlan {
    int64_t chunk, parts;
};

int norm_plan(const marlhip_tensor* t, int32_t count, NormPlan& plan, bool clip) {
    MARL_REQUIRE(count >= 0 && (count == 0 || t != nullptr), "grad_norm: %d tensors", count);
    int64_t total = 0;
    for (int i = 0; i < count; ++i) {
        MARL_REQUIRE(t[i].n >= 0 && t[i].n < (1ll << 40) && (t[i].n == 0 || t[i].data != nullptr), "grad_norm: tensor %d", i);
        MARL_REQUIRE(t[i].dtype >= 0 && t[i].dtype <= 2, "grad_norm: tensor %d: dtype %d (0 f32, 1 bf16, 2 f16)", i, t[i].dtype);
        const int e = t[i].dtype == 0 ? 4 : 2;
        MARL_REQUIRE((uintptr_t)t[i].data % e == 0 && (!clip || (uintptr_t)t[i].out % e == 0), "grad_norm: tensor %d is not aligned to its type", i);
        total += t[i].n;
    }
    // about 2048 workgroups: enough to fill the chip, few enough sums for every one of them to add up
    const int64_t c = (total / 2048 + 4095) / 4096 * 4096;
    plan.chunk = c < 4096 ? 4096 : c;
    plan.parts = 0;
    for (int i = 0; i < count; ++i)
        for (int64_t o = 0; o < t[i].n; o += NORM_PIECE) {
            const int64_t n = t[i].n - o < NORM_PIECE ? t[i].n - o : NORM_PIECE;
            plan.parts += (n + plan.chunk - 1) / plan.chunk;
        }
    MARL_REQUIRE(plan.parts < (1 << 30), "grad_norm: too many tensors");
    return 0;
}

// launch(table, workgroups) for every NORM_ENTRIES pieces
template <class F>
int norm_tables(const marlhip_tensor* t, int32_t count, const NormPlan& plan, float max_norm, F launch) {
    NormTable tab;
    tab.count = 0;
    tab.chunk = (uint32_t)plan.chunk;
    tab.part0 = 0;
    tab.parts = (int)plan.parts;
    tab.max_norm = max_norm;
    uint32_t blocks = 0;
    auto flush = [&]() {
        if (tab.count == 0) return 0;
        const int rc = launch(tab, blocks);
        tab.part0 += (int)blocks;
        tab.count = 0;
        blocks = 0;
        return rc;
    };
    for (int i = 0; i < count; ++i) {
        const int es = t[i].dtype == 0 ? 4 : 2;
        for (int64_t o = 0; o < t[i].n; o += NORM_PIECE) {
            if (tab.count == NORM_ENTRIES && flush() != 0) return -2;
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

int square_pass(const marlhip_tensor* t, int32_t count, const NormPlan& plan, double* part, hipStream_t st) {
    return norm_tables(t, count, plan, 0.f, [&](const NormTable& tab, uint32_t blocks) {
        hipLaunchKernelGGL(grad_square_kernel, dim3(blocks), dim3(256), 0, st, tab, part);
        MARL_CHECK_LAUNCH("grad_square_kernel");
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
    if (square_pass(tensors, count, plan, part, st) != 0) return -2;
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
    if (square_pass(tensors, count, plan, part, st) != 0) return -2;
    return norm_tables(tensors, count, plan, max_norm, [&](const NormTable& tab, uint32_t blocks) {
        hipLaunchKernelGGL(grad_clip_kernel, dim3(blocks), dim3(256), 0, st, tab, part, norm_out);
        MARL_CHECK_LAUNCH("grad_clip_kernel");
        return 0;
    });
}
