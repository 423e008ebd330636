// The global 2-norm of a list of gradients, and the gradients scaled to at most a given norm:
//
//   norm = sqrt(sum over all tensors of sum g^2),   out = g * min(1, max_norm / (norm + 1e-6))
//
// Memory-bound twice over: the norm has to be known before the first value is scaled, so gradients larger than the caches are read
// twice.  The table of tensors travels in the kernels' arguments (nothing is uploaded, a captured graph keeps it); a workgroup takes
// one chunk of one tensor and finds it by bisection.  grad_square_sums writes one 64-bit sum a workgroup, grad_scale adds all of
// them up in a fixed order at its start: two launches for kTensors tensors, no atomics, and a result repeats bit for bit.
// Squares are formed and added in 64 bits, so no gradient's square overflows or vanishes.
#include <algorithm>
#include <vector>

#include "common.h"

namespace msnet {
namespace clip {

constexpr int kThreads = 256;
constexpr int kTensors = 112;          // of one launch: the table keeps below the 4 KB of kernel arguments
constexpr long kChunk = 8192;          // values of a workgroup at least
constexpr long kBlocks = 2048;         // workgroups of a call beyond one a tensor, at most

struct Table {
    const void* in[kTensors];
    void* out[kTensors];
    long n[kTensors];
    unsigned first[kTensors + 1];      // first workgroup of each tensor
    unsigned char types[kTensors];     // input's type + 4 * output's
    int count;
};
static_assert(sizeof(Table) + 64 <= 4096, "kernel arguments");

template <class T, int V> struct Pack { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };      // any view's alignment

__device__ __forceinline__ int tensor_of(const Table& t, unsigned block) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= block) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ double block_sum(double s, double* tab, int tid) {
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((tid & 63) == 0) tab[tid >> 6] = s;
    __syncthreads();
    return (tab[0] + tab[1]) + (tab[2] + tab[3]);
}

template <class T>
__device__ __forceinline__ double square_sum(const T* p, long n, int tid) {
    constexpr int V = 16 / sizeof(T);
    typedef typename Pack<T, V>::type Vec;
    double s[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = 0.;
    const long nv = n / V;
    const Vec* v = reinterpret_cast<const Vec*>(p);
    long i = tid;
    auto add = [&](const Vec& a) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double d = (double)(float)a[e];
            s[e] = fma(d, d, s[e]);
        }
    };
    for (; i + 3 * kThreads < nv; i += 4 * kThreads) {
        const Vec a = v[i], b = v[i + kThreads], c = v[i + 2 * kThreads], d = v[i + 3 * kThreads];
        add(a); add(b); add(c); add(d);
    }
    for (; i < nv; i += kThreads) add(v[i]);
    double r = s[0];
#pragma unroll
    for (int e = 1; e < V; ++e) r += s[e];
    const long at = nv * V + tid;
    if (at < n) { const double d = (double)(float)p[at]; r = fma(d, d, r); }
    return r;
}

__global__ __launch_bounds__(kThreads) void grad_square_sums(Table t, long chunk, double* __restrict__ sums) {
    __shared__ double tab[4];
    const int tid = threadIdx.x, k = tensor_of(t, blockIdx.x);
    const long at = (long)(blockIdx.x - t.first[k]) * chunk, n = min(chunk, t.n[k] - at);
    double s;
    switch (t.types[k] & 3) {
        case 0: s = square_sum(static_cast<const float*>(t.in[k]) + at, n, tid); break;
        case 1: s = square_sum(static_cast<const _Float16*>(t.in[k]) + at, n, tid); break;
        default: s = square_sum(static_cast<const __bf16*>(t.in[k]) + at, n, tid);
    }
    s = block_sum(s, tab, tid);
    if (tid == 0) sums[blockIdx.x] = s;
}

template <class T, class O>
__device__ __forceinline__ void scale(const T* p, O* o, long n, float f, int tid) {
    constexpr int V = 16 / sizeof(T);
    typedef typename Pack<T, V>::type Vec;
    typedef typename Pack<O, V>::type Out;
    const long nv = n / V;
    const Vec* v = reinterpret_cast<const Vec*>(p);
    Out* w = reinterpret_cast<Out*>(o);
    auto put = [&](long i, const Vec& a) {
        Out r;
#pragma unroll
        for (int e = 0; e < V; ++e) r[e] = (O)((float)a[e] * f);
        w[i] = r;
    };
    long i = tid;
    for (; i + 3 * kThreads < nv; i += 4 * kThreads) {
        const Vec a = v[i], b = v[i + kThreads], c = v[i + 2 * kThreads], d = v[i + 3 * kThreads];
        put(i, a); put(i + kThreads, b); put(i + 2 * kThreads, c); put(i + 3 * kThreads, d);
    }
    for (; i < nv; i += kThreads) put(i, v[i]);
    const long at = nv * V + tid;
    if (at < n) o[at] = (O)((float)p[at] * f);
}

// norm: where the first launch's first workgroup leaves it, or null.  scaling: whether there is anything to scale.
__global__ __launch_bounds__(kThreads) void grad_scale(Table t, long chunk, const double* __restrict__ sums, unsigned nsums, double max_norm,
                                                       float* norm, int scaling) {
    __shared__ double tab[4];
    const int tid = threadIdx.x;
    double s = 0.;
#pragma unroll 4
    for (unsigned i = tid; i < nsums; i += kThreads) s += sums[i];
    const double total = sqrt(block_sum(s, tab, tid));
    if (norm && blockIdx.x == 0 && tid == 0) *norm = (float)total;
    if (!scaling) return;
    const double r = max_norm / (total + 1e-6);
    const float f = r > 1. ? 1.f : (float)r;               // (a NaN stays one)
    const int k = tensor_of(t, blockIdx.x);
    if (f == 1.f && t.in[k] == t.out[k]) return;           // short enough already, in place
    const long at = (long)(blockIdx.x - t.first[k]) * chunk, n = min(chunk, t.n[k] - at);
    const void* p = t.in[k];
    void* o = t.out[k];
    switch (t.types[k]) {
        case 0: scale(static_cast<const float*>(p) + at, static_cast<float*>(o) + at, n, f, tid); break;
        case 1: scale(static_cast<const _Float16*>(p) + at, static_cast<float*>(o) + at, n, f, tid); break;
        case 2: scale(static_cast<const __bf16*>(p) + at, static_cast<float*>(o) + at, n, f, tid); break;
        case 5: scale(static_cast<const _Float16*>(p) + at, static_cast<_Float16*>(o) + at, n, f, tid); break;
        default: scale(static_cast<const __bf16*>(p) + at, static_cast<__bf16*>(o) + at, n, f, tid);
    }
}

// The workgroups of a call: chunk values each, more where the whole is large.
struct Cut { long chunk; unsigned long blocks; };

static Cut cut(const int64_t* n, int count) {
    double total = 0;
    for (int i = 0; i < count; ++i) total += (double)n[i];
    Cut c = {kChunk, 0};
    if (total > (double)kChunk * kBlocks) c.chunk = ((long)(total / kBlocks) / kChunk + 1) * kChunk;
    for (int i = 0; i < count; ++i) c.blocks += (unsigned long)((n[i] + c.chunk - 1) / c.chunk);
    return c;
}

// Whether a value would be written that another tensor of the call reads or writes too: workgroups run in any order, so the result
// would depend on it.  (A tensor scaled in place is its own input.)
static bool overlapping(const void* const* in, void* const* out, const int64_t* n, const uint8_t* in_types, const uint8_t* out_types, int count) {
    struct Range { uintptr_t at, end; bool written; };
    std::vector<Range> r;
    r.reserve((size_t)count * 2);
    for (int i = 0; i < count; ++i) {
        if (!n[i]) continue;
        const uintptr_t p = (uintptr_t)in[i], q = (uintptr_t)out[i];
        if (p != q || in_types[i] != out_types[i]) r.push_back({p, p + (uintptr_t)n[i] * (in_types[i] ? 2 : 4), false});
        r.push_back({q, q + (uintptr_t)n[i] * (out_types[i] ? 2 : 4), true});
    }
    const auto before = [](const Range& a, const Range& b) { return a.at < b.at; };
    if (!std::is_sorted(r.begin(), r.end(), before)) std::sort(r.begin(), r.end(), before);
    uintptr_t end = 0, written = 0;                         // of what began so far: all, and what is written
    for (const Range& a : r) {
        if (a.at < written || (a.written && a.at < end)) return true;
        end = std::max(end, a.end);
        if (a.written) written = std::max(written, a.end);
    }
    return false;
}

}  // namespace clip
}  // namespace msnet

using namespace msnet;

static int check_lengths(const char* what, const int64_t* n, int count) {
    if (count < 0 || (count && !n)) return fail("%s: %d tensors", what, count);
    for (int i = 0; i < count; ++i)
        if (n[i] < 0 || n[i] > ((int64_t)1 << 48)) return fail("%s: tensor %d has %lld values", what, i, (long long)n[i]);
    return 0;
}

extern "C" size_t msnet_clip_grads_workspace_bytes(const int64_t* n_host, int count) {
    if (check_lengths("msnet_clip_grads_workspace_bytes", n_host, count)) return 0;
    return (clip::cut(n_host, count).blocks + 1) * sizeof(double);
}

extern "C" int msnet_clip_grads(const void* const* in_host, void* const* out_host, const int64_t* n_host, const uint8_t* in_types_host,
                                const uint8_t* out_types_host, int count, double max_norm, float* norm, void* workspace, size_t workspace_bytes,
                                msnet_stream_t stream) {
    if (int rc = check_lengths("msnet_clip_grads", n_host, count)) return rc;
    if (!norm || (count && (!in_host || !in_types_host)) || (out_host && !out_types_host)) return fail("msnet_clip_grads: null pointer");
    if (out_host && !(max_norm >= 0.)) return fail("msnet_clip_grads: max_norm=%g", max_norm);
    const clip::Cut c = clip::cut(n_host, count);
    if (c.blocks > 0x7ffffffful) return fail("msnet_clip_grads: %lu workgroups are too many", c.blocks);
    if (!workspace || workspace_bytes < (c.blocks + 1) * sizeof(double) || ((uintptr_t)workspace & 7))
        return fail("msnet_clip_grads: workspace of %zu bytes at %p, %zu needed", workspace_bytes, workspace, (size_t)((c.blocks + 1) * sizeof(double)));
    for (int i = 0; i < count; ++i) {
        const int in = in_types_host[i], out = out_host ? out_types_host[i] : in;
        if (in > 2 || (out != in && out != 0)) return fail("msnet_clip_grads: tensor %d: types %d to %d (0 float32, 1 float16, 2 bfloat16; out: the same or float32)", i, in, out);
        if (n_host[i] && (!in_host[i] || (out_host && !out_host[i]))) return fail("msnet_clip_grads: null pointer (tensor %d)", i);
    }
    if (out_host) {
        try {
            if (clip::overlapping(in_host, out_host, n_host, in_types_host, out_types_host, count))
                return fail("msnet_clip_grads: a tensor to be written overlaps another one of the call (is a gradient listed twice?)");
        } catch (...) { return fail("msnet_clip_grads: out of host memory"); }
    }
    hipStream_t s = (hipStream_t)stream;
    double* sums = static_cast<double*>(workspace);
    double bytes_in = 0, bytes_out = 0;
    for (int i = 0; i < count; ++i) {
        bytes_in += (double)n_host[i] * (in_types_host[i] ? 2 : 4);
        if (out_host) bytes_out += (double)n_host[i] * (out_types_host[i] ? 2 : 4);
    }
    // pass 0: the sums; pass 1: the scaled gradients (or the norm alone).  Both cut the tensors the same way.
    for (int pass = 0; pass < 2; ++pass) {
        LaunchScope ls(pass ? "grad_scale" : "grad_square_sums", s, 0, pass ? bytes_out + (out_host ? bytes_in : 0.) : bytes_in);
        clip::Table t;
        unsigned long done = 0;                             // workgroups of this pass's earlier launches
        bool first = true;
        t.count = 0;
        t.first[0] = 0;
        for (int i = 0; i <= count; ++i) {
            if (i < count && n_host[i]) {
                t.in[t.count] = in_host[i];
                t.out[t.count] = out_host ? out_host[i] : nullptr;
                t.n[t.count] = n_host[i];
                t.types[t.count] = (unsigned char)(in_types_host[i] + 4 * (out_host ? out_types_host[i] : in_types_host[i]));
                t.first[t.count + 1] = t.first[t.count] + (unsigned)((n_host[i] + c.chunk - 1) / c.chunk);
                ++t.count;
            }
            if (t.count < clip::kTensors && i < count) continue;
            const unsigned blocks = t.first[t.count];
            if (pass == 0 && blocks)
                hipLaunchKernelGGL(clip::grad_square_sums, dim3(blocks), dim3(clip::kThreads), 0, s, t, c.chunk, sums + done);
            if (pass == 1 && ((blocks && out_host) || first)) {
                const bool scaling = blocks && out_host;
                hipLaunchKernelGGL(clip::grad_scale, dim3(scaling ? blocks : 1), dim3(clip::kThreads), 0, s, t, c.chunk, sums, (unsigned)c.blocks, max_norm,
                                   first ? norm : nullptr, (int)scaling);
                first = false;
            }
            if (int rc = check_launch("msnet_clip_grads")) return rc;
            done += blocks;
            t.count = 0;
        }
    }
    return 0;
}
