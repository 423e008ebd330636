// The global 2-norm of a list of gradients, and the gradients scaled to at most a given norm:
//
//   norm = sqrt(sum over all tensors of sum g^2),   out = g * min(1, max_norm / (norm + 1e-6))
//
// Memory-bound twice over: the norm has to be known before the first value is scaled, so gradients larger than the caches are read
// twice.  Tensors are cut into chunks of kChunk values, and the workgroups take chunks in turn, so that all of them together stream
// through one window of memory.  Up to kTensors tensors travel in the kernels' own arguments; more are written to the workspace
// first, kPart a launch, with every chunk's tensor beside them (so a captured graph needs no host memory either way).
// grad_square_sums leaves one 64-bit sum a workgroup, and each workgroup of grad_scale adds all of them up in a fixed order: no
// atomics, and a result repeats bit for bit.  Squares are formed and added in 64 bits, so no gradient's square overflows or vanishes.
#include <algorithm>
#include <vector>

#include "common.h"

namespace msnet {
namespace clip {

constexpr int kThreads = 256;
constexpr int kTensors = 176;          // in a kernel's arguments, which are 4 KB at most
constexpr int kPart = 216;             // of one launch that writes them to the workspace
constexpr int kChunk = 16384;          // values of a chunk
constexpr unsigned kBlocks = 512;      // workgroups at most, all on the device at once (1024: 2 % slower on 512 MB)

// One tensor.  n: its length, its input's type in bits 44 and 45, its output's in bits 46 and 47.
struct Entry { const void* in; void* out; unsigned long n; };
constexpr int kLengthBits = 44;
__device__ __forceinline__ long length(const Entry& e) { return (long)(e.n & ((1ul << kLengthBits) - 1)); }
__device__ __forceinline__ int types(const Entry& e) { return (int)(e.n >> kLengthBits); }      // input's + 4 * output's

// N of them as kernel arguments, 18 bytes each: addresses and n have 48 bits.
template <int N>
struct Packed {
    unsigned in[N], out[N], n[N];
    unsigned short in_high[N], out_high[N], n_high[N];
    void set(int i, const void* in_, void* out_, unsigned long n_) {
        in[i] = (unsigned)(uintptr_t)in_;
        out[i] = (unsigned)(uintptr_t)out_;
        n[i] = (unsigned)n_;
        in_high[i] = (unsigned short)((uintptr_t)in_ >> 32);
        out_high[i] = (unsigned short)((uintptr_t)out_ >> 32);
        n_high[i] = (unsigned short)(n_ >> 32);
    }
    __device__ __forceinline__ Entry get(int i) const {
        return {reinterpret_cast<const void*>((uintptr_t)in_high[i] << 32 | in[i]), reinterpret_cast<void*>((uintptr_t)out_high[i] << 32 | out[i]),
                (unsigned long)n_high[i] << 32 | n[i]};
    }
};

// The arguments lie in host memory, across the bus: all of them to LDS at once, 16 bytes a thread, and one wait.
template <class A>
__device__ __forceinline__ const A& in_lds(const A& a, uint4* lds, int tid) {
    static_assert(sizeof(A) % 16 == 0 && sizeof(A) <= 16 * kThreads, "one load a thread");
    if (tid < (int)(sizeof(A) / 16)) lds[tid] = reinterpret_cast<const uint4*>(&a)[tid];
    __syncthreads();
    return *reinterpret_cast<const A*>(lds);
}

struct alignas(16) Arguments {
    Packed<kTensors> e;
    unsigned first[kTensors];          // first chunk of each tensor
    int count;
};

// Where a workgroup finds its chunks' tensors: a chunk's is the number of first chunks up to it, three a lane.
struct ArgumentLookup {
    const Arguments& t;
    unsigned f[3];
    __device__ __forceinline__ ArgumentLookup(const Arguments& a, uint4* lds) : t(in_lds(a, lds, threadIdx.x)) {
        static_assert(kTensors <= 192, "three a lane");
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < 3; ++j) f[j] = lane + 64 * j < t.count ? t.first[min(lane + 64 * j, kTensors - 1)] : ~0u;
    }
    __device__ __forceinline__ Entry find(unsigned chunk, long* at) const {
        int k = -1;
#pragma unroll
        for (int j = 0; j < 3; ++j) k += __popcll(__ballot(f[j] <= chunk));
        *at = (long)(chunk - t.first[k]) * kChunk;
        return t.e.get(k);
    }
};

struct Workspace {
    const Entry* e;
    const unsigned* first;
    const unsigned* tensor;            // of each chunk
};

struct WorkspaceLookup {
    Workspace w;
    __device__ __forceinline__ WorkspaceLookup(const Workspace& t, uint4*) : w(t) {}
    __device__ __forceinline__ Entry find(unsigned chunk, long* at) const {
        const unsigned k = w.tensor[chunk];
        *at = (long)(chunk - w.first[k]) * kChunk;
        return w.e[k];
    }
};

template <class Source> struct Lookup;
template <> struct Lookup<Arguments> { typedef ArgumentLookup type; };
template <> struct Lookup<Workspace> { typedef WorkspaceLookup type; };

struct alignas(16) Part {
    Packed<kPart> e;
    int count;
};
static_assert(sizeof(Arguments) + 64 <= 4096 && sizeof(Part) + 64 <= 4096 && kPart <= kThreads, "kernel arguments, one thread a tensor");

__device__ __forceinline__ unsigned chunks_of(const Entry& e) { return (unsigned)((length(e) + kChunk - 1) / kChunk); }

// Tensors at .. at + count of the list, whose first chunk is `before`, and their chunks' places.
__global__ __launch_bounds__(kThreads) void grad_table(Part p, int at, unsigned before, Entry* __restrict__ e, unsigned* __restrict__ first,
                                                       unsigned* __restrict__ tensor) {
    __shared__ unsigned begin[kThreads + 1], wave[kThreads / 64];
    __shared__ uint4 lds[sizeof(Part) / 16];
    const int tid = threadIdx.x, lane = tid & 63;
    Entry mine = {nullptr, nullptr, 0};
    const Part& q = in_lds(p, lds, tid);
    if (tid < q.count) mine = q.e.get(tid);
    const unsigned chunks = tid < q.count ? chunks_of(mine) : 0u;
    unsigned sum = chunks;                                 // of this tensor's chunks and all before it in the wave
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned v = __shfl_up(sum, o);
        if (lane >= o) sum += v;
    }
    if (lane == 63) wave[tid >> 6] = sum;
    __syncthreads();
    for (int w = 0; w < tid >> 6; ++w) sum += wave[w];
    begin[tid + 1] = before + sum;
    if (tid == 0) begin[0] = before;
    __syncthreads();
    const bool writes = blockIdx.x == 0;                   // (every workgroup knows all; the first one writes what is short)
    if (writes && tid < q.count) { e[at + tid] = mine; first[at + tid] = begin[tid]; }
    if (writes && chunks <= 8)                             // a thread its own; a wave together for those of many, the workgroups in turn
        for (unsigned b = 0; b < chunks; ++b) tensor[begin[tid] + b] = (unsigned)(at + tid);
    for (unsigned long many = __ballot(chunks > 8); many; many &= many - 1) {
        const int i = (tid & ~63) + __builtin_ctzl(many);
        if (i % gridDim.x == blockIdx.x)
            for (unsigned b = begin[i] + lane; b < begin[i + 1]; b += 64) tensor[b] = (unsigned)(at + i);
    }
}

template <class T, int V> struct Pack { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };      // any view's alignment

__device__ __forceinline__ double block_sum(double s, double* tab, int tid) {
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((tid & 63) == 0) tab[tid >> 6] = s;
    __syncthreads();
    return (tab[0] + tab[1]) + (tab[2] + tab[3]);
}

template <class T>
__device__ __forceinline__ double square_sum(const T* p, int n, int tid) {
    constexpr int V = 16 / sizeof(T);
    typedef typename Pack<T, V>::type Vec;
    double s[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = 0.;
    const int nv = n / V;
    const Vec* v = reinterpret_cast<const Vec*>(p);
    int i = tid;
    auto add = [&](const Vec& a) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double d = (double)(float)a[e];
            s[e] = fma(d, d, s[e]);
        }
    };
    for (; i + 3 * kThreads < nv; i += 4 * kThreads) {
        const Vec a = v[i], b = v[i + kThreads], c = v[i + 2 * kThreads], d = v[i + 3 * kThreads];
        __builtin_amdgcn_sched_barrier(0);                 // (all four in flight: the compiler would move each down to its use)
        add(a); add(b); add(c); add(d);
    }
    for (; i < nv; i += kThreads) add(v[i]);
    double r = s[0];
#pragma unroll
    for (int e = 1; e < V; ++e) r += s[e];
    const int at = nv * V + tid;
    if (at < n) { const double d = (double)(float)p[at]; r = fma(d, d, r); }
    return r;
}

template <class Source>
__global__ __launch_bounds__(kThreads) void grad_square_sums(Source src, unsigned chunks, double* __restrict__ sums) {
    __shared__ double tab[4];
    __shared__ uint4 lds[sizeof(Arguments) / 16];
    const int tid = threadIdx.x;
    const typename Lookup<Source>::type table(src, lds);
    double s = 0.;
    for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
        long at;
        const Entry e = table.find(c, &at);
        const int n = (int)min((long)kChunk, length(e) - at);
        switch (types(e) & 3) {
            case 0: s += square_sum(static_cast<const float*>(e.in) + at, n, tid); break;
            case 1: s += square_sum(static_cast<const _Float16*>(e.in) + at, n, tid); break;
            default: s += square_sum(static_cast<const __bf16*>(e.in) + at, n, tid);
        }
    }
    s = block_sum(s, tab, tid);
    if (tid == 0) sums[blockIdx.x] = s;
}

__device__ __forceinline__ double total_of(const double* __restrict__ sums, unsigned n, double* tab, int tid) {
    double s = 0.;
#pragma unroll 4
    for (unsigned i = tid; i < n; i += kThreads) s += sums[i];
    return block_sum(s, tab, tid);
}

// One workgroup: the norm alone.
__global__ __launch_bounds__(kThreads) void grad_total(const double* __restrict__ sums, unsigned n, float* norm) {
    __shared__ double tab[4];
    const double s = total_of(sums, n, tab, threadIdx.x);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// A chunk of out = in * f in vectors of 16 bytes of the output, and shifted so that a wave writes whole lines: views into a buffer
// begin anywhere, and the first chunk takes what lies before its first line too.
template <bool STREAM, class T, class O>
__device__ __forceinline__ void scale(const void* in, void* out, long at, long all, float f, int tid) {
    const T* p = static_cast<const T*>(in);
    O* o = static_cast<O*>(out);
    const int head = (int)min(all, (long)((128 - ((uintptr_t)o & 127)) % 128 / sizeof(O)));
    if (at == 0 && tid < head) o[tid] = (O)((float)p[tid] * f);
    p += at + head;
    o += at + head;
    const int n = (int)max(0l, min((long)kChunk, all - at - head));
    constexpr int V = 16 / sizeof(O), U = sizeof(T) < sizeof(O) ? 8 : 4;
    typedef typename Pack<T, V>::type Vec;
    typedef typename Pack<O, V>::type Out;
    const int nv = n / V;
    const Vec* v = reinterpret_cast<const Vec*>(p);
    Out* w = reinterpret_cast<Out*>(o);
    const auto get = [&](int i) {
        if constexpr (STREAM) return __builtin_nontemporal_load(v + i);
        else return v[i];
    };
    const auto put = [&](int i, const Vec& a) {
        Out r;
#pragma unroll
        for (int e = 0; e < V; ++e) r[e] = (O)((float)a[e] * f);
        if constexpr (STREAM) __builtin_nontemporal_store(r, w + i);
        else w[i] = r;
    };
    int i = tid;
    for (; i + (U - 1) * kThreads < nv; i += U * kThreads) {
        Vec a[U];
#pragma unroll
        for (int u = 0; u < U; ++u) a[u] = get(i + u * kThreads);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u) put(i + u * kThreads, a[u]);
    }
    for (; i < nv; i += kThreads) put(i, get(i));
    const int rest = nv * V + tid;
    if (rest < n) o[rest] = (O)((float)p[rest] * f);
}

// The same for a factor below float's normal numbers (gradients near float's largest), where a float would lose the factor's bits: in
// 64 bits, a value at a time.  A loop of its own: a second factor carried along by scale() cost every call 3 % (512 MB to float32:
// 375 us for 363).
template <class T, class O>
__device__ __forceinline__ void scale_tiny(const void* in, void* out, long at, long all, double r, int tid) {
    const T* p = static_cast<const T*>(in) + at;
    O* o = static_cast<O*>(out) + at;
    const int n = (int)min((long)kChunk, all - at);
#pragma unroll 1
    for (int i = tid; i < n; i += kThreads) o[i] = (O)(float)((double)(float)p[i] * r);
}

__device__ __forceinline__ double factor(double total, double max_norm) { return max_norm / (total + 1e-6); }

// STREAM: past the caches, for gradients that do not fit them anyway.
template <class Source, bool STREAM>
__global__ __launch_bounds__(kThreads) void grad_scale(Source src, unsigned chunks, const double* __restrict__ sums, double max_norm, float* norm) {
    __shared__ double tab[4];
    __shared__ uint4 lds[sizeof(Arguments) / 16];
    const int tid = threadIdx.x;
    const typename Lookup<Source>::type table(src, lds);
    const double total = sqrt(total_of(sums, gridDim.x, tab, tid));
    if (blockIdx.x == 0 && tid == 0) *norm = (float)total;
    const double r = factor(total, max_norm);
    const float f = r > 1. ? 1.f : (float)r;               // (a NaN stays one)
    const bool tiny = r > 0. && r < 0x1p-126;
    // last chunks first: what the sums read last is what the caches hold
    for (unsigned c = blockIdx.x + (chunks - 1 - blockIdx.x) / gridDim.x * gridDim.x;; c -= gridDim.x) {
        long at;
        const Entry e = table.find(c, &at);
        if (f != 1.f || e.in != e.out) {                   // (else: short enough already, in place)
            const long all = length(e);
            if (tiny) {
                const double t = factor(sqrt((tab[0] + tab[1]) + (tab[2] + tab[3])), max_norm);      // (r, not kept over the loop)
                switch (types(e)) {
                    case 0: scale_tiny<float, float>(e.in, e.out, at, all, t, tid); break;
                    case 1: scale_tiny<_Float16, float>(e.in, e.out, at, all, t, tid); break;
                    case 2: scale_tiny<__bf16, float>(e.in, e.out, at, all, t, tid); break;
                    case 5: scale_tiny<_Float16, _Float16>(e.in, e.out, at, all, t, tid); break;
                    default: scale_tiny<__bf16, __bf16>(e.in, e.out, at, all, t, tid);
                }
            } else switch (types(e)) {
                case 0: scale<STREAM, float, float>(e.in, e.out, at, all, f, tid); break;
                case 1: scale<STREAM, _Float16, float>(e.in, e.out, at, all, f, tid); break;
                case 2: scale<STREAM, __bf16, float>(e.in, e.out, at, all, f, tid); break;
                case 5: scale<STREAM, _Float16, _Float16>(e.in, e.out, at, all, f, tid); break;
                default: scale<STREAM, __bf16, __bf16>(e.in, e.out, at, all, f, tid);
            }
        }
        if (c < gridDim.x) break;
    }
}

struct Cut {
    unsigned long chunks;
    int tensors;                       // that hold any value
    unsigned blocks() const { return chunks < kBlocks ? (unsigned)chunks : kBlocks; }
    size_t bytes() const {             // the sums, the tensors of a long list and the chunks'
        return (size_t)kBlocks * sizeof(double) + (tensors > kTensors ? (size_t)tensors * (sizeof(Entry) + sizeof(unsigned)) + chunks * sizeof(unsigned) : 0);
    }
};

static long chunks_of_length(int64_t n) { return (long)((n + kChunk - 1) / kChunk); }

static Cut cut(const int64_t* n, int count) {
    Cut c = {0, 0};
    for (int i = 0; i < count; ++i) {
        c.chunks += (unsigned long)chunks_of_length(n[i]);
        c.tensors += n[i] > 0;
    }
    return c;
}

// Whether a value would be written that another tensor of the call reads or writes too: workgroups run in any order, so the result
// would depend on it.  (A tensor scaled in place is its own input.)
static bool overlapping(const void* const* in, void* const* out, const int64_t* n, const uint8_t* in_types, const uint8_t* out_types, int count) {
    struct Range { uintptr_t at, end; };
    std::vector<Range> read, written;
    read.reserve((size_t)count);
    written.reserve((size_t)count);
    for (int i = 0; i < count; ++i) {
        if (!n[i]) continue;
        const uintptr_t p = (uintptr_t)in[i], q = (uintptr_t)out[i];
        if (p != q || in_types[i] != out_types[i]) read.push_back({p, p + (uintptr_t)n[i] * (in_types[i] ? 2 : 4)});
        written.push_back({q, q + (uintptr_t)n[i] * (out_types[i] ? 2 : 4)});
    }
    const auto before = [](const Range& a, const Range& b) { return a.at < b.at; };
    for (auto* r : {&read, &written})                       // (views into one buffer come in order)
        if (!std::is_sorted(r->begin(), r->end(), before)) std::sort(r->begin(), r->end(), before);
    for (size_t i = 1; i < written.size(); ++i)
        if (written[i].at < written[i - 1].end) return true;
    size_t k = 0;                                           // the first written range that ends behind the one read
    for (const Range& a : read) {
        while (k < written.size() && written[k].end <= a.at) ++k;
        if (k < written.size() && written[k].at < a.end) return true;
    }
    return false;
}

}  // namespace clip
}  // namespace msnet

using namespace msnet;

static int check_lengths(const char* what, const int64_t* n, int count) {
    if (count < 0 || (count && !n)) return fail("%s: %d tensors", what, count);
    for (int i = 0; i < count; ++i)
        if (n[i] < 0 || n[i] >= ((int64_t)1 << clip::kLengthBits)) return fail("%s: tensor %d has %lld values", what, i, (long long)n[i]);
    return 0;
}

extern "C" size_t msnet_clip_grads_workspace_bytes(const int64_t* n_host, int count) {
    if (check_lengths("msnet_clip_grads_workspace_bytes", n_host, count)) return 0;
    return clip::cut(n_host, count).bytes();
}

extern "C" int msnet_clip_grads(const void* const* in_host, void* const* out_host, const int64_t* n_host, const uint8_t* in_types_host,
                                const uint8_t* out_types_host, int count, double max_norm, float* norm, void* workspace, size_t workspace_bytes,
                                msnet_stream_t stream) {
    if (int rc = check_lengths("msnet_clip_grads", n_host, count)) return rc;
    if (!norm || (count && (!in_host || !in_types_host)) || (out_host && !out_types_host)) return fail("msnet_clip_grads: null pointer");
    if (out_host && !(max_norm >= 0.)) return fail("msnet_clip_grads: max_norm=%g", max_norm);
    const clip::Cut c = clip::cut(n_host, count);
    if (c.chunks > 0x7ffffffful) return fail("msnet_clip_grads: %lu chunks are too many", c.chunks);
    if (!workspace || workspace_bytes < c.bytes() || ((uintptr_t)workspace & 7))
        return fail("msnet_clip_grads: workspace of %zu bytes at %p, %zu needed", workspace_bytes, workspace, c.bytes());
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
    const unsigned blocks = c.blocks(), chunks = (unsigned)c.chunks;
    const bool past_caches = bytes_out >= 64e6;
    const auto put = [&](auto& packed, int at, int i) {
        const unsigned long in = in_types_host[i], out = out_host ? out_types_host[i] : in_types_host[i];
        packed.set(at, in_host[i], out_host ? out_host[i] : nullptr, (unsigned long)n_host[i] | (in + 4 * out) << clip::kLengthBits);
    };
    const auto run = [&](auto src) {
        if (blocks) {
            LaunchScope ls("grad_square_sums", s, 0, bytes_in);
            hipLaunchKernelGGL((clip::grad_square_sums<decltype(src)>), dim3(blocks), dim3(clip::kThreads), 0, s, src, chunks, sums);
        }
        if (out_host && blocks) {
            LaunchScope ls("grad_scale", s, 0, bytes_in + bytes_out);
            const auto kernel = past_caches ? clip::grad_scale<decltype(src), true> : clip::grad_scale<decltype(src), false>;
            hipLaunchKernelGGL(kernel, dim3(blocks), dim3(clip::kThreads), 0, s, src, chunks, sums, max_norm, norm);
        } else {
            LaunchScope ls("grad_total", s, 0, 8.0 * blocks);
            hipLaunchKernelGGL(clip::grad_total, dim3(1), dim3(clip::kThreads), 0, s, sums, blocks, norm);
        }
        return check_launch("msnet_clip_grads");
    };
    if (c.tensors <= clip::kTensors) {
        clip::Arguments a;
        a.count = 0;
        unsigned first = 0;
        for (int i = 0; i < count; ++i)
            if (n_host[i]) {
                put(a.e, a.count, i);
                a.first[a.count++] = first;
                first += (unsigned)clip::chunks_of_length(n_host[i]);
            }
        return run(a);
    }
    clip::Entry* e = reinterpret_cast<clip::Entry*>(sums + clip::kBlocks);
    unsigned* first = reinterpret_cast<unsigned*>(e + c.tensors);
    unsigned* tensor = first + c.tensors;
    {
        LaunchScope ls("grad_table", s, 0, 28.0 * c.tensors + 4.0 * chunks);
        clip::Part p;
        p.count = 0;
        int at = 0;
        unsigned before = 0, next = 0;
        for (int i = 0; i < count; ++i) {
            if (n_host[i]) {
                put(p.e, p.count++, i);
                next += (unsigned)clip::chunks_of_length(n_host[i]);
            }
            if (p.count == clip::kPart || (i == count - 1 && p.count)) {
                hipLaunchKernelGGL(clip::grad_table, dim3(8), dim3(clip::kThreads), 0, s, p, at, before, e, first, tensor);
                at += p.count;
                before = next;
                p.count = 0;
            }
        }
        if (int rc = check_launch("msnet_clip_grads")) return rc;
    }
    return run(clip::Workspace{e, first, tensor});
}
