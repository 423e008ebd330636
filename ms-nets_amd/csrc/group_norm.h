// What the forward and backward kernels of the group norm share: shapes and chunks, row access, the sums over a group.
//
//   mean_g = (1/m) sum x,  var_g = (1/m) sum (x - mean_g)^2,  m = S * C/G values of one sample and group
//   xhat = (x - mean) / sqrt(var + eps),   z = xhat * gamma_c + beta_c (+ residual),   y = act(z)
//
// Channels-last rows ([N][S][C], S = all spatial positions): one thread keeps the same V channels of a row (one vector of up to
// 16 bytes) and walks down the rows, so its channels' constants stay in registers and a wave reads whole consecutive rows.
#pragma once
#include "common.h"

namespace msnet {
namespace gn {

constexpr int kThreads = 256;          // of the streaming kernels; the channels of a chunk are at most kThreads * V
enum Act { kNone = 0, kRelu = 1, kSilu = 2 };
enum DType { kF32 = 0, kF16 = 1, kBF16 = 2 };

// V values as they lie in memory.  Rows of any stride and views of any offset are taken: gfx950's global loads and stores of up to
// 16 bytes need no more alignment than the element's own.
template <class T, int V> struct Pack { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };
template <class T> struct Pack<T, 1> { typedef T type; };

// STREAM: past the caches, which nobody needs these values from soon (streams(), below).
template <class T, int V, bool STREAM = false>
__device__ __forceinline__ typename Pack<T, V>::type load_raw(const T* p) {
    const auto q = reinterpret_cast<const typename Pack<T, V>::type*>(p);
    if constexpr (STREAM) return __builtin_nontemporal_load(q);
    else return *q;
}

template <class T, int V>
__device__ __forceinline__ float element(const typename Pack<T, V>::type& r, int e) {
    if constexpr (V == 1) return (float)r;
    else return (float)r[e];
}

template <class T, int V, bool STREAM = false>
__device__ __forceinline__ void store(T* p, const float (&f)[V]) {
    typename Pack<T, V>::type o;
    if constexpr (V == 1) o = (T)f[0];
    else
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = (T)f[e];
    const auto q = reinterpret_cast<typename Pack<T, V>::type*>(p);
    if constexpr (STREAM) __builtin_nontemporal_store(o, q);
    else *q = o;
}

struct Rows { long sn, ss; };          // elements from sample to sample and from row to row; channels are consecutive

// How the channels and rows of a call are cut.  A chunk is what one workgroup's row segment covers: `gpc` whole groups (nsub = 1),
// or, where one group is wider than a workgroup, `cw` channels of it (nsub chunks a group, gpc = 1).
struct Shape {
    int N, C, G, cg;                   // cg = C / G
    long S;
    int gpc, nsub, cw, chunks;
    int nblk;                          // workgroups that share a sample's rows: tiles of a few rows a thread, in turn (Walk)
    int rounds;                        // tiles of one of them, at most
};

struct Chunk {
    int n, blk, g0, ng, c0, cw, sub;
};

__device__ __forceinline__ Chunk chunk_of(const Shape& s, unsigned b) {
    Chunk k;
    const unsigned chunk = b % (unsigned)s.chunks, t = b / (unsigned)s.chunks;
    k.blk = (int)(t % (unsigned)s.nblk);
    k.n = (int)(t / (unsigned)s.nblk);
    if (s.nsub > 1) {
        k.g0 = (int)chunk / s.nsub; k.sub = (int)chunk % s.nsub; k.ng = 1;
        k.c0 = k.g0 * s.cg + k.sub * s.cw;
        k.cw = min(s.cw, s.cg - k.sub * s.cw);
    } else {
        k.g0 = (int)chunk * s.gpc; k.sub = 0; k.ng = min(s.gpc, s.G - k.g0);
        k.c0 = k.g0 * s.cg; k.cw = k.ng * s.cg;
    }
    return k;
}

// The rows of one thread: the workgroups of a sample take tiles of U rows a thread in turn, so that all of them together stream
// through one window of memory (each its own contiguous part instead made the finest level's passes 10 to 30 % slower: their
// streams lie at like distances and meet in the same channels).  BACK starts at the last tile.
template <int U, bool BACK>
struct Walk {
    const Shape& s;
    long row;
    int blk, step;
    bool on;
    __device__ __forceinline__ Walk(const Shape& s_, int blk_, int row_, int step_, bool on_) : s(s_), row(row_), blk(blk_), step(step_), on(on_) {}
    // tile(r) for whole tiles, one(r) for the rows of a tile that passes the end
    template <class Whole, class One>
    __device__ __forceinline__ void run(Whole tile, One one) const {
        if (!on) return;
        for (int i = 0; i < s.rounds; ++i) {
            const long r = ((long)(BACK ? s.rounds - 1 - i : i) * s.nblk + blk) * (U * step) + row;
            if (r + (long)(U - 1) * step < s.S) tile(r);
            else
                for (int u = 0; u < U; ++u)
                    if (r + (long)u * step < s.S) one(r + (long)u * step);
        }
    }
};

// U rows of a thread's V channels, loaded at once.  A loads_issued() behind the tiles' loads keeps the compiler from moving them down
// to their uses one by one, as it does for bf16 (sums of the finest level: 136 us with all in flight, 240 without).
__device__ __forceinline__ void loads_issued() { __builtin_amdgcn_sched_barrier(0); }
template <class T, int V, int U, bool STREAM = false>
struct Tile {
    typename Pack<T, V>::type v[U];
    __device__ __forceinline__ void load(const T* p, long r, int step, long ss) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load_raw<T, V, STREAM>(p + (size_t)(r + (long)u * step) * ss);
    }
};

__device__ __forceinline__ double2 shuffle_xor(double2 v, int o) { return make_double2(__shfl_xor(v.x, o), __shfl_xor(v.y, o)); }

// Adds the rows of tab[rows][cols] into row 0, pairwise and in a fixed order; every thread of the workgroup takes part.
__device__ __forceinline__ void sum_rows(double2* tab, int rows, int cols, int tid, int threads) {
    int p = 1;
    while (p < rows) p <<= 1;
    for (int step = p >> 1; step > 0; step >>= 1) {
        __syncthreads();
        for (int i = tid; i < step * cols; i += threads)
            if (i + step * cols < rows * cols) tab[i] = tab[i] + tab[i + step * cols];
    }
    __syncthreads();
}

// f(group, sum of its `per` consecutive entries of tab, each first put through w), called by one thread a group.
template <class W, class F>
__device__ __forceinline__ void sum_groups(const double2* tab, int per, int ng, int tid, int threads, W w, F f) {
    int lanes = 1;                     // threads of a group: a power of two, inside one wave
    while (lanes < 64 && 2 * lanes <= per && 2 * lanes * ng <= threads) lanes <<= 1;
    const int lane = tid & (lanes - 1);
    for (int g = tid / lanes; g < ng; g += threads / lanes) {
        double2 s = make_double2(0., 0.);
        for (int i = lane; i < per; i += lanes) s = s + w(g * per + i, tab[g * per + i]);
        for (int o = lanes >> 1; o > 0; o >>= 1) s = s + shuffle_xor(s, o);
        if (lane == 0) f(g, s);
    }
}

// Whether threads a power of two below a wave's width apart hold the same columns: their rows are added across the wave first.
__device__ __forceinline__ bool in_wave(int columns) { return columns < 64 && (columns & (columns - 1)) == 0; }

// Adds K values a thread over the rows (tid / cv) of threads with the same tid % cv: tab[(tid % cv) * K + j] gets the sums.  Every
// thread takes part; `on` says whether it has a row.  tab: threads * K entries, or threads / 64 * cv * K where in_wave(cv).
template <int K>
__device__ __forceinline__ void sum_threads(double2 (&v)[K], double2* tab, int cv, bool on, int tid, int threads) {
    if (in_wave(cv)) {
#pragma unroll
        for (int j = 0; j < K; ++j)
            for (int o = cv; o < 64; o <<= 1) v[j] = v[j] + shuffle_xor(v[j], o);
        if ((tid & 63) < cv) {
#pragma unroll
            for (int j = 0; j < K; ++j) tab[((tid >> 6) * cv + (tid & 63)) * K + j] = v[j];
        }
        sum_rows(tab, threads >> 6, cv * K, tid, threads);
    } else {
        if (on) {
#pragma unroll
            for (int j = 0; j < K; ++j) tab[tid * K + j] = v[j];
        }
        sum_rows(tab, threads / cv, cv * K, tid, threads);
    }
}

// The sums of groups g0 .. g0 + ng over a sample's slots, part[slot][G]: f(group - g0, sum) by one thread a group.
template <class F>
__device__ __forceinline__ void sum_slots(const double2* __restrict__ part, int slots, int G, int g0, int ng, double2* tab, int tid, F f) {
    for (int gt = 0; gt < ng; gt += kThreads) {
        const int w = min(ng - gt, kThreads), lanes = kThreads / w;
        const int gi = tid % w, lane = tid / w;
        double2 s[1] = {make_double2(0., 0.)};
        if (lane < lanes) {
            const double2* p = part + g0 + gt + gi;
#pragma unroll 4
            for (int i = lane; i < slots; i += lanes) s[0] = s[0] + p[(size_t)i * G];
        }
        sum_threads<1>(s, tab, w, lane < lanes, tid, kThreads);
        if (tid < w) f(gt + tid, tab[tid]);
        __syncthreads();
    }
}

// V channels' gamma or beta, the default's where there are none.  One load from an address chosen before: a load in a branch is waited
// for at the branch's end, and with it everything else in flight.
static __device__ const float kDefaults[8] = {0.f, 0.f, 0.f, 0.f, 1.f, 1.f, 1.f, 1.f};
template <int V>
__device__ __forceinline__ void load_params(const float* params, int c, bool one, float (&out)[V]) {
    const auto v = load_raw<float, V>(params ? params + c : kDefaults + (one ? 4 : 0));
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = element<float, V>(v, e);
}

// 1 / (1 + e^-z).  Below z = -87.4 it is 0, off by less than 2^-126: e^-z or its reciprocal leaves float32's range.
__device__ __forceinline__ float silu_gate(float z) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * z));
}

template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == kRelu) return z < 0.f ? 0.f : z;     // (a NaN stays one)
    else if constexpr (ACT == kSilu) return z * silu_gate(z);
    else return z;
}

// ---- host ------------------------------------------------------------------------------------------------------------
inline int element_bytes(int dtype) { return dtype == kF32 ? 4 : 2; }

// Channels a thread takes at once.  Four of any type: eight 16-bit ones (16-byte lanes, groups of four or fewer inside a vector) were
// no faster on any size once eight rows of four are loaded at once, and 5 us slower on the smallest.
inline int vector_width(int C) { return C % 4 == 0 ? 4 : C % 2 == 0 ? 2 : 1; }
// Rows of a thread's vectors that are loaded at once where bandwidth decides.
constexpr int tile_rows(int V, int bytes) { return V * bytes == 16 ? 4 : 8; }

// Whether a result goes past the caches, and an input that is read for the last time too.  The last-level cache holds 256 MB: a
// result of an eighth of it and more leaves there as a block of dirty lines that the next pass has to push out before it can keep
// what it will read again.  Forward and backward of 94 MB: 222 us through the caches, 203 past them; of 805 MB: 1156 and 1113.
// A smaller result is worth more to whoever reads it next, and lanes of two or four bytes write lines in parts, which only the caches
// put together (33 channels of bf16, forward and backward of 120 MB: 349 us past them, 318 through them).
inline bool streams(double bytes, int lane_bytes) { return bytes >= 32e6 && lane_bytes >= 8; }

int check_shape(const char* what, int dtype, int act, int N, long S, int C, int G, double eps);
// V may be lowered to 1: groups whose edges fall inside vectors and that are too wide to be cut at a common multiple.
Shape make_shape(int N, long S, int C, int G, int* V, long most_cw);
// nblk and rounds: at most most_blocks workgroups in all, each with `tiles` tiles of `tile` rows a thread or more.
void cut_rows(Shape* s, int V, long most_blocks, int tile, int tiles);

}  // namespace gn
}  // namespace msnet
