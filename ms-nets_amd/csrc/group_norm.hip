// Group norm with an activation over channels-last activations, forward: y = act(xhat * gamma + beta (+ residual)).
//
// Two ways, by size:
//   * group_norm_small: a chunk of whole groups of one sample fits the registers of one workgroup; it is read once, in one launch.
//   * group_norm_stats + group_norm_apply: every row block's sums per group go to the workspace, and each workgroup of the second
//     kernel adds up its groups' sums before it normalises; x is read twice, y written once.
//
// Sums are of x - pivot and its square, in 64 bits (pivot: the group's first value): no cancellation for any mean, and the sign of
// a value next to a ReLU's border comes out as in exact arithmetic, which the backward pass relies on.  gfx950 adds doubles at the
// rate of (unpacked) floats: a value costs a conversion or two, a subtraction, an addition and a fused square, and the sums stay below
// the memory's time where a lane has four channels (120 MB of bf16: 5.1 TB/s with 64 channels, 2.5 with 21, one a lane).
#include <type_traits>

#include "group_norm.h"

namespace msnet {
namespace gn {

int check_shape(const char* what, int dtype, int act, int N, long S, int C, int G, double eps) {
    if (dtype < kF32 || dtype > kBF16) return fail("%s: dtype %d is none of 0 (float32), 1 (float16), 2 (bfloat16)", what, dtype);
    if (act < kNone || act > kSilu) return fail("%s: activation %d is none of 0 (none), 1 (ReLU), 2 (SiLU)", what, act);
    if (N < 0 || S < 0 || C <= 0) return fail("%s: bad shape N=%d S=%ld C=%d", what, N, S, C);
    if (G <= 0 || C % G != 0) return fail("%s: %d groups do not divide %d channels", what, G, C);
    if (!(eps >= 0.)) return fail("%s: eps=%g", what, eps);
    return 0;
}

static int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

Shape make_shape(int N, long S, int C, int G, int* V, long most_cw) {
    Shape s = {};
    s.N = N; s.S = S; s.C = C; s.G = G; s.cg = C / G;
    int step = *V / gcd(s.cg, *V);                         // groups between two edges that are edges of vectors too
    if (step > 1 && (long)s.cg * step > (long)kThreads * *V) { *V = 1; step = 1; }
    const long widest = (long)kThreads * *V;
    if ((long)s.cg * step > widest) {
        s.gpc = 1; s.cw = (int)widest; s.nsub = (int)((s.cg + widest - 1) / widest); s.chunks = G * s.nsub;
    } else {
        const long w = most_cw < widest ? most_cw : widest, unit = (long)s.cg * step;
        const int most = (int)(w / unit > 0 ? w / unit : 1) * step;
        s.chunks = (G + most - 1) / most;
        s.gpc = ((G + s.chunks - 1) / s.chunks + step - 1) / step * step;
        s.chunks = (G + s.gpc - 1) / s.gpc;
        s.nsub = 1; s.cw = (s.gpc < G ? s.gpc : G) * s.cg;
    }
    s.nblk = 1;
    return s;
}

void cut_rows(Shape* s, int V, long most_blocks, int tile, int tiles) {
    const long rows = (long)(kThreads / (s->cw / V)) * tile;           // of a tile (of the widest chunk: the last one's are longer)
    const long all = (s->S + rows - 1) / rows, most = (all + tiles - 1) / tiles, nblk = most_blocks / ((long)s->N * s->chunks);
    s->nblk = (int)(nblk < 1 ? 1 : nblk < most ? nblk : most);
    s->rounds = (int)((all + s->nblk - 1) / s->nblk);
}

// mean and 1 / sqrt(var + eps) from the sums of x - pivot and of its square; inv = 1 / m
__device__ __forceinline__ double2 statistics(double2 sum, double pivot, double inv, double eps) {
    const double d = sum.x * inv;
    double var = sum.y * inv - d * d;
    var = var < 0. ? 0. : var;
    return make_double2(pivot + d, 1. / sqrt(var + eps));
}

// What a thread keeps of its channels: z = (x - mean) * scale + shift with the mean's own rounding folded into shift.
template <int V>
struct Affine {
    float mean[V], scale[V], shift[V];
    // gamma and beta first, so that they arrive while the sums are formed
    __device__ __forceinline__ void load(int c, const float* weight, const float* bias) {
        load_params<V>(weight, c, true, scale);
        load_params<V>(bias, c, false, shift);
    }
    __device__ __forceinline__ void set(const double2* st, int c_local, int cg, bool whole) {
        double2 t = st[c_local / cg];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (!whole) t = st[(c_local + e) / cg];
            const double a = t.y * (double)scale[e];
            mean[e] = (float)t.x;
            scale[e] = (float)a;
            shift[e] = (float)((double)shift[e] - (t.x - (double)mean[e]) * a);
        }
    }
};

// One row's V values: normalise, add the residual, activate, store; amax gathers magnitude bits for the range guard.
template <class T, int V, int ACT, bool STREAM>
__device__ __forceinline__ void finish(const Affine<V>& k, const typename Pack<T, V>::type& x, const typename Pack<T, V>::type& res, bool has_res,
                                       T* y, bool guard, unsigned& amax) {
    float o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        float z = fmaf(element<T, V>(x, e) - k.mean[e], k.scale[e], k.shift[e]);
        if (has_res) z += element<T, V>(res, e);
        o[e] = activate<ACT>(z);
    }
    if (guard)
#pragma unroll
        for (int e = 0; e < V; ++e) amax = max(amax, __builtin_bit_cast(unsigned, o[e]) & 0x7fffffffu);
    store<T, V, STREAM>(y, o);
}

// Sums of x - pivot and of its square, a channel.
template <class T, int V>
struct Sums {
    double pivot[V], s[V], q[V];
    __device__ __forceinline__ void start(const T (&first)[V]) {
#pragma unroll
        for (int e = 0; e < V; ++e) { pivot[e] = (double)(float)first[e]; s[e] = q[e] = 0.; }
    }
    __device__ __forceinline__ void add(const typename Pack<T, V>::type& v) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double d = (double)element<T, V>(v, e) - pivot[e];
            s[e] += d;
            q[e] = fma(d, d, q[e]);
        }
    }
    // Over the threads of a workgroup, into tab: one entry a vector where a vector lies in one group, one a channel elsewhere.
    __device__ __forceinline__ void join(double2* tab, bool whole, int cv, bool on, int tid, int threads) {
        if (whole) {
            double2 v[1] = {make_double2(s[0], q[0])};
#pragma unroll
            for (int e = 1; e < V; ++e) { v[0].x += s[e]; v[0].y += q[e]; }
            sum_threads<1>(v, tab, cv, on, tid, threads);
        } else {
            double2 v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = make_double2(s[e], q[e]);
            sum_threads<V>(v, tab, cv, on, tid, threads);
        }
    }
};

template <class T, int V>
__global__ __launch_bounds__(kThreads) void group_norm_stats(const T* __restrict__ x, Rows xr, Shape sh, double2* __restrict__ part,
                                                             double* __restrict__ pivots) {
    extern __shared__ __attribute__((aligned(16))) double2 tab[];
    const Chunk k = chunk_of(sh, blockIdx.x);
    const int tid = threadIdx.x, cv = k.cw / V, per_pass = kThreads / cv;
    const int row = tid / cv, cl = (tid % cv) * V;
    const bool whole = sh.cg % V == 0, on = row < per_pass;
    const T* xn = x + (size_t)k.n * xr.sn;
    const T* p = xn + k.c0 + cl;
    T pivot[V];
    pivot[0] = xn[(size_t)(k.g0 + (k.ng > 1 ? cl / sh.cg : 0)) * sh.cg];
#pragma unroll
    for (int e = 1; e < V; ++e) pivot[e] = whole ? pivot[0] : xn[(size_t)(k.g0 + (k.ng > 1 ? (cl + e) / sh.cg : 0)) * sh.cg];
    if (k.blk == 0 && k.sub == 0)
        for (int g = tid; g < k.ng; g += kThreads) pivots[(size_t)k.n * sh.G + k.g0 + g] = (double)(float)xn[(size_t)(k.g0 + g) * sh.cg];
    Sums<T, V> sums;
    sums.start(pivot);
    constexpr int kTile = tile_rows(V, sizeof(T));
    Walk<kTile, false>(sh, k.blk, row, per_pass, on).run(
        [&](long r) {
            Tile<T, V, kTile> t;
            t.load(p, r, per_pass, xr.ss);
            loads_issued();
#pragma unroll
            for (int u = 0; u < kTile; ++u) sums.add(t.v[u]);
        },
        [&](long r) { sums.add(load_raw<T, V>(p + (size_t)r * xr.ss)); });
    sums.join(tab, whole, cv, on, tid, kThreads);
    const size_t slot = (size_t)k.n * sh.nblk * sh.nsub + (size_t)k.blk * sh.nsub + k.sub;
    sum_groups(tab, (whole ? cv : k.cw) / k.ng, k.ng, tid, kThreads, [](int, double2 v) { return v; },
               [&](int g, double2 v) { part[slot * sh.G + k.g0 + g] = v; });
}

// STREAM: y goes past the caches; without statistics to save (no backward will read them again) x and the residual do too.
template <class T, int V, int ACT, bool STREAM>
__global__ __launch_bounds__(kThreads) void group_norm_apply(const T* x, Rows xr, const float* __restrict__ weight,
                                                             const float* __restrict__ bias, const T* residual, Rows rr, T* y, Rows yr,
                                                             double2* __restrict__ stats, Shape sh, int slots,
                                                             const double2* __restrict__ part, const double* __restrict__ pivots,
                                                             double inv, double eps, unsigned* oflag) {
    extern __shared__ __attribute__((aligned(16))) double2 tab[];      // [kThreads] sums, [ng] statistics
    double2* st = tab + kThreads;
    const bool has_res = residual != nullptr;
    const Chunk k = chunk_of(sh, blockIdx.x);
    const int tid = threadIdx.x, cv = k.cw / V, per_pass = kThreads / cv;
    const int row = tid / cv, cl = (tid % cv) * V;
    const T* px = x + (size_t)k.n * xr.sn + k.c0 + cl;
    const T* pr = has_res ? residual + (size_t)k.n * rr.sn + k.c0 + cl : px;
    const long rs = has_res ? rr.ss : xr.ss;
    T* py = y + (size_t)k.n * yr.sn + k.c0 + cl;
    Affine<V> a;
    a.load(k.c0 + cl, weight, bias);
    const double* mine = pivots + (size_t)k.n * sh.G + k.g0;
    const double pivot = mine[min(tid, k.ng - 1)];         // of the group whose sums this thread will have (of the first kThreads groups)
    sum_slots(part + (size_t)k.n * slots * sh.G, slots, sh.G, k.g0, k.ng, tab, tid, [&](int g, double2 sum) {
        const size_t at = (size_t)k.n * sh.G + k.g0 + g;
        const double2 v = statistics(sum, g < kThreads ? pivot : mine[g], inv, eps);
        st[g] = v;
        if (stats && k.blk == 0 && k.sub == 0) stats[at] = v;
    });
    a.set(st, cl, k.ng > 1 ? sh.cg : k.cw, sh.cg % V == 0);
    unsigned amax = 0u;
    const auto put = [&](long r, const typename Pack<T, V>::type& vx, const typename Pack<T, V>::type& vr) {
        finish<T, V, ACT, STREAM>(a, vx, vr, has_res, py + (size_t)r * yr.ss, oflag != nullptr, amax);
    };
    constexpr int kTile = tile_rows(V, sizeof(T));
    const auto rows = [&](auto last) {                     // last rows first: what the sums read last is what the caches hold
        Walk<kTile, true>(sh, k.blk, row, per_pass, row < per_pass).run(
            [&](long r) {
                Tile<T, V, kTile, decltype(last)::value> x4, r4;
                x4.load(px, r, per_pass, xr.ss);
                if (has_res) r4.load(pr, r, per_pass, rs);
                else r4 = x4;
                loads_issued();
#pragma unroll
                for (int u = 0; u < kTile; ++u) put(r + (long)u * per_pass, x4.v[u], r4.v[u]);
            },
            [&](long r) { put(r, load_raw<T, V>(px + (size_t)r * xr.ss), load_raw<T, V>(pr + (size_t)r * rs)); });
    };
    if constexpr (STREAM) {
        if (stats) rows(std::false_type{});
        else rows(std::true_type{});
    } else rows(std::false_type{});
    if (oflag && amax >= 0x46ffe000u) atomicOr(oflag, 1u);            // |y| >= 32752, inf or NaN: as the convs' epilogues
}

// M: vectors a thread holds.  A workgroup takes all rows of one chunk of one sample; of sh.nblk workgroups that share one (M / 4 or 1)
// each writes its part of them.
template <class T, int V, int M, int ACT>
__global__ __launch_bounds__(1024) void group_norm_small(const T* x, Rows xr, const float* __restrict__ weight, const float* __restrict__ bias,
                                                         const T* residual, Rows rr, T* y, Rows yr, double2* __restrict__ stats, Shape sh,
                                                         double inv, double eps, unsigned* oflag) {
    extern __shared__ __attribute__((aligned(16))) double2 tab[];
    const Chunk k = chunk_of(sh, blockIdx.x);
    const int tid = threadIdx.x, threads = blockDim.x, cv = k.cw / V, per_pass = threads / cv;
    const int row = tid / cv, cl = (tid % cv) * V;
    const bool whole = sh.cg % V == 0, on = row < per_pass;
    double2* st = tab + (whole ? threads : threads * V);  // [ng]: first each group's pivot, then its statistics
    const T* xn = x + (size_t)k.n * xr.sn;
    const T* px = xn + k.c0 + cl;
    const int S = (int)sh.S;
    T pivot[V];
    pivot[0] = xn[(size_t)(k.g0 + cl / sh.cg) * sh.cg];
#pragma unroll
    for (int e = 1; e < V; ++e) pivot[e] = whole ? pivot[0] : xn[(size_t)(k.g0 + (cl + e) / sh.cg) * sh.cg];
    typename Pack<T, V>::type v[M];
#pragma unroll
    for (int i = 0; i < M; ++i)
        if (on && row + i * per_pass < S) v[i] = load_raw<T, V>(px + (size_t)(row + i * per_pass) * xr.ss);
    Affine<V> a;
    a.load(k.c0 + cl, weight, bias);
    loads_issued();
    for (int g = tid; g < k.ng; g += threads) st[g].x = (double)(float)xn[(size_t)(k.g0 + g) * sh.cg];
    Sums<T, V> sums;
    sums.start(pivot);
#pragma unroll
    for (int i = 0; i < M; ++i)
        if (on && row + i * per_pass < S) sums.add(v[i]);
    sums.join(tab, whole, cv, on, tid, threads);
    sum_groups(tab, (whole ? cv : k.cw) / k.ng, k.ng, tid, threads, [](int, double2 u) { return u; }, [&](int g, double2 sum) {
        const double2 t = statistics(sum, st[g].x, inv, eps);
        st[g] = t;
        if (stats && k.blk == 0) stats[(size_t)k.n * sh.G + k.g0 + g] = t;
    });
    __syncthreads();                                       // statistics are there, and nobody reads x any more (y may be x)
    if (!on) return;
    a.set(st, cl, sh.cg, whole);
    const bool has_res = residual != nullptr;
    const T* pr = has_res ? residual + (size_t)k.n * rr.sn + k.c0 + cl : px;
    T* py = y + (size_t)k.n * yr.sn + k.c0 + cl;
    unsigned amax = 0u;
#pragma unroll
    for (int i0 = 0; i0 < M; i0 += 4) {
        if (sh.nblk > 1 && i0 != 4 * k.blk) continue;
        typename Pack<T, V>::type w[4];
        if (has_res) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (row + (i0 + j) * per_pass < S) w[j] = load_raw<T, V>(pr + (size_t)(row + (i0 + j) * per_pass) * rr.ss);
            loads_issued();
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = row + (i0 + j) * per_pass;
            if (r < S) finish<T, V, ACT, false>(a, v[i0 + j], has_res ? w[j] : v[i0 + j], has_res, py + (size_t)r * yr.ss, oflag != nullptr, amax);
        }
    }
    if (oflag && amax >= 0x46ffe000u) atomicOr(oflag, 1u);
}

// ---- host ------------------------------------------------------------------------------------------------------------

struct Forward {
    const void *x, *residual;
    const float *weight, *bias;
    void* y;
    double2* stats;
    Rows xr, rr, yr;
    double eps;
    unsigned* oflag;
    hipStream_t stream;
};

constexpr long kStatsBlocks = 512, kApplyBlocks = 512;
constexpr int kStatsTiles = 2, kApplyTiles = 2;      // tiles of a workgroup at least

// One workgroup a chunk: threads and vectors a thread, or 0 where the chunk does not fit.
static int small_threads(const Shape& s, int V, int* M) {
    const int cv = s.cw / V, most = s.cg % V == 0 ? 1024 : 2048 / V;      // (table of sums and statistics: 64 KB at most)
    for (int m : {4, 16})
        for (int t = 256; t <= most; t <<= 1)
            if (s.S <= (long)m * (t / cv)) { *M = m; return t; }
    return 0;
}

// Chunks of eight channels (or one group) give the single launch the most workgroups and let the longest samples fit: 3060 rows of 32
// channels of bf16 take 9.5 us with their launch, of 16 channels 11.6, of two launches 17.4.  Wider ones once those fill the device.
static Shape small_shape(int N, long S, int C, int G, int* V) {
    long w = 8;
    Shape s = make_shape(N, S, C, G, V, w);
    while ((long)N * s.chunks > 2048 && w < (long)kThreads * *V) {
        w *= 2;
        const Shape t = make_shape(N, S, C, G, V, w);
        int M;
        if (t.nsub > 1 || !small_threads(t, *V, &M)) break;
        s = t;
    }
    return s;
}

static size_t stats_bytes(const Shape& s) { return (size_t)s.N * s.nblk * s.nsub * s.G * sizeof(double2) + (size_t)s.N * s.G * sizeof(double); }

struct Plan {
    Shape shape;                        // of the sums, or of the one launch
    int V, M, threads;                  // threads > 0: the single launch
    size_t bytes;
};

static Plan plan_forward(int N, long S, int C, int G, int dtype) {
    Plan p = {};
    p.V = vector_width(C);
    p.shape = small_shape(N, S, C, G, &p.V);
    p.threads = p.shape.nsub > 1 ? 0 : small_threads(p.shape, p.V, &p.M);
    if (!p.threads) {
        p.V = vector_width(C);
        p.shape = make_shape(N, S, C, G, &p.V, 1l << 40);
        cut_rows(&p.shape, p.V, kStatsBlocks, tile_rows(p.V, element_bytes(dtype)), kStatsTiles);
        p.bytes = stats_bytes(p.shape);
    }
    return p;
}

template <class T, int V, int ACT>
static int forward_act(const Forward& f, const Plan& p, void* ws, double bytes) {
    const Shape& sh = p.shape;
    const double m = (double)sh.S * sh.cg;
    const T *x = (const T*)f.x, *res = (const T*)f.residual;
    const long grid = (long)sh.N * sh.nblk * sh.chunks;
    const size_t per_table = (sh.cg % V == 0 ? 1 : V) * sizeof(double2);
    if (p.threads) {
        Shape cut = sh;
        // Few long chunks: four workgroups a chunk read it and form its statistics, and each writes a quarter (6x17x30x128 in fp32: 8.9 us
        // for 10.5).  Not in place: one would write what another still reads.
        if (p.M == 16 && f.x != f.y && (long)sh.N * sh.chunks <= 64) cut.nblk = 4;
        const dim3 blocks((unsigned)((long)cut.N * cut.nblk * cut.chunks));
        const size_t lds = p.threads * per_table + sh.gpc * sizeof(double2);
        LaunchScope ls("group_norm_small", f.stream, 8.0 * sh.N * m * sh.G, bytes);
        if (p.M == 4)
            hipLaunchKernelGGL((group_norm_small<T, V, 4, ACT>), blocks, dim3(p.threads), lds, f.stream, x, f.xr, f.weight, f.bias,
                               res, f.rr, (T*)f.y, f.yr, f.stats, cut, 1. / m, f.eps, f.oflag);
        else
            hipLaunchKernelGGL((group_norm_small<T, V, 16, ACT>), blocks, dim3(p.threads), lds, f.stream, x, f.xr, f.weight, f.bias,
                               res, f.rr, (T*)f.y, f.yr, f.stats, cut, 1. / m, f.eps, f.oflag);
        return check_launch("msnet_group_norm");
    }
    double2* part = (double2*)ws;
    double* pivots = (double*)(part + (size_t)sh.N * sh.nblk * sh.nsub * sh.G);
    {
        LaunchScope ls("group_norm_stats", f.stream, 4.0 * sh.N * m * sh.G, (double)sh.N * m * sh.G * sizeof(T));
        hipLaunchKernelGGL((group_norm_stats<T, V>), dim3((unsigned)grid), dim3(kThreads), kThreads * per_table, f.stream, x, f.xr, sh, part, pivots);
        if (int rc = check_launch("msnet_group_norm")) return rc;
    }
    Shape out = sh;
    cut_rows(&out, V, kApplyBlocks, tile_rows(V, sizeof(T)), kApplyTiles);
    const long grid2 = (long)out.N * out.nblk * out.chunks;
    LaunchScope ls("group_norm_apply", f.stream, 4.0 * sh.N * m * sh.G, bytes);
    const auto apply = streams((double)sh.N * m * sh.G * sizeof(T), V * sizeof(T)) ? group_norm_apply<T, V, ACT, true> : group_norm_apply<T, V, ACT, false>;
    hipLaunchKernelGGL(apply, dim3((unsigned)grid2), dim3(kThreads), (kThreads + sh.gpc) * sizeof(double2), f.stream, x, f.xr, f.weight, f.bias, res,
                       f.rr, (T*)f.y, f.yr, f.stats, out, sh.nblk * sh.nsub, part, pivots, 1. / m, f.eps, f.oflag);
    return check_launch("msnet_group_norm");
}

template <class T, int V>
static int forward_v(const Forward& f, const Plan& p, int act, void* ws, double bytes) {
    return act == kRelu ? forward_act<T, V, kRelu>(f, p, ws, bytes) : act == kSilu ? forward_act<T, V, kSilu>(f, p, ws, bytes)
                                                                                   : forward_act<T, V, kNone>(f, p, ws, bytes);
}

template <class T>
static int forward_t(const Forward& f, const Plan& p, int act, void* ws, double bytes) {
    return p.V == 4 ? forward_v<T, 4>(f, p, act, ws, bytes) : p.V == 2 ? forward_v<T, 2>(f, p, act, ws, bytes) : forward_v<T, 1>(f, p, act, ws, bytes);
}

}  // namespace gn
}  // namespace msnet

using namespace msnet;

extern "C" size_t msnet_group_norm_workspace_bytes(int dtype, int N, long S, int C, int G) {
    if (gn::check_shape("msnet_group_norm_workspace_bytes", dtype, 0, N, S, C, G, 0.) || N == 0 || S == 0) return 0;
    return gn::plan_forward(N, S, C, G, dtype).bytes;
}

extern "C" int msnet_group_norm(const void* x, const float* weight, const float* bias, const void* residual, void* y, double* stats, int dtype,
                                int act, int N, long S, int C, int G, double eps, long x_sn, long x_ss, long r_sn, long r_ss, long y_sn, long y_ss,
                                void* workspace, size_t workspace_bytes, msnet_stream_t stream) {
    if (int rc = gn::check_shape("msnet_group_norm", dtype, act, N, S, C, G, eps)) return rc;
    if (N == 0 || S == 0) return 0;
    if (!x || !y) return fail("msnet_group_norm: null pointer");
    if (x_sn < 0 || x_ss < 0 || r_sn < 0 || r_ss < 0 || y_sn < 0 || y_ss < 0) return fail("msnet_group_norm: negative stride");
    if (((uintptr_t)stats | (uintptr_t)workspace) & 15) return fail("msnet_group_norm: stats and workspace must be 16-byte aligned");
    const gn::Plan p = gn::plan_forward(N, S, C, G, dtype);
    if (p.bytes && (!workspace || workspace_bytes < p.bytes))
        return fail("msnet_group_norm: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, p.bytes);
    // (a launch has at most 2^32 - 1 threads; row blocks are added only up to a few thousand workgroups in all)
    if (((double)N * p.shape.chunks + 4096) * (p.threads ? p.threads : gn::kThreads) > 4294967295.)
        return fail("msnet_group_norm: N=%d samples of %d channel chunks are too many for one launch", N, p.shape.chunks);
    const gn::Forward f = {x, residual, weight, bias, y, (double2*)stats, {x_sn, x_ss}, {r_sn, r_ss}, {y_sn, y_ss}, eps,
                           dtype == gn::kF32 ? overflow_flag() : nullptr, (hipStream_t)stream};
    const double bytes = (double)N * S * C * gn::element_bytes(dtype) * (residual ? 3 : 2);
    return dtype == gn::kF32 ? gn::forward_t<float>(f, p, act, workspace, bytes) : dtype == gn::kF16 ? gn::forward_t<_Float16>(f, p, act, workspace, bytes)
                                                                                                    : gn::forward_t<__bf16>(f, p, act, workspace, bytes);
}
