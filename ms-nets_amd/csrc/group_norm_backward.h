// Group norm with an activation, backward.  With dz = dy * act'(z), gz = gamma * dz and sums over the m values of a group:
//
//   dbeta_c = sum dz,   dgamma_c = sum dz * xhat          (over samples and rows)
//   c1 = (1/m) sum gz,  c2 = (1/m) sum gz * xhat
//   dx = (gz - c1 - xhat * c2) / sqrt(var + eps),   dresidual = dz
//
// xhat and z are computed again from x (and the residual) and the saved statistics; nothing but those is kept from the forward.
// As in the forward there are two ways: group_norm_grad_small holds a chunk of one sample in registers and reads x and dy once;
// group_norm_grad_sums leaves every row block's sums per channel and per group in the workspace and group_norm_grad_apply adds
// them up, its first workgroups for dgamma and dbeta.  Sums are 64-bit and added in a fixed order: a result repeats bit for bit.
//
// A ReLU's derivative jumps at z = 0.  z in 32 bits is off by at most 2^-22 (|beta + residual| + |what the mean's rounding left|)
// there; a vector with a value within four times that is decided in 64 bits (a few of a million are).
#pragma once
#include "group_norm.h"

namespace msnet {
namespace gn {

struct Backward {
    const void *dy, *x, *residual;
    const float *weight, *bias;
    const double2* stats;              // [N][G] mean, 1 / sqrt(var + eps)
    void *dx, *dresidual;
    float *dweight, *dbias;
    Rows yr, xr, rr;                   // of dy, x, residual; dx and dresidual are dense
    hipStream_t stream;
};

struct BackwardPlan {
    Shape shape;
    int V, M, threads;                 // threads > 0: the single launch
    size_t bytes;
};

BackwardPlan plan_backward(int N, long S, int C, int G, int dtype);
int backward_f32(const Backward& f, const BackwardPlan& p, int act, void* ws);
int backward_f16(const Backward& f, const BackwardPlan& p, int act, void* ws);
int backward_bf16(const Backward& f, const BackwardPlan& p, int act, void* ws);

// vectors of x and dy a thread of the single launch holds (1024 threads leave 128 registers each)
constexpr int kGradFew = 2;
constexpr int grad_many(int V, int bytes) { return V * bytes == 16 ? 4 : 8; }
constexpr int kGradTable = 2048;       // sums of the single launch's threads at a time: 32 KB
constexpr int kParamCols = 16;         // channels of one workgroup that sums dgamma and dbeta
constexpr long kGradApplyBlocks = 512;
constexpr long kGradSumBlocks = 768;   // three of these fit a compute unit's registers
constexpr int kSumTile = 4;            // rows a thread of the sums loads at once (the sums of eight do not fit beside them)
constexpr int kGradSumTiles = 2, kGradApplyTiles = 2;  // tiles of a workgroup at least

// What a thread keeps of its V channels.  WHOLE: they lie in one group, whose constants are kept once.
template <int V, bool WHOLE>
struct Channels {
    static constexpr int W = WHOLE ? 1 : V;
    float mean[W], rstd[W], lo[W], gamma[V], beta[V];
    __device__ __forceinline__ void load(int c, const float* weight, const float* bias) {
        load_params<V>(weight, c, true, gamma);
        load_params<V>(bias, c, false, beta);
    }
    __device__ __forceinline__ void set(const double2* st, int c_local, int cg) {
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const double2 t = st[(c_local + e) / cg];
            mean[e] = (float)t.x;
            rstd[e] = (float)t.y;
            lo[e] = (float)(((double)mean[e] - t.x) * t.y);
        }
    }
};

// dz and xhat of one row's V values.
template <class T, int V, bool WHOLE, int ACT, bool RES>
__device__ __forceinline__ void derive(const Channels<V, WHOLE>& k, const double2* st, int c_local, int cg, const typename Pack<T, V>::type& x,
                                       const typename Pack<T, V>::type& dy, const typename Pack<T, V>::type& res, float (&dz)[V], float (&xhat)[V]) {
    float z[V];
    bool near = false;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int g = WHOLE ? 0 : e;
        xhat[e] = fmaf(element<T, V>(x, e) - k.mean[g], k.rstd[g], k.lo[g]);
        if constexpr (ACT != kNone) {
            const float b = RES ? k.beta[e] + element<T, V>(res, e) : k.beta[e];
            z[e] = fmaf(xhat[e], k.gamma[e], b);
            // (gamma = 0: z is exact, and often 0)
            if constexpr (ACT == kRelu) near |= fabsf(z[e]) <= 0x1p-20f * (fabsf(b) + fabsf(k.lo[g] * k.gamma[e])) && k.gamma[e] != 0.f;
        }
    }
    if constexpr (ACT == kRelu)
        if (near)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                int c = c_local + e;                       // opaque to the compiler, and behind the element before: it would form
                float g = k.gamma[e], b = k.beta[e];       // these doubles outside the loop over the rows and all V at once, for
                asm volatile("" : "+v"(c), "+v"(g), "+v"(b), "+v"(z[e ? e - 1 : 0]));      // a branch hardly any row takes
                const double2 t = st[c / cg];
                double d = ((double)element<T, V>(x, e) - t.x) * t.y * (double)g + (double)b;
                if constexpr (RES) d += (double)element<T, V>(res, e);
                z[e] = d <= 0. ? 0.f : 1.f;
            }
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float g = element<T, V>(dy, e);
        if constexpr (ACT == kRelu) dz[e] = z[e] <= 0.f ? 0.f : g;       // (a NaN passed the forward, and its gradient passes too)
        else if constexpr (ACT == kSilu) {
            const float sig = silu_gate(z[e]);
            dz[e] = g * (sig * fmaf(z[e], 1.f - sig, 1.f));
        } else dz[e] = g;
    }
}

template <int V, bool WHOLE>
__device__ __forceinline__ void grad_input(const Channels<V, WHOLE>& k, const float (&c1)[WHOLE ? 1 : V], const float (&c2)[WHOLE ? 1 : V],
                                           const float (&dz)[V], const float (&xhat)[V], float (&dx)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float gz = k.gamma[e] * dz[e];       // (rounded before the subtraction: a group of one value has gz = c1 and dx = 0)
        const int g = WHOLE ? 0 : e;
        dx[e] = (__fsub_rn(gz, c1[g]) - xhat[e] * c2[g]) * k.rstd[g];
    }
}

// dgamma and dbeta of kParamCols channels from chan[rows][C].
__device__ __forceinline__ void param_grads(const double2* __restrict__ chan, long rows, int C, int block, float* dweight, float* dbias, double2* tab) {
    const int tid = threadIdx.x, col = tid % kParamCols, lane = tid / kParamCols, c = block * kParamCols + col;
    double2 s = make_double2(0., 0.);
    if (c < C)
#pragma unroll 4
        for (long i = lane; i < rows; i += kThreads / kParamCols) s = s + chan[(size_t)i * C + c];
    tab[tid] = s;
    sum_rows(tab, kThreads / kParamCols, kParamCols, tid, kThreads);
    if (tid < kParamCols && c < C) {
        if (dbias) dbias[c] = (float)tab[tid].x;
        if (dweight) dweight[c] = (float)tab[tid].y;
    }
}

template <int UNUSED>
__global__ __launch_bounds__(kThreads) void group_norm_param_grads(const double2* __restrict__ chan, long rows, int C, float* dweight, float* dbias) {
    __shared__ double2 tab[kThreads];
    param_grads(chan, rows, C, blockIdx.x, dweight, dbias, tab);
}

// What a thread reads: x, dy and the residual at its channels of a sample; one row or a tile of them.
template <class T, int V, bool RES>
struct Inputs {
    const T *x, *dy, *r;
    long xs, ys, rs;
    __device__ __forceinline__ Inputs(const T* x_, Rows xr, const T* dy_, Rows yr, const T* r_, Rows rr, int n, int c)
        : x(x_ + (size_t)n * xr.sn + c), dy(dy_ + (size_t)n * yr.sn + c), r(RES ? r_ + (size_t)n * rr.sn + c : x), xs(xr.ss), ys(yr.ss), rs(RES ? rr.ss : xr.ss) {}
    template <class F>
    __device__ __forceinline__ void row(long at, F f) const {
        f(at, load_raw<T, V>(x + (size_t)at * xs), load_raw<T, V>(dy + (size_t)at * ys), load_raw<T, V>(r + (size_t)at * rs));
    }
    template <int U, bool STREAM, class F>
    __device__ __forceinline__ void tile(long at, int step, F f) const {
        Tile<T, V, U, STREAM> tx, td, tr;
        tx.load(x, at, step, xs);
        td.load(dy, at, step, ys);
        if constexpr (RES) tr.load(r, at, step, rs);
        else tr = tx;
        loads_issued();
#pragma unroll
        for (int u = 0; u < U; ++u) f(at + (long)u * step, tx.v[u], td.v[u], tr.v[u]);
    }
};

template <class T, int V, bool WHOLE, int ACT, bool RES>
__global__ __launch_bounds__(kThreads) void group_norm_grad_sums(const T* __restrict__ dy, Rows yr, const T* __restrict__ x, Rows xr,
                                                                 const T* __restrict__ residual, Rows rr, const float* __restrict__ weight,
                                                                 const float* __restrict__ bias, const double2* __restrict__ stats, Shape sh,
                                                                 double2* __restrict__ part, double2* __restrict__ chan) {
    extern __shared__ __attribute__((aligned(16))) double2 tab[];      // [kThreads * V] sums, [ng] statistics
    double2* st = tab + kThreads * V;
    const Chunk k = chunk_of(sh, blockIdx.x);
    const int tid = threadIdx.x, cv = k.cw / V, per_pass = kThreads / cv;
    const int row = tid / cv, cl = (tid % cv) * V, cg = k.ng > 1 ? sh.cg : k.cw;
    const bool on = row < per_pass;
    for (int g = tid; g < k.ng; g += kThreads) st[g] = stats[(size_t)k.n * sh.G + k.g0 + g];
    Channels<V, WHOLE> a;
    a.load(k.c0 + cl, weight, bias);
    __syncthreads();
    a.set(st, cl, cg);
    double s[V], q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = q[e] = 0.;
    const auto add = [&](long, const typename Pack<T, V>::type& vx, const typename Pack<T, V>::type& vd, const typename Pack<T, V>::type& vr) {
        float dz[V], xhat[V];
        derive<T, V, WHOLE, ACT, RES>(a, st, cl, cg, vx, vd, vr, dz, xhat);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            s[e] += (double)dz[e];
            q[e] = fma((double)dz[e], (double)xhat[e], q[e]);
        }
    };
    const Inputs<T, V, RES> in(x, xr, dy, yr, residual, rr, k.n, k.c0 + cl);
    Walk<kSumTile, false>(sh, k.blk, row, per_pass, on).run([&](long r) { in.template tile<kSumTile, false>(r, per_pass, add); }, [&](long r) { in.row(r, add); });
    double2 v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = make_double2(s[e], q[e]);
    sum_threads<V>(v, tab, cv, on, tid, kThreads);
    double2* mine = chan + ((size_t)k.n * sh.nblk + k.blk) * sh.C + k.c0;
    for (int c = tid; c < k.cw; c += kThreads) mine[c] = tab[c];
    const size_t slot = (size_t)k.n * sh.nblk * sh.nsub + (size_t)k.blk * sh.nsub + k.sub;
    sum_groups(tab, k.cw / k.ng, k.ng, tid, kThreads,
               [&](int c, double2 u) { const double g = weight ? (double)weight[k.c0 + c] : 1.; return make_double2(g * u.x, g * u.y); },
               [&](int g, double2 u) { part[slot * sh.G + k.g0 + g] = u; });
}

// STREAM: the gradients go past the caches, and so do the inputs, read for the last time.
template <class T, int V, bool WHOLE, int ACT, bool RES, bool STREAM>
__global__ __launch_bounds__(kThreads) void group_norm_grad_apply(const T* __restrict__ dy, Rows yr, const T* __restrict__ x, Rows xr,
                                                                  const T* __restrict__ residual, Rows rr, const float* __restrict__ weight,
                                                                  const float* __restrict__ bias, const double2* __restrict__ stats, T* __restrict__ dx,
                                                                  T* __restrict__ dresidual, float* dweight, float* dbias, Shape sh, int slots,
                                                                  const double2* __restrict__ part, const double2* __restrict__ chan, long chan_rows,
                                                                  int param_blocks, double inv) {
    extern __shared__ __attribute__((aligned(16))) double2 tab[];      // [kThreads] sums, [ng] statistics, [ng] c1 and c2
    if ((int)blockIdx.x < param_blocks) {
        param_grads(chan, chan_rows, sh.C, blockIdx.x, dweight, dbias, tab);
        return;
    }
    const Chunk k = chunk_of(sh, blockIdx.x - param_blocks);
    double2 *st = tab + kThreads, *coef = st + k.ng;
    const int tid = threadIdx.x, cv = k.cw / V, per_pass = kThreads / cv;
    const int row = tid / cv, cl = (tid % cv) * V, cg = k.ng > 1 ? sh.cg : k.cw;
    Channels<V, WHOLE> a;
    a.load(k.c0 + cl, weight, bias);
    const double2* mine = stats + (size_t)k.n * sh.G + k.g0;
    const double2 first = mine[min(tid, k.ng - 1)];        // of the group whose sums this thread will have (of the first kThreads groups)
    sum_slots(part + (size_t)k.n * slots * sh.G, slots, sh.G, k.g0, k.ng, tab, tid, [&](int g, double2 sum) {
        coef[g] = make_double2(sum.x * inv, sum.y * inv);
        st[g] = g < kThreads ? first : mine[g];
    });
    a.set(st, cl, cg);
    float c1[WHOLE ? 1 : V], c2[WHOLE ? 1 : V];
#pragma unroll
    for (int e = 0; e < (WHOLE ? 1 : V); ++e) { c1[e] = (float)coef[(cl + e) / cg].x; c2[e] = (float)coef[(cl + e) / cg].y; }
    const size_t dense = (size_t)k.n * sh.S * sh.C + k.c0 + cl;
    const auto put = [&](long r, const typename Pack<T, V>::type& vx, const typename Pack<T, V>::type& vd, const typename Pack<T, V>::type& vr) {
        float dz[V], xhat[V], o[V];
        derive<T, V, WHOLE, ACT, RES>(a, st, cl, cg, vx, vd, vr, dz, xhat);
        grad_input<V, WHOLE>(a, c1, c2, dz, xhat, o);
        if (dx) store<T, V, STREAM>(dx + dense + (size_t)r * sh.C, o);
        if (RES && dresidual) store<T, V, STREAM>(dresidual + dense + (size_t)r * sh.C, dz);
    };
    const Inputs<T, V, RES> in(x, xr, dy, yr, residual, rr, k.n, k.c0 + cl);
    constexpr int kTile = tile_rows(V, sizeof(T));
    Walk<kTile, true>(sh, k.blk, row, per_pass, row < per_pass).run(             // last rows first, as in the forward
        [&](long r) { in.template tile<kTile, STREAM>(r, per_pass, put); }, [&](long r) { in.row(r, put); });
}

// All rows of one chunk of one sample in registers, M vectors of x and of dy a thread.  direct: one sample, its channel sums are
// dgamma and dbeta; else they go to chan[N][C].
template <class T, int V, bool WHOLE, int M, int ACT, bool RES>
__global__ __launch_bounds__(1024) void group_norm_grad_small(const T* __restrict__ dy, Rows yr, const T* __restrict__ x, Rows xr,
                                                              const T* __restrict__ residual, Rows rr, const float* __restrict__ weight,
                                                              const float* __restrict__ bias, const double2* __restrict__ stats, T* __restrict__ dx,
                                                              T* __restrict__ dresidual, float* dweight, float* dbias, Shape sh,
                                                              double2* __restrict__ chan, bool direct, double inv) {
    extern __shared__ __attribute__((aligned(16))) double2 tab[];      // [kGradTable] sums, [cw] of the channels, [ng] statistics, [ng] c1 and c2
    const Chunk k = chunk_of(sh, blockIdx.x);
    double2 *st = tab + kGradTable + k.cw, *coef = st + k.ng;
    const int tid = threadIdx.x, threads = blockDim.x, cv = k.cw / V, per_pass = threads / cv;
    const int row = tid / cv, cl = (tid % cv) * V, cg = sh.cg;
    const int S = (int)sh.S;
    const T* px = x + (size_t)k.n * xr.sn + k.c0 + cl;
    const T* pd = dy + (size_t)k.n * yr.sn + k.c0 + cl;
    const T* pr = RES ? residual + (size_t)k.n * rr.sn + k.c0 + cl : px;
    typename Pack<T, V>::type vx[M], vd[M], vr[M];
    const bool on = row < per_pass;
    if (on) {
#pragma unroll
        for (int i = 0; i < M; ++i)
            if (row + i * per_pass < S) {
                vx[i] = load_raw<T, V>(px + (size_t)(row + i * per_pass) * xr.ss);
                vd[i] = load_raw<T, V>(pd + (size_t)(row + i * per_pass) * yr.ss);
                if constexpr (RES) vr[i] = load_raw<T, V>(pr + (size_t)(row + i * per_pass) * rr.ss);
            }
    }
    Channels<V, WHOLE> a;
    a.load(k.c0 + cl, weight, bias);
    loads_issued();
    for (int g = tid; g < k.ng; g += threads) st[g] = stats[(size_t)k.n * sh.G + k.g0 + g];
    __syncthreads();
    a.set(st, cl, cg);
    double2 v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = make_double2(0., 0.);
#pragma unroll
    for (int i = 0; i < M; ++i)
        if (on && row + i * per_pass < S) {
            float dz[V], xhat[V];
            derive<T, V, WHOLE, ACT, RES>(a, st, cl, cg, vx[i], vd[i], RES ? vr[i] : vx[i], dz, xhat);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[e].x += (double)dz[e];
                v[e].y = fma((double)dz[e], (double)xhat[e], v[e].y);
            }
        }
    double2* sums = tab;                                   // of the channels
    if (threads * V <= kGradTable || (in_wave(cv) && (threads >> 6) * k.cw <= kGradTable)) {
        sum_threads<V>(v, tab, cv, on, tid, threads);
    } else {                                               // an element of all vectors at a time, each round's sums put behind the table
        sums = tab + kGradTable;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            double2 u[1] = {v[e]};
            sum_threads<1>(u, tab, cv, on, tid, threads);
            for (int i = tid; i < cv; i += threads) sums[i * V + e] = tab[i];
            __syncthreads();
        }
    }
    for (int c = tid; c < k.cw; c += threads) {
        if (direct) {
            if (dbias) dbias[k.c0 + c] = (float)sums[c].x;
            if (dweight) dweight[k.c0 + c] = (float)sums[c].y;
        } else if (chan) chan[(size_t)k.n * sh.C + k.c0 + c] = sums[c];
    }
    sum_groups(sums, cg, k.ng, tid, threads,
               [&](int c, double2 u) { const double g = weight ? (double)weight[k.c0 + c] : 1.; return make_double2(g * u.x, g * u.y); },
               [&](int g, double2 u) { coef[g] = make_double2(u.x * inv, u.y * inv); });
    __syncthreads();
    if (!on) return;
    float c1[WHOLE ? 1 : V], c2[WHOLE ? 1 : V];
#pragma unroll
    for (int e = 0; e < (WHOLE ? 1 : V); ++e) { c1[e] = (float)coef[(cl + e) / cg].x; c2[e] = (float)coef[(cl + e) / cg].y; }
    const size_t dense = (size_t)k.n * sh.S * sh.C + k.c0 + cl;
#pragma unroll
    for (int i = 0; i < M; ++i) {
        const int r = row + i * per_pass;
        if (r < S) {
            float dz[V], xhat[V], o[V];
            derive<T, V, WHOLE, ACT, RES>(a, st, cl, cg, vx[i], vd[i], RES ? vr[i] : vx[i], dz, xhat);
            grad_input<V, WHOLE>(a, c1, c2, dz, xhat, o);
            if (dx) store<T, V>(dx + dense + (size_t)r * sh.C, o);
            if (RES && dresidual) store<T, V>(dresidual + dense + (size_t)r * sh.C, dz);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------

template <class T, int V, bool WHOLE, int ACT, bool RES>
static int backward_act(const Backward& f, const BackwardPlan& p, void* ws) {
    const Shape& sh = p.shape;
    const double m = (double)sh.S * sh.cg, values = m * sh.N * sh.G;
    const T *dy = (const T*)f.dy, *x = (const T*)f.x, *res = (const T*)f.residual;
    T *dx = (T*)f.dx, *dres = (T*)f.dresidual;
    const bool params = f.dweight || f.dbias;
    // (a multiple of the eight dies, so that a row's workgroup stays on the die whose cache its sums were read into)
    const unsigned param_blocks = params ? (unsigned)((sh.C + kParamCols - 1) / kParamCols + 7) / 8 * 8 : 0;
    const unsigned grid = (unsigned)((long)sh.N * sh.nblk * sh.chunks);
    if (p.threads) {
        const bool direct = sh.N == 1;
        double2* chan = direct || !params ? nullptr : (double2*)ws;
        const size_t lds = (kGradTable + sh.cw + 2 * sh.gpc) * sizeof(double2);
        {
            LaunchScope ls("group_norm_grad_small", f.stream, 16.0 * values, values * sizeof(T) * (RES ? 5 : 3));
            if (p.M == kGradFew)
                hipLaunchKernelGGL((group_norm_grad_small<T, V, WHOLE, kGradFew, ACT, RES>), dim3(grid), dim3(p.threads), lds, f.stream, dy, f.yr, x, f.xr, res, f.rr,
                                   f.weight, f.bias, f.stats, dx, dres, f.dweight, f.dbias, sh, chan, direct, 1. / m);
            else
                hipLaunchKernelGGL((group_norm_grad_small<T, V, WHOLE, grad_many(V, sizeof(T)), ACT, RES>), dim3(grid), dim3(p.threads), lds, f.stream, dy, f.yr, x, f.xr, res, f.rr,
                                   f.weight, f.bias, f.stats, dx, dres, f.dweight, f.dbias, sh, chan, direct, 1. / m);
            if (int rc = check_launch("msnet_group_norm_backward")) return rc;
        }
        if (!chan) return 0;
        LaunchScope ls("group_norm_param_grads", f.stream, 0, 16.0 * sh.N * sh.C);
        hipLaunchKernelGGL(group_norm_param_grads<0>, dim3(param_blocks), dim3(kThreads), 0, f.stream, chan, (long)sh.N, sh.C, f.dweight, f.dbias);
        return check_launch("msnet_group_norm_backward");
    }
    double2* part = (double2*)ws;
    double2* chan = part + (size_t)sh.N * sh.nblk * sh.nsub * sh.G;
    {
        LaunchScope ls("group_norm_grad_sums", f.stream, 8.0 * values, values * sizeof(T) * (RES ? 3 : 2));
        hipLaunchKernelGGL((group_norm_grad_sums<T, V, WHOLE, ACT, RES>), dim3(grid), dim3(kThreads), (kThreads * V + sh.gpc) * sizeof(double2), f.stream, dy,
                           f.yr, x, f.xr, res, f.rr, f.weight, f.bias, f.stats, sh, part, chan);
        if (int rc = check_launch("msnet_group_norm_backward")) return rc;
    }
    if (!dx && !dres) {                                    // the parameters' gradients alone
        LaunchScope ls("group_norm_param_grads", f.stream, 0, 16.0 * sh.N * sh.nblk * sh.C);
        hipLaunchKernelGGL(group_norm_param_grads<0>, dim3(param_blocks), dim3(kThreads), 0, f.stream, chan, (long)sh.N * sh.nblk, sh.C, f.dweight, f.dbias);
        return check_launch("msnet_group_norm_backward");
    }
    Shape out = sh;
    cut_rows(&out, V, kGradApplyBlocks, tile_rows(V, sizeof(T)), kGradApplyTiles);
    const unsigned grid2 = (unsigned)((long)out.N * out.nblk * out.chunks) + param_blocks;
    LaunchScope ls("group_norm_grad_apply", f.stream, 8.0 * values, values * sizeof(T) * (RES ? 5 : 3));
    const auto apply = streams(values * sizeof(T), V * sizeof(T)) ? group_norm_grad_apply<T, V, WHOLE, ACT, RES, true> : group_norm_grad_apply<T, V, WHOLE, ACT, RES, false>;
    hipLaunchKernelGGL(apply, dim3(grid2), dim3(kThreads), (kThreads + 2 * sh.gpc) * sizeof(double2), f.stream, dy, f.yr, x, f.xr, res, f.rr, f.weight,
                       f.bias, f.stats, dx, dres, f.dweight, f.dbias, out, sh.nblk * sh.nsub, part, chan, (long)sh.N * sh.nblk, (int)param_blocks, 1. / m);
    return check_launch("msnet_group_norm_backward");
}

template <class T, int V, bool WHOLE>
static int backward_w(const Backward& f, const BackwardPlan& p, int act, void* ws) {
    if (act == kRelu) return f.residual ? backward_act<T, V, WHOLE, kRelu, true>(f, p, ws) : backward_act<T, V, WHOLE, kRelu, false>(f, p, ws);
    if (act == kSilu) return f.residual ? backward_act<T, V, WHOLE, kSilu, true>(f, p, ws) : backward_act<T, V, WHOLE, kSilu, false>(f, p, ws);
    return backward_act<T, V, WHOLE, kNone, false>(f, p, ws);        // the residual's gradient is dy itself
}

template <class T, int V>
static int backward_v(const Backward& f, const BackwardPlan& p, int act, void* ws) {
    return p.shape.cg % V == 0 ? backward_w<T, V, true>(f, p, act, ws) : backward_w<T, V, false>(f, p, act, ws);
}

template <class T>
static int backward_t(const Backward& f, const BackwardPlan& p, int act, void* ws) {
    return p.V == 4 ? backward_v<T, 4>(f, p, act, ws) : p.V == 2 ? backward_v<T, 2>(f, p, act, ws) : backward_w<T, 1, true>(f, p, act, ws);
}

}  // namespace gn
}  // namespace msnet
