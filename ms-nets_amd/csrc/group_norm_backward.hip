// Group norm backward: the C entry and the float32 kernels (group_norm_backward.h).
#include "group_norm_backward.h"

namespace msnet {
namespace gn {

int backward_f32(const Backward& f, const BackwardPlan& p, int act, void* ws) { return backward_t<float>(f, p, act, ws); }

static int grad_small_threads(const Shape& s, int V, int dtype, int* M) {
    const int cv = s.cw / V;
    if ((kGradTable + s.cw + 2 * s.gpc) * sizeof(double2) > 65536) return 0;
    for (int m : {kGradFew, grad_many(V, element_bytes(dtype))})
        for (int t = 256; t <= 1024; t <<= 1)
            if (s.S <= (long)m * (t / cv)) { *M = m; return t; }
    return 0;
}

BackwardPlan plan_backward(int N, long S, int C, int G, int dtype) {
    BackwardPlan p = {};
    long w = 8;                                            // as in the forward: narrow chunks, wider ones once workgroups abound
    p.V = vector_width(C);
    p.shape = make_shape(N, S, C, G, &p.V, w);
    while ((long)N * p.shape.chunks > 2048 && w < (long)kThreads * p.V) {
        w *= 2;
        int M;
        const Shape t = make_shape(N, S, C, G, &p.V, w);
        if (t.nsub > 1 || !grad_small_threads(t, p.V, dtype, &M)) break;
        p.shape = t;
    }
    p.threads = p.shape.nsub > 1 ? 0 : grad_small_threads(p.shape, p.V, dtype, &p.M);
    if (p.threads) {
        p.bytes = N > 1 ? (size_t)N * C * sizeof(double2) : 0;
    } else {
        p.V = vector_width(C);
        p.shape = make_shape(N, S, C, G, &p.V, (long)kThreads * p.V / 2);
        cut_rows(&p.shape, p.V, kGradSumBlocks, kSumTile, kGradSumTiles);
        p.bytes = ((size_t)N * p.shape.nblk * p.shape.nsub * G + (size_t)N * p.shape.nblk * C) * sizeof(double2);
    }
    return p;
}

}  // namespace gn
}  // namespace msnet

using namespace msnet;

extern "C" size_t msnet_group_norm_backward_workspace_bytes(int dtype, int N, long S, int C, int G) {
    if (gn::check_shape("msnet_group_norm_backward_workspace_bytes", dtype, 0, N, S, C, G, 0.) || N == 0 || S == 0) return 0;
    return gn::plan_backward(N, S, C, G, dtype).bytes;
}

extern "C" int msnet_group_norm_backward(const void* dy, const void* x, const float* weight, const float* bias, const void* residual,
                                         const double* stats, void* dx, void* dresidual, float* dweight, float* dbias, int dtype, int act, int N, long S,
                                         int C, int G, long dy_sn, long dy_ss, long x_sn, long x_ss, long r_sn, long r_ss, void* workspace,
                                         size_t workspace_bytes, msnet_stream_t stream) {
    if (int rc = gn::check_shape("msnet_group_norm_backward", dtype, act, N, S, C, G, 0.)) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (!dx && !dresidual && !dweight && !dbias) return 0;
    if (N == 0 || S == 0) {                                // no rows: the parameters' gradients are zero
        if (!dweight && !dbias) return 0;
        LaunchScope ls("group_norm_param_grads", s, 0, 8.0 * C);
        hipLaunchKernelGGL(gn::group_norm_param_grads<0>, dim3((C + gn::kParamCols - 1) / gn::kParamCols), dim3(gn::kThreads), 0, s,
                           (const double2*)nullptr, 0l, C, dweight, dbias);
        return check_launch("msnet_group_norm_backward");
    }
    if (!dy || !x || !stats) return fail("msnet_group_norm_backward: null pointer");
    if (dresidual && !residual) return fail("msnet_group_norm_backward: a residual's gradient needs the residual");
    if (dresidual && act == gn::kNone) return fail("msnet_group_norm_backward: without an activation the residual's gradient is dy itself");
    if (dy_sn < 0 || dy_ss < 0 || x_sn < 0 || x_ss < 0 || r_sn < 0 || r_ss < 0) return fail("msnet_group_norm_backward: negative stride");
    if (((uintptr_t)stats | (uintptr_t)workspace) & 15) return fail("msnet_group_norm_backward: stats and workspace must be 16-byte aligned");
    const gn::BackwardPlan p = gn::plan_backward(N, S, C, G, dtype);
    if (p.bytes && (!workspace || workspace_bytes < p.bytes))
        return fail("msnet_group_norm_backward: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, p.bytes);
    // (a launch has at most 2^32 - 1 threads; row blocks are added only up to a few thousand workgroups in all)
    if (((double)N * p.shape.chunks + C + 4096) * (p.threads ? p.threads : gn::kThreads) > 4294967295.)
        return fail("msnet_group_norm_backward: N=%d samples of %d channel chunks are too many for one launch", N, p.shape.chunks);
    const gn::Backward f = {dy, x, residual, weight, bias, (const double2*)stats, dx, dresidual, dweight, dbias,
                            {dy_sn, dy_ss}, {x_sn, x_ss}, {r_sn, r_ss}, s};
    return dtype == gn::kF32 ? gn::backward_f32(f, p, act, workspace) : dtype == gn::kF16 ? gn::backward_f16(f, p, act, workspace)
                                                                                         : gn::backward_bf16(f, p, act, workspace);
}
