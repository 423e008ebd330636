"""hipops.group_norm, grad_norm and clip_grads on the GPU at values, views and calls off the ordinary path: each is answered as the
definition has it, or refused."""
import pytest
import torch

import msnets_amd  # noqa: F401
from msnets_amd import hipops
from norm_clip_reference import U, norm64, within

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAN, INF = float("nan"), float("inf")


def make(shape, dtype, residual, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)              # noqa: E731
    c = shape[-1]
    x = (rnd(*shape) * (0.5 + torch.rand(c, device="cuda", generator=g)) + rnd(c)).to(dtype)
    return x, 1 + 0.3 * rnd(c), 0.3 * rnd(c), rnd(*shape).clamp_min(0).to(dtype) if residual else None, rnd(*shape).to(dtype)


def gradients(x, groups, w, b, r, dy, act):
    leaves = {k: t.detach().clone().requires_grad_() for k, t in zip(("x", "weight", "bias", "residual"), (x, w, b, r)) if t is not None}
    y = hipops.group_norm(leaves["x"], groups, leaves["weight"], leaves["bias"], act=act, residual=leaves.get("residual"))
    return {"d" + k: v for k, v in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy))}


# ---- what is not finite, backward: in one launch and in two ---------------------------------------------------------------

BOTH_WAYS = [(2, 60, 16), (2, 30000, 16)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape", BOTH_WAYS)
def test_relu_gradient_at_nonfinite_residuals(gpu, shape, dtype):
    """A NaN passes the ReLU and so does its gradient; +inf passes it, -inf does not.  All gradients stay finite: they are those of
    a residual with +1000 and -1000 in these places."""
    x, w, b, r, dy = make(shape, dtype, True)
    r[1, 7, 5], r[0, 0, 1], r[1, 8, 5], r[0, 3, 2] = NAN, NAN, INF, -INF
    want = norm64(x, 4, w, b, 1e-5, "relu", r.nan_to_num(nan=1000.0, posinf=1000.0, neginf=-1000.0), dy)
    for k, v in gradients(x, 4, w, b, r, dy, "relu").items():
        within(v, want[k], k)


@pytest.mark.parametrize("where", [0, 7])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("shape", BOTH_WAYS)
def test_relu_gradient_of_a_nonfinite_group(gpu, shape, bad, where):
    """Something in x that is not finite makes xhat a NaN in its whole group: dy passes there (dresidual, dbias), dx and dgamma are
    NaN, and nothing else changes."""
    x, w, b, r, dy = make(shape, F32, True)
    lifted = r.clone()
    lifted[1, :, 4:8] = 1000.0                 # a group that passes everywhere, for dresidual and dbias
    want, ordinary = norm64(x, 4, w, b, 1e-5, "relu", lifted, dy), norm64(x, 4, w, b, 1e-5, "relu", r, dy)
    x[1, where, 5] = bad
    got = gradients(x, 4, w, b, r, dy, "relu")
    within(got["dresidual"], want["dresidual"], "dresidual")
    within(got["dbias"], want["dbias"], "dbias")
    assert torch.isnan(got["dx"][1, :, 4:8]).all() and torch.isnan(got["dweight"][4:8]).all()
    rest = torch.ones(16, dtype=torch.bool, device="cuda")
    rest[4:8] = False
    within(got["dweight"][rest], tuple(t[rest] for t in ordinary["dweight"]), "dweight")
    for at in ((0,), (1, slice(None), rest)):
        within(got["dx"][at], tuple(t[at] for t in ordinary["dx"]), "dx")


@pytest.mark.parametrize("act", ["relu", "silu"])
@pytest.mark.parametrize("shape", BOTH_WAYS)
def test_nonfinite_incoming_gradient(gpu, shape, act):
    """In dy: its own value in dresidual, its channel's parameters and its group's dx; with a ReLU only where that passes."""
    x, w, b, r, dy = make(shape, F32, True)
    z = norm64(x, 4, w, b, 1e-5, "none", r)["y"][0]
    on = int((z[1, :, 5] > 0.1).nonzero()[0])
    off = int((z[1, :, 9] < -0.1).nonzero()[0])
    want = norm64(x, 4, w, b, 1e-5, act, r, dy)
    clean = dy.clone()
    clean[1, off, 9] = 0
    blocked = norm64(x, 4, w, b, 1e-5, act, r, clean)
    dy[1, on, 5], dy[1, off, 9] = NAN, (INF if act == "relu" else dy[1, off, 9])
    got = gradients(x, 4, w, b, r, dy, act)
    assert torch.isnan(got["dresidual"][1, on, 5]) and torch.isnan(got["dweight"][5]) and torch.isnan(got["dbias"][5])
    assert torch.isnan(got["dx"][1, :, 4:8]).all()
    ref = blocked if act == "relu" else want
    rest = torch.ones(16, dtype=torch.bool, device="cuda")
    rest[4:8] = False
    for k in ("dweight", "dbias"):
        within(got[k][rest], tuple(t[rest] for t in ref[k]), k)
    for k in ("dx", "dresidual"):
        within(got[k][..., rest], tuple(t[..., rest] for t in ref[k]), k)
        within(got[k][0], tuple(t[0] for t in ref[k]), k)


@pytest.mark.parametrize("shape", BOTH_WAYS)
def test_silu_of_a_nan(gpu, shape):
    """SiLU has no side for a NaN to pass on: everything it reaches is one."""
    x, w, b, r, dy = make(shape, F32, True)
    want = norm64(x, 4, w, b, 1e-5, "silu", r, dy)
    r[1, 7, 5] = NAN
    got = gradients(x, 4, w, b, r, dy, "silu")
    assert torch.isnan(got["dresidual"][1, 7, 5]) and torch.isnan(got["dx"][1, :, 4:8]).all()
    within(got["dx"][0], tuple(t[0] for t in want["dx"]), "dx")
    within(got["dbias"][:4], tuple(t[:4] for t in want["dbias"]), "dbias")


# ---- clipping: gradients at the ends of their types' range -----------------------------------------------------------------

@pytest.mark.parametrize("max_norm", [1e3, 1e-3, 1e-30])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_factors_below_float32s_normal_range(gpu, dtype, max_norm):
    """Gradients near the largest float: max_norm / norm is next to 2^-126 (1e3) or below it, where a float32 has fewer bits the smaller
    it is.  The factor and the products round by half a step each, as for any other factor; results below 2^-126 by half of the last step more."""
    values = [1e38, -3e38, 2.5e37, 1e30, -1e20, 1.0, 1e-20, 0.0]
    t = torch.tensor(values * 4000, device="cuda").to(dtype)
    short = t[:13].clone()
    norm = (t.double().square().sum() + short.double().square().sum()).sqrt()
    assert float(norm) > torch.finfo(F32).max
    before = [t.clone(), short.clone()]
    out = [torch.empty_like(t, dtype=F32), torch.empty_like(short, dtype=F32)]
    assert float(hipops.clip_grads([t, short], max_norm, out=out)) == INF
    hipops.clip_grads([t, short], max_norm)
    for got in (out, [t, short]):
        for v, o in zip(before, got):
            want = v.double() * (max_norm / (float(norm) + 1e-6))
            allowed = 2.1 * U * want.abs() + torch.finfo(o.dtype).eps / 2 * want.abs() * (1 + 3 * U) + 2.0 ** -149 + (2.0 ** -134 if o.dtype == BF16 else 0)
            assert bool(((o.double() - want).abs() <= allowed).all())


# ---- negated views: what .conj().imag of a complex tensor is -----------------------------------------------------------------

def negated(t):
    """t's values as a view whose memory holds their negatives, laid out as t is."""
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


def test_group_norm_of_negated_views(gpu):
    x, w, b, r, dy = make((2, 50, 16), F32, True)
    want = gradients(x, 4, w, b, r, dy, "silu")
    y = hipops.group_norm(x, 4, w, b, act="silu", residual=r)
    for i in range(4):
        args = [negated(t) if k == i else t for k, t in enumerate((x, w, b, r))]
        assert torch.equal(hipops.group_norm(args[0], 4, args[1], args[2], act="silu", residual=args[3]), y), i
        assert torch.equal(hipops.group_norm(args[0], 4, args[1], args[2], act="silu", residual=args[3], out=torch.empty_like(x)), y), i
        got = [t.requires_grad_() for t in args]
        got = torch.autograd.grad(hipops.group_norm(got[0], 4, got[1], got[2], act="silu", residual=got[3]), got, negated(dy))
        assert all(torch.equal(a, c) for a, c in zip(got, want.values())), i
        for t in (x, w, b, r):
            t.requires_grad_(False)
    with pytest.raises(ValueError, match="negated"):
        hipops.group_norm(x, 4, w, b, out=negated(x))
    z = torch.complex(x, -x).conj().imag[..., :1]                # (a stride of two floats, a negated one)
    assert z.is_neg() and torch.equal(hipops.group_norm(z, 1), hipops.group_norm(z.resolve_neg(), 1))


def test_clipping_of_negated_views(gpu):
    a, c = make((40, 8), F32, False)[0], make((7,), F32, False, seed=1)[0]
    want = [torch.empty_like(a), torch.empty_like(c)]
    norm = hipops.clip_grads([a, c], 1.0, out=want)
    na, nc = negated(a), negated(c)
    out = [torch.empty_like(a), torch.empty_like(c)]
    assert torch.equal(hipops.clip_grads([na, c], 1.0, out=out), norm) and all(torch.equal(p, q) for p, q in zip(out, want))
    out = [negated(a), negated(c)]
    assert torch.equal(hipops.clip_grads([a, nc], 1.0, out=out), norm) and all(torch.equal(p, q) for p, q in zip(out, want))
    assert torch.equal(hipops.grad_norm([na, nc]), norm)
    assert torch.equal(hipops.clip_grads([na, nc], 1.0), norm) and torch.equal(na, want[0]) and torch.equal(nc, want[1])


# ---- derivatives that the operators do not have are refused, not dropped -----------------------------------------------------

def test_forward_mode_is_refused(gpu):
    import torch.autograd.forward_ad as forward_ad
    full = make((2, 60, 16), F32, True)[:4]
    for base in (full, [full[0][..., :12].transpose(0, 1), full[1][:12].bfloat16(), full[2][:12].half(), full[3][..., :12].transpose(0, 1)]):
        for i in range(4):
            with forward_ad.dual_level():
                args = [forward_ad.make_dual(t, torch.ones_like(t)) if k == i else t for k, t in enumerate(base)]
                for mode in (torch.enable_grad, torch.no_grad):                   # (tangents do not depend on this mode)
                    for out in (None, torch.empty_like(base[0], memory_format=torch.contiguous_format)):
                        with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                            hipops.group_norm(args[0], 4, args[1], args[2], residual=args[3], out=out)
                hipops.group_norm(*[forward_ad.unpack_dual(args[0]).primal, 4, *base[1:3]])       # nothing is left behind
    with forward_ad.dual_level():
        out = forward_ad.make_dual(torch.empty_like(full[0]), full[0])
        with pytest.raises(NotImplementedError, match="forward-mode"):
            hipops.group_norm(full[0], 4, out=out)
        for t in (full[0], full[0].transpose(0, 1), full[0][:, ::2]):
            d = forward_ad.make_dual(t, torch.ones_like(t))
            for call in (lambda: hipops.grad_norm([d]), lambda: hipops.clip_grads([d], 1.0), lambda: hipops.clip_grads([t], 1.0, out=[d]),
                         lambda: hipops.clip_grads([full[1], d], 1.0, out=[full[1].clone(), torch.empty_like(t)])):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
    for transform in (lambda f, t: torch.func.jvp(f, (t,), (t,)), lambda f, t: torch.func.grad(lambda u: f(u).sum())(t), lambda f, t: torch.func.vmap(f)(t)):
        for f in (lambda t: hipops.group_norm(t, 4), lambda t: hipops.group_norm(t, 4, out=torch.empty_like(full[0][:1])), lambda t: hipops.grad_norm([t])):
            with pytest.raises((RuntimeError, ValueError)):
                transform(f, full[0][None, :1])


def test_gradients_of_the_norm_are_refused(gpu):
    """Gradients that carry a graph, as a penalty on their norm would have them; taken as numbers under no_grad."""
    p = torch.tensor([3.0, 4.0], device="cuda", requires_grad=True)
    g, = torch.autograd.grad(0.5 * p.square().sum(), p, create_graph=True)
    column = (p[:, None] * torch.ones(2, 3, device="cuda"))[:, ::2]             # one of other strides
    for t in (g, p, column):
        out = torch.full_like(t, 7.0).detach()
        for call in (lambda: hipops.grad_norm([t]), lambda: hipops.grad_norm(t), lambda: hipops.clip_grads([t], 1.0, out=[out]),
                     lambda: hipops.clip_grads([out, t], 1.0, out=[out, torch.empty_like(out)])):
            with pytest.raises(ValueError, match="requires a gradient"):
                call()
        assert bool((out == 7).all())
        with torch.no_grad():
            n = hipops.grad_norm([t])
            assert torch.equal(n, hipops.clip_grads([t], 1.0, out=[out])) and float(out.norm()) <= 1 + 1e-6
        assert torch.equal(n, hipops.grad_norm([t.detach()]))
    hipops.clip_grads([p.detach()], 1.0)


# ---- capture: leaves that are cast or laid out before the kernels see them ---------------------------------------------------

def test_capture_beside_a_live_eager_graph_of_other_types_and_strides(gpu):
    """A leaf of another type or stride reaches the kernels as a copy whose graph ends at the leaf: its eager graph stands in a captured
    backward's way as one of a plain leaf does, and the captured forward refuses it likewise."""
    x, w, b, r, dy = make((2, 60, 16), F32, True)
    turned = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)                          # noqa: E731
    for i, leaf in ((0, turned(x)), (1, w.bfloat16()), (1, torch.stack([w, w], 1)[:, 0]), (2, b.half()), (3, turned(r))):
        leaf = leaf.detach().requires_grad_()
        args = [leaf if k == i else t for k, t in enumerate((x, w, b, r))]
        run = lambda: hipops.group_norm(args[0], 4, args[1], args[2], act="relu", residual=args[3])      # noqa: E731,B023
        alive = run()
        with pytest.raises(RuntimeError, match="drop the results"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                run()
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = run()
            d, = torch.autograd.grad(y, leaf, dy)
            y = y.detach()
        for seed in range(3):
            with torch.no_grad():
                leaf.copy_(make((2, 60, 16), F32, True, seed=seed)[i])
            graph.replay()
            torch.cuda.synchronize()
            got = [y.clone(), d.clone()]
            want = run()
            assert torch.equal(got[0], want.detach()) and torch.equal(got[1], torch.autograd.grad(want, leaf, dy)[0]), (i, seed)
            del want


# ---- lists of strided gradients ------------------------------------------------------------------------------------------------

def test_strided_gradients_that_share_memory(gpu):
    base = make((10, 12), F32, False)[0]
    before = base.clone()
    for bad in ([base[:, ::2], base[:, ::2]], [base, base[:, :3]], [base[:, 1:], base[:4, :1], base[3:, 2:3]]):
        with pytest.raises(RuntimeError, match="overlaps"):
            hipops.clip_grads(bad, 1.0)
        with pytest.raises(RuntimeError, match="overlaps"):
            hipops.clip_grads([t.clone() for t in bad], 1.0, out=bad)
        assert torch.equal(base, before)
        assert abs(float(hipops.grad_norm(bad)) - sum(float(t.double().square().sum()) for t in bad) ** 0.5) <= 1e-5      # read only
    shared = base.view(-1).as_strided((4, 3), (2, 1))
    with pytest.raises(ValueError, match="overlaps itself"):
        hipops.clip_grads([shared], 1.0)
    assert torch.equal(base, before)
    norm = hipops.clip_grads([base[:, ::2], base[:, 1:6:2], base[:, 7::2].t()], 1.0)          # beside each other: each value once
    want = float(before.double().norm())
    assert abs(float(norm) - want) <= 2 * U * want
    within(base, (before.double() / (want + 1e-6), 4 * U * before.double().abs()), "values")


# ---- out= ---------------------------------------------------------------------------------------------------------------------

def test_out_over_the_parameters_is_refused(gpu):
    x, w, b, _, _ = make((2, 20, 16), F32, False)
    pool = torch.zeros(2 * 20 * 16 + 16, device="cuda")
    out, beside = pool[:640].view(2, 20, 16), pool[640:]
    for shared in (pool[:16], pool[630:646]):
        for kw in (dict(weight=shared, bias=b), dict(weight=w, bias=shared)):
            with pytest.raises(ValueError, match="weight or bias"):
                hipops.group_norm(x, 4, out=out, **kw)
    assert not pool.any()
    beside.copy_(b)
    assert torch.equal(hipops.group_norm(x, 4, w, beside, out=out), hipops.group_norm(x, 4, w, b))
    cast = pool[:8].view(F16)                  # of another type: read, as a copy, before anything is written
    want = hipops.group_norm(x, 4, cast.clone(), b)
    assert torch.equal(hipops.group_norm(x, 4, cast, b, out=out), want)


@pytest.mark.parametrize("eps", [0.0, 5e-324, 1e30, 1e300, 1e305, 1.7e308])
@pytest.mark.parametrize("shape", BOTH_WAYS)
def test_any_finite_eps(gpu, shape, eps):
    x, w, b, r, dy = make(shape, F32, True)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = hipops.group_norm(x, 4, w, b, eps=eps, act="relu", residual=r)
    grads = torch.autograd.grad(y, leaves, dy)
    want = norm64(x.detach(), 4, w.detach(), b.detach(), eps, "relu", r.detach(), dy)
    within(y.detach(), want["y"], "y")
    for k, v in zip(("dx", "dweight", "dbias", "dresidual"), grads):
        if k == "dweight":                     # beyond eps = 1e76, 1 / sqrt(eps) and xhat are below float32's normal numbers
            value, allowed = want[k]
            want[k] = value, allowed + 2.0 ** -149 * float(dy.abs().sum())
        within(v, want[k], k)


def test_forward_over_reverse_is_refused(gpu):
    """A tangent of the incoming gradient would be lost in the backward as one of x is in the forward."""
    import torch.autograd.forward_ad as forward_ad
    x, w, b, r, dy = make((2, 60, 16), F32, True)
    for act, res in (("relu", None), ("silu", r.clone().requires_grad_()), ("none", r.clone().requires_grad_())):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)] + ([res] if res is not None else [])
        y = hipops.group_norm(leaves[0], 4, leaves[1], leaves[2], act=act, residual=res)
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaves, forward_ad.make_dual(dy, torch.ones_like(dy)), retain_graph=True)
            torch.autograd.grad(y, leaves, dy)


def test_lists_in_one_buffer_are_taken_or_refused(gpu):
    """Contiguous tensors in one buffer, in order and out of it, empty ones among them, in place and not: refused if and only if a
    written byte belongs to another tensor of the call, and right where they are taken."""
    import random
    rng, seen = random.Random(3), [0, 0]
    start = make((4096,), F32, False)[0]
    for trial in range(2000):
        buffer, k = start.clone(), rng.randint(1, 6)

        def views(types):
            at, out = rng.choice([0, 0, 16, 64]), []
            for t in types:
                flat, n = buffer.view(t), rng.choice([0, 1, 2, 3, 5, 8, 40])
                out.append(flat[at * 4 // t.itemsize:][:n])
                at += -(-n * t.itemsize // 4) + rng.choice([0, 0, 1, 3, 16])
            return out
        types = [rng.choice([F32, F32, F16, BF16]) for _ in range(k)]
        outs = views(types)
        grads = [o if rng.random() < 0.6 else start.to(o.dtype if o.dtype != F32 else rng.choice([F32, F16, BF16]))[rng.randint(0, 99):][:o.numel()]
                 for o in outs]
        if rng.random() < 0.3:
            i = rng.randrange(k)
            grads[i] = buffer.view(outs[i].dtype)[rng.randint(0, 200):][:outs[i].numel()]
        both = list(zip(grads, outs))
        if rng.random() < 0.3:
            rng.shuffle(both)
        grads, outs = [t for t, _ in both], [o for _, o in both]
        try:
            hipops._check_overlaps(grads, outs)
            refused = False
        except RuntimeError:
            refused = True
        seen[refused] += 1
        before = [t.double() for t in grads]
        if refused:
            with pytest.raises(RuntimeError, match="overlaps"):
                hipops.clip_grads(grads, 0.5, out=outs)
            assert torch.equal(buffer.view(torch.int32), start.view(torch.int32))
            continue
        if any(not bool(torch.isfinite(t).all()) for t in before):               # (16-bit views of floats)
            continue
        norm = sum(float(t.square().sum()) for t in before) ** 0.5
        got = hipops.clip_grads(grads, 0.5, out=outs)
        assert abs(float(got) - norm) <= 2 * U * norm
        for t, o in zip(before, outs):
            want = t * min(1.0, 0.5 / (norm + 1e-6))
            within(o, (want, (3 * U + torch.finfo(o.dtype).eps / 2) * want.abs() + torch.finfo(o.dtype).smallest_normal * torch.finfo(o.dtype).eps), "values")
    assert min(seen) > 100, seen
