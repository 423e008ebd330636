"""hipops.group_norm on the GPU against its definition in 64 bits, with tolerances from the roundings of its steps
(norm_clip_reference.norm64)."""
import pytest
import torch

import msnets_amd  # noqa: F401
from msnets_amd import hipops
from norm_clip_reference import norm64, within

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAMES = ("x", "weight", "bias", "residual")


def make(shape, dtype, residual, seed=0, mean=1.0, wide=0, affine=True):
    """Inputs as a conv leaves them: every channel its own mean and width.  wide: x is a channel slice of that many more."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)              # noqa: E731
    c = shape[-1]
    x = (rnd(*shape[:-1], c + wide) * (0.5 + torch.rand(c + wide, device="cuda", generator=g)) + mean * rnd(c + wide)).to(dtype)[..., wide:]
    w, b = (1 + 0.3 * rnd(c), 0.3 * rnd(c)) if affine else (None, None)
    r = rnd(*shape).clamp_min(0).to(dtype) if residual else None
    return x, w, b, r, rnd(*shape).to(dtype)


def run_and_check(x, groups, w, b, r, dy, act, eps=1e-5):
    leaves = {k: v.detach().requires_grad_() for k, v in zip(NAMES, (x, w, b, r)) if v is not None}
    y = hipops.group_norm(leaves["x"], groups, leaves.get("weight"), leaves.get("bias"), eps=eps, act=act, residual=leaves.get("residual"))
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    want = norm64(x, groups, w, b, eps, act, r, dy)
    with torch.no_grad():
        served = hipops.group_norm(x, groups, w, b, eps=eps, act=act, residual=r)
    assert torch.equal(served, y.detach()), "with and without gradients"
    within(y.detach(), want["y"], "y")
    for k, v in grads.items():
        assert v.dtype == leaves[k].dtype and v.shape == leaves[k].shape
        within(v, want["d" + k], "d" + k)


# (shape, groups): every vector width, groups inside and across vectors, one launch and two, chunks of channels, groups wider than a
# workgroup, one channel a group, one group, one row, one value a group
SHAPES = [((2, 2, 3, 5, 32), 8), ((1, 6, 17, 30, 128), 8), ((2, 12, 34, 61, 64), 16), ((1, 23, 40, 41, 32), 8), ((3, 50, 60), 12),
          ((2, 701, 33), 3), ((2, 9, 11, 13, 12), 4), ((1, 40000, 20), 5), ((5, 1, 64), 8), ((1, 1, 8), 8), ((4, 3, 2, 640), 1),
          ((2, 3, 4224), 1), ((1, 300, 2112), 2), ((1, 7, 1025), 1), ((2, 5000, 7), 7), ((1, 3001, 96), 32), ((70, 33, 24), 2),
          ((2, 37, 2048), 2048), ((3, 1, 1), 1), ((2, 1100, 514), 257), ((1, 90, 1540), 7), ((3, 64), 4)]


@pytest.mark.parametrize("act,residual", [("none", False), ("relu", False), ("relu", True), ("silu", True)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape,groups", SHAPES, ids=["x".join(map(str, s)) + "g%d" % g for s, g in SHAPES])
def test_forward_and_gradients(gpu, shape, groups, dtype, act, residual):
    x, w, b, r, dy = make(shape, dtype, residual, seed=len(shape) * 1000 + groups)
    run_and_check(x, groups, w, b, r, dy, act)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape,groups", [((2, 4, 9, 60), 12), ((1, 50000, 32), 8), ((2, 300, 5), 5)])
def test_channel_slices_and_other_strides(gpu, shape, groups, dtype):
    x, w, b, r, dy = make(shape, dtype, True, wide=shape[-1])
    assert not x.is_contiguous()
    run_and_check(x, groups, w, b, r, dy, "silu")
    run_and_check(x.contiguous().transpose(0, 1).contiguous().transpose(0, 1), groups, w, b, r, dy.expand_as(x), "relu")
    run_and_check(x, groups, w, b, r[:1].expand_as(x), dy[..., :1].expand_as(x), "relu")           # broadcast inputs
    odd = torch.empty(x.numel() + 3, device="cuda", dtype=dtype)[3:].view(shape).copy_(x)             # no 16-byte alignment
    run_and_check(odd, groups, w, b, r, dy, "relu")


def test_parameters_in_other_types_and_without_any(gpu):
    x, w, b, r, dy = make((2, 100, 48), BF16, False)
    wb, bb = w.bfloat16().requires_grad_(), b.half().requires_grad_()
    y = hipops.group_norm(x, 6, wb, bb, act="relu")
    dw, db = torch.autograd.grad(y, [wb, bb], dy)
    want = norm64(x, 6, wb.detach().float(), bb.detach().float(), 1e-5, "relu", None, dy)
    assert dw.dtype == BF16 and db.dtype == F16
    for got, (v, e) in ((dw, want["dweight"]), (db, want["dbias"])):
        within(got, (v, e + torch.finfo(got.dtype).eps / 2 * (v.abs() + e)), "parameter gradient")
    for one in ((None, None), (w, None), (None, b)):
        run_and_check(x, 6, *one, None, dy, "silu")


@pytest.mark.parametrize("mean", [1e3, 1e5])
@pytest.mark.parametrize("shape,groups", [((1, 40, 32), 8), ((2, 30000, 32), 8)])
def test_mean_far_from_zero(gpu, shape, groups, mean):
    x, w, b, r, dy = make(shape, F32, False, mean=mean)
    run_and_check(x, groups, w, b, None, dy, "none")
    x[:, 0] = 3e7                              # the first row, which the sums are taken against, is the outlier
    run_and_check(x, groups, w, b, None, dy, "relu")


@pytest.mark.parametrize("shape", [(1, 50, 16), (2, 40000, 16)])
def test_constant_and_zero_groups(gpu, shape):
    x = torch.full(shape, 2.5, device="cuda")
    x[..., 8:] = 0
    w, b = torch.linspace(-1, 1, 16, device="cuda"), torch.linspace(1, -1, 16, device="cuda")
    run_and_check(x, 2, w, b, None, torch.ones_like(x), "relu")
    x, _, _, r, dy = make(shape, F32, True)
    zero = torch.zeros(16, device="cuda")      # gamma and beta of a residual branch before its first step: z is the residual, often 0
    run_and_check(x, 2, zero, zero, r, dy, "relu")
    run_and_check(x, 2, zero, zero, None, dy, "relu")


def test_relu_border_is_decided_in_64_bits(gpu):
    """Values at and next to the border, where 32 bits cannot tell the side: symmetric data whose mean is exactly representable, and
    biases that cancel xhat * gamma up to the last bits."""
    for seed in range(3):
        x, w, b, r, dy = make((2, 20011, 8), F32, False, seed)
        want = norm64(x, 2, w, b, 1e-5, "none", None)["y"][0]
        r = -(want.float())                    # z = a rounding error of the residual: +-2^-25 of its size
        run_and_check(x, 2, w, b, r, dy, "relu")


@pytest.mark.parametrize("shape", [(2, 60, 16), (2, 30000, 16)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nonfinite_values_stay_in_their_group(gpu, shape, bad):
    x, w, b, r, _ = make(shape, F32, True)
    clean = hipops.group_norm(x, 4, w, b, act="relu", residual=r)
    x[1, 7, 5] = bad
    y = hipops.group_norm(x, 4, w, b, act="relu", residual=r)
    assert torch.isnan(y[1, :, 4:8]).all()
    y[1, :, 4:8] = clean[1, :, 4:8]
    assert torch.equal(y, clean)


def test_empty(gpu):
    w, b = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda", requires_grad=True)
    for shape in ((0, 4, 8), (3, 0, 8), (2, 0, 5, 8)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y = hipops.group_norm(x, 2, w, b, act="silu")
        dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
        assert y.shape == shape and dx.shape == shape and not dw.any() and not db.any()


@pytest.mark.parametrize("shape", [(2, 50, 32), (1, 40000, 32)])
def test_out(gpu, shape):
    x, w, b, r, _ = make(shape, F32, True)
    args = dict(act="relu")
    want = hipops.group_norm(x, 8, w, b, residual=r, **args)
    wide = torch.full(shape[:-1] + (96,), 7.0, device="cuda")
    hipops.group_norm(x, 8, w, b, residual=r, out=wide[..., 32:64], **args)
    assert torch.equal(wide[..., 32:64], want) and bool((wide[..., :32] == 7).all()) and bool((wide[..., 64:] == 7).all())
    wide[..., :32] = x                         # a slice of the rows that hold the input
    hipops.group_norm(wide[..., :32], 8, w, b, residual=r, out=wide[..., 64:], **args)
    assert torch.equal(wide[..., 64:], want)
    rr = r.clone()
    assert hipops.group_norm(x, 8, w, b, residual=rr, out=rr, **args) is rr and torch.equal(rr, want)
    xx = x.clone()
    hipops.group_norm(xx, 8, w, b, residual=r, out=xx, **args)
    assert torch.equal(xx, want)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 3060, 128), (2, 4097, 32), (1, 2049, 64)])
def test_in_place_and_out_of_place_agree(gpu, shape, dtype):
    """Long chunks: out of place, workgroups share one and each writes its part; in place one writes all of it."""
    x, w, b, r, _ = make(shape, dtype, True)
    want = norm64(x, 8, w, b, 1e-5, "relu", r)["y"]
    y = hipops.group_norm(x, 8, w, b, act="relu", residual=r)
    within(y, want, "y")
    for k, out in enumerate((x.clone(), r.clone())):
        hipops.group_norm(x if k else out, 8, w, b, act="relu", residual=out if k else r, out=out)
        assert torch.equal(out, y)


def test_gradients_against_differences(gpu):
    """d/dt of sum(y * dy) along random directions, by central differences of the operator itself: y is float32, so with step h the
    quotient is off by about |y dy| sqrt(n) 2^-24 / h and h^2 |third derivative| / 6."""
    x, w, b, r, dy = make((2, 400, 24), F32, True, seed=5)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    f = lambda *t: hipops.group_norm(t[0], 6, t[1], t[2], act="silu", residual=t[3])                # noqa: E731
    grads = torch.autograd.grad(f(*leaves), leaves, dy)
    g = torch.Generator(device="cuda").manual_seed(1)
    h = 2.0 ** -7
    with torch.no_grad():
        for i in range(4):
            v = torch.randn(leaves[i].shape, device="cuda", generator=g)
            # inputs on a grid of powers of two: x +- h v is exact to 2^-24 of itself and does not disturb the quotient
            at = lambda s: [t.detach() + s * h * v if k == i else t.detach() for k, t in enumerate(leaves)]      # noqa: E731
            diff = float(((f(*at(1)).double() - f(*at(-1)).double()) * dy.double()).sum()) / (2 * h)
            exact = float((grads[i].double() * v.double()).sum())
            scale = float(grads[i].double().norm() * v.double().norm())
            # the second-order term: |silu'''| < 1, every value moves by at most about |v| <= 5: (5h)^2 / 6 of the terms' size
            assert abs(diff - exact) <= (25 * h * h / 6) * scale + 1e-3 * scale * 2 ** -7, (i, diff, exact, scale)


def test_repeats_bit_for_bit(gpu):
    for shape in ((2, 100, 64), (2, 20000, 64)):
        x, w, b, r, dy = make(shape, BF16, True)
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]

        def once():
            y = hipops.group_norm(leaves[0], 8, leaves[1], leaves[2], act="silu", residual=leaves[3])
            return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
        first = once()
        for _ in range(3):
            torch.empty(1 << 24, device="cuda").normal_()              # other work, other contents of freed memory
            assert all(torch.equal(a, c) for a, c in zip(first, once()))


def test_a_sample_does_not_depend_on_its_batch(gpu):
    """The statistics' sums of a sample are cut by the batch's size, so only their rounding may differ (64-bit sums: none that shows)."""
    x, w, b, r, _ = make((3, 9000, 32), F32, True)
    y = hipops.group_norm(x, 8, w, b, act="relu", residual=r)
    for i in range(3):
        one = hipops.group_norm(x[i:i + 1], 8, w, b, act="relu", residual=r[i:i + 1])
        assert float((one - y[i:i + 1]).abs().max()) <= 2.0 ** -22 * float(y.abs().max())


def test_another_stream_and_two_at_once(gpu):
    xs = [make((1, 30000, 32), F32, True, seed=s) for s in range(4)]
    want = [hipops.group_norm(x, 8, w, b, act="relu", residual=r) for x, w, b, r, _ in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(3):
        for (x, w, b, r, _), s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(hipops.group_norm(x, 8, w, b, act="relu", residual=r))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 4])


@pytest.mark.parametrize("shape,groups", [((70_001, 3, 8), 2), ((70_001, 64), 4), ((1, 2_000_003, 4), 1)])
def test_very_many_samples_or_rows(gpu, shape, groups):
    x, w, b, r, dy = make(shape, BF16, True)
    run_and_check(x, groups, w, b, r, dy, "relu")


def test_two_threads(gpu):
    """Two Python threads, a stream each, forward and backward at once."""
    import threading
    sets = [make((1, 20000, 32), F32, True, seed=s) for s in range(2)]

    def step(k):
        leaves = [t.detach().requires_grad_() for t in sets[k][:4]]
        y = hipops.group_norm(leaves[0], 8, leaves[1], leaves[2], act="silu", residual=leaves[3])
        return [y.detach(), *torch.autograd.grad(y, leaves, sets[k][4])]
    want = [step(0), step(1)]
    torch.cuda.synchronize()
    got, errors = {0: [], 1: []}, []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[k].append(step(k))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                 # noqa: BLE001  (raised again below, on the test's own thread)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    [t.start() for t in threads]
    [t.join(60) for t in threads]
    assert not errors, errors
    for k in (0, 1):
        assert len(got[k]) == 20 and all(torch.equal(a, c) for one in got[k] for a, c in zip(one, want[k]))


@pytest.mark.parametrize("shape", [(2, 60, 32), (2, 12000, 32)])
def test_captured_and_replayed(gpu, shape):
    x, w, b, r, dy = make(shape, F32, True)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b, r)]

    def step():
        y = hipops.group_norm(leaves[0], 8, leaves[1], leaves[2], act="silu", residual=leaves[3])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        with torch.no_grad():
            for t, v in zip(leaves, make(shape, F32, True, seed=seed)[:4]):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, c) for a, c in zip(got, step())), seed


def test_capture_beside_a_live_eager_graph_is_refused(gpu):
    """Captured while an eager graph of the same leaves lives, a backward pass would end the process: the forward refuses."""
    x, w, b, _, dy = make((1, 60, 16), F32, False)
    leaf = x.clone().requires_grad_()
    alive = hipops.group_norm(leaf, 4, w, b, act="relu")
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="drop the results"):
        with torch.cuda.graph(graph):
            hipops.group_norm(leaf, 4, w, b, act="relu")
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx, = torch.autograd.grad(hipops.group_norm(leaf, 4, w, b, act="relu"), leaf, dy)
    graph.replay()
    torch.cuda.synchronize()
    got = dx.clone()
    assert torch.equal(got, torch.autograd.grad(hipops.group_norm(leaf, 4, w, b, act="relu"), leaf, dy)[0])


def test_saved_tensors_are_watched_and_differentiated_once(gpu):
    x, w, b, _, dy = make((1, 20, 8), F32, False)
    leaf = x.clone().requires_grad_()
    mid = leaf * 1
    y = hipops.group_norm(mid, 2, w, b, act="relu")
    with torch.no_grad():
        mid.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)
    leaf2 = x.clone().requires_grad_()
    dx, = torch.autograd.grad(hipops.group_norm(leaf2, 2, w, b, act="silu"), leaf2, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_partial_gradients(gpu):
    x, w, b, r, dy = make((2, 12000, 32), F32, True)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    full = torch.autograd.grad(hipops.group_norm(leaves[0], 8, *leaves[1:3], act="relu", residual=leaves[3]), leaves, dy)
    for i in range(4):
        args = [t if k == i else t.detach() for k, t in enumerate(leaves)]
        one, = torch.autograd.grad(hipops.group_norm(args[0], 8, *args[1:3], act="relu", residual=args[3]), [leaves[i]], dy)
        assert torch.equal(one, full[i]), NAMES[i]


def test_parameters_alone(gpu):
    """Frozen inputs: the same dgamma and dbeta, with one sample and with several, in one launch's reach and beyond it."""
    for shape in ((1, 40, 16), (3, 40, 16), (1, 30000, 16), (2, 30000, 16)):
        x, w, b, r, dy = make(shape, F32, True)
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        full = torch.autograd.grad(hipops.group_norm(leaves[0], 4, *leaves[1:3], act="relu", residual=leaves[3]), leaves, dy)
        both = torch.autograd.grad(hipops.group_norm(x, 4, *leaves[1:3], act="relu", residual=r), leaves[1:3], dy)
        assert torch.equal(both[0], full[1]) and torch.equal(both[1], full[2])
    dr, = torch.autograd.grad(hipops.group_norm(x, 4, w, b, residual=leaves[3]), [leaves[3]], dy)
    assert torch.equal(dr, dy)                 # without an activation


def test_out_is_seen_by_autograd(gpu):
    x, w, b, _, _ = make((1, 20, 8), F32, False)
    leaf = x.clone().requires_grad_()
    mid = leaf * 1
    loss = mid.square().sum()                  # keeps mid
    with torch.no_grad():
        hipops.group_norm(mid, 2, w, b, out=mid)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_refusals_on_the_gpu(gpu):
    x, w, b, r, _ = make((2, 10, 12), F32, True)
    call = hipops.group_norm
    for bad in (dict(groups=5), dict(groups=0), dict(groups=2.5), dict(act="gelu"), dict(eps=-1.0), dict(eps=float("nan")), dict(weight=w[:6]),
                dict(residual=r[:1]), dict(residual=r.half()), dict(out=torch.empty(2, 10, 13, device="cuda")), dict(out=x.half()),
                dict(out=torch.empty(1, device="cuda").expand(2, 10, 12))):
        kw = dict(groups=3, weight=w, bias=b, residual=r)
        kw.update(bad)
        with pytest.raises((ValueError, TypeError)):
            call(x, **kw)
    with pytest.raises(ValueError):
        call(x[0, 0], 3)
    with pytest.raises(TypeError):
        call(x.double(), 3)
    with pytest.raises(RuntimeError, match="MI355X"):
        call(x, 3, w.cpu(), b)
    with pytest.raises(ValueError, match="gradient"):
        call(x.clone().requires_grad_(), 3, out=torch.empty_like(x))
    flat = torch.zeros(2 * 10 * 12 + 12, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        call(flat[:240].view(2, 10, 12), 3, out=flat[12:].view(2, 10, 12))


def test_offsets_beyond_32_bits(gpu):
    """2.2e9 values in one call (a row stride of 64 channels, 8 of them used; and a dense batch), and the last rows exact."""
    rows = (1 << 31) // 64 + 5
    wide = torch.zeros(1, rows, 64, device="cuda", dtype=BF16)
    g = torch.Generator(device="cuda").manual_seed(0)
    x = wide[..., 56:]
    x.copy_(torch.randn(rows, 8, device="cuda", generator=g))
    w, b = torch.rand(8, device="cuda") + 0.5, torch.rand(8, device="cuda")
    y = hipops.group_norm(x, 2, w, b, act="relu", out=wide[..., :8])
    want = norm64(x.contiguous(), 2, w, b, 1e-5, "relu", None)["y"]
    within(y.contiguous(), want, "y")
    assert not wide[..., 8:56].any()
    del wide, x, y, want
    n = (1 << 31) // (4096 * 64) + 1            # dense, past 2^31 values: samples at either end
    x = torch.empty(n, 4096, 64, device="cuda", dtype=BF16)
    x.normal_(generator=g)
    leaf, wl = x.requires_grad_(), torch.ones(64, device="cuda", requires_grad=True)
    y = hipops.group_norm(leaf, 8, wl, None, act="silu")
    dx, _ = torch.autograd.grad(y, [leaf, wl], x.detach())
    for i in (0, n // 2, n - 1):
        one = norm64(x.detach()[i:i + 1], 8, wl.detach(), None, 1e-5, "silu", None, x.detach()[i:i + 1])
        within(y.detach()[i:i + 1], one["y"], "y[%d]" % i)
        within(dx[i:i + 1], one["dx"], "dx[%d]" % i)
