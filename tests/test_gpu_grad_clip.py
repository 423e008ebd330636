"""hipops.grad_norm / clip_grads and driver_utils.clip_grad_norm_ on the GPU against the definition in 64 bits.  The norm's squares
and sums are 64-bit, so it is off by its own rounding to float32; a scaled value by the factor's rounding and its own."""
import pytest
import torch

import msnets_amd  # noqa: F401
from msnets_amd import driver_utils, hipops
from norm_clip_reference import FLOOR, HALF_STEP, U

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def tensors(lengths, dtypes, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, device="cuda", generator=g) * scale).to(dtypes[i % len(dtypes)]) for i, n in enumerate(lengths)]


def norm_of(ts):
    return sum(float(t.double().square().sum()) for t in ts) ** 0.5


def check(before, after, max_norm, norm):
    want = norm_of(before)
    assert norm.dtype == F32 and norm.dim() == 0 and norm.is_cuda
    assert abs(float(norm) - want) <= (U + 1e-12) * want + 1e-45
    f = min(1.0, max_norm / (want + 1e-6))
    for t, o in zip(before, after):
        v = t.double() * f
        # the factor's rounding and the product's, then the output type's
        allowed = 2.1 * U * v.abs() + HALF_STEP[o.dtype] * v.abs() * (1 + 3 * U) + FLOOR[o.dtype]
        assert bool(((o.double() - v).abs() <= allowed).all())
        if f == 1:
            assert torch.equal(o, t.to(o.dtype))


LENGTHS = [[1], [5, 1, 0, 8191, 8192, 8193], [3] * 113, [700_001, 2, 40_000], list(range(1, 260)), [20_000_003, 17]]


@pytest.mark.parametrize("ratio", [0.3, 4.0])
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (F32, BF16, F16)], ids=["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: "%dx%d" % (len(v), max(v)))
def test_norm_and_clip(gpu, lengths, dtypes, ratio):
    ts = tensors(lengths, dtypes)
    before = [t.clone() for t in ts]
    want = norm_of(ts)
    assert abs(float(hipops.grad_norm(ts)) - want) <= (U + 1e-12) * want
    max_norm = want / ratio
    out = [torch.full_like(t, 3, dtype=F32) for t in ts]
    check(before, out, max_norm, hipops.clip_grads(ts, max_norm, out=out))
    assert all(torch.equal(a, b) for a, b in zip(ts, before)), "inputs are left alone"
    check(before, ts, max_norm, hipops.clip_grads(ts, max_norm))


def test_views_into_one_buffer(gpu):
    """Gradients as views of a bucket, of every alignment, and nothing written beside them."""
    for dtype in (F32, BF16):
        flat = tensors([10_050], [dtype])[0]
        before = flat.clone()
        lengths = [1, 2, 3, 5, 8, 13, 21, 34, 55, 89, 7, 4001, 999]
        views, at = [], 1
        for n in lengths:
            views.append(flat[at:at + n])
            at += n + n % 2                                     # gaps behind the odd ones
        old = [v.clone() for v in views]
        check(old, views, 1.5, hipops.clip_grads(views, 1.5))
        for v, o in zip(views, old):
            v.copy_(o)
        assert torch.equal(flat, before)


def test_shapes_and_layouts(gpu):
    g = torch.Generator(device="cuda").manual_seed(0)
    a = torch.randn(8, 4, 3, 3, 3, device="cuda", generator=g).to(memory_format=torch.channels_last_3d)
    b = torch.randn(50, 60, device="cuda", generator=g).t()
    c = torch.randn(40, 40, device="cuda", generator=g)[:, ::2]
    d = torch.randn((), device="cuda", generator=g)
    ts = [a, b, c, d]
    old = [t.clone() for t in ts]
    check(old, ts, 2.0, hipops.clip_grads(ts, 2.0))
    out = [torch.empty(t.shape, device="cuda") for t in ts]
    check([t.clone() for t in ts], out, 0.5, hipops.clip_grads(ts, 0.5, out=out))
    e = torch.ones(3, device="cuda").expand(4, 3)
    assert abs(float(hipops.grad_norm(e)) - 12 ** 0.5) <= 4 * U
    with pytest.raises(ValueError, match="expanded"):
        hipops.clip_grads([e], 1.0)


@pytest.mark.parametrize("value", [1e30, 1e-30])
def test_squares_beyond_float32(gpu, value):
    ts = [torch.full((1000,), value, device="cuda"), torch.full((24,), value, device="cuda", dtype=BF16)]
    old = [t.clone() for t in ts]
    check(old, ts, value, hipops.clip_grads(ts, value))


def test_nonfinite(gpu):
    for bad, rest in ((float("inf"), 0.0), (float("nan"), float("nan"))):
        ts = tensors([5000, 33], [F32])
        ts[1][7] = bad
        norm = hipops.clip_grads(ts, 1.0)
        assert not torch.isfinite(norm)
        assert torch.isnan(ts[1][7])
        for t in (ts[0], ts[1][:7], ts[1][8:]):
            assert bool((t == 0).all()) if rest == 0.0 else bool(torch.isnan(t).all())


def test_nothing_to_scale(gpu):
    z = torch.zeros(100, device="cuda")
    assert float(hipops.clip_grads([z], 1.0)) == 0 and not z.any()
    assert float(hipops.grad_norm([])) == 0 and float(hipops.clip_grads([], 1.0)) == 0
    assert float(hipops.grad_norm([torch.empty(0, device="cuda")])) == 0
    t = tensors([1000], [F32])[0]
    old = t.clone()
    hipops.clip_grads([t], float("inf"))
    assert torch.equal(t, old)
    hipops.clip_grads([t], 0.0)
    assert not t.any()


def test_longer_than_32_bits(gpu):
    n = (1 << 31) + 12_345
    t = torch.zeros(n, device="cuda", dtype=BF16)
    t[-5:] = 3
    t[:4] = 1
    norm = hipops.clip_grads([t], 0.7)
    assert abs(float(norm) - 7.0) <= 7 * U
    f = torch.tensor(0.7 / 7.000001, device="cuda")
    assert bool((t[-5:].float() - 3 * f).abs().max() <= 2 ** -8 * 0.31) and bool((t[:4].float() - f).abs().max() <= 2 ** -8 * 0.11)
    assert not t[4:-5].any()


def test_parameters(gpu):
    net = torch.nn.Sequential(torch.nn.Linear(30, 40), torch.nn.Linear(40, 5), torch.nn.Linear(5, 5)).cuda()
    net[2].requires_grad_(False)
    net[1](net[0](torch.randn(7, 30, device="cuda"))).square().sum().backward()
    grads = [p.grad for p in net.parameters() if p.grad is not None]
    assert len(grads) == 4
    old = [t.clone() for t in grads]
    versions = [t._version for t in grads]
    check(old, grads, 0.1, driver_utils.clip_grad_norm_(net.parameters(), 0.1))
    assert all(t._version > v for t, v in zip(grads, versions))
    one = torch.nn.Parameter(torch.ones(3, device="cuda"))
    assert float(driver_utils.clip_grad_norm_(one, 1.0)) == 0
    one.grad = torch.full((3,), 2.0, device="cuda")
    check([torch.full((3,), 2.0, device="cuda")], [one.grad], 1.0, driver_utils.clip_grad_norm_(one, 1.0))


def test_gradients_with_a_graph(gpu):
    """Of a loss whose gradient is to be differentiated: clipped by the driver's function, refused where a graph would record it."""
    p = torch.nn.Parameter(torch.tensor([3.0, 4.0], device="cuda"))
    p.square().sum().backward(create_graph=True)
    assert p.grad.requires_grad
    with pytest.raises(ValueError, match="requires a gradient"):
        hipops.clip_grads([p.grad], 1.0)
    old = p.grad.detach().clone()
    check([old], [p.grad.detach()], 1.0, driver_utils.clip_grad_norm_([p], 1.0))
    p.grad = None


def test_captured_and_replayed(gpu):
    lengths = [100_000, 7, 64] + [33] * 200                     # more tensors than one launch takes
    ts = tensors(lengths, [F32, BF16])
    out = [torch.zeros_like(t) for t in ts]
    hipops.clip_grads(ts, 3.0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = hipops.clip_grads(ts, 3.0, out=out)
    for seed in range(4):
        for t, v in zip(ts, tensors(lengths, [F32, BF16], seed=seed, scale=10.0 ** -seed)):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        eager = [torch.empty_like(t) for t in ts]
        n2 = hipops.clip_grads(ts, 3.0, out=eager)
        assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(out, eager)), seed


def test_two_streams_at_once(gpu):
    sets = [tensors([300_000, 11], [F32], seed=s) for s in range(4)]
    want = [float(hipops.grad_norm(ts)) for ts in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for ts, s in zip(sets, [torch.cuda.Stream() for _ in sets]):
            with torch.cuda.stream(s):
                got.append(hipops.grad_norm(ts))
    torch.cuda.synchronize()
    assert [float(v) for v in got] == want * 5


def test_refusals(gpu):
    a, b = tensors([100, 50], [F32])
    with pytest.raises(RuntimeError, match="overlaps"):
        hipops.clip_grads([a, b, a], 1.0)
    with pytest.raises(RuntimeError, match="overlaps"):
        hipops.clip_grads([a, a[40:60]], 1.0)
    with pytest.raises(RuntimeError, match="overlaps"):
        hipops.clip_grads([a[:50], b], 1.0, out=[b, torch.empty_like(b)])
    with pytest.raises(RuntimeError, match="overlaps"):
        hipops.clip_grads([a[:50]], 1.0, out=[a[1:51]])
    with pytest.raises(ValueError):
        hipops.clip_grads([a], -1.0)
    with pytest.raises(ValueError):
        hipops.clip_grads([a], float("nan"))
    with pytest.raises(ValueError):
        hipops.clip_grads([a, b], 1.0, out=[torch.empty_like(a)])
    with pytest.raises(ValueError):
        hipops.clip_grads([a], 1.0, out=[torch.empty_like(b)])
    with pytest.raises(ValueError):
        hipops.clip_grads([a.bfloat16()], 1.0, out=[a.half()])
    with pytest.raises(TypeError):
        hipops.clip_grads([a.double()], 1.0)
    with pytest.raises(TypeError):
        hipops.clip_grads([a.to_sparse()], 1.0)
    with pytest.raises(RuntimeError, match="MI355X"):
        hipops.clip_grads([a.cpu()], 1.0)
    assert abs(float(hipops.grad_norm([a, a])) - (2 ** 0.5) * norm_of([a])) <= 3 * U * norm_of([a])       # read only: allowed
