"""hipops.group_norm on the GPU: the ways through its kernels that sizes choose and ordinary tests do not reach -- results past the
caches, more groups in a chunk than a workgroup has threads, vectors narrowed to one channel, offsets past 2^31 in the backward's
two launches, and values next to a ReLU's border in every type.  Against 64 bits, with the tolerances of norm_clip_reference.norm64."""
import pytest
import torch

import msnets_amd  # noqa: F401
from msnets_amd import hipops
from norm_clip_reference import FLOOR, HALF_STEP, U, norm64, within

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make(shape, dtype, residual, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)              # noqa: E731
    c = shape[-1]
    x = (rnd(*shape) * (0.5 + torch.rand(c, device="cuda", generator=g)) + rnd(c)).to(dtype)
    return x, 1 + 0.3 * rnd(c), 0.3 * rnd(c), rnd(*shape).clamp_min(0).to(dtype) if residual else None, rnd(*shape).to(dtype)


def two_launches(x, groups):
    lib, s = msnets_amd._lib.load(), x.numel() // (x.shape[0] * x.shape[-1])
    return lib.msnet_group_norm_workspace_bytes(hipops._DTYPE_CODES[x.dtype], x.shape[0], s, x.shape[-1], groups) > 0


def check(x, groups, w, b, r, dy, act):
    leaves = {k: t.detach().requires_grad_() for k, t in zip(("x", "weight", "bias", "residual"), (x, w, b, r)) if t is not None}
    y = hipops.group_norm(leaves["x"], groups, leaves["weight"], leaves["bias"], act=act, residual=leaves.get("residual"))
    want = norm64(x, groups, w, b, 1e-5, act, r, dy)
    within(y.detach(), want["y"], "y")
    for k, v in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)):
        within(v, want["d" + k], "d" + k)
    with torch.no_grad():
        assert torch.equal(hipops.group_norm(x, groups, w, b, act=act, residual=r), y.detach())


@pytest.mark.parametrize("act,residual", [("relu", False), ("silu", True), ("none", False), ("relu", True)])
@pytest.mark.parametrize("shape,groups,dtype", [((1, 300001, 32), 8, F32), ((1, 600001, 32), 8, BF16), ((3, 90011, 60), 12, F16), ((2, 150003, 30), 5, F32)],
                         ids=["fp32", "bf16", "fp16", "fp32-pairs"])
def test_results_past_the_caches(gpu, shape, groups, dtype, act, residual):
    x, w, b, r, dy = make(shape, dtype, residual)
    assert x.numel() * x.element_size() >= 32e6 and two_launches(x, groups)
    check(x, groups, w, b, r, dy, act)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape,groups", [((1, 9000, 512), 512), ((2, 9001, 1024), 1024), ((1, 12000, 700), 350),      # groups of one and two channels
                                          ((2, 50, 2056), 4), ((1, 300, 1542), 3),                                  # 514 a group: edges inside vectors
                                          ((1, 200, 3081), 3)])                                                     # odd, and wider than a workgroup
def test_many_groups_and_narrowed_vectors(gpu, shape, groups, dtype):
    x, w, b, r, dy = make(shape, dtype, True)
    assert two_launches(x, groups)
    check(x, groups, w, b, r, dy, "silu")
    check(x, groups, w, b, None, dy, "relu")


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("shape,groups", [((2, 61, 16), 4), ((2, 20011, 16), 4), ((1, 3001, 6), 2), ((1, 90001, 6), 6)])
def test_relu_border_in_every_type(gpu, shape, groups, dtype):
    """Few distinct values, so that a channel's beta can cancel xhat * gamma of one of them to the last bit of a float32: a good part
    of all z are +-2^-25 of their terms, and 32 bits cannot tell their side."""
    g = torch.Generator(device="cuda").manual_seed(0)
    c = shape[-1]
    levels = torch.tensor([-1.5, -0.25, 0.5, 1.0, 3.0], device="cuda")
    pick = torch.randint(0, 5, shape, device="cuda", generator=g)
    x, w = levels[pick].to(dtype), 0.7 + torch.rand(c, device="cuda", generator=g)
    dy = torch.randn(*shape, device="cuda", generator=g).to(dtype)
    zero = torch.zeros(c, device="cuda")
    for level in range(5):
        z = norm64(x, groups, w, zero, 1e-5, "none", None)["y"][0]
        at = (pick[0] == level).double()
        b = -((z[0] * at).sum(0) / at.sum(0).clamp_min(1)).float()             # of the first sample, whose groups have one value there
        near = (z + b.double()).abs() < 2.0 ** -22
        assert float(near.double().mean()) > 0.02
        check(x, groups, w, b, None, dy, "relu")
    check(x, groups, w, b, torch.zeros_like(x), dy, "relu")


def test_backward_offsets_beyond_32_bits(gpu):
    """Rows that lie 64 channels apart, x and dy both past 2^31 values of one buffer."""
    rows = (1 << 31) // 64 + 5
    wide = torch.zeros(1, rows, 64, device="cuda", dtype=BF16)
    g = torch.Generator(device="cuda").manual_seed(0)
    x, dy = wide[..., 56:], wide[..., 8:16]
    for t in (x, dy):
        t.copy_(torch.randn(rows, 8, device="cuda", generator=g))
    w, b = torch.rand(8, device="cuda", generator=g) + 0.5, torch.rand(8, device="cuda", generator=g)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(hipops.group_norm(leaves[0], 2, leaves[1], leaves[2], act="relu"), leaves, dy)
    want = norm64(x.detach().contiguous(), 2, w.detach(), b.detach(), 1e-5, "relu", None, dy.contiguous())
    for k, v in zip(("dx", "dweight", "dbias"), grads):
        within(v, want[k], k)


def test_dense_backward_beyond_32_bits(gpu):
    """One dense sample of more than 2^31 values, forward and backward in two launches each; sums from the definition in 64 bits, part
    by part, and both ends compared.  Off by the roundings of gz, c1, xhat c2 (xhat itself by 4u) and the difference: at most 10u of
    their sizes, times rstd; the mean is so small that its own rounding is far below that."""
    rows, c, groups = (1 << 31) // 64 + 1003, 64, 4
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(1, rows, c, device="cuda", dtype=BF16).normal_(generator=g)
    dy = torch.empty_like(x).normal_(generator=g)
    w, b = torch.rand(c, device="cuda", generator=g) + 0.5, torch.rand(c, device="cuda", generator=g)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = hipops.group_norm(leaves[0], groups, leaves[1], leaves[2])
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    xs, ds, wd = x.detach()[0].split(1 << 20), dy[0].split(1 << 20), w.detach().double()
    m = rows * c // groups
    group = lambda per_channel: per_channel.view(groups, -1).sum(1).repeat_interleave(c // groups) / m                # noqa: E731
    mean = group(sum(p.double().sum(0) for p in xs))
    var = group(sum((p.double() - mean).square().sum(0) for p in xs))
    rstd = 1 / torch.sqrt(var + 1e-5)
    sums, dots = torch.zeros(c, dtype=torch.float64, device="cuda"), torch.zeros(c, dtype=torch.float64, device="cuda")
    for p, d in zip(xs, ds):
        sums += d.double().sum(0)
        dots += (d.double() * ((p.double() - mean) * rstd)).sum(0)
    sizes = rows * 1.0                           # of |dy|, |dy xhat|: at most about one each on average
    within(db, (sums, U * sums.abs() + 1e-12 * sizes), "dbias")
    within(dw, (dots, U * dots.abs() + 4 * U * sizes), "dweight")
    c1, c2 = group(wd * sums), group(wd * dots)
    for at in (slice(0, 1000), slice(rows - 1000, rows)):
        xhat, gz = (x.detach()[0, at].double() - mean) * rstd, wd * dy[0, at].double()
        v = (gz - c1 - xhat * c2) * rstd
        e = 10 * U * rstd * (gz.abs() + c1.abs() + (xhat * c2).abs())
        within(dx[0, at], (v, e + HALF_STEP[BF16] * (v.abs() + e) + FLOOR[BF16]), "dx")
        z = xhat * wd + b.detach().double()
        e = 8 * U * ((xhat * wd).abs() + b.detach().double().abs())
        within(y.detach()[0, at], (z, e + HALF_STEP[BF16] * (z.abs() + e) + FLOOR[BF16]), "y")
