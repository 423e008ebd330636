"""The group-normalised aggregators (norm="group") on the GPU against the oracle's forward in 64 bits with its batch norm exchanged,
and a training step of group norm and gradient clipping together."""
import pytest
import torch
import torch.nn.functional as F

import msnets_amd  # noqa: F401
from msnets_amd import driver_utils, hipops
from msnets_amd.gcnet_3dcnn import GCNet_CostVolumeAggre
from msnets_amd.psmnet_3dcnn import PSMNet_CostVolumeAggre
from oracle import aggregators as oracle

pytestmark = pytest.mark.gpu
TOLERANCE = 1e-3                               # of a disparity, as for the batch-normalised aggregators


def randomise(model, seed):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for m in model.modules():
            if isinstance(m, torch.nn.GroupNorm):
                m.weight.copy_(0.5 + torch.rand(m.weight.shape, generator=g))
                m.bias.copy_(0.4 * torch.rand(m.bias.shape, generator=g) - 0.2)
    return model.eval()


def want(monkeypatch, forward, model, x, groups, *args, **kw):
    monkeypatch.setattr(oracle, "_bn", lambda sd, p, t: F.group_norm(t, groups, sd[p + ".weight"], sd[p + ".bias"], 1e-5))
    sd = {k: v.detach().cpu().double() for k, v in model.state_dict().items()}
    with torch.no_grad():
        return forward(sd, x.double(), *args, **kw)


@pytest.mark.parametrize("precision", ["split-fp16", "fp32"])
@pytest.mark.parametrize("shape,groups,quarter", [((1, 8, 16, 16, 32), 8, False), ((2, 8, 32, 32, 64), 4, False), ((1, 8, 16, 48, 80), 16, False),
                                                  ((1, 8, 16, 16, 32), 8, True), ((1, 16, 16, 32, 32), 8, False)])
def test_gcnet(gpu, monkeypatch, shape, groups, quarter, precision):
    torch.manual_seed(3)
    maxdisp = shape[2] * (4 if quarter else 2)
    model = randomise(GCNet_CostVolumeAggre(maxdisp, shape[1], is_quarter_input_size=quarter, norm="group", norm_groups=groups), 1)
    x = torch.rand(shape)
    ref = want(monkeypatch, oracle.gcnet_forward, model, x, groups, maxdisp, is_quarter_input_size=quarter)
    model = model.cuda()
    monkeypatch.setattr(hipops, "_default_precision", precision)
    xc = x.cuda()
    disp = model(xc)
    assert float((disp.cpu().double() - ref).abs().max()) <= TOLERANCE
    assert torch.equal(model(xc), disp), "a second forward from the arena"
    assert torch.equal(model.forward_ndhwc(xc.permute(0, 2, 3, 4, 1).contiguous()), disp)
    model.use_graph = True
    for _ in range(4):
        assert torch.equal(model(xc), disp)
        torch.empty(1 << 22, device="cuda").normal_()


@pytest.mark.parametrize("precision", ["split-fp16", "fp32"])
@pytest.mark.parametrize("shape,planes", [((1, 64, 8, 16, 16), 64), ((2, 8, 8, 16, 32), 8)])
def test_psmnet(gpu, monkeypatch, shape, planes, precision):
    torch.manual_seed(4)
    model = randomise(PSMNet_CostVolumeAggre(32, in_planes=planes, norm="group"), 2)
    x = torch.rand(shape)
    ref = want(monkeypatch, oracle.psmnet_forward, model, x, 8, 32, (4 * shape[3], 4 * shape[4]))
    model = model.cuda()
    monkeypatch.setattr(hipops, "_default_precision", precision)
    disp = model(x.cuda())
    assert float((disp.cpu().double() - ref).abs().max()) <= TOLERANCE
    assert torch.equal(model.forward_ndhwc(x.cuda().permute(0, 2, 3, 4, 1).contiguous()), disp)


def test_a_sample_of_a_batch_is_normalised_by_itself(gpu):
    model = randomise(GCNet_CostVolumeAggre(32, norm="group"), 5).cuda()
    x = torch.rand(2, 8, 16, 32, 32, device="cuda")
    both = model(x)
    assert float((model(x[1:]) - both[1:]).abs().max()) <= TOLERANCE
    x[0] *= 100                                # the other sample's values do not matter
    assert float((model(x)[1:] - both[1:]).abs().max()) <= TOLERANCE


def test_range_guard_sees_the_norms_output(gpu):
    """An activation beyond the fp16 halves of the next conv, made by the norm's own weights: flagged, and repeated on fp32."""
    model = randomise(GCNet_CostVolumeAggre(32, norm="group"), 6).cuda()
    x = torch.rand(1, 8, 16, 16, 32, device="cuda")
    with torch.no_grad():
        model.conv3dbn_1[1].weight.fill_(2.0 ** 15)
    with pytest.warns(RuntimeWarning, match="fp16 range"):
        disp = model(x)
    assert model._forced_precision == "fp32" and torch.isfinite(disp).all()


def test_training_step(gpu):
    """Two group-normalised layers with a skip, a loss, the gradients clipped, a step: against the same in 64 bits, formula by formula
    (torch's own norm and clipping there).  Off by float32's roundings of sums of at most 2 * 480 * 16 terms: 1e-5 of a tensor's norm."""
    g = torch.Generator().manual_seed(0)
    x, target = torch.randn(2, 6, 8, 10, 8, generator=g), torch.randn(2, 6, 8, 10, 16, generator=g)
    params = [0.4 * torch.randn(16, 8, generator=g), 1 + 0.1 * torch.randn(16, generator=g), 0.1 * torch.randn(16, generator=g),
              0.3 * torch.randn(16, 16, generator=g), 1 + 0.1 * torch.randn(16, generator=g), 0.1 * torch.randn(16, generator=g)]

    def step(ps, norm, clip, x, target, max_norm):
        ps = [p.clone().requires_grad_() for p in ps]
        w1, g1, b1, w2, g2, b2 = ps
        h = norm(F.linear(x, w1), g1, b1, "relu", None)
        y = norm(F.linear(h, w2), g2, b2, "silu", h)
        (y - target).square().mean().backward()
        total = clip(ps, max_norm)
        grads = [p.grad.clone() for p in ps]
        with torch.no_grad():
            for p in ps:
                p.sub_(0.5 * p.grad)
        return [total] + grads + [p.detach() for p in ps]

    def plain(t, w, b, act, res):
        z = F.group_norm(t.movedim(-1, 1), 4, w, b, 1e-5).movedim(1, -1)
        z = z if res is None else z + res
        return torch.relu(z) if act == "relu" else F.silu(z)
    ours = lambda t, w, b, act, res: hipops.group_norm(t, 4, w, b, act=act, residual=res)          # noqa: E731
    for max_norm in (0.05, 1e3):
        ref = step([p.double() for p in params], plain, torch.nn.utils.clip_grad_norm_, x.double(), target.double(), max_norm)
        got = step([p.cuda() for p in params], ours, driver_utils.clip_grad_norm_, x.cuda(), target.cuda(), max_norm)
        assert (float(ref[0]) > max_norm) == (max_norm < 1), "the first clips, the second does not"
        for i, (a, b) in enumerate(zip(got, ref)):
            assert float((a.cpu().double() - b).norm()) <= 1e-5 * float(b.norm()), (max_norm, i)
