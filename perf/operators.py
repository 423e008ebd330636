"""The group norm and gradient clipping workloads: what is computed (plain torch), on which sizes, and what it has to move.

Two operators, each as a user of the aggregators meets it:

  norm   group norm with an activation over channels-last activations [N, D, H, W, C], with the residual that the decoder levels
         add before the activation; forward alone (serving), and forward with all gradients (training).
  clip   the global 2-norm over the gradients of a model, and the gradients scaled to at most a given norm.

Activation sizes are those of the cost-volume aggregators at 960x544x192 (levels 96x272x480x32, 48x136x240x64, 24x68x120x64,
12x34x60x64, 6x17x30x128), odd crops of them, and short sequences of rows; parameter sizes are the GCNet aggregator's, and
generic lists.

With `own` false, run() is elementary torch operations in 32 bits: sums over a group, which can be 50 million values long, and the
sign of a value next to a ReLU's border are taken in 64.  With `own` true it calls the package's operators."""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5
MOST_BYTES = 96 * 272 * 480 * 32 * 4         # the finest level's activation in fp32


def _norm(name, n, d, h, w, c, groups, dtype, act, residual, train, sliced=False):
    return {"name": name, "op": "norm", "n": n, "d": d, "h": h, "w": w, "c": c, "groups": groups, "dtype": dtype, "act": act,
            "residual": residual, "train": train, "sliced": sliced}


def _clip(name, model, tensors, total, dtype, out_dtype, ratio):
    """ratio: the gradients' norm over the allowed one (below 1: nothing to scale)."""
    return {"name": name, "op": "clip", "model": model, "tensors": tensors, "total": total, "dtype": dtype, "out_dtype": out_dtype,
            "ratio": ratio}


def listed():
    return [
        # the finest level behind its conv, one 960x544 pair being served
        _norm("norm serve finest", 1, 96, 272, 480, 32, 8, "fp32", "relu", False, False),
        # a decoder level: the skip connection is added inside
        _norm("norm serve decoder", 1, 48, 136, 240, 64, 8, "fp32", "relu", True, False),
        # the coarsest level: one small call among sixty, where its latency is what counts
        _norm("norm serve coarsest", 1, 6, 17, 30, 128, 8, "fp32", "relu", False, False),
        # a training step at the finest level, activations kept in bf16
        _norm("norm train finest", 1, 96, 272, 480, 32, 8, "bf16", "relu", False, True),
        # a training step on two crops of odd size, decoder level, fp32
        _norm("norm train odd crops", 2, 23, 67, 119, 64, 16, "fp32", "silu", True, True),
        # a coarse level of a training crop, mixed precision
        _norm("norm train coarse", 2, 12, 34, 60, 64, 8, "fp16", "silu", False, True),
        # half of the channels of a wider buffer, an odd group width
        _norm("norm serve slice", 2, 24, 68, 120, 60, 12, "bf16", "silu", False, False, sliced=True),
        # the GCNet aggregator's 56 gradients, too long
        _clip("clip aggregator", "gcnet", 56, 0, "fp32", "fp32", 7.5),
        # a gradient bucket of a large model: views of every length into one buffer, bf16 gradients into fp32 master gradients
        _clip("clip large bucket", "mixed", 290, 256_000_001, "bf16", "fp32", 3.0),
        # very many short tensors (norms, biases), short enough already
        _clip("clip short tensors", "mixed", 1000, 400_009, "fp32", "fp32", 0.4),
        # a fine-tuned head: a few tensors
        _clip("clip head", "mixed", 5, 70_001, "bf16", "bf16", 2.0),
    ]


def draw(rng):
    if rng.random() < 0.4:
        total = int(math.exp(rng.uniform(math.log(1000), math.log(256e6))))
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        case = _clip("", "mixed", 0, total, dtype, rng.choice([dtype, "fp32"]), math.exp(rng.uniform(math.log(0.1), math.log(30))))
        case["tensors"] = int(math.exp(rng.uniform(0, math.log(min(1200, total // 8)))))
        if BYTES[dtype] == 4:
            case["total"] = min(total, 190_000_000)
    else:
        dtype, train = rng.choice(["fp32", "bf16", "fp16"]), rng.random() < 0.5
        cg = rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 8, 12, 16, 16, 24, 32, 33, 64])
        groups = rng.choice([g for g in (1, 2, 3, 4, 7, 8, 8, 12, 16, 32) if cg * g <= 640])
        c, n = cg * groups, rng.choice([1, 1, 2, 3, 8])
        residual = rng.random() < 0.4
        most = MOST_BYTES // ((2 * BYTES[dtype] if train else 4) * c * n)
        if residual:
            most //= 2
        # the shortest groups hold 16 values: with fewer, the gradient of a normalised group is all rounding
        least = -(-16 // cg)
        s = int(math.exp(rng.uniform(math.log(least), math.log(min(most, 96 * 272 * 480)))))
        d = max(1, min(96, int(s ** (1 / 3) * rng.uniform(0.3, 1))))
        h = max(1, int((s / d) ** 0.5 * rng.uniform(0.5, 1)))
        w = max(1, s // (d * h))
        if d * h * w < least:
            w = least
        case = _norm("", n, d, h, w, c, groups, dtype, rng.choice(["none", "relu", "relu", "silu"]), residual, train, rng.random() < 0.2)
    del case["name"]
    return case


def _lengths(case):
    """Lengths of the tensors of a clip case: the aggregator's own, or spread over their logarithm with the given sum."""
    if case["model"] == "gcnet":
        convs = [(8, 32), (32, 32), (32, 64)] + [(64, 64)] * 8 + [(64, 128), (128, 128), (128, 128), (128, 64), (64, 64), (64, 64), (64, 32)]
        return [v for ci, co in convs for v in (27 * ci * co, co, co)] + [27 * 32, 1]
    k, total = case["tensors"], case["total"]
    r = random.Random(k * 1_000_003 + total)
    parts = [math.exp(r.uniform(0, 7)) for _ in range(k)]
    scale = (total - k) / sum(parts)
    lengths = [1 + int(p * scale) for p in parts]
    lengths[r.randrange(k)] += total - sum(lengths)
    return lengths


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "clip":
        lengths = _lengths(case)
        # gradients of one model lie next to each other, each layer with a magnitude of its own
        flat = randn(sum(lengths))
        for part in flat.split(lengths):
            part.mul_(0.02 * torch.exp(randn(1)))
        norm = float(flat.double().square().sum().sqrt())
        flat = flat.to(dtype)
        out = torch.empty_like(flat, dtype=DTYPES[case["out_dtype"]])
        return {"case": case, "grads": list(flat.split(lengths)), "out": list(out.split(lengths)), "flat_out": out,
                "max_norm": norm / case["ratio"]}
    shape, c = (case["n"], case["d"], case["h"], case["w"]), case["c"]
    wide = 2 * c if case["sliced"] else c
    x = torch.empty(*shape, wide, device="cuda", dtype=dtype)
    x.copy_(randn(*shape, wide) * (0.5 + torch.rand(wide, device="cuda", generator=g)) + randn(wide))    # a conv's outputs: each channel its own mean and width
    state = {"case": case, "x": x[..., wide - c:], "weight": 1 + 0.3 * randn(c), "bias": 0.3 * randn(c), "residual": None}
    if case["residual"]:
        state["residual"] = randn(*shape, c).clamp_min_(0).to(dtype)
    if case["train"]:
        state["dy"] = randn(*shape, c).to(dtype)
        for k in ("x", "weight", "bias", "residual"):
            if state[k] is not None:
                state[k].requires_grad_()
    return state


def _plain_clip(grads, max_norm, flat_out):
    flat = torch.cat(grads).float()
    total = flat.square().sum(dtype=torch.float64).sqrt()
    factor = (max_norm / (total + 1e-6)).clamp(max=1.0).float()
    flat_out.copy_(flat * factor)
    return total.float()


def _plain_norm(x, groups, weight, bias, act, residual, dy=None):
    shape, c = x.shape, x.shape[-1]
    dtype, n, cg = x.dtype, shape[0], c // groups
    x = x.detach().reshape(n, -1, c).float()
    weight, bias = weight.detach(), bias.detach()
    res = None if residual is None else residual.detach().reshape(n, -1, c)

    def per_channel(v):                        # [n, groups] -> [n, 1, c]
        return v.repeat_interleave(cg, 1).unsqueeze(1)

    def group_mean(v):
        return v.sum(1, dtype=torch.float64).view(n, groups, cg).sum(2) / (v.shape[1] * cg)

    mean = group_mean(x)
    centred = x - per_channel(mean).float()
    off = group_mean(centred)                  # what rounding the mean to 32 bits left
    centred = centred - per_channel(off).float()
    var = group_mean(centred.square())
    rstd = 1 / torch.sqrt(var + EPS)
    xhat = centred * per_channel(rstd).float()
    del centred
    z = xhat * weight + bias
    if res is not None:
        z = z + res.float()
    y = z if act == "none" else z.clamp_min(0) if act == "relu" else z / (1 + torch.exp(-z))
    out = {"y": y.to(dtype).view(shape)}
    if dy is None:
        return out
    dz = dy.reshape(n, -1, c).float()
    if act == "relu":                          # on which side of the border: in 64 bits
        z = (x.double() - per_channel(mean)) * per_channel(rstd) * weight.double() + bias.double()
        if res is not None:
            z = z + res.double()
        dz = torch.where(z > 0, dz, torch.zeros_like(dz))
    elif act == "silu":
        sig = 1 / (1 + torch.exp(-z))
        dz = dz * (sig * (1 + z * (1 - sig)))
    del x, y, z
    out["dbias"] = dz.sum((0, 1), dtype=torch.float64).float()
    out["dweight"] = (dz * xhat).sum((0, 1), dtype=torch.float64).float()
    if res is not None:
        out["dresidual"] = dz.to(dtype).view(shape)
    dz = dz * weight
    c1, c2 = group_mean(dz), group_mean(dz * xhat)
    dx = (dz - per_channel(c1).float() - xhat * per_channel(c2).float()) * per_channel(rstd).float()
    out["dx"] = dx.to(dtype).view(shape)
    return out


def run(state):
    case = state["case"]
    if case["op"] == "clip":
        if own:
            from msnets_amd import hipops
            norm = hipops.clip_grads(state["grads"], state["max_norm"], out=state["out"])
        else:
            norm = _plain_clip(state["grads"], state["max_norm"], state["flat_out"])
        return {"norm": norm, "grads": state["flat_out"]}
    x, weight, bias, residual, dy = state["x"], state["weight"], state["bias"], state["residual"], state.get("dy")
    if not own:
        return _plain_norm(x, case["groups"], weight, bias, case["act"], residual, dy)
    from msnets_amd import hipops
    y = hipops.group_norm(x, case["groups"], weight, bias, eps=EPS, act=case["act"], residual=residual)
    if dy is None:
        return {"y": y}
    names = ["x", "weight", "bias"] + (["residual"] if residual is not None else [])
    grads = torch.autograd.grad(y, [state[k] for k in names], dy)
    return {"y": y.detach(), **{"d" + k: v for k, v in zip(names, grads)}}


def work(case):
    if case["op"] == "clip":
        total = sum(_lengths(case))
        return {"bytes": total * (BYTES[case["dtype"]] + BYTES[case["out_dtype"]]) + 4, "flops": 3 * total}
    values = case["n"] * case["d"] * case["h"] * case["w"] * case["c"]
    tensors = 2 + case["residual"]                          # x, y, the residual
    params = 2
    if case["train"]:
        tensors += 2 + case["residual"]                     # dy, dx, the residual's gradient
        params += 2
    return {"bytes": values * tensors * BYTES[case["dtype"]] + 4 * params * case["c"], "flops": values * (22 if case["train"] else 8)}


def exact(case, seed):
    """The same outputs from the definitions in 64 bits; the gradients by differentiating the forward formula."""
    state = prepare(case, seed)
    if case["op"] == "clip":
        flat = torch.cat(state["grads"]).double()
        norm = torch.linalg.vector_norm(flat)
        factor = min(1.0, state["max_norm"] / (float(norm) + 1e-6))
        return {"norm": norm, "grads": flat * factor}
    leaf = {k: state[k].detach().double().requires_grad_(case["train"]) for k in ("x", "weight", "bias", "residual") if state[k] is not None}
    n, g, c = case["n"], case["groups"], case["c"]
    x = leaf["x"].reshape(n, -1, g, c // g)
    mean = x.mean((1, 3), keepdim=True)
    x = x - mean
    x = x * (x.square().mean((1, 3), keepdim=True) + EPS).rsqrt()
    z = x.reshape(leaf["x"].shape) * leaf["weight"] + leaf["bias"]
    if "residual" in leaf:
        z = z + leaf["residual"]
    y = torch.relu(z) if case["act"] == "relu" else z * torch.sigmoid(z) if case["act"] == "silu" else z
    if not case["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, list(leaf.values()), state["dy"].double())
    return {"y": y.detach(), **{"d" + k: v for k, v in zip(leaf, grads)}}
