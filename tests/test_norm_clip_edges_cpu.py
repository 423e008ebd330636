"""The host side of hipops.group_norm, grad_norm and clip_grads at calls off the ordinary path."""
import pytest
import torch

import msnets_amd  # noqa: F401
from msnets_amd import hipops


def test_graphs_are_refused_in_grad_mode_only():
    p = torch.ones(3, requires_grad=True)
    with pytest.raises(ValueError, match="grads\\[2\\] requires a gradient"):
        hipops._refuse_graph(p * 2, "grads[2]")
    hipops._refuse_graph(p.detach(), "t")
    with torch.no_grad():
        hipops._refuse_graph(p, "t")


def _bytes_of(t):
    first = t.data_ptr()
    at = torch.zeros((), dtype=torch.int64)
    for s, n in zip(t.stride(), t.shape):
        at = at[..., None] + torch.arange(n) * s
    at = at.reshape(-1) * t.element_size() + first
    return at, set((at[:, None] + torch.arange(t.element_size())).reshape(-1).tolist())


def _random_view(base, rng):
    """A view of base's memory, now and then one whose values share places."""
    flat = base.view(torch.bfloat16) if rng.random() < 0.3 else base
    dims = rng.randint(0, 4)
    shape = [rng.randint(1, 4) for _ in range(dims)]
    if rng.random() < 0.6:                     # nested, in any order: a slice of a dense tensor
        at, stride = 1, [0] * dims
        for i in rng.sample(range(dims), dims):
            stride[i] = at * rng.choice([1, 1, 1, 2, 3])
            at = stride[i] * (shape[i] + rng.randint(0, 1))
    else:
        stride = [rng.randint(0, 12) for _ in range(dims)]
    reach = sum((n - 1) * s for n, s in zip(shape, stride))
    if reach >= flat.numel():
        return flat[:5]
    return flat.as_strided(shape, stride, rng.randint(0, min(flat.numel() - reach - 1, 60)))


def test_overlaps_of_any_strides():
    """Against the places listed one by one."""
    import random
    rng, base, seen = random.Random(0), torch.zeros(4000), [0, 0, 0]
    for _ in range(3000):
        a, b = _random_view(base, rng), _random_view(base, rng)
        (pa, sa), (_, sb) = _bytes_of(a), _bytes_of(b)
        assert hipops._overlap(a, b) == hipops._overlap(b, a) == bool(sa & sb), (a.shape, a.stride(), b.shape, b.stride())
        own = len(sa) < a.numel() * a.element_size()
        assert hipops._overlaps_itself(a) == own, (a.shape, a.stride())
        seen[0] += bool(sa & sb)
        seen[1] += not sa & sb and a.data_ptr() < b.data_ptr() < a.data_ptr() + max(sa) - min(sa)
        seen[2] += own
    assert min(seen) > 100, seen
    assert not hipops._overlap(base[:0], base) and not hipops._overlaps_itself(base[:0])
    # hard to say within the budget: taken for an overlap
    wide = torch.empty(1, dtype=torch.float32).as_strided((1,), (1,))
    assert hipops._reaches([(2 ** 20 + 2 * k, 0, 2 ** 12) for k in range(12)], 2 ** 33 + 1) and wide.numel() == 1


def test_overlaps_in_lists():
    """Three outputs and three gradients in the same memory, some in place: refused if a written place belongs to anything else."""
    import random
    rng, base, refused = random.Random(1), torch.zeros(4000), 0
    for _ in range(3000):
        outs = [_random_view(base, rng) for _ in range(3)]
        grads = [o if rng.random() < 0.7 else _random_view(base[500 * rng.randint(0, 1):], rng) for o in outs]
        places = [_bytes_of(t)[1] for t in outs + grads]
        layout = lambda t: (t.data_ptr(), t.dtype, [(k, n) for k, n in zip(t.stride(), t.shape) if n > 1])      # noqa: E731
        want = any(places[i] & places[j] for i in range(3) for j in range(i + 1, 6) if j != i + 3 or layout(outs[i]) != layout(grads[i]))
        try:
            hipops._check_overlaps(grads, outs)
            assert not want
        except RuntimeError:
            assert want
            refused += 1
    assert 500 < refused < 2900, refused


def test_clipping_refuses_overlaps_of_any_strides(monkeypatch):
    monkeypatch.setattr(hipops, "_require_gpu", lambda t, name: t)          # (the layout is host code: any tensors will do)
    base, spare = torch.zeros(10, 12), [torch.zeros(10, 6), torch.zeros(10, 6)]
    even, odd, left = base[:, ::2], base[:, 1::2], base[:, :3]
    for bad in ([even, even], [base, left], [left, base], [even, base[:, 2:4]], [base[:, :6].t(), base[3:4, 5:7]], [even[2], base[:, 4]]):
        with pytest.raises(RuntimeError, match="overlaps"):
            hipops._clip_layout(bad, bad)
        hipops._clip_layout(bad, [torch.zeros_like(t) for t in bad])          # read only
    for src, dst in ((spare, [even, even]), (spare, [base[:, :6], base[:, 5:11]]), ([even, spare[0]], [spare[1], even]), ([base[:, 1:7]], [base[:, :6]]),
                     ([even.bfloat16(), base[:, 6:]], [even, spare[0]])):
        with pytest.raises(RuntimeError, match="overlaps"):
            hipops._clip_layout(src, dst)
    for shared in (torch.zeros(40).as_strided((4, 3), (2, 1)), torch.zeros(40).as_strided((3, 4, 2), (4, 2, 3))):
        with pytest.raises(ValueError, match="overlaps itself"):
            hipops._clip_layout([shared], [shared])
        hipops._clip_layout([shared], [torch.zeros(shared.shape)])
    for good in ([even, odd], [base[:, :6], base[:, 6:]], [base[:, 3 * i:3 * i + 3].t() for i in range(4)], [even[:, None], odd[3:]], [base[:5], base.t()[:, 5:]]):
        src, dst, back = hipops._clip_layout(good, good)
        assert len(src) == len(dst) == len(good)
    wide = torch.zeros(64, 4000)
    columns = [wide[:, i:i + 8] for i in range(0, 4000, 8)]                    # many slices of one matrix
    assert len(hipops._clip_layout(columns, columns)[2]) == 500
    for one in (wide[7:9, 100:101], wide[:, 3992:], wide.t()[3999:]):
        with pytest.raises(RuntimeError, match="overlaps"):
            hipops._clip_layout(columns + [one], columns + [one])
    around = [wide[1:40, :7], wide[:39, 4:4000:4000], wide.view(-1)[4000 * 50:4000 * 50 + 6]]
    around += [torch.as_strided(wide, (38, 8), (4000, 1), 3996)]                # rows that go over a row's end
    with pytest.raises(RuntimeError, match="overlaps"):
        hipops._clip_layout(around, around)
    assert hipops._overlap(around[0], around[3]) and not hipops._overlap(around[1], around[2])


def test_out_over_the_parameters():
    base = torch.zeros(1000)
    out = base[:960].view(2, 20, 24)[..., :8]
    check = hipops._check_out_params
    check(out, None, None)
    check(out, torch.zeros(8), base[960:968])
    check(out, base[8:16], base[24 * 5 + 16:24 * 6])                            # between its rows
    check(out[:0], base[:8])
    for bad in (base[:8], base[4:12], base[17:25], base[24 * 39:24 * 39 + 8], base.view(torch.bfloat16)[14:22]):
        for params in ((bad, None), (None, bad), (torch.zeros(8), bad)):
            with pytest.raises(ValueError, match="weight or bias"):
                check(out, *params)


def test_the_same_memory_with_other_strides_of_single_entries(monkeypatch):
    """In place through another view: the strides of dimensions of one entry do not matter."""
    monkeypatch.setattr(hipops, "_require_gpu", lambda t, name: t)
    base = torch.zeros(40)
    t, o = base[:5].view(1, 5), base.as_strided((1, 5), (99, 1))
    other = torch.zeros(6, 4)[:, ::2]
    assert len(hipops._clip_layout([t, other], [o, other])[0]) == 2
    with pytest.raises(RuntimeError, match="overlaps"):
        hipops._clip_layout([t, other], [base[1:6].view(1, 5), other])


def test_c_entry_overlaps(hiplib):
    """Lists of contiguous tensors, in order and out of it, empty ones among them: refused where a written byte belongs to another
    tensor of the call.  (Lists that are taken are launched: those are compared on the GPU.)"""
    import ctypes
    import random
    rng, seen = random.Random(2), [0, 0]
    size = {0: 4, 1: 2, 2: 2}

    def call(src, dst, n, st, dt, ws):
        k = len(n)
        return hiplib.msnet_clip_grads((ctypes.c_uint64 * k)(*src), (ctypes.c_uint64 * k)(*dst), (ctypes.c_int64 * k)(*n), bytes(st), bytes(dt), k, 1.0,
                                       ctypes.c_void_p(1 << 20), ws, 1 << 16, None)
    for trial in range(4000):
        k = rng.randint(1, 5)
        n = [rng.choice([0, 1, 2, 3, 5, 8]) for _ in range(k)]
        dt = [rng.choice([0, 0, 1, 2]) for _ in range(k)]
        st = [rng.choice([1, 2, 0]) if d == 0 else d for d in dt]
        place = lambda at, t: [at.append(at[-1] + n[i] * size[t[i]] + 4 * rng.choice([0, 0, 1, 3])) or at[-2] for i in range(k)]      # noqa: E731
        dst, src = place([4096], dt), place([rng.choice([4096, 4100, 4160, 8192, 16384])], st)
        for t in (dst, src):
            if rng.random() < 0.3:
                rng.shuffle(t)
        for i in range(k):
            if rng.random() < 0.4 and st[i] == dt[i]:
                src[i] = dst[i]
        if rng.random() < 0.2:
            dst[rng.randrange(k)] += rng.choice([-4, 4])
        out = [set(range(dst[i], dst[i] + n[i] * size[dt[i]])) for i in range(k)]
        read = [set(range(src[i], src[i] + n[i] * size[st[i]])) for i in range(k)]
        want = any(out[i] & out[j] for i in range(k) for j in range(i)) or any(
            out[i] & read[j] for i in range(k) for j in range(k) if not (src[j] == dst[j] and st[j] == dt[j] and i == j))
        if not want:
            seen[0] += 1
            continue
        assert call(src, dst, n, st, dt, ctypes.c_void_p(1 << 20)) != 0 and b"overlaps" in hiplib.msnet_last_error(), (src, dst, n, st, dt)
        seen[1] += 1
    assert min(seen) > 1000, seen
