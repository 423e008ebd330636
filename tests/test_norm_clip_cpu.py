"""What hipops.group_norm, grad_norm and clip_grads refuse before any launch, and the host-side helpers they lay tensors out with."""
import ctypes

import pytest
import torch

import msnets_amd  # noqa: F401
from msnets_amd import driver_utils, hipops
from msnets_amd.gcnet_3dcnn import GCNet_CostVolumeAggre
from msnets_amd.psmnet_3dcnn import PSMNet_CostVolumeAggre

FAKE = ctypes.c_void_p(1 << 20)              # never read: every call below fails on the host


def test_no_cpu_path():
    x = torch.zeros(1, 4, 8)
    with pytest.raises(RuntimeError, match="MI355X"):
        hipops.group_norm(x, 2)
    with pytest.raises(RuntimeError, match="MI355X"):
        hipops.clip_grads([x], 1.0)
    with pytest.raises(RuntimeError, match="MI355X"):
        hipops.grad_norm(x)
    with pytest.raises(TypeError):
        hipops.group_norm([1.0], 2)
    with pytest.raises(TypeError):
        hipops.clip_grads([x.to_sparse()], 1.0)
    p = torch.nn.Parameter(x)
    assert float(driver_utils.clip_grad_norm_([p], 1.0)) == 0


def test_c_entry_refusals_of_the_norm(hiplib):
    def call(x=FAKE, y=FAKE, stats=None, dtype=0, act=0, n=1, s=4, c=8, g=2, eps=1e-5, strides=(32, 8, 0, 0, 32, 8), ws=None, nbytes=0):
        return hiplib.msnet_group_norm(x, None, None, None, y, stats, dtype, act, n, s, c, g, eps, *strides, ws, nbytes, None)
    for bad, word in ((dict(dtype=3), b"dtype"), (dict(dtype=-1), b"dtype"), (dict(act=3), b"activation"), (dict(n=-1), b"shape"), (dict(s=-1), b"shape"),
                      (dict(c=0), b"shape"), (dict(g=3), b"groups"), (dict(g=0), b"groups"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"),
                      (dict(x=None), b"null"), (dict(y=None), b"null"), (dict(strides=(32, -8, 0, 0, 32, 8)), b"stride"),
                      (dict(stats=ctypes.c_void_p(8)), b"aligned"), (dict(s=1 << 22), b"workspace"), (dict(s=1 << 22, ws=FAKE, nbytes=16), b"workspace"),
                      (dict(n=2147483647, c=64, g=64), b"too many")):
        assert call(**bad) != 0 and word in hiplib.msnet_last_error(), bad
    assert call(n=0, x=None, y=None) == 0 and call(s=0, x=None, y=None) == 0
    size = hiplib.msnet_group_norm_workspace_bytes
    assert size(0, 1, 10, 32, 8) == 0 and size(0, 1, 96 * 272 * 480, 32, 8) > 0 and size(0, 1, 96, 32, 7) == 0

    def back(dy=FAKE, stats=FAKE, res=None, dres=None, act=1, s=4, ws=None, nbytes=0):
        return hiplib.msnet_group_norm_backward(dy, FAKE, None, None, res, stats, FAKE, dres, None, None, 0, act, 1, s, 8, 2, 32, 8, 32, 8, 0, 0, ws,
                                                nbytes, None)
    for bad, word in ((dict(dy=None), b"null"), (dict(stats=None), b"null"), (dict(dres=FAKE), b"residual"), (dict(dres=FAKE, res=FAKE, act=0), b"itself"),
                      (dict(s=1 << 22), b"workspace"), (dict(act=7), b"activation")):
        assert back(**bad) != 0 and word in hiplib.msnet_last_error(), bad


def test_c_entry_refusals_of_clipping(hiplib):
    arr = lambda kind, *v: (kind * len(v))(*v)                                          # noqa: E731
    q, n = ctypes.c_uint64, ctypes.c_int64

    def call(src=(1 << 20,), dst=(1 << 20,), lengths=(10,), st=b"\0", dt=b"\0", count=1, max_norm=1.0, norm=FAKE, ws=FAKE, nbytes=1 << 16):
        return hiplib.msnet_clip_grads(arr(q, *src) if src else None, arr(q, *dst) if dst else None, arr(n, *lengths), st, dt, count, max_norm, norm, ws,
                                       nbytes, None)
    for bad, word in ((dict(count=-1), b"tensors"), (dict(lengths=(-1,)), b"values"), (dict(norm=None), b"null"), (dict(src=None), b"null"),
                      (dict(src=(0,)), b"null"), (dict(max_norm=-1.0), b"max_norm"), (dict(max_norm=float("nan")), b"max_norm"), (dict(ws=None), b"workspace"),
                      (dict(nbytes=8), b"workspace"), (dict(st=b"\3"), b"types"), (dict(st=b"\1", dt=b"\2"), b"types"), (dict(st=b"\0", dt=b"\1"), b"types"),
                      (dict(dst=((1 << 20) + 4,)), b"overlaps"), (dict(dst=((1 << 20) - 4,)), b"overlaps")):
        assert call(**bad) != 0 and word in hiplib.msnet_last_error(), bad
    two = dict(count=2, lengths=(10, 10), st=b"\0\0", dt=b"\0\0")
    for src, dst in (((4096, 4096), (4096, 4096)), ((4096, 4136), (8192, 4136 + 36)), ((4096, 8192), (16384, 4100)), ((8192, 4096), (8192, 4096 + 4))):
        assert call(src=src, dst=dst, **two) != 0 and b"overlaps" in hiplib.msnet_last_error(), (src, dst)
    size = hiplib.msnet_clip_grads_workspace_bytes
    assert 0 < size(arr(n, 10, 0, 8193), 3) < size((n * 1000)(*[5] * 1000), 1000) and size(arr(n, -1), 1) == 0


def test_row_strides():
    f = hipops._row_strides
    x = torch.zeros(2, 3, 4, 5, 24)
    assert f(x) == (1440, 24) and f(x[..., 8:16]) == (1440, 24) and f(x[..., :1]) == (1440, 24)
    assert f(x.transpose(1, 2)) is None and f(x[:, :, ::2]) is None and f(x[..., ::2]) is None and f(x[:, :, :, ::2]) is None and f(x[:, :, :, ::5]) == (1440, 120)
    assert f(x[:, :1, :1]) == (1440, 24) and f(x[:1].expand(7, 3, 4, 5, 24)) == (0, 24) and f(x[:, :1, :1, :1]) == (1440, 0)
    assert f(torch.zeros(3, 8)) == (8, 8) and f(torch.zeros(24).expand(2, 5, 24)) == (0, 0)


def test_out_overlaps():
    base = torch.zeros(2, 10, 24)
    ok = hipops._check_out
    ok(base[..., :8], base[..., 8:16], "x")
    ok(base[..., 16:], base[..., :8], "x")
    ok(base, base, "x")
    ok(base[0:1], base[1:2], "x")
    ok(torch.zeros(2, 10, 24), base, "x")
    for a, b in ((base[..., :8], base[..., 4:12]), (base[:, :9], base[:, 1:]), (base[..., 20:], base[..., 18:22]), (base.view(2, 10, 24)[:, :, :8], base)):
        with pytest.raises(ValueError, match="overlaps"):
            ok(a, b, "x")


def test_dense_in_any_order():
    t = torch.zeros(4, 6, 2, 3, 5)
    assert hipops._is_dense(t) and hipops._is_dense(t.to(memory_format=torch.channels_last_3d)) and hipops._is_dense(t.transpose(0, 3))
    assert not hipops._is_dense(t[:, ::2]) and not hipops._is_dense(t[:1].expand(4, 6, 2, 3, 5)) and hipops._is_dense(t[:, :1, :1, :1, :1].contiguous())


def test_group_normalised_aggregators():
    """norm="group": no running statistics, the same keys otherwise, the same convs from the same seed; a bad norm is refused."""
    for make in (lambda **k: GCNet_CostVolumeAggre(32, **k), lambda **k: PSMNet_CostVolumeAggre(32, **k)):
        batch, group = make().state_dict(), make(norm="group").state_dict()
        assert {k for k in batch if "running" not in k and "num_batches" not in k} == set(group)
        with pytest.raises(ValueError, match="norm must be"):
            make(norm="layer")
        with pytest.raises(ValueError):
            make(norm="group", norm_groups=7)
    torch.manual_seed(0)
    a = GCNet_CostVolumeAggre(32).state_dict()
    torch.manual_seed(0)
    b = GCNet_CostVolumeAggre(32, norm="group").state_dict()
    assert all(torch.equal(a[k], b[k]) for k in b), "the same seed gives the same convs"
