"""What the layer-norm and gradient-norm entry points refuse, before anything reaches a device (there is none here)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import multigputrainmlp_b200 as mgt  # noqa: E402
from multigputrainmlp_b200 import _lib  # noqa: E402
from multigputrainmlp_b200.api import _Tensor  # noqa: E402

A = dict(dy=0x100000, x=0x200000, gamma=0x300000, beta=0x310000, y=0x400000, mean=0x500000, rstd=0x510000, dx=0x600000, dgamma=0x700000,
         dbeta=0x710000, dbias=0x720000, workspace=0x800000)


def forward(cfg, **bad):
    a = dict(A, **bad)
    return mgt.launch_layer_norm(cfg, a["x"], a["gamma"], a["beta"], a["y"], a["mean"], a["rstd"], stream=0)


def backward(cfg, floats=None, **bad):
    a = dict(A, **bad)
    floats = mgt.layer_norm_backward_workspace_floats(cfg) if floats is None else floats
    return mgt.launch_layer_norm_backward(cfg, a["dy"], a["x"], a["gamma"], a["mean"], a["rstd"], a["dx"], a["dgamma"], a["dbeta"], a["dbias"], a["workspace"],
                                          floats, stream=0)


@pytest.mark.parametrize("bad", [dict(cols=0), dict(cols=(1 << 20) + 1), dict(cols=-1), dict(rows=-1), dict(rows=2**32), dict(eps=0.0), dict(eps=-1e-5), dict(eps=float("nan")),
                                 dict(eps=float("inf")), dict(x_type=3), dict(x_type=-1), dict(y_type=7), dict(dx_type=5), dict(x_pitch=7), dict(y_pitch=1),
                                 dict(dx_pitch=7), dict(x_pitch=-8), dict(x_type=mgt.F16, y_type=mgt.BF16), dict(x_type=mgt.BF16, y_type=mgt.F16),
                                 dict(x_type=mgt.F16, dx_type=mgt.F32), dict(x_type=mgt.F32, y_type=mgt.F16, dx_type=mgt.F16), dict(dx_type=mgt.F16, y_type=mgt.F16)])
def test_configurations_that_are_refused(bad):
    cfg = mgt.LayerNormConfig(**dict(dict(rows=4, cols=8), **bad))
    assert mgt.validate_layer_norm_config(cfg) == 1
    assert forward(cfg) == 1 and mgt.layer_norm_backward_workspace_floats(cfg) == 0 and backward(cfg, floats=1 << 30) == 1


def test_configurations_that_hold():
    for x, y, dx in ((mgt.F32, mgt.F32, None), (mgt.F32, mgt.F32, mgt.F16), (mgt.F32, mgt.F32, mgt.BF16), (mgt.F32, mgt.F16, None), (mgt.F32, mgt.BF16, None),
                     (mgt.F16, mgt.F16, None), (mgt.F16, mgt.F32, None), (mgt.BF16, mgt.BF16, None), (mgt.BF16, mgt.F32, None)):
        assert mgt.validate_layer_norm_config(mgt.LayerNormConfig(4, 1 << 20, x_type=x, y_type=y, dx_type=dx)) == 0
    assert mgt.validate_layer_norm_config(mgt.LayerNormConfig(0, 1)) == 0


@pytest.mark.parametrize("name", ["x", "y"])
def test_forward_arrays(name):
    cfg = mgt.LayerNormConfig(4, 8)
    assert forward(cfg, **{name: None}) == 1
    assert forward(cfg, **{name: A[name] + 2}) == 1   # half an element
    assert forward(mgt.LayerNormConfig(4, 8, x_type=mgt.F16, y_type=mgt.F16), **{name: A[name] + 1}) == 1
    for other in ("gamma", "beta", "mean", "rstd"):
        assert forward(cfg, **{other: A[other] + 2}) == 1


@pytest.mark.parametrize("name", ["dy", "x", "dx", "mean", "rstd", "workspace"])
def test_backward_arrays(name):
    cfg = mgt.LayerNormConfig(4, 8)
    assert backward(cfg, **{name: None}) == 1
    assert backward(cfg, **{name: A[name] + 2}) == 1
    assert backward(cfg, workspace=A["workspace"] + 4) == 1
    for other in ("gamma", "dgamma", "dbeta", "dbias"):
        assert backward(cfg, **{other: A[other] + 1}) == 1
    assert backward(cfg, floats=mgt.layer_norm_backward_workspace_floats(cfg) - 1) == 3
    assert backward(mgt.LayerNormConfig(4, 9000), floats=mgt.layer_norm_backward_workspace_floats(mgt.LayerNormConfig(4, 8))) == 3


def test_host_tensors_are_refused():
    if torch.cuda.is_available():
        pytest.skip("for machines without a device: here the current device is asked for")
    cfg = mgt.LayerNormConfig(4, 8)
    assert mgt.launch_layer_norm(cfg, torch.zeros(4, 8), None, None, torch.zeros(4, 8), stream=0) == 1
    with pytest.raises(mgt.MgtError):
        mgt.TensorList([torch.zeros(4)])
    with pytest.raises(mgt.MgtError):
        mgt.TensorList([])


def entries(*rows):
    array = (_Tensor * max(1, len(rows)))()
    for e, (data, count, kind) in zip(array, rows):
        e.data, e.count, e.type = data, count, kind
    return array


def test_tensor_lists():
    lib = _lib.load()
    floats = lambda array, n: int(lib.mgt_gradient_norm_workspace_floats(ctypes.cast(array, ctypes.c_void_p), n))  # noqa: E731
    good = entries((0x1000, 10, 0), (0x2002, 3, 1), (0x3002, 0, 2), (None, 0, 0))
    assert floats(good, 4) > 0
    assert floats(good, 0) == 0 and floats(None, 1) == 0
    for bad in ((0x1002, 10, 0), (0x1001, 10, 1), (None, 10, 0), (0x1000, 10, 3), (0x1000, 10, -1), (0x1000, (1 << 40) + 1, 0)):
        assert floats(entries(bad), 1) == 0, bad
    assert floats(entries((0x1000, 1 << 40, 0)), 1) > 0
    assert floats(entries((0x1000, 1 << 40, 0), (0x1000, 1, 0)), 2) == 0  # together too many
    many = entries(*[(0x1000, 4, 0)] * 1025)
    assert floats(many, 1024) > 0 and floats(many, 1025) == 0


def test_gradient_norm_and_clip_arguments():
    lib = _lib.load()
    two = ctypes.cast(entries((0x1000, 10, 0), (0x2002, 3, 1)), ctypes.c_void_p)
    run = lambda max_norm=1.0, result=0x4000, norms=0x5000, ws=0x6000, floats=1 << 20: int(  # noqa: E731
        lib.mgt_launch_gradient_norm(two, 2, max_norm, result, norms, ws, floats, None))
    assert run(max_norm=0.0) == 1 and run(max_norm=-1.0) == 1 and run(max_norm=float("nan")) == 1
    assert run(result=None) == 1 and run(result=0x4002) == 1 and run(norms=0x5002) == 1 and run(ws=None) == 1 and run(ws=0x6004) == 1
    assert run(floats=int(lib.mgt_gradient_norm_workspace_floats(two, 2)) - 1) == 3
    clip = lambda out, n=2, result=0x4000: int(lib.mgt_launch_clip_gradients(two, n, result, ctypes.cast(out, ctypes.c_void_p) if out is not None else None, None))  # noqa: E731
    assert clip(None, n=0) == 1 and clip(None, result=None) == 1 and clip(None, result=0x4001) == 1
    for bad in (((0x1000, 9, 0), (0x2002, 3, 1)), ((0x1000, 10, 0), (0x2002, 3, 2)), ((0x1002, 10, 0), (0x2002, 3, 1)), ((None, 10, 0), (0x2002, 3, 1))):
        assert clip(entries(*bad)) == 1
    cfg = mgt.AdamWKernelConfig(8, 1, 1e-3)
    adamw = lambda clip_at=0x4000, w=0x10000: mgt.launch_adamw_kernel_with_clip(cfg, w, None, 0x20000, clip_at, 0x30000, 0x40000, stream=0)  # noqa: E731
    assert adamw(clip_at=None) == 1 and adamw(clip_at=0x4002) == 1 and adamw(w=0x10004) == 1


def test_workspace_of_layer_norm_never_shrinks_with_the_batch():
    for dims, batches in (((72, 72, 333, 77, 3, 1), range(1, 40000, 401)), ((72, 72, 2560, 224, 16, 1), range(3500, 3800)), ((16, 16, 64, 512, 0, 2), range(1, 300))):
        shape = mgt.CudaMlpShape(*dims)
        for half_table in (True, False):
            sizes = [mgt.mlp_loss_grad_workspace_floats(shape, b, 1, half_table, layer_norm=True) for b in batches]
            assert sizes[0] > 0 and all(x <= y for x, y in zip(sizes, sizes[1:]))
    shape = mgt.CudaMlpShape(16, 16, 64, 64, 1, 1)
    assert mgt.mlp_loss_grad_workspace_floats(shape, 64, layer_norm=True, use_half_linear=False) == 0  # fp32 layers have no normalisation
    assert mgt.mlp_loss_grad_workspace_floats(shape, 64, layer_norm=True, batch_norm=True) == 0
    assert mgt.mlp_loss_grad_workspace_floats(shape, 0, layer_norm=True) == 0


def test_clipping_refuses_tensors_that_share_memory():
    """(On a machine with a GPU only the refusals are made: the addresses are no memory.)"""
    lib = _lib.load()
    clip = lambda rows, out=None: int(lib.mgt_launch_clip_gradients(  # noqa: E731
        ctypes.cast(entries(*rows), ctypes.c_void_p), len(rows), 0x4000, ctypes.cast(entries(*out), ctypes.c_void_p) if out else None, None))
    a, b, c = (0x1000, 10, 0), (0x1028, 8, 1), (0x1038, 8, 2)  # side by side: 40 bytes, 16, 16
    for rows in ((a, a), (a, b, a), ((0x1024, 4, 0), a), (a, (0x1026, 1, 1)), (b, c, (0x1036, 1, 1)), (c, b, (0x1028, 4, 2)), (a, (None, 0, 0), (0x1000, 1, 0))):
        assert clip(rows) == 1, rows
    far = [(0x9000 + d - 0x1000, n, k) for d, n, k in (a, b, c)]
    for out in ([far[0], far[0][:1] + (8, 1), far[2]], [(0x1004, 10, 0), far[1], far[2]], [(0x1038, 10, 0), far[1], far[2]], [far[0], (0x1000, 8, 1), far[2]],
                [far[0], far[1], (0x1028, 8, 2)]):
        assert clip((a, b, c), out) == 1, out
    if not torch.cuda.is_available():  # what fits reaches the launch, which has no device here
        assert clip((a, b, c)) == 4 and clip((c, a, b)) == 4 and clip((a, b, c), far) == 4 and clip((c, a, b), (c, a, b)) == 4
        assert clip((a, (0x1000, 0, 0), b)) == 4 and clip((b, a), ((0xfe0, 8, 1), (0x1038, 10, 0))) == 4
