"""Tensors that do not lie as a call reads them are refused; views that do are taken as they lie."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import multigputrainmlp_b200 as mgt  # noqa: E402
from test_gpu_layer_norm import check_forward  # noqa: E402

DEV = "cuda:0"
ROWS, COLS, PITCH = 12, 40, 48


def buffer(*shape, seed=0, kind=torch.float32):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(kind)


def strided(n):
    """n floats, every second one of a buffer: enough lies behind the first."""
    return torch.full((2 * n, 2), 3.0, device=DEV)[:, 0][:n]


def forward(config=None, **args):
    a = dict(x=buffer(ROWS, COLS), gamma=torch.ones(COLS, device=DEV), beta=torch.zeros(COLS, device=DEV), y=torch.empty(ROWS, COLS, device=DEV),
             mean=torch.empty(ROWS, device=DEV), rstd=torch.empty(ROWS, device=DEV))
    a.update(args)
    return mgt.launch_layer_norm(config or mgt.LayerNormConfig(ROWS, COLS), *a.values())


def backward(config=None, **args):
    config = config or mgt.LayerNormConfig(ROWS, COLS)
    floats = mgt.layer_norm_backward_workspace_floats(config)
    a = dict(dy=buffer(ROWS, COLS, seed=1), x=buffer(ROWS, COLS), gamma=torch.ones(COLS, device=DEV), mean=torch.zeros(ROWS, device=DEV), rstd=torch.ones(ROWS, device=DEV),
             dx=torch.empty(ROWS, COLS, device=DEV), dgamma=torch.empty(COLS, device=DEV), dbeta=torch.empty(COLS, device=DEV), dbias=torch.empty(COLS, device=DEV),
             workspace=torch.empty(floats, device=DEV))
    a.update(args)
    return mgt.launch_layer_norm_backward(config, *a.values(), floats)


def update(**args):
    n = 30
    a = dict(w=torch.ones(n, device=DEV), half=None, grad=torch.ones(n, device=DEV), clip=torch.ones(2, device=DEV), m=torch.zeros(n, device=DEV), v=torch.zeros(n, device=DEV))
    a.update(args)
    return mgt.launch_adamw_kernel_with_clip(mgt.AdamWKernelConfig(n, 1, 1e-3), *a.values())


def test_vectors_are_dense():
    assert forward() == 0 and backward() == 0 and update() == 0
    for name, n in (("gamma", COLS), ("beta", COLS), ("mean", ROWS), ("rstd", ROWS)):
        kept = strided(n)
        assert forward(**{name: kept}) == 1, name
        assert (kept == 3.0).all()
    for name, n in (("gamma", COLS), ("mean", ROWS), ("rstd", ROWS), ("dgamma", COLS), ("dbeta", COLS), ("dbias", COLS),
                    ("workspace", mgt.layer_norm_backward_workspace_floats(mgt.LayerNormConfig(ROWS, COLS)))):
        assert backward(**{name: strided(n)}) == 1, name
    for name, n in (("w", 30), ("grad", 30), ("clip", 2), ("m", 30), ("v", 30)):
        assert update(**{name: strided(n)}) == 1, name
    assert update(half=torch.zeros(60, 2, device=DEV, dtype=torch.float16)[:, 0][:30]) == 1


def test_results_and_workspaces_of_the_norm_are_dense():
    t = torch.ones(100, device=DEV)
    lst = mgt.TensorList([t])
    floats = mgt.gradient_norm_workspace_floats(lst)
    ws, result, norms = torch.empty(floats, device=DEV), torch.empty(2, device=DEV), torch.empty(1, device=DEV)
    assert mgt.launch_gradient_norm(lst, 1.0, result, norms, ws, floats) == 0 and mgt.launch_clip_gradients(lst, result) == 0
    assert mgt.launch_gradient_norm(lst, 1.0, strided(2), norms, ws, floats) == 1
    assert mgt.launch_gradient_norm(lst, 1.0, result, norms, strided(floats), floats) == 1
    assert mgt.launch_clip_gradients(lst, strided(2)) == 1


def wrong_views(kind=torch.float32):
    big = buffer(64, 64, kind=kind)
    yield buffer(COLS, ROWS, kind=kind).T                    # transposed
    yield buffer(ROWS, PITCH, kind=kind)[:, :COLS]           # rows PITCH apart, which the config does not say
    yield buffer(2 * ROWS, COLS, kind=kind)[::2]             # every second row
    yield big[:ROWS, 1::2][:, :COLS]                         # every second column
    yield buffer(1, COLS, kind=kind).expand(ROWS, COLS)      # one row again and again
    yield buffer(2, ROWS, COLS, kind=kind)[:, :ROWS // 2]    # two halves with a gap between them


def test_matrices_lie_in_rows_of_the_config():
    for n, view in enumerate(wrong_views()):
        assert forward(x=view) == 1 and backward(x=view) == 1 and backward(dy=view) == 1, n
        kept = view.clone()
        assert forward(y=view) == 1 and backward(dx=view) == 1 and torch.equal(view, kept), n
    pitched = mgt.LayerNormConfig(ROWS, COLS, x_pitch=PITCH, y_pitch=PITCH, dx_pitch=PITCH)
    short = buffer(ROWS + 4, PITCH)[:ROWS - 1, :COLS]        # a row too few in the view, though not in the memory behind it
    fits = dict(x=buffer(ROWS, PITCH)[:, :COLS], y=buffer(ROWS, PITCH)[:, :COLS])
    assert forward(pitched, **fits) == 0
    assert forward(pitched, **dict(fits, x=short)) == 1 and forward(pitched, **dict(fits, y=short)) == 1
    back = dict(dy=buffer(ROWS, PITCH)[:, :COLS], x=buffer(ROWS, PITCH)[:, :COLS], dx=buffer(ROWS, PITCH)[:, :COLS])
    assert backward(pitched, **back) == 0
    assert all(backward(pitched, **dict(back, **{k: short})) == 1 for k in back)


@pytest.mark.parametrize("kind,code", [(torch.float32, mgt.F32), (torch.bfloat16, mgt.BF16)])
def test_views_that_lie_so_are_taken(kind, code):
    name = {mgt.F32: "f32", mgt.BF16: "bf16"}[code]
    values = buffer(ROWS, COLS, seed=3, kind=kind)
    config = mgt.LayerNormConfig(ROWS, COLS, x_type=code, y_type=code, x_pitch=PITCH, y_pitch=PITCH)
    holds = buffer(3, ROWS // 3, PITCH, kind=kind)
    for x in (buffer(ROWS, PITCH, kind=kind)[:, 5:5 + COLS], holds[:, :, :COLS], holds[:, None, :, 3:3 + COLS], buffer(ROWS + 3, PITCH, kind=kind)[2:, :COLS]):
        into = x[:ROWS] if x.dim() == 2 else x
        into.copy_(values.view(into.shape))
        y = torch.zeros(ROWS, PITCH, device=DEV, dtype=kind)
        assert mgt.launch_layer_norm(config, x, None, None, y[:, :COLS]) == 0
        check_forward(values, name, y[:, :COLS], None, None, None, None)  # (to the bit where x lies on the same boundaries only: sums go by layout)
        assert (y[:, COLS:] == 0).all()
    # dense, of any shape
    dense = mgt.LayerNormConfig(ROWS, COLS, x_type=code, y_type=code)
    for x in (values.view(-1), values.view(ROWS, 5, 8), values.view(ROWS // 2, 2 * COLS)):
        y = torch.empty(ROWS, COLS, device=DEV, dtype=kind)
        assert mgt.launch_layer_norm(dense, x, None, None, y) == 0
        check_forward(values, name, y, None, None, None, None)
    # one column of a matrix
    column = buffer(ROWS, PITCH, seed=4, kind=kind)
    out = torch.full((ROWS,), 9.0, device=DEV, dtype=kind)
    for x in (column[:, 7], column[:, 7:8]):
        assert mgt.launch_layer_norm(mgt.LayerNormConfig(ROWS, 1, x_type=code, y_type=code, x_pitch=PITCH), x, None, None, out) == 0
        assert (out == 0).all()
        assert mgt.launch_layer_norm(mgt.LayerNormConfig(ROWS, 1, x_type=code, y_type=code, x_pitch=PITCH + 1), x, None, None, out) == 1
