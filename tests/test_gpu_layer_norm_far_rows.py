"""Backward pass of rows so far from zero that mean * rstd is beyond the floats, though every x - mean is small: what a thread holds beyond the
row's end must not enter its sums. Bounds as in test_gpu_layer_norm.py."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import multigputrainmlp_b200 as mgt  # noqa: E402
from test_gpu_layer_norm import DEV, TYPES, check_backward  # noqa: E402

TINY = 1e-30  # eps: rstd is 1e15 where a row has no spread


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1, 3, 12, 20, 24, 77, 88, 96, 200, 301, 500, 600, 1000, 1028, 2049, 2056, 3000, 5001, 5004, 6000, 9000, 10001, 12000, 16383, 20000])
@pytest.mark.parametrize("rows", [7, 700])
def test_rows_far_from_zero(rows, cols, kind):
    g = torch.Generator(device=DEV).manual_seed(cols)
    x = torch.randn(rows, cols, device=DEV, generator=g)
    x[::2] = 2.0 ** 90 * (1 + torch.arange((rows + 1) // 2, device=DEV)[:, None] % 3)  # (1.2e27 to 3.7e27: times rstd 1e42; up to 2^100 in a row's sum)
    x = x.to(TYPES[kind][1])
    dy = torch.randn(rows, cols, device=DEV, generator=g).to(x.dtype)
    gamma = 1.0 + 0.3 * torch.randn(cols, device=DEV, generator=g)
    mean = x.double().mean(1)
    mean, rstd = mean.float(), ((x.double() - mean[:, None]).square().mean(1) + TINY).rsqrt().float()
    assert (mean[::2, None] == x[::2].float()).all() and (rstd[::2] > 9e14).all() and torch.isfinite(rstd).all()
    cfg = mgt.LayerNormConfig(rows, cols, TINY, TYPES[kind][0], TYPES[kind][0])
    floats = mgt.layer_norm_backward_workspace_floats(cfg)
    dx, sums = torch.empty_like(x), [torch.empty(cols, device=DEV) for _ in range(3)]
    assert mgt.launch_layer_norm_backward(cfg, dy, x, gamma, mean, rstd, dx, *sums, torch.empty(floats, device=DEV), floats) == 0
    check_backward(dy, x, gamma, mean, rstd, dx, kind, sums)
