"""Layer normalisation of rows whose squares add up to more than a float holds: deviations of 1e18, which the header allows at any width. The
bounds are those of rows of ordinary size, whose derivation does not depend on it."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import multigputrainmlp_b200 as mgt  # noqa: E402
from test_gpu_layer_norm import DEV, EPS, TYPES, check_backward, check_forward, exact_forward, make  # noqa: E402

SHAPES = [(1, 2), (5, 8), (301, 8), (40, 77), (130, 224), (2500, 301), (70, 512), (50, 600), (33, 1024), (9, 2049), (30, 4096), (9, 6143), (5, 8192), (9, 9000), (5, 10001), (3, 16384),
          (3, 16385), (6, 20000), (2, 1 << 20)]


def large_rows(rows, cols, seed):
    """Rows of ordinary size between rows of +-8e17 to +-9e17, which are less than 1e18 away from their mean in all but the narrowest rows."""
    values, gamma, beta, g = make(rows, cols, seed)
    large = (torch.randint(0, 2, (rows, cols), device=DEV, generator=g) * 2 - 1) * (8e17 + 1e17 * torch.rand(rows, cols, device=DEV, generator=g))
    return torch.where(torch.arange(rows, device=DEV)[:, None] % 2 == 0, large, values), gamma, beta, g


@pytest.mark.parametrize("x_kind,y_kind", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(rows, cols, x_kind, y_kind):
    values, gamma, beta, _ = large_rows(rows, cols, rows + cols)
    x = values.to(TYPES[x_kind][1])
    y = torch.empty(rows, cols, device=DEV, dtype=TYPES[y_kind][1])
    mean, rstd = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    assert mgt.launch_layer_norm(mgt.LayerNormConfig(rows, cols, EPS, TYPES[x_kind][0], TYPES[y_kind][0]), x, gamma, beta, y, mean, rstd) == 0
    check_forward(x, y_kind, y, mean, rstd, gamma, beta)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_backward(rows, cols, kind):
    values, gamma, _, g = large_rows(rows, cols, rows + cols)
    x = values.to(TYPES[kind][1])
    dy = (torch.randn(rows, cols, device=DEV, generator=g) * 2.0 ** 60).to(TYPES[kind][1])  # (so that dx, divided by the spread, is no denormal number)
    _, m, r, *_ = exact_forward(x, None, None)
    mean, rstd = m.float(), r.float()
    cfg = mgt.LayerNormConfig(rows, cols, EPS, TYPES[kind][0], TYPES[kind][0])
    floats = mgt.layer_norm_backward_workspace_floats(cfg)
    dx, sums = torch.empty_like(x), [torch.empty(cols, device=DEV) for _ in range(3)]
    assert mgt.launch_layer_norm_backward(cfg, dy, x, gamma, mean, rstd, dx, *sums, torch.empty(floats, device=DEV), floats) == 0
    check_backward(dy, x, gamma, mean, rstd, dx, kind, sums)


@pytest.mark.parametrize("cols", [3, 77, 224, 600, 2049, 9000, 20000, 1 << 20])
def test_large_values_without_large_deviations_are_finite(cols):
    # the mean of values of 1e22 is off by (16 + 10 + cols / 1024) * 2^-24 of them at most, 6e17 for the widest rows: so the squares hold, and what the
    # sums find is the row's spread and those roundings
    x = torch.where(torch.arange(6, device=DEV)[:, None] % 2 == 0, 1e22, -7e21) * torch.ones(6, cols, device=DEV)
    x[4:] *= 1 + 2.0 ** -20 * torch.randn(2, cols, device=DEV, generator=torch.Generator(device=DEV).manual_seed(cols))
    y, mean, rstd = torch.empty_like(x), torch.empty(6, device=DEV), torch.empty(6, device=DEV)
    assert mgt.launch_layer_norm(mgt.LayerNormConfig(6, cols), x, None, None, y, mean, rstd) == 0
    k = (64 + cols / 1024) * 2.0 ** -24
    m = x.double().mean(1)
    assert ((mean.double() - m).abs() <= k * x.double().abs().amax(1)).all()
    assert torch.isfinite(y).all() and torch.isfinite(rstd).all() and (rstd > 0).all()
