"""rstd where a row has no spread and eps is all there is: down to the smallest number that the config takes (1.4e-45)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import multigputrainmlp_b200 as mgt  # noqa: E402

DEV = "cuda:0"


@pytest.mark.parametrize("eps", [1e-45, 3e-45, 1e-42, 1e-39, 1e-38, 1e-30, 1e-5, 1.0, 1e30, 3e38])
@pytest.mark.parametrize("cols", [1, 8, 77, 600, 9000, 20000])
def test_rows_without_spread(cols, eps):
    # the device's reciprocal root is off by 2 units in the last place at most, which one Newton step squares away: what is left are the roundings of
    # its two products and of its sum (1.5 - 0.5, half a unit of 1 each), and of the last product: 4 half units of rstd, 4 * 2^-24
    x = torch.zeros(5, cols, device=DEV)
    beta = torch.randn(cols, device=DEV)
    y, mean, rstd = torch.empty_like(x), torch.empty(5, device=DEV), torch.empty(5, device=DEV)
    assert mgt.launch_layer_norm(mgt.LayerNormConfig(5, cols, eps), x, None, beta, y, mean, rstd) == 0
    want = torch.tensor(eps, dtype=torch.float32).double().rsqrt().item()  # (of the eps that a float argument holds)
    assert ((rstd.double() - want).abs() <= 4 * 2.0 ** -24 * want).all()
    assert (mean == 0).all() and torch.equal(y, beta.expand(5, cols))


@pytest.mark.parametrize("size,eps", [(1e-17, 1e-45), (1e-17, 1e-36), (1e-18, 1e-34), (1e-19, 1e-34), (1e-30, 1e-34), (1e-10, 1e-38)])
@pytest.mark.parametrize("rows,cols", [(7, 8), (40, 77), (33, 224), (9, 600), (5, 4096), (5, 9000), (3, 20000)])
def test_small_rows(rows, cols, size, eps):
    # bounds as in test_gpu_layer_norm.py. What is lost of squares among the smallest numbers: half of 2^-149 a thread, times 2^12 that its sum is divided
    # by, of at least one column a thread: 2^-138 of the variance at most, a 2^-24th of 1e-34 / 2
    x = torch.randn(rows, cols, device=DEV, generator=torch.Generator(device=DEV).manual_seed(cols)) * size
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    assert mgt.launch_layer_norm(mgt.LayerNormConfig(rows, cols, eps), x, None, None, y, mean, rstd) == 0
    m = x.double().mean(1, keepdim=True)
    d = x.double() - m
    want = (d.square().mean(1) + torch.tensor(eps, dtype=torch.float32).double().item()).rsqrt()
    k = (65 + cols / 1024) * 2.0 ** -24
    assert ((rstd.double() - want).abs() <= k * want).all()
    xhat = d * want[:, None]
    assert ((y.double() - xhat).abs() <= k * xhat.abs().amax(1, keepdim=True) + 2.0 ** -24 * xhat.abs()).all()
    assert ((mean.double() - m[:, 0]).abs() <= 2.0 ** -24 * m[:, 0].abs() + k * d.abs().amax(1)).all()
