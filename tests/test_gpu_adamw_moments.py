"""AdamW's first moments that are too small to move their weight, at every step and with second moments of any kind. An update of a weight of zero
takes the whole way (no moment is too small for it) and leaves minus the step itself: what any other weight has to move by."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import multigputrainmlp_b200 as mgt  # noqa: E402

DEV = "cuda:0"


def update(cfg, clip, w, g, m, v):
    t = [torch.from_numpy(a.copy()).to(DEV) for a in (w, g, m, v)]
    if clip:
        assert mgt.launch_adamw_kernel_with_clip(cfg, t[0], None, t[1], torch.ones(2, device=DEV), t[2], t[3]) == 0
    else:
        assert mgt.launch_adamw_kernel(cfg, *t) == 0
    return [x.cpu().numpy() for x in (t[0], t[2], t[3])]


def bits_or_nan(a):
    return np.where(np.isnan(a), np.uint32(0x7fc00000), a.view(np.uint32))


@pytest.mark.parametrize("clip", [False, True])
@pytest.mark.parametrize("lr,eps,beta1,beta2", [(1e-4, 1e-8, 0.9, 0.999), (0.5, 1e-3, 0.9, 0.999), (1e-3, 1e-8, 0.5, 0.5)])
@pytest.mark.parametrize("step", [1, 2, 7, 40, 164, 165, 1000])
def test_moments_of_every_size(step, lr, eps, beta1, beta2, clip):
    rng = np.random.default_rng(step)
    n = 100_000
    m = (np.exp2(rng.uniform(-149, 0, n)) * rng.choice([-1, 1], n)).astype(np.float32)
    v = np.where(rng.random(n) < 0.2, 0.0, np.exp2(rng.uniform(-149, 20, n))).astype(np.float32)
    w = (np.exp2(rng.uniform(-149, 30, n)) * rng.choice([-1, 1], n)).astype(np.float32)
    w[::3] = (rng.standard_normal(w[::3].size) * 0.05).astype(np.float32)
    g = np.where(rng.random(n) < 0.8, 0.0, m[::-1]).astype(np.float32)
    # second moments that have no root, or an infinite one
    v[:50], v[50:100], v[100:150], v[150:200] = np.nan, -1.0, np.inf, -np.float32(1e-30)
    m[:200:2], g[:200] = np.float32(2.0 ** -149), 0.0
    cfg = mgt.AdamWKernelConfig(n, step, lr, beta1=beta1, beta2=beta2, eps=eps)
    moved, m1, v1 = update(cfg, clip, np.zeros(n, np.float32), g, m, v)
    got, m2, v2 = update(cfg, clip, w, g, m, v)
    with np.errstate(over="ignore", invalid="ignore"):
        want = w - (0 - moved)
    assert np.array_equal(bits_or_nan(got), bits_or_nan(want))
    assert np.array_equal(bits_or_nan(m1), bits_or_nan(m2)) and np.array_equal(bits_or_nan(v1), bits_or_nan(v2))
    # (where even lr * m rounds to zero, the step is zero whatever it is divided by)
    assert np.isnan(got[:200]).sum() >= 50 and np.isfinite(got[100:150]).all() and np.isfinite(got[200:]).all()
    assert (got == w).sum() > n // 4 and (got != w).sum() > n // 8
