"""AdamW on moments, weights and gradients at the lower end of the numbers, bit for bit against the update in numpy's fp32, operation by operation."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import multigputrainmlp_b200 as mgt  # noqa: E402

DEV = "cuda:0"
F = np.float32


def plain(w, g, m, v, step, lr, wd=0.0, b1=0.9, b2=0.999, eps=1e-8):
    lr, wd, b1, b2, eps = map(F, (lr, wd, b1, b2, eps))
    decayed = g + wd * w
    m = b1 * m + (F(1) - b1) * decayed
    v = b2 * v + ((F(1) - b2) * decayed) * decayed
    return w, m, v, lr, eps


@pytest.mark.parametrize("lr,wd", [(1e-4, 0.0), (0.5, 0.0), (1e-3, 0.01)])
@pytest.mark.parametrize("clip", [False, True])
def test_update_bit_for_bit(lr, wd, clip):
    # from step 400 on 1 - 0.9^step is 1 in fp32 (0.9^400 = 5e-19), and at step 20000 1 - 0.999^step is 1 as well (2e-9, below half an ulp)
    step = 20000
    rng = np.random.default_rng(5)
    n = 200_000
    tiny = np.exp2(rng.uniform(-149, -110, n)).astype(F) * rng.choice([-1, 1], n).astype(F)
    m = np.where(rng.random(n) < 0.5, tiny, np.where(rng.random(n) < 0.5, F(0), tiny * F(2.0) ** 60)).astype(F)
    v = np.where(rng.random(n) < 0.3, np.exp2(rng.uniform(-149, -100, n)), np.where(rng.random(n) < 0.3, 0.0, np.exp2(rng.uniform(-60, 0, n)))).astype(F)
    w = np.where(rng.random(n) < 0.3, np.exp2(rng.uniform(-149, -40, n)), np.where(rng.random(n) < 0.1, 0.0, rng.standard_normal(n))).astype(F)
    w *= rng.choice([-1, 1], n).astype(F)
    g = np.where(rng.random(n) < 0.6, F(0), np.where(rng.random(n) < 0.5, tiny[::-1], rng.standard_normal(n).astype(F) * F(1e-3))).astype(F)
    dw, dg, dm, dv = (torch.from_numpy(a.copy()).to(DEV) for a in (w, g, m, v))
    cfg = mgt.AdamWKernelConfig(n, step, lr, weight_decay=wd)
    if clip:
        assert mgt.launch_adamw_kernel_with_clip(cfg, dw, None, dg, torch.tensor([1.0, 1.0], device=DEV), dm, dv) == 0
    else:
        assert mgt.launch_adamw_kernel(cfg, dw, dg, dm, dv) == 0
    w0, nm, nv, lr32, eps = plain(w, g, m, v, step, lr, wd)
    want = w0 - lr32 * nm / (np.sqrt(nv) + eps)
    assert np.array_equal(dm.cpu().numpy().view(np.uint32), nm.view(np.uint32)) and np.array_equal(dv.cpu().numpy().view(np.uint32), nv.view(np.uint32))
    assert np.array_equal(dw.cpu().numpy().view(np.uint32), want.view(np.uint32))


def test_moment_that_has_come_to_rest_moves_no_weight():
    # 0.9 of four times the smallest number rounds to it again
    m = torch.full((4096,), 4 * 2.0 ** -149, device=DEV)
    w = torch.linspace(-1, 1, 4096, device=DEV)
    kept, v, g = w.clone(), torch.full((4096,), 1e-12, device=DEV), torch.zeros(4096, device=DEV)
    for step in (1, 100, 5000):
        assert mgt.launch_adamw_kernel(mgt.AdamWKernelConfig(4096, step, 1e-3), w, g, m, v) == 0
    assert (m == 4 * 2.0 ** -149).all() and torch.equal(w, kept)
