"""The gradient norm over many tensors, clipping, and the clipped update, against 64-bit sums.

Tolerances: squares and sums are 64-bit, so a norm is off by the rounding of the result to fp32 (half a step, 2^-24 of it) and by some
2^-50 besides; the scale, computed from the unrounded norm, by half a step. What is multiplied by the scale is compared bit for bit."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import multigputrainmlp_b200 as mgt  # noqa: E402

DEV = "cuda:0"
STEP = 2.0 ** -24 * (1 + 1e-6)


def views(counts, kinds, seed, scale=1e-2, gap=0):
    """Tensors that follow one another (with `gap` elements between) in one buffer a type."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = []
    pools = {}
    for i, n in enumerate(counts):
        kind = kinds[i % len(kinds)]
        pools.setdefault(kind, []).append((i, n))
    got = {}
    for kind, items in pools.items():
        total = sum(n + gap for _, n in items)
        flat = (torch.randn(total + 1, device=DEV, generator=g) * scale).to(kind)
        at = gap
        for i, n in items:
            got[i] = flat[at:at + n]
            at += n + gap
    out = [got[i] for i in range(len(counts))]
    return out


def norm_of(tensors, max_norm=1.0, floats=None):
    lst = mgt.TensorList(tensors)
    floats = mgt.gradient_norm_workspace_floats(lst)
    assert floats > 0
    ws = torch.full((floats + 16,), float("nan"), device=DEV)
    ws[floats:] = 3.0
    result, norms = torch.full((4,), 5.0, device=DEV), torch.full((lst.count + 2,), 5.0, device=DEV)
    assert mgt.launch_gradient_norm(lst, max_norm, result, norms, ws, floats) == 0
    assert (ws[floats:] == 3.0).all() and (result[2:] == 5.0).all() and (norms[lst.count:] == 5.0).all()
    return lst, result, norms[:lst.count]


def exact_norms(tensors):
    squares = [float(t.double().square().sum()) if t.numel() else 0.0 for t in tensors]
    return math.sqrt(math.fsum(squares)), [math.sqrt(s) for s in squares]


CASES = [([1], 0), ([5], 0), ([4096], 0), ([4097], 1), ([1 << 20], 0), ([0, 3, 0, 70000, 1], 0), ([333 * 77, 77, 77 * 77, 77] * 4, 1), ([7] * 96, 0), ([7, 5000] * 49, 3),
         ([33] * 1024, 0), ([2_000_003, 17, 300_001], 0), ([0], 0), ([0, 0], 0)]


@pytest.mark.parametrize("kinds", [[torch.float32], [torch.float16], [torch.bfloat16], [torch.float32, torch.bfloat16, torch.float16]])
@pytest.mark.parametrize("counts,gap", CASES)
def test_norms_and_scale(counts, gap, kinds):
    tensors = views(counts, kinds, len(counts) + counts[0], gap=gap)
    for max_norm in (1e-3, 1e9, float("inf")):
        _, result, norms = norm_of(tensors, max_norm)
        total, each = exact_norms(tensors)
        assert abs(float(result[0]) - total) <= STEP * total
        most = float(np.float32(max_norm))  # the call's argument is a float: 1e-3 reaches it rounded
        scale = most / total if total > most else 1.0
        assert abs(float(result[1]) - scale) <= STEP * scale + 1e-45
        assert np.all(np.abs(norms.double().cpu().numpy() - np.array(each)) <= STEP * np.array(each))


@pytest.mark.parametrize("value", [1e30, 3e38, 1e-30, 1e-44])
def test_squares_beyond_the_floats(value):
    n = 3 if value > 1e38 else 5000
    t = torch.full((n,), value, device=DEV) * torch.where(torch.arange(n, device=DEV) % 3 == 0, -1.0, 0.5)
    _, result, norms = norm_of([t], 1.0)
    total, _ = exact_norms([t])
    small = 2.0 ** -150  # half the smallest fp32 number
    if total > torch.finfo(torch.float32).max:  # 3e38, 1.5e38, 1.5e38: 3.67e38, which no float holds
        assert float(result[0]) == float("inf") and float(result[1]) == 0.0
        return
    assert abs(float(result[0]) - total) <= STEP * total + small and float(norms[0]) == float(result[0])
    scale = min(1.0, 1.0 / total)
    assert abs(float(result[1]) - scale) <= STEP * scale + small


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
def test_gradients_that_are_not_finite(value, kind):
    tensors = views([5000, 3, 777], [kind], 4)
    tensors[2][776] = value
    for max_norm in (1.0, float("inf")):
        lst, result, norms = norm_of(tensors, max_norm)
        assert not math.isfinite(float(result[0])) and float(result[1]) == 0.0 and not math.isfinite(float(norms[2])) and norms[:2].isfinite().all()
    assert mgt.launch_clip_gradients(lst, result) == 0
    assert all((t == 0).all() for t in tensors)


def test_a_norm_that_no_float_holds():
    t = torch.full((100,), 3e38, device=DEV)
    lst, result, _ = norm_of([t], 1.0)
    assert float(result[0]) == float("inf") and float(result[1]) == 0.0
    assert mgt.launch_clip_gradients(lst, result) == 0 and (t == 0).all()


@pytest.mark.parametrize("kinds", [[torch.float32], [torch.float16], [torch.bfloat16], [torch.bfloat16, torch.float32]])
@pytest.mark.parametrize("counts,gap,out_gap", [([1], 0, 0), ([5000, 0, 3], 0, 0), ([333, 77, 4099] * 5, 1, 1), ([333, 77, 4099] * 5, 1, 2), ([9, 5001] * 60, 0, 3), ([300_001], 0, 1)])
def test_clipping(counts, gap, out_gap, kinds):
    tensors = views(counts, kinds, 11, gap=gap)
    for max_norm in (1e-2, 1e9):
        lst, result, _ = norm_of(tensors, max_norm)
        scale = result[1].clone()
        want = [(t.float() * scale).to(t.dtype) for t in tensors]
        out = views(counts, kinds, 12, gap=out_gap)
        around = [o.untyped_storage() for o in out]
        before = {s.data_ptr(): torch.tensor([], device=DEV, dtype=torch.uint8).set_(s).clone() for s in around}
        kept = [t.clone() for t in tensors]
        assert mgt.launch_clip_gradients(lst, result, mgt.TensorList(out)) == 0
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and all(torch.equal(a, b) for a, b in zip(tensors, kept))
        for o in out:
            o.zero_()
        for s in around:  # nothing beside the outputs was written
            now, then = torch.tensor([], device=DEV, dtype=torch.uint8).set_(s), before[s.data_ptr()]
            for o in out:
                if o.untyped_storage().data_ptr() == s.data_ptr():
                    lo = o.storage_offset() * o.element_size()
                    then[lo:lo + o.numel() * o.element_size()] = 0
            assert torch.equal(now, then)
        assert mgt.launch_clip_gradients(lst, result) == 0
        assert all(torch.equal(a, b) for a, b in zip(tensors, want))
        for t, k in zip(tensors, kept):
            t.copy_(k)


@pytest.mark.parametrize("mirror", [False, True])
@pytest.mark.parametrize("n", [1, 3, 4, 1023, 1_000_003])
def test_clipped_update_is_the_update_of_the_clipped_gradient(n, mirror):
    g = torch.Generator(device=DEV).manual_seed(n)
    grad = torch.randn(n, device=DEV, generator=g)
    grad[::7] = 0
    start = [torch.randn(n, device=DEV, generator=g), 0.1 * torch.randn(n, device=DEV, generator=g), torch.rand(n, device=DEV, generator=g)]
    cfg = mgt.AdamWKernelConfig(n, 7, 1e-3, weight_decay=0.01)

    def update(clip=None, gradient=grad):
        w, m, v = (t.clone() for t in start)
        half = torch.full((n,), 9.0, device=DEV, dtype=torch.float16) if mirror else None
        if clip is not None:
            assert mgt.launch_adamw_kernel_with_clip(cfg, w, half, gradient, clip, m, v) == 0
        elif mirror:
            assert mgt.launch_adamw_kernel_with_half_mirror(cfg, w, half, gradient, m, v) == 0
        else:
            assert mgt.launch_adamw_kernel(cfg, w, gradient, m, v) == 0
        return [t for t in (w, m, v, half) if t is not None]

    kept = grad.clone()
    _, clip, _ = norm_of([grad], 0.25)
    assert all(torch.equal(a, b) for a, b in zip(update(clip[:2]), update(gradient=grad * clip[1])))
    assert all(torch.equal(a, b) for a, b in zip(update(torch.tensor([0.5, 1.0], device=DEV)), update()))
    for norm in (float("nan"), float("inf")):  # skipped
        got = update(torch.tensor([norm, 0.0], device=DEV))
        assert all(torch.equal(a, b) for a, b in zip(got, start)) and (not mirror or (got[3] == 9.0).all())
    assert torch.equal(grad, kept)


def test_norm_then_update_from_a_graph_and_on_two_streams():
    counts = [100_000, 17, 40_001]
    g = torch.Generator(device=DEV).manual_seed(1)
    n = sum(counts)
    grad = torch.randn(n, device=DEV, generator=g)
    start = [torch.randn(n, device=DEV, generator=g), torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)]
    lst = mgt.TensorList(grad.split(counts))
    floats = mgt.gradient_norm_workspace_floats(lst)
    cfg = mgt.AdamWKernelConfig(n, 1, 1e-3)

    def state():
        return [*(t.clone() for t in start), torch.empty(2, device=DEV), torch.empty(3, device=DEV), torch.full((floats,), float("nan"), device=DEV)]

    def step(s):
        w, m, v, result, norms, ws = s
        assert mgt.launch_gradient_norm(lst, 1.0, result, norms, ws, floats) == 0
        assert mgt.launch_adamw_kernel_with_clip(cfg, w, None, grad, result, m, v) == 0

    plain = state()
    step(plain)
    streams, both = [torch.cuda.Stream() for _ in range(2)], [state(), state()]
    torch.cuda.synchronize()
    for st, s in zip(streams, both):
        with torch.cuda.stream(st):
            step(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for s in both for a, b in zip(s[:5], plain[:5]))
    captured = state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured)
    grad.mul_(3.0)
    graph.replay()
    other = state()
    step(other)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured[:5], other[:5]))


def test_lists_that_do_not_fit_are_refused():
    t = torch.zeros(10, device=DEV)
    for bad in ([t.double()], [t.cpu()], [torch.zeros(4, 4, device=DEV)[:, 1]], []):
        with pytest.raises(mgt.MgtError):
            mgt.TensorList(bad)
    lst = mgt.TensorList([t])
    floats = mgt.gradient_norm_workspace_floats(lst)
    ws, result = torch.empty(floats, device=DEV), torch.empty(2, device=DEV)
    assert mgt.launch_gradient_norm(lst, 1.0, result, None, ws, floats) == 0
    assert mgt.launch_gradient_norm(lst, 1.0, result[:1], None, ws, floats) == 1
    assert mgt.launch_gradient_norm(lst, 1.0, result, None, ws[:-1], floats) == 1
    assert mgt.launch_gradient_norm(lst, 1.0, result, None, ws, floats - 1) == 3
    assert mgt.launch_clip_gradients(lst, result, mgt.TensorList([t, t])) == 1
    assert mgt.launch_clip_gradients(lst, result, mgt.TensorList([t[:9]])) == 1
    assert mgt.launch_clip_gradients(lst, result, mgt.TensorList([t.half()])) == 1
