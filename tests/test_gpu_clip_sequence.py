"""Gradient norm, clipping and clipped update enqueued one behind the other through one result buffer, with nothing that waits between
them: every call takes the scale of the norm just before it, not the one that lay there."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import multigputrainmlp_b200 as mgt  # noqa: E402

DEV = "cuda:0"


def gradients(counts, kind):
    """Four gradients whose norms differ by factors of three; the third is not finite."""
    g = torch.Generator(device=DEV).manual_seed(sum(counts))
    flats = [(torch.randn(sum(counts), device=DEV, generator=g) * 3.0 ** k).to(kind) for k in range(4)]
    flats[2][-1] = float("inf")
    return flats


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("counts", [[1], [77, 5000], [3, 400_000, 1_000_001]])
def test_each_call_takes_the_norm_before_it(counts, kind, captured):
    flats = gradients(counts, kind)
    lists = [mgt.TensorList(f.split(counts)) for f in flats]
    floats = mgt.gradient_norm_workspace_floats(lists[0])
    ws, result = torch.empty(floats, device=DEV), torch.full((2,), 5.0, device=DEV)
    scales = []
    for lst in lists:  # each by itself
        alone, aside = torch.empty(2, device=DEV), torch.empty(floats, device=DEV)
        assert mgt.launch_gradient_norm(lst, 1e-4, alone, None, aside, floats) == 0
        torch.cuda.synchronize()
        scales.append(alone.clone())
    assert len({float(s[1]) for s in scales}) == 4 and float(scales[2][1]) == 0.0
    out = [torch.empty_like(f) for f in flats]
    out_lists = [mgt.TensorList(o.split(counts)) for o in out]
    in_place = [f.clone() for f in flats]
    in_place_lists = [mgt.TensorList(f.split(counts)) for f in in_place]
    n = sum(counts)
    cfg = mgt.AdamWKernelConfig(n, 3, 1e-3)
    start = [torch.randn(n, device=DEV), torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)]
    updated = [[t.clone() for t in start] for _ in flats]

    def everything():
        for k in range(4):
            assert mgt.launch_gradient_norm(lists[k], 1e-4, result, None, ws, floats) == 0
            assert mgt.launch_clip_gradients(lists[k], result, out_lists[k]) == 0
            if kind == torch.float32:
                assert mgt.launch_adamw_kernel_with_clip(cfg, updated[k][0], None, flats[k], result, updated[k][1], updated[k][2]) == 0
        for k in (1, 3, 2, 0):
            assert mgt.launch_gradient_norm(lists[k], 1e-4, result, None, ws, floats) == 0
            assert mgt.launch_clip_gradients(in_place_lists[k], result) == 0

    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            everything()
        graph.replay()
    else:
        everything()
    torch.cuda.synchronize()
    for k in range(4):
        want = (flats[k].float() * scales[k][1]).to(kind) if k != 2 else torch.zeros_like(flats[k])
        assert torch.equal(out[k], want) and torch.equal(in_place[k], want), k
        if kind == torch.float32:
            w, m, v = (t.clone() for t in start)
            if k != 2:
                assert mgt.launch_adamw_kernel(cfg, w, flats[k] * scales[k][1], m, v) == 0
            assert all(torch.equal(a, b) for a, b in zip(updated[k], (w, m, v))), k
