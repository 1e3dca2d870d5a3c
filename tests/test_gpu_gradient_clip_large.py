"""Norm and clipping of a tensor with more elements than 32 bits count in bytes, and more than 2^31 of them."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import multigputrainmlp_b200 as mgt  # noqa: E402

DEV = "cuda:0"


def test_more_elements_than_an_int_counts():
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 9 GB")
    n = 2 ** 31 + 4099
    flat = torch.zeros(n + 3, device=DEV, dtype=torch.bfloat16)
    t, small = flat[1:n + 1], torch.full((77,), 2.0, device=DEV)
    spots = torch.tensor([0, 5, 2 ** 30 + 1, 2 ** 31 - 1, 2 ** 31, n - 4, n - 1], device=DEV)
    t[spots] = torch.tensor([1.0, -2.0, 3.0, -4.0, 5.0, -6.0, 7.0], device=DEV, dtype=torch.bfloat16)
    flat[n + 1:], flat[0] = 100.0, 100.0  # beside the tensor
    lst = mgt.TensorList([t, small])
    floats = mgt.gradient_norm_workspace_floats(lst)
    ws, result, norms = torch.empty(floats, device=DEV), torch.empty(2, device=DEV), torch.empty(2, device=DEV)
    assert mgt.launch_gradient_norm(lst, 1.0, result, norms, ws, floats) == 0
    squares = 140.0 + 77 * 4.0  # 1 + 4 + 9 + 16 + 25 + 36 + 49
    # squares and sums of these are exact: what is left is half a step of fp32
    assert abs(float(result[0]) - math.sqrt(squares)) <= 2.0 ** -24 * math.sqrt(squares) and abs(float(norms[0]) - math.sqrt(140.0)) <= 2.0 ** -24 * math.sqrt(140.0)
    want = (t[spots].float() * result[1]).bfloat16()
    out = torch.full((n,), 9.0, device=DEV, dtype=torch.bfloat16)  # (lies otherwise to 16 bytes than t does)
    aside = torch.empty_like(small)
    assert mgt.launch_clip_gradients(lst, result, mgt.TensorList([out, aside])) == 0
    assert torch.equal(out[spots], want) and int(out.count_nonzero()) == 7
    del out
    assert mgt.launch_clip_gradients(lst, result) == 0
    assert torch.equal(t[spots], want) and int(t.count_nonzero()) == 7 and torch.equal(aside, small)
    assert (flat[n + 1:] == 100.0).all() and float(flat[0]) == 100.0
