"""A list of tensors keeps the memory that it stands for: a tensor that is given other data does not leave it with an address that others use."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import multigputrainmlp_b200 as mgt  # noqa: E402

DEV = "cuda:0"
N = 1 << 20  # 4 MB: a block of its own


def test_memory_of_a_tensor_that_gets_other_data():
    kept, moved = torch.full((N,), 3.0, device=DEV), torch.full((N,), 4.0, device=DEV)
    lst = mgt.TensorList([kept, moved])
    floats = mgt.gradient_norm_workspace_floats(lst)
    ws, result, norms = torch.empty(floats, device=DEV), torch.empty(2, device=DEV), torch.empty(2, device=DEV)
    moved.data = torch.full((N,), 5.0, device=DEV)
    others = [torch.full((N,), float("inf"), device=DEV) for _ in range(8)]  # (would lie where `moved` lay, were it free)
    assert mgt.launch_gradient_norm(lst, 1024.0, result, norms, ws, floats) == 0
    assert norms.tolist() == [3.0 * 1024, 4.0 * 1024] and result.tolist() == [5.0 * 1024, float(torch.tensor(0.2))]
    assert mgt.launch_clip_gradients(lst, result) == 0
    assert all(o.isinf().all() for o in others) and (moved == 5.0).all() and torch.equal(kept, torch.full_like(kept, 3.0) * result[1])
