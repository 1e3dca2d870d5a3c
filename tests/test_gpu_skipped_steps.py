"""A step of the trainer whose gradient has no finite norm leaves no trace in what is trained or kept beside it."""
import json
import os
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "bin", "mgt_native_train")
MODEL = ["--batch-size", 512, "--k-min", 1, "--k-max", 29, "--hd1", 256, "--hd2", 64, "--nrd", 2, "--lr", 0.001]
HIDDEN_WEIGHTS = 72 * 72 * 256 + 256  # where they begin


def train(out_dir, *flags):
    cmd = [BIN, "--output-dir", out_dir, "--device-id", 0, "--world-size", 1, "--global-rank", 0, "--local-rank", 0, *MODEL, *flags]
    res = subprocess.run([str(c) for c in cmd], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr + res.stdout
    return {name: np.fromfile(out_dir / "checkpoint" / name, np.float32) for name in os.listdir(out_dir / "checkpoint") if name.endswith(".f32.bin")}


@pytest.mark.parametrize("norm", ["--batch-norm", "--layer-norm"])
@pytest.mark.parametrize("mirror", [0, 1])
def test_a_skipped_step_changes_nothing(tmp_path, norm, mirror):
    flags = [norm, 1, "--persistent-half-weights", mirror]
    start = train(tmp_path / "start", "--steps", 2, *flags)
    assert len(start) == 2 and all(np.isfinite(a).all() for a in start.values())
    again = ["--resume-checkpoint", tmp_path / "start" / "checkpoint", "--resume-step", 1]
    # a finite step moves everything, by exactly what it does without clipping
    clipped, plain = train(tmp_path / "clipped", "--steps", 1, *again, *flags, "--max-grad-norm", 1e9), train(tmp_path / "plain", "--steps", 1, *again, *flags)
    assert all(np.array_equal(clipped[k], plain[k]) and not np.array_equal(plain[k], start[k]) for k in start)
    # a weight that no half holds: its layer's pre-activations, and with them the batch's statistics and the gradient, are not finite
    broken = dict(start, **{"state.f32.bin": start["state.f32.bin"].copy()})
    broken["state.f32.bin"][HIDDEN_WEIGHTS] = 1e5
    broken["state.f32.bin"].tofile(tmp_path / "start" / "checkpoint" / "state.f32.bin")
    kept = train(tmp_path / "skipped", "--steps", 3, *again, *flags, "--max-grad-norm", 1.0)
    rows = [json.loads(line) for line in open(tmp_path / "skipped" / "grad_norm.jsonl")]
    assert len(rows) == 3 and all(r["grad_norm"] is None and r["scale"] == 0 for r in rows)
    for k in broken:
        assert np.array_equal(kept[k].view(np.uint32), broken[k].view(np.uint32)), k
