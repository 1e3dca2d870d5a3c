"""Checkpoints of the trainer with layer normalisation: what is resumed is the state of the model that is trained."""
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


def train(out_dir, *flags, hd2=32, nrd=1):
    cmd = [BIN, "--output-dir", out_dir, "--device-id", 0, "--world-size", 1, "--global-rank", 0, "--local-rank", 0, "--batch-size", 64, "--k-min", 1, "--k-max", 29,
           "--hd1", 64, "--hd2", hd2, "--nrd", nrd, "--lr", 0.001, "--steps", 1, *flags]
    return subprocess.run([str(c) for c in cmd], capture_output=True, text=True, timeout=300)


def test_state_of_another_model_is_refused(tmp_path):
    own = tmp_path / "own" / "checkpoint"
    resume = ["--layer-norm", 1, "--resume-checkpoint", own]
    assert train(tmp_path / "own", "--layer-norm", 1).returncode == 0 and train(tmp_path / "again", *resume).returncode == 0
    state, meta = (own / "layer_norm.f32.bin").read_bytes(), (own / "layer_norm.json").read_text()
    for wrong in (state + b"\0" * 4, state * 2, state[:-4], b""):
        (own / "layer_norm.f32.bin").write_bytes(wrong)
        res = train(tmp_path / "wrong", *resume)
        assert res.returncode != 0 and "layer_norm.f32.bin" in res.stderr, len(wrong)
    (own / "layer_norm.f32.bin").write_bytes(state)
    for key, value in (("layers", 4), ("width", 16), ("layers", 22), ("width", 3)):  # (the file alone could be four layers of half the width)
        (own / "layer_norm.json").write_text(json.dumps(dict(json.loads(meta), **{key: value}), indent=2))
        res = train(tmp_path / "wrong", *resume)
        assert res.returncode != 0 and "layer_norm.f32.bin" in res.stderr, (key, value)
    (own / "layer_norm.json").write_text(meta)
    assert train(tmp_path / "again", *resume).returncode == 0
    os.remove(own / "layer_norm.json")  # (the numbers are all in the binary file)
    assert train(tmp_path / "once more", *resume).returncode == 0
    a, b = (np.fromfile(tmp_path / d / "checkpoint" / "layer_norm.f32.bin", np.float32) for d in ("again", "once more"))
    assert np.array_equal(a, b)
    # the state of a deeper or wider model beside the weights of this one
    for size in (dict(hd2=64), dict(nrd=3)):
        assert train(tmp_path / "larger", "--layer-norm", 1, **size).returncode == 0
        (own / "layer_norm.f32.bin").write_bytes((tmp_path / "larger" / "checkpoint" / "layer_norm.f32.bin").read_bytes())
        assert train(tmp_path / "wrong", *resume).returncode != 0, size


def names(folder):
    return sorted(n for n in os.listdir(folder) if "norm" in n)


def test_a_folder_holds_the_state_of_its_last_run_only(tmp_path):
    d = tmp_path / "run"
    layer, batch = ["layer_norm.f32.bin", "layer_norm.json"], ["batch_norm.f32.bin", "batch_norm.json"]
    for flags, in_checkpoint, in_weights in ((["--layer-norm", 1], layer, layer), (["--batch-norm", 1], batch, []), (["--layer-norm", 1], layer, layer), ([], [], []),
                                             (["--batch-norm", 1], batch, []), ([], [], [])):
        assert train(d, *flags).returncode == 0
        assert names(d / "checkpoint") == in_checkpoint and names(d / "weights") == in_weights, flags
    for flag in ("--layer-norm", "--batch-norm"):  # the plain run's checkpoint is no checkpoint of either
        assert train(tmp_path / "next", flag, 1, "--resume-checkpoint", d / "checkpoint").returncode != 0


def test_a_model_with_layer_norm_is_not_resumed_without(tmp_path):
    assert train(tmp_path / "own", "--layer-norm", 1).returncode == 0
    kept = (tmp_path / "own" / "checkpoint" / "state.f32.bin").read_bytes()
    for flags in ([], ["--batch-norm", 1], ["--layer-norm", 0], ["--linear-fp16", 0]):
        res = train(tmp_path / "own", "--resume-checkpoint", tmp_path / "own" / "checkpoint", *flags)
        assert res.returncode != 0 and "--layer-norm 1" in res.stderr, flags
    assert (tmp_path / "own" / "checkpoint" / "state.f32.bin").read_bytes() == kept
