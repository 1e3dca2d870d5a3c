"""The trainer with layer normalisation and clipping on one rank and on two: the gradient is averaged first, its norm taken of the average, and the
update made of what that leaves, the same on every rank, whether the exchange overlaps the backward pass or follows it."""
import json
import os
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from helpers import trainer_init_weights  # noqa: E402
from oracle import MlpShape  # noqa: E402
from test_gpu_layer_norm_step import model  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "bin", "mgt_native_train")
SHAPE = MlpShape(72, 72, 128, 32, 2, 1)
BATCH, STEPS, LR = 256, 3, 1e-3


def train(folder, world, max_norm, overlap):
    """The checkpoint and the rows of every rank."""
    flags = ["--steps", STEPS, "--batch-size", BATCH, "--k-min", 1, "--k-max", 29, "--hd1", 128, "--hd2", 32, "--nrd", 2, "--lr", LR, "--layer-norm", 1,
             "--max-grad-norm", max_norm, "--overlap-allreduce", overlap, "--world-size", world]
    if world > 1:
        flags += ["--nccl-id-file", folder / "ranks.id"]
    folder.mkdir()
    procs = []
    for r in range(world):
        cmd = [BIN, "--output-dir", folder / f"rank{r}", "--device-id", r, "--global-rank", r, "--local-rank", r, *flags]
        procs.append(subprocess.Popen([str(c) for c in cmd], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, env=dict(os.environ, NCCL_NVLS_ENABLE="0")))
    outs = [p.communicate(timeout=300) for p in procs]
    assert all(p.returncode == 0 for p in procs), outs
    ranks = []
    for r in range(world):
        d = folder / f"rank{r}"
        state = {n: (d / "checkpoint" / n).read_bytes() for n in ("state.f32.bin", "layer_norm.f32.bin")}
        ranks.append((state, [json.loads(line) for line in open(d / "grad_norm.jsonl")], [json.loads(line) for line in open(d / "profile.jsonl")]))
    return ranks


def expected(oracle, world, max_norm):
    """Losses of every rank and norms of the averaged gradient, by the 64-bit model."""
    moves, target = oracle.cyclic_puzzle(72, 18)
    p, nn = SHAPE.param_count, 2 * (SHAPE.residual_blocks + 1) * SHAPE.hd2
    w = np.concatenate([trainer_init_weights(p), np.zeros(nn, np.float32)])
    w[p:].reshape(-1, 2, SHAPE.hd2)[:, 0, :] = 1.0
    m, v = np.zeros_like(w), np.zeros_like(w)
    losses, norms = [], []
    for step in range(STEPS):
        parts = []
        for r in range(world):
            _, states, depth, _ = oracle.random_walks(moves, target, seed=1234, epoch=0, step=step, rank=r, k_min=1, k_max=29, samples=BATCH)
            parts.append(model(SHAPE, w, states, depth.reshape(-1, 1), torch.float16))
        grad = np.mean([g for _, g in parts], axis=0)
        norm = np.linalg.norm(grad)
        losses.append([loss for loss, _ in parts])
        norms.append(norm)
        grad = grad * (max_norm / norm if norm > max_norm else 1.0)
        assert oracle.adamw(w, grad.astype(np.float32), m, v, step=step + 1, lr=LR) == 0
    return losses, norms


@pytest.mark.parametrize("world", [1, pytest.param(2, marks=pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs"))])
def test_ranks_clip_the_average(tmp_path, oracle, world):
    max_norm = 0.75
    losses, norms = expected(oracle, world, max_norm)
    runs = [train(tmp_path / f"overlap{o}", world, max_norm, o) for o in (0, 1)]
    for ranks in runs:
        for r, (state, clips, rows) in enumerate(ranks):
            assert state == runs[0][0][0] and clips == runs[0][0][1]  # every rank, both forms of the exchange, to the bit
            assert len(clips) == len(rows) == STEPS
            for step, (clip, row) in enumerate(zip(clips, rows)):
                assert abs(row["loss"] - losses[step][r]) <= 2e-3 * abs(losses[step][r])
                assert abs(clip["grad_norm"] - norms[step]) <= 2e-2 * norms[step]
                assert abs(clip["scale"] - min(1.0, max_norm / clip["grad_norm"])) <= 1e-6
    if world > 1:
        assert all(row["overlap_ranges"] == 2 * 2 + 4 for _, _, rows in runs[1] for row in rows)  # the scale/shift vectors are one more
