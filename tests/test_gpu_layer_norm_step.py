"""Layer normalisation inside the loss+gradient engine and the trainer, and the trainer's clipping, against a 64-bit model of the network
whose products round their operands where the engine does (so that the two differ by fp32 sums and by roundings that fall the other way)."""
import json
import os
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import multigputrainmlp_b200 as mgt  # noqa: E402
from helpers import rel_l2, trainer_init_weights  # noqa: E402
from test_gpu_batch_norm import assert_close, cshape_of, keep_relus_open, make_case  # noqa: E402

from oracle import MlpShape  # noqa: E402

DEV = "cuda:0"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "bin", "mgt_native_train")


def rounded(t, kind):
    return t if kind is None else t.float().to(kind).double()


class Product(torch.autograd.Function):
    """x @ w with both operands rounded, and the incoming gradient rounded before it meets either of them."""

    @staticmethod
    def forward(ctx, x, w, kind):
        x, w = rounded(x, kind), rounded(w, kind)
        ctx.save_for_backward(x, w)
        ctx.kind = kind
        return x @ w

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        dy = rounded(dy, ctx.kind)
        return dy @ w.T, x.T @ dy, None


class Embedding(torch.autograd.Function):
    """Sums of rounded table rows; the table's gradient takes the rounded gradient."""

    @staticmethod
    def forward(ctx, onehot, table, kind, table_kind):
        ctx.save_for_backward(onehot)
        ctx.kind = kind if table_kind == "same" else table_kind
        return onehot @ rounded(table, kind)

    @staticmethod
    def backward(ctx, dy):
        (onehot,) = ctx.saved_tensors
        return None, onehot.T @ rounded(dy, ctx.kind), None, None


class RoundForward(torch.autograd.Function):
    """A value that is rounded on its way, its gradient not."""

    @staticmethod
    def forward(ctx, x, kind):
        return rounded(x, kind)

    @staticmethod
    def backward(ctx, dy):
        return dy, None


def layer_norm(z, gamma, beta, eps):
    d = z - z.mean(1, keepdim=True)
    return d / torch.sqrt((d * d).mean(1, keepdim=True) + eps) * gamma + beta


def model(shape, w, states, labels, kind, ce=False, eps=1e-5, table_kind="same"):
    """(loss, gradient) in 64 bits; kind: the operands' type, None for none; table_kind: what the gradient of the table is taken from."""
    w = torch.from_numpy(np.asarray(w, np.float32)).to(DEV).double().requires_grad_()
    n, h1, h2, r, out = states.shape[0], shape.hd1, shape.hd2, shape.residual_blocks, shape.output_dim
    at = [0]

    def take(*dims):
        size = int(np.prod(dims))
        at[0] += size
        return w[at[0] - size:at[0]].view(*dims)

    rows = shape.state_len * shape.state_value_pad
    table, b_in, wh, bh = take(rows, h1), take(h1), take(h1, h2), take(h2)
    blocks = [(take(h2, h2), take(h2), take(h2, h2), take(h2)) for _ in range(r)]
    w_out, b_out = take(h2, out), take(out)
    assert at[0] == shape.param_count
    norms = [(take(h2), take(h2)) for _ in range(r + 1)]
    index = torch.from_numpy(states[:, :shape.state_len].astype(np.int64)).to(DEV) + torch.arange(shape.state_len, device=DEV) * shape.state_value_pad
    onehot = torch.zeros(n, rows, device=DEV, dtype=torch.float64).scatter_(1, index, 1.0)
    a1 = torch.relu(Embedding.apply(onehot, table, kind, table_kind) + RoundForward.apply(b_in, kind))
    x = torch.relu(layer_norm(Product.apply(a1, wh, kind) + bh, *norms[0], eps))
    for (w1, b1, w2, b2), (gamma, beta) in zip(blocks, norms[1:]):
        inner = torch.relu(Product.apply(x, w1, kind) + b1)
        x = torch.relu(x + layer_norm(Product.apply(inner, w2, kind) + b2, gamma, beta, eps))
    y = (x @ w_out if out == 1 else Product.apply(x, w_out, kind)) + b_out
    target = torch.from_numpy(np.ascontiguousarray(labels)).to(DEV).double().view(n, out)
    if ce:
        loss = torch.nn.functional.cross_entropy(y, target[:, 0].round().long() - 1)
    else:
        loss = ((y - target) ** 2).mean()
    loss.backward()
    return float(loss.detach()), w.grad.cpu().numpy()


def run_engine(eng, shape, w, states, labels, *, callback=None, half_table=True, **more):
    cshape = cshape_of(shape)
    b = states.shape[0]
    dw, ds = torch.from_numpy(w).to(DEV), torch.from_numpy(states).to(DEV)
    dl = torch.from_numpy(np.ascontiguousarray(labels)).to(DEV)
    loss, grad = torch.zeros(1, device=DEV), torch.full((w.size + 16,), float("nan"), device=DEV)
    floats = mgt.mlp_loss_grad_workspace_floats(cshape, b, 1, half_table, layer_norm=True)
    ws = torch.full((floats + 256,), float("nan"), device=DEV)
    ws[floats:] = 5.0
    st = eng.launch_mlp_loss_grad(cshape, dw, None, ds, dl, b, loss, grad, ws, floats, gradient_ready=callback, use_half_input_grad=half_table, **more)
    assert st == 0, mgt.status_name(st)
    st, code = eng.check()
    assert st == 0, f"device status {code}"
    assert (ws[floats:] == 5.0).all() and grad[w.size:].isnan().all()
    return float(loss.item()), grad[:w.size].cpu().numpy()


CASES = [  # dims, samples, bfloat16, cross-entropy, ReLUs held open
    ((72, 72, 128, 224, 3, 1), 600, False, False, False),     # the p888 tower width
    ((72, 72, 128, 224, 3, 1), 600, False, False, True),
    ((72, 72, 64, 64, 2, 5), 257, False, True, False),        # cross-entropy, a ragged last row tile
    ((72, 72, 64, 64, 2, 5), 257, False, False, True),
    ((6, 8, 9, 7, 2, 11), 40, False, False, False),           # widths that are no multiple of four
    ((6, 8, 9, 77, 2, 1), 1000, False, False, True),
    ((72, 72, 96, 224, 2, 29), 300, True, True, False),       # bfloat16 + cross-entropy
    ((72, 72, 64, 32, 0, 1), 128, False, False, False),       # no residual blocks
    ((6, 8, 32, 512, 1, 1), 300, False, False, True),         # the widest tower
    ((8, 8, 32, 40, 1, 1), 20001, False, False, True),
    ((6, 8, 16, 8, 1, 1), 1, False, False, False),            # one sample
]


@pytest.mark.parametrize("dims,n,bf16,ce,smooth", CASES)
def test_engine_with_layer_norm_matches_the_model(oracle, dims, n, bf16, ce, smooth):
    shape, w, states, labels = make_case(oracle, dims, n, seed=41)
    if smooth:
        w = keep_relus_open(shape, w)
    if not ce and shape.output_dim > 1:
        labels = labels * 0.1
    kind = torch.bfloat16 if bf16 else torch.float16
    loss_m, grad_m = model(shape, w, states, labels, kind, ce)
    _, grad_exact = model(shape, w, states, labels, None, ce)
    seen = []
    eng = mgt.Engine(0)
    try:
        assert eng.set_train_options(bf16=bf16, cross_entropy=ce) == 0 and eng.set_layer_norm(True) == 0
        loss_g, grad_g = run_engine(eng, shape, w, states, labels, callback=lambda u, i, off, cnt, s: seen.append((i, off, cnt)) or 0)
        again = run_engine(eng, shape, w, states, labels)
        assert again[0] == loss_g and np.array_equal(again[1], grad_g)
        # without it the same engine is what it was
        assert eng.set_layer_norm(False) == 0
        plain = eng.launch_mlp_loss_grad
        cshape = cshape_of(shape)
        floats = mgt.mlp_loss_grad_workspace_floats(cshape, n)
        args = [torch.from_numpy(w).to(DEV), None, torch.from_numpy(states).to(DEV), torch.from_numpy(np.ascontiguousarray(labels)).to(DEV), n, torch.zeros(1, device=DEV)]
        g1, g2 = torch.zeros(shape.param_count, device=DEV), torch.zeros(shape.param_count, device=DEV)
        assert plain(cshape, *args, g1, torch.empty(floats, device=DEV), floats) == 0
        fresh = mgt.Engine(0)
        assert fresh.set_train_options(bf16=bf16, cross_entropy=ce) == 0
        assert fresh.launch_mlp_loss_grad(cshape, *args, g2, torch.empty(floats, device=DEV), floats) == 0
        assert torch.equal(g1, g2)
        fresh.close()
    finally:
        eng.close()
    assert_close(shape, loss_g, grad_g, loss_m, grad_m, grad_exact, tol=8e-3 if bf16 else 1e-3)
    assert len(seen) == 2 * shape.residual_blocks + 4
    assert seen[-1] == (2 * shape.residual_blocks + 3, shape.param_count, 2 * (shape.residual_blocks + 1) * shape.hd2) and seen[-2][1] == 0


def test_fp32_table_gradient_profile_and_early_range(oracle):
    shape, w, states, labels = make_case(oracle, (72, 72, 96, 40, 2, 1), 333, seed=45)
    loss_m, grad_m = model(shape, w, states, labels, torch.float16, table_kind=None)
    _, grad_exact = model(shape, w, states, labels, None)
    eng = mgt.Engine(0)
    early = []
    try:
        assert eng.set_layer_norm(True) == 0
        loss_g, grad_g = run_engine(eng, shape, w, states, labels, half_table=False)
        assert_close(shape, loss_g, grad_g, loss_m, grad_m, grad_exact, tol=1e-3)
        plain = run_engine(eng, shape, w, states, labels)
        profile = mgt.BackwardProfile()
        timed = run_engine(eng, shape, w, states, labels, profile=profile)
        assert np.array_equal(plain[1], timed[1]) and profile.residual_forward_ms > 0
        assert eng.set_early_range_hook(lambda u, i, off, cnt, s: early.append((off, cnt)) or 0) == 0
        hooked = run_engine(eng, shape, w, states, labels)
        assert np.array_equal(plain[1], hooked[1]) and early == [(0, 72 * 72 * 96 + 96)]
    finally:
        eng.close()


def test_gradient_against_differences_of_the_loss(oracle):
    # every ReLU open, so that the loss is smooth: differences of the 64-bit loss without any rounding. What the operands' rounding does to
    # a gradient here is bounded by the model's own distance from the exact one
    shape, w, states, labels = make_case(oracle, (6, 8, 16, 24, 2, 1), 64, seed=42)
    w = keep_relus_open(shape, w)
    eng = mgt.Engine(0)
    try:
        assert eng.set_layer_norm(True, 1e-5) == 0
        _, grad = run_engine(eng, shape, w, states, labels)
    finally:
        eng.close()
    _, exact = model(shape, w, states, labels, None)
    _, rounded_grad = model(shape, w, states, labels, torch.float16)
    # one direction a section: the slope along a random direction
    rng = np.random.default_rng(1)
    p, h1, h2 = shape.param_count, shape.hd1, shape.hd2
    edges = [0, 48 * h1, 48 * h1 + h1, 48 * h1 + h1 + h1 * h2, p - h2 - 1, p, p + 2 * h2, w.size]
    for lo, hi in zip(edges, edges[1:]):
        d = np.zeros(w.size)
        d[lo:hi] = rng.standard_normal(hi - lo)
        d /= np.linalg.norm(d)
        h = 1e-3
        up = (w + h * d).astype(np.float32).astype(np.float64)
        down = (w - h * d).astype(np.float32).astype(np.float64)
        slope = (model(shape, up, states, labels, None)[0] - model(shape, down, states, labels, None)[0])
        along = float(exact @ (up - down))
        norm = np.linalg.norm(exact[lo:hi]) * np.linalg.norm(up - down)
        assert abs(slope - along) <= 1e-4 * norm + 1e-9
        slack = np.linalg.norm(rounded_grad[lo:hi] - exact[lo:hi]) * np.linalg.norm(up - down)
        assert abs(slope - float(grad.astype(np.float64) @ (up - down))) <= 2 * slack + 2e-3 * norm + 1e-9, (lo, hi)


def test_scale_of_the_layer_in_front_does_not_matter(oracle):
    # every sample is normalised: weights and bias in front of a normalisation scaled by a power of two leave the rest as it is
    shape, w, states, labels = make_case(oracle, (72, 72, 64, 64, 1, 1), 256, seed=43)
    in_w = 72 * 72 * 64
    lo, hi = in_w + 64, in_w + 64 + 64 * 64 + 64
    w2 = w.copy()
    w2[lo:hi] *= 2.0
    eng = mgt.Engine(0)
    try:
        assert eng.set_layer_norm(True, 1e-12) == 0
        la, ga = run_engine(eng, shape, w, states, labels)
        lb, gb = run_engine(eng, shape, w2, states, labels)
    finally:
        eng.close()
    assert abs(la - lb) <= 1e-5 * abs(la) and rel_l2(gb[lo:hi] * 2.0, ga[lo:hi]) <= 1e-4
    rest = np.r_[0:lo, hi:w.size]
    assert rel_l2(gb[rest], ga[rest]) <= 1e-4


def test_option_errors():
    cshape = mgt.CudaMlpShape(8, 8, 16, 16, 2, 1)
    eng = mgt.Engine(0)
    try:
        assert eng.set_layer_norm(True, 0.0) == 1 and eng.set_layer_norm(True, float("nan")) == 1 and eng.set_layer_norm(True, float("inf")) == 1
        assert eng.set_layer_norm(True) == 0
        n = 32
        t = torch.zeros(cshape.param_count + mgt.bn_param_count(cshape), device=DEV)
        st8 = torch.zeros(n, 80, dtype=torch.uint8, device=DEV)
        small = mgt.mlp_loss_grad_workspace_floats(cshape, n)
        ws = torch.zeros(small, device=DEV)
        assert eng.launch_mlp_loss_grad(cshape, t, None, st8, t, n, t, t, ws, small) == 3
        assert eng.launch_mlp_loss_grad(cshape, t, None, st8, t, n, t, t, ws, small, use_half_linear=False) == 1
        assert eng.set_train_options(batch_norm=True) == 0
        assert eng.launch_mlp_loss_grad(cshape, t, None, st8, t, n, t, t, ws, small) == 1  # one normalisation or the other
    finally:
        eng.close()


def test_normalise_clip_and_update_in_one_captured_step(oracle):
    # the operators together, as a training loop runs them: loss and gradient, norm, clipped update, captured and replayed
    shape, w, states, labels = make_case(oracle, (72, 72, 128, 96, 2, 1), 700, seed=44)
    cshape = cshape_of(shape)
    n, total = states.shape[0], w.size
    floats = mgt.mlp_loss_grad_workspace_floats(cshape, n, layer_norm=True)
    ds, dl = torch.from_numpy(states).to(DEV), torch.from_numpy(np.ascontiguousarray(labels)).to(DEV)
    eng = mgt.Engine(0)
    assert eng.set_layer_norm(True) == 0

    def state():
        grad = torch.zeros(total, device=DEV)
        lst = mgt.TensorList([grad[:shape.param_count], grad[shape.param_count:]])
        k = mgt.gradient_norm_workspace_floats(lst)
        return dict(w=torch.from_numpy(w).to(DEV), m=torch.zeros(total, device=DEV), v=torch.zeros(total, device=DEV), grad=grad, lst=lst, loss=torch.zeros(1, device=DEV),
                    clip=torch.zeros(2, device=DEV), ws=torch.empty(floats, device=DEV), nws=torch.empty(k, device=DEV), k=k)

    def step(s):
        assert eng.launch_mlp_loss_grad(cshape, s["w"], None, ds, dl, n, s["loss"], s["grad"], s["ws"], floats) == 0
        assert mgt.launch_gradient_norm(s["lst"], 0.5, s["clip"], None, s["nws"], s["k"]) == 0
        assert mgt.launch_adamw_kernel_with_clip(mgt.AdamWKernelConfig(total, 1, 1e-3), s["w"], None, s["grad"], s["clip"], s["m"], s["v"]) == 0

    try:
        plain, captured = state(), state()
        step(plain)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(captured)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(plain[k], captured[k]) for k in ("w", "m", "v", "grad", "loss", "clip"))
        g = plain["grad"].double()
        norm = float(g.norm())
        assert abs(float(plain["clip"][0]) - norm) <= 1e-6 * norm and abs(float(plain["clip"][1]) - min(1.0, 0.5 / norm)) <= 1e-6
        # the moments tell what gradient the update saw
        seen = plain["m"].double() / 0.1
        assert rel_l2(seen.cpu().numpy(), (g * float(plain["clip"][1])).cpu().numpy()) <= 1e-6
    finally:
        eng.close()


def run_trainer(out_dir, *flags, check=True):
    cmd = [BIN, "--output-dir", str(out_dir), "--device-id", 0, "--world-size", 1, "--global-rank", 0, "--local-rank", 0, *flags]
    res = subprocess.run([str(c) for c in cmd], capture_output=True, text=True, timeout=300)
    if check:
        assert res.returncode == 0, res.stderr + res.stdout
    return res


def model_training(oracle, shape, *, batch, steps, lr, max_norm=0.0, seed=1234):
    moves, target = oracle.cyclic_puzzle(72, 18)
    p, nn = shape.param_count, 2 * (shape.residual_blocks + 1) * shape.hd2
    w = np.concatenate([trainer_init_weights(p), np.zeros(nn, np.float32)])
    w[p:].reshape(-1, 2, shape.hd2)[:, 0, :] = 1.0
    m, v = np.zeros_like(w), np.zeros_like(w)
    losses, norms = [], []
    for step in range(steps):
        _, states, depth, _ = oracle.random_walks(moves, target, seed=seed, epoch=0, step=step, rank=0, k_min=1, k_max=29, samples=batch)
        loss, grad = model(shape, w, states, depth.reshape(-1, 1), torch.float16)
        norm = np.linalg.norm(grad)
        norms.append(norm)
        grad = grad * (max_norm / norm if 0 < max_norm < norm else 1.0)
        assert oracle.adamw(w, grad.astype(np.float32), m, v, step=step + 1, lr=lr) == 0
        losses.append(loss)
    return w, losses, norms


def test_trainer_with_layer_norm_and_clipping(tmp_path, oracle):
    shape = MlpShape(72, 72, 256, 64, 2, 1)
    common = ["--batch-size", 512, "--k-min", 1, "--k-max", 29, "--hd1", 256, "--hd2", 64, "--nrd", 2, "--lr", 0.001, "--layer-norm", 1, "--max-grad-norm", 0.75]
    d = tmp_path / "ln"
    run_trainer(d, "--steps", 3, *common)
    w, losses, norms = model_training(oracle, shape, batch=512, steps=3, lr=1e-3, max_norm=0.75)
    rows = [json.loads(line) for line in open(d / "profile.jsonl")]
    for row, want in zip(rows, losses):
        assert abs(row["loss"] - want) <= 2e-3 * abs(want), (row["loss"], want)
    clips = [json.loads(line) for line in open(d / "grad_norm.jsonl")]
    assert [c["step"] for c in clips] == [0, 1, 2]
    for c, norm in zip(clips, norms):
        assert abs(c["grad_norm"] - norm) <= 2e-2 * norm and abs(c["scale"] - min(1.0, 0.75 / c["grad_norm"])) <= 1e-6
    p, nn = shape.param_count, 2 * 3 * 64
    state = np.fromfile(d / "checkpoint" / "state.f32.bin", np.float32)
    extra = np.fromfile(d / "checkpoint" / "layer_norm.f32.bin", np.float32)
    assert state.size == 3 * p and extra.size == 3 * nn
    meta = json.load(open(d / "checkpoint" / "layer_norm.json"))
    assert meta["layers"] == 3 and meta["width"] == 64 and meta["section_floats"] == nn
    # weights/ holds the network as it is, the scale/shift vectors beside it, and says so
    assert np.array_equal(np.fromfile(d / "weights" / "weights.f32.bin", np.float32), state[:p])
    assert np.array_equal(np.fromfile(d / "weights" / "layer_norm.f32.bin", np.float32), extra[:nn])
    assert json.load(open(d / "weights" / "manifest.json"))["normalization"] == "layer_norm"
    # 2 + 1 steps through a checkpoint end in the state of 3 steps in one run
    run_trainer(tmp_path / "two", "--steps", 2, *common)
    run_trainer(tmp_path / "third", "--steps", 1, "--resume-checkpoint", tmp_path / "two" / "checkpoint", "--resume-step", 1, *common)
    assert np.array_equal(np.fromfile(tmp_path / "third" / "checkpoint" / "state.f32.bin", np.float32), state)
    assert np.array_equal(np.fromfile(tmp_path / "third" / "checkpoint" / "layer_norm.f32.bin", np.float32), extra)
    # a norm far above the gradient's changes nothing: bit for bit the run without clipping
    a, b = tmp_path / "loose", tmp_path / "none"
    run_trainer(a, "--steps", 2, *common[:-1], 1e9)
    run_trainer(b, "--steps", 2, *common[:-2])
    assert np.array_equal(np.fromfile(a / "checkpoint" / "state.f32.bin", np.float32), np.fromfile(b / "checkpoint" / "state.f32.bin", np.float32))
    assert not os.path.exists(b / "grad_norm.jsonl")
    # without a mirror of the weights, with the stages timed, without files
    run_trainer(tmp_path / "other", "--steps", 2, *common, "--persistent-half-weights", 0, "--backward-profile", 1, "--write-artifacts", 0)
    other = [json.loads(line)["grad_norm"] for line in open(tmp_path / "other" / "grad_norm.jsonl")]
    assert other == [c["grad_norm"] for c in clips[:2]]  # (the mirror holds what the step rounds itself)
    for bad in (("--ln-eps", 0), ("--max-grad-norm", -1), ("--batch-norm", 1), ("--linear-fp16", 0)):
        assert run_trainer(tmp_path / "bad", "--steps", 1, *common, *bad, check=False).returncode != 0, bad
    # without the normalisation's checkpoint a run with it cannot be resumed
    run_trainer(tmp_path / "plain", "--steps", 1, *common[:-4])
    assert run_trainer(tmp_path / "bad2", "--steps", 1, "--resume-checkpoint", tmp_path / "plain" / "checkpoint", *common, check=False).returncode != 0
