"""Operator cases: layer normalisation with its backward pass, the norm of a gradient over all tensors of a model, clipping, and
the clipped AdamW update, over the range of batches, widths, models and types that training meets.

`run` makes one pass through one operator: in its plain form (elementary torch operations), or by the framework's calls when `own`
is set. Everything comes from the seed. Buffers that the calls write are made by `prepare`, as a training program makes them once;
the tensors of a gradient are views of one flat buffer in the order of the model's parameters, so their addresses are what they are.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the smallest batch through the narrowest model: launch latency
        dict(name="norm_layer_64x8", op="layer_norm", rows=64, cols=8, x="f32", y="f32", pad=0),
        # a ragged batch of a width that is a multiple of nothing, in half precision
        dict(name="norm_layer_9001x77_f16", op="layer_norm", rows=9001, cols=77, x="f16", y="f16", pad=0),
        # pre-activations of the p888 hidden layer to the 16-bit operand of the next product
        dict(name="norm_layer_53248x224_f32_f16", op="layer_norm", rows=53248, cols=224, x="f32", y="f16", pad=0),
        # the widest residual stream and the largest batch, in bfloat16
        dict(name="norm_layer_131072x512_bf16", op="layer_norm", rows=131072, cols=512, x="bf16", y="bf16", pad=0),
        # backward: the tiny model
        dict(name="norm_grad_1024x64", op="layer_norm_grad", rows=1024, cols=64, x="f32", y="f32", pad=0),
        # backward: p888, fp32 gradients and pre-activations in rows with a pitch
        dict(name="norm_grad_53248x224_pitch", op="layer_norm_grad", rows=53248, cols=224, x="f32", y="f32", pad=8),
        # backward: as wide as the widest hidden layer, bfloat16
        dict(name="norm_grad_16384x4096_bf16", op="layer_norm_grad", rows=16384, cols=4096, x="bf16", y="bf16", pad=0),
        # the gradient norm of the tiny model (1.36 M parameters) and of p888 (15.5 M in 70 tensors)
        dict(name="grad_norm_tiny", op="grad_norm", state_len=72, values=72, hd1=256, hd2=64, blocks=2, outputs=1, x="f32"),
        dict(name="grad_norm_p888", op="grad_norm", state_len=72, values=72, hd1=2560, hd2=224, blocks=16, outputs=1, x="f32"),
        # norm and clipping, bfloat16 gradients of a model of odd sizes: most tensors begin off any boundary
        dict(name="clip_odd_bf16", op="clip", state_len=72, values=72, hd1=1333, hd2=177, blocks=9, outputs=29, x="bf16"),
        # norm and clipped update: a small puzzle's model, and p888 with the fp16 mirror of the weights
        dict(name="update_cube54", op="update", state_len=54, values=6, hd1=1024, hd2=256, blocks=4, outputs=1, mirror=False, decay=0.01),
        dict(name="update_p888", op="update", state_len=72, values=72, hd1=2560, hd2=224, blocks=16, outputs=1, mirror=True, decay=0.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm_grad", "grad_norm", "clip", "update"])
    if op.startswith("layer_norm"):
        cols = _log_int(rng, 1, 16384)
        if rng.random() < 0.5:  # widths as models have them
            cols = (cols + 7) // 8 * 8
        x = rng.choice(["f32", "f16", "bf16"])
        y = rng.choice(["f32", "f16", "bf16"]) if x == "f32" else rng.choice([x, x, "f32"])
        rows = _log_int(rng, 1, min(131072, 60_000_000 // cols))
        return dict(op=op, rows=rows, cols=cols, x=x, y=y, pad=rng.choice([0, 0, 0, 8, rng.randint(1, 40)]))
    case = dict(op=op, state_len=rng.randint(16, 72), values=rng.randint(4, 72), hd1=_log_int(rng, 8, 4096), hd2=_log_int(rng, 8, 512),
                blocks=rng.randint(0, 32), outputs=rng.choice([1, 1, rng.randint(2, 40)]))
    if rng.random() < 0.5:
        case["hd1"], case["hd2"] = (case["hd1"] + 7) // 8 * 8, (case["hd2"] + 7) // 8 * 8
    if op == "update":
        case.update(mirror=rng.random() < 0.5, decay=rng.choice([0.0, 0.01]))
    else:
        case["x"] = rng.choice(["f32", "f32", "f16", "bf16"])
    return case


def _counts(c):
    """Elements of every parameter tensor, in the order of the flat parameters."""
    h1, h2 = c["hd1"], c["hd2"]
    return [c["state_len"] * c["values"] * h1, h1, h1 * h2, h2] + [h2 * h2, h2] * (2 * c["blocks"]) + [h2 * c["outputs"], c["outputs"]]


def _prepare_layer_norm(c, dev, g):
    rows, cols, pitch = c["rows"], c["cols"], c["cols"] + c["pad"]

    def rows_of(kind):
        return torch.empty(rows, pitch, dtype=TYPES[kind], device=dev)

    # pre-activations: features of unlike scale and offset, samples of unlike size
    x = torch.randn(rows, pitch, device=dev, generator=g)
    x *= 0.5 + torch.rand(pitch, device=dev, generator=g)
    x += 0.5 * torch.randn(pitch, device=dev, generator=g)
    x *= 0.25 + 2.0 * torch.rand(rows, 1, device=dev, generator=g)
    x = x.to(TYPES[c["x"]])
    s = {"op": c["op"], "rows": rows, "cols": cols, "x": x, "gamma": 1.0 + 0.2 * torch.randn(cols, device=dev, generator=g),
         "beta": 0.1 * torch.randn(cols, device=dev, generator=g), "mean": torch.empty(rows, device=dev), "rstd": torch.empty(rows, device=dev)}
    if own:
        import multigputrainmlp_b200 as mgt
        kinds = {"f32": mgt.F32, "f16": mgt.F16, "bf16": mgt.BF16}
        s["mgt"] = mgt
        s["config"] = mgt.LayerNormConfig(rows, cols, EPS, x_type=kinds[c["x"]], y_type=kinds[c["y"]], x_pitch=pitch, y_pitch=pitch, dx_pitch=pitch)
    if c["op"] == "layer_norm":
        s["y"] = rows_of(c["y"])
        return s
    for lo in range(0, rows, 16384):  # the statistics that the forward pass left
        part = x[lo:lo + 16384, :cols].double()
        m = part.mean(1, keepdim=True)
        s["mean"][lo:lo + 16384] = m[:, 0]
        s["rstd"][lo:lo + 16384] = ((part - m).square().mean(1) + EPS).rsqrt()
    s["dy"] = (torch.randn(rows, pitch, device=dev, generator=g) / rows).to(TYPES[c["y"]])
    s["dx"] = rows_of(c["x"])
    for k in ("dgamma", "dbeta", "dbias"):
        s[k] = torch.empty(cols, device=dev)
    if own:
        s["floats"] = s["mgt"].layer_norm_backward_workspace_floats(s["config"])
        s["workspace"] = torch.empty(s["floats"], device=dev)
    return s


def prepare(case, seed):
    c = dict(case)
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    if c["op"].startswith("layer_norm"):
        return _prepare_layer_norm(c, dev, g)
    counts = _counts(c)
    total = sum(counts)
    flat = torch.randn(total, device=dev, generator=g) * 1e-3
    # units whose ReLU never opens: a seventh of the gradient is exactly zero
    flat *= torch.rand(total // 64 + 1, device=dev, generator=g).gt(1 / 7).repeat_interleave(64)[:total]
    flat = flat.to(TYPES[c.get("x", "f32")])
    s = {"op": c["op"], "total": total, "flat": flat, "parts": flat.split(counts), "max_norm": 1.0 if c["op"] != "grad_norm" else 1e9,
         "result": torch.empty(2, device=dev), "norms": torch.empty(len(counts), device=dev)}
    if c["op"] == "clip":
        s["out"] = torch.empty_like(flat)
    if c["op"] == "update":
        s["max_norm"] = 0.5
        s["step"], s["decay"] = 101, c["decay"]
        s["w"] = torch.randn(total, device=dev, generator=g) * 0.05
        s["m"] = torch.randn(total, device=dev, generator=g) * 1e-4
        s["v"] = 1e-6 * (0.5 + torch.rand(total, device=dev, generator=g))
        s["w_half"] = s["w"].half() if c["mirror"] else None
    if own:
        import multigputrainmlp_b200 as mgt
        s["mgt"] = mgt
        s["tensors"] = mgt.TensorList(s["parts"])  # built once by a program whose gradients stay where they are
        if c["op"] == "clip":
            s["out_tensors"] = mgt.TensorList(s["out"].split(counts))
        s["floats"] = mgt.gradient_norm_workspace_floats(s["tensors"])
        s["workspace"] = torch.empty(s["floats"], device=dev)
        if c["op"] == "update":
            s["adamw"] = mgt.AdamWKernelConfig(total, s["step"], 1e-4, weight_decay=c["decay"])
    return s


def _checked(status):
    if status != 0:
        raise RuntimeError("status %d" % status)


def _run_own(s):
    mgt = s["mgt"]
    if s["op"] == "layer_norm":
        _checked(mgt.launch_layer_norm(s["config"], s["x"], s["gamma"], s["beta"], s["y"], s["mean"], s["rstd"]))
        return {"y": s["y"][:, :s["cols"]], "mean": s["mean"], "rstd": s["rstd"]}
    if s["op"] == "layer_norm_grad":
        _checked(mgt.launch_layer_norm_backward(s["config"], s["dy"], s["x"], s["gamma"], s["mean"], s["rstd"], s["dx"], s["dgamma"], s["dbeta"],
                                                s["dbias"], s["workspace"], s["floats"]))
        return {"dx": s["dx"][:, :s["cols"]], "dgamma": s["dgamma"], "dbeta": s["dbeta"], "dbias": s["dbias"]}
    _checked(mgt.launch_gradient_norm(s["tensors"], s["max_norm"], s["result"], s["norms"], s["workspace"], s["floats"]))
    out = {"result": s["result"], "norms": s["norms"]}
    if s["op"] == "clip":
        _checked(mgt.launch_clip_gradients(s["tensors"], s["result"], s["out_tensors"]))
        out["clipped"] = s["out"]
    if s["op"] == "update":
        _checked(mgt.launch_adamw_kernel_with_clip(s["adamw"], s["w"], s["w_half"], s["flat"], s["result"], s["m"], s["v"]))
        out.update({k: s[k] for k in ("w", "m", "v", "w_half") if s[k] is not None})
    return out


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "layer_norm":
        x = s["x"][:, :s["cols"]].float()
        mean = x.mean(1)
        d = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((d * d).mean(1) + EPS)
        y = d * rstd[:, None] * s["gamma"] + s["beta"]
        return {"y": y.to(s["y"].dtype), "mean": mean, "rstd": rstd}
    if s["op"] == "layer_norm_grad":
        dy, x = s["dy"][:, :s["cols"]].float(), s["x"][:, :s["cols"]].float()
        xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
        gy = dy * s["gamma"]
        dx = s["rstd"][:, None] * (gy - gy.mean(1, keepdim=True) - xhat * (gy * xhat).mean(1, keepdim=True))
        return {"dx": dx.to(s["dx"].dtype), "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0), "dbias": dx.sum(0)}
    squares = torch.stack([p.double().square().sum() for p in s["parts"]])
    norm = squares.sum().sqrt().float()
    scale = torch.where(norm.isfinite(), (s["max_norm"] / norm.double()).clamp(max=1.0), 0.0).float()
    out = {"result": torch.stack([norm, scale]), "norms": squares.sqrt().float()}
    if s["op"] == "clip":
        out["clipped"] = (s["flat"].float() * scale).to(s["flat"].dtype)
    if s["op"] == "update":
        w, m, v = s["w"], s["m"], s["v"]
        grad = s["flat"] * scale + s["decay"] * w
        m.mul_(0.9).add_(0.1 * grad)
        v.mul_(0.999).add_((1.0 - _f32(0.999)) * grad * grad)
        m_hat, v_hat = m / (1.0 - 0.9 ** s["step"]), v / (1.0 - _f32(0.999) ** s["step"])
        w.sub_(1e-4 * m_hat / (v_hat.sqrt() + 1e-8))
        out.update(w=w, m=m, v=v)
        if s["w_half"] is not None:
            s["w_half"].copy_(w)
            out["w_half"] = s["w_half"]
    return out


def _f32(value):
    """The value that a 32-bit argument holds."""
    return torch.tensor(value, dtype=torch.float32).item()


def work(case):
    c = dict(case)
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["op"].startswith("layer_norm"):
        n, sx, sy = c["rows"] * c["cols"], size[c["x"]], size[c["y"]]
        if c["op"] == "layer_norm":
            return {"bytes": n * (sx + sy) + 8 * c["rows"] + 8 * c["cols"], "flops": 8 * n}
        return {"bytes": n * (2 * sx + sy) + 8 * c["rows"] + 16 * c["cols"], "flops": 18 * n}
    total, tensors = sum(_counts(c)), len(_counts(c))
    if c["op"] == "update":
        return {"bytes": total * (30 if c["mirror"] else 28) + 4 * tensors + 8, "flops": 20 * total}
    per = size[c["x"]] * (2 if c["op"] == "clip" else 1)
    return {"bytes": total * per + 4 * tensors + 8, "flops": (3 if c["op"] == "clip" else 2) * total}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "layer_norm":
        x = s["x"].double()[:, :s["cols"]]
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = (var + EPS) ** -0.5
        y = torch.addcmul(s["beta"].double(), (x - mean.unsqueeze(1)) * s["gamma"].double(), rstd.unsqueeze(1))
        return {"y": y, "mean": mean, "rstd": rstd}
    if s["op"] == "layer_norm_grad":
        dy, gamma, rstd = s["dy"].double()[:, :s["cols"]], s["gamma"].double(), s["rstd"].double()
        xhat = (s["x"].double()[:, :s["cols"]] - s["mean"].double().unsqueeze(1)) * rstd.unsqueeze(1)
        n = float(s["cols"])
        along = torch.einsum("rc,rc,c->r", dy, xhat, gamma) / n
        dx = torch.addmm((dy * gamma), (torch.mv(dy, gamma) / -n).unsqueeze(1), torch.ones(1, s["cols"], dtype=torch.float64, device=dy.device))
        dx = (dx - along.unsqueeze(1) * xhat) * rstd.unsqueeze(1)
        return {"dx": dx, "dgamma": torch.einsum("rc,rc->c", dy, xhat), "dbeta": dy.sum(0), "dbias": dx.sum(0)}
    g = s["flat"].double()
    norms = torch.cat([torch.linalg.vector_norm(p.double()).reshape(1) for p in s["parts"]])
    norm = torch.linalg.vector_norm(g)
    scale = s["max_norm"] / norm if norm > s["max_norm"] else torch.ones_like(norm)
    out = {"result": torch.cat([norm.reshape(1), scale.reshape(1)]), "norms": norms}
    if s["op"] == "clip":
        out["clipped"] = g * scale
    if s["op"] == "update":
        b1, b2, t = _f32(0.9), _f32(0.999), s["step"]
        w = s["w"].double()
        g = torch.add(g * scale, w, alpha=_f32(s["decay"]))
        m = torch.lerp(g, s["m"].double(), b1)
        v = torch.lerp(g.square(), s["v"].double(), b2)
        out.update(w=w - _f32(1e-4) * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + _f32(1e-8)), m=m, v=v)
        if s["w_half"] is not None:
            out["w_half"] = out["w"]
    return out
