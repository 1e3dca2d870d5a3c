"""Layer normalisation against plain 64-bit arithmetic, over types, widths, pitches and alignments.

Tolerances. With u = 2^-24 a sum of n fp32 terms, each thread adding at most e = 16 (or cols / 1024 in the widest rows) of them in order and
the threads by trees of at most 10 levels, is off by at most (e + 10) u of the sum of absolute values; a product or difference adds u. A
row's mean (twice corrected), variance, rstd and the two means of the backward pass are such sums and some single operations beside
them, so K = 64 + cols / 1024 times u bounds each of the errors below relative to the absolute terms that it is made of. Results in 16
bits are off by half a step more (2^-11 and 2^-8 of the value, and half the smallest fp16 number)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

import multigputrainmlp_b200 as mgt  # noqa: E402

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = {"f32": (mgt.F32, torch.float32), "f16": (mgt.F16, torch.float16), "bf16": (mgt.BF16, torch.bfloat16)}
EPS = 1e-5
MARK = 7.0  # what lies beyond the columns


def half_step(kind, value):
    if kind == "f32":
        return U * value.abs()
    return torch.finfo(TYPES[kind][1]).eps / 2 * value.abs() + (2.0 ** -25 if kind == "f16" else 0.0)


class Rows:
    """A [rows][cols] matrix whose rows lie `pitch` apart, `offset` elements behind an allocation's begin; the rest is MARK."""

    def __init__(self, rows, cols, kind, pad=0, offset=0, values=None):
        self.pitch, self.cols, self.offset, self.kind = cols + pad, cols, offset, kind
        self.buffer = torch.full((offset + rows * self.pitch + 8,), MARK, device=DEV, dtype=TYPES[kind][1])
        self.at = self.buffer[offset:]
        self.view = self.at[:rows * self.pitch].view(rows, self.pitch)[:, :cols]
        if values is not None:
            self.view.copy_(values)

    def rest_untouched(self):
        copy = self.buffer.clone()
        copy[self.offset:][:self.view.shape[0] * self.pitch].view(-1, self.pitch)[:, :self.cols] = MARK
        return bool((copy == MARK).all())


def exact_forward(x, gamma, beta):
    x = x.double()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((d * d).mean(1) + EPS)
    g = torch.ones(x.shape[1], device=DEV, dtype=torch.float64) if gamma is None else gamma.double()
    b = torch.zeros_like(g) if beta is None else beta.double()
    return d * rstd[:, None] * g + b, mean, rstd, d * rstd[:, None], g, b


def check_forward(x, y_kind, y, mean, rstd, gamma, beta):
    cols = x.shape[1]
    k = (64 + cols / 1024) * U
    want, m, r, xhat, g, b = exact_forward(x, gamma, beta)
    spread = xhat.abs().amax(1, keepdim=True)
    tol = k * (g.abs() * spread + b.abs())
    assert ((y.double() - want).abs() <= tol + half_step(y_kind, want.abs() + tol)).all()
    if mean is not None:
        assert ((mean.double() - m).abs() <= U * m.abs() + k * (x.double() - m[:, None]).abs().amax(1)).all()
    if rstd is not None:
        assert ((rstd.double() - r).abs() <= k * r).all()


def make(rows, cols, seed, offset=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, cols, device=DEV, generator=g) * (0.5 + torch.rand(cols, device=DEV, generator=g)) + offset
    gamma = 1.0 + 0.3 * torch.randn(cols, device=DEV, generator=g)
    beta = 0.2 * torch.randn(cols, device=DEV, generator=g)
    return x, gamma, beta, g


FORWARD_TYPES = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")]
SHAPES = [(1, 1), (5, 2), (1, 224), (64, 8), (3, 31), (33, 77), (129, 224), (257, 512), (1300, 224), (100, 513), (40, 1000), (9, 4096), (5, 4097), (700, 2048),
          (3, 8192), (3, 8193), (2, 16384), (301, 9000), (3, 16385), (40, 20000), (1, 16386)]
# one of each layout: single columns by 8 and by 32 lanes, packs of four in 16 bits, whole warps of packs
SHAPES += [(10000, 11), (10000, 27), (10000, 61), (10000, 125), (6000, 77), (2500, 131), (2500, 231), (2500, 301), (2500, 501), (3000, 100), (50, 1004), (5, 5004),
           (3000, 512), (2000, 1024), (500, 2050)]


@pytest.mark.parametrize("x_kind,y_kind", FORWARD_TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(rows, cols, x_kind, y_kind):
    values, gamma, beta, _ = make(rows, cols, rows * 31 + cols)
    for pad, offset in ((0, 0), (8, 8), (3, 1)):
        x = Rows(rows, cols, x_kind, pad, offset, values)
        y = Rows(rows, cols, y_kind, pad, offset)
        mean, rstd = Rows(1, rows, "f32"), Rows(1, rows, "f32")
        cfg = mgt.LayerNormConfig(rows, cols, EPS, TYPES[x_kind][0], TYPES[y_kind][0], x_pitch=x.pitch, y_pitch=y.pitch)
        assert mgt.launch_layer_norm(cfg, x.at, gamma, beta, y.at, mean.at, rstd.at) == 0
        check_forward(x.view, y_kind, y.view, mean.view[0], rstd.view[0], gamma, beta)
        assert all(b.rest_untouched() for b in (x, y, mean, rstd))


def test_forward_without_scale_shift_statistics():
    values, gamma, beta, _ = make(70, 224, 1)
    cfg = mgt.LayerNormConfig(70, 224)
    for g, b in ((None, None), (gamma, None), (None, beta)):
        y = torch.empty_like(values)
        assert mgt.launch_layer_norm(cfg, values, g, b, y) == 0
        check_forward(values, "f32", y, None, None, g, b)
    one = torch.full((1, 20000), 3.0, device=DEV)
    y = torch.empty_like(one)
    assert mgt.launch_layer_norm(mgt.LayerNormConfig(1, 20000), one, None, None, y) == 0
    assert (y == 0.0).all()  # a row of one value has no spread


@pytest.mark.parametrize("offset", [1e3, -1e4])
@pytest.mark.parametrize("cols", [7, 224, 4096, 9000])
def test_rows_far_from_zero(cols, offset):
    values, gamma, beta, _ = make(50, cols, cols, offset)
    cfg = mgt.LayerNormConfig(50, cols)
    y, mean, rstd = torch.empty_like(values), torch.empty(50, device=DEV), torch.empty(50, device=DEV)
    assert mgt.launch_layer_norm(cfg, values, gamma, beta, y, mean, rstd) == 0
    check_forward(values, "f32", y, mean, rstd, gamma, beta)


def exact_backward(dy, x, gamma, mean, rstd):
    dy, x, mean, rstd = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    g = dy if gamma is None else dy * gamma.double()
    xhat = (x - mean) * rstd
    c1, c2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    dx = rstd * (g - c1 - xhat * c2)
    terms = rstd * (g.abs() + g.abs().mean(1, keepdim=True) + xhat.abs() * (g * xhat).abs().mean(1, keepdim=True))  # what dx's error is relative to
    return dx, xhat, terms


def check_backward(dy, x, gamma, mean, rstd, dx, dx_kind, sums):
    rows, cols = x.shape
    k = (64 + cols / 1024) * U
    # a column's sum: in order over a thread's rows (a slice of 1 / 37 at most) and over up to 256 groups of a CTA, then 5 in order and a tree
    ks = (64 + rows / 37 + 256) * U
    want, xhat, terms = exact_backward(dy, x, gamma, mean, rstd)
    assert ((dx.double() - want).abs() <= k * terms + half_step(dx_kind, want.abs() + k * terms)).all()
    d = dy.double()
    for got, exact, size in zip(sums, (d * xhat, d, want), (d * xhat, d, terms)):
        if got is not None:
            assert ((got.double() - exact.sum(0)).abs() <= (ks + k) * size.abs().sum(0) + 1e-37).all()


BACKWARD_TYPES = [("f32", "f32", "f32"), ("f32", "f32", "f16"), ("f32", "f32", "bf16"), ("f16", "f32", "f32"), ("bf16", "f32", "f32"), ("f16", "f16", "f16"),
                  ("f32", "f16", "f16"), ("bf16", "bf16", "bf16"), ("f32", "bf16", "bf16")]  # dy, x, dx


@pytest.mark.parametrize("dy_kind,x_kind,dx_kind", BACKWARD_TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES + [(5000, 24), (2500, 1)])
def test_backward(rows, cols, dy_kind, x_kind, dx_kind):
    values, gamma, _, g = make(rows, cols, rows * 17 + cols)
    dvalues = torch.randn(rows, cols, device=DEV, generator=g)
    for pad, offset in ((0, 0), (8, 8), (3, 1)):
        x, dy, dx = Rows(rows, cols, x_kind, pad, offset, values), Rows(rows, cols, dy_kind, pad, offset, dvalues), Rows(rows, cols, dx_kind, pad, offset)
        _, m, r, *_ = exact_forward(x.view, None, None)
        mean, rstd = m.float(), r.float()
        sums = [Rows(1, cols, "f32") for _ in range(3)]
        cfg = mgt.LayerNormConfig(rows, cols, EPS, TYPES[x_kind][0], TYPES[dy_kind][0], TYPES[dx_kind][0], x.pitch, dy.pitch, dx.pitch)
        floats = mgt.layer_norm_backward_workspace_floats(cfg)
        ws = torch.full((floats + 64,), float("nan"), device=DEV)
        ws[floats:] = MARK
        assert mgt.launch_layer_norm_backward(cfg, dy.at, x.at, gamma, mean, rstd, dx.at, *[s.at for s in sums], ws, floats) == 0
        check_backward(dy.view, x.view, gamma, mean, rstd, dx.view, dx_kind, [s.view[0] for s in sums])
        assert all(b.rest_untouched() for b in (x, dy, dx, *sums)) and (ws[floats:] == MARK).all()


@pytest.mark.parametrize("rows,cols", [(64, 8), (900, 224), (4, 9000)])
def test_backward_sums_that_are_not_wanted(rows, cols):
    values, gamma, _, g = make(rows, cols, 3)
    dy = torch.randn(rows, cols, device=DEV, generator=g)
    _, m, r, *_ = exact_forward(values, None, None)
    cfg = mgt.LayerNormConfig(rows, cols)
    floats = mgt.layer_norm_backward_workspace_floats(cfg)
    for wanted in range(8):
        sums = [torch.full((cols,), MARK, device=DEV) if wanted >> k & 1 else None for k in range(3)]
        dx, ws = torch.empty_like(values), torch.empty(floats, device=DEV)
        scale = gamma if wanted & 1 else None
        assert mgt.launch_layer_norm_backward(cfg, dy, values, scale, m.float(), r.float(), dx, *sums, ws, floats) == 0
        check_backward(dy, values, scale, m.float(), r.float(), dx, "f32", sums)


@pytest.mark.parametrize("cols", [1, 6, 40])
def test_gradients_against_differences(cols):
    rows = 5
    values, gamma, beta, g = make(rows, cols, cols)
    dy = torch.randn(rows, cols, device=DEV, generator=g)
    y, mean, rstd = torch.empty_like(values), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    cfg = mgt.LayerNormConfig(rows, cols)
    assert mgt.launch_layer_norm(cfg, values, gamma, beta, y, mean, rstd) == 0
    dx, dgamma, dbeta, dbias = torch.empty_like(values), *[torch.empty(cols, device=DEV) for _ in range(3)]
    floats = mgt.layer_norm_backward_workspace_floats(cfg)
    assert mgt.launch_layer_norm_backward(cfg, dy, values, gamma, mean, rstd, dx, dgamma, dbeta, dbias, torch.empty(floats, device=DEV), floats) == 0

    def loss(x, ga, be):
        return float((exact_forward(x, ga, be)[0] * dy.double()).sum())

    h = 1e-4
    x64, g64, b64 = values.double(), gamma.double(), beta.double()
    for r in range(rows):
        for c in range(cols):
            step = torch.zeros_like(x64)
            step[r, c] = h
            slope = (loss(x64 + step, g64, b64) - loss(x64 - step, g64, b64)) / (2 * h)
            assert abs(slope - float(dx[r, c])) <= 1e-5 * (1 + float(dx.abs().max()))  # third derivatives times h^2 / 6, fp32 results
    for c in range(cols):
        step = torch.zeros_like(g64)
        step[c] = h
        assert abs((loss(x64, g64 + step, b64) - loss(x64, g64 - step, b64)) / (2 * h) - float(dgamma[c])) <= 1e-5 * (1 + float(dgamma.abs().max()))
        assert abs((loss(x64, g64, b64 + step) - loss(x64, g64, b64 - step)) / (2 * h) - float(dbeta[c])) <= 1e-5 * (1 + float(dbeta.abs().max()))


def test_no_rows():
    cfg = mgt.LayerNormConfig(0, 40)
    empty = torch.empty(0, 40, device=DEV)
    assert mgt.launch_layer_norm(cfg, empty, None, None, empty, None, None) == 0
    sums = [torch.full((40,), MARK, device=DEV) for _ in range(3)]
    floats = mgt.layer_norm_backward_workspace_floats(cfg)
    assert mgt.launch_layer_norm_backward(cfg, empty, empty, None, None, None, empty, *sums, torch.empty(floats, device=DEV), floats) == 0
    assert all((s == 0).all() for s in sums)


@pytest.mark.parametrize("rows,cols,kind", [(600, 224, "f32"), (301, 77, "f16"), (50, 4096, "bf16"), (7, 9000, "f32"), (700, 8, "bf16")])
def test_in_place(rows, cols, kind):
    values, gamma, beta, g = make(rows, cols, 9)
    x = values.to(TYPES[kind][1])
    dy = torch.randn(rows, cols, device=DEV, generator=g).to(x.dtype)
    cfg = mgt.LayerNormConfig(rows, cols, EPS, TYPES[kind][0], TYPES[kind][0])
    y, mean, rstd = torch.empty_like(x), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    assert mgt.launch_layer_norm(cfg, x, gamma, beta, y, mean, rstd) == 0
    same = x.clone()
    assert mgt.launch_layer_norm(cfg, same, gamma, beta, same) == 0
    assert torch.equal(same, y)
    floats = mgt.layer_norm_backward_workspace_floats(cfg)
    ws, sums = torch.empty(floats, device=DEV), [torch.empty(cols, device=DEV) for _ in range(3)]
    dx = torch.empty_like(x)
    assert mgt.launch_layer_norm_backward(cfg, dy, x, gamma, mean, rstd, dx, *sums, ws, floats) == 0
    for over_dy in (True, False):
        a, b, again = dy.clone(), x.clone(), [torch.empty(cols, device=DEV) for _ in range(3)]
        assert mgt.launch_layer_norm_backward(cfg, a, b, gamma, mean, rstd, a if over_dy else b, *again, ws, floats) == 0
        assert torch.equal(a if over_dy else b, dx) and all(torch.equal(p, q) for p, q in zip(sums, again))


@pytest.mark.parametrize("cols", [8, 224, 2048, 9000])
def test_rows_that_are_not_finite_stay_alone(cols):
    values, gamma, beta, _ = make(20, cols, 2)
    bad = values.clone()
    bad[3, cols - 1], bad[7, 0], bad[8, cols // 2] = float("nan"), float("inf"), float("-inf")
    cfg = mgt.LayerNormConfig(20, cols)
    a, b, mean, rstd = torch.empty_like(values), torch.empty_like(values), torch.empty(20, device=DEV), torch.empty(20, device=DEV)
    assert mgt.launch_layer_norm(cfg, values, gamma, beta, a) == 0
    assert mgt.launch_layer_norm(cfg, bad, gamma, beta, b, mean, rstd) == 0
    rows = torch.tensor([3, 7, 8], device=DEV)
    keep = torch.ones(20, dtype=torch.bool, device=DEV)
    keep[rows] = False
    assert torch.equal(a[keep], b[keep]) and b[rows].isnan().all() and rstd[rows].isnan().all() and rstd[keep].isfinite().all()


@pytest.mark.parametrize("rows,cols", [(4000, 224), (900, 1024), (40, 9000)])
def test_same_results_every_time_on_any_stream_and_from_a_graph(rows, cols):
    values, gamma, beta, g = make(rows, cols, 5)
    dy = torch.randn(rows, cols, device=DEV, generator=g)
    cfg = mgt.LayerNormConfig(rows, cols)
    floats = mgt.layer_norm_backward_workspace_floats(cfg)

    def buffers():
        return [torch.empty_like(values), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV), torch.empty_like(values),
                *[torch.empty(cols, device=DEV) for _ in range(3)], torch.full((floats,), float("nan"), device=DEV)]

    def step(b, x=values):
        assert mgt.launch_layer_norm(cfg, x, gamma, beta, b[0], b[1], b[2]) == 0
        assert mgt.launch_layer_norm_backward(cfg, dy, x, gamma, b[1], b[2], *b[3:7], b[7], floats) == 0

    first = buffers()
    step(first)
    side = [torch.cuda.Stream() for _ in range(2)]
    both = [buffers() for _ in side]
    torch.cuda.synchronize()
    for s, b in zip(side, both):  # two at once, each with a workspace
        with torch.cuda.stream(s):
            step(b)
    torch.cuda.synchronize()
    for b in both:
        assert all(torch.equal(p, q) for p, q in zip(first[:7], b[:7]))
    captured, x = buffers(), values.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured, x)
    x.copy_(values.flip(0) * 2)
    graph.replay()
    other = buffers()
    step(other, x)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(other[:7], captured[:7]))


def test_widest_rows():
    rows, cols = 3, 1 << 20
    values, gamma, beta, g = make(rows, cols, 12)
    y, mean, rstd = torch.empty_like(values), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    cfg = mgt.LayerNormConfig(rows, cols)
    assert mgt.launch_layer_norm(cfg, values, gamma, beta, y, mean, rstd) == 0
    check_forward(values, "f32", y, mean, rstd, gamma, beta)
    dy = torch.randn(rows, cols, device=DEV, generator=g)
    dx, sums = torch.empty_like(values), [torch.empty(cols, device=DEV) for _ in range(3)]
    floats = mgt.layer_norm_backward_workspace_floats(cfg)
    ws = torch.full((floats + 64,), MARK, device=DEV)
    assert mgt.launch_layer_norm_backward(cfg, dy, values, gamma, mean, rstd, dx, *sums, ws, floats) == 0
    check_backward(dy, values, gamma, mean, rstd, dx, "f32", sums)
    assert (ws[floats:] == MARK).all()


def test_workspace_that_begins_off_16_bytes():
    rows, cols = 900, 222
    values, gamma, _, g = make(rows, cols, 13)
    dy = torch.randn(rows, cols, device=DEV, generator=g)
    _, m, r, *_ = exact_forward(values, None, None)
    cfg = mgt.LayerNormConfig(rows, cols)
    floats = mgt.layer_norm_backward_workspace_floats(cfg)
    ws = torch.full((floats + 66,), MARK, device=DEV)
    dx, sums = torch.empty_like(values), [torch.empty(cols, device=DEV) for _ in range(3)]
    assert mgt.launch_layer_norm_backward(cfg, dy, values, gamma, m.float(), r.float(), dx, *sums, ws[2:], floats) == 0
    check_backward(dy, values, gamma, m.float(), r.float(), dx, "f32", sums)
    assert (ws[floats + 2:] == MARK).all() and (ws[:2] == MARK).all()


def test_rows_beyond_32_bit_offsets():
    rows, cols, pitch = 18, 300, 1 << 27  # the last row begins at element 17 * 2^27 > 2^31
    free, _ = torch.cuda.mem_get_info()
    if free < 8 << 30:
        pytest.skip("needs 5 GB")
    x = torch.empty(rows * pitch, device=DEV, dtype=torch.float16)
    view = x.view(rows, pitch)[:, :cols]
    values, gamma, beta, g = make(rows, cols, 8)
    view.copy_(values)
    kept = view.clone()
    cfg = mgt.LayerNormConfig(rows, cols, EPS, mgt.F16, mgt.F16, x_pitch=pitch, y_pitch=pitch, dx_pitch=pitch)
    mean, rstd = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    assert mgt.launch_layer_norm(cfg, x, gamma, beta, x, mean, rstd) == 0
    check_forward(kept, "f16", view, mean, rstd, gamma, beta)
    dense = mgt.LayerNormConfig(rows, cols, EPS, mgt.F16, mgt.F16, x_pitch=cols, y_pitch=pitch, dx_pitch=pitch)
    view.copy_(torch.randn(rows, cols, device=DEV, generator=g))
    dy = view.clone()
    floats = mgt.layer_norm_backward_workspace_floats(dense)
    sums = [torch.empty(cols, device=DEV) for _ in range(3)]
    assert mgt.launch_layer_norm_backward(dense, x, kept, gamma, mean, rstd, x, *sums, torch.empty(floats, device=DEV), floats) == 0
    check_backward(dy, kept, gamma, mean, rstd, view, "f16", sums)


def test_tensors_that_do_not_fit_are_refused():
    x = torch.zeros(10, 40, device=DEV)
    cfg = mgt.LayerNormConfig(10, 40)
    run = lambda c=cfg, **bad: mgt.launch_layer_norm(c, *[bad.get(k, v) for k, v in (("x", x), ("gamma", None), ("beta", None), ("y", torch.zeros_like(x)), ("mean", None), ("rstd", None))])  # noqa: E731
    assert run() == 0
    assert run(x=x.half()) == 1 and run(y=x[:9]) == 1 and run(x=x.cpu()) == 1 and run(gamma=torch.ones(39, device=DEV)) == 1 and run(beta=torch.ones(40, device=DEV).half()) == 1
    assert run(mean=torch.zeros(9, device=DEV)) == 1 and run(x=x[:, :20].expand(10, 20)) == 0  # (a view of the same rows: enough lies behind it)
    assert run(x=torch.zeros(1, 1, device=DEV).expand(10, 40)) == 1
    assert run(mgt.LayerNormConfig(10, 40, x_pitch=41)) == 1
    assert run(mgt.LayerNormConfig(10, 40, x_type=3)) == 1 and run(mgt.LayerNormConfig(10, 40, y_type=-1)) == 1


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 376), (70, 77), (301, 224), (40, 512), (33, 600), (9, 2049), (1346, 5304), (5, 12000), (3, 20000), (2, 20001)])
def test_means_far_below_the_spread_have_the_sums_precision(kind, rows, cols):
    """Values of 1/32 up to 127/32: with up to 20001 of them every partial sum is a multiple of 1/32 below 2^24 / 32, so fp32 adds them up
    exactly in any order, and the mean is off by the roundings of 1 / cols and of the product: 2 u, and their product."""
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    x = (torch.randint(-127, 128, (rows, cols), device=DEV, generator=g) / 32.0).to(TYPES[kind][1])
    mean = torch.empty(rows, device=DEV)
    assert mgt.launch_layer_norm(mgt.LayerNormConfig(rows, cols, EPS, TYPES[kind][0], TYPES[kind][0]), x, None, None, torch.empty_like(x), mean, None) == 0
    want, var = x.double().mean(1), x.double().var(1, correction=0)
    assert (want.square() < 0.5 * var).all()
    assert ((mean.double() - want).abs() <= 2.001 * U * want.abs()).all()


# rows whose threads hold three packs: of eight columns (1 to 512 lanes a row), of four (8 to 512 lanes); enough rows not to be spread further
THREE_PACKS = [(75800, 24), (20001, 88), (9500, 160), (9500, 96), (4801, 304), (4740, 384), (600, 768), (299, 1280), (151, 2056), (150, 2560), (9, 6000), (7, 12000)]


@pytest.mark.parametrize("x_kind,y_kind", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f32"), ("f32", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,cols", THREE_PACKS)
def test_forward_with_three_packs(rows, cols, x_kind, y_kind):
    test_forward(rows, cols, x_kind, y_kind)


@pytest.mark.parametrize("dy_kind,x_kind,dx_kind", [("f16", "f16", "f16"), ("bf16", "bf16", "bf16"), ("f32", "f32", "f32"), ("f32", "f32", "bf16"), ("f16", "f32", "f32")])
@pytest.mark.parametrize("rows,cols", THREE_PACKS)
def test_backward_with_three_packs(rows, cols, dy_kind, x_kind, dx_kind):
    test_backward(rows, cols, dy_kind, x_kind, dx_kind)


# single columns, 9 to 16 a thread, in CTAs of 256, 512 and 1024 threads (or two of 512), at the ends of what each layout holds
SINGLE = [(150, 2049), (150, 2559), (9, 4097), (9, 6143), (9, 6145), (9, 8191), (7, 8193), (7, 12287), (7, 12289), (7, 16383), (5000, 289), (5000, 319)]


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,cols", SINGLE)
def test_single_columns_of_wide_rows(rows, cols, kind):
    test_forward(rows, cols, kind, kind)
    test_backward(rows, cols, kind, kind, kind)
