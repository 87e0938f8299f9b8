"""The norms around a residual block, forward and backward, on the GPU against the float64 oracle; the operators of a
block in a row, on streams and in captured graphs."""
import numpy as np
import pytest
import torch

from oracle import block_oracle as O
from tests import block_cases as B

pytestmark = pytest.mark.gpu

SCALE, EPS = 0.875, 1e-6


@pytest.fixture(scope="module")
def H(pkg):
    from ascend_mlir_amd import hip_kernels
    hip_kernels.load()
    assert torch.cuda.is_available(), "no GPU visible"
    return hip_kernels


def inputs(m, n, rows_per_gate, kind, seed):
    rng = np.random.default_rng(seed)
    gates = -(-m // rows_per_gate) if rows_per_gate else 0
    t = lambda a: B.tensor(a, kind, "cuda")
    return dict(x=t(rng.normal(size=(m, n)) * 3), f=t(rng.normal(size=(m, n)) * 2), dy=t(rng.normal(size=(m, n)) * 0.5),
                dh=t(rng.normal(size=(m, n)) * 0.5), post_weight=t(1 + 0.2 * rng.normal(size=n)),
                pre_weight=t(1 + 0.2 * rng.normal(size=n)),
                gate=t(rng.uniform(0.1, 0.9, size=(gates, n))) if gates else None)


def reference(v):
    return {k: None if t is None else B.numbers(t) for k, t in v.items()}


def check_forward(v, got, kind, rows_per_gate, f=True, pre=True):
    r = reference(v)
    m, n = r["x"].shape
    args = (r["x"], r["f"] if f else None, r["post_weight"], r["gate"], r["pre_weight"] if pre else None, SCALE, EPS,
            rows_per_gate or m)
    y, h = O.norm(*args)
    s = B.row_sum_steps(n)
    g = np.abs(O.gate_of_rows(r["gate"], m, rows_per_gate or m))
    size = np.abs(SCALE * r["x"]) + g * np.abs(r["f"] * O.rstd(r["f"], EPS) * r["post_weight"])
    if f:
        # the branch carries half the relative error of its row sum (the root) and five roundings of its own
        B.close(got[0], y, size, kind, s / 2 + 8)
    if pre:
        if not f:
            size = np.abs(y)
        # h carries y's errors through y itself and, at most as strongly, through the row's rstd
        ry, w = O.rstd(y, EPS), np.abs(r["pre_weight"])
        through = (size + np.abs(y) * ry ** 2 * (np.abs(y) * size).mean(axis=1, keepdims=True)) * ry * w
        B.close(got[1], h, through, kind, s + 12)


def check_backward(v, y, got, kind, rows_per_gate, dy=True, dh=True, f=True):
    r = reference(v)
    y = B.numbers(y)
    m, n = y.shape
    want, size = O.norm_grad(r["dy"] if dy else None, r["dh"] if dh else None, y, r["f"] if f else None, r["post_weight"],
                             r["gate"], r["pre_weight"], SCALE, EPS, rows_per_gate or m)
    got = dict(zip(("dx", "df", "dpost_weight", "dgate", "dpre_weight"), got))
    assert {k for k, t in got.items() if t is not None} == set(want)
    # a chain of two rounds of row sums and about twenty operations of its own; columns add m terms on top
    s = 3 * B.row_sum_steps(n) + 24
    for name, w in want.items():
        B.close(got[name], w, size[name], kind, s if name in ("dx", "df") else s + m)


def forward(H, v, rows_per_gate, **kw):
    return H.norm_gate_residual(v["x"], v["f"], v["post_weight"], v["gate"], v["pre_weight"], residual_scale=SCALE, eps=EPS,
                                rows_per_gate=rows_per_gate or None, **kw)


def backward(H, v, y, rows_per_gate, **kw):
    return H.norm_gate_residual_backward(v["dy"], v["dh"], y, v["f"], v["post_weight"], v["gate"], v["pre_weight"],
                                         residual_scale=SCALE, eps=EPS, rows_per_gate=rows_per_gate or None, **kw)


@pytest.mark.parametrize("kind", B.TYPES)
@pytest.mark.parametrize("m,n,rows_per_gate", [
    (1, 1, 1), (1, 7, 0), (2, 8, 1), (3, 9, 2), (5, 64, 5), (33, 255, 4), (7, 513, 3), (9, 1000, 1), (4, 1024, 0),
    (6, 2048, 6), (5, 2052, 2), (3, 4096, 1), (11, 5000, 4), (2, 8192, 2), (3, 8200, 1), (2, 16384, 0), (3, 16381, 2),
    (700, 72, 1), (2500, 40, 7), (2111, 136, 500), (600, 1030, 600), (1030, 520, 0)])
def test_forward_and_backward(H, kind, m, n, rows_per_gate):
    v = inputs(m, n, rows_per_gate, kind, 100 * m + n)
    got = forward(H, v, rows_per_gate)
    check_forward(v, got, kind, rows_per_gate)
    check_backward(v, got[0], backward(H, v, got[0], rows_per_gate), kind, rows_per_gate)


@pytest.mark.parametrize("kind,m,n,rows_per_gate", [
    # rows of one, two and four wavefronts, whose workgroups walk several stretches; gates shorter than a stretch, a
    # little longer, split over stretches with some left idle, and one for all
    ("bf16", 8192, 40, 3), ("f32", 8200, 72, 10), ("f16", 8191, 256, 20), ("bf16", 4097, 513, 2), ("f32", 5000, 260, 1),
    ("f16", 4100, 900, 9), ("bf16", 6001, 600, 700), ("f32", 3000, 1000, 11), ("f16", 2600, 2048, 3), ("bf16", 2100, 1100, 7),
    ("f32", 2049, 600, 2049), ("bf16", 8192, 64, 0), ("f16", 4099, 33, 4099)])
def test_gradients_of_many_short_rows(H, kind, m, n, rows_per_gate):
    v = inputs(m, n, rows_per_gate, kind, m + n)
    y, _ = forward(H, v, rows_per_gate)
    got = backward(H, v, y, rows_per_gate)
    check_backward(v, y, got, kind, rows_per_gate)
    for a, b in zip(backward(H, v, y, rows_per_gate, block_dim=3), got):
        assert (a is None and b is None) or torch.equal(a, b)


@pytest.mark.parametrize("m,n,rows_per_gate", [(37, 300, 5), (300, 2048, 1), (515, 96, 129)])
def test_parts_left_out(H, m, n, rows_per_gate):
    kind = "bf16"
    v = inputs(m, n, rows_per_gate, kind, 5)
    # no second norm
    y, h = H.norm_gate_residual(v["x"], v["f"], v["post_weight"], v["gate"], residual_scale=SCALE, eps=EPS,
                                rows_per_gate=rows_per_gate)
    assert h is None
    check_forward(v, (y, None), kind, rows_per_gate, pre=False)
    got = H.norm_gate_residual_backward(v["dy"], None, y, v["f"], v["post_weight"], v["gate"], residual_scale=SCALE, eps=EPS,
                                        rows_per_gate=rows_per_gate)
    check_backward(v, y, got, kind, rows_per_gate, dh=False)
    # the norm ahead of the first block
    same, h = H.norm_gate_residual(v["x"], pre_weight=v["pre_weight"], eps=EPS)
    assert same is v["x"]
    nogate = dict(v, gate=None)
    check_forward(nogate, (None, h), kind, 0, f=False)
    got = H.norm_gate_residual_backward(v["dy"], v["dh"], v["x"], pre_weight=v["pre_weight"], residual_scale=SCALE, eps=EPS)
    check_backward(nogate, v["x"], got, kind, 0, f=False)
    # no gradient into y but h's
    y, h = forward(H, v, rows_per_gate)
    check_backward(v, y, backward(H, dict(v, dy=None), y, rows_per_gate), kind, rows_per_gate, dy=False)


def test_rows_of_zeros_and_of_large_numbers(H):
    for kind in B.TYPES:
        v = inputs(6, 260, 1, kind, 8)
        v["x"][1] = 0
        v["f"][1] = 0
        v["f"][2] = 0
        v["f"][3] *= 1000
        v["x"][4] *= 100
        got = forward(H, v, 1)
        assert not got[0][1].any() and not got[1][1].any()
        check_forward(v, got, kind, 1)
        check_backward(v, got[0], backward(H, v, got[0], 1), kind, 1)


def test_a_nan_stays_in_its_row(H):
    v = inputs(9, 300, 3, "bf16", 9)
    v["f"][4, 7] = float("nan")
    y, h = forward(H, v, 3)
    rows = torch.arange(9, device="cuda") == 4
    assert torch.equal(torch.isnan(y).any(1), rows) and torch.equal(torch.isnan(h).any(1), rows)
    dx, df, *_ = backward(H, inputs(9, 300, 3, "bf16", 9) | {"f": v["f"]}, forward(H, inputs(9, 300, 3, "bf16", 9), 3)[0], 3)
    assert not torch.isnan(dx).any() and torch.equal(torch.isnan(df).any(1), rows)


@pytest.mark.parametrize("kind", B.TYPES)
def test_rows_with_strides_and_off_alignment(H, kind):
    m, n, per = 21, 301, 4
    v = inputs(m, n, per, kind, 11)
    wide = {}
    for i, name in enumerate(("x", "f", "dy", "dh", "gate")):
        rows = v[name].shape[0]
        big = torch.full((rows, n + 5 + 2 * i), 55.0, dtype=B.TYPES[kind], device="cuda")
        wide[name] = big[:, 1 + i:1 + i + n]
        wide[name].copy_(v[name])
    dense = forward(H, v, per)
    y = torch.full((m, n + 9), 77.0, dtype=B.TYPES[kind], device="cuda")
    h = torch.full((m, n + 3), 77.0, dtype=B.TYPES[kind], device="cuda")
    s = dict(v, **wide)
    got = forward(H, s, per, y=y[:, 3:3 + n], h=h[:, 1:1 + n])
    assert torch.equal(got[0], dense[0]) and torch.equal(got[1], dense[1])
    assert (y[:, :3] == 77).all() and (y[:, 3 + n:] == 77).all() and (h[:, 0] == 77).all() and (h[:, 1 + n:] == 77).all()
    want = backward(H, v, dense[0], per)
    for a, b in zip(backward(H, s, got[0], per), want):
        assert torch.equal(a, b)


def test_in_place(H):
    for n in (200, 4096, 9000):
        v = inputs(50, n, 7, "bf16", 12)
        y, h = forward(H, v, 7)
        x, f = v["x"].clone(), v["f"].clone()
        got = forward(H, dict(v, x=x, f=f), 7, y=x, h=f)
        assert got[0] is x and got[1] is f and torch.equal(x, y) and torch.equal(f, h)


def test_few_workgroups_and_repeated_calls_give_the_same(H):
    for m, n, per in ((300, 520, 1), (300, 4100, 50), (3000, 64, 0)):
        v = inputs(m, n, per, "f16", 13)
        y, h = forward(H, v, per)
        a = forward(H, v, per, block_dim=3)
        assert torch.equal(a[0], y) and torch.equal(a[1], h)
        want = backward(H, v, y, per)
        for other in (backward(H, v, y, per, block_dim=5), backward(H, v, y, per)):
            for p, q in zip(other, want):
                assert (p is None and q is None) or torch.equal(p, q)


def test_gradients_against_differences(H):
    """The kernels alone: differences of the forward kernel's results against the backward kernel's, in float32."""
    m, n, per = 6, 48, 4
    v = inputs(m, n, per, "f32", 14)
    y, _ = forward(H, v, per)
    grads = dict(zip(("x", "f", "post_weight", "gate", "pre_weight"), backward(H, v, y, per)))

    def loss(u):
        y, h = forward(H, u, per)
        return float((y.double() * v["dy"].double()).sum() + (h.double() * v["dh"].double()).sum())

    gen = torch.Generator(device="cuda").manual_seed(1)
    for name, g in grads.items():
        direction = torch.randn(g.shape, generator=gen, device="cuda")
        step = 2.0 ** -7
        slope = (loss(dict(v, **{name: v[name] + step * direction})) - loss(dict(v, **{name: v[name] - step * direction}))) / (2 * step)
        want = float((g.double() * direction.double()).sum())
        # 2 m n results of size 3 with a rounding each, added at random: sqrt(576) * 3 * 2^-24 / step = 6e-4; the third
        # derivative's term, step^2 / 6 times the slopes' own size (at most a few times |g|): 1e-5 * |g|
        assert abs(slope - want) < 2e-3 + 1e-3 * float(g.double().abs().sum()) ** 0.5, name


def test_gate_of_one_dimension(H):
    v = inputs(12, 96, 12, "bf16", 15)
    y, h = forward(H, v, 12)
    one = dict(v, gate=v["gate"][0])
    got = forward(H, one, 0)
    assert torch.equal(got[0], y) and torch.equal(got[1], h)
    grads = backward(H, one, y, 0)
    assert grads[3].shape == (96,) and torch.equal(grads[3], backward(H, v, y, 12)[3][0])


def test_two_results_in_one_tensor_are_refused(H):
    v = inputs(4, 64, 1, "f32", 20)
    t = torch.empty(4, 64, device="cuda")
    with pytest.raises(H.AfirHipError, match="two results"):
        H.norm_gate_residual(v["x"], v["f"], v["post_weight"], v["gate"], v["pre_weight"], y=t, h=t)


def test_two_results_in_one_buffer(H):
    """Views that share numbers are refused, whatever objects they are; views side by side are not."""
    m, n = 5, 96
    v = inputs(m, n, 1, "bf16", 21)
    y, h = forward(H, v, 1)
    t = torch.full((m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    wide = torch.full((m + 1, 3 * n), 7.0, dtype=torch.bfloat16, device="cuda")
    for a, b in ((t, t.view(m, n)), (t.view(m, n), t), (wide[:m, :n], wide[:m, n - 1:2 * n - 1]),
                 (wide[1:, :n], wide.as_strided((m, n), (3 * n, 1), 2 * n + 1)),
                 (wide[:m, :n], wide[1:, :n])):
        with pytest.raises(H.AfirHipError, match="must not overlap"):
            forward(H, v, 1, y=a, h=b)
    assert (t == 7).all() and (wide == 7).all()
    stacked = torch.empty((2 * m, n), dtype=torch.bfloat16, device="cuda")
    for a, b in ((wide[:m, :n], wide[:m, n:2 * n]), (wide[1:, n:2 * n], wide[1:, :n]), (wide[:m, 2 * n:], wide[1:, :n]),
                 (wide[1:, :n], wide[:m, n:2 * n]), (stacked[:m], stacked[m:]), (stacked[m:], stacked[:m])):
        forward(H, v, 1, y=a, h=b)
        assert torch.equal(a, y) and torch.equal(b, h)


def test_refusals(H):
    v = inputs(8, 64, 2, "bf16", 16)
    x, f, w, gate = v["x"], v["f"], v["post_weight"], v["gate"]
    N = H.norm_gate_residual
    for args, kw, word in (((x[0],), dict(pre_weight=w), "two dimensions"), ((x.int(),), dict(pre_weight=w), "float32"),
                           ((x,), {}, "without f"), ((x, None, w), dict(pre_weight=w), "without f"),
                           ((x, f.half(), w), {}, "bfloat16"), ((x, f[:4], w), {}, "shape"), ((x, f, w[:3]), {}, "shape"),
                           ((x, f, w, gate), {}, "do not cover"), ((x, f, w, gate), dict(rows_per_gate=3), "do not cover"),
                           ((x, f, w, gate), dict(rows_per_gate=0), "do not cover"),
                           ((x, f, w, gate.float()), dict(rows_per_gate=2), "bfloat16"),
                           ((x, f, w), dict(y=x.t().contiguous().t()), "adjacent"),
                           ((x, f, w), dict(h=torch.empty_like(x)), "pre_weight"),
                           ((x, f, w), dict(eps=-1.0), "eps"), ((x, f, w), dict(eps=float("nan")), "eps"),
                           ((x, f, w, None, w.cpu()), {}, "device tensor"),
                           ((x, f, w), dict(y=x[:1].expand(8, 64)), "overlap")):
        with pytest.raises(H.AfirHipError, match=word):
            N(*args, **kw)
    G = H.norm_gate_residual_backward
    for args, kw, word in (((x, x, x, f, w), {}, "together"), ((None, None, x, f, w), {}, "dy or dh"),
                           ((x, None, x), {}, "f or dh"), ((x, x, x, None, w, None, w), {}, "need f"),
                           ((x, x[:4], x, f, w, None, w), {}, "shape"), ((x[:0], x[:0], x[:0], None, None, None, w), {}, "empty")):
        with pytest.raises(H.AfirHipError, match=word):
            G(*args, **kw)
    long = torch.zeros((2, 16385), device="cuda")
    with pytest.raises(H.AfirHipError, match="16384"):
        N(long, pre_weight=long[0])


# ---- the operators of a block in a row ----

def block_weights(n, hidden, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
    return dict(pre=(1 + 0.1 * r(n)).bfloat16(), post=(1 + 0.1 * r(n)).bfloat16(), nxt=(1 + 0.1 * r(n)).bfloat16(),
                up=(r(n, hidden) / n ** 0.5).bfloat16(), down=(r(hidden, n) / hidden ** 0.5).bfloat16(),
                up_bias=(0.1 * r(hidden)).bfloat16(), gate=torch.sigmoid(r(1, n)).bfloat16())


def run_block(H, w, x, q=None):
    """x -> (y, h): norm, up product with leaky relu, down product, norm with gate and residual, the next norm."""
    up, down = q if q else (H.mxfp4_quantize(w["up"], axis=0), H.mxfp4_quantize(w["down"], axis=0))
    _, h = H.norm_gate_residual(x, pre_weight=w["pre"])
    mid = H.mxfp4_matmul_add_leakyrelu(*H.mxfp4_quantize(h), *up, w["up_bias"], alpha=0.1)
    f = H.mxfp4_matmul_add_leakyrelu(*H.mxfp4_quantize(mid), *down, alpha=1.0)
    y, h = H.norm_gate_residual(x, f, w["post"], w["gate"], w["nxt"], residual_scale=SCALE)
    return h, mid, f, y


@pytest.mark.parametrize("m", [1, 37, 300])
def test_a_block_in_a_row(H, m):
    n, hidden = 264, 520
    w = block_weights(n, hidden, 1)
    x = torch.randn(m, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).bfloat16()
    h2, mid, f, y = run_block(H, w, x)
    # each step against the oracle at the tensors that the step before gave
    h = H.norm_gate_residual(x, pre_weight=w["pre"])[1]
    num = B.numbers
    for a, weight, bias, alpha, got in ((h, "up", "up_bias", 0.1, mid), (mid, "down", None, 1.0, f)):
        qa, qb = O.quantize(num(a))[2], O.quantize(num(w[weight]).T)[2]
        want, size = O.matmul(qa, qb, num(w[bias]) if bias else None, alpha)
        B.close(got, want, size, "bf16", qa.shape[1] / 32 + 11)
    want, _ = O.norm(num(x), num(f), num(w["post"]), num(w["gate"]), num(w["nxt"]), SCALE, EPS, m)
    assert np.abs(num(y) - want).max() < 2 ** -7 * np.abs(want).max()


def test_a_block_replayed_from_a_captured_graph(H):
    w = block_weights(256, 512, 3)
    q = H.mxfp4_quantize(w["up"], axis=0), H.mxfp4_quantize(w["down"], axis=0)
    x = torch.randn(70, 256, device="cuda").bfloat16()
    dy, dh = torch.randn(2, 70, 256, device="cuda").bfloat16().unbind(0)

    def step():
        h, mid, f, y = run_block(H, w, x, q)
        grads = H.norm_gate_residual_backward(dy, dh, y, f, w["post"], w["gate"], w["nxt"], residual_scale=SCALE)
        return h, y, *grads

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for replay in range(4):
        x.copy_(torch.randn(70, 256, device="cuda").bfloat16())
        dy.mul_(1.5)
        want = [t.clone() for t in step()]
        for t in captured:
            t.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, expected in zip(captured, want):
            assert torch.equal(got, expected), replay


def test_two_streams_at_once(H):
    """Calls on two streams overlap; each has its own results and workspaces."""
    w = block_weights(520, 1032, 4)
    q = H.mxfp4_quantize(w["up"], axis=0), H.mxfp4_quantize(w["down"], axis=0)
    xs = [torch.randn(400, 520, device="cuda").bfloat16() for _ in range(2)]

    def step(x):
        h, mid, f, y = run_block(H, w, x, q)
        return (h, y, *H.norm_gate_residual_backward(x, h, y, f, w["post"], w["gate"], w["nxt"], residual_scale=SCALE))

    want = [[t.clone() for t in step(x)] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    results = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                results[i].append(step(xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for got in results[i]:
            assert all(torch.equal(a, b) for a, b in zip(got, want[i]))


def test_a_given_stream(H):
    v = inputs(300, 512, 1, "bf16", 17)
    y, h = forward(H, v, 1)
    want = backward(H, v, y, 1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = backward(H, v, y, 1, stream=s.cuda_stream)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_default_stream_given_by_its_handle(H, monkeypatch):
    """stream=0 is the default stream, as for every other launcher, from whatever stream the call is made."""
    assert torch.cuda.default_stream().cuda_stream == 0
    v = inputs(40, 96, 1, "bf16", 18)
    y, h = forward(H, v, 1)
    grads = backward(H, v, y, 1)
    q = H.mxfp4_quantize(v["x"])
    out = H.mxfp4_matmul_add_leakyrelu(*q, *q)
    torch.cuda.synchronize()
    used, launch = [], H._launch_on

    def recorded(index, *rest):
        used.append(torch.cuda.current_stream(index).cuda_stream)
        return launch(index, *rest)

    monkeypatch.setattr(H, "_launch_on", recorded)
    for place in (torch.cuda.default_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(place):
            got = (*forward(H, v, 1, stream=0), *backward(H, v, y, 1, stream=0), *H.mxfp4_quantize(v["x"], stream=0),
                   H.mxfp4_matmul_add_leakyrelu(*q, *q, stream=0))
            assert torch.cuda.current_stream() == place
        torch.cuda.synchronize()
        for a, b in zip(got, (y, h, *grads, *q, out)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert used == [0] * 8


def signs(rng, shape):
    return rng.integers(0, 2, shape) * 2.0 - 1


def terms(rng, m, n):
    """m rows of +-1 whose column sums stay small: half of the rows undo the other half, but for sixty at the end."""
    c = signs(rng, (m, n))
    half = (m - 60) // 2
    if half > 0:
        c[half:2 * half] = -c[rng.permutation(half)]
    return c


@pytest.mark.parametrize("kind,m,n,rows_per_gate", [
    ("bf16", 8192, 64, 3), ("f32", 8200, 64, 10), ("f16", 8191, 256, 20), ("bf16", 4097, 512, 2), ("f32", 5000, 256, 1),
    ("f16", 4100, 1024, 9), ("bf16", 6001, 1024, 700), ("f32", 3000, 1024, 11), ("f16", 2600, 2048, 3), ("bf16", 2100, 2048, 7),
    ("f32", 2049, 512, 2049), ("bf16", 8192, 64, 0), ("bf16", 1500, 4096, 0), ("f16", 1100, 8192, 300), ("bf16", 700, 16384, 0),
    ("f32", 600, 8192, 5), ("f32", 520, 16384, 100), ("bf16", 513, 4096, 17), ("f16", 40, 2048, 0), ("f32", 3, 64, 2)])
def test_column_sums_miss_no_row_and_take_none_twice(H, kind, m, n, rows_per_gate):
    """Rows of +-1 have the norm 1, so with weights and gates of 1 every term of a column sum is +-1: the sums are whole
    numbers that each of the types holds, compared without a tolerance."""
    rng = np.random.default_rng(m + n)
    per = rows_per_gate or m
    t = lambda a: B.tensor(a, kind, "cuda")
    f, y, c, d = signs(rng, (m, n)), signs(rng, (m, n)), terms(rng, m, n), terms(rng, m, n)
    one, starts = t(np.ones(n)), np.arange(0, m, per)
    gate = t(np.ones((len(starts), n))) if rows_per_gate else None
    sums, dgate = c.sum(axis=0), np.add.reduceat(c, starts, axis=0)
    assert np.abs(sums).max() <= 256 and np.abs(dgate).max() <= 256
    got = H.norm_gate_residual_backward(t(c * f), None, t(y), t(f), one, gate, eps=0.0, rows_per_gate=rows_per_gate or None)
    assert np.array_equal(B.numbers(got[2]), sums)
    if gate is not None:
        assert np.array_equal(B.numbers(got[3]), dgate)
    got = H.norm_gate_residual_backward(t(c * f), t(d * y), t(y), t(f), one, gate, one, eps=0.0,
                                        rows_per_gate=rows_per_gate or None)
    assert np.array_equal(B.numbers(got[4]), d.sum(axis=0))
    got = H.norm_gate_residual_backward(None, t(d * y), t(y), pre_weight=one, eps=0.0)
    assert np.array_equal(B.numbers(got[4]), d.sum(axis=0))


GRAD = "afir_hip_launch_norm_gate_residual_backward"


def launch_backward(H, v, y, kind, rows_per_gate, dx, df, dy, f):
    """The C launcher: results in given places, whose rows have the strides that they have."""
    m, n = y.shape
    gate = v["gate"]
    dpost, dpre = torch.empty_like(v["post_weight"]), torch.empty_like(v["pre_weight"])
    dgate = None if gate is None else torch.empty_like(gate)
    tiling = H.pack_tiling(m, n, rows_per_gate or m, dy.stride(0), n, n, f.stride(0), n, dx.stride(0), df.stride(0),
                           H.f32_bits(SCALE), H.f32_bits(EPS), list(B.TYPES).index(kind))
    size = H.load().afir_hip_norm_gate_residual_backward_workspace_bytes(tiling)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    ptrs = [0 if t is None else t.data_ptr() for t in (dy, v["dh"], y, f, v["post_weight"], gate, v["pre_weight"], dx, df,
                                                       dpost, dgate, dpre, workspace)]
    assert H.launch_raw(GRAD, 0, None, ptrs, tiling) == 0
    torch.cuda.synchronize()
    return dx, df, dpost, dgate, dpre


@pytest.mark.parametrize("kind,m,n,rows_per_gate", [
    # rows of 1 to 16 wavefronts and of 1, 2 and 4 pieces per lane; gates within a stretch, over several, and none
    ("bf16", 900, 200, 1), ("f32", 1500, 200, 700), ("f16", 2500, 600, 7), ("bf16", 1200, 2000, 0), ("f32", 700, 2048, 3),
    ("f16", 600, 5000, 600), ("bf16", 1030, 9000, 40), ("f32", 530, 16000, 1), ("f16", 50, 16384, 7), ("bf16", 1, 300, 1)])
def test_gradients_in_place_and_with_strides(H, kind, m, n, rows_per_gate):
    v = inputs(m, n, rows_per_gate, kind, 22)
    y, _ = forward(H, v, rows_per_gate)
    want = backward(H, v, y, rows_per_gate)

    def same(got):
        for a, b in zip(got, want):
            assert (a is None and b is None) or torch.equal(a, b)

    # dx in dy's place, df in f's
    dy, f = v["dy"].clone(), v["f"].clone()
    same(launch_backward(H, v, y, kind, rows_per_gate, dy, f, dy, f))

    def wide(t, left, right):
        big = torch.full((m, left + n + right), 77.0, dtype=t.dtype, device="cuda")
        big[:, left:left + n] = t
        return big, big[:, left:left + n]

    def untouched(big, left):
        return (big[:, :left] == 77).all() and (big[:, left + n:] == 77).all()

    # rows with strides of their own, off every boundary but an element's
    (big_dx, dx), (big_df, df) = wide(torch.zeros_like(y), 3, 6), wide(torch.zeros_like(y), 1, 4)
    same(launch_backward(H, v, y, kind, rows_per_gate, dx, df, v["dy"], v["f"]))
    assert untouched(big_dx, 3) and untouched(big_df, 1)
    # ... and in place with them
    (big_dy, dy), (big_f, f) = wide(v["dy"], 3, 6), wide(v["f"], 1, 4)
    same(launch_backward(H, v, y, kind, rows_per_gate, dy, f, dy, f))
    assert untouched(big_dy, 3) and untouched(big_f, 1)


def test_beyond_32_bit_offsets(H):
    m, n, per, kind = 133000, 16384, 1000, "bf16"      # 2^31 numbers are 131072 rows
    r = lambda rows, spread: torch.randn(rows, n, device="cuda", dtype=torch.bfloat16) * spread
    v = dict(x=r(m, 3), f=r(m, 2), dy=r(m, 0.5), dh=r(m, 0.5), post_weight=r(1, 1)[0], pre_weight=r(1, 1)[0],
             gate=torch.sigmoid(r(m // per, 1)))
    got = forward(H, v, per)
    grads = backward(H, v, got[0], per)
    for first, last in ((0, 20), (131000, 131100), (132980, 133000)):
        part = {k: t if t.dim() == 1 else t[first:last] for k, t in v.items()}
        part["gate"] = v["gate"][first // per:first // per + 1]
        check_forward(part, [t[first:last] for t in got], kind, per)
        ref, y = reference(part), B.numbers(got[0][first:last])
        want, size = O.norm_grad(ref["dy"], ref["dh"], y, ref["f"], ref["post_weight"], ref["gate"], ref["pre_weight"], SCALE,
                                 EPS, per)
        for name, g in zip(("dx", "df"), grads):
            B.close(g[first:last], want[name], size[name], kind, 3 * B.row_sum_steps(n) + 24)
