"""The oracle of the block operators against definitions worked out by hand, and its gradients against differences;
the operators' refusals, which need no GPU."""
import ctypes

import numpy as np
import pytest

from oracle import block_oracle as O


def test_every_code_and_tie_of_the_format():
    # a block whose largest number is 6 (scale 1): grid points, ties to the even code, saturation above 6
    x = np.zeros((1, 32))
    x[0, :16] = [0, .25, .26, .5, .75, .74, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5]
    x[0, 16:24] = [5.01, 6, 7.9, -0.25, -0.75, -1.25, -5, -7]
    _, scales, values = O.quantize(x)
    assert scales.tolist() == [[127]]
    assert values[0, :16].tolist() == [0, 0, .5, .5, 1, .5, 1, 1, 1.5, 2, 2, 2, 3, 4, 4, 4]
    assert values[0, 16:24].tolist() == [6, 6, 6, -0.0, -1, -1, -4, -6]


@pytest.mark.parametrize("top,byte", [(1.0, 125), (1.999, 125), (2.0, 126), (4.0, 127), (7.99, 127), (8.0, 128),
                                      (2.0 ** -126, 0), (2.0 ** -125, 0), (2.0 ** -124, 1), (2.0 ** 127, 252), (0.0, 0),
                                      (2.0 ** -149, 0), (np.inf, 255), (np.nan, 255)])
def test_scale_of_a_block(top, byte):
    x = np.zeros((1, 40))
    x[0, 3] = top
    x[0, 33] = 1.0
    codes, scales, values = O.quantize(x)
    assert scales.tolist() == [[byte, 125]]
    assert values[0, 33] == 1.0 and values.shape == (1, 40) and codes.shape == (1, 32)
    assert np.isnan(values[0, :32]).all() == (byte == 255)


def test_decode_reads_what_quantize_wrote():
    rng = np.random.default_rng(0)
    x = rng.normal(size=(9, 75)) * np.exp(rng.normal(size=(9, 75)) * 4)
    codes, scales, values = O.quantize(x)
    assert np.array_equal(O.decode(codes, scales)[:, :75], values)
    assert not O.decode(codes, scales)[:, 75:].any()
    # an element is off by at most a quarter of its block's largest magnitude (7.99 saturates to 6)
    top = np.abs(np.pad(x, ((0, 0), (0, 21)))).reshape(9, 3, 32).max(axis=2).repeat(32, axis=1)[:, :75]
    assert (np.abs(values - x) <= top / 4).all()


@pytest.mark.parametrize("rows_per_gate", [1, 2, 3, 5])
def test_gradients_against_differences(rows_per_gate):
    rng = np.random.default_rng(1)
    m, n, scale, eps = 5, 11, 0.7, 1e-3
    x, f, dy, dh = (rng.normal(size=(m, n)) for _ in range(4))
    post, pre = (1 + 0.3 * rng.normal(size=n) for _ in range(2))
    gate = rng.uniform(0.2, 1, size=(-(-m // rows_per_gate), n))
    inputs = {"x": x, "f": f, "post_weight": post, "gate": gate, "pre_weight": pre}

    def loss():
        y, h = O.norm(inputs["x"], inputs["f"], inputs["post_weight"], inputs["gate"], inputs["pre_weight"], scale, eps,
                      rows_per_gate)
        return (y * dy).sum() + (h * dh).sum()

    y, _ = O.norm(x, f, post, gate, pre, scale, eps, rows_per_gate)
    grads, _ = O.norm_grad(dy, dh, y, f, post, gate, pre, scale, eps, rows_per_gate)
    for name, array in inputs.items():
        got = grads["d" + name]
        for at in np.ndindex(array.shape):
            keep, step = array[at], 1e-5
            array[at] = keep + step
            up = loss()
            array[at] = keep - step
            down = loss()
            array[at] = keep
            # the third derivative's term is about step^2 = 1e-10, the cancellation 1e-16 / 1e-5
            assert abs((up - down) / (2 * step) - got[at]) < 1e-7 * (1 + abs(got[at])), (name, at)


# ---- refusals of the C ABI: all on the host, before anything is launched ----

FAKE = 1 << 20   # an aligned address that is never followed


def refusal(H, symbol, args, fields, bad_tiling=False):
    L = H.load()
    til = H.pack_tiling(*fields)
    rc = getattr(L, symbol)(0, None, *[ctypes.c_void_p(a) for a in args], None if bad_tiling else til)
    assert rc == 1, rc
    return L.afir_hip_last_error().decode()


@pytest.fixture(scope="module")
def H(pkg):
    from ascend_mlir_amd import hip_kernels
    hip_kernels.load()
    return hip_kernels


QUANT = "afir_hip_launch_mxfp4_quantize"


@pytest.mark.parametrize("args,fields,word", [
    ((0, FAKE, FAKE, 0, 0), (4, 64, 64, 1, 0), "null"),
    ((FAKE, 0, FAKE, 0, 0), (4, 64, 64, 1, 0), "null"),
    ((FAKE, FAKE, 0, 0, 0), (4, 64, 64, 1, 0), "null"),
    ((FAKE, FAKE, FAKE, 0, 0), (-4, 64, 64, 1, 0), "negative"),
    ((FAKE, FAKE, FAKE, 0, 0), (4, 64, 63, 1, 0), "stride"),
    ((FAKE, FAKE, FAKE, 0, 0), (4, 64, 1 << 62, 1, 0), "stride"),
    ((FAKE, FAKE, FAKE, 0, 0), (4, 64, 64, 2, 0), "axis"),
    ((FAKE, FAKE, FAKE, 0, 0), (4, 64, 64, 1, 3), "elem_type"),
    ((FAKE, FAKE, FAKE, 0, 0), (4, 64, 64, 1, -1), "elem_type"),
    ((FAKE, FAKE, FAKE, 0, 0), (1 << 40, 64, 64, 1, 0), "2^31"),
    ((FAKE, FAKE, FAKE, 0, 0), (4, 1 << 40, 1 << 40, 1, 0), "2^31"),
    ((FAKE + 1, FAKE, FAKE, 0, 0), (4, 64, 64, 1, 1), "alignment"),
    ((FAKE, FAKE, FAKE, FAKE + 2, 0), (4, 64, 64, 1, 0), "alignment"),
    ((FAKE, FAKE + 8, FAKE, 0, 0), (4, 64, 64, 1, 1), "16-byte"),
])
def test_quantize_refuses(H, args, fields, word):
    assert word in refusal(H, QUANT, args, fields)
    assert "null tiling" in refusal(H, QUANT, args, fields, bad_tiling=True)


MATMUL = "afir_hip_launch_mxfp4_matmul_add_leakyrelu"


@pytest.mark.parametrize("args,fields,word", [
    ((0, FAKE, FAKE, FAKE, 0, FAKE, 0), (4, 64, 8, 0, 2), "null"),
    ((FAKE, 0, FAKE, FAKE, 0, FAKE, 0), (4, 64, 8, 0, 2), "null"),
    ((FAKE, FAKE, 0, FAKE, 0, FAKE, 0), (4, 64, 8, 0, 2), "null"),
    ((FAKE, FAKE, FAKE, 0, 0, FAKE, 0), (4, 64, 8, 0, 2), "null"),
    ((FAKE, FAKE, FAKE, FAKE, 0, 0, 0), (4, 64, 8, 0, 2), "null"),
    ((FAKE, FAKE, FAKE, FAKE, 0, FAKE, 0), (4, -64, 8, 0, 2), "negative"),
    ((FAKE, FAKE, FAKE, FAKE, 0, FAKE, 0), (4, 64, 1 << 33, 0, 2), "2^31"),
    ((FAKE, FAKE, FAKE, FAKE, 0, FAKE, 0), (4, 64, 8, 0, 7), "elem_type"),
    ((FAKE + 4, FAKE, FAKE, FAKE, 0, FAKE, 0), (4, 64, 8, 0, 2), "16-byte"),
    ((FAKE, FAKE, FAKE + 4, FAKE, 0, FAKE, 0), (4, 64, 8, 0, 2), "16-byte"),
    ((FAKE, FAKE, FAKE, FAKE, FAKE + 1, FAKE, 0), (4, 64, 8, 0, 2), "alignment"),
    ((FAKE, FAKE, FAKE, FAKE, 0, FAKE + 2, 0), (4, 64, 8, 0, 0), "alignment"),
])
def test_matmul_refuses(H, args, fields, word):
    assert word in refusal(H, MATMUL, args, fields)
    assert "null tiling" in refusal(H, MATMUL, args, fields, bad_tiling=True)


NORM = "afir_hip_launch_norm_gate_residual"
ALL = dict(x=FAKE, f=FAKE, post=FAKE, gate=FAKE, pre=FAKE, y=FAKE, h=FAKE)
FIELDS = dict(m=4, n=64, rpg=2, ld_x=64, ld_f=64, ld_gate=64, ld_y=64, ld_h=64, scale=0, eps=0, type=2)


@pytest.mark.parametrize("args,fields,word", [
    (dict(x=0), {}, "null"),
    (dict(post=0), {}, "post_weight"),
    (dict(y=0), {}, "y"),
    (dict(pre=0), {}, "pre_weight"),
    (dict(f=0), {}, "without f"),
    (dict(f=0, y=0, gate=0, h=0), {}, "neither"),
    ({}, dict(m=-1), "negative"),
    ({}, dict(n=16385, ld_x=1 << 20, ld_f=1 << 20, ld_gate=1 << 20, ld_y=1 << 20, ld_h=1 << 20), "16384"),
    ({}, dict(rpg=0), "rows_per_gate"),
    ({}, dict(ld_x=63), "stride"),
    ({}, dict(ld_f=63), "stride"),
    ({}, dict(ld_gate=63), "stride"),
    ({}, dict(ld_y=0), "stride"),
    ({}, dict(ld_h=1 << 62), "stride"),
    ({}, dict(eps=0xbf800000), "eps"),
    ({}, dict(eps=0x7fc00000), "eps"),
    ({}, dict(type=3), "elem_type"),
    (dict(gate=FAKE + 1), {}, "alignment"),
])
def test_norm_refuses(H, args, fields, word):
    a, f = dict(ALL, **args), dict(FIELDS, **fields)
    assert word in refusal(H, NORM, (*a.values(), 0), f.values())
    assert "null tiling" in refusal(H, NORM, (*a.values(), 0), f.values(), bad_tiling=True)


GRAD = "afir_hip_launch_norm_gate_residual_backward"
GALL = dict(dy=FAKE, dh=FAKE, y=FAKE, f=FAKE, post=FAKE, gate=FAKE, pre=FAKE, dx=FAKE, df=FAKE, dpost=FAKE, dgate=FAKE,
            dpre=FAKE, ws=FAKE)
GFIELDS = dict(m=4, n=64, rpg=2, ld_dy=64, ld_dh=64, ld_y=64, ld_f=64, ld_gate=64, ld_dx=64, ld_df=64, scale=0, eps=0, type=2)


@pytest.mark.parametrize("args,fields,word", [
    (dict(dx=0), {}, "null"),
    (dict(dy=0, dh=0), {}, "null"),
    (dict(y=0), {}, "dh needs"),
    (dict(dpre=0), {}, "dh needs"),
    (dict(df=0), {}, "f needs"),
    (dict(dpost=0), {}, "f needs"),
    (dict(dgate=0), {}, "together"),
    (dict(gate=0), {}, "together"),
    (dict(f=0), {}, "without f"),
    (dict(f=0, dh=0), {}, "neither"),
    (dict(ws=0), {}, "workspace"),
    (dict(ws=FAKE + 2), {}, "workspace"),
    ({}, dict(m=0), "empty"),
    ({}, dict(n=16385), "16384"),
    ({}, dict(rpg=-1), "rows_per_gate"),
    ({}, dict(ld_dx=63), "stride"),
    ({}, dict(ld_df=63), "stride"),
    ({}, dict(ld_dh=63), "stride"),
    ({}, dict(eps=0xbf800000), "eps"),
    ({}, dict(type=-1), "elem_type"),
    (dict(df=FAKE + 1), {}, "alignment"),
])
def test_norm_backward_refuses(H, args, fields, word):
    a, f = dict(GALL, **args), dict(GFIELDS, **fields)
    assert word in refusal(H, GRAD, a.values(), f.values())
    assert "null tiling" in refusal(H, GRAD, a.values(), f.values(), bad_tiling=True)


# y and h, dx and df: (bytes from the first result to the second, their row strides), m = 4, n = 64, two bytes a number
@pytest.mark.parametrize("apart,ld_first,ld_second", [
    (0, 64, 64), (2, 64, 64), (126, 64, 64), (3 * 128, 64, 64), (4 * 128 - 2, 64, 64),   # dense rows
    (0, 200, 200), (126, 200, 200), (200 * 2 - 126, 200, 200), (2 * 400 + 126, 200, 200), (3 * 400 + 126, 200, 200),
    (2 * 400 + 400 - 126, 200, 200), (0, 64, 200), (128, 200, 64), (3 * 400 + 126, 200, 64)])
def test_norms_refuse_two_results_that_overlap(H, apart, ld_first, ld_second):
    for first, second in (("y", "h"), ("h", "y")):
        a = dict(ALL, **{first: FAKE, second: FAKE + apart})
        f = dict(FIELDS, **{"ld_" + first: ld_first, "ld_" + second: ld_second})
        assert "must not overlap" in refusal(H, NORM, (*a.values(), 0), f.values())
    for first, second in (("dx", "df"), ("df", "dx")):
        a = dict(GALL, **{first: FAKE, second: FAKE + apart})
        f = dict(GFIELDS, **{"ld_" + first: ld_first, "ld_" + second: ld_second})
        assert "must not overlap" in refusal(H, GRAD, a.values(), f.values())


def test_empty_calls_launch_nothing(H):
    L = H.load()
    null = [ctypes.c_void_p(0)]
    assert L.afir_hip_launch_mxfp4_quantize(0, None, *null * 5, H.pack_tiling(0, 64, 64, 1, 0)) == 0
    assert L.afir_hip_launch_mxfp4_quantize(0, None, *null * 5, H.pack_tiling(4, 0, 0, 1, 0)) == 0
    assert L.afir_hip_launch_mxfp4_matmul_add_leakyrelu(0, None, *null * 7, H.pack_tiling(0, 64, 8, 0, 2)) == 0
    assert L.afir_hip_launch_norm_gate_residual(0, None, *null * 8, H.pack_tiling(0, 64, 1, 64, 64, 64, 64, 64, 0, 0, 2)) == 0


def test_host_tensors_are_refused(H):
    import torch
    x = torch.zeros(4, 64)
    with pytest.raises(H.AfirHipError, match="device tensor"):
        H.mxfp4_quantize(x)
    with pytest.raises(H.AfirHipError, match="device tensor"):
        H.norm_gate_residual(x, pre_weight=x[0])
    with pytest.raises(H.AfirHipError, match="device tensor"):
        H.norm_gate_residual_backward(x, x, x, pre_weight=x[0])
    with pytest.raises(H.AfirHipError, match="device tensor"):
        H.mxfp4_matmul_add_leakyrelu(x, x, x, x)


@pytest.mark.parametrize("gate,rows_per_gate", [((24,), None), ((1, 24), None), ((1, 24), 7), ((0, 24), None), ((0, 24), 3),
                                                (None, None)])
def test_a_batch_of_no_rows_goes_with_a_learned_gate(H, monkeypatch, gate, rows_per_gate):
    """The host side alone: what would be launched is recorded."""
    import torch
    launched = []
    monkeypatch.setattr(H, "_device_of", lambda t, what: -1)   # host tensors pass for those of one device
    monkeypatch.setattr(H, "_launch_on", lambda index, symbol, block_dim, tiling, *rest: launched.append(tiling))
    x, w = torch.zeros(0, 24), torch.ones(24)
    gate = None if gate is None else torch.ones(gate)
    y, h = H.norm_gate_residual(x, x.clone(), w, gate, w, rows_per_gate=rows_per_gate)
    assert y.shape == h.shape == (0, 24) and len(launched) == 1
    for bad, per in ((torch.ones(2, 24), None), (torch.ones(2, 24), 1), (torch.ones(1, 24), 0)):
        with pytest.raises(H.AfirHipError, match="do not cover"):
            H.norm_gate_residual(x, x.clone(), w, bad, w, rows_per_gate=per)
