"""Cases of the four-bit block products and of the norms around a block: what a pass costs and what it computes.

Four operators, as a residual block of a language model runs them at 4-bit weights and activations:

  quantize   x -> MXFP4: blocks of 32 along one axis share a scale 2^e (e8m0), elements are e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6);
             the pass also returns the numbers the codes stand for (what a calibration or a straight-through gradient uses)
  product    out = leakyrelu(A B^T + bias), A [M, K] and B [N, K] both MXFP4 along K
  norm       y = residual_scale * x + gate * rmsnorm(f) * post_weight;  h = rmsnorm(y) * pre_weight
  norm_grad  the gradients of all of its inputs, given those of y and h

`own` selects the framework's kernels; without it everything is computed with elementary torch operations in 32 bits.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32
EPS = 1e-6


# ---- cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the activations of one new token on their way into a 4-bit product
        {"name": "quantize one token", "op": "quantize", "type": "bf16", "rows": 1, "k": 8192, "axis": -1},
        # the activations of a long batch
        {"name": "quantize activations", "op": "quantize", "type": "bf16", "rows": 8192, "k": 8192, "axis": -1},
        # a weight kept [K, N] in float32, quantised along K and laid out [N, K]: once per load or per training step
        {"name": "quantize weight kn", "op": "quantize", "type": "f32", "rows": 4099, "k": 8192, "axis": 0},
        # one token through a square layer: bound by reading the weight
        {"name": "product one token", "op": "product", "m": 1, "n": 8192, "k": 8192, "type": "bf16", "bias": True},
        # a batch of decoding sequences, through a layer whose width is no multiple of a tile
        {"name": "product 48 tokens", "op": "product", "m": 48, "n": 8200, "k": 4096, "type": "bf16", "bias": True},
        # a prompt of odd length, a width and a depth that end inside tiles, float32 out as logits are kept
        {"name": "product ragged", "op": "product", "m": 1003, "n": 2056, "k": 1376, "type": "f32", "bias": False},
        # a large square product, every extent a whole number of tiles
        {"name": "product 8192", "op": "product", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "bias": True},
        # one token between two blocks
        {"name": "norm one token", "op": "norm", "type": "bf16", "m": 1, "n": 4096, "rows_per_gate": 1},
        # a batch of four sequences, one gate row per sequence (as a modulated block has it)
        {"name": "norm batch", "op": "norm", "type": "bf16", "m": 8192, "n": 4096, "rows_per_gate": 2048},
        # float32, a gate per element, a width that is no multiple of a vector
        {"name": "norm ragged f32", "op": "norm", "type": "f32", "m": 4097, "n": 1001, "rows_per_gate": 1},
        # the backward pass of the batch
        {"name": "norm_grad batch", "op": "norm_grad", "type": "bf16", "m": 8192, "n": 4096, "rows_per_gate": 2048},
        # a short ragged batch in half precision, one learned gate row for all of it
        {"name": "norm_grad ragged f16", "op": "norm_grad", "type": "f16", "m": 333, "n": 5000, "rows_per_gate": 333},
    ]


def _log_size(rng, low, high):
    """A size spread over the logarithm of its range; about a third are multiples of 32."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.35:
        v = max(32, v // 32 * 32)
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["quantize", "quantize", "product", "product", "product", "norm", "norm", "norm_grad"])
    if op == "quantize":
        return {"op": op, "type": rng.choice(["f32", "f16", "bf16"]), "rows": _log_size(rng, 1, 8192),
                "k": _log_size(rng, 1, 8192), "axis": rng.choice([-1, 0])}
    if op == "product":
        return {"op": op, "m": _log_size(rng, 1, 8192), "n": _log_size(rng, 1, 8192), "k": _log_size(rng, 1, 8192),
                "type": rng.choice(["bf16", "bf16", "f16", "f32"]), "bias": rng.random() < 0.7}
    m, n = _log_size(rng, 1, 8192), _log_size(rng, 1, 4096)
    per = rng.choice([1, m, max(1, m // rng.randint(2, 9)), rng.randint(1, m)])
    return {"op": op, "type": rng.choice(["f32", "f16", "bf16"]), "m": m, "n": n, "rows_per_gate": per}


def _blocks(k):
    return -(-k // BLOCK)


def work(case):
    op = case["op"]
    if op == "quantize":
        rows, k, e = case["rows"], case["k"], SIZE[case["type"]]
        kb = _blocks(k)
        return {"bytes": rows * (2 * k * e + kb * 17), "flops": 4 * rows * k}
    if op == "product":
        m, n, k, e = case["m"], case["n"], case["k"], SIZE[case["type"]]
        return {"bytes": (m + n) * _blocks(k) * 17 + m * n * e + (n * e if case["bias"] else 0), "flops": 2 * m * n * k}
    m, n, e = case["m"], case["n"], SIZE[case["type"]]
    gates = -(-m // case["rows_per_gate"])
    if op == "norm":
        return {"bytes": (4 * m * n + gates * n + 2 * n) * e, "flops": 12 * m * n}
    return {"bytes": (6 * m * n + 2 * gates * n + 4 * n) * e, "flops": 30 * m * n}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _normal(shape, gen, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale


def _activations(rows, k, gen):
    """Rows as a model's activations are: a scale of their own per row, a few channels far above the others, some
    blocks of zeros (padding)."""
    x = _normal((rows, k), gen)
    x *= torch.exp(_normal((rows, 1), gen))
    x *= torch.where(torch.rand((1, k), generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    x[torch.rand((rows,), generator=gen, device="cuda") < 0.02] = 0.0
    return x


def _mx_operand(rows, k, gen, scale):
    """Codes and scale bytes of a normal matrix: what a program holds after it has quantised a weight or a batch."""
    codes, exponent, _ = _plain_quantize(_normal((rows, k), gen, scale))
    return _pack(codes), (exponent + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    state = dict(case)
    if case["op"] == "quantize":
        x = _activations(case["rows"], case["k"], gen).to(TYPES[case["type"]])
        state["x"] = x if case["axis"] == -1 else x.t().contiguous()
    elif case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        state["a"] = _mx_operand(m, k, gen, 1.0)
        state["b"] = _mx_operand(n, k, gen, 1.0 / math.sqrt(k))
        state["bias_row"] = _normal((n,), gen, 0.1).to(TYPES[case["type"]]) if case["bias"] else None
    else:
        m, n, t = case["m"], case["n"], TYPES[case["type"]]
        gates = -(-m // case["rows_per_gate"])
        state["f"] = _normal((m, n), gen, 2.0).to(t)
        state["post_weight"] = (1.0 + _normal((n,), gen, 0.2)).to(t)
        state["pre_weight"] = (1.0 + _normal((n,), gen, 0.2)).to(t)
        state["gate"] = torch.sigmoid(_normal((gates, n), gen)).to(t)
        if case["op"] == "norm":
            state["x"] = _normal((m, n), gen, 3.0).to(t)
        else:
            state["y"] = _normal((m, n), gen, 3.0).to(t)
            state["dy"] = _normal((m, n), gen, 0.5).to(t)
            state["dh"] = _normal((m, n), gen, 0.5).to(t)
    return state


RESIDUAL_SCALE = 0.875
ALPHA = 0.01


# ---- the plain forms --------------------------------------------------------------------------------------------

def _plain_quantize(x):
    """x [R, K] float32 -> (codes [R, Kb*32] of 0..15, exponents [R, Kb], values [R, K] float32)."""
    rows, k = x.shape
    kb = _blocks(k)
    padded = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).reshape(rows, kb, BLOCK)
    top = padded.abs().amax(dim=2)
    finite = torch.isfinite(top)
    exponent = torch.where(top > 0, torch.frexp(torch.where(finite, top, 1.0))[1] - 3, -127).clamp(-127, 127)
    v = torch.ldexp(padded, -exponent.unsqueeze(2))
    size = v.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    near = (torch.round(size / step) * step).clamp(max=6.0)
    near = torch.where(finite.unsqueeze(2), near, 0.0)
    code = torch.where(near < 2, near * 2, torch.where(near < 4, near + 2, near / 2 + 4)).to(torch.uint8)
    code = code + 8 * (torch.signbit(v) & finite.unsqueeze(2)).to(torch.uint8)
    exponent = torch.where(finite, exponent, 128)
    values = torch.ldexp(torch.copysign(near, v), exponent.unsqueeze(2))
    values = torch.where(finite.unsqueeze(2), values, math.nan).reshape(rows, kb * BLOCK)[:, :k]
    return code.reshape(rows, kb * BLOCK), exponent, values


def _pack(codes):
    """Two codes a byte, the lower k in the lower four bits."""
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def _plain_decode(packed, scales):
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    codes = torch.stack([packed & 15, packed >> 4], dim=2).reshape(packed.shape[0], -1, BLOCK)
    return (table[codes.int()] * scales.float().unsqueeze(2)).reshape(packed.shape[0], -1)


def _plain_rms(x):
    return torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS)


def _gate_rows(gate, m, per):
    return gate.float().repeat_interleave(per, dim=0)[:m]


def _plain_norm(s):
    t, f, x = TYPES[s["type"]], s["f"].float(), s["x"].float()
    gate = _gate_rows(s["gate"], s["m"], s["rows_per_gate"])
    y = RESIDUAL_SCALE * x + gate * (f * _plain_rms(f)) * s["post_weight"].float()
    h = y * _plain_rms(y) * s["pre_weight"].float()
    return {"y": y.to(t), "h": h.to(t)}


def _plain_norm_grad(s):
    t, m, n, per = TYPES[s["type"]], s["m"], s["n"], s["rows_per_gate"]
    y, f, dy, dh = (s[k].float() for k in ("y", "f", "dy", "dh"))
    gate = _gate_rows(s["gate"], m, per)
    post, pre = s["post_weight"].float(), s["pre_weight"].float()
    ry, rf = _plain_rms(y), _plain_rms(f)
    yn, fn = y * ry, f * rf
    a = dh * pre
    total = dy + ry * (a - yn * (a * yn).mean(dim=1, keepdim=True))
    b = total * gate * post
    df = rf * (b - fn * (b * fn).mean(dim=1, keepdim=True))
    groups = -(-m // per)
    dgate = total * fn * post
    dgate = torch.nn.functional.pad(dgate, (0, 0, 0, groups * per - m)).reshape(groups, per, n).sum(dim=1)
    return {"dx": (RESIDUAL_SCALE * total).to(t), "df": df.to(t), "dpost_weight": (total * gate * fn).sum(dim=0).to(t),
            "dgate": dgate.to(t), "dpre_weight": (dh * yn).sum(dim=0).to(t)}


# ---- one pass ---------------------------------------------------------------------------------------------------

_kernels = None


def _framework():
    global _kernels
    if _kernels is None:
        from __graft_entry__ import load_package
        load_package()
        from ascend_mlir_amd import hip_kernels
        _kernels = hip_kernels
    return _kernels


def run(state):
    s, op = state, state["op"]
    if own:
        H = _framework()
        if op == "quantize":
            _, scales, values = H.mxfp4_quantize(s["x"], axis=s["axis"], return_values=True)
            return {"values": values, "scales": scales}
        if op == "product":
            return H.mxfp4_matmul_add_leakyrelu(*s["a"], *s["b"], s["bias_row"], alpha=ALPHA, out_dtype=TYPES[s["type"]])
        if op == "norm":
            y, h = H.norm_gate_residual(s["x"], s["f"], s["post_weight"], s["gate"], s["pre_weight"],
                                        residual_scale=RESIDUAL_SCALE, eps=EPS, rows_per_gate=s["rows_per_gate"])
            return {"y": y, "h": h}
        dx, df, dpost, dgate, dpre = H.norm_gate_residual_backward(
            s["dy"], s["dh"], s["y"], s["f"], s["post_weight"], s["gate"], s["pre_weight"],
            residual_scale=RESIDUAL_SCALE, eps=EPS, rows_per_gate=s["rows_per_gate"])
        return {"dx": dx, "df": df, "dpost_weight": dpost, "dgate": dgate, "dpre_weight": dpre}
    if op == "quantize":
        x = s["x"] if s["axis"] == -1 else s["x"].t()
        _, exponent, values = _plain_quantize(x.float())
        values = values if s["axis"] == -1 else values.t().contiguous()
        scales = (exponent + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
        return {"values": values.to(s["x"].dtype), "scales": scales}
    if op == "product":
        out = torch.mm(_plain_decode(*s["a"]), _plain_decode(*s["b"]).t())
        if s["bias_row"] is not None:
            out += s["bias_row"].float()
        return torch.maximum(out, out * ALPHA).to(TYPES[s["type"]])
    return _plain_norm(s) if op == "norm" else _plain_norm_grad(s)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------

def _exact_quantize(x):
    """Nearest of the representable values, by their midpoints; a midpoint goes to the even neighbour."""
    rows, k = x.shape
    kb = _blocks(k)
    x = torch.nn.functional.pad(x.double(), (0, kb * BLOCK - k)).reshape(rows, kb, BLOCK)
    top = x.abs().amax(dim=2, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -149)))
    e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e))
    scale = torch.exp2(torch.where(top > 0, (e - 2).clamp(min=-127), -127.0))
    z = x.abs() / scale
    value = torch.zeros_like(z)
    for edge, above, wins in ((.25, .5, False), (.75, 1, True), (1.25, 1.5, False), (1.75, 2, True), (2.5, 3, False),
                              (3.5, 4, True), (5, 6, False)):
        value = torch.where(z >= edge if wins else z > edge, float(above), value)
    return (torch.sign(x) * value * scale).reshape(rows, kb * BLOCK)[:, :k], scale.squeeze(2)


def _exact_decode(packed, scales):
    nibble = torch.stack([packed & 15, packed >> 4], dim=2).reshape(packed.shape[0], -1).to(torch.int16)
    e, m = (nibble >> 1) & 3, (nibble & 1).double()
    size = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e.double() - 1))
    value = torch.where(nibble >= 8, -size, size)
    power = torch.exp2(scales.view(torch.uint8).double() - 127)
    return value * power.repeat_interleave(BLOCK, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        values, scale = _exact_quantize(s["x"] if case["axis"] == -1 else s["x"].t())
        return {"values": values if case["axis"] == -1 else values.t().contiguous(), "scales": scale}
    if case["op"] == "product":
        out = torch.mm(_exact_decode(*s["a"]), _exact_decode(*s["b"]).t().contiguous())
        if s["bias_row"] is not None:
            out += s["bias_row"].double()
        return torch.where(out > 0, out, out * ALPHA)
    m, n, per = case["m"], case["n"], case["rows_per_gate"]
    at = torch.arange(m, device="cuda") // per
    f, post, pre, gate = (s[k].double() for k in ("f", "post_weight", "pre_weight", "gate"))
    f.requires_grad_(), post.requires_grad_(), pre.requires_grad_(), gate.requires_grad_()

    def normed(v):
        return v / torch.sqrt(v.square().sum(dim=1, keepdim=True) / n + EPS)

    branch = gate[at] * normed(f) * post
    if case["op"] == "norm":
        y = RESIDUAL_SCALE * s["x"].double() + branch
        return {"y": y.detach(), "h": (normed(y) * pre).detach()}
    # the gradient by automatic differentiation, at the y that the forward pass wrote
    y = s["y"].double().requires_grad_()
    through_h, dpre = torch.autograd.grad((normed(y) * pre * s["dh"].double()).sum(), (y, pre))
    total = s["dy"].double() + through_h
    df, dpost, dgate = torch.autograd.grad((branch * total).sum(), (f, post, gate))
    return {"dx": RESIDUAL_SCALE * total, "df": df, "dpost_weight": dpost, "dgate": dgate, "dpre_weight": dpre}
