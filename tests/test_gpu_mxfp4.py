"""MXFP4 quantisation and products on the GPU against the float64 oracle."""
import numpy as np
import pytest
import torch

from oracle import block_oracle as O
from tests import block_cases as B

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def H(pkg):
    from ascend_mlir_amd import hip_kernels
    hip_kernels.load()
    assert torch.cuda.is_available(), "no GPU visible"
    return hip_kernels


def check_quantize(H, x, axis, **kw):
    """Codes, scales and values are exact: no tolerance."""
    want = O.quantize(B.numbers(x) if axis else B.numbers(x).T)
    codes, scales, values = H.mxfp4_quantize(x, axis=axis, return_values=True, **kw)
    torch.cuda.synchronize()
    assert np.array_equal(scales.view(torch.uint8).cpu().numpy(), want[1])
    assert np.array_equal(codes.cpu().numpy(), want[0])
    got = B.numbers(values)
    back = want[2] if axis else want[2].T
    assert np.array_equal(got, back, equal_nan=True)
    fine = ~np.isnan(back)
    assert np.array_equal(np.signbit(got[fine]), np.signbit(back[fine]))
    two = H.mxfp4_quantize(x, axis=axis, **kw)          # without the values: the same codes
    assert len(two) == 2 and torch.equal(two[0], codes) and torch.equal(two[1].view(torch.uint8), scales.view(torch.uint8))


@pytest.mark.parametrize("kind", B.TYPES)
@pytest.mark.parametrize("axis", [1, 0])
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (64, 64), (7, 1000), (130, 257), (1, 8192),
                                   (300, 129), (33, 2050), (2, 5)])
def test_quantize(H, kind, axis, shape):
    rng = np.random.default_rng(shape[0] * 1000 + shape[1])
    x = rng.normal(size=shape) * np.exp2(rng.integers(-12, 8, (shape[0], 1)))
    x[rng.random(shape) < 0.1] = 0
    x[rng.random(shape[0]) < 0.2] = 0
    check_quantize(H, B.tensor(x, kind, "cuda"), axis)


@pytest.mark.parametrize("kind", B.TYPES)
@pytest.mark.parametrize("axis", [1, 0])
def test_quantize_ties_and_special_numbers(H, kind, axis):
    t = B.TYPES[kind]
    info = torch.finfo(t)
    grid = np.concatenate([np.arange(0, 33) / 4, [0.126, 0.2499, 1.2499, 5.0001, 7.99]])
    rows = []
    for e in (0, 3, -5, -9):
        block = np.resize(grid, 64) * np.exp2(float(e)) * np.resize([1, -1, 1], 64)
        block[31] = block[63] = 4 * np.exp2(float(e))
        rows.append(block)
    x = B.tensor(np.array(rows), kind, "cpu")
    extra = torch.zeros((9, 64), dtype=t)
    extra[0, :] = -0.0
    extra[1, 5], extra[1, 40] = float("inf"), 1.0
    extra[2, 5], extra[2, 40] = float("nan"), -3.0
    extra[3, 63], extra[3, 62] = -float("inf"), info.max
    extra[4, :] = info.max
    extra[5, :] = info.smallest_normal
    extra[6, :] = info.smallest_normal * info.eps      # the smallest subnormal
    extra[6, 3] *= 3
    extra[7, 1], extra[7, 33] = info.smallest_normal * 1.5, info.smallest_normal * 4
    extra[8, ::2], extra[8, 1::2] = -info.max, info.smallest_normal
    x = torch.cat([x, extra]).cuda()
    check_quantize(H, x if axis else x.t().contiguous(), axis)


@pytest.mark.parametrize("kind", B.TYPES)
def test_quantize_every_16_bit_number(H, kind):
    if kind == "f32":
        bits = torch.arange(0, 1 << 16, dtype=torch.int32) * 65537 + 12345    # spread over the float32 patterns
        x = bits.view(torch.float32)
    else:
        x = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(B.TYPES[kind])
    # neighbours in value share a block, and every number meets a block of far larger ones too
    x = torch.cat([x.reshape(-1, 64), x.reshape(64, -1).t()]).cuda()
    check_quantize(H, x.contiguous(), 1)
    check_quantize(H, x.t().contiguous(), 0)


@pytest.mark.parametrize("axis", [1, 0])
def test_quantize_rows_with_a_stride_and_off_alignment(H, axis):
    rng = np.random.default_rng(5)
    for kind in B.TYPES:
        wide = B.tensor(rng.normal(size=(65, 403)), kind, "cuda")
        check_quantize(H, wide[:, 1:258], axis)          # rows start off every boundary but an element's
        check_quantize(H, wide[3:4, 2:100], axis)
        check_quantize(H, wide[::2, :64], axis)


def test_quantize_into_given_tensors_and_few_workgroups(H):
    x = torch.randn(40, 200, device="cuda", dtype=torch.bfloat16)
    guard = torch.full((42, 7 * 16), 77, dtype=torch.uint8, device="cuda")
    scales = torch.full((42, 7), 77, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    values = torch.full((42, 200), 77.0, dtype=torch.bfloat16, device="cuda")
    want = H.mxfp4_quantize(x, return_values=True)
    got = H.mxfp4_quantize(x, codes=guard[1:41], scales=scales[1:41], values=values[1:41], block_dim=1)
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for t in (guard, scales.view(torch.uint8), values):   # the rows around are left as they were
        assert (t[0] == 77).all() and (t[41] == 77).all()
    xt = x.t().contiguous()
    got = H.mxfp4_quantize(xt, axis=0, codes=guard[1:41], scales=scales[1:41], block_dim=2)
    assert torch.equal(got[0], want[0])
    assert (guard[0] == 77).all() and (guard[41] == 77).all()


def test_quantize_refuses(H):
    x = torch.zeros(8, 64, device="cuda")
    for bad, word in ((dict(x=x.int()), "float32"), (dict(x=x[0]), "two dimensions"), (dict(x=x, axis=2), "axis"),
                      (dict(x=x.t()), "adjacent"), (dict(x=x[:1].expand(8, 64)), "overlap"),
                      (dict(x=x, codes=torch.zeros(8, 31, dtype=torch.uint8, device="cuda")), "shape"),
                      (dict(x=x, codes=torch.zeros(8, 32, device="cuda")), "uint8"),
                      (dict(x=x, scales=torch.zeros(8, 2, dtype=torch.uint8, device="cuda")), "e8m0"),
                      (dict(x=x, values=torch.zeros(8, 64, device="cuda").half()), "float32"),
                      (dict(x=x, values=torch.zeros(64, 8, device="cuda").t()), "contiguous")):
        with pytest.raises(H.AfirHipError, match=word):
            H.mxfp4_quantize(**bad)


# ---- products ----

def operand(rng, rows, k, spread=3):
    kb = -(-k // 32)
    codes = rng.integers(0, 256, (rows, kb * 16), dtype=np.uint8)
    scales = (127 + rng.integers(-spread, spread + 1, (rows, kb))).astype(np.uint8)
    return codes, scales


def check_matmul(H, m, n, k, kind, bias=True, alpha=0.01, seed=0, **kw):
    rng = np.random.default_rng(seed + 7 * m + 11 * n + 13 * k)
    (ac, asc), (bc, bsc) = operand(rng, m, k), operand(rng, n, k)
    size_of_sum = np.sqrt(k) * 10
    bias_t = B.tensor(rng.normal(size=n) * size_of_sum, kind, "cuda") if bias else None
    want, size = O.matmul(O.decode(ac, asc), O.decode(bc, bsc), None if bias_t is None else B.numbers(bias_t), alpha)
    dev = [torch.from_numpy(t).cuda() for t in (ac, asc, bc, bsc)]
    guard = torch.full((m + 2, n), 77.0, dtype=B.TYPES[kind], device="cuda")
    got = H.mxfp4_matmul_add_leakyrelu(dev[0], dev[1].view(torch.float8_e8m0fnu), dev[2], dev[3].view(torch.float8_e8m0fnu),
                                       bias_t, alpha=alpha, out=guard[1:m + 1] if n % 8 == 0 else None,
                                       out_dtype=B.TYPES[kind], **kw)
    torch.cuda.synchronize()
    # numbers of a block are multiples of 1/4 up to 36, their sum over a block is exact in float32; what rounds is the
    # sum over ceil(k / 32) blocks, the joining of eight partial sums, the bias and the slope
    B.close(got, want, size, kind, -(-k // 32) + 10)
    if n % 8 == 0:
        assert (guard[0] == 77).all() and (guard[m + 1] == 77).all()
    return got


@pytest.mark.parametrize("kind", B.TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 32), (1, 40, 33), (3, 31, 96), (15, 257, 512), (16, 32, 544),
                                   (17, 48, 1056), (33, 100, 4096), (48, 72, 8192), (64, 33, 640), (65, 17, 256),
                                   (130, 264, 288)])
def test_matmul(H, kind, m, n, k):
    check_matmul(H, m, n, k, kind)
    check_matmul(H, m, n, k, kind, bias=False, alpha=1.0)


@pytest.mark.parametrize("m,n,k", [(1, 24, 2048), (64, 520, 1000), (200, 1032, 776)])
def test_matmul_on_few_workgroups(H, m, n, k):
    a = check_matmul(H, m, n, k, "bf16", block_dim=3)
    assert torch.equal(a, check_matmul(H, m, n, k, "bf16"))


@pytest.mark.parametrize("kind,m,n,k,blocks", [
    ("bf16", 66, 130, 32, 0), ("f32", 129, 127, 256, 0), ("f16", 128, 128, 512, 0), ("bf16", 257, 300, 768, 2),
    ("f32", 500, 1029, 1376, 0), ("bf16", 1000, 520, 2080, 5), ("f16", 384, 640, 8192, 3),
    # as many tiles of 256 x 256 as the chip has compute units, and more
    ("bf16", 4100, 4090, 288, 0), ("f32", 4096, 4096, 160, 0), ("f16", 4097, 4104, 1024, 0), ("bf16", 4350, 4601, 32, 0),
    ("bf16", 4096, 4352, 608, 7), ("bf16", 4100, 4090, 256, 0), ("f16", 4300, 4100, 4384, 100), ("bf16", 4352, 4096, 512, 0), ("f32", 4129, 4353, 1312, 200)])
def test_matmul_on_tiles(H, kind, m, n, k, blocks):
    check_matmul(H, m, n, k, kind, block_dim=blocks)
    # the tiled kernels take whole lines of 256 numbers, shallower products have a kernel of their own, and few
    # tiles go to the kernel with a workgroup per tile
    few = -(-m // 128) * -(-n // 128) <= 256
    assert H.last_launch()["kernel"] == ("mxfp4_matmul_direct" if k <= 224 else
                                         "mxfp4_matmul_ring" if few else "mxfp4_matmul_tiles")


@pytest.mark.parametrize("kind,m,n,k,blocks", [
    # one to many slices of 256, the last one whole or of half the blocks; few and many tiles
    ("bf16", 65, 64, 256, 0), ("f32", 70, 130, 384, 0), ("f16", 128, 200, 512, 0), ("bf16", 129, 257, 640, 0),
    ("bf16", 66, 72, 768, 1), ("f32", 200, 100, 1024, 0), ("f16", 257, 520, 1152, 0), ("bf16", 300, 1030, 2176, 3),
    ("f32", 1000, 2050, 640, 0), ("bf16", 1025, 1796, 1408, 0), ("f16", 2000, 1500, 256, 0), ("bf16", 2048, 2048, 384, 100),
    ("bf16", 130, 8200, 1024, 0),
    # scale rows of whole 16-byte pieces, of whole words and of neither; more slices than a tile's scales are held for
    ("f32", 80, 96, 8192 + 512, 0), ("bf16", 80, 96, 8192 + 384, 0), ("f16", 80, 96, 8192 + 416, 0),
    ("f32", 257, 130, 16384 + 32, 0), ("f32", 70, 65, 1376, 0), ("bf16", 150, 300, 8192 + 256, 2), ("f32", 66, 70, 255, 0),
    ("f16", 300, 2048, 992, 0), ("bf16", 500, 4100, 736, 0),
    # tiles of 32 and 64 rows, below and above a full chip
    ("bf16", 17, 16, 256, 0), ("f32", 31, 33, 384, 0), ("f16", 32, 8200, 512, 0), ("bf16", 33, 40, 1376, 0),
    ("f32", 48, 8200, 768, 0), ("bf16", 64, 16400, 1056, 0), ("f16", 64, 32, 8192 + 640, 2), ("bf16", 18, 130, 8192 + 416, 1),
    # more slices than the scales held: 1 to 32 of them beyond, rows of scales whole, of words and of bytes
    ("f32", 40, 70, 8192 + 4096, 0), ("bf16", 65, 64, 8192 + 512, 0), ("f16", 150, 260, 8192 + 4096 + 128, 0),
    ("bf16", 33, 100, 16384, 0), ("f32", 70, 40, 16384 + 256, 1), ("bf16", 20, 48, 16384 + 4096 + 32, 0),
    ("f16", 260, 4100, 8192 + 2048 + 384, 0), ("f32", 130, 130, 4096 + 96, 0), ("bf16", 40, 40, 4096 + 128, 0),
    ("f32", 40, 24600, 640, 0), ("bf16", 96, 2048, 2048, 0), ("bf16", 64, 8192, 512, 0)])
def test_matmul_with_a_workgroup_per_tile(H, kind, m, n, k, blocks):
    check_matmul(H, m, n, k, kind, block_dim=blocks)
    assert H.last_launch()["kernel"] == "mxfp4_matmul_ring"
    check_matmul(H, m, n, k, kind, bias=False, alpha=1.0, seed=1)


@pytest.mark.parametrize("kind", B.TYPES)
@pytest.mark.parametrize("m,n,k,blocks", [(17, 300, 1, 0), (17, 1, 31, 0), (40, 33, 70, 0), (64, 64, 64, 0), (129, 127, 128, 3),
                                          (70, 2000, 160, 0), (1000, 1031, 224, 0), (3000, 3010, 97, 0), (4096, 2056, 33, 40)])
def test_matmul_of_little_depth(H, kind, m, n, k, blocks):
    check_matmul(H, m, n, k, kind, block_dim=blocks)
    assert H.last_launch()["kernel"] == "mxfp4_matmul_direct"
    check_matmul(H, m, n, k, kind, bias=False, alpha=1.0, seed=1)


@pytest.mark.parametrize("kind,m,n,k", [("bf16", 4200, 1100, 288), ("f32", 2100, 2100, 512), ("f16", 70, 33000, 256)])
def test_matmul_without_a_workspace(H, monkeypatch, kind, m, n, k):
    a = check_matmul(H, m, n, k, kind)
    monkeypatch.setattr(H, "_workspace", lambda *query: None)
    b = check_matmul(H, m, n, k, kind)
    assert H.last_launch()["kernel"] == "mxfp4_matmul_ring"
    # both add the blocks of a row in one order, onto the bias
    assert torch.equal(a, b)


def test_matmul_without_depth_is_the_bias(H):
    a = torch.zeros((5, 0), dtype=torch.uint8, device="cuda")
    b = torch.zeros((24, 0), dtype=torch.uint8, device="cuda")
    s = lambda t: torch.zeros((t.shape[0], 0), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    bias = torch.randn(24, device="cuda").bfloat16()
    got = H.mxfp4_matmul_add_leakyrelu(a, s(a), b, s(b), bias, alpha=0.5)
    want = torch.maximum(bias.float(), bias.float() * 0.5).bfloat16().expand(5, 24)
    assert torch.equal(got, want)
    assert not H.mxfp4_matmul_add_leakyrelu(a, s(a), b, s(b)).any()


@pytest.mark.parametrize("m", [1, 17, 300])
def test_matmul_without_depth_for_any_number_of_rows(H, m):
    a, b = (torch.zeros((r, 0), dtype=torch.uint8, device="cuda") for r in (m, 40))
    scales = [t.view(torch.float8_e8m0fnu) for t in (a, b)]
    bias = torch.linspace(-3, 5, 40, device="cuda")
    got = H.mxfp4_matmul_add_leakyrelu(a, scales[0], b, scales[1], bias, alpha=0.5, out_dtype=torch.float32)
    assert torch.equal(got, torch.maximum(bias, bias * 0.5).expand(m, 40))
    assert not H.mxfp4_matmul_add_leakyrelu(a, scales[0], b, scales[1]).any()


def test_matmul_keeps_nan_to_the_rows_and_columns_that_hold_it(H):
    rng = np.random.default_rng(3)
    for m, n, k in ((5, 40, 320), (70, 80, 1056)):
        (ac, asc), (bc, bsc) = operand(rng, m, k), operand(rng, n, k)
        asc[2, -1] = 255
        bsc[7, 0] = 255
        bc[7, :16] = 0                       # as quantisation writes such a block
        dev = [torch.from_numpy(t).cuda() for t in (ac, asc, bc, bsc)]
        got = H.mxfp4_matmul_add_leakyrelu(dev[0], dev[1].view(torch.float8_e8m0fnu), dev[2],
                                           dev[3].view(torch.float8_e8m0fnu), out_dtype=torch.float32)
        want = np.zeros((m, n), dtype=bool)
        want[2, :] = want[:, 7] = True
        assert np.array_equal(np.isnan(got.cpu().numpy()), want)


def test_matmul_scales_at_their_ends(H):
    # scale bytes 0 and 254: the sums stay in range because the other operand's scales answer them
    k, m, n = 576, 9, 33
    rng = np.random.default_rng(4)
    (ac, asc), (bc, bsc) = operand(rng, m, k), operand(rng, n, k)
    asc[:], bsc[:] = 0, 254
    asc[:, ::2], bsc[:, ::2] = 250, 4
    want, size = O.matmul(O.decode(ac, asc), O.decode(bc, bsc), None, 1.0)
    dev = [torch.from_numpy(t).cuda() for t in (ac, asc, bc, bsc)]
    got = H.mxfp4_matmul_add_leakyrelu(dev[0], dev[1].view(torch.float8_e8m0fnu), dev[2], dev[3].view(torch.float8_e8m0fnu),
                                       alpha=1.0, out_dtype=torch.float32)
    B.close(got, want, size, "f32", k // 32 + 10)


@pytest.mark.parametrize("m,n,k", [(4100, 4200, 1056), (260, 8300, 608), (40, 300, 1184), (300, 200, 640), (90, 70, 192), (4100, 4200, 160)])
def test_matmul_of_many_rows_keeps_nan_and_scales_at_their_ends(H, m, n, k):
    # in rows, columns and blocks of both operands: on tiles (the first two), on a workgroup per tile, of little depth
    rng = np.random.default_rng(5)
    (ac, asc), (bc, bsc) = operand(rng, m, k), operand(rng, n, k)
    asc[:], bsc[:] = 0, 254
    asc[:, ::2], bsc[:, ::2] = 250, 4
    asc[m - 1, -1] = asc[2, -4] = 255
    bsc[7, 0] = bsc[n - 2, max(-9, -bsc.shape[1])] = 255
    want, size = O.matmul(O.decode(ac, asc), O.decode(bc, bsc), None, 1.0)
    dev = [torch.from_numpy(t).cuda() for t in (ac, asc, bc, bsc)]
    got = H.mxfp4_matmul_add_leakyrelu(dev[0], dev[1].view(torch.float8_e8m0fnu), dev[2], dev[3].view(torch.float8_e8m0fnu),
                                       alpha=1.0, out_dtype=torch.float32)
    lost = np.zeros((m, n), dtype=bool)
    lost[m - 1] = lost[2] = lost[:, 7] = lost[:, n - 2] = True
    assert np.array_equal(np.isnan(got.cpu().numpy()), lost)
    keep = torch.from_numpy(~lost).cuda()
    B.close(got[keep], want[~lost], size[~lost], "f32", k // 32 + 10)


@pytest.mark.parametrize("kind", B.TYPES)
@pytest.mark.parametrize("axis", [1, 0])
def test_quantize_in_place(H, kind, axis):
    x = torch.randn(170, 300, device="cuda").to(B.TYPES[kind])
    want = H.mxfp4_quantize(x, axis=axis, return_values=True)
    got = H.mxfp4_quantize(x, axis=axis, values=x)
    assert got[2] is x
    for a, b in zip(got, want):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def test_results_on_a_given_stream_come_from_its_memory(H):
    # memory freed on the current stream may still be written by what runs there
    x = torch.randn(256, 2048, device="cuda").bfloat16()
    (qa, sa), (qb, sb) = H.mxfp4_quantize(x), H.mxfp4_quantize(x[:72].contiguous())
    want = H.mxfp4_matmul_add_leakyrelu(qa, sa, qb, sb)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    freed = [torch.empty_like(t) for t in (qa, sa, want)]
    places = {t.data_ptr() for t in freed}
    del freed
    codes, scales = H.mxfp4_quantize(x, stream=side.cuda_stream)
    got = H.mxfp4_matmul_add_leakyrelu(codes, scales, qb, sb, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(codes, qa) and torch.equal(got, want)
    assert not places & {t.data_ptr() for t in (codes, scales, got)}


def test_matmul_refuses(H):
    u8 = dict(dtype=torch.uint8, device="cuda")
    a, b = torch.zeros(4, 32, **u8), torch.zeros(8, 32, **u8)
    sa, sb = (torch.zeros(t.shape[0], 2, **u8).view(torch.float8_e8m0fnu) for t in (a, b))
    bias = torch.zeros(8, device="cuda", dtype=torch.bfloat16)
    H.mxfp4_matmul_add_leakyrelu(a, sa, b, sb, bias, k=63)
    for args, kw, word in (((a, sa, b[:, :16], sb), {}, "shape"), ((a, sa, b, sa), {}, "shape"),
                           ((a[:, :24], sa, b, sb), {}, "whole blocks"), ((a.int(), sa, b, sb), {}, "uint8"),
                           ((a, sa.view(torch.uint8), b, sb), {}, "e8m0"), ((a, sa, b, sb, bias.float()), {}, "bfloat16"),
                           ((a, sa, b, sb, bias[:4]), {}, "shape"), ((a, sa, b, sb), dict(k=65), "blocks"),
                           ((a, sa, b, sb), dict(k=32), "blocks"), ((a, sa, b, sb), dict(out_dtype=torch.int32), "float32"),
                           ((a, sa, b, sb), dict(out=bias.reshape(1, 8)), "shape"),
                           ((torch.zeros(32, 4, **u8).t(), sa, b, sb), {}, "contiguous"),
                           ((torch.zeros(4 * 32 + 1, **u8)[1:].view(4, 32), sa, b, sb), {}, "16-byte")):
        with pytest.raises(H.AfirHipError, match=word):
            H.mxfp4_matmul_add_leakyrelu(*args, **kw)


def random_operand(rows, kb, gen):
    """Codes and scales made on the GPU: any code, scales of 2^-3 to 2^3."""
    codes = torch.randint(0, 256, (rows, kb * 16), dtype=torch.uint8, device="cuda", generator=gen)
    return codes, torch.randint(124, 131, (rows, kb), dtype=torch.uint8, device="cuda", generator=gen)


def decoded(operand, rows):
    return O.decode(operand[0][rows].cpu().numpy(), operand[1][rows].cpu().numpy())


def test_matmul_of_more_columns_than_a_launch_has_threads(H):
    # 2^28 columns and some: 2^23 tiles of 32 columns and 512 threads each
    n, gen = (1 << 28) + 77, torch.Generator(device="cuda").manual_seed(6)
    a, b = random_operand(1, 1, gen), random_operand(n, 1, gen)
    e8 = torch.float8_e8m0fnu
    out = torch.full((n + 64,), 77.0, dtype=torch.bfloat16, device="cuda")
    got = H.mxfp4_matmul_add_leakyrelu(a[0], a[1].view(e8), b[0], b[1].view(e8), alpha=0.25, out=out[:n].view(1, n))
    assert H.last_launch()["kernel"] == "mxfp4_matmul_rows"
    torch.cuda.synchronize()
    assert (out[n:] == 77).all()
    # the first and the last columns, both sides of each bound on the way, and some from everywhere
    some = torch.cat([torch.arange(at - 70, at + 70) for at in (70, 1 << 25, 1 << 26, 1 << 27, 1 << 28, n - 70)] +
                     [torch.randint(0, n, (20000,))]).cuda()
    want, size = O.matmul(decoded(a, slice(None)), decoded(b, some), None, 0.25)
    B.close(got[:, some], want, size, "bf16", 11)


@pytest.mark.parametrize("kind", B.TYPES)
@pytest.mark.parametrize("m,n,k,blocks", [
    # 32 columns a workgroup (n above 16 per compute unit), the last ones partly past the end; more steps of 512 numbers
    # than the eight wavefronts take in one go, the last step whole or not
    (1, 4097, 4096, 0), (7, 4129, 4128, 0), (16, 8200, 608, 0), (16, 4128, 8192, 0), (1, 5003, 8192 + 416, 0),
    (7, 4100, 8192 + 512, 37), (16, 4129, 32, 5), (1, 8224, 65, 0),
    # 16 columns a workgroup, as deep
    (1, 520, 8192 + 416, 0), (16, 72, 4096 + 512, 0), (7, 4096, 4128, 3), (3, 17, 3 * 4096 + 32, 0)])
def test_matmul_of_few_rows(H, kind, m, n, k, blocks):
    check_matmul(H, m, n, k, kind, block_dim=blocks)
    last, tiles = H.last_launch(), -(-n // (32 if n > 4096 else 16))
    assert last["kernel"] == "mxfp4_matmul_rows" and last["workgroups"] == (blocks or -(-tiles // 8) * 8)
    check_matmul(H, m, n, k, kind, bias=False, alpha=1.0, seed=1, block_dim=blocks)


@pytest.mark.parametrize("m,n,k", [(1, 4129, 8192 + 416), (16, 4100, 4128), (5, 300, 8192 + 96)])
def test_matmul_of_few_rows_keeps_nan_and_scales_at_their_ends(H, m, n, k):
    rng = np.random.default_rng(7)
    (ac, asc), (bc, bsc) = operand(rng, m, k), operand(rng, n, k)
    asc[:], bsc[:] = 0, 254
    asc[:, ::2], bsc[:, ::2] = 250, 4
    if m > 1:
        asc[m - 1, -1] = 255
    bsc[n - 1, -1] = bsc[7, -9] = bsc[40, 128] = 255
    want, size = O.matmul(O.decode(ac, asc), O.decode(bc, bsc), None, 1.0)
    dev = [torch.from_numpy(t).cuda() for t in (ac, asc, bc, bsc)]
    got = H.mxfp4_matmul_add_leakyrelu(dev[0], dev[1].view(torch.float8_e8m0fnu), dev[2], dev[3].view(torch.float8_e8m0fnu),
                                       alpha=1.0, out_dtype=torch.float32)
    lost = np.zeros((m, n), dtype=bool)
    lost[:, [7, 40, n - 1]] = True
    if m > 1:
        lost[m - 1] = True
    assert np.array_equal(np.isnan(got.cpu().numpy()), lost)
    if not lost.all():
        B.close(got[torch.from_numpy(~lost).cuda()], want[~lost], size[~lost], "f32", -(-k // 32) + 10)


@pytest.mark.parametrize("m,n,k,threads", [(4100, 4200, 1056, 512), (2100, 2100, 608, 256), (2200, 2050, 1280, 256)])
def test_matmul_on_tiles_keeps_nan_and_scales_at_their_ends(H, m, n, k, threads):
    """Both tiles of the kernel with persistent workgroups: 256 x 256 with eight wavefronts, 128 x 128 with four."""
    test_matmul_of_many_rows_keeps_nan_and_scales_at_their_ends(H, m, n, k)
    last = H.last_launch()
    assert last["kernel"] == "mxfp4_matmul_tiles" and last["threads"] == threads


# ---- more than 2^31 numbers ----

@pytest.mark.parametrize("axis", [1, 0])
def test_quantize_beyond_32_bit_offsets(H, axis):
    rows, k = 133000, 16416
    x = torch.randn((rows, k) if axis else (k, rows), device="cuda", dtype=torch.bfloat16)
    codes, scales, values = H.mxfp4_quantize(x, axis=axis, return_values=True)
    for part in (slice(0, 40), slice(130780, 130860), slice(rows - 40, rows)):   # 2^31 numbers are 130816 rows and some
        piece = x[part] if axis else x[:, part]
        want = O.quantize(B.numbers(piece) if axis else B.numbers(piece).T)
        assert np.array_equal(codes[part].cpu().numpy(), want[0])
        assert np.array_equal(scales[part].view(torch.uint8).cpu().numpy(), want[1])
        assert np.array_equal(B.numbers(values[part] if axis else values[:, part]), want[2] if axis else want[2].T)


def test_quantize_more_rows_than_one_launch_takes(H):
    rows = (1 << 29) + 70     # of one number: a launch indexes 2^31 groups of eight, four to a block
    x = torch.randint(-8, 9, (rows, 1), device="cuda", dtype=torch.int8).to(torch.float16)
    codes, scales = H.mxfp4_quantize(x)
    some = torch.cat([torch.arange(200), torch.arange((1 << 29) - 100, rows), torch.randint(0, rows, (5000,))]).cuda()
    want = O.quantize(B.numbers(x[some]))
    assert np.array_equal(codes[some].cpu().numpy(), want[0])
    assert np.array_equal(scales[some].view(torch.uint8).cpu().numpy(), want[1])


def test_matmul_beyond_32_bit_offsets(H):
    m, n, gen = 66000, 33000, torch.Generator(device="cuda").manual_seed(8)
    a, b = random_operand(m, 9, gen), random_operand(n, 9, gen)
    e8 = torch.float8_e8m0fnu
    got = H.mxfp4_matmul_add_leakyrelu(a[0], a[1].view(e8), b[0], b[1].view(e8), alpha=0.5)
    assert H.last_launch()["kernel"] == "mxfp4_matmul_tiles"
    for part in (slice(0, 20), slice(65060, 65090), slice(m - 20, m)):   # 2^31 numbers are 65075 rows and some
        want, size = O.matmul(decoded(a, part), decoded(b, slice(None)), None, 0.5)
        B.close(got[part], want, size, "bf16", 19)
