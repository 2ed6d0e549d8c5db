"""Block-scaled FP8 on the GPU against plain implementations in 64 bits.

Tolerances. Whole-number results (codes, scales, lists) are equal. A product's
sum differs from the 64-bit one in two ways.
* The FP8 matrix instruction adds eight neighbouring products at a time, each
  cut (towards zero) to a multiple of 2^(E - 13), E the largest sum of the two
  exponents among the eight (measured on the device with single products beside
  a large pair that cancels). The largest of them is at least 2^E and an exact
  multiple, so eight products are off by less than 7 * 2^-13 of the largest:
  C = 7 * 2^-13 * (sum over the eights of the largest magnitude).
* The eights of a block, and the blocks, are added in f32: at most G = (16 +
  blocks + 4) * 2^-23 times the sum of the terms' magnitudes, each addition
  taken as off by a whole unit in case it is cut, the scales' product and its
  fma two more.
bf16 then rounds by at most 2^-8 of the value. SwiGLU passes a gate error on by
at most 1.1 |u| (the largest slope of silu is below 1.1) and an up error by
|silu(g)|, and its own exp2, reciprocal and products add less than 2^-20 of the
value. Products of small whole numbers lose nothing in any of these steps and
are compared bit for bit.
"""
import pytest
import torch

import clef_i4

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
BF = torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, std, seed, dtype=BF):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * std).to(dtype)


def quantize64(x):
    """(codes as f64 values [rows][width], scales f64 [rows][kb]) of bf16 rows."""
    rows, width = x.shape
    v = torch.nn.functional.pad(x.cpu().double(), (0, -width % 128)).unflatten(1, (-1, 128))
    mag = v.abs()
    mag = torch.where(torch.isfinite(mag), mag, torch.zeros_like(mag))
    part, e = torch.frexp(mag.amax(-1).clamp(min=2.0 ** -118) / 448.0)
    e = torch.where(part == 0.5, e - 1, e)
    scale = torch.ldexp(torch.ones_like(part), e)
    q = (v / scale[..., None]).float()  # exact: a power of two
    q = torch.where(torch.isfinite(v), q, torch.full_like(q, float("nan")))
    return q.flatten(1)[:, :width].to(F8).double(), scale


def weight(matrices, n, k, kind, seed):
    """e4m3 codes [matrices][n][k] and scales as a checkpoint holds them."""
    codes = randn((matrices, n, k), 60.0, seed, torch.float32).clamp(-448, 448).to(F8)
    scales = torch.exp(torch.randn((matrices, -(-n // 128), -(-k // 128)), generator=gen(seed + 1), device="cuda") - 6)
    if kind == "e8m0":
        scales = torch.exp2(torch.round(torch.log2(scales))).to(torch.float8_e8m0fnu)
    return codes, scales


def weight64(codes, scales):
    m, n, k = codes.shape
    wide = scales.float().double().repeat_interleave(128, 1)[:, :n].repeat_interleave(128, 2)[:, :, :k]
    return codes.double() * wide


def rows64(a):
    return a.codes.double() * a.scales.double().repeat_interleave(128, 1)[:, : a.width]


def check(got, want, slack):
    """|got - want| <= 2^-8 |want| + slack (1 + 2^-8), elementwise."""
    got, want = got.double(), want.double()
    off = (got - want).abs() - (2.0 ** -8 * want.abs() + slack * (1 + 2.0 ** -8))
    assert torch.isfinite(got).all()
    assert (off <= 0).all(), f"{(off > 0).sum().item()} of {off.numel()} off, worst by {off.max().item()}"


def product64(x, w):
    """x [m][k] times w [n][k] in f64, and how far off an f32 sum by FP8
    matrix instructions may be (C + G above)."""
    m, k = x.shape
    n = w.shape[0]
    pad = (0, -k % 8)
    xe = torch.nn.functional.pad(x.abs().float(), pad).unflatten(1, (-1, 8))
    we = torch.nn.functional.pad(w.abs().float(), pad).unflatten(1, (-1, 8))
    largest = torch.zeros((m, n), device="cuda")
    step = max(1, (1 << 27) // (8 * max(m * n, 1)))
    for c in range(0, xe.shape[1], step):
        largest += (xe[:, None, c: c + step] * we[None, :, c: c + step]).amax(-1).sum(-1)
    mag = x.abs() @ w.abs().t()
    return x @ w.t(), 7 * 2.0 ** -13 * largest.double() * (1 + 2.0 ** -10) + (20 + -(-k // 128)) * 2.0 ** -23 * mag


def swiglu64(x, wg, wu):
    (g, dg), (u, du) = product64(x, wg), product64(x, wu)
    s = g * torch.sigmoid(g)
    h = s * u
    return h, 1.1 * dg * (u.abs() + du) + s.abs() * du + 2.0 ** -20 * h.abs()


# ---------------------------------------------------------------- quantizer

@pytest.mark.parametrize("rows,width", [(0, 128), (1, 8), (1, 2048), (2, 136), (3, 768), (7, 1000), (8, 128), (9, 4160),
                                        (37, 264), (130, 2176), (16, 32768)])
def test_prepare_matches_definition(rows, width):
    x = randn((rows, width), 3.0, rows * 7 + width)
    if rows:
        x[0, : width // 2] = 0
        x[-1] *= 1e-3
    a = clef_i4.prepare_f8(x)
    codes, scales = quantize64(x)
    assert torch.equal(a.codes.cpu().double(), codes)
    assert torch.equal(a.scales.cpu().double(), scales)
    blocks = -(-width // 128)
    exps = a.storage[rows * a.pitch:].view(-1)[: rows * (-(-blocks // 16) * 16)].view(rows, -(-blocks // 16) * 16)
    assert torch.equal(torch.ldexp(torch.ones((), dtype=torch.float64), exps[:, :blocks].cpu().int() - 127), scales)
    pad = a.storage[: rows * a.pitch].view(rows, a.pitch)[:, width:]
    assert (pad == 0).all()


def test_prepare_every_bf16_value():
    """Every bf16 bit pattern, in blocks whose largest finite magnitude is each
    binade's: normal, subnormal, zero, infinite, NaN."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF)
    x = torch.cat([bits.view(512, 128), bits.view(128, 512).t().contiguous()]).cuda().contiguous()
    a = clef_i4.prepare_f8(x[:, :128])
    codes, scales = quantize64(x[:, :128])
    assert torch.equal(a.scales.cpu().double(), scales)
    got = a.codes.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(codes))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(codes))


def test_prepare_edges_of_the_scale():
    """amax at, just below and just above 448 * 2^e, ties of e4m3, e4m3
    subnormals, blocks of nothing but zeros or non-finite values."""
    x = torch.zeros((8, 256), dtype=BF, device="cuda")
    x[0, 0], x[0, 1:5] = 448.0, torch.tensor([17.0, 19.0, 2.0 ** -9, 3 * 2.0 ** -10])
    x[1, 0], x[1, 1] = 450.0, 1.0
    x[2, 0], x[2, 1] = 446.0, 2.0 ** -10
    x[3, 5] = float("inf")
    x[4, 7], x[4, 9] = float("nan"), 5.0
    x[5, :128] = float("-inf")
    x[6, 0] = 3.3895313892515355e38
    x[7, 0] = 1e-40
    a = clef_i4.prepare_f8(x)
    codes, scales = quantize64(x)
    assert torch.equal(a.scales.cpu().double(), scales)
    got = a.codes.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(codes)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(codes))


def test_prepare_strided_rows_and_reused_buffer():
    wide = randn((19, 1024), 2.0, 5)
    buffer = torch.full((100000,), 0xAB, dtype=torch.uint8, device="cuda")
    for first, width in [(0, 512), (8, 520), (256, 768)]:
        x = wide[:, first: first + width]
        a = clef_i4.prepare_f8(x, out=buffer)
        b = clef_i4.prepare_f8(x.contiguous())
        n = b.storage.numel()
        assert torch.equal(a.storage[:n], b.storage) and (a.storage[n:] == 0xAB).all()


@pytest.mark.parametrize("rows", [(1 << 24) + 5, 1 << 27])
def test_prepare_more_rows_than_one_dimension_of_a_launch(rows):
    """2^27 rows, the most there may be: every row as in a call of its own."""
    some = randn((4096, 8), 1.0, 5)
    x = some.repeat(-(-rows // 4096), 1)[:rows]
    x[-3:] = some[7:10] * 3
    a = clef_i4.prepare_f8(x)
    del x
    want = clef_i4.prepare_f8(some)
    codes, scales = a.codes.view(torch.uint8), a.scales
    whole_parts = rows // 4096 - 1  # the last rows differ
    for first in range(0, whole_parts, 2048):
        count = min(2048, whole_parts - first)
        at = slice(first * 4096, (first + count) * 4096)
        assert (codes[at].view(count, 4096, 8) == want.codes.view(torch.uint8)).all()
        assert (scales[at].view(count, 4096) == want.scales[:, 0]).all()
    last = clef_i4.prepare_f8(some[7:10] * 3)
    assert torch.equal(codes[-3:], last.codes.view(torch.uint8)) and torch.equal(scales[-3:], last.scales)
    exps = a.storage[rows * 128: rows * 144].view(rows, 16)
    assert torch.equal(exps[-3:], last.storage[3 * 128: 3 * 144].view(3, 16))


def test_views_of_a_prepared_activation():
    """On the buffer's memory, which they keep; refused where they do not fit."""
    buffer = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    a = clef_i4.prepare_f8(randn((5, 264), 1.0, 1), out=buffer[4096:])
    codes, scales = a.codes, a.scales
    assert codes.shape == (5, 264) and codes.stride() == (384, 1) and codes.dtype == F8 and not codes.requires_grad
    assert scales.shape == (5, 3) and scales.stride() == (1, 5) and scales.dtype == torch.float32
    assert codes.data_ptr() == buffer.data_ptr() + 4096
    assert scales.data_ptr() == buffer.data_ptr() + 4096 + 5 * (384 + 16)
    at = 4096 + torch.arange(5, device="cuda")[:, None] * 384 + torch.arange(264, device="cuda")
    assert torch.equal(codes.view(torch.uint8), buffer[at])
    want = buffer[4096 + 5 * 400: 4096 + 5 * 400 + 60].view(torch.float32).view(3, 5).t()
    assert torch.equal(scales, want)
    kept = scales.clone()
    del buffer, a
    torch.full((1 << 16,), 0xAB, dtype=torch.uint8, device="cuda")
    assert torch.equal(scales, kept)
    for wrong in (clef_i4.PreparedF8(codes.view(torch.uint8), 5, 264), clef_i4.PreparedF8(torch.zeros(2000, dtype=torch.uint8, device="cuda"), 5, 264),
                  clef_i4.PreparedF8(torch.empty(4099, dtype=torch.uint8, device="cuda")[3:], 1, 1280)):
        with pytest.raises(ValueError):
            wrong.scales


# ---------------------------------------------------------------- weights

@pytest.mark.parametrize("matrices,n,k", [(1, 8, 8), (1, 128, 128), (2, 264, 392), (3, 40, 136)])
def test_weight_layout(matrices, n, k):
    """Tiled codes byte by byte, and the quantizer's rule on 128 x 128 blocks."""
    nb, kb = -(-n // 128), -(-k // 128)
    r, c = torch.meshgrid(torch.arange(nb * 128), torch.arange(kb * 128), indexing="ij")
    at = ((r // 128 * kb + c // 128) * 16384 + r % 128 // 16 * 2048 + c % 128 // 64 * 1024 +
          (c // 16 % 4 * 16 + r % 16) * 16 + c % 16)

    def tiled(codes):
        wide = torch.zeros((matrices, nb * 128, kb * 128), dtype=torch.uint8)
        wide[:, :n, :k] = codes.view(torch.uint8).cpu()
        out = torch.empty((matrices, nb * kb * 16384), dtype=torch.uint8)
        out[:, at.reshape(-1)] = wide.view(matrices, -1)
        return out.view(-1)

    codes, scales = weight(matrices, n, k, "f32", 3)
    w = clef_i4.f8_weight(codes, scales)
    assert torch.equal(w.codes.cpu(), tiled(codes)) and torch.equal(w.scales, scales)
    dense = randn((matrices, n, k), 0.05, 9)
    w = clef_i4.load_f8_weight(dense)
    blocks = torch.zeros((matrices, nb * 128, kb * 128))
    blocks[:, :n, :k] = dense.float().cpu()
    blocks = blocks.view(matrices, nb, 128, kb, 128).permute(0, 1, 3, 2, 4).reshape(-1, 128 * 128)
    part, e = torch.frexp(blocks.double().abs().amax(-1).clamp(min=2.0 ** -118) / 448.0)
    e = torch.where(part == 0.5, e - 1, e)
    scale = torch.ldexp(torch.ones_like(part), e)
    q = (blocks.double() / scale[:, None]).float().to(F8)
    q = q.view(matrices, nb, kb, 128, 128).permute(0, 1, 3, 2, 4).reshape(matrices, nb * 128, kb * 128)[:, :n, :k]
    assert torch.equal(w.codes.cpu(), tiled(q.contiguous()))
    assert torch.equal(w.scales.cpu().view(-1).double(), scale)


# ---------------------------------------------------------------- projections

SHAPES = [(1, 128, 128), (1, 4096, 1024), (3, 136, 8), (16, 1000, 264), (17, 264, 1352), (37, 4160, 1352),
          (64, 512, 128), (65, 2048, 520), (129, 1024, 2048), (257, 768, 1288), (300, 17408, 256),
          (20, 1200, 6848), (31, 392, 4104), (24, 520, 4000),
          # 128 x 128 tiles: one, two, three and nine blocks of k, and (two
          # at a time) 16, 17, 33, 40 and 43
          (700, 128, 4104), (700, 256, 4104), (700, 384, 4104), (1030, 1152, 1032),
          (700, 2048, 1544), (650, 2064, 2056), (140, 4224, 8200), (620, 5120, 2504),
          (600, 5384, 2504),
          # 256 x 256 tiles: one, two, three and eight blocks
          (2300, 128, 3608), (2300, 256, 3608), (2300, 392, 3608), (2060, 1000, 4104)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("kind,res", [("f32", False), ("e8m0", True)])
def test_project_matches_64_bits(m, k, n, kind, res):
    x = randn((m, k), 1.0, m + k)
    codes, scales = weight(1, n, k, kind, n)
    w = clef_i4.f8_weight(codes[0], scales[0])
    residual = randn((m, n), 30.0, 4) if res else None
    a = clef_i4.prepare_f8(x)
    want, slack = product64(rows64(a), weight64(codes, scales)[0])
    if res:
        want = want + residual.double()
        slack += 2.0 ** -23 * want.abs()
    out = torch.full((m + 1, n), 7.0, dtype=BF, device="cuda")
    got = clef_i4.project_f8(a, w, residual, out=out[:m])
    check(got, want, slack)
    assert (out[m:] == 7.0).all()
    again = clef_i4.project_quantized_f8(x, w, residual)
    check(again, want, slack)
    assert torch.equal(again, clef_i4.project_quantized_f8(x, w, residual))


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_project_gate_up_matches_64_bits(m, k, n, kind):
    x = randn((m, k), 1.0, m + k)
    (gc, gs), (uc, us) = weight(1, n, k, kind, n), weight(1, n, k, "e8m0", n + 2)
    gs = (gs.float() * 2.0 ** -6).to(gs.dtype)
    a = clef_i4.prepare_f8(x)
    want, slack = swiglu64(rows64(a), weight64(gc, gs)[0], weight64(uc, us)[0])
    gate, up = clef_i4.f8_weight(gc[0], gs[0]), clef_i4.f8_weight(uc[0], us[0])
    out = torch.full((m + 1, n), 7.0, dtype=BF, device="cuda")
    check(clef_i4.project_gate_up_f8(a, gate, up, out=out[:m]), want, slack)
    assert (out[m:] == 7.0).all()


# Shapes of the kernels that SHAPES does not reach, or not with more than 16 blocks
# of k (whose row scales are loaded anew): test_f8.py holds by the library's
# rule that every kernel is among these lists.
MORE = [(40, 264, 5000), (50, 2120, 4000), (130, 264, 5128), (250, 2184, 4072), (60, 2312, 8000), (20, 2312, 6848),
        (2300, 2312, 3608), (2060, 4232, 4104), (1030, 2312, 4104)]
MORE_GU = [(40, 264, 2504), (1000, 392, 6136), (1100, 128, 6136), (1100, 2312, 6136), (1000, 4232, 6136),
           (20, 2312, 3000), (60, 2312, 4000), (130, 2312, 2504)]


@pytest.mark.parametrize("m,k,n", MORE)
@pytest.mark.parametrize("kind,res", [("f32", False), ("e8m0", True)])
def test_project_matches_64_bits_on_every_kernel(m, k, n, kind, res):
    test_project_matches_64_bits(m, k, n, kind, res)


@pytest.mark.parametrize("m,k,n", MORE_GU)
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_project_gate_up_matches_64_bits_on_every_kernel(m, k, n, kind):
    test_project_gate_up_matches_64_bits(m, k, n, kind)


@pytest.mark.parametrize("m,k,n", MORE)
@pytest.mark.parametrize("kind", ["f32", "e8m0"])
def test_project_of_whole_numbers_is_exact_on_every_kernel(m, k, n, kind):
    test_project_of_whole_numbers_is_exact(m, k, n, kind)


def whole(shape, top, seed):
    return torch.randint(-top, top + 1, shape, generator=gen(seed), device="cuda").float()


@pytest.mark.parametrize("kind", ["f32", "e8m0"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_project_of_whole_numbers_is_exact(m, k, n, kind):
    """Whole numbers up to 15: products at most 2^8 apart, sums below 2^24, so
    nothing is lost before the rounding to bf16."""
    x = whole((m, k), 15, m + k)
    w = whole((n, k), 15, n)
    x[:, ::128] = 15.0
    nb, kb = -(-n // 128), -(-k // 128)
    scales = torch.exp2(torch.randint(-3, 1, (nb, kb), generator=gen(3), device="cuda").float())
    packed = clef_i4.f8_weight(w.to(F8), scales.to(torch.float8_e8m0fnu) if kind == "e8m0" else scales)
    assert packed.pow2 == (kind == "e8m0")
    res = whole((m, n), 255, 5)
    wide = w.double() * scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    want = x.double() @ wide.t()
    assert torch.equal(clef_i4.project_quantized_f8(x.to(BF), packed), want.float().to(BF))
    assert torch.equal(clef_i4.project_f8(clef_i4.prepare_f8(x.to(BF)), packed, res.to(BF)),
                       (want + res.double()).float().to(BF))


@pytest.mark.parametrize("m,k,n", [
    # one launch on 16 x 32, 32 x 32, 16 x 64 and 32 x 64 tiles: one row to many tiles of
    # rows, the last of them short; blocks that end inside; one pass to ten
    (1, 8, 8), (1, 16384, 256), (2, 20480, 264), (3, 12288, 520), (5, 8192, 136), (9, 4104, 1000), (10, 4096, 2048),
    (16, 2560, 32), (17, 2560, 392), (33, 128, 3992), (130, 1000, 520), (250, 512, 1096), (255, 1280, 1016),
    (513, 1032, 1000), (1000, 264, 520), (4095, 128, 64), (20, 1200, 6848), (31, 1280, 4104),
    # and rows or widths just past it
    (11, 4096, 2048), (16, 2568, 32), (3, 20480, 264), (64, 1400, 5000)])
@pytest.mark.parametrize("res", [False, True])
def test_project_quantizing_rows_itself_is_the_two_steps(m, k, n, res):
    """The same codes, scales and order of sums whether the rows are quantized
    by the product or before it, non-finite values and column ranges included."""
    wide = randn((m, k + 24), 1.0, m + k)
    wide *= torch.exp2(torch.randint(-140, 100, (m, 1), generator=gen(3), device="cuda").float()).to(BF)
    wide[m // 2, 8 + k // 2] = float("nan")
    wide[-1, 8 + k - 1] = float("-inf")
    codes, scales = weight(1, n, k, "f32", n)
    w = clef_i4.f8_weight(codes[0], scales[0])
    residual = randn((m, n), 3.0, 4) if res else None
    for x in (wide[:, 8: 8 + k], wide[:, 8: 8 + k].contiguous()):
        want = clef_i4.project_f8(clef_i4.prepare_f8(x), w, residual)
        out = torch.full((m + 1, n), 7.0, dtype=BF, device="cuda")
        clef_i4.project_quantized_f8(x, w, residual, out=out[:m])
        assert torch.equal(out[:m].view(torch.int16), want.view(torch.int16)) and (out[m:] == 7.0).all()
    if res:  # the output may be the residual itself
        clef_i4.project_quantized_f8(x, w, residual, out=residual)
        assert torch.equal(residual.view(torch.int16), want.view(torch.int16))


def test_project_loaded_weight_and_strided_rows():
    wide = randn((21, 800), 1.0, 1)
    x = wide[:, 16: 16 + 520]
    dense = randn((392, 520), 0.05, 2)
    w = clef_i4.load_f8_weight(dense)
    got = clef_i4.project_quantized_f8(x, w)
    assert torch.equal(got, clef_i4.project_quantized_f8(x.contiguous(), w))
    rel = (got.double() - x.double() @ dense.double().t()).norm() / (x.double() @ dense.double().t()).norm()
    assert rel < 2 * 2.0 ** -4  # each operand's codes are off by at most 2^-4


def test_project_non_finite_rows_and_values():
    """A row with NaN or infinity gives NaN in its own outputs only; saturated
    sums become infinite, SwiGLU's far tails its limits."""
    x = randn((40, 256), 1.0, 1)
    x[3, 5], x[17, 200] = float("nan"), float("inf")
    codes, scales = weight(1, 264, 256, "f32", 2)
    w = clef_i4.f8_weight(codes[0], scales[0])
    got = clef_i4.project_quantized_f8(x, w)
    bad = torch.isnan(got).all(1)
    assert bad.nonzero().flatten().tolist() == [3, 17] and torch.isfinite(got[~bad]).all()
    big = clef_i4.f8_weight(codes[0].float().abs().clamp(min=1).to(F8), torch.full_like(scales[0], 3e38))
    assert torch.isinf(clef_i4.project_quantized_f8(torch.ones_like(x), big)).all()
    eye = torch.zeros((8, 256), device="cuda")
    eye[:, 0] = torch.tensor([448.0, -448.0, 100, -100, 20, -20, 0, 1])
    ones = torch.zeros((8, 256), device="cuda")
    ones[:, 1] = 1.0
    one = torch.ones((1, 2), device="cuda")
    v = torch.zeros((1, 256), dtype=BF, device="cuda")
    v[0, :2] = 1.0
    a = clef_i4.prepare_f8(v)
    h = clef_i4.project_gate_up_f8(a, clef_i4.f8_weight(eye.to(F8), one), clef_i4.f8_weight(ones.to(F8), one))
    g = eye[:, 0].to(F8).double()
    want = g * torch.sigmoid(g)
    assert ((h[0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-30).all()


@pytest.mark.parametrize("m,k,n", [(5, 4104, 264), (64, 512, 2000), (700, 256, 4104), (620, 5120, 2504),
                                   (2300, 392, 3608)])
def test_project_onto_its_residual(m, k, n):
    x, residual = randn((m, k), 1.0, m), randn((m, n), 30.0, 4)
    codes, scales = weight(1, n, k, "f32", n)
    w = clef_i4.f8_weight(codes[0], scales[0])
    want = clef_i4.project_quantized_f8(x, w, residual)
    assert torch.equal(clef_i4.project_quantized_f8(x, w, residual, out=residual), want)


@pytest.mark.parametrize("m", [3, 300, 1030, 8200])
def test_project_scales_at_their_limits(m):
    """e8m0 from 2^-127 to 2^127 and NaN. One product of ones per output: exact."""
    k, n = 384, 1280
    exponents = torch.tensor([0, 1, 2, 120, 127, 140, 252, 253, 254, 255], dtype=torch.uint8, device="cuda")
    scales = exponents[:, None].expand(10, 3).contiguous().view(torch.float8_e8m0fnu)
    w = clef_i4.f8_weight(torch.ones((n, k), device="cuda").to(F8), scales)
    x = torch.zeros((m, k), dtype=BF, device="cuda")
    x[torch.arange(m, device="cuda"), torch.arange(m, device="cuda") * 37 % k] = 448.0  # a row scale of one
    got = clef_i4.project_quantized_f8(x, w).double()
    want = 448.0 * scales[:, 0].double().repeat_interleave(128)
    want = want.float().to(BF).double().expand(m, n)  # past the largest bf16: infinity
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


# one of each kernel: quantizing its rows itself, few rows, 128 x 128 tiles (two
# blocks of k at a time, one at a time), 256 x 256 tiles and their shape of half the rows
ENDS = [(5, 4104, 264), (64, 512, 2000), (700, 2064, 1544), (700, 256, 4104), (2300, 392, 3608), (2100, 392, 4104)]


def scaled_weight(matrices, n, k, kind, p, seed):
    """The same codes for every p, scales (of full mantissas in f32) times 2^p."""
    codes = randn((matrices, n, k), 60.0, seed, torch.float32).clamp(-448, 448).to(F8)
    scales = torch.rand((matrices, -(-n // 128), -(-k // 128)), generator=gen(seed + 1), device="cuda")
    scales = torch.exp2(-torch.floor(4 * scales)) if kind == "e8m0" else 0.6 + 0.9 * scales
    scales = torch.ldexp(scales * 2.0 ** -6, torch.tensor(p + 6, device="cuda"))
    return clef_i4.f8_weight(codes, scales.to(torch.float8_e8m0fnu) if kind == "e8m0" else scales)


def one(w):
    return clef_i4.F8Weight(w.codes, w.scales[0], w.rows, w.cols, 1, w.pow2)


@pytest.mark.parametrize("kind", ["f32", "e8m0"])
@pytest.mark.parametrize("p", [123, -118])
@pytest.mark.parametrize("m,k,n", ENDS)
def test_project_rows_at_the_ends_of_bf16(m, k, n, p, kind):
    """Rows times 2^p against weights times 2^-p: the same bits as without, since
    every step only multiplies by powers of two in between, while a row's scale
    times a sum of codes is far outside f32 (p = 123) or the weight's scale large."""
    x = whole((m, k), 15, m + k)
    far = torch.ldexp(x, torch.tensor(p, device="cuda")).to(BF)
    assert torch.equal(torch.ldexp(far.double(), torch.tensor(-p, device="cuda")).float(), x)
    x, res = x.to(BF), randn((m, n), 300.0, 3)
    near_w, far_w = (one(scaled_weight(1, n, k, kind, e, 5)) for e in (0, -p))
    want = clef_i4.project_quantized_f8(x, near_w, res)
    assert torch.isfinite(want).all()
    assert torch.equal(clef_i4.project_quantized_f8(far, far_w, res), want)
    near_u, far_u = (one(scaled_weight(1, n, k, kind, e, 7)) for e in (0, -p))
    want = clef_i4.project_gate_up_f8(clef_i4.prepare_f8(x), near_w, near_u)
    assert torch.isfinite(want).all()
    assert torch.equal(clef_i4.project_gate_up_f8(clef_i4.prepare_f8(far), far_w, far_u), want)


def same_bits(got, want64):
    """want64 has at most 24 bits: f32 holds it, and bf16 rounds it once."""
    assert torch.equal(want64.float().double(), want64)
    assert torch.equal(got.view(torch.int16), want64.float().to(BF).view(torch.int16))


@pytest.mark.parametrize("kind", ["f32", "e8m0"])
@pytest.mark.parametrize("m,k,n", ENDS)
def test_project_scales_whose_product_leaves_f32(m, k, n, kind):
    """Sums in f32's range whose scales multiply to more than its largest value
    (2^119 times 2^10: each block's largest value meets a weight of zero) or to
    less than its smallest normal (2^-126 times 2^-18). Whole numbers, blocks and
    rows chosen so that f32 loses nothing: bit for bit."""
    nb, kb = -(-n // 128), -(-k // 128)

    def product(x, w, scale):
        scales = torch.full((nb, kb), scale, device="cuda")
        packed = clef_i4.f8_weight(w.to(F8), scales.to(torch.float8_e8m0fnu) if kind == "e8m0" else scales)
        want = x.double() @ w.to(F8).double().t() * scales[0, 0].double()
        same_bits(clef_i4.project_quantized_f8(x.to(BF), packed), want)
        h = clef_i4.project_gate_up_f8(clef_i4.prepare_f8(x.to(BF)), packed, packed)
        assert not torch.isnan(h).any()

    # two of a block's values count, in an eight of their own: sums of few bits
    x = torch.zeros((m, k), device="cuda")
    x[:, 9::128] = whole((m, x[:, 9::128].shape[1]), 7, m) * 2.0 ** 110
    x[:, 13::128] = whole((m, x[:, 13::128].shape[1]), 7, m + 1) * 2.0 ** 110
    x[:, 0::128] = 2.0 ** 127
    w = whole((n, k), 7, n) * 2.0 ** -9
    w[:, 0::128] = 0
    product(x, w, 1.375 * 2.0 ** 10 if kind == "f32" else 2.0 ** 10)
    x = (7.5 + whole((m, k), 7, m) / 2).floor() * 2.0 ** -122  # 4 .. 11
    x[:, 0::128] = 15 * 2.0 ** -122
    w = 32 * (12 + whole((n, k), 2, n))  # 320 .. 448
    w = w * (torch.arange(k, device="cuda") % 128 < 8)
    product(x, w, 85 * 2.0 ** -24 if kind == "f32" else 2.0 ** -18)


@pytest.mark.parametrize("m,k,n", ENDS)
def test_project_blocks_with_a_scale_of_zero(m, k, n):
    """Such blocks add nothing, however large the rows; subnormal scales count."""
    codes = whole((n, k), 15, n).to(F8)
    x = whole((m, k), 15, m)
    x[:, ::128] = 15.0
    far = torch.ldexp(x, torch.tensor(123, device="cuda")).to(BF)
    scales = torch.full((-(-n // 128), -(-k // 128)), 85 * 2.0 ** -139, device="cuda")  # 2.66 * 2^-134
    scales[:, ::2] = 0
    scales[:, 2::4] = -0.0
    wide = scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    want = far.double() @ (codes.double() * wide).t()
    got = clef_i4.project_quantized_f8(far, clef_i4.f8_weight(codes, scales))
    # sums of whole numbers below 2^24 times 85 and a power of two
    slack = 2.0 ** -23 * (far.double().abs() @ (codes.double() * wide).abs().t())
    check(got, want, slack)


@pytest.mark.parametrize("m,k,n", ENDS)
def test_project_infinite_scale(m, k, n):
    """A block of infinite scale makes its sums infinite with their sign,
    whatever the number of blocks."""
    codes = torch.ones((n, k), device="cuda")
    codes[1::2] = -1.0
    scales = torch.ones((-(-n // 128), -(-k // 128)), device="cuda")
    scales[:, 0] = float("inf")
    w = clef_i4.f8_weight(codes.to(F8), scales)
    got = clef_i4.project_quantized_f8(torch.ones((m, k), dtype=BF, device="cuda"), w)
    assert torch.equal(got.float(), (codes[:, 0] * float("inf")).expand(m, n))


@pytest.mark.parametrize("kind", ["f32", "e8m0"])
@pytest.mark.parametrize("p", [123, -118])
@pytest.mark.parametrize("tokens,experts,k,n", [(20, 16, 264, 520), (900, 5, 256, 392), (3000, 4, 264, 3000)])
def test_experts_rows_at_the_ends_of_bf16(tokens, experts, k, n, p, kind):
    """The same over lists."""
    (offsets, slots), _ = lists(tokens, 1, experts, tokens)
    x = whole((tokens, k), 15, tokens + k)
    far = clef_i4.prepare_f8(torch.ldexp(x, torch.tensor(p, device="cuda")).to(BF))
    near = clef_i4.prepare_f8(x.to(BF))
    near_w, far_w = (scaled_weight(experts, n, k, kind, e, 5) for e in (0, -p))
    want = clef_i4.expert_f8(near, near_w, offsets, slots, 1, True)
    assert torch.isfinite(want).all()
    assert torch.equal(clef_i4.expert_f8(far, far_w, offsets, slots, 1, True), want)
    want = clef_i4.expert_gate_up_f8(near, near_w, near_w, offsets, slots, 1, True)
    assert torch.equal(clef_i4.expert_gate_up_f8(far, far_w, far_w, offsets, slots, 1, True), want)


def test_rows_and_slots_beyond_4_gib():
    """Activations whose bytes do not fit 32 bits (rows of a projection) or
    just do (an expert's), read at their end."""
    n, k, m = 8, 4224, 1048576
    codes, scales = weight(2, n, k, "f32", 3)
    last = randn((300, k), 1.0, 7)
    x = torch.zeros((m, k), dtype=BF, device="cuda")
    x[-300:] = last
    want, slack = product64(rows64(clef_i4.prepare_f8(last)), weight64(codes, scales)[0])
    w = clef_i4.f8_weight(codes[0], scales[0])
    got = clef_i4.project_quantized_f8(x, w)
    check(got[-300:], want, slack)
    assert not got[:-300].any()
    del got
    rows = 1000000  # 4.22e9 bytes of codes
    a = clef_i4.prepare_f8(x[-rows:])
    two = clef_i4.f8_weight(codes, scales)
    count = 250
    slots = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    slots[:count] = torch.arange(rows - count, rows, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 0, count], dtype=torch.int32, device="cuda")
    out = clef_i4.expert_f8(a, two, offsets, slots, 1, True, out=torch.full((rows, n), 7.0, dtype=BF, device="cuda"))
    want, slack = product64(rows64(clef_i4.prepare_f8(last[-count:])), weight64(codes, scales)[1])
    check(out[-count:], want, slack)
    assert (out[:-count] == 7.0).all()
    with pytest.raises(clef_i4.ClefError):
        clef_i4.expert_f8(clef_i4.prepare_f8(x), two, offsets, slots, 1, True)


@pytest.mark.parametrize("kind", ["f32", "e8m0"])
@pytest.mark.parametrize("m,n", [(3, 264), (60, 2000), (250, 4072), (700, 1544), (1030, 4104), (2100, 3608)])
def test_project_of_the_widest_rows(m, n, kind):
    """32768 columns: 256 blocks of k, whole numbers, exact."""
    test_project_of_whole_numbers_is_exact(m, 32768, n, kind)


@pytest.mark.parametrize("m", [1, 40, 700])
def test_project_onto_the_most_columns(m):
    """1048576 columns of which a few are looked at, exact."""
    n, k = 1 << 20, 136
    x, w = whole((m, k), 7, m).to(BF), whole((n, k), 15, 2)
    scales = torch.exp2(torch.randint(-3, 1, (n // 128, 2), generator=gen(3), device="cuda").float())
    packed = clef_i4.f8_weight(w.to(F8), scales)
    got = clef_i4.project_quantized_f8(x, packed)
    for at in (slice(0, 300), slice(n // 2 - 130, n // 2 + 130), slice(n - 300, n)):
        wide = scales.repeat_interleave(128, 0)[at].repeat_interleave(128, 1)[:, :k]
        want = x.double() @ (w[at] * wide).double().t()
        assert torch.equal(got[:, at], want.float().to(BF))


def test_outputs_beyond_4_gib():
    """150000 rows of 16384 columns (4.9e9 bytes), projected, onto themselves as
    the residual, and over lists whose slots run backwards."""
    m, n, k = 150000, 16384, 8
    x, w = whole((m, k), 7, 1).to(BF), whole((n, k), 7, 2).to(BF)
    packed = clef_i4.f8_weight(w.to(F8), torch.ones((n // 128, 1), device="cuda"))
    a = clef_i4.prepare_f8(x)
    got = clef_i4.project_f8(a, packed)

    def holds(out, factor):
        for at in range(0, m, 15000):
            want = x[at: at + 15000].float() @ w.float().t() * factor
            assert torch.equal(out[at: at + 15000], want.to(BF))

    holds(got, 1)
    holds(clef_i4.project_f8(a, packed, got, out=got), 2)
    two = clef_i4.f8_weight(torch.stack([w.to(F8)] * 2), torch.tensor([1.0, 2.0], device="cuda")[:, None, None].repeat(1, n // 128, 1))
    slots = torch.arange(m - 1, -1, -1, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, m, m], dtype=torch.int32, device="cuda")
    holds(clef_i4.expert_f8(a, two, offsets, slots, 1, True, out=got), 1)
    offsets = torch.tensor([0, 0, m], dtype=torch.int32, device="cuda")
    holds(clef_i4.expert_f8(a, two, offsets, slots, 1, True, out=got), 2)


@pytest.mark.parametrize("m,n", [(2100, 3608), (2100, 264), (9, 264)])
def test_rows_that_lie_far_apart(m, n):
    """Row pitches of 2^21 and more elements: addresses past 32 bits."""
    k = 264
    pitch = (1 << 21) if m > 9 else (1 << 29) + 8
    base = torch.empty((m - 1) * pitch + k, dtype=BF, device="cuda")
    x = base.as_strided((m, k), (pitch, 1))
    near = randn((m, k), 1.0, 3)
    x.copy_(near)
    w = clef_i4.load_f8_weight(randn((n, k), 0.1, 2))
    assert torch.equal(clef_i4.prepare_f8(x).storage, clef_i4.prepare_f8(near).storage)
    assert torch.equal(clef_i4.project_quantized_f8(x, w), clef_i4.project_quantized_f8(near, w))


def test_two_streams_at_once():
    """Calls in flight side by side have workspaces of their own."""
    w = clef_i4.load_f8_weight(randn((2048, 1032), 0.05, 8))
    inputs = [randn((700, 1032), 1.0, 20 + i) for i in range(6)] + [randn((9, 1032), 1.0, 40 + i) for i in range(6)]
    want = [clef_i4.project_quantized_f8(x, w) for x in inputs]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for i, x in enumerate(inputs):
        with torch.cuda.stream(streams[i % 3]):
            got.append(clef_i4.project_quantized_f8(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------- lists

@pytest.mark.parametrize("tokens,topk,experts", [(0, 8, 128), (1, 1, 1), (1, 8, 128), (2, 3, 8), (63, 1, 2), (235, 8, 128),
                                                 (256, 8, 60), (257, 8, 128), (700, 6, 300), (5000, 8, 128),
                                                 (3000, 4, 1024), (70000, 8, 64)])
def test_group_slots_is_a_stable_sort(tokens, topk, experts):
    g = gen(tokens + experts)
    ids = torch.randint(0, experts, (tokens, topk), generator=g, device="cuda")
    if tokens > 60:
        ids[tokens // 2:] = torch.randint(0, max(1, experts // 9), (tokens - tokens // 2, topk), generator=g, device="cuda")
    ids = ids.float()
    if tokens > 2:
        ids[1, 0], ids[2, -1], ids[tokens // 3, 0] = -1.0, float(experts), float("nan")
    routes = torch.cat([ids, torch.rand((tokens, topk), generator=g, device="cuda")], 1)
    offsets, slots = clef_i4.omni_group_slots(routes, experts)
    flat = ids.reshape(-1).cpu()
    valid = (flat > -1) & (flat < experts)
    key = torch.where(valid, torch.nan_to_num(flat), torch.tensor(float(experts))).long()
    order = torch.argsort(key, stable=True)[: int(valid.sum())]
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    assert offsets.cpu().tolist() == [0] + counts.cumsum(0).tolist()
    assert torch.equal(slots[: order.numel()].cpu().long(), order)
    assert (slots[order.numel():] == -1).all()


@pytest.mark.parametrize("tokens,topk,experts", [(1 << 20, 16, 1024), (1 << 20, 16, 3), ((1 << 17) - 1, 128, 128)])
def test_group_slots_of_the_most_routes(tokens, topk, experts):
    """16777216 slots: chunks of many batches."""
    ids = torch.randint(-1, experts + 1, (tokens, topk), generator=gen(experts), device="cuda")
    offsets, slots = clef_i4.omni_group_slots(torch.cat([ids, ids], 1).float(), experts)
    flat = ids.reshape(-1)
    key, order = torch.sort(torch.where(flat < 0, experts, flat), stable=True)
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    count = int(counts.sum())
    assert offsets.tolist() == [0] + counts.cumsum(0).tolist()
    assert torch.equal(slots[:count].long(), order[:count]) and (slots[count:] == -1).all()


# ---------------------------------------------------------------- experts

def lists(tokens, topk, experts, seed, empty=()):
    """Distinct random experts per token, none of `empty`."""
    score = torch.rand((tokens, experts), generator=gen(seed), device="cuda")
    score += 2.0 * torch.rand(experts, generator=gen(seed + 1), device="cuda")
    for e in empty:
        score[:, e] = -1
    ids = score.topk(topk, 1)[1].float()
    return clef_i4.omni_group_slots(torch.cat([ids, torch.ones_like(ids)], 1), experts), ids.long()


EXPERTS = [(1, 8, 128, 256, 136), (1, 1, 1, 8, 8), (5, 2, 4, 384, 200), (37, 8, 60, 264, 136), (235, 4, 16, 768, 264),
           (300, 1, 3, 1152, 128), (900, 2, 5, 256, 392), (2100, 8, 24, 136, 128), (900, 1, 200, 264, 136),
           (3000, 1, 4, 264, 3000), (3000, 1, 4, 128, 3000)]


@pytest.mark.parametrize("kind", ["f32", "e8m0"])
@pytest.mark.parametrize("tokens,topk,experts,k,n", EXPERTS)
def test_experts_match_64_bits(tokens, topk, experts, k, n, kind):
    empty = (0, experts - 1) if experts > topk + 2 else ()
    (offsets, slots), ids = lists(tokens, topk, experts, tokens + n, empty)
    total = tokens * topk
    codes, scales = weight(experts, n, k, kind, 5)
    uc, us = weight(experts, n, k, "e8m0", 7)
    w, up = clef_i4.f8_weight(codes, scales), clef_i4.f8_weight(uc, us)
    gate = clef_i4.f8_weight(codes, (scales.float() * 2.0 ** -6).to(scales.dtype))
    w64, u64 = weight64(codes, scales), weight64(uc, us)
    a = clef_i4.prepare_f8(randn((tokens, k), 1.0, 1))
    routed = clef_i4.prepare_f8(randn((total, k), 1.0, 2))
    x, xr = rows64(a), rows64(routed)
    want = torch.empty((total, n), dtype=torch.float64, device="cuda")
    want_t, want_h = torch.empty_like(want), torch.empty_like(want)
    slack, slack_t, slack_h = torch.empty_like(want), torch.empty_like(want), torch.empty_like(want)
    flat = ids.reshape(-1)
    for e in range(experts):
        s = (flat == e).nonzero().flatten()
        want[s], slack[s] = product64(xr[s], w64[e])
        want_t[s], slack_t[s] = product64(x[s // topk], w64[e])
        want_h[s], slack_h[s] = swiglu64(x[s // topk], w64[e] * 2.0 ** -6, u64[e])
    out = torch.full((total + 1, n), 7.0, dtype=BF, device="cuda")
    check(clef_i4.expert_f8(routed, w, offsets, slots, topk, True, out=out[:total]), want, slack)
    assert (out[total] == 7.0).all()
    check(clef_i4.expert_f8(a, w, offsets, slots, topk, False), want_t, slack_t)
    h = clef_i4.expert_gate_up_f8(a, gate, up, offsets, slots, topk, out=out[:total])
    check(h, want_h, slack_h)
    assert (out[total] == 7.0).all()
    assert torch.equal(h, clef_i4.expert_gate_up_f8(a, gate, up, offsets, slots, topk))
    # rows sorted by expert, lists without slots
    order = slots.long()
    sorted_a = clef_i4.prepare_f8(randn((total, k), 1.0, 2)[order])
    got = clef_i4.expert_f8(sorted_a, w, offsets, None, 1, True)
    check(got, want[order], slack[order])


MORE_EXPERTS = [(1, 8, 128, 2312, 136), (37, 8, 60, 2312, 136), (900, 1, 200, 2312, 136), (900, 2, 5, 2312, 392),
                (3000, 1, 4, 2312, 3000)]


@pytest.mark.parametrize("kind", ["f32", "e8m0"])
@pytest.mark.parametrize("tokens,topk,experts,k,n", MORE_EXPERTS)
def test_experts_match_64_bits_with_more_than_16_blocks(tokens, topk, experts, k, n, kind):
    test_experts_match_64_bits(tokens, topk, experts, k, n, kind)


@pytest.mark.parametrize("n", [136, 2600, 4104])
def test_experts_leave_unlisted_rows_and_odd_lists(n):
    """Rows behind the last list, slots outside the table and offsets outside
    it or descending: nothing else is written."""
    k, experts, total = 256, 4, 70
    codes, scales = weight(experts, n, k, "f32", 5)
    w = clef_i4.f8_weight(codes, scales)
    a = clef_i4.prepare_f8(randn((total, k), 1.0, 2))
    w64, x = weight64(codes, scales), rows64(a)

    def run(offsets, slots):
        out = torch.full((total, n), 7.0, dtype=BF, device="cuda")
        clef_i4.expert_f8(a, w, torch.tensor(offsets, dtype=torch.int32, device="cuda"),
                          None if slots is None else torch.tensor(slots, dtype=torch.int32, device="cuda"), 1, True, out)
        return out

    def same(out, rows):
        left = torch.ones(total, dtype=torch.bool)
        for row, e in rows.items():
            want, slack = product64(x[row: row + 1], w64[e])
            check(out[row: row + 1], want, slack)
            left[row] = False
        assert (out[left.cuda()] == 7.0).all()

    same(run([0, 3, 3, 20, 41], None), {**{r: 0 for r in range(3)}, **{r: 2 for r in range(3, 20)},
                                        **{r: 3 for r in range(20, 41)}})
    same(run([0, 0, 0, 0, 0], None), {})
    slots = list(range(total))
    slots[1], slots[2], slots[5] = -1, total, 1 << 30
    same(run([0, 4, 4, 4, 8], slots), {0: 0, 3: 0, 4: 3, 6: 3, 7: 3})
    same(run([-5, 2, 2, 60, 1 << 30], None), {**{r: 0 for r in range(2)}, **{r: 2 for r in range(2, 60)},
                                              **{r: 3 for r in range(60, total)}})
    same(run([10, 5, 8, 8, 8], None), {r: 1 for r in range(5, 8)})


@pytest.mark.parametrize("tokens,experts", [(12, 1024), (5000, 1024), (20000, 130)])
def test_experts_past_the_first_128(tokens, experts):
    """Whole numbers, each expert's weight its number: exact."""
    k, n = 136, 8
    ids = torch.randint(0, experts, (tokens, 1), generator=gen(experts), device="cuda")
    ids[0], ids[-1] = 128, experts - 1
    offsets, slots = clef_i4.omni_group_slots(torch.cat([ids, torch.ones_like(ids)], 1).float(), experts)
    codes = torch.zeros((experts, n, k), device="cuda")
    codes[:, :, 0] = (torch.arange(experts, device="cuda") // 64)[:, None]
    codes[:, :, 130] = (torch.arange(experts, device="cuda") % 64 // 4)[:, None]
    w = clef_i4.f8_weight(codes.to(F8), torch.ones((experts, 1, 2), device="cuda"))
    assert torch.equal(codes.to(F8).float(), codes)
    x = torch.zeros((tokens, k), dtype=BF, device="cuda")
    x[:, 0], x[:, 130] = 16.0, 1.0
    got = clef_i4.expert_f8(clef_i4.prepare_f8(x), w, offsets, slots, 1, True)
    assert torch.equal(got.float(), (ids // 64 * 16 + ids % 64 // 4).float().expand(tokens, n).to(BF).float())


def test_experts_of_the_most_slots():
    """16777216 slots of 8 experts, each expert's weight its number: exact."""
    total, experts, k, n = 1 << 24, 8, 8, 8
    bounds = [0, 5, 5, 1 << 20, (1 << 20) + 129, 1 << 22, 1 << 23, total - 1, total]
    offsets = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    values = torch.arange(1, experts + 1, device="cuda").float()
    w = clef_i4.f8_weight(values[:, None, None].expand(experts, n, k).to(F8), torch.ones((experts, 1, 1), device="cuda"))
    x = torch.zeros((total, k), dtype=BF, device="cuda")
    x[:, 5] = (torch.arange(total, device="cuda") % 15 + 1).to(BF)
    got = clef_i4.expert_f8(clef_i4.prepare_f8(x), w, offsets, None, 1, True)
    counts = torch.tensor(bounds, device="cuda").diff()
    want = x[:, 5].float() * torch.repeat_interleave(values, counts)
    assert (got.float() == want[:, None]).all()


@pytest.mark.parametrize("n", [136, 2048])
def test_experts_overlapping_lists_stay_inside(n):
    """Lists that name places twice make more tiles than sound ones can: a row
    is one of its experts', nothing else is written."""
    k, total = 128, 1000
    w = clef_i4.f8_weight(torch.ones((6, n, k), device="cuda").to(F8),
                          torch.arange(1, 7, device="cuda").float()[:, None, None].expand(6, -(-n // 128), 1).contiguous())
    x = torch.zeros((total, k), dtype=BF, device="cuda")
    x[:, 3] = 1.0
    offsets = torch.tensor([0, total, 0, total, 0, total, 1], dtype=torch.int32, device="cuda")
    out = torch.full((total + 1, n), 7.0, dtype=BF, device="cuda")
    clef_i4.expert_f8(clef_i4.prepare_f8(x), w, offsets, None, 1, True, out=out[:total])
    assert torch.isin(out, torch.tensor([1.0, 3.0, 5.0, 7.0], dtype=BF, device="cuda")).all() and (out[total] == 7.0).all()


# ---------------------------------------------------------------- together

def moe(experts=16, d=264, f=136, topk=4):
    gate, up = (clef_i4.load_f8_weight(randn((experts, f, d), 0.05, s)) for s in (1, 2))
    down = clef_i4.load_f8_weight(randn((experts, d, f), 0.05, 3))
    return clef_i4.MoeLayerF8(gate, up, down, topk), (gate, up, down)


@pytest.mark.parametrize("tokens", [1, 30, 500])
def test_moe_layer_is_its_steps(tokens):
    """The layer equals its operators called one by one, and stays within the
    FP8 roundings of the block in 64 bits."""
    layer, (gate, up, down) = moe()
    x, logits = randn((tokens, 264), 1.0, 4), randn((tokens, 16), 1.0, 5)
    got = layer(x, logits)
    routes = clef_i4.omni_route(logits, 4)
    offsets, slots = clef_i4.omni_group_slots(routes, 16)
    a = clef_i4.prepare_f8(x)
    h = clef_i4.expert_gate_up_f8(a, gate, up, offsets, slots, 4)
    values = clef_i4.expert_f8(clef_i4.prepare_f8(h), down, offsets, slots, 4, True)
    assert torch.equal(got, clef_i4.omni_combine(values, routes))
    wg, wu = (randn((16, 136, 264), 0.05, s).double() for s in (1, 2))
    wd = randn((16, 264, 136), 0.05, 3).double()
    want = torch.zeros((tokens, 264), dtype=torch.float64, device="cuda")
    for r in range(4):
        e = routes[:, r].long()
        g = torch.bmm(wg[e], x.double()[:, :, None])[..., 0]
        u = torch.bmm(wu[e], x.double()[:, :, None])[..., 0]
        y = torch.bmm(wd[e], (g * torch.sigmoid(g) * u)[:, :, None])[..., 0]
        want += routes[:, 4 + r, None].double() * y
    # five codes on the way (x, gate, up, h, down), each off by at most 2^-4
    assert (got.double() - want).norm() / want.norm() < 5 * 2.0 ** -4


@pytest.mark.parametrize("tokens", [1, 40, 600])
def test_moe_layer_rows_without_experts(tokens):
    """Tokens whose logits leave fewer experts than topk, or none (all masked,
    NaN): the other tokens' outputs are as without them."""
    layer, _ = moe()
    x, logits = randn((tokens + 4, 264), 1.0, 4), randn((tokens + 4, 16), 1.0, 5)
    want = layer(x, logits)
    at = [0, tokens // 2, tokens + 1, tokens + 3]
    logits[at[0]] = float("nan")
    logits[at[1]] = float("-inf")
    logits[at[2], 2:] = torch.finfo(BF).min
    logits[at[3], 1:] = float("-inf")
    kept = [i for i in range(tokens + 4) if i not in at]
    torch.full((tokens * 16 + 64, 264), float("nan"), dtype=BF, device="cuda")  # what the intermediates may find
    got = layer(x, logits)
    assert got.shape == want.shape and torch.equal(got[kept], want[kept])


@pytest.mark.parametrize("tokens", [3, 200])
def test_graph_replays_match_eager(tokens):
    """A captured layer and projections, replayed between eager calls on other
    inputs; two graphs, each with its own intermediates."""
    layer, _ = moe()
    w = clef_i4.load_f8_weight(randn((520, 264), 0.05, 8))
    gate, up = (clef_i4.load_f8_weight(randn((392, 264), 0.05, s)) for s in (9, 10))
    inputs = [(randn((tokens, 264), 1.0, 20 + i), randn((tokens, 16), 1.0, 30 + i)) for i in range(4)]

    def step(x, logits):
        y = layer(x, logits)
        return y, clef_i4.project_quantized_f8(y, w), clef_i4.project_gate_up_f8(clef_i4.prepare_f8(y), gate, up)

    want = [step(*i) for i in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step(*inputs[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, want[1]))
    graphs = []
    for _ in range(2):
        x, logits = (t.clone() for t in inputs[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(x, logits)
        graphs.append((graph, x, logits, out))
    for i in (0, 1, 2, 3, 1, 0):
        for g, (graph, x, logits, out) in enumerate(graphs):
            j = (i + g) % 4
            x.copy_(inputs[j][0])
            logits.copy_(inputs[j][1])
            graph.replay()
        step(*inputs[(i + 2) % 4])
        torch.cuda.synchronize()
        for g, (_, _, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(i + g) % 4]))


def test_binding_refusals():
    x = randn((4, 256), 1.0, 1)
    a = clef_i4.prepare_f8(x)
    w = clef_i4.load_f8_weight(randn((128, 256), 0.1, 2))
    two = clef_i4.load_f8_weight(randn((2, 128, 256), 0.1, 2))
    other = clef_i4.load_f8_weight(randn((128, 264), 0.1, 2))
    offsets = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    refused = [
        lambda: clef_i4.prepare_f8(x.float()),
        lambda: clef_i4.prepare_f8(x[:, :252]),
        lambda: clef_i4.prepare_f8(x[:, 4:252].t()),
        lambda: clef_i4.prepare_f8(x[:, 4:252]),  # rows that do not start on 16 bytes
        lambda: clef_i4.prepare_f8(x, out=torch.empty(10, dtype=torch.uint8, device="cuda")),
        lambda: clef_i4.prepare_f8(x.cpu()),
        lambda: clef_i4.load_f8_weight(x.float()),
        lambda: clef_i4.f8_weight(x, torch.ones((1, 2), device="cuda")),
        lambda: clef_i4.f8_weight(x.to(F8), torch.ones((2, 1), device="cuda")),
        lambda: clef_i4.project_f8(a, other),
        lambda: clef_i4.project_f8(a, two),
        lambda: clef_i4.project_f8(a, w, residual=randn((4, 120), 1.0, 1)),
        lambda: clef_i4.project_f8(a, w, out=torch.empty((4, 128), device="cuda")),
        lambda: clef_i4.project_quantized_f8(x, two),
        lambda: clef_i4.project_gate_up_f8(a, w, other),
        lambda: clef_i4.expert_f8(a, two, offsets[:2], None, 1, True),
        lambda: clef_i4.expert_f8(a, two, offsets.long(), None, 1, True),
        lambda: clef_i4.expert_f8(a, two, offsets, torch.zeros(9, dtype=torch.int32, device="cuda"), 2, False),
        lambda: clef_i4.expert_f8(a, two, offsets.cpu(), None, 1, True),
        lambda: clef_i4.omni_group_slots(torch.zeros((4, 3), device="cuda")),
        lambda: clef_i4.omni_group_slots(torch.zeros((4, 4), device="cuda"), 2000),
    ]
    for i, f in enumerate(refused):
        with pytest.raises(clef_i4.ClefError):
            f()
            pytest.fail(f"refusal {i} did not raise")


def test_weights_smaller_than_they_say_are_refused():
    x = randn((4, 256), 1.0, 1)
    a = clef_i4.prepare_f8(x)
    two = clef_i4.load_f8_weight(randn((2, 136, 256), 0.1, 2))
    w = one(clef_i4.F8Weight(two.codes[: 4 * 16384], two.scales, 136, 256))
    clef_i4.project_f8(a, w)
    offsets = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    F8Weight = clef_i4.F8Weight
    for codes, scales in ((w.codes[:-16], w.scales), (w.codes, w.scales[:1]), (w.codes.cpu(), w.scales),
                          (w.codes, w.scales.cpu()), (w.codes.view(torch.int32), w.scales), (w.codes, w.scales.bfloat16())):
        bad = F8Weight(codes, scales, 136, 256)
        for f in (lambda: clef_i4.project_f8(a, bad), lambda: clef_i4.project_quantized_f8(x, bad),
                  lambda: clef_i4.project_gate_up_f8(a, bad, w), lambda: clef_i4.project_gate_up_f8(a, w, bad)):
            with pytest.raises(clef_i4.ClefError):
                f()
    for bad in (F8Weight(two.codes, two.scales, 136, 264, 2), F8Weight(two.codes, two.scales, 264, 256, 2)):
        with pytest.raises(clef_i4.ClefError):
            clef_i4.expert_f8(clef_i4.prepare_f8(randn((4, bad.cols), 1.0, 1)), bad, offsets, None, 1, True)
    three = F8Weight(two.codes, two.scales, 136, 256, 3)
    for f in (lambda: clef_i4.expert_f8(a, three, torch.zeros(4, dtype=torch.int32, device="cuda"), None, 1, True),
              lambda: clef_i4.expert_gate_up_f8(a, two, F8Weight(two.codes, two.scales[:1], 136, 256, 2), offsets, None, 1, True)):
        with pytest.raises(clef_i4.ClefError):
            f()


@pytest.mark.parametrize("m,n", [(4, 128), (700, 2056)])
def test_outputs_over_their_inputs_are_refused(m, n):
    """Views of one buffer, as a caller saving memory would pass them."""
    k = 256
    x, w = randn((m, k), 1.0, 1), clef_i4.load_f8_weight(randn((n, k), 0.1, 2))
    a = clef_i4.prepare_f8(x)
    kept, both = x.clone(), randn((m + 1, n), 1.0, 3)
    for f in (lambda: clef_i4.prepare_f8(x[: m // 2], out=x.view(torch.uint8).view(-1)),
              lambda: clef_i4.project_f8(a, w, both[:m], out=both[1:]),
              lambda: clef_i4.project_quantized_f8(x, w, both[1:], out=both[:m])):
        with pytest.raises(clef_i4.ClefError):
            f()
    assert torch.equal(x, kept)
    want = clef_i4.project_f8(a, w, both[:m])
    assert torch.equal(clef_i4.project_f8(a, w, both[:m], out=both[:m]), want)
