"""Products with bf16 activations on the GPU against plain implementations in
64 bits.

Tolerances. Products of two bf16 values are exact in f32. A sum of k of them is
off by at most G = (k + 16) * 2^-23 times the sum of their magnitudes: each
addition taken as off by a whole unit in case it is cut, the bias' and the join
of partial sums among the 16. An activation passes an error of its argument on
by its largest slope (1.13 for both GELUs, 1.1 for SiLU, 1 for ReLU, 0.25 for
the logistic function) and adds its own: the argument z of its exponential is
rounded (at most 2^-22 |z| in the exponent, so of the value), and sixteen more
roundings and one-ulp functions are below 2^-19: E = (|z| + 8) 2^-21 of the
value, 2^-100 where the value underflows. Adding the residual and multiplying by
the up sum round once each, and bf16 by at most 2^-8 of the value, f32 by none
that is not counted. Sums of small whole numbers lose nothing and are compared
bit for bit.
"""
import math

import pytest
import torch

import clef_i4

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
BF = torch.bfloat16
F32 = torch.float32
NAN, INF = float("nan"), float("inf")
SLOPE = {None: 1.0, "relu": 1.0, "gelu": 1.13, "gelu_tanh": 1.13, "silu": 1.1, "sigmoid": 0.25}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, std, seed, dtype=BF):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * std).to(dtype)


def whole(shape, most, seed, dtype=BF):
    return torch.randint(-most, most + 1, shape, generator=gen(seed), device="cuda").to(dtype)


def act64(v, name):
    """(value, argument of the exponential) in 64 bits."""
    if name == "relu":
        return v.clamp(min=0.0), torch.zeros_like(v)
    if name == "gelu":
        # (erfc: 1 + erf loses its last 2^-53, which counts below v = -8)
        return 0.5 * v * torch.erfc(-v * math.sqrt(0.5)), v * v / 2
    if name == "gelu_tanh":
        z = math.sqrt(8.0 / math.pi) * (v + 0.044715 * v ** 3)
        return v * torch.sigmoid(z), z
    if name == "silu":
        return v * torch.sigmoid(v), v
    if name == "sigmoid":
        return torch.sigmoid(v), v
    return v, torch.zeros_like(v)


def activated(v, slack, name):
    """act of sums that are off by `slack`: (value, how far off)."""
    y, z = act64(v, name)
    own = (z.abs() + 8) * 2.0 ** -21 * y.abs() + 2.0 ** -100 if name not in (None, "relu") else 0.0
    return y, SLOPE[name] * slack + own


def sums64(x, w, bias):
    """x @ w.T + bias in 64 bits, and G."""
    xd, wd = x.double(), w.double()
    y, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return y, (x.shape[1] + 16) * 2.0 ** -23 * mag


def check(got, want, slack):
    half = 2.0 ** -8 if got.dtype == BF else 2.0 ** -24
    off = (got.double() - want).abs() - (half * want.abs() + slack * (1 + half))
    assert torch.isfinite(got).all()
    assert (off <= 0).all(), f"{(off > 0).sum().item()} of {off.numel()} off, worst by {off.max().item()}"


def linear64(x, w, bias=None, act=None, residual=None):
    y, slack = activated(*sums64(x, w, bias), act)
    if residual is not None:
        y = y + residual.double()
        slack = slack + 2.0 ** -23 * y.abs()
    return y, slack


def gate_up64(x, wg, wu, act="silu", bg=None, bu=None):
    a, da = activated(*sums64(x, wg, bg), act)
    u, du = sums64(x, wu, bu)
    h = a * u
    return h, da * (u.abs() + du) + a.abs() * du + 2.0 ** -22 * h.abs()


def make_bias(n, kind, seed):
    return None if kind is None else randn((n,), 1.0, seed, BF if kind == "bf16" else F32)


# ---------------------------------------------------------------- linear

# rows, k, columns: one of each, ends of every tile, k that ends inside a step, k
# and n not multiples of 8, many rows and columns
SHAPES = [(1, 1, 1), (1, 8, 8), (1, 2048, 128), (2, 7, 3), (3, 64, 17), (15, 72, 40), (16, 128, 64), (17, 136, 65),
          (31, 1000, 333), (37, 4160, 1353), (63, 200, 63), (64, 512, 256), (65, 520, 257), (127, 1001, 130),
          (128, 264, 384), (129, 2048, 127), (200, 4096, 520), (255, 328, 511), (257, 1024, 1000), (300, 776, 2056),
          (520, 1032, 1288)]
EPILOGUES = [(None, None, False, BF), ("bf16", "relu", False, BF), ("f32", None, True, BF), (None, "gelu", True, F32),
             ("f32", "gelu_tanh", False, BF), ("bf16", "silu", True, BF), (None, "sigmoid", False, F32)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("bias,act,res,dtype", EPILOGUES)
def test_linear_matches_64_bits(m, k, n, bias, act, res, dtype):
    seed = m * 31 + k * 7 + n
    x, w, b = randn((m, k), 1.0, seed), randn((n, k), k ** -0.5, seed + 1), make_bias(n, bias, seed + 2)
    r = randn((m, n), 1.0, seed + 3) if res else None
    got = clef_i4.linear(x, w, bias=b, activation=act, residual=r, dtype=dtype)
    assert got.dtype == dtype and got.shape == (m, n)
    check(got, *linear64(x, w, b, act, r))


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_of_whole_numbers_is_exact(m, k, n):
    """|sums| <= 3 k + 9 < 2^24: exact in f32 in any order."""
    x, w = whole((m, k), 3, m + k), whole((n, k), 1, n + k)
    b, r = whole((n,), 4, 5), whole((m, n), 5, 6)
    got = clef_i4.linear(x, w, bias=b, residual=r, dtype=F32)
    assert torch.equal(got.double(), x.double() @ w.double().t() + b.double() + r.double())
    assert torch.equal(clef_i4.linear(x, w, bias=b, residual=r), got.to(BF))


# rows, k, columns, the kernel that the rule picks and the parts of k: every kernel
# with ends inside its tile and its last step (projections, gate/up)
KERNELS = ([(3, 776, 41, "8x8", 1), (9, 8200, 45, "8x8", 1), (7, 648, 2563, "8x16", 1), (11, 72, 45, "16x16", 1),
            (11, 72, 4099, "16x32", 1), (29, 72, 2981, "32x16", 1), (29, 72, 4141, "32x32", 1), (45, 72, 5483, "64x32", 1),
            (51, 648, 8203, "64x64", 1), (525, 136, 6003, "128x128", 1), (9, 6152, 8097, "128x128", 4),
            (133, 2056, 8203, "128x128x2", 1), (131, 8200, 3001, "128x128x2", 4), (403, 1032, 8203, "128x256", 1),
            (131, 8200, 4107, "128x256", 6), (1303, 264, 6001, "256x256", 1), (401, 4104, 8203, "256x256", 3)],
           [(5, 392, 43, "8x16", 1), (9, 4104, 43, "8x16", 1), (11, 72, 45, "16x32", 1), (29, 72, 2059, "32x32", 1),
            (45, 72, 2837, "64x32", 1), (51, 648, 4155, "64x64", 1), (141, 72, 9001, "128x128", 1), (9, 6472, 3991, "128x128", 4),
            (131, 2056, 4107, "128x128x2", 1), (131, 4104, 3001, "128x128x2", 2), (133, 1032, 8203, "128x256", 1),
            (131, 4104, 4107, "128x256", 3), (403, 264, 8203, "256x256", 1), (131, 4104, 8203, "256x256", 3)])
# the same for rows that start at any even byte
ODD_KERNELS = ([(3, 349, 43, "8x8"), (7, 913, 2059, "8x16"), (11, 73, 45, "16x16"), (11, 73, 4099, "16x32"), (17, 77, 3269, "32x16"),
                (29, 85, 4115, "32x32"), (45, 89, 4099, "64x32"), (500, 1001, 2059, "any"), (901, 137, 5003, "any128")],
               [(5, 77, 43, "8x16"), (11, 81, 45, "8x16"), (17, 81, 41, "16x32"), (29, 89, 2067, "32x32"), (45, 85, 2075, "64x32"),
                (300, 1001, 2059, "any"), (901, 137, 3003, "any128")])


# weights of 16 MiB and more that one row of tiles reads
ONCE = ([(1, 16880, 499, "8x8"), (1, 3368, 2497, "8x16"), (9, 3256, 2579, "16x16"), (1, 152, 55189, "16x32"),
         (17, 1160, 7235, "32x32"), (33, 1984, 4277, "64x32"), (33, 592, 14251, "64x64")],
        [(1, 6504, 645, "8x16"), (1, 640, 6555, "16x32"), (17, 824, 5141, "32x32"), (33, 2088, 2065, "64x32"),
         (33, 608, 6903, "64x64")])


@pytest.mark.parametrize("m,k,n", [c[:3] for c in KERNELS[0] + ODD_KERNELS[0] + ONCE[0]])
def test_linear_on_every_kernel(m, k, n):
    seed = m * 17 + k * 3 + n
    x, w, r = randn((m, k), 1.0, seed), randn((n, k), k ** -0.5, seed + 1), randn((m, n), 1.0, seed + 3)
    for bias, act, res, dtype in EPILOGUES:
        b = make_bias(n, bias, seed + 2)
        got = clef_i4.linear(x, w, bias=b, activation=act, residual=r if res else None, dtype=dtype)
        check(got, *linear64(x, w, b, act, r if res else None))
    again = r.clone()
    clef_i4.linear(x, w, residual=again, out=again)
    assert torch.equal(again, clef_i4.linear(x, w, residual=r))
    x, w, b = whole((m, k), 3, m + k), whole((n, k), 1, n + k), whole((n,), 4, 5)
    want = x.double() @ w.double().t() + b.double() + r.double()
    assert torch.equal(clef_i4.linear(x, w, bias=b, residual=r), want.float().to(BF))


@pytest.mark.parametrize("m,k,n", [c[:3] for c in KERNELS[0] + ODD_KERNELS[0]])
def test_linear_non_finite_values_on_every_kernel(m, k, n):
    """A NaN row and a NaN weight row touch their row and column alone; the columns
    behind the last one and the rows behind the last stay as they were."""
    x, w = randn((m, k), 1.0, 1), randn((n, k), 0.05, 2)
    clean = clef_i4.linear(x, w)
    wide = torch.full((m + 1, n + 5), 7.0, dtype=BF, device="cuda")
    x[m // 2, k - 1], w[n - 2, 0] = NAN, INF
    clef_i4.linear(x, w, out=wide[:m, :n])
    keep = torch.ones((m, n), dtype=torch.bool, device="cuda")
    keep[m // 2], keep[:, n - 2] = False, False
    assert torch.equal(wide[:m, :n][keep], clean[keep])
    assert torch.isnan(wide[m // 2, :n]).all() and not torch.isfinite(wide[:m, n - 2]).any()
    assert (wide[m] == 7.0).all() and (wide[:, n:] == 7.0).all()


@pytest.mark.parametrize("m,k,n", [c[:3] for c in KERNELS[1] + ODD_KERNELS[1] + ONCE[1]])
def test_gate_up_on_every_kernel(m, k, n):
    seed = m * 11 + k * 3 + n
    x, wg, wu = randn((m, k), 1.0, seed), randn((n, k), k ** -0.5, seed + 1), randn((n, k), k ** -0.5, seed + 2)
    bg, bu = randn((n,), 1.0, seed + 3), randn((n,), 1.0, seed + 4)
    check(clef_i4.linear_gate_up(x, wg, wu), *gate_up64(x, wg, wu))
    check(clef_i4.linear_gate_up(x, wg, wu, activation="gelu", gate_bias=bg, up_bias=bu), *gate_up64(x, wg, wu, "gelu", bg, bu))
    x = (whole((m, k), 1, m + k).float() * (torch.arange(k, device="cuda") % 8 == 0)).to(BF)
    wg, wu = whole((n, k), 1, 1), whole((n, k), 1, 2)
    want = (x.double() @ wg.double().t()) * (x.double() @ wu.double().t())
    assert torch.equal(clef_i4.linear_gate_up(x, wg, wu, activation=None), want.float().to(BF))


@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_tanh", "silu", "sigmoid"])
def test_activations_over_their_range(act):
    """Every bf16 value between -2^7 and 2^7 through a weight of one."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF).cuda()
    x = bits[torch.isfinite(bits) & (bits.abs() <= 128)].view(-1, 1)
    w = torch.ones((1, 1), dtype=BF, device="cuda")
    y, z = act64(x.double(), act)
    exact = act in (None, "relu")
    got = clef_i4.linear(x, w, activation=act, dtype=F32).double()
    tiny = 2.0 ** -100 if not exact else 2.0 ** -126  # values below f32's normal range may become zero
    off = (got - y).abs() - ((0.0 if exact else (z.abs() + 8) * 2.0 ** -21) * y.abs() + tiny)
    assert (off <= 0).all(), off.max()


def test_activations_keep_nan_and_limits():
    x = torch.tensor([[NAN], [INF], [-INF], [0.0]], dtype=BF, device="cuda")
    w = torch.ones((1, 1), dtype=BF, device="cuda")
    relu = clef_i4.linear(x, w, activation="relu").flatten().tolist()
    assert math.isnan(relu[0]) and relu[1:] == [INF, 0.0, 0.0]
    sig = clef_i4.linear(x, w, activation="sigmoid").flatten().tolist()
    assert math.isnan(sig[0]) and sig[1:] == [1.0, 0.0, 0.5]
    for act in ("gelu", "gelu_tanh", "silu"):
        y = clef_i4.linear(x, w, activation=act).flatten().tolist()
        assert math.isnan(y[0]) and y[1] == INF and y[3] == 0.0


STRIDED = [(5, 128, 64, 136, 0), (37, 1000, 333, 1007, 3), (70, 512, 96, 1024, 8), (130, 264, 200, 272, 8), (64, 63, 65, 129, 1),
           (300, 520, 260, 1048, 16)]


@pytest.mark.parametrize("m,k,n,pitch,skip", STRIDED)
def test_linear_of_column_ranges(m, k, n, pitch, skip):
    """Operands that are columns of wider rows of NaN, an output among columns
    that stay as they were, rows of it behind the last one too."""
    def part(rows, cols, wide, at, seed):
        t = torch.full((rows, wide), NAN, dtype=BF, device="cuda")
        t[:, at:at + cols] = randn((rows, cols), 1.0, seed)
        return t[:, at:at + cols]

    x, w = part(m, k, pitch, skip, 1), part(n, k, pitch + 8, skip, 2)
    r = part(m, n, n + 24, skip, 3)
    b = randn((n,), 1.0, 4)
    wide = torch.full((m + 3, n + 40), 7.0, dtype=BF, device="cuda")
    out = wide[:m, skip:skip + n]
    assert clef_i4.linear(x, w, bias=b, residual=r, out=out) is out
    check(out, *linear64(x, w, b, None, r))
    whole_rows = clef_i4.linear(x.contiguous(), w.contiguous(), bias=b, residual=r.contiguous())
    check(whole_rows, *linear64(x, w, b, None, r))
    if skip % 8 == 0 and pitch % 8 == 0 and k % 8 == 0:  # rows of another alignment run another kernel: other bits
        assert torch.equal(out, whole_rows)
    rest = wide.clone()
    rest[:m, skip:skip + n] = 7.0
    assert (rest == 7.0).all()


@pytest.mark.parametrize("k", [*range(1, 20), 63, 64, 65, 127, 129, 513, 1023, 1025])
@pytest.mark.parametrize("skip", [0, 1, 2, 8])
def test_linear_of_every_width_and_start(k, skip):
    """Whole numbers in rows that start at any even byte, between NaN columns, on the
    kernels for few rows, some and many."""
    for m, n in ((1, 9), (8, 40), (23, 70), (150, 200), (500, 600)):
        x, w = whole((m, k + skip), 3, m + k), whole((n, k + skip + 1), 1, n + k)
        x[:, :skip], w[:, :skip], w[:, k + skip:] = NAN, NAN, NAN
        x, w = x[:, skip:], w[:, skip:k + skip]
        assert torch.equal(clef_i4.linear(x, w, dtype=F32).double(), x.double() @ w.double().t()), (m, n)


def pitched(which):
    """(rows, k, columns, first column, columns behind) of operands in wider rows, on
    every kernel: rows on multiples of 16 bytes as in KERNELS and ONCE, and at any
    even byte."""
    aligned = [c[:3] for c in KERNELS[which] + ONCE[which]]
    return [(*c, 8, 16) for c in aligned] + [(*c, 3, 6) for c in aligned[::3]] + [(*c[:3], 5, 2) for c in ODD_KERNELS[which]]


def columns(t, skip, behind):
    """t as a column range of wider rows of NaN."""
    wide = torch.full((t.shape[0], skip + t.shape[1] + behind), NAN, dtype=t.dtype, device="cuda")
    wide[:, skip:skip + t.shape[1]] = t
    return wide[:, skip:skip + t.shape[1]]


class Guarded:
    """An output among rows and columns that stay as they are."""

    def __init__(self, m, n, skip, behind, dtype=BF):
        self.wide = torch.full((m + 3, skip + n + behind), 7.0, dtype=dtype, device="cuda")
        self.out = self.wide[1:m + 1, skip:skip + n]

    def result(self):
        got = self.out.clone()
        self.out.fill_(7.0)
        assert (self.wide == 7.0).all()
        return got


@pytest.mark.parametrize("m,k,n,skip,behind", pitched(0))
def test_linear_of_column_ranges_on_every_kernel(m, k, n, skip, behind):
    seed = m * 19 + k * 5 + n + skip
    x, w, r = randn((m, k), 1.0, seed), randn((n, k), k ** -0.5, seed + 1), randn((m, n), 1.0, seed + 2)
    b = randn((n,), 1.0, seed + 3)
    cx, cw, cr = columns(x, skip, behind), columns(w, skip, behind + 8), columns(r, skip, behind + 1)
    # whole rows run the same kernel where both start on 16 bytes, or neither
    alike = (skip % 8 == 0) == (k % 8 == 0)
    for act, res, dtype in ((None, True, BF), ("silu", False, BF), ("gelu", True, F32), (None, False, F32)):
        to = Guarded(m, n, skip, behind, dtype)
        clef_i4.linear(cx, cw, bias=b, activation=act, residual=cr if res else None, out=to.out)
        got = to.result()
        check(got, *linear64(x, w, b, act, r if res else None))
        if alike:
            assert torch.equal(got, clef_i4.linear(x, w, bias=b, activation=act, residual=r if res else None, dtype=dtype))
    to = Guarded(m, n, skip, behind)
    to.out.copy_(r)
    clef_i4.linear(cx, cw, residual=to.out, out=to.out)
    got = to.result()
    check(got, *linear64(x, w, residual=r))


@pytest.mark.parametrize("m,k,n,skip,behind", pitched(1))
def test_gate_up_of_column_ranges_on_every_kernel(m, k, n, skip, behind):
    seed = m * 23 + k * 5 + n + skip
    x, wg, wu = randn((m, k), 1.0, seed), randn((n, k), k ** -0.5, seed + 1), randn((n, k), k ** -0.5, seed + 2)
    bg, bu = randn((n,), 1.0, seed + 3, F32), randn((n,), 1.0, seed + 4, F32)
    cx = columns(x, skip, behind)
    gap = 8 - k % 8 if skip % 8 == 0 else 2
    both = columns(torch.cat((wg, torch.full((n, gap), NAN, dtype=BF, device="cuda"), wu), 1), skip, behind)  # side by side
    cg, cu = both[:, :k], both[:, k + gap:]
    for act, biases in (("silu", (None, None)), ("gelu_tanh", (bg, bu))):
        to = Guarded(m, n, skip, behind)
        clef_i4.linear_gate_up(cx, cg, cu, activation=act, gate_bias=biases[0], up_bias=biases[1], out=to.out)
        got = to.result()
        check(got, *gate_up64(x, wg, wu, act, *biases))
        if (skip % 8 == 0) == (k % 8 == 0):
            assert torch.equal(got, clef_i4.linear_gate_up(x, wg, wu, act, *biases))


@pytest.mark.parametrize("k,pitch,skip", [(8192, 8200, 1), (8192, 8201, 0), (8191, 8191, 0)])
def test_rows_off_16_bytes_take_no_workspace(k, pitch, skip):
    """A caller of the C entries with rows that do not lie on 16 bytes hands none over."""
    m, n, lib, _n = 200, 2048, clef_i4.lib(), clef_i4._n
    x = randn((m * pitch + 8,), 1.0, 1).as_strided((m, k), (pitch, 1), skip)
    w, up = randn((n, k), k ** -0.5, 2), randn((n, k), k ** -0.5, 3)
    out = torch.empty((m, n), dtype=BF, device="cuda")
    _n.launch(_n.clef_linear, x.data_ptr(), m, k, pitch, w, n, k, None, 0, 0, None, n, out, 0, n, None, 0)
    assert torch.equal(out, clef_i4.linear(x, w))
    check(out, *linear64(x, w))
    _n.launch(_n.clef_linear_gate_up, x.data_ptr(), m, k, pitch, w, up, n, k, None, None, 0, 4, out, n, None, 0)
    check(out, *gate_up64(x, w, up))


def test_one_row_onto_its_residual_whatever_the_pitches():
    """One row has no second that the pitches could place elsewhere."""
    k, n, _n = 256, 64, clef_i4._n
    x, w, r = randn((1, k), 1.0, 1), randn((n, k), 0.05, 2), randn((1, n), 1.0, 3)
    want = clef_i4.linear(x, w, residual=r)
    _n.launch(_n.clef_linear, x, 1, k, k, w, n, k, None, 0, 0, r, n, r, 0, n + 64, None, 0)
    assert torch.equal(r, want)
    with pytest.raises(clef_i4.ClefError, match="overlaps"):  # two do
        both = randn((3, n + 64), 1.0, 4)
        _n.launch(_n.clef_linear, x.expand(2, k).contiguous(), 2, k, k, w, n, k, None, 0, 0, both, n, both, 0, n + 64, None, 0)


@pytest.mark.parametrize("m,k,n", [(1, 256, 64), (37, 520, 129), (300, 1024, 512)])
def test_linear_onto_its_residual_and_beside_its_rows(m, k, n):
    x, w, r = randn((m, k), 1.0, 1), randn((n, k), 0.05, 2), randn((m, n), 1.0, 3)
    want = clef_i4.linear(x, w, activation="silu", residual=r)
    again = r.clone()
    clef_i4.linear(x, w, activation="silu", residual=again, out=again)
    assert torch.equal(again, want)
    both = torch.zeros((m, k + n), dtype=BF, device="cuda")  # x and the output in rows of one buffer
    both[:, :k] = x
    if m > 1:
        clef_i4.linear(both[:, :k], w, activation="silu", residual=r, out=both[:, k:])
        check(both[:, k:].contiguous(), *linear64(x, w, None, "silu", r))
        assert torch.equal(both[:, :k], x)
        if (k + n) % 8 == 0:  # rows of another alignment run another kernel: other bits
            assert torch.equal(both[:, k:], want)


@pytest.mark.parametrize("m,k,n", [(3, 256, 64), (40, 520, 129), (300, 1032, 512)])
def test_linear_non_finite_rows_and_columns_stay_alone(m, k, n):
    x, w = randn((m, k), 1.0, 1), randn((n, k), 0.05, 2)
    clean = clef_i4.linear(x, w)
    x[1, k - 1], w[n - 2, 0] = INF, NAN
    got = clef_i4.linear(x, w)
    assert not torch.isfinite(got[1]).any() and torch.isnan(got[:, n - 2]).all()
    keep = torch.ones((m, n), dtype=torch.bool, device="cuda")
    keep[1] = False
    keep[:, n - 2] = False
    assert torch.equal(got[keep], clean[keep])


def test_linear_of_no_rows():
    x, w = torch.empty((0, 64), dtype=BF, device="cuda"), randn((8, 64), 1.0, 1)
    assert clef_i4.linear(x, w).shape == (0, 8)
    assert clef_i4.linear_gate_up(x, w, w).shape == (0, 8)
    moe, _ = layer(8, 64, 128, 2, "f32", 1, router=w)
    assert moe.decode(x).shape == (0, 64)
    assert moe.decode(x, torch.empty((0, 8), device="cuda"), residual=x).shape == (0, 64)


@pytest.mark.parametrize("m,k", [(5, 72), (130, 1032), (300, 77)])
def test_one_tensor_as_several_operands(m, k):
    """x is its own weight and its own residual; gate and up are x too."""
    x = randn((m, max(m, k)), 0.1, m)[:, :k]
    check(clef_i4.linear(x, x, x[0, :1].expand(m).contiguous(), "silu"), *linear64(x, x, x[0, :1].expand(m), "silu"))
    check(clef_i4.linear_gate_up(x, x, x), *gate_up64(x, x, x))
    w = randn((k, k), 0.1, k)
    check(clef_i4.linear(x, w, residual=x), *linear64(x, w, residual=x))


def test_linear_rows_far_apart():
    """Rows more than 2^31 elements into their buffers."""
    m, k, n, pitch = 5, 64, 40, 1 << 29
    rows, w = randn((m, k), 1.0, 1), randn((n, k), 0.1, 2)
    buf = torch.empty(4 * pitch + k + n, dtype=BF, device="cuda")
    x = buf.as_strided((m, k), (pitch, 1))
    x.copy_(rows)
    out = buf.as_strided((m, n), (pitch, 1), k)  # beside the rows
    clef_i4.linear(x, w, out=out)
    check(out.contiguous(), *linear64(rows, w))
    far = buf.as_strided((n, k), (pitch // 16, 1))
    far.copy_(w)
    for m in (1, 5):
        check(clef_i4.linear(rows[:m], far), *linear64(rows[:m], w))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_linear_output_beyond_4_gib(dtype):
    m, k, n = (1 << 20), 8, 2056
    x, w = whole((m, k), 3, 1), whole((n, k), 2, 2)
    got = clef_i4.linear(x, w, dtype=dtype)
    for at in (0, m // 2 - 5, m - 300):
        assert torch.equal(got[at:at + 300].double(), x[at:at + 300].double() @ w.double().t())


# ---------------------------------------------------------------- gate/up

@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("act,bias", [("silu", None), ("gelu_tanh", "bf16"), ("gelu", "f32"), ("sigmoid", None), (None, None)])
def test_gate_up_matches_64_bits(m, k, n, act, bias):
    seed = m * 13 + k * 5 + n
    x = randn((m, k), 1.0, seed)
    wg, wu = randn((n, k), k ** -0.5, seed + 1), randn((n, k), k ** -0.5, seed + 2)
    bg, bu = make_bias(n, bias, seed + 3), make_bias(n, bias, seed + 4)
    got = clef_i4.linear_gate_up(x, wg, wu, activation=act, gate_bias=bg, up_bias=bu)
    check(got, *gate_up64(x, wg, wu, act, bg, bu))


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_gate_up_of_whole_numbers_is_exact(m, k, n):
    """Sums below 2^12 (entries 0 or 1 in 1 of 8 places at most), products below 2^24."""
    x = (whole((m, k), 1, m + k).float() * (torch.arange(k, device="cuda") % 8 == 0)).to(BF)
    wg, wu = whole((n, k), 1, 1), whole((n, k), 1, 2)
    assert k <= 8 * 4095
    want = (x.double() @ wg.double().t()) * (x.double() @ wu.double().t())
    assert torch.equal(clef_i4.linear_gate_up(x, wg, wu, activation=None), want.float().to(BF))


@pytest.mark.parametrize("m,k,n,pitch,skip", STRIDED)
def test_gate_up_of_column_ranges_and_one_bias(m, k, n, pitch, skip):
    x = torch.full((m, pitch), NAN, dtype=BF, device="cuda")
    x[:, skip:skip + k] = randn((m, k), 1.0, 1)
    x = x[:, skip:skip + k]
    both = torch.full((2 * n, pitch), NAN, dtype=BF, device="cuda")  # gate and up as rows of one weight
    both[:, skip:skip + k] = randn((2 * n, k), 0.05, 2)
    wg, wu = both[:n, skip:skip + k], both[n:, skip:skip + k]
    b = randn((n,), 1.0, 3)
    wide = torch.full((m + 2, n + 40), 7.0, dtype=BF, device="cuda")
    out = wide[:m, skip:skip + n]
    clef_i4.linear_gate_up(x, wg, wu, up_bias=b, out=out)
    check(out, *gate_up64(x, wg, wu, "silu", None, b))
    rest = wide.clone()
    rest[:m, skip:skip + n] = 7.0
    assert (rest == 7.0).all()
    check(clef_i4.linear_gate_up(x, wg, wu, gate_bias=b), *gate_up64(x, wg, wu, "silu", b, None))


# ---------------------------------------------------------------- a MoE layer of few tokens

def expert_weight(matrices, n, k, kind, seed):
    codes = randn((matrices, n, k), 60.0, seed, F32).clamp(-448, 448).to(F8)
    scales = torch.exp(torch.randn((matrices, -(-n // 128), -(-k // 128)), generator=gen(seed + 1), device="cuda") * 0.5 - 7)
    if kind == "e8m0":
        scales = torch.exp2(torch.round(torch.log2(scales))).to(torch.float8_e8m0fnu)
    return codes, scales


def weight64(codes, scales):
    m, n, k = codes.shape
    return codes.double() * scales.float().double().repeat_interleave(128, 1)[:, :n].repeat_interleave(128, 2)[:, :, :k]


def chosen(logits, topk):
    """Per token [(expert, probability)] in 64 bits."""
    out = []
    for row in logits.double().tolist():
        row = [-INF if math.isnan(v) else v for v in row]
        best = sorted(range(len(row)), key=lambda e: (-row[e], e))[:topk]
        best = [e for e in best if row[e] > -INF]
        p = [1.0 if row[e] == row[best[0]] else math.exp(row[e] - row[best[0]]) for e in best]
        out.append([(e, v / sum(p)) for e, v in zip(best, p)])
    return out


def moe64(x, logits, gate, up, down, topk, residual=None):
    """The definition in 64 bits, and how far off f32 sums may be: gate and up by
    (hidden + 16) 2^-23 of their magnitudes, SiLU as above, probabilities by
    (topk + 40) 2^-23 (differences of logits up to 40, the sum, a division), h
    held to 2^-16, the sum over the experts by (topk * inter * 2 + 32) 2^-23."""
    y = torch.zeros((x.shape[0], down.shape[1]), dtype=torch.float64, device="cuda")
    slack = torch.zeros_like(y)
    for t, names in enumerate(chosen(logits, topk)):
        for e, p in names:
            a, da = activated(*sums64(x[t:t + 1], gate[e], None), "silu")
            u, du = sums64(x[t:t + 1], up[e], None)
            h = a * u * p
            dh = p * (da * (u.abs() + du) + a.abs() * du) + h.abs() * (2.0 ** -16 + (topk + 44) * 2.0 ** -23)
            y[t] += (h @ down[e].t())[0]
            slack[t] += (dh @ down[e].abs().t())[0]
            slack[t] += (topk * down.shape[2] * 2 + 32) * 2.0 ** -23 * (h.abs() @ down[e].abs().t())[0]
    if residual is not None:
        y += residual.double()
        slack += 2.0 ** -23 * y.abs()
    return y, slack


def layer(experts, hidden, inter, topk, kind, seed, router=None):
    raw = [expert_weight(experts, r, c, kind, seed + 10 * i)
           for i, (r, c) in enumerate(((inter, hidden), (inter, hidden), (hidden, inter)))]
    packed = [clef_i4.f8_weight(*w) for w in raw]
    return clef_i4.MoeLayerF8(*packed, topk=topk, router=router), [weight64(*w) for w in raw]


MOE = [(1, 2048, 768, 128, 8, "e8m0"), (1, 8, 8, 1, 1, "f32"), (2, 136, 72, 3, 2, "f32"), (3, 256, 128, 8, 1, "f32"),
       (5, 1000, 520, 60, 4, "f32"), (7, 128, 2048, 8, 6, "e8m0"), (8, 512, 256, 128, 8, "e8m0"), (13, 4096, 264, 32, 2, "f32"),
       (2, 5000, 136, 8, 2, "f32"), (12, 4232, 72, 12, 3, "e8m0"), (2, 32768, 8, 4, 2, "f32"), (11, 32768, 16, 4, 2, "f32"),
       (3, 8, 32768, 4, 2, "f32"), (9, 256, 2048, 32, 4, "e8m0"), (16, 200, 1032, 24, 8, "f32"), (16, 264, 136, 16, 16, "f32"), (16, 640, 384, 128, 8, "f32"), (16, 128, 8, 128, 128, "f32"), (4, 256, 136, 65, 3, "e8m0")]


@pytest.mark.parametrize("t,hidden,inter,experts,topk,kind", MOE)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_decode_matches_64_bits(t, hidden, inter, experts, topk, kind, dtype):
    moe, w = layer(experts, hidden, inter, topk, kind, t + hidden)
    x, logits, r = randn((t, hidden), 1.0, 1), randn((t, experts), 2.0, 2, dtype), randn((t, hidden), 1.0, 3)
    check(moe.decode(x, logits), *moe64(x, logits, *w, topk))
    check(moe.decode(x, logits, residual=r), *moe64(x, logits, *w, topk, r))


# 64 MB of experts' weights and more (named by evenly chosen routes), every width of hidden
@pytest.mark.parametrize("t,hidden,inter,experts,topk", [(16, 200, 5128, 32, 4), (16, 504, 2056, 32, 4), (16, 1000, 1032, 32, 4),
                                                         (2, 2048, 776, 32, 8), (5, 4096, 520, 16, 4), (5, 5000, 1032, 6, 2)])
def test_decode_of_large_weights(t, hidden, inter, experts, topk):
    assert experts * (1 - (1 - topk / experts) ** t) * 3 * hidden * inter >= 64e6
    moe, w = layer(experts, hidden, inter, topk, "f32", t + hidden)
    x, logits, r = randn((t, hidden), 1.0, 1), randn((t, experts), 2.0, 2, F32), randn((t, hidden), 1.0, 3)
    check(moe.decode(x, logits, residual=r), *moe64(x, logits, *w, topk, r))


def test_decode_of_whole_numbers_is_exact():
    """One expert per token (p = 1), gate sums of 2^15 and more (silu(g) = g in
    f32: exp(-g) is 0), up sums that make h a multiple of 2^15 with 16 bits."""
    t, hidden, inter, experts = 9, 256, 128, 5
    gate = torch.zeros((experts, inter, hidden), device="cuda")
    gate[:, :, 0] = 256.0
    up = whole((experts, inter, hidden), 1, 1, F32)
    down = whole((experts, hidden, inter), 3, 2, F32)
    one = [torch.ones((experts, -(-r // 128), -(-c // 128)), device="cuda") for r, c in ((inter, hidden), (hidden, inter))]
    moe = clef_i4.MoeLayerF8(clef_i4.f8_weight(gate.to(F8), one[0]), clef_i4.f8_weight(up.to(F8), one[0]),
                             clef_i4.f8_weight(down.to(F8), one[1]), topk=1)
    x = whole((t, hidden), 1, 3)
    x[:, 0] = 128.0
    logits = randn((t, experts), 1.0, 4, F32)
    e = logits.argmax(1)
    u = (up.double()[e] * x.double()[:, None]).sum(-1)
    assert (u.abs() < 2 ** 16).all()
    want = (down.double()[e] * (u * 2.0 ** 15)[:, None]).sum(-1)
    assert torch.equal(moe.decode(x, logits), want.float().to(BF))


@pytest.mark.parametrize("t,experts,hidden,inter", [(1, 4, 96, 128), (8, 3, 264, 136), (5, 8, 1000, 72), (16, 1, 48, 520),
                                                    (9, 8, 256, 2048), (16, 12, 520, 1032)])
def test_decode_keeps_every_bit_of_h(t, experts, hidden, inter):
    """One expert per token (p = 1) and sums of whole numbers from 2^10 to 2^11, where
    silu(g) = g in f32, so h = g u needs up to 22 bits. An output is the difference of
    two columns of h, g u - (g - 1)(u + 1) = u + 1 - g, at most 100: every sum on the
    way is a whole number below 2^23, the output itself a bf16."""
    rng = torch.Generator().manual_seed(t * 1000 + inter)
    triples, pairs = hidden // 3, inter // 2
    g = torch.randint(1100, 1900, (experts, pairs, triples), generator=rng)
    want = torch.randint(-100, 101, (experts, pairs, triples), generator=rng)
    u = want + g - 1

    def digits(a, b):
        """Weights [experts][inter][hidden]: columns of h 2 i with sums a, 2 i + 1 with b, of three hexadecimal digits."""
        v = torch.stack((a, b), 2).reshape(experts, inter, triples)
        w = torch.zeros((experts, inter, hidden))
        for at, shift in enumerate((8, 4, 0)):
            w[:, :, at:3 * triples:3] = (v >> shift & 15).float()
        return w

    order = torch.randperm(inter, generator=rng)  # the columns of a pair lie anywhere
    pair = torch.randint(0, pairs, (hidden,), generator=rng)
    down = torch.zeros((experts, hidden, inter))
    down[:, torch.arange(hidden), 2 * pair], down[:, torch.arange(hidden), 2 * pair + 1] = 1.0, -1.0
    ones = [torch.ones((experts, -(-r // 128), -(-c // 128)), device="cuda") for r, c in ((inter, hidden), (hidden, inter))]
    moe = clef_i4.MoeLayerF8(clef_i4.f8_weight(digits(g, g - 1)[:, order].to(F8).cuda(), ones[0]),
                             clef_i4.f8_weight(digits(u, u + 1)[:, order].to(F8).cuda(), ones[0]),
                             clef_i4.f8_weight(down[:, :, order].to(F8).cuda(), ones[1]), topk=1)
    at = torch.arange(t) * 37 % triples
    x = torch.zeros((t, hidden))
    for i, place in enumerate((256.0, 16.0, 1.0)):
        x[torch.arange(t), 3 * at + i] = place
    e = torch.randint(0, experts, (t,), generator=rng)
    logits = torch.nn.functional.one_hot(e, experts).float().cuda()
    got = moe.decode(x.to(BF).cuda(), logits)
    assert torch.equal(got.cpu().float(), want[e[:, None], pair[None, :], at[:, None]].float())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_decode_masked_logits(dtype):
    t, hidden, inter, experts, topk = 8, 256, 136, 12, 4
    moe, w = layer(experts, hidden, inter, topk, "f32", 5)
    x, r = randn((t, hidden), 1.0, 1), randn((t, hidden), 1.0, 3)
    logits = randn((t, experts), 1.0, 2, dtype)
    low = torch.finfo(dtype).min
    logits[0] = -INF
    logits[1] = NAN
    logits[2, :9] = -INF          # three left
    logits[3, ::2] = NAN
    logits[4] = low               # all at the lowest value: the first four, evenly
    logits[5, 3:] = low           # three, and one of probability zero
    logits[6] = 0.5               # ties
    logits[7, 5], logits[7, 6] = INF, -INF
    want, slack = moe64(x, logits, *w, topk, r)
    got = moe.decode(x, logits, residual=r)
    check(got, want, slack)
    assert torch.equal(got[:2], r[:2])
    assert (moe.decode(x, logits)[:2] == 0).all()


def test_decode_takes_nothing_of_other_experts_and_tokens():
    """NaN weights and scales of experts that a token does not name, and another
    token's NaN row, leave it as it is."""
    t, hidden, inter, experts, topk = 6, 264, 136, 8, 2
    raw = [expert_weight(experts, a, b, "f32", s) for s, (a, b) in enumerate(((inter, hidden), (inter, hidden), (hidden, inter)))]
    x = randn((t, hidden), 1.0, 1)
    logits = torch.full((t, experts), -5.0, device="cuda")
    for i in range(t):
        logits[i, i % 4] = 1.0
        logits[i, (i + 1) % 4] = 0.5
    logits[5] = -5.0
    logits[5, 6], logits[5, 7] = 1.0, 2.0
    clean = clef_i4.MoeLayerF8(*[clef_i4.f8_weight(*w) for w in raw], topk=topk).decode(x, logits)
    for codes, scales in raw:
        codes.view(torch.uint8)[6] = 0x7F
        scales[7] = NAN
    x[3] = NAN
    got = clef_i4.MoeLayerF8(*[clef_i4.f8_weight(*w) for w in raw], topk=topk).decode(x, logits)
    keep = [0, 1, 2, 4]
    assert torch.equal(got[keep], clean[keep])
    assert torch.isnan(got[3]).all() and torch.isnan(got[5]).all()


@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** -117, 1.0, 2.0 ** 100, 1.5 * 2.0 ** 112])
def test_decode_scales_at_their_limits(scale):
    """Gate and up scales of any size with rows that bring the sums back."""
    t, hidden, inter = 3, 256, 128
    codes = [randn((2, a, b), 60.0, s, F32).clamp(-448, 448).to(F8) for s, (a, b) in
             enumerate(((inter, hidden), (inter, hidden), (hidden, inter)))]
    size = 2.0 ** -round(math.log2(scale))
    x = (randn((t, hidden), 1.0, 4, F32) * min(size, 2.0 ** 120)).to(BF)
    ones = torch.ones((2, 1, 2), device="cuda") * scale
    down = torch.ones((2, 2, 1), device="cuda") * 2.0 ** -10
    raw = list(zip(codes, (ones, ones, down)))
    moe = clef_i4.MoeLayerF8(*[clef_i4.f8_weight(*w) for w in raw], topk=1)
    logits = randn((t, 2), 1.0, 5, F32)
    check(moe.decode(x, logits), *moe64(x, logits, *[weight64(*w) for w in raw], 1))


def test_decode_in_place_strided_and_with_its_router():
    t, hidden, inter, experts, topk = 5, 512, 256, 24, 3
    router = randn((experts, hidden), 0.05, 9)
    moe, w = layer(experts, hidden, inter, topk, "f32", 3, router)
    x = randn((t, hidden), 1.0, 1)
    many = randn((9, 25), 1.0, 7)
    part = many.flatten()[1:1 + t * experts].view(t, experts)  # logits that start at any element
    assert torch.equal(moe.decode(x, part), moe.decode(x, part.clone()))
    logits = clef_i4.linear(x, router, dtype=F32)
    want = moe.decode(x, logits, residual=x)
    assert torch.equal(moe.decode(x, residual=x), want)
    wide = torch.full((t, hidden + 24), NAN, dtype=BF, device="cuda")
    wide[:, 8:8 + hidden] = x
    assert torch.equal(moe.decode(wide[:, 8:8 + hidden], residual=x), want)
    again = x.clone()
    assert moe.decode(again, residual=again, out=again) is again
    assert torch.equal(again, want)
    check(want, *moe64(x, logits, *w, topk, x))
    assert moe.decode(x[:0]).shape == (0, hidden)


@pytest.mark.parametrize("t", [1, 16])
def test_decode_does_not_depend_on_its_scratch(t):
    """Two calls of different tokens through the same freed memory, and the rows
    of a call one by one."""
    moe, _ = layer(32, 512, 264, 4, "e8m0", 1)
    x, logits = randn((t, 512), 1.0, 2), randn((t, 32), 1.0, 3, F32)
    first = moe.decode(x, logits)
    torch.full((1 << 22,), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(moe.decode(x, logits), first)
    for i in range(t):
        one = moe.decode(x[i:i + 1], logits[i:i + 1])
        off = (one[0].double() - first[i].double()).abs()
        assert (off <= 2.0 ** -7 * first[i].double().abs() + 1e-3 * first[i].double().abs().mean()).all()


def decode_on(scratch, moe, x, logits):
    """decode on a workspace of the caller's."""
    out, n = torch.full_like(x, NAN), clef_i4._n
    n.launch(n.clef_moe_layer_f8, x, x.shape[1], logits, int(logits.dtype == F32), x.shape[0], x.shape[1], moe.gate.rows,
             moe.gate.matrices, moe.topk, moe.gate.codes, moe.gate.scales, moe.up.codes, moe.up.scales, moe.down.codes,
             moe.down.scales, None, out, scratch, scratch.numel())
    return out


def workspace(moe, t, hidden):
    nbytes = clef_i4.lib().clef_moe_layer_f8_workspace_bytes(t, hidden, moe.gate.rows, moe.gate.matrices, moe.topk)
    return torch.zeros((nbytes,), dtype=torch.uint8, device="cuda")


# widths whose down products are split in many parts: 8 columns a workgroup, 32
PARTS = [(4, 64, 8192, 4, 4), (3, 8, 32768, 4, 2), (9, 256, 2048, 32, 4), (16, 128, 4096, 8, 2)]


@pytest.mark.parametrize("t,hidden,inter,experts,topk", PARTS)
def test_decode_adds_parts_that_have_arrived(t, hidden, inter, experts, topk):
    """A part's sum read before it is there would be the NaN that the
    scratch held."""
    moe, w = layer(experts, hidden, inter, topk, "f32", t)
    x, logits = randn((t, hidden), 1.0, 1), randn((t, experts), 2.0, 2, F32)
    scratch = workspace(moe, t, hidden)
    first = decode_on(scratch, moe, x, logits)
    check(first, *moe64(x, logits, *w, topk))
    for _ in range(20):
        scratch.fill_(255)
        assert torch.equal(decode_on(scratch, moe, x, logits), first)


@pytest.mark.parametrize("t,hidden,inter,experts,topk", [(1, 512, 264, 32, 4), (16, 512, 264, 32, 4), *PARTS])
def test_decode_takes_nothing_from_its_scratch(t, hidden, inter, experts, topk):
    """A call on what a call of other tokens left (their table, h, parts' sums and
    counts), or on all bits set, is a call on zeros, bit for bit. Some tokens name
    fewer experts than topk, and one none."""
    moe, w = layer(experts, hidden, inter, topk, "f32", t)
    sets = []
    for seed in (1, 2):
        logits = randn((t, experts), 2.0, seed, F32)
        if seed == 2:
            logits[::2, :experts - 1] = -INF
            logits[t // 2] = NAN
        sets.append((randn((t, hidden), 1.0, seed + 2), logits))
    wants = []
    for x, logits in sets:
        wants.append(decode_on(workspace(moe, t, hidden), moe, x, logits))
        check(wants[-1], *moe64(x, logits, *w, topk))
    assert not torch.equal(*wants)
    scratch = workspace(moe, t, hidden)
    for turn in (0, 1, 0, 1, 1, 0):
        assert torch.equal(decode_on(scratch, moe, *sets[turn]), wants[turn])
    for turn in (0, 1):
        scratch.fill_(255)
        assert torch.equal(decode_on(scratch, moe, *sets[turn]), wants[turn])


# ---------------------------------------------------------------- together

def block(moe, x, wg, wu, wd, wo, bo):
    """An output projection onto its residual, then a MoE block with a shared expert."""
    y = clef_i4.linear(x, wo, bias=bo, residual=x)
    shared = clef_i4.linear(clef_i4.linear_gate_up(y, wg, wu), wd, residual=y)
    return moe.decode(y, residual=shared), y, shared


@pytest.fixture(scope="module")
def parts():
    hidden, inter, experts, topk = 768, 256, 16, 4
    moe, w = layer(experts, hidden, inter, topk, "f32", 3, randn((experts, hidden), 0.05, 9))
    dense = (randn((inter, hidden), 0.03, 11), randn((inter, hidden), 0.03, 12), randn((hidden, inter), 0.06, 13),
             randn((hidden, hidden), 0.03, 14), randn((hidden,), 1.0, 15))
    return moe, w, dense


@pytest.mark.parametrize("t", [1, 3, 16])
def test_block_of_all_matches_64_bits(parts, t):
    moe, w, (wg, wu, wd, wo, bo) = parts
    x = randn((t, 768), 1.0, t)
    got, y, shared = block(moe, x, wg, wu, wd, wo, bo)
    check(y, *linear64(x, wo, bo, None, x))
    h = clef_i4.linear_gate_up(y, wg, wu)
    check(h, *gate_up64(y, wg, wu))
    check(shared, *linear64(h, wd, None, None, y))
    check(got, *moe64(y, clef_i4.linear(y, moe.router, dtype=F32), *w, moe.topk, shared))


def test_block_graphs_replay_beside_eager_calls(parts):
    """Two captured graphs and eager calls in between, on new inputs each time."""
    moe, _, dense = parts
    sizes = (2, 16)
    xs = [torch.zeros((t, 768), dtype=BF, device="cuda") for t in sizes]
    for x in xs:
        block(moe, x, *dense)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(block(moe, x, *dense)[0])
        graphs.append(g)
    for turn in range(4):
        for t, x in zip(sizes, xs):
            x.copy_(randn((t, 768), 1.0, 100 * turn + t))
        wants = [block(moe, x.clone(), *dense)[0] for x in xs]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, wants):
            assert torch.equal(out, want)


def test_split_products_in_graphs_and_on_two_streams():
    """Products whose parts meet in scratch of their own: two captured graphs, eager
    calls in between, then two streams."""
    shapes = [(131, 8200, 3001), (300, 8200, 1040)]
    ws = [randn((n, k), 0.02, n) for _, k, n in shapes]
    xs = [torch.zeros((m, k), dtype=BF, device="cuda") for m, k, _ in shapes]
    assert all(clef_i4.lib().clef_linear_workspace_bytes(m, n, k, g) > 0 for m, k, n in shapes for g in (0, 1))

    def both(i, x):
        return clef_i4.linear(x, ws[i], activation="silu"), clef_i4.linear_gate_up(x, ws[i], ws[i])

    for i, x in enumerate(xs):
        both(i, x)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i, x in enumerate(xs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both(i, x))
        graphs.append(g)
    for turn in range(4):
        for i, x in enumerate(xs):
            x.copy_(randn(x.shape, 1.0, 10 * turn + i))
        wants = [both(i, x.clone()) for i, x in enumerate(xs)]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for out, want in zip(outs, wants) for o, w in zip(out, want))
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
    for _ in range(5):
        for i, (s, x) in enumerate(zip(streams, xs)):
            with torch.cuda.stream(s):
                got[i].append(both(i, x))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for g, want in zip(got, wants) for out in g for o, w in zip(out, want))


def test_block_on_two_streams_at_once(parts):
    moe, _, dense = parts
    xs = [randn((t, 768), 1.0, t) for t in (16, 9)]
    wants = [block(moe, x, *dense)[0] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
    for _ in range(10):
        for i, (s, x) in enumerate(zip(streams, xs)):
            with torch.cuda.stream(s):
                got[i].append(block(moe, x, *dense)[0])
    torch.cuda.synchronize()
    for outs, want in zip(got, wants):
        assert all(torch.equal(o, want) for o in outs)


def test_binding_refusals():
    x, w = randn((4, 64), 1.0, 1), randn((32, 64), 1.0, 2)
    good = dict(x=x, weight=w)

    def refused(match, fn=clef_i4.linear, **kw):
        with pytest.raises((clef_i4.ClefError, AssertionError), match=match):
            fn(**kw)

    shape = "linear shape/dtype"
    refused(shape, **{**good, "x": x.float()})
    refused(shape, **{**good, "weight": w.float()})
    refused(shape, **{**good, "x": x[:, :32]})
    refused(shape, **{**good, "weight": w[None]})
    refused(shape, **{**good, "weight": w[0]})
    refused(shape, **{**good, "x": x.t().contiguous().t()})
    refused(shape, **{**good, "x": x[:1].expand(4, 64)})
    refused(shape, **good, bias=randn((31,), 1.0, 3))
    refused(shape, **good, bias=randn((32,), 1.0, 3).half())
    refused(shape, **good, dtype=torch.float16)
    refused("contiguous", **good, bias=randn((64,), 1.0, 3)[::2])
    refused("unknown activation", **good, activation="swish")
    refused("residual", **good, residual=randn((3, 32), 1.0, 3))
    refused(shape, **good, residual=randn((4, 31), 1.0, 3))
    refused(shape, **good, residual=randn((4, 32), 1.0, 3, F32))
    refused("current device", **{**good, "x": x.cpu()})
    refused("current device", **{**good, "weight": w.cpu()})
    refused("current device", **good, bias=torch.zeros(32, dtype=BF))
    refused("current device", **good, residual=torch.zeros((4, 32), dtype=BF))
    refused("current device", **good, out=torch.zeros((4, 32), dtype=BF))
    refused("output shape/dtype", **good, out=torch.zeros((4, 31), dtype=BF, device="cuda"))
    refused("output shape/dtype", **good, out=torch.zeros((4, 32), dtype=F32, device="cuda"), dtype=BF)
    refused("output shape/dtype", **good, out=torch.zeros((32, 4), dtype=BF, device="cuda").t())
    refused("overlaps", x=x, weight=randn((64, 64), 1.0, 2), out=x)
    gu = clef_i4.linear_gate_up
    refused(shape, gu, x=x, gate=w, up=w[:31])
    refused(shape, gu, x=x, gate=w, up=randn((32, 128), 1.0, 1)[:, :64])
    refused(shape, gu, x=x, gate=w, up=w, gate_bias=torch.zeros(32, device="cuda"), up_bias=torch.zeros(32, dtype=BF, device="cuda"))
    refused("unknown activation", gu, x=x, gate=w, up=w, activation="geglu")
    moe, _ = layer(8, 256, 128, 2, "f32", 1)
    x, logits = randn((4, 256), 1.0, 1), randn((4, 8), 1.0, 2)
    few = moe.decode
    refused("few tokens", few, x=randn((17, 256), 1.0, 1), logits=randn((17, 8), 1.0, 2))
    refused("few tokens", few, x=x[:, :128], logits=logits)
    refused("needs router logits", few, x=x)
    refused("router logits", few, x=x, logits=logits[:3])
    refused("logits dtype", few, x=x, logits=logits.half())
    refused("current device", few, x=x, logits=logits.cpu())
    refused("residual", few, x=x, logits=logits, residual=x[:3])
    refused("output", few, x=x, logits=logits, out=x.float())
    refused("contiguous", few, x=x, logits=randn((4, 16), 1.0, 2)[:, ::2])
    moe.topk = 9
    refused("few tokens", few, x=x, logits=logits)
