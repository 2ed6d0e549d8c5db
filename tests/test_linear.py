"""Products with bf16 activations without a GPU: sizes, refusals."""
import math
import os
import re

import pytest
import torch

import clef_i4

FAKE = 1 << 20  # never dereferenced: every call below fails its checks first
FAR = 1 << 44
SHAPE = "linear shape/dtype mismatch"
OVERLAP = "linear output overlaps an operand"
FEW = "unsupported MoE shape for few tokens"


def call(name, *args):
    rc = getattr(clef_i4.lib(), name)(*args)
    return rc, clef_i4.lib().clef_last_error().decode()


def linear(x=FAKE, m=4, k=128, xs=None, w=FAR, n=64, ws=None, bias=None, bias_dtype=0, act=0, res=None, rs=None, out=2 * FAR,
           out_dtype=0, os=None, ws_at=5 * FAR, nbytes=1 << 40):
    xs, ws, rs, os = (d if v is None else v for v, d in ((xs, k), (ws, k), (rs, n), (os, n)))
    return call("clef_linear", x, m, k, xs, w, n, ws, bias, bias_dtype, act, res, rs, out, out_dtype, os, ws_at,
                nbytes, None)


def gate_up(x=FAKE, m=4, k=128, xs=None, gate=FAR, up=3 * FAR, n=64, ws=None, gb=None, ub=None, bias_dtype=0, act=4,
            h=2 * FAR, hs=None, ws_at=5 * FAR, nbytes=1 << 40):
    xs, ws, hs = (d if v is None else v for v, d in ((xs, k), (ws, k), (hs, n)))
    return call("clef_linear_gate_up", x, m, k, xs, gate, up, n, ws, gb, ub, bias_dtype, act, h, hs, ws_at,
                nbytes, None)


BAD = [dict(m=-1), dict(m=(1 << 20) + 1), dict(k=0), dict(k=(1 << 20) + 1), dict(n=0), dict(n=(1 << 20) + 1), dict(xs=127),
       dict(ws=127), dict(xs=1 << 31), dict(ws=1 << 31), dict(bias_dtype=2), dict(bias_dtype=-1), dict(act=-1), dict(act=6)]


@pytest.mark.parametrize("bad", BAD + [dict(out_dtype=2), dict(os=63), dict(os=1 << 31), dict(res=FAKE, rs=63)])
def test_linear_rejects(bad):
    assert linear(**bad) == (-1, SHAPE)


@pytest.mark.parametrize("bad", BAD + [dict(hs=63), dict(hs=1 << 31)])
def test_gate_up_rejects(bad):
    assert gate_up(**bad) == (-1, SHAPE)


def test_no_rows_do_nothing():
    assert linear(x=None, w=None, out=None, m=0)[0] == 0
    assert gate_up(x=None, gate=None, up=None, h=None, m=0)[0] == 0


@pytest.mark.parametrize("bad", [dict(x=None), dict(x=FAKE + 1), dict(w=None), dict(w=FAR + 1), dict(out=None),
                                 dict(out=FAR * 2 + 1), dict(out=FAR * 2 + 2, out_dtype=1), dict(bias=FAR * 3 + 1),
                                 dict(bias=FAR * 3 + 2, bias_dtype=1), dict(res=FAR * 3 + 1)])
def test_linear_pointers(bad):
    rc, msg = linear(**bad)
    assert rc == -1 and "aligned" in msg


def test_gate_up_pointers():
    for bad in (dict(up=None), dict(gate=FAR + 1), dict(h=FAKE + 1), dict(gb=FAKE * 9 + 1), dict(ub=FAKE * 9 + 2, bias_dtype=1)):
        rc, msg = gate_up(**bad)
        assert rc == -1 and "aligned" in msg


def test_outputs_over_operands_are_refused():
    # x: 4 rows of 128 at FAKE; the output 4 rows of 64
    assert linear(out=FAKE) == (-1, OVERLAP)
    assert linear(out=FAKE + 4 * 256 - 2) == (-1, OVERLAP)
    assert linear(out=FAR) == (-1, OVERLAP)
    assert linear(bias=2 * FAR + 64) == (-1, OVERLAP)
    assert linear(res=2 * FAR, out_dtype=1) == (-1, OVERLAP)      # f32 over its bf16 residual
    assert linear(res=2 * FAR, rs=128) == (-1, OVERLAP)           # the same memory in other rows
    assert linear(res=2 * FAR + 16) == (-1, OVERLAP)
    assert linear(xs=192, out=FAKE + 254, os=192) == (-1, OVERLAP)  # columns 127 .. of the same wide rows
    assert linear(xs=192, out=FAKE - 2, os=192) == (-1, OVERLAP)
    assert gate_up(h=FAKE) == (-1, OVERLAP)
    assert gate_up(h=3 * FAR + 64 * 256 - 2) == (-1, OVERLAP)
    assert gate_up(ub=2 * FAR) == (-1, OVERLAP)


@pytest.mark.parametrize("call_it,gate_up_it", [(linear, 0), (gate_up, 1)])
def test_workspace(call_it, gate_up_it):
    shape = dict(m=200, n=2048, k=8192)
    need = clef_i4.lib().clef_linear_workspace_bytes(200, 2048, 8192, gate_up_it)
    assert need > 0 and need % (200 * 2048 * 4 * (1 + gate_up_it)) == 0
    assert call_it(**shape, nbytes=need - 1) == (-1, "workspace too small")
    for ws_at in (None, 5 * FAR + 8):
        rc, msg = call_it(**shape, ws_at=ws_at)
        assert rc == -1 and "aligned" in msg
    for at in (FAKE, FAR, 2 * FAR):  # x, a weight, the output
        assert call_it(**shape, ws_at=at + 16) == (-1, "linear workspace overlaps an operand")
    for bad in ((0, 2048, 8192), (200, 0, 8192), (200, 2048, 0), (1 << 21, 2048, 8192), (8, 2048, 8192), (200, 2048, 64)):
        assert clef_i4.lib().clef_linear_workspace_bytes(*bad, gate_up_it) == 0


def test_kernel_name_and_every_kernel_is_compared_with_a_reference():
    """The GPU tests' shapes run every kernel of either product, split and whole."""
    from test_gpu_linear import KERNELS, ODD_KERNELS, ONCE

    lib = clef_i4.lib()
    few = {"8x16", "16x32", "32x32", "64x32"}
    for bad in ((0, 8, 8), (8, 0, 8), (8, 8, 0), (1 << 21, 8, 8)):
        assert lib.clef_linear_kernel_name(*bad, 0, 1) == b""
    for gate_up_it in (0, 1):
        seen = set()
        for m, k, n, name, parts in KERNELS[gate_up_it]:
            need = lib.clef_linear_workspace_bytes(m, n, k, gate_up_it)
            assert lib.clef_linear_kernel_name(m, n, k, gate_up_it, 1).decode() == name, (m, k, n)
            assert need == (parts * (1 + gate_up_it) * m * -(-n // 4) * 16 if parts > 1 else 0), (m, k, n)
            seen.add((name, parts > 1))
        tiles = {"128x128", "128x128x2", "128x256", "256x256"}
        whole = few | {"64x64"} | tiles | (set() if gate_up_it else {"8x8", "16x16", "32x16"})
        assert seen == {(t, False) for t in whole} | {(t, True) for t in tiles}
        for m, k, n, name in ONCE[gate_up_it]:
            assert lib.clef_linear_kernel_name(m, n, k, gate_up_it, 1).decode() == name, (m, k, n)
            assert m <= int(name.split("x")[0]) and n * k * 2 * (1 + gate_up_it) >= 1 << 24
        assert {c[3] for c in ONCE[gate_up_it]} == few | {"64x64"} | (set() if gate_up_it else {"8x8", "16x16"})
        odd = set()
        for m, k, n, name in ODD_KERNELS[gate_up_it]:
            assert lib.clef_linear_kernel_name(m, n, k, gate_up_it, 1).decode() == name, (m, k, n)
            odd.add(name)
        assert odd == few | {"any", "any128"} | (set() if gate_up_it else {"8x8", "16x16", "32x16"})


@pytest.mark.parametrize("which", [0, 1])
def test_column_ranges_reach_every_kernel(which):
    """Operands in wider rows run every kernel on the GPU, split and whole, on 16 bytes
    and at any even byte."""
    from test_gpu_linear import pitched

    lib = clef_i4.lib()
    seen = {True: set(), False: set()}
    for m, k, n, skip, behind in pitched(which):
        on16 = all(v % 8 == 0 for v in (skip, k, skip + k + behind))
        split = on16 and lib.clef_linear_workspace_bytes(m, n, k, which) > 0
        seen[on16].add((lib.clef_linear_kernel_name(m, n, k, which, on16).decode(), split))
    few = {"8x16", "16x32", "32x32", "64x32"} | (set() if which else {"8x8", "16x16", "32x16"})
    tiles = {"128x128", "128x128x2", "128x256", "256x256"}
    assert seen[True] == {(t, False) for t in few | {"64x64"} | tiles} | {(t, True) for t in tiles}
    assert seen[False] == {(t, False) for t in few | {"any", "any128"}}


def few(x=FAKE, xs=None, logits=FAR, dtype=0, t=4, hidden=256, inter=128, experts=8, topk=2, gate=2 * FAR, gs=3 * FAR,
        up=4 * FAR, us=5 * FAR, down=6 * FAR, ds=7 * FAR, res=None, out=8 * FAR, ws=9 * FAR, nbytes=1 << 30):
    xs = hidden if xs is None else xs
    return call("clef_moe_layer_f8", x, xs, logits, dtype, t, hidden, inter, experts, topk, gate, gs, up, us, down, ds, res,
                out, ws, nbytes, None)


@pytest.mark.parametrize("bad", [dict(t=-1), dict(t=17), dict(hidden=0), dict(hidden=12), dict(hidden=32776), dict(inter=0),
                                 dict(inter=12), dict(inter=32776), dict(experts=129), dict(experts=1), dict(topk=0),
                                 dict(topk=9), dict(xs=248), dict(xs=260), dict(xs=(1 << 24) + 8), dict(dtype=2)])
def test_moe_layer_f8_rejects(bad):
    assert few(**bad) == (-1, FEW)


@pytest.mark.parametrize("name", ["x", "logits", "gate", "gs", "up", "us", "down", "ds", "out", "ws", "res"])
def test_moe_layer_f8_pointers(name):
    at = dict(x=FAKE, logits=FAR, gate=2 * FAR, gs=3 * FAR, up=4 * FAR, us=5 * FAR, down=6 * FAR, ds=7 * FAR, res=10 * FAR,
              out=8 * FAR, ws=9 * FAR)[name]
    for bad in ([] if name == "res" else [None]) + [at + (1 if name == "logits" else 8)]:
        rc, msg = few(**{name: bad})
        assert rc == -1 and "aligned" in msg


def test_moe_layer_f8_workspace_and_overlaps():
    need = clef_i4.lib().clef_moe_layer_f8_workspace_bytes(4, 256, 128, 8, 2)
    assert need >= 4 * 2 * 128 * 4
    for bad in ((0, 256, 128, 8, 2), (17, 256, 128, 8, 2), (4, 12, 128, 8, 2), (4, 256, 128, 8, 9), (4, 256, 128, 129, 2)):
        assert clef_i4.lib().clef_moe_layer_f8_workspace_bytes(*bad) == 0
    assert few(nbytes=need - 1) == (-1, "workspace too small")
    assert few(t=0, x=None, logits=None, gate=None, out=None, ws=None, nbytes=0)[0] == 0
    for name in ("x", "logits", "out", "gate", "up", "down", "res"):
        assert few(**{name: 9 * FAR + 16}) == (-1, "MoE workspace overlaps an operand"), name
    assert few(out=FAKE + 16) == (-1, "MoE output overlaps an operand")
    assert few(out=FAR) == (-1, "MoE output overlaps an operand")
    assert few(res=8 * FAR + 16) == (-1, "MoE output overlaps an operand")


@pytest.mark.parametrize("name,bytes_", [("gate", 8 * 1 * 2 * 16384), ("up", 8 * 1 * 2 * 16384), ("down", 8 * 2 * 1 * 16384),
                                         ("gs", 8 * 1 * 2 * 4), ("us", 8 * 1 * 2 * 4), ("ds", 8 * 2 * 1 * 4)])
def test_moe_layer_f8_weights_and_scales_lie_apart(name, bytes_):
    """The output and the workspace over the first and the last 16 bytes of each."""
    at = dict(gate=2, gs=3, up=4, us=5, down=6, ds=7)[name] * FAR
    need = clef_i4.lib().clef_moe_layer_f8_workspace_bytes(4, 256, 128, 8, 2)
    result = 4 * 256 * 2
    for first in (at + 16 - result, at, at + bytes_ - 16):
        assert few(out=first) == (-1, "MoE output overlaps an operand"), (name, first - at)
    for first in (at + 16 - need // 16 * 16, at, at + bytes_ - 16):
        assert few(ws=first, nbytes=need) == (-1, "MoE workspace overlaps an operand"), (name, first - at)


def test_moe_layer_f8_output_over_rows_of_another_pitch():
    assert few(out=FAKE, xs=264) == (-1, "MoE output overlaps an operand")


@pytest.mark.parametrize("residual", [torch.zeros((), dtype=torch.bfloat16), torch.zeros(4, dtype=torch.bfloat16),
                                      torch.zeros((1, 4, 32), dtype=torch.bfloat16), torch.zeros((3, 32), dtype=torch.bfloat16)])
def test_residuals_of_other_dimensions_are_refused(residual, monkeypatch):
    """What linear says to them (here with the host as the device)."""
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((32, 64), dtype=torch.bfloat16)
    with pytest.raises(clef_i4.ClefError, match="residual shape/dtype mismatch"):
        clef_i4._refuse_linear(x, (w,), (None,), residual, None, None, None)


@pytest.mark.parametrize("gate_up_it", [0, 1])
def test_widths_off_16_bytes_need_no_workspace(gate_up_it):
    lib = clef_i4.lib()
    for k in (8185, 8190, 8191, 8193, 8196):
        assert lib.clef_linear_workspace_bytes(200, 2048, k, gate_up_it) == 0, k
    assert lib.clef_linear_workspace_bytes(200, 2048, 8184, gate_up_it) > 0


def test_gelu_polynomial_is_as_near_as_its_comment_says():
    """The coefficients in the source, rounded to f32, against the normal distribution's
    tail in 64 bits (14 is where exp(-a^2 / 2) leaves f32's normal range)."""
    with open(os.path.join(os.path.dirname(clef_i4.__file__), "csrc", "linear.hpp")) as f:
        source = f.read()
    body = source[source.index("float gelu_f32(float v) {"):]
    body = body[:body.index("\n}\n")]
    c = [torch.tensor(float(v)).item() for v in [re.search(r"float p = ([-\d.e]+)f;", body)[1]]
         + re.findall(r"p = __builtin_fmaf\(p, t, ([-\d.e]+)f\)", body)]
    slope = torch.tensor(float(re.search(r"__builtin_fmaf\(a, ([\d.]+)f, 1.0f\)", body)[1])).item()
    stated = float(re.search(r"\(([\d.]+e-7) of the value for a in 0 \.\. 14", source)[1])
    assert len(c) == 8 and stated < 1e-6
    worst = 0.0
    for i in range(14001):
        a = i / 1000
        t, p = 1.0 / (1.0 + slope * a), 0.0
        for v in c:
            p = p * t + v
        worst = max(worst, abs(p * t / (math.exp(a * a / 2) * math.erfc(a / math.sqrt(2.0)) / 2) - 1.0))
    assert 0.9 * stated < worst <= stated
