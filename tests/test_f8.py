"""Block-scaled FP8 entry points without a GPU: sizes, refusals."""
import types

import numpy as np
import pytest
import torch

import clef_i4

FAKE = 1 << 20  # never dereferenced: every call below fails its checks first
SHAPE = "unsupported FP8 block shape"


def call(name, *args):
    rc = getattr(clef_i4.lib(), name)(*args)
    return rc, clef_i4.lib().clef_last_error().decode()


def test_sizes():
    lib = clef_i4.lib()
    assert lib.clef_f8_prepared_bytes(5, 128) == 5 * (128 + 16 + 4)
    assert lib.clef_f8_prepared_bytes(5, 136) == 5 * (256 + 16 + 2 * 4)
    assert lib.clef_f8_prepared_bytes(5, 2056) == 5 * (17 * 128 + 32 + 17 * 4)
    assert lib.clef_f8_prepared_bytes(0, 136) == 0
    assert lib.clef_f8_prepared_bytes(1 << 20, 32768) == (1 << 20) * (32768 + 256 + 1024)
    assert lib.clef_f8_prepared_bytes(5, 130) == -1 and lib.clef_f8_prepared_bytes(5, 32776) == -1
    assert lib.clef_f8_weight_bytes(3, 136, 264) == 3 * 2 * 3 * 16384
    assert lib.clef_f8_weight_bytes(0, 136, 264) == -1 and lib.clef_f8_weight_bytes(1, 136, 0) == -1
    assert lib.clef_f8_project_workspace_bytes(0, 256, 256) == 0
    assert lib.clef_f8_project_workspace_bytes(4096, 256, 264) == 4096 * (384 + 16 + 12)
    assert lib.clef_moe_group_slots_workspace_bytes(1 << 20, 16, 1024) > 0
    assert lib.clef_moe_group_slots_workspace_bytes(1, 8, 128) == 0


@pytest.mark.parametrize("rows,width,stride", [(4, 0, 8), (4, 12, 16), (4, 32776, 32776), (4, 256, 248), (4, 256, 260),
                                               (-1, 256, 256), ((1 << 27) + 1, 256, 256)])
def test_prepare_rejects(rows, width, stride):
    rc, msg = call("clef_f8_prepare", FAKE, rows, width, stride, FAKE, None)
    assert rc == -1 and msg == SHAPE


def test_prepare_pointers_and_no_rows():
    assert call("clef_f8_prepare", None, 0, 256, 256, None, None)[0] == 0
    for x, out in [(None, FAKE), (FAKE + 2, FAKE), (FAKE, FAKE + 8)]:
        rc, msg = call("clef_f8_prepare", x, 4, 256, 256, out, None)
        assert rc == -1 and "aligned" in msg


@pytest.mark.parametrize("matrices,n,k", [(0, 128, 128), (1025, 128, 128), (1, 0, 128), (1, 12, 128), (1, 128, 4),
                                          (1, 128, 32776), (1, 1048584, 128), (1024, 1048576, 32768)])
def test_weight_rejects(matrices, n, k):
    rc, msg = call("clef_f8_pack_weight", FAKE, matrices, n, k, FAKE, FAKE, None)
    assert rc == -1 and msg == SHAPE
    rc, msg = call("clef_f8_retile", FAKE, matrices, n, k, FAKE, None)
    assert rc == -1 and msg == SHAPE


@pytest.mark.parametrize("m,n,k", [(-1, 128, 128), ((1 << 20) + 1, 128, 128), (4, 0, 128), (4, 100, 128), (4, 128, 12)])
def test_products_reject(m, n, k):
    assert call("clef_f8_gemm", FAKE, FAKE, FAKE, m, n, k, 0, None, FAKE, None) == (-1, SHAPE)
    assert call("clef_f8_gemm_gate_up", FAKE, FAKE, FAKE, FAKE, FAKE, m, n, k, 0, FAKE, None) == (-1, SHAPE)
    assert call("clef_f8_project", FAKE, m, k, max(k, 16), FAKE, FAKE, n, 0, None, FAKE, FAKE, 1 << 40, None) == (-1, SHAPE)


def test_products_pointers_workspace_and_no_rows():
    assert call("clef_f8_gemm", None, None, None, 0, 128, 128, 1, None, None, None)[0] == 0
    assert call("clef_f8_gemm_gate_up", *[None] * 5, 0, 128, 128, 1, None, None)[0] == 0
    assert call("clef_f8_project", None, 0, 128, 128, None, None, 128, 1, None, None, None, 0, None)[0] == 0
    good = [FAKE] * 3
    for i in range(3):
        bad = list(good)
        bad[i] = FAKE + 4
        rc, msg = call("clef_f8_gemm", *bad, 4, 128, 128, 0, None, FAKE, None)
        assert rc == -1 and "aligned" in msg
    rc, msg = call("clef_f8_gemm", *good, 4, 128, 128, 0, FAKE + 2, FAKE, None)
    assert rc == -1 and "aligned" in msg
    need = clef_i4.lib().clef_f8_project_workspace_bytes(4096, 256, 256)
    rc, msg = call("clef_f8_project", FAKE, 4096, 256, 256, FAKE, FAKE, 256, 0, None, FAKE, FAKE, need - 1, None)
    assert rc == -1 and msg == "workspace too small"
    rc, msg = call("clef_f8_project", FAKE, 4096, 256, 252, FAKE, FAKE, 256, 0, None, FAKE, FAKE, need, None)
    assert rc == -1 and msg == SHAPE


@pytest.mark.parametrize("m", [4, 4096])
def test_project_rejects_an_output_over_its_rows(m):
    far = FAKE + (1 << 40)
    for x, out in ((FAKE, FAKE), (FAKE, FAKE + (m - 1) * 1024 + 496), (FAKE + 512 * m - 16, FAKE)):
        rc, msg = call("clef_f8_project", x, m, 256, 512, far, far, 256, 0, None, out, far, 1 << 40, None)
        assert rc == -1 and msg == "FP8 output overlaps its input rows"


def test_group_slots_rejects():
    args = (FAKE, FAKE, FAKE, 1 << 30, None)
    assert call("clef_moe_group_slots", FAKE, (1 << 20) + 1, 8, 128, *args)[1] == "unsupported Omni route grouping shape"
    assert call("clef_moe_group_slots", FAKE, 1 << 20, 17, 128, *args)[1] == "unsupported Omni route grouping shape"
    for experts in (0, 1025):
        assert call("clef_moe_group_slots", FAKE, 4, 8, experts, *args)[1] == "invalid grouped expert lists"
    assert call("clef_moe_group_slots", FAKE, 4, 8, 128, None, FAKE, FAKE, 1 << 30, None)[0] == -1
    assert call("clef_moe_group_slots", FAKE, 4, 8, 128, FAKE, None, FAKE, 1 << 30, None)[0] == -1
    need = clef_i4.lib().clef_moe_group_slots_workspace_bytes(65536, 8, 128)
    rc, msg = call("clef_moe_group_slots", FAKE, 65536, 8, 128, FAKE, FAKE, FAKE, need - 1, None)
    assert rc == -1 and msg == "workspace too small"


@pytest.mark.parametrize("a_rows,experts,total,topk,routed,k,n,message", [
    (4, 0, 8, 2, 0, 128, 128, "invalid grouped expert lists"),
    (4, 1025, 8, 2, 0, 128, 128, "invalid grouped expert lists"),
    (4, 8, -1, 2, 0, 128, 128, "invalid grouped expert lists"),
    (4, 8, 1 << 25, 2, 0, 128, 128, "invalid grouped expert lists"),
    (4, 8, 8, 0, 0, 128, 128, "invalid grouped expert lists"),
    (4, 8, 8, 129, 0, 128, 128, "invalid grouped expert lists"),
    (4, 8, 8, 2, 0, 130, 128, SHAPE),
    (4, 8, 8, 2, 0, 128, 130, SHAPE),
    (3, 8, 8, 2, 0, 128, 128, "expert lists name more rows than the activation has"),
    (7, 8, 8, 2, 1, 128, 128, "expert lists name more rows than the activation has"),
    (131073, 8, 8, 2, 0, 32768, 128, "expert activation operand of 4 GiB or more (split the tokens into chunks)"),
])
def test_experts_reject(a_rows, experts, total, topk, routed, k, n, message):
    rest = (FAKE, FAKE, experts, total, topk, routed, k, n, 0, FAKE, None)
    assert call("clef_moe_expert_f8", FAKE, a_rows, FAKE, FAKE, *rest) == (-1, message)
    assert call("clef_moe_expert_gate_up_f8", FAKE, a_rows, FAKE, FAKE, FAKE, FAKE, *rest) == (-1, message)


def test_experts_pointers_and_no_slots():
    none = (None, 4, None, None, None, None, 8, 0, 2, 0, 128, 128, 1, None, None)
    assert call("clef_moe_expert_f8", *none)[0] == 0
    rc, msg = call("clef_moe_expert_f8", FAKE, 4, FAKE, FAKE, None, FAKE, 8, 8, 2, 0, 128, 128, 0, FAKE, None)
    assert rc == -1 and "list pointer" in msg
    rc, msg = call("clef_moe_expert_f8", FAKE, 4, FAKE, FAKE, FAKE, FAKE + 2, 8, 8, 2, 0, 128, 128, 0, FAKE, None)
    assert rc == -1 and "list pointer" in msg
    rc, msg = call("clef_moe_expert_f8", FAKE, 4, FAKE, None, FAKE, FAKE, 8, 8, 2, 0, 128, 128, 0, FAKE, None)
    assert rc == -1 and "aligned" in msg


def test_operand_order_is_a_permutation():
    """The byte formula of a weight block (include/clef_i4.h) names each of the
    16384 bytes once, and a lane's 16 bytes are 16 consecutive k of one row."""
    r, k = np.meshgrid(np.arange(128), np.arange(128), indexing="ij")
    at = (r // 16) * 2048 + (k // 64) * 1024 + ((k // 16) % 4 * 16 + r % 16) * 16 + k % 16
    assert np.array_equal(np.sort(at.ravel()), np.arange(16384))
    assert (np.diff(at.reshape(128, 8, 16), axis=2) == 1).all()


def weight(matrices=1, rows=136, cols=264, codes=None, scales=None, dtype=torch.float32):
    blocks = matrices * -(-rows // 128) * -(-cols // 128)
    return clef_i4.F8Weight(torch.zeros(blocks * 16384 if codes is None else codes, dtype=torch.uint8),
                            torch.zeros(blocks if scales is None else scales, dtype=dtype), rows, cols, matrices)


@pytest.mark.parametrize("bad", [dict(codes=6 * 16384 - 1), dict(scales=5), dict(codes=0), dict(scales=0),
                                 dict(dtype=torch.bfloat16)])
def test_weights_smaller_than_they_say_do_not_reach_the_library(monkeypatch, bad):
    """Every call that takes a weight, on host tensors with the library's entry
    points replaced by one that records."""
    reached = []
    holds = clef_i4._n.holds
    fake = types.SimpleNamespace(holds=holds, value=lambda *a: 0, launch=lambda *a: reached.append(a),
                                 empty=lambda like, dtype, *size: torch.empty(size, dtype=dtype))
    for name in clef_i4.SIGNATURES:
        setattr(fake, name, name)
    monkeypatch.setattr(clef_i4, "_n", fake)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1)
    good, wrong = weight(), weight(**bad)
    goods = weight(2)
    bad = {k: 2 * v if isinstance(v, int) else v for k, v in bad.items()}
    wrongs = weight(2, **bad)
    x = torch.zeros((4, 264), dtype=torch.bfloat16)
    a = clef_i4.PreparedF8(torch.zeros(clef_i4.lib().clef_f8_prepared_bytes(4, 264), dtype=torch.uint8), 4, 264)
    offsets = torch.zeros(3, dtype=torch.int32)
    clef_i4.project_f8(a, good), clef_i4.project_quantized_f8(x, good), clef_i4.project_gate_up_f8(a, good, good)
    clef_i4.expert_f8(a, goods, offsets, None, 1, True), clef_i4.expert_gate_up_f8(a, goods, goods, offsets, None, 1, True)
    assert len(reached) == 5
    for f in (lambda: clef_i4.project_f8(a, wrong), lambda: clef_i4.project_quantized_f8(x, wrong),
              lambda: clef_i4.project_gate_up_f8(a, wrong, good), lambda: clef_i4.project_gate_up_f8(a, good, wrong),
              lambda: clef_i4.expert_f8(a, wrongs, offsets, None, 1, True),
              lambda: clef_i4.expert_gate_up_f8(a, wrongs, goods, offsets, None, 1, True),
              lambda: clef_i4.expert_gate_up_f8(a, goods, wrongs, offsets, None, 1, True)):
        with pytest.raises(clef_i4.ClefError):
            f()
    assert len(reached) == 5


def test_holds():
    t, u = torch.zeros((4, 6), dtype=torch.int32), torch.zeros(3)
    holds = clef_i4._n.holds
    assert holds(-1) and holds(-1, t, torch.int32, 24) and holds(-1, t, torch.int32, -1, u, torch.float32, 3)
    assert not holds(-1, t, torch.int32, 25) and not holds(-1, t, torch.float32, 24) and not holds(0, t, torch.int32, 24)
    assert not holds(-1, t.t(), torch.int32, 24) and not holds(-1, t.to("meta"), torch.int32, 24)
    assert not holds(-1, t, torch.int32, 25, u, torch.float32, 3) and not holds(-1, t, torch.int32, 24, u, torch.float32, 4)
    for wrong in ((), (-1, t), (-1, t, torch.int32), (-1, None, torch.int32, 0), (-1, t, 4, 24), (-1, t, torch.int32, "24"),
                  (None, t, torch.int32, 24)):
        with pytest.raises(TypeError):
            holds(*wrong)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64, torch.int32, torch.int8])
def test_router_logits_of_other_types_are_refused(dtype):
    """The library knows bf16 and f32: logits of a narrower type would be read
    past their end, wider ones as other values."""
    logits = torch.zeros((4, 128), dtype=dtype)
    with pytest.raises(clef_i4.ClefError, match="router logits dtype"):
        clef_i4.omni_route(logits)
    x = torch.zeros((4, 264), dtype=torch.bfloat16)
    gate, down = weight(128, 136, 264), weight(128, 264, 136)
    with pytest.raises(clef_i4.ClefError, match="router logits dtype"):
        clef_i4.MoeLayerF8(gate, gate, down)(x, logits)
    q = clef_i4.QuantizedWeight(torch.zeros(1), torch.zeros(1), 128 * 256, 512, 512, 4)
    with pytest.raises(clef_i4.ClefError, match="router logits dtype"):
        clef_i4.MoeLayer(q, q, q)(x, logits)


SPLIT_K = ("16x32", "32x32", "16x64", "32x64", "64x64")
TILED = ("128x128", "128x128x2", "256x256")


def kernel(rows, n, k, gate_up=0, pow2=0, experts=0):
    return clef_i4.lib().clef_f8_kernel_name(rows, n, k, gate_up, pow2, experts).decode()


def test_kernel_name():
    assert kernel(1, 128, 128) == "16x32" and kernel(4096, 12288, 4096) == "256x256"
    assert kernel(620, 5120, 17408) == "128x128x2" and kernel(620, 5120, 4096, pow2=1) == "128x128"
    for bad in ((0, 128, 128), ((1 << 20) + 1, 128, 128), (4, 100, 128), (4, 128, 12), (4, 128, 32776)):
        assert kernel(*bad) == ""
    assert kernel(1 << 24, 128, 128, experts=8) == "128x128" and kernel((1 << 24) + 1, 128, 128, experts=8) == ""
    assert kernel(4, 128, 128, experts=1025) == "" and kernel(4, 128, 128, experts=-1) == ""


@pytest.mark.parametrize("pow2", [0, 1])
def test_every_kernel_is_compared_with_a_reference(pow2):
    """The shapes of the GPU tests reach, by the library's rule, every kernel of
    every product; the tiled ones with up to 16 blocks of k and more, the 256 x
    256 one with a last tile of at most half the rows and of more."""
    import test_gpu_f8 as gpu

    def reached(shapes, gate_up, experts=False):
        found = {}
        for s in shapes:
            rows, k, n = (s[0] * s[1], s[3], s[4]) if experts else s
            found.setdefault(kernel(rows, n, k, gate_up, pow2, s[2] if experts else 0), []).append((rows, k))
        return found

    for found in (reached(gpu.SHAPES + gpu.MORE, 0), reached(gpu.SHAPES + gpu.MORE_GU, 1)):
        assert set(found) == set(SPLIT_K + TILED)
        for name in TILED:
            blocks = [-(-k // 128) for _, k in found[name]]
            assert max(blocks) > 16 and (min(blocks) <= 16 or (name == "128x128x2" and pow2))
        for name in SPLIT_K:  # eight waves, a block each, and a second one
            assert max(k for _, k in found[name]) > 8 * 128
        assert {0 < rows % 256 <= 128 for rows, _ in found["256x256"]} == {True, False}
    for gate_up in (0, 1):
        found = reached(gpu.EXPERTS + gpu.MORE_EXPERTS, gate_up, experts=True)
        assert set(found) == {"16x32", "16x64", "128x128", "256x256"}
        for name, shapes in found.items():
            assert max(k for _, k in shapes) > 16 * 128
    # and the rows quantized by the product itself, against the two steps
    mark = next(m for m in gpu.test_project_quantizing_rows_itself_is_the_two_steps.pytestmark if m.args[0] == "m,k,n")
    fused = {kernel(m, n, k, 0, pow2) for m, k, n in mark.args[1]
             if clef_i4.lib().clef_f8_project_workspace_bytes(m, n, k) == 0}
    assert fused == set(SPLIT_K[:4])


APART = 1 << 34


def test_outputs_over_their_inputs_are_refused():
    """Kernels read and write in parallel: an output over what other workgroups
    still read would hold anything."""
    rows_message, residual_message = "FP8 output overlaps its input rows", "FP8 output overlaps a part of its residual"
    weight_message = "FP8 weight output overlaps its input"
    need = clef_i4.lib().clef_f8_prepared_bytes(64, 256)
    for out in (FAKE, FAKE + 64 * 512 - 16, FAKE - need + 16):
        assert call("clef_f8_prepare", FAKE, 64, 256, 256, out, None) == (-1, rows_message)
    assert call("clef_f8_prepare", FAKE, 64, 256, 1024, FAKE + 63 * 2048, None) == (-1, rows_message)
    for codes in (FAKE, FAKE + 256 * 256 - 16, FAKE - 4 * 16384 + 16):
        assert call("clef_f8_retile", FAKE, 1, 256, 256, codes, None) == (-1, weight_message)
        assert call("clef_f8_pack_weight", FAKE, 1, 256, 256, codes, FAKE + APART, None) == (-1, weight_message)
    assert call("clef_f8_pack_weight", FAKE, 1, 256, 256, FAKE + APART, FAKE, None) == (-1, weight_message)
    assert call("clef_f8_pack_weight", FAKE, 1, 256, 256, FAKE + APART, FAKE + APART, None) == (-1, weight_message)
    a, w, s, far = FAKE, FAKE + APART, FAKE + 2 * APART, FAKE + 3 * APART
    for out in (a, a + need - 16, a - 64 * 128 * 2 + 16):
        assert call("clef_f8_gemm", a, w, s, 64, 128, 256, 0, None, out, None) == (-1, rows_message)
        assert call("clef_f8_gemm_gate_up", a, w, s, w, s, 64, 128, 256, 0, out, None) == (-1, rows_message)
        assert call("clef_moe_expert_f8", a, 64, w, s, far, far, 8, 64, 1, 1, 256, 128, 0, out, None) == (-1, rows_message)
        assert call("clef_moe_expert_gate_up_f8", a, 64, w, s, w, s, far, far, 8, 64, 1, 1, 256, 128, 0, out, None) == \
            (-1, rows_message)
    for m, n in ((64, 128), (4096, 256)):
        for shift in (256, -256, m * n * 2 - 16):
            assert call("clef_f8_gemm", a, w, s, m, n, 256, 0, far + shift, far, None) == (-1, residual_message)
            assert call("clef_f8_project", a, m, 256, 256, w, s, n, 0, far + shift, far, far + APART, 1 << 30, None) == \
                (-1, residual_message)
    assert call("clef_f8_project", a, 4096, 256, 256, w, s, 256, 0, None, far, far, 1 << 30, None) == (-1, rows_message)
    assert call("clef_f8_project", a, 4096, 256, 256, w, s, 256, 0, far, far + APART, far, 1 << 30, None) == \
        (-1, "FP8 workspace overlaps an operand")
