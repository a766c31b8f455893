"""Channels-last layers at the ends of their types' ranges and next to callers' modes (no GPU)."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch
from torch.autograd import forward_ad

from oracle import ref_cl as R
from textboxgan_amd import build, native, ops_cl


def test_the_format_read_as_fp16():
    """every finite fp16 value, alone in its block, comes back finite and within half a step"""
    x = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.float16).reshape(-1, 1)
    x = x[torch.isfinite(x[:, 0])]
    q, e = R.pack(x)
    v = R.unpack_as(q, e, x.shape, torch.float16)
    assert torch.isfinite(v).all()
    # half a step (amax / 127.5 at most), and fp16's rounding where its own steps are wider (2^-24 below 2^-14: half of that)
    assert ((v.double() - x.double()).abs() <= torch.clamp(x.double().abs() / 127.5, min=2.0 ** -25)).all()
    far = torch.tensor([[66560.0], [-70000.0], [3e38]])  # what no fp16 value can have been stays beyond its range
    assert torch.isinf(R.unpack_as(*R.pack(far), far.shape, torch.float16)).all()


def a8(shape, dtype=torch.float32):
    rows, nb = shape[0], (shape[-1] + 31) // 32
    return ops_cl.Act8(torch.zeros(rows, nb * 32, dtype=torch.int8), torch.zeros(rows, nb, dtype=torch.uint8), shape, dtype)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", range(3))
def test_a_group_norm_refuses_forward_mode(which, grad):
    """no result that has lost its tangent: refused before anything runs, whether or not reverse mode is on as well"""
    ops = [torch.ones(2, 3, 8), torch.ones(8), torch.zeros(8)]
    with forward_ad.dual_level():
        ops[which] = forward_ad.make_dual(ops[which], torch.ones_like(ops[which]))
        if grad:
            ops[0].requires_grad_()
        with pytest.raises(native.TbgError, match="forward-mode"):
            ops_cl.group_norm_act(*ops, 2)
        with torch.no_grad(), pytest.raises(native.TbgError, match="forward-mode"):
            ops_cl.group_norm_act(*ops, 2)
        with pytest.raises(native.TbgError, match="device tensors"):  # (no operand has a tangent)
            ops_cl.group_norm_act(torch.ones(2, 3, 8), torch.ones(8), torch.zeros(8), 2)


def test_backward_passes_refuse_forward_mode(monkeypatch):
    """a dual output gradient: the kernels would answer with its value alone"""
    monkeypatch.setattr(ops_cl, "_gn_fwd", lambda x, *a: (x.detach().clone(), torch.zeros(1), None, None, None))
    x, w = torch.ones(4, 8, requires_grad=True), torch.ones(8, 8)
    y = ops_cl._GroupNormAct.apply(x, torch.ones(8), torch.zeros(8), (2, 0, 1e-5), False, False, [])
    z = ops_cl._DenseAct8.apply(x, w, None, 1.0, None, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(4, 8), torch.ones(4, 8))
        for out in (y, z):
            with pytest.raises(native.TbgError, match="forward-mode"):
                torch.autograd.grad(out, x, dual, retain_graph=True)
        with pytest.raises(native.TbgError, match="forward-mode"):
            ops_cl.act8_wgrad(a8((4, 40)), dual)
    assert torch.equal(torch.autograd.grad(z, x, torch.ones(4, 8))[0], torch.full((4, 8), 8.0))


def test_a_dense_layer_without_reverse_mode_keeps_tangents(monkeypatch):
    monkeypatch.setattr(ops_cl, "_placed", lambda *a: None)
    x, w, t = torch.randn(4, 8), torch.randn(8, 3), torch.randn(4, 8)
    with forward_ad.dual_level():
        y = ops_cl.dense_act8(forward_ad.make_dual(x, t), w, coef=0.5)
        assert torch.allclose(forward_ad.unpack_dual(y).tangent, 0.5 * t @ w, atol=1e-6)
        with pytest.raises(RuntimeError, match="jvp"):  # (torch's own refusal of a function that has none)
            ops_cl.dense_act8(forward_ad.make_dual(x, t), w.clone().requires_grad_(), x8=a8((4, 8)))


def test_a_data_gradient_inside_autocast():
    """the product of the backward pass runs in its operands' type, as that of the forward pass does"""
    x, w = torch.randn(40, 72, requires_grad=True), torch.randn(72, 30)
    dy = torch.randn(40, 30)
    want = torch.autograd.grad(ops_cl._DenseAct8.apply(x, w, None, 0.5, None, None), x, dy)[0]
    with torch.autocast("cpu", dtype=torch.bfloat16):
        y = ops_cl._DenseAct8.apply(x, w, None, 0.5, None, None)
        got = torch.autograd.grad(y, x, dy)[0]
    assert y.dtype == got.dtype == torch.float32 and torch.equal(got, want)


def test_rows_are_moved_at_their_own_alignment(tmp_path):
    """the 8-channel loads and stores of the channels-last kernels promise the compiler no more than a row's element alignment (rows begin at any
    element), and the header compiles without a word about it"""
    src = tmp_path / "rows.hip"
    src.write_text('#include "act8.h"\n' + "\n".join(f"""
__global__ void copy_{e}_{past}(const {e}::type *x, {e}::type *y) {{
  const Pack8<{e}> r = ld8<{e}, {past}>(x + threadIdx.x * 9);
  st8<{e}, {past}>(y + threadIdx.x * 9, r);
}}""" for e in ("ElF32", "ElBf16", "ElF16") for past in ("false", "true")) + "\n")
    out = tmp_path / "rows.ll"
    run = subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *build.FLAGS, "-I", build.CSRC, "--cuda-device-only", "-S", "-emit-llvm", str(src),
                          "-o", str(out)], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
    assert "aligned" not in run.stderr, run.stderr
    moves = re.findall(r"(?:load|store) <4 x (i32|float)>.*align (\d+)", out.read_text())
    assert len(moves) == 2 * 2 * (2 + 1 + 1) and all(int(a) <= (4 if t == "float" else 2) for t, a in moves), moves


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_checkpoint_of_another_type_is_refused(dtype):
    for other in (torch.float32, torch.bfloat16, torch.float16):
        with pytest.raises(native.TbgError, match="device tensors" if other == dtype else "is not one of"):
            ops_cl.dense_act8(torch.zeros(2, 40, dtype=dtype), torch.zeros(40, 4), x8=a8((2, 40), other))


@pytest.mark.parametrize("dtype, terms", [(0, 3), (1, 1), (2, 2)])
@pytest.mark.parametrize("cin, cout, tk, tn, regs", [(128, 128, 128, 128, 2), (256, 256, 128, 128, 2), (128, 64, 128, 64, 2), (64, 128, 64, 128, 2), (64, 64, 64, 64, 4)])
def test_weight_gradients_fill_the_card_once(dtype, terms, cin, cout, tk, tn, regs):
    """many rows are split over as many blocks as 256 CUs hold at once (by registers, and by the 160 KB of LDS that three buffers of 32 rows share)"""
    if dtype == 1 and cin == cout == 256:
        tk, tn, regs = 256, 256, 1  # (bf16 has a wider tile)
    lds = 3 * 32 * (tk + 32 + terms * (tn + 32)) * 2
    rows = 1 << 20
    splits, left = divmod(native.lib().tbg_act8_wgrad_workspace_bytes(rows, cin, cout, dtype), (cin + 1) * cout * 4)
    assert left == 0 and splits * -(-cin // tk) * -(-cout // tn) == 256 * min(regs, 160 * 1024 // lds)


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_weight_gradients_of_few_rows_take_one_launch(dtype):
    """no partial sums up to 512 rows, whatever the type and the widths"""
    space = native.lib().tbg_act8_wgrad_workspace_bytes
    for cin, cout in ((512, 512), (64, 64), (512, 1023), (512, 1024), (1024, 1024)):
        assert space(512, cin, cout, dtype) == 0 < space(1024, cin, cout, dtype), (cin, cout)


def test_column_sums_entry_checks_its_arguments():
    lib, p, odd = native.lib(), C.c_void_p(256), C.c_void_p(264)
    space = lib.tbg_column_sums_workspace_bytes
    assert space(1, 1, 0) == 0 and space(0, 1, 0) == -1 and space(1, 0, 0) == -1 and space(1, 1, 3) == -1 and space(1, (1 << 30) + 1, 0) == -2
    need = space(100000, 72, 1)
    assert need > 0 and need % (72 * 4) == 0
    call = lambda x, dt, rows, cols, ld, out, ws, n: lib.tbg_column_sums(x, dt, rows, cols, ld, out, ws, n, None)
    assert call(None, 1, 100000, 72, 72, p, p, need) == -1 and call(p, 1, 100000, 72, 72, None, p, need) == -1
    assert call(p, 1, 100000, 72, 71, p, p, need) == -1 and call(p, 1, 0, 72, 72, p, p, need) == -1 and call(p, 3, 100000, 72, 72, p, p, need) == -1
    assert call(p, 1, 100000, 72, 72, p, p, need - 1) == -1 and call(p, 1, 100000, 72, 72, p, None, need) == -1 and call(p, 1, 100000, 72, 72, p, odd, need) == -1
