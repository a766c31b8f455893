"""Channels-last layers: refusals, the C entries' argument checks, the struct layout and the oracle's format (no GPU)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from oracle import ref_cl as R
from textboxgan_amd import native, ops_cl

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD = native.TbgError


@pytest.mark.parametrize("call, says", [
    (lambda: ops_cl.act8_pack([1.0]), "a tensor is wanted"),
    (lambda: ops_cl.act8_pack(torch.zeros(2, 8, dtype=torch.float64)), "unsupported dtype"),
    (lambda: ops_cl.act8_pack(torch.zeros(())), "channels"),
    (lambda: ops_cl.act8_pack(torch.zeros(3, 0)), "channels"),
    (lambda: ops_cl.act8_pack(torch.zeros(2, 8)), "device tensors"),
    (lambda: ops_cl.act8_unpack(torch.zeros(2)), "Act8"),
    (lambda: ops_cl.act8_unpack(_a8((2, 40))), "device tensors"),
    (lambda: ops_cl.act8_unpack(_a8((2, 40)), torch.int32), "unsupported dtype"),
    (lambda: ops_cl.act8_unpack(_a8((2, 40))._replace(shape=(3, 40))), "do not fit"),
    (lambda: ops_cl.act8_unpack(_a8((2, 40))._replace(shape=(2, 65))), "do not fit"),
    (lambda: ops_cl.act8_unpack(_a8((2, 40))._replace(q=torch.zeros(2, 64))), "unsupported dtype"),
    (lambda: ops_cl.act8_wgrad(_a8((2, 40)), torch.zeros(3, 8)), "does not belong"),
    (lambda: ops_cl.act8_wgrad(_a8((2, 40)), torch.zeros(2, 0)), "does not belong"),
    (lambda: ops_cl.act8_wgrad(_a8((2, 40)), torch.zeros(2, 8, dtype=torch.int8)), "unsupported dtype"),
    (lambda: ops_cl.act8_wgrad(_a8((2, 40)), torch.zeros(2, 8)), "device tensors"),
    (lambda: _gn(groups=3), "do not divide"),
    (lambda: _gn(groups=0), "do not divide"),
    (lambda: _gn(groups=2.0), "do not divide"),
    (lambda: _gn(act="gelu"), "unknown activation"),
    (lambda: _gn(save="fp8"), "save is"),
    (lambda: _gn(eps=0.0), "eps"),
    (lambda: _gn(eps=float("nan")), "eps"),
    (lambda: _gn(x=torch.zeros(8)), "is wanted"),
    (lambda: _gn(x=torch.zeros(2, 3, 8, dtype=torch.float64)), "unsupported dtype"),
    (lambda: _gn(gamma=torch.ones(8, dtype=torch.bfloat16)), "gamma: unsupported dtype"),
    (lambda: _gn(gamma=torch.ones(7)), "have to be"),
    (lambda: _gn(gamma=torch.ones(2, 8)), "have to be"),
    (lambda: _gn(gamma=torch.ones(3, 8), beta=torch.ones(3, 8)), "have to be"),
    (lambda: _gn(), "device tensors"),
    (lambda: ops_cl.act8_unpack(ops_cl.Act8(torch.zeros(0, 0, dtype=torch.int8), torch.zeros(0, 0, dtype=torch.uint8), (), torch.float32)), "is wanted"),
    (lambda: ops_cl.act8_pack(torch.zeros(1, 1).expand(1, 2 ** 32 + 8)), "channels, at most"),
    (lambda: ops_cl.act8_wgrad(_a8((2, 2 ** 20 + 1)), torch.zeros(2, 8)), "channels, at most"),
    (lambda: ops_cl.act8_wgrad(_a8((2, 8)), torch.zeros(1, 1).expand(2, 2 ** 32 + 1)), "channels, at most"),
    (lambda: _gn(x=torch.zeros(1, 1, 8).expand(1, 2 ** 32 + 3, 8)), "positions, at most"),
    (lambda: _gn(x=torch.zeros(1, 1, 8).expand(2 ** 32 + 3, 1, 8)), "samples, at most"),
    (lambda: _gn(x=torch.zeros(1, 1, 1).expand(1, 1, 2 ** 32 + 8)), "channels, at most"),
    (lambda: ops_cl.dense_act8(torch.zeros(2, 8), torch.zeros(7, 4)), "do not fit"),
    (lambda: ops_cl.dense_act8(torch.zeros(2, 8), torch.zeros(8, 4, dtype=torch.float16)), "w: unsupported dtype"),
    (lambda: ops_cl.dense_act8(torch.zeros(2, 8), torch.zeros(8, 4), torch.zeros(5)), "bias"),
    (lambda: ops_cl.dense_act8(torch.zeros(2, 40), torch.zeros(40, 4), x8=_a8((3, 40))), "is not one of"),
    (lambda: ops_cl.dense_act8(torch.zeros(2, 8), torch.zeros(8, 4)), "device tensors"),
])
def test_refusals(call, says):
    with pytest.raises(BAD, match=says):
        call()


def _a8(shape):
    rows, nb = shape[0], (shape[-1] + 31) // 32
    return ops_cl.Act8(torch.zeros(rows, nb * 32, dtype=torch.int8), torch.zeros(rows, nb, dtype=torch.uint8), shape, torch.float32)


def _gn(x=None, gamma=None, beta=None, groups=2, **kw):
    x = torch.zeros(2, 3, 8) if x is None else x
    return ops_cl.group_norm_act(x, torch.ones(8) if gamma is None else gamma, torch.zeros(8) if beta is None else beta, groups, **kw)


def _desc(**kw):
    d = dict(xn=24, xs=8, dn=24, ds=8, N=2, S=3, C=8, G=2, dtype=0, act=0, per_sample=0, eps=1e-5)
    d.update(kw)
    return native.GnDesc(*[d[f] for f, _ in native.GnDesc._fields_])


@pytest.mark.parametrize("kw", [dict(N=0), dict(S=0), dict(C=0), dict(G=0), dict(G=3), dict(dtype=3), dict(dtype=-1), dict(act=3), dict(act=-1),
                                dict(per_sample=2), dict(eps=0.0), dict(eps=float("nan")), dict(xs=7), dict(ds=7), dict(xn=-1), dict(dn=-1)])
def test_group_norm_entry_checks_its_descriptor(kw):
    lib, p = native.lib(), C.c_void_p(256)
    assert lib.tbg_group_norm_workspace_bytes(C.byref(_desc(**kw)), 0) == -1
    assert lib.tbg_group_norm_fwd(C.byref(_desc(**kw)), p, p, p, p, None, None, None, None, None, p, 1 << 20, None) == -1
    assert lib.tbg_group_norm_bwd(C.byref(_desc(**kw)), p, None, None, p, p, p, p, p, p, p, p, 1 << 20, None) == -1


def test_entries_check_pointers_and_workspaces():
    lib, p, odd = native.lib(), C.c_void_p(256), C.c_void_p(264)
    d = C.byref(_desc())
    fwd = lambda *a: lib.tbg_group_norm_fwd(d, *a)
    assert fwd(None, p, p, p, None, None, None, None, None, p, 1 << 20, None) == -1
    assert fwd(p, p, p, p, None, p, None, None, None, p, 1 << 20, None) == -1        # values without scales
    assert fwd(p, p, p, p, None, None, None, p, None, p, 1 << 20, None) == -1
    assert fwd(p, p, p, p, None, odd, p, None, None, p, 1 << 20, None) == -1         # misaligned checkpoint
    big = C.byref(_desc(S=100000, xn=800000, dn=800000))                             # (one launch, for few positions, takes no workspace)
    assert lib.tbg_group_norm_workspace_bytes(big, 0) > 8 and lib.tbg_group_norm_workspace_bytes(d, 0) == 0
    assert lib.tbg_group_norm_fwd(big, p, p, p, p, None, None, None, None, None, p, 8, None) == -1         # workspace too small
    assert lib.tbg_group_norm_fwd(big, p, p, p, p, None, None, None, None, None, None, 1 << 20, None) == -1
    assert fwd(p, p, p, p, odd, None, None, None, None, p, 1 << 20, None) == -1      # misaligned statistics
    bwd = lambda *a: lib.tbg_group_norm_bwd(d, *a)
    assert bwd(p, p, p, p, p, p, p, p, p, p, p, 1 << 20, None) == -1                 # both the input and a checkpoint
    assert bwd(None, None, None, p, p, p, p, p, p, p, p, 1 << 20, None) == -1        # neither
    assert bwd(p, None, None, p, p, p, p, p, p, p, p, 8, None) == -1
    assert lib.tbg_group_norm_workspace_bytes(C.byref(_desc(S=(1 << 30) + 1)), 0) == -2
    assert lib.tbg_act8_pack(p, 0, 4, 8, 7, p, p, None) == -1 and lib.tbg_act8_pack(p, 3, 4, 8, 8, p, p, None) == -1
    assert lib.tbg_act8_pack(p, 0, 4, 8, 8, odd, p, None) == -1 and lib.tbg_act8_pack(None, 0, 4, 8, 8, p, p, None) == -1
    assert lib.tbg_act8_unpack(p, p, 0, 8, p, 0, 8, None) == -1 and lib.tbg_act8_unpack(p, None, 4, 8, p, 0, 8, None) == -1
    assert lib.tbg_act8_pack(p, 0, 1 << 38, 64, 64, p, p, None) == -2
    # launches of 2^32 threads
    for kw, backward in ((dict(N=1 << 30, S=1, C=1024), 0), (dict(N=1 << 30, S=300, C=1024), 1), (dict(N=1 << 15, S=1, C=1 << 17), 0)):
        wide = dict(xs=kw.get("C", 8), ds=kw.get("C", 8), **kw)
        assert lib.tbg_group_norm_workspace_bytes(C.byref(_desc(**wide)), backward) == -2, kw
    assert lib.tbg_act8_wgrad_workspace_bytes(1 << 10, 1 << 16, 1 << 15, 1) >= 0
    ws = lib.tbg_act8_wgrad_workspace_bytes(1 << 16, 256, 256, 1)
    assert ws > 0 and lib.tbg_act8_wgrad_workspace_bytes(1, 1, 1, 0) == 0
    assert lib.tbg_act8_wgrad_workspace_bytes(0, 1, 1, 0) == -1 and lib.tbg_act8_wgrad_workspace_bytes(1, 1, 1, 3) == -1
    assert lib.tbg_act8_wgrad_workspace_bytes(1, 1 << 21, 1, 0) == -2
    wg = lambda *a: lib.tbg_act8_wgrad(*a)
    assert wg(p, p, p, 1, 1 << 16, 256, 256, 256, 1.0, p, p, p, ws - 1, None) == -1
    assert wg(p, p, p, 1, 1 << 16, 256, 256, 255, 1.0, p, p, p, ws, None) == -1
    assert wg(odd, p, p, 1, 1 << 16, 256, 256, 256, 1.0, p, p, p, ws, None) == -1
    assert wg(p, p, p, 1, 1 << 16, 256, 256, 256, 1.0, None, p, p, ws, None) == -1


def test_descriptor_layout_matches_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "tbg.h"', 'int main(void) {', '  printf("%zu\\n", sizeof(tbg_gn_desc));']
    lines += [f'  printf("%zu\\n", offsetof(tbg_gn_desc, {f}));' for f, _ in native.GnDesc._fields_] + ['  return 0;', '}']
    (tmp_path / "l.c").write_text("\n".join(lines))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "l")], text=True).split()]
    assert got == [C.sizeof(native.GnDesc)] + [getattr(native.GnDesc, f).offset for f, _ in native.GnDesc._fields_]


def test_the_format_keeps_what_it_says():
    """the oracle's own format: at most half a step of error, amax / 127 or better, the whole of fp32's range, NaN blocks"""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(500, 70, generator=g) * torch.exp(20 * torch.randn(500, 1, generator=g))
    x[7] = 0
    x[8, 3] = float("inf")
    x[9, 40] = float("nan")
    x[10, 0] = torch.finfo(torch.float32).max
    v = R.round_trip(x)
    nan = torch.zeros(500, 70, dtype=torch.bool)
    nan[8, :32] = True
    nan[9, 32:64] = True
    assert torch.equal(torch.isnan(v), nan)
    for b in range(0, 70, 32):
        xb, vb = x[:, b:b + 32].double(), v[:, b:b + 32]
        fine = ~nan[:, b]
        big = xb[fine].abs().amax(dim=1, keepdim=True)
        # half a step: the scale is at most amax / 63.75; below 2^-120 the step is 2^-126
        assert ((vb - xb)[fine].abs() <= torch.maximum(big / 127.5, torch.tensor(2.0 ** -127, dtype=torch.float64))).all()
    assert (v[7] == 0).all()
