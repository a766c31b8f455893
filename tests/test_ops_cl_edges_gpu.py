"""-m gpu: channels-last layers at the ends of their types' ranges, against their definitions in 64 bits (oracle/ref_cl.py).  Tolerances are those of test_ops_cl_gpu.py."""
import pytest
import torch

from oracle import ref_cl as R
from textboxgan_amd import ops_cl
from test_ops_cl_gpu import values

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------- 8-bit checkpoints
def test_fp16_values_stay_finite(dev):
    """the top of fp16's range: its largest values lie within half a step of 65536 = 64 2^10, which the type does not hold"""
    x = torch.zeros(12, 70, dtype=torch.float16)
    for i, v in enumerate((65504.0, 65472.0, 65312.0, 65280.0, 65248.0, 65024.0, 64992.0)):
        x[i, 0], x[i, 33], x[i, 40], x[i, 69] = v, -v, v / 2, v
    x[8] = 65504.0
    x[9] = -65504.0
    x = x.to(dev)
    a = ops_cl.act8_pack(x)
    back = ops_cl.act8_unpack(a)
    assert torch.isfinite(back).all()
    assert torch.equal(back, R.unpack_as(a.q, a.e, x.shape, torch.float16))
    assert (back[8] == 65504).all() and (back[9] == -65504).all()
    # half a step: the scale is at most amax / 63.75
    assert ((back.double() - x.double()).abs() <= x.double().abs().amax(dim=1, keepdim=True) / 127.5).all()
    assert torch.equal(ops_cl.act8_unpack(a, torch.float32).double(), R.unpack(a.q, a.e, x.shape))


def test_wider_values_become_infinite_in_fp16(dev):
    """checkpoints of the wider types read as fp16: what may stand for one of its values is one, the others are beyond its range"""
    x = torch.tensor([[65504.0], [65536.0], [66047.0], [66560.0], [70000.0], [131072.0], [3e38], [-65600.0], [-70000.0], [float("inf")], [65535.0]], device=dev)
    for t in (torch.float32, torch.bfloat16):
        for wide in (x, torch.cat([x, x / 2, 1000 + 0 * x], dim=1), torch.cat([x, 4 * x], dim=1)):
            a = ops_cl.act8_pack(wide.to(t))
            got, want = ops_cl.act8_unpack(a, torch.float16), R.unpack_as(a.q, a.e, wide.shape, torch.float16)
            assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got.double()), torch.nan_to_num(want.double()))
    a = ops_cl.act8_pack(x[3:6])
    assert torch.isinf(ops_cl.act8_unpack(a, torch.float16)[1:]).all()


def test_fp16_output_checkpoint_stays_finite(dev):
    """the checkpoint that a norm writes of its output, at the top of the type's range"""
    x = values((2, 64, 64), torch.float16, dev, 200)
    gamma, beta = torch.full((64,), 30.0, device=dev), torch.full((64,), 65400.0, device=dev)
    y, y8 = ops_cl.group_norm_act(x, gamma, beta, 8, sink=True)
    back = ops_cl.act8_unpack(y8)
    fine = torch.isfinite(y).reshape(-1, 2, 32).all(dim=2, keepdim=True).expand(-1, 2, 32).reshape(y.shape)  # (blocks without an infinity)
    assert fine.any() and (y[fine] >= 65280).any()
    assert torch.isfinite(back[fine]).all() and torch.isnan(back[~fine]).all()
    assert ((back.double() - y.double())[fine].abs() <= 65504 / 127.5).all()
