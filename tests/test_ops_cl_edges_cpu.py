"""Channels-last layers at the ends of their types' ranges and next to callers' modes (no GPU)."""
import torch

from oracle import ref_cl as R


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
