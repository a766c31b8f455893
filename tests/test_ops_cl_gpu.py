"""-m gpu: the channels-last layers (8-bit activation checkpoints, group norm with an activation, dense layer on a checkpoint) against
their definitions in 64 bits (oracle/ref_cl.py).

Tolerances.  A result rounded to type t is off by at most eps(t) / 2 of its value.  Before that rounding the arithmetic is fp32 (statistics
fp64): an element goes through at most 16 roundings of 2^-24, each relative to the magnitude of the terms it is made of (`*_amp`), plus the
exponential's 2^-20: ARITH = 2^-19 of the magnitude.  Sums over positions are accumulated by lanes over at most 64 values in these tests,
then joined in a tree: at most 64 + 32 more roundings of the sum of magnitudes, 2^-17.  Weight gradients: every product is exact in fp32 and
the matrix pipe adds 8 or more products at a time; the tests' chains are at most 2^6 long (512 rows in two terms, 16 rows at a time) in additions
that are off by 2^-23 of the partial sum if they truncate, and partial sums of magnitudes grow to the whole over the chain, half of it on
average: 2^6 2^-1 2^-23 = 2^-18."""
import pytest
import torch

from oracle import ref_cl as R
from textboxgan_amd import native, ops_cl

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None
ARITH, SUMS, WG = 2.0 ** -19, 2.0 ** -17, 2.0 ** -18


def near(got, want, amp, arith, what):
    got, want = got.double(), want.double()
    half = 0.0 if got.dtype is None else torch.finfo(near.dtype).eps / 2
    tol = half * want.abs() * (1 + arith) + arith * (1 + half) * amp + torch.finfo(near.dtype).smallest_normal * torch.finfo(near.dtype).eps
    # what lies beyond the type's largest value by half a step (of eps / 2 of it, at most) or more rounds to an infinity, what lies below stays finite:
    # an infinity of the right sign is due where `want` is beyond it by more than `tol`, allowed where it comes within `tol` of it
    top = torch.finfo(near.dtype).max
    inf = torch.isinf(got) & (got.sign() == want.sign()) & (want.abs() + tol >= top)
    assert (torch.isfinite(got) | inf).all(), what
    over = torch.where(inf, 0.0, (torch.where(inf, 0.0, got) - want).abs() - tol)
    assert over.max() <= 0, f"{what}: {float((got - want).abs().max()):.3g} off, {float((over > 0).double().mean()):.2g} of the values"


def check(got, want, amp, arith, what):
    near.dtype = got.dtype
    near(got, want, amp, arith, what)


def values(shape, dtype, dev, seed, spread=1.0, offset=0.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    ch = shape[-1]
    s = torch.exp(spread * torch.randn(ch, generator=g, device=dev))
    return ((torch.randn(shape, generator=g, device=dev) + offset * torch.randn(ch, generator=g, device=dev)) * s).to(dtype)


# ---------------------------------------------------------------------------------------- 8-bit checkpoints
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (5, 33), (7, 40), (2, 3, 64), (257, 96), (1000, 250), (64, 128), (2, 4096), (33, 7)])
def test_pack_and_unpack(dev, dtype, shape):
    x = values(shape, dtype, dev, 1)
    a = ops_cl.act8_pack(x)
    q, e = R.pack(x)
    assert torch.equal(a.q, q) and torch.equal(a.e, e) and a.shape == shape and a.dtype == dtype
    want = R.unpack(q, e, shape)
    got = ops_cl.act8_unpack(a)
    assert got.dtype == dtype and torch.equal(got.double(), want.to(dtype).double())
    for t in TYPES:
        assert torch.equal(ops_cl.act8_unpack(a, t).double(), want.to(t).double())


def test_pack_special_values(dev):
    f = torch.finfo(torch.float32)
    x = torch.zeros(24, 70)
    rows = [f.max, -f.max, f.max / 2, f.tiny, 1e-45, 2.0 ** -133, 127.5, 127.49999, 127.0, 64.0, 1.9921875, 63.75, float("inf"), -float("inf"), float("nan"),
            2.0 ** -120, 2.0 ** -119, 2.0 ** 127, -0.0]
    for i, v in enumerate(rows):
        x[i, 0], x[i, 5], x[i, 40], x[i, 69] = v, v / 3, v, v / 2
    x[20, :32] = (torch.arange(32) - 16).float() + 0.5   # ties
    x[20, 0] = 127.0
    for t in TYPES:
        v = x.to(t).to(dev)
        a = ops_cl.act8_pack(v)
        q, e = R.pack(v)
        assert torch.equal(a.e, e)
        assert torch.equal(a.q, q)
        want = R.unpack(q, e, v.shape).to(t)
        assert torch.equal(torch.isnan(want), torch.isnan(ops_cl.act8_unpack(a)))
        assert torch.equal(torch.nan_to_num(want.double()), torch.nan_to_num(ops_cl.act8_unpack(a).double()))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_pack_of_slices(dev, dtype):
    wide = values((50, 200), dtype, dev, 2)
    for v in (wide[:, 8:72], wide[:, 1:66], wide[3::2, 16:48], wide[:, ::2], wide.t(), wide.reshape(10, 5, 200)[:, :, 40:104], wide.reshape(10, 5, 200)[:, 1:3, :64],
              wide[:1, 24:88], wide[7]):
        before = v.clone()
        a = ops_cl.act8_pack(v)
        q, e = R.pack(v)
        assert torch.equal(a.q, q) and torch.equal(a.e, e) and torch.equal(v, before)


def test_pack_beyond_32_bit_offsets(dev):
    rows, ch = (1 << 22) + 5, 520
    x = torch.empty(rows, ch, dtype=torch.bfloat16, device=dev).normal_(generator=torch.Generator(device=dev).manual_seed(4))
    a = ops_cl.act8_pack(x)
    y = ops_cl.act8_unpack(a)
    for r in (slice(0, 9), slice(rows - 9, rows), slice(rows // 2, rows // 2 + 9)):
        q, e = R.pack(x[r])
        assert torch.equal(a.q[r], q) and torch.equal(a.e[r], e)
        assert torch.equal(y[r].double(), R.unpack(q, e, x[r].shape))


def test_pack_of_more_rows_than_a_launch_takes(dev):
    """2^30 + 70 rows of one channel: 2^32 lanes and some"""
    rows = (1 << 30) + 70
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    x = torch.ones((rows, 1), dtype=torch.float16, device=dev)
    at = [0, 1, (1 << 29) - 1, 1 << 29, (1 << 30) - 1, 1 << 30, rows - 1]
    for k, r in enumerate(at):
        x[r] = k - 2.5
    a = ops_cl.act8_pack(x)
    q, e = R.pack(x[at])
    assert torch.equal(a.q[at], q) and torch.equal(a.e[at], e)
    assert int(a.q[:, 0].view(-1, 2).eq(64).sum()) >= rows - 2 * len(at)
    back = ops_cl.act8_unpack(a)
    assert torch.equal(back, x)


def test_empty_tensors(dev):
    for shape in ((0, 40), (3, 0, 40)):
        x = torch.zeros(shape, device=dev, dtype=torch.bfloat16)
        a = ops_cl.act8_pack(x)
        assert a.rows == 0 and ops_cl.act8_unpack(a).shape == x.shape
        dw, db = ops_cl.act8_wgrad(a, torch.zeros(*shape[:-1], 8, device=dev))
        assert dw.shape == (40, 8) and not dw.any() and not db.any()
        if len(shape) > 1:
            x.requires_grad_()
            g = torch.ones(40, device=dev, requires_grad=True)
            b = torch.zeros(40, device=dev, requires_grad=True)
            y, y8 = ops_cl.group_norm_act(x, g, b, 4, sink=True)
            dx, dg, db = torch.autograd.grad(y, (x, g, b), torch.zeros_like(y))
            assert y.shape == x.shape and y.dtype == x.dtype and y8.shape == x.shape and not dg.any() and not db.any() and dx.shape == x.shape
    w = torch.zeros(40, 8, device=dev, requires_grad=True)
    y = ops_cl.dense_act8(torch.zeros(0, 40, device=dev), w)
    assert y.shape == (0, 8) and not torch.autograd.grad(y.sum(), w)[0].any()


# ---------------------------------------------------------------------------------------- group norm
SHAPES = [  # N, positions, C, groups
    (1, 1, 1, 1), (2, 1, 8, 8), (1, 1, 64, 2), (2, 3, 32, 32), (3, 5, 24, 8), (1, 7, 33, 11), (2, 17, 40, 5), (2, 100, 96, 3), (4, 64, 128, 32),
    (1, 300, 160, 5), (2, 33, 250, 10), (3, 65, 120, 8), (1, 40, 1024, 1), (1, 9, 2056, 2), (2, 1000, 64, 4), (5, 130, 256, 16), (1, 4097, 48, 6), (300, 2, 16, 2),
    (2, 64, 256, 1), (1, 128, 384, 2), (3, 512, 64, 1), (1, 1024, 32, 4), (2, 1025, 40, 8), (1, 70, 136, 17), (2, 33, 7, 7), (2, 5, 5, 1), (1, 600, 100, 4),
]


def affine(n, ch, per_sample, dev, seed=5):
    g = torch.Generator(device=dev).manual_seed(seed)
    shape = (n, ch) if per_sample else (ch,)
    return 1 + 0.4 * torch.randn(shape, generator=g, device=dev), 0.4 * torch.randn(shape, generator=g, device=dev)


def train(x, gamma, beta, groups, dy, **kw):
    leaves = [t.detach().clone().requires_grad_() for t in (x, gamma, beta)] if x.is_contiguous() else \
        [x.detach().requires_grad_(), gamma.detach().clone().requires_grad_(), beta.detach().clone().requires_grad_()]
    y = ops_cl.group_norm_act(*leaves, groups, **kw)
    out = y[0] if kw.get("sink") else y
    return (y, *torch.autograd.grad(out, leaves, dy))


@pytest.mark.parametrize("save", ["input", "act8"])
@pytest.mark.parametrize("act", ["linear", "lrelu", "silu"])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_group_norm_forward_and_gradients(dev, dtype, act, save):
    for i, (n, s, ch, groups) in enumerate(SHAPES):
        what = f"{n}x{s}x{ch} groups {groups}"
        x = values((n, s, ch), dtype, dev, 10 + i)
        gamma, beta = affine(n, ch, i % 2 == 1, dev)
        dy = values((n, s, ch), dtype, dev, 50 + i, 0.3)
        y, dx, dg, db = train(x, gamma, beta, groups, dy, act=act, save=save)
        o = R.group_norm(x, gamma, beta, groups, act, 1e-5, dy, save)
        assert y.dtype == dtype and dx.dtype == dtype and dg.dtype == db.dtype == torch.float32 and dg.shape == gamma.shape
        check(y, o["y"], o["y_amp"], ARITH, f"{what} y")
        check(dx, o["dx"], o["dx_amp"], SUMS, f"{what} dx")
        check(dg, o["dgamma"], o["dgamma_amp"], SUMS, f"{what} dgamma")
        check(db, o["dbeta"], o["dbeta_amp"], SUMS, f"{what} dbeta")
        with torch.no_grad():
            assert torch.equal(ops_cl.group_norm_act(x, gamma, beta, groups, act=act), y.detach()), f"{what}: without gradients"


@pytest.mark.parametrize("save", ["input", "act8"])
@pytest.mark.parametrize("per_sample", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_group_norm_of_many_small_samples(dev, dtype, per_sample, save):
    """samples that share blocks, some of them taken in turn"""
    for i, (n, s, ch, groups) in enumerate([(700, 1, 256, 8), (1100, 3, 33, 11), (5000, 1, 40, 5), (601, 20, 64, 2), (20000, 1, 32, 1), (2100, 4, 100, 4),
                                            (17001, 2, 256, 8), (700, 7, 1000, 8), (70001, 1, 24, 3), (1030, 9, 520, 1), (800, 3, 130, 130), (3000, 60, 32, 2), (4200, 200, 32, 2)]):
        what = f"{n}x{s}x{ch} groups {groups}"
        x = values((n, s, ch), dtype, dev, 110 + i)
        gamma, beta = affine(n, ch, per_sample, dev)
        dy = values((n, s, ch), dtype, dev, 150 + i, 0.3)
        act = ("linear", "lrelu", "silu")[i % 3]
        y, dx, dg, db = train(x, gamma, beta, groups, dy, act=act, save=save)
        o = R.group_norm(x, gamma, beta, groups, act, 1e-5, dy, save)
        check(y, o["y"], o["y_amp"], ARITH, f"{what} y")
        check(dx, o["dx"], o["dx_amp"], SUMS, f"{what} dx")
        check(dg, o["dgamma"], o["dgamma_amp"], SUMS, f"{what} dgamma")
        check(db, o["dbeta"], o["dbeta_amp"], SUMS, f"{what} dbeta")
        y2, y8 = ops_cl.group_norm_act(x, gamma, beta, groups, act=act, sink=True)
        q, e = R.pack(y2)
        assert torch.equal(y2, y) and torch.equal(y8.q, q) and torch.equal(y8.e, e), what


@pytest.mark.parametrize("ch", [128, 250])
def test_group_norm_of_a_large_tensor(dev, ch):
    """more than the card's caches hold (results are written past them): sample by sample against the definition"""
    n, s = 3, 38400000 // ch
    x = values((n, s, ch), torch.bfloat16, dev, 58)
    gamma, beta = affine(n, ch, True, dev)
    dy = values((n, s, ch), torch.bfloat16, dev, 59, 0.3)
    (y, y8), dx, dg, db = train(x, gamma, beta, 2, dy, act="silu", save="act8", sink=True)
    for i in range(n):
        o = R.group_norm(x[i:i + 1], gamma[i:i + 1], beta[i:i + 1], 2, "silu", 1e-5, dy[i:i + 1], "act8")
        check(y[i:i + 1].detach(), o["y"], o["y_amp"], ARITH, f"{i} y")
        # (a lane's chain: 300000 rows over at most 32 row ranges of 32 rows at a time are 300 values, 5 times the 64 of SUMS, joined as there)
        check(dx[i:i + 1], o["dx"], o["dx_amp"], 5 * SUMS, f"{i} dx")
        check(dg[i:i + 1], o["dgamma"], o["dgamma_amp"], 5 * SUMS, f"{i} dgamma")
        check(db[i:i + 1], o["dbeta"], o["dbeta_amp"], 5 * SUMS, f"{i} dbeta")
        del o
        q, e = R.pack(y[i].detach())
        assert torch.equal(y8.q.view(n, s, -1)[i], q) and torch.equal(y8.e.view(n, s, -1)[i], e)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_group_norm_sink_is_the_outputs_checkpoint(dev, dtype):
    for n, s, ch, groups in SHAPES:
        x = values((n, s, ch), dtype, dev, 3)
        gamma, beta = affine(n, ch, False, dev)
        y, y8 = ops_cl.group_norm_act(x, gamma, beta, groups, act="silu", sink=True)
        q, e = R.pack(y)
        assert torch.equal(y8.q, q) and torch.equal(y8.e, e) and y8.shape == y.shape and y8.dtype == dtype
        z, z8 = train(x, gamma, beta, groups, torch.ones_like(x), act="silu", save="act8", sink=True)[0]
        assert torch.equal(z.detach(), y) and torch.equal(z8.q, q) and torch.equal(z8.e, e)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("save", ["input", "act8"])
def test_group_norm_takes_slices(dev, dtype, save):
    wide = values((4, 30, 3, 200), dtype, dev, 6)
    dwide = values((4, 30, 3, 200), dtype, dev, 7)
    for cut in (lambda t: t[..., 8:72], lambda t: t[..., 1:65], lambda t: t[1:3, ..., 40:104], lambda t: t[:, ::2, :, :64], lambda t: t[::2, :, :, 16:80],
                lambda t: t.permute(0, 2, 1, 3)[..., :64], lambda t: t[:1, :, :, 8:72], lambda t: t[:, 0, 0, :64], lambda t: t[..., :1].expand(4, 30, 3, 64)):
        x, dy = cut(wide), cut(dwide)
        gamma, beta = affine(x.shape[0], 64, True, dev)
        before = wide.clone()
        y, dx, dg, db = train(x, gamma, beta, 4, dy, act="lrelu", save=save)
        y2, dx2, dg2, db2 = train(x.contiguous(), gamma, beta, 4, dy.contiguous(), act="lrelu", save=save)
        o = R.group_norm(x, gamma, beta, 4, "lrelu", 1e-5, dy, save)
        check(y, o["y"], o["y_amp"], ARITH, "y")
        check(dx, o["dx"], o["dx_amp"], SUMS, "dx")
        check(dg, o["dgamma"], o["dgamma_amp"], SUMS, "dgamma")
        check(dx2, o["dx"], o["dx_amp"], SUMS, "dx of the copy")
        assert torch.equal(wide, before)


@pytest.mark.parametrize("act", ["linear", "lrelu", "silu"])
def test_group_norm_far_from_zero(dev, act):
    """a mean of thousands of standard deviations: the statistics lose nothing (ARITH is relative to |mean| rstd)"""
    x = values((2, 500, 64), torch.float32, dev, 8, 0.0) + 3000.0
    gamma, beta = affine(2, 64, False, dev)
    dy = values((2, 500, 64), torch.float32, dev, 9)
    for save in ("input", "act8"):
        y, dx, dg, db = train(x, gamma, beta, 4, dy, act=act, save=save)
        o = R.group_norm(x, gamma, beta, 4, act, 1e-5, dy, save)
        assert (y.double() - o["y"]).abs().max() < 2e-3  # 3000 in fp32 has steps of 2^-12; a sum in 32 bits would be 0.1 off
        check(y, o["y"], o["y_amp"], ARITH, "y")
        if act != "lrelu":  # (values next to the kink may fall on either side)
            check(dx, o["dx"], o["dx_amp"], SUMS, "dx")
            check(dg, o["dgamma"], o["dgamma_amp"], SUMS, "dgamma")


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_group_norm_of_extreme_values(dev, dtype):
    """a position filled with the type's lowest value, and values at both ends of the type's range"""
    for fill in (torch.finfo(dtype).min, torch.finfo(dtype).max / 4, torch.finfo(dtype).tiny):
        x = values((2, 200, 64), dtype, dev, 18)
        x[1, 7] = fill
        if fill > 0:
            x[0] = (x[0].double() / x[0].double().abs().max() * fill).to(dtype)
        gamma, beta = affine(2, 64, False, dev)
        with torch.no_grad():
            y = ops_cl.group_norm_act(x, gamma, beta, 4, act="silu")
        o = R.group_norm(x, gamma, beta, 4, "silu", 1e-5)
        check(y, o["y"], o["y_amp"], ARITH, f"fill {fill}")


def test_group_norm_of_constant_groups(dev):
    for dtype in TYPES:
        x = torch.full((2, 20, 32), 3.0, device=dev, dtype=dtype)
        gamma, beta = affine(2, 32, False, dev)
        for save in ("input", "act8"):
            y, dx, dg, db = train(x, gamma, beta, 4, torch.ones_like(x), act="silu", save=save)
            o = R.group_norm(x, gamma, beta, 4, "silu", 1e-5, torch.ones_like(x), save)
            check(y, o["y"], o["y_amp"], ARITH, "y")
            check(dx, o["dx"], o["dx_amp"], SUMS, "dx")
            assert not dg.any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("save", ["input", "act8"])
def test_group_norm_keeps_bad_values_in_their_group(dev, bad, save):
    for dtype in TYPES:
        x = values((3, 50, 96), dtype, dev, 11)
        gamma, beta = affine(3, 96, True, dev)
        dy = values((3, 50, 96), dtype, dev, 12)
        clean = train(x, gamma, beta, 3, dy, act="silu", save=save)
        x[1, 7, 40] = bad
        dirty = train(x, gamma, beta, 3, dy, act="silu", save=save)
        hit = torch.zeros(3, 1, 96, dtype=torch.bool, device=dev)
        hit[1, 0, 32:64] = True
        for c, d in zip(clean, dirty):
            m = hit.expand(c.shape) if c.dim() == 3 else hit[:, 0]
            assert torch.isnan(d[m]).all() and torch.equal(c[~m], d[~m])


def test_group_norm_gradient_against_differences(dev):
    """along a random direction, in fp32: central differences of the loss, whose third derivative bounds their own error"""
    for act in ("linear", "silu"):
        x = values((2, 40, 48), torch.float32, dev, 13, 0.3)
        gamma, beta = affine(2, 48, False, dev)
        dy = values((2, 40, 48), torch.float32, dev, 14, 0.3)
        _, *grads = train(x, gamma, beta, 6, dy, act=act)
        for i, t in enumerate((x, gamma, beta)):
            v = torch.randn(t.shape, generator=torch.Generator(device=dev).manual_seed(15), device=dev)
            h = 2.0 ** -7
            loss = lambda s: (ops_cl.group_norm_act(*[u + s * v if j == i else u for j, u in enumerate((x, gamma, beta))], 6, act=act).double() * dy.double()).sum()
            diff = (loss(h) - loss(-h)) / (2 * h)
            slope = (grads[i].double() * v.double()).sum()
            size = (grads[i].double().abs() * v.double().abs()).sum()
            # h^2 / 6 times third derivatives of O(10) a value, and 2^-22 of the loss' terms over h
            assert abs(diff - slope) < 2e-3 * size, (act, i, float(diff), float(slope))


def test_runs_repeat_bit_for_bit(dev):
    x = values((4, 700, 128), torch.bfloat16, dev, 16)
    gamma, beta = affine(4, 128, False, dev)
    dy = values((4, 700, 128), torch.bfloat16, dev, 17)
    first = train(x, gamma, beta, 32, dy, act="lrelu", save="act8")
    a = ops_cl.act8_pack(x)
    w1 = ops_cl.act8_wgrad(a, dy)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, train(x, gamma, beta, 32, dy, act="lrelu", save="act8")))
        assert all(torch.equal(p, q) for p, q in zip(w1, ops_cl.act8_wgrad(a, dy)))


# ---------------------------------------------------------------------------------------- weight gradient
WSHAPES = [(1, 1, 1), (1, 32, 8), (3, 33, 5), (31, 64, 64), (32, 65, 72), (100, 128, 128), (129, 200, 72), (500, 17, 300), (1000, 256, 256), (4099, 200, 72),
           (2048, 512, 40), (777, 40, 512), (2000, 520, 264), (300, 1, 1000), (300, 1000, 1),
           (16400, 512, 512), (20011, 384, 264), (16400, 400, 512), (66000, 256, 144)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows, cin, cout", WSHAPES)
def test_wgrad(dev, dtype, rows, cin, cout):
    a = ops_cl.act8_pack(values((rows, cin), torch.float32, dev, 20))
    dy = values((rows, cout), dtype, dev, 21)
    x = R.unpack(a.q, a.e, a.shape)
    for coef, want_db in ((1.0, True), (-0.3, False)):
        dw, db = ops_cl.act8_wgrad(a, dy, coef, want_db)
        ref, rdb, amp, damp = R.wgrad(x, dy, coef)
        check(dw, ref, amp, WG, "dw")
        assert (db is None) == (not want_db)
        if want_db:
            check(db, rdb, damp, SUMS, "db")


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_wgrad_products_are_exact(dev, dtype):
    """one row: every entry is one product of 7 bits by the type's own, so only its rounding to fp32 may show"""
    a = ops_cl.act8_pack(values((1, 96), torch.float32, dev, 22))
    dy = values((1, 80), dtype, dev, 23)
    dw, db = ops_cl.act8_wgrad(a, dy)
    want = R.unpack(a.q, a.e, a.shape).t() @ dy.double()
    assert ((dw.double() - want).abs() <= 3 * 2.0 ** -24 * want.abs()).all()  # three terms are added: two roundings more
    assert torch.equal(db, dy[0].float())


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_wgrad_takes_slices(dev, dtype):
    wide = values((60, 200), dtype, dev, 24)
    a = ops_cl.act8_pack(values((60, 70), torch.bfloat16, dev, 25))
    x = R.unpack(a.q, a.e, a.shape)
    for dy in (wide[:, 8:72], wide[:, 1:66], wide[:, ::2], values((200, 60), dtype, dev, 26).t(), wide[:, :1].expand(60, 24)):
        dw, db = ops_cl.act8_wgrad(a, dy)
        ref, rdb, amp, damp = R.wgrad(x, dy, 1.0)
        check(dw, ref, amp, WG, "dw")
        check(db, rdb, damp, SUMS, "db")
    a3 = ops_cl.Act8(a.q, a.e, (4, 15, 70), a.dtype)
    dw3, _ = ops_cl.act8_wgrad(a3, wide[:, 8:72].reshape(4, 15, 64))
    assert torch.equal(dw3, ops_cl.act8_wgrad(a, wide[:, 8:72])[0])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_wgrad_of_bad_values(dev, dtype):
    """a NaN block of the checkpoint reaches its 32 rows of dw, a bad dy its column; nothing else changes"""
    x = values((40, 96), torch.float32, dev, 27)
    dy = values((40, 24), dtype, dev, 28)
    clean, cdb = ops_cl.act8_wgrad(ops_cl.act8_pack(x), dy)
    x[3, 40] = float("inf")
    for bad in (float("inf"), -float("inf"), float("nan")):
        d = dy.clone()
        d[5, 7] = bad
        dw, db = ops_cl.act8_wgrad(ops_cl.act8_pack(x), d)
        hit = torch.zeros(96, 24, dtype=torch.bool, device=dev)
        hit[32:64] = True
        hit[:, 7] = True
        assert not torch.isfinite(dw[hit]).any() and torch.equal(dw[~hit], clean[~hit])
        assert not torch.isfinite(db[7]) and torch.equal(db[:7], cdb[:7]) and torch.equal(db[8:], cdb[8:])


# ---------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("pos", [(), (5, 9)])
def test_dense_layer(dev, dtype, pos):
    x = values((6, *pos, 72), dtype, dev, 30).requires_grad_()
    w = (0.1 * values((72, 40), torch.float32, dev, 31)).requires_grad_()
    b = values((40,), torch.float32, dev, 32).requires_grad_()
    dy = values((6, *pos, 40), dtype, dev, 33)
    y = ops_cl.dense_act8(x, w, b, coef=0.5)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    xq = R.round_trip(x.detach()).reshape(-1, 72)
    ref, rdb, amp, damp = R.wgrad(xq, dy, 0.5)
    check(dw, ref, amp, WG, "dw")
    check(db, rdb, damp, SUMS, "db")
    # the library products run in x's type on operands of x's type: weight, result and (y only) bias are rounded once each, and the
    # product's 72 (40) terms are added in fp32, each addition rounding by 2^-24 of a partial sum that the sum of magnitudes bounds
    eps = torch.finfo(dtype).eps + 72 * 2.0 ** -24 / 2
    wd, xd = 0.5 * w.detach().double(), x.detach().double()
    yr = xd @ wd + b.detach().double()
    assert ((y.detach().double() - yr).abs() <= 2 * eps * (xd.abs() @ wd.abs() + b.detach().double().abs()) + 1e-7).all()
    dr = dy.double() @ wd.t()
    assert dx.shape == x.shape and ((dx.double() - dr).abs() <= 2 * eps * (dy.double().abs() @ wd.abs().t()) + 1e-7).all()
    with torch.no_grad():
        assert torch.equal(ops_cl.dense_act8(x, w, b, coef=0.5), y)


def block(x, p, save="act8"):
    """norm -> act -> 1x1 -> norm -> act -> 1x1, added to the input: what is kept of the activations is 8 bits wide"""
    h, h8 = ops_cl.group_norm_act(x, p[0], p[1], 8, act="silu", save=save, sink=True)
    h = ops_cl.dense_act8(h, p[2], p[3], coef=0.2, x8=h8)
    h, h8 = ops_cl.group_norm_act(h, p[4], p[5], 4, act="lrelu", save=save, sink=True)
    return x + ops_cl.dense_act8(h, p[6], p[7], coef=0.1, x8=h8)


def block_params(n, ch, mid, dev):
    g = torch.Generator(device=dev).manual_seed(40)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)
    return [t.requires_grad_() for t in (1 + 0.2 * r(ch), 0.2 * r(ch), r(ch, mid), 0.1 * r(mid), 1 + 0.2 * r(n, mid), 0.2 * r(n, mid), r(mid, ch), 0.1 * r(ch))]


def test_a_block_of_them_trains(dev):
    """the whole chain in fp32 against the same chain in 64 bits whose gradients read the same 8-bit values"""
    n, s, ch, mid = 3, 70, 64, 48
    p = block_params(n, ch, mid, dev)
    x = values((n, s, ch), torch.float32, dev, 41, 0.3).requires_grad_()
    dy = values((n, s, ch), torch.float32, dev, 42, 0.3)
    y = block(x, p)
    grads = torch.autograd.grad(y, [x, *p], dy)
    d = [t.detach().double() for t in p]
    xd = x.detach()
    f1 = R.group_norm(xd, p[0].detach(), p[1].detach(), 8, "silu", 1e-5)["y"]
    h1 = 0.2 * (f1 @ d[2]) + d[3]
    f2 = R.group_norm(h1.float(), p[4].detach(), p[5].detach(), 4, "lrelu", 1e-5)["y"]
    yr = xd.double() + 0.1 * (f2 @ d[6]) + d[7]
    close = lambda a, b, tol, what: (_ for _ in ()).throw(AssertionError(f"{what}: {float((a.double() - b).norm() / b.norm()):.3g}")) if (a.double() - b).norm() > tol * b.norm() else None
    close(y.detach(), yr, 1e-5, "y")
    g2 = 0.1 * (dy.double() @ d[6].t())
    w2, b2, _, _ = R.wgrad(R.round_trip(f2.float()), dy, 0.1)
    o2 = R.group_norm(h1.float(), p[4].detach(), p[5].detach(), 4, "lrelu", 1e-5, g2, "act8")
    g1 = 0.2 * (o2["dx"] @ d[2].t())
    w1, b1, _, _ = R.wgrad(R.round_trip(f1.float()), o2["dx"], 0.2)
    o1 = R.group_norm(xd, p[0].detach(), p[1].detach(), 8, "silu", 1e-5, g1, "act8")
    want = [dy.double() + o1["dx"], o1["dgamma"], o1["dbeta"], w1, b1, o2["dgamma"], o2["dbeta"], w2, b2]
    # a value on the border between two 8-bit steps may fall to either side: 2^-24 of its size next to steps of 2^-6, some 1e-4 of the values,
    # each off by one step of about 1 / 100: 1e-4 in the 2-norm
    for i, (a, b) in enumerate(zip(grads, want)):
        close(a, b, 3e-4, f"gradient {i}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=ids)
def test_a_block_keeps_eight_bits(dev, dtype):
    """what the graph holds between forward and backward, and how far 8 bits move the gradients"""
    n, s, ch, mid = 2, 4096, 128, 128
    p = block_params(n, ch, mid, dev)
    x = values((n, s, ch), dtype, dev, 43, 0.3).requires_grad_()
    dy = values((n, s, ch), dtype, dev, 44, 0.3)
    got = {}
    for save in ("input", "act8"):
        y = block(x, p, save)
        got[save] = torch.autograd.grad(y, [x, *p], dy)
    for a, b in zip(got["act8"], got["input"]):
        # a step of amax / 64 to amax / 127.5 in blocks of 32: errors of at most amax / 127.5 (rms a third to a half of that) beside values of
        # rms about amax / 2.5
        assert (a.double() - b.double()).norm() <= 0.03 * b.double().norm()
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        y = block(x, p)
    big = [t for t in {t.data_ptr(): t for t in kept}.values() if t.numel() >= n * s * ch // 32]
    assert all(t.dtype in (torch.int8, torch.uint8) for t in big) and sum(t.numel() * t.element_size() for t in big) <= 4 * n * s * ch * 33 // 32


def test_captured_and_replayed(dev):
    """forward and backward in one graph, replayed with new inputs between eager runs of the same and of other sizes"""
    p = block_params(2, 64, 48, dev)
    static_x = values((2, 300, 64), torch.bfloat16, dev, 50).requires_grad_()
    static_dy = values((2, 300, 64), torch.bfloat16, dev, 51)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            out = torch.autograd.grad(block(static_x, p), [static_x, *p], static_dy)
    del out
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = block(static_x, p)
            grads = torch.autograd.grad(y, [static_x, *p], static_dy)
        graphs.append((g, y.detach(), grads))
        del y
    for k in range(4):
        x, dy = values((2, 300, 64), torch.bfloat16, dev, 60 + k), values((2, 300, 64), torch.bfloat16, dev, 70 + k)
        with torch.no_grad():
            static_x.copy_(x)
            static_dy.copy_(dy)
        for g, *_ in graphs:
            g.replay()
        other = ops_cl.act8_unpack(ops_cl.act8_pack(values((64, 300), torch.float32, dev, 80 + k)))
        torch.cuda.synchronize()
        got = [(a.clone(), [t.clone() for t in b]) for _, a, b in graphs]
        xe = x.clone().requires_grad_()
        ye = block(xe, p)
        ge = torch.autograd.grad(ye, [xe, *p], dy)
        for a, b in got:
            assert torch.equal(a, ye.detach()) and all(torch.equal(u, v) for u, v in zip(b, ge)), k
        assert torch.isfinite(other).all()


def test_a_backward_pass_is_not_captured_over_an_eager_graph(dev):
    """leaves that an eager graph of the default stream holds: the capture is refused while it lives, and works once it is gone"""
    p = block_params(1, 64, 32, dev)
    x, dy = values((1, 50, 64), torch.bfloat16, dev, 52), values((1, 50, 64), torch.bfloat16, dev, 53)
    want = torch.autograd.grad(block(x, p), p, dy)
    eager = block(x, p)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(native.TbgError, match="is alive"):
        with torch.cuda.graph(g):
            block(x, p)
    with torch.no_grad():  # no backward pass: nothing to refuse
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = block(x, p)
    g.replay()
    assert torch.equal(y, eager.detach())
    del eager
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        grads = torch.autograd.grad(block(x, p), p, dy)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_checkpoints_are_no_part_of_a_graph(dev):
    """operands that want gradients, contiguous and not"""
    x, dy = values((40, 96), torch.float32, dev, 56).requires_grad_(), values((40, 64), torch.float32, dev, 57).requires_grad_()
    for xs, ds in ((x, dy), (x[:, 1:34], dy[:, 3:20]), (x.t()[:40].t(), dy.t()[:8].t())):
        a = ops_cl.act8_pack(xs)
        dw, db = ops_cl.act8_wgrad(a, ds)
        y = ops_cl.act8_unpack(a)
        assert not any(t.requires_grad for t in (a.q, a.e, dw, db, y))
        w, b = ops_cl.act8_wgrad(ops_cl.act8_pack(xs.detach().contiguous()), ds.detach().contiguous())
        assert torch.equal(dw, w) and torch.equal(db, b)


def test_under_autocast(dev):
    """types are the operands' own, whatever the caller's autocast"""
    p = block_params(2, 64, 48, dev)
    for dtype in (torch.float32, torch.bfloat16):
        x, dy = values((2, 30, 64), dtype, dev, 54), values((2, 30, 64), dtype, dev, 55)
        want_y = block(x, p)
        want = torch.autograd.grad(want_y, p, dy)
        with torch.autocast("cuda", dtype=torch.float16):
            y = block(x, p)
        got = torch.autograd.grad(y, p, dy)
        assert y.dtype == dtype and torch.equal(y, want_y) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_weight_gradients(dev):
    """every form of the weight gradient in a graph, replayed with new inputs between eager calls"""
    cases = [(values((r, i), torch.float32, dev, 100 + k), values((r, o), t, dev, 110 + k)) for k, (r, i, o, t) in enumerate(
        [(16400, 512, 512, torch.bfloat16), (9000, 256, 200, torch.float32), (5000, 70, 130, torch.float16), (40, 33, 7, torch.float32)])]
    static = [(ops_cl.act8_pack(x), dy.clone()) for x, dy in cases]
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = [ops_cl.act8_wgrad(a, dy) for a, dy in static]
    for k in range(3):
        for (a, dy), (x, y) in zip(static, cases):
            new = ops_cl.act8_pack(x * (1 + k))
            a.q.copy_(new.q)
            a.e.copy_(new.e)
            dy.copy_(y * (2 - k))
        g.replay()
        want = [ops_cl.act8_wgrad(a, dy) for a, dy in static]
        torch.cuda.synchronize()
        for got, ref in zip(out, want):
            assert all(torch.equal(u, v) for u, v in zip(got, ref)), k


def test_on_another_stream(dev):
    x = values((4, 2000, 128), torch.bfloat16, dev, 90)
    gamma, beta = affine(4, 128, False, dev)
    dy = values((4, 2000, 128), torch.bfloat16, dev, 91)
    want = train(x, gamma, beta, 32, dy, act="silu", save="act8")
    want_w = ops_cl.act8_wgrad(ops_cl.act8_pack(x), dy)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for st in (a, b, a, b):
        with torch.cuda.stream(st):
            got.append((train(x, gamma, beta, 32, dy, act="silu", save="act8"), ops_cl.act8_wgrad(ops_cl.act8_pack(x), dy)))
    torch.cuda.synchronize()
    for t, w in got:
        assert all(torch.equal(u, v) for u, v in zip(t, want)) and all(torch.equal(u, v) for u, v in zip(w, want_w))


def test_nothing_is_written_outside(dev):
    """results land in their own memory only: the bytes around them stay (C entries on slices of a guarded buffer)"""
    lib, ld = native.lib(), native
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 2)):
        for n, s, ch, groups in ((2, 7, 40, 5), (1, 5, 33, 11), (3, 9, 160, 5), (1, 3, 250, 10), (2, 11, 64, 4), (1, 700, 33, 3), (601, 2, 7, 7)):
            nb, rows = (ch + 31) // 32, n * s
            x, dy = values((n, s, ch), dtype, dev, 95), values((n, s, ch), dtype, dev, 96)
            gamma, beta = affine(n, ch, False, dev)
            sizes = {"y": rows * ch * x.element_size(), "q": rows * nb * 32, "e": rows * nb, "yq": rows * nb * 32, "ye": rows * nb, "stats": n * groups * 16,
                     "dx": rows * ch * x.element_size(), "dg": ch * 4, "db": ch * 4, "dw": ch * ch * 4, "dwb": ch * 4}
            d = ld.GnDesc(s * ch, ch, s * ch, ch, n, s, ch, groups, code, 2, 0, 1e-5)
            ref = __import__("ctypes").byref(d)
            sizes["wf"], sizes["wb"] = lib.tbg_group_norm_workspace_bytes(ref, 0), lib.tbg_group_norm_workspace_bytes(ref, 1)
            sizes["ww"] = max(16, lib.tbg_act8_wgrad_workspace_bytes(rows, ch, ch, code))
            at, total = {}, 256
            for k, b in sizes.items():
                at[k] = total
                total += (b + 255) // 256 * 256 + 256
            buf = torch.full((total,), 0x5A, dtype=torch.uint8, device=dev)
            P = lambda k: buf.data_ptr() + at[k]
            st = ld.stream()
            ld.check(lib.tbg_group_norm_fwd(ref, x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), P("y"), P("stats"), P("q"), P("e"), P("yq"), P("ye"), P("wf"), sizes["wf"], st), "fwd")
            ld.check(lib.tbg_group_norm_bwd(ref, None, P("q"), P("e"), dy.data_ptr(), gamma.data_ptr(), beta.data_ptr(), P("stats"), P("dx"), P("dg"), P("db"), P("wb"), sizes["wb"], st), "bwd")
            ld.check(lib.tbg_act8_wgrad(P("yq"), P("ye"), dy.data_ptr(), code, rows, ch, ch, ch, 1.0, P("dw"), P("dwb"), P("ww"), sizes["ww"], st), "wgrad")
            out = buf.cpu()
            for k, b in sizes.items():
                assert (out[at[k] - 256:at[k]] == 0x5A).all() and (out[at[k] + b:at[k] + (b + 255) // 256 * 256 + 256] == 0x5A).all(), (k, ch, dtype)
            y, dx, dg, db = train(x, gamma, beta, groups, dy, act="silu", save="act8")
            got = out[at["dx"]:at["dx"] + sizes["dx"]].view(dtype).reshape(dx.shape)
            assert torch.equal(got, dx.cpu())
