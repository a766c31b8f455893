"""-m gpu: channels-last layers at the ends of their types' ranges and next to callers' modes, against their definitions in 64 bits (oracle/ref_cl.py).  Tolerances are those of test_ops_cl_gpu.py."""
import pytest
import torch

from oracle import ref_cl as R
from textboxgan_amd import native, ops_cl
from test_ops_cl_gpu import ARITH, SUMS, TYPES, affine, check, ids, train, values

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


# ---------------------------------------------------------------------------------------- group norm
@pytest.mark.parametrize("save", ["input", "act8"])
@pytest.mark.parametrize("act", ["linear", "lrelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
def test_gradients_over_the_whole_range(dev, dtype, act, save):
    """one launch, a block of its own for every sample, and two launches; all groups of one size, and neighbouring groups far apart"""
    for i, (n, s, ch, groups) in enumerate([(1, 40, 64, 4), (3, 30, 48, 12), (3, 700, 64, 4), (2, 1500, 40, 10), (2, 900, 35, 7)]):
        for k in (-60, 60, 73, 100, 120):
            for mixed in (False, True):
                what = f"{n}x{s}x{ch} groups {groups} 2^{k} mixed {mixed}"
                x = values((n, s, ch), torch.float32, dev, 210 + i, 0.2)
                size = torch.full((ch,), 2.0 ** k, device=dev)
                if mixed:
                    size = torch.where(torch.arange(ch, device=dev) // (ch // groups) % 2 == 0, size, 1.0)
                x = (x * size).to(dtype)
                gamma, beta = affine(n, ch, i % 2 == 1, dev)
                dy = values((n, s, ch), dtype, dev, 220 + i, 0.3)
                eps = 1e-5 if k > 0 else 2.0 ** -130
                y, dx, dg, db = train(x, gamma, beta, groups, dy, act=act, save=save, eps=eps)
                o = R.group_norm(x, gamma, beta, groups, act, eps, dy, save)
                check(y, o["y"], o["y_amp"], ARITH, f"{what} y")
                check(dg, o["dgamma"], o["dgamma_amp"], SUMS, f"{what} dgamma")
                check(db, o["dbeta"], o["dbeta_amp"], SUMS, f"{what} dbeta")
                check(dx, o["dx"], o["dx_amp"], SUMS, f"{what} dx")


# ---------------------------------------------------------------------------------------- callers' modes
def test_backward_inside_autocast(dev):
    """the gradients of a dense layer do not hang on an autocast region around the backward pass"""
    for dtype in TYPES:
        x = values((50, 72), dtype, dev, 230).requires_grad_()
        w = (0.1 * values((72, 40), torch.float32, dev, 231)).requires_grad_()
        b = values((40,), torch.float32, dev, 232).requires_grad_()
        dy = values((50, 40), dtype, dev, 233)
        want = torch.autograd.grad(ops_cl.dense_act8(x, w, b, coef=0.5), (x, w, b), dy)
        for low in (torch.float16, torch.bfloat16):
            with torch.autocast("cuda", dtype=low):
                y = ops_cl.dense_act8(x, w, b, coef=0.5)
                got = torch.autograd.grad(y, (x, w, b), dy)
            assert all(torch.equal(u, v) and u.dtype == v.dtype for u, v in zip(got, want)), (dtype, low)


# ---------------------------------------------------------------------------------------- dense layer with a frozen weight
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 8), (3, 5), (7, 33), (33, 64), (255, 72), (257, 256), (1000, 264), (4099, 130), (100000, 72), (50001, 3), (20000, 512), (40, 5000)])
def test_bias_gradient_alone(dev, dtype, rows, cols):
    """the weight is frozen: db is the sum of dy's rows.  (A lane adds at most 64 rows in these cases, then 8 to 256 lanes and 4 to 128 splits are joined:
    SUMS.)"""
    dy = values((rows, cols), dtype, dev, 240)
    x, w = torch.zeros(rows, 4, device=dev, dtype=dtype), torch.zeros(4, cols, device=dev)
    b = torch.zeros(cols, device=dev, requires_grad=True)
    db, = torch.autograd.grad(ops_cl.dense_act8(x, w, b), b, dy)
    assert db.dtype == torch.float32 and torch.equal(db, torch.autograd.grad(ops_cl.dense_act8(x, w, b), b, dy)[0])
    check(db, dy.double().sum(dim=0), dy.double().abs().sum(dim=0), SUMS, "db")


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_bias_gradient_alone_of_slices(dev, dtype):
    wide = values((60, 200), dtype, dev, 241)
    b = torch.zeros(64, device=dev, requires_grad=True)
    x, w = torch.zeros(60, 4, device=dev, dtype=dtype), torch.zeros(4, 64, device=dev)
    for dy in (wide[:, 8:72], wide[:, 1:65], wide[:, :128:2], values((64, 60), dtype, dev, 242).t(), wide[:, :1].expand(60, 64)):
        before = wide.clone()
        db, = torch.autograd.grad(ops_cl.dense_act8(x, w, b), b, dy)
        check(db, dy.double().sum(dim=0), dy.double().abs().sum(dim=0), SUMS, "db")
        assert torch.equal(wide, before)
    none, = torch.autograd.grad(ops_cl.dense_act8(x[:0], w, b), b, wide[:0, :64])
    assert not none.any()


def test_column_sums_write_nothing_outside(dev):
    """the bytes around the result and the workspace stay"""
    lib = native.lib()
    for code, dtype in enumerate(TYPES):
        for rows, cols in ((5, 7), (3000, 33), (700, 264), (9000, 130)):
            x = values((rows, cols), dtype, dev, 243)
            need = lib.tbg_column_sums_workspace_bytes(rows, cols, code)
            buf = torch.full((256 + (4 * cols + 255) // 256 * 256 + 256 + need + 256,), 0x5A, dtype=torch.uint8, device=dev)
            at = 256 + (4 * cols + 255) // 256 * 256 + 256
            native.check(lib.tbg_column_sums(x.data_ptr(), code, rows, cols, cols, buf.data_ptr() + 256, buf.data_ptr() + at, need, native.stream()), "sums")
            out = buf.cpu()
            assert (out[:256] == 0x5A).all() and (out[256 + 4 * cols:at] == 0x5A).all() and (out[at + need:] == 0x5A).all()
            got = out[256:256 + 4 * cols].view(torch.float32)
            check(got.to(dev), x.double().sum(dim=0), x.double().abs().sum(dim=0), SUMS, "sums")


def warmed(call):
    """one call on a side stream first, as a graph's first capture wants it"""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()


def test_no_layer_records_a_memset(dev, tmp_path):
    """memsets in a captured graph are not replayed reliably: forward and backward passes record kernels only"""
    for rows, cin, cout in ((100000, 64, 72), (262144, 128, 128), (5000, 1024, 8)):
        for need in ((0, 0, 1), (1, 0, 1), (1, 1, 1)):
            x, dy = values((2, rows // 2, cin), torch.float32, dev, 250), values((2, rows // 2, cout), torch.float32, dev, 251)
            w, b = 0.1 * values((cin, cout), torch.float32, dev, 252), values((cout,), torch.float32, dev, 253)
            gamma, beta = torch.ones(cin, device=dev), torch.zeros(cin, device=dev)
            leaves = [t.requires_grad_() for t, f in zip((x, w, b), need) if f]

            def call():
                h, h8 = ops_cl.group_norm_act(x, gamma, beta, 8, act="silu", save="act8", sink=True)
                return torch.autograd.grad(ops_cl.dense_act8(h, w, b, x8=h8), leaves, dy)

            warmed(call)
            g = torch.cuda.CUDAGraph(keep_graph=True)  # (to be printed)
            g.enable_debug_mode()
            with torch.cuda.graph(g):
                out = call()
            g.debug_dump(str(tmp_path / "graph.dot"))
            nodes = (tmp_path / "graph.dot").read_text(errors="replace").lower()
            assert "column_sums" in nodes or need[1], need
            assert "memset" not in nodes, (rows, cin, cout, need)
            del out


@pytest.mark.parametrize("need", [(0, 0, 1), (1, 0, 1), (1, 1, 1)])
@pytest.mark.parametrize("rows, cin, cout", [(100000, 64, 72), (5000, 1024, 8), (16, 512, 512)])
def test_captured_dense_layers(dev, rows, cin, cout, need):
    """with the weight frozen or not: a graph's replays answer as eager calls do, with eager work between them"""
    for dtype in (torch.float32, torch.bfloat16):
        x, dy = values((rows, cin), dtype, dev, 250), values((rows, cout), dtype, dev, 251)
        w, b = 0.1 * values((cin, cout), torch.float32, dev, 252), values((cout,), torch.float32, dev, 253)
        leaves = [t.requires_grad_() for t, f in zip((x, w, b), need) if f]
        warmed(lambda: torch.autograd.grad(ops_cl.dense_act8(x, w, b, coef=0.5), leaves, dy))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops_cl.dense_act8(x, w, b, coef=0.5)
            grads = torch.autograd.grad(y, leaves, dy)
        got = [y.detach(), *grads]
        del y
        for k in range(4):
            with torch.no_grad():
                x.copy_(values((rows, cin), dtype, dev, 260 + k))
                dy.copy_(values((rows, cout), dtype, dev, 270 + k))
            g.replay()
            ye = ops_cl.dense_act8(x, w, b, coef=0.5)
            want = [ye.detach(), *torch.autograd.grad(ye, leaves, dy)]
            del ye
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(got, want)), (dtype, k)
