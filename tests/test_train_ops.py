"""The training operators (commux_b200.ops.train) against their formulas in 64
bits, and their gradients against differences.

A result may be off by its own rounding, u |want| with u half a unit of its
type, and by the 32-bit arithmetic before it: c 2^-24 times the sum of the
magnitudes that the formula adds up, where c bounds the roundings on the
longest path from an input to the result (stated at each test)."""

import math

import pytest
import torch

from commux_b200 import ops

gpu = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # absolute, near zero
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def close(got, want, mag, c, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    tol = U[got.dtype] * want.abs() * 1.01 + c * 2.0 ** -24 * mag + LEAST[got.dtype]
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol)[bad].max()):.3g} "
                           f"times the tolerance")


def held64(x):
    """Values of the 8-bit form of 64-bit rows, by its definition."""
    x = x.double()
    n, d = x.shape
    v = torch.nn.functional.pad(x, (0, -d % 32)).view(n, -1, 32)
    big = v.abs().amax(2, keepdim=True)
    e = torch.full_like(big, -126.0)
    for _ in range(3):  # the smallest that fits, from below
        e = torch.maximum(e, torch.ceil(torch.log2(big / 127)).nan_to_num(neginf=-126.0, posinf=0.0) - 1)
    while True:
        grow = (127 * torch.exp2(e) < big) & big.isfinite()
        if not grow.any():
            break
        e = e + grow
    s = torch.exp2(e)
    q = torch.round(v / s)
    q = torch.where(e == 122, q.clamp(-63, 63), q)  # 64 * 2^122 is no fp32 value: finite values stay finite
    out = torch.where(big.isfinite(), q * s, math.nan)
    return out.view(n, -1)[:, :d]


# --- layer norm --------------------------------------------------------------

def norm64(x, w, b, eps=1e-5):
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    h = (x - mean) * rstd
    size = (x.abs() + x.abs().mean(1, keepdim=True)) * rstd  # of what h is a difference of
    return h, rstd, h * w + (b if b is not None else 0), size


NORM_TYPES = [(F32, F32, F32, F32), (F32, BF16, F32, BF16), (BF16, BF16, BF16, BF16), (F16, F16, F32, F16),
              (F32, F32, F32, BF16), (BF16, F32, F16, F32)]  # x, y, weight, residual


@gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 768), (3, 31), (5, 33), (257, 768), (64, 1000), (33, 1001),
                                       (7, 4096), (5, 5003), (3, 8192), (2, 20011), (2, 40000), (1300, 8),
                                       (900, 200), (1100, 2056), (700, 4100), (650, 6001)])
@pytest.mark.parametrize("xt,yt,wt,rt", NORM_TYPES)
@pytest.mark.parametrize("residual,pack", [(False, False), (True, False), (False, True), (True, True)])
def test_layer_norm(rows, cols, xt, yt, wt, rt, residual, pack):
    # longest paths: a row's sum (cols / 32 terms a lane at most, 16 for the
    # wide rows' blocks, then 10 joins), twice; a column's sum over <= 1300 rows
    g = gen(rows * 7 + cols)
    x = randn(g, rows, cols, dtype=xt, scale=3.0).add_(1.0).requires_grad_()
    r = randn(g, rows, cols, dtype=rt).requires_grad_() if residual else None
    w = (1 + 0.3 * randn(g, cols)).to(wt).requires_grad_()
    b = randn(g, cols, dtype=wt).requires_grad_()
    got = ops.layer_norm(x, w, b, residual=r, out_dtype=yt, pack=pack)
    got = got if isinstance(got, tuple) else (got,)
    y, s = got[0], got[1] if residual else x
    x64 = x.detach().double()
    if residual:
        close(s.detach(), x64 + r.detach().double(), (x64.abs() + r.detach().double().abs()), 1, "s")
        x64 = s.detach().double()
    c = 96 + cols / 512
    h, rstd, want, size = norm64(x64, w.detach().double(), b.detach().double())
    close(y.detach(), want, size * w.detach().double().abs() + b.detach().double().abs(), c, "y")
    dy, ds = randn(g, rows, cols, dtype=yt), randn(g, rows, cols, dtype=xt) if residual else None
    if pack:
        kept = got[-1]
        assert kept.nbytes == rows * (-(-cols // 32)) * 33
        v = ops.Act8(kept.q, kept.scale, kept.shape, F32).unpack().double()
        step = torch.exp2(kept.scale.double() - 127).repeat_interleave(32, 1)[:, :cols]
        # half a step from h as computed in 32 bits
        assert ((v - h).abs() <= step / 2 + c * 2.0 ** -24 * size).all()
        big = torch.nn.functional.pad(h.abs(), (0, -cols % 32)).view(rows, -1, 32).amax(2)
        top = torch.exp2(kept.scale.double() - 127) * 127
        err = c * 2.0 ** -24 * torch.nn.functional.pad(size, (0, -cols % 32)).view(rows, -1, 32).amax(2)
        assert ((top + err >= big) & ((top / 2 <= big + err) | (kept.scale == 1))).all()
        close(kept.unpack().detach(), v * w.detach().double() + b.detach().double(),
              v.abs() * w.detach().double().abs() + b.detach().double().abs(), 2, "unpacked")
        h, size = v, torch.maximum(size, v.abs())
    ins = [t for t in (x, r, w, b) if t is not None]
    grads = torch.autograd.grad([y, s] if residual else [y], ins, [dy, ds] if residual else [dy])
    dx, dw, db = grads[0], grads[-2], grads[-1]
    gy = dy.double() * w.detach().double()
    c2 = (gy * h).mean(1, keepdim=True)
    want = rstd * (gy - gy.mean(1, keepdim=True) - h * c2)
    mag = rstd * (gy.abs() + gy.abs().mean(1, keepdim=True) + size * (gy.abs() * size).mean(1, keepdim=True))
    if residual:
        want, mag = want + ds.double(), mag + ds.double().abs()
        close(grads[1], want, mag, 2 * c, "dr")
    close(dx, want, mag, 2 * c, "dx")
    close(dw, (dy.double() * h).sum(0), (dy.double().abs() * size).sum(0), 2 * c + 256, "dw")
    close(db, dy.double().sum(0), dy.double().abs().sum(0), 256, "db")


@gpu
@pytest.mark.parametrize("pack", [False, True])
def test_layer_norm_optional_parts(pack):
    g = gen(1)
    x, w = randn(g, 5, 7, 96).requires_grad_(), randn(g, 96).requires_grad_()
    r = randn(g, 5, 7, 96)
    out = ops.layer_norm(x, w, pack=pack)
    y = out[0] if pack else out
    h, _, want, size = norm64(x.detach().double().view(35, 96), w.detach().double(), None)
    close(y.detach().view(35, 96), want, size * w.detach().double().abs(), 96, "no bias")
    # only some gradients wanted
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y), retain_graph=True)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert dw.shape == w.shape and dx.shape == x.shape
    # only the stream used, only the norm used
    y, s = ops.layer_norm(x, w, residual=r)
    (dx,) = torch.autograd.grad(s, x, torch.full_like(s, 2.0))
    assert torch.equal(dx, torch.full_like(x, 2.0))
    y, s = ops.layer_norm(x, w, residual=r)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    y2 = ops.layer_norm((x + r).detach().requires_grad_(), w)
    assert torch.equal(y, y2)
    # no graph: nothing kept, the same values
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, residual=r)[0], y)


@gpu
@pytest.mark.parametrize("cols", [768, 77])
def test_layer_norm_constant_and_far_rows(cols):
    # a constant row has no variance: y is the bias; a mean 1000 times the
    # deviation costs log2(1000) of the 24 bits and no more
    w, b = torch.full((cols,), 2.0, device="cuda"), torch.full((cols,), 0.5, device="cuda")
    x = torch.full((4, cols), 3.0, device="cuda")
    assert torch.equal(ops.layer_norm(x, w, b), torch.full_like(x, 0.5))
    x = randn(gen(2), 64, cols) + 1000.0
    _, _, want, size = norm64(x.double(), w.double(), b.double())
    close(ops.layer_norm(x, w, b), want, size * 2 + 0.5, 96, "far")
    x[1, 3] = math.nan
    x[2, 5] = math.inf
    y = ops.layer_norm(x, w, b)
    assert y[1:3].isnan().all() and y[0].isfinite().all() and y[3:].isfinite().all()
    _, kept = ops.layer_norm(x, w, b, pack=True)
    v = kept.unpack()
    assert v[1:3].isnan().all() and v[3:].isfinite().all()


# --- 8-bit form --------------------------------------------------------------

@gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 31), (3, 32), (5, 33), (129, 768), (17, 1001), (4, 4096), (0, 64)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_pack8_is_the_definition(rows, cols, dtype):
    g = gen(cols)
    x = randn(g, rows, cols, dtype=dtype) * torch.exp(2 * randn(g, rows, 1)).to(dtype)
    kept = ops.pack8(x)
    assert kept.q.shape == (rows, -(-cols // 32) * 32) and kept.scale.shape == (rows, -(-cols // 32))
    if rows == 0:
        assert kept.unpack().shape == x.shape
        return
    want = held64(x.double())
    assert torch.equal(kept.unpack(F32).double(), want)
    assert torch.equal(kept.unpack(BF16).double(), want)  # 7 bits: bf16 holds them all
    assert kept.unpack().dtype == dtype
    pad = kept.q[:, cols:]
    assert not pad.any()


@gpu
def test_pack8_edges():
    big = torch.finfo(F32).max
    rows = [
        [0.0] * 4,
        [127.0, -127.0, 1.0, 0.5],  # the last that step 1 holds; ties go to the even value
        [127.00001, 1.0, -1.0, 3.0],  # one more: step 2
        [big, -big, big / 254, 0.0],
        [2.0 ** -149, 2.0 ** -126, 0.0, -2.0 ** -127],  # below the least step
        [127 * 2.0 ** -126, 2.0 ** -126, 0.6 * 2.0 ** -126, 0.0],
        [math.inf, 1.0, 2.0, 3.0],
        [math.nan, 1.0, 2.0, -math.inf],
        [-128.0, 64.0, 1.0, 2.5],
    ]
    x = torch.tensor(rows, device="cuda")
    kept = ops.pack8(x)
    got, want = kept.unpack().double(), held64(x.double())
    assert torch.equal(got[:6], want[:6]) and torch.equal(got[8], want[8])
    assert got[6:8].isnan().all() and kept.scale[6:8].eq(255).all()
    assert kept.q.min() >= -127
    # float16 too: 65504 is held as 2^16
    x = torch.tensor([[65504.0, -65504.0, 1.0]], device="cuda", dtype=F16)
    assert torch.equal(ops.pack8(x).unpack()[:, :2], x[:, :2])
    # only the group with the infinity is lost
    x = torch.ones(1, 96, device="cuda")
    x[0, 40] = math.inf
    v = ops.pack8(x).unpack()
    assert v[0, 32:64].isnan().all() and v[0, :32].eq(1).all() and v[0, 64:].eq(1).all()


def _orders(x):
    """The same matrix in other orders: rows apart, shifted, transposed, repeated."""
    n, d = x.shape
    wide = torch.zeros(n, d + 24, dtype=x.dtype, device="cuda")
    wide[:, 8:8 + d] = x
    odd = torch.zeros(n, d + 5, dtype=x.dtype, device="cuda")
    odd[:, 3:3 + d] = x
    flat = torch.zeros(n * d + 1, dtype=x.dtype, device="cuda")
    flat[1:] = x.reshape(-1)
    return {"apart": wide[:, 8:8 + d], "odd": odd[:, 3:3 + d], "shifted": flat[1:].view(n, d),
            "transposed": x.t().contiguous().t()}


@gpu
@pytest.mark.parametrize("cols", [64, 768, 1000, 77])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_other_orders_give_the_same(cols, dtype):
    g = gen(3)
    x, dy = randn(g, 37, cols, dtype=dtype), randn(g, 37, cols, dtype=dtype)
    w, b = randn(g, cols), randn(g, cols)
    target = torch.randint(0, cols, (37,), generator=g, device="cuda")

    def everything(x, dy):
        x = x.detach().requires_grad_()
        y, s, kept = ops.layer_norm(x, w, b, residual=dy, pack=True)
        z = ops.gelu8(x)
        loss = ops.cross_entropy(x, target)
        p = ops.pack8(x)
        out = [y, s, kept.q, kept.scale, z, loss, p.q, p.scale, ops.weight_grad8(dy, p)]
        out += torch.autograd.grad([y, z, loss], x, [dy, dy, torch.ones((), device="cuda")])
        return [t.detach() for t in out]

    want = everything(x, dy)
    for name, other in _orders(x).items():
        for k, (u, v) in enumerate(zip(everything(other, _orders(dy)[name]), want)):
            if u.dtype.is_floating_point:  # another order may take another path through a sum
                assert torch.allclose(u.float(), v.float(), rtol=2 * U[u.dtype], atol=4e-6 * float(v.abs().max())), \
                    (name, k)
            else:
                assert (u != v).double().mean() < 1e-3, (name, k)
    one = x[:1].expand(5, cols)  # rows at distance zero
    assert torch.equal(ops.pack8(one).q, ops.pack8(one.contiguous()).q)
    assert torch.equal(ops.layer_norm(one, w, b), ops.layer_norm(one.contiguous(), w, b))


# --- GELU --------------------------------------------------------------------

def gelu64(x, form):
    if form == "tanh":
        u = math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
        sig = torch.sigmoid(2 * u)
        return x * sig, sig + x * sig * (1 - sig) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x ** 2)
    cdf = 0.5 * torch.erfc(-x / math.sqrt(2))
    return x * cdf, cdf + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)


@gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 33), (16, 3072), (129, 768), (31, 1000), (9, 10001), (0, 32)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("form", ["tanh", "none"])
@pytest.mark.parametrize("pack", [False, True])
def test_gelu8(rows, cols, dtype, form, pack):
    # a dozen roundings; the exponent's own error is a few of them times an
    # argument z whose weight sigmoid(-z) z stays under 0.3
    g = gen(cols + rows)
    x = randn(g, rows, cols, dtype=dtype, scale=2.0).requires_grad_()
    dy = randn(g, rows, cols, dtype=dtype)
    got = ops.gelu8(x, approximate=form, pack=pack)
    y, kept = got if pack else (got, None)
    x64 = x.detach().double()
    close(y.detach(), gelu64(x64, form)[0], x64.abs(), 16, "y")
    (dx,) = torch.autograd.grad(y, x, dy)
    if rows == 0:
        assert dx.shape == x.shape
        return
    h = held64(x64)
    slope = gelu64(h, form)[1]
    close(dx, dy.double() * slope, dy.double().abs() * (1 + h.abs()), 32, "dx")
    if pack:
        v = kept.unpack(F32).double()
        step = torch.exp2(kept.scale.double() - 127).repeat_interleave(32, 1)[:, :cols]
        assert ((v - gelu64(x64, form)[0]).abs() <= step / 2 + 16 * 2.0 ** -24 * x64.abs()).all()


@gpu
@pytest.mark.parametrize("form", ["tanh", "none"])
def test_gelu8_extremes(form):
    x = torch.tensor([[0.0, -0.0, 30.0, -30.0, 1e4, -1e4, 3e38, -3e38]], device="cuda")
    y = ops.gelu8(x, approximate=form)
    assert torch.equal(y, torch.tensor([[0.0, 0.0, 30.0, 0.0, 1e4, 0.0, 3e38, 0.0]], device="cuda"))
    for v in (1e4, 1e19, 3e38):
        x = torch.full((1, 32), v, device="cuda")
        x[0, ::2] *= -1
        x.requires_grad_()
        (dx,) = torch.autograd.grad(ops.gelu8(x, approximate=form).nan_to_num().sum(), x)
        assert torch.equal(dx, (x > 0).float()), v
    x = torch.zeros(1, 64, device="cuda")
    x[0, 3] = math.nan
    x.requires_grad_()
    y = ops.gelu8(x, approximate=form)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert dx[0, :32].isnan().all() and dx[0, 32:].eq(0.5).all()


# --- weight gradient ---------------------------------------------------------

@gpu
@pytest.mark.parametrize("rows,cols,outs", [(1, 1, 1), (1, 100, 61), (37, 100, 61), (64, 256, 128), (65, 257, 129),
                                            (63, 255, 127), (200, 768, 384), (1024, 128, 1000), (130, 2049, 40),
                                            (4096, 64, 64), (2500, 33, 7), (513, 300, 520), (0, 40, 24)])
@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16), (F16, F32), (F32, BF16)])
def test_weight_grad8(rows, cols, outs, dtype, out):
    # a product of exact factors, at most `rows` roundings in its sum
    g = gen(rows + cols + outs)
    x = randn(g, rows, cols, dtype=dtype) * torch.exp(randn(g, cols)).to(dtype)
    dy = randn(g, rows, outs, dtype=dtype) * torch.exp(randn(g, rows, 1)).to(dtype)
    kept = ops.pack8(x)
    dw, db = ops.weight_grad8(dy, kept, bias=True, out_dtype=out)
    assert dw.dtype == out and torch.equal(dw, ops.weight_grad8(dy, kept, out_dtype=out))
    v = kept.unpack(F32).double() if rows else x.double()
    close(dw, dy.double().t() @ v, dy.double().abs().t() @ v.abs(), rows + 64, "dw")
    close(db, dy.double().sum(0), dy.double().abs().sum(0), rows + 64, "db")


@gpu
@pytest.mark.parametrize("rows,cols,outs,out", [(4000, 2050, 9000, F32), (2000, 2100, 9000, BF16),
                                                (6000, 700, 1500, F32)])
@pytest.mark.parametrize("after_norm", [False, True])
def test_weight_grad8_many_tiles(rows, cols, outs, out, after_norm):
    # tiles that one pair holds whole, tiles that several share, and sums that are cut
    g = gen(rows)
    x, dy = randn(g, rows, cols, dtype=BF16), randn(g, rows, outs, dtype=BF16)
    w, b = (1 + 0.2 * randn(g, cols), randn(g, cols)) if after_norm else (None, None)
    kept = ops.layer_norm(x, w, b, pack=True)[1] if after_norm else ops.pack8(x)
    dw, db = ops.weight_grad8(dy, kept, bias=True, out_dtype=out)
    v = ops.Act8(kept.q, kept.scale, kept.shape, F32).unpack().double()
    mag = v.abs()
    if after_norm:
        v, mag = v * w.double() + b.double(), mag * w.double().abs() + b.double().abs()
    close(dw, dy.double().t() @ v, dy.double().abs().t() @ mag, rows + 64, "dw")
    close(db, dy.double().sum(0), dy.double().abs().sum(0), rows + 64, "db")
    if out == F32 and not after_norm:
        # A sum of 16 tokens' products is cut off, not rounded, when it is added to
        # the others: half a unit (2^-24 to 2^-25 of the sum) each on average, over
        # 96 additions at most. Twice that holds the error's norm.
        off = (dw.double() - dy.double().t() @ v).norm() / (dy.double().t() @ v).norm()
        assert float(off) <= 2 * 96 * 2.0 ** -24.5, float(off)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("with_bias", [False, True])
def test_weight_grad8_after_a_norm(dtype, with_bias):
    g = gen(11)
    x = randn(g, 300, 200, dtype=dtype)
    w, b = randn(g, 200), randn(g, 200) if with_bias else None
    y, kept = ops.layer_norm(x, w, b, pack=True)
    dy = randn(g, 300, 150, dtype=dtype)
    dw, db = ops.weight_grad8(dy, kept, bias=True, out_dtype=F32)
    h = ops.Act8(kept.q, kept.scale, kept.shape, F32).unpack().double()
    v = h * w.double() + (b.double() if with_bias else 0)
    mag = dy.double().abs().t() @ (h.abs() * w.double().abs() + (b.double().abs() if with_bias else 0))
    close(dw, dy.double().t() @ v, mag, 400, "dw")
    close(db, dy.double().sum(0), dy.double().abs().sum(0), 364, "db")


@gpu
def test_weight_grad8_wide_range():
    # fp32 and fp16 gradients keep all their bits, large and small; a NaN or an
    # infinity reaches the entries that its row and column meet, and no others
    g = gen(5)
    x = randn(g, 96, 64)
    for dtype, lo, hi in ((F32, 2.0 ** -60, 2.0 ** 60), (F16, 2.0 ** -20, 2.0 ** 8), (BF16, 2.0 ** -60, 2.0 ** 60)):
        dy = randn(g, 96, 48)
        dy[:, ::2] *= lo
        dy[:, 1::2] *= hi
        dy = dy.to(dtype)
        kept = ops.pack8(x)
        v = kept.unpack(F32).double()
        close(ops.weight_grad8(dy, kept, out_dtype=F32), dy.double().t() @ v, dy.double().abs().t() @ v.abs(), 160)
    for bad in (math.nan, math.inf, -math.inf):
        for dtype in (F32, BF16, F16):
            dy = randn(g, 96, 48, dtype=dtype)
            dy[7, 5] = bad
            dw = ops.weight_grad8(dy, ops.pack8(x))
            assert not dw[5].isfinite().any() and dw[:5].isfinite().all() and dw[6:].isfinite().all()
    x[9, 40] = math.inf
    dw = ops.weight_grad8(randn(g, 96, 48, dtype=BF16), ops.pack8(x))
    assert dw[:, 32:].isnan().all() and dw[:, :32].isfinite().all()


@gpu
@pytest.mark.parametrize("dtype,wt", [(BF16, F32), (F32, F32), (F16, F16)])
@pytest.mark.parametrize("given", [False, True])
def test_linear8(dtype, wt, given):
    g = gen(21)
    x = randn(g, 3, 50, 96, dtype=dtype).requires_grad_()
    w, b = randn(g, 40, 96, dtype=wt).requires_grad_(), randn(g, 40, dtype=wt).requires_grad_()
    dy = randn(g, 3, 50, 40, dtype=dtype)
    kept = ops.pack8(x)
    y = ops.linear8(x, w, b, act8=kept if given else None)
    assert torch.equal(y, torch.nn.functional.linear(x, w.to(dtype), b.to(dtype)))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert torch.equal(dx, dy @ w.to(dtype)) and dw.dtype == wt and db.dtype == wt
    d2, v = dy.double().view(150, 40), kept.unpack(F32).double().view(150, 96)
    close(dw, d2.t() @ v, d2.abs().t() @ v.abs(), 214, "dw")
    close(db, d2.sum(0), d2.abs().sum(0), 214, "db")
    y = ops.linear8(x.detach(), w.detach(), b)  # only the bias has a gradient
    (db2,) = torch.autograd.grad(y, b, dy)
    assert torch.allclose(db2.float(), db.float(), rtol=1e-2, atol=1e-2)


# --- cross entropy -----------------------------------------------------------

def xent64(x, target, ignore):
    valid = target != ignore
    z = x - x.amax(1, keepdim=True)
    ls = torch.log(torch.exp(z).sum(1, keepdim=True))
    at = torch.where(valid, target, 0)[:, None]
    rows = torch.where(valid, (ls - z.gather(1, at))[:, 0], 0)
    p = torch.exp(z - ls)
    one = torch.zeros_like(x).scatter_(1, at, 1.0)
    mag = p * (z.abs().nan_to_num(posinf=0) + ls + 4) + one
    return rows, (p - one) * valid[:, None], mag * valid[:, None], valid


@gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32000), (8, 32000), (300, 1000), (33, 1001), (5, 50001), (2, 128257),
                                       (3, 300000), (700, 40)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy(rows, cols, dtype, reduction):
    # an exponent's argument carries one rounding of its size, the sums few
    g = gen(rows + cols)
    x = randn(g, rows, cols, dtype=dtype, scale=3.0).requires_grad_()
    target = torch.randint(0, cols, (rows,), generator=g, device="cuda")
    if rows > 2:
        target[1] = -100
    loss = ops.cross_entropy(x, target, reduction=reduction)
    each, grad, mag, valid = xent64(x.detach().double(), target, -100)
    n = valid.sum() if reduction == "mean" else 1
    size = x.detach().double().abs().amax(1) + 16
    want, lm = (each, size) if reduction == "none" else (each.sum() / n, (size * valid).sum() / n)
    assert loss.dtype == F32
    close(loss.detach(), want, lm, 32 + rows / 32, "loss")
    up = randn(g, rows).abs() + 0.5 if reduction == "none" else torch.ones((), device="cuda")
    f = up.double()[:, None] if reduction == "none" else 1.0 / n
    (dx,) = torch.autograd.grad(loss, x, up, retain_graph=True)
    close(dx, grad * f, mag * f, 16, "dx")
    # another upstream gradient, on the kept graph; the first result stays as it was
    was = dx.clone()
    (dx3,) = torch.autograd.grad(loss, x, up * 3.7)
    close(dx3, grad * (up * 3.7).double()[:, None] if reduction == "none" else grad * float(up * 3.7) / n,
          mag * f * 3.7, 16, "dx, 3.7")
    assert torch.equal(dx, was)
    with torch.no_grad():
        assert torch.equal(ops.cross_entropy(x, target, reduction=reduction), loss)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [40, 1001, 32000, 50001, 140001])
def test_cross_entropy_masks(dtype, cols):
    g = gen(cols)
    low = torch.finfo(dtype).min
    x = randn(g, 9, cols, dtype=dtype)
    target = torch.randint(0, cols // 2, (9,), generator=g, device="cuda")
    x[0, cols // 2:] = -math.inf
    x[1, cols // 2:] = low
    x[2, :] = -math.inf  # nothing left
    x[3, :] = low  # uniform
    x[4, 1] = math.nan
    x[5, 2] = math.inf
    x[6, target[6]] = -math.inf  # a target that cannot be
    x[7, 0], target[7] = -low, cols // 2  # one certain class, and not the target
    x[8, :], target[8] = math.nan, -100  # ignored, whatever it holds
    x.requires_grad_()
    loss = ops.cross_entropy(x, target, reduction="none")
    (dx,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
    ok = [0, 1, 3]
    each, grad, mag, _ = xent64(x.detach().double()[ok], target[ok], -100)
    close(loss.detach()[ok], each, torch.full_like(each, 32.0), 32, "loss")
    close(dx[ok], grad, grad.abs() * 40 + 4.0 / cols, 32, "dx")
    assert loss[2].isnan() and dx[2].isnan().all()
    assert loss[4].isnan() and dx[4].isnan().all() and loss[5].isnan()
    assert loss[6] == math.inf and dx[6, target[6]] == -1 and dx[6].isfinite().all()
    assert loss[7] > -low * 0.99 and dx[7, 0] == 1 and dx[7, target[7]] == -1
    assert loss[8] == 0 and dx[8].eq(0).all()
    # the mean over the rest, its gradient in the same call
    keep = [0, 1, 3, 8]
    y = x.detach()[keep].requires_grad_()
    mean = ops.cross_entropy(y, target[keep])
    (dy,) = torch.autograd.grad(mean, y)
    close(mean.detach(), each.mean(), torch.tensor(32.0, device="cuda").double(), 32, "mean")
    close(dy[:3], grad / 3, grad.abs() * 40 + 4.0 / cols, 32, "dy")
    assert dy[3].eq(0).all()


@gpu
def test_cross_entropy_targets():
    x = randn(gen(9), 6, 500).requires_grad_()
    target = torch.tensor([3, 500, -1, 7, 10 ** 12, 499], device="cuda")
    loss = ops.cross_entropy(x, target, reduction="none")
    assert loss.isnan().tolist() == [False, True, True, False, True, False]
    (dx,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
    assert dx.isnan().all(1).tolist() == loss.isnan().tolist()
    # another ignored value, also one that names a class
    a = ops.cross_entropy(x, torch.tensor([3, 7, 7, 1, 2, 7], device="cuda"), ignore_index=7)
    b = ops.cross_entropy(x[[0, 3, 4]], torch.tensor([3, 1, 2], device="cuda"))
    assert torch.allclose(a, b, rtol=1e-6)
    none = torch.full((6,), -100, device="cuda")
    loss = ops.cross_entropy(x, none)
    (dx,) = torch.autograd.grad(loss, x)
    assert loss.isnan() and dx.eq(0).all()  # the mean over no rows; no row has a gradient
    assert ops.cross_entropy(x, none, reduction="sum") == 0
    empty = torch.zeros(0, 500, device="cuda", requires_grad=True)
    nothing = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert ops.cross_entropy(empty, nothing).isnan()
    loss = ops.cross_entropy(empty, nothing, reduction="sum")
    (dx,) = torch.autograd.grad(loss, empty)
    assert loss == 0 and dx.shape == (0, 500)
    y = randn(gen(10), 2, 3, 50)  # more dimensions
    t = torch.randint(0, 50, (2, 3), device="cuda")
    assert torch.allclose(ops.cross_entropy(y, t), ops.cross_entropy(y.view(6, 50), t.view(6)), rtol=1e-6)
    assert ops.cross_entropy(y, t, reduction="none").shape == (2, 3)


@gpu
@pytest.mark.parametrize("rows,cols", [(700, 3000), (900, 5003), (600, 8192), (400, 9001), (300, 20000), (310, 16379),
                                       (200, 32001), (160, 60000), (150, 120001)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_cross_entropy_many_rows(rows, cols, dtype):
    # several rows to a block: what one row leaves behind must not reach the next
    g = gen(rows + cols)
    x = randn(g, rows, cols, dtype=dtype, scale=2.0)
    target = torch.randint(0, cols, (rows,), generator=g, device="cuda")
    target[::7] = -100
    target[0] = 0
    target[2], target[3] = cols - 1, cols - 2
    x[5::11, cols // 3:] = -math.inf
    target[5::11] %= cols // 3
    x[7] = math.nan
    target[7] = -100  # ignored, whatever it holds
    x.requires_grad_()
    loss = ops.cross_entropy(x, target)
    (dx,) = torch.autograd.grad(loss, x)
    keep = torch.arange(rows, device="cuda") != 7
    each, grad, mag, valid = xent64(x.detach().double()[keep], target[keep], -100)
    n = valid.sum()
    size = x.detach().double()[keep].abs().nan_to_num(posinf=0).amax(1) + 16
    close(loss.detach(), each.sum() / n, (size * valid).sum() / n, 32 + rows / 32, "loss")
    close(dx[keep], grad / n, mag.nan_to_num() / n, 16, "dx")
    assert dx[7].eq(0).all()


@gpu
@pytest.mark.parametrize("rows,cols", [(80, 5003), (80, 9001), (80, 16385), (160, 32001), (150, 32004), (75, 64001),
                                       (75, 128257), (75, 9000)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_cross_entropy_targets_at_ends(rows, cols, dtype):
    # the first and last elements of a row, and of what each of 2, 4 or 8 blocks has of it
    g = gen(rows + 2 * cols)
    x = randn(g, rows, cols, dtype=dtype, scale=2.0).requires_grad_()
    places = [*range(9), *range(cols - 9, cols)]
    for n in (2, 4, 8):
        for k in range(1, n):
            at = (-(-cols // n) + 7) // 8 * 8 * k
            places += [at - 1, at]
    places = [q for q in places if q < cols]
    target = torch.tensor([places[i % len(places)] for i in range(rows)], device="cuda")
    target[3::13] = -100
    loss = ops.cross_entropy(x, target)
    (dx,) = torch.autograd.grad(loss, x)
    each, grad, mag, valid = xent64(x.detach().double(), target, -100)
    n = valid.sum()
    size = x.detach().double().abs().amax(1) + 16
    close(loss.detach(), each.sum() / n, (size * valid).sum() / n, 32 + rows / 32, "loss")
    close(dx, grad / n, mag / n, 16, "dx")


@gpu
@pytest.mark.parametrize("rows,cols", [(9000, 512), (6000, 768), (6000, 1024), (5000, 1001), (3000, 3000), (2500, 4096),
                                       (1500, 6001)])
@pytest.mark.parametrize("pack,residual", [(False, False), (True, False), (True, True)])
def test_layer_norm_rows_alone(rows, cols, pack, residual):
    # a row's results do not depend on which rows are there besides it
    g = gen(rows + cols)
    x, dy = randn(g, rows, cols, dtype=BF16), randn(g, rows, cols, dtype=BF16)
    r = randn(g, rows, cols, dtype=BF16) if residual else None
    w, b = randn(g, cols, dtype=BF16), randn(g, cols, dtype=BF16)

    def run(part):
        xs = x[part].clone().requires_grad_()
        y, *rest = ops.layer_norm(xs, w, b, residual=r[part] if residual else None, pack=True) if pack else (
            ops.layer_norm(xs, w, b),)
        return [y.detach(), torch.autograd.grad(y, xs, dy[part])[0]] + ([rest[-1].q] if pack else [])

    whole = run(slice(0, rows))
    for first in (0, rows // 2, rows - 40):
        part = slice(first, first + 40)
        for got, want in zip(whole, run(part)):
            assert torch.equal(got[part], want)


# --- gradients against differences -------------------------------------------

def _differences(f, xs, seed, step=2.0 ** -7):
    """<gradient, v> against (f(x + step v) - f(x - step v)) / 2 step. The
    quotient is off by step^2 / 6 of the third derivative (2^-16 of a result of
    order one here) and by 2^-24 / step of f's rounding: 2 % holds both."""
    g = gen(seed)
    xs = [x.clone().requires_grad_() for x in xs]
    grads = torch.autograd.grad(f(*xs), xs)
    for k, (x, grad) in enumerate(zip(xs, grads)):
        v = randn(g, *x.shape)
        v /= v.double().norm().float() / math.sqrt(8)

        def at(t):
            moved = [y.detach() for y in xs]
            moved[k] = moved[k] + t * v
            return f(*moved).double()

        quotient = (at(step) - at(-step)) / (2 * step)
        along = (grad.double() * v.double()).sum()
        size = grad.double().norm() * v.double().norm()
        assert abs(float(quotient - along)) <= 0.02 * float(size) / math.sqrt(8) + 2e-4, (k, float(quotient),
                                                                                          float(along), float(size))


@gpu
def test_gradients_against_differences():
    g = gen(31)
    c = randn(g, 6, 48).double()
    x, r = randn(g, 6, 48), randn(g, 6, 48)
    w, b = randn(g, 48), randn(g, 48)

    def norm(x, r, w, b):
        y, s = ops.layer_norm(x, w, b, residual=r)
        return (y.double() * c).sum() / 8 + (s.double() * c.flip(0)).sum() / 8

    _differences(norm, [x, r, w, b], 1)
    target = torch.randint(0, 48, (6,), generator=g, device="cuda")
    _differences(lambda x: ops.cross_entropy(x, target), [x * 2], 2)
    _differences(lambda x: ops.cross_entropy(x, target, reduction="sum") * 0.5, [x * 2], 3)
    # the 8-bit backward passes read the checkpoint: at inputs that it holds
    # exactly, that is the gradient itself
    x = ops.pack8(x).unpack()
    for form in ("tanh", "none"):
        _differences(lambda x: (ops.gelu8(x, approximate=form).double() * c).sum() / 8, [x], 4)
    wt = randn(g, 20, 48)
    up = randn(g, 6, 20).double()
    _differences(lambda w, b: (ops.linear8(x, w, b).double() * up).sum() / 8, [wt, randn(g, 20)], 5)


# --- where and when they run -------------------------------------------------

@gpu
def test_other_streams_and_repeated_calls():
    g = gen(41)
    x, w, b = randn(g, 512, 768, dtype=BF16), randn(g, 768), randn(g, 768)
    wl, target = randn(g, 320, 768), torch.randint(0, 768, (512,), generator=g, device="cuda")

    def step():
        xs, ws = x.clone().requires_grad_(), wl.clone().requires_grad_()
        y, kept = ops.layer_norm(xs, w, b, pack=True)
        z = ops.linear8(y, ws, act8=kept)
        loss = ops.cross_entropy(z, target % 320)
        return [loss.detach(), *torch.autograd.grad(loss, [xs, ws])]

    want = step()
    torch.cuda.synchronize()
    for _ in range(3):  # sums are in a fixed order: the same bits every time
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("what", ["norm", "gelu8", "pack8", "xent", "wgrad8"])
def test_offsets_past_32_bits(what):
    rows, cols = 70001, 32768  # 2.3e9 elements
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB of free device memory")
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    tail = randn(gen(51), 3, cols, dtype=BF16)
    x[-3:] = tail
    if what == "norm":
        w, b = torch.ones(cols, device="cuda"), torch.zeros(cols, device="cuda")
        y, kept = ops.layer_norm(x, w, b, pack=True)
        y3, kept3 = ops.layer_norm(tail, w, b, pack=True)
        assert torch.equal(y[-3:], y3) and torch.equal(kept.q[-3:], kept3.q) and not y[:-3].any()
    elif what == "gelu8":
        x.requires_grad_()
        y = ops.gelu8(x)
        (dx,) = torch.autograd.grad(y, x, x.detach())
        t = tail.clone().requires_grad_()
        y3 = ops.gelu8(t)
        (dx3,) = torch.autograd.grad(y3, t, tail)
        assert torch.equal(y[-3:], y3) and torch.equal(dx[-3:], dx3) and not dx[:-3].any()
    elif what == "pack8":
        assert torch.equal(ops.pack8(x).unpack()[-3:], ops.pack8(tail).unpack())
    elif what == "xent":
        x.requires_grad_()
        target = torch.full((rows,), -100, device="cuda")
        target[-3:] = torch.tensor([5, 6, 7], device="cuda")
        loss = ops.cross_entropy(x, target)
        (dx,) = torch.autograd.grad(loss, x)
        t = tail.clone().requires_grad_()
        loss3 = ops.cross_entropy(t, target[-3:])
        (dx3,) = torch.autograd.grad(loss3, t)
        assert torch.allclose(loss, loss3, rtol=1e-5) and torch.allclose(dx[-3:], dx3, rtol=1e-2, atol=1e-9)
        assert not dx[:-3].any()
    else:
        dy = torch.zeros(rows, 8, dtype=BF16, device="cuda")
        dy[-3:] = randn(gen(52), 3, 8, dtype=BF16)
        got = ops.weight_grad8(dy, ops.pack8(x), out_dtype=F32)
        want = dy[-3:].double().t() @ ops.pack8(tail).unpack(F32).double()
        close(got, want, dy[-3:].double().abs().t() @ tail.double().abs() * 1.02, 64)


@gpu
def test_no_wait_gave_up():
    # the status word of the kernels' bounded waits, after a few of each that wait
    from commux_b200 import _ops

    g = gen(61)
    for rows, cols in ((300, 500), (40, 40000)):
        x = randn(g, rows, cols, dtype=BF16).requires_grad_()
        loss = ops.cross_entropy(x, torch.randint(0, cols, (rows,), generator=g, device="cuda"))
        torch.autograd.grad(loss, x)
        ops.weight_grad8(randn(g, rows, 700, dtype=BF16), ops.pack8(x))
        ops.weight_grad8(randn(g, rows, 70), ops.pack8(x))
    torch.cuda.synchronize()
    assert _ops.kernel_status() == 0


@gpu
def test_refusals_on_device():
    x, w = torch.zeros(4, 32, device="cuda"), torch.ones(32, device="cuda")
    for bad in (dict(weight=torch.ones(31, device="cuda")), dict(weight=w.double()), dict(weight=w.cpu()),
                dict(weight=w, bias=w.half()), dict(weight=w, residual=x[:2]), dict(weight=w, out_dtype=torch.float64)):
        with pytest.raises(RuntimeError, match="layer_norm: "):
            ops.layer_norm(x, **bad)
    with pytest.raises(RuntimeError, match="layer_norm: "):
        ops.layer_norm(x.double(), w)
    with pytest.raises(RuntimeError, match="pack8: "):
        ops.pack8(torch.zeros(4, 0, device="cuda"))
    kept = ops.pack8(x)
    with pytest.raises(ValueError, match="weight_grad8: "):
        ops.weight_grad8(torch.zeros(5, 3, device="cuda"), kept)
    with pytest.raises(RuntimeError, match="weight_grad8: "):
        ops.weight_grad8(torch.zeros(4, 3, device="cuda"), ops.Act8(kept.q[:, :16], kept.scale, x.shape, x.dtype))
    with pytest.raises(RuntimeError, match="weight_grad8: "):
        ops.weight_grad8(torch.zeros(4, 3, device="cuda", dtype=torch.int32), kept, out_dtype=F32)
    with pytest.raises(ValueError, match="linear8: "):
        ops.linear8(x[:2], torch.zeros(8, 32, device="cuda"), act8=kept)
    with pytest.raises(RuntimeError, match="linear8: "):
        ops.linear8(x, torch.zeros(8, 31, device="cuda"))
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for targets in (t.int(), t[:3], t.cpu()):
        with pytest.raises(RuntimeError, match="cross_entropy: "):
            ops.cross_entropy(x, targets)
    x.requires_grad_()
    for f in (lambda: ops.layer_norm(x, w).sum(), lambda: ops.gelu8(x).sum(), lambda: ops.cross_entropy(x, t),
              lambda: ops.linear8(x, torch.ones(8, 32, device="cuda")).sum()):
        with pytest.raises(RuntimeError, match="no derivative"):
            torch.autograd.grad(f(), x, create_graph=True)


def test_refusals():
    x, w = torch.zeros(4, 32), torch.ones(32)
    with pytest.raises(RuntimeError, match="layer_norm: x must be a CUDA tensor"):
        ops.layer_norm(x, w)
    with pytest.raises(RuntimeError, match="pack8: x must be a CUDA tensor"):
        ops.pack8(x)
    with pytest.raises(RuntimeError, match="gelu8: x must be a CUDA tensor"):
        ops.gelu8(x)
    with pytest.raises(RuntimeError, match="linear8: x must be a CUDA tensor"):
        ops.linear8(x, torch.zeros(8, 32))
    with pytest.raises(RuntimeError, match="cross_entropy: logits must be a CUDA tensor"):
        ops.cross_entropy(x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="weight_grad8: dy must be a CUDA tensor"):
        held = ops.Act8(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8), (4, 32), F32)
        ops.weight_grad8(x, held)
    with pytest.raises(RuntimeError, match="unpack8: "):
        held.unpack()
    with pytest.raises(ValueError, match="gelu8: approximate"):
        ops.gelu8(x, approximate="erf")
    with pytest.raises(ValueError, match="cross_entropy: reduction"):
        ops.cross_entropy(x, torch.zeros(4, dtype=torch.int64), reduction="batchmean")


# --- together ----------------------------------------------------------------

@gpu
@pytest.mark.parametrize("autocast", [False, True])
def test_gpt_step(autocast):
    # The same weights and tokens with and without the operators. A checkpoint's
    # values are off by about 0.8 % of their size (a step of 2 max / 127 at most,
    # evenly spread), which a weight's gradient averages over its tokens; bf16
    # products add 0.4 %. The gradients of a whole model stay within 5 % of
    # their norm, the loss, which no checkpoint enters, within bf16's rounding.
    from commux_b200.models.gpt import GPT, GPTConfig

    torch.manual_seed(3)
    sizes = dict(n_layer=2, n_head=4, d_model=160, d_ff=448, vocab=1003, seq_len=96)
    plain = GPT(GPTConfig(**sizes)).cuda()
    held = GPT(GPTConfig(**sizes, act8=True)).cuda()
    held.load_state_dict(plain.state_dict())
    idx = torch.randint(0, 1003, (3, 96), device="cuda")
    target = torch.randint(0, 1003, (3, 96), device="cuda")
    target[0, :20] = -100
    losses = []
    for m in (plain, held):
        with torch.autocast("cuda", dtype=BF16, enabled=autocast):
            loss = m(idx, target)
        loss.backward()
        losses.append(float(loss.detach()))
    assert abs(losses[0] - losses[1]) <= (2e-2 if autocast else 1e-4), losses
    for (name, p), q in zip(plain.named_parameters(), held.parameters()):
        assert q.grad.dtype == p.grad.dtype
        off = float((p.grad.double() - q.grad.double()).norm() / p.grad.double().norm())
        assert off <= 0.05, (name, off)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16, enabled=autocast):
        a, b = plain(idx[:, :7]), held(idx[:, :7])
    assert a.shape == b.shape and torch.allclose(a.float(), b.float(), rtol=2e-2, atol=2e-2)
