"""The training operators (commux_b200.ops.train) at the edges of their ranges:
long sums, constant and far rows, orders that are copied, devices' waits that
give up, rows of more than 2^31 elements, and the ways through the kernels that
common sizes do not take."""

import math
import os
import subprocess
import sys
import os
import subprocess
import sys

import pytest
import torch

from commux_b200 import ops

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


# --- layer norm of rows whose mean is far from their deviation ------------------

@gpu
@pytest.mark.parametrize("cols", [7, 41, 96, 768, 1000, 3001, 4100, 8192, 10007])
@pytest.mark.parametrize("value", [1000.0, 1000.1, -0.3, 12345.678])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_layer_norm_constant_rows(cols, value, dtype):
    # A constant row is its own mean. The mean of its sum (25 roundings one after the
    # other at most) is off by 2^-19 of it, what corrects the mean by 2^-19 of that, and
    # the normalised values are the rest times rstd = eps^-1/2 = 316. Its 8-bit form too.
    x = torch.full((3, cols), value, dtype=dtype, device="cuda").requires_grad_()
    w, b = torch.full((cols,), 2.0, device="cuda"), torch.full((cols,), 0.5, device="cuda")
    far = 2.0 ** -38 * abs(value) * 317
    y, kept = ops.layer_norm(x, w, b, pack=True)
    assert ((y.detach().float() - 0.5).abs() <= 2 * far + 2.0 ** -24).all(), float((y.float() - 0.5).abs().max())
    assert (ops.Act8(kept.q, kept.scale, kept.shape, F32).unpack().abs() <= 1.01 * far).all()
    y = ops.layer_norm(x, w, b)
    dy = randn(gen(cols), 3, cols, dtype=dtype)
    (dx,) = torch.autograd.grad(y, x, dy)
    # the mean that the backward pass keeps is the value itself: h = 0
    g = dy.double() * 2
    want = (g - g.mean(1, keepdim=True)) / math.sqrt(1e-5)
    tol = 2.0 ** {F32: -20, BF16: -8, F16: -10}[dtype] * 317 * (g.abs() + g.abs().mean(1, keepdim=True))
    assert ((dx.double() - want).abs() <= tol).all()


@gpu
@pytest.mark.parametrize("cols", [7, 33, 77, 100])
def test_layer_norm_backward_of_huge_rows(cols):
    # 2^120 / sqrt(eps) is no fp32 number, and no element of the row has it: a constant
    # row's normalised values are zero, and so is all that the columns beyond it add
    x = torch.full((3, cols), 2.0 ** 120, device="cuda").requires_grad_()
    w = torch.ones(cols, device="cuda").requires_grad_()
    dy = randn(gen(1), 3, cols)
    dx, dw = torch.autograd.grad(ops.layer_norm(x, w), (x, w), dy)
    g = dy.double()
    want = (g - g.mean(1, keepdim=True)) / math.sqrt(1e-5)
    assert ((dx.double() - want).abs() <= 2.0 ** -20 * 317 * (g.abs() + g.abs().mean(1, keepdim=True))).all()
    assert dw.eq(0).all()


# --- long sums of the weight gradient -------------------------------------------

def _one_sign(rows, dtype, out):
    """weight_grad8 of products of one sign, whose losses add up, and its values in 64 bits
    (some columns). So many columns that every pair of blocks has sums over all tokens."""
    cols, outs = 74 * 256, 512
    g = gen(rows)
    q = torch.randint(1, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int8)
    scale = torch.full((rows, cols // 32), 120, dtype=torch.uint8, device="cuda")
    spread = 1 + torch.rand(outs, generator=g, device="cuda")  # results all over a binade
    dy = (torch.rand(rows, outs, generator=g, device="cuda") * spread / 16).to(dtype)
    dw = ops.weight_grad8(dy, ops.Act8(q, scale, (rows, cols), dtype), out_dtype=out)
    some = torch.arange(0, cols, 37, device="cuda")
    want = torch.zeros(outs, len(some), dtype=torch.float64, device="cuda")
    for k in range(0, rows, 50_000):
        want += dy[k:k + 50_000].double().t() @ (q[k:k + 50_000][:, some].double() / 128)
    return dw[:, some].double(), want


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows", [1536, 5000])
def test_weight_grad8_sums_do_not_shrink(rows, dtype):
    # What tensor memory cuts off is half a unit on average at each of 96 additions of
    # a sum, which is half its final size on average, and 2^-24 of that size is half a
    # unit at most. It does not depend on the number of terms that dy comes in.
    dw, want = _one_sign(rows, dtype, F32)
    off = float((dw - want).norm() / want.norm())
    assert off <= 96 * 2.0 ** -25, off


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_weight_grad8_long_sums_in_16_bits(dtype):
    # Rounded to nearest, results are off to both sides alike: the mean of 262144 relative
    # errors (over 512 different sizes) is u / 50 by chance. Cut-off sums stay under a
    # tenth of u, half a unit of the type.
    u = {F16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype]
    dw, want = _one_sign(200_000, dtype, dtype)
    off = float(((dw - want) / want).mean())
    assert dw.isfinite().all() and abs(off) <= u * (0.1 + 0.02), off / u


@gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,cols,outs", [(3000, 2050, 9000), (700, 2100, 9000), (5000, 700, 1500)])
def test_weight_grad8_terms_in_shared_tiles(rows, cols, outs, dtype):
    # pairs' parts that begin and end among the lower terms, with and without cuts; each
    # addition of a sum in tensor memory is off by a unit, 2^-23 of what has been added up
    g = gen(rows)
    x, dy = randn(g, rows, cols, dtype=BF16), randn(g, rows, outs, dtype=dtype)
    kept = ops.pack8(x)
    dw, db = ops.weight_grad8(dy, kept, bias=True, out_dtype=F32)
    v, d = kept.unpack(F32).double(), dy.double()
    want = d.t() @ v
    assert ((dw.double() - want).abs() <= (rows / 8 + 64) * 2.0 ** -24 * (d.abs().t() @ v.abs())).all()
    assert float((dw.double() - want).norm() / want.norm()) <= 2 * 96 * 2.0 ** -24.5
    assert ((db.double() - d.sum(0)).abs() <= (rows / 8 + 64) * 2.0 ** -24 * d.abs().sum(0)).all()


# --- waits that run out -------------------------------------------------------------

def _wait_worker(what, limit_ms):
    worker = os.path.join(ROOT, "tests", "workers", "train_waits.py")
    env = dict(os.environ, COMMUX_KERNEL_WAIT_MS=limit_ms, PYTHONPATH=ROOT)
    r = subprocess.run([sys.executable, worker, what], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "PASS" in r.stdout, r.stdout[-3000:] + r.stderr[-3000:]


@gpu
def test_weight_grad8_waits_that_run_out():
    _wait_worker("weight_grad8", "0")


@gpu
@pytest.mark.parametrize("limit_ms", ["0", "0.004"])
def test_cross_entropy_waits_that_run_out(limit_ms):
    _wait_worker("cross_entropy", limit_ms)


@gpu
def test_the_call_after_a_wait_that_ran_out_raises():
    _wait_worker("raises", "0")


# --- the exact GELU ---------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gelu8_exact_form_keeps_its_relative_accuracy(dtype):
    # Phi(x) of a negative x is small, and the product keeps its relative accuracy: half
    # a unit of the type, and 32 bits' in the exponential's argument z = x^2 / 2 log2(e)
    # (four roundings of z <= 18 for x >= -5, times ln 2) and about ten beside it.
    x = -torch.linspace(0.001, 5, 40_000, device="cuda").to(dtype).view(40, 1000)
    y = ops.gelu8(x, approximate="none").double()
    x64 = x.double()
    want = x64 * 0.5 * torch.erfc(-x64 / math.sqrt(2))
    u, least = {F32: (2.0 ** -24, 2.0 ** -149), BF16: (2.0 ** -8, 2.0 ** -133), F16: (2.0 ** -11, 2.0 ** -24)}[dtype]
    tol = want.abs() * (u + (4 * 18 * 0.7 + 10) * 2.0 ** -24) + least
    worst = float(((y - want).abs() / tol).max())
    assert worst <= 1, worst


@gpu
def test_gelu8_exact_form_against_torch():
    # no further from 64 bits, in norm, than one and a half times torch's own 32-bit form
    g = gen(3)
    x = randn(g, 500, 1000) * torch.where(torch.rand(1000, generator=g, device="cuda") < 0.01, 6.0, 1.0)
    want = x.double() * 0.5 * torch.erfc(-x.double() / math.sqrt(2))
    plain = 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    off = [float((y.double() - want).norm() / want.norm()) for y in (ops.gelu8(x, approximate="none"), plain)]
    assert off[0] <= 1.5 * off[1], off


# --- orders that are copied -------------------------------------------------------

def _peak_of(f):
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = f()
    torch.cuda.synchronize()
    return got, torch.cuda.max_memory_allocated() - before


@gpu
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_cross_entropy_of_a_shifted_slice_copies_once(reduction):
    # logits[:, :-1] has outer dimensions that do not merge: the forward pass's copy
    # serves the backward pass too
    g = gen(1)
    x = randn(g, 6, 65, 2000).requires_grad_()
    target = torch.randint(0, 2000, (6, 64), generator=g, device="cuda")
    part = x[:, :-1]
    loss = ops.cross_entropy(part, target, reduction=reduction)
    up = torch.rand_like(loss)
    size = 6 * 64 * 2000 * 4
    (dx,), peak = _peak_of(lambda: torch.autograd.grad(loss, part, up, retain_graph=True))
    made = size if reduction == "none" else 0  # the mean's is there since the forward pass
    assert peak <= made + size // 4, (peak, size)
    ref = part.detach().double().requires_grad_()
    want = torch.nn.functional.cross_entropy(ref.flatten(0, 1), target.flatten(), reduction=reduction)
    (wx,) = torch.autograd.grad(want, ref, up.flatten().double() if reduction == "none" else up.double())
    assert torch.allclose(dx.double(), wx, rtol=1e-5, atol=1e-8)
    (again,) = torch.autograd.grad(loss, part, up)
    assert torch.allclose(again, dx, rtol=1e-6, atol=1e-9)


@gpu
def test_layer_norm_of_a_shifted_slice_copies_once():
    g = gen(2)
    x, w = randn(g, 6, 129, 1000).requires_grad_(), randn(g, 1000)
    part = x[:, :-1]
    y = ops.layer_norm(part, w)
    dy = randn(g, 6, 128, 1000)
    size = dy.numel() * 4
    (dx,), peak = _peak_of(lambda: torch.autograd.grad(y, part, dy))
    assert peak <= size + size // 4, (peak, size)
    ref = part.detach().double().requires_grad_()
    (want,) = torch.autograd.grad(torch.nn.functional.layer_norm(ref, (1000,), w.double()), ref, dy.double())
    assert torch.allclose(dx.double(), want, rtol=1e-4, atol=1e-5)


# --- linear8 whose bias has another type than its weight ---------------------------

@gpu
@pytest.mark.parametrize("dtype,wt,bt", [(BF16, BF16, F32), (F16, F16, F32), (F32, BF16, F32), (BF16, F32, BF16)])
def test_linear8_bias_gradient_in_its_own_type(dtype, wt, bt):
    # the sum over 150 tokens in 32 bits, rounded once, to the bias's type
    g = gen(8)
    x = randn(g, 150, 96, dtype=dtype)
    w, b = randn(g, 40, 96, dtype=wt).requires_grad_(), randn(g, 40, dtype=bt).requires_grad_()
    dy = randn(g, 150, 40, dtype=dtype)
    dw, db = torch.autograd.grad(ops.linear8(x, w, b), (w, b), dy)
    assert dw.dtype == wt and db.dtype == bt
    u = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}[bt]
    want = dy.double().sum(0)
    assert ((db.double() - want).abs() <= 1.01 * u * want.abs() + 160 * 2.0 ** -24 * dy.double().abs().sum(0)).all()


# --- the model that uses them -------------------------------------------------------

def _small_gpt(**more):
    from commux_b200.models.gpt import GPT, GPTConfig

    torch.manual_seed(3)
    return GPT(GPTConfig(n_layer=2, n_head=4, d_model=160, d_ff=448, vocab=1003, seq_len=96, **more))


def test_gpt_has_the_same_parameters_with_and_without():
    plain, held = _small_gpt(), _small_gpt(act8=True)
    assert {k: v.shape for k, v in plain.state_dict().items()} == {k: v.shape for k, v in held.state_dict().items()}
    assert all(torch.equal(a, b) for a, b in zip(plain.state_dict().values(), held.state_dict().values()))


@gpu
def test_gpt_without_a_gradient_holds_no_checkpoints(monkeypatch):
    made = []
    init = ops.Act8.__init__
    monkeypatch.setattr(ops.Act8, "__init__", lambda self, *a, **k: (made.append(1), init(self, *a, **k))[1])
    m = _small_gpt(act8=True).cuda()
    idx = torch.randint(0, 1003, (2, 96), device="cuda")
    with torch.no_grad():
        a = m(idx)
    assert not made
    b = m(idx)
    assert made and torch.equal(a, b)


@gpu
def test_gpt_hooks_and_checkpointing_see_every_layer():
    m = _small_gpt(act8=True).cuda()
    idx, target = (torch.randint(0, 1003, (2, 96), device="cuda") for _ in range(2))
    seen = set()
    handles = [sub.register_forward_hook(lambda mod, i, o, name=name: seen.add(name))
               for name, sub in m.named_modules() if name and not isinstance(sub, torch.nn.ModuleList)]
    loss = m(idx, target)
    loss.backward()
    for h in handles:
        h.remove()
    assert seen == {name for name, sub in m.named_modules() if name and not isinstance(sub, torch.nn.ModuleList)}
    want = [p.grad.clone() for p in m.parameters()]
    # blocks that are run again in the backward pass
    from torch.utils.checkpoint import checkpoint

    for b in m.blocks:
        run = b.forward
        b.forward = lambda *a, run=run: checkpoint(run, *a, use_reentrant=False)
    m.zero_grad()
    m(idx, target).backward()
    for p, g in zip(m.parameters(), want):
        assert torch.allclose(p.grad, g, rtol=1e-5, atol=1e-8)


# --- rows of more than 2^31 elements ---------------------------------------------------

def _room(n):
    if torch.cuda.mem_get_info()[0] < n:
        pytest.skip(f"needs {n / 1e9:.0f} GB of free device memory")


@gpu
@pytest.mark.parametrize("extra", [37, 64, 72])
def test_packing_and_gelu_of_rows_past_31_bits(extra):
    # a group's results do not depend on where in the row it lies
    _room(60e9)
    cols = 2 ** 31 + extra
    x = torch.zeros(1, cols, dtype=BF16, device="cuda")
    places = [(2 ** 31 - 4096, 4096 + extra), (2 ** 30 - 96, 4096), (0, 4096)]
    g = gen(extra)
    for at, n in places:
        x[0, at:at + n] = randn(g, n, dtype=BF16)
    kept = ops.pack8(x)
    values = kept.unpack()
    for at, n in places:
        small = ops.pack8(x[:, at:at + n].clone())
        assert torch.equal(kept.q[:, at:at + n], small.q[:, :n])
        assert torch.equal(kept.scale[:, at // 32:-(-(at + n) // 32)], small.scale)
        assert torch.equal(values[:, at:at + n], small.unpack())
    assert not kept.q[:, cols:].any() and not values[0, 2 ** 31 - 8192:2 ** 31 - 4096].any()
    del kept, values
    x.requires_grad_()
    y = ops.gelu8(x)
    (dx,) = torch.autograd.grad(y, x, x.detach())
    for at, n in places:
        t = x.detach()[:, at:at + n].clone().requires_grad_()
        z = ops.gelu8(t)
        (dz,) = torch.autograd.grad(z, t, t.detach())
        assert torch.equal(y[:, at:at + n], z) and torch.equal(dx[:, at:at + n], dz)


@gpu
def test_weight_grad8_refuses_sizes_past_31_bits():
    _room(30e9)
    dy = torch.zeros(1, 2 ** 31, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="weight_grad8: at most"):
        ops.weight_grad8(dy, ops.pack8(torch.ones(1, 1, dtype=BF16, device="cuda")))
    with pytest.raises(RuntimeError, match="weight_grad8: at most"):
        ops.weight_grad8(torch.ones(1, 1, dtype=BF16, device="cuda"), ops.pack8(dy))


# --- ways through the kernels that common sizes do not take ---------------------------

@gpu
@pytest.mark.parametrize("rows,cols", [(400, 9001), (200, 32000), (160, 32001), (60, 40000), (20, 128257)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("ahead,behind", [(0, 8), (0, 5), (8, 8), (3, 4)])
def test_cross_entropy_of_a_slice(rows, cols, dtype, ahead, behind):
    # rows apart, off 16-byte boundaries, and lying otherwise than dx's: the same results
    g = gen(rows + cols)
    wide = torch.full((rows, ahead + cols + behind), math.nan, dtype=dtype, device="cuda")
    wide[:, ahead:ahead + cols] = randn(g, rows, cols, dtype=dtype, scale=2.0)
    x = wide[:, ahead:ahead + cols]
    target = torch.randint(0, cols, (rows,), generator=g, device="cuda")
    target[::9] = -100
    for reduction in ("mean", "none"):
        got, want = [], []
        for t, to in ((x.detach(), got), (x.detach().contiguous(), want)):
            t.requires_grad_()
            loss = ops.cross_entropy(t, target, reduction=reduction)
            (dx,) = torch.autograd.grad(loss.sum(), t)
            to += [loss.detach(), dx]
        # sums in another order: 2^-20 of a loss of order 10; a probability's and its rounding
        assert torch.allclose(got[0], want[0], rtol=1e-6, atol=1e-5)
        assert torch.allclose(got[1].float(), want[1].float(), rtol=2.0 ** -7 if dtype == BF16 else 1e-5, atol=1e-12)


@gpu
@pytest.mark.parametrize("pack", [False, True])
def test_layer_norm_rows_past_32_bits(pack):
    # the kernels that hold a row in registers, with their gradients
    rows, cols = 1_100_001, 2048  # 2.25e9 elements
    if torch.cuda.mem_get_info()[0] < 60e9:
        pytest.skip("needs 60 GB of free device memory")
    g = gen(4)
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    tail, w, b = randn(g, 3, cols, dtype=BF16), randn(g, cols, dtype=BF16), randn(g, cols, dtype=BF16)
    x[-3:] = tail
    x.requires_grad_()
    got = ops.layer_norm(x, w, b, pack=pack)
    y = got[0] if pack else got
    (dx,) = torch.autograd.grad(y, x, x.detach())
    t = tail.clone().requires_grad_()
    got3 = ops.layer_norm(t, w, b, pack=pack)
    y3 = got3[0] if pack else got3
    (dx3,) = torch.autograd.grad(y3, t, tail)
    assert torch.equal(y[-3:], y3) and torch.equal(dx[-3:], dx3)
    assert not dx[:1000].any() and not dx[rows // 2:rows // 2 + 1000].any()
    assert torch.equal(y[rows // 2], b)
    if pack:
        assert torch.equal(got[-1].q[-3:], got3[-1].q)


@gpu
def test_operators_from_two_threads():
    # each thread on a stream of its own, the same results as alone
    import threading

    g = gen(5)
    xs = [randn(g, 300, 768, dtype=BF16) for _ in range(2)]
    w, b, wl = randn(g, 768), randn(g, 768), randn(g, 9000, 768)
    target = torch.randint(0, 9000, (300,), generator=g, device="cuda")
    torch.cuda.synchronize()

    def step(x):
        x, ws = x.clone().requires_grad_(), wl.clone().requires_grad_()
        y, kept = ops.layer_norm(x, w, b, pack=True)
        loss = ops.cross_entropy(ops.linear8(ops.gelu8(y), ws, act8=None), target)
        return [loss.detach(), *torch.autograd.grad(loss, [x, ws])]

    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(8):
                    got[k] = step(xs[k])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    for a, c in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, c))
