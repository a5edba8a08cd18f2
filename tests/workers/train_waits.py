"""Bounded waits of the training operators' kernels that run out: run with
COMMUX_KERNEL_WAIT_MS=0, where a wait gives up after its first looks (a look
blocks for 4 us), or a few microseconds. No result may look like one that is not: each is right or NaN, the
status says so, and the device stays usable."""

import os
import sys

import torch

from commux_b200 import _ops, ops

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
g = torch.Generator(device="cuda").manual_seed(1)


def randn(*shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def right_or_nan(got, want, tol, what):
    torch.cuda.synchronize()
    status = _ops.kernel_status(True)
    bad = ~(got.isnan() | ((got.double() - want).abs() <= tol))
    assert not bad.any(), (what, int(bad.sum()), bad.numel())
    assert status != 0 or not got.isnan().any(), what
    return status != 0, float(got.isnan().double().mean())


def weight_grad8():
    nans = []
    for rows, cols, outs, dtype, out, norm in [(8192, 768, 3072, BF16, F32, False),
                                               (4096, 74 * 256, 512, BF16, BF16, True),
                                               (4096, 700, 500, F32, F32, True), (3000, 1000, 90, F16, F16, False)]:
        x, dy = randn(rows, cols, dtype=BF16), randn(rows, outs, dtype=dtype)
        w, b = (1 + 0.2 * randn(cols), randn(cols)) if norm else (None, None)
        kept = ops.layer_norm(x, w, b, pack=True)[1] if norm else ops.pack8(x)
        v = ops.Act8(kept.q, kept.scale, kept.shape, F32).unpack()
        mag = v.abs()
        if norm:
            v, mag = v * w + b, mag * w.abs() + b.abs()
        d = dy.double()
        want, size = d.t() @ v.double(), d.abs().t() @ mag.double()
        dw, db = ops.weight_grad8(dy, kept, bias=True, out_dtype=out)
        ran_out, some = right_or_nan(dw, want, 1.01 * U[out] * want.abs() + (rows + 64) * 2.0 ** -24 * size, "dw")
        want = d.sum(0)
        assert (db.isnan() | ((db.double() - want).abs() <= 1.01 * U[out] * want.abs()
                              + (rows + 64) * 2.0 ** -24 * d.abs().sum(0))).all()
        print(f"weight_grad8 {rows} {cols} {outs}: {100 * some:.1f} % NaN", flush=True)
        nans.append(ran_out and some)
    # in a short sum nothing takes longer than one look, which itself waits for 4 us
    assert max(nans) > 0


def raises():
    """The call after one whose wait ran out says so, in both directions; then all is as before."""
    x, w, t = randn(500, 32001).requires_grad_(), torch.ones(32001, device="cuda"), torch.zeros(500, dtype=torch.int64,
                                                                                                device="cuda")
    y, kept = ops.layer_norm(x, w, pack=True)
    z, u = ops.gelu8(x), ops.linear8(x, w[None].requires_grad_(), act8=kept)
    assert ops.kernel_status() == 0
    loss = ops.cross_entropy(x, t)
    torch.cuda.synchronize()
    assert loss.isnan() and ops.kernel_status() == 1
    for f in (lambda: ops.layer_norm(x, w), lambda: ops.gelu8(x), lambda: ops.pack8(x), kept.unpack,
              lambda: ops.linear8(x, w[None]), lambda: ops.weight_grad8(u.detach(), kept),
              lambda: ops.cross_entropy(x, t), *(lambda y=y: torch.autograd.grad(y.sum(), x) for y in (loss, y, z, u))):
        try:
            f()
        except RuntimeError as e:
            assert "wait has run out" in str(e) and "kernel_status(reset=True)" in str(e), e
        else:
            raise AssertionError("no error")
    assert ops.kernel_status(reset=True) == 1 and ops.kernel_status() == 0
    assert torch.equal(ops.layer_norm(x, w), ops.layer_norm(x, w)) and ops.kernel_status() == 0


def cross_entropy():
    given_up = 0
    for rows, cols, dtype in [(700, 9001, BF16), (600, 32000, BF16), (500, 32001, F32), (300, 20000, F32),
                              (160, 120001, BF16), (150, 128256, BF16), (20, 32000, F32), (9, 140001, F16)]:
        x = randn(rows, cols, dtype=dtype).requires_grad_()
        target = torch.randint(0, cols, (rows,), generator=g, device="cuda")
        target[::7] = -100
        z = x.detach().double()
        ls = torch.log_softmax(z, 1)
        valid = target != -100
        at = torch.where(valid, target, 0)[:, None]
        each = torch.where(valid, -ls.gather(1, at)[:, 0], 0)
        p = torch.exp(ls)
        grad = (p - torch.zeros_like(p).scatter_(1, at, 1.0)) * valid[:, None]
        # its rounding, a dozen roundings of an exponent's argument under 30, and float16's least
        tol, least = (1.01 * U[dtype] + 512 * 2.0 ** -24) * grad.abs(), 2.0 ** -24 * (dtype == F16) + 2.0 ** -133
        for reduction in ("none", "mean"):
            loss = ops.cross_entropy(x, target, reduction=reduction)
            torch.cuda.synchronize()
            first = _ops.kernel_status(True)
            want = each if reduction == "none" else each.sum() / valid.sum()
            assert (loss.isnan() | ((loss.double() - want).abs() <= 1e-4)).all(), (rows, cols, reduction)
            assert first != 0 or not loss.isnan().any()
            (dx,) = torch.autograd.grad(loss.sum(), x)
            n = 1 if reduction == "none" else valid.sum()
            torch.cuda.synchronize()
            bad = ~(dx.isnan() | ((dx.double() - grad / n).abs() <= tol / n + least))
            assert not bad.any(), (rows, cols, reduction, int(bad.sum()))
            assert first != 0 or not dx.isnan().any()
            given_up += first != 0
            print(f"cross_entropy {rows} {cols} {reduction}: {100 * float(dx.isnan().double().mean()):.2f} % NaN",
                  flush=True)
    # the GPU's memory does not fill every block's shared memory within a look
    assert given_up > 0 or os.environ["COMMUX_KERNEL_WAIT_MS"] != "0"


if __name__ == "__main__":
    globals()[sys.argv[1]]()
    x = torch.arange(1000, device="cuda")
    assert int(x.sum()) == 499500
    print("PASS")
