"""GPU tests of the residual RMS norm at both ends of fp32's range. The sums of squares are made of rows scaled by a power of two there, which rounds
nothing, so the bounds are those of ordinary rows: rstd 48 u, y 52 u and the stored result's own half step (u = 2^-24; see test_gpu_i8_ops.py); a
result below 2^-100, where steps stop shrinking at 2^-149, gets 2^-126 beside it."""
import pytest
import torch

from test_gpu_i8_ops import check_i8, norm_ref, rnd, rt
from test_gpu_seq_ops import BF, U, within

pytestmark = pytest.mark.gpu
DT = pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])


@pytest.fixture(scope="module")
def cb(built_lib):
    from celebbasis_amd import lib
    ctx = lib.Context()
    yield lib, ctx
    ctx.sync()


@DT
@pytest.mark.parametrize("rows,C", [(3, 40), (5, 513), (4, 1024), (3, 2048), (2, 5000), (2, 16384)])
@pytest.mark.parametrize("scale,eps", [(1e19, 1e-6), (3e25, 1e-6), (1e36, 0.0), (1e-16, 0.0), (1e-25, 0.0), (1e-30, 1e-38), (1e-30, 1e-6)])
def test_rms_norm_of_very_large_and_small_rows(cb, dtype, rows, C, scale, eps):
    lib, ctx = cb
    x, r, g = rnd(rows, C, seed=1, scale=scale, dtype=dtype), rnd(rows, C, seed=3, scale=2 * scale, dtype=dtype), 1 + rnd(C, seed=2, scale=0.3)
    x[0] = 0.0
    r[0] = rnd(C, seed=4, dtype=dtype)                                    # (an ordinary row among them)
    n = lib.rms_norm(ctx, x, g, residual=r, eps=eps, need_grad=True)
    held = (x.float() + r.float()).to(dtype)
    assert torch.equal(n.h, held)
    y, rstd = norm_ref(held, g, eps)
    assert ((n.rstd.double() - rstd[..., 0]).abs() <= 48 * U * rstd[..., 0]).all()
    within("y", n.y, y, (52 * U + rt(dtype)) * y.abs() + 2.0 ** -126)
    e = lib.rms_norm(ctx, x, g, residual=r, eps=eps, out="i8")
    check_i8(e.y, e.scale, y, 52 * U)
    dy = rnd(rows, C, seed=5, scale=scale if scale > 1 else 1.0, dtype=dtype)
    dh, dg = lib.rms_norm_backward(ctx, dy, n.h, g, n.rstd)
    xh, w = held.double() * rstd, dy.double() * g.double()
    m = (w * xh).mean(-1, keepdim=True)
    want = rstd * (w - xh * m)
    b = rstd * (60 * U * w.abs() + xh.abs() * (140 * U * (w * xh).abs().mean(-1, keepdim=True) + 60 * U * m.abs())) + 4 * U * w.abs() * rstd
    within("dh", dh, want, b + rt(dtype) * (want.abs() + b) + 2.0 ** -126)
    within("dg", dg, (dy.double() * xh).sum(0), (rows / 512 + 200) * U * (dy.double() * xh).abs().sum(0) + 2.0 ** -126)
