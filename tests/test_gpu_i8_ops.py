"""GPU tests of the residual RMS norm, of rows in 8 bits and of the 8-bit product, against 64 bits, and of a block that chains them with the
sequence attention.

Bounds (u = 2^-24, r = 2^-8 for a stored bf16 result, else u). A row sum runs over at most 64 terms a thread and 10 joining steps: its relative
error is at most 80 u of the sum of magnitudes; rstd, behind the mean, the addition, the root and the division, at most 48 u. Integer sums are
exact; a product's result takes 4 roundings of its parts and the stored one."""
import math

import pytest
import torch

from test_gpu_seq_ops import Ref, within

pytestmark = pytest.mark.gpu
U, R = 2.0 ** -24, 2.0 ** -8
BF = torch.bfloat16
DT = pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])


def _dev():
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def cb(built_lib):
    from celebbasis_amd import lib
    ctx = lib.Context()
    yield lib, ctx
    ctx.sync()


def rnd(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(_dev())


def rt(dtype):
    return R if dtype == BF else U


def norm_ref(h, g, eps):
    h = h.double()
    rstd = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    return h * rstd * g.double(), rstd


def check_i8(q, s, y, y_err):
    """q * s stands for y within half a step; y_err bounds the error of the values that were rounded"""
    C = y.shape[-1]
    assert q.shape[-1] == (C + 15) // 16 * 16 and not q[..., C:].any()
    s64 = s.double()[..., None]
    amax = y.abs().amax(-1, keepdim=True)
    assert ((s64 * 127 - amax).abs() <= (y_err + 4 * U) * amax).all()
    assert ((q[..., :C].double() * s64 - y).abs() <= 0.5 * s64 * (1 + 2.0 ** -20) + 2 * (y_err + 4 * U) * amax).all()
    assert (q[..., :C].abs().amax(-1) == 127)[amax[..., 0] > 0].all()


@DT
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 7), (1, 768), (5, 512), (4, 513), (77, 1024), (9, 1000), (33, 2048), (3, 2049), (17, 4096), (6, 5000),
                                    (2, 8192), (2, 16384), (3, 16383), (2050, 64)])
@pytest.mark.parametrize("res", [True, False])
def test_rms_norm(cb, dtype, rows, C, res):
    lib, ctx = cb
    x, g = rnd(rows, C, seed=1, dtype=dtype), 1 + rnd(C, seed=2, scale=0.3)
    r = rnd(rows, C, seed=3, scale=2.0, dtype=dtype) if res else None
    n = lib.rms_norm(ctx, x, g, residual=r, eps=1e-6, need_grad=True)
    held = (x.float() + r.float()).to(dtype) if res else x
    assert torch.equal(n.h, held)
    y, rstd = norm_ref(held, g, 1e-6)
    assert ((n.rstd.double() - rstd[..., 0]).abs() <= 48 * U * rstd[..., 0]).all()
    within("y", n.y, y, (52 * U + rt(dtype)) * y.abs() + 2.0 ** -126)
    e = lib.rms_norm(ctx, x, g, residual=r, eps=1e-6, out="i8")
    assert torch.equal(e.h, held)
    check_i8(e.y, e.scale, y, 52 * U)


@DT
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 7), (1, 768), (4, 513), (77, 1024), (9, 1000), (700, 2048), (5, 2049), (530, 4096), (6, 5000), (2, 16384), (5000, 72)])
@pytest.mark.parametrize("dres", [True, False])
def test_rms_norm_backward(cb, dtype, rows, C, dres):
    lib, ctx = cb
    h, g, dy = rnd(rows, C, seed=1, dtype=dtype, scale=2.0), 1 + rnd(C, seed=2, scale=0.3), rnd(rows, C, seed=3, dtype=dtype)
    dr = rnd(rows, C, seed=4, dtype=dtype) if dres else None
    n = lib.rms_norm(ctx, h, g, need_grad=True)
    dh, dg = lib.rms_norm_backward(ctx, dy, n.h, g, n.rstd, dres=dr)
    h64, g64 = h.double().requires_grad_(), g.double().requires_grad_()
    y, rstd = norm_ref(h64, g64, 1e-6)
    want, wg = torch.autograd.grad((y * dy.double()).sum(), (h64, g64))
    want = want + dr.double() if dres else want
    xh, w, rstd = (h64 * rstd).detach(), dy.double() * g.double(), rstd.detach()
    m = (w * xh).mean(-1, keepdim=True)
    me = 140 * U * (w * xh).abs().mean(-1, keepdim=True)
    b = rstd * (60 * U * w.abs() + xh.abs() * (me + 60 * U * m.abs())) + 4 * U * (w.abs() * rstd + (dr.double().abs() if dres else 0))
    within("dh", dh, want, b + rt(dtype) * (want.abs() + b) + 2.0 ** -126)
    within("dg", dg, wg, (rows / 512 + 200) * U * (dy.double() * xh).abs().sum(0) + 2.0 ** -126)
    dh2, dg2 = lib.rms_norm_backward(ctx, dy, n.h, g, n.rstd, dres=dr)
    assert torch.equal(dh, dh2) and torch.equal(dg, dg2)
    only, none = lib.rms_norm_backward(ctx, dy, n.h, g, n.rstd, dres=dr, want_dweight=False)
    assert none is None and torch.equal(only, dh)


def test_rms_norm_gradient_by_differences(cb):
    lib, ctx = cb
    x, g, w = rnd(6, 96, seed=1).double(), 1 + rnd(96, seed=2, scale=0.2).double(), rnd(6, 96, seed=3).double()
    f = lambda x, g: float((lib.rms_norm(ctx, x.float(), g.float()).y.double() * w).sum())
    n = lib.rms_norm(ctx, x.float(), g.float(), need_grad=True)
    dh, dg = lib.rms_norm_backward(ctx, w.float(), n.h, g.float(), n.rstd)
    h = 2.0 ** -7
    for v, d, at in ((x, dh, 0), (g, dg, 1)):
        e = torch.sign(rnd(*v.shape, seed=5)).double()
        hi, lo = ([x + h * e, g], [x - h * e, g]) if at == 0 else ([x, g + h * e], [x, g - h * e])
        num, ana = (f(*hi) - f(*lo)) / (2 * h), float((d.double() * e).sum())
        # |y| < 8: each sum is off by at most sum |w| * 8 * 56 u; the second-order remainder is h^2 of the gradient's magnitudes
        assert abs(num - ana) <= float(w.abs().sum()) * 8 * 56 * U / h + h * h * float(d.double().abs().sum()), (at, num, ana)


@DT
def test_norm_strides_aliases_and_shapes(cb, dtype):
    lib, ctx = cb
    g = 1 + rnd(96, seed=2, scale=0.3)
    wide = rnd(20, 200, seed=1, dtype=dtype)
    a = lib.rms_norm(ctx, wide[:, 3:99], g, need_grad=True)              # rows that start off a 16-byte piece
    b = lib.rms_norm(ctx, wide[:, 3:99].contiguous(), g, need_grad=True)
    # (the order of a row's sum differs between the two paths)
    assert ((a.y.double() - b.y.double()).abs() <= (104 * U + 2 * rt(dtype)) * b.y.double().abs()).all()
    c = lib.rms_norm(ctx, b.h.view(4, 5, 96), g, out="i8")
    assert c.y.shape == (4, 5, 96) and c.scale.shape == (4, 5)
    q, s = lib.quantize_rows(ctx, wide[:, 3:99])
    q2, s2 = lib.quantize_rows(ctx, wide[:, 3:99].contiguous())
    assert torch.equal(q, q2) and torch.equal(s, s2)
    for rows in (0, 1):
        z = torch.zeros(rows, 96, dtype=dtype, device=_dev())
        n = lib.rms_norm(ctx, z, g, residual=z, need_grad=True)
        dh, dg = lib.rms_norm_backward(ctx, z, n.h, g, n.rstd)
        assert not n.y.any() and not dh.any() and not dg.any() and dg.shape == (96,)
        assert lib.quantize_rows(ctx, z)[0].shape == (rows, 96)
    # in place: h over the residual, dh over dy
    import ctypes as C
    x, r = rnd(9, 96, seed=5, dtype=dtype), rnd(9, 96, seed=6, dtype=dtype)
    n = lib.rms_norm(ctx, x, g, residual=r, need_grad=True)
    y = torch.empty_like(x)
    d = lib.RmsNormDesc()
    d.dtype, d.rows, d.C, d.eps = lib.dtype_code(dtype), 9, 96, 1e-6
    for k, t in (("x", x), ("residual", r), ("h", r), ("y", y), ("gamma", g)):
        setattr(d, k, t.data_ptr())
    d.ldx = d.ldres = d.ldh = d.ldy = 96
    lib.check(lib.load().cb_rmsnorm_fwd(ctx.h, C.byref(d)))
    assert torch.equal(r, n.h) and torch.equal(y, n.y)


@DT
@pytest.mark.parametrize("rows,K", [(1, 1), (5, 15), (5, 16), (3, 100), (64, 768), (7, 4096), (2, 16384), (3, 16385), (2, 20000)])
def test_quantize_rows(cb, dtype, rows, K):
    lib, ctx = cb
    x = rnd(rows, K, seed=1, dtype=dtype, scale=3.0)
    q, s = lib.quantize_rows(ctx, x)
    check_i8(q, s, x.double(), 0.0)
    f = x.float()
    amax = f.abs().amax(1, keepdim=True)
    want = torch.round(f * (torch.full_like(amax, 127.0) / amax))         # ties to even, the formula in fp32 (127.0 / amax would be 127 times a reciprocal)
    assert torch.equal(q[:, :K].float(), want)


@DT
def test_quantize_edges(cb, dtype):
    lib, ctx = cb
    x = rnd(6, 64, seed=1, dtype=dtype)
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 9] = -math.inf
    x[4] = 1e-38
    x[5] = torch.finfo(dtype).max
    q, s = lib.quantize_rows(ctx, x)
    assert not q[1:5].any() and s[1] == 0 and torch.isnan(s[2]) and torch.isinf(s[3]) and s[4] == 0
    assert (q[5] == 127).all() and torch.isfinite(s[5])
    w = torch.ones(32, 64, dtype=torch.int8, device=_dev())
    y = lib.linear_i8(ctx, q, s, w, torch.ones(32, device=_dev()), dtype="f32")
    assert torch.isfinite(y[[0, 1, 4]]).all() and torch.isnan(y[[2, 3]]).all() and not y[1].any()


def i8(*shape, seed=0, lo=-127, hi=127):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi + 1, shape, generator=g).to(torch.int8).to(_dev())


def product64(a, b):
    return torch.matmul(a.double(), b.double().t().contiguous())


SIZES = [(1, 1, 16), (1, 64, 64), (2, 7, 48), (3, 2304, 768), (4, 130, 144), (5, 768, 4096), (8, 4100, 128), (15, 33, 80), (16, 512, 2048), (17, 100, 512), (31, 257, 272),
         (32, 64, 16), (33, 1000, 256), (64, 768, 768), (65, 65, 4112), (77, 2304, 768), (128, 128, 128), (129, 127, 144), (200, 1280, 5120), (256, 256, 256),
         (300, 4096, 1024), (513, 515, 528), (616, 768, 768), (1024, 1000, 640), (2000, 333, 96),
         (48, 2056, 16400), (250, 4090, 8208), (2500, 4100, 64),
         (2050, 2100, 400), (3500, 3600, 16), (3500, 3600, 144), (3500, 3601, 272), (4001, 3307, 528)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_is_exact(cb, M, N, K):
    lib, ctx = cb
    a, b = i8(M, K, seed=M + K, lo=-128), i8(N, K, seed=N)
    one = torch.ones(max(M, N), device=_dev())
    got = lib.linear_i8(ctx, a, one[:M], b, one[:N], dtype="f32")
    want = product64(a, b)
    assert torch.equal(got.double(), want.float().double())               # one rounding of the whole number to fp32


def test_more_rows_than_a_launch_holds(cb):
    """17 million rows of 8 elements, a wave each: the first, the last and those around 2^23 and 2^24"""
    lib, ctx = cb
    n, c = (1 << 24) + 5, 8
    x = torch.empty(n, c, dtype=torch.bfloat16, device=_dev())
    at = torch.tensor([0, 1, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, (1 << 24) - 1, 1 << 24, n - 1], device=_dev())
    x.fill_(1.0)
    x[at] = rnd(len(at), c, seed=9, dtype=torch.bfloat16)
    g = rnd(c, seed=10)
    few = lib.rms_norm(ctx, x[at].contiguous(), g, residual=x[at].contiguous(), need_grad=True)
    all_ = lib.rms_norm(ctx, x, g, residual=x, need_grad=True)
    assert torch.equal(all_.y[at], few.y) and torch.equal(all_.h[at], few.h) and torch.equal(all_.rstd[at], few.rstd)
    q, s = lib.quantize_rows(ctx, x)
    q0, s0 = lib.quantize_rows(ctx, x[at].contiguous())
    assert torch.equal(q[at], q0) and torch.equal(s[at], s0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_epilogue(cb, dtype, M, N, K):
    lib, ctx = cb
    a, b = i8(M, K, seed=M), i8(N, K, seed=N + 1)
    sa, sb, bias = rnd(M, seed=1).abs() * 0.01, rnd(N, seed=2).abs() * 0.01, rnd(N, seed=3)
    res = rnd(M, N, seed=4).to(lib.torch_dtype(lib.dtype_code(dtype)))
    got = lib.linear_i8(ctx, a, sa, b, sb, bias=bias, residual=res, dtype=dtype)
    v = product64(a, b) * sa.double()[:, None] * sb.double()[None]
    want = v + bias.double() + res.double()
    bnd = 4 * U * (v.abs() + bias.double().abs() + res.double().abs())
    within("C", got, want, bnd + rt(got.dtype) * (want.abs() + bnd))
    assert torch.equal(got, lib.linear_i8(ctx, a, sa, b, sb, bias=bias, residual=res, dtype=dtype))


@pytest.mark.parametrize("M,N", [(40, 300), (300, 80), (300, 40000)])
def test_product_offsets_past_31_bits(cb, M, N):
    """300 rows that lie 2^23 - 16 bytes apart: the same numbers as in a small buffer"""
    lib, ctx = cb
    a, b = i8(M, 128, seed=5), i8(N, 128, seed=6)
    one = torch.ones(max(M, N), device=_dev())
    want = lib.linear_i8(ctx, a, one[:M], b, one[:N], dtype="f32")
    far = torch.empty(300, (1 << 23) - 16, dtype=torch.int8, device=_dev())
    if M == 300:
        a = far[:, :128].copy_(a)
    else:
        b = far[:, :128].copy_(b)
    assert torch.equal(lib.linear_i8(ctx, a, one[:M], b, one[:N], dtype="f32"), want)


def test_product_largest_sum_and_strides(cb):
    lib, ctx = cb
    K = 131056
    a = torch.full((3, K), -128, dtype=torch.int8, device=_dev())
    b = torch.full((5, K), -128, dtype=torch.int8, device=_dev())
    b[1] = 127
    one = torch.ones(5, device=_dev())
    got = lib.linear_i8(ctx, a, one[:3], b, one, dtype="f32")
    assert torch.equal(got.double(), product64(a, b).float().double())
    # rows of a wider buffer, output and residual with odd strides through the descriptor, R = C
    import ctypes as C
    M, N, K = 70, 45, 64
    wa, wb = i8(M, 96, seed=1), i8(N, 80, seed=2)
    out = rnd(M, 53, seed=3)
    keep = out.clone()
    s = torch.rand(128, device=_dev())
    d = lib.GemmI8Desc()
    d.dtype, d.M, d.N, d.K, d.lda, d.ldb, d.ldc, d.ldr = lib.DTYPE_F32, M, N, K, 96, 80, 53, 53
    d.A, d.B, d.C, d.R, d.a_scale, d.b_scale = wa.data_ptr() + 16, wb.data_ptr() + 16, out.data_ptr() + 4, out.data_ptr() + 4, s.data_ptr(), s.data_ptr() + 4
    n = C.c_int64()
    lib.check(lib.load().cb_gemm_i8_workspace(ctx.h, C.byref(d), C.byref(n)))
    ws = torch.empty(n.value + 16, dtype=torch.uint8, device=_dev())
    d.workspace, d.workspace_bytes = ws.data_ptr(), n.value
    lib.check(lib.load().cb_gemm_i8(ctx.h, C.byref(d)))
    v = product64(wa[:, 16:80], wb[:, 16:80]) * s[:M].double()[:, None] * s[1:N + 1].double()[None]
    want = v + keep[:, 1:46].double()
    assert ((out[:, 1:46].double() - want).abs() <= 5 * U * (v.abs() + want.abs() + keep[:, 1:46].double().abs())).all()
    assert torch.equal(out[:, :1], keep[:, :1]) and torch.equal(out[:, 46:], keep[:, 46:])


def test_zero_sizes(cb):
    lib, ctx = cb
    z = torch.empty(0, 64, dtype=torch.int8, device=_dev())
    w, one = i8(8, 64), torch.ones(8, device=_dev())
    assert lib.linear_i8(ctx, z, one[:0], w, one).shape == (0, 8)
    assert lib.linear_i8(ctx, w, one, z, one[:0]).shape == (8, 0)


@pytest.mark.parametrize("T,S", [(40, 25), (1, 9)])
def test_block(cb, T, S):
    """a block as it is used: norm -> 8-bit q/k/v projection -> biased self attention -> 8 bits -> projection onto the residual -> norm -> cross
    attention to states of another length. Each stage is held to its own bound on what the stage before it gave."""
    lib, ctx = cb
    B, H, d = 3, 4, 32
    W = H * d
    x, res = rnd(B, T, W, seed=1, dtype=BF), rnd(B, T, W, seed=2, dtype=BF)
    g = 1 + rnd(W, seed=3, scale=0.2)
    wqkv, sqkv = lib.quantize_rows(ctx, rnd(3 * W, W, seed=4, scale=W ** -0.5))
    wo, so = lib.quantize_rows(ctx, rnd(W, W, seed=5, scale=W ** -0.5))
    table, rp = rnd(32, H, seed=6), lib.RelPos(ctx)
    tl = torch.tensor([T, (T + 1) // 2, T], dtype=torch.int32, device=_dev())
    states = rnd(B, S, 2 * W, seed=7, dtype=BF).view(B, S, 2 * H, d)
    sl = torch.tensor([S, 3, 0], dtype=torch.int32, device=_dev())
    n = lib.rms_norm(ctx, x, g, residual=res, out="i8")
    y, _ = norm_ref((x.float() + res.float()).to(BF), g, 1e-6)
    check_i8(n.y, n.scale, y, 52 * U)
    qkv = lib.linear_i8(ctx, n.y, n.scale, wqkv, sqkv)
    v = product64(n.y.view(-1, W), wqkv).view(B, T, -1) * n.scale.double()[..., None] * sqkv.double()
    within("qkv", qkv, v, (4 * U + R + 4 * U * R) * v.abs())
    q = qkv.view(B, T, 3 * H, d)
    a = lib.seq_attention(ctx, q[:, :, :H], q[:, :, H:2 * H], q[:, :, 2 * H:], relpos=rp, table=table, q_len=tl, kv_len=tl)
    ref = Ref(q[:, :, :H], q[:, :, H:2 * H], q[:, :, 2 * H:], d ** -0.5, rel=(32, 128, True), table=table, q_len=tl, kv_len=tl)
    within("self", a, ref.out, ref.out_bound)
    aq, as_ = lib.quantize_rows(ctx, a.view(B, T, W))
    h = lib.linear_i8(ctx, aq, as_, wo, so, residual=n.h)
    v = product64(aq.view(-1, W), wo).view(B, T, -1) * as_.double()[..., None] * so.double()
    want = v + n.h.double()
    within("h", h, want, 4 * U * (v.abs() + n.h.double().abs()) + R * (1 + 4 * U) * want.abs() + 4 * U * R * (v.abs() + n.h.double().abs()))
    m = lib.rms_norm(ctx, h, g)
    c = lib.seq_attention(ctx, m.y.view(B, T, H, d), states[:, :, :H], states[:, :, H:], kv_len=sl)
    ref = Ref(m.y.view(B, T, H, d), states[:, :, :H], states[:, :, H:], d ** -0.5, kv_len=sl)
    within("cross", c, ref.out, ref.out_bound)
    assert not c[2].any()


def test_training_chain_gradients(cb):
    """fp32: residual norm -> biased self attention -> cross attention, the gradients of the whole chain against 64-bit differentiation"""
    lib, ctx = cb
    B, T, S, H, d = 2, 30, 17, 2, 32
    W = H * d
    x, res, g = rnd(B, T, W, seed=1), rnd(B, T, W, seed=2), 1 + rnd(W, seed=3, scale=0.2)
    table, rp = rnd(32, H, seed=4), lib.RelPos(ctx)
    st, w = rnd(B, S, 2 * H, d, seed=5), rnd(B, T, H, d, seed=6)
    sl = torch.tensor([S, 5], dtype=torch.int32, device=_dev())
    n = lib.rms_norm(ctx, x, g, residual=res, need_grad=True)
    y = n.y.view(B, T, H, d)
    a, t1 = lib.seq_attention(ctx, y, y, y, relpos=rp, table=table, need_grad=True)
    c, t2 = lib.seq_attention(ctx, a, st[:, :, :H], st[:, :, H:], kv_len=sl, need_grad=True)
    g2 = lib.seq_attention_backward(ctx, t2, w)
    g1 = lib.seq_attention_backward(ctx, t1, g2.dq)
    dh, dg = lib.rms_norm_backward(ctx, (g1.dq + g1.dk + g1.dv).view(B, T, W), n.h, g, n.rstd)
    leaves = [v.double().requires_grad_() for v in (x, res, g, table, st)]
    X, RS, Gm, Tb, St = leaves
    from test_gpu_seq_ops import buckets
    h = X + RS
    yy = (h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * Gm).view(B, T, H, d).transpose(1, 2)
    i = torch.arange(T, device=_dev())
    s = torch.matmul(yy, yy.transpose(-1, -2).contiguous()) * d ** -0.5 + Tb[buckets(i[None] - i[:, None], 32, 128, True)].permute(2, 0, 1)
    aa = torch.matmul(torch.softmax(s, -1), yy)
    kk, vv = St[:, :, :H].transpose(1, 2), St[:, :, H:].transpose(1, 2)
    s = torch.matmul(aa, kk.transpose(-1, -2).contiguous()) * d ** -0.5
    s = s.masked_fill((torch.arange(S, device=_dev())[None] >= sl[:, None])[:, None, None], -math.inf)
    cc = torch.matmul(torch.softmax(s, -1), vv)
    want = torch.autograd.grad((cc.transpose(1, 2) * w.double()).sum(), leaves)
    # four fp32 stages of sums of at most d + T terms, amplified by at most the row count: 1e-4 of the largest entry is 2^10 u a stage with room
    for name, got, ref in (("x", dh, want[0]), ("res", dh, want[1]), ("g", dg, want[2]), ("table", g1.dtable, want[3]), ("states", torch.cat([g2.dk, g2.dv], 2), want[4])):
        assert (got.double() - ref).abs().max() <= 1e-4 * ref.abs().max(), name


def test_captured_block_replays(cb):
    """the serving block captured once, replayed on changing inputs with eager calls and synchronisation in between"""
    lib, _ = cb
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ctx = lib.Context()
        x, g = rnd(33, 768, seed=1, dtype=BF), 1 + rnd(768, seed=2, scale=0.1)
        r = rnd(33, 768, seed=3, dtype=BF)
        w, ws = lib.quantize_rows(ctx, rnd(1000, 768, seed=4))
        dy = rnd(33, 768, seed=5, dtype=BF)

        def block():
            n = lib.rms_norm(ctx, x, g, residual=r, out="i8")
            y = lib.linear_i8(ctx, n.y, n.scale, w, ws)
            q, sc = lib.quantize_rows(ctx, y)
            m = lib.rms_norm(ctx, x, g, residual=r, need_grad=True)
            dh, dg = lib.rms_norm_backward(ctx, dy, m.h, g, m.rstd)
            return n.h, y, q, sc, dh, dg
        block()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            res = block()
        for turn in range(4):
            x.copy_(rnd(33, 768, seed=20 + turn, dtype=BF))
            graph.replay()
            want = block()
            s.synchronize()
            for a, b in zip(res, want):
                assert torch.equal(a, b)
