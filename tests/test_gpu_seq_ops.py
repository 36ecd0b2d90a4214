"""GPU tests of the sequence operators against a plain implementation in 64 bits.

Bounds are derived, element by element, from the arithmetic (u = 2^-24 half a step of fp32, r = 2^-8 half a step of bf16):
  a score is a sum of d products: off by e_s <= (d + 8) u (scale |q|.|k| + |bias|); with exp2's own error a probability is off by the share
  e_P = 2 max e_s + 2^-21 (both numerator and denominator), a sum of N terms by N u of the sum of magnitudes;
  numbers below 2^-126 may be taken as zero: a probability is off by up to F = 2^-126 more, a product with it by F times the other factor + 1;
  bf16: an operand rounded for the matrix unit (probabilities, dS) adds r of its magnitude, the stored result r of its own.
Nothing else is allowed for: the bound of each output is written where it is used."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U, R, F = 2.0 ** -24, 2.0 ** -8, 2.0 ** -126
BF = torch.bfloat16


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


def buckets(rel, nb, D, two):
    n = rel.abs() if two else (-rel).clamp(min=0)
    half = nb // 2 if two else nb
    E = half // 2
    m = half - E
    x = n.clamp(min=1).double()
    far = E + torch.floor(torch.log(x / E) / math.log(D / E) * m + 1e-9).clamp(max=m - 1).long()
    b = torch.where(n < E, n, far)
    return b + half * (rel > 0) if two else b


class Ref:
    """64-bit forward and backward of attention with everything visible spelled out, and the bounds of the fp32 / bf16 kernels' errors"""

    def __init__(self, q, k, v, scale, causal=False, q_pos=None, q_len=None, kv_len=None, kv_mask=None, rel=None, table=None, dout=None):
        B, Nq, H, d = q.shape
        Nk, Hkv = k.shape[1:3]
        G = H // Hkv
        dev = q.device
        r = R if q.dtype == BF else 0.0
        rT = R if q.dtype == BF else U
        j, i = torch.arange(Nk, device=dev), torch.arange(Nq, device=dev)
        pos = i[None] + (q_pos.long()[:, None] if q_pos is not None else 0)
        pos = pos.expand(B, Nq)
        ok = torch.ones(B, Nq, Nk, dtype=torch.bool, device=dev)
        if kv_len is not None:
            ok &= (j[None] < kv_len[:, None])[:, None, :]
        if kv_mask is not None:
            ok &= kv_mask.bool()[:, None, :]
        if q_len is not None:
            ok &= (i[None] < q_len[:, None])[:, :, None]
        if causal:
            ok &= j[None, None, :] <= pos[:, :, None]
        seen = ok.any(1)                                                  # [B, Nk]
        live = (i[None] < q_len[:, None]) if q_len is not None else torch.ones(B, Nq, dtype=torch.bool, device=dev)
        vis = torch.ones(B, Nk, dtype=torch.bool, device=dev)             # what lengths and mask let through: the rest may hold anything
        if kv_len is not None:
            vis &= j[None] < kv_len[:, None]
        if kv_mask is not None:
            vis &= kv_mask.bool()
        q64 = torch.where(live[:, :, None, None], q.double(), 0.0).transpose(1, 2)
        k64 = torch.where(vis[:, :, None, None], k.double(), 0.0).transpose(1, 2).repeat_interleave(G, 1)
        v64 = torch.where(vis[:, :, None, None], v.double(), 0.0).transpose(1, 2).repeat_interleave(G, 1)
        T = lambda x: x.transpose(-1, -2).contiguous()
        s = torch.matmul(q64, T(k64)) * scale
        mag = torch.matmul(q64.abs(), T(k64.abs())) * scale
        if rel is not None:
            nb, D, two = rel
            bk = buckets(j[None, None, :] - pos[:, :, None], nb, D, two)          # [B, Nq, Nk]
            bias = table.double()[bk].permute(0, 3, 1, 2)
            s = s + bias
            mag = mag + torch.where(torch.isfinite(bias), bias, 0.0).abs()
        okh = ok[:, None]
        s = s.masked_fill(~okh, -math.inf)
        top = s.amax(-1, keepdim=True) if Nk else s.new_full((B, H, Nq, 1), -math.inf)
        top = torch.where(torch.isfinite(top), top, 0.0)
        e = torch.exp(s - top)
        tot = e.sum(-1, keepdim=True)
        p = torch.where(tot > 0, e / tot, 0.0)
        self.lse = torch.where(tot > 0, top + torch.log(tot), -math.inf)[..., 0]
        mmax = float(torch.where(okh, mag, 0.0).max()) if Nk and Nq else 0.0
        es = (d + 8) * U * mmax
        eP = 2 * es + 2.0 ** -21
        self.lse_bound = es + 2.0 ** -21 + 4 * U * (1 + self.lse.abs().nan_to_num(0, 0, 0))
        o = torch.matmul(p, v64)
        pv = torch.matmul(p, v64.abs())
        vis64 = okh.double().expand_as(p)
        o32_bound = (eP + (Nk + 4) * U + r) * pv + F * torch.matmul(vis64, v64.abs() + 1)
        self.out = o.transpose(1, 2)
        self.out_bound = (o32_bound + rT * (o.abs() + o32_bound)).transpose(1, 2)
        if dout is None:
            return
        do = torch.where(live[:, :, None, None], dout.double(), 0.0).transpose(1, 2)
        dp = torch.matmul(do, T(v64))
        Dr = (do * o).sum(-1, keepdim=True)
        ds = p * (dp - Dr)
        e_dp = (d + 2) * U * torch.matmul(do.abs(), T(v64.abs()))
        # the row sums dO.O: from the output as stored, or (bf16 with a table) from out32, whose probabilities carry r^2
        o_used = (eP + (Nk + 4) * U + R * R) * pv + F * torch.matmul(vis64, v64.abs() + 1) if rel is not None and r else o32_bound + rT * (o.abs() + o32_bound)
        e_D = (do.abs() * ((d + 2) * U * o.abs() + o_used)).sum(-1, keepdim=True)
        bs = p * (eP * (dp.abs() + Dr.abs()) + e_dp + e_D) + 4 * U * ds.abs() + F * vis64 * (dp.abs() + Dr.abs() + 1)
        a = ds.abs()
        fold = lambda x: x.view(B, Hkv, G, *x.shape[2:]).sum(2)
        self.dq = (torch.matmul(ds, k64) * scale).transpose(1, 2)
        self.dq_bound = (scale * torch.matmul(bs + (r + (Nk + 4) * U) * (a + bs) + F * vis64, k64.abs() + 1)).transpose(1, 2)
        self.dq_bound = self.dq_bound + rT * (self.dq.abs() + self.dq_bound)
        dk = fold(torch.matmul(T(ds), q64)) * scale
        bk_ = scale * fold(torch.matmul(T(bs + (r + (G * Nq + 4) * U) * (a + bs)), q64.abs())) + F * scale * fold(torch.matmul(T(vis64), q64.abs() + 1))
        dv = fold(torch.matmul(T(p), do))
        bv = fold(torch.matmul(T(p * (eP + r + (G * Nq + 4) * U) + F * vis64), do.abs() + 1))
        self.dk, self.dk_bound = dk.transpose(1, 2), (bk_ + rT * (dk.abs() + bk_)).transpose(1, 2)
        self.dv, self.dv_bound = dv.transpose(1, 2), (bv + rT * (dv.abs() + bv)).transpose(1, 2)
        self.seen = seen
        if rel is not None:
            hot = torch.nn.functional.one_hot(bk, nb).double()                      # [B, Nq, Nk, nb]
            ein = lambda x: torch.matmul(hot.reshape(-1, nb).t().contiguous(), x.permute(0, 2, 3, 1).reshape(-1, H).contiguous())
            self.dtable, self.dtable_bound = ein(ds), ein(bs) + (hot.sum((0, 1, 2))[:, None].clamp(max=4096) + 64) * U * ein(a)


def within(name, got, ref, bound):
    got = got.double()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - ref).abs() - bound
    assert (over <= 0).all(), f"{name}: {int((over > 0).sum())} of {over.numel()} outside, worst {float(((got - ref).abs() / bound).max()):.2f} of the bound"


def check(cb, dtype, B, Nq, Nk, H, Hkv, d, causal=False, rel=None, seed=0, grad=True, scale=None, hide_nan=True, amp=1.0, **kw):
    """one call, forward and backward, against Ref; hidden places of K, V, Q and dout hold NaN"""
    lib, ctx = cb
    q, k, v = rnd(B, Nq, H, d, seed=seed, dtype=dtype, scale=amp), rnd(B, Nk, Hkv, d, seed=seed + 1, dtype=dtype, scale=amp), rnd(B, Nk, Hkv, d, seed=seed + 2, dtype=dtype)
    dout = rnd(B, Nq, H, d, seed=seed + 3, dtype=dtype)
    t = {n: (torch.tensor(x, dtype=torch.int32, device=_dev()) if isinstance(x, list) else x) for n, x in kw.items()}
    relpos = table = None
    if rel is not None:
        relpos = lib.RelPos(ctx, *rel)
        table = rnd(rel[0], H, seed=seed + 4)
    scale = d ** -0.5 if scale is None else scale
    ref = Ref(q, k, v, scale, causal=causal, rel=rel, table=table, dout=dout if grad else None, **t)
    if hide_nan:
        j, i = torch.arange(Nk, device=_dev()), torch.arange(Nq, device=_dev())
        hid = torch.zeros(B, Nk, dtype=torch.bool, device=_dev())
        if t.get("kv_len") is not None:
            hid |= j[None] >= t["kv_len"][:, None]
        if t.get("kv_mask") is not None:
            hid |= ~t["kv_mask"].bool()
        k[hid], v[hid] = float("nan"), float("nan")
        if t.get("q_len") is not None:
            q[i[None] >= t["q_len"][:, None]] = float("inf")
            dout[i[None] >= t["q_len"][:, None]] = float("nan")
    got = lib.seq_attention(ctx, q, k, v, scale=scale, causal=causal, relpos=relpos, table=table, need_grad=grad, **t)
    out, tape = got if grad else (got, None)
    within("out", out, ref.out, ref.out_bound)
    if not grad:
        return
    fin = torch.isfinite(ref.lse)
    assert torch.equal(fin, torch.isfinite(tape.lse)) and (tape.lse[~fin] == -math.inf).all()
    assert ((tape.lse.double() - ref.lse)[fin].abs() <= ref.lse_bound[fin]).all()
    g = lib.seq_attention_backward(ctx, tape, dout)
    within("dq", g.dq, ref.dq, ref.dq_bound)
    within("dk", g.dk, ref.dk, ref.dk_bound)
    within("dv", g.dv, ref.dv, ref.dv_bound)
    assert not g.dk[~ref.seen].any() and not g.dv[~ref.seen].any()
    if rel is not None:
        within("dtable", g.dtable, ref.dtable, ref.dtable_bound)
    again = lib.seq_attention_backward(ctx, tape, dout)                            # no sum depends on the order of arrival
    for x in ("dq", "dk", "dv"):
        assert torch.equal(getattr(g, x), getattr(again, x)), x
    assert rel is None or torch.equal(g.dtable, again.dtable)


DT = pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])


@DT
@pytest.mark.parametrize("Nq,Nk", [(1, 1), (1, 65), (77, 77), (64, 64), (65, 63), (130, 200), (5, 300), (300, 5)])
def test_attention_sizes(cb, dtype, Nq, Nk):
    check(cb, dtype, 2, Nq, Nk, 3, 3, 64)


@DT
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 48, 56, 64, 72, 80, 96, 120, 128, 136, 160])
def test_attention_head_dims(cb, dtype, d):
    check(cb, dtype, 1, 70, 90, 2, 1, d, kv_len=[83])


@DT
@pytest.mark.parametrize("H,Hkv", [(4, 4), (4, 2), (6, 1), (8, 2)])
def test_attention_shared_heads(cb, dtype, H, Hkv):
    check(cb, dtype, 2, 100, 140, H, Hkv, 32, causal=True)
    check(cb, dtype, 2, 100, 140, H, Hkv, 32, rel=(32, 128, True))


@DT
@pytest.mark.parametrize("causal", [False, True])
def test_attention_lengths(cb, dtype, causal):
    check(cb, dtype, 5, 130, 130, 2, 2, 64, causal=causal, kv_len=[130, 0, 1, 64, 65], q_len=[130, 130, 1, 0, 65])


@DT
def test_attention_lengths_out_of_range_are_held(cb, dtype):
    lib, ctx = cb
    q, k, v = rnd(3, 20, 2, 32, dtype=dtype), rnd(3, 30, 2, 32, seed=1, dtype=dtype), rnd(3, 30, 2, 32, seed=2, dtype=dtype)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=_dev())
    a = lib.seq_attention(ctx, q, k, v, kv_len=i32(10 ** 9, -5, 30), q_len=i32(10 ** 9, 20, -7))
    b = lib.seq_attention(ctx, q, k, v, kv_len=i32(30, 0, 30), q_len=i32(20, 20, 0))
    assert torch.equal(a, b) and not a[1].any() and not a[2].any()


@DT
@pytest.mark.parametrize("rel", [None, (32, 128, True)])
def test_attention_masks(cb, dtype, rel):
    m = torch.rand(4, 200, generator=torch.Generator().manual_seed(3)) < 0.5
    m[0] = False                                      # a sample that sees nothing
    m[1, :130] = False                                # whole tiles without a visible key
    m[2] = True
    check(cb, dtype, 4, 90, 200, 2, 2, 64, kv_mask=m.to(_dev()), kv_len=[200, 190, 77, 200], rel=rel)
    check(cb, dtype, 4, 90, 200, 2, 2, 64, kv_mask=m.to(_dev()).to(torch.uint8) * 7, causal=True, rel=rel)


@DT
@pytest.mark.parametrize("rel", [(32, 128, True), (32, 128, False), (16, 64, True), (64, 256, False), (4, 2, True), (2, 2, False), (256, 1024, True), (64, 33, False)])
@pytest.mark.parametrize("causal", [False, True])
def test_relative_bias(cb, dtype, rel, causal):
    check(cb, dtype, 2, 150, 150, 2, 2, 64, rel=rel, causal=causal, kv_len=[150, 101])


@DT
@pytest.mark.parametrize("d", [40, 80, 128, 160])
def test_relative_bias_head_dims(cb, dtype, d):
    check(cb, dtype, 1, 140, 200, 2, 1, d, rel=(32, 64, True))
    check(cb, dtype, 1, 70, 70, 2, 1, d, rel=(64, 1024, True))


@DT
def test_relative_bias_far_distances(cb, dtype):
    """tiles on both sides of the table's range, and queries that start far into (or before) the keys"""
    check(cb, dtype, 1, 700, 700, 1, 1, 32, rel=(32, 64, True))
    check(cb, dtype, 4, 90, 400, 2, 2, 32, rel=(32, 128, False), causal=True, q_pos=[0, 310, 1000000, -50])
    check(cb, dtype, 4, 90, 400, 2, 2, 32, rel=(32, 128, True), q_pos=[-2 ** 31, 2 ** 31 - 1, 5, 399])


@DT
@pytest.mark.parametrize("rel", [None, (32, 128, True)])
def test_split_axes(cb, dtype, rel):
    """few blocks: the long axis is split over blocks, with parts that hold nothing; and the key counts where the row sums change their source"""
    check(cb, dtype, 2, 77, 2500, 2, 1, 64, rel=rel, kv_len=[2500, 70])
    check(cb, dtype, 1, 40, 1100, 2, 2, 40, rel=rel, causal=True, q_pos=[600], kv_len=[900])
    check(cb, dtype, 2, 2500, 77, 2, 1, 64, rel=rel, kv_len=[77, 0])
    m = torch.zeros(1, 1300, dtype=torch.bool, device=_dev())
    m[0, 700:720] = True
    check(cb, dtype, 1, 100, 1300, 2, 2, 80, rel=rel, kv_mask=m)
    for Nk in (127, 128, 129):
        check(cb, dtype, 1, 70, Nk, 2, 2, 32, rel=rel)
    check(cb, dtype, 6, 2100, 70, 16, 16, 32, rel=rel)              # enough blocks for 32 queries a wave


@DT
def test_wide_blocks(cb, dtype):
    """enough work for the kernels that hold 32 rows a wave, at an odd length"""
    check(cb, dtype, 8, 650, 650, 12, 12, 64, causal=True, rel=(32, 128, False), kv_len=[650, 1, 64, 65, 333, 640, 0, 512])
    check(cb, dtype, 4, 600, 700, 40, 10, 32, kv_len=[700, 130, 650, 9])


@DT
def test_table_entries_at_the_edge(cb, dtype):
    """-inf hides a bucket; the type's lowest value in every bucket leaves the plain softmax (all scores are absorbed alike)"""
    lib, ctx = cb
    q, k, v = (rnd(1, 100, 2, 64, seed=i, dtype=dtype) for i in range(3))
    rp = lib.RelPos(ctx, 32, 128, True)
    t = rnd(32, 2, seed=5)
    t[3] = -math.inf
    ref = Ref(q, k, v, 0.125, rel=(32, 128, True), table=t)
    within("hidden bucket", lib.seq_attention(ctx, q, k, v, relpos=rp, table=t), ref.out, ref.out_bound)
    t = torch.full((32, 2), torch.finfo(torch.float32).min, device=_dev())
    mean = v.double().mean(1, keepdim=True).expand_as(v)
    got = lib.seq_attention(ctx, q, k, v, relpos=rp, table=t).double()
    assert ((got - mean).abs() <= (R if dtype == BF else U) * 3 + 200 * U * v.double().abs().mean(1, keepdim=True) + (R if dtype == BF else 0) * v.double().abs().mean(1, keepdim=True)).all()
    t[:] = -math.inf
    out, tape = lib.seq_attention(ctx, q, k, v, relpos=rp, table=t, need_grad=True)
    assert not out.any() and (tape.lse == -math.inf).all()
    g = lib.seq_attention_backward(ctx, tape, rnd(1, 100, 2, 64, seed=9, dtype=dtype))
    assert not g.dq.any() and not g.dk.any() and not g.dv.any() and not g.dtable.any()


@DT
def test_large_scores(cb, dtype):
    """scores of some hundreds: the running maximum has to move, and rows whose weight is on one key"""
    check(cb, dtype, 1, 130, 260, 2, 2, 64, amp=6.0, scale=1.0)


@DT
def test_nan_in_a_visible_place_shows(cb, dtype):
    lib, ctx = cb
    q, k, v = (rnd(1, 80, 1, 32, seed=i, dtype=dtype) for i in range(3))
    k[0, 70] = float("nan")
    out = lib.seq_attention(ctx, q, k, v, causal=True)
    assert torch.isfinite(out[0, :70]).all() and torch.isnan(out[0, 70:]).all()


@DT
def test_strides_and_fused_buffers(cb, dtype):
    lib, ctx = cb
    B, N, H, d = 2, 90, 3, 40
    fused = rnd(B, N, 3 * H + 1, d, dtype=dtype)                                  # q | k | v and a head that is not ours
    q, k, v = fused[:, :, :H], fused[:, :, H:2 * H], fused[:, :, 2 * H:3 * H]
    c = [x.contiguous() for x in (q, k, v)]
    want, tape0 = lib.seq_attention(ctx, *c, need_grad=True)
    do = rnd(B, N, H, d, seed=8, dtype=dtype)
    g0 = lib.seq_attention_backward(ctx, tape0, do)
    got, tape = lib.seq_attention(ctx, q, k, v, need_grad=True)
    assert torch.equal(want, got)
    grad = torch.full_like(fused, 7.0)
    wide = rnd(B, N, H + 2, d, seed=8, dtype=dtype)
    wide[:, :, 1:H + 1] = do
    lib.seq_attention_backward(ctx, tape, wide[:, :, 1:H + 1], dq=grad[:, :, :H], dk=grad[:, :, H:2 * H], dv=grad[:, :, 2 * H:3 * H])
    assert torch.equal(grad[:, :, :3 * H], torch.cat([g0.dq, g0.dk, g0.dv], 2)) and (grad[:, :, 3 * H] == 7.0).all()
    t = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in c]                # head-major storage
    out = torch.zeros(B, H, N, d, dtype=dtype, device=_dev())
    r = lib.seq_attention(ctx, *t, out=out.transpose(1, 2))
    assert torch.equal(r, want) and torch.equal(out.transpose(1, 2), want)
    one = [x[:1].expand(B, N, H, d) for x in c]                                    # one sample broadcast: stride 0
    assert torch.equal(lib.seq_attention(ctx, *one), lib.seq_attention(ctx, *[x.contiguous() for x in one]))


@pytest.mark.parametrize("Nq", [1, 70])
def test_offsets_past_32_bits(cb, Nq):
    """keys, values and their gradients of one sample 5 GB apart: the same numbers as in a small buffer"""
    lib, ctx = cb
    N, H, d, row = 5000, 2, 64, 1 << 19
    far = torch.empty(N, row, dtype=torch.bfloat16, device=_dev())
    view = lambda buf, at: buf[:, at:at + H * d].unflatten(1, (H, d))[None]
    q, k, v = rnd(1, Nq, H, d, dtype=torch.bfloat16), rnd(1, N, H, d, seed=1, dtype=torch.bfloat16), rnd(1, N, H, d, seed=2, dtype=torch.bfloat16)
    kf, vf = view(far, 0), view(far, 1024)
    kf.copy_(k); vf.copy_(v)
    do = rnd(1, Nq, H, d, seed=3, dtype=torch.bfloat16)
    want, t0 = lib.seq_attention(ctx, q, k, v, need_grad=True)
    got, t1 = lib.seq_attention(ctx, q, kf, vf, need_grad=True)
    assert torch.equal(want, got)
    g0 = lib.seq_attention_backward(ctx, t0, do)
    grad = torch.empty(N, row, dtype=torch.bfloat16, device=_dev())
    g1 = lib.seq_attention_backward(ctx, t1, do, dk=view(grad, 512), dv=view(grad, 4096))
    assert torch.equal(g0.dq, g1.dq) and torch.equal(g0.dk, view(grad, 512)) and torch.equal(g0.dv, view(grad, 4096))


@DT
def test_one_token_over_a_cache(cb, dtype):
    check(cb, dtype, 6, 1, 700, 4, 2, 64, rel=(32, 128, False), causal=True, kv_len=[700, 1, 129, 640, 0, 333], q_pos=[699, 0, 128, 639, -1, 332], grad=False)
    check(cb, dtype, 3, 1, 5000, 8, 2, 128, kv_len=[5000, 4097, 17], grad=False)
    check(cb, dtype, 2, 1, 3000, 4, 4, 64, rel=(32, 128, False), causal=True, kv_len=[3000, 2000], q_pos=[2999, 1999])


@DT
@pytest.mark.parametrize("d", [8, 24, 40, 64, 80, 128, 160])
@pytest.mark.parametrize("H,Hkv", [(2, 2), (4, 2), (6, 2), (8, 1), (16, 1)])
def test_one_token_shapes(cb, dtype, d, H, Hkv):
    """head dims and head sharing of the one-token kernel (and 16 heads on one: the tile kernel), masks, empty samples, the statistics it keeps"""
    m = torch.rand(4, 600, generator=torch.Generator().manual_seed(3)) < 0.5
    m[1] = False
    check(cb, dtype, 4, 1, 600, H, Hkv, d, kv_mask=m.to(_dev()), kv_len=[600, 600, 0, 33], rel=(32, 64, True), q_pos=[300, 5, 7, 40], q_len=[1, 1, 1, 1])
    check(cb, dtype, 2, 1, 2100, H, Hkv, d, kv_len=[2100, 257], q_len=[1, 0])


@DT
def test_difference_quotient(cb, dtype):
    """gradients against differences of the forward pass: the loss sum(out * w) along a random direction, in fp32 inputs"""
    if dtype == BF:
        pytest.skip("a step that bf16 resolves is too coarse for differences")
    lib, ctx = cb
    B, N, H, d = 1, 40, 2, 32
    q, k, v, w = (rnd(B, N, H, d, seed=i).double() for i in range(4))
    rp = lib.RelPos(ctx, 16, 32, True)
    t = rnd(16, H, seed=7).double()
    out, tape = lib.seq_attention(ctx, q.float(), k.float(), v.float(), relpos=rp, table=t.float(), need_grad=True)
    g = lib.seq_attention_backward(ctx, tape, w.float())
    h = 2.0 ** -7
    for name, x, gr in (("q", q, g.dq), ("k", k, g.dk), ("v", v, g.dv), ("table", t, g.dtable)):
        dirn = torch.sign(rnd(*x.shape, seed=11)).double()
        val = []
        for s in (-h, h):
            a = dict(q=q, k=k, v=v, table=t)
            a[name] = x + s * dirn
            o = lib.seq_attention(ctx, *(a[n].float().contiguous() for n in ("q", "k", "v")), relpos=rp, table=a["table"].float())
            val.append(float((o.double() * w).sum()))
        num, ana = (val[1] - val[0]) / (2 * h), float((gr.double() * dirn).sum())
        # fp32 outputs: each sum(out * w) is off by at most sum |w| * 2^-20 (|out| <= 4); the third derivative leaves h^2 of the gradient's scale
        tol = float(w.abs().sum()) * 4 * 2.0 ** -20 / h + 40 * h * h * float(gr.double().abs().sum()) / 40
        assert abs(num - ana) <= tol, (name, num, ana, tol)


def test_stream_and_device_are_checked(cb):
    lib, ctx = cb
    q, k, v = (rnd(1, 8, 1, 32, seed=i) for i in range(3))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        with pytest.raises(ValueError, match="stream"):
            lib.seq_attention(ctx, q, k, v)
    with pytest.raises(ValueError, match="is on cpu"):
        lib.seq_attention(ctx, q.cpu(), k, v)


def test_captured_training_step_replays(cb):
    """two graphs of one context, replayed in turn with eager calls between: every replay equals the eager result for the inputs of the time"""
    lib, _ = cb
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ctx = lib.Context()
        rp = lib.RelPos(ctx)
        table = rnd(32, 4, seed=3)
        sets = []
        for n in (100, 300):
            q, k, v, do = (rnd(2, n, 4, 64, seed=i, dtype=BF) for i in range(4))
            kl = torch.tensor([n, n // 2], dtype=torch.int32, device=_dev())

            def step(q=q, k=k, v=v, do=do, kl=kl):
                out, tape = lib.seq_attention(ctx, q, k, v, relpos=rp, table=table, kv_len=kl, need_grad=True)
                g = lib.seq_attention_backward(ctx, tape, do)
                return out, g.dq, g.dk, g.dv, g.dtable
            step()
            s.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                res = step()
            sets.append((graph, res, step, q, kl))
        for turn in range(4):
            for graph, res, step, q, kl in sets:
                q.copy_(rnd(*q.shape, seed=50 + turn, dtype=BF))
                kl.sub_(1)
                graph.replay()
                want = step()
                s.synchronize()
                for a, b in zip(res, want):
                    assert torch.equal(a, b)
