"""GPU tests of the sequence attention at the edges of its definition: table entries of -inf and of very large magnitude over whole key tiles, and
their gradients.

Bounds as in test_gpu_seq_ops.py (u = 2^-24, r = 2^-8 for bf16 operands and results). A table entry b of magnitude 1e8 and more takes every score
|s| < ulp(b) / 2 up whole: s + b rounds to b, so all keys of such entries weigh alike; against keys of ordinary entries their weight is 0 exactly. What is
left of a probability's error is that of the ordinary scores (2 (d + 8) u of their magnitude), of a logarithm of at most 16 (2^-20 before the
exponential, ln 2 2^-20 behind it) and of the exponentials: 2^-19 in all."""
import math

import pytest
import torch

from test_gpu_seq_ops import BF, F, R, U, buckets, check, rnd, within

pytestmark = pytest.mark.gpu
DT = pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
LOWEST = torch.finfo(torch.float32).min


def _dev():
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def cb(built_lib):
    from celebbasis_amd import lib
    ctx = lib.Context()
    yield lib, ctx
    ctx.sync()


T = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731


def check_table(cb, dtype, B, Nq, Nk, H, d, rel, table, causal=False, q_pos=None, kv_mask=None, scale=None, amp=1.0, seed=0):
    """forward and backward with the given table against 64 bits (one key head a query head)"""
    lib, ctx = cb
    dev = _dev()
    q, k = rnd(B, Nq, H, d, seed=seed, dtype=dtype, scale=amp), rnd(B, Nk, H, d, seed=seed + 1, dtype=dtype, scale=amp)
    v, do = rnd(B, Nk, H, d, seed=seed + 2, dtype=dtype), rnd(B, Nq, H, d, seed=seed + 3, dtype=dtype)
    scale = d ** -0.5 if scale is None else scale
    pos32 = torch.tensor(q_pos, dtype=torch.int32, device=dev) if q_pos is not None else None
    rp = lib.RelPos(ctx, *rel)
    nb, D, two = rel
    i, j = torch.arange(Nq, device=dev), torch.arange(Nk, device=dev)
    at = (i[None] + (pos32.long()[:, None] if pos32 is not None else 0)).expand(B, Nq)
    dist = j[None, None] - at[:, :, None]
    ok = torch.ones(B, Nq, Nk, dtype=torch.bool, device=dev)
    if causal:
        ok &= dist <= 0
    if kv_mask is not None:
        ok &= kv_mask[:, None]
    bk = buckets(dist, nb, D, two)
    bias = table.double()[bk].permute(0, 3, 1, 2)
    q64, k64, v64, do64 = (x.double().transpose(1, 2).contiguous() for x in (q, k, v, do))
    s = torch.matmul(q64, T(k64)) * scale
    mag = torch.matmul(q64.abs(), T(k64.abs())) * scale + bias.abs()
    huge = bias.abs() >= 1e8                                             # -inf among them
    s = torch.where(huge, bias, s + bias).masked_fill(~ok[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    tot = e.sum(-1, keepdim=True)
    p = torch.where(tot > 0, e / tot, 0.0)
    none = (tot == 0)[..., 0]                                            # rows that see nothing
    plain = ok[:, None] & ~huge
    eP = 2 * (d + 8) * U * (float(mag[plain].max()) if plain.any() else 0.0) + 2.0 ** -19
    r, rT = (R, R) if dtype == BF else (0.0, U)
    vis = ok[:, None].double().expand_as(p)
    o = torch.matmul(p, v64)
    ob = (eP + (Nk + 4) * U + r) * torch.matmul(p, v64.abs()) + F * torch.matmul(vis, v64.abs() + 1)
    ob = ob + rT * (o.abs() + ob)
    dp = torch.matmul(do64, T(v64))
    Dr = (do64 * o).sum(-1, keepdim=True)
    ds = p * (dp - Dr)
    e_dp = (d + 2) * U * torch.matmul(do64.abs(), T(v64.abs()))
    e_D = (do64.abs() * ((d + 2) * U * o.abs() + ob)).sum(-1, keepdim=True)
    bs = p * (eP * (dp.abs() + Dr.abs()) + e_dp + e_D) + 4 * U * ds.abs() + F * vis * (dp.abs() + Dr.abs() + 1)
    a = ds.abs()
    dq = torch.matmul(ds, k64) * scale
    dqb = scale * torch.matmul(bs + (r + (Nk + 4) * U) * (a + bs) + F * vis, k64.abs() + 1)
    dk = torch.matmul(T(ds), q64) * scale
    dkb = scale * torch.matmul(T(bs + (r + (Nq + 4) * U) * (a + bs) + F * vis), q64.abs() + 1)
    dv = torch.matmul(T(p), do64)
    dvb = torch.matmul(T(p * (eP + r + (Nq + 4) * U) + F * vis), do64.abs() + 1)

    out, tape = lib.seq_attention(ctx, q, k, v, scale=scale, causal=causal, q_pos=pos32, kv_mask=kv_mask, relpos=rp, table=table, need_grad=True)
    heads = lambda x: x.transpose(1, 2)                                   # noqa: E731
    within("out", out, heads(o), heads(ob))
    assert not heads(out)[none].any() and (tape.lse[none] == -math.inf).all() and torch.isfinite(tape.lse[~none]).all()
    bare = lib.seq_attention(ctx, q, k, v, scale=scale, causal=causal, q_pos=pos32, kv_mask=kv_mask, relpos=rp, table=table)
    assert torch.equal(bare, out)
    g = lib.seq_attention_backward(ctx, tape, do)
    for name, got, want, bnd in (("dq", g.dq, dq, dqb), ("dk", g.dk, dk, dkb), ("dv", g.dv, dv, dvb)):
        within(name, got, heads(want), heads(bnd + rT * (want.abs() + bnd)))
    hot = torch.nn.functional.one_hot(bk, nb).double().reshape(-1, nb).t().contiguous()
    by_bucket = lambda x: torch.matmul(hot, x.permute(0, 2, 3, 1).reshape(-1, H).contiguous())      # noqa: E731
    within("dtable", g.dtable, by_bucket(ds), by_bucket(bs) + (4096 + 64) * U * by_bucket(a) + F)
    assert not heads(g.dq)[none].any()
    again = lib.seq_attention_backward(ctx, tape, do)
    assert all(torch.equal(getattr(g, n), getattr(again, n)) for n in ("dq", "dk", "dv", "dtable"))


def _table(rel, H, value, which, seed=7):
    """a random table whose outermost buckets, or all of them, hold `value`"""
    nb, _, two = rel
    t = rnd(nb, H, seed=seed)
    if which == "all":
        t[:] = value
    else:
        t[nb // 2 - 1 if two else nb - 1] = value
        if two:
            t[nb - 1] = value
    return t


# keys in one short tile run, over tiles whole, over tiles split, and with 32 rows a wave (bf16)
SHAPES = [(2, 90, 100, 2), (2, 90, 200, 2), (1, 100, 700, 2), (8, 700, 700, 12)]


@DT
@pytest.mark.parametrize("value", [-math.inf, LOWEST, -1e9])
@pytest.mark.parametrize("B,Nq,Nk,H", SHAPES)
def test_outermost_bucket_hidden(cb, dtype, value, B, Nq, Nk, H):
    """a window: keys past the table's range carry -inf (or next to nothing) while near ones are ordinary; small and large scores"""
    for rel, causal in (((32, 64, True), False), ((32, 64, False), True)):
        t = _table(rel, H, value, "outer")
        check_table(cb, dtype, B, Nq, Nk, H, 64, rel, t, causal=causal)
        if value != -1e9:                      # (scores of hundreds are not absorbed by 1e9)
            check_table(cb, dtype, B, Nq, Nk, H, 64, rel, t, causal=causal, amp=6.0, scale=1.0)


@DT
@pytest.mark.parametrize("value", [-math.inf, LOWEST, -1e9])
def test_rows_that_see_only_hidden_buckets(cb, dtype, value):
    """queries far from every key, and a key mask that leaves far keys alone"""
    rel = (32, 64, True)
    t = _table(rel, 2, value, "outer")
    for Nk in (100, 200, 700):
        check_table(cb, dtype, 4, 70, Nk, 2, 64, rel, t, q_pos=[0, 2000, -2000, 300])
        m = torch.zeros(2, Nk, dtype=torch.bool, device=_dev())
        m[:, Nk - 20:] = True
        check_table(cb, dtype, 2, Nk - 10, Nk, 2, 64, rel, t, kv_mask=m)
    check_table(cb, dtype, 16, 520, 700, 16, 40, rel, _table(rel, 16, value, "outer"), q_pos=[1500] * 8 + [0] * 8)


@DT
@pytest.mark.parametrize("value", [LOWEST, -1e30, -1e9, 1e9, -math.inf])
@pytest.mark.parametrize("B,Nq,Nk,H", SHAPES)
def test_every_bucket_alike(cb, dtype, value, B, Nq, Nk, H):
    """all entries take the scores up whole: every visible key weighs the same, in the gradients too"""
    rel = (32, 64, True)
    check_table(cb, dtype, B, Nq, Nk, H, 64, rel, _table(rel, H, value, "all"))
    check_table(cb, dtype, B, Nq, Nk, H, 40, (16, 700, False), _table((16, 700, False), H, value, "all"), causal=True)
    if abs(value) != 1e9:
        check_table(cb, dtype, B, Nq, Nk, H, 64, rel, _table(rel, H, value, "all"), amp=6.0, scale=1.0)


@DT
def test_one_token_row_of_lowest_entries(cb, dtype):
    """the one-token kernel's statistics in the tile kernels' backward"""
    rel = (32, 64, True)
    for value in (LOWEST, -1e9, -math.inf):
        for Nk in (90, 600, 3000):
            check_table(cb, dtype, 3, 1, Nk, 2, 64, rel, _table(rel, 2, value, "all"), q_pos=[0, 50, 4000])
            check_table(cb, dtype, 3, 1, Nk, 2, 64, rel, _table(rel, 2, value, "outer"), q_pos=[0, 50, 4000])


@DT
@pytest.mark.parametrize("amp", [12.0, 24.0])
@pytest.mark.parametrize("rel", [None, (32, 64, True)])
def test_scores_of_thousands(cb, dtype, amp, rel):
    """ordinary rows on both sides of the magnitude at which the backward pass makes its statistics anew"""
    check(cb, dtype, 1, 130, 100, 2, 2, 64, amp=amp, scale=1.0, rel=rel)
    check(cb, dtype, 2, 130, 260, 2, 1, 64, amp=amp, scale=1.0, rel=rel, causal=True, kv_len=[260, 201])
    check(cb, dtype, 1, 70, 900, 2, 2, 80, amp=amp, scale=1.0, rel=rel)


@DT
@pytest.mark.parametrize("rel", [None, (32, 64, True)])
@pytest.mark.parametrize("Nq,Nk,H", [(100, 77, 2), (100, 200, 2), (100, 700, 2), (520, 700, 64), (1, 700, 2)])
def test_rows_without_keys_are_zero_beside_values_that_overflowed(cb, dtype, rel, Nq, Nk, H):
    """rows behind q_len, and rows before the first key in causal order, give 0 and take 0 where a value that other rows see is infinite"""
    lib, ctx = cb
    q, k, v = (rnd(2, n, H, 64, seed=i, dtype=dtype) for i, n in enumerate((Nq, Nk, Nk)))
    v[:, 3] = math.inf
    do = rnd(2, Nq, H, 64, seed=3, dtype=dtype)
    extra = dict(relpos=lib.RelPos(ctx, *rel), table=rnd(rel[0], H, seed=4)) if rel else {}
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=_dev())              # noqa: E731
    for kw, rows in ((dict(q_len=i32(Nq - Nq // 3 - 1, Nq)), [(0, slice(Nq - Nq // 3 - 1, Nq)), (1, slice(0, 0))]),
                     (dict(causal=True, q_pos=i32(-(Nq // 3) - 1, 8)), [(0, slice(0, Nq // 3 + 1)), (1, slice(0, 0))])):
        out, tape = lib.seq_attention(ctx, q, k, v, need_grad=True, **kw, **extra)
        g = lib.seq_attention_backward(ctx, tape, do)
        for b, r in rows:
            assert not out[b, r].any() and (tape.lse[b, :, r] == -math.inf).all() and not g.dq[b, r].any()
        assert not torch.isfinite(out[1, :, :]).all()                               # the infinity shows where it is seen


def _key_block(cb, B, Nq, Nk, H, Hkv, d, nb):
    """keys a block of the dK/dV kernel takes (64 or 128), told from what its parts of dtable need: whole key axes, so parts = blocks of keys"""
    import ctypes as C
    lib, ctx = cb
    rp = lib.RelPos(ctx, nb, 64, True)
    t = torch.zeros(16, device=_dev())
    D = lib.SeqAttentionDesc()
    D.dtype, D.B, D.Nq, D.Nk, D.heads, D.kv_heads, D.d, D.scale = lib.DTYPE_BF16, B, Nq, Nk, H, Hkv, d, 1.0
    D.relpos, D.table = rp.h, t.data_ptr()
    sizes = []
    for dtable in (None, t.data_ptr()):
        D.dtable = dtable
        n = C.c_int64()
        lib.check(lib.load().cb_seq_attention_workspace(ctx.h, C.byref(D), 1, C.byref(n)))
        sizes.append(n.value)
    parts = [b for b in (64, 128) if abs(sizes[1] - sizes[0] - B * H * -(-Nk // b) * nb * 4) < 256]
    assert len(parts) == 1, sizes
    return parts[0]


@pytest.mark.parametrize("d", [32, 40, 64])
@pytest.mark.parametrize("kind", ["causal", "two_sided", "shared", "plain"])
def test_backward_of_wide_blocks(cb, d, kind):
    """bf16, enough work for the backward kernels that hold 32 rows a wave (both take the same rule, on queries and on keys), odd lengths"""
    B, N, H, Hkv, kw = 11, 650, 12, 12, {}
    lens = [650, 1, 64, 65, 333, 640, 0, 512, 649, 129, 650]
    if kind == "causal":
        kw = dict(rel=(32, 64, False), causal=True, kv_len=lens, q_len=lens)
    elif kind == "two_sided":
        m = torch.rand(B, N, generator=torch.Generator().manual_seed(5)) < 0.6
        m[3] = False
        m[4, :300] = False
        kw = dict(rel=(32, 64, True), kv_mask=m.to(_dev()))
    elif kind == "shared":
        H, Hkv = 24, 12
        kw = dict(rel=(16, 128, True), kv_len=lens)
    else:
        kw = dict(kv_len=lens, causal=True, q_pos=[0, 5, 700, 0, -30, 0, 0, 100, 0, 0, 1])
    nb = kw.get("rel", (32,))[0]
    assert _key_block(cb, B, N, N, H, Hkv, d, nb) == 128 and _key_block(cb, 10, N, N, 12, 12, d, nb) == 64
    check(cb, BF, B, N, N, H, Hkv, d, **kw)
    if kind == "two_sided":
        check_table(cb, BF, B, N, N, H, d, kw["rel"], _table(kw["rel"], H, LOWEST, "outer"), kv_mask=kw["kv_mask"])


@DT
@pytest.mark.parametrize("d", [8, 40, 128, 160])
@pytest.mark.parametrize("Nk", [60, 120, 300, 900])
def test_large_entries_with_shared_heads(cb, dtype, d, Nk):
    """key / value heads shared by three query heads, lengths, a mask, causal order: the call with the heads repeated gives the same rows, and the
    gradients of the shared heads are the sums of its own (each stored with one rounding, the sum with another, in at most 4 more of fp32)"""
    lib, ctx = cb
    B, Nq, Hkv, G = 2, 90, 2, 3
    H, rel = Hkv * G, (32, 64, False)
    q, k, v = rnd(B, Nq, H, d, seed=1, dtype=dtype), rnd(B, Nk, Hkv, d, seed=2, dtype=dtype), rnd(B, Nk, Hkv, d, seed=3, dtype=dtype)
    do, rp = rnd(B, Nq, H, d, seed=4, dtype=dtype), lib.RelPos(ctx, *rel)
    m = torch.rand(B, Nk, generator=torch.Generator().manual_seed(6)).to(_dev()) < 0.7
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=_dev())              # noqa: E731
    t = rnd(rel[0], H, seed=5)
    t[:, 1], t[rel[0] - 1, 2], t[:, 4], t[3, 5] = LOWEST, -1e9, 3e9, -math.inf      # heads of one group differ
    kw = dict(causal=True, q_pos=i32(Nk - Nq + 20, 10), q_len=i32(Nq, 77), kv_len=i32(Nk, Nk - 9), kv_mask=m, relpos=rp, table=t, need_grad=True)
    out, tape = lib.seq_attention(ctx, q, k, v, **kw)
    g = lib.seq_attention_backward(ctx, tape, do)
    ke, ve = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2)
    want, tape2 = lib.seq_attention(ctx, q, ke, ve, **kw)
    w = lib.seq_attention_backward(ctx, tape2, do)
    for x in (out, tape.lse.nan_to_num(neginf=0.0), g.dq, g.dk, g.dv, g.dtable):
        assert torch.isfinite(x).all()
    assert torch.equal(tape.lse == -math.inf, tape2.lse == -math.inf)
    rt = R if dtype == BF else U
    near = lambda a, b, bound: ((a.double() - b.double()).abs() <= bound).all()     # noqa: E731
    # (how the axes are split may differ between the two calls: bf16 probabilities stay, fp32 sums move by their own rounding)
    assert near(out, want, 2 * rt * want.double().abs() + 2 * (Nk + 8) * U * v.double().abs().max())
    assert near(g.dq, w.dq, 2 * rt * w.dq.double().abs() + 2 * rt * w.dq.double().abs().amax(-1, keepdim=True) + 2 * (Nk + 64) * U * w.dq.double().abs().max())
    for a, b in ((g.dk, w.dk), (g.dv, w.dv)):
        parts = b.double().view(B, Nk, Hkv, G, d)
        assert near(a, parts.sum(3), rt * parts.abs().sum(3) + rt * a.double().abs() + 2 * (G * Nq + 64) * U * parts.abs().max())
