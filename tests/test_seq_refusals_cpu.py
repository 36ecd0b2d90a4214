"""CPU tests of what the sequence operators refuse: gradients laid over each other, and grids beyond a launch (a dry context: no GPU, all checks)."""
import itertools

import pytest
import torch


@pytest.fixture(scope="module")
def dry(built_lib):
    from celebbasis_amd import lib
    return lib, lib.Context(device=-1)


def _tape(dry, B=2, Nq=5, Nk=7, H=4, Hkv=2, d=16):
    lib, ctx = dry
    q, k, v = torch.zeros(B, Nq, H, d), torch.zeros(B, Nk, Hkv, d), torch.zeros(B, Nk, Hkv, d)
    out, tape = lib.seq_attention(ctx, q, k, v, need_grad=True)
    return tape, torch.zeros_like(out)


def test_gradients_over_each_other_are_refused(dry):
    lib, ctx = dry
    tape, do = _tape(dry)
    same = torch.zeros(2, 7, 2, 16)
    with pytest.raises(lib.CBError, match="dk overlaps dv"):
        lib.seq_attention_backward(ctx, tape, do, dk=same, dv=same)
    wide = torch.zeros(2, 7, 8, 16)
    with pytest.raises(lib.CBError, match="dk overlaps dv"):
        lib.seq_attention_backward(ctx, tape, do, dk=wide[:, :, 1:3], dv=wide[:, :, 2:4])
    both = torch.zeros(2, 9, 4, 16)
    with pytest.raises(lib.CBError, match="dq overlaps dk"):
        lib.seq_attention_backward(ctx, tape, do, dq=both[:, :5], dk=both[:, 2:, 1:3])
    with pytest.raises(lib.CBError, match="dq overlaps dv"):
        lib.seq_attention_backward(ctx, tape, do, dq=both[:, :5], dv=both[:, 2:, 1:3])


def test_gradients_side_by_side_are_taken(dry):
    """slices of heads, of tokens, of samples, of the head dim, and head-major buffers"""
    lib, ctx = dry
    tape, do = _tape(dry)
    x = torch.zeros(2, 7, 4, 16)
    lib.seq_attention_backward(ctx, tape, do, dk=x[:, :, :2], dv=x[:, :, 2:])
    lib.seq_attention_backward(ctx, tape, do, dk=x[:, :, 0::2], dv=x[:, :, 1::2])
    x = torch.zeros(2, 7, 2, 32)
    lib.seq_attention_backward(ctx, tape, do, dk=x[..., :16], dv=x[..., 16:])
    x = torch.zeros(2, 14, 2, 16)
    lib.seq_attention_backward(ctx, tape, do, dk=x[:, :7], dv=x[:, 7:])
    lib.seq_attention_backward(ctx, tape, do, dk=x[:, 0::2], dv=x[:, 1::2])
    x = torch.zeros(2, 4, 7, 16).transpose(1, 2)
    lib.seq_attention_backward(ctx, tape, do, dk=x[:, :, :2], dv=x[:, :, 2:])
    tape, do = _tape(dry, Nq=7)
    x = torch.zeros(2, 7, 8, 16)
    lib.seq_attention_backward(ctx, tape, do, dq=x[:, :, :4], dk=x[:, :, 4:6], dv=x[:, :, 6:])
    x = torch.zeros(2, 2, 7, 4, 16)
    lib.seq_attention_backward(ctx, tape, do, dq=x[0], dk=x[1][:, :, :2], dv=x[1][:, :, 2:])
    tape, do = _tape(dry, B=1, Nq=1, Nk=1, H=2, Hkv=2)
    x = torch.zeros(1, 1, 6, 16)
    lib.seq_attention_backward(ctx, tape, do, dq=x[:, :, :2], dk=x[:, :, 2:4], dv=x[:, :, 4:])
    tape, do = _tape(dry, B=0)
    lib.seq_attention_backward(ctx, tape, do, dk=torch.zeros(0, 7, 2, 16), dv=torch.zeros(0, 7, 2, 16))


def test_every_small_layout_against_its_addresses(dry):
    """dk and dv as views of one buffer at all offsets and a range of strides: refused if and only if an element is in both"""
    lib, ctx = dry
    B, N, H, d = 2, 3, 2, 8
    tape, do = _tape(dry, B=B, Nq=2, Nk=N, H=H, Hkv=H, d=d)
    buf = torch.zeros(4096)
    seen = [0, 0]
    orders = [(8, 16, 48), (16, 32, 96), (24, 8, 72), (8, 40, 120), (48, 16, 8), (16, 96, 32), (32, 8, 104)]      # (head, row, batch) strides
    idx = lambda st, o: {o + b * st[2] + n * st[1] + h * st[0] + c for b in range(B) for n in range(N) for h in range(H) for c in range(0, d, 4)}      # noqa: E731
    for st in orders:
        if len(idx(st, 0)) < B * N * H * 2:                             # overlaps itself: refused for that
            continue
        for off in range(0, 400, 4):
            dk = torch.as_strided(buf, (B, N, H, d), (st[2], st[1], st[0], 1), 0)
            dv = torch.as_strided(buf, (B, N, H, d), (st[2], st[1], st[0], 1), off)
            clash = bool(idx(st, 0) & idx(st, off))
            try:
                lib.seq_attention_backward(ctx, tape, do, dk=dk, dv=dv)
                said = ""
            except lib.CBError as e:
                said = str(e)
            assert ("dk overlaps dv" in said) == clash, (st, off, said)
            seen[clash] += 1
    assert min(seen) > 20
    for a, b in itertools.permutations(orders, 2):                      # other strides: never accepted where they meet
        for off in (0, 4, 8, 16, 24, 40):
            dk = torch.as_strided(buf, (B, N, H, d), (a[2], a[1], a[0], 1), 0)
            dv = torch.as_strided(buf, (B, N, H, d), (b[2], b[1], b[0], 1), off)
            if idx(a, 0) & idx(b, off):
                with pytest.raises(lib.CBError, match="overlaps"):
                    lib.seq_attention_backward(ctx, tape, do, dk=dk, dv=dv)


def test_product_grids_beyond_a_launch_are_refused(dry):
    """a launch holds fewer than 2^32 threads; 2^31 - 1 rows onto one channel would be 2^23 blocks of 512"""
    import ctypes as C
    lib, ctx = dry
    for m, n, ok in (((1 << 31) - 1, 1, False), ((1 << 31) - 600, 1, True), (1, 1 << 27, True), (1 << 30, 1, True)):
        d = lib.GemmI8Desc()
        d.M, d.N, d.K, d.lda, d.ldb, d.ldc = m, n, 16, 16, 16, n
        for name in ("A", "B", "C", "a_scale", "b_scale"):
            setattr(d, name, 0x1000)
        rc = lib.load().cb_gemm_i8(ctx.h, C.byref(d))
        assert (rc == 0) == ok and (ok or rc == -3 and b"too many" in lib.load().cb_last_error()), (m, n, rc, lib.load().cb_last_error())
