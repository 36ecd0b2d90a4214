"""CPU tests of the sequence operators' host side: bucket borders in exact arithmetic, refusals through a dry context, descriptor layout."""
import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def dry(built_lib):
    from celebbasis_amd import lib
    return lib, lib.Context(device=-1)


def exact_bucket(rel, num_buckets, D, two):
    """the definition, in whole numbers"""
    nb = num_buckets // 2 if two else num_buckets
    E, base = nb // 2, nb if two and rel > 0 else 0
    n = abs(rel) if two else max(-rel, 0)
    if n < E:
        return base + n
    m = nb - E
    return base + E + sum(n ** m * E ** k >= E ** m * D ** k for k in range(1, m))


@pytest.mark.parametrize("nb,D,two", [(32, 128, True), (32, 128, False), (64, 256, True), (16, 64, True), (16, 64, False), (4, 2, True), (2, 2, False),
                                      (256, 1024, False), (8, 1024, True), (64, 33, False)])
def test_relpos_buckets_are_exact(dry, nb, D, two):
    lib, ctx = dry
    rp = lib.RelPos(ctx, nb, D, two)
    for rel in list(range(-min(D, 300) - 3, min(D, 300) + 4)) + [-D - 1, -D, D, D + 1, -10 ** 12, 10 ** 12]:
        assert rp.bucket(rel) == exact_bucket(max(-D, min(D, rel)), nb, D, two), rel
    # past the range everything shares the outermost bucket
    assert rp.bucket(-D) == rp.bucket(-10 ** 9) and rp.bucket(D) == rp.bucket(10 ** 9)


@pytest.mark.parametrize("nb,D,two", [(30, 128, True), (258, 128, False), (0, 128, True), (32, 8, True), (32, 1025, True), (3, 128, False)])
def test_relpos_refusals(dry, nb, D, two):
    lib, ctx = dry
    with pytest.raises(lib.CBError) as e:
        lib.RelPos(ctx, nb, D, two)
    assert e.value.code == -1


def test_sequence_descriptors_match_the_header(built_lib, tmp_path):
    from celebbasis_amd import lib
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    pairs = [("cb_seq_tensor", lib.SeqTensor), ("cb_seq_attention_desc", lib.SeqAttentionDesc)]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "celebbasis_hip.h"', "int main(void) {"]
    for cname, cls in pairs:
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        lines += [f'  printf("%zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for _, cls in pairs:
        want += [C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


def qkv(B=2, Nq=5, Nk=7, H=4, Hkv=2, d=16, dtype=torch.float32):
    return torch.zeros(B, Nq, H, d, dtype=dtype), torch.zeros(B, Nk, Hkv, d, dtype=dtype), torch.zeros(B, Nk, Hkv, d, dtype=dtype)


def test_seq_attention_accepts_what_it_documents(dry):
    lib, ctx = dry
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v = qkv(dtype=dtype)
        rp = lib.RelPos(ctx)
        out, tape = lib.seq_attention(ctx, q, k, v, relpos=rp, table=torch.zeros(32, 4), causal=True, kv_len=torch.zeros(2, dtype=torch.int32),
                                      kv_mask=torch.ones(2, 7, dtype=torch.bool), need_grad=True)
        g = lib.seq_attention_backward(ctx, tape, torch.zeros_like(out))
        assert out.shape == q.shape and g.dk.shape == k.shape and g.dtable.shape == (32, 4)
    for kw in (dict(B=0), dict(Nq=0), dict(Nk=0), dict(Nq=1, Nk=1, H=1, Hkv=1, d=8)):
        q, k, v = qkv(**kw)
        out, tape = lib.seq_attention(ctx, q, k, v, need_grad=True)
        lib.seq_attention_backward(ctx, tape, torch.zeros_like(out))
    x = torch.zeros(2, 5, 8, 16)                                     # slices of one fused projection, and a transposed cache
    lib.seq_attention(ctx, x[:, :, :4], x[:, :, 4:6], x[:, :, 6:])
    cache = torch.zeros(2, 2, 7, 16).transpose(1, 2)
    lib.seq_attention(ctx, qkv()[0], cache, cache)
    lib.seq_attention(ctx, qkv()[0], cache[:1].expand(2, -1, -1, -1), cache)


@pytest.mark.parametrize("change,exc", [
    (dict(d=12), "head dim"), (dict(d=168), "head dim"), (dict(H=3), "kv_heads"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(kv_len=torch.zeros(3, dtype=torch.int32)), "kv_len"),
    (dict(kv_len=torch.zeros(2, dtype=torch.int64)), "kv_len"), (dict(kv_mask=torch.zeros(2, 6, dtype=torch.bool)), "kv_mask"),
    (dict(kv_mask=torch.zeros(2, 7)), "kv_mask"), (dict(table=torch.zeros(32, 4)), "together"), (dict(dtype=torch.float16), "float"),
    (dict(v_shape=(2, 6, 2, 16)), "v has shape"), (dict(v_dtype=torch.bfloat16), "v: expected dtype"), (dict(stride=True), "contiguous"),
    (dict(odd=True), "16 bytes"), (dict(shift=True), "aligned"), (dict(overlap=True), "overlaps"),
])
def test_seq_attention_refusals(dry, change, exc):
    lib, ctx = dry
    q, k, v = qkv(**{x: y for x, y in change.items() if x in ("d", "H", "dtype")})
    kw = {x: y for x, y in change.items() if x in ("scale", "kv_len", "kv_mask", "table")}
    if "v_shape" in change:
        v = torch.zeros(change["v_shape"])
    if "v_dtype" in change:
        v = v.to(change["v_dtype"])
    if "stride" in change:
        k = torch.zeros(2, 7, 16, 2).transpose(2, 3)
    if "odd" in change:
        k = torch.zeros(2, 7, 2, 18)[..., :16]
    if "shift" in change:
        k = torch.zeros(2 * 7 * 2 * 16 + 1)[1:].view(2, 7, 2, 16)
    if "overlap" in change:
        kw["out"] = torch.zeros(1, 5, 4, 16).expand(2, 5, 4, 16)
    with pytest.raises((ValueError, TypeError, lib.CBError), match=exc):
        lib.seq_attention(ctx, q, k, v, **kw)


def test_seq_attention_refuses_results_over_inputs(dry):
    lib, ctx = dry
    q, k, v = qkv()
    with pytest.raises(lib.CBError, match="out overlaps q"):
        lib.seq_attention(ctx, q, k, v, out=q)
    out, tape = lib.seq_attention(ctx, q, k, v, need_grad=True)
    do = torch.zeros_like(out)
    for kw, what in ((dict(dq=q), "dq overlaps q"), (dict(dk=k), "dk overlaps k"), (dict(dv=k), "dv overlaps k"), (dict(dq=do), "dq overlaps dout"), (dict(dq=out), "dq overlaps out")):
        with pytest.raises(lib.CBError, match=what):
            lib.seq_attention_backward(ctx, tape, do, **kw)
    same = torch.zeros(2, 7, 4, 16)                                   # dk and dv as slices of one buffer
    lib.seq_attention_backward(ctx, tape, do, dk=same[:, :, :2], dv=same[:, :, 2:])


def test_seq_attention_descriptor_refusals(dry):
    """what the Python wrapper cannot express: a foreign struct size, a short or misaligned workspace, gradients of a table that is not there"""
    lib, ctx = dry
    q, k, v = qkv()
    D = lib.SeqAttentionDesc()
    D.B, D.Nq, D.Nk, D.heads, D.kv_heads, D.d, D.scale = 2, 5, 7, 4, 2, 16, 0.25
    out, lse, keep = torch.zeros_like(q), torch.zeros(2, 4, 5), []
    D.lse = lse.data_ptr()
    for x, t in (("q", q), ("k", k), ("v", v), ("out", out), ("dout", out.clone()), ("dq", q.clone()), ("dk", k.clone()), ("dv", v.clone())):
        keep.append(t)
        setattr(D, x, lib.SeqTensor(t.data_ptr(), t.stride(1), t.stride(2), t.stride(0)))
    so = lib.load()
    D.struct_size -= 8
    assert so.cb_seq_attention_fwd(ctx.h, C.byref(D)) == -1 and b"struct_size" in so.cb_last_error()
    D.struct_size += 8
    assert so.cb_seq_attention_fwd(ctx.h, None) == -1 and so.cb_seq_attention_fwd(None, C.byref(D)) == -1
    need = C.c_int64()
    assert so.cb_seq_attention_workspace(ctx.h, C.byref(D), 1, C.byref(need)) == 0 and need.value > 0
    D.workspace_bytes = need.value - 1
    assert so.cb_seq_attention_bwd(ctx.h, C.byref(D)) == -1 and b"workspace" in so.cb_last_error()
    D.workspace_bytes, D.workspace = need.value, 0x1008
    assert so.cb_seq_attention_bwd(ctx.h, C.byref(D)) == -1 and b"aligned" in so.cb_last_error()
    D.workspace, D.dtable = 0x1000, 0x1000
    assert so.cb_seq_attention_bwd(ctx.h, C.byref(D)) == -1 and b"dtable" in so.cb_last_error()
    D.dtable, D.dtype = None, 7
    assert so.cb_seq_attention_bwd(ctx.h, C.byref(D)) == -1


def test_norm_and_product_descriptors_match_the_header(built_lib, tmp_path):
    from celebbasis_amd import lib
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    pairs = [("cb_rmsnorm_desc", lib.RmsNormDesc), ("cb_gemm_i8_desc", lib.GemmI8Desc)]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "celebbasis_hip.h"', "int main(void) {"]
    for cname, cls in pairs:
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        lines += [f'  printf("%zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for _, cls in pairs:
        want += [C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


def test_norm_accepts_and_refuses(dry):
    lib, ctx = dry
    x, g = torch.zeros(3, 4, 40), torch.ones(40)
    n = lib.rms_norm(ctx, x, g, residual=x, need_grad=True)
    assert n.y.shape == x.shape and n.rstd.shape == (3, 4)
    dh, dg = lib.rms_norm_backward(ctx, x, n.h, g, n.rstd, dres=x)
    assert dh.shape == x.shape and dg.shape == (40,)
    assert lib.rms_norm(ctx, x.to(torch.bfloat16), g, out="i8").y.shape == (3, 4, 48)
    lib.rms_norm(ctx, torch.zeros(5, 50)[:, :40], g)
    for bad, kw, what in ((x.half(), {}, "float"), (x, dict(residual=x[:2]), "residual has shape"), (x, dict(residual=x.to(torch.bfloat16)), "residual"),
                          (x, dict(eps=-1.0), "eps"), (x, dict(eps=float("nan")), "eps"), (x, dict(out="i4"), "i8"), (x.transpose(0, 1), {}, "contiguous"),
                          (torch.zeros(5, 80)[:, ::2], {}, "contiguous"), (torch.zeros(2, 16385), {}, "shape|C ="), (torch.zeros(2, 39), {}, "weight")):
        w = torch.ones(16385) if bad.shape[-1] == 16385 else g
        with pytest.raises((ValueError, TypeError, lib.CBError), match=what):
            lib.rms_norm(ctx, bad, w, **kw)
    with pytest.raises(ValueError, match="shape"):
        lib.rms_norm_backward(ctx, x[:, :3], n.h, g, n.rstd)
    with pytest.raises(ValueError, match="rstd"):
        lib.rms_norm_backward(ctx, x, n.h, g, n.rstd[:1])
    so = lib.load()
    d = lib.RmsNormDesc()
    d.rows, d.C, d.ldx, d.ldy, d.ldi8 = 4, 40, 40, 40, 40
    y = torch.zeros(4, 48)
    p = lambda t: t.data_ptr()
    d.x, d.gamma, d.y, d.y_i8 = p(y), p(g), p(y), p(y)
    assert so.cb_rmsnorm_fwd(ctx.h, C.byref(d)) == -1 and b"exactly one" in so.cb_last_error()
    d.y = None
    assert so.cb_rmsnorm_fwd(ctx.h, C.byref(d)) == -3 and b"16-byte" in so.cb_last_error()       # ldi8 = 40
    d.ldi8, d.ldx = 48, 39
    assert so.cb_rmsnorm_fwd(ctx.h, C.byref(d)) == -3 and b"shorter" in so.cb_last_error()
    d.ldx, d.struct_size = 40, 8
    assert so.cb_rmsnorm_fwd(ctx.h, C.byref(d)) == -1
    d.struct_size = C.sizeof(d)
    d.h = d.dy = d.dh = p(y)
    d.ldh = d.lddy = d.lddh = 40
    d.dgamma, d.workspace_bytes = p(y), 0
    assert so.cb_rmsnorm_bwd(ctx.h, C.byref(d)) == -1 and b"workspace" in so.cb_last_error()


def test_rows_and_product_accept_and_refuse(dry):
    lib, ctx = dry
    q, s = lib.quantize_rows(ctx, torch.zeros(2, 3, 100))
    assert q.shape == (2, 3, 112) and q.dtype == torch.int8 and s.shape == (2, 3)
    w, ws = lib.quantize_rows(ctx, torch.zeros(50, 100))
    assert lib.linear_i8(ctx, q, s, w, ws, bias=torch.zeros(50), residual=torch.zeros(2, 3, 50, dtype=torch.bfloat16)).shape == (2, 3, 50)
    assert lib.linear_i8(ctx, q, s, w, ws, dtype="f32").dtype == torch.float32
    for args, kw, what in (((q, s, w[:, :96], ws), {}, "expected"), ((q, s[:1], w, ws), {}, "a_scale"), ((q, s, w, ws.double()), {}, "w_scale"),
                           ((q.float(), s, w, ws), {}, "int8"), ((q, s, w, ws), dict(bias=torch.zeros(49)), "bias"),
                           ((q, s, w, ws), dict(residual=torch.zeros(2, 3, 50)), "residual"), ((q, s, w[0], ws), {}, "w has shape"),
                           ((q[..., :100].contiguous(), s, w[:, :100].contiguous(), ws), {}, "multiple of 16"), ((q, s, w, ws), dict(dtype="f16"), "dtype")):
        with pytest.raises((ValueError, TypeError, lib.CBError), match=what):
            lib.linear_i8(ctx, *args, **kw)
    with pytest.raises(lib.CBError, match="at most"):
        lib.quantize_rows(ctx, torch.zeros(1, 131057))
    so = lib.load()
    d = lib.GemmI8Desc()
    d.M, d.N, d.K, d.lda, d.ldb, d.ldc = 4, 4, 32, 40, 32, 4
    t = torch.zeros(4, 64)
    for k in ("A", "B", "C", "a_scale", "b_scale"):
        setattr(d, k, t.data_ptr())
    assert so.cb_gemm_i8(ctx.h, C.byref(d)) == -3 and b"16-byte" in so.cb_last_error()
    d.lda, d.K = 32, 131072
    assert so.cb_gemm_i8(ctx.h, C.byref(d)) == -3 and b"at most" in so.cb_last_error()
    d.K, d.ldc = 32, 3
    assert so.cb_gemm_i8(ctx.h, C.byref(d)) == -3 and b"shorter" in so.cb_last_error()
    d.ldc, d.struct_size = 4, 1
    assert so.cb_gemm_i8(ctx.h, C.byref(d)) == -1


@pytest.mark.parametrize("m,n", [(0, 70), (70, 0), (0, 0), (300, 0)])
def test_product_of_nothing(dry, m, n):
    """no rows or no outputs: nothing to ask a workspace for, nothing to divide a split by"""
    lib, ctx = dry
    k = 8192
    d = lib.GemmI8Desc()
    d.M, d.N, d.K, d.lda, d.ldb, d.ldc = m, n, k, k, k, max(n, 1)
    t = torch.zeros(16, dtype=torch.int32)
    for name in ("A", "B", "C", "a_scale", "b_scale"):
        setattr(d, name, t.data_ptr())
    need = C.c_int64(-1)
    assert lib.load().cb_gemm_i8_workspace(ctx.h, C.byref(d), C.byref(need)) == 0 and need.value == 0
    assert lib.load().cb_gemm_i8(ctx.h, C.byref(d)) == 0
    got = lib.linear_i8(ctx, torch.zeros(m, k, dtype=torch.int8), torch.zeros(m), torch.zeros(n, k, dtype=torch.int8), torch.zeros(n))
    assert got.shape == (m, n)


@pytest.mark.parametrize("b,h,nq,nk", [(0, 4, 9, 9), (2, 4, 0, 9), (2, 4, 9, 0), (2, 4, 0, 0), (2, 4, 1, 0), (0, 4, 1, 300), (2, 4, 300, 0), (2, 4, 0, 300)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_of_nothing(dry, dtype, b, h, nq, nk):
    """empty samples, queries or keys pass through the plans of both directions"""
    lib, ctx = dry
    q, k, v = torch.zeros(b, nq, h, 64, dtype=dtype), torch.zeros(b, nk, 2, 64, dtype=dtype), torch.zeros(b, nk, 2, 64, dtype=dtype)
    out, tape = lib.seq_attention(ctx, q, k, v, need_grad=True)
    g = lib.seq_attention_backward(ctx, tape, torch.zeros_like(out))
    assert out.shape == q.shape and g.dq.shape == q.shape and g.dk.shape == k.shape and g.dv.shape == v.shape
