"""GPU tests of the 8-bit product of few tokens with very many output channels (a projection onto a vocabulary): exact sums on both sides of the
row counts at which the tile changes, and the whole epilogue."""
import pytest
import torch

from test_gpu_i8_ops import i8, product64, rnd
from test_gpu_seq_ops import R, U, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cb(built_lib):
    from celebbasis_amd import lib
    ctx = lib.Context()
    yield lib, ctx
    ctx.sync()


@pytest.mark.parametrize("N,K", [(49152, 768), (40961, 528), (33000, 1040)])
@pytest.mark.parametrize("M", [17, 64, 65, 100, 128, 129])
def test_few_tokens_onto_many_channels(cb, M, N, K):
    lib, ctx = cb
    a, b = i8(M, K, seed=M, lo=-128), i8(N, K, seed=N)
    v = product64(a, b)
    one = torch.ones(N, device=a.device)
    assert torch.equal(lib.linear_i8(ctx, a, one[:M], b, one, dtype="f32").double(), v.float().double())
    sa, sb, bias, res = rnd(M, seed=1).abs() * 0.01, rnd(N, seed=2).abs() * 0.01, rnd(N, seed=3), rnd(M, N, seed=4).to(torch.bfloat16)
    got = lib.linear_i8(ctx, a, sa, b, sb, bias=bias, residual=res)
    v = v * sa.double()[:, None] * sb.double()[None]
    want = v + bias.double() + res.double()
    bnd = 4 * U * (v.abs() + bias.double().abs() + res.double().abs())
    within("C", got, want, bnd + R * (want.abs() + bnd))
