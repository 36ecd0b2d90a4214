"""CPU tests of the build's flags of the sequence operators."""


def test_flags_of_the_sequence_operators():
    """the attention kernels are built with the accumulators beside the vector registers and all of these files without packed fp32 instructions"""
    from celebbasis_amd import build
    for src in ("cb_seq_fwd.hip", "cb_seq_bwd.hip", "cb_seq_short.hip", "cb_seq_token.hip", "cb_norm_i8.hip", "cb_gemm_i8.hip"):
        assert src in build.SOURCES and "-packed-fp32-ops" in build.EXTRA[src], src
    for src in ("cb_seq_fwd.hip", "cb_seq_bwd.hip", "cb_seq_short.hip"):
        assert build.EXTRA[src][:len(build.EXTRA["cb_flash.hip"])] == build.EXTRA["cb_flash.hip"], src
    assert "-amdgpu-mfma-vgpr-form" in build.EXTRA["cb_flash.hip"]
