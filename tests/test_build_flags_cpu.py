"""CPU tests of the build's flags of the sequence operators."""
import json
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_flags_of_the_sequence_operators():
    """the attention kernels are built with the accumulators beside the vector registers and all of these files without packed fp32 instructions"""
    from celebbasis_amd import build
    for src in ("cb_seq_fwd.hip", "cb_seq_bwd.hip", "cb_seq_short.hip", "cb_seq_token.hip", "cb_norm_i8.hip", "cb_gemm_i8.hip"):
        assert src in build.SOURCES and "-packed-fp32-ops" in build.EXTRA[src], src
    for src in ("cb_seq_fwd.hip", "cb_seq_bwd.hip", "cb_seq_short.hip"):
        assert build.EXTRA[src][:len(build.EXTRA["cb_flash.hip"])] == build.EXTRA["cb_flash.hip"], src
    assert "-amdgpu-mfma-vgpr-form" in build.EXTRA["cb_flash.hip"]


def _build_with(tmp_path, rejected):
    """the build against a stub compiler that rejects one flag: (return code, output, commands by source)"""
    stub = tmp_path / "hipcc_stub.py"
    stub.write_text("""#!/usr/bin/env python3
import json, os, sys
a = sys.argv[1:]
if os.environ['STUB_REJECTS'] in a:
    sys.exit('unknown argument')
out = a[a.index('-o') + 1]
if '-c' in a:
    with open(os.environ['STUB_LOG'], 'a') as f:
        f.write(json.dumps([os.path.basename(a[a.index('-c') + 1]), a]) + '\\n')
if '-Rpass-analysis=kernel-resource-usage' in a:
    for k in ('gemm_glds_stub', 'gemm_bf16_p8_stub'):
        sys.stderr.write('x.hip:1:1: remark: Function Name: ' + k + ' [-Rpass]\\nx.hip:1:1: remark:     ScratchSize [bytes/lane]: 0 [-Rpass]\\n')
open(out, 'w').write('stub')
""")
    stub.chmod(0o755)
    code = (f"import sys; sys.path.insert(0, {ROOT!r})\nfrom celebbasis_amd import build\n"
            f"build.BUILD = {str(tmp_path / '_build')!r}; build.LIB = {str(tmp_path / 'lib.so')!r}\nbuild.build(verbose=False)\n")
    log = tmp_path / "log.txt"
    log.write_text("")
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, HIPCC=str(stub), STUB_LOG=str(log), STUB_REJECTS=rejected),
                       capture_output=True, text=True, timeout=120)
    return r.returncode, r.stdout + r.stderr, dict(json.loads(line) for line in log.read_text().splitlines())


def test_a_rejected_tuning_flag_leaves_the_others(tmp_path):
    """a compiler without the accumulator flag still builds the sequence operators without packed fp32 instructions"""
    rc, out, cmds = _build_with(tmp_path, "-amdgpu-mfma-vgpr-form")
    assert rc == 0 and "rejects" in out, out[-400:]
    for src in ("cb_seq_fwd.hip", "cb_seq_bwd.hip", "cb_seq_short.hip", "cb_seq_token.hip", "cb_norm_i8.hip", "cb_gemm_i8.hip"):
        assert "-packed-fp32-ops" in cmds[src] and "-amdgpu-mfma-vgpr-form" not in cmds[src], src


def test_a_rejected_guard_flag_fails_the_build(tmp_path):
    rc, out, cmds = _build_with(tmp_path, "-packed-fp32-ops")
    assert rc != 0 and "packed" in out and "cb_seq_fwd.hip" not in cmds, out[-400:]
