"""The build invariants of the hand-scheduled kernels on the code that is built: compiled with the commands of sfm_amd/csrc/Makefile
(tests/test_build_invariants.py has flags of its own, without the Makefile's -packed-fp32-ops), and those of the group norm and dropout."""
import concurrent.futures
import os
import re
import shlex
import subprocess

import pytest

import test_build_invariants as B


def _asm_as_built(src, contract, tmp_path):
    if not os.path.exists(B.HIPCC):
        pytest.skip("hipcc not available")
    obj = src.replace(".hip", ".o")
    lines = subprocess.check_output(["make", "-n", "-B", "--no-print-directory", obj], cwd=B.CSRC, text=True).replace("\\\n", " ").splitlines()
    (line,) = [v for v in lines if f"-c {src}" in v]
    args = shlex.split(line)
    assert [a for a in args if a.startswith("-ffp-contract")][-1] == f"-ffp-contract={contract}" and "-packed-fp32-ops" in args
    at = args.index("-c")
    assert args[at:at + 4] == ["-c", src, "-o", obj] and len(args) == at + 4
    out = str(tmp_path / (src + ".s"))
    subprocess.check_call([*args[:at], "--cuda-device-only", "-S", src, "-o", out], cwd=B.CSRC, stderr=subprocess.DEVNULL)
    return open(out).read()


@pytest.mark.parametrize("test", [B.test_stencil_kernels_have_no_scratch_and_no_exec_writing_valu, B.test_loss_kernels_have_no_scratch])
def test_of_the_loss(test, tmp_path, monkeypatch):
    monkeypatch.setattr(B, "_asm", _asm_as_built)
    test(tmp_path)


# bytes of scratch: masked kernels of the backward, whose registers are held down to the number of workgroups that their pass is launched with
# (type, elements of a vector, adjacent channels of one group in it; 0: any)
SCRATCH = {("sums", "16", 8, 1): 48, ("sums", "16", 8, 2): 16, ("sums", "16", 2, 1): 36, ("sums", "16", 2, 2): 24, ("sums", "32", 1, 1): 8,
           ("apply", "16", 8, 1): 84, ("apply", "16", 4, 0): 20, ("apply", "32", 4, 0): 20}


def test_group_norm_and_dropout(tmp_path):
    """no scratch and no packed fp32 instruction, but for the masked kernels named above"""
    sources = ["group_norm_fwd.hip", "group_norm_bwd.hip", "dropout.hip"]
    with concurrent.futures.ThreadPoolExecutor() as pool:
        texts = list(pool.map(lambda s: _asm_as_built(s, "off", tmp_path), sources))
    count = 0
    for text in texts:
        assert not re.search(r"\bv_pk_(add|mul|fma|mov)_(f32|b32)\b", text)
        for name, priv, spill, vgpr in B._kernels(text):
            count += 1
            allowed = 0
            m = re.search(r"gn_bwd_(sums|apply)_kernelILi(\d)ELi(\d)ELi(\d)ELb1E", name)
            if m:
                which, dt, v, e = m[1], "32" if m[2] == "0" else "16", int(m[3]), int(m[4])
                allowed = SCRATCH.get((which, dt, v, e), SCRATCH.get((which, dt, v, 0), 0))
            assert priv <= allowed, f"{name}: {priv} bytes of scratch, {spill} spilled VGPRs"
    assert count


def test_build_compiles_whatever_is_there(monkeypatch):
    import __graft_entry__ as g
    ran = []
    monkeypatch.setattr(g.subprocess, "check_call", lambda args, **kw: ran.append(args))
    g.build()
    assert len(ran) == 1 and ran[0][0] == "make" and "-B" in ran[0]
