"""CPU tier: properties of the generated gfx950 code of the 4-bit cache's kernels.

No kernel uses private (scratch) memory, and none packed fp32 arithmetic.  The
attention's loops keep a next tile's loads under way while they work on this
one: a wait for all loads (vmcnt(0)) in a block that holds matrix instructions
would mean that a branch around the loads has come back."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    if not shutil.which(HIPCC) and not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    from zeninfer_amd.build import FLAGS
    tmp = tmp_path_factory.mktemp("asm")
    out = {}
    for src in ("zq_kv.hip", "zq_attn_q4.hip"):
        path = tmp / (src + ".s")
        r = subprocess.run([HIPCC, *[f for f in FLAGS if f not in ("-shared", "-fPIC")], "--cuda-device-only", "-S", "-o",
                            str(path), os.path.join(ROOT, "zeninfer_amd", "csrc", src)], capture_output=True, text=True,
                           timeout=900)
        assert r.returncode == 0, r.stderr[-2000:]
        out[src] = path.read_text()
    return out


def test_no_scratch_and_no_packed_fp32(asm):
    for src, text in asm.items():
        kernels = re.findall(r"^\s*\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", text, re.M | re.S)
        assert len(kernels) >= 8
        for name, body in kernels:
            assert re.search(r"\.amdhsa_private_segment_fixed_size 0\b", body), (src, name)
        assert not re.search(r"^\s*v_pk_(?:fma|add|mul)_f32\b", text, re.M), src


def test_decode_attention_keeps_loads_under_way(asm):
    found = 0
    for m in re.finditer(r"^(_Z\S*attn_q4_few_kernel\S*):", asm["zq_attn_q4.hip"], re.M):
        body = asm["zq_attn_q4.hip"][m.end():asm["zq_attn_q4.hip"].find(".Lfunc_end", m.end())]
        blocks = re.split(r"^\.LBB\S+:", body, flags=re.M)
        loop = [b for b in blocks if "v_mfma" in b]
        assert loop, m.group(1)
        found += 1
        for b in loop:
            waits = [int(n) for n in re.findall(r"s_waitcnt[^\n]*vmcnt\((\d+)\)", b)]
            assert 0 not in waits, (m.group(1), waits)
    assert found == 3
