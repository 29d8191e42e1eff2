"""CPU tier: properties of the generated gfx950 code of the paged cache's kernels.

No private (scratch) memory, no packed fp32 arithmetic, and attention loops that keep the next tile's loads under way: a
wait for all loads (vmcnt(0)) in a block that both loads and multiplies would mean that they are not."""
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
    runs = {}
    for src in ("zq_paged.hip", "zq_attn_paged.hip", "zq_page_select.hip"):
        path = tmp / (src + ".s")
        runs[src] = path, subprocess.Popen(
            [HIPCC, *[f for f in FLAGS if f not in ("-shared", "-fPIC")], "--cuda-device-only", "-S", "-o", str(path),
             os.path.join(ROOT, "zeninfer_amd", "csrc", src)], stderr=subprocess.PIPE, text=True)
    out = {}
    for src, (path, r) in runs.items():
        err = r.communicate(timeout=900)[1]
        assert r.returncode == 0, err[-2000:]
        out[src] = path.read_text()
    return out


def functions(text):
    for m in re.finditer(r"^(_Z\S+):", text, re.M):
        yield m.group(1), text[m.end():text.find(".Lfunc_end", m.end())]


def test_scratch_and_packed_fp32(asm):
    for src, text in asm.items():
        kernels = re.findall(r"^\s*\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", text, re.M | re.S)
        assert len(kernels) >= 4
        for name, body in kernels:
            assert re.search(r"\.amdhsa_private_segment_fixed_size 0\b", body), (src, name)
        assert not re.search(r"^\s*v_pk_(?:fma|add|mul)_f32\b", text, re.M), src


def test_attention_keeps_loads_under_way(asm):
    found = 0
    for name, body in functions(asm["zq_attn_paged.hip"]):
        if "attn_paged_kernel" not in name and "attn_paged_pair_kernel" not in name:
            continue
        for b in re.split(r"^\.LBB\S+:", body, flags=re.M):
            if "v_mfma" not in b:
                continue
            if b.count("global_load") > 2:  # (the last tile's block asks for the next tiles' places alone)
                found += 1
                waits = [int(n) for n in re.findall(r"s_waitcnt[^\n]*vmcnt\((\d+)\)", b)]
                assert 0 not in waits, (name, waits)
    assert found >= 27  # three types, three dimensions, three kernels
