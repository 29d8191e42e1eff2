"""CPU tier: properties of the generated gfx950 code of the paged cache's kernels.

No private (scratch) memory, no packed fp32 arithmetic, and attention loops that keep the next tile's loads under way: a
wait for all loads (vmcnt(0)) in a block that both loads and multiplies would mean that they are not."""
import bisect
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


# ---- what a load brings is read before the next load takes its registers -----------
_REG = re.compile(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])")


def _regs(ops):
    out = set()
    for kind, one, a, b in (r for o in ops for r in _REG.findall(o)):
        out |= {(kind, int(one))} if one else {(kind, i) for i in range(int(a), int(b) + 1)}
    return out


def lost_loads(body):
    """(vector loads of a kernel's body, those of them of which some register is loaded again on a path without having been
    read, with whether their basic block multiplies).  Other writes count as reads: what they mean depends on the lanes."""
    ins, labels = [], {}
    for line in body.split("\n"):
        line = line.split(";")[0].strip()
        label = re.match(r"(\.?\w+):$", line)
        if label:
            labels[label.group(1)] = len(ins)
        elif line and not line.startswith("."):
            name, _, ops = line.partition(" ")
            ins.append((name, re.split(r",(?![^\[]*\])", ops)))
    touched, loads = [], {}
    for i, (name, ops) in enumerate(ins):
        load = re.match(r"(global|buffer|flat)_load", name)
        touched.append(_regs(ops[1:] if load else ops) if not name.startswith("s_") else set())
        if load:
            loads[i] = _regs(ops[:1])

    def after(i):
        name, ops = ins[i]
        if name.startswith(("s_branch", "s_cbranch")):
            return [labels[ops[0].strip()]] + ([i + 1] if name != "s_branch" else [])
        return [i + 1] if name != "s_endpgm" and i + 1 < len(ins) else []
    edges = [after(i) for i in range(len(ins))]
    starts = sorted(set(labels.values()) | {i + 1 for i in range(len(ins)) if len(edges[i]) != 1 or edges[i][0] != i + 1})
    block = lambda i: bisect.bisect_right(starts, i)
    multiplies = {block(i) for i, (name, _) in enumerate(ins) if "mfma" in name}
    wide = [i for i in loads if "dwordx" in ins[i][0]]
    lost = []
    for i in wide:
        for reg in loads[i]:
            todo, seen, gone = list(edges[i]), set(), False
            while todo and not gone:
                j = todo.pop()
                if j in seen or reg in touched[j]:
                    continue
                seen.add(j)
                gone = reg in loads.get(j, ())
                todo += edges[j]
            if gone:
                lost.append((i, block(i) in multiplies))
                break
    return len(wide), lost


def test_loaded_tiles_are_read_before_the_next_load_takes_their_registers(asm):
    """A register allocation that overwrote half of a V load has been met once (in a build that was not kept).  In kernels
    of one pair a workgroup no loaded register may be loaded again unread on any path; in those of several pairs a
    share, whose first tile is loaded before it is known that there is one, none that the tiles' loop loads."""
    pairs = shares = 0
    for name, body in functions(asm["zq_attn_paged.hip"]):
        if "attn_paged_pair_kernel" in name:
            loads, lost = lost_loads(body)
            assert loads and not lost, (name, lost)
            pairs += 1
        elif "attn_paged_kernel" in name:
            loads, lost = lost_loads(body)
            assert loads and not [i for i, in_loop in lost if in_loop], (name, lost)
            shares += 1
    assert pairs == 18 and shares == 27


def test_a_lost_load_is_found(asm):
    """The same kernel with one load repeated before its value is read."""
    name, body = next((n, b) for n, b in functions(asm["zq_attn_paged.hip"]) if "attn_paged_pair_kernel" in n)
    lines = body.split("\n")
    at = [i for i, line in enumerate(lines) if re.search(r"global_load_dwordx4", line)]
    for i in (at[0], at[len(at) // 2], at[-1]):
        assert lost_loads("\n".join(lines[:i + 1] + lines[i:]))[1]
