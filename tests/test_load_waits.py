"""Loads into LDS are written as assembly, whose waits the compiler does not count.  A load may read a scalar register five wait states after a
vector instruction wrote it; the built library's kernels are walked along all their branches for loads that come sooner."""
import os
import re
import shutil
import struct
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

WAIT_STATES = 5
LOADS = ("global_", "buffer_", "flat_", "scratch_")
NO_NEXT = ("s_branch", "s_endpgm", "s_setpc_b64")
SCALARS = re.compile(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b|\b(vcc)")
LINE = re.compile(r"\t(\S+)\s*(.*?)\s*// ([0-9A-F]+):.*?(?:<[^>+]*(?:\+0x([0-9a-f]+))?>)?$")


def scalars(operand):
    out = set()
    for first, last, single, vcc in SCALARS.findall(operand):
        out |= {106, 107} if vcc else set(range(int(first), int(last) + 1)) if first else {int(single)}
    return out


def written_by_vector(name, operands):
    """Scalar registers that a vector instruction writes: lanes read out, comparisons' and carries' masks."""
    if not name.startswith("v_"):
        return set()
    parts = operands.split(",")
    out = scalars(parts[0])
    if len(parts) > 1 and ("_co_" in name or name.startswith(("v_div_scale", "v_mad_u64", "v_mad_i64"))):
        out |= scalars(parts[1])
    return out | ({106, 107} if name.startswith("v_cmp") and parts[0].strip().startswith("v") else set())


def too_early(lines):
    """(vector instruction, load) of every load that reads a scalar register too soon, and how many loads into LDS there are."""
    code, place = [], {}
    for line in lines:
        found = LINE.match(line)
        if found:
            name, operands, address, target = found.groups()
            jump = int(target or "0", 16) if name == "s_branch" or name.startswith("s_cbranch") else None
            place[int(address, 16)] = len(code)
            code.append((name, operands, jump))
    start = min(place) if place else 0
    before = [[] for _ in code]
    for i, (name, _, jump) in enumerate(code):
        if i + 1 < len(code) and name not in NO_NEXT:
            before[i + 1].append(i)
        if jump is not None:
            before[place[start + jump]].append(i)
    writes, bad = [written_by_vector(name, operands) for name, operands, _ in code], []
    for i, (name, operands, _) in enumerate(code):
        reads = scalars(operands) if name.startswith(LOADS) else set()
        todo, least = [(j, 0) for j in before[i]] if reads else [], {}
        while todo:
            j, waited = todo.pop()
            if waited >= WAIT_STATES or least.get(j, WAIT_STATES) <= waited:
                continue
            least[j] = waited
            if writes[j] & reads:
                bad.append((" ".join(code[j][:2]), " ".join(code[i][:2])))
                continue
            states = int(code[j][1].split()[0], 0) + 1 if code[j][0] == "s_nop" else 1
            todo += [(k, waited + states) for k in before[j]]
    return bad, sum("load_lds" in name for name, _, _ in code)


def kernels(text):
    name, lines = None, []
    for line in text.split("\n"):
        head = re.match(r"(?:[0-9a-f]+ )?<(.+)>:$", line)
        if head:
            if name:
                yield name, lines
            name, lines = head.group(1), []
        else:
            lines.append(line)
    if name:
        yield name, lines


def test_the_walk_finds_what_it_looks_for():
    def listing(*code):
        return [f"\t{c} // {4 * i:012X}: 00000000" + (f" <k+0x{to:x}>" if to else "") for i, (c, to) in enumerate(code)]
    lane, load = ("v_readlane_b32 s5, v2, 3", 0), ("global_load_lds_dwordx4 v1, s[4:5]", 0)
    moves, more = ("s_mov_b32 m0, s9", 0), lambda n: (f"s_nop {n}", 0)
    assert too_early(listing(lane, moves, more(0), load)) == ([(lane[0], load[0])], 1)
    assert too_early(listing(lane, moves, more(2), load))[0] and not too_early(listing(lane, moves, more(3), load))[0]
    assert not too_early(listing(("v_readlane_b32 s6, v2, 3", 0), load))[0]
    # behind a branch: the load follows the lane's number by two on one way and by six on the other
    assert too_early(listing(lane, ("s_cbranch_scc1 2", 12), more(4), moves, load))[0]
    assert not too_early(listing(lane, ("s_branch 2", 16), load, more(0), more(4), load))[0]


def test_no_load_reads_a_scalar_too_early(tmp_path):
    from sprout_lm_amd.csrc.build import ensure_built
    tools = [shutil.which(name, path=os.environ.get("PATH", "") + ":/opt/rocm/llvm/bin") for name in ("llvm-objcopy", "llvm-objdump")]
    if not all(tools):
        pytest.skip("llvm-objcopy and llvm-objdump are not here")
    subprocess.run([tools[0], "--dump-section", f".hip_fatbin={tmp_path}/all", ensure_built(), f"{tmp_path}/copy"], check=True)
    data, at, objects = (tmp_path / "all").read_bytes(), 0, []
    while (at := data.find(b"__CLANG_OFFLOAD_BUNDLE__", at)) >= 0:      # one a source: number of entries, then offset, size and name of each
        entry = at + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            offset, size, name = struct.unpack_from("<QQQ", data, entry)
            if b"gfx950" in data[entry + 24:entry + 24 + name]:
                objects.append(tmp_path / f"{len(objects)}.co")
                objects[-1].write_bytes(data[at + offset:at + offset + size])
            entry += 24 + name
        at += 24

    def walk(path):
        text = subprocess.run([tools[1], "-d", str(path)], check=True, capture_output=True, text=True).stdout
        return [(name, *too_early(lines)) for name, lines in kernels(text) if any("load_lds" in line for line in lines)] if "load_lds" in text else []
    with ThreadPoolExecutor(8) as pool:
        found = [kernel for of_source in pool.map(walk, objects) for kernel in of_source]
    for part in ("attention_shared_kernel", "attention_rows", "gemm_q4_staged_kernel", "gemm_pipe", "gemm_quad"):
        assert any(part in name and loads for name, _, loads in found), part
    assert [(name, bad[0], len(bad)) for name, bad, _ in found if bad] == []
