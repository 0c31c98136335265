"""The built library's kernels as instructions, for tests of the waits between them: the AMD assembly of code that is compiled here."""
import os
import re
import shutil
import struct
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

NO_NEXT = ("s_branch", "s_endpgm", "s_setpc_b64")
LINE = re.compile(r"\t(\S+)\s*(.*?)\s*// ([0-9A-F]+):.*?(?:<[^>+]*(?:\+0x([0-9a-f]+))?>)?$")


def instructions(lines):
    """(name, operands) of every instruction, and the places that may follow each."""
    code, place, jumps = [], {}, []
    for line in lines:
        found = LINE.match(line)
        if found:
            name, operands, address, target = found.groups()
            if name == "s_branch" or name.startswith("s_cbranch"):
                jumps.append((len(code), int(target or "0", 16)))
            place[int(address, 16)] = len(code)
            code.append((name, operands))
    after = [[i + 1] if i + 1 < len(code) and name not in NO_NEXT else [] for i, (name, _) in enumerate(code)]
    start = min(place, default=0)
    for i, jump in jumps:
        after[i].append(place[start + jump])
    return code, after


def wait_states(name, operands):
    return int(operands.split()[0], 0) + 1 if name == "s_nop" else 1


def listing(*code):
    """Lines as the disassembler writes them, of (instruction, address to branch to or 0)."""
    return [f"\t{c} // {4 * i:012X}: 00000000" + (f" <k+0x{to:x}>" if to else "") for i, (c, to) in enumerate(code)]


def kernels_with(word, look, folder):
    """`look(lines)` of every kernel of the built library that has `word` in its assembly, by name."""
    from sprout_lm_amd.csrc.build import ensure_built
    tools = [shutil.which(name, path=os.environ.get("PATH", "") + ":/opt/rocm/llvm/bin") for name in ("llvm-objcopy", "llvm-objdump")]
    if not all(tools):
        pytest.skip("llvm-objcopy and llvm-objdump are not here")
    subprocess.run([tools[0], "--dump-section", f".hip_fatbin={folder}/all", ensure_built(), f"{folder}/copy"], check=True)
    data, at, objects = (folder / "all").read_bytes(), 0, []
    while (at := data.find(b"__CLANG_OFFLOAD_BUNDLE__", at)) >= 0:      # one a source: number of entries, then offset, size and name of each
        entry = at + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            offset, size, name = struct.unpack_from("<QQQ", data, entry)
            if b"gfx950" in data[entry + 24:entry + 24 + name]:
                objects.append(folder / f"{len(objects)}.co")
                objects[-1].write_bytes(data[at + offset:at + offset + size])
            entry += 24 + name
        at += 24

    def walk(path):
        text = subprocess.run([tools[1], "-d", str(path)], check=True, capture_output=True, text=True).stdout
        parts = re.split(r"^(?:[0-9a-f]+ )?<(.+)>:$", text, flags=re.MULTILINE) if word in text else [""]
        return [(name, look(body.split("\n"))) for name, body in zip(parts[1::2], parts[2::2]) if word in body]
    with ThreadPoolExecutor(8) as pool:
        return [kernel for of_source in pool.map(walk, objects) for kernel in of_source]
