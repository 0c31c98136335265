"""Loads into LDS are written as assembly, whose waits the compiler does not count.  A load may read a scalar register five wait states after a
vector instruction wrote it; the built library's kernels are walked along all their branches for loads that come sooner."""
import re

from tests.assembly_helpers import instructions, kernels_with, listing, wait_states

WAIT_STATES = 5
LOADS = ("global_", "buffer_", "flat_", "scratch_")
SCALARS = re.compile(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b|\b(vcc)")


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
    code, after = instructions(lines)
    before = [[] for _ in code]
    for i, places in enumerate(after):
        for j in places:
            before[j].append(i)
    writes, bad = [written_by_vector(*c) for c in code], []
    for i, (name, operands) in enumerate(code):
        reads = scalars(operands) if name.startswith(LOADS) else set()
        todo, least = [(j, 0) for j in before[i]] if reads else [], {}
        while todo:
            j, waited = todo.pop()
            if waited >= WAIT_STATES or least.get(j, WAIT_STATES) <= waited:
                continue
            least[j] = waited
            if writes[j] & reads:
                bad.append((" ".join(code[j]), " ".join(code[i])))
                continue
            todo += [(k, waited + wait_states(*code[j])) for k in before[j]]
    return bad, sum("load_lds" in name for name, _ in code)


def test_the_walk_finds_what_it_looks_for():
    lane, load = ("v_readlane_b32 s5, v2, 3", 0), ("global_load_lds_dwordx4 v1, s[4:5]", 0)
    moves, more = ("s_mov_b32 m0, s9", 0), lambda n: (f"s_nop {n}", 0)
    assert too_early(listing(lane, moves, more(0), load)) == ([(lane[0], load[0])], 1)
    assert too_early(listing(lane, moves, more(2), load))[0] and not too_early(listing(lane, moves, more(3), load))[0]
    assert not too_early(listing(("v_readlane_b32 s6, v2, 3", 0), load))[0]
    # behind a branch: the load follows the lane's number by two on one way and by six on the other
    assert too_early(listing(lane, ("s_cbranch_scc1 2", 12), more(4), moves, load))[0]
    assert not too_early(listing(lane, ("s_branch 2", 16), load, more(0), more(4), load))[0]


def test_no_load_reads_a_scalar_too_early(tmp_path):
    found = kernels_with("load_lds", too_early, tmp_path)
    for part in ("attention_shared_kernel", "attention_rows", "gemm_q4_staged_kernel", "gemm_pipe", "gemm_quad"):
        assert any(part in name and loads for name, (_, loads) in found), part
    assert [(name, bad[0], len(bad)) for name, (bad, _) in found if bad] == []
