"""A matrix instruction's result may be read some wait states after its issue; no hardware holds a reader back, and behind branches the compiler has left
fewer.  The built library's kernels are walked along all their branches."""
import re

from tests.assembly_helpers import instructions, kernels_with, listing, wait_states

# From a matrix instruction to a vector or memory instruction, or another matrix instruction's operands (not its sum), that reads or overwrites the result
WAITS = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_32x32x16_bf16": 12, "v_mfma_f32_16x16x4_f32": 10, "v_mfma_f32_32x32x2_f32": 18}
READERS = ("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")
VECTORS = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def registers(text):
    out = set()
    for kind, first, last, single in VECTORS.findall(text):
        out |= {kind + single} if single else {f"{kind}{n}" for n in range(int(first), int(last) + 1)}
    return out


def too_early(lines):
    """(matrix instruction, reader, wait states between them) of every result that is taken too soon, and the matrix instructions met."""
    code, after = instructions(lines)
    read, bad, met = {}, [], set()
    for i, (name, operands) in enumerate(code):
        if not name.startswith("v_mfma"):
            continue
        met.add(name)
        result = registers(operands.split(",")[0])
        todo, least = [(j, 0) for j in after[i]], {}
        while todo:
            j, waited = todo.pop()
            if waited >= WAITS[name] or least.get(j, WAITS[name]) <= waited:
                continue
            least[j] = waited
            reader, its = code[j]
            if reader.startswith(READERS):
                if j not in read:
                    matrix = reader.startswith("v_mfma")
                    parts = its.split(",")
                    read[j] = registers(",".join(parts[1:3]) if matrix else its), registers(parts[0] + parts[3]) if matrix else set()
                if read[j][0] & result:
                    bad.append((f"{name} {operands}", f"{reader} {its}", waited))
                    continue
                if read[j][1] & result:      # the next product of the same sum: the matrix cores take them in order
                    continue
            todo += [(k, waited + wait_states(reader, its)) for k in after[j]]
    return bad, met


def test_the_walk_finds_what_it_looks_for():
    product, reader, more = ("v_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], 0", 0), ("v_mul_f32_e32 v40, s1, v9", 0), lambda n: (f"s_nop {n}", 0)
    assert too_early(listing(product, more(7), more(2), reader))[0] == [(product[0], reader[0], 11)]
    assert not too_early(listing(product, more(7), more(3), reader))[0]
    assert not too_early(listing(product, ("v_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], v[0:15]", 0), more(7), more(3), reader))[0]
    assert too_early(listing(product, ("v_mfma_f32_16x16x32_bf16 v[50:53], v[0:3], v[20:23], v[50:53]", 0)))[0]
    assert too_early(listing(product, ("ds_write_b128 v30, v[12:15]", 0)))[0]
    # twelve states on the way that does not branch, two on the other
    assert [w for _, _, w in too_early(listing(product, ("s_cbranch_vccnz 2", 16), more(7), more(1), ("s_nop 0", 0), reader))[0]] == [2]


def test_no_result_is_read_too_early(tmp_path):
    found = kernels_with("v_mfma", too_early, tmp_path)
    assert set().union(*(met for _, (_, met) in found)) == set(WAITS)
    for part in ("attention_shared_kernel", "attention_prefill", "gemm_q4_staged_kernel", "split_product_kernel", "delta_chunk"):
        assert any(part in name for name, _ in found), part
    assert [(name, bad[0], len(bad)) for name, (bad, _) in found if bad] == []
