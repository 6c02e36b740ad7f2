"""The key/value cache's kernels keep all they hold in registers and shared memory.

Register spills are not only slow here: hipcc has put the store of one into the block that ends a divergent region, before
the execution mask is restored there, so that only some lanes stored what all lanes loaded again later, and kernels went on
with wild addresses.  Code without spills and without indexed private arrays has no such stores."""

from comp_amd import isa


def kernels():
    return [(n, k) for co in isa.library_code_objects() for n, k in co.kernels.items() if "kv_" in n]


def test_kernels_are_there():
    names = " ".join(n for n, _ in kernels())
    for name in ("kv_write_kernel", "kv_read_kernel", "kv_attend_few_kernel", "kv_attend_many_kernel", "kv_attend_join_kernel"):
        assert name in names
    assert len(kernels()) >= 200


def test_no_kernel_uses_scratch_memory():
    """(SGPRs spilled to lanes of a VGPR are whole whatever the mask: v_writelane and v_readlane do not look at it.)"""
    bad = [(n, k["vgpr_spill"], k["scratch"]) for n, k in kernels() if k["vgpr_spill"] or k["scratch"]]
    assert not bad, bad


def before_restore(instructions, kept):
    """The instructions of `kept` that run before an s_or_b64 exec, exec, ... of their own block."""
    leaders = {t for _, _, _, t in instructions if t is not None}
    found = []
    for i, (addr, name, ops, _) in enumerate(instructions):
        if name not in kept:
            continue
        for a, n, o, t in instructions[i + 1 :]:
            if a in leaders or t is not None or n.endswith("saveexec_b64"):
                break
            if n == "s_or_b64" and o.startswith("exec, exec"):
                found.append((hex(addr), name, ops))
                break
    return found


def test_before_restore_reads_blocks():
    code = [(0, "s_and_saveexec_b64", "s[0:1], vcc", None), (4, "s_cbranch_execz", "2", 16), (8, "v_mov_b32_e32", "v1, 0", None),
            (12, "v_accvgpr_write_b32", "a1, v1", None), (16, "v_accvgpr_write_b32", "a0, v2", None),
            (20, "s_or_b64", "exec, exec, s[0:1]", None), (24, "v_accvgpr_write_b32", "a2, v2", None),
            (28, "s_and_saveexec_b64", "s[0:1], vcc", None), (32, "s_or_b64", "exec, exec, s[0:1]", None)]  # fmt: skip
    assert before_restore(code, {"v_accvgpr_write_b32"}) == [("0x10", "v_accvgpr_write_b32", "a0, v2")]


def test_values_held_in_accumulation_registers_are_whole():
    """Where a kernel parks values in AGPRs, no such write comes before its block restores the execution mask."""
    for co in isa.library_code_objects():
        for name, k in co.kernels.items():
            if "kv_" in name and k["agpr"]:
                found = before_restore(co.disassemble(k["symbol"]), {"v_accvgpr_write_b32"})
                assert not found, (name, found)
