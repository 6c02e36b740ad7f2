"""The microscaled rows' kernels keep all they hold in registers and shared memory (see test_kv_registers.py for why)."""

from comp_amd import isa


def kernels():
    return [(n, k) for co in isa.library_code_objects() for n, k in co.kernels.items() if "mx_" in n]


def test_kernels_are_there():
    names = " ".join(n for n, _ in kernels())
    for name in ("mx_quantize_kernel", "mx_lookup_kernel", "mx_pack_kernel", "mx_step_kernel", "mx_stream_kernel", "mx_tile_kernel"):
        assert name in names


def test_no_kernel_uses_scratch_memory():
    bad = [(n, k["vgpr_spill"], k["scratch"]) for n, k in kernels() if k["vgpr_spill"] or k["scratch"]]
    assert not bad, bad

