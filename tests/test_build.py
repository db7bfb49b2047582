"""What the build checks about the kernels that it compiles; no compiler is run here."""
import pytest

from rocm_sgemm_b200 import build

SOURCE = (build.CSRC / "mx4_gemm.cu").read_text()


def log(*kernels):
    """What nvcc -Xptxas -v prints, for (template arguments, registers)."""
    return "".join(f"ptxas info    : Compiling entry function '_ZN12_GLOBAL__N_115mx4_gemm_kernel{args}EEvNS_5GArgsE' for 'sm_100a'\n"
                   f"ptxas info    : Function properties\n    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads\n"
                   f"ptxas info    : Used {n} registers, used 1 barriers, 4112 bytes smem\n" for args, n in kernels)


def test_registers_that_add_up():
    build.check_registers(SOURCE, log(("ILi0ELi64ELi1ELb0", 96), ("ILi1ELi256ELi2ELb1", 168), ("ILi0ELi256ELi2ELb1", 168)))
    build.check_registers("int x;", "")  # a source without such a kernel


def test_registers_that_do_not():
    for bad in (log(("ILi1ELi256ELi2ELb1", 168), ("ILi0ELi256ELi2ELb1", 160)), log(("ILi0ELi64ELi1ELb0", 168)), ""):
        with pytest.raises(RuntimeError, match="168"):
            build.check_registers(SOURCE, bad)
