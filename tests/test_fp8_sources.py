"""What the 8-bit product's source has to keep: properties that no run shows when they are lost."""
import re
from pathlib import Path

SOURCE = (Path(__file__).resolve().parent.parent / "cormorant_b200" / "csrc" / "cm_fp8_gemm.cu").read_text()


def test_a_tensor_memory_load_and_its_wait_are_one_statement():
    """The registers of a load are written until its wait: a copy or a spill that the compiler places between two
    statements would read them too early."""
    statements = re.findall(r"asm volatile\((.*?)\);\n", SOURCE, re.S)
    loads = [s for s in statements if "tcgen05.ld." in s]
    assert len(loads) >= 4
    for s in loads:
        assert "tcgen05.wait::ld" in s[s.rindex("tcgen05.ld."):]
    assert SOURCE.count("tcgen05.ld.") == sum(s.count("tcgen05.ld.") for s in loads)
    assert "tmem_ld_wait" not in SOURCE
