"""What shows only in the gfx950 code that hipcc makes of the 4-bit cache's attention (compiled here; no GPU needed): its
kernels keep everything in registers.  A variant of the kernel for heads of 256 that did not, with 160 registers in scratch
memory, once read an illegal address for a reason that was not found."""
import os
import re
import subprocess

import pytest

from flaggems_vllm import _native


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    out = tmp_path_factory.mktemp("asm") / "mxfp4.s"
    flags = [f for f in _native.HIPCC_FLAGS if f not in ("-fPIC", "-shared")]
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *flags, "-S", "--cuda-device-only",
                    f"-I{_native._INCLUDE}", f"-I{_native._CSRC}", os.path.join(_native._CSRC, "mxfp4_attention.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    return open(out).read()


def test_nothing_in_scratch(assembly):
    seen = {"mxfp4_attend_kernel": 0, "mxfp4_attend_wide_kernel": 0, "mxfp4_combine_kernel": 0}
    for m in re.finditer(r"\.name:\s+\S*?\d(mxfp4_\w+?_kernel)I\S*\n(.*?)\.wavefront_size", assembly, re.S):
        number = {k: int(re.search(rf"\.{k}:\s+(\d+)", m.group(2)).group(1))
                  for k in ("private_segment_fixed_size", "vgpr_spill_count", "vgpr_count")}
        assert number["private_segment_fixed_size"] == 0 and number["vgpr_spill_count"] == 0, (m.group(0)[:200], number)
        assert number["vgpr_count"] <= 256
        seen[m.group(1)] += 1
    # head sizes and types; 128-row tiles up to 128; joining for each kind of tile, by rows or by cuts
    assert seen == {"mxfp4_attend_kernel": 6, "mxfp4_attend_wide_kernel": 4, "mxfp4_combine_kernel": 20}
    assert "scratch_load" not in assembly and "scratch_store" not in assembly


def test_no_packed_float_arithmetic(assembly):
    assert not re.search(r"v_pk_(add|mul|fma)_f32", assembly)
