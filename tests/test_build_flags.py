"""What larder_amd.build hands the compiler."""
import re

from larder_amd import build


def test_every_matrix_core_source_keeps_its_sums_in_arch_vgprs():
    """Whatever multiplies on the matrix cores, itself or by a header's function, is compiled with them in arch VGPRs."""
    headers = {h.name: "mfma" in h.read_text() for h in build.SRC.glob("*.h")}
    with_cores = set()
    for src in build.sources():
        text = src.read_text()
        if "mfma" in text and ("__builtin_amdgcn_mfma" in text or any(headers[h] for h in re.findall(r'#include "(\w+\.h)"', text))):
            with_cores.add(src.name)
    assert {"chunk.hip", "prompt.hip", "attend.hip", "grouped.hip"} <= with_cores
    for name in with_cores:
        assert "-amdgpu-mfma-vgpr-form" in build.FILE_FLAGS.get(name, ()), name
