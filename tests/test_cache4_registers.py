"""What the compiler makes of the attention that decoding calls most (csrc/cache4_attend_impl.h): with prefixes or without, the kernel of few rows is another one, and without them it
has no registers in memory."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-kmeans_amd", "csrc")


@pytest.mark.parametrize("groups", [2, 4])
def test_plain_decoding_keeps_its_registers(tmp_path, groups):
    with open(os.path.join(CSRC, "Makefile")) as f:
        text = f.read().replace("\\\n", " ")
    setting = lambda name: re.search(r"^%s\s*\??=(.*)$" % name, text, re.M).group(1).strip()  # noqa: E731
    flags = setting("HIPFLAGS").replace("$(ARCH)", "gfx950").split()
    hipcc = os.environ.get("HIPCC") or setting("HIPCC")
    out = str(tmp_path / "attend.s")
    subprocess.run([hipcc, *flags, "--cuda-device-only", "-S", "-DKMX_J=%d" % groups, "cache4_attend_inst.hip", "-o", out], cwd=CSRC, check=True, capture_output=True, timeout=600)
    with open(out) as f:
        kernels = {m.group(1): m.group(0) for m in re.finditer(r"^    \.name:\s+(\S+)(?:\n    .*)+", f.read(), re.M)}
    plain = [body for name, body in kernels.items() if "attend4_kernelILi%dELb0E" % groups in name]
    assert len(plain) == 1 and any("attend4_kernelILi%dELb1E" % groups in name for name in kernels), list(kernels)
    for what in ("private_segment_fixed_size", "sgpr_spill_count", "vgpr_spill_count"):
        assert re.search(r"\.%s:\s+(\d+)" % what, plain[0]).group(1) == "0", what
