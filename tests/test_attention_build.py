"""The attention kernels' registers (device passes of hipcc, no GPU): two waves a SIMD, 256 vector
registers a lane each, and nothing in scratch memory, whose loads would wait behind the tiles in
flight."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "lightdelta_amd" / "csrc"
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

pytestmark = pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not available")


@pytest.mark.parametrize("source,count", [("attention_decode", 5), ("attention_prefill", 4)])
def test_attention_keeps_its_registers(tmp_path, source, count):
    from lightdelta_amd.build import EXTRA_FLAGS, HIPCC_FLAGS

    listing = tmp_path / f"{source}.s"
    subprocess.run([HIPCC, *HIPCC_FLAGS, *EXTRA_FLAGS.get(f"{source}.hip", []), "--cuda-device-only",
                    "-S", "-o", str(listing), str(CSRC / f"{source}.hip")], check=True,
                   capture_output=True, timeout=300)
    kernels = re.findall(r"\.name: +(\S*attention_\w+_kernel\S*)\n +\.private_segment_fixed_size: +(\d+)"
                         r"\n(?:.*\n)*? +\.vgpr_count: +(\d+)\n +\.vgpr_spill_count: +(\d+)",
                         listing.read_text())
    assert len(kernels) == count
    for name, scratch, registers, spilled in kernels:
        assert int(scratch) == 0 and int(registers) <= 256 and int(spilled) == 0, name
