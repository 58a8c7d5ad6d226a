"""Wait states around inline assembly in the shared-prefix kernels (no GPU): the
rules and the reader of tests/test_asm_waits.py on their listing."""

import subprocess

from gaudirt_amd import build
from tests.test_asm_waits import faults, kernels


def test_waits_around_asm(tmp_path):
    out = tmp_path / "shared_prefix.s"
    subprocess.run([build.HIPCC, *build.COMMON, *build.DEVICE_FLAGS, "--offload-device-only", "-S",
                    str(build.CSRC / "shared_prefix.hip"), "-o", str(out)], check=True, capture_output=True)
    checked, bad = 0, []
    for name, (body, before) in kernels(out.read_text()).items():
        checked += sum(ins.in_asm and ins.vector for ins in body)
        bad += [f"{name}: {fault}" for fault in sorted(set(faults(body, before)))]
    assert checked, "no asm vector instruction found: the listing is not read as it is written"
    assert not bad, f"{len(bad)} faults, the first:\n" + "\n".join(bad[:10])
