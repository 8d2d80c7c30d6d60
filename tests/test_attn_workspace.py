"""CPU test: the attention kernels do not compile where their workspace is too small for the counters and parts that they index."""
import os
import shutil
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
@pytest.mark.parametrize("source", ["exl3_attn8.hip", "exl3_attn8_prefill.hip"])
def test_half_the_counters_are_refused(tmp_path, source):
    """The 8-bit cache's kernels count in both halves: a tile's parts in the first, a group's in the second."""
    shutil.copytree(os.path.join(REPO, "include"), tmp_path / "include")
    shutil.copytree(os.path.join(REPO, "qwen38-27b-exl3-rdna4_amd", "csrc"), tmp_path / "package" / "csrc")
    header = tmp_path / "include" / "exl3_mi355x.h"

    def errors(nbytes):
        text = header.read_text()
        now = next(line for line in text.splitlines() if line.startswith("#define EXL3_ATTN_COUNTER_BYTES "))
        header.write_text(text.replace(now, f"#define EXL3_ATTN_COUNTER_BYTES {nbytes}"))
        r = subprocess.run([HIPCC, "--offload-arch=gfx950", "--cuda-device-only", "-std=c++17", "-fsyntax-only", str(tmp_path / "package" / "csrc" / source)],
                           capture_output=True, text=True)
        assert r.returncode == 0 or "error: static assertion failed" in r.stderr, r.stderr[-2000:]
        return r.returncode != 0

    assert not errors(4096) and errors(2048)
