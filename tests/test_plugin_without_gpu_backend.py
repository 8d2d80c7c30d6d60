"""The plugin's registration under a torch that was built without a GPU backend, which has no raw-stream lookup."""
import os
import subprocess
import sys

from exl3rocm import _lib

CODE = """
import torch
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    del torch._C._cuda_getCurrentRawStream
from exl3rocm import plugin
plugin.register()
print([hasattr(torch.ops.exl3rocm, n) for n in ("linear", "batch_plan", "rope_kv_write", "paged_attention")])
"""


def test_register():
    package = os.path.dirname(os.path.dirname(os.path.abspath(_lib.__file__)))
    r = subprocess.run([sys.executable, "-c", CODE], capture_output=True, text=True, timeout=300, env={**os.environ, "PYTHONPATH": package})
    assert r.returncode == 0 and r.stdout.strip() == "[True, True, True, True]", r.stderr[-500:]
