"""The package imports where torch has no GPU functions at all; only a call on a GPU needs them."""

import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_import():
    code = ("import torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, name)\n"
            "import apexw_amd\n"
            "try:\n"
            "    apexw_amd.layer_norm_forward(torch.randn(2, 8))\n"
            "except ValueError as e:\n"
            "    assert 'GPU' in str(e)\n"
            "else:\n"
            "    raise SystemExit('not refused')\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
