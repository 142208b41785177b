"""The package loads on a torch without GPU bindings: its loader, layouts and build need none, and its calls say that their tensors
are on no GPU."""
from __future__ import annotations

import os
import subprocess
import sys

CHILD = r"""
import sys
sys.path.insert(0, sys.argv[1])
import torch
gone = [n for n in dir(torch._C) if n.startswith("_cuda")]
assert gone
for n in gone:
    delattr(torch._C, n)
import mi355moe
from mi355moe import build, dispatch, ffn, layer, loader, norm, ops
assert ops.ids_dtype_code(torch.int64) == mi355moe._lib.I64 and build.SOURCES and loader and layer
x = torch.zeros(2, 8).half()
for f in (lambda: dispatch.sort_tokens(torch.zeros(2, 2, dtype=torch.int32), 4), lambda: ffn.linear(x, x), lambda: ffn.gated(x, torch.zeros(16, 8).half()),
          lambda: norm.rms(x, x[0])):
    try:
        f()
    except ValueError as e:
        assert "GPU" in str(e), e
    else:
        raise AssertionError("no refusal")
print("loaded")
"""


def test_without_gpu_bindings():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "glm-5.3-flash-dgx-spark-vllm-optimization_amd")
    r = subprocess.run([sys.executable, "-c", CHILD, pkg], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "loaded", r.stderr[-2000:]
