"""CPU: the wrappers of the paged key / value cache (merv_amd/ops.py) where no GPU is needed to see what they do."""
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_a_torch_without_a_gpu_imports_the_wrappers():
    """They are missed at the call, where the tensors are refused, not at the import."""
    code = """
import torch
for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
from merv_amd import ops
pages, ints = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32)
try:
    ops.paged_decode_attention(torch.zeros(3, 4, 64, dtype=torch.bfloat16), pages, pages, ints, ints[:, 0])
except ValueError as e:
    assert "CUDA" in str(e), e
    print("refused")
"""
    got = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout.strip().endswith("refused"), got.stderr
