"""CPU: the wrappers of the paged key / value cache (merv_amd/ops.py) where no GPU is needed to see what they do."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as fwd

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


def test_gradients_and_tangents_are_refused():
    """Of rows and of the rotary tables (through the checks themselves: on the CPU a call ends at its pages)."""
    from merv_amd import ops
    x = torch.ones(3, 2, 64, dtype=torch.bfloat16)
    c = torch.ones(8, 64, dtype=torch.bfloat16)
    wants, c_wants = x.clone().requires_grad_(), c.clone().requires_grad_()
    rows = lambda t: ops._paged_rows("call", "k", t, (3, 2, 64), -1)  # noqa: E731
    assert rows(x) == (x.data_ptr(), 128, 64)
    assert ops._paged_tables("call", c, c, 64, -1) == (c.data_ptr(), c.data_ptr(), 8, 64)
    for bad in (lambda: rows(wants), lambda: ops._paged_tables("call", c_wants, c, 64, -1), lambda: ops._paged_tables("call", c, c_wants, 64, -1)):
        with pytest.raises(ValueError, match="requires a gradient"):
            bad()
        with torch.no_grad():
            bad()
    with fwd.dual_level():
        rows(x)
        ops._paged_tables("call", c, c, 64, -1)
        dual, c_dual = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(c, torch.ones_like(c))
        for bad in (lambda: rows(dual), lambda: ops._paged_tables("call", c_dual, c, 64, -1), lambda: ops._paged_tables("call", c, c_dual, 64, -1)):
            with pytest.raises(ValueError, match="tangent"):
                bad()


def test_outputs_that_are_other_operands_are_refused():
    """A workgroup would write over rows that another one still reads (C entries, host checks alone)."""
    from merv_amd import _lib
    from test_paged_cpu import _cache
    lib, c = _lib.load(), _cache()

    def write(**kw):
        a = dict(k=1 << 20, ks=128, kh=64, v=2 << 20, vs=128, vh=64, q=3 << 20, qs=128, qh=64, cos=64, sin=64, rl=10, rs=64, qo=4 << 20, qos=128, qoh=64, ko=5 << 20, kos=128,
                 koh=64, off=64, start=64, T=5, H=2, st=0)
        a.update(kw)
        return lib.merv_paged_cache_write(c, *a.values())

    for kw in (dict(qo=1 << 20), dict(qo=2 << 20), dict(qo=5 << 20), dict(ko=2 << 20), dict(ko=3 << 20), dict(ko=1 << 20, kos=256), dict(qo=3 << 20, qoh=128),
               dict(v=1 << 20, ko=1 << 20)):
        with pytest.raises(ValueError, match="must not share memory"):
            _lib.check(write(**kw), "write")
    with pytest.raises(ValueError, match="must not share memory"):
        _lib.check(lib.merv_paged_cache_read(c, 64, 128, 64, 64, 128, 64, 64, 0, 3, 0), "read")
    with pytest.raises(ValueError, match="must not share memory"):
        _lib.check(lib.merv_paged_decode_attention(c, 64, 256, 64, 64, 512, 64, 0, 64, 4, 0, 1.0, 4096, 1 << 30, 0), "attention")
