"""GPU: the decode's scratch needs no initialisation, whatever it held before;
outputs that it cannot write are refused.

The arrival counters in it are told from leftovers by a tag of the launch, so
a process's first launches are tried on scratch full of 64-bit words whose
upper half is a small number, as lengths, page ids and pairs of int32 leave
them.  In a process of its own, so that they are its first launches."""

import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

CODE = """
import torch
from kessie_b200 import ops

def inputs(dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    kv = torch.randn(600, 16, 2, 2, 128, generator=g, device="cuda").to(dtype)
    table = torch.randperm(600, generator=g, device="cuda").int().view(3, 200)
    q = torch.randn(3, 8, 128, generator=g, device="cuda").to(dtype)
    return q, kv[:, :, 0], kv[:, :, 1], table, torch.tensor([3200, 2999, 700], dtype=torch.int32, device="cuda")

LOW = (0, 1, 2, 1000, 1 << 31)
launch = 0
for dtype in (torch.bfloat16, torch.float16, torch.float32):
    args, got = inputs(dtype), []
    for low in LOW:
        launch += 1
        ws = torch.full((4 << 20,), (launch << 32) + low, dtype=torch.int64, device="cuda").view(torch.uint8)
        out = torch.full_like(args[0], 7.0)
        ops.paged_fog_decode(*args, out=out, ws=ws)
        got.append(out)
    launch += 1
    want = ops.paged_fog_decode(*args, ws=torch.zeros(32 << 20, dtype=torch.uint8, device="cuda"))
    for low, x in zip(LOW, got):
        assert torch.equal(x, want), (dtype, low, (x != want).any(-1).sum().item())
assert ops.read_device_status() == 0
print("ok")
"""


def test_decode_on_scratch_full_of_small_numbers():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CODE], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stderr[-2000:]


def test_decode_refuses_outputs_it_would_write_past():
    """The rows are written next to one another: an output with gaps between
    them, of another type or another size is not what the kernel writes."""
    from kessie_b200 import ops
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    kv = torch.randn(4, 16, 2, 2, 128, device="cuda").half()
    table, lens = torch.arange(4, device="cuda").int().view(2, 2), torch.tensor([20, 32], device="cuda").int()
    q = torch.randn(2, 8, 128, device="cuda").half()
    wide = torch.zeros(2, 10, 128, device="cuda", dtype=torch.float16)
    for out in (wide[:, 1:9], torch.zeros(2, 8, 128, device="cuda"), wide[:1, :8], torch.zeros(2, 8, 128).half()):
        with pytest.raises(ValueError, match="out must be"):
            ops.paged_fog_decode(q, kv[:, :, 0], kv[:, :, 1], table, lens, out=out)
    flat = torch.zeros(2, 8 * 128, device="cuda", dtype=torch.float16)
    ops.paged_fog_decode(q, kv[:, :, 0], kv[:, :, 1], table, lens, out=flat)
    assert torch.equal(flat.view(2, 8, 128), ops.paged_fog_decode(q, kv[:, :, 0], kv[:, :, 1], table, lens))
