"""The attention cache's binding on the host: which device and stream a call takes,
and what it needs of torch (no GPU needed)."""
import os
import subprocess
import sys
from types import SimpleNamespace

import pytest
import torch


def test_stream_of_another_device_refused(ofb):
    # the call would go to the tensors' device, unordered with the stream that was named
    called = []
    stream = SimpleNamespace(device=torch.device("cuda:1"))
    with pytest.raises(ofb.OfbError) as e:
        ofb._elsewhere(torch.device("cuda:0"), stream, called.append, 1)
    assert e.value.status == ofb.EINVAL and not called


def test_module_loads_where_torch_has_no_cuda():
    # a torch built without CUDA lacks these; what works on the host has to work there
    code = """
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
import conftest
ofb = conftest.load_ofb()
assert ofb.synth_blocks_host(ofb.TYPE_Q4_K, 1, 1, 1).nbytes == 144
z = lambda *s: torch.zeros(*s, dtype=torch.int32)
k = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
cache = ofb.KvCache(k, k.clone(), z(1, 2))
try:
    ofb.attn_decode(cache, k[:1, :, 0], z(1))
except ofb.OfbError as e:
    assert e.status == ofb.EINVAL
else:
    raise AssertionError("host tensors were taken")
print("loaded")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=os.path.dirname(os.path.abspath(__file__)))
    assert r.stdout.strip() == "loaded", r.stderr
