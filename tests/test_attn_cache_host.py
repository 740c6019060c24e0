"""The attention cache's binding on the host: which device and stream a call takes,
and what it needs of torch (no GPU needed)."""
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
