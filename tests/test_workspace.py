"""The shim's stream and device handling, without a GPU."""
import importlib.util
from pathlib import Path
from types import SimpleNamespace

import torch

from auto_gpu_kernel_b200 import workspace


def test_calls_without_the_raw_stream_query(monkeypatch):
    """A torch that does not offer the query of the raw handle: both ways to a stream go through torch.cuda."""
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=4711))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    spec = importlib.util.spec_from_file_location("workspace_without_raw_stream", Path(workspace.__file__))
    fresh = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(fresh)
    word = fresh._status[0] = torch.zeros(1, dtype=torch.int32)
    got = []
    assert fresh.call_on(0, lambda *args: got.append(args) or 5, 1, 2) == 5
    assert got == [(1, 2, word.data_ptr(), 4711)]
    assert fresh.stream_handle(torch.device("cuda", 0)) == 4711
