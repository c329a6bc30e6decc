"""The torch wrappers' host side, without a GPU."""
import types

from cuda_hgemm_b200 import api


def test_the_stream_is_found_without_torchs_private_call(monkeypatch):
    import torch

    tensor = types.SimpleNamespace(device=torch.device("cuda:3"), get_device=lambda: 3)
    asked = []

    def current_stream(device):
        asked.append(device)
        return types.SimpleNamespace(cuda_stream=77)

    monkeypatch.setattr(torch.cuda, "current_stream", current_stream)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    assert api._stream_of(tensor) == 103 and asked == []
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream")
    assert api._stream_of(tensor) == 77 and asked == [torch.device("cuda:3")]
