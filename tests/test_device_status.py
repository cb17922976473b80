"""Which workspace a status is read from, without a GPU: "cuda" is the current device."""
import pytest
import torch

from mlc_decode_b200 import MlaDecodeKernel, MlaPagedDecodeKernel


@pytest.mark.parametrize("kind", ["plain", "paged", "int4"])
def test_a_device_without_an_index_is_the_current_one(monkeypatch, kind):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 2)
    k = MlaDecodeKernel(1, 16, 1, 64) if kind == "plain" else MlaPagedDecodeKernel(1, 16, 64)
    ws = torch.zeros(64, dtype=torch.uint8)
    dt = torch.bfloat16
    k._ws[(2, dt, "int4") if kind == "int4" else (2, dt)] = ws
    for device in ("cuda", torch.device("cuda"), "cuda:2", torch.device("cuda", 2)):
        ws.zero_()
        assert k.device_status(device, dt) == 0
        ws[0] = 5
        assert k.device_status(device, dt) == 5 and k.device_status("cuda:1", dt) == 0
        if kind != "int4":
            ws[8] = 7
            assert k.clock_probe(device, dt) == (7, 0, 0)
