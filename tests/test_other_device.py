"""Calls on tensors of another device than the current one: every C entry point a paged step
enqueues through runs with the tensors' device current and on that device's stream.  No GPU:
tensors that say they are on device 1, and recorders in the entry points' places."""
import contextlib
import types

import pytest
import torch

from mlc_decode_b200 import MlaPagedDecodeKernel, Rotary, capi, decode

DEV = torch.device("cuda", 1)


class OnDevice1(torch.Tensor):
    device = property(lambda self: DEV)

    def get_device(self):
        return 1


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnDevice1)


@pytest.fixture
def calls(monkeypatch):
    """[(entry point, device current at the call, stream)]; device 0 is current outside."""
    current, made = [0], []

    @contextlib.contextmanager
    def device(d):
        current.append(torch.device(d).index)
        try:
            yield
        finally:
            current.pop()

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[-1], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 1000 + i, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: types.SimpleNamespace(cuda_stream=1000 + d.index))
    for name in ("extend_block_tables", "extend_block_tables_whole", "cache_append", "cache_gather", "rotary",
                 "decode_ext", "decode_ext_fp8kv", "decode_ext_int4kv"):
        monkeypatch.setattr(capi, name, lambda *a, _n=name: made.append((_n, current[-1], a[-1])))
    return made


@pytest.mark.parametrize("form", ["model", "fp8", "int4"])
def test_step(calls, form):
    b, h, i32 = 2, 16, torch.int32
    dt = torch.bfloat16
    k, rot = MlaPagedDecodeKernel(b, h, 128), Rotary(64)
    ws = _t(1 << 16, dtype=torch.uint8)
    k._ws.update({(1, dt): ws, (1, dt, "int4"): ws,
                  (1, dt, "step"): (_t(b, dtype=i32), _t(b, dtype=i32), _t(b, dtype=i32), _t(b, h, 64))})
    rot._dev[DEV] = _t(32, dtype=torch.float64)
    extra = {"model": {}, "fp8": {"kv_scale": 0.5}, "int4": {"kv_scales": _t(4, 64, 1, 16, dtype=torch.half)}}[form]
    cache = {"model": _t(4, 64, 1, 512), "fp8": _t(4, 64, 1, 512, dtype=torch.uint8),
             "int4": _t(4, 64, 1, 256, dtype=torch.uint8)}[form]
    k.step(_t(b, h, 512), _t(b, h, 64), _t(b, 1, 512), _t(b, 1, 64), cache, _t(4, 64, 1, 64), _t(b, 2, dtype=i32),
           _t(b, dtype=i32), _t(4, dtype=i32), _t(1, dtype=i32), _t(b, h, 512), rotary=rot, **extra)
    last = {"model": "decode_ext", "fp8": "decode_ext_fp8kv", "int4": "decode_ext_int4kv"}[form]
    assert calls == [(n, 1, 1001) for n in ("extend_block_tables_whole", "cache_append", "rotary", last)]
    assert decode.torch._C._cuda_getDevice() == 0
