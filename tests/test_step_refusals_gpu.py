"""A refused step changes nothing: not the tables, the lengths or the free list, not the cache, and
not a graph that was being captured."""
import pytest
import torch

from mlc_decode_b200 import MlaPagedDecodeKernel, Rotary

pytestmark = pytest.mark.gpu


def _args(b, h, form):
    dt = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(5)

    def rn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dt)

    a = dict(q=rn(b, h, 512), q_pe=rn(b, h, 64), kv=rn(b, 1, 512), k_pe=rn(b, 1, 64),
             k_pe_cache=torch.zeros(4, 64, 1, 64, dtype=dt, device="cuda"),
             block_table=torch.full((b, 2), -1, dtype=torch.int32, device="cuda"),
             cache_seqlens=torch.zeros(b, dtype=torch.int32, device="cuda"),
             free_pages=torch.arange(4, dtype=torch.int32, device="cuda"),
             free_pos=torch.zeros(1, dtype=torch.int32, device="cuda"), out=torch.empty(b, h, 512, dtype=dt, device="cuda"))
    if form == "int4":
        a["kv_cache"] = torch.zeros(4, 64, 1, 256, dtype=torch.uint8, device="cuda")
        a["kv_scales"] = torch.zeros(4, 64, 1, 16, dtype=torch.half, device="cuda")
    elif form == "fp8":
        a["kv_cache"], a["kv_scale"] = torch.zeros(4, 64, 1, 512, device="cuda").to(torch.float8_e4m3fn), 1 / 32
    else:
        a["kv_cache"] = torch.zeros(4, 64, 1, 512, dtype=dt, device="cuda")
    return a


@pytest.mark.parametrize("scale", [1e39, 1e-50, float("nan"), -1.0])
def test_scales_outside_float32(scale):
    a = _args(2, 16, "fp8")
    with pytest.raises(ValueError, match="kv_scale"):
        MlaPagedDecodeKernel(2, 16, 128).step(**{**a, "kv_scale": scale})
    assert a["cache_seqlens"].tolist() == [0, 0] and a["free_pos"].item() == 0 and (a["block_table"] == -1).all()


@pytest.mark.parametrize("form", ["model", "fp8", "int4"])
def test_a_rotary_first_met_in_a_capture(form):
    a = _args(2, 16, form)
    k = MlaPagedDecodeKernel(2, 16, 128)
    known = Rotary(64)
    k.step(**a, rotary=known)                     # everything but the new rotary is in place
    assert a["cache_seqlens"].tolist() == [1, 1]
    held = a["free_pos"].item()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before the capture"):
            k.step(**a, rotary=Rotary(64, base=500.0))
        a["out"].zero_()                          # (a graph of its own, without the step)
    graph.replay()
    torch.cuda.synchronize()
    assert a["cache_seqlens"].tolist() == [1, 1] and a["free_pos"].item() == held
    other = Rotary(64, base=500.0)
    other.turns(torch.device("cuda", torch.cuda.current_device()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k.step(**a, rotary=other)
    graph.replay()
    torch.cuda.synchronize()
    assert a["cache_seqlens"].tolist() == [2, 2] and torch.isfinite(a["out"]).all()
