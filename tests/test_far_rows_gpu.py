"""Cache rows whose byte and element offsets pass 32 bits: what is written and read there is what a
small cache gives."""
import pytest
import torch

from mlc_decode_b200 import MlaPagedDecodeKernel, cache_append, cache_gather

pytestmark = pytest.mark.gpu

KERNELS = {"simt": {"kernel": "simt"}, "pair": {"block_H": 128}, "mma16": {"block_H": 16}, "mma32": {"block_H": 32}}


@pytest.mark.parametrize("kvh", [1, 2])
def test_far_pages(kvh):
    page, per, rows, dt = 64, 8, 500, torch.bfloat16
    pages = 140000 // kvh                       # 2.3 GB of codes, 9.2 GB of 16-bit rows
    g = torch.Generator(device="cuda").manual_seed(kvh)

    def caches(n):
        return (torch.zeros(n, page, kvh, 256, dtype=torch.uint8, device="cuda"),
                torch.zeros(n, page, kvh, 16, dtype=torch.half, device="cuda"),
                torch.zeros(n, page, kvh, 64, dtype=dt, device="cuda"))

    far, near = caches(pages), caches(2 * per)
    last = torch.arange(pages - 1, pages - 1 - 2 * per, -1, device="cuda").int().view(2, per)
    first = torch.arange(2 * per, device="cuda").int().view(2, per)
    r = torch.arange(rows, device="cuda")

    def slots(table):
        return torch.cat([t.long()[r // page] * page + r % page for t in table]).int()

    kv = torch.randn(2 * rows, kvh, 512, generator=g, device="cuda").to(dt)
    kp = torch.randn(2 * rows, kvh, 64, generator=g, device="cuda").to(dt)
    back = []
    for (codes, scales, pe), table in ((far, last), (near, first)):
        cache_append(kv, kp, slots(table), codes, pe, kv_scales=scales)
        got = torch.empty_like(kv), torch.empty_like(kp)
        cache_gather(slots(table), codes, pe, *got, kv_scales=scales)
        back.append(got)
    assert torch.equal(back[0][0], back[1][0]) and torch.equal(back[0][1], kp)
    lens = torch.tensor([rows, rows - 300], dtype=torch.int32, device="cuda")
    for ql in (1, 2):
        lead = (2, 8 * kvh) if ql == 1 else (2, ql, 8 * kvh)
        q = torch.randn(*lead, 512, generator=g, device="cuda").to(dt)
        qp = torch.randn(*lead, 64, generator=g, device="cuda").to(dt)
        for cfg in KERNELS.values():
            k = MlaPagedDecodeKernel(2, 8 * kvh, per * page, cfg=cfg, q_len=ql, kv_heads=kvh)
            outs = []
            for (codes, scales, pe), table in ((far, last), (near, first)):
                outs.append((torch.empty_like(q), torch.empty(lead, device="cuda")))
                k.decode_int4(q, qp, codes, scales, pe, lens, outs[-1][0], outs[-1][1], block_table=table)
            # (pieces that meet in order of arrival may differ in a rounding of the last bit)
            assert ((outs[0][0] - outs[1][0]).abs().float() <= 2.0 ** -8 * outs[1][0].abs().float() + 1e-6).all()
            assert (outs[0][1] - outs[1][1]).abs().max() <= 1e-5 and outs[0][0].abs().max() > 0
    del far
    model = torch.zeros(pages, page, kvh, 512, dtype=dt, device="cuda")
    pe = torch.zeros(pages, page, kvh, 64, dtype=dt, device="cuda")
    cache_append(kv, kp, slots(last), model, pe)
    got = torch.empty_like(kv), torch.empty_like(kp)
    cache_gather(slots(last), model, pe, *got)
    assert torch.equal(got[0], kv) and torch.equal(got[1], kp)
