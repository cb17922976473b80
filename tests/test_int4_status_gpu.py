"""The status word of a 4-bit decode's workspace: zero after every call that was not cut short,
whichever kernel ran and however many splits it took."""
import pytest
import torch

from mlc_decode_b200 import MlaPagedDecodeKernel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cfg", [{"kernel": "simt"}, {"kernel": "simt", "num_split": 1}, {"kernel": "simt", "num_split": 7},
                                 {}, {"block_H": 16}, {"block_H": 32}, {"block_H": 128}], ids=str)
@pytest.mark.parametrize("s", [40, 3000])
def test_status_word_stays_zero(s, cfg):
    g = torch.Generator(device="cuda").manual_seed(s)
    b, h, dt = 2, 16, torch.bfloat16
    q, qp = torch.randn(b, h, 512, generator=g, device="cuda").to(dt), torch.randn(b, h, 64, generator=g, device="cuda").to(dt)
    codes = torch.randint(0, 256, (b, s, 1, 256), generator=g, dtype=torch.uint8, device="cuda")
    scales, pe = torch.ones(b, s, 1, 16, device="cuda").half(), torch.randn(b, s, 1, 64, generator=g, device="cuda").to(dt)
    k = MlaPagedDecodeKernel(b, h, s, cfg=cfg)
    out = torch.empty_like(q)
    for _ in range(3):
        k.decode_int4(q, qp, codes, scales, pe, None, out)
        assert k.device_status(q.device, dt) == 0
