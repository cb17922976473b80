"""Small softmax weights in decode over a 4-bit latent cache: many rows far below one that
dominates."""
import math

import pytest
import torch

from mlc_decode_b200 import MlaPagedDecodeKernel

pytestmark = pytest.mark.gpu

KERNELS = {"pair": {"block_H": 128}, "mma16": {"block_H": 16}, "mma32": {"block_H": 32}}
SCALE = 576 ** -0.5


@pytest.mark.parametrize("kernel", list(KERNELS))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("e", [14.3, 20.6, 24.6, 25.1, 27.0])
def test_many_small_weights_beside_a_dominant_one(e, dtype, kernel):
    """Row 0 has value 0 and the largest score, the s - 1 others value 1 and weights 2^-e beside
    it: the output is the others' share.  A stored weight is a half of 2^7 x its value, so below
    2^-21 it is off by at most half a step of 2^-24 / 2^7, 2^-32, and by 2^-11 of itself above."""
    s, h = 20000, 16
    codes = torch.full((1, s, 1, 256), 0x99, dtype=torch.uint8, device="cuda")
    codes[0, 0] = 0x88
    scales = torch.ones(1, s, 1, 16, dtype=torch.half, device="cuda")
    pe = torch.zeros(1, s, 1, 64, dtype=dtype, device="cuda")
    pe[0, 0, 0, :2] = torch.tensor([1.0, 2.0 ** -7], dtype=dtype)
    q, qp = torch.zeros(1, h, 512, dtype=dtype, device="cuda"), torch.zeros(1, h, 64, dtype=dtype, device="cuda")
    want = e * math.log(2) / SCALE
    qp[0, :, 0] = want
    qp[0, :, 1] = (want - qp[0, 0, 0].item()) * 2 ** 7      # (what the type leaves of it)
    score = SCALE * (qp[0, 0, 0].double() + qp[0, 0, 1].double() * 2 ** -7).item()
    w = math.exp(-score)
    ref, ref_lse = (s - 1) * w / (1 + (s - 1) * w), score + math.log1p((s - 1) * w)
    out, lse = torch.empty_like(q), torch.empty(1, h, device="cuda")
    k = MlaPagedDecodeKernel(1, h, s, cfg={**KERNELS[kernel], "num_split": 1})    # one running maximum
    k.decode_int4(q, qp, codes, scales, pe, None, out, lse)
    # float32 roundings, 2^-24 of the value each: the sum l of about 1 takes up to s / 64 tiles one
    # after another and 64 weights within each, (20000 / 64 + 64) x 2^-24 = 2.2e-5 of it; the score
    # of up to 19 takes eight (its two products, the scale's and ln 2's factors, the sums)
    sums, scores = (s / 64 + 64) * 2.0 ** -24, 8 * 2.0 ** -24 * (1 + ref_lse)
    # the weights' rounding, the result's, and these
    tol = (s - 1) * max(2.0 ** -32, w * 2.0 ** -11) + (torch.finfo(dtype).eps / 2 + sums + scores) * ref
    assert (out.double() - ref).abs().max().item() <= tol, (out[0, 0, 0].item(), ref)
    assert (lse.double() - ref_lse).abs().max().item() <= sums + scores
