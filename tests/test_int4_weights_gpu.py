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


@pytest.mark.parametrize("kernel", ["mma16", "mma32"])
@pytest.mark.parametrize("b, h, s", [(8, 96, 500), (16, 64, 1000), (4, 16, 300)])
def test_fp16_results_are_near_their_own_rounding(b, h, s, kernel):
    """fp16 results of the warp-level kernel: the weights are taken in two parts, so what is left
    beside the result's own rounding is the values', (n - 8) s to fp16.  Each value's relative error
    has at most the result's spread (some products are exact), and results are sums of values with
    independent errors: at most sqrt(2) times the result's rounding in the root mean square, and 3 %
    for the sample (weights in one part: 1.46 to 1.52)."""
    g = torch.Generator(device="cuda").manual_seed(b * h)
    dt = torch.float16
    x = torch.randn(b, s, 16, 32, generator=g, device="cuda")
    scales = (x.abs().amax(-1) / 7).half()
    n = (x / scales.float().unsqueeze(-1)).round().clamp(-8, 7)
    nib = [0, 2, 4, 6, 1, 3, 5, 7]
    c = (n + 8).to(torch.uint8).view(b, s, 64, 8)[..., nib].view(b, s, 64, 4, 2)
    codes = (c[..., 0] | (c[..., 1] << 4)).reshape(b, s, 1, 256).contiguous()
    rows = (n.double() * scales.double().unsqueeze(-1)).view(b, s, 512)
    q, qp = torch.randn(b, h, 512, generator=g, device="cuda").to(dt), torch.randn(b, h, 64, generator=g, device="cuda").to(dt)
    pe = torch.randn(b, s, 1, 64, generator=g, device="cuda").to(dt)
    scores = (q.double() @ rows.transpose(1, 2) + qp.double() @ pe[:, :, 0].double().transpose(1, 2)) * SCALE
    ref = torch.softmax(scores, -1) @ rows
    out = torch.empty_like(q)
    MlaPagedDecodeKernel(b, h, s, cfg=KERNELS[kernel]).decode_int4(q, qp, codes, scales.view(b, s, 1, 16), pe, None, out)
    own = (ref.half().double() - ref).norm()
    assert (out.double() - ref).norm() <= 1.03 * math.sqrt(2) * own, ((out.double() - ref).norm() / own).item()
