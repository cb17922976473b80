"""Queries and cache rows that are not finite, or leave fp16's range, in decode over a 4-bit
latent cache: what sees them answers NaN whichever kernel and split the call takes, and
nothing else changes."""
import pytest
import torch

from mlc_decode_b200 import MlaDecodeKernel, MlaPagedDecodeKernel, combine

pytestmark = pytest.mark.gpu

KERNELS = {"simt": {"kernel": "simt"}, "auto": {}, "pair": {"block_H": 128}, "mma16": {"block_H": 16},
           "mma32": {"block_H": 32}}
NAN = float("nan")


def _call(b, ql, h, s, dtype, cfg, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lead = (b, h) if ql == 1 else (b, ql, h)
    q = torch.randn(*lead, 512, generator=g, device="cuda").to(dtype)
    qp = torch.randn(*lead, 64, generator=g, device="cuda").to(dtype)
    codes = torch.randint(0, 256, (b, s, 1, 256), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.05 + 0.3 * torch.rand(b, s, 1, 16, generator=g, device="cuda")).half()
    pe = torch.randn(b, s, 1, 64, generator=g, device="cuda").to(dtype)
    k = MlaPagedDecodeKernel(b, h, s, cfg=cfg, q_len=ql)

    def run(lens=None):
        out, lse = torch.full_like(q, -7.0), torch.full(lead, -7.0, device="cuda")
        k.decode_int4(q, qp, codes, scales, pe, lens, out, lse)
        return out, lse

    return q, qp, codes, scales, pe, run


@pytest.mark.parametrize("kernel", list(KERNELS))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b, h, s", [(1, 16, 60), (1, 16, 300), (2, 16, 9000), (1, 130, 700), (80, 16, 90)])
def test_nan_queries_answer_nan(b, h, s, dtype, kernel):
    """A NaN in a query's latent or rope dims: that row is NaN, its LSE too, whether its
    sequence is whole on one CTA, cut in a few pieces or in many; the other rows are what
    they are without it."""
    q, qp, _, _, _, run = _call(b, 1, h, s, dtype, KERNELS[kernel], seed=s)
    clean, clean_lse = run()
    rows = [(0, 3), (0, h - 1), (b - 1, 7)]
    q[rows[0]][5] = NAN
    qp[rows[1]][63] = NAN
    q[rows[2]][511] = NAN
    out, lse = run()
    hit = torch.zeros(b, h, dtype=torch.bool, device="cuda")
    for r in rows:
        hit[r] = True
    assert out[hit].isnan().all() and lse[hit].isnan().all()
    assert torch.isfinite(out[~hit]).all()
    # (pieces that meet in order of arrival may differ in a rounding of the last bit)
    eps = torch.finfo(dtype).eps
    assert ((out[~hit].float() - clean[~hit].float()).abs() <= eps * clean[~hit].float().abs() + 1e-6).all()
    assert ((lse[~hit] - clean_lse[~hit]).abs() <= 1e-5).all()


@pytest.mark.parametrize("kernel", ["auto", "pair", "mma16", "mma32"])
@pytest.mark.parametrize("s", [60, 9000])
def test_queries_past_fp16_are_not_silent(s, kernel):
    """A bfloat16 query value that fp16 cannot hold: never a finite answer."""
    q, _, _, _, _, run = _call(1, 1, 16, s, torch.bfloat16, KERNELS[kernel], seed=1)
    q[0, 2, 40] = 1e5
    out, lse = run()
    assert not torch.isfinite(out[0, 2]).any() and not torch.isfinite(lse[0, 2])
    assert not (out[0, 2] == 0).any() and torch.isfinite(out[0, 3]).all()


@pytest.mark.parametrize("kernel", list(KERNELS))
def test_nan_queries_beside_sequences_without_rows(kernel):
    """Zeros and -inf remain the answer of a sequence without rows, whatever its query holds."""
    q, _, _, _, _, run = _call(3, 1, 16, 300, torch.bfloat16, KERNELS[kernel], seed=2)
    q[0, 1, 0] = q[1, 1, 0] = NAN
    out, lse = run(torch.tensor([300, 0, 129], dtype=torch.int32, device="cuda"))
    assert out[0, 1].isnan().all() and lse[0, 1].isnan()
    assert (out[1] == 0).all() and torch.isneginf(lse[1]).all()
    assert torch.isfinite(out[2]).all() and torch.isfinite(lse[2]).all()


@pytest.mark.parametrize("b, h, s", [(1, 128, 20000), (8, 128, 1024), (2, 128, 200)])
@pytest.mark.parametrize("kernel", ["auto", "simt"])
def test_nan_queries_of_a_16_bit_cache(b, h, s, kernel):
    g = torch.Generator(device="cuda").manual_seed(3)
    q, qp, kv, kp = (torch.randn(*shape, generator=g, device="cuda").bfloat16()
                     for shape in ((b, h, 512), (b, h, 64), (b, s, 1, 512), (b, s, 1, 64)))
    q[0, 9, 9] = NAN
    out, lse = torch.empty_like(q), torch.empty(b, h, device="cuda")
    MlaDecodeKernel(b, h, 1, s, cfg={"kernel": kernel})(q, qp, kv, kp, out, lse)
    assert out[0, 9].isnan().all() and lse[0, 9].isnan()
    assert torch.isfinite(out[0, 10:]).all() and torch.isfinite(lse[0, 10:]).all()


def test_combine_of_nan_parts():
    """A row whose parts are all NaN is not a row without parts."""
    lse = torch.zeros(3, 1, 4, device="cuda")
    o = torch.ones(3, 1, 4, 512, device="cuda")
    lse[:, 0, 1], o[:, 0, 1] = NAN, NAN
    lse[:, 0, 2], o[:, 0, 2] = -float("inf"), 0.0
    lse[1, 0, 3], o[1, 0, 3] = NAN, NAN
    out, total = torch.empty(1, 4, 512, device="cuda"), torch.empty(1, 4, device="cuda")
    combine(lse, o, out, total)
    assert out[0, 1].isnan().all() and total[0, 1].isnan() and out[0, 3].isnan().all() and total[0, 3].isnan()
    assert (out[0, 2] == 0).all() and torch.isneginf(total[0, 2])
    assert (out[0, 0] - 1).abs().max() < 1e-6 and abs(total[0, 0].item() - 1.0986123) < 1e-6


@pytest.mark.parametrize("kernel", list(KERNELS))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ql, h, s", [(2, 16, 129), (3, 16, 200), (3, 40, 66), (5, 3, 64), (70, 1, 100), (4, 16, 3)])
def test_rows_a_position_does_not_see_may_hold_anything(ql, h, s, dtype, kernel):
    """The rows of a step's later positions: infinite or NaN scales and rope values, and values
    past fp16's range, change nothing for the positions before them, to the bit; the
    tensor-core kernels answer NaN or infinity to those that see them."""
    _, _, codes, scales, pe, run = _call(2, ql, h, s, dtype, KERNELS[kernel], seed=ql + s)
    clean, clean_lse = run()
    for back, scale, rope in ((1, 65504.0, 0.0), (2, NAN, float("inf")), (3, float("inf"), NAN), (4, 9362.0, 0.0)):
        if back >= min(ql, s):
            continue
        keep = scales.clone(), pe.clone(), codes.clone()
        codes[0, s - back] = 0xff                # the largest code everywhere: 7 x the scale
        scales[0, s - back, 0, 3::5] = scale     # (7 x 9362 rounds to infinity, 7 x 9352 does not)
        if rope != 0.0:
            pe[0, s - back, 0, 11] = rope
        out, lse = run()
        blind = ql - back                        # positions [0, blind) do not see the row
        if kernel in ("auto", "pair") and s > 128:   # (pieces met in order of arrival: the last bit)
            eps = torch.finfo(dtype).eps
            assert ((out[0, :blind] - clean[0, :blind]).abs().float() <= eps * clean[0, :blind].abs().float() + 1e-6).all()
        else:
            assert torch.equal(out[0, :blind], clean[0, :blind]) and torch.equal(lse[0, :blind], clean_lse[0, :blind])
        assert torch.isfinite(out[1]).all()
        if kernel != "simt":
            assert not torch.isfinite(out[0, blind:]).all(-1).any()
        scales.copy_(keep[0]), pe.copy_(keep[1]), codes.copy_(keep[2])


@pytest.mark.parametrize("kernel", ["auto", "pair", "mma16", "mma32"])
def test_the_largest_values_fp16_holds_are_values(kernel):
    """Scales above 8188 whose codes keep the values within fp16's range are ordinary values, for
    the last positions' rows too."""
    q, qp, codes, scales, pe, run = _call(1, 3, 16, 80, torch.float16, KERNELS[kernel], seed=9)
    q.zero_()
    codes[0, 70:] = 0xff
    codes[0, 79] = 0x11
    scales[0, 70:, 0, ::4] = 9352.0
    ref, ref_lse = torch.empty_like(q), torch.empty(1, 3, 16, device="cuda")
    MlaPagedDecodeKernel(1, 16, 80, cfg=KERNELS["simt"], q_len=3).decode_int4(q, qp, codes, scales, pe, None, ref, ref_lse)
    out, lse = run()
    assert torch.isfinite(ref).all() and torch.isfinite(out).all()
    # weights and values rounded to fp16 once each, and the result: three times 2^-11 of the largest value
    assert ((out.float() - ref.float()).abs() <= 3 * 2.0 ** -11 * 65504).all()
    assert ((lse - ref_lse).abs() <= 1e-4).all()
