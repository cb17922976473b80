"""A ragged call whose sequences have fewer tiles than the launch has CTA pairs: the pairs
without tiles wait for nothing (no bounded wait runs out, the status word stays zero)."""
import time

import pytest
import torch

from mlc_decode_b200 import MlaPagedDecodeKernel
from oracle import mla_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["bf16", "fp16", "fp8"])
def test_pairs_without_tiles(form):
    b, h, smax, lens = 4, 128, 2000, [1, 0, 130, 64]
    dtype = "fp16" if form == "fp16" else "bf16"
    q, qp, kv, kp = O.make_inputs(b, h, smax, dtype, seed=3)
    kw = {}
    kv_d = kv.cuda()
    if form == "fp8":
        kw["kv_scale"] = 0.02
        kv_d = (kv.float() / 0.02).clamp(-448, 448).to(torch.float8_e4m3fn)
        kv, kv_d = kv_d.float() * 0.02, kv_d.cuda()
    k = MlaPagedDecodeKernel(b, h, smax)
    out, lse = torch.empty_like(q, device="cuda"), torch.empty(b, h, device="cuda")
    args = (q.cuda(), qp.cuda(), kv_d, kp.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), out, lse)
    k(*args, **kw)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    k(*args, **kw)
    torch.cuda.synchronize()
    assert time.perf_counter() - t0 < 1.0      # a wait that runs out takes 2 s
    assert k.device_status(torch.device("cuda"), q.dtype) == 0
    for i, n in enumerate(lens):
        if n:
            ref, ref_lse = O.ref_program_f64(q[i:i + 1], qp[i:i + 1], kv[i:i + 1, :n], kp[i:i + 1, :n])
            assert O.check_parity(out[i:i + 1].float().cpu().numpy(), lse[i:i + 1].cpu().numpy(), ref, ref_lse,
                                  dtype)["ok"], i


def test_block_table_that_covers_less_than_max_seqlen():
    """Without lengths every sequence has the rows its block table covers."""
    b, h, page, per = 2, 128, 64, 3
    q, qp, kv, kp = O.make_inputs(b, h, page * per, "bf16", seed=8)
    table = torch.tensor([[3, 0, 5], [1, 4, 2]], dtype=torch.int32)
    kv_c, kp_c = torch.empty(6, page, 1, 512).bfloat16(), torch.empty(6, page, 1, 64).bfloat16()
    for i in range(b):
        for j in range(per):
            kv_c[table[i, j]], kp_c[table[i, j]] = kv[i, j * page:(j + 1) * page], kp[i, j * page:(j + 1) * page]
    k = MlaPagedDecodeKernel(b, h, 256)
    out, lse = torch.empty_like(q, device="cuda"), torch.empty(b, h, device="cuda")
    k(q.cuda(), qp.cuda(), kv_c.cuda(), kp_c.cuda(), None, out, lse, block_table=table.cuda())
    ref, ref_lse = O.ref_program_f64(q, qp, kv, kp)
    assert O.check_parity(out.float().cpu().numpy(), lse.cpu().numpy(), ref, ref_lse, "bf16")["ok"]
