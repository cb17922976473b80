"""A request's new rows in a step: all of them or none, and then every position of the step
sees its own row and those before it, whatever the cache's form and KV heads."""
import numpy as np
import pytest
import torch

from mlc_decode_b200 import MlaPagedDecodeKernel, cache_gather, extend_block_tables
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

SCALE = 576 ** -0.5


def _i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device="cuda")


@pytest.mark.parametrize("q_len", [1, 2, 3, 70])
@pytest.mark.parametrize("b", [1, 5, 130, 3000])
@pytest.mark.parametrize("num_free", [0, 1, 40, 100000])
def test_whole_rows(b, q_len, num_free):
    if b * q_len > 20000:
        b = 200
    rng = np.random.default_rng(q_len + b)
    max_pages, page = 7, 64
    lens = rng.integers(-2, 7 * 64 + 3, b).tolist()
    new = rng.integers(-1, q_len + 3, b).tolist()
    num_pages = b * max_pages + num_free
    ids = rng.permutation(num_pages)
    table, free = ids[:b * max_pages].reshape(b, max_pages), ids[b * max_pages:]
    n = b * q_len
    for free_pos in (0, 3):
        ref = P.extend_tables(table.tolist(), lens, new, free.tolist(), free_pos, page, num_pages, n, q_len, whole=True)
        t, fp, sl = _i32(table), _i32([free_pos]), _i32(lens)
        slots, pos = (torch.full((n,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
        cu = torch.full((b + 1,), -7, dtype=torch.int32, device="cuda")
        extend_block_tables(t, sl, _i32(new), _i32(free), fp, sl, fp, slots, pos, page_size=page, num_pages=num_pages,
                            cu_new=cu, q_len=q_len, whole=True)
        got = (t.cpu().tolist(), sl.cpu().tolist(), int(fp), slots.cpu().tolist(), pos.cpu().tolist(), cu.cpu().tolist())
        for name, g, r in zip(("table", "lens", "free_pos", "slots", "positions", "cu"), got, ref):
            assert g == r, name


def test_whole_needs_q_len():
    i = _i32([0, 0])
    with pytest.raises(Exception, match="q_len"):
        extend_block_tables(i.view(2, 1), i, i, i, i[:1], i, i[:1], i, i, page_size=64, num_pages=4, whole=True)


@pytest.mark.parametrize("form", ["model", "fp8", "int4"])
@pytest.mark.parametrize("h, kvh", [(16, 1), (128, 1), (8, 2)])
def test_step_places_all_rows_or_none(form, h, kvh):
    """Request 0 has 62 rows on its only page and finds the free list empty, request 1's table
    row ends after one more row, request 2 has its page: 0 and 1 are left as they are, cache
    included, and all of 2's positions see their own rows."""
    dt, b, ql, page, per, num = torch.bfloat16, 3, 3, 64, 2, 6
    g = torch.Generator(device="cuda").manual_seed(h + kvh)

    def rn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dt)

    lead = (num, page, kvh)
    if form == "int4":
        cache = torch.randint(0, 256, (*lead, 256), generator=g, dtype=torch.uint8, device="cuda")
        extra = {"kv_scales": (0.1 + 0.3 * torch.rand(*lead, 16, generator=g, device="cuda")).half()}
    elif form == "fp8":
        cache, extra = (rn(*lead, 512) * 64).to(torch.float8_e4m3fn), {"kv_scale": 1 / 64}
    else:
        cache, extra = rn(*lead, 512), {}
    pe = rn(*lead, 64)
    table = _i32([[4, -1], [1, 3], [0, -1]])
    lens, free_pos = _i32([62, 127, 50]), _i32([0])
    q, qp, kv, kp = rn(b, ql, h, 512), rn(b, ql, h, 64), rn(b, ql, kvh, 512), rn(b, ql, kvh, 64)
    out, lse = torch.empty_like(q), torch.empty(b, ql, h, device="cuda")
    before = [t.clone().view(torch.uint8) for t in (cache, pe)]
    k = MlaPagedDecodeKernel(b, h, per * page, q_len=ql, kv_heads=kvh)
    k.step(q, qp, kv, kp, cache, pe, table, lens, _i32([]), free_pos, out, lse, **extra)
    assert lens.tolist() == [62, 127, 53] and free_pos.item() == 0
    assert table.tolist() == [[4, -1], [1, 3], [0, -1]]
    for t, old in zip((cache, pe), before):
        same = (t.view(torch.uint8) == old).view(num, page, -1).all(-1)
        assert (~same).nonzero().tolist() == [[0, 50], [0, 51], [0, 52]]
    rows = torch.arange(53, dtype=torch.int32, device="cuda")
    v, kpe = torch.empty(53, kvh, 512, dtype=dt, device="cuda"), torch.empty(53, kvh, 64, dtype=dt, device="cuda")
    cache_gather(rows, cache, pe, v, kpe, **extra)
    assert torch.equal(kpe[50:], kp[2])
    v, kpe = v.double().cpu().numpy(), kpe.double().cpu().numpy()
    if form == "int4":
        code = P.unpack_int4(cache[0, :53].cpu().numpy())
        v = P.dequantise_int4(code, extra["kv_scales"][0, :53].cpu().numpy())
    gr = h // kvh
    for t in range(ql):
        m = 51 + t
        for j in range(kvh):
            hs = slice(j * gr, (j + 1) * gr)
            qq, qqp = (x[2, t, hs].double().cpu().numpy() for x in (q, qp))
            ref, ref_lse, spread, ds = P.decode(qq, qqp, v[:m, j], kpe[:m, j], SCALE)
            assert (np.abs(out[2, t, hs].double().cpu().numpy() - ref) <= spread + 2.0 ** -8 * np.abs(ref) + 1e-6).all()
            assert (np.abs(lse[2, t, hs].double().cpu().numpy() - ref_lse) <= ds[:, 0] + 1e-4).all()
