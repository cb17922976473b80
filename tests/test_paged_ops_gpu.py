"""GPU tests of block tables, rotary positions and cache rows against the 64-bit oracle."""
import numpy as np
import pytest
import torch

from mlc_decode_b200 import Rotary, cache_append, cache_gather, extend_block_tables
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

TDT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device="cuda")


# ---------------------------------------------------------------- tables
def _run_tables(lens, new, page, max_pages, num_free, num_tokens, q_len=0, free_pos=0, in_place=False, skew=0, seed=0):
    rng = np.random.default_rng(seed)
    b = len(lens)
    num_pages = b * max_pages + num_free
    ids = rng.permutation(num_pages)
    table, free = ids[:b * max_pages].reshape(b, max_pages), ids[b * max_pages:]
    ref = P.extend_tables(table.tolist(), lens, new, free.tolist(), free_pos, page, num_pages, num_tokens, q_len)
    t, fp = _i32(table), _i32([free_pos])
    sl, nl = _i32(lens), _i32(new)
    out_sl = sl if in_place else torch.full((b,), -7, dtype=torch.int32, device="cuda")
    out_fp = fp if in_place else torch.full((1,), -7, dtype=torch.int32, device="cuda")
    slots, pos = (torch.full((num_tokens + skew,), -7, dtype=torch.int32, device="cuda")[skew:] for _ in range(2))
    cu = torch.full((b + 1,), -7, dtype=torch.int32, device="cuda")
    extend_block_tables(t, sl, nl, _i32(free), fp, out_sl, out_fp, slots, pos, page_size=page, num_pages=num_pages,
                        cu_new=cu, q_len=q_len)
    got = (t.cpu().tolist(), out_sl.cpu().tolist(), int(out_fp), slots.cpu().tolist(), pos.cpu().tolist(),
           cu.cpu().tolist())
    for name, g, r in zip(("table", "lens", "free_pos", "slots", "positions", "cu"), got, ref):
        assert g == r, name


@pytest.mark.parametrize("b", [1, 2, 3, 64, 257, 2048, 2049])
@pytest.mark.parametrize("page, tokens_per", [(64, 1), (192, 40), (64, 300)])
def test_tables(b, page, tokens_per):
    if b > 300 and tokens_per > 1:
        tokens_per = 5
    rng = np.random.default_rng(b * 1000 + page)
    max_pages = 7
    lens = rng.integers(0, 5 * page, b).tolist()
    new = rng.integers(0, tokens_per + 1, b).tolist()
    total = sum(new)
    _run_tables(lens, new, page, max_pages, 6 * b, total + 9, seed=b)
    _run_tables(lens, new, page, max_pages, 6 * b, max(total - 3, 0), in_place=True, free_pos=2, seed=b)


@pytest.mark.parametrize("big", [False, True])
def test_tables_where_room_ends(big):
    """Free list or table row full, lengths outside the row, negative counts, page borders."""
    pad = 9000 if big else 0      # past one CTA's token budget
    lens = [0, 63, 64, 65, 448, 447, 500, -5, 128, 1]
    new = [0, 1, 64, 200, 1, 2, 3, 65, -4, 447]
    for num_free in (0, 1, 3, 5, 100):
        for free_pos in (0, 2, -3, 1000):
            _run_tables(lens, new, 64, 7, num_free, sum(max(n, 0) for n in new) + pad, free_pos=free_pos)
            _run_tables(lens, new, 64, 7, num_free, 70 + pad, free_pos=free_pos, in_place=True, skew=1)


@pytest.mark.parametrize("q_len", [1, 2, 3, 8])
@pytest.mark.parametrize("b", [1, 5, 130, 3000])
def test_tables_step_layout(q_len, b):
    rng = np.random.default_rng(q_len)
    lens = rng.integers(0, 400, b).tolist()
    new = rng.integers(-1, q_len + 3, b).tolist()
    _run_tables(lens, new, 64, 7, b // 2 + 1, b * q_len, q_len=q_len, in_place=True)


def test_tables_no_rows():
    _run_tables([5, 70], [0, 0], 64, 4, 3, 0)


def test_tables_page_ids_outside_the_cache():
    table = _i32([[1 << 30, -1], [0, -1]])
    slots, pos = (torch.empty(4, dtype=torch.int32, device="cuda") for _ in range(2))
    lens = _i32([3, 63])
    extend_block_tables(table, lens, _i32([2, 2]), _i32([-9]), _i32([0]), lens, _i32([0]), slots, pos, page_size=64,
                        num_pages=5)
    assert slots.tolist() == [-1, -1, 63, -1] and pos.tolist() == [3, 4, 63, 64]
    assert table.tolist() == [[1 << 30, -1], [0, -9]] and lens.tolist() == [5, 65]


# ---------------------------------------------------------------- rotary
def _check_rotary(got, x, pos, rot, offset):
    freq, gain = P.frequencies(rot.rot_dim, rot.base, rot.scaling)
    ref = P.rotate(x.double().cpu().numpy(), pos.cpu().numpy(), freq, gain, rot.interleaved, offset)
    g = got.double().cpu().numpy()
    eps = torch.finfo(got.dtype).eps
    # half a step of the result's type, and float32 cosines, sines, products and sums: the
    # angle's fraction 2^-26 of a turn (1e-7), sincospi 2 ulp (2.4e-7), gain, product and
    # sum half an ulp each (1.8e-7): below 1e-6 of |a| + |b|; fp16's smallest step below that
    tol = eps / 2 * np.abs(ref) * (1 + 1e-5) + 1e-6 * P.rotate_bound(x.double().cpu().numpy(), freq, gain, offset,
                                                                     rot.interleaved) + 2.0 ** -25
    bad = np.abs(g - ref) > tol
    assert not bad.any(), (np.abs(g - ref) / tol).max()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens, heads, dim, rot_dim, offset", [
    (1, 1, 64, 64, 0), (5, 128, 64, 64, 0), (33, 16, 192, 64, 128), (7, 3, 10, 6, 3), (300, 1, 64, 64, 0),
    (2, 5, 66, 64, 1), (9, 40, 80, 32, 16), (3, 2, 24, 24, 0), (1, 300, 128, 128, 0), (2, 1, 1030, 1024, 4)])
def test_rotary(dtype, interleaved, tokens, heads, dim, rot_dim, offset):
    g = torch.Generator().manual_seed(tokens + dim)
    x = torch.randn(tokens, heads, dim, generator=g).to(TDT[dtype]).cuda()
    pos = torch.randint(-1000, 1 << 20, (tokens,), generator=g, dtype=torch.int32).cuda()
    rot = Rotary(rot_dim, interleaved=interleaved)
    out = torch.full_like(x, float("nan"))
    keep = x.clone()
    rot(x, pos, out, offset=offset)
    assert torch.equal(x, keep)
    _check_rotary(out, x, pos, rot, offset)
    rot(x, pos, x, offset=offset)                     # in place
    assert torch.equal(x, out)


@pytest.mark.parametrize("scaling", [{"type": "linear", "factor": 8.0}, {"type": "ntk", "factor": 4.0},
                                     {"type": "yarn", "factor": 40.0, "original_max_position": 4096}])
def test_rotary_scaled_far(scaling):
    x = torch.randn(40, 4, 64, device="cuda").bfloat16()
    pos = torch.randint(0, 2**31 - 1, (40,), dtype=torch.int32, device="cuda")
    # at position 2^31 a float64 angle is itself off by 2^-53 x 2^31 (2.4e-7): both sides
    # hold positions up to 2^24 to 2e-9
    pos = pos % (1 << 24)
    rot = Rotary(64, base=1e5, interleaved=False, scaling=scaling)
    out = torch.empty_like(x)
    rot(x, pos, out)
    _check_rotary(out, x, pos, rot, 0)


def test_rotary_strided_and_back():
    base = torch.randn(6, 9, 200, device="cuda").half()
    pos = torch.arange(9, dtype=torch.int32, device="cuda") * 777
    x = base.transpose(0, 1)[:, :, 8:136]              # heads outermost, a slice of the dims
    rot = Rotary(64)
    out = torch.zeros(9, 12, 128, dtype=torch.half, device="cuda")
    rot(x, pos, out[:, ::2], offset=64)
    _check_rotary(out[:, ::2], x, pos, rot, 64)
    assert not out[:, 1::2].any()                      # the rows between stay as they were
    back = torch.empty(9, 6, 128, dtype=torch.half, device="cuda")
    rot(out[:, ::2], -pos, back, offset=64)
    # two roundings to fp16 of values up to |a| + |b| <= 2 max
    assert (back.float() - x.float()).abs().max() <= 2 * 2.0 ** -11 * 2 * x.float().abs().max()


def test_rotary_refusals():
    rot, x, pos = Rotary(), torch.zeros(4, 2, 64, device="cuda").half(), _i32([0, 1, 2, 3])
    out = torch.empty_like(x)
    with pytest.raises(ValueError, match="inside"):
        rot(x, pos, out, offset=1)
    with pytest.raises(ValueError, match="shape"):
        rot(x, pos[:3], out)
    with pytest.raises(ValueError, match="int32"):
        rot(x, pos.long(), out)
    with pytest.raises(ValueError, match="dtype"):
        rot(x, pos, out.float())
    with pytest.raises(ValueError, match="rows overlap"):
        rot(x, pos, out[:1].expand(4, 2, 64))
    with pytest.raises(ValueError, match="overlap it"):
        buf = torch.zeros(5, 2, 64, device="cuda").half()
        rot(buf[:4], pos, buf[1:])
    with pytest.raises(ValueError, match="contiguous"):
        rot(x.transpose(1, 2).contiguous().transpose(1, 2), pos, out)
    rot(x[:0], pos[:0], out[:0])


# ---------------------------------------------------------------- cache rows
def _cache(form, dtype, pages, page, kvh):
    lead = (pages, page, kvh)
    if form == "int4":
        kv, sc = torch.randint(0, 256, (*lead, 256), dtype=torch.uint8, device="cuda"), \
            torch.randn(*lead, 16, device="cuda").half()
    else:
        sc = None
        kv = torch.randn(*lead, 512, device="cuda").to(torch.float8_e4m3fn if form == "fp8" else TDT[dtype])
    return kv, sc, torch.randn(*lead, 64, device="cuda").to(TDT[dtype])


def _bytes(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


@pytest.mark.parametrize("form", ["model", "fp8", "int4"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens, kvh, layout, turn", [
    (1, 1, "dense", None), (7, 1, "fused", True), (300, 1, "dense", False), (33, 2, "heads", True), (64, 3, "dense", True)])
def test_append_and_gather(form, dtype, tokens, kvh, layout, turn):
    dt = TDT[dtype]
    g = torch.Generator(device="cuda").manual_seed(tokens)
    fused = torch.randn(tokens, kvh, 576 if layout != "heads" else 592, generator=g, device="cuda").to(dt)
    if layout == "heads":
        fused = fused.transpose(0, 1).contiguous().transpose(0, 1)
    kv, pe = fused[..., :512], fused[..., 512:576]
    if layout == "dense":
        kv, pe = kv.contiguous(), pe.contiguous()
    pages, page = 7, 64
    rows = pages * page
    slots = torch.randperm(rows, generator=g, device="cuda")[:tokens].to(torch.int32)
    if tokens > 3:
        slots[1], slots[2], slots[3] = -1, rows, 2**31 - 1       # skipped
    cache, scales, pec = _cache(form, dtype, pages, page, kvh)
    old = [None if t is None else _bytes(t).reshape(rows, kvh, -1) for t in (cache, scales, pec)]
    scale = 0.043 if form == "fp8" else None
    rot = None if turn is None else Rotary(64, interleaved=turn)
    pos = torch.randint(0, 1 << 17, (tokens,), generator=g, dtype=torch.int32, device="cuda")
    cache_append(kv, pe, slots, cache, pec, kv_scale=scale, kv_scales=scales, rotary=rot,
                 positions=None if rot is None else pos)
    x = kv.double().cpu().numpy()
    keep = (slots >= 0) & (slots < rows)
    idx, sel = slots[keep].long().cpu().numpy(), keep.cpu().numpy()
    new = [None if t is None else _bytes(t).reshape(rows, kvh, -1) for t in (cache, scales, pec)]
    if form == "int4":
        n, s = P.quantise_int4(x)
        assert np.array_equal(new[0][idx], P.pack_int4(n)[sel])
        assert np.array_equal(new[1][idx], np.ascontiguousarray(s).view(np.uint8).reshape(tokens, kvh, -1)[sel])
        value = P.dequantise_int4(n, s)
    elif form == "fp8":
        want = (kv.float() / scale).clamp(-448, 448).to(torch.float8_e4m3fn)
        assert np.array_equal(new[0][idx], _bytes(want)[sel])
        # float32 product of an e4m3 value and the scale
        value = (want.float() * torch.tensor(scale, dtype=torch.float32, device="cuda")).double().cpu().numpy()
    else:
        value = x
        assert np.array_equal(new[0][idx], _bytes(kv).reshape(tokens, kvh, -1)[sel])
    stay = np.ones(rows, bool)
    stay[idx] = False
    for a, b in zip(old, new):
        assert a is None or np.array_equal(a[stay], b[stay])      # other rows as they were
    if rot is None:
        assert np.array_equal(new[2][idx], _bytes(pe).reshape(tokens, kvh, -1)[sel])
    else:
        _check_rotary(pec.view(rows, kvh, 64)[slots[keep].long()], pe[keep], pos[keep], rot, 0)
    back = torch.full((tokens, kvh, 1024), float("nan"), dtype=dt, device="cuda")
    kv_b, pe_b = back[..., 256:768], back[..., 960:]
    cache_gather(slots, cache, pec, kv_b, pe_b, kv_scale=scale, kv_scales=scales)
    want = torch.from_numpy(np.where(sel[:, None, None], value, 0.0)).to(torch.float32).cuda().to(dt)
    assert torch.equal(kv_b, want)
    want_pe = torch.where(keep[:, None, None], pec.view(rows, kvh, 64)[slots.long().clamp(0, rows - 1)], 0)
    assert torch.equal(pe_b, want_pe)
    assert torch.isnan(back[..., :256]).all() and torch.isnan(back[..., 768:960]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_int4_special_values(dtype):
    """Zeros, one value, tiny and huge groups, ties between codes, infinities and NaN."""
    x = torch.zeros(12, 1, 512)
    x[1, 0, 5] = 3.0
    x[2] = 7.0 * torch.arange(512).remainder(2).sub(0.5)         # +-3.5
    x[3] = 1e-7
    x[4] = 6e4 if dtype == "fp16" else 3e38
    x[5, 0, ::32] = 7.0                                           # scale 1: codes tie at halves
    x[5, 0, 1::32], x[5, 0, 2::32], x[5, 0, 3::32] = 2.5, 3.5, -0.5
    x[6, 0, 40], x[6, 0, 41], x[6, 0, 42] = float("inf"), -float("inf"), 5.0
    x[7, 0, 70], x[7, 0, 71] = float("nan"), 2.0
    x[8] = float("nan")
    x[9] = -8.0
    x[10] = torch.linspace(-1, 1, 512)
    x[11] = -0.0
    x = x.to(TDT[dtype]).cuda()
    cache, scales, pec = _cache("int4", dtype, 1, 64, 1)
    slots = torch.arange(12, dtype=torch.int32, device="cuda") * 5
    pe = torch.zeros(12, 1, 64, dtype=TDT[dtype], device="cuda")
    cache_append(x, pe, slots, cache, pec, kv_scales=scales)
    n, s = P.quantise_int4(x.double().cpu().numpy())
    at = slots.long()
    assert np.array_equal(cache.view(64, 1, 256)[at].cpu().numpy(), P.pack_int4(n))
    assert np.array_equal(scales.view(64, 1, 16)[at].cpu().numpy().view(np.uint16), s.view(np.uint16))


def test_fp8_special_values():
    x = torch.zeros(1, 1, 512)
    x[0, 0, :8] = torch.tensor([float("inf"), -float("inf"), float("nan"), 1e4, -1e4, 448.0, 2.0 ** -9, 2.0 ** -11])
    x = x.bfloat16().cuda()
    cache, _, pec = _cache("fp8", "bf16", 1, 64, 1)
    slots = _i32([9])
    cache_append(x, torch.zeros(1, 1, 64, device="cuda").bfloat16(), slots, cache, pec, kv_scale=1.0)
    got = cache.view(64, 512)[9].float().cpu()
    assert got[:2].tolist() == [448.0, -448.0] and torch.isnan(got[2])
    assert got[3:8].tolist() == [448.0, -448.0, 448.0, 2.0 ** -9, 0.0]


def test_cache_refusals():
    kv, pe = torch.zeros(4, 1, 512, device="cuda").bfloat16(), torch.zeros(4, 1, 64, device="cuda").bfloat16()
    slots = _i32([0, 1, 2, 3])
    c4, s4, p4 = _cache("int4", "bf16", 2, 64, 1)
    c16, _, _ = _cache("model", "bf16", 2, 64, 1)
    for bad in (dict(kv_scale=1.0), dict(), dict(kv_scales=s4[..., :8]), dict(kv_scales=s4.float()),
                dict(kv_scales=s4, rotary=Rotary()), dict(kv_scales=s4, positions=slots),
                dict(kv_scales=s4, rotary=Rotary(32), positions=slots),
                dict(kv_scales=s4, rotary=Rotary(), positions=slots[:2])):
        with pytest.raises(ValueError):
            cache_append(kv, pe, slots, c4, p4, **bad)
    with pytest.raises(ValueError, match="dtype"):
        cache_append(kv, pe, slots, c16.half(), p4)
    with pytest.raises(ValueError, match="kv_scale"):
        cache_append(kv, pe, slots, c16, p4, kv_scale=1.0)
    with pytest.raises(ValueError, match="KV heads"):
        cache_append(kv.expand(4, 2, 512), pe.expand(4, 2, 64), slots, c4, p4, kv_scales=s4)
    with pytest.raises(ValueError, match="boundary"):
        odd = torch.zeros(4 * 520, device="cuda").bfloat16()
        cache_append(odd.as_strided((4, 1, 512), (516, 516, 1)), pe, slots, c4, p4, kv_scales=s4)
    with pytest.raises(ValueError, match="rows overlap"):
        cache_gather(slots, c16, p4, kv[:1].expand(4, 1, 512), pe)
    cache_append(kv[:0], pe[:0], slots[:0], c16, p4)
    cache_append(kv[:1].expand(4, 1, 512), pe[:1].expand(4, 1, 64), slots, c16, p4)   # one row to four slots
