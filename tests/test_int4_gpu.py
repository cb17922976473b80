"""GPU tests of decode over a 4-bit latent cache and of the whole paged decode step."""
import numpy as np
import pytest
import torch

from mlc_decode_b200 import MlaPagedDecodeKernel, Rotary, cache_gather
from oracle import mla_oracle as O
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

TDT = {"fp16": torch.float16, "bf16": torch.bfloat16}
SCALE = 576 ** -0.5
# the CUDA-core kernel, the library's choice, and each of the two tensor-core kernels
KERNELS = {"simt": {"kernel": "simt"}, "auto": {}, "pair": {"block_H": 128}, "mma16": {"block_H": 16},
           "mma32": {"block_H": 32}}


def _inputs(b, ql, h, kvh, smax, dtype, seed, peak=1.0):
    rng = np.random.default_rng(seed)

    def t(*shape, s=1.0):
        return torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * s).to(TDT[dtype])

    q, qp = t(b, ql, h, 512, s=peak), t(b, ql, h, 64, s=peak)
    n, s = P.quantise_int4(rng.standard_normal((b, smax, kvh, 512)).astype(np.float32))
    return q, qp, n, s, t(b, smax, kvh, 64)


def _caches(n, s, kp, lens, page, seed):
    """Contiguous (page 0) or shuffled pages; rows past a length hold NaN scales and rope
    values, table entries past it page ids the cache does not have."""
    b, smax, kvh = n.shape[:3]
    g = np.random.default_rng(seed + 1)
    kp = kp.clone()
    codes, s = P.pack_int4(n), s.copy()
    for i, L in enumerate(lens):
        codes[i, max(L, 0):], s[i, max(L, 0):], kp[i, max(L, 0):] = 255, np.nan, float("nan")
    if page == 0:
        return torch.from_numpy(codes).cuda(), torch.from_numpy(s).cuda(), kp.cuda(), None
    per = -(-smax // page)
    num = b * per + 2
    ids = g.permutation(num)[:b * per].reshape(b, per)
    pc = np.full((num, page, kvh, 256), 255, np.uint8)
    ps = np.full((num, page, kvh, 16), np.nan, np.float16)
    pk = torch.full((num, page, kvh, 64), float("nan"), dtype=kp.dtype)
    table = np.full((b, per), 1 << 29, np.int32)
    for i, L in enumerate(lens):
        for j in range(-(-max(L, 0) // page)):
            m = min(page, smax - j * page)
            pc[ids[i, j], :m], ps[ids[i, j], :m] = codes[i, j * page:j * page + m], s[i, j * page:j * page + m]
            pk[ids[i, j], :m] = kp[i, j * page:j * page + m]
            table[i, j] = ids[i, j]
    return torch.from_numpy(pc).cuda(), torch.from_numpy(ps).cuda(), pk.cuda(), torch.from_numpy(table).cuda()


def _check(out, lse, q, qp, n, s, kp, lens, dtype, scale=SCALE, v=None):
    b, ql, h = q.shape[:3]
    kvh = kp.shape[2]
    g = h // kvh
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    eps = torch.finfo(TDT[dtype]).eps
    q, qp, kp = (t.double().cpu().numpy() for t in (q, qp, kp))
    err = ref2 = gate = 0.0
    for i in range(b):
        rows = P.dequantise_int4(n[i], s[i]) if v is None else v[i]
        for t in range(ql):
            m = max(min(max(lens[i], 0), kp.shape[1]) - (ql - 1 - t), 0)
            for j in range(kvh):
                hs = slice(j * g, (j + 1) * g)
                ref, ref_lse, spread, ds = P.decode(q[i, t, hs], qp[i, t, hs], rows[:m, j], kp[i, :m, j], scale)
                got, got_lse = out[i, t, hs], lse[i, t, hs]
                if m == 0:
                    assert not got.any() and np.isneginf(got_lse).all()
                    continue
                tol = spread + eps / 2 * np.abs(ref) + 1e-6
                assert (np.abs(got - ref) <= tol).all(), (i, t, j, (np.abs(got - ref) / tol).max())
                assert (np.abs(got_lse - ref_lse) <= ds[:, 0] + 1e-4).all(), (i, t, j)
                want = O.round_to(ref, dtype)
                err += ((got - want) ** 2).sum()
                ref2 += (want ** 2).sum()
                gate += (want ** 2).sum() * P.rounding_gate(q[i, t, hs], qp[i, t, hs], rows[:m, j], kp[i, :m, j],
                                                            scale, dtype)
    # over the whole call: the expected distance of a kernel whose weights and row values are
    # fp16, and half as much again
    assert err <= 1.5 ** 2 * gate, ((err / ref2) ** 0.5, (gate / ref2) ** 0.5)


CASES = [
    # b, q_len, heads, kv_heads, smax, lens, page
    (1, 1, 1, 1, 1, [1], 0),
    (1, 1, 16, 1, 300, [300], 64),
    (3, 1, 128, 1, 257, [257, 1, 128], 64),
    (6, 1, 128, 1, 700, [0, 1, 130, 700, 64, 257], 0),
    (5, 1, 40, 1, 513, [513, 512, 511, 0, 65], 192),
    (2, 1, 200, 1, 333, [333, 129], 128),
    (4, 3, 16, 1, 400, [400, 2, 1, 0], 64),
    (2, 2, 128, 1, 1000, [1000, 129], 256),
    (3, 1, 32, 2, 200, [200, 64, 0], 64),
    (2, 2, 24, 3, 130, [130, 5], 0),
    (1, 1, 128, 1, 5000, [4999], 64),
    (64, 1, 8, 1, 130, [(37 * i) % 131 for i in range(64)], 64),
    (2, 1, 64, 1, 128, [-3, 400], 0),              # lengths outside [0, max]
    (300, 1, 16, 1, 70, [(11 * i) % 71 for i in range(300)], 64),   # more sequences than workers
    (3, 5, 3, 1, 300, [300, 4, 70], 64),           # query rows of several positions in one tile
    (1, 1, 16, 1, 30000, [29999], 64),             # one sequence over every worker
]


@pytest.mark.parametrize("kernel", list(KERNELS))
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"b{c[0]}q{c[1]}h{c[2]}k{c[3]}s{c[4]}p{c[6]}")
def test_decode_int4(case, dtype, kernel):
    b, ql, h, kvh, smax, lens, page = case
    q, qp, n, s, kp = _inputs(b, ql, h, kvh, smax, dtype, seed=smax + h)
    codes, scales, pe, table = _caches(n, s, kp, [min(L, smax) for L in lens], page, seed=smax)
    k = MlaPagedDecodeKernel(b, h, smax, cfg=KERNELS[kernel], q_len=ql, kv_heads=kvh)
    qq, qpp = (t.cuda().squeeze(1) if ql == 1 else t.cuda() for t in (q, qp))
    out = torch.full(qq.shape, float("nan"), dtype=TDT[dtype], device="cuda")
    lse = torch.full(qq.shape[:-1], float("nan"), device="cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for _ in range(2):       # the workspace is left ready for the next call
        k.decode_int4(qq, qpp, codes, scales, pe, sl, out, lse, block_table=table)
    _check(out.view(b, ql, h, 512), lse.view(b, ql, h), q, qp, n, s, kp, lens, dtype)
    first = out.clone()
    k.decode_int4(qq, qpp, codes, scales, pe, sl, out, block_table=table)      # no lse
    if kernel in ("simt", "mma16", "mma32"):
        assert torch.equal(out, first)       # (the pair kernel merges split sequences in order of arrival)
    assert k.device_status(torch.device("cuda"), TDT[dtype]) == 0


@pytest.mark.parametrize("kernel", list(KERNELS))
def test_decode_int4_no_lengths_scale_and_peaks(kernel):
    """All rows of every sequence, a softmax scale of the caller's, peaky scores."""
    q, qp, n, s, kp = _inputs(3, 1, 48, 1, 390, "bf16", seed=4, peak=3.0)
    codes, scales, pe, _ = _caches(n, s, kp, [390] * 3, 0, seed=1)
    k = MlaPagedDecodeKernel(3, 48, 390, cfg=KERNELS[kernel], softmax_scale=0.1)
    out, lse = torch.empty(3, 48, 512, device="cuda").bfloat16(), torch.empty(3, 48, device="cuda")
    k.decode_int4(q.cuda().squeeze(1), qp.cuda().squeeze(1), codes, scales, pe, None, out, lse)
    _check(out.unsqueeze(1), lse.unsqueeze(1), q, qp, n, s, kp, [390] * 3, "bf16", scale=0.1)


@pytest.mark.parametrize("kernel", list(KERNELS))
def test_decode_int4_pages_outside_the_cache_read_as_zeros(kernel):
    q, qp, n, s, kp = _inputs(2, 1, 16, 1, 256, "bf16", seed=9)
    codes, scales, pe, table = _caches(n, s, kp, [256, 256], 64, seed=3)
    for (i, j), bad in (((0, 1), -1), ((0, 3), 1 << 30), ((1, 0), codes.shape[0]), ((1, 2), -(2**31))):
        table[i, j] = bad
        n[i, 64 * j:64 * j + 64], kp[i, 64 * j:64 * j + 64] = 8, 0.0
    k = MlaPagedDecodeKernel(2, 16, 256, cfg=KERNELS[kernel])
    out, lse = torch.empty(2, 16, 512, device="cuda").bfloat16(), torch.empty(2, 16, device="cuda")
    sl = torch.tensor([256, 256], dtype=torch.int32, device="cuda")
    k.decode_int4(q.cuda().squeeze(1), qp.cuda().squeeze(1), codes, scales, pe, sl, out, lse, block_table=table)
    _check(out.unsqueeze(1), lse.unsqueeze(1), q, qp, n, s, kp, [256, 256], "bf16")


def test_decode_int4_extreme_scales():
    """Groups of zeros, of the largest scale whose values fit fp16, and of tiny scales."""
    q, qp, n, s, kp = _inputs(1, 1, 16, 1, 200, "fp16", seed=5, peak=1e-3)
    s[:, ::3, :, ::2] = 0
    s[:, 1::3, :, 1::4] = 8000.0
    s[:, 2::3, :, ::5] = 6e-8
    codes, scales, pe, _ = _caches(n, s, kp, [200], 0, seed=1)
    for kernel in KERNELS:
        k = MlaPagedDecodeKernel(1, 16, 200, cfg=KERNELS[kernel])
        out, lse = torch.empty(1, 16, 512, device="cuda").half(), torch.empty(1, 16, device="cuda")
        k.decode_int4(q.cuda().squeeze(1), qp.cuda().squeeze(1), codes, scales, pe, None, out, lse)
        _check(out.unsqueeze(1), lse.unsqueeze(1), q, qp, n, s, kp, [200], "fp16")


def test_decode_int4_on_a_side_stream_and_in_a_graph():
    q, qp, n, s, kp = _inputs(4, 1, 128, 1, 640, "bf16", seed=21)
    lens = [640, 33, 0, 500]
    codes, scales, pe, table = _caches(n, s, kp, lens, 64, seed=2)
    k = MlaPagedDecodeKernel(4, 128, 640)
    qq, qpp = q.cuda().squeeze(1), qp.cuda().squeeze(1)
    out, lse = torch.empty_like(qq), torch.empty(4, 128, device="cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        k.decode_int4(qq, qpp, codes, scales, pe, sl, out, lse, block_table=table)
    side.synchronize()
    _check(out.unsqueeze(1), lse.unsqueeze(1), q, qp, n, s, kp, lens, "bf16")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k.decode_int4(qq, qpp, codes, scales, pe, sl, out, lse, block_table=table)
    lens = [5, 640, 129, 0]
    codes2, scales2, pe2, table2 = _caches(n, s, kp, [640] * 4, 64, seed=2)
    for dst, src in ((codes, codes2), (scales, scales2), (pe, pe2), (table, table2)):
        dst.copy_(src)
    sl.copy_(torch.tensor(lens))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    _check(out.unsqueeze(1), lse.unsqueeze(1), q, qp, n, s, kp, lens, "bf16")


def test_decode_int4_refusals():
    k = MlaPagedDecodeKernel(2, 16, 128)
    q, qp = torch.zeros(2, 16, 512, device="cuda").half(), torch.zeros(2, 16, 64, device="cuda").half()
    codes = torch.zeros(2, 128, 1, 256, dtype=torch.uint8, device="cuda")
    scales, pe = torch.zeros(2, 128, 1, 16, device="cuda").half(), torch.zeros(2, 128, 1, 64, device="cuda").half()
    out = torch.empty_like(q)
    ok = dict(q=q, q_pe=qp, kv_codes=codes, kv_scales=scales, k_pe_cache=pe, cache_seqlens=None, out=out)
    for bad in (dict(q=q.float()), dict(q_pe=qp.bfloat16()), dict(kv_codes=codes.char()), dict(kv_codes=codes[:1]),
                dict(kv_scales=scales.float()), dict(kv_scales=scales[:, :64]), dict(k_pe_cache=pe.bfloat16()),
                dict(out=out[:1]), dict(cache_seqlens=torch.zeros(2, device="cuda")),
                dict(lse=torch.zeros(2, 15, device="cuda")), dict(q=q.transpose(0, 1)),
                dict(block_table=torch.zeros(1, 2, dtype=torch.int32, device="cuda")),
                dict(block_table=torch.zeros(2, 2, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError):
            k.decode_int4(**{**ok, **bad})
    k.decode_int4(**ok)


# ---------------------------------------------------------------- the whole step
@pytest.mark.parametrize("form", ["model", "fp8", "int4"])
@pytest.mark.parametrize("ql, h", [(1, 128), (3, 16)])
def test_step(form, ql, h):
    """Steps from an empty cache, some of them without rows for some requests: after each the
    output is the decode over what the cache stands for, with rotated queries and keys; the
    last steps run from a captured graph, and one request finds the free list empty."""
    dt, b, page, per = torch.bfloat16, 3, 64, 3
    num = 6
    g = torch.Generator().manual_seed(ql)
    lead = (num, page, 1)
    if form == "int4":
        kv_cache = torch.full((*lead, 256), 255, dtype=torch.uint8, device="cuda")
        extra = {"kv_scales": torch.full((*lead, 16), float("nan"), dtype=torch.half, device="cuda")}
    elif form == "fp8":
        kv_cache = torch.full((*lead, 512), 0x7f, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        extra = {"kv_scale": 1 / 64}
    else:
        kv_cache, extra = torch.full((*lead, 512), float("nan"), dtype=dt, device="cuda"), {}
    pe_cache = torch.full((*lead, 64), float("nan"), dtype=dt, device="cuda")
    table = torch.full((b, per), -1, dtype=torch.int32, device="cuda")
    lens = torch.tensor([0, 62, 0], dtype=torch.int32, device="cuda")
    table[1, 0] = 4
    for c in (kv_cache, *([extra["kv_scales"]] if form == "int4" else []), pe_cache):   # request 1's first rows
        c[4].view(torch.uint8).zero_()
    free = torch.tensor([2, 0, 5], dtype=torch.int32, device="cuda")
    free_pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    rot = Rotary(64, scaling={"type": "yarn", "factor": 4.0, "original_max_position": 64})
    k = MlaPagedDecodeKernel(b, h, per * page, q_len=ql)
    qs = (b, h) if ql == 1 else (b, ql, h)
    rs = (b, 1) if ql == 1 else (b, ql, 1)
    q, qp = torch.empty(*qs, 512, dtype=dt, device="cuda"), torch.empty(*qs, 64, dtype=dt, device="cuda")
    kv, kp = torch.empty(*rs, 512, dtype=dt, device="cuda"), torch.empty(*rs, 64, dtype=dt, device="cuda")
    new = torch.empty(b, dtype=torch.int32, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(qs, device="cuda")

    def call():
        k.step(q, qp, kv, kp, kv_cache, pe_cache, table, lens, free, free_pos, out, lse, new_lens=new, rotary=rot, **extra)

    freq, gain = P.frequencies(64, 10000.0, rot.scaling)
    graph = None
    held = [0, 62, 0]
    for it in range(40):
        for t in (q, qp, kv, kp):
            t.copy_(torch.randn(t.shape, generator=g).to(dt))
        n = [min(ql, 1 + it % 2), ql, 0 if it % 3 == 0 else 1]
        new.copy_(torch.tensor(n, dtype=torch.int32))
        if it == 35:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                call()
        keep_qp = qp.clone()
        graph.replay() if graph is not None else call()
        assert torch.equal(qp, keep_qp)
        before, held = held, lens.tolist()
        assert all(0 <= a - c <= m for a, c, m in zip(held, before, n))
        if it not in (0, 1, 5, 34, 35, 36, 39):
            continue
        for i in range(b):
            if held[i] == 0:
                continue
            r = torch.arange(held[i], device="cuda")
            slots = (table[i].long()[r // page] * page + r % page).int()
            v, pe = torch.empty(held[i], 1, 512, dtype=dt, device="cuda"), torch.empty(held[i], 1, 64, dtype=dt, device="cuda")
            cache_gather(slots, kv_cache, pe_cache, v, pe, **extra)
            # the step's own rows, as the cache holds them: rotated to their positions
            for t in range(held[i] - before[i]):
                p = before[i] + t
                src = kp.view(b, ql, 1, 64)[i, ql - n[i] + t].double().cpu().numpy()
                want = P.rotate(src[None], [p], freq, gain, True)[0]
                tol = 2.0 ** -8 * np.abs(want) + 1e-6 * P.rotate_bound(src[None], freq, gain)[0]
                assert (np.abs(pe[p].double().cpu().numpy() - want) <= tol).all()
            if form == "int4":
                code = P.unpack_int4(kv_cache.view(-1, 256)[slots.long()].cpu().numpy())
                rows = P.dequantise_int4(code, extra["kv_scales"].view(-1, 16)[slots.long()].cpu().numpy())
            else:
                rows = v[:, 0].double().cpu().numpy()
            if n[i] < ql or held[i] - before[i] < n[i]:
                last = [ql - 1] if n[i] else []      # a shorter step: its last position sees every row
            else:
                last = range(ql)
            if held[i] - before[i] < n[i]:
                continue                             # no place for all rows: the positions do not line up
            for t in last:
                m = held[i] - (ql - 1 - t)
                qq, qqp = (x.view(b, ql, h, -1)[i, t].double().cpu().numpy() for x in (q, qp))
                turned = O.round_to(P.rotate(qqp[None], [m - 1], freq, gain, True)[0], "bf16")
                ref, ref_lse, spread, bound = P.decode(qq, turned, rows[:m], pe[:m, 0].double().cpu().numpy(), SCALE)
                got = out.view(b, ql, h, 512)[i, t].double().cpu().numpy()
                got_lse = lse.view(b, ql, h)[i, t].double().cpu().numpy()
                # a query value beside a tie may round the other way: one bf16 step of it
                # times the keys moves a score by at most this
                ds = (2.0 ** -8 * np.abs(turned) @ np.abs(pe[:m, 0].double().cpu().numpy()).T).max() * SCALE * 1e-2
                tol = spread + 2.0 ** -8 * np.abs(ref) + 2 * ds * np.abs(rows[:m]).max() + 1e-6
                assert (np.abs(got - ref) <= tol).all(), (it, i, t)
                assert (np.abs(got_lse - ref_lse) <= bound[:, 0] + 1e-4 + ds).all()
    assert sum(-(-x // page) for x in held) <= 4 and int(free_pos) <= 3


def test_step_refused_changes_nothing():
    b, h = 2, 16
    k = MlaPagedDecodeKernel(b, h, 128)
    dt = torch.bfloat16
    q, qp = torch.zeros(b, h, 512, dtype=dt, device="cuda"), torch.zeros(b, h, 64, dtype=dt, device="cuda")
    kv, kp = torch.zeros(b, 1, 512, dtype=dt, device="cuda"), torch.zeros(b, 1, 64, dtype=dt, device="cuda")
    cache, pe = torch.zeros(4, 64, 1, 512, dtype=dt, device="cuda"), torch.zeros(4, 64, 1, 64, dtype=dt, device="cuda")
    table = torch.full((b, 2), -1, dtype=torch.int32, device="cuda")
    lens, free_pos = torch.zeros(b, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    free = torch.arange(4, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    ok = dict(q=q, q_pe=qp, kv=kv, k_pe=kp, kv_cache=cache, k_pe_cache=pe, block_table=table, cache_seqlens=lens,
              free_pages=free, free_pos=free_pos, out=out)
    for bad in (dict(q=q.float()), dict(kv=kv.half()), dict(kv=kv[:1]), dict(k_pe=kp.unsqueeze(1)),
                dict(kv_cache=cache[:, :32].contiguous(), k_pe_cache=pe[:, :32].contiguous()),
                dict(kv_cache=cache.to(torch.float8_e4m3fn)), dict(kv_cache=cache.to(torch.float8_e4m3fn), kv_scale=0.0),
                dict(kv_scale=1.0), dict(rotary=Rotary(32)), dict(new_lens=lens[:1]), dict(out=out.half()),
                dict(block_table=torch.zeros(b, 3, dtype=torch.int32, device="cuda")),
                dict(lse=torch.zeros(b, h, dtype=dt, device="cuda")), dict(free_pages=free.long()),
                dict(free_pos=free)):
        with pytest.raises(ValueError):
            k.step(**{**ok, **bad})
        assert lens.tolist() == [0, 0] and free_pos.item() == 0 and (table == -1).all()
    simt = MlaPagedDecodeKernel(b, h, 128, cfg={"kernel": "simt"})
    with pytest.raises(Exception, match="tensor-core"):
        simt.step(**ok)
    assert lens.tolist() == [0, 0] and free_pos.item() == 0
    k.step(**ok)
    assert lens.tolist() == [1, 1]
