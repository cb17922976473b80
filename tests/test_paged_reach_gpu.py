"""GPU tests of the paged operators where they are reached differently: long row lists, many
sequences with one of them widely split, call after call on other tensors, captured graphs,
streams of their own."""
import numpy as np
import pytest
import torch

from mlc_decode_b200 import MlaPagedDecodeKernel, Rotary, cache_append, cache_gather, extend_block_tables
from oracle import mla_oracle as O
from oracle import paged_oracle as P
from test_int4_gpu import KERNELS, _caches, _check, _inputs

pytestmark = pytest.mark.gpu

SCALE = 576 ** -0.5


@pytest.mark.parametrize("form", ["model", "fp8", "int4"])
@pytest.mark.parametrize("tokens, kvh", [(20001, 1), (6667, 3)])
def test_long_append_and_gather(form, tokens, kvh):
    """More rows than the GPU has warps, an odd number of them: what a gather returns is what
    the appended rows became."""
    dt = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(tokens)
    pages, page = 330, 64
    rows = pages * page
    kv = torch.randn(tokens, kvh, 512, generator=g, device="cuda").to(dt)
    pe = torch.randn(tokens, kvh, 64, generator=g, device="cuda").to(dt)
    slots = torch.randperm(rows, generator=g, device="cuda")[:tokens].to(torch.int32)
    slots[tokens // 2] = -1
    lead = (pages, page, kvh)
    extra = {"model": {}, "fp8": {"kv_scale": 0.02},
             "int4": {"kv_scales": torch.zeros(*lead, 16, dtype=torch.half, device="cuda")}}[form]
    cache = {"model": torch.zeros(*lead, 512, dtype=dt, device="cuda"),
             "fp8": torch.zeros(*lead, 512, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
             "int4": torch.full((*lead, 256), 0x88, dtype=torch.uint8, device="cuda")}[form]
    pec = torch.zeros(*lead, 64, dtype=dt, device="cuda")
    cache_append(kv, pe, slots, cache, pec, **extra)
    if form == "model":
        want = kv.clone()
    elif form == "fp8":
        code = (kv.float() / 0.02).clamp(-448, 448).to(torch.float8_e4m3fn)
        want = (code.float() * torch.tensor(0.02, device="cuda")).to(dt)
    else:
        x = kv.float().view(tokens, kvh, 16, 32)
        s = (x.abs().amax(-1, keepdim=True).double() / 7).half().double()
        n = (x.double() / s).float().round().clamp(-8, 7)      # (a float32 quotient, ties to even)
        want = (n * s.float()).view(tokens, kvh, 512).to(dt)
    want[tokens // 2] = 0
    want_pe = pe.clone()
    want_pe[tokens // 2] = 0
    got, got_pe = torch.full_like(kv, float("nan")), torch.full_like(pe, float("nan"))
    cache_gather(slots, cache, pec, got, got_pe, **extra)
    assert torch.equal(got, want) and torch.equal(got_pe, want_pe)


LENS = [40, 0, 129, 64, 9000, 1, 300, 77, 128, 513, 2, 256]


@pytest.mark.parametrize("ql, h", [(1, 128), (2, 24), (1, 200)])
@pytest.mark.parametrize("form", ["bf16", "fp8", "int4"])
def test_one_long_sequence_among_many(form, ql, h):
    """Twelve sequences, one of them over many CTA pairs: its partials are merged by the
    combine launch, everyone else's in the decode launch."""
    b, smax = len(LENS), max(LENS)
    q, qp, n, s, kp = _inputs(b, ql, h, 1, smax, "bf16", seed=h)
    sl = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    qq, qpp = (t.cuda().squeeze(1) if ql == 1 else t.cuda() for t in (q, qp))
    out = torch.full(qq.shape, float("nan"), dtype=torch.bfloat16, device="cuda")
    lse = torch.full(qq.shape[:-1], float("nan"), device="cuda")
    k = MlaPagedDecodeKernel(b, h, smax, cfg={"block_H": 128} if form == "int4" else None, q_len=ql)
    if form == "int4":
        codes, scales, pe, table = _caches(n, s, kp, LENS, 64, seed=3)
        for _ in range(2):
            k.decode_int4(qq, qpp, codes, scales, pe, sl, out, lse, block_table=table)
        _check(out.view(b, ql, h, 512), lse.view(b, ql, h), q, qp, n, s, kp, LENS, "bf16")
        return
    # the rows themselves: small integers times a power of two, exact in bf16 and in e4m3
    kv = torch.from_numpy((n.astype(np.float32) - 8) / 4)
    if form == "fp8":
        cache, extra = (kv * 4).to(torch.float8_e4m3fn).cuda(), {"kv_scale": 0.25}
    else:
        cache, extra = kv.bfloat16().cuda(), {}
    for _ in range(2):
        k(qq, qpp, cache, kp.cuda(), sl, out, lse, **extra)
    o, l = out.view(b, ql, h, 512).float().cpu().numpy(), lse.view(b, ql, h).cpu().numpy()
    for i in range(b):
        for t in range(ql):
            m = max(LENS[i] - (ql - 1 - t), 0)
            if m == 0:
                assert not o[i, t].any() and np.isneginf(l[i, t]).all()
                continue
            ref, ref_lse = O.ref_program_f64(q[i:i + 1, t], qp[i:i + 1, t], kv[i:i + 1, :m].bfloat16(), kp[i:i + 1, :m])
            res = O.check_parity(o[i:i + 1, t], l[i:i + 1, t], ref, ref_lse, "bf16")
            assert res["ok"], (i, t, res)


@pytest.mark.parametrize("kernel", ["mma16", "mma32", "auto"])
def test_more_sequences_than_threads(kernel):
    b = 1100
    lens = [(13 * i) % 71 for i in range(b)]
    q, qp, n, s, kp = _inputs(b, 1, 4, 1, 70, "fp16", seed=8)
    codes, scales, pe, table = _caches(n, s, kp, lens, 64, seed=8)
    k = MlaPagedDecodeKernel(b, 4, 70, cfg=KERNELS[kernel])
    qq, qpp = q.cuda().squeeze(1), qp.cuda().squeeze(1)
    out, lse = torch.empty_like(qq), torch.empty(b, 4, device="cuda")
    k.decode_int4(qq, qpp, codes, scales, pe, torch.tensor(lens, dtype=torch.int32, device="cuda"), out, lse,
                  block_table=table)
    _check(out.unsqueeze(1), lse.unsqueeze(1), q, qp, n, s, kp, lens, "fp16")


@pytest.mark.parametrize("kernel", list(KERNELS))
def test_calls_on_other_tensors_of_the_same_shape(kernel):
    """Two sets of inputs in turn through one object: each call reads and writes its own."""
    k = MlaPagedDecodeKernel(2, 32, 200, cfg=KERNELS[kernel])
    sets = []
    for seed in (1, 2):
        q, qp, n, s, kp = _inputs(2, 1, 32, 1, 200, "bf16", seed=seed)
        codes, scales, pe, _ = _caches(n, s, kp, [200, 200], 0, seed=1)
        sets.append((q, qp, n, s, kp, q.cuda().squeeze(1), qp.cuda().squeeze(1), codes, scales, pe,
                     torch.zeros(2, 32, 512, device="cuda").bfloat16(), torch.zeros(2, 32, device="cuda")))
    for it in range(2):
        for x in sets:
            k.decode_int4(*x[5:10], None, x[10], x[11])
    for q, qp, n, s, kp, *_, out, lse in sets:
        _check(out.unsqueeze(1), lse.unsqueeze(1), q, qp, n, s, kp, [200, 200], "bf16")


def test_model_type_calls_on_other_tensors_of_the_same_shape():
    k = MlaPagedDecodeKernel(2, 128, 300)
    sets = []
    for seed in (5, 6):
        q, qp, kv, kp = O.make_inputs(2, 128, 300, "bf16", seed=seed)
        sets.append((q, qp, kv, kp, [t.cuda() for t in (q, qp, kv, kp)],
                     torch.zeros(2, 128, 512, device="cuda").bfloat16(), torch.zeros(2, 128, device="cuda")))
    for it in range(2):
        for *_, dev, out, lse in sets:
            k(*dev, None, out, lse)
    for q, qp, kv, kp, _, out, lse in sets:
        ref, ref_lse = O.ref_program_f64(q, qp, kv, kp)
        res = O.check_parity(out.float().cpu().numpy(), lse.cpu().numpy(), ref, ref_lse, "bf16")
        assert res["ok"], res


@pytest.mark.parametrize("kernel", ["pair", "mma16"])
def test_two_objects_on_two_streams(kernel):
    """Each with a workspace of its own; their launches may overlap."""
    objs = []
    for seed in (11, 12):
        q, qp, n, s, kp = _inputs(3, 1, 16, 1, 2000, "bf16", seed=seed)
        lens = [2000, 700, 65]
        codes, scales, pe, table = _caches(n, s, kp, lens, 64, seed=seed)
        objs.append((q, qp, n, s, kp, lens, MlaPagedDecodeKernel(3, 16, 2000, cfg=KERNELS[kernel]),
                     [q.cuda().squeeze(1), qp.cuda().squeeze(1), codes, scales, pe,
                      torch.tensor(lens, dtype=torch.int32, device="cuda")],
                     torch.zeros(3, 16, 512, device="cuda").bfloat16(), torch.zeros(3, 16, device="cuda"), table,
                     torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for *_, k, args, out, lse, table, stream in objs:
            with torch.cuda.stream(stream):
                k.decode_int4(*args, out, lse, block_table=table)
    torch.cuda.synchronize()
    for q, qp, n, s, kp, lens, k, _, out, lse, _, _ in objs:
        _check(out.unsqueeze(1), lse.unsqueeze(1), q, qp, n, s, kp, lens, "bf16")
        assert k.device_status(torch.device("cuda"), torch.bfloat16) == 0


@pytest.mark.parametrize("batch, per", [(9, 40), (2100, 6)])
def test_prompt_rows_in_a_graph(batch, per):
    """Tables, append and gather of packed prompt rows captured together (the second size
    takes the two-launch form with its workspace), replayed on other lengths and rows."""
    dt, page, max_pages = torch.float16, 64, 3
    tokens = batch * per
    rng = np.random.default_rng(batch)
    num_pages = 2 * batch + 7
    table = torch.full((batch, max_pages), -1, dtype=torch.int32, device="cuda")
    lens, new = (torch.zeros(batch, dtype=torch.int32, device="cuda") for _ in range(2))
    free = torch.from_numpy(rng.permutation(num_pages).astype(np.int32)).cuda()
    pos0 = torch.zeros(1, dtype=torch.int32, device="cuda")
    slots, positions = (torch.empty(tokens, dtype=torch.int32, device="cuda") for _ in range(2))
    kv, pe = torch.zeros(tokens, 1, 512, dtype=dt, device="cuda"), torch.zeros(tokens, 1, 64, dtype=dt, device="cuda")
    cache = torch.zeros(num_pages, page, 1, 512, dtype=dt, device="cuda")
    pec = torch.zeros(num_pages, page, 1, 64, dtype=dt, device="cuda")
    back, back_pe = torch.empty_like(kv), torch.empty_like(pe)
    rot = Rotary(64)
    rot.turns(torch.device("cuda", 0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        extend_block_tables(table, lens, new, free, pos0, lens, pos0, slots, positions, page_size=page,
                            num_pages=num_pages)
        cache_append(kv, pe, slots, cache, pec, rotary=rot, positions=positions)
        cache_gather(slots, cache, pec, back, back_pe)
    state = (table.tolist(), lens.tolist(), 0)
    for it in range(3):
        n = rng.integers(0, per + 1, batch)
        new.copy_(torch.from_numpy(n.astype(np.int32)))
        kv.normal_()
        pe.normal_()
        graph.replay()
        ref = P.extend_tables(state[0], state[1], n.tolist(), free.tolist(), state[2], page, num_pages, tokens)
        assert (table.tolist(), lens.tolist(), int(pos0)) == ref[:3]
        assert slots.tolist() == ref[3] and positions.tolist() == ref[4]
        state = ref[:3]
        has = slots >= 0
        assert torch.equal(back[has], kv[has]) and not back[~has].any()
        turned = torch.empty_like(pe)
        rot(pe, positions, turned)
        assert torch.equal(back_pe[has], turned[has])


def _step_args(b, h, int4):
    dt = torch.bfloat16
    z = lambda *shape, dtype=dt: torch.zeros(*shape, dtype=dtype, device="cuda")   # noqa: E731
    args = dict(q=z(b, h, 512), q_pe=z(b, h, 64), kv=z(b, 1, 512), k_pe=z(b, 1, 64), k_pe_cache=z(4, 64, 1, 64),
                block_table=z(b, 2, dtype=torch.int32) - 1, cache_seqlens=z(b, dtype=torch.int32),
                free_pages=torch.arange(4, dtype=torch.int32, device="cuda"), free_pos=z(1, dtype=torch.int32),
                out=z(b, h, 512))
    if int4:
        return dict(args, kv_cache=z(4, 64, 1, 256, dtype=torch.uint8), kv_scales=z(4, 64, 1, 16, dtype=torch.half))
    return dict(args, kv_cache=z(4, 64, 1, 512))


@pytest.mark.parametrize("int4", [False, True])
def test_first_call_inside_a_capture_is_refused(int4):
    """The workspace, the step's scratch and a rotary's frequencies are made (and given their
    first values) by an eager call; a capture that would make them is refused."""
    args = _step_args(2, 16, int4)
    k, rot = MlaPagedDecodeKernel(2, 16, 128), Rotary(64)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        args["out"].zero_()
        with pytest.raises(RuntimeError, match="before the capture"):
            k.step(**args)
        with pytest.raises(RuntimeError, match="before the capture"):
            rot(args["q_pe"], args["cache_seqlens"], args["q_pe"])
    graph.replay()
    assert args["cache_seqlens"].tolist() == [0, 0]
    k.step(**args, rotary=rot)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k.step(**args, rotary=rot)
    graph.replay()
    assert args["cache_seqlens"].tolist() == [2, 2]


@pytest.mark.parametrize("kernel", ["simt", "mma16", "mma32"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scores_of_short_sequences_are_exact_products(kernel, dtype):
    """Sequences of a few rows, where one score is the log-sum-exp: codes times scales are not
    rounded in the scores.  What is left: float32 sums of 576 products (off by at most 2^-23
    of the magnitudes' sum each, 2^-13 of it together at the very worst; a random walk of
    their roundings stays below 2^-20 of it), a float32 exponential and logarithm (1e-6)."""
    b, h, lens = 6, 16, [1, 2, 3, 5, 1, 8]
    q, qp, n, s, kp = _inputs(b, 1, h, 1, 8, dtype, seed=31)
    codes, scales, pe, _ = _caches(n, s, kp, lens, 0, seed=1)
    k = MlaPagedDecodeKernel(b, h, 8, cfg=KERNELS[kernel])
    qq, qpp = q.cuda().squeeze(1), qp.cuda().squeeze(1)
    out, lse = torch.empty_like(qq), torch.empty(b, h, device="cuda")
    k.decode_int4(qq, qpp, codes, scales, pe, torch.tensor(lens, dtype=torch.int32, device="cuda"), out, lse)
    for i, m in enumerate(lens):
        v = P.dequantise_int4(n[i], s[i])[:m, 0]
        qd, qpd, kd = (t.double().numpy() for t in (q[i, 0], qp[i, 0], kp[i, :m, 0]))
        _, ref, _, _ = P.decode(qd, qpd, v, kd, SCALE)
        sums = (np.abs(qd) @ np.abs(v).T + np.abs(qpd) @ np.abs(kd).T).max(-1) * SCALE
        err = np.abs(lse[i].double().cpu().numpy() - ref)
        assert (err <= 2.0 ** -20 * sums + 1e-6 * (1 + np.abs(ref))).all(), (i, err.max())


@pytest.mark.parametrize("kernel", ["mma16", "mma32"])
@pytest.mark.parametrize("b, h, q_len, smax", [(1, 16, 1, 300), (1, 1, 1, 512), (5, 40, 2, 512), (3, 100, 1, 513),
                                               (40, 16, 1, 500), (2, 48, 3, 129)])
def test_short_sequences_cut_over_ctas(kernel, b, h, q_len, smax):
    """Sequences of a few tiles, cut over CTAs and merged: call after call with other lengths,
    the same values each time."""
    q, qp, n, s, kp = _inputs(b, q_len, h, 1, smax, "fp16", seed=b + h)
    k = MlaPagedDecodeKernel(b, h, smax, cfg=KERNELS[kernel], q_len=q_len)
    qq, qpp = (t.cuda().squeeze(1) if q_len == 1 else t.cuda() for t in (q, qp))
    out, lse = torch.empty_like(qq), torch.empty(qq.shape[:-1], device="cuda")
    rng = np.random.default_rng(smax)
    for it in range(4):
        lens = [smax] * b if it == 0 else rng.integers(0, smax + 1, b).tolist()
        codes, scales, pe, table = _caches(n, s, kp, lens, 64, seed=it)
        sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        out.fill_(float("nan"))
        k.decode_int4(qq, qpp, codes, scales, pe, sl, out, lse, block_table=table)
        _check(out.view(b, q_len, h, 512), lse.view(b, q_len, h), q, qp, n, s, kp, lens, "fp16")
        first = out.clone()
        k.decode_int4(qq, qpp, codes, scales, pe, sl, out, block_table=table)
        assert torch.equal(out, first)
    assert k.device_status(torch.device("cuda"), torch.float16) == 0
