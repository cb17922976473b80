"""Workloads of the paged latent-cache operators, for measurement.

The operators: block tables and slots from request lengths, rotary positions, latent
rows written to and read back from a paged cache (16-bit, e4m3 or 4-bit), and decode
attention over a cache held in 4 bits.  ``run`` computes one pass in elementary torch
operations, or, with ``own`` set, through this repository's kernels; ``exact`` gives the
same outputs from the definitions in 64 bits.

A latent row is 512 values (keys and values at once) and a rope row 64.  The 4-bit form
of a latent row: 16 groups of 32 dims, each with a float16 scale s = half(max|x| / 7) and
codes n = clamp(rint(x / s), -8, 7) + 8, so that a dim stands for (n - 8) s; eight
consecutive dims d0..d7 share a 32-bit word whose nibbles, lowest first, are
d0 d2 d4 d6 d1 d3 d5 d7.
"""
import math

import torch

own = False

DIM, PE, GROUP = 512, 64, 32
SCALE = (DIM + PE) ** -0.5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
YARN = {"type": "yarn", "factor": 40.0, "original_max_position": 4096, "beta_fast": 32.0, "beta_slow": 1.0}
NIBBLE_DIM = (0, 2, 4, 6, 1, 3, 5, 7)   # dim (of eight) held by each nibble, lowest first


def listed():
    return [
        # a decode step of the serving batch: one new row per request
        {"name": "tables_step_b64", "op": "tables", "batch": 64, "max_len": 8192, "new": 1, "ragged": False,
         "page": 64},
        # prompts of up to 16384 tokens admitted together
        {"name": "tables_prompts_b132", "op": "tables", "batch": 132, "max_len": 16384, "new": 16384, "ragged": True,
         "page": 64},
        # the rope part of a decode step's queries
        {"name": "rotary_step_b64_h128", "op": "rotary", "tokens": 64, "heads": 128, "head_dim": 64, "offset": 0,
         "interleaved": True, "scaling": "none", "max_pos": 131072, "dtype": "bf16"},
        # a prompt chunk's query heads, 64 rope dims behind 128 others, scaled for long contexts
        {"name": "rotary_prompt_8192_h128", "op": "rotary", "tokens": 8192, "heads": 128, "head_dim": 192,
         "offset": 128, "interleaved": False, "scaling": "yarn", "max_pos": 131072, "dtype": "fp16"},
        # a decode step's new rows into the 4-bit cache
        {"name": "append_step_int4_b64", "op": "append", "tokens": 64, "form": "int4", "rotary": True, "page": 64,
         "dtype": "bf16"},
        # an odd prompt chunk into an e4m3 cache
        {"name": "append_5003_fp8", "op": "append", "tokens": 5003, "form": "fp8", "rotary": True, "page": 128,
         "dtype": "fp16"},
        # a long context's rows into the 4-bit cache and back
        {"name": "append_131072_int4", "op": "append", "tokens": 131072, "form": "int4", "rotary": True, "page": 64,
         "dtype": "bf16"},
        # the smallest call: one short sequence, sixteen heads
        {"name": "decode_b1_h16_s300", "op": "decode", "batch": 1, "q_len": 1, "heads": 16, "kv_heads": 1,
         "max_len": 300, "ragged": False, "page": 64, "dtype": "bf16"},
        # a few drafted tokens per sequence, odd head count and lengths
        {"name": "decode_b6_q3_h40_s3001", "op": "decode", "batch": 6, "q_len": 3, "heads": 40, "kv_heads": 1,
         "max_len": 3001, "ragged": True, "page": 192, "dtype": "fp16"},
        # heads split over eight GPUs: sixteen on each
        {"name": "decode_b128_h16_s4096", "op": "decode", "batch": 128, "q_len": 1, "heads": 16, "kv_heads": 1,
         "max_len": 4096, "ragged": False, "page": 64, "dtype": "bf16"},
        # one long context
        {"name": "decode_b1_h128_s131072", "op": "decode", "batch": 1, "q_len": 1, "heads": 128, "kv_heads": 1,
         "max_len": 131072, "ragged": False, "page": 0, "dtype": "bf16"},
        # the serving batch at full context
        {"name": "decode_b64_h128_s8192", "op": "decode", "batch": 64, "q_len": 1, "heads": 128, "kv_heads": 1,
         "max_len": 8192, "ragged": False, "page": 64, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "rotary", "append", "decode", "decode"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "tables":
        return {"op": op, "batch": _log(rng, 1, 132), "max_len": _log(rng, 64, 16384), "new": _log(rng, 1, 8192),
                "ragged": rng.random() < 0.7, "page": 64 * rng.randint(1, 4)}
    if op == "rotary":
        head_dim = rng.choice([64, 128, 192])
        return {"op": op, "tokens": _log(rng, 1, 4096), "heads": rng.randint(1, 128), "head_dim": head_dim,
                "offset": rng.choice([0, head_dim - 64]), "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "max_pos": _log(rng, 1000, 1000000),
                "dtype": dtype}
    if op == "append":
        return {"op": op, "tokens": _log(rng, 1, 65536), "form": rng.choice(["model", "fp8", "int4", "int4"]),
                "rotary": rng.random() < 0.7, "page": 64 * rng.randint(1, 4), "dtype": dtype}
    batch, q_len = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 3])
    heads = rng.choice([1, 8, 16, 24, 32, 40, 64, 96, 128])
    kv_heads = 2 if heads % 2 == 0 and rng.random() < 0.15 else 1
    # at most a third of the work of the largest listed case
    longest = 64 * 8192 * 128 // (3 * batch * q_len * max(heads, 32))
    return {"op": op, "batch": batch, "q_len": q_len, "heads": heads, "kv_heads": kv_heads,
            "max_len": _log(rng, 8, max(16, min(65536, longest))), "ragged": rng.random() < 0.7,
            "page": 64 * rng.randint(0, 4), "dtype": dtype}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)


def _ceil(a, b):
    return -(-a // b)


def _pack(n):
    """Codes 0..15 [..., 512] -> bytes [..., 256]."""
    n = n.reshape(*n.shape[:-1], DIM // 8, 8)[..., list(NIBBLE_DIM)].to(torch.uint8)
    n = n.reshape(*n.shape[:-1], 4, 2)
    return (n[..., 0] | (n[..., 1] << 4)).reshape(*n.shape[:-3], DIM // 2)


def _quantise(x):
    """Rows [..., 512] -> (codes 0..15 [..., 512], scales float16 [..., 16]), in 32 bits."""
    g = x.float().reshape(*x.shape[:-1], DIM // GROUP, GROUP)
    s = (g.abs().amax(-1) / 7.0).to(torch.float16)
    sf = s.float().unsqueeze(-1)
    n = torch.where(sf > 0, torch.round(g / torch.where(sf > 0, sf, 1.0)), torch.zeros_like(g)).clamp(-8, 7) + 8
    return n.reshape(x.shape), s


def _dequantise(codes, scales):
    """Bytes [..., 256] and scales [..., 16] -> float32 rows [..., 512]."""
    n = torch.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], DIM // 8, 8)
    order = [NIBBLE_DIM.index(d) for d in range(8)]
    n = n[..., order].reshape(*codes.shape[:-1], DIM // GROUP, GROUP).float() - 8.0
    return (n * scales.float().unsqueeze(-1)).reshape(*codes.shape[:-1], DIM)


def _scaling(case):
    return {"none": None, "linear": {"type": "linear", "factor": 8.0}, "ntk": {"type": "ntk", "factor": 8.0},
            "yarn": YARN}[case["scaling"]]


def _tables_inputs(case, seed):
    g = _gen(seed)
    b, page = case["batch"], case["page"]
    total = _ceil(case["max_len"] + case["new"], page) * page
    lens = _randint(g, 0, case["max_len"] + 1, b)
    # ragged: evenly spread counts in a random order, their rows padded to a fixed token budget
    new = torch.full_like(lens, case["new"])
    if case["ragged"]:
        order = torch.randperm(b, generator=g, device="cuda").to(torch.int32)
        new = ((order + 1) * case["new"] // b).clamp(min=1)
    max_pages = total // page
    ids = torch.randperm(b * max_pages, generator=g, device="cuda").to(torch.int32)
    held = (lens + page - 1) // page
    table = ids.reshape(b, max_pages).clone()
    keep = torch.arange(max_pages, device="cuda") < held.unsqueeze(1)
    free = table[~keep]
    table[~keep] = -1
    return {"table": table, "lens": lens, "new": new, "free": free, "page": page, "pages": b * max_pages,
            "tokens": _ceil(int(new.sum()), 128) * 128 if case["ragged"] else int(new.sum())}


def _rotary_inputs(case, seed):
    g = _gen(seed)
    x = _randn(g, case["tokens"], case["heads"], case["head_dim"]).to(DTYPES[case["dtype"]])
    return {"x": x, "pos": _randint(g, 0, case["max_pos"], case["tokens"])}


def _append_inputs(case, seed):
    g = _gen(seed)
    n, dt = case["tokens"], DTYPES[case["dtype"]]
    kv, pe = _randn(g, n, 1, DIM).to(dt), _randn(g, n, 1, PE).to(dt)
    pages = _ceil(n, case["page"]) + 1
    slots = torch.randperm(pages, generator=g, device="cuda").unsqueeze(1) * case["page"] \
        + torch.arange(case["page"], device="cuda")
    return {"kv": kv, "pe": pe, "slots": slots.reshape(-1)[:n].to(torch.int32).contiguous(), "pages": pages,
            "pos": _randint(g, 0, 131072, n)}


def _decode_inputs(case, seed):
    g = _gen(seed)
    b, h, kvh, page, dt = case["batch"], case["heads"], case["kv_heads"], case["page"], DTYPES[case["dtype"]]
    smax = max(case["max_len"], case["q_len"])
    q = _randn(g, b, case["q_len"], h, DIM).to(dt)
    q_pe = _randn(g, b, case["q_len"], h, PE).to(dt)
    lens = _randint(g, case["q_len"], smax + 1, b) if case["ragged"] else \
        torch.full((b,), smax, dtype=torch.int32, device="cuda")
    if page:
        per = _ceil(smax, page)
        lead = (b * per, page)
        table = torch.randperm(b * per, generator=g, device="cuda").to(torch.int32).reshape(b, per)
    else:
        lead, table = (b, smax), None
    codes = torch.empty(*lead, kvh, DIM // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(*lead, kvh, DIM // GROUP, dtype=torch.float16, device="cuda")
    step = max(1, (1 << 17) // (lead[1] * kvh))
    for i in range(0, lead[0], step):
        m = min(step, lead[0] - i)
        n, s = _quantise(_randn(g, m, lead[1], kvh, DIM))
        codes[i:i + m], scales[i:i + m] = _pack(n), s
    pe = _randn(g, *lead, kvh, PE).to(dt)
    return {"q": q, "q_pe": q_pe, "codes": codes, "scales": scales, "pe": pe, "lens": lens, "table": table,
            "smax": smax}


_INPUTS = {"tables": _tables_inputs, "rotary": _rotary_inputs, "append": _append_inputs, "decode": _decode_inputs}


def prepare(case, seed):
    st = _INPUTS[case["op"]](case, seed)
    st["case"] = case
    if case["op"] == "decode":
        ql = case["q_len"]
        if ql == 1:
            st["q"], st["q_pe"] = st["q"].squeeze(1), st["q_pe"].squeeze(1)
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty(st["q"].shape[:-1], dtype=torch.float32, device="cuda")
        st["host_lens"] = st["lens"].tolist()
        if own:
            from mlc_decode_b200 import MlaPagedDecodeKernel
            st["kernel"] = MlaPagedDecodeKernel(case["batch"], case["heads"], st["smax"], q_len=ql,
                                                kv_heads=case["kv_heads"])
    elif case["op"] == "append":
        form, n, dt = case["form"], st["pages"] * case["page"], DTYPES[case["dtype"]]
        lead = (st["pages"], case["page"], 1)
        if form == "int4":
            st["cache"] = torch.zeros(*lead, DIM // 2, dtype=torch.uint8, device="cuda")
            st["scales"] = torch.zeros(*lead, DIM // GROUP, dtype=torch.float16, device="cuda")
        else:
            st["cache"] = torch.zeros(*lead, DIM, dtype=torch.float8_e4m3fn if form == "fp8" else dt, device="cuda")
            st["scales"] = None
        st["scale"] = 1.0 / 32.0 if form == "fp8" else None
        st["pe_cache"] = torch.zeros(*lead, PE, dtype=dt, device="cuda")
        st["kv_back"], st["pe_back"] = torch.empty_like(st["kv"]), torch.empty_like(st["pe"])
    elif case["op"] == "rotary":
        st["out"] = torch.empty_like(st["x"])
    else:
        n = st["tokens"]
        st["slots"] = torch.empty(n, dtype=torch.int32, device="cuda")
        st["positions"] = torch.empty(n, dtype=torch.int32, device="cuda")
        st["new_lens"] = torch.empty_like(st["lens"])
        st["cu"] = torch.empty(case["batch"] + 1, dtype=torch.int32, device="cuda")
        st["free_pos"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        st["new_free_pos"] = torch.empty(1, dtype=torch.int32, device="cuda")
    if case["op"] == "rotary" or (case["op"] == "append" and case["rotary"]):
        rotary = case["op"] == "rotary"
        st["freq"], st["gain"] = _frequencies(_scaling(case) if rotary else None, "cuda")
        if own:
            from mlc_decode_b200 import Rotary
            st["rotary"] = Rotary(PE, base=10000.0, interleaved=case["interleaved"] if rotary else True,
                                  scaling=_scaling(case) if rotary else None)
    else:
        st["rotary"] = None
    return st


# ---------------------------------------------------------------- the plain forms
def _frequencies(scaling, device, base=10000.0):
    """Angle per position of the 32 rotated pairs (64 bits), and the factor on cos and sin."""
    i = torch.arange(PE // 2, dtype=torch.float64, device=device)
    kind = None if scaling is None else scaling["type"]
    if kind == "ntk":
        base = base * scaling["factor"] ** (PE / (PE - 2))
    freq = base ** (-2.0 * i / PE)
    if kind == "linear":
        freq = freq / scaling["factor"]
    if kind != "yarn":
        return freq, 1.0

    def turn_dim(turns):
        return PE * math.log(scaling["original_max_position"] / (turns * 2 * math.pi)) / (2 * math.log(base))

    low = max(math.floor(turn_dim(scaling["beta_fast"])), 0)
    high = min(math.ceil(turn_dim(scaling["beta_slow"])), PE - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return freq / scaling["factor"] * ramp + freq * (1 - ramp), 0.1 * math.log(scaling["factor"]) + 1.0


def _rotate(x, pos, freq, gain, interleaved):
    """x [tokens, heads, 64] rotated, in x's type: angles in 64 bits, the rest in 32."""
    angle = pos.double().unsqueeze(1) * freq
    c, s = (torch.cos(angle) * gain).float().unsqueeze(1), (torch.sin(angle) * gain).float().unsqueeze(1)
    xf = x.float()
    a, b = (xf[..., 0::2], xf[..., 1::2]) if interleaved else (xf[..., :PE // 2], xf[..., PE // 2:])
    ra, rb = a * c - b * s, a * s + b * c
    return (torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)).to(x.dtype)


def _plain_tables(st):
    table, page, n = st["table"], st["page"], st["tokens"]
    b, max_pages = table.shape
    lens, new = st["lens"].long(), st["new"].long()
    held = (lens + page - 1) // page
    need = (lens + new + page - 1) // page - held
    first = st["free_pos"].long() + need.cumsum(0) - need
    cu = torch.cat((torch.zeros_like(new[:1]), new.cumsum(0)))
    col = torch.arange(max_pages, device=table.device).unsqueeze(0)
    fresh = (col >= held.unsqueeze(1)) & (col < (held + need).unsqueeze(1))
    src = (first.unsqueeze(1) + col - held.unsqueeze(1)).clamp(0, max(st["free"].numel() - 1, 0))
    table.copy_(torch.where(fresh, st["free"][src] if st["free"].numel() else src.int(), table))
    k = torch.arange(n, device=table.device)
    real = k < cu[-1]
    req = (torch.searchsorted(cu, k, right=True) - 1).clamp(max=b - 1)
    pos = torch.where(real, lens[req] + k - cu[req], 0)
    slot = torch.where(real, table[req, pos // page].long() * page + pos % page, -1)
    return {"table": table, "slots": slot.int(), "positions": pos.int(), "lens": (lens + new).int(), "cu": cu.int(),
            "free_pos": (st["free_pos"] + need.sum()).int()}


def _plain_rotary(st):
    case, x = st["case"], st["x"]
    o = case["offset"]
    out = x.clone()
    out[..., o:o + PE] = _rotate(x[..., o:o + PE], st["pos"], st["freq"], st["gain"], case["interleaved"])
    return out


def _plain_append(st):
    case, kv, slots = st["case"], st["kv"], st["slots"].long()
    cache, pe_cache = st["cache"].flatten(0, 1), st["pe_cache"].flatten(0, 1)
    pe = _rotate(st["pe"], st["pos"], st["freq"], st["gain"], True) if case["rotary"] else st["pe"]
    pe_cache[slots] = pe
    if case["form"] == "int4":
        scales = st["scales"].flatten(0, 1)
        n, s = _quantise(kv)
        cache[slots], scales[slots] = _pack(n), s
        back = _dequantise(cache[slots], scales[slots]).to(kv.dtype)
    elif case["form"] == "fp8":
        bytes_ = cache.view(torch.uint8)
        bytes_[slots] = (kv.float() / st["scale"]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        back = (bytes_[slots].view(torch.float8_e4m3fn).float() * st["scale"]).to(kv.dtype)
    else:
        cache[slots] = kv
        back = cache[slots]
    return {"kv": back, "pe": pe_cache[slots]}


def _plain_decode(st):
    case = st["case"]
    b, ql, h, kvh, page = case["batch"], case["q_len"], case["heads"], case["kv_heads"], case["page"]
    g = h // kvh
    q, q_pe = st["q"].reshape(b, ql, kvh, g, DIM), st["q_pe"].reshape(b, ql, kvh, g, PE)
    out, lse = st["out"].view(b, ql, kvh, g, DIM), st["lse"].view(b, ql, kvh, g)
    for i, n in enumerate(st["host_lens"]):
        if page:
            ids = st["table"][i, :_ceil(n, page)].long()
            codes, scales, pe = (st[k][ids].flatten(0, 1)[:n] for k in ("codes", "scales", "pe"))
        else:
            codes, scales, pe = (st[k][i, :n] for k in ("codes", "scales", "pe"))
        v = _dequantise(codes, scales).transpose(0, 1)                # [kvh, n, 512]
        k = torch.cat((v, pe.float().transpose(0, 1)), -1)
        qq = torch.cat((q[i].float(), q_pe[i].float()), -1).transpose(0, 1).reshape(kvh, ql * g, DIM + PE)
        s = torch.matmul(qq, k.transpose(1, 2)).view(kvh, ql, g, n) * SCALE
        seen = n - ql + 1 + torch.arange(ql, device=s.device)         # rows each position attends to
        s = torch.where(torch.arange(n, device=s.device) < seen.view(1, ql, 1, 1), s, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - top)
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p.view(kvh, ql * g, n), v).view(kvh, ql, g, DIM) / total
        out[i].copy_(o.transpose(0, 1))
        lse[i].copy_((top + torch.log(total)).squeeze(-1).transpose(0, 1))
    return {"out": st["out"], "lse": st["lse"]}


_PLAIN = {"tables": _plain_tables, "rotary": _plain_rotary, "append": _plain_append, "decode": _plain_decode}


# ---------------------------------------------------------------- this repository's kernels
def _own_tables(st):
    from mlc_decode_b200 import extend_block_tables
    extend_block_tables(st["table"], st["lens"], st["new"], st["free"], st["free_pos"], st["new_lens"],
                        st["new_free_pos"], st["slots"], st["positions"], page_size=st["page"],
                        num_pages=st["pages"], cu_new=st["cu"])
    return {"table": st["table"], "slots": st["slots"], "positions": st["positions"], "lens": st["new_lens"],
            "cu": st["cu"], "free_pos": st["new_free_pos"]}


def _own_rotary(st):
    st["rotary"](st["x"], st["pos"], st["out"], offset=st["case"]["offset"])
    return st["out"]


def _own_append(st):
    from mlc_decode_b200 import cache_append, cache_gather
    cache_append(st["kv"], st["pe"], st["slots"], st["cache"], st["pe_cache"], kv_scale=st["scale"],
                 kv_scales=st["scales"], rotary=st["rotary"], positions=st["pos"] if st["rotary"] else None)
    cache_gather(st["slots"], st["cache"], st["pe_cache"], st["kv_back"], st["pe_back"], kv_scale=st["scale"],
                 kv_scales=st["scales"])
    return {"kv": st["kv_back"], "pe": st["pe_back"]}


def _own_decode(st):
    st["kernel"].decode_int4(st["q"], st["q_pe"], st["codes"], st["scales"], st["pe"], st["lens"], st["out"],
                             st["lse"], block_table=st["table"])
    return {"out": st["out"], "lse": st["lse"]}


_OWN = {"tables": _own_tables, "rotary": _own_rotary, "append": _own_append, "decode": _own_decode}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ---------------------------------------------------------------- the work of a pass
def work(case):
    op = case["op"]
    if op == "tables":
        b, per = case["batch"], ((case["new"] + 1) / 2 if case["ragged"] else case["new"])
        tokens = b * per
        # lengths read and written, a slot and a position per token, page ids read and written
        return {"bytes": 20 * b + 8 * tokens + 8 * b * (per / case["page"]), "flops": 0}
    if op == "rotary":
        n = case["tokens"] * case["heads"]
        return {"bytes": 4 * n * case["head_dim"] + 4 * case["tokens"], "flops": 3 * n * PE}
    if op == "append":
        row = {"model": 2 * DIM, "fp8": DIM, "int4": DIM // 2 + 2 * DIM // GROUP}[case["form"]] + 2 * PE
        # rows in, cache rows written, rows back
        return {"bytes": case["tokens"] * (2 * 2 * (DIM + PE) + row + 8), "flops": 2 * case["tokens"] * DIM}
    b, ql, h = case["batch"], case["q_len"], case["heads"]
    rows = b * ((case["max_len"] + ql) / 2 if case["ragged"] else max(case["max_len"], ql))
    cache = rows * case["kv_heads"] * (DIM // 2 + 2 * DIM // GROUP + 2 * PE)
    return {"bytes": cache + b * ql * h * (2 * (DIM + PE) + 2 * DIM + 4),
            "flops": 2.0 * rows * ql * h * (2 * DIM + PE)}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_tables(case, seed):
    st = _tables_inputs(case, seed)
    table, lens, new = st["table"].tolist(), st["lens"].tolist(), st["new"].tolist()
    free, page, taken = st["free"].tolist(), st["page"], 0
    slots, positions, cu = [], [], [0]
    for i, (length, count) in enumerate(zip(lens, new)):
        for k in range(_ceil(length, page), _ceil(length + count, page)):
            table[i][k] = free[taken]
            taken += 1
        for p in range(length, length + count):
            positions.append(p)
            slots.append(table[i][p // page] * page + p % page)
        cu.append(cu[-1] + count)
    slots += [-1] * (st["tokens"] - cu[-1])
    positions += [0] * (st["tokens"] - cu[-1])

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    return {"table": ints(table), "slots": ints(slots), "positions": ints(positions),
            "lens": ints([a + c for a, c in zip(lens, new)]), "cu": ints(cu), "free_pos": ints([taken])}


def _exact_turn(x, pos, scaling, interleaved):
    """The rotation of x's 64 dims as complex numbers, pair i by pos * frequency i."""
    f, d = [], PE
    factor = 1.0 if scaling is None else scaling["factor"]
    kind = "none" if scaling is None else scaling["type"]
    theta = 10000.0 * (factor ** (d / (d - 2.0)) if kind == "ntk" else 1.0)
    for i in range(d // 2):
        w = math.exp(-2.0 * i / d * math.log(theta))
        if kind == "linear":
            w /= factor
        elif kind == "yarn":
            edges = [d / 2.0 * math.log(scaling["original_max_position"] / (2 * math.pi * scaling[e])) / math.log(theta)
                     for e in ("beta_fast", "beta_slow")]
            lo, hi = max(math.floor(edges[0]), 0), min(math.ceil(edges[1]), d - 1)
            t = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            w = w * (1.0 - t) + w * t / factor
        f.append(w)
    gain = 1.0 + 0.1 * math.log(factor) if kind == "yarn" else 1.0
    phase = torch.outer(pos.double(), torch.tensor(f, dtype=torch.float64, device=x.device))
    turn = torch.polar(torch.full_like(phase, gain), phase).unsqueeze(1)
    xd = x.double()
    pairs = xd.unflatten(-1, (d // 2, 2)) if interleaved else xd.unflatten(-1, (2, d // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.complex(pairs[..., 0].contiguous(), pairs[..., 1].contiguous()) * turn)
    return z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)


def _exact_rotary(case, seed):
    st, o = _rotary_inputs(case, seed), case["offset"]
    x = st["x"].double()
    x[..., o:o + PE] = _exact_turn(st["x"][..., o:o + PE], st["pos"], _scaling(case), case["interleaved"])
    return x


def _exact_append(case, seed):
    st = _append_inputs(case, seed)
    kv = st["kv"].double()
    if case["form"] == "int4":
        groups = kv.unflatten(-1, (DIM // GROUP, GROUP))
        s = (groups.abs().amax(-1, keepdim=True) / 7).to(torch.float16).double()
        kv = (torch.clamp(torch.round(groups / s), -8, 7) * s).nan_to_num(0.0).flatten(-2)
    elif case["form"] == "fp8":
        kv = torch.clamp(kv * 32, -448, 448).to(torch.float8_e4m3fn).double() / 32
    pe = _exact_turn(st["pe"], st["pos"], None, True) if case["rotary"] else st["pe"].double()
    return {"kv": kv, "pe": pe}


def _exact_decode(case, seed):
    st = _decode_inputs(case, seed)
    b, ql, h, kvh, page = case["batch"], case["q_len"], case["heads"], case["kv_heads"], case["page"]
    q = torch.cat((st["q"], st["q_pe"]), -1).double()
    out = torch.empty(b, ql, h, DIM, dtype=torch.float64, device="cuda")
    lse = torch.empty(b, ql, h, dtype=torch.float64, device="cuda")
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device="cuda")   # of dims d0..d7 in their word
    for i, n in enumerate(st["lens"].tolist()):
        r = torch.arange(n, device="cuda")
        row = (st["table"][i].long()[r // page] * page + r % page) if page else i * st["smax"] + r
        words = st["codes"].flatten(0, 1)[row].view(torch.int32).long()          # [n, kvh, 64]
        code = ((words.unsqueeze(-1) >> shift) & 15).flatten(-2) - 8
        scale = st["scales"].flatten(0, 1)[row].double().repeat_interleave(GROUP, -1)
        v = code.double() * scale
        k = torch.cat((v, st["pe"].flatten(0, 1)[row].double()), -1)
        for t in range(ql):
            m = n - (ql - 1 - t)
            for j in range(kvh):
                heads = slice(j * h // kvh, (j + 1) * h // kvh)
                s = q[i, t, heads] @ k[:m, j].T * SCALE
                lse[i, t, heads] = torch.logsumexp(s, -1)
                out[i, t, heads] = torch.softmax(s, -1) @ v[:m, j]
    if ql == 1:
        out, lse = out.squeeze(1), lse.squeeze(1)
    return {"out": out, "lse": lse}


def exact(case, seed):
    return {"tables": _exact_tables, "rotary": _exact_rotary, "append": _exact_append,
            "decode": _exact_decode}[case["op"]](case, seed)
