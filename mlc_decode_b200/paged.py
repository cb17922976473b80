"""The paged latent cache around a decode call: block tables and slots from request
lengths, rotary positions, and latent rows into and out of the cache.

Everything is enqueued on the current stream of the tensors' device, allocates at most
small temporaries, never synchronises the host and can be captured into a CUDA graph.
No counterpart in the reference, whose cache is one contiguous tensor per call and whose
inputs come rotated (baseline_mla.py:167-191).  C entry points: mla_extend_block_tables,
mla_rotary, mla_cache_append, mla_cache_gather (include/mla_decode_b200.h).
"""
from __future__ import annotations

import math
import threading

import torch

from . import capi
from .decode import _DTYPES, _FP8, DIM, PE_DIM, _check_tensor, _fits, _not_capturing, _on_device

INT4_GROUP = 32                      # dims per scale of the 4-bit form
INT4_GROUPS = DIM // INT4_GROUP      # scales per row
INT4_BYTES = DIM // 2                # code bytes per row

_ROTARY_DTYPES = {**_DTYPES, torch.float32: capi.MLA_DTYPE_F32}


def extend_block_tables(block_table, cache_seqlens, new_lens, free_pages, free_pos, new_seqlens, new_free_pos, slots,
                        positions, page_size, num_pages, cu_new=None, q_len=0, whole=False):
    """Give every request ``new_lens[i]`` more cache rows (mla_extend_block_tables).

    All tensors int32 on one device.  ``block_table`` [batch, max_pages] is extended in
    place with page ids taken from ``free_pages[free_pos[0]:]`` in request order;
    ``cache_seqlens`` [batch] are the rows held.  Written: ``new_seqlens`` [batch] (rows held
    afterwards; fewer than asked for when the table row or the free list is full),
    ``new_free_pos`` [1], ``slots`` [num_tokens] (cache row of every new row, -1 where there is
    none), ``positions`` [num_tokens] (index in its sequence) and ``cu_new`` [batch + 1]
    (first new row of every request; optional).  New rows are packed, request after request,
    or, with ``q_len``, the last rows of each request's q_len.  ``whole`` (with ``q_len``
    only): a request gets all of its rows or none, as a decode over them needs it (its causal
    rule counts back from the last row); from the first one on that does not find its pages
    nobody gets new pages (mla_extend_block_tables_whole).  ``new_seqlens`` may be
    ``cache_seqlens`` and ``new_free_pos`` may be ``free_pos``; nothing else may overlap.
    """
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise ValueError("block_table must be an int32 tensor [batch, max_pages]")
    b, max_pages = block_table.shape
    dev = block_table.device
    i32, index = torch.int32, dev.index
    # all at once; one by one, with names, only if something is wrong
    if not (type(cache_seqlens) is type(new_lens) is type(free_pages) is type(free_pos) is type(new_seqlens)
            is type(new_free_pos) is type(slots) is type(positions) is torch.Tensor and dev.type == "cuda"
            and block_table.dtype is cache_seqlens.dtype is new_lens.dtype is free_pages.dtype is free_pos.dtype
            is new_seqlens.dtype is new_free_pos.dtype is slots.dtype is positions.dtype is i32
            and cache_seqlens.shape == new_lens.shape == new_seqlens.shape == (b,)
            and free_pos.shape == new_free_pos.shape == (1,) and slots.shape == positions.shape
            and slots.dim() == free_pages.dim() == 1
            and cache_seqlens.get_device() == new_lens.get_device() == free_pages.get_device()
            == free_pos.get_device() == new_seqlens.get_device() == new_free_pos.get_device() == slots.get_device()
            == positions.get_device() == index
            and block_table.is_contiguous() and cache_seqlens.is_contiguous() and new_lens.is_contiguous()
            and free_pages.is_contiguous() and free_pos.is_contiguous() and new_seqlens.is_contiguous()
            and new_free_pos.is_contiguous() and slots.is_contiguous() and positions.is_contiguous()
            and (cu_new is None or _fits(cu_new, (b + 1,), i32, index))):
        _check_tensor("block_table", block_table, (b, max_pages), i32, None)
        n, nf = (t.numel() if isinstance(t, torch.Tensor) else -1 for t in (slots, free_pages))
        for name, t, k in (("cache_seqlens", cache_seqlens, b), ("new_lens", new_lens, b),
                           ("free_pages", free_pages, nf), ("free_pos", free_pos, 1),
                           ("new_seqlens", new_seqlens, b), ("new_free_pos", new_free_pos, 1), ("slots", slots, n),
                           ("positions", positions, n), ("cu_new", cu_new, b + 1)):
            if t is not None or name != "cu_new":
                _check_tensor(name, t, (k,), i32, dev)
    n, nf = slots.numel(), free_pages.numel()
    nbytes = capi.block_tables_workspace_bytes(b, n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    call = capi.extend_block_tables_whole if whole else capi.extend_block_tables
    _on_device(dev, call, block_table.data_ptr(), cache_seqlens.data_ptr(), new_lens.data_ptr(),
               free_pages.data_ptr(), free_pos.data_ptr(), new_seqlens.data_ptr(), new_free_pos.data_ptr(),
               slots.data_ptr(), positions.data_ptr(), None if cu_new is None else cu_new.data_ptr(),
               None if ws is None else ws.data_ptr(), nbytes, b, max_pages, int(page_size), int(num_pages), nf, n,
               int(q_len))


def rotary_frequencies(rot_dim, base=10000.0, scaling=None):
    """(angles per position of the rot_dim / 2 pairs, gain on cos and sin) in 64 bits.

    Unscaled: base ** (-2 i / rot_dim), gain 1.  ``scaling`` (a dict) stretches them for
    contexts longer than the trained one:
      {"type": "linear", "factor": f}   every frequency / f
      {"type": "ntk", "factor": f}      base * f ** (rot_dim / (rot_dim - 2))
      {"type": "yarn", "factor": f, "original_max_position": n, "beta_fast": 32, "beta_slow": 1,
       "gain": ...}                     pairs that turn more than beta_fast times in n positions
                                        stay, those below beta_slow turns are / f, a linear ramp
                                        between them; gain defaults to 0.1 ln f + 1
    """
    if rot_dim < 2 or rot_dim % 2 or not base > 1.0 or not math.isfinite(base):
        raise ValueError(f"rot_dim must be even and >= 2 and base finite and > 1 (got {rot_dim}, {base})")
    s = dict(scaling or {})
    kind = s.get("type")
    if kind not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown rotary scaling {kind!r}")
    known = {None: set(), "linear": {"factor"}, "ntk": {"factor"},
             "yarn": {"factor", "original_max_position", "beta_fast", "beta_slow", "gain"}}[kind]
    if set(s) - known - {"type"}:
        raise ValueError(f"unknown rotary scaling parameters {sorted(set(s) - known - {'type'})}")
    factor = float(s.get("factor", 1.0))
    if not factor >= 1.0 or not math.isfinite(factor):
        raise ValueError(f"rotary scaling factor must be finite and >= 1, got {factor}")
    if kind == "ntk":
        if rot_dim == 2:
            raise ValueError("ntk scaling needs rot_dim > 2")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freq = [base ** (-2.0 * i / rot_dim) for i in range(rot_dim // 2)]
    if kind == "linear":
        return [f / factor for f in freq], 1.0
    if kind != "yarn":
        return freq, 1.0
    trained = float(s.get("original_max_position", 0))
    fast, slow = float(s.get("beta_fast", 32.0)), float(s.get("beta_slow", 1.0))
    if not trained >= 1 or not fast >= slow > 0:
        raise ValueError("yarn needs original_max_position >= 1 and beta_fast >= beta_slow > 0")

    def pair_of(turns):   # the (fractional) pair that makes `turns` turns in the trained context
        return rot_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rot_dim - 1)
    out = []
    for i, f in enumerate(freq):
        ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
        out.append(f * (1.0 - ramp) + f / factor * ramp)
    return out, float(s.get("gain", 0.1 * math.log(factor) + 1.0))


class Rotary:
    """Rotary positions of ``rot_dim`` dims of every head (mla_rotary).

    ``rot(x, positions, out, offset=0)``: x, out [tokens, heads, head_dim] in float16,
    bfloat16 or float32 (any token and head strides, last dim contiguous), positions int32
    [tokens]; dims [offset, offset + rot_dim) turn, the others are copied; out may be x, or have no
    element in common with it (slices of one buffer with the same strides will do).
    ``interleaved``: pairs are dims (2 i, 2 i + 1), else (i, i + rot_dim / 2).  ``scaling``: see
    ``rotary_frequencies``.  The frequencies are uploaded by the first call on a device (make
    it, or ``rot.turns(device)``, before a graph capture: a capture refuses).
    """

    def __init__(self, rot_dim=PE_DIM, base=10000.0, interleaved=True, scaling=None):
        self.rot_dim, self.base, self.interleaved = int(rot_dim), float(base), bool(interleaved)
        self.scaling = dict(scaling) if scaling else None
        freq, self.gain = rotary_frequencies(self.rot_dim, self.base, self.scaling)
        if self.rot_dim > 1024:
            raise ValueError(f"rot_dim must be at most 1024, got {rot_dim}")
        if not math.isfinite(self.gain):
            raise ValueError(f"gain must be finite, got {self.gain}")
        self._turns = [f / (2 * math.pi) for f in freq]
        self._dev = {}
        self._lock = threading.Lock()
        capi.load()

    def turns(self, device):
        """Turns per position of every pair, float64 on ``device`` (kept)."""
        t = self._dev.get(device)
        if t is not None:
            return t
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        t = self._dev.get(device)
        if t is None:
            with self._lock:
                t = self._dev.get(device)
                if t is None:
                    _not_capturing("the frequencies' copy")
                    t = self._dev[device] = torch.tensor(self._turns, dtype=torch.float64, device=device)
        return t

    def __call__(self, x, positions, out, offset=0):
        if not isinstance(x, torch.Tensor) or x.dim() != 3 or x.dtype not in _ROTARY_DTYPES:
            raise ValueError("x must be a float16, bfloat16 or float32 tensor [tokens, heads, head_dim]")
        n, h, d = shape = x.shape
        if not 0 <= int(offset) <= d - self.rot_dim:
            raise ValueError(f"dims [{offset}, {offset} + {self.rot_dim}) must lie inside the head's {d}")
        dev, dtype = x.device, x.dtype
        index = dev.index
        dense = _fits(x, shape, dtype, index)
        if not dense:
            _check_rows("x", x, shape, dtype, None)
        if not _fits(out, shape, dtype, index):
            dense = False
            _check_rows("out", out, shape, dtype, dev, written=True)
        if not _fits(positions, (n,), torch.int32, index):
            _check_tensor("positions", positions, (n,), torch.int32, dev)
        if n == 0:
            return
        xp, op = x.data_ptr(), out.data_ptr()
        if dense:     # the same strides; apart if the starts are a whole tensor apart
            xs = os_ = (h * d, d)
            meet = xp != op and abs(xp - op) < n * h * d * dtype.itemsize
        else:
            xs, os_ = _strides(x), _strides(out)
            meet = xs != os_ if xp == op else _share_elements(x, out)
        if meet:
            raise ValueError("out must be x itself or must not overlap it")
        _on_device(dev, capi.rotary, xp, op, positions.data_ptr(), self.turns(dev).data_ptr(), self.gain, n, h, d,
                   self.rot_dim, int(offset), self.interleaved, xs[0], xs[1], os_[0], os_[1], _ROTARY_DTYPES[dtype])


def _strides(t):
    """Token and head stride; of a dimension of one entry any stride will do."""
    (n, h, _), (sn, sh, _) = t.shape, t.stride()
    return sn if n > 1 else 0, sh if h > 1 else 0


def _share_elements(a, b):
    """Whether two 3-D tensors of one shape and type (last dim contiguous) have an element in
    common.  Exact where their strides are the same, as those of slices of one buffer are; True
    where it would take more to tell."""
    apart = (b.data_ptr() - a.data_ptr()) // a.element_size()
    dims = sorted(((sa, sb, n) for sa, sb, n in zip(a.stride()[:2], b.stride()[:2], a.shape[:2]) if n > 1), reverse=True)

    def meet(apart, dims):       # rows of a from 0, of b from `apart`
        ends = [sum((n - 1) * d[k] for *d, n in dims) + a.shape[2] for k in (0, 1)]
        if apart >= ends[0] or -apart >= ends[1]:
            return False
        if not dims:
            return True
        (sa, sb, n), inner = dims[0], dims[1:]
        if sa != sb or sa == 0:
            return True
        # entries i apart along the outermost dim whose inner extents overlap
        ends = [e - (n - 1) * sa for e in ends]
        low, high = max(-((apart + ends[1] - 1) // sa), 1 - n), min((ends[0] - 1 - apart) // sa, n - 1)
        return high - low > 16 or any(meet(apart + i * sa, inner) for i in range(low, high + 1))

    return meet(apart, dims)


def _check_rows(name, t, shape, dtype, device, written=False, align=1):
    """A 3-D CUDA tensor with contiguous last dim; its rows start on ``align`` elements, and
    do not overlap one another when they are written."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor (got {t.device})")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.numel() == 0:
        return
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    if align > 1:
        bad = [s for d, s in enumerate(t.stride()[:2]) if t.shape[d] > 1 and s % align]
        if bad or t.data_ptr() % (align * t.element_size()):
            raise ValueError(f"{name}: every row must start on a {align * t.element_size()}-byte boundary")
    if written:
        need = t.shape[2]
        for s, size in sorted((t.stride(d), t.shape[d]) for d in (0, 1) if t.shape[d] > 1):
            if s < need:
                raise ValueError(f"{name}: rows overlap (strides {t.stride()})")
            need = s * (size - 1) + need


def _check_cache(kv_cache, k_pe_cache, kv_scale, kv_scales, dtype, device):
    """(form, rows, kv_heads) of a cache [a, b, kv_heads, width] in any of its forms."""
    def need(name, t, shape, want):
        if not _fits(t, shape, want, device.index):
            _check_tensor(name, t, shape, want, device)

    if not isinstance(kv_cache, torch.Tensor) or kv_cache.dim() != 4:
        raise ValueError("kv_cache must be [num_pages, page_size, kv_heads, width] (or [batch, max_seqlen, ...])")
    lead = kv_cache.shape[:3]
    if kv_scales is not None:
        if kv_scale is not None:
            raise ValueError("kv_scale belongs to an e4m3 cache, kv_scales to a 4-bit one: pass one of them")
        form = capi.MLA_CACHE_INT4
        need("kv_cache", kv_cache, (*lead, INT4_BYTES), torch.uint8)
        need("kv_scales", kv_scales, (*lead, INT4_GROUPS), torch.float16)
    elif kv_cache.dtype in (torch.uint8, _FP8):
        if kv_scale is None:
            raise ValueError("an e4m3 kv_cache needs kv_scale, a 4-bit one kv_scales")
        form = capi.MLA_CACHE_FP8
        need("kv_cache", kv_cache, (*lead, DIM), kv_cache.dtype)
    else:
        if kv_scale is not None:
            raise ValueError("kv_scale belongs to an e4m3 cache")
        form = capi.MLA_CACHE_MODEL
        need("kv_cache", kv_cache, (*lead, DIM), dtype)
    need("k_pe_cache", k_pe_cache, (*lead, PE_DIM), dtype)
    return form, lead[0] * lead[1], lead[2]


def _check_dense(kv, k_pe, slots, written):
    dtype = kv.dtype if isinstance(kv, torch.Tensor) else None
    if dtype not in _DTYPES or kv.dim() != 3:
        raise ValueError("kv must be a float16 or bfloat16 tensor [tokens, kv_heads, 512]")
    n, h = kv.shape[:2]
    dev = kv.device
    for name, t, shape in (("kv", kv, (n, h, DIM)), ("k_pe", k_pe, (n, h, PE_DIM))):
        if not (_fits(t, shape, dtype, dev.index) and dev.type == "cuda" and t.data_ptr() % 16 == 0):
            _check_rows(name, t, shape, dtype, None if name == "kv" else dev, written, align=8)
    if not _fits(slots, (n,), torch.int32, dev.index):
        _check_tensor("slots", slots, (n,), torch.int32, dev)
    return n, h, dtype


def _quick_rows(kv, k_pe, slots, kv_cache, k_pe_cache, kv_scale, kv_scales):
    """(tokens, KV heads, cache rows, form, type, strides) of arguments that are all dense and as
    they should be, in one go; None for any others, which the checks above then take up (a
    third of the time of a call of 64 rows went into them)."""
    if not (type(kv) is type(k_pe) is type(slots) is type(kv_cache) is type(k_pe_cache) is torch.Tensor):
        return None
    dtype, index, lead, shape = kv.dtype, kv.get_device(), kv_cache.shape, kv.shape
    if dtype not in _DTYPES or index < 0 or len(lead) != 4 or len(shape) != 3:
        return None
    n, h, width = shape
    pages, page, kvh, held = lead
    if kv_scales is not None:
        if not (kv_scale is None and held == INT4_BYTES and kv_cache.dtype is torch.uint8
                and _fits(kv_scales, (pages, page, kvh, INT4_GROUPS), torch.float16, index)):
            return None
        form = capi.MLA_CACHE_INT4
    elif held != DIM:
        return None
    elif kv_scale is not None:
        if kv_cache.dtype is not _FP8 and kv_cache.dtype is not torch.uint8:
            return None
        form = capi.MLA_CACHE_FP8
    elif kv_cache.dtype is dtype:
        form = capi.MLA_CACHE_MODEL
    else:
        return None
    if (width == DIM and h == kvh and k_pe.dtype is dtype and k_pe_cache.dtype is dtype and slots.dtype is torch.int32
            and k_pe.shape == (n, h, PE_DIM) and slots.shape == (n,) and k_pe_cache.shape == (pages, page, kvh, PE_DIM)
            and kv.is_contiguous() and k_pe.is_contiguous() and slots.is_contiguous() and kv_cache.is_contiguous()
            and k_pe_cache.is_contiguous() and k_pe.get_device() == index and slots.get_device() == index
            and kv_cache.get_device() == index and k_pe_cache.get_device() == index
            and (kv.data_ptr() | k_pe.data_ptr()) & 15 == 0):
        return n, h, pages * page, form, dtype, (h * DIM, DIM, h * PE_DIM, PE_DIM)
    return None


def _rows(kv, k_pe, slots, kv_cache, k_pe_cache, kv_scale, kv_scales, written):
    """What ``_quick_rows`` returns, of any arguments; raises for wrong ones."""
    got = _quick_rows(kv, k_pe, slots, kv_cache, k_pe_cache, kv_scale, kv_scales)
    if got is None:
        n, h, dtype = _check_dense(kv, k_pe, slots, written)
        form, rows, kvh = _check_cache(kv_cache, k_pe_cache, kv_scale, kv_scales, dtype, kv.device)
        if kvh != h:
            raise ValueError(f"kv has {h} KV heads, the cache {kvh}")
        got = n, h, rows, form, dtype, (*_strides(kv), *_strides(k_pe))
    return got


def cache_append(kv, k_pe, slots, kv_cache, k_pe_cache, kv_scale=None, kv_scales=None, rotary=None, positions=None):
    """Write rows kv [tokens, kv_heads, 512] and k_pe [tokens, kv_heads, 64] to cache rows
    ``slots`` (int32 [tokens]; outside the cache, e.g. -1: skipped; slots are distinct).

    The cache ([num_pages, page_size, kv_heads, ...], or [batch, max_seqlen, kv_heads, ...])
    is 16-bit (kv's type), e4m3 (``kv_scale``: codes of kv / kv_scale) or 4-bit (``kv_cache``
    uint8 [..., 256] with ``kv_scales`` float16 [..., 16]); k_pe_cache is in kv's type.  With
    ``rotary`` (a ``Rotary`` of 64 dims) and ``positions`` (int32 [tokens]) k_pe turns on the
    way.  kv and k_pe may be strided (rows on 16-byte boundaries).
    """
    n, h, rows, form, dtype, strides = _rows(kv, k_pe, slots, kv_cache, k_pe_cache, kv_scale, kv_scales, False)
    dev = kv.device
    if (rotary is None) != (positions is None):
        raise ValueError("rotary and positions go together")
    turns, gain, inter = None, 1.0, False
    if rotary is not None:
        if rotary.rot_dim != PE_DIM:
            raise ValueError(f"rotary must turn {PE_DIM} dims, not {rotary.rot_dim}")
        if not _fits(positions, (n,), torch.int32, dev.index):
            _check_tensor("positions", positions, (n,), torch.int32, dev)
        turns, gain, inter = rotary.turns(dev).data_ptr(), rotary.gain, rotary.interleaved
    _on_device(dev, capi.cache_append, kv.data_ptr(), k_pe.data_ptr(), slots.data_ptr(), kv_cache.data_ptr(),
               None if kv_scales is None else kv_scales.data_ptr(), k_pe_cache.data_ptr(),
               1.0 if kv_scale is None else float(kv_scale), None if rotary is None else positions.data_ptr(), turns, gain,
               inter, n, h, rows, *strides, form, _DTYPES[dtype])


def cache_gather(slots, kv_cache, k_pe_cache, kv, k_pe, kv_scale=None, kv_scales=None):
    """Read cache rows ``slots`` back into kv [tokens, kv_heads, 512] and k_pe [tokens,
    kv_heads, 64]: what the cache stands for, in the model's type (zeros for a slot outside
    the cache).  The cache and its forms as in ``cache_append``.
    """
    n, h, rows, form, dtype, strides = _rows(kv, k_pe, slots, kv_cache, k_pe_cache, kv_scale, kv_scales, True)
    _on_device(kv.device, capi.cache_gather, slots.data_ptr(), kv_cache.data_ptr(),
               None if kv_scales is None else kv_scales.data_ptr(), k_pe_cache.data_ptr(),
               1.0 if kv_scale is None else float(kv_scale), kv.data_ptr(), k_pe.data_ptr(), n, h, rows, *strides,
               form, _DTYPES[dtype])
