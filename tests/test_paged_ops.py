"""Paged-cache operators without a GPU: refusals of the C entry points and of the Python
calls, the rotary frequencies and the oracle's own 4-bit form.  Nothing here launches."""
import ctypes
import math

import numpy as np
import pytest
import torch

from mlc_decode_b200 import MlaPagedDecodeKernel, Rotary, cache_append, cache_gather, capi, extend_block_tables, \
    rotary_frequencies
from oracle import paged_oracle as P

PTR = 4096   # a non-null aligned address that no refused call touches


@pytest.fixture(scope="module")
def lib():
    return capi.load()


def _tables(lib, **kw):
    a = dict(table=PTR, lens=PTR, new=PTR, free=PTR, pos=PTR, nlens=PTR, npos=PTR, slots=PTR, positions=PTR, cu=None,
             ws=None, wsb=0, batch=4, max_pages=8, page=64, pages=32, nfree=10, tokens=4, q_len=0)
    a.update(kw)
    return lib.mla_extend_block_tables(*a.values(), None)


@pytest.mark.parametrize("kw, status, word", [
    (dict(batch=0), 1, "size"), (dict(max_pages=0), 1, "size"), (dict(page=0), 1, "size"), (dict(pages=0), 1, "size"),
    (dict(nfree=-1), 1, "size"), (dict(tokens=-1), 1, "size"), (dict(q_len=-1), 1, "size"),
    (dict(page=1 << 20, pages=1 << 12), 1, "2^31"), (dict(page=1 << 20, max_pages=1 << 12), 1, "2^31"),
    (dict(q_len=2), 1, "batch x q_len"), (dict(table=None), 1, "null"), (dict(lens=None), 1, "null"),
    (dict(new=None), 1, "null"), (dict(free=None), 1, "null"), (dict(pos=None), 1, "null"),
    (dict(slots=None), 1, "null"), (dict(positions=None), 1, "null"), (dict(npos=None), 1, "null"),
    (dict(batch=4000), 2, "workspace"), (dict(tokens=100000), 2, "workspace"),
    (dict(tokens=100000, ws=PTR + 8, wsb=1 << 20), 2, "workspace"),
])
def test_tables_refusals(lib, kw, status, word):
    assert _tables(lib, **kw) == status and word in capi.last_error()


def test_tables_workspace_rule():
    assert capi.block_tables_workspace_bytes(64, 64) == 0
    assert capi.block_tables_workspace_bytes(2048, 8192) == 0
    assert capi.block_tables_workspace_bytes(2049, 1) == 2049 * 16
    assert capi.block_tables_workspace_bytes(3, 8193) == 3 * 16
    with pytest.raises(capi.MlaError):
        capi.block_tables_workspace_bytes(0, 4)


def _rotary(lib, **kw):
    a = dict(x=PTR, out=2 * PTR, pos=PTR, turns=PTR, gain=1.0, tokens=4, heads=2, dim=64, rot=64, offset=0, inter=1,
             xt=128, xh=64, ot=128, oh=64, dtype=1)
    a.update(kw)
    return lib.mla_rotary(*a.values(), None)


@pytest.mark.parametrize("kw, word", [
    (dict(tokens=-1), "size"), (dict(heads=0), "size"), (dict(rot=63), "size"), (dict(rot=0), "size"),
    (dict(rot=2048, dim=4096), "size"), (dict(offset=1), "size"), (dict(offset=-1), "size"), (dict(dtype=5), "dtype"),
    (dict(xt=-1), "strides"), (dict(x=None), "null"), (dict(pos=None), "null"), (dict(turns=None), "null"),
    (dict(out=PTR, ot=256), "in place"), (dict(x=PTR + 1), "aligned"), (dict(turns=PTR + 4), "aligned"),
])
def test_rotary_refusals(lib, kw, word):
    assert _rotary(lib, **kw) == 1 and word in capi.last_error()


def _append(lib, **kw):
    a = dict(kv=PTR, pe=PTR, slots=PTR, cache=PTR, scales=PTR, pec=PTR, scale=1.0, pos=None, turns=None, gain=1.0,
             inter=0, tokens=4, kvh=1, rows=128, kt=512, kh=512, pt=64, ph=64, form=2, dtype=1)
    a.update(kw)
    return lib.mla_cache_append(*a.values(), None)


@pytest.mark.parametrize("kw, word", [
    (dict(tokens=-1), "size"), (dict(kvh=0), "size"), (dict(rows=0), "size"), (dict(rows=1 << 31), "size"),
    (dict(dtype=2), "dtype"), (dict(form=3), "form"), (dict(form=1, scale=0.0), "kv_scale"),
    (dict(form=1, scale=math.inf), "kv_scale"), (dict(form=1, scale=math.nan), "kv_scale"),
    (dict(kt=-8), "strides"), (dict(kt=516), "strides"), (dict(ph=4), "strides"), (dict(kv=None), "null"),
    (dict(slots=None), "null"), (dict(scales=None), "null"), (dict(pos=PTR), "null"), (dict(cache=PTR + 8), "aligned"),
    (dict(kv=PTR + 2), "aligned"), (dict(scales=PTR + 2), "aligned"),
])
def test_append_refusals(lib, kw, word):
    assert _append(lib, **kw) == 1 and word in capi.last_error()


def test_empty_calls_launch_nothing(lib):
    assert _append(lib, tokens=0) == 0
    assert _rotary(lib, tokens=0) == 0


def _int4(lib, cfg=None, **kw):
    a = dict(q=PTR, qpe=PTR, codes=PTR, scales=PTR, pe=PTR, table=None, lens=None, out=PTR, lse=None, ws=PTR,
             wsb=1 << 40, batch=2, q_len=1, heads=16, kvh=1, smax=300, page=0, pages=0, maxp=0, dtype=1)
    a.update(kw)
    return lib.mla_decode_ext_int4kv(*a.values(), ctypes.byref(capi.make_cfg(cfg or {})), None)


@pytest.mark.parametrize("kw, status, word", [
    (dict(batch=0), 1, ">= 1"), (dict(q_len=0), 1, ">= 1"), (dict(heads=3, kvh=2), 1, "multiple"),
    (dict(smax=0), 1, ">= 1"), (dict(dtype=2), 1, "dtype"), (dict(batch=1 << 16), 3, "large"),
    (dict(q=None), 1, "null"), (dict(scales=None), 1, "null"), (dict(codes=PTR + 8), 1, "aligned"),
    (dict(table=PTR, page=32, pages=4, maxp=4), 1, "page_size"), (dict(table=PTR, page=64, pages=0, maxp=4), 1, "page_size"),
    (dict(table=PTR, page=64, pages=1 << 26, maxp=4), 1, "page_size"), (dict(ws=None), 2, "workspace"),
    (dict(wsb=64), 2, "workspace"), (dict(ws=PTR + 16), 2, "workspace"),
    (dict(cfg={"softmax_scale": -1.0}), 1, "softmax_scale"), (dict(cfg={"softmax_scale": math.inf}), 1, "softmax_scale"),
    (dict(cfg={"num_split": -1}), 1, "num_split"), (dict(cfg={"kernel": 9}), 1, "kernel"),
])
def test_int4_refusals(lib, kw, status, word):
    assert _int4(lib, **kw) == status and word in capi.last_error()


def test_cpu_tensors_are_refused():
    i = torch.zeros(4, dtype=torch.int32)
    kv, pe = torch.zeros(4, 1, 512, dtype=torch.bfloat16), torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    cache = torch.zeros(2, 64, 1, 256, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        extend_block_tables(i.view(2, 2), i, i, i, i, i, i, i, i, page_size=64, num_pages=4)
    with pytest.raises(ValueError, match="CUDA"):
        cache_append(kv, pe, i, cache, pe, kv_scales=cache)
    with pytest.raises(ValueError, match="CUDA"):
        cache_gather(i, cache, pe, kv, pe, kv_scales=cache)
    with pytest.raises(ValueError, match="CUDA"):
        Rotary()(pe, i, pe)
    k = MlaPagedDecodeKernel(4, 1, 64)
    with pytest.raises(ValueError, match="CUDA"):
        k.decode_int4(kv, pe, cache, cache, pe, None, kv)
    with pytest.raises(ValueError, match="CUDA"):
        k.step(kv, pe, kv, pe, cache, pe, i, i, i, i, kv)


@pytest.mark.parametrize("kw", [
    dict(rot_dim=63), dict(rot_dim=0), dict(rot_dim=2048), dict(base=1.0), dict(base=math.inf),
    dict(scaling={"type": "other"}), dict(scaling={"type": "linear", "factor": 0.5}),
    dict(scaling={"type": "linear", "factor": math.inf}), dict(scaling={"type": "linear", "fcator": 2.0}),
    dict(scaling={"type": "yarn", "factor": 4.0}), dict(scaling={"factor": 4.0}),
    dict(scaling={"type": "yarn", "factor": 4.0, "original_max_position": 4096, "beta_fast": 0.5}),
    dict(scaling={"type": "yarn", "factor": 4.0, "original_max_position": 4096, "gain": math.nan}),
    dict(rot_dim=2, scaling={"type": "ntk", "factor": 2.0}),
])
def test_rotary_parameter_refusals(kw):
    with pytest.raises(ValueError):
        Rotary(**kw)


@pytest.mark.parametrize("scaling", [
    None, {"type": "linear", "factor": 8.0}, {"type": "ntk", "factor": 4.0},
    {"type": "yarn", "factor": 40.0, "original_max_position": 4096},
    {"type": "yarn", "factor": 1.0, "original_max_position": 10, "beta_fast": 1.0, "beta_slow": 1.0, "gain": 2.0},
])
@pytest.mark.parametrize("rot_dim, base", [(64, 10000.0), (4, 500.0), (128, 1e6)])
def test_rotary_frequencies(rot_dim, base, scaling):
    freq, gain = rotary_frequencies(rot_dim, base, scaling)
    ref, ref_gain = P.frequencies(rot_dim, base, scaling)
    # a handful of float64 roundings
    np.testing.assert_allclose(freq, ref, rtol=1e-13)
    assert gain == pytest.approx(ref_gain, rel=1e-14)


def test_int4_form_round_trip():
    rng = np.random.default_rng(3)
    codes = rng.integers(0, 16, (5, 512)).astype(np.uint8)
    assert np.array_equal(P.unpack_int4(P.pack_int4(codes)), codes)
    x = rng.standard_normal((7, 512))
    n, s = P.quantise_int4(x)
    # half a step of the scale, and what the scale's own rounding (2^-11) leaves past code 7
    err = np.abs(P.dequantise_int4(n, s) - x).reshape(7, 16, 32)
    assert np.all(err <= s.astype(np.float64)[..., None] * (0.5 + 7 * 2.0 ** -11))
