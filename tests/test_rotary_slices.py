"""Which pairs of strided tensors share elements: the rotary's check of its operands against
a listing of every element's address, and slices of one buffer on the GPU."""
import itertools
import random

import pytest
import torch

from mlc_decode_b200 import Rotary
from mlc_decode_b200.paged import _share_elements


def _elements(t):
    return {t.storage_offset() + sum(i * s for i, s in zip(at, t.stride()))
            for at in itertools.product(*(range(n) for n in t.shape))}


def test_shared_elements_against_a_listing():
    rng = random.Random(7)
    buf = torch.zeros(4000)
    told = 0
    for _ in range(3000):
        n, h, d = rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 6)
        inner, outer = rng.randint(d, 12), 0
        outer = inner * (h - 1) + d + rng.randint(0, 20)
        st = (outer, inner) if rng.random() < 0.7 else (d + rng.randint(0, 3), (n - 1) * (d + 3) + d + rng.randint(0, 9))
        st2 = st if rng.random() < 0.7 else (outer + rng.randint(0, 9), inner)
        a = buf.as_strided((n, h, d), (*st, 1), rng.randint(0, 200))
        b = buf.as_strided((n, h, d), (*st2, 1), rng.randint(0, 200))
        true = bool(_elements(a) & _elements(b))
        got = _share_elements(a, b)
        assert got or not true, (a.shape, st, st2, a.storage_offset(), b.storage_offset())
        norm = [tuple(s for s, k in zip(s2, (n, h)) if k > 1) for s2 in (st, st2)]
        if norm[0] == norm[1]:
            assert got == true, (a.shape, st, st2, a.storage_offset(), b.storage_offset())
            told += not true
    assert told > 100


def test_shared_elements_of_broadcast_rows():
    buf = torch.zeros(100)
    x = buf.as_strided((5, 2, 4), (0, 4, 1))
    assert _share_elements(x, buf.as_strided((5, 2, 4), (8, 4, 1)))
    assert not _share_elements(x, buf.as_strided((5, 2, 4), (8, 4, 1), 8))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [True, False])
def test_slices_of_one_buffer(interleaved):
    g = torch.Generator(device="cuda").manual_seed(3)
    rot = Rotary(64, interleaved=interleaved)
    pos = torch.randint(0, 5000, (37,), generator=g, device="cuda", dtype=torch.int32)

    def rn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").bfloat16()

    for buf, cut in ((rn(37, 5, 128), lambda t: (t[:, :, :64], t[:, :, 64:])),          # halves of every head
                     (rn(37, 10, 64), lambda t: (t[:, 5:], t[:, :5])),                  # two ranges of heads
                     (rn(37, 10, 64), lambda t: (t[:, ::2], t[:, 1::2])),               # every other head
                     (rn(74, 5, 64), lambda t: (t[1::2], t[::2])),                      # every other token
                     (rn(37, 640 + 24), lambda t: (t[:, :320].unflatten(1, (5, 64)),
                                                   t[:, 344:].unflatten(1, (5, 64))))):   # parts of a fused row
        before = buf.clone()
        x, out = cut(buf)
        want = torch.empty(37, 5, 64, dtype=buf.dtype, device="cuda")
        rot(x.contiguous(), pos, want)
        rot(x, pos, out)
        assert torch.equal(out, want)
        cut(before)[1].copy_(want)
        assert torch.equal(buf, before)


@pytest.mark.gpu
def test_overlapping_slices_are_refused():
    rot = Rotary(64)
    buf = torch.zeros(9, 4, 128, device="cuda").bfloat16()
    pos = torch.zeros(9, dtype=torch.int32, device="cuda")
    for x, out in ((buf[:, :, :64], buf[:, :, 32:96]), (buf[:, :, :64], buf[:, :, 63:127]),
                   (buf[:, :3, :64], buf[:, 1:, :64]), (buf[:8, :, :64], buf[1:, :, :64])):
        with pytest.raises(ValueError, match="overlap"):
            rot(x, pos[:x.shape[0]], out)


@pytest.mark.gpu
def test_in_place_with_other_strides_of_single_entries():
    """Of a dim of one entry any stride will do, in place too."""
    g = torch.Generator(device="cuda").manual_seed(4)
    buf = torch.randn(600, generator=g, device="cuda").bfloat16()
    rot = Rotary(64)
    for shape, s1, s2 in (((1, 4, 64), (256, 64, 1), (7, 64, 1)), ((5, 1, 64), (64, 64, 1), (64, 999, 1))):
        pos = torch.arange(1, shape[0] + 1, dtype=torch.int32, device="cuda") * 77
        x, out = buf.as_strided(shape, s1), buf.as_strided(shape, s2)
        want = torch.empty(shape, dtype=buf.dtype, device="cuda")
        rot(x.clone(), pos, want)
        rot(x, pos, out)
        assert torch.equal(x, want)
