"""All-or-nothing rows of a step's block tables, without a GPU: refusals of the C entry point,
and the oracle's rule on cases worked out by hand."""
import pytest

from mlc_decode_b200 import capi
from oracle import paged_oracle as P

PTR = 4096   # a non-null aligned address that no refused call touches


def _whole(**kw):
    a = dict(table=PTR, lens=PTR, new=PTR, free=PTR, pos=PTR, nlens=PTR, npos=PTR, slots=PTR, positions=PTR, cu=None,
             ws=None, wsb=0, batch=4, max_pages=8, page=64, pages=32, nfree=10, tokens=12, q_len=3)
    a.update(kw)
    return capi.load().mla_extend_block_tables_whole(*a.values(), None)


@pytest.mark.parametrize("kw, status, word", [
    (dict(q_len=0, tokens=4), 1, "q_len"), (dict(q_len=-1), 1, "q_len"), (dict(q_len=2), 1, "batch x q_len"),
    (dict(batch=0), 1, "size"), (dict(page=0), 1, "size"), (dict(page=1 << 20, pages=1 << 12), 1, "2^31"),
    (dict(table=None), 1, "null"), (dict(slots=None), 1, "null"),
    (dict(batch=4000, tokens=12000), 2, "workspace"),
])
def test_refusals(kw, status, word):
    assert _whole(**kw) == status
    assert word in capi.last_error() and "mla_extend_block_tables_whole" in capi.last_error()


def test_the_rule_by_hand():
    # 62 rows on a page of 64, three more asked for, no page free: two would fit, none is placed
    table, lens, pos, slots, positions, cu = P.extend_tables([[4, -1]], [62], [3], [], 0, 64, 8, 3, 3, whole=True)
    assert (table, lens, pos, slots, positions, cu) == ([[4, -1]], [62], 0, [-1] * 3, [62, 63, 64], [0, 3])
    # one page free: the second request lacks one more than there is, the third lacks one and
    # gets none behind it, the fourth lacks none and is placed, the first has taken its page
    got = P.extend_tables([[0, 9], [9, 9], [1, 9], [2, 9]], [64, 0, 64, 10], [1, 65, 2, 70], [5, 6], 0, 64, 8, 280, 70,
                          whole=True)
    assert got[0] == [[0, 5], [9, 9], [1, 9], [2, 9]] and got[1] == [65, 0, 64, 10] and got[2] == 1
    got = P.extend_tables([[0, 9], [9, 9], [1, 9], [2, 9]], [64, 0, 64, 10], [1, 65, 2, 54], [5, 6], 0, 64, 8, 280, 70,
                          whole=True)
    assert got[1] == [65, 0, 64, 64] and got[3][226:] == [2 * 64 + r for r in range(10, 64)]
    # a table row that is too short is refused by itself: the next request still finds its page
    got = P.extend_tables([[3], [0]], [63, 0], [2, 2], [7], 0, 64, 8, 4, 2, whole=True)
    assert got[:4] == ([[3], [7]], [63, 2], 1, [-1, -1, 7 * 64, 7 * 64 + 1])


def test_append_takes_every_float32_scale():
    """What the decode takes as an e4m3 scale the append takes too (no rows: nothing launches)."""
    lib = capi.load()
    for scale, status in ((3.4028e38, 0), (1e-45, 0), (1e39, 1), (1e-50, 1), (-1.0, 1)):
        got = lib.mla_cache_append(PTR, PTR, PTR, PTR, None, PTR, scale, None, None, 1.0, 0, 0, 1, 128, 512, 512, 64, 64,
                                   1, 1, None)
        assert got == status, scale
