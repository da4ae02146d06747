"""CPU: the oracle of the key-value cache against the format's definition, the workspace sizes, and the refusals of the
C ABI (all decided on the host, before any GPU work)."""
import ctypes

import numpy as np
import pytest

from oracle import kv_oracle as orc


@pytest.fixture(scope="module")
def lib():
    import rans_b200 as rb
    return rb.build()


def test_oracle_quantises_the_grid_and_its_midpoints():
    # a block whose largest value is 6 has scale 1; grid values keep, midpoints go to the even code, 7 saturates
    x = np.zeros(32)
    x[:8] = orc.GRID
    x[8:15] = -(orc.GRID[:-1] + orc.GRID[1:]) / 2
    x[15] = 7.0
    index, scale = orc.quantise(x)
    assert scale[0] == 127
    assert list(index[:8]) == list(range(8))
    assert [int(i) & 7 for i in index[8:15]] == [0, 2, 2, 4, 4, 6, 6]
    assert all(i >= 8 for i in index[8:15])
    assert index[15] == 7
    got = orc.values(index, scale)
    assert np.array_equal(got[:8], orc.GRID) and got[15] == 6.0


def test_oracle_scale_clamps_and_marks_what_is_not_finite():
    for value, byte in ((0.0, 64), (2.0 ** -80, 64), (2.0 ** 80, 190), (np.inf, 255), (np.nan, 255), (4.0, 127), (3.99, 126)):
        x = np.zeros(32)
        x[5] = value
        assert orc.quantise(x)[1][0] == byte
    assert np.isnan(orc.values(*orc.quantise(np.full(32, np.nan)))).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_stored_bytes_hold_every_code_once(dim):
    index = (np.arange(dim) * 7 % 16).astype(np.uint8)
    stored = orc.pack(index)
    assert stored.shape == (dim // 2,)
    back = [(stored[d % 32 // 8 * (dim // 8) + d // 32 * 4 + d % 8 // 2] >> (4 * (d % 2))) & 15 for d in range(dim)]
    assert back == list(index)


def test_oracle_eviction():
    w, p = np.array([5.0, 1.0, 1.0, 9.0, 0.0, 2.0]), np.arange(6)
    # newest two stay (4, 5), then 3 (9.0) and 0 (5.0): freed 1, 2 take 4, 5
    assert orc.evict_moves(w, p, 6, 4, 2) == [(1, 4), (2, 5)]
    assert orc.evict_moves(w, p, 6, 6, 2) == []
    # a tie at 1.0 keeps the lower place
    assert orc.evict_moves(w, p, 6, 4, 0) == [(2, 5)]
    assert orc.evict_moves(np.array([1.0, np.nan, 2.0]), np.arange(3), 3, 1, 0) == [(0, 1)]


# ------------------------------------------------------------------ refusals
FAKE = 1 << 20          # an aligned address that is never followed


def _cache(**change):
    import rans_cache as rc
    d = dict(k=FAKE, v=FAKE, k_scale=None, v_scale=None, weight=FAKE, position=FAKE, table=FAKE, length=FAKE, seen=FAKE,
             status=FAKE, workspace=FAKE, workspace_bytes=1 << 40, k_page=1 << 16, k_head=1 << 12, k_slot=256, v_page=1 << 16,
             v_head=1 << 12, v_slot=256, pages=4, page=16, kv_heads=2, dim=128, batch=3, table_cols=2, kind=0, reserved=0)
    d.update(change)
    return rc.RansKvCache(**d)


BAD = [(dict(kind=3), -1), (dict(dim=96), -1), (dict(dim=0), -1), (dict(page=8), -2), (dict(page=24), -2), (dict(page=0), -2),
       (dict(pages=0), -2), (dict(kv_heads=0), -2), (dict(batch=0), -2), (dict(batch=2049), -2),
       (dict(batch=2048, kv_heads=32), -2), (dict(table_cols=0), -2), (dict(table_cols=1 << 30), -2), (dict(reserved=1), -2),
       (dict(k=None), -2), (dict(v=None), -2), (dict(k=FAKE + 2), -2), (dict(table=None), -2), (dict(length=None), -2),
       (dict(seen=None), -2), (dict(status=None), -2), (dict(workspace=None), -2), (dict(k_slot=264), -2),
       (dict(v_page=8), -2), (dict(kind=2), -2), (dict(workspace_bytes=64), -3)]


@pytest.mark.parametrize("change,code", BAD, ids=[",".join(f"{k}={v}" for k, v in c.items()) for c, _ in BAD])
def test_bad_caches_are_refused(lib, change, code):
    c = _cache(**change)
    p = ctypes.addressof(c)
    assert lib.rans_kv_append(p, FAKE, FAKE, 0, 512, 256, 512, 256, None, c.batch, None) == code
    assert lib.rans_kv_read(p, FAKE, FAKE, None, c.batch, None) == code
    assert lib.rans_kv_attend(p, FAKE, 0, 4096, 256, 16, 1.0, FAKE, FAKE, 0, None) == code
    assert lib.rans_kv_evict(p, 8, 2, None) == code


def test_no_cache_is_refused(lib):
    assert lib.rans_kv_append(None, FAKE, FAKE, 0, 512, 256, 512, 256, None, 3, None) == -2
    assert lib.rans_kv_evict(None, 8, 2, None) == -2
    assert lib.rans_kv_attend_bytes(None, 16, 0) == -2
    assert lib.rans_kv_counter_bytes(None) == -2
    assert lib.rans_kv_evict_bytes(None, 4) == -2


def test_bad_calls_are_refused(lib):
    c = _cache()
    p = ctypes.addressof(c)
    append = lambda **d: lib.rans_kv_append(p, *[{**dict(k=FAKE, v=FAKE, given=0, a=512, b=256, c=512, d=256, starts=None, n=3,    # noqa: E731
                                                         stream=None), **d}[x] for x in ("k", "v", "given", "a", "b", "c", "d", "starts", "n", "stream")])
    assert append(given=2) == -1 and append(given=7) == -1
    assert append(n=2) == -2 and append(n=-1) == -2 and append(k=None) == -2 and append(v=FAKE + 8) == -2 and append(b=264) == -2
    assert append(starts=FAKE, n=0) == 0                       # nothing to do, nothing launched
    assert lib.rans_kv_read(p, None, FAKE, None, 3, None) == -2
    assert lib.rans_kv_read(p, FAKE, FAKE, None, 2, None) == -2
    attend = lambda **d: lib.rans_kv_attend(p, *[{**dict(q=FAKE, kind=0, qb=4096, qh=256, heads=16, scale=1.0, out=FAKE, ls=None,   # noqa: E731
                                                         weigh=0, stream=None), **d}[x] for x in ("q", "kind", "qb", "qh", "heads", "scale", "out", "ls", "weigh", "stream")])
    assert attend(kind=1) == -1 and attend(kind=3) == -1
    assert attend(heads=15) == -2 and attend(heads=0) == -2 and attend(heads=2 * 16 * 16 + 2) == -2
    assert attend(q=None) == -2 and attend(out=None) == -2 and attend(q=FAKE + 4) == -2 and attend(qh=250) == -2
    assert lib.rans_kv_evict(p, 0, 0, None) == -2 and lib.rans_kv_evict(p, 8, 9, None) == -2 and lib.rans_kv_evict(p, 8, -1, None) == -2
    bare = _cache(weight=None)
    assert lib.rans_kv_attend(ctypes.addressof(bare), FAKE, 0, 4096, 256, 16, 1.0, FAKE, None, 1, None) == -2
    assert lib.rans_kv_evict(ctypes.addressof(bare), 8, 2, None) == -2
    small = _cache(workspace_bytes=lib.rans_kv_counter_bytes(p))
    assert lib.rans_kv_attend(ctypes.addressof(small), FAKE, 0, 4096, 256, 16, 1.0, FAKE, None, 0, None) == -3
    assert lib.rans_kv_evict(ctypes.addressof(small), 8, 2, None) == -3


def test_workspace_sizes(lib):
    c = _cache()
    p = ctypes.addressof(c)
    base = lib.rans_kv_counter_bytes(p)
    assert base >= c.batch * c.kv_heads * 4
    plain, weighed = lib.rans_kv_attend_bytes(p, 16, 0), lib.rans_kv_attend_bytes(p, 16, 1)
    assert base < plain < weighed
    assert weighed - plain >= c.pages * c.page * c.kv_heads * 8 * 4          # a score per token and padded query head
    assert lib.rans_kv_attend_bytes(p, 15, 0) == -2
    assert lib.rans_kv_evict_bytes(p, 8) > base and lib.rans_kv_evict_bytes(p, 0) == -2


def test_struct_mirror_has_the_headers_layout():
    import rans_cache as rc
    assert ctypes.sizeof(rc.RansKvCache) == 12 * 8 + 6 * 8 + 8 * 4
    assert rc.RansKvCache.k_page.offset == 96 and rc.RansKvCache.pages.offset == 144 and rc.RansKvCache.kind.offset == 168


def test_eviction_to_more_than_the_table_holds_needs_no_lists(lib):
    """A (sequence, kv head) has at most as many moves as the budget and the places above it."""
    c = _cache(table_cols=4)                               # 64 places
    p = ctypes.addressof(c)
    none = lib.rans_kv_evict_bytes(p, 64)
    assert all(lib.rans_kv_evict_bytes(p, budget) == none for budget in (65, 10 ** 6, 2 ** 31 - 1))
    assert none < lib.rans_kv_evict_bytes(p, 63) <= lib.rans_kv_evict_bytes(p, 32)
    wide = _cache(table_cols=1 << 14, batch=128, kv_heads=8)
    p = ctypes.addressof(wide)
    room = 16 << 14
    keys = (1 << 14) * 16 * 128 * 8 * 4                    # more than shared memory takes
    assert lib.rans_kv_evict_bytes(p, room - 10) < lib.rans_kv_counter_bytes(p) + keys + 2 * 128 * 8 * 10 * 4 + (1 << 16)
