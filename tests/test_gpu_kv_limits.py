"""GPU: the paged key-value cache at the ends of its types, its row ranges and its pages, against the 64-bit oracle."""
import numpy as np
import pytest

from oracle import kv_oracle as orc
from test_gpu_kv_cache import APART, check_attend, fill, rc, seeded, torch     # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu


def i32(torch, x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ probabilities
@pytest.mark.parametrize("dim,heads", [(64, 8), (128, 8), (128, 24), (256, 4)])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "4-bit values far apart"])
def test_attend_rounds_the_output_and_little_else(torch, rc, kind, dim, heads):
    """The error's root mean square beside that of the exact result rounded once to the output's type.  Probabilities held to
    2^-16 (bf16) or 2^-22 (fp16) of themselves and fp32 sums add less than a hundredth of it; probabilities rounded once to
    the type would add about a fifth.  (The squares add up: 2 % is an error of a fifth of the rounding's.)"""
    lens = [2000, 1777, 3001]
    apart = kind.startswith("4-bit")
    cache, truth, _ = fill(torch, rc, lens, 2, dim, 16, "mxfp4" if apart else kind, seed=dim + heads, exponents=APART["far apart"] if apart else None)
    q = torch.randn(len(lens), heads, dim, device="cuda").to(torch.float16 if kind == "fp16" else torch.bfloat16)
    scale = dim ** -0.5 * (0.05 if apart else 1.0)
    out = cache.attend(q, scale=scale)[0].double().cpu()
    want = torch.from_numpy(np.stack([orc.attend(q[b].double().cpu().numpy(), truth["k"][b], truth["v"][b], scale)[0] for b in range(len(lens))]))
    size = want.abs().amax(-1, keepdim=True) if apart else 1.0             # (a row's largest blocks decide)
    rms = lambda x: float((x / size).square().mean().sqrt())                # noqa: E731
    assert rms(out - want) <= 1.02 * rms(want.to(q.dtype).double() - want)


@pytest.mark.parametrize("lens", [[1], [300], [9000], [1, 0, 33, 700]])
@pytest.mark.parametrize("spread", [8.0e37, 2.0 ** -70], ids=["large", "small"])
def test_attend_over_bf16_values_near_the_ends_of_the_type(torch, rc, lens, spread):
    """Sums of values up to the type's largest stay finite, and tiny ones keep their digits, in one part and in many."""
    cache, truth, table = fill(torch, rc, lens, 2, 128, 16, "bf16", seed=sum(lens))
    v = (cache.v.float() * spread).clamp(-3.38e38, 3.38e38).bfloat16()
    cache.v.copy_(v)
    pages = lambda b, n: torch.from_numpy(table[b, :-(-n // 16)]).long().cuda()     # noqa: E731
    for b, n in enumerate(lens):
        truth["v"][b] = v[pages(b, n)].transpose(0, 1).reshape(2, -1, 128)[:, :n].double().cpu().numpy() if n else truth["v"][b]
    q = torch.randn(len(lens), 14, 128, device="cuda").bfloat16()
    got = cache.attend(q, weigh=True)
    check_attend(torch, cache, truth, q, lens, 128 ** -0.5, got, cache.weight, table)


def test_attend_over_bf16_values_that_are_all_the_largest(torch, rc):
    lens = [1, 40, 5000]
    cache, _, _ = fill(torch, rc, lens, 1, 64, 16, "bf16", seed=1)
    top = torch.finfo(torch.bfloat16).max
    cache.v.fill_(top)
    cache.v[..., ::2] = -top
    out, _ = cache.attend(torch.randn(3, 8, 64, device="cuda").bfloat16())
    # the exact answer is the value itself; fp32 sums are off by less than half a unit of bf16
    assert (out[..., 1::2] == top).all() and (out[..., ::2] == -top).all()


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("n", [1, 17, 600])
def test_attend_with_scores_near_the_lowest_number(torch, rc, kind, n):
    """Equal scores of -2.2e38 (finite in powers of two as well): the mean of the values."""
    cache, truth, table = fill(torch, rc, [n], 1, 64, 16, kind, seed=n)
    cache.k.fill_(0.0)
    cache.k[..., 0] = 2.0 ** 10
    q = torch.zeros(1, 4, 64, device="cuda", dtype=cache.k.dtype)
    q[..., 0] = -1.3046875
    scale = 2.0 ** 117                                     # -1.3046875 * 2^127 = -2.2198e38, times log2 e -3.2026e38
    out, log_sum = cache.attend(q, scale=scale, weigh=True)
    want = truth["v"][0][0].mean(0)
    size = np.abs(truth["v"][0][0]).mean(0)
    assert (np.abs(out[0].double().cpu().numpy() - want) <= 2.0 ** -7 * size).all()
    assert np.abs(log_sum.double().cpu().numpy() / (-1.3046875 * 2.0 ** 127) - 1).max() <= 2.0 ** -21
    t = np.arange(n)
    weight = cache.weight.cpu().numpy()[table[0, t // 16], 0, t % 16]
    assert np.abs(weight * n / 4 - 1).max() <= 2.0 ** -18


@pytest.mark.parametrize("dim,heads", [(64, 4), (128, 8), (128, 24), (256, 8)])
def test_attend_over_key_blocks_that_are_not_finite(torch, rc, dim, heads):
    """Scale byte 255 is NaN whatever the block's codes are: the scores, so all of the head's output, are NaN."""
    lens = [40, 40, 40]
    cache, _, table = fill(torch, rc, lens, 2, dim, 16, "mxfp4", seed=dim)
    for b, code in ((0, 0x77), (1, 0xff)):                 # 6 and -6 throughout the row
        cache.k[int(table[b, 1]), 1, 3] = code
        cache.k_scale[int(table[b, 1]), 1, 3, 1] = 255
    q = torch.randn(3, heads, dim, device="cuda").abs().bfloat16()
    out, log_sum = cache.attend(q)
    half = heads // 2
    assert torch.isnan(out[:2, half:]).all() and torch.isnan(log_sum[:2, half:]).all()
    assert torch.isfinite(out[:2, :half]).all() and torch.isfinite(out[2]).all() and torch.isfinite(log_sum[2]).all()


# ------------------------------------------------------------------ row ranges
STARTS = {"past the rows": ([0, 2, 9], [42, 22]), "past the rows at once": ([0, 100, 200], [44, 20]),
          "not from zero": ([1, 2, 4], [41, 22]), "from below zero": ([-3, 2, 4], [42, 22]),
          "falling": ([0, 3, 1], [40, 20]), "falling below zero": ([0, -2, 4], [40, 20])}


@pytest.mark.parametrize("what", list(STARTS))
@pytest.mark.parametrize("kind", ["bf16", "mxfp4"])
def test_append_of_bad_row_ranges_counts_what_it_stored(torch, rc, what, kind):
    """4 rows: those inside both the ranges and the rows are stored and counted, none where the ranges fall; check() tells."""
    starts, lens = STARTS[what]
    cache, _, table = fill(torch, rc, [40, 20], 1, 64, 16, kind, seed=3)
    rows = torch.randn(4, 1, 64, device="cuda").bfloat16()
    cache.append(rows, rows, i32(torch, starts))
    with pytest.raises(rc.CacheError, match="rows"):
        cache.check()
    assert cache.length.tolist() == lens and cache.seen.tolist() == lens
    # what was counted can be read back: the rows of the clamped ranges
    new = [n - m for n, m in zip(lens, (40, 20))]
    got = cache.read(i32(torch, np.cumsum([0] + new)), sum(new))[0].double().cpu().numpy()
    first = [min(max(s, 0), 4) for s in starts]
    want = np.concatenate([rows[first[b]:first[b] + new[b]].double().cpu().numpy() for b in range(2)])
    assert np.array_equal(got, want if kind == "bf16" else orc.values(*orc.quantise(want)))
    cache.check()


@pytest.mark.parametrize("starts", [[0, 2, 9], [1, 2, 4], [0, 3, 1], [-1, 2, 4]])
def test_read_of_bad_row_ranges_is_reported(torch, rc, starts):
    cache, truth, _ = fill(torch, rc, [40, 20], 1, 64, 16, "bf16", seed=3)
    k, _ = cache.read(i32(torch, starts), 4)
    assert torch.isfinite(k).all()
    with pytest.raises(rc.CacheError, match="rows"):
        cache.check()


def test_append_of_falling_ranges_over_many_sequences(torch, rc):
    """Ranges in no order over more sequences than one round of the search takes."""
    batch = 300
    cache, _, _ = fill(torch, rc, [5] * batch, 1, 64, 16, "bf16", seed=4)
    rng = np.random.default_rng(0)
    rows = torch.ones(200, 1, 64, device="cuda")
    for _ in range(5):
        cache.append(rows, rows, i32(torch, rng.integers(0, 201, batch + 1)))
        with pytest.raises(rc.CacheError, match="rows"):
            cache.check()
        assert cache.length.tolist() == [5] * batch and cache.seen.tolist() == [5] * batch
        assert torch.isfinite(cache.read(i32(torch, rng.integers(0, 201, batch + 1)), 200)[0]).all()
        with pytest.raises(rc.CacheError, match="rows"):
            cache.check()


# ------------------------------------------------------------------ pages of the cache's own
def _rows(torch, n, kv=2, dim=64):
    return [torch.randn(n, kv, dim, device="cuda").bfloat16() for _ in range(2)]


def _pages_of(cache, b, n):
    return [int(p) for p in cache.table[b, :-(-n // cache.page)]]


def test_what_an_eviction_gives_back_is_never_shared(torch, rc):
    """After an eviction another sequence takes the freed pages; an append without reserve by the first is left out and
    reported, and harms nobody."""
    cache = rc.KVCache(pages=6, page=16, kv_heads=2, dim=64, batch=2, max_tokens=96)
    cache.reserve([64, 0])
    cache.append(*_rows(torch, 64), i32(torch, [0, 64, 64]))
    cache.evict(16, 4)
    assert cache.free_pages == 5
    cache.reserve([0, 80])                                 # all that is free
    assert cache.free_pages == 0
    k, v = _rows(torch, 80)
    cache.append(k, v, i32(torch, [0, 0, 80]))
    used = _pages_of(cache, 0, 16) + _pages_of(cache, 1, 80)
    assert len(set(used)) == 6 and min(used) >= 0
    cache.check()
    cache.append(*_rows(torch, 1), i32(torch, [0, 1, 1]))  # place 16 of sequence 0: not reserved
    got = cache.read(i32(torch, [0, 0, 80]), 80)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    with pytest.raises(rc.CacheError, match="page"):
        cache.check()


def test_pages_reserved_for_tokens_to_come_survive_an_eviction(torch, rc):
    cache = rc.KVCache(pages=8, page=16, kv_heads=2, dim=64, batch=2, max_tokens=128)
    cache.reserve([100, 10])                               # 7 pages and 1
    cache.append(*_rows(torch, 60), i32(torch, [0, 50, 60]))
    cache.evict(32, 4)                                     # 32 left, 50 more are to come: 6 pages
    assert cache.length.tolist() == [32, 10] and cache.free_pages == 1
    with pytest.raises(rc.CacheError):
        cache.reserve([0, 30])
    k, v = _rows(torch, 50)
    cache.append(k, v, i32(torch, [0, 50, 50]))
    got = cache.read(i32(torch, [0, 50, 50]), 50)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    assert cache.length.tolist() == [82, 10]
    cache.check()
    cache.evict(32, 4)                                     # of 110 tokens 10 are to come, of which sequence the host cannot tell
    assert cache.length.tolist() == [32, 10] and cache.free_pages == 8 - 3 - 1
    cache.check()


def test_pages_change_hands_many_times(torch, rc):
    """A random history of reservations, appends, evictions and releases beside what each sequence should hold."""
    rng = np.random.default_rng(5)
    batch, page, pages = 4, 16, 14
    cache = rc.KVCache(pages=pages, page=page, kv_heads=1, dim=64, batch=batch, max_tokens=128, kind="fp16")
    held = [np.zeros(0, np.int64) for _ in range(batch)]   # every token's own number, in places
    number = 0
    refused = 0
    for turn in range(150):
        what = rng.integers(0, 10)
        if what < 6:
            new = [int(x) for x in rng.integers(0, 30, batch)]
            if any(len(h) + n > 128 for h, n in zip(held, new)):
                continue
            try:
                cache.reserve(new)
            except rc.CacheError:
                refused += 1
                assert sum(-(-(len(h) + n) // page) for h, n in zip(held, new)) > pages
                continue
            total = sum(new)
            ids = np.arange(number, number + total)
            number += total
            rows = torch.from_numpy((ids % 2048).astype(np.float32))[:, None, None].expand(total, 1, 64).contiguous().cuda()
            starts = np.cumsum([0] + new)
            cache.append(rows, -rows, i32(torch, starts))
            held = [np.concatenate([h, ids[starts[b]:starts[b + 1]]]) for b, h in enumerate(held)]
        elif what < 9:
            budget = int(rng.integers(1, 60))
            cache.evict(budget, budget)                    # the newest stay, in the order of the moves
            for b, h in enumerate(held):
                if len(h) > budget:
                    newest = set(np.sort(h)[-budget:])
                    holes = [t for t in range(budget) if h[t] not in newest]
                    movers = [t for t in range(budget, len(h)) if h[t] in newest]
                    out = h[:budget].copy()
                    out[holes] = h[movers]
                    held[b] = out
        else:
            b = int(rng.integers(0, batch))
            cache.release(b)
            held[b] = held[b][:0]
        lens = [len(h) for h in held]
        assert cache.length.tolist() == lens
        assert cache.free_pages == pages - sum(-(-n // page) for n in lens)
        used = [p for b, n in enumerate(lens) for p in _pages_of(cache, b, n)]
        assert len(set(used)) == len(used) and all(0 <= p < pages for p in used)
        got = cache.read(i32(torch, np.cumsum([0] + lens)), sum(lens))[0][:, 0, 0].cpu().numpy()
        assert np.array_equal(got, np.concatenate(held).astype(np.int64) % 2048)
        cache.check()
    assert refused > 3


def test_a_step_at_the_budget_does_not_wait_for_the_gpu(torch, rc):
    """Budget a multiple of the page: the page that an eviction frees is the one that the next token takes."""
    cache = rc.KVCache(pages=20, page=16, kv_heads=2, dim=64, batch=3, max_tokens=512)
    q = torch.randn(3, 8, 64, device="cuda").bfloat16()
    k, v = _rows(torch, 3)

    def step():
        cache.reserve([1] * 3)
        cache.append(k, v)
        cache.attend(q, weigh=True)
        cache.evict(48, 8)

    for _ in range(52):
        step()
    torch.cuda.synchronize()
    before = cache.table.clone()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(40):
            step()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert torch.equal(cache.table, before) and cache.length.tolist() == [48] * 3 and cache.seen.tolist() == [92] * 3
    cache.check()


def test_new_pages_do_not_wait_for_the_gpu(torch, rc):
    cache = rc.KVCache(pages=60, page=16, kv_heads=2, dim=64, batch=3, max_tokens=320)
    cache.reserve([1, 0, 0])
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(12):
            cache.reserve([17, 3, 20])
    finally:
        torch.cuda.set_sync_debug_mode("default")
    used = [p for b, n in enumerate(cache.most) for p in _pages_of(cache, b, n)]
    assert cache.most == [205, 36, 240] and len(set(used)) == len(used) == 13 + 3 + 15 and min(used) >= 0


def test_a_captured_step_of_a_cache_with_pages_of_its_own(torch, rc):
    """Append, attention and eviction of two sequences, some turns as they are and then replayed from a graph, while a third
    one holds all pages that are free; the oracle goes along."""
    budget, recent, steps = 48, 8, 40
    cache = rc.KVCache(pages=11, page=16, kv_heads=2, dim=64, batch=3, max_tokens=176, kind="fp16")
    now = [torch.zeros(n, h, 64, device="cuda", dtype=torch.float16) for n, h in ((2, 2), (2, 2), (3, 4))]
    starts = i32(torch, [0, 1, 2, 2])
    cache.reserve([60, 60, 0])                             # 4 pages each

    def step():
        cache.append(now[0], now[1], starts)
        out = cache.attend(now[2], weigh=True)[0]
        cache.evict(budget, recent)
        return out

    # what each sequence and kv head should hold, in places
    hold = [[dict(k=np.zeros((0, 64)), v=np.zeros((0, 64)), w=np.zeros(0), p=np.zeros(0, int)) for _ in range(2)] for _ in range(2)]

    def follow(seen, out):
        k, v, q = (x.double().cpu().numpy() for x in now)
        for b in range(2):
            for h in range(2):
                s = hold[b][h]
                s["k"], s["v"] = np.vstack([s["k"], k[b, h]]), np.vstack([s["v"], v[b, h]])
                s["w"], s["p"] = np.append(s["w"], 0.0), np.append(s["p"], seen)
                want, _, share, size = orc.attend(q[b, 2 * h:2 * h + 2], s["k"][None], s["v"][None], 0.125)
                got = out[b, 2 * h:2 * h + 2].double().cpu().numpy()
                assert (np.abs(got - want) <= 2.0 ** -10 * size + 2.0 ** -24).all()
                s["w"] = s["w"] + share[0]
                n = len(s["p"])
                if n > budget:
                    # the kept ones by the cache's own weights: fp32 sums may part near ties the other way
                    pages = torch.tensor(_pages_of(cache, b, budget)).cuda()
                    place = cache.position[pages][:, h].reshape(-1)[:budget].cpu().numpy()
                    assert set(range(seen + 1 - recent, seen + 1)) <= set(place.tolist())
                    gone = sorted(set(s["p"].tolist()) - set(place.tolist()))
                    assert len(gone) == n - budget
                    for g in gone:
                        i = int(np.nonzero(s["p"] == g)[0][0])
                        old = s["p"] < seen + 1 - recent
                        assert old[i] and s["w"][i] <= s["w"][old].min() * (1 + 1e-5)
                        for name in s:                     # the last place moves into the freed one
                            if i < budget:
                                s[name][i] = s[name][-1]
                            s[name] = s[name][:-1]
                    assert np.array_equal(place, s["p"])

    gen = torch.Generator(device="cuda").manual_seed(7)
    graph, out = None, None
    for i in range(50 + steps):
        for x in now:
            x.normal_(generator=gen)
        if i < 50:
            out = step()
        else:
            if graph is None:
                cache.reserve([0, 0, 48])
                third = [r.half() for r in _rows(torch, 48)]
                cache.append(*third, i32(torch, [0, 0, 0, 48]))
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                before = cache.length.tolist(), cache.free_pages, cache.most
                with torch.cuda.graph(graph):
                    out = step()
                assert (cache.length.tolist(), cache.free_pages, cache.most) == before      # nothing ran, nothing is given back
            graph.replay()
        torch.cuda.synchronize()
        follow(i, out)
    assert cache.length.tolist() == [budget, budget, 48] and cache.seen.tolist() == [50 + steps, 50 + steps, 48]
    got = cache.read(i32(torch, [0, 0, 0, 48]), 48)
    assert torch.equal(got[0], third[0]) and torch.equal(got[1], third[1])
    cache.check()


def test_a_layer_lets_its_sequences_grow_by_the_slack_whatever_is_reserved(torch, rc):
    """Pages reserved ahead are not tokens: evictions come when budget + slack are passed."""
    import rans_model as rm

    class Same(torch.nn.Module):
        def __init__(self, rows):
            super().__init__()
            self.out_features, self.in_features = rows, 128

        def forward(self, x):
            return x[:, :self.out_features]

    cache = rc.KVCache(pages=20, page=16, kv_heads=1, dim=64, batch=2, max_tokens=160)
    layer = rm.RansAttention(Same(128), Same(64), Same(64), Same(128), cache, 2, budget=24, recent=8, slack=4)
    cache.reserve([100, 60])
    lens = []
    for _ in range(45):
        layer(torch.randn(2, 128, device="cuda").bfloat16())
        lens.append(cache.length.tolist())
        assert cache.held == lens[-1]
    want = list(range(1, 29)) + [24, 25, 26, 27, 28] * 4
    assert lens == [[n, n] for n in want[:45]]
    cache.check()


# ------------------------------------------------------------------ eviction's workspace
def test_evicting_to_more_than_the_table_holds(torch, rc):
    """Nothing can be over such a budget: no lists of that size are kept."""
    cache, _, _ = fill(torch, rc, [100, 64], 2, 64, 16, "bf16")
    cache.weight.uniform_()
    before = cache.k.clone(), torch.cuda.memory_allocated()
    for budget in (10 ** 6, 2 ** 31 - 1, 112):
        cache.evict(budget, 5)
    assert torch.equal(torch.nan_to_num(cache.k), torch.nan_to_num(before[0])) and cache.length.tolist() == [100, 64]
    assert torch.cuda.memory_allocated() - before[1] < 1 << 20
    cache.check()


# ------------------------------------------------------------------ sharing
@pytest.mark.parametrize("kind", ["bf16", "mxfp4"])
def test_attend_over_shared_pages(torch, rc, kind):
    """Two sequences with the same first pages, as after a fork, and one that is all of another's."""
    cache, truth, table = fill(torch, rc, [100, 70, 48], 2, 128, 16, kind, seed=6)
    table = table.copy()
    table[1, :3] = table[0, :3]                            # 48 tokens in common
    table[2, :3] = table[0, :3]
    for name in "kv":
        truth[name][1] = np.concatenate([truth[name][0][:, :48], truth[name][1][:, 48:]], 1)
        truth[name][2] = truth[name][0][:, :48]
    cache.table.copy_(torch.from_numpy(table))
    q = torch.randn(3, 8, 128, device="cuda").bfloat16()
    check_attend(torch, cache, truth, q, [100, 70, 48], 0.03, cache.attend(q, scale=0.03))
    cache.check()


def test_two_caches_on_two_streams(torch, rc):
    """Caches share nothing: the same passes side by side give the bits that they give alone."""
    lens = [3000, 17, 900]
    made = [fill(torch, rc, lens, 2, 128, 16, kind, seed=s)[0] for s, kind in ((1, "bf16"), (2, "mxfp4"))]
    q = torch.randn(3, 8, 128, device="cuda").bfloat16()
    alone = []
    for cache in made:
        for _ in range(20):
            out, log_sum = cache.attend(q, weigh=True)
        alone.append((out, log_sum, cache.weight.clone()))
        cache.weight.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    got = [None, None]
    for _ in range(20):
        for i, (cache, stream) in enumerate(zip(made, streams)):
            with torch.cuda.stream(stream):
                got[i] = cache.attend(q, weigh=True)
    torch.cuda.synchronize()
    for cache, one, two in zip(made, alone, got):
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1]) and torch.equal(one[2], cache.weight)
