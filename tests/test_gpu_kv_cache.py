"""GPU: the paged key-value cache (append, read, attend, evict) against the 64-bit oracle on the same stored values.

Tolerances, from the operations.  u is the unit roundoff of the 16-bit type that probabilities and outputs are rounded
to (bf16 2^-8; fp16 2^-11; 4-bit rows: bf16 probabilities).  Scores are sums of dim fp32 products: their error is at most
delta = 2^-21 (sum |q k| scale + 1), and a probability's relative error at most 2 delta + 2^-20.  So an output is within
(u_p + u_out + 2 delta + 2^-20) sum p |v| of the oracle's; fp16 probabilities below 2^-14 add n 2^-25 max |v|.  What lies
below the formats' smallest numbers adds n 2^-126 max |v| (fp32 probabilities) and 2^-133 (bf16 outputs).
"""
import numpy as np
import pytest

from oracle import kv_oracle as orc

pytestmark = pytest.mark.gpu

BF16, FP16 = 2.0 ** -8, 2.0 ** -11


@pytest.fixture(scope="module")
def torch(cuda_ok):
    import torch as t
    import rans_b200
    rans_b200.load()
    return t


@pytest.fixture(autouse=True)
def seeded(torch):
    torch.manual_seed(1)


@pytest.fixture(scope="module")
def rc():
    import rans_cache
    return rans_cache


def fill(torch, rc, lens, kv_heads, dim, page, kind, seed=0, spread=1.0, tail=2, layout="head", exponents=None, cols=1):
    """A cache over tensors whose unused slots and pages hold NaN, and the stored rows of each sequence in 64 bits."""
    rng = np.random.default_rng(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + tail
    order = rng.permutation(pages)
    cols = max(max(need) + 1, cols)
    table = np.full((len(lens), cols), -1, np.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    rows = {}
    truth = {"k": [], "v": []}
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16}.get(kind)
    for name in "kv":
        full = rng.standard_normal((pages, kv_heads, page, dim)) * spread
        used = np.zeros((pages, page), bool)
        for b, n in enumerate(lens):
            for i in range(need[b]):
                used[table[b, i], :min(page, n - i * page)] = True
        if kind == "mxfp4":
            e = rng.integers(-6, 7, (pages, kv_heads, page, dim // 32))
            if name == "v" and exponents is not None:
                for b, n in enumerate(lens):
                    for t in range(n):
                        e[table[b, t // page], :, t % page] = exponents(rng, t, e.shape[1::2])
            full = full * np.exp2(e.repeat(32, -1))
            index, scale = orc.quantise(full)
            stored = orc.values(index, scale)
            scale[~used[:, None, :].repeat(kv_heads, 1)] = 255
            rows[name] = torch.from_numpy(orc.pack(index)).cuda()
            rows[name + "_scale"] = torch.from_numpy(scale).cuda()
        else:
            t = torch.from_numpy(full).to(dtype)
            stored = t.double().numpy()
            t[torch.from_numpy(~used)[:, None, :].repeat(1, kv_heads, 1)] = float("nan")
            if layout == "token":           # [pages, page, kv_heads, dim] memory
                t = t.transpose(1, 2).contiguous().cuda().transpose(1, 2)
            elif layout == "wide":          # rows apart by more than their size, pages by more than their rows
                big = torch.full((pages, kv_heads + 1, page, dim + 8), float("nan"), dtype=dtype).cuda()
                big[:, :kv_heads, :, :dim] = t.cuda()
                t = big[:, :kv_heads, :, :dim]
            rows[name] = t.cuda()
        for b, n in enumerate(lens):
            x = stored[table[b, :need[b]]].transpose(1, 0, 2, 3).reshape(kv_heads, need[b] * page, dim)[:, :n]
            truth[name].append(x)
    i32 = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()     # noqa: E731
    weight = torch.zeros(pages, kv_heads, page, device="cuda")
    position = torch.zeros(pages, kv_heads, page, dtype=torch.int32, device="cuda")
    cache = rc.KVCache.from_tensors(rows["k"], rows["v"], i32(table), i32(lens), i32(lens), weight, position,
                                    rows.get("k_scale"), rows.get("v_scale"))
    return cache, truth, table


def check_attend(torch, cache, truth, q, lens, scale, got, weight=None, table=None, before=0.0, floor=0.0):
    out, log_sum = got[0].double().cpu().numpy(), got[1].double().cpu().numpy()
    qn = q.double().cpu().numpy()
    u_out = FP16 if q.dtype == torch.float16 else BF16
    u_p = FP16 if cache.kind == "fp16" else BF16
    w = None if weight is None else weight.double().cpu().numpy()
    for b, n in enumerate(lens):
        k, v = truth["k"][b], truth["v"][b]
        want, ls, share, size = orc.attend(qn[b], k, v, scale)
        if n == 0:
            assert (out[b] == 0).all() and np.isneginf(log_sum[b]).all()
            continue
        group = q.shape[1] // cache.kv_heads
        reach = np.einsum("hgd,hnd->hgn", np.abs(qn[b]).reshape(cache.kv_heads, group, -1), np.abs(k)) * abs(scale)
        delta = 2.0 ** -21 * (reach.max() + 1)
        bound = (u_p + u_out + 2 * delta + 2.0 ** -20) * size
        if cache.kind == "fp16":
            bound = bound + n * 2.0 ** -25 * np.abs(v).max()
        bound = bound + floor * np.repeat(np.abs(v).sum(1), group, axis=0)
        bound = bound + n * 2.0 ** -126 * np.abs(v).max() + (2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -133)
        assert (np.abs(out[b] - want) <= bound).all(), (b, n, (np.abs(out[b] - want) / bound).max())
        assert np.abs(log_sum[b] - ls).max() <= delta + 2.0 ** -20 * (1 + np.abs(ls).max())
        if w is not None:
            t = np.arange(n)
            mine = w[table[b, t // cache.page], :, t % cache.page].T
            err = np.abs(mine - before - share)
            assert (err <= (2 * delta + 2.0 ** -18) * share + 2.0 ** -23 * (before + share) + 1e-12).all()


LENS = [0, 1, 15, 16, 17, 31, 33, 64, 100, 257, 1000, 0]


@pytest.mark.parametrize("kind", ["bf16", "fp16", "mxfp4"])
@pytest.mark.parametrize("dim,heads,kv_heads,page", [(64, 8, 8, 16), (64, 6, 2, 32), (64, 48, 4, 16), (128, 12, 2, 16), (128, 8, 1, 64),
                                                     (128, 20, 2, 48), (128, 33, 1, 16), (256, 16, 1, 16), (256, 6, 2, 128)])
def test_attend(torch, rc, kind, dim, heads, kv_heads, page):
    cache, truth, table = fill(torch, rc, LENS, kv_heads, dim, page, kind, seed=dim + heads)
    q = torch.randn(len(LENS), heads, dim, device="cuda").to(torch.float16 if kind == "fp16" else torch.bfloat16)
    scale = dim ** -0.5 * (0.2 if kind == "mxfp4" else 1.0)
    check_attend(torch, cache, truth, q, LENS, scale, cache.attend(q, scale=scale))
    cache.weight.fill_(0.25)
    got = cache.attend(q, scale=scale, weigh=True)
    check_attend(torch, cache, truth, q, LENS, scale, got, cache.weight, table, before=0.25)
    cache.check()


@pytest.mark.parametrize("kind", ["bf16", "mxfp4"])
@pytest.mark.parametrize("lens", [[1], [16], [129], [4097], [20000], [3, 9001], [1] * 300, [40, 0, 0, 5000, 1, 0]])
def test_attend_lengths(torch, rc, kind, lens):
    """Few and many blocks a sequence, parts that end inside a warp's run, more sequences than blocks."""
    cache, truth, table = fill(torch, rc, lens, 2, 128, 16, kind, seed=len(lens) + lens[0])
    q = torch.randn(len(lens), 14, 128, device="cuda").bfloat16()
    got = cache.attend(q, scale=0.05, weigh=True)
    check_attend(torch, cache, truth, q, lens, 0.05, got, cache.weight, table)
    again = cache.attend(q, scale=0.05)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])        # joins do not depend on the order of blocks
    cache.check()


@pytest.mark.parametrize("q_type", ["bf16", "fp16"])
def test_attend_over_4_bits_takes_both_query_types(torch, rc, q_type):
    lens = [300, 5]
    cache, truth, _ = fill(torch, rc, lens, 2, 128, 32, "mxfp4", seed=9)
    q = (torch.randn(2, 8, 128, device="cuda") * torch.tensor([[[1e-3]], [[100.0]]], device="cuda"))
    q = q.to(torch.float16 if q_type == "fp16" else torch.bfloat16)
    check_attend(torch, cache, truth, q, lens, 0.01, cache.attend(q, scale=0.01))


APART = {
    "far apart": lambda rng, t, shape: rng.integers(-60, 60, shape),
    "rising": lambda rng, t, shape: np.full(shape, min(-50 + t // 3, 55)),
    "falling": lambda rng, t, shape: np.full(shape, max(50 - t // 3, -55)),
    "one large": lambda rng, t, shape: np.full(shape, 40 if t == 37 else -1),
    "one small": lambda rng, t, shape: np.full(shape, -50 if t == 21 else 2),
    "blocks apart": lambda rng, t, shape: np.broadcast_to(np.arange(shape[1]) * 12 - 20, shape),
    "zeros": lambda rng, t, shape: np.full(shape, -63 if t % 2 else 3),
}


@pytest.mark.parametrize("exponents", list(APART))
@pytest.mark.parametrize("dim,heads", [(64, 4), (128, 8), (128, 24), (256, 8)])
def test_attend_over_4_bit_values_of_very_different_scales(torch, rc, exponents, dim, heads):
    """Tiles inside and outside what fp16 operands take, in both directions, and the units that O is held in.  Probabilities
    in fp16 are whole multiples of 2^-24 where the largest is at least 2^11 (the kernel keeps it between 2^0 and 2^15, and
    above 2^11 at the last rise): each is off by up to 2^-36 of the largest, which shows where the tokens that dominate hold
    zeros in a column."""
    lens = [45, 333, 16, 1]
    cache, truth, table = fill(torch, rc, lens, 2, dim, 16, "mxfp4", seed=dim, exponents=APART[exponents])
    q = torch.randn(len(lens), heads, dim, device="cuda").bfloat16()
    got = cache.attend(q, scale=0.05, weigh=True)
    check_attend(torch, cache, truth, q, lens, 0.05, got, cache.weight, table, floor=2.0 ** -36)


@pytest.mark.parametrize("layout", ["token", "wide"])
def test_attend_strides(torch, rc, layout):
    lens = [50, 333, 0]
    cache, truth, table = fill(torch, rc, lens, 3, 128, 16, "bf16", seed=4, layout=layout)
    q = torch.randn(3, 2, 12, 128, device="cuda").bfloat16()[:, 1]                # a strided query
    got = cache.attend(q, weigh=True)
    check_attend(torch, cache, truth, q, lens, 128 ** -0.5, got, cache.weight, table)
    odd = torch.randn(3, 12, 129, device="cuda").bfloat16()[:, :, 1:]             # unaligned: copied
    check_attend(torch, cache, truth, odd, lens, 128 ** -0.5, cache.attend(odd))


def test_attend_sharp_and_flat(torch, rc):
    """Scores far apart (one token takes all, the maximum rising late) and all equal."""
    lens = [700, 700]
    cache, truth, table = fill(torch, rc, lens, 1, 64, 16, "bf16", seed=2)
    k = torch.zeros(cache.k.shape).bfloat16()
    for b in range(2):
        for t in range(700):
            k[table[b, t // 16], 0, t % 16, 0] = t / 16 if b == 0 else 1.0
            truth["k"][b][0, t] = 0
            truth["k"][b][0, t, 0] = float(k[table[b, t // 16], 0, t % 16, 0])
    cache.k.copy_(k)
    q = torch.zeros(2, 4, 64, device="cuda").bfloat16()
    q[:, :, 0] = torch.tensor([1.0, 8.0, -8.0, 0.0])
    got = cache.attend(q, scale=4.0, weigh=True)
    check_attend(torch, cache, truth, q, lens, 4.0, got, cache.weight, table)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "mxfp4"])
def test_attend_carries_nan_and_infinity_of_its_own_tokens_only(torch, rc, kind):
    lens = [40, 40]
    cache, truth, table = fill(torch, rc, lens, 2, 64, 16, kind, seed=5)
    page, slot = table[0, 1], 3
    if kind == "mxfp4":
        cache.v[page, 1, slot] = 0
        cache.v_scale[page, 1, slot, 0] = 255
    else:
        cache.v[page, 1, slot, 5] = float("nan")
    q = torch.randn(2, 4, 64, device="cuda").to(torch.float16 if kind == "fp16" else torch.bfloat16)
    out, log_sum = cache.attend(q)
    assert torch.isfinite(out[1]).all() and torch.isfinite(out[0, :2]).all() and torch.isfinite(log_sum).all()
    bad = torch.isnan(out[0, 2:])
    assert bad[:, :32].all() and not bad[:, 32:].any() if kind == "mxfp4" else bad[:, 5].all() and int(bad.sum()) == 2
    if kind != "mxfp4":
        # keys of -infinity in one channel: every score of a query that is positive there is -infinity
        cache.v[page, 1, slot, 5] = 0
        for i in range(3):
            cache.k[table[0, i], 0, :, 0] = -float("inf")
        q[0, :2, 0] = 1.0
        out, log_sum = cache.attend(q)
        assert (out[0, :2] == 0).all() and torch.isneginf(log_sum[0, :2]).all()
        assert torch.isfinite(out[0, 2:]).all()


def test_attend_past_4_gigabytes(torch, rc):
    """Pages whose byte offsets need more than 32 bits, in the cache and in the weights' scores."""
    pages, kv, page, dim = 36000, 8, 64, 128                # a page is 128 KB: offsets pass 2^32 from page 32768 on
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB of free memory")
    k = torch.empty(pages, kv, page, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    used = torch.tensor([35999, 1, 33000, 32768], dtype=torch.int32, device="cuda")
    for x in (k, v):
        x[used.long()] = torch.randn(4, kv, page, dim, device="cuda").bfloat16()
    n = 250
    one = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")     # noqa: E731
    cache = rc.KVCache.from_tensors(k, v, used[None].contiguous(), one(n), one(n))
    truth = {name: [x[used.long()].transpose(0, 1).reshape(kv, 4 * page, dim)[:, :n].double().cpu().numpy()]
             for name, x in (("k", k), ("v", v))}
    q = torch.randn(1, 64, dim, device="cuda").bfloat16()
    check_attend(torch, cache, truth, q, [n], dim ** -0.5, cache.attend(q))
    cache.append(torch.ones(1, kv, dim, device="cuda"), torch.ones(1, kv, dim, device="cuda") * 2)
    assert (v[32768, :, 250 % 64] == 2).all() and int(cache.length) == 251


def test_4_bit_pages_past_4_gigabytes(torch, rc):
    """Every operator on 4-bit pages whose byte offsets need more than 32 bits."""
    pages, kv, page, dim = 70000, 8, 64, 256                # a page is 64 KB: offsets pass 2^32 from page 65536 on
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB of free memory")
    empty = lambda last, dtype=torch.uint8: torch.empty(pages, kv, page, *last, dtype=dtype, device="cuda")     # noqa: E731
    table = torch.tensor([[69999, 3, 65537, 68000]], dtype=torch.int32, device="cuda")
    zero = lambda: torch.zeros(1, dtype=torch.int32, device="cuda")     # noqa: E731
    cache = rc.KVCache.from_tensors(empty([128]), empty([128]), table, zero(), zero(), empty([], torch.float32),
                                    empty([], torch.int32), empty([8]), empty([8]))
    n = 250
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(n, kv, dim, device="cuda").bfloat16() for _ in range(2))
    cache.append(k, v, starts)
    truth = {}
    for name, x, got in (("k", k, cache.read(starts, n)[0]), ("v", v, cache.read(starts, n)[1])):
        want = orc.values(*orc.quantise(x.double().cpu().numpy()))
        assert np.array_equal(got.double().cpu().numpy(), want)
        truth[name] = [want.transpose(1, 0, 2)]
    q = torch.randn(1, 16, dim, device="cuda").bfloat16()
    got = cache.attend(q, weigh=True)
    check_attend(torch, cache, truth, q, [n], dim ** -0.5, got, cache.weight, table.cpu().numpy())
    cache.weight[table[0].long()] = torch.rand(4, kv, page, device="cuda")
    weight = cache.weight[table[0].long()].transpose(0, 1).reshape(kv, -1).cpu().numpy()
    cache.evict(130, 20)
    left = torch.tensor([0, 130], dtype=torch.int32, device="cuda")
    k2 = cache.read(left, 130)[0].double().cpu().numpy()
    position = cache.position[table[0].long()].transpose(0, 1).reshape(kv, -1).cpu().numpy()
    for h in range(kv):
        order = np.arange(n)
        for to, of in orc.evict_moves(weight[h, :n], np.arange(n), n, 130, 20):
            order[to] = of
        assert np.array_equal(position[h, :130], order[:130])
        assert np.array_equal(k2[:, h], truth["k"][0][h][order[:130]])
    cache.check()


# ------------------------------------------------------------------ append, read
@pytest.mark.parametrize("kind", ["bf16", "fp16", "mxfp4"])
@pytest.mark.parametrize("given", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dim,kv_heads,counts", [(128, 2, [1, 1, 1]), (64, 3, [0, 5, 40]), (256, 1, [17, 0, 100]), (128, 8, [333, 1, 0])])
def test_append_and_read(torch, rc, kind, given, dim, kv_heads, counts):
    start = [0, 7, 30]
    page = 16
    cache = rc.KVCache(pages=64, page=page, kv_heads=kv_heads, dim=dim, batch=3, max_tokens=512, kind=kind)
    gen = torch.Generator(device="cuda").manual_seed(dim + sum(counts))
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[given]
    make = lambda n: [(torch.randn(n, kv_heads, dim, device="cuda", generator=gen) * 3).to(dtype) for _ in range(2)]   # noqa: E731
    starts = lambda c: torch.tensor(np.cumsum([0] + c), dtype=torch.int32, device="cuda")     # noqa: E731
    cache.reserve(start)
    first = make(sum(start))
    cache.append(*first, starts(start))
    cache.reserve(counts)
    k, v = make(sum(counts))
    if counts == [1, 1, 1]:
        cache.append(k, v)
        got = cache.read()
    else:
        wide = [torch.cat([x, x], 1)[:, kv_heads:] for x in (k, v)]         # a strided source
        cache.append(*wide, starts(counts))
        got = cache.read(starts(counts), sum(counts))
    for x, y in ((k, got[0]), (v, got[1])):
        if kind == "mxfp4":
            want = torch.from_numpy(orc.values(*orc.quantise(x.double().cpu().numpy())))
        else:
            want = x.to(torch.bfloat16 if kind == "bf16" else torch.float16).double().cpu()
        assert torch.equal(y.double().cpu(), want)
    total = [a + b for a, b in zip(start, counts)]
    assert cache.length.tolist() == total and cache.seen.tolist() == total
    table = cache.table.cpu()
    for b, n in enumerate(total):
        t = torch.arange(n)
        assert (cache.position.cpu()[table[b, t // page].long(), :, t % page] == t[:, None]).all()
    everything = cache.read(starts(total), sum(total))
    at = np.cumsum([0] + total)
    tail = torch.cat([everything[0][at[b + 1] - counts[b]:at[b + 1]] for b in range(3)])
    assert torch.equal(tail, got[0])
    cache.check()


def test_append_4_bits_of_every_kind_of_block(torch, rc):
    """Ties, saturation, zeros of both signs, tiny and huge blocks, infinities and NaN."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((64, 1, 128)).astype(np.float32)
    x[0] = 0.0
    x[1] = -0.0
    x[2, 0, :8] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5]
    x[3, 0, :9] = [7.9, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -7]
    x[4] *= 2.0 ** -70
    x[5] *= 2.0 ** 70
    x[6] = 1e-41
    x[7, 0, 3] = np.inf
    x[8, 0, 40] = -np.inf
    x[9, 0, 127] = np.nan
    x[10] = 3.0e38
    x[11:40] = np.round(x[11:40] * 8) / 4                    # many ties
    cache = rc.KVCache(pages=8, page=16, kv_heads=1, dim=128, batch=1, max_tokens=64, kind="mxfp4")
    cache.reserve([64])
    starts = torch.tensor([0, 64], dtype=torch.int32, device="cuda")
    t = torch.from_numpy(x).cuda()
    cache.append(t, -t, starts)
    for sign, y, codes, scales in ((1, cache.read(starts, 64)[0], cache.k, cache.k_scale), (-1, cache.read(starts, 64)[1], cache.v, cache.v_scale)):
        index, scale = orc.quantise(sign * x.astype(np.float64))
        want = orc.values(index, scale)
        assert np.array_equal(y.double().cpu().numpy(), want, equal_nan=True)
        pages = cache.table[0, :4].long()
        assert np.array_equal(scales[pages].reshape(64, 1, 4).cpu().numpy(), scale)
        assert np.array_equal(codes[pages].reshape(64, 1, 64).cpu().numpy(), orc.pack(index))


# ------------------------------------------------------------------ evict
def _evict_case(torch, rc, lens, kv_heads, dim, page, kind, weights, budget, recent, seed=0, cols=1):
    cache, truth, table = fill(torch, rc, lens, kv_heads, dim, page, kind, seed=seed, cols=cols)
    rng = np.random.default_rng(seed)
    w = np.full(cache.weight.shape, np.nan, np.float32)
    pos = np.full(cache.weight.shape, 1 << 30, np.int32)
    for b, n in enumerate(lens):
        for t in range(n):
            for h in range(kv_heads):
                w[table[b, t // page], h, t % page] = weights(rng, b, h, t)
                pos[table[b, t // page], h, t % page] = 2 * t + h           # gaps, as after earlier evictions
    cache.weight.copy_(torch.from_numpy(w))
    cache.position.copy_(torch.from_numpy(pos))
    seen = [2 * n + 3 for n in lens]
    cache.seen.copy_(torch.tensor(seen, dtype=torch.int32))
    names = [n for n in ("k", "v", "k_scale", "v_scale", "weight", "position") if getattr(cache, n) is not None]
    raw = lambda x: x.cpu().contiguous().view(torch.uint8).numpy().copy()    # noqa: E731
    want = {n: raw(getattr(cache, n)) for n in names}
    for b, n in enumerate(lens):
        at = lambda t: (table[b, t // page], h, t % page)                    # noqa: E731
        for h in range(kv_heads):
            t = np.arange(n)
            moves = orc.evict_moves(w[table[b, t // page], h, t % page], pos[table[b, t // page], h, t % page], seen[b], budget, recent)
            for name in names:
                x = want[name].reshape(*cache.weight.shape, -1)
                old = x.copy()
                for to, of in moves:
                    x[at(to)] = old[at(of)]
    cache.evict(budget, recent)
    cache.check()
    assert cache.length.tolist() == [min(n, budget) for n in lens]
    for name in names:
        assert np.array_equal(raw(getattr(cache, name)).reshape(-1), want[name].reshape(-1)), name


SOME = {
    "random": lambda rng, b, h, t: rng.exponential(),
    "equal": lambda rng, b, h, t: 1.0,
    "few values": lambda rng, b, h, t: float(rng.integers(0, 3)),
    "zeros of both signs": lambda rng, b, h, t: [0.0, -0.0][int(rng.integers(0, 2))],
    "odd": lambda rng, b, h, t: [np.nan, np.inf, -np.inf, -1.0, 1e-45, 3e38, 0.5][int(rng.integers(0, 7))],
    "rising": lambda rng, b, h, t: float(t),
    "close": lambda rng, b, h, t: np.float32(1.0) + np.float32(2.0 ** -23) * np.float32(rng.integers(0, 1000)),
}


@pytest.mark.parametrize("weights", list(SOME))
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (7, 3), (32, 0), (100, 100), (255, 40)])
def test_evict(torch, rc, weights, budget, recent):
    _evict_case(torch, rc, [0, 1, budget, budget + 1, 300], 2, 64, 16, "bf16", SOME[weights], budget, recent, seed=budget)


@pytest.mark.parametrize("weights", list(SOME))
@pytest.mark.parametrize("budget,recent", [(1, 1), (5, 0), (64, 60), (200, 3)])
def test_evict_a_few(torch, rc, weights, budget, recent):
    """One to five tokens over the budget: the search one by one and the first one beyond it."""
    _evict_case(torch, rc, [budget + i for i in range(1, 6)], 2, 64, 16, "bf16", SOME[weights], budget, recent, seed=budget)


@pytest.mark.parametrize("over", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("weights", ["random", "equal", "few values"])
def test_evict_a_few_of_many(torch, rc, over, weights):
    """The same with several blocks to a head."""
    _evict_case(torch, rc, [30000 + over], 1, 64, 64, "fp16", SOME[weights], 30000, 100, seed=over)


@pytest.mark.parametrize("kind,dim,page", [("fp16", 128, 32), ("mxfp4", 64, 16), ("mxfp4", 128, 48), ("mxfp4", 256, 16), ("bf16", 256, 64)])
def test_evict_kinds(torch, rc, kind, dim, page):
    _evict_case(torch, rc, [200, 90, 33], 3, dim, page, kind, SOME["random"], 60, 16)


@pytest.mark.parametrize("n,budget", [(20000, 5000), (33333, 33332), (60000, 1)])
def test_evict_long(torch, rc, n, budget):
    _evict_case(torch, rc, [n], 1, 64, 64, "bf16", SOME["random"], budget, min(64, budget))


@pytest.mark.parametrize("kind,dim", [("bf16", 256), ("fp16", 256)])
def test_evict_many_rows_of_few_heads(torch, rc, kind, dim):
    """Enough rows for the moves to get a grid of their own (32 MB over 8 heads, by the table's room)."""
    _evict_case(torch, rc, [6000], 8, dim, 64, kind, SOME["random"], 4096, 64, cols=129)


@pytest.mark.parametrize("weights", ["random", "few values"])
def test_evict_with_keys_in_the_workspace(torch, rc, weights):
    """More places in the table than a block's shared memory has keys for, over more heads than there are SMs for clusters."""
    _evict_case(torch, rc, [150, 33, 0], 30, 64, 16, "bf16", SOME[weights], 50, 10, cols=2700)
    _evict_case(torch, rc, [52], 150, 64, 16, "bf16", SOME[weights], 50, 10, cols=2700)


def test_evicting_again_moves_nothing(torch, rc):
    cache, _, _ = fill(torch, rc, [100], 2, 64, 16, "bf16")
    cache.weight.uniform_()
    cache.evict(50, 5)
    before = [cache.k.clone(), cache.weight.clone(), cache.position.clone()]
    cache.evict(50, 5)
    assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(before, (cache.k, cache.weight, cache.position)))


# ------------------------------------------------------------------ the cache as a whole
def test_pages_are_handed_out_and_come_back(torch, rc):
    cache = rc.KVCache(pages=6, page=16, kv_heads=1, dim=64, batch=2, max_tokens=64)
    cache.reserve([33, 1])
    assert cache.free_pages == 2
    with pytest.raises(rc.CacheError):
        cache.reserve([0, 48])
    with pytest.raises(ValueError):
        cache.reserve([32, 0])              # past max_tokens
    assert cache.free_pages == 2
    starts = torch.tensor([0, 33, 34], dtype=torch.int32, device="cuda")
    cache.append(torch.randn(34, 1, 64, device="cuda"), torch.randn(34, 1, 64, device="cuda"), starts)
    cache.evict(16, 4)
    assert cache.free_pages == 4 and cache.length.tolist() == [16, 1]
    cache.reserve([1, 0])
    assert cache.free_pages == 3
    cache.release(0)
    assert cache.free_pages == 5 and cache.length.tolist() == [0, 1] and cache.seen.tolist() == [0, 1]
    cache.check()


def test_bad_pages_lengths_and_rows_are_left_out_and_reported(torch, rc):
    """What a kernel cannot follow it leaves out; check() says so once."""
    cache, truth, table = fill(torch, rc, [40, 20], 1, 64, 16, "bf16", seed=3)
    q = torch.randn(2, 2, 64, device="cuda").bfloat16()
    good = cache.attend(q)[0]
    for bad in (-1, 10 ** 6):
        cache.table[0, 1] = bad
        out, _ = cache.attend(q, weigh=True)
        assert torch.equal(out[1], good[1]) and torch.isfinite(out).all()
        some = {n: [np.concatenate([truth[n][0][:, :16], truth[n][0][:, 32:]], 1)] for n in "kv"}
        check_attend(torch, cache, some, q[:1], [24], 64 ** -0.5, [out[:1], cache.attend(q)[1][:1]])
        with pytest.raises(rc.CacheError, match="page"):
            cache.check()
        cache.check()
    cache.table[0, 1] = int(table[0, 1])
    cache.length[1] = 10 ** 6
    cache.append(torch.zeros(2, 1, 64, device="cuda"), torch.zeros(2, 1, 64, device="cuda"))
    with pytest.raises(rc.CacheError, match="length"):
        cache.check()
    cache.length.copy_(torch.tensor([40, -5]))
    assert (cache.attend(q)[0][1] == 0).all()
    with pytest.raises(rc.CacheError, match="length"):
        cache.check()
    cache.length.copy_(torch.tensor([40, 20]))
    cache.append(torch.zeros(3, 1, 64, device="cuda"), torch.zeros(3, 1, 64, device="cuda"),
                 torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"))
    with pytest.raises(rc.CacheError, match="rows"):
        cache.check()
    assert cache.length.tolist() == [41, 21]


def _decode(torch, rc, steps, graph):
    torch.manual_seed(1)
    cache = rc.KVCache(pages=40, page=16, kv_heads=2, dim=128, batch=3, max_tokens=160, kind="mxfp4")
    fed = [torch.randn(steps, 3, h, 128, device="cuda").bfloat16() for h in (2, 2, 8)]
    now = [x[0].clone() for x in fed]
    outs = []
    cache.reserve([100, 100, 100])

    def step():
        cache.append(now[0], now[1])
        out, _ = cache.attend(now[2], weigh=True)
        cache.evict(48, 8)
        return out

    g = out = None
    for i in range(steps):
        for a, x in zip(now, fed):
            a.copy_(x[i])
        if not graph or i == 0:
            out = step()
            cache.reserve([0, 0, 0])
        else:
            if g is None:
                torch.cuda.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    out = step()
            g.replay()
        cache._most = [100] * 3
        outs.append(out.clone())
    torch.cuda.synchronize()
    cache.check()
    return torch.stack(outs), cache.position.clone(), cache.weight.clone(), cache.length.tolist()


def test_decode_loop_in_a_graph_and_out(torch, rc):
    a, b = _decode(torch, rc, 70, False), _decode(torch, rc, 70, True)
    assert all(torch.equal(x, y) for x, y in zip(a[:3], b[:3])) and a[3] == b[3] == [48, 48, 48]


def test_another_stream(torch, rc):
    lens = [500, 3]
    cache, truth, table = fill(torch, rc, lens, 2, 128, 16, "bf16", seed=8)
    q = torch.randn(2, 8, 128, device="cuda").bfloat16()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = cache.attend(q, weigh=True)
    side.synchronize()
    check_attend(torch, cache, truth, q, lens, 128 ** -0.5, got, cache.weight, table)


def test_refusals(torch, rc):
    make = lambda **d: rc.KVCache(**{**dict(pages=4, page=16, kv_heads=2, dim=64, batch=2, max_tokens=32), **d})     # noqa: E731
    for d in (dict(page=8), dict(page=20), dict(dim=80), dict(kind="fp8"), dict(pages=0), dict(batch=0), dict(max_tokens=0)):
        with pytest.raises(ValueError):
            make(**d)
    c = make()
    rows = torch.zeros(2, 2, 64, device="cuda")
    for k, v, starts in ((rows[:1], rows[:1], None), (rows, rows[:, :1], None), (rows.double(), rows.double(), None), (rows, rows.half(), None),
                         (rows.cpu(), rows.cpu(), None), (rows, rows, torch.zeros(3, device="cuda")), (rows, rows, torch.zeros(2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            c.append(k, v, starts)
    q = torch.zeros(2, 4, 64, device="cuda").bfloat16()
    for x in (q[:1], q[:, :3], q.half(), q.float(), q.cpu(), q[..., :32]):
        with pytest.raises(ValueError):
            c.attend(x)
    for d in (dict(out=q.float()), dict(out=q[:, :2]), dict(log_sum=torch.zeros(2, 3, device="cuda"))):
        with pytest.raises(ValueError):
            c.attend(q, **d)
    for budget, recent in ((0, 0), (4, 5), (4, -1)):
        with pytest.raises(ValueError):
            c.evict(budget, recent)
    with pytest.raises(ValueError):
        c.read(torch.zeros(3, dtype=torch.int32, device="cuda"))
    bare = rc.KVCache.from_tensors(c.k, c.v, c.table, c.length, c.seen)
    for call in (lambda: bare.attend(q, weigh=True), lambda: bare.evict(4), lambda: bare.reserve([1, 1]), lambda: bare.release(0)):
        with pytest.raises(ValueError):
            call()
    f = rc.KVCache.from_tensors
    for args, more in (((c.k, c.v[:3], c.table, c.length, c.seen), {}), ((c.k[..., :60], c.v[..., :60], c.table, c.length, c.seen), {}),
                       ((c.k.float(), c.v.float(), c.table, c.length, c.seen), {}), ((c.k, c.v, c.table.long(), c.length, c.seen), {}),
                       ((c.k, c.v, c.table, c.length, c.seen[:1]), {}), ((c.k, c.v, c.table, c.length, c.seen), dict(weight=c.weight.half())),
                       ((c.k.cpu(), c.v.cpu(), c.table, c.length, c.seen), {}), ((c.k.view(torch.uint8), c.v.view(torch.uint8), c.table, c.length, c.seen), {}),
                       ((c.k[:, :, ::2], c.v, c.table, c.length, c.seen), {})):
        with pytest.raises(ValueError):
            f(*args, **more)
