"""The paged key-value cache's operators, as cases to be measured: appending tokens (16-bit or microscaled 4-bit
storage), attention of one new token per sequence over the pages (with or without the weight that each cached token
received), eviction by that weight, and a decode step of all three.

`run` computes them in a plain form from elementary torch operations, or with `own` through rans_cache.KVCache.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

GOLDEN = 0.6180339887498949
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step of four users of a small model: a token each into their caches; pure latency
        dict(name="append 4 tokens bf16", op="append", kind="bf16", given="bf16", batch=4, heads=12, kv_heads=2, dim=128,
             page=16, longest=1, shortest=1, held=777),
        # three prompts of uneven length, one of them empty, stored in 4 bits as a long-context service does
        dict(name="append prompts mxfp4", op="append", kind="mxfp4", given="bf16", batch=3, heads=64, kv_heads=8, dim=128,
             page=64, longest=8191, shortest=0, held=5),
        # a chat turn on a 1.5B-class model: one user, short history, odd group of six heads; latency
        dict(name="attend 1x777 g6 bf16", op="attend", kind="bf16", batch=1, heads=12, kv_heads=2, dim=128, page=16,
             longest=777, shortest=777, weigh=False),
        # one user of a 70B-class model with a long document
        dict(name="attend 1x32768 g8 bf16", op="attend", kind="bf16", batch=1, heads=64, kv_heads=8, dim=128, page=64,
             longest=32768, shortest=32768, weigh=False),
        # a full serving batch of uneven histories, one slot empty
        dict(name="attend 48 ragged g8 bf16", op="attend", kind="bf16", batch=48, heads=64, kv_heads=8, dim=128, page=64,
             longest=16384, shortest=0, weigh=False),
        # a small-head model without grouped heads, half precision
        dict(name="attend 16 ragged g1 d64 fp16", op="attend", kind="fp16", batch=16, heads=16, kv_heads=16, dim=64, page=32,
             longest=4099, shortest=1, weigh=False),
        # the longest context: a cache that only fits comfortably in 4 bits
        dict(name="attend 1x131071 g8 mxfp4", op="attend", kind="mxfp4", batch=1, heads=64, kv_heads=8, dim=128, page=64,
             longest=131071, shortest=131071, weigh=False),
        # a batch over a 4-bit cache
        dict(name="attend 32 ragged g8 mxfp4", op="attend", kind="mxfp4", batch=32, heads=64, kv_heads=8, dim=128, page=64,
             longest=16000, shortest=0, weigh=False),
        # attention that also keeps the books which eviction goes by
        dict(name="attend 8 ragged weights", op="attend", kind="bf16", batch=8, heads=64, kv_heads=8, dim=128, page=64,
             longest=9001, shortest=1, weigh=True),
        # a long prompt cut to a quarter once, before decoding goes on
        dict(name="evict 1x65536 to 16384", op="evict", kind="bf16", batch=1, heads=64, kv_heads=8, dim=128, page=64,
             longest=65536, shortest=65536, budget=16384, recent=256),
        # a batch that is brought back to its budget every 64 tokens
        dict(name="evict 32x4160 to 4096", op="evict", kind="bf16", batch=32, heads=12, kv_heads=2, dim=128, page=16,
             longest=4160, shortest=4160, budget=4096, recent=128),
        # a decode step at the budget: a token in, attention with weights, a token out
        dict(name="step 16x4096", op="step", kind="bf16", batch=16, heads=64, kv_heads=8, dim=128, page=64,
             longest=4096, shortest=4096, budget=4096, recent=64),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "evict", "step"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    case = dict(op=op, batch=_spread(rng, 1, 64), kv_heads=kv_heads, heads=kv_heads * rng.choice([1, 3, 4, 6, 7, 8, 8, 12, 16]),
                dim=dim, page=rng.choice([16, 32, 64, 128]))
    room = 400_000_000 // (case["batch"] * kv_heads * dim)     # tokens a sequence, so that no case is over the largest
    if op == "append":
        case.update(kind=rng.choice(["bf16", "fp16", "mxfp4"]), given=rng.choice(["bf16", "fp32"]),
                    longest=_spread(rng, 1, max(1, min(room // 16, 8191))), held=rng.randrange(200))
        case["shortest"] = rng.choice([0, 1, case["longest"]])
    elif op == "attend":
        case.update(kind=rng.choice(["bf16", "fp16", "mxfp4"]), longest=_spread(rng, 1, max(1, min(room, 131071))),
                    weigh=rng.random() < 0.3)
        case["shortest"] = rng.choice([0, 1, case["longest"]])
    else:
        case.update(kind=rng.choice(["bf16", "fp16"]), budget=_spread(rng, 8, max(8, min(room // 4, 16384))))
        case["recent"] = rng.randrange(case["budget"] // 2 + 1)
        case["longest"] = case["budget"] if op == "step" else case["budget"] + _spread(rng, 1, max(1, min(3 * case["budget"], 49152)))
        case["shortest"] = case["longest"] if op == "step" else rng.choice([1, case["budget"], case["longest"]])
    return case


def lengths(case):
    """Tokens of each sequence (new ones for `append`): uneven, the first the longest, the second the shortest."""
    low, high = case["shortest"], case["longest"]
    return [high if b == 0 else low if b == 1 else low + int((high - low + 1) * ((b * GOLDEN) % 1.0)) for b in range(case["batch"])]


def held(case):
    """Tokens of each sequence that are in the cache before the pass."""
    return [case["held"] + b % 7 for b in range(case["batch"])] if case["op"] == "append" else lengths(case)


def _row_bytes(case):
    return case["dim"] * 17 / 32 if case["kind"] == "mxfp4" else case["dim"] * 2


def work(case):
    n, row, hk, hq, dim = lengths(case), _row_bytes(case), case["kv_heads"], case["heads"], case["dim"]

    def append(tokens, size):
        # the rows in, the stored rows out, position and weight out
        return tokens * hk * (2 * dim * size + 2 * row + 8)

    def attend(lens, weigh):
        # every cached row in, queries in, outputs and log-sums out, accumulated weights in and out
        return sum(lens) * hk * (2 * row + (8 if weigh else 0)) + case["batch"] * hq * (4 * dim + 4), 4.0 * sum(lens) * hq * dim

    def evict(lens, budget, recent):
        total = 0.0
        for k in lens:
            if k > budget:
                late = min(recent, k - budget)
                moved = late + max(0, budget - recent) * max(0, k - budget - late) / max(1, k - recent)
                total += k * 8 + moved * (4 * row + 16)      # weights and positions in; the moved rows and books in and out
        return total * hk

    if case["op"] == "append":
        bytes_ = append(sum(n), 4 if case["given"] == "fp32" else 2)
        if case["kind"] == "mxfp4":
            bytes_ += sum(n) * hk * 2 * (row + 2 * dim)      # read back as bf16
        return {"bytes": bytes_, "flops": 0}
    if case["op"] == "attend":
        bytes_, flops = attend(n, case["weigh"])
        return {"bytes": bytes_, "flops": flops}
    if case["op"] == "evict":
        return {"bytes": evict(n, case["budget"], case["recent"]), "flops": 0}
    more = [k + 1 for k in n]
    bytes_, flops = attend(more, True)
    return {"bytes": bytes_ + append(case["batch"], 2) + evict(more, case["budget"], case["recent"]), "flops": flops}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    """Pages in shuffled order, filled as far as the sequences go and full of NaN elsewhere, and the new token's rows."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev)   # noqa: E731
    op, batch, hk, dim, page = case["op"], case["batch"], case["kv_heads"], case["dim"], case["page"]
    now, new = held(case), lengths(case) if op == "append" else [1] * batch if op == "step" else [0] * batch
    most = [-(-(a + b) // page) for a, b in zip(now, new)]
    pages = sum(most) + 1
    order = torch.randperm(pages, generator=gen, device=dev).int()
    table = torch.full((batch, max(max(most), 1)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, k in enumerate(most):
        table[b, :k] = order[at:at + k]
        at += k
    # length, seen and the books of the tokens in one buffer, so that one copy takes the cache back to where it was
    books = torch.zeros(2 * batch + 2 * pages * hk * page, dtype=torch.int32, device=dev)
    length, seen = books[:batch], books[batch:2 * batch]
    position, weight = books[2 * batch:].view(2, pages, hk, page)
    weight = weight.view(torch.float32)
    length.copy_(torch.tensor(now, dtype=torch.int32))
    seen.copy_(length)
    s = dict(case=case, table=table, books=books, length=length, seen=seen, position=position, weight=weight, scale=1 / math.sqrt(dim))
    inside = torch.arange(table.shape[1] * page, device=dev)[None, :] < length[:, None]
    filled = torch.zeros(pages, page, dtype=torch.bool, device=dev)
    real = table >= 0
    filled[table[real].long()] = inside.view(batch, -1, page)[real]
    where = torch.zeros(pages, page, dtype=torch.int32, device=dev)
    where[table[real].long()] = torch.arange(table.shape[1] * page, dtype=torch.int32, device=dev).view(1, -1, page).expand(batch, -1, -1)[real]
    position.copy_(where[:, None, :].expand(-1, hk, -1))
    # some tokens are attended to far more than others
    weight.copy_(torch.where(filled[:, None, :], normal(pages, hk, page).mul(2).exp(), 0.0))
    # a few channels of the keys are much larger than the others, as in trained models
    channel = normal(hk, 1, dim).mul(0.5).exp()
    for name, form in (("k", channel), ("v", torch.ones_like(channel))):
        rows = normal(pages, hk, page, dim) * form
        if case["kind"] == "mxfp4":
            s[name], s[name + "_scale"] = pack(rows)
            s[name + "_scale"].masked_fill_(~filled[:, None, :, None], 255)
        else:
            s[name] = rows.to(TYPES[case["kind"]])
            s[name].masked_fill_(~filled[:, None, :, None], float("nan"))
        del rows
    if op in ("append", "step"):
        given = TYPES[case.get("given", case["kind"])]
        s["new_k"], s["new_v"] = ((normal(sum(new), hk, dim) * f).to(given) for f in (channel[None, :, 0, :], 1.0))
        s["starts"] = torch.tensor(np.cumsum([0] + new), dtype=torch.int32).to(dev)
    if op in ("attend", "step"):
        s["q"] = (normal(batch, case["heads"], dim) * 1.5).to(torch.float16 if case["kind"] == "fp16" else torch.bfloat16)
    s["before"] = books.clone()
    if own:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vram-compression_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        import rans_cache
        s["cache"] = rans_cache.KVCache.from_tensors(s["k"], s["v"], table, length, seen, weight=weight, position=position,
                                                     k_scale=s.get("k_scale"), v_scale=s.get("v_scale"))
    return s


# ------------------------------------------------------------------ 4-bit rows
# A row of `dim` values is stored as dim/2 bytes of e2m1 codes and dim/32 scale bytes (2 to the power of byte - 127; 255 for
# a block with a value that is not finite). Value d, of block n = d // 32, lies in byte (d % 32 // 8) * dim/8 + 4 n + d % 8 // 2,
# in the low half where d is even.
def pack(x):
    blocks = x.float().unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(top)
    exponent = (torch.frexp(torch.where(finite, top, 1.0))[1] - 3).clamp(-63, 63)
    exponent = torch.where(top == 0, -63, exponent)
    a = torch.where(finite, blocks, 0.0) * ((127 - exponent) << 23).view(torch.float32)
    m = a.abs()
    code = ((m > 0.25).byte() + (m >= 0.75).byte() + (m > 1.25).byte() + (m >= 1.75).byte() + (m > 2.5).byte() + (m >= 3.5).byte() + (m > 5).byte())
    code = code | (torch.signbit(a).byte() << 3)
    code = code.unflatten(-1, (4, 4, 2)).transpose(-4, -3)          # [.., n, c, 4, 2] -> [.., c, n, 4, 2]
    code = (code[..., 0] | (code[..., 1] << 4)).flatten(-3)
    return code.contiguous(), torch.where(finite, exponent + 127, 255).byte().flatten(-2)


def unpack(code, scale):
    values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
    n = scale.shape[-1]
    pairs = code.unflatten(-1, (4, n, 4)).transpose(-3, -2)
    pairs = torch.stack((pairs & 15, pairs >> 4), -1).flatten(-3)
    factor = torch.where(scale == 255, float("nan"), (scale.int() << 23).view(torch.float32))
    return (values[pairs.int()] * factor[..., None]).flatten(-2)


# ------------------------------------------------------------------ the plain form
def _place(s, lens):
    """Page and slot of every place of every sequence, and whether it holds one of its first `lens` tokens."""
    page = s["case"]["page"]
    t = torch.arange(s["table"].shape[1] * page, device=lens.device)
    return s["table"].clamp(min=0).long(), t, t[None, :] < lens[:, None]


def _rows(s, name, pages):
    """All rows of the sequences' pages in 32 bits: [batch, kv_heads, places, dim]."""
    x = s[name][pages]
    x = unpack(x, s[name + "_scale"][pages]) if s["case"]["kind"] == "mxfp4" else x.float()
    return x.transpose(1, 2).flatten(2, 3)


def plain_append(s):
    page, length = s["case"]["page"], s["length"]
    starts, token = s["starts"].long(), torch.arange(s["new_k"].shape[0], device=length.device)
    seq = torch.searchsorted(starts, token, right=True) - 1
    place = length[seq] + token - starts[seq]
    at = (s["table"][seq, place // page].long(), slice(None), place % page)
    for name in ("k", "v"):
        x = s["new_" + name]
        if s["case"]["kind"] == "mxfp4":
            s[name][at], s[name + "_scale"][at] = pack(x)
        else:
            s[name][at] = x.to(s[name].dtype)
    s["position"][at] = (s["seen"][seq] + token - starts[seq])[:, None].int()
    s["weight"][at] = 0.0
    more = (starts[1:] - starts[:-1]).int()
    length += more
    s["seen"] += more
    return at


def plain_attend(s, weigh):
    case = s["case"]
    pages, t, valid = _place(s, s["length"])
    q = s["q"].float().unflatten(1, (case["kv_heads"], -1))
    k, v = (torch.where(valid[:, None, :, None], _rows(s, name, pages), 0.0) for name in ("k", "v"))
    score = torch.where(valid[:, None, None, :], q @ k.transpose(-1, -2) * s["scale"], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = (p @ v).flatten(1, 2).to(s["q"].dtype)
    log_sum = (top + torch.log(total)).flatten(1)
    if weigh:
        add = p.sum(2).unflatten(-1, (-1, case["page"])).transpose(1, 2)
        s["weight"].index_put_((pages,), add, accumulate=True)
    return out, log_sum


def plain_evict(s):
    case = s["case"]
    length, budget = s["length"], case["budget"]
    pages, t, valid = _place(s, length)
    weight, position = (s[name][pages].transpose(1, 2).flatten(2) for name in ("weight", "position"))
    late = position >= (s["seen"] - case["recent"])[:, None, None]
    key = torch.where(valid[:, None, :], torch.where(late, math.inf, weight), -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    keep = torch.zeros_like(valid)[:, None, :].repeat(1, key.shape[1], 1)
    keep.scatter_(-1, order[..., :budget], True)
    after = length.clamp(max=budget)
    keep &= valid[:, None, :]
    low = t[None, None, :] < after[:, None, None]
    b, h, hole = torch.nonzero(low & ~keep, as_tuple=True)
    mover = torch.nonzero(keep & ~low, as_tuple=True)[2]
    page = case["page"]
    to, of = ((pages[b, x // page], h, x % page) for x in (hole, mover))
    for name in ("k", "v", "weight", "position"):
        s[name][to] = s[name][of]
    length.copy_(after)


# ------------------------------------------------------------------ one pass
def run(s):
    case, cache = s["case"], s.get("cache")
    op = case["op"]
    if op in ("append", "evict"):
        s["books"].copy_(s["before"])      # the cache as it was: every pass appends, or evicts, the same tokens
    books = dict(length=s["length"], seen=s["seen"], position=s["position"], weight=s["weight"])
    if op == "append":
        if case["kind"] == "mxfp4":
            if own:
                cache.append(s["new_k"], s["new_v"], s["starts"])
                k, v = cache.read(s["starts"], s["new_k"].shape[0])
            else:
                at = plain_append(s)
                k, v = (unpack(s[name][at], s[name + "_scale"][at]).bfloat16() for name in ("k", "v"))
            return dict(books, k=k, v=v)
        if own:
            cache.append(s["new_k"], s["new_v"], s["starts"])
        else:
            plain_append(s)
        return dict(books, k=s["k"], v=s["v"])
    if op == "attend":
        if own:
            out, log_sum = cache.attend(s["q"], scale=s["scale"], weigh=case["weigh"])
        else:
            out, log_sum = plain_attend(s, case["weigh"])
        return dict(out=out, log_sum=log_sum, **({"weight": s["weight"]} if case["weigh"] else {}))
    if op == "evict":
        if own:
            cache.evict(case["budget"], case["recent"])
        else:
            plain_evict(s)
        return dict(books, k=s["k"], v=s["v"])
    if own:
        cache.append(s["new_k"], s["new_v"])
        out, log_sum = cache.attend(s["q"], scale=s["scale"], weigh=True)
        cache.evict(case["budget"], case["recent"])
    else:
        plain_append(s)
        out, log_sum = plain_attend(s, True)
        plain_evict(s)
    return dict(books, out=out, log_sum=log_sum, k=s["k"], v=s["v"])


# ------------------------------------------------------------------ 64 bits
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _power(e):
    """2 to the whole power e in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_block_values(rows):
    """What rows in 64 bits stand for once stored in 4 bits: the nearest value of each block's grid, ties to the even code."""
    x = rows.double().reshape(-1, 32)
    top = x.abs().max(1).values
    e = (top.view(torch.int64) >> 52) - 1023 - 2      # floor(log2(top)) - 2 by the exponent's bits: a rounded logarithm is off at powers of two
    e = torch.where(top > 0, e.clamp(-63, 63), torch.full_like(e, -63))
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    y = x * _power(-e)[:, None]
    up = torch.bucketize(y.abs(), grid).clamp(1, 7)
    low, high = grid[up - 1], grid[up]
    mid = (low + high) / 2
    pick = torch.where((y.abs() > mid) | ((y.abs() == mid) & (up % 2 == 0)), high, low)
    return (torch.sign(y) * pick * _power(e)[:, None]).reshape(rows.shape)


def _exact_rows(s, name, b, n):
    """The first n rows of sequence b in 64 bits: [kv_heads, n, dim]."""
    page, dim = s["case"]["page"], s["case"]["dim"]
    pages = s["table"][b, :-(-n // page)].long()
    x = s[name][pages].transpose(0, 1).flatten(1, 2)[:, :n]
    if s["case"]["kind"] != "mxfp4":
        return x.double()
    scale = s[name + "_scale"][pages].transpose(0, 1).flatten(1, 2)[:, :n]
    d = torch.arange(dim, device=x.device)
    byte = (d % 32) // 8 * (dim // 8) + d // 32 * 4 + d % 8 // 2
    code = (x[..., byte].int() >> (4 * (d % 2)).int()) & 15
    grid = torch.tensor(E2M1 + [-g for g in E2M1], dtype=torch.float64, device=x.device)
    return grid[code] * _power(scale.int() - 127)[..., d // 32]


def _exact_attend(s, lens, q, out, log_sum, weight):
    case = s["case"]
    group = case["heads"] // case["kv_heads"]
    for b, n in enumerate(lens):
        if not n:
            continue
        k, v = _exact_rows(s, "k", b, n), _exact_rows(s, "v", b, n)
        score = torch.bmm(q[b].double().reshape(case["kv_heads"], group, -1), k.transpose(1, 2)) * s["scale"]
        log_sum[b] = torch.logsumexp(score, -1).reshape(-1)
        p = torch.softmax(score, -1)
        out[b] = torch.bmm(p, v).reshape(case["heads"], -1)
        if weight is not None:
            at = torch.arange(n, device=k.device)
            pages = s["table"][b, at // case["page"]].long()
            weight[pages, :, at % case["page"]] += p.sum(1).T


def _exact_evict(s, lens, seen, weight, position, rows):
    """Moves kept tokens into the places of evicted ones in `weight`, `position` and `rows`, one head at a time, on the host."""
    case = s["case"]
    budget, table = case["budget"], s["table"].cpu().numpy()
    w, p = weight.cpu().numpy().copy(), position.cpu().numpy().copy()
    for b, n in enumerate(lens):
        if n <= budget:
            continue
        at = np.arange(n)
        pages, slots = table[b, at // case["page"]], at % case["page"]
        for h in range(case["kv_heads"]):
            key = np.where(p[pages, h, slots] >= seen[b] - case["recent"], np.inf, w[pages, h, slots])
            keep = np.zeros(n, bool)
            keep[np.argsort(-key, kind="stable")[:budget]] = True
            hole, mover = np.nonzero(~keep[:budget])[0], budget + np.nonzero(keep[budget:])[0]
            to, of = ((pages[x], h, slots[x]) for x in (hole, mover))
            w[to], p[to] = w[of], p[of]
            to, of = (tuple(torch.as_tensor(y, device=s["table"].device) if isinstance(y, np.ndarray) else y for y in x) for x in (to, of))
            for r in rows:
                r[to] = r[of]
    return torch.from_numpy(w), torch.from_numpy(p)


def exact(case, seed):
    s = prepare(case, seed)
    op, lens, dev = case["op"], held(case), s["table"].device
    none = dict(length=None, seen=None, position=None)
    if op in ("append", "step"):
        new = lengths(case) if op == "append" else [1] * case["batch"]
        k, v = s["new_k"].double(), s["new_v"].double()
        if case["kind"] == "mxfp4":
            return dict(none, k=_exact_block_values(k), v=_exact_block_values(v), weight=None)
        at = torch.tensor([(b, lens[b] + i) for b, m in enumerate(new) for i in range(m)], device=dev).reshape(-1, 2)
        pages, slots = s["table"][at[:, 0], at[:, 1] // case["page"]].long(), at[:, 1] % case["page"]
        for name, x in (("k", k), ("v", v)):
            s[name] = s[name].double()
            s[name][pages, :, slots] = x
        weight = s["weight"].double()
        weight[pages, :, slots] = 0.0
        s["position"][pages, :, slots] = at[:, 1:].int()
        if op == "append":
            return dict(none, k=s["k"], v=s["v"], weight=weight)
        lens = [a + b for a, b in zip(lens, new)]
    else:
        weight = s["weight"].double()
    if op in ("attend", "step"):
        weigh = op == "step" or case["weigh"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
        log_sum = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=dev)
        _exact_attend(s, lens, s["q"], out, log_sum, weight if weigh else None)
        if op == "attend":
            return dict(out=out, log_sum=log_sum, **({"weight": weight} if weigh else {}))
    weight, position = _exact_evict(s, lens, lens, weight, s["position"], [s["k"], s["v"]])
    result = dict(none, weight=weight, k=s["k"].double(), v=s["v"].double())
    return dict(result, out=out, log_sum=log_sum) if op == "step" else result
