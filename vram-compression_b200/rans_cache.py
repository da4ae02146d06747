"""The paged key-value cache of a decoder step (librans_b200.so, include/rans_kv.h).

The weight products of a step run from compressed weights (rans_b200.RansChain,
rans_model.RansLinear); between the v and the o projection stands the attention,
and its cache is what else fills the memory.  KVCache holds it in pages of 16-bit
or microscaled 4-bit rows (4.25 bits a value), and runs on it:

  append   new tokens' rows (one per sequence, or whole prompts), quantised on the way
  attend   attention of one new token per sequence, split over the length and joined;
           on request it adds up the weight that each cached token receives
  evict    back to a budget of tokens by that weight, the newest always kept
  read     stored rows back as dense ones

    cache = KVCache(pages=1024, page=64, kv_heads=8, dim=128, batch=4, max_tokens=32768, kind="mxfp4")
    cache.reserve([1] * 4)                  # host: pages for one more token of each sequence
    cache.append(k, v)                      # [4, 8, 128] each
    out, log_sum = cache.attend(q, weigh=True)      # q, out [4, 64, 128]
    cache.evict(budget=4096, recent=64)     # when it is time

Every method but reserve, release and check is one asynchronous call on the
current stream (capturable in a CUDA graph once the workspace has its size: run it
once before).  What the host knows of a cache's own pages does not move while a graph
is captured or replayed: an eviction in a graph gives no pages back, and the pages for
the tokens that replays append are reserved before.  Calls on one cache share its books
and workspace, so they have to be ordered: one stream, or events between streams.
Sequences may share pages for attend alone; append, attend(weigh=True) and evict want
every page in one place.  Page numbers, lengths and row ranges are checked inside the
kernels: what would lie outside is left out and check() raises.
There is no CPU fallback.
"""
from __future__ import annotations

import ctypes

import rans_b200 as rb

_vp, _i32, _i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64

KINDS = {"bf16": 0, "fp16": 1, "mxfp4": 2}
_FP32 = 3
BAD_PAGE, BAD_LENGTH, BAD_STARTS = 1, 2, 4


class RansKvCache(ctypes.Structure):
    """ctypes mirror of the C struct RansKvCache (include/rans_kv.h)."""
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("weight", _vp), ("position", _vp),
                ("table", _vp), ("length", _vp), ("seen", _vp), ("status", _vp), ("workspace", _vp),
                ("workspace_bytes", _i64),
                ("k_page", _i64), ("k_head", _i64), ("k_slot", _i64), ("v_page", _i64), ("v_head", _i64), ("v_slot", _i64),
                ("pages", _i32), ("page", _i32), ("kv_heads", _i32), ("dim", _i32), ("batch", _i32),
                ("table_cols", _i32), ("kind", _i32), ("reserved", _i32)]


class CacheError(RuntimeError):
    """A kernel met a page number, length or row range that the cache does not have; the tokens concerned were left out."""


def _need(ok, what):
    if not ok:
        raise ValueError(what)


class KVCache:
    """A paged key-value cache on one GPU.

    k, v       [pages, kv_heads, page, dim] rows (bf16, fp16), or uint8 codes [.., dim/2] with
               k_scale, v_scale uint8 [.., dim/32] (the 4-bit layout of include/rans_kv.h)
    table      int32 [batch, columns], the pages of each sequence in order
    length     int32 [batch], tokens in the cache; seen: tokens ever appended
    position   int32 [pages, kv_heads, page], each token's place in its sequence
    weight     fp32 [pages, kv_heads, page], the attention weight that it has received
    """

    def __init__(self, pages, page, kv_heads, dim, batch, max_tokens, kind="bf16", device=None, lib=None):
        torch = rb._torch()
        _need(kind in KINDS, f"kind must be one of {sorted(KINDS)}")
        _need(pages > 0 and page >= 16 and page % 16 == 0, "pages > 0 of a multiple of 16 tokens")
        _need(kv_heads > 0 and batch > 0 and max_tokens > 0, "kv_heads, batch and max_tokens must be positive")
        _need(dim in (64, 128, 256), "dim must be 64, 128 or 256")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        shape = (pages, kv_heads, page)
        scale = [None, None]
        if kind == "mxfp4":
            rows = [torch.zeros(*shape, dim // 2, dtype=torch.uint8, device=dev) for _ in range(2)]
            scale = [torch.zeros(*shape, dim // 32, dtype=torch.uint8, device=dev) for _ in range(2)]
        else:
            rows = [torch.zeros(*shape, dim, dtype=torch.bfloat16 if kind == "bf16" else torch.float16, device=dev)
                    for _ in range(2)]
        table = torch.full((batch, -(-max_tokens // page)), -1, dtype=torch.int32, device=dev)
        self._set(rows[0], rows[1], table, torch.zeros(batch, dtype=torch.int32, device=dev),
                  torch.zeros(batch, dtype=torch.int32, device=dev), torch.zeros(shape, device=dev),
                  torch.zeros(shape, dtype=torch.int32, device=dev), scale[0], scale[1], lib)
        # Pages: `_free` ones are in no row of the table.  `_owned` ones are in their sequence's row and in no other; those behind
        # what the sequence needs (_needed) are free too, but stay where they are until another sequence takes them, so that a
        # sequence at its budget, which gives a page back and takes one with every few tokens, leaves the table alone.
        self._free = list(range(pages - 1, -1, -1))
        self._owned = [[] for _ in range(batch)]
        self._most = [0] * batch            # no sequence is longer than this, with all the tokens that are reserved
        self._to_come = [0] * batch         # of those, no more than this are still to be appended
        self._held = [0] * batch            # no sequence holds more than this, unless graphs append too

    @classmethod
    def from_tensors(cls, k, v, table, length, seen, weight=None, position=None, k_scale=None, v_scale=None, lib=None):
        """A cache over tensors that the caller lays out and whose pages the caller hands out.

        16-bit k and v are [pages, kv_heads, page, dim] views with any strides that are multiples of 16 bytes
        and contiguous rows (so [pages, page, kv_heads, dim] memory is fine, transposed); everything else is
        contiguous.  weight and position are needed by attend(weigh=True) and evict only."""
        self = cls.__new__(cls)
        self._set(k, v, table, length, seen, weight, position, k_scale, v_scale, lib)
        self._free = self._owned = self._most = self._to_come = self._held = None
        return self

    def _set(self, k, v, table, length, seen, weight, position, k_scale, v_scale, lib):
        torch = rb._torch()
        self._torch = torch
        self.lib = rb._lib(lib)
        tensors = [t for t in (k, v, table, length, seen, weight, position, k_scale, v_scale) if t is not None]
        _need(all(t.is_cuda and t.device == k.device for t in tensors), "all tensors must be on one CUDA device")
        _need(k.dim() == 4 and v.shape == k.shape and v.dtype == k.dtype, "k and v must be [pages, kv_heads, page, dim] alike")
        pages, heads, page, dim = k.shape
        if k.dtype == torch.uint8:
            self.kind, dim = "mxfp4", dim * 2
            _need(k_scale is not None and v_scale is not None, "4-bit rows need k_scale and v_scale")
            for t in (k_scale, v_scale):
                _need(t.dtype == torch.uint8 and t.shape == (pages, heads, page, dim // 32) and t.is_contiguous(),
                      "scales must be contiguous uint8 [pages, kv_heads, page, dim / 32]")
            _need(k.is_contiguous() and v.is_contiguous(), "4-bit rows must be contiguous")
        else:
            _need(k.dtype in (torch.bfloat16, torch.float16), "k and v must be bf16, fp16 or uint8 codes")
            _need(k_scale is None and v_scale is None, "scales belong to 4-bit rows")
            self.kind = "bf16" if k.dtype == torch.bfloat16 else "fp16"
            for t in (k, v):
                _need(t.stride(3) == 1 and all(s > 0 and s * 2 % 16 == 0 for s in t.stride()[:3]) and t.data_ptr() % 16 == 0,
                      "rows must be contiguous, 16-byte aligned and apart by multiples of 16 bytes")
        _need(dim in (64, 128, 256), "dim must be 64, 128 or 256")
        _need(pages > 0 and page >= 16 and page % 16 == 0, "pages > 0 of a multiple of 16 tokens")
        batch = length.numel()
        _need(table.dim() == 2 and table.shape[0] == batch and table.shape[1] > 0, "table must be [batch, columns]")
        _need(1 <= batch <= 2048 and batch * heads <= 65535, "at most 2048 sequences, and 65535 of sequence times kv head")
        for t, n in ((table, "table"), (length, "length"), (seen, "seen")):
            _need(t.dtype == torch.int32 and t.is_contiguous(), f"{n} must be contiguous int32")
        _need(seen.numel() == batch, "seen must have one entry per sequence")
        for t, d, n in ((weight, torch.float32, "weight"), (position, torch.int32, "position")):
            _need(t is None or (t.dtype == d and t.shape == (pages, heads, page) and t.is_contiguous()),
                  f"{n} must be a contiguous [pages, kv_heads, page] tensor of {d}")
        self.device = k.device
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.table, self.length, self.seen, self.weight, self.position = table, length, seen, weight, position
        self.pages, self.kv_heads, self.page, self.dim, self.batch = pages, heads, page, dim, batch
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        ptr = lambda t: None if t is None else t.data_ptr()      # noqa: E731
        strides = [0] * 6 if self.kind == "mxfp4" else [s * 2 for t in (k, v) for s in t.stride()[:3]]
        self._c = RansKvCache(ptr(k), ptr(v), ptr(k_scale), ptr(v_scale), ptr(weight), ptr(position), ptr(table), ptr(length),
                              ptr(seen), ptr(self.status), None, 0, *strides, pages, page, heads, dim, batch, table.shape[1],
                              KINDS[self.kind], 0)
        self._p = ctypes.addressof(self._c)
        self._index = self.device.index
        self._current_device, self._raw_stream = torch.cuda.current_device, torch._C._cuda_getCurrentRawStream
        self._capturing, self._in_graphs = torch.cuda.is_current_stream_capturing, False
        self._workspaces = []               # replaced ones stay: kernels in flight and captured graphs may use them
        self._sizes = {}                    # what a call's shapes have been found to be good for
        self._room(self.lib.rans_kv_counter_bytes(self._p))

    def _room(self, nbytes):
        if nbytes < 0:
            raise ValueError(f"bad cache description ({nbytes})")
        if nbytes > self._c.workspace_bytes:
            ws = self._torch.empty(nbytes, dtype=self._torch.uint8, device=self.device)
            ws[:self.lib.rans_kv_counter_bytes(self._p)].zero_()
            self._workspaces.append(ws)
            self._c.workspace, self._c.workspace_bytes = ws.data_ptr(), nbytes

    def _stream(self):
        if self._current_device() != self._index:
            raise ValueError(f"the cache is on {self.device}; make it the current device")
        return self._raw_stream(self._index)

    def _rows(self, k, v):
        """Checks of append's rows, which depend on their shapes alone: (type, strides are usable, strides in bytes)."""
        torch = self._torch
        for x, what in ((k, "k"), (v, "v")):
            _need(x.device == self.device and x.dim() == 3 and tuple(x.shape[1:]) == (self.kv_heads, self.dim),
                  f"{what} must be [tokens, {self.kv_heads}, {self.dim}] on {self.device}")
        _need(k.dtype == v.dtype and k.shape == v.shape, "k and v must be alike")
        given = {torch.bfloat16: 0, torch.float16: 1, torch.float32: _FP32}.get(k.dtype)
        _need(given is not None, "k and v must be bf16, fp16 or fp32")
        size = k.element_size()
        usable = lambda x: x.stride(2) == 1 and x.stride(0) * size % 16 == 0 and x.stride(1) * size % 16 == 0   # noqa: E731
        return given, usable(k), usable(v), *(x.stride(i) * size for x in (k, v) for i in range(2))

    @staticmethod
    def _aligned(x, usable):
        """x itself, or a contiguous copy, so that rows can be read 16 bytes at a time."""
        if usable and x.data_ptr() % 16 == 0:
            return x
        return x.clone() if x.is_contiguous() else x.contiguous()

    def _starts(self, starts, tokens):
        if starts is None:
            if tokens != self.batch:
                raise ValueError(f"without starts there is one token for each of the {self.batch} sequences")
            return None
        if (starts.dtype != self._torch.int32 or starts.get_device() != self._index or starts.numel() != self.batch + 1
                or not starts.is_contiguous()):
            raise ValueError(f"starts must be contiguous int32 [{self.batch + 1}] on {self.device}")
        return starts.data_ptr()

    # ---------------------------------------------------------------- pages
    def _needed(self, b):
        return -(-self._most[b] // self.page)

    def _write_table(self, entries):
        """{(row, column): page} into the device table: one asynchronous copy from pinned memory, whatever their number."""
        torch, cols = self._torch, self.table.shape[1]
        at = torch.tensor([[r * cols + c for r, c in entries], list(entries.values())], dtype=torch.int64, pin_memory=True)
        at = at.to(self.device, non_blocking=True)
        self.table.view(-1).scatter_(0, at[0], at[1].int())

    def reserve(self, tokens):
        """Hand out the pages for tokens[b] more tokens of each sequence.  They stay reserved, whatever is evicted meanwhile,
        until as many tokens have been appended.  (Host; one asynchronous copy where the table changes.)"""
        _need(self._free is not None, "the caller hands out the pages of a cache made from tensors")
        _need(len(tokens) == self.batch and all(t >= 0 for t in tokens), "one count per sequence")
        want = [m + t for m, t in zip(self._most, tokens)]
        _need(all(w <= self.table.shape[1] * self.page for w in want), "a sequence would outgrow max_tokens")
        need = [-(-w // self.page) for w in want]
        more = sum(n - self._needed(b) for b, n in enumerate(need))
        if more > self.free_pages:
            raise CacheError(f"{more} pages needed, {self.free_pages} free")
        self._most = want
        self._to_come = [t + n for t, n in zip(self._to_come, tokens)]
        entries = {}
        for b, n in enumerate(need):
            own = self._owned[b]
            while len(own) < n:
                entries[b, len(own)] = page = self._free.pop() if self._free else self._take_back(entries)
                own.append(page)
        if entries:
            self._write_table(entries)

    def _take_back(self, entries):
        """A page that a sequence no longer needs, out of the table."""
        b = next(b for b, own in enumerate(self._owned) if len(own) > self._needed(b))
        page = self._owned[b].pop()
        entries[b, len(self._owned[b])] = -1
        return page

    def release(self, b):
        """Forget sequence b and take its pages back."""
        _need(self._free is not None, "the caller hands out the pages of a cache made from tensors")
        self._free += reversed(self._owned[b])
        self._owned[b], self._most[b], self._to_come[b], self._held[b] = [], 0, 0, 0
        self.table[b].fill_(-1)
        self.length[b].zero_()
        self.seen[b].zero_()

    @property
    def free_pages(self):
        return self.pages - sum(self._needed(b) for b in range(self.batch))

    def _appended(self, tokens, by_sequence):
        """Of the reserved tokens `tokens` have come: one of each sequence, or the host does not know whose."""
        self._held = [min(h + (1 if by_sequence else tokens), m) for h, m in zip(self._held, self._most)]
        if by_sequence:
            self._to_come = [max(t - 1, 0) for t in self._to_come]
        else:
            left = max(sum(self._to_come) - tokens, 0)
            self._to_come = [min(t, left) for t in self._to_come]

    @property
    def most(self):
        """What the host knows of the lengths: no sequence is longer than this, even with all the tokens that are reserved and
        still to come."""
        return list(self._most)

    @property
    def held(self):
        """No sequence holds more tokens than this: what was appended, as far as the host can tell, less what was evicted.
        Once an append has been captured in a graph: as `most`."""
        return list(self._most if self._in_graphs else self._held)

    def nbytes(self):
        """Bytes of rows, scales and books (not of the workspace)."""
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale, self.weight, self.position)
                   if t is not None)

    # ---------------------------------------------------------------- operators
    def append(self, k, v, starts=None):
        """Append rows k, v [tokens, kv_heads, dim] (bf16, fp16 or fp32): row b to sequence b, or with starts (int32
        [batch + 1] on the device, rising from 0 to tokens) rows starts[b]..starts[b+1]-1.  Their pages have to be
        reserved."""
        key = (k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype)
        known = self._sizes.get(key)
        if known is None:
            known = self._sizes[key] = self._rows(k, v)
        given, k_usable, v_usable, kt, kh, vt, vh = known
        if k.get_device() != self._index or v.get_device() != self._index:
            raise ValueError(f"k and v must be on {self.device}")
        n, row = k.shape[0], self.dim * (4 if given == _FP32 else 2)
        if not k_usable or k.data_ptr() % 16:
            k, kt, kh = self._aligned(k, k_usable), self.kv_heads * row, row
        if not v_usable or v.data_ptr() % 16:
            v, vt, vh = self._aligned(v, v_usable), self.kv_heads * row, row
        rc = self.lib.rans_kv_append(self._p, k.data_ptr(), v.data_ptr(), given, kt, kh, vt, vh, self._starts(starts, n), n,
                                     self._stream())
        rb._check(rc, "rans_kv_append")
        if self._free is not None:
            if self._capturing():
                self._in_graphs = True
            else:
                self._appended(n, starts is None)

    def read(self, starts=None, tokens=None):
        """The last starts[b+1]-starts[b] tokens of each sequence (without starts: the last one) as dense rows k, v
        [tokens, kv_heads, dim], bf16 (fp16 from an fp16 cache).  tokens = starts[batch], known to the host."""
        torch = self._torch
        _need(starts is None or tokens is not None, "tokens must be given with starts")
        n = self.batch if starts is None else int(tokens)
        _need(n >= 0, "tokens must not be negative")
        k, v = (torch.empty(n, self.kv_heads, self.dim, dtype=torch.float16 if self.kind == "fp16" else torch.bfloat16,
                            device=self.device) for _ in range(2))
        rb._check(self.lib.rans_kv_read(self._p, k.data_ptr(), v.data_ptr(), self._starts(starts, n), n, self._stream()),
                  "rans_kv_read")
        return k, v

    def attend(self, q, scale=None, weigh=False, out=None, log_sum=None):
        """Attention of one query per sequence over its cached tokens: q [batch, heads, dim] in the cache's type (bf16 or
        fp16 over 4-bit rows) -> out (alike) and log_sum (fp32 [batch, heads], natural logarithm).  scale defaults to
        dim ** -0.5.  An empty sequence gives zeros and -inf.  weigh: also add each token's share of the attention,
        summed over a kv head's query heads, to `weight`."""
        torch = self._torch
        key = (q.shape, q.stride(), q.dtype, weigh)
        known = self._sizes.get(key)
        if known is None:
            known = self._sizes[key] = self._query(q, weigh)
        kind, heads, usable, q_batch, q_head, sums = known
        if q.get_device() != self._index:
            raise ValueError(f"q must be on {self.device}")
        if not usable or q.data_ptr() % 16:
            q = self._aligned(q, usable)
            q_batch, q_head = heads * self.dim * 2, self.dim * 2
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            _need(out.shape == q.shape and out.dtype == q.dtype and out.device == self.device and out.is_contiguous()
                  and out.data_ptr() % 16 == 0, "out must be contiguous and like q")
        if log_sum is None:
            log_sum = torch.empty_like(sums)
        else:
            _need(log_sum.shape == (self.batch, heads) and log_sum.dtype == torch.float32 and log_sum.device == self.device
                  and log_sum.is_contiguous(), "log_sum must be contiguous fp32 [batch, heads]")
        rc = self.lib.rans_kv_attend(self._p, q.data_ptr(), kind, q_batch, q_head, heads,
                                     self.dim ** -0.5 if scale is None else scale, out.data_ptr(), log_sum.data_ptr(),
                                     1 if weigh else 0, self._stream())
        rb._check(rc, "rans_kv_attend")
        return out, log_sum

    def _query(self, q, weigh):
        """Checks of attend's query, which depend on its shape alone, and the workspace for it: (type, heads, strides are
        usable, strides in bytes, a tensor like log_sum)."""
        torch = self._torch
        _need(q.dim() == 3 and q.shape[0] == self.batch and q.shape[2] == self.dim and q.device == self.device
              and q.shape[1] > 0 and q.shape[1] % self.kv_heads == 0,
              f"q must be [{self.batch}, a multiple of {self.kv_heads}, {self.dim}] on {self.device}")
        kind = 0 if q.dtype == torch.bfloat16 else 1
        _need(q.dtype in (torch.bfloat16, torch.float16) and (self.kind == "mxfp4" or kind == KINDS[self.kind]),
              f"q must be of the cache's type ({self.kind})")
        _need(not weigh or self.weight is not None, "this cache has no weight tensor")
        size = self.lib.rans_kv_attend_bytes(self._p, q.shape[1], int(weigh))
        _need(size > 0, f"{q.shape[1]} query heads on {self.kv_heads}, or the table's size, are more than the kernel counts")
        self._room(size)
        return (kind, q.shape[1], q.stride(2) == 1 and q.stride(0) % 8 == 0 and q.stride(1) % 8 == 0, q.stride(0) * 2,
                q.stride(1) * 2, torch.empty((self.batch, q.shape[1]), dtype=torch.float32, device=self.device))

    def evict(self, budget, recent=0):
        """Bring sequences with more than `budget` tokens back to it, per kv head: the `recent` newest tokens and the
        heaviest others stay (ties: the lower place).  Kept tokens from above the budget fill the freed places below, so
        pages past the budget are free again (to this cache's other sequences, or to the caller who hands them out), but for
        those that are reserved for tokens to come."""
        _need(self.weight is not None and self.position is not None, "this cache has no weight and position tensors")
        budget, recent = int(budget), int(recent)
        _need(budget >= 1 and 0 <= recent <= budget, "budget must be positive and recent between 0 and budget")
        size = self._sizes.get(budget)
        if size is None:
            size = self._sizes[budget] = self.lib.rans_kv_evict_bytes(self._p, budget)
            self._room(size)
        rb._check(self.lib.rans_kv_evict(self._p, budget, recent, self._stream()), "rans_kv_evict")
        if self._free is not None and not self._capturing():
            self._most = [min(m, budget + t) for m, t in zip(self._most, self._to_come)]
            self._held = [min(h, budget) for h in self._held]

    def check(self):
        """Synchronise and raise CacheError if a kernel so far met a bad page, length or row range (reading clears it)."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            names = [n for bit, n in ((BAD_PAGE, "a page number outside the cache"),
                                      (BAD_LENGTH, "a length beyond the table"),
                                      (BAD_STARTS, "rows outside starts")) if bits & bit]
            raise CacheError("tokens were left out: " + ", ".join(names))
