"""An 8-bit cache in pages for the kept (not converted) full-attention layers.

The reference quotes its decode figures with an 8-bit key and value cache (README.md:15, 60), and its port copies and removes
sequences of the cache (llamacpp/README.md:77-78).  Here a pool of pages of ``page`` tokens holds e4m3 codes with one power-of-two
scale per (layer, page, KV head), for keys and for values; the host gives out pages (lowest index first, with reference
counts) and the device holds the page table and the lengths, so that ``append`` and ``attend`` read nothing from the
host and can be captured into a CUDA graph:

    c = PagedKV(layers=4, pages=4096, heads=4, slots=64, max_len=131072)
    c.reserve(slots, 1)                       # host: room for the next token of each sequence, once per step
    for layer in range(4):
        c.append(layer, k, v, slot_ids)       # device
        o, _ = c.attend(layer, q, slot_ids)   # device

``fork`` shares pages between sequences, ``free`` and ``truncate`` give them back, ``compact`` closes the pool up.  Where a batch has forks of
one prompt, or of a tree of them, ``share`` finds which pages its sequences have in common, and ``attend`` reads those once for all:

    plan = c.share(slots)                     # host: again after forks, and when the plan is no longer good
    o, _ = c.attend(layer, q, shared=plan)    # device

Calls on one cache belong on one stream, or on streams that the caller orders, and on one host thread at a time.  There is no
CPU path.
"""
from __future__ import annotations

import ctypes
import weakref

import numpy as np
import torch

from . import _lib
from .functional import (heads_16bit, int32_on, kernel_dtype, on_device, prompt_attention, ptr, score_scale, serving_inputs,
                         stream_handle)
from .structs import BfPagePool, BfPageTable

PAGE_SIZES = (16, 32, 64, 128)
MAX_GROUP = 24                  # query heads per KV head of attend
# Tokens of reading that a shared run has to save, and all runs of n sequences together: WORTH[0] + WORTH[1] n.  The way over shared pages has more to start
# (15 us against 8 for the smallest calls) and spends more on each sequence's own tokens.  Decode steps, us without and with a plan: 24 heads
# of 4, two sequences that share 16384 tokens 21 and 25; eight, 28672 saved 19 and 21, 57344 saved 27 and 23; 64, 32256 saved 22 and 28, 64512 saved 32 and 30 (with 1000
# tokens of their own 47 and 56, then at 129024 64 and 54); 24 heads of one, 32 sequences, 31744 saved 20 and 21, 126976 saved 30 and 26.
# (24 heads of one and up to eight sequences gain from 2000 on, 26 against 17: min_saved is for those.)
MIN_SAVED, WORTH = 1024, (32768, 512)


_REASONS = {1: "a slot is outside [0, {slots})", 2: "a slot is named twice", 3: "a number of tokens is negative",
            4: "a sequence would be longer than the cache's max_len ({tokens})", 5: "a slot is both taken from and filled",
            6: "a slot to fill holds a sequence: free it first", 7: "truncate cannot lengthen a sequence"}


class PageTable:
    """The host's side of the cache: which slot holds which pages (``bf_page_table_*``, over numpy arrays).  Every method
    returns what the device has to do, as the int32 lists of ``bf_paged_pages``, good until the next call; a call that raises has
    changed nothing."""

    def __init__(self, pages: int, slots: int, page: int, width: int):
        self.pages, self.slots, self.page, self.width = pages, slots, page, width
        self.refs = np.zeros(pages, np.int32)
        self.table = np.full((slots, width), -1, np.int32)
        self.lens = np.zeros(slots, np.int64)
        self._mark = np.zeros(slots, np.int32)
        self._set = np.empty((slots * (width + 1), 2), np.int32)
        self._fork = np.empty((slots, 5), np.int32)
        self._move = np.empty((pages, 2), np.int32)
        self._out = np.zeros(8, np.int32)                   # [0:3] info, [4] and [5] list lengths
        self._state = BfPageTable(*(x.ctypes.data for x in (self.refs, self.table, self.lens, self._mark)), pages, slots, page,
                                  width, pages, 0, 0)
        self._lib = _lib.load()
        # addresses of what stays where it is
        self._t, self._info = ctypes.addressof(self._state), self._out.ctypes.data
        self._n0, self._n1 = self._info + 16, self._info + 20
        self._to_set, self._to_fork, self._to_move = (x.ctypes.data for x in (self._set, self._fork, self._move))

    @property
    def n_free(self) -> int:
        return self._state.n_free

    def _whole(self, x, like=None) -> np.ndarray:
        """x as int64 [n], or, beside slots, one number for each of them."""
        x = np.asarray(x)
        if x.dtype.kind not in "iu" and x.size:
            raise ValueError("whole numbers are needed")
        if like is not None:
            if x.ndim == 0:
                return np.full(like.shape, x, np.int64)
            if x.shape != like.shape:
                raise ValueError("one whole number, or one for each slot, is needed")
        elif x.ndim > 1:
            raise ValueError("slots must be a list of whole numbers")
        return np.ascontiguousarray(x.reshape(-1), np.int64)

    def _call(self, name, *args) -> None:
        rc = getattr(self._lib, name)(self._t, *args)
        if rc:
            reason = int(self._out[0])
            if reason == 8:
                raise RuntimeError(f"heimdall_b200: the page pool is full ({self._out[1]} pages needed, {self._out[2]} of "
                                   f"{self.pages} free)")
            raise ValueError(_REASONS[reason].format(slots=self.slots, tokens=self.width * self.page))

    def reserve(self, slots, n) -> dict:
        s = self._whole(slots)
        n = self._whole(n, s)
        if s.size > self.slots:
            raise ValueError(_REASONS[2])
        self._call("bf_page_table_reserve", s.ctypes.data, n.ctypes.data, s.size, self._to_set, self._n0, self._info)
        return {"set": self._set[:self._out[4]]}

    def free(self, slots) -> dict:
        s = self._whole(slots)
        self._call("bf_page_table_free", s.ctypes.data, s.size, self._info)
        return {"release": s.astype(np.int32)}

    def fork(self, src, dst) -> dict:
        a, b = self._whole(src), self._whole(dst)
        if a.size != b.size:
            raise ValueError("fork needs as many slots to fill as slots to take from")
        if b.size > self.slots:
            raise ValueError(_REASONS[2])
        self._call("bf_page_table_fork", a.ctypes.data, b.ctypes.data, a.size, self._to_fork, self._info)
        return {"fork": self._fork[:a.size]}

    def truncate(self, slots, lens) -> dict:
        s = self._whole(slots)
        n = self._whole(lens, s)
        if s.size > self.slots:
            raise ValueError(_REASONS[2])
        self._call("bf_page_table_truncate", s.ctypes.data, n.ctypes.data, s.size, self._to_fork, self._n0, self._to_set,
                   self._n1, self._info)
        return {"fork": self._fork[:self._out[4]], "set": self._set[:self._out[5]]}

    def share(self, slots, min_saved: int) -> np.ndarray:
        s = self._whole(slots)
        if s.size < 1:
            raise ValueError("share needs at least one sequence")
        plan, scratch = np.empty(self._lib.bf_share_words(s.size), np.int32), np.empty(7 * s.size, np.int32)
        self._call("bf_page_table_share", s.ctypes.data, s.size, min_saved, plan.ctypes.data, scratch.ctypes.data, self._info)
        return plan

    def compact(self) -> dict:
        self._call("bf_page_table_compact", self._to_move, self._n0)
        return {"move": self._move[:self._out[4]]}


class SharedPages:
    """Which pages the sequences of a batch have in common (``PagedKV.share``): ``slots``, in the order of the batch, and ``runs``, the number of
    page runs that are read once for several sequences.  A plan does not keep its cache: ``cache`` is None once that is gone."""

    def __init__(self, cache: "PagedKV", slots: np.ndarray, plan: np.ndarray):
        self._cache = weakref.ref(cache)         # the cache has plans of its own: with references both ways the pool would wait for the cycle collector
        self._page = cache.page
        self.n = slots.size
        self.plan = torch.empty(plan.size, dtype=torch.int32, device=cache.device)
        self._slot_ids = self.plan[4:4 + self.n]
        self._fill(slots, plan)
        cache._plans.add(self)

    @property
    def cache(self):
        return self._cache()

    def _fill(self, slots: np.ndarray, plan: np.ndarray) -> None:
        self.slots, self.runs, self.good = slots.tolist(), int(plan[0]), True
        # the tokens of each slot that are read as shared pages
        self._covered = dict(zip(self.slots, (plan[4 + 4 * self.n:4 + 5 * self.n] * self._page).tolist()))
        self.plan.copy_(torch.from_numpy(plan))

    def _cut(self, slots, lens) -> None:
        if self.good and any(n < self._covered.get(s, 0) for s, n in zip(slots, lens)):
            self.good = False


class PagedKV:
    """Keys and values of ``layers`` kept layers in 8-bit pages (see the module's docstring).

    ``pages`` of ``page`` tokens (16, 32, 64 or 128) for ``slots`` sequences of up to ``max_len`` tokens, rounded up to whole
    pages (default: the whole pool), ``heads`` KV heads of 256.  Device tensors, for reading: ``k_pages``, ``v_pages``
    [layers,pages,heads,page,256] float8_e4m3fn, ``k_scale``, ``v_scale`` [layers,pages,heads] fp32 (value = code * scale), ``table`` [slots,width] int32
    (-1: no page), ``lens`` [slots] int32."""

    def __init__(self, layers: int, pages: int, heads: int, slots: int, page: int = 64, dim: int = 256, max_len=None,
                 device="cuda"):
        if dim != 256:
            raise NotImplementedError("PagedKV is built for head dim 256")
        if page not in PAGE_SIZES:
            raise NotImplementedError(f"PagedKV has pages of {', '.join(map(str, PAGE_SIZES))} tokens")
        if min(layers, pages, heads, slots) < 1 or (max_len is not None and max_len < 1):
            raise ValueError("layers, pages, heads, slots and max_len must be positive")
        max_len = pages * page if max_len is None else max_len
        width = -(-max_len // page)
        if slots * (width + 1) >= 2 ** 31 or width * page >= 2 ** 31 - 256 or pages * heads * page >= 2 ** 31 or layers * heads > 65535:
            raise ValueError("the cache is too large for 32-bit row numbers")
        dev = torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError("heimdall_b200 runs on CUDA tensors only (there is no CPU fallback)")
        self.layers, self.heads, self.page, self.dim = layers, heads, page, dim
        self.host = PageTable(pages, slots, page, width)
        code = lambda: torch.zeros(layers, pages, heads, page, dim, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        self.k_pages, self.v_pages = code(), code()
        self.device = self.k_pages.device
        self.k_scale = torch.zeros(layers, pages, heads, device=dev)
        self.v_scale = torch.zeros(layers, pages, heads, device=dev)
        self.table = torch.full((slots, width), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(slots, dtype=torch.int32, device=dev)
        self._pool = BfPagePool(ptr(self.k_pages), ptr(self.v_pages), ptr(self.k_scale), ptr(self.v_scale), ptr(self.table),
                                ptr(self.lens), layers, pages, heads, page, dim, slots, width)
        self._pool_ptr = ctypes.addressof(self._pool)
        self._ws = {}                       # workspace bytes by (B, t, H), with True behind them for shared pages
        self._plans = weakref.WeakSet()     # plans of shared pages, good until a slot is cut below what they cover of it
        self._layer_plans = {}              # those of layer(share=True) by the number of sequences, with the forks that they know of
        self._forks = 0
        self._ended = False                 # a change has reached the host's table and not the device's
        self._appended = set()              # layers that the caller's own append has written, for as long as no layer() is out
        self._progress = None               # what retrieval.teacher has written, from the first layer() on

    # -------------------------------------------------------------------------------------------- sequences and pages
    @property
    def free_pages(self) -> int:
        return self.host.n_free

    def length(self, slot: int) -> int:
        """Tokens of a slot, as the host knows them (no device read)."""
        if not 0 <= slot < self.host.slots:
            raise ValueError(_REASONS[1].format(slots=self.host.slots))
        return int(self.host.lens[slot])

    def _apply(self, change, *args) -> None:
        """The host's change, then the device's.  Not for a capture: a replay would not repeat the host's part.  A change that
        fails on the device leaves its table behind the host's, so the cache ends there."""
        self._check()
        with on_device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("heimdall_b200: pages are given out on the host: reserve, fork, free, truncate and compact "
                                   "cannot be captured into a CUDA graph")
            todo = change(*args)
            self._ended = True
            flat, some = [], 0
            for name in ("release", "fork", "move", "set"):
                x = todo.get(name)
                n = 0 if x is None else x.shape[0]
                flat += (x.ctypes.data, n) if n else (0, 0)
                some += n
            if some:
                _lib.call("bf_paged_pages", self._pool_ptr, *flat, stream_handle())
            self._ended = False

    def _check(self) -> None:
        if self._ended:
            raise RuntimeError("heimdall_b200: a change of pages failed on the device, whose table is behind the host's: this "
                               "cache cannot be used any more")

    def reserve(self, slots, n) -> None:
        """Room for n more tokens (one number, or one per slot) of each slot; they belong to the sequences from here on.
        Raises RuntimeError, with nothing changed, when the pool has too few free pages."""
        self._apply(self.host.reserve, slots, n)

    def free(self, slots) -> None:
        """End the sequences of these slots: their pages return to the pool unless another sequence shares them."""
        self._apply(self.host.free, slots)
        self._cut(slots)
        if self._progress is not None:
            self._progress.free(slots)

    def fork(self, src, dst) -> None:
        """The (empty) slots dst continue the sequences of src: full pages are shared, the tokens of a partly filled last
        page are copied, in every layer."""
        self._apply(self.host.fork, src, dst)
        self._forks += 1
        if self._progress is not None:
            self._progress.fork(src, dst)

    def truncate(self, slots, lens) -> None:
        """Shorten the sequences of these slots to lens tokens (rejected drafts); a shared page that becomes partly filled
        is copied.  The scale of the page that is cut stays as it is."""
        self._apply(self.host.truncate, slots, lens)
        self._cut(slots, lens)
        if self._progress is not None:
            self._progress.truncate(slots, lens)

    def _cut(self, slots, lens=0) -> None:
        if self._plans:
            slots = self.host._whole(slots)
            lens = self.host._whole(lens, slots).tolist()
            for plan in self._plans:
                plan._cut(slots.tolist(), lens)

    def compact(self) -> int:
        """Move the live pages at or above their number into the holes below it (both in ascending order), so that the
        pool is in use from page 0 on.  Returns the number of live pages."""
        self._apply(self.host.compact)
        return self.host.pages - self.host.n_free

    def share(self, slots, into: SharedPages = None, min_saved: int = None) -> SharedPages:
        """Which pages these sequences (slots, a list of whole numbers; one may come several times) have in common, for ``attend(shared=)``: the
        runs of pages that are read once for several of them.  The plan is good until a slot of it is freed or truncated into the pages that it
        shares (attend refuses it after that); everything else leaves it good, though sequences forked later are not in it.  ``into``: a plan of as many sequences,
        whose device memory takes the new one, so that a captured attend goes on with it.  Runs that save fewer than
        ``min_saved`` tokens of reading ((sequences - 1) * tokens) are left out; None: those that are not worth their start, which is all of them if
        together they save fewer than 32768 and 512 for each sequence (attend is then the call without a plan).  At most four
        runs to a sequence; deeper ones are read sequence by sequence."""
        self._check()
        if into is not None and (not isinstance(into, SharedPages) or into.cache is not self):
            raise ValueError("into must be a plan of this cache")
        if min_saved is not None and min_saved < 1:
            raise ValueError("min_saved must be positive")
        slots = self.host._whole(slots)
        if into is not None and into.n != slots.size:
            raise ValueError(f"into is a plan of {into.n} sequences, not of {slots.size}")
        with on_device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("heimdall_b200: what is shared is found on the host: share cannot be captured into a CUDA graph")
            plan = self.host.share(slots, MIN_SAVED if min_saved is None else min(int(min_saved), 2 ** 31 - 1))
            if min_saved is None:
                n = slots.size
                runs = plan[4 + 5 * n:4 + 5 * n + 6 * int(plan[0])].reshape(-1, 6).astype(np.int64)
                if ((runs[:, 1] - 1) * (runs[:, 3] - runs[:, 2])).sum() * self.page < WORTH[0] + WORTH[1] * n:
                    plan = self.host.share(slots, 2 ** 31 - 1)
            if into is None:
                return SharedPages(self, slots, plan)
            into._fill(slots, plan)
        return into

    # -------------------------------------------------------------------------------------------- keys and values
    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} is outside [0, {self.layers})")
        return int(layer)

    def _ids(self, slots, B: int):
        if slots is None:
            if B > self.host.slots:
                raise ValueError("more sequences than the cache has slots")
            return None
        serving_inputs("PagedKV", self.k_pages, slots)
        slots = int32_on(self.device, "slots", slots)
        if slots.numel() != B:
            raise ValueError("slots needs one entry per sequence")
        return slots

    def append(self, layer: int, k, v, slots=None, cu_seqlens=None) -> None:
        """Write the newest tokens of each sequence, already reserved: k, v [B,t,G,D], or [T,G,D] packed with cu_seqlens
        [B+1], whose entries must not descend (one below 0 counts as 0, one beyond T as T; after a descending one, which
        prompt_attention takes for the one before it, not all tokens may be written).  Sequence b (slot
        slots[b], an int tensor on the device; None: slot b) gets its n_b tokens at the positions lens - n_b .. lens - 1,
        which are to be its own: tokens from before a fork may lie in pages that it shares.
        A page's scale covers what was written to it; earlier codes of a page whose scale grows are rounded to the new one.
        Infinities are stored as the largest code, NaN as NaN.  A slot named twice is written by its first sequence, a
        number outside the cache's slots by none."""
        B = self._append(layer, k, v, slots, cu_seqlens)
        if B and self._progress is None:
            self._appended.add(layer)
        elif B:
            self._progress.appended(int(layer), slots, B)

    def _append(self, layer: int, k, v, slots=None, cu_seqlens=None) -> int:
        self._check()
        dev = serving_inputs("PagedKV.append", self.k_pages, k, v)
        layer, shape, packed = self._layer(layer), k.shape, cu_seqlens is not None
        if shape != v.shape or k.dtype != v.dtype or len(shape) != (3 if packed else 4):
            raise ValueError("append takes k and v alike: [B,t,G,D], or [T,G,D] with cu_seqlens")
        if shape[-2] != self.heads or shape[-1] != self.dim:
            raise ValueError(f"append takes {self.heads} heads of {self.dim}")
        with on_device(dev):
            cu = int32_on(dev, "cu_seqlens", cu_seqlens) if packed else None
            B = cu.numel() - 1 if packed else shape[0]
            if B < 0:
                raise ValueError("cu_seqlens needs one entry more than there are sequences")
            ids = self._ids(slots, B)
            k, kp, ks = heads_16bit("k", k)
            v, vp, vs = heads_16bit("v", v)
            if packed:
                ks, vs = [0] + ks, [0] + vs
            _lib.call("bf_paged_append", self._pool_ptr, layer, kp, *ks, vp, *vs, ptr(ids), ptr(cu), B, shape[-3], kernel_dtype(k),
                      stream_handle())
        return B if shape[-3] else 0        # the sequences that tokens may have been written of

    def attend(self, layer: int, q, slots=None, scale=None, with_lse: bool = False, shared: SharedPages = None):
        """Attention of each sequence's last t tokens over its pages: q [B,t,H,D] (bf16 or fp16; H a multiple of the KV
        heads) at the positions lens - t .. lens - 1, each seeing the positions up to its own.  Returns o [B,t,H,D] in q's
        dtype and lse [B,H,t] fp32 (None unless ``with_lse``); a token that sees nothing has o = 0 and lse = -inf.  What the
        pages hold behind a sequence's last token has no part in it; a NaN among a sequence's stored values reaches all t
        tokens.  A component of q is held to 2^-25 of the largest of its row and head (exactly, where it is above about 2^-14 of
        that).  A token's weight times its V scale is held to 2^-11 of itself or 2^-26 of (largest weight) * (largest V scale) among
        the 128 tokens of its tile, whichever is more.  Made for decode steps and drafts: 24 rows (tokens times query heads per KV
        head) share one way through the pages, so t tokens take as long as t / floor(24 / (H / G)) of them.

        ``shared``: a plan of ``share`` in the place of slots: its sequences, in its order, each shared page read once for all of them.  There a
        component of q is held to 2^-17 of the largest of its row and head (exactly, where its own bits do not end below that), a token's weight times
        its V scale to 2^-9 (fp16: 2^-12) of itself or 2^-18 of the largest among the 128 tokens of its tile, and V scales of
        a sequence may be 2^100 apart."""
        self._check()
        dev = serving_inputs("PagedKV.attend", self.k_pages, q)
        layer, shape = self._layer(layer), q.shape
        if len(shape) != 4 or shape[3] != self.dim or shape[2] % self.heads or shape[2] < 1:
            raise ValueError(f"attend takes q [B,t,H,{self.dim}] with H a multiple of {self.heads}")
        B, t, H, D = shape
        if H // self.heads > MAX_GROUP:
            raise NotImplementedError(f"attend takes at most {MAX_GROUP} query heads per KV head")
        scale = score_scale(scale, D)
        if shared is not None:
            self._check_plan(shared, slots, B)
        with on_device(dev):
            if shared is None:
                ids = self._ids(slots, B)
            elif not shared.runs:
                ids, shared = shared._slot_ids, None                 # nothing to share
            q, qp, qs = heads_16bit("q", q)
            o = q.new_empty(shape)
            lse = q.new_empty((B, H, t), dtype=torch.float32) if with_lse else None
            if shared is not None:
                nws = self._ws.get((B, t, H, True))
                if nws is None:
                    nws = self._ws[B, t, H, True] = max(_lib.size("bf_paged_attend_shared_workspace", B, t, H, self.heads, D), 16)
                ws = q.new_empty((nws,), dtype=torch.uint8)
                _lib.call("bf_paged_attend_shared", self._pool_ptr, layer, qp, *qs, shared.plan.data_ptr(), B, t, H, kernel_dtype(q), scale,
                          o.data_ptr(), ptr(lse), ws.data_ptr(), nws, stream_handle())
                return o, lse
            nws = self._ws.get((B, t, H))
            if nws is None:
                nws = self._ws[B, t, H] = max(_lib.size("bf_paged_attend_workspace", B, t, H, self.heads, D), 16)
            ws = q.new_empty((nws,), dtype=torch.uint8)
            _lib.call("bf_paged_attend", self._pool_ptr, layer, qp, *qs, ptr(ids), B, t, H, kernel_dtype(q), scale, o.data_ptr(),
                      ptr(lse), ws.data_ptr(), nws, stream_handle())
        return o, lse

    def _check_plan(self, shared, slots, B: int) -> None:
        if not isinstance(shared, SharedPages) or shared.cache is not self:
            raise ValueError("shared must be a plan of this cache's share")
        if slots is not None:
            raise ValueError("the plan of shared pages has its own slots")
        if shared.n != B:
            raise ValueError(f"the plan is of {shared.n} sequences, not of {B}")
        if not shared.good:
            raise ValueError("slots were freed, or truncated into shared pages, since this plan was made: share again")

    def layer(self, layer: int, share: bool = False) -> "PagedLayer":
        """This cache as one kept layer's ``cache`` argument of ``retrieval.teacher`` (slots 0 .. B-1).  How far the layer
        is belongs to the cache: fetched once or for every call, a layer goes on where it was.  ``share``: pages that
        the sequences have in common are read once for all of them (``attend(shared=)``, with its precision there); the plan, one for
        all layers, is made at the first call that needs it and after forks, and again when it is no longer good.  That is host work: before such a call is captured,
        one has to have run.  One plan is kept for each number of sequences, for the calls captured with it."""
        return PagedLayer(self, self._layer(layer), share)

    def _layer_plan(self, B: int):
        plan, forks = self._layer_plans.get(B, (None, -1))
        if forks != self._forks or not plan.good:
            plan = self.share(range(B), into=plan)
            self._layer_plans[B] = plan, self._forks
        return plan if plan.runs else None


class _Progress:
    """What ``retrieval.teacher`` has written: the tokens of each slot in each layer, UNKNOWN where the host cannot tell, because the
    caller's own ``append`` may have written a sequence's newest tokens there."""

    UNKNOWN = -2 ** 40              # so far below any length that no number of new tokens makes one of it

    def __init__(self, cache: PagedKV):
        self.host = cache.host
        self.n = np.zeros((cache.layers, self.host.slots), np.int64)
        self.room = np.zeros(self.host.slots, np.int64)     # a slot's length when teacher last made room in it
        for layer in cache._appended:
            self.n[layer, self.host.lens > 0] = self.UNKNOWN

    def free(self, slots) -> None:
        s = self.host._whole(slots)
        self.n[:, s] = self.room[s] = 0

    def fork(self, src, dst) -> None:
        a, b = self.host._whole(src), self.host._whole(dst)
        self.n[:, b], self.room[b] = self.n[:, a], self.room[a]

    def truncate(self, slots, lens) -> None:
        s = self.host._whole(slots)
        m = self.host._whole(lens, s)
        self.n[:, s], self.room[s] = np.minimum(self.n[:, s], m), np.minimum(self.room[s], m)
        self.n[:, s[m == 0]] = 0

    def appended(self, layer: int, slots, B: int) -> None:
        """The caller's own append of B sequences to a layer: what was reserved by the caller, and not by teacher, may be
        written now.  (Which slots it named is read back from the device where that matters, but not in a capture.)"""
        n, lens = self.n[layer], self.host.lens
        may = (n >= 0) & (n < lens) & (lens != self.room)
        if slots is None:
            may[B:] = False
        elif may.any() and not (slots.is_cuda and torch.cuda.is_current_stream_capturing()):
            named = np.asarray(slots.tolist(), np.int64)
            may &= np.isin(np.arange(n.size), named)
        n[may] = self.UNKNOWN


class PagedLayer:
    """One layer of a ``PagedKV`` as the cache of ``retrieval.teacher``: every call brings the next t tokens of each of the
    sequences in the slots 0 .. B-1.  The first layer that needs room reserves it (or the caller has, for exactly these tokens), and
    every layer takes the same tokens.  ``free``, ``truncate`` and ``fork`` of the cache are followed.  A sequence whose tokens were
    written to the layer with ``append`` is not gone on with: ``attend`` is the call for those.  (Beside
    teacher, an ``append`` to sequences whose room the caller reserved waits for its slot numbers to be read back.)  Replays of a captured
    call are not seen by the host; what was captured goes on by replays, or anew after ``free``."""

    def __init__(self, cache: PagedKV, layer: int, share: bool = False):
        self.cache, self.index, self.share = cache, layer, bool(share)
        if cache._progress is None:
            cache._progress = _Progress(cache)

    @property
    def n(self) -> int:
        """Tokens of the longest sequence that this layer holds.  Setting it says that the layer holds n tokens of each sequence."""
        return max(int(self.cache._progress.n[self.index].max()), 0)

    @n.setter
    def n(self, tokens: int) -> None:
        p = self.cache._progress
        p.n[self.index, p.host.lens > 0] = tokens

    def teacher(self, qr, kr, v, retrieval=None):
        c = self.cache
        B, H, t, D = qr.shape
        # what would be refused after the keys and values are written (append refuses kr and v before that)
        if qr.device != c.device or (qr.requires_grad and torch.is_grad_enabled()):
            serving_inputs("retrieval.teacher over pages", c.k_pages, qr)
        if v.shape != (B, t, c.heads, c.dim) or D != c.dim or H % c.heads or H < 1:
            raise ValueError(f"teacher over pages takes qr [B,H,t,{c.dim}], kr [B,{c.heads},t,{c.dim}] and v [B,t,{c.heads},{c.dim}] "
                             f"with H a multiple of {c.heads}")
        if B > c.host.slots:
            raise ValueError("more sequences than the cache has slots")
        p, lens = c._progress, c.host.lens[:B]
        had = p.n[self.index, :B]
        later = bool(had.any())
        if retrieval is not None and (t == 1 or retrieval.get("prefill")) and \
                int(had.max(initial=0)) + t - retrieval["sinks"] - retrieval["window"] >= retrieval["k"] * retrieval["block"]:
            raise NotImplementedError("heimdall_b200 retrieval: block selection over 8-bit pages is not built")
        if later and H // c.heads > MAX_GROUP:
            raise NotImplementedError(f"attend takes at most {MAX_GROUP} query heads per KV head")
        make_room = had.tobytes() == lens.tobytes()            # (a fifth of the time of comparing the arrays)
        if make_room:
            c.reserve(np.arange(B), t)
            p.room[:B] = lens
        elif (had + t).tobytes() != lens.tobytes():
            if (had < 0).any():
                raise ValueError("a sequence's tokens in this layer were written with append: attend goes on from there, not teacher")
            raise ValueError("the layers of a paged cache must take the same tokens in step")
        try:
            o = self._attend(qr, kr, v, later)
        except BaseException:
            if make_room:                 # nothing of the sequences has changed but their room
                c.truncate(np.arange(B), had.copy())
            raise
        had[:] = lens
        return o

    def _attend(self, qr, kr, v, later: bool):
        c, (B, H, t, D) = self.cache, qr.shape
        dt = kr.dtype if kr.dtype == torch.float16 else torch.bfloat16
        q, k, v = qr.transpose(1, 2).to(dt), kr.transpose(1, 2).to(dt), v.to(dt)
        plan = c._layer_plan(B) if later and self.share else None      # (a capture that has none is refused before it writes)
        c._append(self.index, k, v)
        if later:
            return c.attend(self.index, q, shared=plan)[0].to(qr.dtype)
        # a whole prompt: attention over the keys and values as they are, not over their codes
        cu = torch.arange(B + 1, device=qr.device, dtype=torch.int32) * t
        o, _ = prompt_attention(q.reshape(B * t, H, D), k.reshape(B * t, c.heads, D), v.reshape(B * t, c.heads, D), cu)
        return o.reshape(B, t, H, D).to(qr.dtype)
