"""Low-rank adapters of many requests at once beside one shared projection.

A server that answers requests with adapters of their own runs one projection for the whole batch and adds to every token what its
request's adapter says: y + s_a B_a (A_a x).  ``Adapters`` holds the adapters of one projection on the device; ``BifrostAttention`` takes one for each of
its projections (``adapters=``, and each call's ``adapter_ids``).  There is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from .functional import heads_16bit, kernel_dtype, on_device, ptr, serving_inputs, stream_handle

MAX_RANK = 128
MAX_ADAPTERS = 4096


class Adapters:
    """The adapters of one projection: ``a`` a list of [r_i, d_in] and ``b`` of [d_out, r_i] tensors (bf16 or fp16, all of one dtype, ranks 1 to
    128, each its own), ``scale`` a number or one for each (usually alpha / r).  Laid out once on ``device`` (default: where a[0]
    is); later changes of the given tensors have no part in it.  d_in and d_out are multiples of 8."""

    def __init__(self, a, b, scale=1.0, device=None):
        a, b = list(a), list(b)
        if not a or len(a) != len(b) or any(t.dim() != 2 for t in a + b):
            raise ValueError("Adapters takes as many a [r,d_in] as b [d_out,r], at least one")
        d_in, d_out, dtype = a[0].shape[1], b[0].shape[0], a[0].dtype
        if any(x.shape[1] != d_in or y.shape[0] != d_out or x.shape[0] != y.shape[1] for x, y in zip(a, b)):
            raise ValueError("all a are [r,d_in] and all b [d_out,r], each pair of one rank")
        if any(t.dtype != dtype for t in a + b):
            raise ValueError("all adapters must have one dtype")
        if dtype not in (torch.bfloat16, torch.float16):
            raise NotImplementedError(f"adapters are {dtype}: built for bfloat16 and float16")
        ranks = [x.shape[0] for x in a]
        if min(ranks) < 1 or max(ranks) > MAX_RANK or len(a) > MAX_ADAPTERS:
            raise NotImplementedError(f"Adapters holds up to {MAX_ADAPTERS} adapters of ranks 1 to {MAX_RANK}")
        if d_in % 8 or d_out % 8 or min(d_in, d_out) < 8:
            raise NotImplementedError("Adapters is built for d_in and d_out that are multiples of 8")
        scale = [float(scale)] * len(a) if isinstance(scale, (int, float)) else [float(s) for s in scale]
        if len(scale) != len(a):
            raise ValueError("scale is one number, or one for each adapter")
        dev = torch.device(a[0].device if device is None else device)
        if dev.type != "cuda":
            raise RuntimeError("heimdall_b200 runs on CUDA tensors only (there is no CPU fallback)")
        self.n, self.d_in, self.d_out, self.dtype = len(a), d_in, d_out, dtype
        rows = [0]
        for r in ranks:                     # whole steps of 16 ranks, the rest zeros
            rows.append(rows[-1] + -(-r // 16) * 16)
        self.rmax = max(y - x for x, y in zip(rows, rows[1:]))
        self.a = torch.zeros(rows[-1], d_in, dtype=dtype, device=dev)
        self.b = torch.zeros(rows[-1] * d_out, dtype=dtype, device=dev)
        with torch.no_grad():
            for x, y, r, lo, hi in zip(a, b, ranks, rows, rows[1:]):
                self.a[lo:lo + r] = x
                part = torch.zeros(d_out, hi - lo, dtype=dtype, device=dev)       # in blocks of 8 columns and 8 ranks, as the tensor core reads them
                part[:, :r] = y
                self.b[lo * d_out:hi * d_out] = part.view(d_out // 8, 8, -1, 8).transpose(1, 2).reshape(-1)
        self.device = self.a.device
        self.rows = torch.tensor(rows, dtype=torch.int32, device=dev)
        self.scale = torch.tensor(scale, dtype=torch.float32, device=dev)
        self._at = tuple(ptr(t) for t in (self.a, self.b, self.rows, self.scale))
        self._ws = {}                       # workspace bytes by T

    def add(self, y, x, ids, out=None):
        """y + s_a B_a (A_a x) for every token: x [...,d_in] and y [...,d_out] in the adapters' dtype (any strides), ids [...] int32 or int64, the number of
        each token's adapter (outside 0 .. n - 1: none, out = y).  Returns ``out``: a new contiguous tensor, or the one given, which
        may be y itself.  A token's result does not depend on the other tokens beyond rounding.  A x is summed in fp32 and enters the
        second product to 2^-16 of itself (fp16: 2^-22); the sum with y is rounded once.  A token whose A x is not finite gets NaN."""
        dev = serving_inputs("Adapters.add", self.a, x, y)
        lead = x.shape[:-1]
        if x.shape[-1:] != (self.d_in,) or y.shape != (*lead, self.d_out) or ids.shape != lead:
            raise ValueError(f"Adapters.add takes y [...,{self.d_out}], x [...,{self.d_in}] and ids [...]")
        if x.dtype != self.dtype or y.dtype != self.dtype:
            raise ValueError(f"x and y must be {self.dtype}, as the adapters are")
        if ids.dtype not in (torch.int32, torch.int64):
            raise ValueError("ids must be int32 or int64")
        if out is not None and (out.shape != y.shape or out.dtype != y.dtype or out.device != dev or not out.is_contiguous() or out.data_ptr() % 16):
            raise ValueError("out must be contiguous, on a 16-byte boundary, of y's shape, dtype and device")
        with on_device(dev):
            if ids.dtype != torch.int32 or ids.device != dev or not ids.is_contiguous():
                # numbers above 31 bits name no adapter either
                ids = ids.to(device=dev).clamp(-1, self.n).to(torch.int32).contiguous()
            T = ids.numel()
            flat = len(lead) == 1
            x, xp, xs = heads_16bit("x", x if flat else x.reshape(T, self.d_in))
            y2, yp, ys = heads_16bit("y", y if flat else y.reshape(T, self.d_out))
            if out is None:
                out = torch.empty_like(y, memory_format=torch.contiguous_format)
            elif (out.data_ptr() != yp or (T > 1 and ys[0] != self.d_out)) and _overlap(out, y2):
                raise ValueError("out may be y, but not overlap it")
            nws = self._ws.get(T)
            if nws is None:
                nws = self._ws[T] = max(_lib.size("bf_adapter_workspace", T, self.n, self.d_in, self.rmax), 16)
            ws = x.new_empty((nws,), dtype=torch.uint8)
            a, b, rows, scale = self._at
            _lib.call("bf_adapter_add", xp, xs[0], ptr(ids), T, self.d_in, self.d_out, a, b, rows, scale, self.n, self.rmax, yp, ys[0],
                      out.data_ptr(), self.d_out, kernel_dtype(x), ws.data_ptr(), nws, stream_handle())
        return out


def _overlap(a, b) -> bool:
    def ends(t):
        lo = t.data_ptr()
        return lo, lo + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
    (a0, a1), (b0, b1) = ends(a), ends(b)
    return a0 < b1 and b0 < a1
