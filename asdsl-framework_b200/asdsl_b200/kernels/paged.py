"""A batch of requests over a paged key/value cache, on the sm_100a kernels.

One serving step of a layer:

    plan = StepPlan(max_requests, max_tokens, max_pages, page_size)
    plan_step(plan, kv_lens, new_lens, free_pages)        # block table, slots, row starts
    kv_write(cache, k, v, plan.slots)                     # the new keys and values
    out = attention_paged(q, cache, plan.block_table, plan.total_lens, plan.cu_q, window=4096, sinks=4)

``attention_shared_prefix`` serves requests that begin with the same positions (a system prompt, a
document): those are attended once for the whole batch.

All tensors are CUDA tensors on one device; calls enqueue work on torch's current stream of that
device and do not synchronize.  Lengths and tables are read on the device, so a step can be captured
in a CUDA graph.  There is no CPU path: without the library or a GPU the calls raise.  The operators
are for inference: what they return carries no gradient, whatever the inputs require.
"""

from __future__ import annotations

import ctypes
import math

import torch

from asdsl_b200 import _lib

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.int8: _lib.I8}
_I32 = torch.int32
MAX_REQUESTS = 12288  # of one plan_step

# A step of a small batch is a few microseconds of GPU work, so the checks below are written to cost
# little: messages are built only where a check fails, the entry points are looked up once.
_entries: dict = {}


def _entry(name: str):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    return fn


def _not_cuda(t, name: str):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")


def _check(t, name: str, dtype, dims: int, device) -> None:
    """t is a CUDA tensor of this type and number of dimensions, on `device` (None: any)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got {t.dim()}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the call on {device}")


def _vector(t, name: str, n: int, device, dtype=_I32) -> None:
    """t is a contiguous vector of n entries (n < 0: any number)."""
    _check(t, name, dtype, 1, device)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if n >= 0 and t.numel() != n:
        raise ValueError(f"{name} must have {n} entries, got {t.numel()}")


def _call(device: torch.device, name: str, *args) -> None:
    """Run an entry point on torch's current stream of `device` (its last argument)."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = _entry(name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = _entry(name)(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


# the current stream's handle without building a Stream object
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


class StepPlan:
    """The buffers of a step's plan, kept from step to step.

    ``block_table`` [max_requests, max_pages] int32 is the state: row b names the pages of the request
    in row b, in order; ``plan_step`` appends to it and the caller resets the rows of requests that
    left.  The rest is rewritten by each ``plan_step`` of n requests: ``cu_q`` [n + 1], ``total_lens``
    [n], and ``slots``, ``positions``, ``requests`` [max_tokens] of the new tokens (-1, 0, -1 past the
    last), ``counts`` = (pages taken, new tokens, flags).

    ``total_lens`` may be the next step's kv_lens: a step that reads it writes its totals to another buffer,
    which ``total_lens`` then names.  (A captured step replays with the buffers of its capture: give it lengths
    in a buffer of the caller's.)
    """

    FREE_SHORT, TABLE_NARROW, TOKENS_OVER = 1, 2, 4  # counts[2]

    def __init__(self, max_requests: int, max_tokens: int, max_pages: int, page_size: int, device=None):
        if not 0 < max_requests <= MAX_REQUESTS:
            raise ValueError(f"max_requests must be 1 to {MAX_REQUESTS}")
        if max_tokens <= 0 or max_pages <= 0 or page_size <= 0:
            raise ValueError("max_tokens, max_pages and page_size must be positive")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.page_size, self.max_tokens = page_size, max_tokens
        self._table = torch.full((max_requests, max_pages), -1, dtype=torch.int32, device=device)
        self._cu = torch.zeros(max_requests + 1, dtype=torch.int32, device=device)
        self._totals = torch.zeros(2, max_requests, dtype=torch.int32, device=device)
        self.slots = torch.full((max_tokens,), -1, dtype=torch.int32, device=device)
        self.positions = torch.zeros(max_tokens, dtype=torch.int32, device=device)
        self.requests = torch.full((max_tokens,), -1, dtype=torch.int32, device=device)
        self.counts = torch.zeros(3, dtype=torch.int32, device=device)
        self._total_ptrs = self._totals[0].data_ptr(), self._totals[1].data_ptr()
        self._buffers = tuple((self._table.data_ptr(), self._table.stride(0), max_pages, self._cu.data_ptr(), total,
                               self.slots.data_ptr(), self.positions.data_ptr(), self.requests.data_ptr(), max_tokens,
                               self.counts.data_ptr()) for total in self._total_ptrs)
        self._set(max_requests, 0)

    def _set(self, n: int, which: int) -> None:
        self.n, self._which = n, which
        self.block_table, self.cu_q, self.total_lens = self._table[:n], self._cu[: n + 1], self._totals[which, :n]


def plan_step(plan: StepPlan, kv_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor) -> StepPlan:
    """Fill `plan` for a step of ``len(kv_lens)`` requests that hold kv_lens tokens and gain new_lens.

    The pages a request gains come from the front of `free_pages` in request order (``counts[0]`` of
    them in all).  Lengths, tables and slots stay on the device; the flags in ``counts[2]`` tell of a
    free list that was too short, a request past max_pages, or tokens past max_tokens -- what did not
    fit has page and slot -1, which ``kv_write`` and the attention pass over.  kv_lens may be the last
    step's ``plan.total_lens``; otherwise the inputs must not share memory with the plan's buffers.
    """
    table = plan._table
    device = table.device
    _vector(kv_lens, "kv_lens", -1, device)
    n = kv_lens.numel()
    _vector(new_lens, "new_lens", n, device)
    _vector(free_pages, "free_pages", -1, device)
    if n > table.shape[0]:
        raise ValueError(f"{n} requests, the plan has rows for {table.shape[0]}")
    kv = kv_lens.data_ptr()
    first, second = plan._total_ptrs
    which = 1 if first <= kv < second else 0  # the totals of the last step may be read here
    if plan.n != n or plan._which != which:
        plan._set(n, which)
    _call(device, "asdsl_b200_plan_step", kv, new_lens.data_ptr(), n, free_pages.data_ptr(), free_pages.numel(),
          plan.page_size, *plan._buffers[which])
    return plan


class PagedKV:
    """One layer's cache in pages: k and v [pages, page_size, kv_heads, head_dim].

    bf16, fp16, or int8 codes with fp32 scales [pages, page_size, kv_heads, head_dim / 64], one for each
    64 dims as in the decode engine's cache.  k and v may be strided alike (the halves of one tensor, heads before positions), with
    consecutive head_dim and strides of multiples of 16 bytes; scales are contiguous.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor | None = None,
                 v_scales: torch.Tensor | None = None):
        _not_cuda(k, "k")
        if k.dtype not in (torch.bfloat16, torch.float16, torch.int8):
            raise ValueError(f"a cache of {k.dtype} is not supported")
        _check(k, "k", k.dtype, 4, None)
        _check(v, "v", k.dtype, 4, k.device)
        if k.shape != v.shape or k.stride() != v.stride():
            raise ValueError("k and v must have the same shape and strides")
        if k.stride(3) != 1:
            raise ValueError("head_dim must be consecutive in memory")
        if k.dtype == torch.int8:
            shape = (*k.shape[:3], k.shape[3] // 64)
            for name, s in (("k_scales", k_scales), ("v_scales", v_scales)):
                _check(s, name, torch.float32, 4, k.device)
                if tuple(s.shape) != shape or not s.is_contiguous():
                    raise ValueError(f"{name} must be contiguous {shape}")
        elif k_scales is not None or v_scales is not None:
            raise ValueError("scales belong to an int8 cache")
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self.pages, self.page_size, self.kv_heads, self.head_dim = k.shape
        self.dtype, self.device = k.dtype, k.device
        self._c = _lib.PagedCacheC(k.data_ptr(), v.data_ptr(), _ptr(k_scales), _ptr(v_scales), k.stride(0), k.stride(1),
                                   k.stride(2), _TYPES[k.dtype], *k.shape)
        self._ref = ctypes.addressof(self._c)

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.int8, device=None) -> "PagedKV":
        """A cache without contents (a position is read only after it was written)."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        shape = (pages, page_size, kv_heads, head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        if dtype != torch.int8:
            return cls(k, v)
        if head_dim % 64:
            raise ValueError("head_dim must be 64 or 128")
        ks, vs = (torch.empty((*shape[:3], head_dim // 64), dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs)


def kv_write(cache: PagedKV, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Write k and v [tokens, kv_heads, head_dim] to the cache's slots (``plan.slots``; -1 is skipped).

    fp32, bf16 or fp16 into an int8 cache, a 16-bit type or fp32 into a cache of that 16-bit type.  int8: per
    64 dims the scale is max / 127 and the code the nearest multiple, with the decode engine's scales bit for
    bit and its codes but where a value lies within 2^-22 of the boundary between two of them.  Both may be
    strided alike, as columns of one projection.  A slot named twice in one call holds one of the two tokens.
    """
    _not_cuda(k, "k")
    dtype, device = k.dtype, cache.device
    if dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"k and v of {dtype} are not supported")
    _check(k, "k", dtype, 3, device)
    _check(v, "v", dtype, 3, device)
    n, heads, dim = k.shape
    if heads != cache.kv_heads or dim != cache.head_dim:
        raise ValueError(f"k must be [tokens, {cache.kv_heads}, {cache.head_dim}]")
    stride = k.stride()
    if v.shape != k.shape or v.stride() != stride:
        raise ValueError("k and v must have the same shape and strides")
    if n and stride[2] != 1:
        raise ValueError("head_dim must be consecutive in memory")
    _vector(slots, "slots", -1, device)
    if slots.numel() < n:
        raise ValueError(f"{n} tokens, {slots.numel()} slots")
    _call(cache.device, "asdsl_b200_kv_write", cache._ref, k.data_ptr(), v.data_ptr(), _TYPES[dtype], stride[0],
          stride[1], slots.data_ptr(), n)


class AttentionWorkspace:
    """Device scratch of the attention calls of ONE stream; grows to the largest call.

    Calls that may overlap in time (on several streams) need one each.  Grown outside graph capture
    only: run a step once on it before capturing one.  A captured graph goes on using the buffers that it was
    captured with, so keep the workspace as long as the graph: buffers that a later, larger call outgrew
    stay with it.  A captured call that brings no workspace takes its scratch from the graph's own memory
    (one more small launch, which clears the arrival counters).
    """

    def __init__(self):
        self._ws: torch.Tensor | None = None
        self._merge: torch.Tensor | None = None
        self._outgrown: list[torch.Tensor] = []
        self._bytes: dict[tuple, int] = {}

    def _grown(self, t, n: int, dtype, device, fill: bool):
        if t is not None and t.numel() >= n and t.device == device:
            return t
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the attention workspace must grow: run the step once before capturing it")
        if t is not None:
            self._outgrown.append(t)
            if t.device == device:
                n = max(n, t.numel() + t.numel() // 2)  # what is outgrown adds up to twice the buffer in use at most
        return (torch.zeros if fill else torch.empty)(n, dtype=dtype, device=device)

    def _size(self, device, entry: str, *key) -> int:
        n = self._bytes.get(key)
        if n is None:
            with torch.cuda.device(device):
                n = getattr(_lib.load(), entry)(*key)
            if len(self._bytes) > 4096:
                self._bytes.clear()
            self._bytes[key] = n
        return n

    def sized(self, device, n_req: int, tokens: int, heads: int, kv_heads: int) -> torch.Tensor:
        n = self._size(device, "asdsl_b200_attention_workspace_bytes", n_req, tokens, heads, kv_heads)
        self._ws = self._grown(self._ws, n, torch.uint8, device, True)
        return self._ws

    def merge(self, device, tokens: int, heads: int, dim: int) -> torch.Tensor:
        n = self._size(device, "asdsl_b200_attention_merge_bytes", tokens, heads, dim)
        self._merge = self._grown(self._merge, n, torch.uint8, device, False)
        return self._merge


class _CaptureWorkspace(AttentionWorkspace):
    """Scratch of one captured call, from the graph's own pool: it lives as long as the graph and is no other
    call's.  The arrival counters are cleared by the graph."""

    def sized(self, device, n_req: int, tokens: int, heads: int, kv_heads: int) -> torch.Tensor:
        n = self._size(device, "asdsl_b200_attention_workspace_bytes", n_req, tokens, heads, kv_heads)
        counters = self._size(device, "asdsl_b200_attention_workspace_bytes", 0, 0, heads, kv_heads)  # their offset
        ws = torch.empty(n, dtype=torch.uint8, device=device)
        ws[counters:].zero_()
        return ws

    def merge(self, device, tokens: int, heads: int, dim: int) -> torch.Tensor:
        n = self._size(device, "asdsl_b200_attention_merge_bytes", tokens, heads, dim)
        return torch.empty(n, dtype=torch.uint8, device=device)


_stream_workspaces: dict[tuple, AttentionWorkspace] = {}
_MAX_STREAM_WORKSPACES = 16  # about 30 MB each; the oldest goes, in its stream's order, and is made anew when wanted
_capture_workspace = _CaptureWorkspace()  # holds sizes, no buffers


def _workspace(device) -> AttentionWorkspace:
    """The workspace of torch's current stream, kept for calls that bring none."""
    if torch.cuda.is_current_stream_capturing():
        return _capture_workspace
    key = (device.index, _raw_stream(device.index))
    ws = _stream_workspaces.get(key)
    if ws is None:
        if len(_stream_workspaces) >= _MAX_STREAM_WORKSPACES:
            del _stream_workspaces[next(iter(_stream_workspaces))]
        ws = _stream_workspaces[key] = AttentionWorkspace()
    return ws


def _attention_inputs(q, cache, block_table, kv_lens, cu_q, scale, out, lse, return_lse):
    _not_cuda(q, "q")
    dtype, device = q.dtype, q.device
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"q must be bfloat16 or float16, got {dtype}")
    if cache.dtype is not dtype and cache.dtype is not torch.int8:
        raise ValueError(f"a cache of {cache.dtype} needs q of that type, got {dtype}")
    if cache.device != device:
        raise ValueError(f"the cache is on {cache.device}, q on {device}")
    if q.dim() != 3:
        raise ValueError(f"q must have 3 dimensions, got {q.dim()}")
    tokens, heads, d = q.shape
    if d != cache.head_dim:
        raise ValueError(f"q has head_dim {d}, the cache {cache.head_dim}")
    if heads <= 0 or heads % cache.kv_heads:
        raise ValueError(f"{heads} heads are not a multiple of {cache.kv_heads} kv heads")
    if tokens and q.stride(2) != 1:
        raise ValueError("head_dim of q must be consecutive in memory")
    _check(block_table, "block_table", _I32, 2, device)
    n, width = block_table.shape
    if width > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table's rows must be consecutive in memory")
    _vector(kv_lens, "kv_lens", n, device)
    if cu_q is not None:
        _vector(cu_q, "cu_q", n + 1, device)
    elif tokens != n:
        raise ValueError(f"without cu_q every request has one row: {tokens} rows, {n} requests")
    if out is None:
        out = q.new_empty((tokens, heads, d))
    else:
        _check(out, "out", dtype, 3, device)
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError("out must be contiguous and of q's shape")
    if lse is not None:
        _check(lse, "lse", torch.float32, 2, device)
        if tuple(lse.shape) != (tokens, heads) or not lse.is_contiguous():
            raise ValueError(f"lse must be contiguous {(tokens, heads)}")
    elif return_lse:
        lse = q.new_empty((tokens, heads), dtype=torch.float32)
    scale = d**-0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("scale must be positive and finite")
    return out, lse, scale


def attention_paged(q: torch.Tensor, cache: PagedKV, block_table: torch.Tensor, kv_lens: torch.Tensor,
                    cu_q: torch.Tensor | None = None, *, window: int = 0, sinks: int = 0, scale: float | None = None,
                    out: torch.Tensor | None = None, lse: torch.Tensor | None = None, return_lse: bool = False,
                    workspace: AttentionWorkspace | None = None):
    """Causal attention of new tokens over their requests' pages, grouped heads, with an optional
    sliding window and sink tokens.

    q [tokens, heads, head_dim] (bf16 or fp16) holds the new tokens of request b in rows cu_q[b] ..
    cu_q[b + 1] - 1 (cu_q None: one row per request); kv_lens[b] counts its keys, the new ones among
    them.  The i-th of n new tokens stands at p = kv_len - n + i and sees keys j <= p; with window > 0
    only those with j > p - window or j < sinks.  Returns out (of q's shape and type), or (out, lse)
    with return_lse: lse [tokens, heads] is the log of the sum of exp(scale * q . k).  A row that sees no
    key gives 0 and -inf; a key whose table entry names no page, or that lies past the table, is not seen
    (positions come from kv_lens all the same).  Rows of q past cu_q[-1] are not written.  Softmax weights
    take part in the second product as 16-bit numbers, for fp16 products (fp16 queries; int8 caches with few
    rows) lifted by a power of two: all bits down to 2^-25 of the row's largest (int8: with each weight's V
    scale over the largest one among the keys so far).
    """
    out, lse, scale = _attention_inputs(q, cache, block_table, kv_lens, cu_q, scale, out, lse, return_lse)
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    tokens, heads, _ = q.shape
    n, width = block_table.shape
    device = q.device
    ws = (workspace or _workspace(device)).sized(device, n, tokens, heads, cache.kv_heads)
    _call(device, "asdsl_b200_attention_paged", q.data_ptr(), _TYPES[q.dtype], q.stride(0), q.stride(1), cache._ref,
          block_table.data_ptr(), block_table.stride(0), width, kv_lens.data_ptr(), _ptr(cu_q), n, tokens,
          heads, min(window, 2**31 - 1), min(sinks, 2**31 - 1), scale, out.data_ptr(), _ptr(lse), ws.data_ptr(), ws.numel())
    return (out, lse) if return_lse else out


def attention_shared_prefix(q: torch.Tensor, cache: PagedKV, prefix_pages: torch.Tensor, prefix_len: int,
                            block_table: torch.Tensor, kv_lens: torch.Tensor, cu_q: torch.Tensor | None = None, *,
                            scale: float | None = None, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                            return_lse: bool = False, workspace: AttentionWorkspace | None = None):
    """Attention of a batch whose requests all begin with the same `prefix_len` positions, held once in
    `prefix_pages`; block_table and kv_lens describe each request's own positions after them.

    Every row sees the whole prefix and, causally, its request's own keys -- the result of
    ``attention_paged`` over the joined keys -- but the prefix is read once for the batch.
    """
    out, lse, scale = _attention_inputs(q, cache, block_table, kv_lens, cu_q, scale, out, lse, return_lse)
    device = q.device
    _vector(prefix_pages, "prefix_pages", -1, device)
    if not 0 <= prefix_len <= prefix_pages.numel() * cache.page_size:
        raise ValueError(f"prefix_len {prefix_len} does not lie within {prefix_pages.numel()} pages of {cache.page_size}")
    tokens, heads, d = q.shape
    n = block_table.shape[0]
    space = workspace or _workspace(device)
    ws = space.sized(device, max(n, 1), tokens, heads, cache.kv_heads)
    merge = space.merge(device, tokens, heads, d)
    _call(device, "asdsl_b200_attention_shared_prefix", q.data_ptr(), _TYPES[q.dtype], q.stride(0), q.stride(1),
          cache._ref, prefix_pages.data_ptr(), prefix_pages.numel(), int(prefix_len), block_table.data_ptr(),
          block_table.stride(0), block_table.shape[1], kv_lens.data_ptr(), _ptr(cu_q), n, tokens, heads, scale,
          out.data_ptr(), _ptr(lse), merge.data_ptr(), merge.numel(), ws.data_ptr(), ws.numel())
    return (out, lse) if return_lse else out
