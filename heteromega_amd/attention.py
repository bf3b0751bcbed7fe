"""Attention over a paged key-value cache: the operators between a layer's Q/K/V projection and its O projection, over the
C ABI (include/hm_w4a16.h), and a layer's attention block made of them.

The reference's model keeps one contiguous cache per sequence and runs RoPE and decode attention on it
(src/hipkernels/flash_attn_decode.cu); here a step's requests share a cache of pages. A serving loop calls page_plan once
per step, and each layer then qk_norm_rope and paged_attention (or AttnLayer.block_forward, which calls both). Nothing waits for
the host: lengths, page ids and counters stay in device memory, so a step can be captured in a graph.
"""

import contextlib
import ctypes
import math

import torch

from . import _lib
from .ffn import (_DTYPES, _call, _current_raw_stream, _hm_dtype, _on, _stream, _workspace, packed_linear, residual_add2, rmsnorm)


class _MissingHost:
    """In the place of the compiled module where it is not built: the attention calls say so, and the rest of the package works without it."""

    def __init__(self, error):
        self._error = error

    def __getattr__(self, name):
        raise ImportError("heteromega_amd._attention_host is missing: run `python heteromega_amd/build.py` (or __graft_entry__.build()) first") from self._error


kPagePlanMaxRequests = 4096


def _bind():
    L = _lib.load()
    address = lambda f: ctypes.cast(f, ctypes.c_void_p).value
    current = _current_raw_stream or (lambda index: torch.cuda.current_stream(index).cuda_stream)
    _host.bind(address(L.hm_page_plan), address(L.hm_qk_norm_rope), address(L.hm_paged_attention), current, _stream)


try:
    # The checks and calls of the three operators, compiled: at few rows they took longer in Python than the kernels run.
    from . import _attention_host as _host
except ImportError as e:
    _host = _MissingHost(e)
else:
    _bind()


def _guard(device):
    """`device` as the current one, for a call that allocates or launches there."""
    if device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def rope_frequencies(rotary_dim, base=10000.0, device=None, llama3_scaling=None):
    """Radians per position of the rotary_dim / 2 pairs, base^(-2 i / rotary_dim), fp64 (qk_norm_rope's frequencies).
    llama3_scaling: (factor, low_freq_factor, high_freq_factor, original_context), as in the configuration of Llama 3.1 and 3.2
    models: pairs that turn less than low_freq_factor times in the original context are slowed down by factor, those that turn more than
    high_freq_factor times are kept, and those between are interpolated."""
    freq = []
    for i in range(rotary_dim // 2):
        f = base ** (-2.0 * i / rotary_dim)
        if llama3_scaling is not None:
            factor, low, high, context = llama3_scaling
            turns = context * f / (2.0 * math.pi)
            keep = min(1.0, max(0.0, (turns - low) / (high - low)))
            f = f * keep + f / factor * (1.0 - keep)
        freq.append(f)
    return torch.tensor(freq, dtype=torch.float64, device=device)


class PagedCache:
    """One layer's keys and values in pages, k and v [pages, kv_heads, page_size, head_dim] of one shape and one set of strides, the
    last dimension contiguous (a [pages, page_size, kv_heads, head_dim] array fits as its transpose(1, 2))."""

    def __init__(self, k, v):
        device = k.device
        if k.numel() == 0:
            raise ValueError(f"PagedCache: k and v must not be empty, got {list(k.shape)}")
        if device.type != "cuda":
            raise ValueError(f"PagedCache: needs device tensors, got one on {device}")
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or v.device != device:
            raise ValueError("PagedCache: k and v must be [pages, kv_heads, page_size, head_dim] alike in shape, strides, type and device")
        if k.stride(3) != 1:
            raise ValueError("PagedCache: the head dimension must be contiguous")
        self.k, self.v, self.device, self.dtype = k, v, device, k.dtype
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        # a dimension of one element may have any stride
        strides = [s if n > 1 else self.head_dim for s, n in zip(k.stride()[:3], k.shape[:3])]
        self._c = _lib.KvCache(k.data_ptr(), v.data_ptr(), self.pages, self.page_size, *strides, self.kv_heads, self.head_dim, _hm_dtype(k.dtype))
        self._ref, self._address = ctypes.byref(self._c), ctypes.addressof(self._c)

    @classmethod
    def empty(cls, pages, page_size, kv_heads, head_dim, dtype=torch.bfloat16, device="cuda"):
        """A new cache; its contents are read only where tokens were written."""
        device = torch.device(device)
        return cls(*(torch.empty((pages, kv_heads, page_size, head_dim), dtype=dtype, device=device) for _ in range(2)))

    def attention_workspace_bytes(self, q_heads):
        return _lib.load().hm_paged_attention_workspace_bytes(self._ref, q_heads)

    def attention_workspace(self, q_heads, stream=None):
        """A workspace for paged_attention calls on one stream, for any rows and lengths."""
        with _guard(self.device):
            return _workspace(self.attention_workspace_bytes(q_heads), self.device, stream)


class PagePlan:
    """What page_plan works out for a step of up to `rows` new tokens of `requests` requests, kept from step to step (a captured
    step's layers read these tensors): slots, positions and requests of each row, starts of the requests' rows, and their lengths
    and the page queue's counters after the step."""

    def __init__(self, requests, rows, page_size, device="cuda"):
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        new = lambda n, t: torch.full((n,), -1, dtype=t, device=device)
        self.page_size, self.device = page_size, device
        self.slots, self.positions, self.requests = new(rows, torch.int64), new(rows, torch.int32), new(rows, torch.int32)
        self.starts, self.lengths, self.queue = new(requests + 1, torch.int32), new(requests, torch.int32), new(4, torch.int64)


def page_plan(plan, lengths, added, block_table, free_pages, queue, lengths_out=None, queue_out=None, stream=None):
    """Pages, cache slots and positions of a step's new tokens (hm_page_plan), into `plan`. lengths, added int32 [requests]: cached tokens
    and new ones (0: none, -1: the request has ended and gives its pages back); block_table int32 [requests, pages of a request] and
    the ring of free pages free_pages int32 are updated in place; queue int64 [4] holds the ring's head and tail. The lengths
    and counters after the step go to plan.lengths and plan.queue, or to lengths_out and queue_out, which may be lengths and queue.
    plan.queue[2] counts the requests that got nothing because pages, rows or table entries did not suffice, and those that could not end: free_pages
    should have an entry for every page that is free or held, or pages given back may not fit it, and their request keeps them."""
    status = _host.page_plan(plan.slots, plan.positions, plan.requests, plan.starts, plan.lengths, plan.queue, plan.page_size, lengths, added,
                             block_table, free_pages, queue, lengths_out, queue_out, stream)
    if status != _lib.HM_OK:
        _call(status)
    return plan


def qk_norm_rope(q_out, qkv, frequencies, positions, cache=None, slots=None, k_out=None, kv_heads=None, head_dim=None, q_weight=None, k_weight=None,
                 bias=None, eps=1e-6, interleaved=False, stream=None):
    """Q/K/V rows made ready for attention (hm_qk_norm_rope): bias, RMSNorm of each query and key head (q_weight, k_weight
    [head_dim]; None: no norm), rotation by position * frequencies (fp64 radians per position; fewer than head_dim / 2: only that part of the head),
    fp32 with one rounding. qkv [rows, (q_heads + 2 kv_heads) * head_dim]; queries go to q_out [rows, q_heads (x) head_dim]. With a
    cache, keys and values go to their slots; without one, keys go to k_out and kv_heads and head_dim are given. q_out and
    k_out may be their columns of qkv. Rows with a negative position are left as they are."""
    address, index = (0, 0) if cache is None else (cache._address, cache.device.index)
    status = _host.qk_norm_rope(q_out, qkv, frequencies, positions, address, index, slots, k_out, kv_heads or 0, head_dim or 0, q_weight, k_weight, bias, eps,
                                interleaved, stream)
    if status != _lib.HM_OK:
        _call(status)
    return q_out


def paged_attention(out, q, cache, block_table, positions, requests=None, scale=None, window=0, stream=None, workspace=None):
    """out[t, h] = softmax(scale q[t, h] K^T) V over keys 0..positions[t] (its last `window` ones, if not 0) of row t's request in the
    paged cache (hm_paged_attention). q, out [rows, q_heads, head_dim]; block_table int32 [requests, pages of a request]; row t is of request
    requests[t], or t. Position -1: zeros; a negative request: the row is left as it is; a row outside the table or the
    cache: NaN. Rows of one request share their reads of the cache where there are more rows than the table has: block_table[:n] of the requests
    in use is faster for prompts and drafts than a taller table. scale: 1 / sqrt(head_dim) by default. workspace: cache.attention_workspace(q_heads), one per stream."""
    d = cache.head_dim
    if workspace is None:
        workspace = cache.attention_workspace(q.size(1) if q.dim() == 3 else q.size(-1) // d, stream)
    status = _host.paged_attention(out, q, cache._address, cache.device.index, block_table, positions, requests, 1.0 / math.sqrt(d) if scale is None else scale,
                                   window, workspace, stream)
    if status != _lib.HM_OK:
        _call(status)
    return out


class _Scratch:
    """An attention block's buffers on one stream."""

    def __init__(self, rows, linear, attention):
        self.rows, self.linear, self.attention, self.captured = rows, linear, attention, False


class AttnLayer:
    """A layer's attention block over its paged cache, the counterpart of FfnLayer.block_forward: x += attention(RMSNorm(x)) Wo.
    wqkv [hidden, (q_heads + 2 kv_heads) * head_dim] and wo [q_heads * head_dim, hidden] are RepackedMatrix (RepackedMatrix.concat makes
    wqkv of three); frequencies as rope_frequencies gives them; bias of the Q/K/V columns, q_weight and k_weight of normed heads or None.
    head_dim: 64, 96, 128 or 256."""

    def __init__(self, wqkv, wo, q_heads, kv_heads, head_dim, frequencies, bias=None, q_weight=None, k_weight=None, qk_eps=1e-6, scale=None, window=0,
                 interleaved=False):
        if wqkv.dtype not in _DTYPES or min(q_heads, kv_heads) <= 0 or q_heads > 65536 or q_heads % kv_heads:
            raise ValueError(f"AttnLayer: query heads (up to 65536) must be a multiple of key heads, got {q_heads} and {kv_heads}")
        if head_dim not in (64, 96, 128, 256):
            raise ValueError(f"AttnLayer: paged_attention takes heads of 64, 96, 128 or 256, got {head_dim}")
        if (scale is not None and not math.isfinite(ctypes.c_float(scale).value)) or window < 0:
            raise ValueError(f"AttnLayer: scale must be finite and window not negative, got {scale} and {window}")
        if wo.device != wqkv.device:
            raise ValueError(f"AttnLayer: wqkv and wo must be on one device, got {wqkv.device} and {wo.device}")
        if wqkv.n != (q_heads + 2 * kv_heads) * head_dim or wo.k != q_heads * head_dim or wo.n != wqkv.k or wo.dtype != wqkv.dtype:
            raise ValueError(f"AttnLayer: wqkv [{wqkv.k}, {wqkv.n}] and wo [{wo.k}, {wo.n}] do not fit {q_heads} + 2 x {kv_heads} heads of {head_dim}")
        self.wqkv, self.wo, self.q_heads, self.kv_heads, self.head_dim = wqkv, wo, q_heads, kv_heads, head_dim
        self.hidden, self.dtype, self.device = wqkv.k, wqkv.dtype, wqkv.device
        self.frequencies, self.bias, self.q_weight, self.k_weight, self.qk_eps = frequencies, bias, q_weight, k_weight, qk_eps
        self.scale, self.window, self.interleaved = scale, window, interleaved
        self._buffers = {}
        self._outgrown = []  # those that a captured step still uses

    def _scratch(self, rows, cache, stream):
        """(normed or projected rows, Q/K/V rows, attention rows, workspaces) of calls on this stream, grown as needed."""
        key = _stream(stream, self.device)
        kept = self._buffers.get(key)
        with _on(stream, self.device):
            capturing = torch.cuda.is_current_stream_capturing()
            if kept is None or kept.rows[0].size(0) < rows:
                if kept is not None and kept.captured:
                    self._outgrown.append(kept)
                new = lambda n: torch.empty((rows, n), dtype=self.dtype, device=self.device)
                linear = max(w.workspace_bytes(m) for w in (self.wqkv, self.wo) for m in (rows, min(rows, 16)))
                # attention's workspace does not depend on the rows
                attention = cache.attention_workspace(self.q_heads) if kept is None else kept.attention
                kept = self._buffers[key] = _Scratch((new(self.hidden), new(self.wqkv.n), new(self.wo.k)), _workspace(linear, self.device, None), attention)
        kept.captured |= capturing
        return tuple(t[:rows] for t in kept.rows) + (kept.linear, kept.attention)

    def block_forward(self, x, norm_weight, cache, plan, block_table, eps=1e-5, stream=None):
        """In place: x [rows, hidden] += attention(RMSNorm(x) * norm_weight) Wo. The rows are those of `plan` (page_plan of this step): their keys and values
        are written to `cache` first, and each row sees its request's tokens up to its own. Rows that the plan left empty stay as they are. The buffers in between are
        the stream's, also those of a step that was captured on it: such steps, wherever they are replayed, and other calls on the stream must not run at the same
        time."""
        rows = plan.slots.size(0)
        if x.dim() != 2 or x.size(0) != rows or x.size(1) != self.hidden or x.stride(1) != 1 or x.dtype != self.dtype:
            raise ValueError(f"AttnLayer.block_forward: x must be {self.dtype} [{rows}, {self.hidden}]")
        for t in (x, norm_weight, plan, cache, block_table):
            if t.device != self.device:
                raise ValueError(f"AttnLayer.block_forward: needs everything on {self.device}, got x, norm_weight, plan, cache and block_table on "
                                 f"{x.device}, {norm_weight.device}, {plan.device}, {cache.device}, {block_table.device}")
        if norm_weight.numel() != self.hidden or norm_weight.dtype != x.dtype or not norm_weight.is_contiguous():
            raise ValueError(f"norm_weight must be a contiguous {x.dtype} vector of {self.hidden} elements")
        if (cache.kv_heads, cache.head_dim, cache.page_size) != (self.kv_heads, self.head_dim, plan.page_size):
            raise ValueError("AttnLayer.block_forward: the cache's heads and page size must be the layer's and the plan's")
        if block_table.dtype != torch.int32 or block_table.dim() != 2 or 0 in block_table.shape or (block_table.size(1) > 1 and block_table.stride(1) != 1):
            raise ValueError(f"AttnLayer.block_forward: block_table must be int32 [requests, pages of a request] with contiguous rows, got {block_table.dtype} "
                             f"{list(block_table.shape)}")
        with _guard(self.device):
            normed, qkv, heads, linear_ws, attention_ws = self._scratch(rows, cache, stream)
            rmsnorm(normed, x, norm_weight, eps, stream)
            packed_linear(qkv, normed, self.wqkv, stream=stream, workspace=linear_ws)
            q = qkv[:, :self.q_heads * self.head_dim]
            qk_norm_rope(q, qkv, self.frequencies, plan.positions, cache=cache, slots=plan.slots, q_weight=self.q_weight, k_weight=self.k_weight,
                         bias=self.bias, eps=self.qk_eps, interleaved=self.interleaved, stream=stream)
            with _on(stream, self.device):
                heads.zero_()  # the rows that the plan left empty add nothing
            paged_attention(heads, q, cache, block_table, plan.positions, plan.requests, self.scale, self.window, stream, attention_ws)
            packed_linear(normed, heads, self.wo, stream=stream, workspace=linear_ws)
            residual_add2(x, normed, stream=stream)
        return x


__all__ = ["kPagePlanMaxRequests", "rope_frequencies", "PagedCache", "PagePlan", "page_plan", "qk_norm_rope", "paged_attention", "AttnLayer"]
