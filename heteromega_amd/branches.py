"""Requests that branch over a paged key-value cache: the beams of a search, several samples of one prompt, requests on one system prompt. Over the C ABI
(include/hm_w4a16.h), next to the attention operators (attention.py).

A step of a beam search: beam_select takes the logits of the last step's rows and gives each beam's parent, token and score; page_fork makes each request
what its parent was, sharing full pages, and copy_pages copies the last, partly filled ones in all layers' caches; then page_plan as for any step,
share_plan for the step, and in each layer qk_norm_rope and shared_attention (or AttnLayer.block_forward with the plan), which reads pages that rows share once.
page_compact moves the pages in use to the front of a cache that is to be cut. Nothing waits for the host.
"""

import ctypes
import math

import torch

from . import _lib
from .attention import PagedCache, _guard, _host, kPagePlanMaxRequests
from .ffn import _call, _workspace

kBeamMaxBeams = 256
kBeamMaxK = 64
kBeamMaxRows, kBeamMaxVocabulary = 65535, 1 << 24
kShareMaxRows = 4096


def _bind():
    L = _lib.load()
    address = lambda f: ctypes.cast(f, ctypes.c_void_p).value
    _host.bind_branches(address(L.hm_beam_select), address(L.hm_page_fork), address(L.hm_page_compact), address(L.hm_copy_pages), address(L.hm_share_plan),
                        address(L.hm_shared_attention))


try:
    _bind()
except ImportError:
    pass  # without the compiled module the calls say so


def _device(device):
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        return torch.device("cuda", torch.cuda.current_device())
    return device


def _new_workspace(nbytes, device):
    """An object's own workspace; on the CPU, where no call goes, an empty one."""
    if device.type != "cuda":
        return torch.empty(0, dtype=torch.uint8)
    with _guard(device):
        return _workspace(nbytes, device, None)


def _check_page_size(what, page_size):
    if not 16 <= page_size <= 1 << 30 or page_size & (page_size - 1):
        raise ValueError(f"{what}: page_size must be a power of two from 16 to 2^30, got {page_size}")


class BeamStep:
    """What beam_select works out for `requests` requests of `beams` beams each, kept from step to step: parents (rows of the logits), tokens, scores
    and ended [requests, k], best first. Its workspace is its own: calls with one step object must not run at the same time."""

    def __init__(self, requests, beams, k, vocabulary, device="cuda"):
        self.device = device = _device(device)
        if min(requests, beams, k, vocabulary) < 1 or beams > kBeamMaxBeams or k > kBeamMaxK:
            raise ValueError(f"BeamStep: needs requests, 1 to {kBeamMaxBeams} beams, k of 1 to {kBeamMaxK} and a vocabulary, got {requests}, {beams}, {k}, {vocabulary}")
        if requests * beams > kBeamMaxRows or vocabulary > kBeamMaxVocabulary:
            raise ValueError(f"BeamStep: at most {kBeamMaxRows} rows and {kBeamMaxVocabulary} tokens, got {requests} x {beams} and {vocabulary}")
        self.requests, self.beams, self.k, self.vocabulary = requests, beams, k, vocabulary
        new = lambda v, t: torch.full((requests, k), v, dtype=t, device=device)
        self.parents, self.tokens, self.scores, self.ended = new(-1, torch.int32), new(-1, torch.int32), new(-math.inf, torch.float32), new(True, torch.bool)
        bytes_of = _lib.load().hm_beam_select_workspace_bytes
        self._workspace = _new_workspace(max(bytes_of(requests, beams, vocabulary, k, t) for t in (_lib.HM_FP16, _lib.HM_LOGITS_FP32)), device)


def beam_select(step, logits, scores, ended=None, end_token=-1, stream=None):
    """The k best continuations of each request's beams (hm_beam_select), into `step`: by scores[row] + log_softmax(logits[row]), or for a row that has ended its
    end_token at scores[row]; equal scores by the lower beam and token. logits [requests * beams, vocabulary], fp16, bf16 or fp32; scores fp32 and ended bool
    [requests * beams]. With k = beams, step.scores and step.ended of the last call may be this one's scores and ended (view(-1))."""
    status = _host.beam_select(step.parents, step.tokens, step.scores, step.ended, step._workspace, step.requests, step.beams, step.vocabulary, step.k, logits, scores,
                               ended, end_token, stream)
    if status != _lib.HM_OK:
        _call(status)
    return step


class PageFork:
    """What page_fork works out for a block table [requests, up to width], kept from step to step: copies [requests, 3] (source page, target page, tokens; -1 behind the
    last) for copy_pages, lengths and queue after the call. Its workspace is its own: calls with one object must not run at the same time."""

    def __init__(self, requests, width, page_size, device="cuda"):
        self.device = device = _device(device)
        if not 1 <= requests <= kPagePlanMaxRequests or width < 1:
            raise ValueError(f"PageFork: needs 1 to {kPagePlanMaxRequests} requests and a table of some pages, got {requests}, {width}")
        _check_page_size("PageFork", page_size)
        new = lambda shape, t: torch.full(shape, -1, dtype=t, device=device)
        self.width, self.page_size = width, page_size
        self.copies, self.lengths, self.queue = new((requests, 3), torch.int32), new((requests,), torch.int32), new((4,), torch.int64)
        self._workspace = _new_workspace(_lib.load().hm_page_fork_workspace_bytes(requests, width), device)


def page_fork(fork, sources, lengths, block_table, free_pages, queue, keep=None, table_out=None, lengths_out=None, queue_out=None, stream=None):
    """Requests become copies of others, all at once (hm_page_fork): request r what sources[r] was before the call (r: it stays, negative: it ends), cut to its
    first keep[r] tokens if keep is given. Full pages are shared; a last page that is not full goes to one request, and the others get fresh ones from the
    ring, listed in fork.copies for copy_pages of each layer's cache. block_table (or table_out) and free_pages are updated; lengths and counters after the call go to
    fork.lengths and fork.queue, or to lengths_out and queue_out, which may be lengths and queue. queue[2] is 1 where the call was refused as a whole (a bad
    source, keep or length, or too few pages or places in the ring), and then nothing has changed. Requests that share pages end here, not in page_plan."""
    if block_table.dim() == 2 and block_table.size(1) > fork.width:
        raise ValueError(f"page_fork: the fork is too small, made for {fork.width} blocks of each request, the table has {block_table.size(1)}")
    status = _host.page_fork(fork.copies, fork.lengths, fork.queue, fork._workspace, fork.page_size, sources, lengths, block_table, free_pages, queue, keep, table_out,
                             lengths_out, queue_out, stream)
    if status != _lib.HM_OK:
        _call(status)
    return fork


class PageCompact:
    """What page_compact works out for a cache of `pages` pages: copies [pages // 2, 3] for copy_pages, and the queue after the call. Its workspace is its own: calls with
    one object must not run at the same time."""

    def __init__(self, pages, page_size, device="cuda"):
        self.device = device = _device(device)
        if pages < 1:
            raise ValueError(f"PageCompact: needs a cache of some pages, got {pages}")
        _check_page_size("PageCompact", page_size)
        self.pages, self.page_size = pages, page_size
        self.copies = torch.full((max(1, pages // 2), 3), -1, dtype=torch.int32, device=device)
        self.queue = torch.full((4,), -1, dtype=torch.int64, device=device)
        self._workspace = _new_workspace(_lib.load().hm_page_compact_workspace_bytes(pages), device)


def page_compact(compact, limit, lengths, block_table, free_pages, queue, table_out=None, queue_out=None, stream=None):
    """The pages that requests hold move to ids below `limit` (hm_page_compact), and the ring holds the ids below it that are left: block_table (or table_out) and free_pages
    are updated, compact.copies lists the moves for copy_pages, counters go to compact.queue or queue_out (which may be queue). queue[2] is 1 where the call was
    refused as a whole (more than `limit` pages are held, or the ring is too small), queue[3] the moves."""
    status = _host.page_compact(compact.copies, compact.queue, compact._workspace, compact.pages, compact.page_size, limit, lengths, block_table, free_pages, queue,
                                table_out, queue_out, stream)
    if status != _lib.HM_OK:
        _call(status)
    return compact


def copy_pages(caches, copies, to=None, stream=None):
    """The first `tokens` tokens of page `source` to page `target`, keys and values of all heads, for each (source, target, tokens) of copies int32 [n, 3] whose pages
    lie in the caches, in each of `caches` (a PagedCache or a list, one per layer, alike in shape and strides), or from each to that of `to`
    (hm_copy_pages)."""
    caches = [caches] if isinstance(caches, PagedCache) else list(caches)
    to = [] if to is None else [to] if isinstance(to, PagedCache) else list(to)
    if not caches or (to and len(to) != len(caches)):
        raise ValueError(f"copy_pages: needs caches, and as many to copy to, got {len(caches)} and {len(to)}")
    device = caches[0].device
    if any(c.device != device for c in caches) or any(c.device != device for c in to):
        raise ValueError(f"copy_pages: the caches must be on one device, the first is on {device}")
    status = _host.copy_pages([c._address for c in caches], [c._address for c in to], device.index, copies, stream)
    if status != _lib.HM_OK:
        _call(status)


class SharePlan:
    """What share_plan finds for a step of `rows` rows, kept from step to step (a captured step's layers read it): shared [rows], the leading tokens
    that a row reads from the same pages as the row before it, and what shared_attention of these heads, page size and window works on."""

    def __init__(self, rows, page_size, q_heads, kv_heads, device="cuda", window=0):
        self.device = device = _device(device)
        if not 1 <= rows <= kShareMaxRows or kv_heads < 1 or q_heads < 1 or q_heads % kv_heads or q_heads // kv_heads > 128 or window < 0:
            raise ValueError(f"SharePlan: needs 1 to {kShareMaxRows} rows, query heads that are a multiple (up to 128) of the key heads and a window that is not negative, got "
                             f"{rows}, {q_heads}, {kv_heads}, {window}")
        _check_page_size("SharePlan", page_size)
        self.rows, self.page_size, self.q_heads, self.kv_heads, self.window = rows, page_size, q_heads, kv_heads, window
        self.shared = torch.zeros(rows, dtype=torch.int32, device=device)
        self._plan = _new_workspace(_lib.load().hm_share_plan_bytes(rows), device)
        self._plan.zero_()  # no plan yet


def share_plan(share, block_table, positions, requests=None, stream=None):
    """What neighbouring rows share of their pages (hm_share_plan), once per step for shared_attention of all layers, into `share`. block_table, positions and
    requests as for paged_attention; rows that share pages should follow each other."""
    status = _host.share_plan(share.shared, share._plan, share.page_size, share.q_heads, share.kv_heads, share.window, block_table, positions, requests, stream)
    if status != _lib.HM_OK:
        _call(status)
    return share


def shared_attention(out, q, cache, block_table, positions, share, requests=None, scale=None, stream=None, workspace=None):
    """paged_attention with the window of `share`, reading pages that rows share once for all of them (hm_shared_attention). share: of share_plan with the same
    block_table, positions and requests. workspace: cache.shared_attention_workspace(q_heads, rows), one per stream."""
    if workspace is None:
        workspace = cache.shared_attention_workspace(share.q_heads, share.rows, stream)
    status = _host.shared_attention(out, q, cache._address, cache.device.index, block_table, positions, requests,
                                    1.0 / math.sqrt(cache.head_dim) if scale is None else scale, share.rows, share.q_heads, share.kv_heads, share.page_size,
                                    share._plan, workspace, stream)
    if status != _lib.HM_OK:
        _call(status)
    return out


__all__ = ["kBeamMaxBeams", "kBeamMaxK", "kBeamMaxRows", "kBeamMaxVocabulary", "kShareMaxRows", "BeamStep", "beam_select", "PageFork", "page_fork", "PageCompact", "page_compact", "copy_pages", "SharePlan",
           "share_plan", "shared_attention"]
