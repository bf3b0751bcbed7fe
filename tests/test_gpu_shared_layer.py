"""GPU: an attention block's steps that share pages, next to longer steps that do not, and what it holds for them."""

import pytest
import torch

from test_gpu_beam_search import D, KV_HEADS, PS, Q_HEADS, Model, State

pytestmark = pytest.mark.gpu

REQUESTS, PROMPT = 6, 5000


@pytest.fixture
def served(oracle, hm, device):
    """A prompt of more rows than a plan of shared pages takes, forked into all requests, whose next step is planned; and a run of the first layer on it."""
    model = Model(oracle, hm, device, "bf16", 11)
    width = PROMPT // PS + 3
    s = State(hm, device, torch.bfloat16, REQUESTS, REQUESTS, width + 30, width)
    s.added[0] = PROMPT
    plan, s.plan = s.plan, hm.PagePlan(REQUESTS, PROMPT, PS, device)
    s.take()
    model.forward(s, torch.arange(PROMPT, device=device) % 1000, None)
    fork = hm.PageFork(REQUESTS, width, PS, device)
    hm.page_fork(fork, torch.zeros(REQUESTS, dtype=torch.int32, device=device), s.lengths, s.table, s.ring, s.queue, lengths_out=s.lengths, queue_out=s.queue)
    hm.copy_pages(s.caches, fork.copies)
    s.plan = plan
    s.added.fill_(1)
    s.take()
    assert int(s.queue[2]) == 0
    return model, s


def _padded(hm, s, rows):
    """The planned step with rows of padding behind it, and its plan of shared pages."""
    device = s.table.device
    plan = hm.PagePlan(REQUESTS, rows, PS, device)
    for name in ("slots", "positions", "requests"):
        getattr(plan, name)[:REQUESTS] = getattr(s.plan, name)
    share = hm.share_plan(hm.SharePlan(rows, PS, Q_HEADS, KV_HEADS, device), s.table, plan.positions, plan.requests)
    return plan, share


def _held(layer, stream=0):
    return layer._buffers[stream]


def test_a_shared_steps_workspace_is_of_its_rows(hm, device, served):
    model, s = served
    layer, cache = model.attn[0], s.caches[0]
    assert _held(layer).rows[0].size(0) == PROMPT and _held(layer).shared is None
    results = []
    for rows, most in ((REQUESTS, REQUESTS), (REQUESTS, REQUESTS), (40, 40), (REQUESTS, 40)):
        before = _held(layer).shared
        plan, share = _padded(hm, s, rows)
        x = torch.zeros((rows, 512), dtype=torch.bfloat16, device=device)
        x[:REQUESTS] = model.embedding[:REQUESTS]
        layer.block_forward(x, model.norm, cache, plan, s.table, share=share)
        torch.cuda.synchronize()
        held = _held(layer)
        assert held.shared.numel() == cache.shared_attention_workspace_bytes(Q_HEADS, most) + 256, rows
        assert before is None or (held.shared is before) == (before.numel() == held.shared.numel())
        assert (x[REQUESTS:] == 0).all()
        results.append(x[:REQUESTS].clone())
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[3])
    # the same step without a plan of shared pages
    x = model.embedding[:REQUESTS].clone()
    layer.block_forward(x, model.norm, cache, s.plan, s.table)
    torch.cuda.synchronize()
    for r in results:
        assert (r - x).float().norm() <= 2 * 12 * 2.0 ** -8 * x.float().norm()  # an attention block's roundings, 12 half steps, of both
    # a longer step keeps it
    before = _held(layer).shared
    plan = hm.PagePlan(REQUESTS, PROMPT + 1000, PS, device)
    layer.block_forward(torch.zeros((PROMPT + 1000, 512), dtype=torch.bfloat16, device=device), model.norm, cache, plan, s.table)
    assert _held(layer).rows[0].size(0) == PROMPT + 1000 and _held(layer).shared is before and not layer._outgrown


def test_a_captured_shared_step_keeps_its_workspace_when_others_outgrow_it(hm, device, served):
    model, s = served
    layer, cache = model.attn[0], s.caches[0]
    stream = torch.cuda.Stream()
    plan, share = _padded(hm, s, REQUESTS)
    x = torch.zeros((REQUESTS, 512), dtype=torch.bfloat16, device=device)
    torch.cuda.synchronize()

    def step():
        x.copy_(model.embedding[:REQUESTS])
        layer.block_forward(x, model.norm, cache, plan, s.table, share=share)

    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    want = x.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        step()
    captured = _held(layer, stream.cuda_stream).shared
    for i, rows in enumerate((20, 70, 200)):
        with torch.cuda.stream(stream):
            other, of_other = _padded(hm, s, rows)
            layer.block_forward(torch.ones((rows, 512), dtype=torch.bfloat16, device=device), model.norm, cache, other, s.table, share=of_other)
            junk = [torch.full((n.numel() // 4,), float("nan"), device=device) for n in (captured,) * 3]
        torch.cuda.synchronize()
        del junk
        x.fill_(0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want), i
        print(float(x.float().sum()), flush=True)  # work of the program's own between replays
    held = _held(layer, stream.cuda_stream)
    assert any(t is captured for t in layer._outgrown) and held.shared is not captured
    assert sum(isinstance(t, torch.Tensor) for t in layer._outgrown) == 1, "the captured step's workspace alone is kept"


def test_workspaces_that_no_call_would_take_are_refused(hm, device, served):
    model, s = served
    cache = s.caches[0]
    for q_heads, rows in ((Q_HEADS, 4097), (Q_HEADS, -1), (Q_HEADS + 1, 4), (0, 4)):
        with pytest.raises(ValueError, match="shared_attention_workspace"):
            cache.shared_attention_workspace(q_heads, rows)
    assert cache.shared_attention_workspace(Q_HEADS, 4096).numel() > cache.shared_attention_workspace(Q_HEADS, 64).numel()
    # without a workspace too: the cache's heads are not the plan's
    three = hm.PagedCache.empty(9, PS, 3, D, torch.bfloat16, device)
    q = torch.zeros((REQUESTS, Q_HEADS, D), dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError):
        hm.shared_attention(torch.zeros_like(q), q, three, s.table, s.plan.positions, hm.SharePlan(REQUESTS, PS, Q_HEADS, KV_HEADS, device), s.plan.requests)


def test_a_workspace_that_could_not_be_had_is_taken_again(hm, device, served):
    model, s = served
    layer, cache = model.attn[0], s.caches[0]
    assert layer._scratch(40, cache, None, True)[-1] is _held(layer).shared

    class Full:
        def shared_attention_workspace(self, q_heads, rows):
            raise torch.OutOfMemoryError

    with pytest.raises(torch.OutOfMemoryError):
        layer._scratch(80, Full(), None, True)
    workspace = layer._scratch(REQUESTS, cache, None, True)[-1]
    assert workspace is _held(layer).shared and workspace.numel() == cache.shared_attention_workspace_bytes(Q_HEADS, REQUESTS) + 256
