"""GPU: beam searches of several prompts over one paged cache, as a serving loop runs them: selection, forked pages, page plan, what rows share, and layers whose
attention reads shared pages once. Each hypothesis is run again as a request of its own, without shared pages."""

import math

import numpy as np
import pytest
import torch

import attention_ref as ref
from gpu_util import TORCH, logical_to_device

pytestmark = pytest.mark.gpu

HIDDEN, INTER, Q_HEADS, KV_HEADS, D, PS, V, LAYERS = 512, 1024, 8, 2, 64, 16, 1024, 2


class Model:
    def __init__(self, oracle, hm, device, dtype, seed):
        rng = np.random.default_rng(seed)
        self.hm, self.device, self.dtype = hm, device, TORCH[dtype]
        make = lambda k, n, lo=0.002, hi=0.006: logical_to_device(oracle.random_weights(rng, k, n, 128, dtype, lo, hi), dtype, device)
        packed = lambda k, n, *s: hm.RepackedMatrix.from_logical(*make(k, n, *s), 128, dtype=self.dtype)
        freq = hm.rope_frequencies(D, 10000.0, device=device)
        self.attn = [hm.AttnLayer(packed(HIDDEN, (Q_HEADS + 2 * KV_HEADS) * D), packed(Q_HEADS * D, HIDDEN), Q_HEADS, KV_HEADS, D, freq) for _ in range(LAYERS)]
        self.ffn = [hm.FfnLayer.from_logical(make(HIDDEN, INTER), make(HIDDEN, INTER), make(INTER, HIDDEN), 128, dtype=self.dtype) for _ in range(LAYERS)]
        self.head = packed(HIDDEN, V, 0.004, 0.012)
        gen = torch.Generator(device=device).manual_seed(seed)
        self.embedding = torch.randn((V, HIDDEN), generator=gen, device=device).to(self.dtype)
        self.norm = torch.ones(HIDDEN, dtype=self.dtype, device=device)

    def forward(self, state, tokens, share):
        """Logits of a step's rows (those of padding rows mean nothing)."""
        hm = self.hm
        x = self.embedding[tokens.long().clamp(min=0)]
        for attn, ffn, cache in zip(self.attn, self.ffn, state.caches):
            attn.block_forward(x, self.norm, cache, state.plan, state.table, share=share)
            ffn.block_forward(x, self.norm)
        h = hm.rmsnorm(torch.empty_like(x), x, self.norm, 1e-5)
        return hm.packed_linear(torch.empty((x.size(0), V), dtype=self.dtype, device=self.device), h, self.head)


class State:
    """Requests, their pages and the layers' caches."""

    def __init__(self, hm, device, dtype, requests, rows, pages, width, seed=0):
        self.lengths, self.added = (torch.zeros(requests, dtype=torch.int32, device=device) for _ in range(2))
        self.table = torch.full((requests, width), -1, dtype=torch.int32, device=device)
        self.ring = torch.tensor(np.random.default_rng(seed).permutation(pages), dtype=torch.int32, device=device)
        self.queue = torch.tensor([0, pages, 0, 0], dtype=torch.int64, device=device)
        self.caches = [hm.PagedCache.empty(pages, PS, KV_HEADS, D, dtype, device) for _ in range(LAYERS)]
        for c in self.caches:
            c.k.fill_(float("nan"))
            c.v.fill_(float("nan"))
        self.plan = hm.PagePlan(requests, rows, PS, device)
        self.hm, self.pages = hm, pages

    def take(self):
        self.hm.page_plan(self.plan, self.lengths, self.added, self.table, self.ring, self.queue, self.lengths, self.queue)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("captured", [False, True])
def test_beam_searches(oracle, hm, device, dtype, captured):
    model = Model(oracle, hm, device, dtype, 31)
    groups, beams, steps, end = 3, 4, 40, 9
    prompts = [np.random.default_rng(40 + g).integers(0, V, n).tolist() for g, n in enumerate((150, 17, 64))]
    count = groups * beams
    s = State(hm, device, TORCH[dtype], count, count, 150, 16)
    # the prompts, one request of each group in a step of their own
    most = max(map(len, prompts))
    first = hm.PagePlan(count, sum(map(len, prompts)), PS, device)
    s.added.copy_(torch.tensor([len(prompts[r // beams]) if r % beams == 0 else 0 for r in range(count)], dtype=torch.int32))
    plan, s.plan = s.plan, first
    s.take()
    out = model.forward(s, torch.tensor(sum(prompts, []), device=device), None)
    s.plan = plan
    last = np.cumsum([len(p) for p in prompts]) - 1
    logits = torch.zeros((count, V), dtype=TORCH[dtype], device=device)
    logits[::beams] = out[torch.from_numpy(last).to(device)]

    step = hm.BeamStep(groups, beams, beams, V, device)
    step.scores.fill_(-math.inf)
    step.scores[:, 0] = 0
    step.ended.fill_(False)
    fork, share = hm.PageFork(count, 16, PS, device), hm.SharePlan(count, PS, Q_HEADS, KV_HEADS, device)
    s.added.fill_(1)

    def go():
        hm.beam_select(step, logits, step.scores.view(-1), ended=step.ended.view(-1), end_token=end)
        hm.page_fork(fork, step.parents.view(-1), s.lengths, s.table, s.ring, s.queue, lengths_out=s.lengths, queue_out=s.queue)
        hm.copy_pages(s.caches, fork.copies)
        s.take()
        hm.share_plan(share, s.table, s.plan.positions, s.plan.requests)
        logits.copy_(model.forward(s, step.tokens.view(-1), share))

    paths = [[] for _ in range(count)]  # (token, the logits it was chosen from)
    shared = graph = 0
    for i in range(steps):
        before = logits.clone()
        if captured and i == 2:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                go()
        if graph and i % 7 != 6:
            graph.replay()
        else:
            go()
        torch.cuda.synchronize()
        parents, tokens = step.parents.view(-1).tolist(), step.tokens.view(-1).tolist()
        assert int(s.queue[2]) == 0 and min(parents) >= 0
        paths = [paths[p] + [(t, before[p])] for p, t in zip(parents, tokens)]
        shared += int((share.shared > 0).sum())
        held = {int(p) for r in range(count) for p in s.table[r, :ref.pages_of(int(s.lengths[r]), PS)].tolist()}
        assert len(held) + int(s.queue[1] - s.queue[0]) == s.pages, "every page is held or free"
    assert shared > steps * groups * (beams - 1) * 0.9, "beams share their prompt's pages"

    # each hypothesis as one request of its own, its prompt and tokens in one step
    assert most + steps < 16 * PS
    n = [len(prompts[r // beams]) + steps for r in range(count)]
    alone = State(hm, device, TORCH[dtype], count, sum(n), count * 16, 16, 1)
    alone.added.copy_(torch.tensor(n, dtype=torch.int32))
    alone.take()
    tokens = sum((prompts[r // beams] + [t for t, _ in paths[r]] for r in range(count)), [])
    again = model.forward(alone, torch.tensor(tokens, device=device), None)
    at, worst = 0, 0.0
    scores = step.scores.view(-1).cpu()
    for r in range(count):
        # Roundings, in half steps: 12 for an attention block (test_gpu_attn_layer.py); norm, gate and up, product, down, sum 6 for the other; the last norm and
        # the head 2. Each at most that much of the whole in the L2 sense, in both runs.
        bar = 2 * (LAYERS * (12 + 6) + 2) * ref.half_step(TORCH[dtype])
        chosen = torch.stack([x for _, x in paths[r]]).double()
        begin = at + len(prompts[r // beams]) - 1
        other = again[begin:begin + steps].double()
        e = float((chosen - other).norm() / other.norm())
        worst = max(worst, e / bar)
        assert e <= bar, (r, e, bar)
        # the score is the sum of what was chosen from: fp32 sums of `steps` numbers, logs of sums off by 1e-5, until the path ends
        total = 0.0
        for token, x in paths[r]:
            total += float(torch.log_softmax(x.double(), 0)[token])
            if token == end:
                break
        assert abs(total - float(scores[r])) <= steps * (1e-5 + 2.0 ** -24 * abs(total)), (r, total, float(scores[r]))
        at += n[r]
    print(f"{dtype} captured {captured}: worst {worst:.3f} of the bar", flush=True)


def test_a_layer_with_a_share_plan_is_its_operators(oracle, hm, device):
    model = Model(oracle, hm, device, "bf16", 5)
    s = State(hm, device, torch.bfloat16, 6, 6, 60, 10)
    s.added.copy_(torch.tensor([0, 0, 0, 0, 0, 0], dtype=torch.int32))
    long = hm.PagePlan(6, 100, PS, device)
    s.added[0] = 100
    plan, s.plan = s.plan, long
    s.take()
    model.forward(s, torch.arange(100, device=device), None)
    fork = hm.PageFork(6, 10, PS, device)
    hm.page_fork(fork, torch.zeros(6, dtype=torch.int32, device=device), s.lengths, s.table, s.ring, s.queue, lengths_out=s.lengths, queue_out=s.queue)
    hm.copy_pages(s.caches, fork.copies)
    s.plan = plan
    s.added.fill_(1)
    s.take()
    share = hm.share_plan(hm.SharePlan(6, PS, Q_HEADS, KV_HEADS, device), s.table, s.plan.positions, s.plan.requests)
    assert share.shared.tolist() == [0] + [96] * 5
    layer, cache = model.attn[0], s.caches[0]
    x = model.embedding[:6].clone()
    y = x.clone()
    layer.block_forward(x, model.norm, cache, s.plan, s.table, share=share)
    normed = hm.rmsnorm(torch.empty_like(y), y, model.norm, 1e-5)
    qkv = hm.packed_linear(torch.empty((6, layer.wqkv.n), dtype=y.dtype, device=device), normed, layer.wqkv)
    q = torch.zeros((6, Q_HEADS, D), dtype=y.dtype, device=device)
    hm.qk_norm_rope(q, qkv, layer.frequencies, s.plan.positions, cache=cache, slots=s.plan.slots)
    heads = hm.shared_attention(torch.zeros_like(q), q, cache, s.table, s.plan.positions, share, s.plan.requests)
    hm.residual_add2(y, hm.packed_linear(torch.empty_like(y), heads.view(6, -1), layer.wo))
    torch.cuda.synchronize()
    assert torch.equal(x, y)
    for bad in (hm.SharePlan(5, PS, Q_HEADS, KV_HEADS, device), hm.SharePlan(6, PS, Q_HEADS, KV_HEADS, device, window=5), hm.SharePlan(6, 32, Q_HEADS, KV_HEADS, device)):
        with pytest.raises(ValueError, match="share must"):
            layer.block_forward(x, model.norm, cache, s.plan, s.table, share=bad)
