"""GPU: the attention block over a paged cache as a serving loop runs it: plan, norm, projection, rotation and cache write, attention,
projection and residual, over steps in which requests start, decode and end."""

import math

import numpy as np
import pytest
import torch

import attention_ref as ref
from gpu_util import TORCH, logical_to_device

pytestmark = pytest.mark.gpu

HIDDEN, Q_HEADS, KV_HEADS, D, PS = 512, 8, 2, 64, 16


class Serving:
    """A layer, its cache and the state of a serving loop, with each request's inputs kept for the float64 form."""

    def __init__(self, oracle, hm, device, dtype, seed, requests, rows, norm, window=0):
        rng = np.random.default_rng(seed)
        self.hm, self.device, self.dtype, self.rng = hm, device, TORCH[dtype], rng
        mats = [oracle.random_weights(rng, k, n, 128, dtype, 0.002, 0.006) for k, n in
                ((HIDDEN, Q_HEADS * D), (HIDDEN, KV_HEADS * D), (HIDDEN, KV_HEADS * D), (Q_HEADS * D, HIDDEN))]
        packed = [hm.RepackedMatrix.from_logical(*logical_to_device(w, dtype, device), 128, dtype=self.dtype) for w in mats]
        self.w64 = [torch.from_numpy(oracle.weights_f64(*w, 128, dtype)) for w in mats]
        gen = torch.Generator().manual_seed(seed)
        randn = lambda *s: torch.randn(s, generator=gen).to(self.dtype)
        self.randn = randn
        self.norm_weight = 1 + 0.1 * randn(HIDDEN)
        self.nw = self.norm_weight.to(device)
        self.bias = 0.5 * randn((Q_HEADS + 2 * KV_HEADS) * D) if norm else None
        self.qk = [1 + 0.2 * randn(D) if norm else None for _ in range(2)]
        self.freq = hm.rope_frequencies(D, 10000.0)
        to = lambda t: None if t is None else t.to(device)
        self.window = window
        self.layer = hm.AttnLayer(hm.RepackedMatrix.concat(packed[:3]), packed[3], Q_HEADS, KV_HEADS, D, to(self.freq), bias=to(self.bias),
                                  q_weight=to(self.qk[0]), k_weight=to(self.qk[1]), window=window)
        pages = 64
        self.cache = hm.PagedCache.empty(pages, PS, KV_HEADS, D, self.dtype, device)
        self.cache.k.fill_(float("nan"))
        self.cache.v.fill_(float("nan"))
        self.table = torch.full((requests, 16), -1, dtype=torch.int32, device=device)
        self.ring = torch.tensor(rng.permutation(pages), dtype=torch.int32, device=device)
        self.queue = torch.tensor([0, pages, 0, 0], dtype=torch.int64, device=device)
        self.lengths, self.added = (torch.zeros(requests, dtype=torch.int32, device=device) for _ in range(2))
        self.plan = hm.PagePlan(requests, rows, PS, device)
        self.x = torch.zeros((rows, HIDDEN), dtype=self.dtype, device=device)
        self.history = [[] for _ in range(requests)]

    def inputs(self, added):
        """The step's rows: random values for new tokens, a marker in the padding."""
        rows = self.x.size(0)
        x = torch.full((rows, HIDDEN), 3.0, dtype=self.dtype)
        at = 0
        for r, a in enumerate(added):
            if a < 0:
                self.history[r] = []
            for _ in range(max(a, 0)):
                x[at] = self.randn(HIDDEN)
                self.history[r].append(x[at].double())
                at += 1
        self.added.copy_(torch.tensor(added, dtype=torch.int32))
        self.x.copy_(x)
        return x, at

    def step(self):
        hm = self.hm
        hm.page_plan(self.plan, self.lengths, self.added, self.table, self.ring, self.queue, self.lengths, self.queue)
        self.layer.block_forward(self.x, self.nw, self.cache, self.plan, self.table)

    def expected(self, added):
        """x + attention block, float64, of the step's rows, from each request's whole history."""
        out = []
        for r, a in enumerate(added):
            if a <= 0:
                continue
            x = torch.stack(self.history[r])
            n = x.size(0)
            h = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5) * self.norm_weight.double()
            qkv = torch.cat([h @ w for w in self.w64[:3]], 1)
            if self.bias is not None:
                qkv = qkv + self.bias.double()
            heads = qkv.view(n, Q_HEADS + 2 * KV_HEADS, D)
            pos = torch.arange(n)
            q, _ = ref.norm_rope(heads[:, :Q_HEADS], pos, self.freq, self.qk[0], 1e-6, D, False)
            k, _ = ref.norm_rope(heads[:, Q_HEADS:Q_HEADS + KV_HEADS], pos, self.freq, self.qk[1], 1e-6, D, False)
            v = heads[:, Q_HEADS + KV_HEADS:]
            group = Q_HEADS // KV_HEADS
            s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(group, 1)) / math.sqrt(D)
            seen = pos[None, :] <= pos[:, None]
            if self.window:
                seen &= pos[None, :] > pos[:, None] - self.window
            p = torch.softmax(torch.where(seen, s, -math.inf), -1)
            o = torch.einsum("hqk,khd->qhd", p, v.repeat_interleave(group, 1)).reshape(n, -1) @ self.w64[3]
            out.append((x + o)[n - a:])
        return torch.cat(out)

    def check(self, added, given, used, tag):
        torch.cuda.synchronize()
        got, want = self.x.cpu().double(), self.expected(added)
        # Roundings on the way, in half steps, each at most that much of the whole in the L2 sense: the norm (through q, k and v: 3), the
        # projection and rotation of q and of k (through the scores, of order 1: 4), v, the attention's output, the O
        # projection and the sum: 11.
        bar = 12 * ref.half_step(self.dtype)
        e = float((got[:used] - want).norm() / want.norm())
        print(f"{tag}: {used} rows, relative L2 {e:.2e} of {bar:.2e}", flush=True)
        assert e <= bar and torch.isfinite(got).all()
        assert torch.equal(self.x.cpu()[used:], given[used:]), "padding rows stay as they are"
        assert int(self.queue[2]) == 0


STEPS = [[5, 0, 30, 0], [1, 17, 1, 0], [1, 1, 1, 9], [-1, 1, 1, 1], [40, 1, -1, 1], [1, 1, 2, 1], [1, 1, 1, 1]]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("norm,window", [(False, 0), (True, 0), (True, 20)])
def test_serving_steps(oracle, hm, device, dtype, norm, window):
    s = Serving(oracle, hm, device, dtype, 21, 4, 48, norm, window)
    for i, added in enumerate(STEPS):
        given, used = s.inputs(added)
        s.step()
        s.check(added, given, used, f"step {i}")


def test_the_block_is_its_operators(oracle, hm, device):
    s = Serving(oracle, hm, device, "bf16", 22, 4, 48, True)
    t = Serving(oracle, hm, device, "bf16", 22, 4, 48, True)
    for added in STEPS[:4]:
        s.inputs(added)
        t.inputs(added)
        s.step()
        t.hm.page_plan(t.plan, t.lengths, t.added, t.table, t.ring, t.queue, t.lengths, t.queue)
        layer, rows = t.layer, t.x.size(0)
        normed = hm.rmsnorm(torch.empty_like(t.x), t.x, t.nw, 1e-5)
        qkv = hm.packed_linear(torch.empty((rows, layer.wqkv.n), dtype=t.dtype, device=device), normed, layer.wqkv)
        q = torch.zeros((rows, Q_HEADS, D), dtype=t.dtype, device=device)
        hm.qk_norm_rope(q, qkv, layer.frequencies, t.plan.positions, cache=t.cache, slots=t.plan.slots, q_weight=layer.q_weight, k_weight=layer.k_weight,
                        bias=layer.bias)
        heads = hm.paged_attention(torch.zeros_like(q), q, t.cache, t.table, t.plan.positions, t.plan.requests)
        o = hm.packed_linear(torch.empty_like(t.x), heads.view(rows, -1), layer.wo)
        hm.residual_add2(t.x, o)
        torch.cuda.synchronize()
        assert torch.equal(s.x, t.x)


def test_a_captured_step_is_replayed_with_other_requests(oracle, hm, device):
    s = Serving(oracle, hm, device, "fp16", 23, 4, 16, True)
    first = [3, 4, 0, 1]
    given, used = s.inputs(first)
    s.step()
    s.check(first, given, used, "eager")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):  # the capture stream's buffers
        s.inputs([0, 0, 0, 0])
        s.step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        s.step()
    for i, added in enumerate([[1, 1, 0, 1], [1, 1, 12, 1], [-1, 1, 1, 1], [10, 1, 1, -1], [1, 1, 1, 5]]):
        given, used = s.inputs(added)
        g.replay()
        s.check(added, given, used, f"replay {i}")


def test_on_a_stream_of_the_calls(oracle, hm, device):
    s = Serving(oracle, hm, device, "fp16", 24, 4, 48, False)
    stream = torch.cuda.Stream()
    for added in STEPS[:3]:
        given, used = s.inputs(added)
        torch.cuda.synchronize()
        s.hm.page_plan(s.plan, s.lengths, s.added, s.table, s.ring, s.queue, s.lengths, s.queue, stream=stream)
        s.layer.block_forward(s.x, s.nw, s.cache, s.plan, s.table, stream=stream)
        stream.synchronize()
        s.check(added, given, used, "on another stream")


def test_refusals(oracle, hm, device):
    s = Serving(oracle, hm, device, "fp16", 25, 4, 16, False)
    with pytest.raises(ValueError, match="AttnLayer"):
        hm.AttnLayer(s.layer.wqkv, s.layer.wo, Q_HEADS, KV_HEADS + 1, D, s.layer.frequencies)
    with pytest.raises(ValueError, match="x must be"):
        s.layer.block_forward(s.x[:5], s.nw, s.cache, s.plan, s.table)
    with pytest.raises(ValueError, match="norm_weight"):
        s.layer.block_forward(s.x, s.nw[:8], s.cache, s.plan, s.table)
    with pytest.raises(ValueError, match="page size"):
        s.layer.block_forward(s.x, s.nw, hm.PagedCache.empty(2, 32, KV_HEADS, D, torch.float16, device), s.plan, s.table)
    k = torch.zeros((2, 2, 16, 64), dtype=torch.float16, device=device)
    for bad in (k[..., ::2], k.to(torch.float32), k[0], k.expand(2, 2, 16, 64)[:, :1].expand(2, 2, 16, 64)):
        with pytest.raises(ValueError):
            c = hm.PagedCache(bad, bad)
            hm.paged_attention(torch.zeros((1, 2, 64), dtype=torch.float16, device=device), torch.zeros((1, 2, 64), dtype=torch.float16, device=device), c,
                               s.table, s.added)
    q = torch.zeros((2, 4, 64), dtype=torch.float16, device=device)
    cache = hm.PagedCache(k, k.clone())
    for kw in (dict(q=q.to(torch.bfloat16)), dict(out=q[:, :2]), dict(positions=s.added.long()), dict(positions=s.added[:1]), dict(block_table=s.table.long()),
               dict(requests=s.added[::2]), dict(q=q.cpu())):
        args = dict(out=q.clone(), q=q, cache=cache, block_table=s.table, positions=s.added, **{})
        args.update(kw)
        with pytest.raises(ValueError):
            hm.paged_attention(**args)


def test_a_wrong_number_of_heads_without_a_workspace(hm, device):
    k = torch.zeros((2, 4, 16, 64), dtype=torch.float16, device=device)
    cache, n = hm.PagedCache(k, k.clone()), torch.zeros(2, dtype=torch.int32, device=device)
    for heads in (0, 3, 6):
        q = torch.zeros((2, heads, 64), dtype=torch.float16, device=device)
        with pytest.raises(ValueError, match="multiple of the 4 key heads"):
            hm.paged_attention(q.clone(), q, cache, n[:, None], n)


def test_tensors_of_other_devices_are_refused(oracle, hm, device):
    s = Serving(oracle, hm, device, "fp16", 26, 4, 16, False)
    cpu_plan = hm.PagePlan(4, 16, PS, "cpu")
    for x, nw, plan, table in ((s.x.cpu(), s.nw, cpu_plan, s.table), (s.x, s.nw, cpu_plan, s.table), (s.x.cpu(), s.nw, s.plan, s.table),
                               (s.x, s.nw.cpu(), s.plan, s.table), (s.x, s.nw, s.plan, s.table.cpu())):
        before = x.clone()
        with pytest.raises(ValueError):
            s.layer.block_forward(x, nw, s.cache, plan, table)
        assert torch.equal(x, before)


@pytest.mark.parametrize("shape", [(2048, 32, 8, 64), (4096, 32, 8, 128), (512, 8, 2, 64)])
def test_a_step_of_fewer_rows_has_its_workspace(oracle, hm, device, shape):
    hidden, q_heads, kv_heads, d = shape
    rng = np.random.default_rng(27)
    new = lambda k, n: hm.RepackedMatrix.from_logical(*logical_to_device(oracle.random_weights(rng, k, n, 128, "fp16", 0.002, 0.006), "fp16", device), 128,
                                                      dtype=torch.float16)
    wqkv, wo = new(hidden, (q_heads + 2 * kv_heads) * d), new(q_heads * d, hidden)
    cache = hm.PagedCache.empty(2, 16, kv_heads, d, torch.float16, device)
    for most in (1, 2, 5, 8, 16, 17, 100):
        layer = hm.AttnLayer(wqkv, wo, q_heads, kv_heads, d, hm.rope_frequencies(d, device=device))
        linear_ws = layer._scratch(most, cache, None)[3]
        for rows in range(1, most + 1):
            need = max(wqkv.workspace_bytes(rows), wo.workspace_bytes(rows))
            assert need == 0 or linear_ws.numel() >= need + 256, (most, rows)


def test_outgrown_buffers_go_back(oracle, hm, device):
    # steps of more and more rows, no graph: what is held is what the largest needs
    s = Serving(oracle, hm, device, "fp16", 28, 4, 16, False)
    new = lambda: hm.AttnLayer(s.layer.wqkv, s.layer.wo, Q_HEADS, KV_HEADS, D, s.layer.frequencies)
    held = []
    for sizes in ([2000], range(1, 2001, 37), [2000]):
        layer, before = new(), torch.cuda.memory_allocated()
        for rows in sizes:
            layer._scratch(rows, s.cache, None)
        held.append(torch.cuda.memory_allocated() - before)
        del layer
    print(f"held: {held[0]} bytes at once, {held[1]} after 55 sizes", flush=True)
    # Each of the five tensors may lie in a block that torch had freed and hands out whole where less than 1 MiB of it would be left.
    assert all(abs(h - held[0]) <= 5 * 2 ** 20 for h in held)


def test_a_captured_step_keeps_its_buffers_when_others_outgrow_them(oracle, hm, device):
    s = Serving(oracle, hm, device, "bf16", 29, 4, 16, True)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        s.inputs([0, 0, 0, 0])
        s.step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        s.step()
    for i, added in enumerate([[3, 4, 0, 1], [1, 1, 12, 1], [-1, 1, 1, 1]]):
        with torch.cuda.stream(stream):  # a larger eager step of the same layer on the same stream, of requests that see nothing
            rows = 40 * (i + 1)
            plan = hm.PagePlan(4, rows, PS, device)
            s.layer.block_forward(torch.full((rows, HIDDEN), 2.0, dtype=s.dtype, device=device), s.nw, s.cache, plan, s.table)
            junk = [torch.full((rows, n), float("nan"), dtype=s.dtype, device=device) for n in (HIDDEN, s.layer.wqkv.n, s.layer.wo.k) * 3]
        torch.cuda.synchronize()
        del junk
        given, used = s.inputs(added)
        g.replay()
        s.check(added, given, used, f"replay {i}")
    assert len(s.layer._outgrown) == 1, "the captured step's buffers alone are kept"


def test_a_refused_table_leaves_the_cache_as_it_was(oracle, hm, device):
    s = Serving(oracle, hm, device, "fp16", 31, 4, 16, False)
    s.inputs([3, 1, 1, 1])
    s.hm.page_plan(s.plan, s.lengths, s.added, s.table, s.ring, s.queue)
    for table in (s.table.long(), s.table[0], s.table[:, ::2], s.table[:0], s.table[:, :0]):
        with pytest.raises(ValueError, match="block_table"):
            s.layer.block_forward(s.x, s.nw, s.cache, s.plan, table)
    torch.cuda.synchronize()
    assert torch.isnan(s.cache.k).all() and torch.isnan(s.cache.v).all()
