"""The operators of a serving step as a program runs them: ragged prompts, then token by token, a linear before and after, eagerly on
a side stream and as a replayed graph; what every operator gave, and the whole cache, against the formulas in 64 bits."""
import math
import os
import subprocess
import sys

import pytest
import torch

from test_sample_gpu import expected

pytestmark = pytest.mark.gpu
HEADS, KV, VOCAB, PAGE = 8, 2, 501, 16
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


class Layer:
    """x + W_o attention(rope(W_q x), rope(W_k x), W_v x), and logits of it."""

    def __init__(self, xn, cuda, dtype, hd, interleaved, streams, pages, window):
        g = torch.Generator(device=cuda).manual_seed(hd + interleaved)
        self.xn, self.hd, self.interleaved, self.window, d = xn, hd, interleaved, window, 256

        def weight(n, k):
            return (torch.randn(n, k, generator=g, device=cuda) / math.sqrt(k)).to(dtype)

        self.embed = weight(VOCAB, d) * math.sqrt(d)
        self.qkv, self.out, self.logits = weight((HEADS + 2 * KV) * hd, d), weight(d, HEADS * hd), weight(VOCAB, d)
        self.freqs = xn.rope_frequencies(hd, device=cuda)
        self.k, self.v = (torch.full((streams * pages + 1, KV, PAGE, hd), math.nan, device=cuda, dtype=dtype) for _ in range(2))
        # page 0 is nobody's, the streams' pages lie in turns and backwards
        self.table = (torch.arange(pages * streams, device=cuda).flip(0).view(pages, streams).t() + 1).to(torch.int32).contiguous()
        self.scale = 1 / math.sqrt(hd)

    def step(self, tokens, positions, slots, context, starts, max_query, last, uniform, filters):
        xn = self.xn
        r = dict(x=self.embed[tokens])
        r["qkv"] = xn.Linear(self.qkv)(r["x"]).view(-1, HEADS + 2 * KV, self.hd)
        q, k, v = r["qkv"].split((HEADS, KV, KV), 1)
        r["q"] = xn.paged_append_(self.k, self.v, k, v, slots, q=q, positions=positions, freqs=self.freqs, interleaved=self.interleaved)
        r["o"] = xn.attention_paged(r["q"], self.k, self.v, self.table, context, self.scale, query_starts=starts, max_query=max_query,
                                    window=self.window)
        r["z"] = xn.Linear(self.out)(r["o"].view(-1, HEADS * self.hd))
        r["y"] = xn.ops.add(r["x"], r["z"])
        r["logits"] = xn.Linear(self.logits)(r["y"] if last is None else r["y"][last])
        r["drawn"] = xn.sample(r["logits"], uniform, **filters)
        return r

    def slots(self, stream, positions):
        return self.table[stream, positions // PAGE].long() * PAGE + positions % PAGE

    def turned(self, x, positions):  # [n, heads, hd] in 64 bits
        a = positions.double()[:, None] * self.freqs
        c, s = a.cos()[:, None], a.sin()[:, None]
        x0, x1 = (x[..., 0::2], x[..., 1::2]) if self.interleaved else x.chunk(2, -1)
        y0, y1 = x0 * c - x1 * s, x0 * s + x1 * c
        return torch.stack((y0, y1), -1).flatten(-2) if self.interleaved else torch.cat((y0, y1), -1)

    def check(self, r, raw, history, starts, positions, last, uniform, filters):
        """r: what a step gave, raw: the projections [tokens, heads, hd] of a stream so far, the step's among them.  Bounds: u, half a
        step of the element type, for a stored value; n 2^-24 of the magnitudes for an f32 sum of n products."""
        u = torch.finfo(self.embed.dtype).eps / 2

        def near(got, want, size, n):
            err, bound = (got.double() - want).abs(), want.abs() * u * (1 + u) + size * (n * 2.0 ** -24 * (1 + u)) + 2.0 ** -25
            assert bool((err <= bound).all()), (err / bound).max().item()

        def linear(got, x, w):
            x, w = x.double(), w.double()
            near(got, x @ w.t(), x.abs() @ w.abs().t(), x.shape[1])

        linear(r["qkv"].flatten(1), r["x"], self.qkv)
        for b, all_raw in enumerate(raw):
            mine, n = slice(starts[b], starts[b + 1]), len(history[b])
            assert torch.equal(r["x"][mine], self.embed[history[b][n - (starts[b + 1] - starts[b]):]])
            pages = self.table[b, :-(-n // PAGE)].long()
            k, v = (pool[pages].transpose(1, 2).reshape(-1, KV, self.hd) for pool in (self.k, self.v))
            assert bool(k[n:].isnan().all()) and bool(v[n:].isnan().all())
            k, v, where = k[:n], v[:n], torch.arange(n, device=k.device)
            raw_k, size = all_raw[:, HEADS:HEADS + KV].double(), all_raw.double().abs().amax(-1, keepdim=True)
            near(k, self.turned(raw_k, where), size[:, HEADS:HEADS + KV], 8)
            assert torch.equal(v, all_raw[:, HEADS + KV:])
            near(r["q"][mine], self.turned(r["qkv"][mine, :HEADS].double(), positions[mine]), size[n - (starts[b + 1] - starts[b]):, :HEADS], 8)
            k, v = (t.double().repeat_interleave(HEADS // KV, 1) for t in (k, v))
            s = torch.einsum("ihd,jhd->hij", r["q"][mine].double(), k) * self.scale
            at, key = positions[mine][:, None], where[None]
            s = s.masked_fill((key > at) | ((key <= at - self.window) if self.window else False), -math.inf)
            p = s.softmax(-1)
            # every weight is rounded once, and so is the result; scores and sums in f32 move a weight by 2^-13 at most (head_dim
            # 2^-24 of the sum of |q k|, below 80, and as much again); f16 weights below 2^-14 are off by half a subnormal step
            o, size = torch.einsum("hij,jhd->ihd", p, v), torch.einsum("hij,jhd->ihd", p, v.abs())
            tol = u * o.abs() + (u + 2.0 ** -13) * size + 2.0 ** -13 * o.abs()
            if r["o"].dtype == torch.float16:
                tol = tol + 2.0 ** -25 * torch.einsum("hij,jhd->ihd", (p > 0).double(), v.abs()) + 2.0 ** -24
            assert bool(((r["o"][mine].double() - o).abs() <= tol).all()), b
        linear(r["z"], r["o"].flatten(1), self.out)
        near(r["y"], r["x"].double() + r["z"].double(), 0, 0)
        linear(r["logits"], r["y"] if last is None else r["y"][last], self.logits)
        for b in range(len(raw)):
            one = dict(t=filters["temperature"][b].double().item(), k=int(filters["top_k"][b]), p=filters["top_p"][b].double().item(),
                       m=filters["min_p"][b].double().item())
            assert int(r["drawn"][b]) == expected(r["logits"][b].float().cpu().numpy(), uniform[b].double().item(), **one), b
            history[b] = torch.cat((history[b], r["drawn"][b:b + 1]))


@pytest.mark.parametrize("dtype,hd,interleaved,window",
                         [("bf16", 64, False, 0), ("f16", 128, True, 0), ("bf16", 128, False, 20), ("f16", 64, True, 0)])
def test_prompts_and_then_token_by_token(xn, cuda, dtype, hd, interleaved, window):
    prompts, steps = [37, 1, 70, 16], 6
    streams, pages = len(prompts), 6
    layer = Layer(xn, cuda, DTYPES[dtype], hd, interleaved, streams, pages, window)
    g = torch.Generator(device=cuda).manual_seed(5)
    history = [torch.randint(VOCAB, (n,), generator=g, device=cuda) for n in prompts]
    filters = dict(temperature=torch.tensor([0.0, 0.8, 1.3, 1.0], device=cuda), top_k=torch.tensor([0, 40, 0, 7], dtype=torch.int32, device=cuda),
                   top_p=torch.tensor([1.0, 1.0, 0.9, 0.8], device=cuda), min_p=torch.tensor([0.0, 0.05, 0.0, 0.0], device=cuda))

    where = [torch.arange(n, device=cuda) for n in prompts]
    starts = torch.tensor([0, 37, 38, 108, 124], dtype=torch.int32, device=cuda)
    context = torch.tensor(prompts, dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    uniform = torch.rand(streams, generator=g, device=cuda)
    last = (starts[1:] - 1).long()
    inputs = torch.cat(history), torch.cat(where), torch.cat([layer.slots(b, p) for b, p in enumerate(where)])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        r = layer.step(*inputs, context, starts, 70, last, uniform, filters)
    torch.cuda.synchronize()
    raw = [r["qkv"][starts[b]:starts[b + 1]] for b in range(streams)]
    layer.check(r, raw, history, starts.tolist(), torch.cat(where), last, uniform, filters)

    # a token per stream: eagerly on the side stream, then captured once and replayed
    rows = torch.arange(streams, device=cuda)
    state = dict(tokens=r["drawn"].clone(), positions=context.long(), context=context + 1, uniform=torch.rand(streams, generator=g, device=cuda))
    state["slots"] = layer.slots(rows, state["positions"])

    def run():
        return layer.step(state["tokens"], state["positions"], state["slots"], state["context"], None, None, None, state["uniform"], filters)

    def check_and_advance(r):
        for b in range(streams):
            raw[b] = torch.cat((raw[b], r["qkv"][b:b + 1]))
        layer.check(r, raw, history, range(streams + 1), state["positions"], None, state["uniform"], filters)
        state["tokens"].copy_(r["drawn"])
        state["positions"].add_(1)
        state["context"].add_(1)
        state["slots"].copy_(layer.slots(rows, state["positions"]))
        state["uniform"].copy_(torch.rand(streams, generator=g, device=cuda))

    for _ in range(2):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            r = run()
        torch.cuda.synchronize()
        check_and_advance(r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = run()
    for _ in range(steps):
        graph.replay()
        again = run()  # the same rows into the same slots
        assert all(torch.equal(again[name], r[name]) for name in r)
        check_and_advance(r)
    used = torch.cat([layer.table[b, :-(-int(state["context"][b] - 1) // PAGE)] for b in range(streams)]).long()
    others = torch.ones(layer.k.shape[0], dtype=torch.bool, device=cuda)
    others[used] = False
    assert bool(layer.k[others].isnan().all()) and bool(layer.v[others].isnan().all())


def test_two_streams_at_once(xn, cuda):
    """Appends and draws of two programs overlap, each on its own stream and tensors, and captured into graphs that are replayed at once."""
    g = torch.Generator(device=cuda).manual_seed(3)
    freqs = xn.rope_frequencies(64, device=cuda)
    programs = []
    for i in range(2):
        p = dict(qkv=torch.randn(300, 6, 64, generator=g, device=cuda).bfloat16(), pools=torch.zeros(2, 24, 1, 16, 64, device=cuda, dtype=torch.bfloat16),
                 slots=torch.randperm(24 * 16, generator=g, device=cuda)[:300], at=torch.arange(300, device=cuda) * (7 + i),
                 logits=torch.randn(20 + 30 * i, 30000, generator=g, device=cuda) * 3, top_p=torch.full((20 + 30 * i,), 0.9, device=cuda))
        p["u"] = torch.rand(len(p["logits"]), generator=g, device=cuda)
        programs.append(p)

    def run(p):
        q = xn.paged_append_(*p["pools"], p["qkv"][:, 4:5], p["qkv"][:, 5:], p["slots"], q=p["qkv"][:, :4], positions=p["at"], freqs=freqs)
        return q, xn.rope(q, p["at"], -freqs), p["pools"].clone(), xn.sample(p["logits"], p["u"], top_p=p["top_p"])

    want = [run(p) for p in programs]
    for p, w in zip(programs, want):
        # turned back: two roundings of at most half a step of the pair's length
        length = p["qkv"][:, :4].double().unflatten(-1, (2, 32)).norm(dim=-2, keepdim=True).expand(-1, -1, 2, -1).flatten(-2)
        assert bool(((w[1].double() - p["qkv"][:, :4].double()).abs() <= length * (2.5 * torch.finfo(torch.bfloat16).eps)).all())
    streams = [torch.cuda.Stream() for _ in programs]
    graphs, replayed = [torch.cuda.CUDAGraph() for _ in programs], []
    torch.cuda.synchronize()
    for p, graph in zip(programs, graphs):
        with torch.cuda.graph(graph):
            replayed.append(run(p))
    for _ in range(5):
        got = []
        for p, s in zip(programs, streams):
            with torch.cuda.stream(s):
                got.append(run(p))
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for w, a, b in zip(want, got, replayed):
            assert all(torch.equal(x, y) for x, y in zip(w, a)) and all(torch.equal(x, y) for x, y in zip(w, b))


FIRST_IN_A_CAPTURE = """
import torch, xn_b200 as xn
d = torch.device("cuda:0")
g = torch.Generator(device=d).manual_seed(0)
rand = lambda *s: torch.randn(*s, generator=g, device=d)
whole = lambda v: torch.tensor(v, dtype=torch.int32, device=d)
qkv, pools, x = rand(64, 12, 64).bfloat16(), torch.zeros(2, 9, 2, 16, 64, device=d, dtype=torch.bfloat16), rand(4, 40000)
at, freqs, table = torch.arange(64, device=d), xn.rope_frequencies(64, device=d), torch.arange(9, dtype=torch.int32, device=d)[None]
u, p, context, starts, one = torch.rand(4, device=d), torch.full((4,), 0.9, device=d), whole([64]), whole([0, 64]), whole([50])
def step():
    q = xn.paged_append_(*pools, qkv[:, 8:10], qkv[:, 10:], at, q=qkv[:, :8], positions=at, freqs=freqs)
    return (q, xn.rope(q, at, freqs), xn.attention_paged(q, *pools, table, context, 0.1, query_starts=starts),
            xn.attention_paged(q[:1], *pools, table, one, 0.1), xn.sample(x, u, top_p=p))
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
"""


def test_the_first_calls_of_a_process_in_a_capture(cuda):
    """Nothing that a call sets up once is refused while a stream is captured."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", FIRST_IN_A_CAPTURE], cwd=root, capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr[-2000:]
