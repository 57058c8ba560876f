"""Attention over a paged cache against softmax in 64 bits, sequence by sequence, at the lengths, pages, heads and masks where it
can go wrong."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


class Batch:
    """Sequences of (new tokens, context) on pages handed out in no order; what pages hold beyond a context is NaN, and so are
    the pages that nobody uses."""

    def __init__(self, cuda, dtype, lengths, heads, kv, hd, page, seed=0, extra_rows=0, spread=1.0):
        g = torch.Generator(device=cuda).manual_seed(seed)
        self.lengths, self.page, self.group = lengths, page, heads // kv
        per = [-(-ctx // page) for _, ctx in lengths]
        n = sum(per) + 2
        ids = torch.randperm(n, generator=g, device=cuda)
        self.table = torch.full((len(lengths), max(per + [1])), -7, dtype=torch.int32, device=cuda)
        self.k, self.v = (torch.full((n, kv, page, hd), math.nan, device=cuda, dtype=dtype) for _ in range(2))
        at = 0
        for b, (_, ctx) in enumerate(lengths):
            mine = ids[at:at + per[b]]
            at += per[b]
            self.table[b, :per[b]] = mine
            for pool in (self.k, self.v):
                rows = torch.full((per[b] * page, kv, hd), math.nan, device=cuda, dtype=dtype)
                rows[:ctx] = (torch.randn(ctx, kv, hd, generator=g, device=cuda) * spread).to(dtype)
                pool[mine] = rows.view(per[b], page, kv, hd).transpose(1, 2)
        starts = [0]
        for q, _ in lengths:
            starts.append(starts[-1] + q)
        self.rows = starts[-1]
        self.q = (torch.randn(self.rows + extra_rows, heads, hd, generator=g, device=cuda) * spread).to(dtype)
        self.starts = torch.tensor(starts, dtype=torch.int32, device=cuda)
        self.context = torch.tensor([c for _, c in lengths], dtype=torch.int32, device=cuda)
        self.scale = 1.0 / math.sqrt(hd)

    def run(self, xn, **kw):
        a = dict(query_starts=self.starts)
        a.update(kw)
        return xn.attention_paged(self.q, self.k, self.v, self.table, self.context, self.scale, **a)

    def check(self, got, window=0):
        half = torch.finfo(got.dtype).eps / 2
        for b, (n, ctx) in enumerate(self.lengths):
            if n == 0:
                continue
            mine = got[int(self.starts[b]):int(self.starts[b]) + n].double()
            pages = self.table[b, :-(-ctx // self.page)].long()
            last = torch.arange(ctx - n, ctx, device=got.device)[:, None]
            key = torch.arange(ctx, device=got.device)
            seen = key <= last
            if window:
                seen &= key > last - window
            some = seen.any(1)
            assert bool((mine[~some] == 0).all())
            if not bool(some.any()):
                continue
            for h in range(self.q.shape[1]):
                k, v = (p[pages, h // self.group].flatten(0, 1)[:ctx].double() for p in (self.k, self.v))
                s = self.q[int(self.starts[b]):int(self.starts[b]) + n, h].double() @ k.T * self.scale
                p = torch.softmax(s.masked_fill(~seen, -math.inf)[some], 1)
                want, size = p @ v, p @ v.abs()
                # The output and every probability are rounded once (half a step each); scores and sums in f32 move a probability by
                # 2^-13 at most: head_dim * 2^-24 of the sum of |q k| (below 80), and as much again in the exponential and the sums.
                # f16 probabilities below 2^-14 are off by half a subnormal step, 2^-25, instead, beside a sum of at least 1.
                tol = half * want.abs() + (half + 2.0 ** -13) * size + 2.0 ** -13 * want.abs()
                if got.dtype == torch.float16:
                    tol = tol + 2.0 ** -25 * (seen[some].double() @ v.abs()) + 2.0 ** -24
                off = (mine[some, h] - want).abs()
                assert bool((off <= tol).all()), (b, h, float((off - tol).max()))


def one(*contexts):
    return [(1, c) for c in contexts]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (8, 1), (6, 2), (10, 2), (32, 2), (40, 2)])
@pytest.mark.parametrize("page", [16, 64])
def test_one_token_per_sequence(xn, cuda, dtype, hd, heads, kv, page):
    b = Batch(cuda, DTYPES[dtype], one(1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000, 0, 333), heads, kv, hd, page)
    b.check(b.run(xn))
    b.check(b.run(xn, query_starts=None))
    b.check(b.run(xn, window=40, max_query=1), window=40)


@pytest.mark.parametrize("page", [1, 3, 5, 8, 24, 48, 100, 128, 256, 1000])
@pytest.mark.parametrize("hd", [64, 128])
def test_pages_of_any_size(xn, cuda, page, hd):
    b = Batch(cuda, torch.bfloat16, [(1, 700), (5, 131), (40, 300), (200, 517), (1, 1)], 8, 2, hd, page)
    b.check(b.run(xn))
    b.check(b.run(xn, window=100), window=100)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 2), (6, 2), (5, 1), (7, 1), (64, 1), (200, 1)])
def test_chunks(xn, cuda, dtype, hd, heads, kv):
    lengths = [(3, 3), (1, 64), (17, 200), (128, 128), (129, 700), (0, 50), (64, 64), (33, 1111), (2, 0), (5, 3), (260, 261)]
    b = Batch(cuda, DTYPES[dtype], lengths, heads, kv, hd, 16)
    b.check(b.run(xn, max_query=260))
    b.check(b.run(xn, window=50), window=50)
    b.check(b.run(xn, window=1), window=1)


@pytest.mark.parametrize("window", [0, 300])
def test_a_long_chunk_on_a_long_context(xn, cuda, window):
    b = Batch(cuda, torch.bfloat16, [(700, 5000), (1, 3000), (1000, 1000)], 8, 2, 128, 64)
    b.check(b.run(xn, max_query=1000, window=window), window=window)


@pytest.mark.parametrize("hd,page,heads,kv", [(128, 64, 4, 1), (64, 16, 2, 2), (128, 7, 16, 1)])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_a_context_shared_by_the_whole_machine(xn, cuda, hd, page, heads, kv, n):
    b = Batch(cuda, torch.bfloat16, [(n, 70001), (n, 19)], heads, kv, hd, page)
    b.check(b.run(xn, max_query=n))


def test_many_short_sequences(xn, cuda):
    lengths = one(*[(7 * i) % 41 for i in range(700)])
    b = Batch(cuda, torch.float16, lengths, 4, 2, 64, 16)
    b.check(b.run(xn, query_starts=None))
    lengths = [((5 * i) % 4, (5 * i) % 4 + (7 * i) % 90) for i in range(900)]
    b = Batch(cuda, torch.bfloat16, lengths, 2, 1, 128, 16)
    b.check(b.run(xn, max_query=3))


@pytest.mark.parametrize("n", [1, 30])
def test_scores_that_move_the_maximum(xn, cuda, n):
    """Scores of hundreds, rising along the context: the running maximum moves again and again, and one key takes everything."""
    b = Batch(cuda, torch.bfloat16, [(n, 900), (n, 2000)], 4, 2, 128, 16, spread=1.0)
    ramp = torch.linspace(0.1, 6.0, b.k.shape[0] * 16, device=cuda).view(-1, 1, 16, 1)
    b.k.copy_((b.k.float() * ramp).bfloat16())
    got = b.run(xn, max_query=n)
    assert not bool(got.isnan().any())
    want = []
    for i, (m, ctx) in enumerate(b.lengths):
        pages = b.table[i, :-(-ctx // 16)].long()
        hidden = torch.arange(ctx, device=cuda) > torch.arange(ctx - m, ctx, device=cuda)[:, None]
        for h in range(4):
            k, v = (p[pages, h // 2].flatten(0, 1)[:ctx].double() for p in (b.k, b.v))
            s = b.q[i * n:i * n + m, h].double() @ k.T * b.scale
            want.append(torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v)
    want = torch.stack(want).view(2, 4, n, 128).transpose(1, 2).reshape(2 * n, 4, 128)
    # scores up to about 60 x 6 wide in f32: 128 * 2^-24 of sums of |q k| up to 500 moves a probability by 2^-8
    assert float((got.double() - want).abs().max()) <= (2.0 ** -8 + 2.0 ** -8 + 2.0 ** -7) * float(b.v[~b.v.isnan()].abs().max())


def test_views_of_larger_tensors(xn, cuda):
    """Queries as a slice of the fused projection's rows, both pools in one tensor, tables and outputs wider than the call."""
    g = torch.Generator(device=cuda).manual_seed(2)
    b = Batch(cuda, torch.bfloat16, [(4, 90), (1, 33), (30, 30)], 8, 2, 64, 16)
    want = b.run(xn)
    b.check(want)
    pools = torch.stack([b.k, b.v], 1)
    fused = torch.randn(b.rows, 12, 64, generator=g, device=cuda).bfloat16()
    fused[:, 2:10] = b.q
    wide = torch.zeros(3, 20, dtype=torch.int32, device=cuda)
    wide[:, 3:3 + b.table.shape[1]] = b.table
    out = torch.full((b.rows, 9, 64), 3.0, dtype=torch.bfloat16, device=cuda)
    got = xn.attention_paged(fused[:, 2:10], pools[:, 0], pools[:, 1], wide[:, 3:3 + b.table.shape[1]], b.context, b.scale,
                             query_starts=b.starts, out=out[:, 1:])
    assert got.data_ptr() == out[:, 1:].data_ptr() and torch.equal(got, want) and bool((out[:, 0] == 3).all())
    odd = torch.randn(b.rows, 8 * 64 + 3, generator=g, device=cuda).bfloat16()  # rows that start anywhere
    odd[:, 1:513] = b.q.flatten(1)
    assert torch.equal(xn.attention_paged(odd[:, 1:513].unflatten(1, (8, 64)), b.k, b.v, b.table, b.context, b.scale, query_starts=b.starts), want)
    nhd = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in (b.k, b.v)]  # (pages, page_size, kv_heads, head_dim) storage
    assert torch.equal(xn.attention_paged(b.q, nhd[0], nhd[1], b.table, b.context, b.scale, query_starts=b.starts), want)
    with pytest.raises(xn.XnError):
        xn.attention_paged(b.q, b.k, b.v, b.table, b.context, b.scale, query_starts=b.starts, out=odd[:, 1:513].unflatten(1, (8, 64)))


@pytest.mark.parametrize("n", [1, 50])
def test_rows_behind_the_last_sequence_stay(xn, cuda, n):
    b = Batch(cuda, torch.bfloat16, [(n, 77), (n, 200)], 4, 2, 128, 16, extra_rows=5)
    out = torch.full_like(b.q, 9.0)
    b.run(xn, out=out)
    b.check(out)
    assert bool((out[b.rows:] == 9).all())


@pytest.mark.parametrize("n", [1, 40])
def test_lengths_and_indexes_that_lead_nowhere(xn, cuda, n):
    """What the device's integers say is bounded by the tensors: contexts longer than the table, rows beyond the queries, pages
    outside the pool (zeros)."""
    b = Batch(cuda, torch.float16, [(n, 100), (n, 64)], 4, 2, 64, 16)
    b.check(b.run(xn, max_query=n))
    dense = [torch.nan_to_num(p) for p in (b.k, b.v)]
    zero = [torch.cat([p, torch.zeros_like(p[:1])]) for p in dense]
    t, z = b.table.clone(), b.table.clone()
    t[0, 1], t[0, 3], t[1, 0] = -1, 2 ** 30, len(dense[0])
    z[0, 1] = z[0, 3] = z[1, 0] = len(dense[0])
    got = xn.attention_paged(b.q, *dense, t, b.context, b.scale, query_starts=b.starts)
    assert torch.equal(got, xn.attention_paged(b.q, *zero, z, b.context, b.scale, query_starts=b.starts))
    # the whole table at most, and nothing below zero
    full = torch.tensor([7 * 16, 7 * 16], dtype=torch.int32, device=cuda)
    long = torch.tensor([2 ** 31 - 1, 7 * 16 + 1], dtype=torch.int32, device=cuda)
    assert b.table.shape[1] == 7
    z = z.clamp(min=0)
    assert torch.equal(xn.attention_paged(b.q, *zero, z, long, b.scale, query_starts=b.starts),
                       xn.attention_paged(b.q, *zero, z, full, b.scale, query_starts=b.starts))
    low = torch.tensor([-5, -2 ** 31], dtype=torch.int32, device=cuda)
    assert bool((xn.attention_paged(b.q, *zero, z, low, b.scale, query_starts=b.starts) == 0).all())
    # rows: starts that fall, or lie outside
    for starts in ([0, 2 * n + 100, 5], [-3, n, 2 ** 31 - 1], [2 * n + 9, 2 * n + 10, 3], [n, 0, n]):
        out = torch.zeros_like(b.q)
        xn.attention_paged(b.q, *dense, b.table, b.context, b.scale, query_starts=torch.tensor(starts, dtype=torch.int32, device=cuda), out=out)
        assert bool(out.isfinite().all())


def test_empty_calls(xn, cuda):
    k = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16, device=cuda)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda)  # noqa: E731
    q = torch.ones(4, 4, 64, dtype=torch.bfloat16, device=cuda)
    assert xn.attention_paged(q[:0], k, k, i(0, 5), i(0), 0.1).shape == (0, 4, 64)
    assert xn.attention_paged(q[:, :0], k, k, i(4, 5), i(4), 0.1).shape == (4, 0, 64)
    assert bool((xn.attention_paged(q, k[:0], k[:0], i(4, 5), i(4), 0.1) == 0).all())
    assert bool((xn.attention_paged(q, k, k, i(4, 0), i(4) + 9, 0.1) == 0).all())
    assert bool((xn.attention_paged(q, k[:0], k[:0], i(4, 5), i(4) + 9, 0.1) == 0).all())
    out = torch.full_like(q, 2.0)
    xn.attention_paged(q, k, k, i(0, 5), i(0), 0.1, query_starts=i(1), out=out)
    assert bool((out == 2).all())


@pytest.mark.parametrize("n", [1, 40])
def test_pools_beyond_32_bit_offsets(xn, cuda, n):
    """The pages of the sequence lie behind the first 2^31 elements of the pool."""
    heads, kv, hd, page = 4, 2, 128, 64
    pages = 2 ** 31 // (kv * page * hd) + 40
    pool = torch.empty(pages, kv, page, hd, dtype=torch.bfloat16, device=cuda)
    b = Batch(cuda, torch.bfloat16, [(n, 2000)], heads, kv, hd, page)
    want = torch.nan_to_num(b.k)
    pool[-40:] = 0
    pool[-b.k.shape[0]:] = want
    t = b.table + (pages - b.k.shape[0])
    got = xn.attention_paged(b.q, pool, pool, t, b.context, b.scale, query_starts=b.starts)
    assert torch.equal(got, xn.attention_paged(b.q, want, want, b.table, b.context, b.scale, query_starts=b.starts))


@pytest.mark.parametrize("n", [1, 60])
def test_two_streams_at_once_and_a_replayed_graph(xn, cuda, n):
    bs = [Batch(cuda, torch.bfloat16, [(n, 900 + 37 * i), (n, 3000), (n, 64)], 8, 2, 128, 16, seed=i) for i in range(2)]
    want = [b.run(xn, max_query=n) for b in bs]
    for b, w in zip(bs, want):
        b.check(w)
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(bs[i].run(xn, max_query=n))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(x, w) for x in g)
    graph = torch.cuda.CUDAGraph()
    b = bs[0]
    out = torch.empty_like(b.q)
    with torch.cuda.graph(graph):
        b.run(xn, max_query=n, out=out)
    other = torch.tensor([900, 64 + n, 64], dtype=torch.int32, device=cuda)  # other lengths, the same pages
    for ctx in (b.context.clone(), other, torch.zeros_like(other), b.context.clone()):
        b.context.copy_(ctx)
        out.fill_(5)
        graph.replay()
        assert torch.equal(out, b.run(xn, max_query=n))


def test_the_bound_on_rows_changes_no_result_beyond_rounding(xn, cuda):
    """max_query chooses a kernel; one that is too small is slower, not wrong."""
    b = Batch(cuda, torch.bfloat16, [(150, 400), (1, 300)], 8, 2, 128, 16)
    for m in (None, 0, 1, 2, 4, 16, 150, 10 ** 6):
        b.check(b.run(xn, max_query=m))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n,heads,kv,hd,window", [(3, 2, 2, 64, 0), (5, 4, 2, 128, 0), (7, 4, 2, 128, 20), (4, 8, 2, 64, 3), (40, 8, 2, 128, 0),
                                                  (200, 4, 2, 64, 0), (300, 2, 2, 128, 0), (100, 8, 2, 128, 30), (300, 2, 2, 128, 250), (1, 40, 2, 64, 9)])
def test_what_is_not_finite_stays_with_the_rows_that_see_it(xn, cuda, dtype, n, heads, kv, hd, window):
    """An infinity or NaN in a key or a value that some of a sequence's rows see: the others get what they get without it."""
    b = Batch(cuda, DTYPES[dtype], [(n, n + 100), (n, n), (n, 5000 + n)], heads, kv, hd, 16)
    want = b.run(xn, max_query=n, window=window)
    b.check(want, window=window)
    for pool, value in ((b.v, math.nan), (b.v, math.inf), (b.v, -math.inf), (b.k, math.nan)):
        saved = pool.clone()
        seen = torch.zeros(b.rows, dtype=torch.bool, device=cuda)
        for s, (rows, ctx) in enumerate(b.lengths):
            at = torch.arange(ctx - rows, ctx, device=cuda)  # the last key that each row sees
            keys = [ctx - 1, ctx - rows // 2, ctx - rows - (window // 2 if window else -1)] if s != 1 else [rows // 2 + 1]
            for key in keys:
                key = min(max(key, 0), ctx - 1)
                pool[int(b.table[s, key // 16]), 0, key % 16, 5] = value
                seen[int(b.starts[s]):int(b.starts[s]) + rows] |= (key <= at) & ((key > at - window) if window else True)
        got = b.run(xn, max_query=n, window=window)
        pool.copy_(saved)
        mine = got[:, :heads // kv]
        assert not bool(mine[seen][:, :, 5].isfinite().any())
        assert torch.equal(mine[~seen], want[~seen][:, :heads // kv])
        assert torch.equal(got[:, heads // kv:], want[:, heads // kv:])


@pytest.mark.parametrize("n", [1, 5, 70])
def test_broadcast_queries_and_pools(xn, cuda, n):
    """Dimensions of stride 0 are read like any other: one query for all heads or tokens, one key head or page for all."""
    b = Batch(cuda, torch.bfloat16, [(n, 150), (n, 90), (n, n)], 8, 2, 64, 16)
    k, v = (torch.nan_to_num(t) for t in (b.k, b.v))
    run = lambda q, k, v: xn.attention_paged(q, k, v, b.table, b.context, b.scale, query_starts=b.starts, max_query=n)  # noqa: E731
    for q in (b.q[:, :1].expand_as(b.q), b.q[:1].expand_as(b.q), b.q[:1, :1].expand_as(b.q)):
        wide = Batch.__new__(Batch)
        wide.__dict__.update(b.__dict__, q=q.contiguous(), k=k, v=v)
        wide.check(run(q, k, v))
    for kk, vv in ((k[:, :1].expand_as(k), v[:, :1].expand_as(v)), (k[3:4].expand_as(k), v[3:4].expand_as(v))):
        wide = Batch.__new__(Batch)
        wide.__dict__.update(b.__dict__, k=kk.contiguous(), v=vv.contiguous())
        wide.check(run(b.q, kk, vv))
    assert torch.equal(xn.attention_paged(b.q, k, v, b.table[:1].expand_as(b.table), b.context, b.scale, query_starts=b.starts, max_query=n),
                       xn.attention_paged(b.q, k, v, b.table[:1].expand_as(b.table).contiguous(), b.context, b.scale, query_starts=b.starts, max_query=n))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("streams,n,heads,kv,ctx", [(1, 5, 8, 2, 90), (3, 40, 8, 2, 200), (2, 37, 3, 1, 600), (4, 100, 6, 2, 131), (6, 24, 24, 24, 24), (1, 300, 8, 1, 300),
                                                    (49, 17, 1, 1, 50), (50, 17, 1, 1, 50), (2, 600, 2, 2, 1300)])
def test_small_calls_on_either_side_of_the_line(xn, cuda, streams, n, heads, kv, hd, ctx):
    """Items of 16 rows from a few to hundreds, over short and long contexts, with tables that fit and tables that have room."""
    b = Batch(cuda, torch.bfloat16, [(n - i % 2, ctx + 3 * i) for i in range(streams)], heads, kv, hd, 16, spread=0.7)
    b.check(b.run(xn, max_query=n))
    b.check(b.run(xn, max_query=n, window=20), window=20)
    b.table = torch.nn.functional.pad(b.table, (0, 3000), value=-1)
    b.check(b.run(xn, max_query=n))
