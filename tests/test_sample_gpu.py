"""The draw of the next token against sorting, cumulative sums and 64-bit exponentials, row by row: tokens are equal."""
import numpy as np
import pytest
import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def expected(row, u, t=1.0, k=0, p=1.0, m=0.0):
    x = np.where(np.isnan(row), -np.inf, row.astype(np.float64))
    if np.all(x == -np.inf):
        return -1
    if not t > 0:
        return int(np.argmax(x))
    top = x.max()
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / t))
    w[x == -np.inf] = 0
    order = np.lexsort((np.arange(len(x)), -x))
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        c = np.cumsum(w[order])
        order = order[(c - w[order] < p * c[-1]) | (np.arange(len(order)) == 0)]
    if m > 0:
        order = order[w[order] >= min(m, 1.0)]
    order = np.sort(order)
    c = np.cumsum(w[order])
    return int(order[np.searchsorted(c, u * c[-1], side="right")])


def check(xn, x, u, **kw):
    got = xn.sample(x, u, **kw).tolist()
    rows = x.float().cpu().numpy()
    names = dict(temperature="t", top_k="k", top_p="p", min_p="m")
    for r in range(x.shape[0]):
        one = {names[n]: v[r].double().item() if n != "top_k" else int(v[r]) for n, v in kw.items() if v is not None}
        assert got[r] == expected(rows[r], u[r].double().item(), **one), (r, one)


def settings(rows, cuda, g):
    f = lambda *a: torch.rand(rows, generator=g, device=cuda)  # noqa: E731
    t = 0.3 + 1.5 * f()
    t[::5] = 0.0
    k = (f() * 300).to(torch.int32)
    k[::4] = 0
    p = 0.3 + 0.9 * f()
    return dict(temperature=t, top_k=k, top_p=p, min_p=(f() - 0.5).clamp(min=0) * 0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 31), (40, 1000), (7, 4097), (2, 32000), (33, 32001), (1, 151936), (160, 5003), (3, 2 ** 20)])
def test_all_filters_together(xn, cuda, dtype, rows, vocab):
    g = torch.Generator(device=cuda).manual_seed(rows * 7 + vocab)
    x = (torch.randn(rows, vocab, generator=g, device=cuda) * 3).to(DTYPES[dtype])
    x[:, 3::17] = -torch.inf
    u = torch.rand(rows, generator=g, device=cuda)
    check(xn, x, u, **settings(rows, cuda, g))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["none", "temperature", "top_k", "top_p", "min_p"])
@pytest.mark.parametrize("vocab", [50, 6000, 128001])
def test_each_filter_alone(xn, cuda, which, vocab):
    rows = 24
    g = torch.Generator(device=cuda).manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=g, device=cuda) * 2.5
    every = settings(rows, cuda, g)
    check(xn, x, torch.rand(rows, generator=g, device=cuda), **({which: every[which]} if which != "none" else {}))


@pytest.mark.gpu
def test_equal_logits_are_cut_by_index(xn, cuda):
    """Ties everywhere: whole rows of one value (more of them than the sorted list holds), and a handful of levels."""
    rows, vocab = 16, 30000
    g = torch.Generator(device=cuda).manual_seed(5)
    u = torch.rand(rows, generator=g, device=cuda)
    u[0], u[1], u[2], u[3] = 0.0, 1.0 - 2.0 ** -24, 0.5, 0.25
    k = torch.tensor([1, 2, 3, 100, 2047, 2048, 2049, 5000, 29999, 30000, 30001, 0, 4096, 12345, 7, 50], dtype=torch.int32, device=cuda)
    p = torch.linspace(0.05, 1.0, rows, device=cuda)
    flat = torch.full((rows, vocab), -3.5, device=cuda)
    levels = torch.randint(-4, 5, (rows, vocab), generator=g, device=cuda).float()
    for x in (flat, levels, levels.bfloat16()):
        check(xn, x, u)
        check(xn, x, u, top_k=k)
        check(xn, x, u, top_p=p)
        check(xn, x, u, top_k=k, top_p=p)
        check(xn, x, u, temperature=torch.zeros(rows, device=cuda))


@pytest.mark.gpu
def test_values_that_differ_in_their_last_bits(xn, cuda):
    """One histogram step holds thousands of distinct logits."""
    rows, vocab = 6, 40000
    g = torch.Generator(device=cuda).manual_seed(6)
    x = 1.0 + torch.randint(0, 30000, (rows, vocab), generator=g, device=cuda).float() * 2.0 ** -23
    u = torch.rand(rows, generator=g, device=cuda)
    k = torch.tensor([5, 500, 2500, 20000, 39999, 1], dtype=torch.int32, device=cuda)
    check(xn, x, u, top_k=k)
    check(xn, x, u, top_k=k, top_p=torch.full((rows,), 0.5, device=cuda))


@pytest.mark.gpu
def test_special_values(xn, cuda):
    inf, nan = torch.inf, torch.nan
    low = torch.finfo(torch.float32).min
    x = torch.full((10, 300), -inf, device=cuda)
    x[1, 77] = 1.0
    x[2, 5], x[2, 6], x[2, 200] = nan, 2.0, 2.0
    x[3] = low
    x[4], x[4, 9] = low, 0.0
    x[5, 3], x[5, 100], x[5, 7] = inf, inf, 5.0
    x[6] = nan
    x[7], x[7, ::2] = 0.0, -0.0
    x[8] = torch.arange(300, device=cuda) * 1e36
    x[9] = torch.linspace(-200, 200, 300, device=cuda)
    u = torch.tensor([0.3, 0.3, 0.7, 0.9, 0.5, 0.6, 0.1, 0.55, 0.2, 0.999], device=cuda)
    ones = torch.ones(10, device=cuda)
    for kw in ({}, dict(top_k=torch.full((10,), 2, dtype=torch.int32, device=cuda)), dict(top_p=0.6 * ones), dict(min_p=0.5 * ones),
               dict(temperature=0 * ones), dict(temperature=1e-30 * ones), dict(temperature=1e30 * ones), dict(top_p=0 * ones),
               dict(min_p=7 * ones), dict(top_p=-1 * ones, top_k=torch.full((10,), -3, dtype=torch.int32, device=cuda))):
        check(xn, x, u, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rows_of_any_pitch_and_alignment(xn, cuda, dtype):
    g = torch.Generator(device=cuda).manual_seed(8)
    wide = (torch.randn(9, 5013, generator=g, device=cuda) * 2).to(DTYPES[dtype])
    u = torch.rand(9, generator=g, device=cuda)
    kw = settings(9, cuda, g)
    for lo, hi in ((0, 5013), (1, 5000), (3, 3 + 64), (5, 12), (2, 3)):
        check(xn, wide[:, lo:hi], u, **kw)
    check(xn, wide.t()[:9, :9], u, **kw)
    check(xn, wide[:1].expand(9, 5013), u, **kw)


@pytest.mark.gpu
def test_uniform_out_of_range_draws_a_kept_token(xn, cuda):
    x = torch.randn(5, 1000, device=cuda)
    u = torch.tensor([1.0, 2.0, -1.0, torch.nan, torch.inf], device=cuda)
    k = torch.full((5,), 10, dtype=torch.int32, device=cuda)
    got = xn.sample(x, u, top_k=k)
    kept = x.topk(10, 1).indices.sort(1).values
    assert got.tolist() == [int(kept[0, -1]), int(kept[1, -1]), int(kept[2, 0]), int(kept[3, 0]), int(kept[4, -1])]


@pytest.mark.gpu
def test_no_rows(xn, cuda):
    assert xn.sample(torch.zeros(0, 10, device=cuda), torch.zeros(0, device=cuda)).shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [300, 9000, 128001])
def test_top_p_wherever_its_border_lies(xn, cuda, vocab):
    """Borders among the likeliest tokens, far down, between clumps of tokens and in the middle of one."""
    rows = 24
    g = torch.Generator(device=cuda).manual_seed(vocab + 1)
    n = lambda s: torch.randn(rows, vocab, generator=g, device=cuda) * s  # noqa: E731
    clumps = torch.randint(0, 5, (rows, vocab), generator=g, device=cuda).float() * 0.7
    p = torch.cat([torch.linspace(0.02, 0.98, rows - 8, device=cuda),
                   torch.tensor([1e-9, 1e-30, 0.0, -1.0, 0.999, 0.99999, 1 - 2.0 ** -24, 0.5], device=cuda)])
    u = torch.rand(rows, generator=g, device=cuda)
    steep, two = n(1.0) * 30, n(0.01)
    two[:, ::3] -= 9.0
    for x in (n(0.02), n(3.0), steep, clumps, clumps + n(1e-5), clumps + n(0.003), two, two - 300 * (n(1.0) > 1.5).float()):
        check(xn, x, u, top_p=p)
        check(xn, x, u, top_p=p, min_p=torch.full((rows,), 0.2, device=cuda), temperature=0.2 + u)
    check(xn, n(1e-37), u, top_p=p, temperature=torch.full((rows,), 1e-38, device=cuda))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [8192, 16411, 70001])
@pytest.mark.parametrize("rows", [1, 2, 9, 18, 19, 37, 38, 74, 75])
def test_rows_that_several_ctas_share(xn, cuda, rows, vocab):
    """Clusters of every size, on a machine that earlier launches still fill, so that the CTAs of a cluster do not begin together: short
    stretches, rows that end after the first pass beside rows that go on, and rows of nothing."""
    g = torch.Generator(device=cuda).manual_seed(rows + vocab)
    x = torch.randn(rows, vocab, generator=g, device=cuda) * 2
    x[rows // 2] = -torch.inf
    u = torch.rand(rows, generator=g, device=cuda)
    kw = settings(rows, cuda, g)
    check(xn, x, u, **kw)
    want = xn.sample(x, u, **kw)
    heads = torch.randn(300, 32, 128, generator=g, device=cuda).bfloat16()
    pos, freqs = torch.arange(300, device=cuda), xn.rope_frequencies(128, device=cuda)
    got = []
    for i in range(20):
        xn.rope(heads[:1 + 15 * i], pos[:1 + 15 * i], freqs)
        got.append(xn.sample(x, u, **kw))
        got.append(xn.sample(x, u, **kw))
    assert all(torch.equal(t, want) for t in got)
