"""The scale at both ends of what is accepted: queries of zeros give the mean of the values that a row sees."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 1e-45, 1.0, 2.3e38, 2.5e38, 3.0e38])
@pytest.mark.parametrize("n", [1, 7, 150])
def test_equal_scores(xn, cuda, scale, n):
    g = torch.Generator(device=cuda).manual_seed(n)
    ctx, page, hd = 500, 16, 64
    k, v = (torch.randn(ctx // page + 1, 2, page, hd, generator=g, device=cuda).bfloat16() for _ in range(2))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    q = torch.zeros(n, 4, hd, dtype=torch.bfloat16, device=cuda)
    table = torch.arange(len(k), dtype=torch.int32, device=cuda)[None]
    got = xn.attention_paged(q, k, v, table, ints(ctx), scale, query_starts=ints(0, n), max_query=n)
    rows = v.transpose(1, 2).flatten(0, 1).double()  # [keys, kv_heads, hd]
    last = torch.arange(ctx - n, ctx, device=cuda)
    want = (rows.cumsum(0)[last] / (last + 1)[:, None, None]).repeat_interleave(2, 1)
    # every probability is 1 and exact; sums of 500 values below 6 in f32, one rounding of the result
    assert float((got.double() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) + 500 * 6 * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 7, 150])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores_of_minus_infinity(xn, cuda, n, hd):
    """A key whose score is -inf weighs nothing; a row that sees no others is zeros."""
    g = torch.Generator(device=cuda).manual_seed(n)
    page, ctx = 16, 400
    k, v = (torch.randn(ctx // page, 1, page, hd, generator=g, device=cuda).bfloat16() for _ in range(2))
    q = torch.randn(n, 2, hd, generator=g, device=cuda).bfloat16()
    q[..., 3] = 1.0 + q[..., 3].abs()
    table = torch.arange(len(k), dtype=torch.int32, device=cuda)[None]
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    run = lambda k, c: xn.attention_paged(q, k, v, table, ints(c), 0.1, query_starts=ints(0, n), max_query=n)  # noqa: E731
    far = k.clone()
    far[:, 0, ::3, 3] = -torch.inf
    want = k.clone()
    want[:, 0, ::3, 3] = -3.0e38  # a score below -10^37: a probability of 0 likewise
    assert torch.equal(run(far, ctx), run(want, ctx)) and bool(run(far, ctx).isfinite().all())
    far[:, 0, :, 3] = -torch.inf
    assert bool((run(far, ctx) == 0).all())
