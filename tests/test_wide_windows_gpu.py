"""Windows of 2^30 keys and more: they hide what lies behind them, and nothing else."""
import pytest
import torch

pytestmark = pytest.mark.gpu
PAGE, HD = 128, 64
CTX = 2 ** 30 + 1000


@pytest.mark.parametrize("n,page", [(1, PAGE), (40, PAGE), (40, 2 ** 17 - 1)])  # the streaming kernel, the tensor-memory kernel, the former again
def test_windows_around_a_context_beyond_2_to_30(xn, cuda, n, page):
    """Key 0 outweighs all others together (e^40 against 2^30) where it is seen; every other key is page 1 again and again."""
    pages = -(-CTX // page)
    k, v = (torch.zeros(2, 1, page, HD, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    k[0, 0, 0, 0], v[0, 0, 0, :] = 5.0, 3.0
    q = torch.zeros(n, 1, HD, dtype=torch.bfloat16, device=cuda)
    q[:, :, 0] = 8.0
    table = torch.ones(1, pages, dtype=torch.int32, device=cuda)
    table[0, 0] = 0
    starts, context = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, n], [CTX]))
    room = pages * page
    for window in (0, CTX - n // 2, CTX, CTX + 1, room - 1, room, 2 ** 31 - 1, 2 ** 40, 2 ** 63 - 1):
        got = xn.attention_paged(q, k, v, table, context, 1.0, query_starts=starts, max_query=n, window=window)
        last = torch.arange(CTX - n, CTX, device=cuda)
        seen = (last < window) if window else torch.ones_like(last, dtype=torch.bool)  # key 0 > last - window
        # what the others weigh beside it, 2^30 e^-40, is below a quarter of a millionth; 3 is exact in bf16
        assert bool((got[seen] == 3.0).all()), window
        assert bool((got[~seen] == 0.0).all()), window
        if window == CTX - n // 2 and n > 1:
            assert 0 < int(seen.sum()) < n


@pytest.mark.parametrize("n", [1, 5, 40])
@pytest.mark.parametrize("hd", [64, 128])
def test_windows_that_hide_nothing(xn, cuda, n, hd):
    """With a table wider than 2^30 keys and without: the result of no window, also for rows before the first key."""
    g = torch.Generator(device=cuda).manual_seed(n)
    page = 16
    k, v = (torch.randn(40, 2, page, hd, generator=g, device=cuda).bfloat16() for _ in range(2))
    context = torch.tensor([300, n, max(n - 3, 0)], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, n, 2 * n, 3 * n], dtype=torch.int32, device=cuda)
    q = torch.randn(3 * n, 4, hd, generator=g, device=cuda).bfloat16()
    table = torch.randint(0, 40, (3, 2 ** 26 + 2 ** 20), generator=g, device=cuda, dtype=torch.int32)
    for t in (table, table[:, :19]):
        want = xn.attention_paged(q, k, v, t, context, 0.1, query_starts=starts, max_query=n)
        for window in (400, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 5, 2 ** 31 - 1, 2 ** 62):
            got = xn.attention_paged(q, k, v, t, context, 0.1, query_starts=starts, max_query=n, window=window)
            # the bound on the keys that are read chooses the kernel, so the two may differ by their roundings: a half step of the
            # output and of every probability on each side, values below 6
            assert float((got.float() - want.float()).abs().max()) <= 4 * 2.0 ** -8 * 6, window
