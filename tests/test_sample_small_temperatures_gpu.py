"""The draw at temperatures down to the smallest number there is: logits as close together as the temperature is small, so that several
tokens weigh something, around 0 and elsewhere."""
import numpy as np
import pytest
import torch

from test_sample_gpu import check

pytestmark = pytest.mark.gpu
LEAST = 2.0 ** -149


def logits(rows, vocab, unit, seed, top=0.0):
    """The largest is `top`, the others lie 0 to 40 units below it, many equal ones among them."""
    rng = np.random.default_rng(seed)
    x = top - rng.integers(0, 41, (rows, vocab)) * unit
    x[:, vocab // 3] = top
    return x


@pytest.mark.parametrize("vocab", [2, 300, 9000, 40000])
@pytest.mark.parametrize("steps", [1, 3, 100, 714, 50000])  # the temperature in units of 2^-149: 1.4e-45 to 7e-41
@pytest.mark.parametrize("top", [0, 17, -60])
def test_subnormal_temperatures(xn, cuda, vocab, steps, top):
    rows = 12
    t = torch.full((rows,), steps * LEAST, dtype=torch.float64).float()
    assert float(t[0].double()) == steps * LEAST
    unit = max(1, steps // 4) * LEAST
    x = torch.from_numpy(logits(rows, vocab, unit, vocab + steps, top * unit)).float().to(cuda)
    g = torch.Generator(device=cuda).manual_seed(vocab)
    u = torch.rand(rows, generator=g, device=cuda)
    k = torch.tensor([2, 3, 1, 40, 200, 257, 1000, 2049, 5000, vocab - 1, vocab, 7], dtype=torch.int32, device=cuda)
    p = torch.linspace(0.2, 0.97, rows, device=cuda)
    m = torch.linspace(0.0, 0.9, rows, device=cuda)
    t = t.to(cuda)
    check(xn, x, u, temperature=t)
    check(xn, x, u, temperature=t, top_k=k)
    check(xn, x, u, temperature=t, top_p=p)
    check(xn, x, u, temperature=t, min_p=m)
    check(xn, x, u, temperature=t, top_k=k, top_p=p)
    check(xn, x, u, temperature=t, top_k=k, top_p=p, min_p=m)


def test_two_tokens_a_smallest_step_apart(xn, cuda):
    """Weights 1 and e^-1: the second is drawn from 1 / (1 + e^-1) = 0.731 on."""
    x = torch.tensor([[0.0, -LEAST], [0.0, -LEAST], [-LEAST, 0.0], [5 * LEAST, 4 * LEAST]], dtype=torch.float64).float().to(cuda)
    u = torch.tensor([0.73, 0.74, 0.26, 0.74], device=cuda)
    t = torch.full((4,), LEAST, dtype=torch.float64).float().to(cuda)
    k = torch.full((4,), 2, dtype=torch.int32, device=cuda)
    wide = torch.nn.functional.pad(x, (0, 5000), value=-1.0)
    for y, kw in ((x, {}), (wide, {}), (wide, dict(top_k=k)), (wide, dict(top_k=k, top_p=torch.full((4,), 0.999, device=cuda)))):
        assert xn.sample(y, u, temperature=t, **kw).tolist() == [0, 1, 0, 1]


@pytest.mark.parametrize("top", [0.0, 1.0, -3.0e38, 5.0])
def test_temperatures_far_below_the_logits_spacing(xn, cuda, top):
    """Of the logits only those equal to the largest weigh anything, and there are more of them than are ever listed."""
    rows, vocab = 6, 20000
    x = torch.full((rows, vocab), top, dtype=torch.float32)
    below = torch.nextafter(torch.tensor(top), torch.tensor(-torch.inf))
    x[:, ::2] = below if top else -1e-30
    u = torch.linspace(0.01, 0.99, rows, device=cuda)
    for t in (1e-38, 1e-40, LEAST):
        ts = torch.full((rows,), t, dtype=torch.float64).float().to(cuda)
        k = torch.tensor([1, 2, 300, 3000, 9999, 15000], dtype=torch.int32, device=cuda)
        check(xn, x.to(cuda), u, temperature=ts, top_k=k)
        check(xn, x.to(cuda), u, temperature=ts, top_k=k, top_p=torch.linspace(0.1, 0.9, rows, device=cuda))
