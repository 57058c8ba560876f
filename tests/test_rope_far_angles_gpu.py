"""Angles of far positions against whole-number arithmetic: a position loses nothing however far it is."""
import math
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu


def pi_digits(bits):
    """floor(pi * 2^bits): Machin, pi = 16 arctan(1/5) - 4 arctan(1/239)."""
    guard = bits + 32

    def arctan(n):
        term, total, i = (1 << guard) // n, 0, 1
        while term:
            total += term // i if i % 4 == 1 else -(term // i)
            term //= n * n
            i += 2
        return total

    return (16 * arctan(5) - 4 * arctan(239)) >> 32


TWO_PI = Fraction(pi_digits(200), 2 ** 199)


def sine_cosine(position, freq):
    """Of the product of a whole number and an f64, reduced by whole turns without rounding."""
    angle = Fraction(position) * Fraction(freq)
    rest = float(angle - round(angle / TWO_PI) * TWO_PI)
    return math.sin(rest), math.cos(rest)


@pytest.mark.parametrize("first", [1, 12345, 2 ** 24 + 1, 2 ** 31 + 12345, 2 ** 40 + 7, -2 ** 45 - 3, 2 ** 50 + 11])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_at_any_position(xn, cuda, first, interleaved):
    g = torch.Generator(device=cuda).manual_seed(4)
    tokens, heads, hd = 9, 2, 32
    freqs = torch.cat([xn.rope_frequencies(24), torch.tensor([1.0 / 3.0, 0.9999999, 2.0 ** -30, 1e-8], dtype=torch.float64)]).to(cuda)
    assert freqs.numel() == hd // 2
    x = torch.randn(tokens, heads, hd, generator=g, device=cuda)
    pos = torch.arange(first, first + 3 * tokens, 3, device=cuda)
    sc = torch.tensor([[sine_cosine(p, f) for f in freqs.tolist()] for p in pos.tolist()], dtype=torch.float64, device=cuda)[:, None]
    sn, cs = sc[..., 0], sc[..., 1]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :hd // 2], x[..., hd // 2:])
    a, b = a.double(), b.double()
    want = [a * cs - b * sn, a * sn + b * cs]
    want = torch.stack(want, -1).flatten(-2) if interleaved else torch.cat(want, -1)
    got = xn.rope(x, pos, freqs, interleaved=interleaved)
    # The angle is rounded to f32 half turns, of which there is one at most: 2^-25 pi radians, below 2^-23.  Its sine and cosine are off
    # by 2^-23 at most together with that rounding's like, and each of two products and their sum by 2^-24 of the larger one.
    tol = (2 * (2.0 ** -23 + 2.0 ** -23) + 4 * 2.0 ** -24) * float(x.abs().max())
    assert float((got.double() - want).abs().max()) <= tol
