"""Rotary positions, alone and on the way into a paged cache, against the rotation of complex numbers in 64 bits."""
import pytest
import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def turned(x, positions, freqs, interleaved):
    """f64: every pair as a complex number, times e^(i position frequency); the rest of the head as it is."""
    n = freqs.numel()
    z = torch.polar(torch.ones(1, 1, dtype=torch.float64, device=x.device), positions.double()[:, None] * freqs)[:, None]
    y = x.double().clone()
    if interleaved:
        w = torch.complex(y[..., 0:2 * n:2].contiguous(), y[..., 1:2 * n:2].contiguous()) * z
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = w.real, w.imag
    else:
        w = torch.complex(y[..., :n].contiguous(), y[..., n:2 * n].contiguous()) * z
        y[..., :n], y[..., n:2 * n] = w.real, w.imag
    return y


def close(got, want, x):
    # two products with a sine and a cosine of relative error 2^-22 together at most, one rounding to the type
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    tol = 2.0 ** -22 * 2 * x.double().abs().amax() + half * want.abs() + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,head_dim,rotated", [
    (1, 32, 128, 128), (1, 1, 64, 16), (7, 3, 64, 64), (33, 5, 128, 64), (300, 8, 80, 40), (5, 2, 6, 2), (4, 3, 34, 30), (2, 2, 64, 0),
    (2000, 32, 128, 128), (9000, 4, 64, 32), (0, 4, 64, 64), (3, 0, 64, 64)])
def test_rope_against_complex_numbers(xn, cuda, dtype, interleaved, tokens, heads, head_dim, rotated):
    g = torch.Generator(device=cuda).manual_seed(tokens + heads)
    x = torch.randn(tokens, heads, head_dim, generator=g, device=cuda).to(DTYPES[dtype])
    pos = torch.randint(0, 100000, (tokens,), generator=g, device=cuda)
    freqs = xn.rope_frequencies(rotated, device=cuda) if rotated else torch.zeros(0, dtype=torch.float64, device=cuda)
    y = xn.rope(x, pos, freqs, interleaved=interleaved)
    assert y.shape == x.shape and y.dtype == x.dtype
    if x.numel():
        close(y, turned(x, pos, freqs, interleaved), x)
        assert torch.equal(y[..., rotated:], x[..., rotated:])


@pytest.mark.gpu
@pytest.mark.parametrize("first", [0, 2 ** 20, 2 ** 31 + 12345, 2 ** 40, -5])
def test_far_positions_lose_nothing(xn, cuda, first):
    """Products of a position and a frequency in 64 bits: an angle of 2^40 radians is known to 2^-12 of a turn's 2^-24 there."""
    x = torch.randn(64, 4, 64, device=cuda)
    pos = torch.arange(first, first + 64, device=cuda)
    freqs = xn.rope_frequencies(64, device=cuda)
    want = turned(x, pos, freqs, False)
    # beyond 2^31 the reference's own product, rounded at 2^-53 of the angle, is what limits both sides
    tol = 2.0 ** -20 * float(x.abs().max()) + abs(first) * 2.0 ** -51 * float(x.abs().max())
    assert float((xn.rope(x, pos, freqs).double() - want).abs().max()) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_strides_offsets_and_in_place(xn, cuda, dtype):
    g = torch.Generator(device=cuda).manual_seed(3)
    qkv = torch.randn(19, 3 * 4 * 64 + 5, generator=g, device=cuda).to(DTYPES[dtype])
    pos, freqs = torch.arange(19, device=cuda) * 7, xn.rope_frequencies(64, device=cuda)
    for off in (0, 1, 3, 256):  # rows of an odd pitch, heads at any offset
        x = qkv[:, off:off + 256].unflatten(1, (4, 64))
        close(xn.rope(x, pos, freqs), turned(x, pos, freqs, False), x)
    x = torch.randn(4, 19, 64, generator=g, device=cuda).to(DTYPES[dtype]).transpose(0, 1)
    close(xn.rope(x, pos, freqs, interleaved=True), turned(x, pos, freqs, True), x)
    x = torch.randn(64, 4, 19, generator=g, device=cuda).to(DTYPES[dtype]).permute(2, 1, 0)  # heads of scattered elements
    close(xn.rope(x, pos, freqs), turned(x, pos, freqs, False), x)
    x = torch.randn(1, 4, 64, generator=g, device=cuda).to(DTYPES[dtype]).expand(19, 4, 64)
    close(xn.rope(x, pos, freqs), turned(x, pos, freqs, False), x)
    x = torch.randn(19, 4, 64, generator=g, device=cuda).to(DTYPES[dtype])
    for inter in (False, True):
        want = xn.rope(x, pos, freqs, interleaved=inter)
        y = x.clone()
        assert xn.rope(y, pos, freqs, interleaved=inter, out=y).data_ptr() == y.data_ptr() and torch.equal(y, want)
        wide = torch.full((19, 4, 72), 5.0, device=cuda, dtype=DTYPES[dtype])
        xn.rope(x, pos, freqs, interleaved=inter, out=wide[..., 8:])
        assert torch.equal(wide[..., 8:], want) and bool((wide[..., :8] == 5).all())


def test_frequencies(xn):
    f = xn.rope_frequencies(64, base=500000.0)
    assert f.dtype == torch.float64 and f.shape == (32,)
    assert torch.allclose(f, 500000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64), rtol=1e-14)
    assert torch.allclose(xn.rope_frequencies(64, scaling="linear", factor=4.0), xn.rope_frequencies(64) / 4, rtol=1e-14)
    b = xn.rope_frequencies(64, scaling="base", factor=4.0) / xn.rope_frequencies(64)
    assert abs(float(b[0]) - 1) < 1e-12 and abs(float(b[-1]) - 0.25) < 1e-12 and bool((b.diff() < 0).all())
    r = xn.rope_frequencies(128, scaling="bands", factor=8.0, context=8192) / xn.rope_frequencies(128)
    turns = 8192 * xn.rope_frequencies(128) / (2 * torch.pi)
    assert bool((r[turns > 4] == 1).all()) and torch.allclose(r[turns < 1], torch.tensor(0.125, dtype=torch.float64), rtol=1e-14)
    assert bool((r.diff() <= 1e-15).all())
    for bad in (dict(rotated=7), dict(rotated=0), dict(rotated=64, scaling="other"), dict(rotated=64, scaling="linear", factor=0.0),
                dict(rotated=64, scaling="bands", low_turns=4.0, high_turns=1.0)):
        with pytest.raises(xn.XnError):
            xn.rope_frequencies(**bad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens,heads,kv,head_dim,page", [(1, 8, 8, 64, 16), (32, 32, 8, 128, 16), (77, 6, 2, 64, 5), (500, 4, 1, 128, 64),
                                                          (3, 1, 1, 6, 1), (2500, 16, 16, 128, 128)])
def test_append_writes_its_slots_and_nothing_else(xn, cuda, dtype, tokens, heads, kv, head_dim, page):
    g = torch.Generator(device=cuda).manual_seed(tokens)
    dt = DTYPES[dtype]
    qkv = torch.randn(tokens, heads + 2 * kv, head_dim, generator=g, device=cuda).to(dt)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    pages = tokens // page + 4
    pools = torch.randn(pages, 2, kv, page, head_dim, generator=g, device=cuda).to(dt)  # both pools in one tensor
    before = pools.clone()
    slots = torch.randperm(pages * page, generator=g, device=cuda)[:tokens]
    if tokens > 2:  # padding, on either side of the pool
        slots[1], slots[2] = -1, pages * page
    pos = torch.randint(0, 5000, (tokens,), generator=g, device=cuda)
    freqs = xn.rope_frequencies(head_dim // 2 // 2 * 2, device=cuda)
    out = xn.paged_append_(pools[:, 0], pools[:, 1], k, v, slots, q=q, positions=pos, freqs=freqs)
    close(out, turned(q, pos, freqs, False), q)
    ok = (slots >= 0) & (slots < pages * page)
    at, row = slots[ok] // page, slots[ok] % page
    close(pools[at, 0, :, row], turned(k, pos, freqs, False)[ok], k)
    assert torch.equal(pools[at, 1, :, row], v[ok])
    untouched = torch.ones(pages, page, dtype=torch.bool, device=cuda)
    untouched[at, row] = False
    assert torch.equal(pools.permute(0, 3, 1, 2, 4)[untouched], before.permute(0, 3, 1, 2, 4)[untouched])
    # without frequencies nothing turns, and without queries nothing comes back
    assert xn.paged_append_(pools[:, 0], pools[:, 1], k, v, slots) is None
    assert torch.equal(pools[at, 0, :, row], k[ok]) and torch.equal(pools[at, 1, :, row], v[ok])
    # pools of their own strides: (pages, page_size, kv_heads, head_dim) storage
    other = torch.zeros(2, pages, page, kv, head_dim, device=cuda, dtype=dt).transpose(2, 3)
    xn.paged_append_(other[0], other[1], k, v, slots, positions=pos, freqs=freqs, interleaved=True)
    close(other[0][at, :, row], turned(k, pos, freqs, True)[ok], k)
    assert torch.equal(other[1][at, :, row], v[ok])
