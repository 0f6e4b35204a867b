"""How precise attention over the 8-bit cache is, as a 2-norm over many results: a bound per entry has to allow for every rounding going the
same way, so it does not see the loss of a part of the weights or of a digit of the queries."""
import math

import pytest
import torch

import plain_q8
from test_attention_q8 import BF, F32, check, decode, make, ops, prefill      # noqa: F401 (ops: a fixture)


def reference(c, window=0, rows=None):
    """Results in 64 bits, and sums of weight * |value|."""
    H, G, hd = c["H"], c["G"], c["hd"]
    rows = range(len(c["positions"])) if rows is None else rows
    ref, size = (torch.zeros(len(rows), H * hd, dtype=torch.float64) for _ in range(2))
    for i, r in enumerate(rows):
        s, p = int(c["seq"][r]), int(c["positions"][r])
        keys = plain_q8.seen_keys(p, window, 0)
        for h in range(H):
            cols, g = slice(h * hd, (h + 1) * hd), h // (H // G)
            ref[i, cols], size[i, cols], _ = plain_q8.attend(c["q"][r, cols].double(), c["held"][0][s][:, g], c["held"][1][s][:, g], p, keys, hd ** -0.5)
    return ref, size


def norm(x):
    return x.pow(2).sum().sqrt().item()


def bound_16(ref, size):
    """For bfloat16 results, of |out - the result rounded once| over |result|.  What the kernel rounds is off by e <= 2^-16 sum w |v|
    (2^-17 from the weights' two parts, and no more from the rest, which is done in 32 bits).  That only shows where a border between two
    bfloat16 numbers lies in between: with borders a step d <= 2^-7 |result| apart in e / d of the entries, each then off by d, so the
    mean square is d e.  (Weights in one part are off by up to 2^-8, by 2^-10 or so in the mean.)"""
    return math.sqrt(2.0 ** -7 * 2.0 ** -16 * (ref.abs() * size).sum().item()) / norm(ref)


# For 32-bit results, of |out - result| over |result|: a score of some units takes four roundings of 2^-24 of itself, an exponential is off by
# up to 2^-22, a weight's three parts by 2^-25, the sums by a rounding per tile: 2^-21.5 or so in the mean, 2^-20 with all of them at once.
# (Weights in two parts are off by up to 2^-17, by 2^-18.6 in the mean.)
BOUND_32 = 2.0 ** -20


def test_the_bounds_see_a_part_that_is_lost():
    """The mistakes are planted in the plain form."""
    g = torch.Generator().manual_seed(1)
    for n in (17, 300, 2000):
        w = torch.softmax(torch.randn(64, n, generator=g, dtype=torch.float64), -1)
        v = torch.randn(n, 64, generator=g, dtype=torch.float64)
        ref, size = w @ v, w @ v.abs()
        first = w.to(BF).double()
        second = (w - first).to(BF).double()
        off = lambda x: norm((x @ v).to(BF).double() - ref.to(BF).double()) / norm(ref)      # noqa: E731
        assert off(first) > bound_16(ref, size) > off(first + second)
        assert norm((first + second) @ v - ref) / norm(ref) > BOUND_32


@pytest.mark.gpu
@pytest.mark.parametrize("H,G,hd,ps,window", [(4, 4, 128, 16, 0), (4, 2, 64, 16, 0), (4, 2, 128, 32, 100), (4, 1, 64, 64, 70)])
def test_long_chunks(ops, H, G, hd, ps, window):      # noqa: F811
    """The chunk's length decides which kernel takes it, but not how precise the results are."""
    c = make(ops, BF, H, G, hd, ps, [400, 700], [150, 130], seed=hd + ps)
    rows = range(0, 280, 4)
    ref, size = reference(c, window, rows)
    for work in (True, False):
        out = prefill(ops, c, window, work=work).cpu().double()[list(rows)]
        assert norm(out - ref.to(BF).double()) / norm(ref) <= bound_16(ref, size), work


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,G,hd,ps", [(4, 4, 128, 16), (8, 2, 64, 16), (12, 1, 128, 16), (4, 1, 256, 16), (4, 4, 32, 16), (6, 3, 80, 5)])
def test_decoding_rows_and_few_rows(ops, dtype, H, G, hd, ps):      # noqa: F811
    c = make(ops, dtype, H, G, hd, ps, [17, 300, 700, 2000, 129, 64], [1] * 6, seed=hd)
    ref, size = reference(c)
    chunk = make(ops, dtype, H, G, hd, ps, [300, 700], [9, 30], seed=hd + 1)
    chunk_ref, chunk_size = reference(chunk)
    for out, ref, size in ((decode(ops, c), ref, size), (prefill(ops, chunk), chunk_ref, chunk_size)):
        out = out.cpu().double()
        if dtype == BF:
            assert norm(out - ref.to(BF).double()) / norm(ref) <= bound_16(ref, size)
        else:
            assert norm(out - ref) / norm(ref) <= BOUND_32


def with_a_large_channel(c, channel, large):
    """One channel of the queries is far larger than the others, and no key has anything in it."""
    c["q"].view(len(c["positions"]), c["H"], c["hd"])[:, :, channel] = large
    c["k"].codes[..., channel] = 0
    for k in c["held"][0]:
        k[..., channel] = 0
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,G,hd,ps", [(4, 4, 64, 16), (4, 1, 128, 16), (2, 2, 32, 8), (12, 1, 64, 16), (2, 1, 256, 16), (2, 2, 48, 5)])
@pytest.mark.parametrize("large,spread", [(3000.0, 1.0), (3000.0, 20.0), (-16000.0, 1.0)])
def test_a_large_channel_costs_the_others_nothing(ops, dtype, H, G, hd, ps, large, spread):      # noqa: F811
    """A dot product in 32 bits keeps every channel's own bits, and so the tolerance is the one of all other tests."""
    c = with_a_large_channel(make(ops, dtype, H, G, hd, ps, [17, 300, 64], [1] * 3, seed=hd, spread=spread), 5, large)
    check(c, decode(ops, c), hd ** -0.5)
    c = with_a_large_channel(make(ops, dtype, H, G, hd, ps, [90, 200], [9, 20], seed=hd, spread=spread), hd - 1, large)
    check(c, prefill(ops, c), hd ** -0.5)
    if spread == 1.0 and dtype == F32:
        ref, _ = reference(c)
        assert norm(prefill(ops, c).cpu().double() - ref) / norm(ref) <= BOUND_32
