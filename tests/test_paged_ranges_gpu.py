"""Attention over a paged cache where scores and weights leave their ordinary range: long tails
of small weights, and scores far from zero."""
import math

import pytest
import torch

from flexkv_amd import c_ext

from test_paged_gpu import BF16, DEV, FP16, Case, _gen

pytestmark = pytest.mark.gpu


# -- many small weights ----------------------------------------------------------------

@pytest.mark.parametrize("below", [0, 2.0 ** -7])
@pytest.mark.parametrize("batch,queries,G,D", [
    (257, 1, 4, 64), (257, 2, 8, 128), (260, 3, 8, 64), (257, 1, 4, 256),   # few rows, uncut
    (1, 1, 4, 64), (3, 3, 8, 128),                                          # and dealt out
    (1, 4096, 16, 64), (1, 4096, 16, 128), (2, 3000, 16, 256),              # many rows, uncut
    (1, 60, 1, 64), (1, 20, 8, 128), (2, 9, 8, 256)])                       # and cut
def test_a_long_tail_of_small_weights_keeps_its_part_in_fp16(batch, queries, G, D, below):
    """The first token has nearly all of the attention, and tens of thousands of others e^-16.3 of
    that each, together 0.5 %: 1.4 * 2^-24, or a little less, with the same rounding for all, so that
    roundings do not average out.  `below`: how much lower a quarter of the tokens score than the others.
    A weight is rounded to 11 bits, or by half of 2^-24 of a 2^7th of the largest, 2^-32 of it."""
    n, T = 65536, 64
    g = _gen(queries)
    cache = torch.zeros(2, n // T, T, 1, D, dtype=FP16)
    flat = cache.view(2, n, D)
    flat[0, :, 0] = torch.where(torch.arange(n) < n // 4, -below, 0.0)
    flat[0, 0, 0] = 16.296875
    flat[1] = torch.randn(D, generator=g) + 1.0          # a token's values are all others'
    flat[1, 0] = 0.0
    q = torch.zeros(batch * queries, G, D, dtype=FP16)
    q[..., 0] = 1.0
    table = torch.randperm(n // T, generator=g).to(torch.int32)
    dev = torch.empty_like(cache, device=DEV)
    dev[:, table.to(DEV).long()] = cache.to(DEV)
    w = torch.zeros(batch, 1, n, device=DEV)
    lse = torch.empty(batch * queries, G, device=DEV)
    out = c_ext.paged_attention(q.to(DEV), dev[0], dev[1], table.expand(batch, -1).to(DEV),
                                torch.full((batch,), n, dtype=torch.int32, device=DEV),
                                queries * torch.arange(batch + 1, dtype=torch.int32, device=DEV),
                                scale=1.0, causal=False, lse=lse, weights=w)
    s = flat[0, :, 0].double()
    p = torch.exp(s - s.max())
    total = p.sum()
    want = (p / total) @ flat[1].double()
    half = torch.finfo(FP16).eps / 2
    # A row's sum grows by 32 keys at a time or more, and is off by at most 2^-24 of it each time.  The
    # result's rounding; a weight's of 11 bits, or 2^-32; scores are exact but for the scale, which
    # their differences of up to 2^5 take 2^-22 of, and the exponential.
    sums = n / 32 * 2.0 ** -24
    tail = ((p / total)[:, None] * flat[1].double().abs()).sum(0)
    tol = half * want.abs() + tail * (half + 2.0 ** -16 + 2 * sums) \
        + n * 2.0 ** -32 * flat[1].double().abs().max()
    off = (out.double() - want.to(DEV)).abs()
    assert (off <= tol.to(DEV)).all(), (off.max(), tol.min())
    assert ((lse.double() - (s.max() + math.log(total))).abs() <= sums + 2.0 ** -15).all()
    share = (queries * G * p / total).to(DEV)
    for b in range(0, batch, 64):
        assert ((w[b, 0].double() - share).abs() <= share * (sums + 2.0 ** -14)).all()


# -- scores far from zero --------------------------------------------------------------

@pytest.mark.parametrize("scale", [2.0 ** 12, 2.0 ** 16, -2.0 ** 17, 2.0 ** 24])
@pytest.mark.parametrize("kw", [
    dict(keys=[400, 90], queries=[1, 1]),
    dict(keys=[300], queries=[2], G=8, D=64, dtype=FP16),
    dict(keys=[300], queries=[3], D=256),
    dict(keys=[5000], queries=[1], H=1, G=8),
    dict(keys=[400, 90], queries=[6, 7], D=64),
    dict(keys=[300], queries=[8], dtype=FP16),
    dict(keys=[2600, 31], queries=[1, 1], H=1, G=23, D=256),
    dict(keys=[300], queries=[3], H=1, G=9, D=256, dtype=FP16),
    dict(keys=[3000], queries=[2], H=1, G=8, T=1024, width=16500),
    dict(keys=[400, 90], queries=[40, 60], D=64),
    dict(keys=[400], queries=[70], dtype=FP16),
    dict(keys=[2300], queries=[30], H=1, D=256),
], ids=lambda kw: "-".join(str(v) for v in kw.values()))
def test_the_weights_a_row_gives_add_up_to_one(kw, scale):
    """Scores of 2^17 to 2^30 in units of log 2, whose last bits are worth up to a factor of 2^64
    of a weight: the shares are those that the row's sum is of."""
    c = Case(seed=7, **kw)
    c.w = torch.zeros_like(c.w)
    out, lse, w = c.run(scale=scale)
    assert out.isfinite().all() and lse.isfinite().all()
    for b, n in enumerate(c.queries):
        # two sums of up to 5000 terms, half of 2^-24 of it each time; quotient and exponentials 2^-20
        got = w[b].double().sum(1) / (n * c.G)
        assert ((got - 1).abs() <= 2.0 ** -10).all(), (b, got)


@pytest.mark.parametrize("queries", [1, 50])
@pytest.mark.parametrize("scale", [2.0 ** 127, -(2.0 ** 127), 2.0 ** -149])
def test_the_largest_and_smallest_scales(queries, scale):
    """With scores of 0 every key weighs alike."""
    c = Case([200], [queries], H=1, G=2, D=64)
    c.q = torch.zeros_like(c.q)
    c.check(c.run(scale=scale), scale=scale)
