"""The paged attention on values and scores at and past the ends of their types (csrc/paged.hip): which outputs turn NaN, in
every form of the call alike, and that the others keep their bits."""

import numpy as np
import pytest
import torch

from skinny_mlx import kernels as K

pytestmark = pytest.mark.gpu

BF16, I32 = torch.bfloat16, torch.int32
NAN_BITS = 0x7FC0


def _ints(v, dev):
    return torch.tensor(v, dtype=I32, device=dev)


def _bits(t):
    return t.contiguous().view(torch.int16)


def _cache(dev, seed, hkv, d, page, lengths, width):
    """Pools whose first pages hold `lengths` tokens each, in a shuffled order; every other slot is NaN."""
    need = [-(-n // page) for n in lengths]
    order = np.random.default_rng(seed).permutation(sum(need))
    table = np.full((len(lengths), width), -1, dtype=np.int32)
    at = 0
    g = torch.Generator().manual_seed(seed)
    k = torch.full((sum(need), hkv, page, d), float("nan"), dtype=BF16)
    vt = torch.full((sum(need), hkv, d, page), float("nan"), dtype=BF16)
    for i, (n, m) in enumerate(zip(lengths, need)):
        table[i, :m] = order[at:at + m]
        at += m
        kk = torch.randn((m * page, hkv, d), generator=g).to(BF16)
        vv = torch.randn((m * page, hkv, d), generator=g).to(BF16)
        kk[n:], vv[n:] = float("nan"), float("nan")
        where = torch.from_numpy(table[i, :m].astype(np.int64))
        k[where] = kk.view(m, page, hkv, d).transpose(1, 2)
        vt[where] = vv.view(m, page, hkv, d).permute(0, 2, 3, 1)
    return table, k.to(dev), vt.to(dev)


@pytest.mark.parametrize("d,page", [(64, 16), (64, 64), (128, 16), (128, 32), (128, 256), (256, 32), (256, 64)])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_values_that_are_not_finite_make_nan_in_every_form(dev, d, page, bad):
    """One dim of one position is not finite, in a block before the last, at a block's edges, or among the new tokens. Every row
    that sees it is NaN there and has the clean bits elsewhere; rows before it are clean: as one of several new tokens, alone
    with the others cached, and however the bound cuts the keys. 16 heads weigh the position by as many weights."""
    hq, hkv, T, dim = 16, 2, 4, d - 3
    n = 700                                     # cached before the step; blocks end at multiples of 64 and 128
    hits = [0, 5, 63, 64, 127, 128, 300, 511, 639, 640, n - 1, n, n + 1, n + T - 1]
    width = (1 << 16) // page
    table, k, vt = _cache(dev, d + page, hkv, d, page, [n + T] * len(hits), width)
    pages = torch.tensor(table, device=dev)
    q = torch.randn((len(hits) * T, hq, d), generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    gate = torch.randn((len(hits) * T, hq, d), generator=torch.Generator().manual_seed(2)).to(BF16).to(dev)
    gate[:, 3] = float("-inf")                  # a closed gate hides nothing
    lens = _ints([n] * len(hits), dev)
    hit_vt = vt.clone()
    for i, p in enumerate(hits):
        hit_vt[int(table[i, p // page]), :, dim, p % page] = bad
    sees = torch.tensor([[n + t >= p for t in range(T)] for p in hits], device=dev)
    for g in (None, gate):
        clean = K.paged_attention(q, lens, pages, k, vt, d ** -0.5, gate=g, keys=n + T).view(len(hits), T, hq, d)
        assert torch.isfinite(clean).all()
        want = _bits(clean).clone()
        want[..., dim] = torch.where(sees[..., None], NAN_BITS, want[..., dim])
        for keys in (n + T, 1 << 13, 1 << 16):
            got = K.paged_attention(q, lens, pages, k, hit_vt, d ** -0.5, gate=g, keys=keys).view(len(hits), T, hq, d)
            assert torch.equal(_bits(got), want), keys
            for t in range(T):                  # every sequence's token t alone
                one = K.paged_attention(q[t::T].contiguous(), lens + t, pages, k, hit_vt, d ** -0.5,
                                        gate=None if g is None else g[t::T], keys=keys).view(len(hits), hq, d)
                assert torch.equal(_bits(one), want[:, t]), (keys, t)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf")])
def test_infinite_values_of_short_sequences(dev, d, bad):
    """The same where one workgroup finishes a sequence and no merge follows: single tokens over at most a block of keys."""
    hq, hkv, page, n = 16, 2, 16, 60
    hits = [0, 1, 15, 16, 33, n - 1, n]
    table, k, vt = _cache(dev, d, hkv, d, page, [n + 1] * len(hits), 4)
    pages, lens = torch.tensor(table, device=dev), _ints([n] * len(hits), dev)
    assert K.paged_attn_workspace(len(hits), 1, hq, hkv, d, n + 1, dev).numel() == 16  # none needed
    q = torch.randn((len(hits), hq, d), generator=torch.Generator().manual_seed(3)).to(BF16).to(dev)
    want = _bits(K.paged_attention(q, lens, pages, k, vt, d ** -0.5, keys=n + 1)).view(len(hits), hq, d).clone()
    for i, p in enumerate(hits):
        vt[int(table[i, p // page]), :, 7, p % page] = bad
    want[..., 7] = NAN_BITS
    got = K.paged_attention(q, lens, pages, k, vt, d ** -0.5, keys=n + 1).view(len(hits), hq, d)
    assert torch.equal(_bits(got), want)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("T", [1, 3])
def test_scores_that_the_scale_takes_to_minus_infinity(dev, d, T):
    """Finite products of query and key that the scale takes past fp32's range weigh nothing, as ones that are -inf themselves:
    the same bits, whether whole blocks, joins of blocks or single keys are such, and NaN where nothing else is seen."""
    hq, hkv, page, n, scale = 8, 2, 32, 1300, 64.0
    block = 64 if d == 256 else 128
    low = [range(0, block), range(block, 2 * block), range(0, 4 * block), range(0, 1024), range(1024, n), range(7, n),
           range(0, n, 3), range(n - n % block, n + T), range(0, n + T)]
    table, k, vt = _cache(dev, d + T, hkv, d, page, [n + T] * len(low), (1 << 16) // page)
    pages, lens = torch.tensor(table, device=dev), _ints([n] * len(low), dev)
    g = torch.Generator().manual_seed(4)
    q = (torch.rand((len(low) * T, hq, d), generator=g) + 0.5).to(BF16).to(dev)
    k = k * (2.0 ** -6 * d ** -0.5)             # ordinary scores of a few units
    finite, infinite = k.clone(), k.clone()
    for i, these in enumerate(low):
        p = torch.tensor(list(these))
        at = torch.from_numpy(table[i].astype(np.int64))[p // page]
        finite[at.to(dev), :, (p % page).to(dev)] = -(2.0 ** 124) / d  # a product of -2^124, half as much again or less
        infinite[at.to(dev), :, (p % page).to(dev)] = float("-inf")
    for keys in (n + T, 1 << 13, 1 << 16):
        got = K.paged_attention(q, lens, pages, finite, vt, scale, keys=keys).view(len(low), -1)
        ref = K.paged_attention(q, lens, pages, infinite, vt, scale, keys=keys).view(len(low), -1)
        assert torch.isfinite(ref[:-1]).all() and torch.isnan(ref[-1]).all(), keys
        assert torch.equal(_bits(got), _bits(ref)), keys
        over = K.paged_attention(q, lens, pages, -finite, vt, scale, keys=keys)  # past the other end: a score of +inf
        assert (_bits(over) == NAN_BITS).all(), keys

