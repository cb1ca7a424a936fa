"""Attention behind a shared prefix (csrc/paged_shared.hip), in each form of the prefix's kernel: how exact a row is, and that its
bits are its own."""

import pytest
import torch

from test_paged_shared_gpu import BF16, HALF, NAN, U, Shared, _bits

pytestmark = pytest.mark.gpu

# (head dim, sequences): of four query rows a kv head each, so 12 rows to 280, which is every form, and more than one block of rows
FORMS = [(64, 3), (64, 7), (64, 15), (64, 30), (64, 70), (128, 3), (128, 7), (128, 15), (128, 30), (128, 70), (256, 7), (256, 15),
         (256, 40)]


def _batch(dev, d, batch):
    lengths = [(37 * i) % 91 for i in range(batch)]
    return Shared(dev, d + batch, 4, 2, d, 32, 1000, lengths, 2, counts=[1 + i % 3 % 2 for i in range(batch)])


def _exact(s, i):
    """Sequence i's rows in 64 bits, and how far a kernel may be off before it rounds its outputs: scores of d products in fp32
    (d + 4 steps of 2^-24 of the products' absolute sum, twice since the maximum or the sum has as much); weights of two bf16 terms,
    2^-8 of 2^-8; fp32 sums, and the exponentials and joins of parts (64 steps for all of these)."""
    n, c, d, hq = s.lengths[i], s.counts[i], s.d, s.hq
    keys, vals = (torch.cat([p, o]).double() for p, o in zip((s.pk, s.pv), s.own[i]))
    rep, total = hq // keys.shape[1], s.prefix + n + c
    q = s.q.view(-1, s.T, hq, d)[i, :c].double()
    seen = torch.arange(total) <= s.prefix + n + torch.arange(c)[:, None]
    out, err = torch.zeros((c, hq, d), dtype=torch.float64), torch.zeros((c, hq, d), dtype=torch.float64)
    for h in range(hq):
        kh, vh = keys[:, h // rep], vals[:, h // rep]
        w = torch.softmax(torch.where(seen, q[:, h] @ kh.t() * d ** -0.5, -torch.inf), -1)
        ds = (q[:, h].abs() @ kh.abs().t()).amax(-1, keepdim=True) * d ** -0.5 * (d + 4) * U
        out[:, h] = w @ vh
        err[:, h] = (2 * ds + 2.0 ** -16 + 2 * (total + 64) * U) * (w @ vh.abs())
    return out, err


@pytest.mark.parametrize("d,batch", FORMS)
def test_weights_of_the_prefix_are_as_exact_as_the_own_keys(dev, d, batch):
    """No more than the outputs' own rounding, and what fp32 and two bf16 terms of a weight leave: paged_attention's bound."""
    s = _batch(dev, d, batch)
    got = s.run().view(batch, 2, 4, d)
    for i in range(0, batch, max(1, batch // 5)):
        c = s.counts[i]
        out, err = _exact(s, i)
        off = (got[i, :c].double().cpu() - out).abs()
        worst = (off / (HALF * (out.abs() + err) + err)).max().item()
        assert worst <= 1, f"sequence {i}: {worst:.3f} of the bound"


@pytest.mark.parametrize("d,batch", FORMS)
@pytest.mark.parametrize("padding", [NAN, 3e38, 0.0])
def test_bits_do_not_depend_on_other_rows(dev, d, batch, padding):
    """One sequence's queries made so long that its maximum is raised all along the prefix, and padding rows that hold anything:
    the other sequences keep their bits."""
    s = _batch(dev, d, batch)
    clean = _bits(s.run()).view(batch, -1)
    for i in (0, batch // 2, batch - 1):
        q = s.q.view(batch, 2, 4, d).clone()
        q[i] = (q[i].float() * 20).to(BF16)
        for j, c in enumerate(s.counts):
            q[j, c:] = padding
        y = _bits(s.run(q=q.view(-1, 4, d).to(dev))).view(batch, -1)
        others = [j for j in range(batch) if j != i]
        assert torch.equal(y[others], clean[others]), f"sequence {i}"
