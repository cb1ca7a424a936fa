"""The cache in pages and the attention over it (csrc/paged.hip) against plain implementations in 64 bits.

Tolerances are counted, not measured. A value rounded once to bf16 is off by at most half a step, 2^-8 of it; what fp32 adds
before that is counted beside each check. Slots that hold no token are NaN or infinite throughout, so that anything that
leaks from them shows. What the kernels promise beyond that is checked bit for bit: a row's result does not depend on the
batch, on how many tokens share the step, on the page size or on where the pages lie."""

import math

import numpy as np
import pytest
import torch

from skinny_mlx import kernels as K

pytestmark = pytest.mark.gpu

BF16, I32 = torch.bfloat16, torch.int32
HALF = 2.0 ** -8    # half a bf16 step, relative
U = 2.0 ** -24      # half an fp32 step, relative
EPS = 1e-6


def _ints(v, dev):
    return torch.tensor(v, dtype=I32, device=dev)


class Cache:
    """A pool in pages and the sequences in it, with the same keys and values as dense arrays per sequence."""

    def __init__(self, dev, seed, hkv, d, page, lengths, new, spare=3, fill=True, width=None):
        g = np.random.default_rng(seed)
        self.page, self.lengths, self.new, self.hkv, self.d, self.dev = page, lengths, new, hkv, d, dev
        need = [-(-(n + t) // page) for n, t in zip(lengths, new)]
        self.width = width or max(max(need), 1)
        n_pages = sum(need) + spare
        order = g.permutation(n_pages)
        table = np.full((len(lengths), self.width), -7, dtype=np.int32)  # entries that no token needs: nonsense
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        self.table = table
        self.pages = torch.tensor(table, device=dev)
        self.k = torch.full((n_pages, hkv, page, d), float("nan"), dtype=BF16)
        self.vt = torch.full((n_pages, hkv, d, page), float("inf"), dtype=BF16)
        gen = torch.Generator().manual_seed(seed)
        self.keys, self.vals = [], []
        for i, (n, t) in enumerate(zip(lengths, new)):
            m = n + t if fill else n
            kk = torch.randn((m, hkv, d), generator=gen).to(BF16)
            vv = torch.randn((m, hkv, d), generator=gen).to(BF16)
            self.keys.append(kk)
            self.vals.append(vv)
            for p in range(m):
                pg = int(table[i, p // page])
                self.k[pg, :, p % page] = kk[p]
                self.vt[pg, :, :, p % page] = vv[p]
        self.k, self.vt = self.k.to(dev), self.vt.to(dev)

    def len_t(self):
        return _ints(self.lengths, self.dev)


def _reference(q, keys, vals, first, scale, gate=None):
    """64-bit attention of one sequence: q [c, Hq, D], keys, vals [n, Hkv, D], token t sees first + t + 1 keys. Returns the
    outputs and, per value, the bound on what fp32 and the split weights add before the last rounding."""
    c, hq, d = q.shape
    hkv = keys.shape[1]
    q64, k64, v64 = q.double().cpu(), keys.double(), vals.double()
    out = torch.zeros((c, hq, d), dtype=torch.float64)
    err = torch.zeros_like(out)
    for t in range(c):
        n = first + t + 1
        for h in range(hq):
            kh, vh = k64[:n, h // (hq // hkv)], v64[:n, h // (hq // hkv)]
            s = kh @ q64[t, h] * scale
            p = torch.softmax(s, 0)
            # a score: d products summed in fp32, each partial sum off by U; times 2 for numerator and sum. A weight: exp
            # 2 steps, its two bf16 terms 2^-16. Sums over n keys and the joins: 2(n + 16) U. Division, gate: 8 U.
            ds = (kh.abs() @ q64[t, h].abs()).max() * scale * (d + 4) * U
            rel = 2 * float(ds) + 2.0 ** -16 + 2 * (n + 16) * U + 16 * U
            out[t, h] = p @ vh
            err[t, h] = rel * (p @ vh.abs())
    if gate is not None:
        sg = torch.sigmoid(gate.double().cpu())
        out, err = out * sg, err * sg + out.abs() * 8 * U
    return out, err


def _check(got, out, err, what):
    diff = (got.double().cpu() - out).abs()
    bound = HALF * (out.abs() + err) + err
    worst = (diff / bound.clamp(min=1e-30)).max().item() if out.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1.0, f"{what}: {worst:.3f} of the bound"


LAYOUTS = [(4, 1, 128), (32, 8, 128), (16, 4, 256), (8, 8, 64), (6, 2, 64), (64, 1, 128), (12, 4, 256)]
LENGTHS = [0, 1, 15, 16, 31, 63, 64, 100, 127, 128, 129, 255, 256, 300, 511, 700]


@pytest.mark.parametrize("hq,hkv,d", LAYOUTS)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_attention_of_single_tokens(dev, hq, hkv, d, page):
    lengths = LENGTHS if hq <= 16 else LENGTHS[::3]
    c = Cache(dev, page + d + hq, hkv, d, page, lengths, [1] * len(lengths))
    q = torch.randn((len(lengths), hq, d), generator=torch.Generator().manual_seed(1)).to(BF16)
    got = K.paged_attention(q.to(dev), c.len_t(), c.pages, c.k, c.vt, d ** -0.5).view(-1, hq, d)
    for i, n in enumerate(lengths):
        out, err = _reference(q[i:i + 1], c.keys[i], c.vals[i], n, d ** -0.5)
        _check(got[i:i + 1], out, err, f"length {n}")


@pytest.mark.parametrize("hq,hkv,d,T", [(4, 1, 128, 3), (32, 8, 128, 8), (16, 4, 256, 5), (16, 4, 256, 16), (8, 8, 64, 16), (4, 4, 64, 64),
                                        (6, 2, 128, 7)])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("gated", [False, True])
def test_attention_of_several_tokens(dev, hq, hkv, d, T, page, gated):
    lengths = [0, 60, 250, 125, 300, 63, 7]
    counts = [T, T, max(1, T - 2), 1, T, 0, T - 1]
    c = Cache(dev, T + d, hkv, d, page, lengths, counts)
    g = torch.Generator().manual_seed(2)
    rows = len(lengths) * T
    q = (2 * torch.randn((rows, hq, d), generator=g)).to(BF16)
    wide = torch.randn((rows, hq, 2, d), generator=g).to(BF16).to(dev)
    gate = wide[:, :, 1] if gated else None  # as q_proj's rows hold it
    got = K.paged_attention(q.to(dev), c.len_t(), c.pages, c.k, c.vt, d ** -0.5, counts=_ints(counts, dev), gate=gate)
    got = got.view(len(lengths), T, hq, d)
    for i, n in enumerate(lengths):
        m = counts[i]
        assert (got[i, m:] == 0).all()
        if m:
            out, err = _reference(q[i * T:i * T + m], c.keys[i], c.vals[i], n, d ** -0.5,
                                  gate[i * T:i * T + m] if gated else None)
            _check(got[i, :m], out, err, f"sequence {i}")


def _bits(t):
    return t.contiguous().view(torch.int16)


def test_rows_do_not_depend_on_batch_step_or_pages(dev):
    """The same tokens in a batch and alone, in one step and one by one, over other page sizes, places and bounds: the same bits."""
    hq, hkv, d, T = 8, 2, 128, 6
    lengths, counts = [500, 3, 250, 1020], [6, 6, 4, 6]
    q = torch.randn((len(lengths) * T, hq, d), generator=torch.Generator().manual_seed(3)).to(BF16).to(dev)
    base = None
    for page in (16, 64, 256):
        c = Cache(dev, 5, hkv, d, page, lengths, counts)
        got = K.paged_attention(q, c.len_t(), c.pages, c.k, c.vt, 0.1, counts=_ints(counts, dev)).view(len(lengths), T, -1)
        base = got if base is None else base
        assert torch.equal(_bits(got), _bits(base)), page
        bound = K.paged_attention(q, c.len_t(), c.pages, c.k, c.vt, 0.1, counts=_ints(counts, dev), keys=1026)
        assert torch.equal(_bits(bound), _bits(base.view(bound.shape)))
        for i in range(len(lengths)):
            alone = K.paged_attention(q[i * T:(i + 1) * T], c.len_t()[i:i + 1], c.pages[i:i + 1], c.k, c.vt, 0.1,
                                      counts=_ints(counts[i:i + 1], dev))
            assert torch.equal(_bits(alone), _bits(base[i])), (page, i)
            for t in range(counts[i]):
                one = K.paged_attention(q[i * T + t:i * T + t + 1], _ints([lengths[i] + t], dev), c.pages[i:i + 1], c.k, c.vt, 0.1)
                assert torch.equal(_bits(one[0]), _bits(base[i, t])), (page, i, t)


def test_short_sequences_alone_and_beside_long_ones(dev):
    """A sequence of one block of keys is finished without a join when the bound allows it: the same bits."""
    hq, hkv, d = 4, 1, 128
    c = Cache(dev, 6, hkv, d, 32, [100, 5000], [1, 1])
    q = torch.randn((2, hq, d), generator=torch.Generator().manual_seed(4)).to(BF16).to(dev)
    both = K.paged_attention(q, c.len_t(), c.pages, c.k, c.vt, 0.1)
    alone = K.paged_attention(q[:1], c.len_t()[:1], c.pages[:1], c.k, c.vt, 0.1, keys=101)
    assert torch.equal(_bits(both[:1]), _bits(alone))
    out, err = _reference(q[1:].cpu(), c.keys[1], c.vals[1], 5000, 0.1)
    _check(both[1:].view(1, hq, d), out, err, "5001 keys")


@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (256, 32)])
def test_values_that_are_no_numbers_stay_with_the_rows_that_see_them(dev, d, page):
    """A draft's NaN key or infinite value reaches its own row and the later ones, and no earlier one."""
    hq, hkv, T = 4, 2, 7
    lengths = [0, 59, 130, 255]
    c = Cache(dev, 7, hkv, d, page, lengths, [T] * 4)
    q = torch.randn((4 * T, hq, d), generator=torch.Generator().manual_seed(5)).to(BF16).to(dev)
    clean = K.paged_attention(q, c.len_t(), c.pages, c.k, c.vt, 0.1).view(4, T, hq, d)
    hit = 4
    for what in ("k", "v", "v inf"):
        k, vt = c.k.clone(), c.vt.clone()
        for i, n in enumerate(lengths):
            p = n + hit
            if what == "k":
                k[int(c.table[i, p // page]), :, p % page] = float("nan")
            else:
                vt[int(c.table[i, p // page]), :, :, p % page] = float("nan" if what == "v" else "inf")
        got = K.paged_attention(q, c.len_t(), c.pages, k, vt, 0.1).view(4, T, hq, d)
        assert torch.equal(_bits(got[:, :hit]), _bits(clean[:, :hit])), what
        assert not torch.isfinite(got[:, hit:]).any(), what


def test_scores_of_minus_infinity(dev):
    """Keys whose score is -inf weigh nothing; a row with only such keys has no distribution: NaN, as a softmax gives."""
    hq, hkv, d, n = 2, 1, 64, 200
    c = Cache(dev, 8, hkv, d, 32, [n - 1, n - 1], [1, 1])
    q = torch.ones((2, hq, d), dtype=BF16, device=dev)
    k = c.k.clone()
    for p in range(n):
        if p % 3 or p >= 100:
            k[int(c.table[0, p // 32]), :, p % 32] = float("-inf")
        k[int(c.table[1, p // 32]), :, p % 32] = float("-inf")
    got = K.paged_attention(q, c.len_t(), c.pages, k, c.vt, 0.1).view(2, hq, d)
    seen = [p for p in range(100) if p % 3 == 0]
    out, err = _reference(q[:1].cpu(), c.keys[0][seen], c.vals[0][seen], len(seen) - 1, 0.1)
    _check(got[:1], out, err, "33 keys of 200")
    assert torch.isnan(got[1]).all()


def test_sequences_that_cannot_be_are_nan_and_the_others_are_right(dev):
    """Lengths, counts and pages out of range: NaN rows for that sequence, nothing read or written for it."""
    hq, hkv, d, T, page = 4, 2, 128, 2, 32
    lengths, counts = [40] * 7, [2] * 7
    c = Cache(dev, 9, hkv, d, page, lengths, counts, width=4)
    q = torch.randn((7 * T, hq, d), generator=torch.Generator().manual_seed(6)).to(BF16).to(dev)
    good = K.paged_attention(q, c.len_t(), c.pages, c.k, c.vt, 0.1).view(7, T, -1)
    bad_len = _ints([40, -1, 127, 2 ** 31 - 1, 40, 40, 40], dev)
    bad_count = _ints([2, 2, 2, 2, 3, -1, 2], dev)
    table = c.table.copy()
    table[6, 1] = c.k.shape[0]  # one past the pool; positions 32.. lie there
    got = K.paged_attention(q, bad_len, torch.tensor(table, device=dev), c.k, c.vt, 0.1, counts=bad_count).view(7, T, -1)
    assert torch.equal(_bits(got[0]), _bits(good[0]))
    assert torch.isnan(got[1:]).all()
    # keys: a bound under the sequence's tokens
    low = K.paged_attention(q[:2 * T], _ints([40, 20], dev), c.pages[:2], c.k, c.vt, 0.1, keys=41).view(2, T, -1)
    assert torch.isnan(low[0]).all() and torch.isfinite(low[1]).all()
    low = K.paged_attention(q[:2 * T], _ints([400, 20], dev), c.pages[:2], c.k, c.vt, 0.1, keys=128).view(2, T, -1)
    assert torch.isnan(low[0]).all() and torch.isfinite(low[1]).all()
    # a row that does not see the missing page is not touched by it: tokens at 31 and 32
    early = K.paged_attention(q[:T], _ints([31], dev), torch.tensor(table[6:], device=dev), c.k, c.vt, 0.1).view(T, -1)
    assert torch.isfinite(early[0]).all() and torch.isnan(early[1]).all()


def _turned(x, w, cos, sin, rd):
    """64-bit norm and rotation of heads x [n, h, D] at table rows cos, sin [n, rd / 2], and the bound on fp32's part."""
    x = x.double()
    d = x.shape[-1]
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
    a, b, c, s = x[..., :rd // 2], x[..., rd // 2:rd], cos.double()[:, None], sin.double()[:, None]
    out = torch.cat([a * c - b * s, b * c + a * s, x[..., rd:]], -1)
    # the sum of d squares d U at most, halved by the root; root, scale, weight, two products and a sum: 16 U more
    size = torch.cat([a.abs() + b.abs(), a.abs() + b.abs(), x[..., rd:].abs()], -1)
    return out, (d / 2 + 16) * U * size


@pytest.mark.parametrize("hq,hkv,d,rd,gated", [(4, 1, 128, 128, False), (16, 4, 256, 64, True), (6, 2, 64, 64, False), (3, 3, 128, 50, False),
                                               (2, 2, 64, 2, True), (5, 1, 256, 256, False), (4, 2, 128, 126, False)])
@pytest.mark.parametrize("T,page", [(1, 16), (1, 256), (5, 32), (16, 16), (37, 64), (130, 16), (61, 128)])
@pytest.mark.parametrize("norm", [True, False])
def test_store(dev, hq, hkv, d, rd, gated, T, page, norm):
    lengths = [0, 9, 100, 31, 17]
    counts = [T, max(0, T - 1), T, 0, (T + 1) // 2]
    c = Cache(dev, T + d + rd, hkv, d, page, lengths, counts, fill=False)
    g = torch.Generator().manual_seed(7)
    qs = (2 if gated else 1) * d
    cols = hq * qs + 2 * hkv * d
    # rows of a wider buffer, keys after values
    wide = torch.randn((5 * T, cols + 24), generator=g).to(BF16)
    rows = wide[:, 8:8 + cols]
    qn = (1 + 0.1 * torch.randn(d, generator=g)).to(BF16) if norm else None
    kn = (1 + 0.1 * torch.randn(d, generator=g)).to(BF16) if norm else None
    table = K.rope_table_dim(1e4, rd, c.width * page, dev)
    k0, vt0 = c.k.clone(), c.vt.clone()
    voff, koff = hq * qs, hq * qs + hkv * d
    put = lambda t: None if t is None else t.to(dev)  # noqa: E731
    out = torch.full((5 * T, hq, d), 7.0, dtype=BF16, device=dev)
    q = K.paged_store(wide.to(dev)[:, 8:8 + cols], hq, hkv, d, qs, koff, voff, put(qn), put(kn), EPS, rd, table, c.len_t(),
                      c.pages, c.k, c.vt, counts=_ints(counts, dev), out=out)
    assert q is out
    q = q.cpu().view(5, T, hq, d)
    k1, vt1 = c.k.cpu(), c.vt.cpu()
    touched = torch.zeros(k1.shape[0], page, dtype=torch.bool)
    tab = table.cpu()
    rows = rows.view(5, T, cols)
    for i, (n, m) in enumerate(zip(lengths, counts)):
        assert (q[i, m:] == 0).all()
        if not m:
            continue
        cos, sin = tab[n:n + m].unbind(-1)
        r = rows[i, :m]
        ref, err = _turned(r[:, :hq * qs].view(m, hq, qs)[..., :d], qn, cos, sin, rd)
        assert ((q[i, :m].double() - ref).abs() <= HALF * (ref.abs() + err) + err).all(), ("q", i)
        at = torch.tensor([int(c.table[i, p // page]) for p in range(n, n + m)])
        slot = torch.arange(n, n + m) % page
        touched[at, slot] = True
        ref, err = _turned(r[:, koff:koff + hkv * d].reshape(m, hkv, d), kn, cos, sin, rd)
        assert ((k1[at, :, slot].double() - ref).abs() <= HALF * (ref.abs() + err) + err).all(), ("k", i)
        assert torch.equal(_bits(vt1[at, :, :, slot]), _bits(r[:, voff:voff + hkv * d].reshape(m, hkv, d))), ("v", i)
    same = ~touched
    assert torch.equal(_bits(k1.transpose(1, 2)[same]), _bits(k0.cpu().transpose(1, 2)[same]))
    assert torch.equal(_bits(vt1.permute(0, 3, 1, 2)[same]), _bits(vt0.cpu().permute(0, 3, 1, 2)[same]))


def test_store_of_sequences_that_cannot_be(dev):
    """Nothing is written for them, and their queries are NaN; a token whose page is missing is dropped alone."""
    hq, hkv, d, T, page = 2, 1, 64, 3, 16
    c = Cache(dev, 11, hkv, d, page, [14] * 6, [T] * 6, fill=False, width=2)
    k0, vt0 = c.k.clone(), c.vt.clone()
    rows = torch.randn((6 * T, 4 * d), generator=torch.Generator().manual_seed(8)).to(BF16).to(dev)
    table = K.rope_table_dim(1e4, d, 32, dev)
    pages = c.table.copy()
    pages[5, 1] = -1
    q = K.paged_store(rows, hq, hkv, d, d, 2 * d, 3 * d, None, None, EPS, d, table, _ints([-1, 30, 2 ** 31 - 1, 14, 14, 14], dev),
                      torch.tensor(pages, device=dev), c.k, c.vt, counts=_ints([3, 3, 3, 4, -1, 3], dev)).view(6, T, hq, d)
    assert torch.isnan(q[:5]).all() and torch.isnan(q[5, 2]).all() and torch.isfinite(q[5, :2]).all()
    changed = (_bits(c.k) != _bits(k0)).any(-1).any(1)  # [page, slot]
    assert changed.sum() == 2 and changed[int(pages[5, 0]), 14:16].all()
    changed = (_bits(c.vt) != _bits(vt0)).any(2).any(1)
    assert changed.sum() == 2 and changed[int(pages[5, 0]), 14:16].all()


def test_pages_between_other_layers_pages(dev):
    """A pool of [n_pages, layers, ...] with one layer's pages apart, tables with a row stride, a transposed gate."""
    hq, hkv, d, page, T = 4, 2, 128, 32, 2
    lengths = [70, 33, 5]
    c = Cache(dev, 12, hkv, d, page, lengths, [T] * 3)
    n = c.k.shape[0]
    kk = torch.full((n, 3, hkv, page, d), float("nan"), dtype=BF16, device=dev)
    vv = torch.full((n, 3, hkv, d, page), float("nan"), dtype=BF16, device=dev)
    kk[:, 1], vv[:, 1] = c.k, c.vt
    wide = torch.full((3, c.width + 5), -1, dtype=I32, device=dev)
    wide[:, 2:2 + c.width] = c.pages
    pages = wide[:, 2:2 + c.width]
    g = torch.Generator().manual_seed(9)
    q = torch.randn((3 * T, hq, d), generator=g).to(BF16).to(dev)
    gate = torch.randn((hq, 3 * T, d), generator=g).to(BF16).to(dev).transpose(0, 1)
    ref = K.paged_attention(q, c.len_t(), c.pages, c.k, c.vt, 0.1, gate=gate.contiguous())
    assert torch.equal(_bits(K.paged_attention(q, c.len_t(), pages, kk[:, 1], vv[:, 1], 0.1, gate=gate)), _bits(ref))
    rows = torch.randn((3 * T, 8 * d), generator=g).to(BF16).to(dev)
    table = K.rope_table_dim(1e6, d, c.width * page, dev)
    args = (rows, hq, hkv, d, d, 4 * d, 6 * d, None, None, EPS, d, table, c.len_t())
    k0, v0 = kk.clone(), vv.clone()
    q1 = K.paged_store(*args, c.pages, c.k, c.vt)
    q2 = K.paged_store(*args, pages, kk[:, 1], vv[:, 1])
    assert torch.equal(_bits(q1), _bits(q2)) and torch.equal(_bits(kk[:, 1]), _bits(c.k)) and torch.equal(_bits(vv[:, 1]), _bits(c.vt))
    for layer in (0, 2):
        assert torch.equal(_bits(kk[:, layer]), _bits(k0[:, layer])) and torch.equal(_bits(vv[:, layer]), _bits(v0[:, layer]))


def test_pages_past_32_bits_of_elements(dev):
    """A pool of 2^32 keys' elements and more: the last pages are found."""
    hq, hkv, d, page = 2, 1, 256, 256
    n = (1 << 32) // (hkv * page * d) + 40
    k = torch.empty((n, hkv, page, d), dtype=BF16, device=dev)
    vt = torch.empty((n, hkv, d, page), dtype=BF16, device=dev)
    pages = _ints([[n - 1, 3, n - 2]], dev)
    small = _ints([[0, 1, 2]], dev)
    ks = torch.zeros((3, hkv, page, d), dtype=BF16, device=dev)
    vs = torch.zeros((3, hkv, d, page), dtype=BF16, device=dev)
    g = torch.Generator().manual_seed(10)
    table = K.rope_table_dim(1e7, 64, 3 * page, dev)
    rows = torch.randn((700, 4 * d), generator=g).to(BF16).to(dev)
    outs = []
    for p, kk, vv in ((pages, k, vt), (small, ks, vs)):
        q = K.paged_store(rows, hq, hkv, d, d, 2 * d, 3 * d, None, None, EPS, 64, table, _ints([0], dev), p, kk, vv)
        outs.append((q, K.paged_attention(q[-1:], _ints([699], dev), p, kk, vv, 0.06)))
    assert torch.equal(_bits(outs[0][0]), _bits(outs[1][0])) and torch.equal(_bits(outs[0][1]), _bits(outs[1][1]))
    assert torch.isfinite(outs[0][1]).all()


def test_long_cache(dev):
    """A sequence of 40000 tokens beside a short one, against 64 bits, in few heads."""
    hq, hkv, d = 2, 1, 128
    c = Cache(dev, 13, hkv, d, 256, [40000, 12], [1, 1])
    q = (2 * torch.randn((2, hq, d), generator=torch.Generator().manual_seed(11))).to(BF16)
    got = K.paged_attention(q.to(dev), c.len_t(), c.pages, c.k, c.vt, d ** -0.5).view(2, hq, d)
    for i, n in enumerate(c.lengths):
        out, err = _reference(q[i:i + 1], c.keys[i], c.vals[i], n, d ** -0.5)
        _check(got[i:i + 1], out, err, f"length {n}")


def test_captured_steps_follow_the_lengths(dev):
    """A step of store, attention and the lengths' advance, captured once and replayed with eager work between the replays:
    every replay has the bits of the eager steps. Two graphs that share a workspace replay in turn."""
    hq, hkv, d, page, T = 8, 2, 128, 16, 2
    lengths = [3, 250, 120]
    steps = 8
    g = torch.Generator().manual_seed(12)
    rows = torch.randn((steps, 3 * T, 12 * d), generator=g).to(BF16).to(dev)
    counts = _ints([2, 2, 1], dev)
    qn = (1 + 0.1 * torch.randn(d, generator=g)).to(BF16).to(dev)

    def fresh():
        c = Cache(dev, 14, hkv, d, page, lengths, [T * steps] * 3, fill=False)
        return c, c.len_t(), K.rope_table_dim(1e6, d, c.width * page, dev)

    def step(x, c, ln, table, ws):
        q = K.paged_store(x, hq, hkv, d, d, 8 * d, 10 * d, qn, None, EPS, d, table, ln, c.pages, c.k, c.vt, counts=counts)
        o = K.paged_attention(q, ln, c.pages, c.k, c.vt, d ** -0.5, counts=counts, workspace=ws)
        ln.add_(counts)
        return o

    ws = K.paged_attn_workspace(3, T, hq, hkv, d, (fresh()[0]).width * page, dev)
    c, ln, table = fresh()
    eager = [step(rows[i], c, ln, table, ws).clone() for i in range(steps)]
    sides = []
    for _ in range(2):
        c2, ln2, table2 = fresh()
        x = rows[0].clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = step(x, c2, ln2, table2, ws)
        sides.append((graph, x, o, c2, ln2, table2))
    for i in range(steps):
        for graph, x, o, c2, ln2, _ in sides:
            x.copy_(rows[i])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(_bits(o), _bits(eager[i])), i
            (torch.ones(1000, device=dev) * 2).sum()  # eager work between the replays
    for _, _, _, c2, ln2, _ in sides:
        assert torch.equal(ln2, ln)
        assert torch.equal(_bits(c2.k), _bits(c.k)) and torch.equal(_bits(c2.vt), _bits(c.vt))


def test_calls_on_two_streams_at_once(dev):
    """Calls that allocate their own workspaces may overlap."""
    hq, hkv, d = 8, 2, 128
    c = Cache(dev, 15, hkv, d, 64, [3000, 2900], [1, 1])
    q = torch.randn((2, hq, d), generator=torch.Generator().manual_seed(13)).to(BF16).to(dev)
    ref = K.paged_attention(q, c.len_t(), c.pages, c.k, c.vt, 0.1)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ln = c.len_t()
    torch.cuda.synchronize()
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(K.paged_attention(q, ln, c.pages, c.k, c.vt, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(_bits(o), _bits(ref)) for o in outs)


def test_wrappers_refuse(dev):
    hq, hkv, d, page = 4, 2, 64, 16
    k = torch.zeros((6, hkv, page, d), dtype=BF16, device=dev)
    vt = torch.zeros((6, hkv, d, page), dtype=BF16, device=dev)
    ln, pages = _ints([3, 4], dev), _ints([[0, 1], [2, 3]], dev)
    rows = torch.zeros((4, 8 * d), dtype=BF16, device=dev)
    table = K.rope_table_dim(1e4, d, 32, dev)
    q = torch.zeros((4, hq, d), dtype=BF16, device=dev)

    def store(match, **change):
        a = dict(qkv=rows, n_q=hq, n_kv=hkv, head_dim=d, q_stride=d, k_offset=4 * d, v_offset=6 * d, q_norm=None, k_norm=None,
                 eps=EPS, rotary_dim=d, table=table, lengths=ln, pages=pages, k_pages=k, vt_pages=vt)
        a.update(change)
        with pytest.raises(ValueError, match=match):
            K.paged_store(**a)

    def attend(match, **change):
        a = dict(q=q, lengths=ln, pages=pages, k_pages=k, vt_pages=vt, scale=1.0)
        a.update(change)
        with pytest.raises(ValueError, match=match):
            K.paged_attention(**a)

    for call in (store, attend):
        call("k_pages", k_pages=k.float())
        call("k_pages", k_pages=k[0])
        call("vt_pages", vt_pages=k)
        call("contiguous", k_pages=torch.zeros((6, page, hkv, d), dtype=BF16, device=dev).transpose(1, 2))
        call("lengths", lengths=ln.long())
        call("lengths", lengths=ln.cpu())
        call("counts", counts=ln[:1])
        call("pages must", pages=pages.long())
        call("pages must", pages=pages.t())
        call("do not divide", lengths=_ints([1, 2, 3], dev), pages=_ints([[0], [1], [2]], dev))
        call("page strides", k_pages=k[:1].expand(6, -1, -1, -1))
    store("have 1 of 64", n_kv=1, n_q=hq)
    store("do not fit", v_offset=6 * d + 1)
    store("do not fit", q_stride=63)
    store("table", table=table[:, :31])
    store("RoPE table", table=table[:31])
    store("table", rotary_dim=62)
    store("q_norm", q_norm=torch.ones(d + 1, dtype=BF16, device=dev))
    store("k_norm", k_norm=torch.ones(d, device=dev))
    store("out must", out=torch.zeros((4, hq, d), device=dev))
    store("qkv", qkv=rows.t())
    attend("q must", q=q.float())
    attend("q must", q=q[:, ::2])
    attend("has 128", q=torch.zeros((4, 2, 128), dtype=BF16, device=dev))
    attend("multiple of Hkv", q=torch.zeros((4, 3, d), dtype=BF16, device=dev))
    attend("query rows", q=torch.zeros((2 * 33, hq, d), dtype=BF16, device=dev))
    attend("gate", gate=q[:2])
    attend("keys=33", keys=33)
    attend("keys=0", keys=0)
    attend("out must", out=q)
    big = torch.full((2, 20), 0, dtype=I32, device=dev)
    attend("workspace", pages=big, workspace=torch.zeros(8, device=dev))


def _layers(model, x, ln, pages, pools, table, counts, T):
    """The dense decoder's layers over B sequences' rows, from its own modules and the paged calls."""
    a = model.args
    h = x
    for layer, (k, vt) in zip(model.layers, pools):
        at = layer.self_attn
        y = K.rmsnorm(h, layer.input_layernorm, a.rms_norm_eps)
        qkv = torch.cat([at.q_proj(y), at.k_proj(y), at.v_proj(y)], -1)
        hq, hkv, d = a.num_attention_heads, a.num_key_value_heads, a.head_dim
        q = K.paged_store(qkv, hq, hkv, d, d, hq * d, (hq + hkv) * d, at.q_norm, at.k_norm, a.rms_norm_eps, d, table, ln, pages,
                          k, vt, counts=counts)
        o = K.paged_attention(q, ln, pages, k, vt, d ** -0.5, counts=counts)
        h = h + at.o_proj(o)
        y = K.rmsnorm(h, layer.post_attention_layernorm, a.rms_norm_eps)
        gu = torch.cat([layer.mlp.gate_proj(y), layer.mlp.up_proj(y)], -1)
        h = h + layer.mlp.down_proj(K.silu_mul(gu))
    return K.rmsnorm(h, model.norm, a.rms_norm_eps)


def test_a_batch_decodes_and_scores_as_its_sequences_do(dev):
    """The operators together on the small dense decoder: three prompts of different lengths fed in steps of up to 8 tokens, then
    decoded greedily with every answer's log-probability. The same as each sequence alone, bit for bit, in tokens and in
    numbers; and the scores of the last step are the model's own over its contiguous cache, as near as its oracle tests ask."""
    from skinny_mlx.cache import make_prompt_cache
    from skinny_mlx.model import build_model
    from skinny_mlx.patch import patch_model
    from skinny_mlx.spec import forward

    model = build_model("tiny-dense", device=dev)
    patch_model(model, fuse=False)
    a = model.args
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, a.vocab_size, n).tolist() for n in (5, 70, 23)]
    page, width = 16, 8

    def serve(ids, T):
        b = len(ids)
        pools = [(torch.full((b * width, a.num_key_value_heads, page, a.head_dim), float("nan"), dtype=BF16, device=dev),
                  torch.full((b * width, a.num_key_value_heads, a.head_dim, page), float("nan"), dtype=BF16, device=dev))
                 for _ in model.layers]
        pages = torch.arange(b * width, dtype=I32, device=dev).view(width, b).t().contiguous()
        ln = torch.zeros(b, dtype=I32, device=dev)
        table = K.rope_table_dim(a.rope_theta, a.head_dim, width * page, dev)
        left = [list(p) for p in ids]
        last = torch.zeros((b, a.hidden_size), dtype=BF16, device=dev)
        while any(left):
            take = [p[:T] for p in left]
            counts = _ints([len(p) for p in take], dev)
            rows = _ints([p + [0] * (T - len(p)) for p in take], dev).view(-1)
            h = _layers(model, K.embed(rows, model.embed_tokens), ln, pages, pools, table, counts, T).view(b, T, -1)
            for i, p in enumerate(take):
                if p:
                    last[i] = h[i, len(p) - 1]
            ln += counts
            left = [p[T:] for p in left]
        out = []
        for _ in range(10):
            logits = model.lm_head(last)
            tok = K.argmax_rows(logits)
            lp, ent, ids_, alt = K.token_logprobs(logits, tok, 3)
            out.append((tok.clone(), lp.clone(), ent, ids_, alt, logits))
            last = _layers(model, K.embed(tok, model.embed_tokens), ln, pages, pools, table, None, 1)
            ln += 1
        return out

    together = serve(prompts, 8)
    for i, p in enumerate(prompts):
        for T in (8, 1):
            alone = serve([p], T)
            for s, (x, y) in enumerate(zip(together, alone)):
                for n in range(5):
                    assert torch.equal(x[n][i], y[n][0]), (i, T, s, n)
        for tok, lp, ent, ids_, alt, logits in together:
            assert ids_[i, 0] == tok[i] and alt[i, 0] == lp[i] and lp[i] < 0 and ent[i] > 0
        # the model's own pass over the prompt and the tokens answered
        answered = [int(x[0][i]) for x in together]
        _, own = forward(model, p + answered[:-1], make_prompt_cache(model))
        ref = own[len(p) - 1:].float()
        got = torch.stack([x[5][i] for x in together]).float()
        assert (got - ref).norm() <= 2e-2 * ref.norm()


def _runs(c, b, T, hq, keys):
    """Blocks per workgroup and whether a merge follows, from the workspace's size."""
    n = K.paged_attn_workspace(b, T, hq, c.hkv, c.d, keys, c.dev).numel()
    nblk = -(-keys // (64 if c.d == 256 else 128))
    slots = n // (b * T * hq * (c.d + 2) * 4)
    return nblk if slots == 0 else next(s for s in (1, 4, 8) if -(-nblk // s) == slots)


@pytest.mark.parametrize("d,G,T,b", [(64, 1, 1, 3), (64, 2, 16, 40), (128, 4, 1, 3), (128, 4, 4, 40), (128, 4, 8, 20), (128, 4, 16, 9),
                                     (256, 4, 1, 5), (256, 4, 5, 30), (256, 3, 16, 12)])
def test_bits_do_not_depend_on_how_the_keys_are_cut(dev, d, G, T, b):
    """The host's bound decides how many blocks a workgroup takes and who joins them; the rows keep their bits, alone too."""
    hkv = 2
    hq = hkv * G
    pattern = [2300, 0, 1025, 513, 64, 1100, 2047 - T, 7, 300, 1536]
    lengths = [pattern[i % 10] for i in range(b)]
    counts = [T - (i % 3 if T > 2 else 0) for i in range(b)]
    c = Cache(dev, d + T, hkv, d, 32, lengths, counts, width=(1 << 18) // 32)
    q = torch.randn((b * T, hq, d), generator=torch.Generator().manual_seed(20)).to(BF16).to(dev)
    ln, cn = c.len_t(), _ints(counts, dev)
    seen, ref = set(), None
    for keys in (2400, 1 << 14, 1 << 15, 1 << 16, 1 << 18):
        seen.add(_runs(c, b, T, hq, keys))
        got = K.paged_attention(q, ln, c.pages, c.k, c.vt, d ** -0.5, counts=cn, keys=keys)
        ref = got if ref is None else ref
        assert torch.isfinite(got).all() and torch.equal(_bits(got), _bits(ref)), keys
    assert 8 in seen and len(seen) > 1
    for i in sorted({0, 2, b // 2, b - 1}):
        seen.add(_runs(c, 1, T, hq, 2400))
        for t in sorted({0, counts[i] - 1}):  # one token at a time, the others before it in the cache
            one = K.paged_attention(q[i * T + t:i * T + t + 1], ln[i:i + 1] + t, c.pages[i:i + 1], c.k, c.vt, d ** -0.5, keys=2400)
            assert torch.equal(_bits(one[0]), _bits(ref[i * T + t])), (i, t)
    assert 1 in seen or 4 in seen


@pytest.mark.parametrize("hkv,d,b,keys", [(64, 64, 4, 1000), (32, 256, 8, 500), (32, 128, 4, 400)])
def test_sequences_of_one_part(dev, hkv, d, b, keys):
    """Enough heads that a workgroup takes a whole sequence and writes its rows itself."""
    lengths = [keys - 2, 0, keys // 2, 130, 63, keys - 70, 300, 1][:b]
    counts = [2, 1, 2, 0, 2, 1, 2, 2][:b]
    c = Cache(dev, d, hkv, d, 16, lengths, counts)
    assert _runs(c, b, 2, hkv, keys) > 1 and _runs(c, 1, 2, hkv, keys) == 1
    q = torch.randn((2 * b, hkv, d), generator=torch.Generator().manual_seed(21)).to(BF16).to(dev)
    ln, cn = c.len_t(), _ints(counts, dev)
    got = K.paged_attention(q, ln, c.pages, c.k, c.vt, d ** -0.5, counts=cn, keys=keys).view(b, 2, -1)
    for i in range(b):
        one = K.paged_attention(q[2 * i:2 * i + 2], ln[i:i + 1], c.pages[i:i + 1], c.k, c.vt, d ** -0.5, counts=cn[i:i + 1], keys=keys)
        assert torch.equal(_bits(got[i]), _bits(one)) and (got[i, counts[i]:] == 0).all(), i


def test_sequences_that_share_pages(dev):
    """A prefix held once: the same pages in several rows of the table, each sequence's last page its own."""
    hq, hkv, d, page = 8, 2, 128, 32
    c = Cache(dev, 30, hkv, d, page, [200, 200, 200], [1, 1, 1])
    pages = c.pages.clone()
    pages[1:, :6] = pages[0, :6]  # 192 tokens of the first sequence
    k, vt = c.k.clone(), c.vt.clone()
    for i in (1, 2):
        for p in range(6):
            k[c.pages[i, p]], vt[c.pages[i, p]] = c.k[c.pages[0, p]], c.vt[c.pages[0, p]]
    q = torch.randn((3, hq, d), generator=torch.Generator().manual_seed(22)).to(BF16).to(dev)
    ref = K.paged_attention(q, c.len_t(), c.pages, k, vt, d ** -0.5)
    assert torch.equal(_bits(K.paged_attention(q, c.len_t(), pages, c.k, c.vt, d ** -0.5)), _bits(ref))


def test_the_most_sequences(dev):
    """65535 of them, none with a cache: a row's output is its own value."""
    b, d = 65535, 64
    k = torch.empty((b, 1, 16, d), dtype=BF16, device=dev)
    vt = torch.empty((b, 1, d, 16), dtype=BF16, device=dev)
    ln = torch.zeros(b, dtype=I32, device=dev)
    pages = torch.arange(b - 1, -1, -1, dtype=I32, device=dev).view(b, 1)
    rows = torch.randn((b, 4 * d), device=dev, generator=torch.Generator(dev).manual_seed(23)).to(BF16)
    q = K.paged_store(rows, 2, 1, d, d, 2 * d, 3 * d, None, None, EPS, d, K.rope_table_dim(1e4, d, 16, dev), ln, pages, k, vt)
    assert torch.equal(_bits(q), _bits(rows[:, :2 * d].reshape(b, 2, d)))  # position 0: cos 1, sin 0
    got = K.paged_attention(q, ln, pages, k, vt, d ** -0.5).view(b, 2, d)
    assert torch.equal(_bits(got), _bits(rows[:, None, 3 * d:].expand(-1, 2, -1)))


def test_the_most_tokens_at_once(dev):
    """65535 new tokens stored in one call: the bits of storing them in pieces."""
    T, d, page = 65535, 64, 16
    rows = torch.randn((T, 4 * d), device=dev, generator=torch.Generator(dev).manual_seed(24)).to(BF16)
    w = -(-(T + 5) // page)
    pages = torch.randperm(w, device=dev, generator=torch.Generator(dev).manual_seed(25)).to(I32).view(1, w)
    table = K.rope_table_dim(1e6, d, w * page, dev)
    outs = []
    for step in (T, 9001):
        k = torch.zeros((w, 1, page, d), dtype=BF16, device=dev)
        vt = torch.zeros((w, 1, d, page), dtype=BF16, device=dev)
        q = [K.paged_store(rows[i:i + step], 2, 1, d, d, 2 * d, 3 * d, None, None, EPS, d, table, _ints([5 + i], dev), pages, k, vt)
             for i in range(0, T, step)]
        outs.append((torch.cat(q), k, vt))
    assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip(*outs))


def test_calls_on_another_stream(dev):
    """Each call runs on the current stream: a store and an attention behind a slow write of their rows on a side stream."""
    hq, hkv, d = 8, 2, 128
    c = Cache(dev, 31, hkv, d, 64, [300, 5], [1, 1], fill=False)
    rows = torch.randn((2, 12 * d), generator=torch.Generator().manual_seed(26)).to(BF16).to(dev)
    table = K.rope_table_dim(1e6, d, c.width * 64, dev)
    ln = c.len_t()

    def step(x, k, vt):
        q = K.paged_store(x, hq, hkv, d, d, 8 * d, 10 * d, None, None, EPS, d, table, ln, c.pages, k, vt)
        return K.paged_attention(q, ln, c.pages, k, vt, d ** -0.5)

    ref = step(rows, c.k.clone(), c.vt.clone())
    x, k, vt = torch.zeros_like(rows), c.k.clone(), c.vt.clone()
    busy = torch.randn((4096, 4096), device=dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(8):
            busy = busy @ busy * 1e-2
        x.copy_(rows)
        got = step(x, k, vt)
    torch.cuda.synchronize()
    assert torch.equal(_bits(got), _bits(ref))


def test_scale_must_be_positive(dev):
    c = Cache(dev, 32, 1, 64, 16, [3], [1])
    q = torch.zeros((1, 1, 64), dtype=BF16, device=dev)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            K.paged_attention(q, c.len_t(), c.pages, c.k, c.vt, scale)
