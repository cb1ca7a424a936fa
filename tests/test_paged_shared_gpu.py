"""Attention behind a shared prefix (csrc/paged_shared.hip) against a plain implementation in 64 bits, and what it promises beyond.

Tolerances are counted. The prefix's weights are rounded to bf16, 2^-8 of each at most, and divided by the sum of the rounded
ones: sum |w| |v - out| 2^-8 of an output; the rest as for paged_attention: scores of d products in fp32, weights of two bf16
terms for the own keys, fp32 sums; the output's own rounding, half a bf16 step."""

import numpy as np
import pytest
import torch

from skinny_mlx import kernels as K

pytestmark = pytest.mark.gpu

BF16, I32 = torch.bfloat16, torch.int32
HALF, U = 2.0 ** -8, 2.0 ** -24
NAN = float("nan")


def _ints(v, dev):
    return torch.tensor(v, dtype=I32, device=dev)


def _bits(t):
    return t.contiguous().view(torch.int16)


class Shared:
    """A prefix and sequences after it in one pool, pages dealt in no order; slots without a token hold NaN and infinities."""

    def __init__(self, dev, seed, hq, hkv, d, page, prefix, lengths, T, counts=None, spare=2):
        rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        counts = [T] * len(lengths) if counts is None else counts
        self.dev, self.d, self.hq, self.T, self.prefix, self.lengths, self.counts = dev, d, hq, T, prefix, lengths, counts
        need = [-(-(n + c) // page) for n, c in zip(lengths, counts)]
        front = max(-(-prefix // page), 1)
        total = front + sum(need) + spare
        order = rng.permutation(total)
        table = np.full((len(lengths), max(max(need), 1)), -5, dtype=np.int32)
        k = torch.full((total, hkv, page, d), NAN, dtype=BF16)
        vt = torch.full((total, hkv, d, page), float("inf"), dtype=BF16)
        at = front
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n

        def fill(pages, n):
            kk, vv = torch.randn((n, hkv, d), generator=g).to(BF16), torch.randn((n, hkv, d), generator=g).to(BF16)
            for j in range(0, n, page):
                m = min(page, n - j)
                k[pages[j // page], :, :m] = kk[j:j + m].transpose(0, 1)
                vt[pages[j // page], :, :, :m] = vv[j:j + m].permute(1, 2, 0)
            return kk, vv

        self.front = order[:front].astype(np.int32)
        self.pk, self.pv = fill(self.front, prefix)
        self.own = [fill(table[i], n + c) for i, (n, c) in enumerate(zip(lengths, counts))]
        self.k, self.vt = k.to(dev), vt.to(dev)
        self.pages, self.front_pages = torch.tensor(table, device=dev), torch.tensor(self.front, device=dev)
        self.q = (1.5 * torch.randn((len(lengths) * T, hq, d), generator=g)).to(BF16)
        self.gate = torch.randn((len(lengths) * T, hq, 2, d), generator=g).to(BF16).to(dev)[:, :, 1]

    def run(self, gate=None, **kw):
        for name, of in (("counts", self.counts), ("lengths", self.lengths), ("prefix", [self.prefix])):
            if name not in kw:
                kw[name] = _ints(of, self.dev)
        q = kw.pop("q") if "q" in kw else self.q.to(self.dev)
        at = [kw.pop(name, own) for name, own in (("front", self.front_pages), ("lengths", None), ("pages", self.pages),
                                                  ("k", self.k), ("vt", self.vt))]
        return K.paged_attention_shared(q, kw.pop("prefix"), *at, self.d ** -0.5, gate=gate, **kw)

    def check(self, got, gate=None, rows=None):
        b, T, hq, d = len(self.lengths), self.T, self.hq, self.d
        got = got.view(b, T, hq, d)
        for i in range(b) if rows is None else rows:
            n, c = self.lengths[i], self.counts[i]
            assert (got[i, c:] == 0).all()
            if not c:
                continue
            out, err = self._reference(i, gate)
            diff = (got[i, :c].double().cpu() - out).abs()
            worst = (diff / (HALF * (out.abs() + err) + err)).max().item()
            assert torch.isfinite(got[i, :c]).all() and worst <= 1, f"sequence {i}: {worst:.3f} of the bound"

    def _reference(self, i, gate):
        n, c, d, hq = self.lengths[i], self.counts[i], self.d, self.hq
        keys, vals = (torch.cat([p, o]).double() for p, o in zip((self.pk, self.pv), self.own[i]))
        hkv = keys.shape[1]
        rep = hq // hkv
        q = self.q.view(-1, self.T, hq, d)[i, :c].double()
        total = self.prefix + n + c
        out = torch.zeros((c, hq, d), dtype=torch.float64)
        err = torch.zeros_like(out)
        seen = torch.arange(total) <= self.prefix + n + torch.arange(c)[:, None]
        first = (torch.arange(total) < self.prefix).double()
        for h in range(hq):
            kh, vh = keys[:, h // rep], vals[:, h // rep]
            s = torch.where(seen, q[:, h] @ kh.t() * d ** -0.5, -torch.inf)
            w = torch.softmax(s, -1)
            o = w @ vh
            ds = (q[:, h].abs() @ kh.abs().t()).amax(-1, keepdim=True) * d ** -0.5 * (d + 4) * U
            rel = 2 * ds + 2.0 ** -16 + 2 * (total + 64) * U
            wp = w * first
            # sum of w |v - out| by Cauchy: sqrt(sum w) sqrt(sum w (v - out)^2)
            spread = (wp @ vh ** 2 - 2 * o * (wp @ vh) + wp.sum(-1, keepdim=True) * o ** 2).clamp(min=0)
            out[:, h] = o
            err[:, h] = rel * (w @ vh.abs()) + 1.01 * HALF * (wp.sum(-1, keepdim=True) * spread).sqrt()
        if gate is not None:
            sg = torch.sigmoid(gate.view(-1, self.T, hq, d)[i, :c].double().cpu())
            out, err = out * sg, err * sg + (out * sg).abs() * 8 * U
        return out, err


LAYOUTS = [(4, 1, 128), (16, 4, 128), (16, 4, 256), (8, 8, 64), (6, 2, 64), (64, 1, 128), (12, 4, 256)]


@pytest.mark.parametrize("hq,hkv,d", LAYOUTS)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_single_tokens(dev, hq, hkv, d, page):
    lengths = [0, 1, 15, 16, 40, 127, 128, 300, 63]
    s = Shared(dev, hq + page, hq, hkv, d, page, 333, lengths, 1)
    s.check(s.run())


@pytest.mark.parametrize("prefix", [0, 1, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 200, 256, 1000, 2049])
@pytest.mark.parametrize("d,page", [(128, 16), (256, 32), (64, 64)])
def test_prefixes(dev, prefix, d, page):
    """Every end of a prefix inside a page, a tile and a run, and none at all; with the tight bound and a loose one."""
    s = Shared(dev, prefix + d, 4, 2, d, page, prefix, [0, 5, 77], 2, counts=[2, 1, 2])
    s.check(s.run(prefix_keys=max(prefix, 1)))
    s.check(s.run())


@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 128), (8, 4, 64), (8, 2, 256)])
@pytest.mark.parametrize("batch", [1, 2, 4, 7, 8, 16, 31, 33, 64, 65, 100])
def test_batches(dev, hq, hkv, d, batch):
    """One to 400 query rows per kv head: every form of the prefix's kernel, full and with rows to spare."""
    rng = np.random.default_rng(batch)
    lengths = [int(n) for n in rng.integers(0, 50, batch)]
    s = Shared(dev, batch + d, hq, hkv, d, 32, 517, lengths, 1)
    s.check(s.run(), rows=range(0, batch, max(1, batch // 7)))


@pytest.mark.parametrize("hq,hkv,d,T", [(4, 1, 128, 3), (32, 8, 128, 8), (16, 4, 256, 4), (16, 4, 256, 16), (4, 4, 64, 64), (6, 2, 128, 7)])
@pytest.mark.parametrize("gated", [False, True])
def test_several_tokens(dev, hq, hkv, d, T, gated):
    lengths = [0, 60, 250, 125, 63, 7]
    counts = [T, T, max(1, T - 2), 1, 0, T - 1]
    s = Shared(dev, T + d, hq, hkv, d, 32, 401, lengths, T, counts)
    gate = s.gate if gated else None
    s.check(s.run(gate), gate)


def test_many_sequences(dev):
    """More blocks of rows than CUs; more own runs than rows of a workgroup's waves."""
    rng = np.random.default_rng(5)
    s = Shared(dev, 16, 4, 1, 64, 16, 33, [int(n) for n in rng.integers(0, 20, 1500)], 1)
    s.check(s.run(), rows=(0, 1, 700, 1498, 1499))
    s = Shared(dev, 17, 8, 8, 128, 32, 150, [int(n) for n in rng.integers(0, 90, 500)], 3)
    s.check(s.run(), rows=(0, 255, 499))


def test_a_prefix_of_many_runs(dev):
    s = Shared(dev, 3, 4, 2, 128, 256, 40001, [3, 900], 1)
    s.check(s.run())
    s = Shared(dev, 4, 8, 1, 256, 64, 20000, [3, 90] * 20, 1)
    s.check(s.run(), rows=(0, 19, 39))


def test_peaked_and_flat_scores(dev):
    """One key far above the rest, in the prefix or among the own keys; scores that rise along the prefix, so that the maximum
    moves; all scores alike; all -inf but the own."""
    for kind in ("prefix", "own", "rising", "flat"):
        s = Shared(dev, 5, 4, 1, 128, 64, 700, [100, 3], 1)
        q0 = s.q[0, 0].float()
        if kind == "prefix":
            s.pk[333, 0] = (q0 * 4).to(BF16)
        elif kind == "own":
            s.own[0][0][50, 0] = (q0 * 4).to(BF16)
        elif kind == "rising":
            s.pk[:, 0] = (q0 * torch.linspace(-3, 3, 700)[:, None]).to(BF16)
        else:
            s.pk[:] = 0
        k = s.k.clone()
        for i in range(700):
            k[s.front[i // 64], :, i % 64] = s.pk[i].to(dev)
        for i in range(101):
            k[int(s.pages[0, i // 64]), :, i % 64] = s.own[0][0][i].to(dev)
        s.check(s.run(k=k))


def test_rows_are_those_of_one_long_cache(dev):
    """The prefix's pages listed in front of each sequence's own are the same attention by paged_attention."""
    s = Shared(dev, 6, 8, 2, 128, 64, 640, [10, 200, 0], 2)
    got = s.run().float()
    table = torch.cat([s.front_pages.expand(3, -1), s.pages], 1)
    ref = K.paged_attention(s.q.to(dev), _ints([640 + n for n in s.lengths], dev), table, s.k, s.vt, 128 ** -0.5).float()
    s.check(got.to(BF16))
    s.check(ref.to(BF16))


def test_values_that_are_no_numbers(dev):
    """A value that is not finite makes its dim NaN in every row (the prefix is everyone's), a key of NaN the rows of its kv
    head, and an infinite score likewise; the other kv heads keep their bits."""
    s = Shared(dev, 7, 8, 2, 128, 32, 300, [5, 40], 1)
    clean = s.run().view(2, 2, 4, 128)
    for bad in (NAN, float("inf"), -float("inf")):
        vt = s.vt.clone()
        vt[s.front[100 // 32], 0, 9, 100 % 32] = bad
        y = s.run(vt=vt).view(2, 2, 4, 128)
        assert torch.isnan(y[:, 0, :, 9]).all() and torch.equal(_bits(y[:, 1]), _bits(clean[:, 1]))
        rest = [d for d in range(128) if d != 9]
        assert torch.equal(_bits(y[:, 0][..., rest]), _bits(clean[:, 0][..., rest]))
    k = s.k.clone()
    k[s.front[3], 1, 2, 5] = NAN
    y = s.run(k=k).view(2, 2, 4, 128)
    assert torch.isnan(y[:, 1]).all() and torch.equal(_bits(y[:, 0]), _bits(clean[:, 0]))
    k[s.front[3], 1, 2, 5] = float("inf")  # scores of +inf and of -inf, by the sign of the query's dim
    y = s.run(k=k).view(2, 2, 4, 128)
    up = s.q.view(2, 2, 4, 128)[:, 1, :, 5] > 0
    assert torch.isnan(y[:, 1].cpu()[up]).all() and torch.isfinite(y[:, 1].cpu()[~up]).all()
    own = s.vt.clone()  # in one sequence's own keys: its rows alone
    own[int(s.pages[1, 0]), 0, 3, 4] = NAN
    y = s.run(vt=own).view(2, 2, 4, 128)
    assert torch.isnan(y[1, 0, :, 3]).all() and torch.equal(_bits(y[0]), _bits(clean[0]))


@pytest.mark.parametrize("hq,hkv,d,page", [(8, 2, 128, 32), (16, 4, 256, 16), (4, 4, 64, 64), (4, 1, 128, 256)])
def test_new_tokens_that_are_no_numbers(dev, hq, hkv, d, page):
    """A new token's value or key that is not finite reaches its own row and the later ones; the rows before it, and the other
    sequences, keep their bits. At every place of a step of 32 keys."""
    T, lengths = 5, [0, 27, 61, 300, 1023]
    s = Shared(dev, 14, hq, hkv, d, page, 150, lengths, T)
    clean = _bits(s.run().view(5, T, hq, d))
    rep = hq // hkv
    for i, n in enumerate(lengths):
        for at, bad in ((1, NAN), (T - 1, float("inf")), (3, -float("inf"))):
            where = int(s.pages[i, (n + at) // page]), (n + at) % page
            vt = s.vt.clone()
            vt[where[0], 0, 7, where[1]] = bad
            y = s.run(vt=vt).view(5, T, hq, d)
            hit = torch.zeros((5, T, hq, d), dtype=torch.bool, device=dev)
            hit[i, at:, :rep, 7] = True
            assert not torch.isfinite(y[hit]).any() and torch.equal(_bits(y)[~hit], clean[~hit])
            k = s.k.clone()
            k[where[0], hkv - 1, where[1], 3] = NAN
            y = s.run(k=k).view(5, T, hq, d)
            hit[:] = False
            hit[i, at:, hq - rep:] = True
            assert torch.isnan(y[hit]).all() and torch.equal(_bits(y)[~hit], clean[~hit])


@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 128), (16, 4, 256), (2, 2, 64)])
def test_own_keys_of_many_runs(dev, hq, hkv, d):
    """Own caches far longer than the prefix, their ends at and beside a run's, with a bound on the keys that is far too loose."""
    lengths = [5000, 63, 64, 2047, 2048, 0]
    s = Shared(dev, 15, hq, hkv, d, 64, 40, lengths, 2, counts=[2, 2, 1, 1, 2, 0])
    s.check(s.run())
    wide = torch.full((6, 4096), -7, dtype=I32, device=dev)
    wide[:, :s.pages.shape[1]] = s.pages
    s.check(s.run(pages=wide))


def test_what_cannot_be_is_nan_and_reads_nothing(dev):
    s = Shared(dev, 8, 8, 2, 128, 32, 300, [5, 40, 9], 2)
    clean = s.run()
    for prefix in (-1, 320 + 1, 2 ** 31 - 1):
        assert torch.isnan(s.run(prefix=_ints([prefix], dev))).all()
    assert torch.isnan(s.run(prefix_keys=299)).all()
    for bad in (-1, s.k.shape[0], 2 ** 31 - 1):
        front = s.front_pages.clone()
        front[4] = bad
        assert torch.isnan(s.run(front=front)).all()
        wide = torch.cat([s.front_pages, _ints([bad, bad], dev)])  # not needed: may hold anything
        assert torch.equal(_bits(s.run(front=wide, prefix_keys=300)), _bits(s.run(front=s.front_pages, prefix_keys=300)))
        pages = s.pages.clone()
        pages[1, 1] = bad
        y = s.run(pages=pages).view(3, 2, -1)
        assert torch.isnan(y[1]).all() and torch.equal(_bits(y[[0, 2]]), _bits(clean.view(3, 2, -1)[[0, 2]]))
    y = s.run(lengths=_ints([5, -2, 9], dev), counts=_ints([2, 2, 3], dev)).view(3, 2, -1)
    assert torch.isnan(y[1:]).all() and torch.equal(_bits(y[0]), _bits(clean.view(3, 2, -1)[0]))
    assert (s.run(counts=_ints([0, 0, 0], dev)) == 0).all()


def test_pages_past_32_bits_of_elements(dev):
    hq, hkv, d, page = 2, 1, 256, 256
    n = (1 << 32) // (hkv * page * d) + 40
    s = Shared(dev, 9, hq, hkv, d, page, 300, [20], 1)
    k = torch.empty((n, hkv, page, d), dtype=BF16, device=dev)
    vt = torch.empty((n, hkv, d, page), dtype=BF16, device=dev)
    far = lambda t: torch.where(t >= 0, n - 1 - t, t)  # noqa: E731
    for i in range(s.k.shape[0]):
        k[n - 1 - i], vt[n - 1 - i] = s.k[i], s.vt[i]
    ref = s.run()
    assert torch.equal(_bits(s.run(k=k, vt=vt, front=far(s.front_pages), pages=far(s.pages))), _bits(ref))


def test_captured_steps_and_a_shared_workspace(dev):
    """Captured with loose bounds and replayed while the prefix, the lengths and the counts change, with eager work between; a
    second graph with the same workspace replays in turn. Every replay has the eager call's bits."""
    s = Shared(dev, 10, 8, 2, 128, 32, 900, [5, 40, 90], 2)
    ws = K.paged_attn_shared_workspace(3, 2, 8, 2, 128, 928, 96, dev)
    q = s.q.to(dev)
    prefix, lengths, counts = _ints([900], dev), _ints(s.lengths, dev), _ints(s.counts, dev)
    kw = dict(prefix=prefix, lengths=lengths, counts=counts, prefix_keys=928, keys=96)
    graphs = []
    for scale in (1.0, 0.5):
        qs = (q.float() * scale).to(BF16)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.run(q=qs, workspace=ws, **kw)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = s.run(q=qs, workspace=ws, **kw)
        graphs.append((graph, y, qs))
    for i in range(5):
        prefix.fill_([900, 1, 0, 33, 899][i])
        lengths.copy_(_ints([5 - i, 40 + i, 90 - 2 * i], dev))
        counts.copy_(_ints([2, i % 3, 1], dev))
        for graph, y, qs in graphs:
            graph.replay()
            ref = s.run(q=qs, **kw)
            torch.cuda.synchronize()
            assert torch.equal(_bits(y), _bits(ref))


def test_strides_streams_and_outputs(dev):
    """One layer's pages of a pool of several, a table with a row stride, a gate with odd strides, an output given, another
    stream: the same bits."""
    s = Shared(dev, 11, 4, 2, 128, 32, 130, [70, 33, 5], 2)
    ref = s.run(s.gate)
    n = s.k.shape[0]
    kk = torch.full((n, 3, *s.k.shape[1:]), NAN, dtype=BF16, device=dev)
    vv = torch.full((n, 3, *s.vt.shape[1:]), NAN, dtype=BF16, device=dev)
    kk[:, 1], vv[:, 1] = s.k, s.vt
    wide = torch.full((3, s.pages.shape[1] + 5), -1, dtype=I32, device=dev)
    wide[:, 2:2 + s.pages.shape[1]] = s.pages
    gate = s.gate.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.full_like(ref, NAN)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y = s.run(gate, k=kk[:, 1], vt=vv[:, 1], pages=wide[:, 2:2 + s.pages.shape[1]], out=out)
    torch.cuda.synchronize()
    assert y is out and torch.equal(_bits(y), _bits(ref))


def test_refusals(dev):
    s = Shared(dev, 12, 8, 2, 128, 32, 100, [7, 3], 2)
    q = s.q.to(dev)
    for change in (dict(q=q.float()), dict(q=q[:3]), dict(q=q[:, :, :64]), dict(q=q.transpose(0, 1)), dict(prefix=_ints([1, 2], dev)),
                   dict(prefix=_ints([100], "cpu")), dict(prefix=torch.tensor([100], device=dev)), dict(front=s.front_pages[:0]),
                   dict(front=s.front_pages.long()), dict(front=s.front_pages.cpu()), dict(front=s.front_pages[None]),
                   dict(lengths=_ints([7], dev)), dict(pages=s.pages.long()), dict(k=s.k[:, :1]), dict(vt=s.vt.float()),
                   dict(counts=_ints([1], dev)), dict(keys=0), dict(keys=33), dict(prefix_keys=0), dict(prefix_keys=129),
                   dict(out=torch.empty((4, 1024), device=dev)), dict(workspace=torch.empty(64, dtype=torch.uint8, device=dev)),
                   dict(workspace=torch.empty(1 << 20, dtype=torch.uint8)), dict(gate=s.gate[:, :7])):
        with pytest.raises(ValueError):
            s.run(**change)
    wide = torch.zeros((2 * 17, 8, 128), dtype=BF16, device=dev)
    with pytest.raises(ValueError):
        s.run(q=wide)
