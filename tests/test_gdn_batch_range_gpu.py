"""The Gated-DeltaNet recurrence of several sequences in chunks (csrc/gdn_batch.hip): each form of its kernel over many chunks, values
and states whose size changes from token to token, and values that are no numbers, against the rule in 64 bits."""

import pytest
import torch

from test_gdn_batch_gpu import D, NAN, Mixer, _ints, _same

pytestmark = pytest.mark.gpu

# Value heads, key heads, sequences: 4, 40, 96 and 160 heads in all, one for each form, of 16, 32, 64 and 128 columns a workgroup.
FORMS = [(2, 1, 2), (8, 4, 5), (16, 8, 6), (32, 16, 5)]


def _rule(m, i, state, heads=None):
    """The rule in 64 bits over sequence i and `heads` (None: all) from `state` [H, Dv, Dk] -> y, the last state, and how far y, and
    a column of the state (2-norm over the key dims), may be off.

    The error of a column is carried on by the tokens' decay and (I - beta k k^T), which lengthen nothing, and each token adds its
    own, of its present sizes alone: 128 products in fp32, k.S, of the decayed state; 32 of a chunk's corrections, in the system's
    inverse and again where it is applied: 2^-17 of the correction's parts, beta (|v| + decay |S|), of this token and of the chunk's
    earlier ones as far as the decays have left them; unit vectors, gates and what is rounded on the way, as much again: 2^-16. A
    decay's logarithm is a product of two exponentials' results, 2^-21 of it: so much of the decayed state. y: 128 products in fp32
    and the query's own rounding, 2^-16 of |q| |S|."""
    n, T = m.counts[i], m.T
    heads = range(m.heads) if heads is None else heads
    x = m.qkv.view(-1, T, 2 * m.key_heads + m.heads, D)[i, :n].double().cpu()
    rep = m.heads // m.key_heads
    unit = lambda h: h / torch.sqrt((h * h).sum(-1, keepdim=True) + 1e-6)  # noqa: E731
    hs = torch.tensor(list(heads))
    q, k = unit(x[:, hs // rep]) * D ** -0.5, unit(x[:, m.key_heads + hs // rep])
    v = x[:, 2 * m.key_heads + hs]
    a = (m.a.view(-1, T, m.heads)[i, :n].double().cpu() + m.dt.double().cpu())[:, hs]
    log_decay = -m.a_log.double().cpu().exp()[hs] * torch.nn.functional.softplus(a, threshold=40)
    decay, beta = torch.exp(log_decay), torch.sigmoid(m.b.reshape(-1, T, m.heads)[i, :n].double().cpu()[:, hs])
    s = state.double().cpu()[hs].clone()
    y = torch.zeros((n, len(hs), D), dtype=torch.float64)
    yerr, err, recent = torch.zeros_like(y), torch.zeros_like(y[0]), torch.zeros_like(y[0])
    for t in range(n):
        g, b = decay[t, :, None], beta[t, :, None]
        s = s * g[..., None]
        left = s.norm(dim=-1)
        delta = b * (v[t] - (s @ k[t][..., None])[..., 0])
        s = s + delta[..., None] * k[t][:, None]
        y[t] = (s @ q[t][..., None])[..., 0]
        recent = (0 if t % 32 == 0 else recent * g) + b * (v[t].abs() + left)
        add = 2.0 ** -16 * (recent + left) + 2.0 ** -21 * log_decay[t, :, None].abs() * left
        err = err * g + add
        yerr[t] = q[t].norm(dim=-1)[:, None] * (err + 2.0 ** -16 * s.norm(dim=-1))
    return y, s, yerr, err


def _check(m, i, y, state, begin, rows=None, heads=None, cols=None, what=""):
    """Sequence i's rows (and its state, where rows is None) by the rule, in some heads and columns."""
    ry, rs, yerr, serr = _rule(m, i, begin, heads)
    n = m.counts[i]
    hs = list(range(m.heads)) if heads is None else list(heads)
    cs = list(range(D)) if cols is None else cols
    at = slice(0, n) if rows is None else rows
    got = y.view(-1, m.T, m.heads, D)[i, :n].double().cpu()[:, hs]
    worst = ((got - ry).abs()[at][..., cs] / (yerr[at][..., cs] + 1e-30)).max().item()
    assert worst <= 1, f"{what} sequence {i}: y off by {worst:.3g} of the bound"
    if rows is None:
        off = (state.double().cpu()[hs] - rs).norm(dim=-1)[:, cs]
        worst = (off / (serr[:, cs] + 1e-30)).max().item()
        assert worst <= 1, f"{what} sequence {i}: state off by {worst:.3g} of the bound"


@pytest.mark.parametrize("heads,key_heads,batch", FORMS)
def test_every_form_over_many_chunks(dev, heads, key_heads, batch):
    """Prompts of ten chunks and a part, so that each preparing wave takes its second chunk; shorter ones beside them, one without
    tokens."""
    T = 331
    counts = ([331, 289] + [33, 64, 0, 17])[:batch]
    m = Mixer(dev, 50 + heads, heads, key_heads, T, counts)
    pool = m.pool.clone()
    y = m.run(pool)
    for i in (0, 1, batch - 1):
        if counts[i]:
            _check(m, i, y, pool[m.slots[i]], m.pool[m.slots[i]])
    for i, n in enumerate(counts):
        assert (y.view(batch, T, heads, D)[i, n:] == 0).all()
        if n == 0:
            assert _same(pool[m.slots[i]], m.pool[m.slots[i]])
    again = m.pool.clone()
    assert _same(m.run(again), y) and _same(again, pool)


KINDS = ["fall 8", "fall 12", "fall 20", "rise 12", "rise 20", "outlier 12", "state 16", "columns", "vanish"]


@pytest.mark.parametrize("heads,key_heads,batch", FORMS)
@pytest.mark.parametrize("kind", KINDS)
def test_sizes_that_change_inside_a_prompt(dev, heads, key_heads, batch, kind):
    """Behind decays of about 0.4 a token, values that fall or rise by a power of two inside the first and the third chunk, one token
    far above the rest, a starting state that is soon forgotten, columns of unlike sizes; and values that rise to 1e10 and are zero
    from then on while the state all but vanishes."""
    T = 200
    m = Mixer(dev, 70 + heads, heads, key_heads, T, [T] * batch)
    m.a_log.zero_()
    m.dt.zero_()
    m.a[:] = (torch.randn(m.a.shape, generator=torch.Generator().manual_seed(3)) * 0.2 + 0.5).to(m.a)  # decays 1 / (1 + e^a)
    v = m.qkv.view(batch, T, 2 * key_heads + heads, D)[:, :, 2 * key_heads:]
    name, _, power = kind.partition(" ")
    f = 2.0 ** int(power or 0)
    if name == "fall":
        v[:, 11:70] /= f
        v[:, 85:] /= f
    elif name == "rise":
        v[:, 20:40] *= f
        v[:, 77:] *= f
    elif name == "outlier":
        v[:, ::50] *= f
    elif name == "state":
        m.pool *= f
    elif name == "columns":
        v *= 2.0 ** (torch.arange(D, device=dev) % 41 - 20)
    else:
        v[:] = 0
        v[:, 0] = 1e10
        m.pool[m.slots] = 0
        a = m.a.view(batch, T, heads)
        a[:, :32] = -4.6
        a[:, 32:] = 0.45
    pool = m.pool.clone()
    y = m.run(pool)
    assert torch.isfinite(y).all() and torch.isfinite(pool[m.slots]).all()
    for i in (0, batch - 1):
        _check(m, i, y, pool[m.slots[i]], m.pool[m.slots[i]], heads=[0, heads - 1], what=kind)


@pytest.mark.parametrize("heads,key_heads,batch", FORMS)
@pytest.mark.parametrize("where,col", [("v", 36), ("v", 37), ("k", 5), ("q", 5), ("a", 0), ("b", 0), ("state", 36), ("state", 101)])
@pytest.mark.parametrize("bad", [NAN, float("inf")])
def test_values_that_are_no_numbers_in_every_form(dev, heads, key_heads, batch, where, col, bad):
    """In a token of the third chunk, or the state, of one head: the rows before it, the columns that do not meet it, and their
    states are right; the other sequences keep their bits, and so do heads of other key heads."""
    T, at, last = 130, 75, heads - 1
    m = Mixer(dev, 90 + heads, heads, key_heads, T, [T] * batch)
    clean_pool = m.pool.clone()
    clean = m.run(clean_pool).view(batch, T, heads, D)
    kept = {name: getattr(m, name).clone() for name in ("qkv", "wide", "pool")}
    row = T + at
    if where == "v":
        m.qkv[row, (2 * key_heads + last) * D + col] = bad
    elif where in "qk":
        m.qkv[row, (key_heads - 1 + (key_heads if where == "k" else 0)) * D + col] = bad
    elif where in "ab":
        (m.a if where == "a" else m.b)[row, last] = bad
    else:
        m.pool[m.slots[1], last, col, 5] = bad
    pool = m.pool.clone()
    y = m.run(pool).view(batch, T, heads, D)
    for i in range(batch):
        if i != 1:
            assert _same(y[i], clean[i]) and _same(pool[m.slots[i]], clean_pool[m.slots[i]])
    hit = heads // key_heads if where in "qk" else 1
    assert _same(y[1, :, :heads - hit], clean[1, :, :heads - hit])
    assert _same(pool[m.slots[1], :heads - hit], clean_pool[m.slots[1], :heads - hit])
    for name, of in kept.items():
        getattr(m, name).copy_(of)
    begin, state = m.pool[m.slots[1]], pool[m.slots[1]]
    if where in ("v", "state"):
        others = [c for c in range(D) if c != col]
        _check(m, 1, y, state, begin, heads=[last], cols=others, what="other columns")
        if where == "state":
            assert not torch.isfinite(y[1, :, last, col]).any()
            return
        assert not torch.isfinite(y[1, at:, last, col]).any() and not torch.isfinite(state[last, col]).all()
    _check(m, 1, y, state, begin, rows=slice(0, at), heads=[last], what="rows before")
    if where == "q":
        assert torch.isnan(y[1, at, last]).all()
        _check(m, 1, y, state, begin, rows=slice(at + 1, T), heads=[last], what="rows after")
        assert torch.isfinite(state).all()
    elif where in "ka":
        if not (where == "a" and bad > 0):  # (a decay of 0 is a number)
            assert not torch.isfinite(y[1, at:, last]).any()


@pytest.mark.parametrize("heads,key_heads,batch", FORMS)
@pytest.mark.parametrize("T", [9, 130])
def test_rows_past_the_range_of_their_squares_are_zero(dev, heads, key_heads, batch, T):
    """Queries and keys of finite values whose squares pass 32 bits count as zeros, in chunks as token by token; rows just inside
    that range are right."""
    m = Mixer(dev, 110 + heads, heads, key_heads, T, [T] * batch)
    rows = m.qkv.view(batch, T, 2 * key_heads + heads, D)
    inside = m.qkv.clone().view(rows.shape)
    rows[:, 1::2, :2 * key_heads] *= 2.0 ** 59  # lengths of 11 * 2^59: squares of 2^125
    pool = m.pool.clone()
    y = m.run(pool)
    _check(m, 1, y, pool[m.slots[1]], m.pool[m.slots[1]], heads=[0, heads - 1], what="inside")
    rows.copy_(inside)
    rows[:, 4::7, :key_heads] *= 2.0 ** 66
    rows[:, 5::9, key_heads:2 * key_heads] *= 2.0 ** 100
    long_pool = m.pool.clone()
    long = m.run(long_pool)
    rows[:, 4::7, :key_heads] = 0
    rows[:, 5::9, key_heads:2 * key_heads] = 0
    pool = m.pool.clone()
    y = m.run(pool)
    assert torch.isfinite(long).all() and torch.equal(long, y) and torch.equal(long_pool[m.slots], pool[m.slots])


@pytest.mark.parametrize("heads,key_heads,batch", FORMS)
@pytest.mark.parametrize("kind", ["reset", "kept", "same", "zero"])
def test_hard_gates_and_keys_in_every_form(dev, heads, key_heads, batch, kind):
    """Decays of zero inside chunks, decays of one, one key for all tokens with betas of one, keys of zero."""
    T = 170
    m = Mixer(dev, 130 + heads, heads, key_heads, T, [T - 13 * (i % 2) for i in range(batch)])
    keys = m.qkv.view(batch, T, 2 * key_heads + heads, D)[:, :, key_heads:2 * key_heads]
    if kind == "reset":
        m.a[5::7] = 3000.0
        m.a[6::11] = 40.0
    elif kind == "kept":
        m.a[:] = -100.0
    elif kind == "same":
        keys[:] = keys[:, :1].clone()
        m.b[:], m.a[:] = 20.0, -100.0
    else:
        keys[:, 3::5] = 0
    pool = m.pool.clone()
    y = m.run(pool)
    assert torch.isfinite(y).all()
    for i in (0, 1):
        _check(m, i, y, pool[m.slots[i]], m.pool[m.slots[i]], heads=[0, heads - 1], what=kind)


@pytest.mark.parametrize("heads,key_heads,batch", FORMS)
def test_states_apart_in_every_form(dev, heads, key_heads, batch):
    """Read from one shared state or from none and written elsewhere, in a pool between other layers' states; a sequence without tokens
    passes its state on. What is only read, and what is free, stays as it was; in place and in a dense pool, the same bits."""
    T = 70
    counts = [T, 0, 33, T, 64, 1][:batch]
    m = Mixer(dev, 150 + heads, heads, key_heads, T, counts, extra=batch)
    n = m.pool.shape[0]
    free = [s for s in range(n) if s not in m.slots]
    read = [m.slots[0] if i % 3 < 2 else -1 for i in range(batch)]
    pool = m.pool.clone()
    y = m.run(pool, read, slots_out=_ints(free, dev))
    for i, c in enumerate(counts):
        begin = m.pool[read[i]] if read[i] >= 0 else torch.zeros_like(m.pool[0])
        if c:
            _check(m, i, y, pool[free[i]], begin, heads=[0, heads - 1])
        else:
            assert _same(pool[free[i]], begin)
    assert _same(pool[m.slots], m.pool[m.slots])
    wide = torch.full((n, 3, heads, D, D), 7.0, device=dev)
    wide[:, 1] = m.pool
    assert _same(m.run(wide[:, 1], read, slots_out=_ints(free, dev)), y) and _same(wide[:, 1], pool)
    assert (wide[:, 0] == 7).all() and (wide[:, 2] == 7).all()
    own = m.pool.clone()
    for i, s in enumerate(m.slots):
        own[s] = m.pool[read[i]] if read[i] >= 0 else 0
    assert _same(m.run(own), y)
    for i, s in enumerate(m.slots):
        assert _same(own[s], pool[free[i]])
