"""The Gated-DeltaNet mixer of several sequences (csrc/gdn_batch.hip): its conv and its recurrence, states in a pool.

The conv, and the recurrence of up to 16 tokens, have the bits of the one-sequence kernels on each sequence alone. Longer
runs go in chunks and are held to the rule in 64 bits, with a bound that is counted: see _bound."""

import numpy as np
import pytest
import torch

from skinny_mlx import kernels as K

pytestmark = pytest.mark.gpu

BF16, I32 = torch.bfloat16, torch.int32
D = 128
NAN = float("nan")


def _ints(v, dev):
    return torch.tensor(v, dtype=I32, device=dev)


def _bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


def _same(a, b):
    return torch.equal(_bits(a), _bits(b))


class Mixer:
    """A batch's rows (padding rows NaN), gates as columns of wider rows, and a pool whose free states are NaN."""

    def __init__(self, dev, seed, heads, key_heads, T, counts, extra=2, k_std=1.0, state_std=0.1):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.heads, self.key_heads, self.T, self.counts = dev, heads, key_heads, T, counts
        b = len(counts)
        c = (2 * key_heads + heads) * D
        qkv = torch.randn((b, T, c), generator=g)
        qkv[..., key_heads * D:2 * key_heads * D] *= k_std
        gates = torch.randn((b, T, 2 * heads + 3), generator=g)
        for i, n in enumerate(counts):
            qkv[i, n:] = NAN
            gates[i, n:] = NAN
        self.qkv = qkv.view(b * T, c).to(BF16).to(dev)
        self.wide = gates.view(b * T, -1).to(BF16).to(dev)
        self.b, self.a = self.wide[:, 1:1 + heads], self.wide[:, 2 + heads:2 + 2 * heads]
        self.a_log = torch.log(torch.rand((heads,), generator=g) * 15 + 1).to(dev)
        self.dt = (torch.rand((heads,), generator=g) * 2 - 1).to(dev)
        n = b + extra
        self.slots = np.random.default_rng(seed).permutation(n)[:b].tolist()
        pool = torch.full((n, heads, D, D), NAN)
        pool[self.slots] = torch.randn((b, heads, D, D), generator=g) * state_std
        self.pool = pool.to(dev)

    def run(self, pool, slots=None, **kw):
        counts = kw.pop("counts", self.counts)
        return K.gdn_recurrence_batch(self.qkv, self.b, self.a, self.a_log, self.dt, pool,
                                      _ints(self.slots if slots is None else slots, self.dev), self.heads, D, D,
                                      counts=_ints(counts, self.dev), n_key_heads=self.key_heads, **kw)

    def alone(self, i, state):
        """Sequence i by the one-sequence kernel -> y; `state` advanced."""
        rows = slice(i * self.T, i * self.T + self.counts[i])
        return K.gdn_recurrence(self.qkv[rows], self.b[rows], self.a[rows], self.a_log, self.dt, state, None, self.heads, D, D,
                                n_key_heads=self.key_heads)


def _rule(m, i, state, chunk):
    """The rule in 64 bits over sequence i from `state` [H, Dv, Dk] -> y, the last state, and how far each may be off.

    _bound: the error of a value column, E (2-norm over the key dims), is carried on by the tokens' (I - beta k k^T) and
    decay, none of which lengthens it, and each token adds its own. Token by token (chunk 0) all is fp32: k.S and q.S over
    128 products and the update, 2 * (128 + 16) steps of 2^-24 of |v| + |S|; the unit vectors and gates, another 2 * 140, the
    exponentials 2 ulp of an argument's worth: 2^-14 in all. In chunks, the state, the corrections and the triangular matrices
    go into their products as two fp16 terms: 2^-22 of a value, and 2^-25 of a power of two that is at most 4 times the
    column's largest, so 2^-21.4 of that, 2^-18 of the column's length over 128 dims; the products are summed in fp32, 128 and 32
    steps of 2^-24, 2^-17 of theirs; a correction takes the errors of the chunk's tokens before it, each of at most 1 times its
    beta (|v| + |S|), from the system's inverse (32 substitution steps of 2^-24, and its terms) and its own two terms: 2^-16 of
    the sum of beta (|v| + |S|) over the chunk and of the token's own."""
    n, T = m.counts[i], m.T
    x = m.qkv.view(-1, T, 2 * m.key_heads + m.heads, D)[i, :n].double().cpu()
    rep = m.heads // m.key_heads
    unit = lambda h: (h / torch.sqrt((h * h).sum(-1, keepdim=True) + 1e-6)).repeat_interleave(rep, 1)  # noqa: E731
    q, k, v = unit(x[:, :m.key_heads]) * D ** -0.5, unit(x[:, m.key_heads:2 * m.key_heads]), x[:, 2 * m.key_heads:]
    a = m.a.view(-1, T, m.heads)[i, :n].double().cpu() + m.dt.double().cpu()
    decay = torch.exp(-m.a_log.double().cpu().exp() * torch.nn.functional.softplus(a, threshold=1e9))
    beta = torch.sigmoid(m.b.reshape(-1, T, m.heads)[i, :n].double().cpu())
    s = state.double().cpu().clone()
    y = torch.zeros((n, m.heads, D), dtype=torch.float64)
    err = torch.zeros((m.heads, D), dtype=torch.float64)
    yerr = torch.zeros_like(y)
    recent = torch.zeros_like(err)
    for t in range(n):
        before = s.norm(dim=-1)
        s = s * decay[t, :, None, None]
        delta = beta[t, :, None] * (v[t] - (s @ k[t][..., None])[..., 0])
        s = s + delta[..., None] * k[t][:, None]
        y[t] = (s @ q[t][..., None])[..., 0]
        size = v[t].abs() + before
        if chunk:
            recent = (0 if t % chunk == 0 else recent) + beta[t, :, None] * size
            add = 2.0 ** -16 * (recent + size)
        else:
            add = 2.0 ** -14 * size
        err = err * decay[t, :, None] + add
        yerr[t] = q[t].norm(dim=-1)[:, None] * (err + (2.0 ** -16 if chunk else 2.0 ** -14) * s.norm(dim=-1) + add)
    return y, s, yerr, err


def _near(m, y, states, begin, chunk, what=""):
    """y and the written states against the rule; padding rows zero. begin[i] = sequence i's first state."""
    y = y.view(-1, m.T, m.heads, D)
    for i, n in enumerate(m.counts):
        ry, rs, yerr, serr = _rule(m, i, begin[i], chunk)
        assert (y[i, n:] == 0).all(), f"{what} sequence {i}: padding"
        if n:
            worst = ((y[i, :n].double().cpu() - ry).abs() / yerr).max().item()
            assert worst <= 1, f"{what} sequence {i} of {n} tokens: y off by {worst:.3f} of the bound"
        off = (states[i].double().cpu() - rs).norm(dim=-1)
        worst = (off / (serr + 1e-30)).max().item() if n else off.max().item()
        assert worst <= (1 if n else 0), f"{what} sequence {i} of {n} tokens: state off by {worst:.3f} of the bound"


HEADS = [(4, 2), (16, 16), (3, 1), (32, 16)]


@pytest.mark.parametrize("heads,key_heads", HEADS)
@pytest.mark.parametrize("T", [1, 2, 5, 16])
@pytest.mark.parametrize("batch", [1, 5, 40])
def test_few_tokens_have_the_bits_of_each_sequence_alone(dev, heads, key_heads, T, batch):
    rng = np.random.default_rng(T + batch)
    counts = [T] + [int(c) for c in rng.integers(0, T + 1, batch - 1)]
    m = Mixer(dev, heads + T, heads, key_heads, T, counts)
    pool = m.pool.clone()
    y = m.run(pool).view(batch, T, heads, D)
    free = [i for i in range(m.pool.shape[0]) if i not in m.slots]
    assert torch.isnan(pool[free]).all()
    for i, n in enumerate(counts):
        assert (y[i, n:] == 0).all()
        state = m.pool[m.slots[i]].clone()
        if n:
            assert _same(y[i, :n], m.alone(i, state)), f"sequence {i}"
        assert _same(pool[m.slots[i]], state), f"sequence {i}"


LENGTHS = [1, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 96, 97, 100, 0, 130]


@pytest.mark.parametrize("heads,key_heads", [(4, 2), (2, 2), (3, 1)])
@pytest.mark.parametrize("T", [17, 24, 33, 64, 130])
def test_many_tokens_against_the_rule(dev, heads, key_heads, T):
    counts = [min(n, T) for n in LENGTHS]
    m = Mixer(dev, 3 * T + heads, heads, key_heads, T, counts)
    pool = m.pool.clone()
    y = m.run(pool)
    assert torch.isfinite(y).all()
    _near(m, y, [pool[s] for s in m.slots], [m.pool[s] for s in m.slots], 32)
    again = m.pool.clone()
    assert _same(m.run(again), y) and _same(again, pool)


def test_a_long_prompt(dev):
    m = Mixer(dev, 5, 2, 1, 1500, [1500, 1, 777])
    pool = m.pool.clone()
    y = m.run(pool)
    _near(m, y, [pool[s] for s in m.slots], [m.pool[s] for s in m.slots], 32)


@pytest.mark.parametrize("T", [1, 7, 40])
def test_states_that_are_read_and_written_apart(dev, T):
    """From one shared state, from none (zeros), and from its own; a sequence without tokens passes its state on. What is
    only read stays as it was, and so does what is free."""
    counts = [T, max(1, T // 2), 0, T, 0]
    m = Mixer(dev, 11, 4, 2, T, counts, extra=6)
    shared, own = m.slots[0], m.slots[3]
    free = [i for i in range(m.pool.shape[0]) if i not in m.slots]
    read = [shared, -1, shared, own, -1]
    written = free[:3] + [own, free[3]]
    pool = m.pool.clone()
    y = m.run(pool, read, slots_out=_ints(written, dev))
    zeros = torch.zeros_like(m.pool[0])
    begin = [m.pool[r] if r >= 0 else zeros for r in read]
    _near(m, y, [pool[w] for w in written], begin, 32 if T > 16 else 0)
    rest = [i for i in range(m.pool.shape[0]) if i not in written]
    assert _same(pool[rest], m.pool[rest])


@pytest.mark.parametrize("T", [1, 9, 50])
def test_sequences_that_cannot_be_touch_nothing(dev, T):
    """A slot outside the pool, zeros with nowhere to go, a count outside [0, T]: NaN rows, no state written; the others as alone."""
    counts = [T, T, T, T + 1, -1, T, T]
    m = Mixer(dev, 12, 4, 4, T, [T] * 7)
    n = m.pool.shape[0]
    slots = list(m.slots)
    slots[1], slots[2], slots[6] = n, -1, -2
    pool = m.pool.clone()
    y = m.run(pool, slots, counts=counts).view(7, T, -1)
    whole = m.pool.clone()
    ref = m.run(whole).view(7, T, -1)
    for i in range(7):
        if i in (0, 5):
            assert _same(y[i], ref[i]) and _same(pool[m.slots[i]], whole[m.slots[i]])
        else:
            assert torch.isnan(y[i]).all() and _same(pool[m.slots[i]], m.pool[m.slots[i]])
    out = list(m.slots)
    out[1], out[5] = n, -1
    pool = m.pool.clone()
    y = m.run(pool, slots_out=_ints(out, dev)).view(7, T, -1)
    for i in range(7):
        assert torch.isnan(y[i]).all() if i in (1, 5) else _same(y[i], ref[i])
    assert _same(pool[[m.slots[1], m.slots[5]]], m.pool[[m.slots[1], m.slots[5]]])


@pytest.mark.parametrize("T", [16, 80])
@pytest.mark.parametrize("where", ["v", "k", "q", "b", "a", "state"])
@pytest.mark.parametrize("bad", [NAN, float("inf"), -float("inf")])
def test_values_that_are_no_numbers_stay_where_they_are_seen(dev, T, where, bad):
    """In a token: the rows before it, the other value columns (for v and the state) and the other sequences keep their bits."""
    m = Mixer(dev, 13, 2, 2, T, [T, T, T])
    at, col = 2 * T // 3, 37
    clean_pool = m.pool.clone()
    clean = m.run(clean_pool).view(3, T, 2, D)
    row = T + at
    if where in "qkv":
        m.qkv[row, {"q": 0, "k": 2 * D, "v": 4 * D}[where] + col] = bad
    elif where in "ab":
        (m.a if where == "a" else m.b)[row, 0] = bad
    else:
        m.pool[m.slots[1], 0, col, 5] = bad
    pool = m.pool.clone()
    y = m.run(pool).view(3, T, 2, D)
    for i in (0, 2):
        assert _same(y[i], clean[i]) and _same(pool[m.slots[i]], clean_pool[m.slots[i]])
    assert _same(y[1, :, 1], clean[1, :, 1])  # the other head
    if where == "state":
        others = [c for c in range(D) if c != col]
        assert torch.isfinite(y[1, :, 0][:, others]).all() and not torch.isfinite(y[1, :, 0, col]).any()
        _columns_near(m, y, clean, others, 0, T)
        return
    _columns_near(m, y, clean, list(range(D)), 0, at)
    if where == "v":
        others = [c for c in range(D) if c != col]
        _columns_near(m, y, clean, others, 0, T)
        assert not torch.isfinite(y[1, at:, 0, col]).any()
    if where == "q":  # the row alone, and no state
        assert torch.isnan(y[1, at, 0]).all() and torch.isfinite(y[1, at + 1:]).all() and torch.isfinite(pool[m.slots[1]]).all()


def _columns_near(m, y, clean, cols, t0, t1):
    """Sequence 1's columns agree with the clean run's: the same rule, by whichever kernel form, so to twice its bound."""
    if t1 <= t0:
        return
    n = m.counts[1]
    assert n
    off = (y[1, t0:t1, 0][:, cols].double() - clean[1, t0:t1, 0][:, cols].double()).abs().max().item()
    assert off <= 2.0 ** -9, off  # of values around 0.1 to 1; the bound of _rule at 80 tokens is above


@pytest.mark.parametrize("T", [16, 100])
def test_hard_gates_and_keys(dev, T):
    """Decays that are zero in the middle of a run, decays of one, keys that all are the same with betas of one (each token
    replaces what the one before it wrote), keys of zero, keys too long and too short for their squares."""
    for kind in ("reset", "kept", "same", "zero", "long", "short"):
        m = Mixer(dev, 17, 2, 2, T, [T, T - 3])
        if kind == "reset":
            m.a[5::7] = 3000.0
            m.a[6::11] = 40.0
        elif kind == "kept":
            m.a[:] = -100.0
        elif kind == "same":
            keys = m.qkv.view(-1, 6, D)[:, 2:4]
            keys[:] = keys[:1].clone()
            m.b[:], m.a[:] = 20.0, -100.0
        elif kind == "zero":
            m.qkv.view(-1, 6, D)[3::5, 2:4] = 0
        elif kind == "long":
            m.qkv.view(-1, 6, D)[:, 0:4] *= 2.0 ** 50
        else:
            m.qkv.view(-1, 6, D)[:, 0:4] *= 2.0 ** -50
        pool = m.pool.clone()
        y = m.run(pool)
        assert torch.isfinite(y).all(), kind
        _near(m, y, [pool[s] for s in m.slots], [m.pool[s] for s in m.slots], 32 if T > 16 else 0, kind)


def test_one_prompt_in_pieces(dev):
    """A prompt in one call, and in calls of unlike lengths, the state carried on between them: both within the bound."""
    m = Mixer(dev, 19, 2, 1, 200, [200])
    whole = m.pool.clone()
    y = m.run(whole)
    pool, rows, at = m.pool.clone(), [], 0
    for n in (3, 64, 33, 100):
        part = slice(at, at + n)
        rows.append(K.gdn_recurrence_batch(m.qkv[part], m.b[part], m.a[part], m.a_log, m.dt, pool, _ints(m.slots, dev), 2, D, D,
                                           n_key_heads=1))
        at += n
    for got, state in ((y, whole), (torch.cat(rows), pool)):
        _near(m, got, [state[m.slots[0]]], [m.pool[m.slots[0]]], 32)


@pytest.mark.parametrize("T", [2, 40])
def test_states_between_other_layers_states(dev, T):
    m = Mixer(dev, 23, 4, 2, T, [T, T - 1, 1])
    pool = m.pool.clone()
    y = m.run(pool)
    wide = torch.full((m.pool.shape[0], 3, 4, D, D), 7.0, device=dev)
    wide[:, 1] = m.pool
    assert _same(m.run(wide[:, 1]), y) and _same(wide[:, 1], pool)
    assert (wide[:, 0] == 7).all() and (wide[:, 2] == 7).all()


def test_a_pool_past_32_bits_of_elements(dev):
    heads, n = 16, (1 << 32) // (16 * D * D) + 3
    pool = torch.empty((n, heads, D, D), device=dev)
    for T in (2, 40):
        m = Mixer(dev, 29, heads, 16, T, [T, T])
        small = m.pool.clone()
        y = m.run(small)
        far = [n - 1, n - 3]
        pool[far] = m.pool[m.slots]
        assert _same(m.run(pool, far), y) and _same(pool[far], small[m.slots])
    del pool
    c = 64
    n = (1 << 32) // (3 * c) + 3
    pool = torch.empty((n, 3, c), dtype=BF16, device=dev)
    x, w = torch.randn((10, c), device=dev).to(BF16), torch.randn((c, 4), device=dev).to(BF16)
    pool[[n - 1, n - 3]] = torch.randn((2, 3, c), device=dev).to(BF16)
    small = pool[[n - 1, n - 3]].clone()
    assert _same(K.gdn_conv_silu_batch(x, pool, w, _ints([n - 1, n - 3], dev)), K.gdn_conv_silu_batch(x, small, w, _ints([0, 1], dev)))
    assert _same(pool[[n - 1, n - 3]], small)


# --- the conv -----------------------------------------------------------------------------------

@pytest.mark.parametrize("C", [8, 37, 768, 6144])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 16, 17, 50])
def test_conv_has_the_bits_of_each_sequence_alone(dev, C, T):
    g = torch.Generator().manual_seed(C + T)
    counts = [T, 0, min(T, 1), min(T, 2), min(T, 3), T // 2, T]
    b = len(counts)
    x = torch.randn((b, T, C + 3), generator=g)
    for i, n in enumerate(counts):
        x[i, n:] = NAN
    x = x.view(b * T, -1).to(BF16).to(dev)[:, 1:1 + C]
    w = torch.randn((C, 4), generator=g).to(BF16).to(dev)
    pool = torch.randn((b + 3, 3, C), generator=g).to(BF16).to(dev)
    slots = np.random.default_rng(T).permutation(b + 3)[:b].tolist()
    for read, written in ((slots, None), ([slots[0]] * 4 + [-1] * 3, slots)):
        # the state that is shared is also the first sequence's own: give that one another to write
        out_slots = None if written is None else [s for s in range(b + 3) if s != slots[0]][:b]
        left = pool.clone()
        y = K.gdn_conv_silu_batch(x, left, w, _ints(read, dev), counts=_ints(counts, dev),
                                  slots_out=None if out_slots is None else _ints(out_slots, dev)).view(b, T, C)
        expected = pool.clone()
        for i, n in enumerate(counts):
            state = pool[read[i]].clone() if read[i] >= 0 else torch.zeros_like(pool[0])
            assert (y[i, n:] == 0).all()
            if n:
                assert _same(y[i, :n], K.gdn_conv_silu(x[i * T:i * T + n], state, w, None)), f"sequence {i}"
            expected[(out_slots or read)[i]] = state
        assert _same(left, expected)


@pytest.mark.parametrize("C,T", [(64, 5), (130, 21), (63, 3)])
def test_conv_of_rows_at_odd_places(dev, C, T):
    """Rows, states and results that begin at odd elements and lie odd strides apart: the bits of the same at even ones."""
    g = torch.Generator().manual_seed(C)
    b, n = 3, 5
    x = torch.randn((b * T, C), generator=g).to(BF16).to(dev)
    w = torch.randn((C, 4), generator=g).to(BF16).to(dev)
    state = torch.randn((n, 3, C), generator=g).to(BF16).to(dev)
    slots, counts = _ints([4, 0, 2], dev), _ints([T, T - 1, 1], dev)
    ref_state = state.clone()
    ref = K.gdn_conv_silu_batch(x, ref_state, w, slots, counts=counts)
    wide = torch.full((b * T, (C | 1) + 2), NAN, dtype=BF16, device=dev)
    odd_x = wide[:, 1:1 + C]
    odd_x.copy_(x)
    flat = torch.full((1 + n * (3 * C | 1) + 8,), NAN, dtype=BF16, device=dev)
    odd_state = flat.as_strided((n, 3, C), (3 * C | 1, C, 1), 1)
    odd_state.copy_(state)
    odd_w = torch.full((4 * C + 1,), NAN, dtype=BF16, device=dev)[1:].view(C, 4)
    odd_w.copy_(w)
    out = torch.full((b * T * C + 1,), NAN, dtype=BF16, device=dev)[1:].view(b * T, C)
    y = K.gdn_conv_silu_batch(odd_x, odd_state, odd_w, slots, counts=counts, out=out)
    assert y is out and _same(y, ref) and _same(odd_state, ref_state)


def test_conv_of_sequences_that_cannot_be(dev):
    C, T = 24, 20
    x = torch.randn((4 * T, C), device=dev).to(BF16)
    w = torch.randn((C, 4), device=dev).to(BF16)
    pool = torch.randn((3, 3, C), device=dev).to(BF16)
    left = pool.clone()
    y = K.gdn_conv_silu_batch(x, left, w, _ints([0, 3, -1, 1], dev), counts=_ints([T, T, T, T + 1], dev)).view(4, T, C)
    assert torch.isnan(y[1:]).all() and torch.isfinite(y[0]).all() and _same(left[1:], pool[1:])


# --- as a program runs them -----------------------------------------------------------------------

@pytest.mark.parametrize("T", [1, 33])
def test_captured_steps_follow_slots_and_counts(dev, T):
    """A step of conv and recurrence captured once, replayed with other slots, counts and rows and eager work between the
    replays: the bits of the eager steps."""
    heads, b = 4, 3
    c = 3 * heads * D
    g = torch.Generator().manual_seed(31)
    steps = [(torch.randn((b * T, c + 2 * heads), generator=g).to(BF16).to(dev),
              _ints(np.random.default_rng(i).permutation(b + 2)[:b].tolist(), dev), _ints([T, T - i % 2, max(T - i, 0)], dev))
             for i in range(6)]
    w = (torch.randn((c, 4), generator=g) * 0.5).to(BF16).to(dev)
    a_log, dt = torch.rand(heads, generator=g).to(dev), torch.rand(heads, generator=g).to(dev)

    def step(x, slots, counts, conv, state):
        xc = K.gdn_conv_silu_batch(x[:, :c], conv, w, slots, counts=counts)
        return K.gdn_recurrence_batch(xc, x[:, c:c + heads], x[:, c + heads:], a_log, dt, state, slots, heads, D, D, counts=counts)

    pools = lambda: (torch.zeros((b + 2, 3, c), dtype=BF16, device=dev), torch.zeros((b + 2, heads, D, D), device=dev))  # noqa: E731
    eager = pools()
    x, slots, counts = (t.clone() for t in steps[0])
    graphed = pools()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, slots, counts, *graphed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(x, slots, counts, *graphed)
    for t in graphed:
        t.zero_()
    for rows, sl, ct in steps:
        for to, of in ((x, rows), (slots, sl), (counts, ct)):
            to.copy_(of)
        graph.replay()
        ref = step(rows, sl, ct, *eager)
        torch.cuda.synchronize()
        assert _same(y, ref) and _same(graphed[0], eager[0]) and _same(graphed[1], eager[1])


@pytest.mark.parametrize("T", [1, 7, 40])
def test_a_padded_batch(dev, T):
    """Sequences without tokens that name a state which another one writes, several of them the same: they touch nothing, and the
    others have the bits of the batch without them."""
    m = Mixer(dev, 37 + T, 8, 4, T, [0, T, 0, max(T - 3, 1), 0])
    one, three = m.slots[1], m.slots[3]
    slots = [three, one, three, three, one]
    pool = m.pool.clone()
    y = m.run(pool, slots).view(5, T, -1)
    small = Mixer(dev, 37 + T, 8, 4, T, [T, max(T - 3, 1)])
    keep = torch.tensor([1, 3], device=dev)
    small.qkv, small.wide = (t.view(5, T, -1)[keep].reshape(2 * T, -1) for t in (m.qkv, m.wide))
    small.b, small.a, small.a_log, small.dt = small.wide[:, 1:9], small.wide[:, 10:18], m.a_log, m.dt
    ref_pool = m.pool.clone()
    ref = small.run(ref_pool, [one, three]).view(2, T, -1)
    assert _same(y[keep], ref) and _same(pool, ref_pool) and (y[[0, 2, 4]] == 0).all()
    g = torch.Generator().manual_seed(T)
    c = 320
    x, w = torch.randn((5 * T, c), generator=g).to(BF16).to(dev), torch.randn((c, 4), generator=g).to(BF16).to(dev)
    state = torch.randn((6, 3, c), generator=g).to(BF16).to(dev)
    mine, theirs = state.clone(), state.clone()
    out = K.gdn_conv_silu_batch(x, mine, w, _ints([4, 2, 4, 4, 2], dev), counts=_ints([0, T, 0, T, 0], dev)).view(5, T, c)
    alone = K.gdn_conv_silu_batch(x.view(5, T, c)[keep].reshape(2 * T, c), theirs, w, _ints([2, 4], dev)).view(2, T, c)
    assert _same(out[keep], alone) and _same(mine, theirs) and (out[[0, 2, 4]] == 0).all()


@pytest.mark.parametrize("T", [1, 9, 33])
def test_many_sequences(dev, T):
    """Hundreds of sequences: some of them against themselves in a small batch, bit for bit (in chunks, 2^-18 of the
    norm: sixteen times what a product of terms is off)."""
    rng = np.random.default_rng(T)
    b, heads, some = 700, 2, [0, 1, 350, 698, 699]
    m = Mixer(dev, 41 + T, heads, 1, T, [int(n) for n in rng.integers(0, T + 1, b)])
    pool = m.pool.clone()
    y = m.run(pool).view(b, T, heads, D)
    small = Mixer(dev, 41 + T, heads, 1, T, [m.counts[i] for i in some])
    keep = torch.tensor(some, device=dev)
    small.qkv, small.wide = (t.view(b, T, -1)[keep].reshape(len(some) * T, -1) for t in (m.qkv, m.wide))
    small.b, small.a, small.a_log, small.dt = small.wide[:, 1:1 + heads], small.wide[:, 2 + heads:2 + 2 * heads], m.a_log, m.dt
    ref_pool = m.pool.clone()
    ref = small.run(ref_pool, [m.slots[i] for i in some]).view(len(some), T, heads, D)
    for i, j in enumerate(some):
        got, want = (torch.cat([t.flatten(), p[m.slots[j]].flatten()]) for t, p in ((y[j], pool), (ref[i], ref_pool)))
        assert _same(got, want) if T <= 16 else (got - want).norm() <= 2.0 ** -18 * want.norm()


def test_two_streams_at_once(dev):
    m = [Mixer(dev, s, 4, 2, 60, [60, 41]) for s in (37, 41)]
    refs = []
    for x in m:
        pool = x.pool.clone()
        refs.append((x.run(pool), pool))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    pools = [x.pool.clone() for x in m]
    torch.cuda.synchronize()
    for x, s, pool in zip(m, streams, pools):
        with torch.cuda.stream(s):
            got.append(x.run(pool))
    torch.cuda.synchronize()
    for (y, pool), z, left in zip(refs, got, pools):
        assert _same(y, z) and _same(pool, left)


def test_refusals(dev):
    m = Mixer(dev, 43, 4, 2, 3, [3, 3])
    slots = _ints(m.slots, dev)

    def call(**change):
        f = dict(qkv=m.qkv, b=m.b, a=m.a, A_log=m.a_log, dt_bias=m.dt, state=m.pool, slots=slots, n_heads=4, dk=D, dv=D, n_key_heads=2)
        f.update(change)
        return K.gdn_recurrence_batch(**f)

    for change in (dict(qkv=m.qkv.float()), dict(qkv=m.qkv[:, :-8]), dict(qkv=m.qkv[:5]), dict(b=m.b[:, :3]), dict(a=m.a.contiguous()),
                   dict(a=m.a.float()), dict(A_log=m.a_log.double()), dict(dt_bias=m.dt[:3]), dict(state=m.pool[:, :2]),
                   dict(state=m.pool.transpose(2, 3)), dict(state=m.pool[:0]), dict(slots=slots.long()), dict(slots=slots[:0]),
                   dict(slots=slots.cpu()), dict(slots_out=slots[:1]), dict(counts=slots[:1]), dict(counts=slots.long()),
                   dict(out=torch.empty((6, 4, D), dtype=BF16, device=dev)), dict(n_key_heads=3), dict(dk=64), dict(state=m.pool.cpu())):
        with pytest.raises(ValueError):
            call(**change)
    x, w, pool = m.qkv[:, :768], torch.zeros((768, 4), dtype=BF16, device=dev), torch.zeros((4, 3, 768), dtype=BF16, device=dev)
    for args in ((x.float(), pool, w, slots), (x, pool.float(), w, slots), (x, pool[:, :2], w, slots), (x, pool, w[:, :3], slots),
                 (x, pool, w.t(), slots), (x, pool[..., ::2], w, slots), (x[:5], pool, w, slots), (x, pool, w, slots.long()),
                 (x.t(), pool, w, slots), (x, pool[:0], w, slots)):
        with pytest.raises(ValueError):
            K.gdn_conv_silu_batch(*args)
    with pytest.raises(ValueError):
        K.gdn_conv_silu_batch(x, pool, w, slots, out=torch.empty((6, 767), dtype=BF16, device=dev))
