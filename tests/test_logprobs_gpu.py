"""Token log-probabilities, entropy and alternatives (csrc/logprobs.hip) against 64 bits.

fp32 sums of non-negative terms: a slice's 8192 are added over at most 45 levels, the slices over 6, each off by U = 2^-24
relative; an exponential is off by 2 steps and by its argument's rounding, which weighs at most |a| e^-a < 1 step. So Z is within
64 U, ln Z within 64 U + a step of itself, and W / Z within 128 U + 8 U relative. A logprob adds the rounding of (x - m) / T."""

import numpy as np
import pytest
import torch

from skinny_mlx import kernels as K

pytestmark = pytest.mark.gpu

BF16, I32 = torch.bfloat16, torch.int32
U = 2.0 ** -24


def _scores(rows, v, seed, std=3.0):
    return (torch.randn((rows, v), generator=torch.Generator().manual_seed(seed)) * std).to(BF16)


def _check(x, tokens, top, T, got, what=""):
    lp, ent, ids, alt = (t.cpu() for t in got)
    rows, v = x.shape
    assert lp.shape == ent.shape == (rows,) and ids.shape == alt.shape == (rows, top)
    assert lp.dtype == ent.dtype == alt.dtype == torch.float32 and ids.dtype == I32
    x64 = x.double() / T
    m = x64.amax(-1, keepdim=True)
    d = x64 - m
    e = d.exp()
    z = e.sum(-1, keepdim=True)
    ln_z = z.log()
    w = torch.where(e > 0, -e * d.clamp(min=-1e300), 0).sum(-1) / z[:, 0]
    tol_z = 64 * U + 2 * U * ln_z[:, 0].abs()
    ref = d.gather(1, tokens.long()[:, None])[:, 0] - ln_z[:, 0]
    fin = torch.isfinite(ref)
    tol = tol_z + 4 * U * (d.gather(1, tokens.long()[:, None])[:, 0].abs() + ref.abs())
    assert ((lp.double() - ref).abs() <= tol)[fin].all() and torch.equal(lp[~fin].double(), ref[~fin]), what
    assert ((ent.double() - (ln_z[:, 0] + w)).abs() <= tol_z + 140 * U * w + 2 * U * (ln_z[:, 0] + w)).all(), what
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(ids.long(), order), what
    dt = d.gather(1, order)
    ref = dt - ln_z
    fin = torch.isfinite(ref)
    assert ((alt.double() - ref).abs() <= tol_z[:, None] + 4 * U * (dt.abs() + ref.abs()))[fin].all(), what
    assert torch.equal(alt[~fin].double(), ref[~fin]), what


@pytest.mark.parametrize("rows,v", [(1, 1), (2, 2), (3, 7), (5, 63), (4, 1000), (2, 8191), (2, 8192), (3, 8193), (2, 16385),
                                    (7, 32768), (5, 151936), (2, 248320), (1, 524288), (4, 100003)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
@pytest.mark.parametrize("T", [1.0, 0.7])
def test_against_64_bits(dev, rows, v, top, T):
    top = min(top, v)
    x = _scores(rows, v, v + top)
    tokens = torch.randint(0, v, (rows,), generator=torch.Generator().manual_seed(v), dtype=I32)
    tokens[0] = int(x[0].float().argmax())
    _check(x, tokens, top, T, K.token_logprobs(x.to(dev), tokens.to(dev), top, T), f"{rows} x {v}")


@pytest.mark.parametrize("offset", range(8))
def test_rows_off_the_grid(dev, offset):
    """Rows that begin at any even address, with any stride, and neighbours that must not be read as scores."""
    v, rows, top = 9001, 3, 9
    wide = torch.full((rows, v + 24), float("nan"), dtype=BF16)
    x = _scores(rows, v, 5)
    wide[:, offset:offset + v] = x
    tokens = torch.tensor([0, v - 1, 4500], dtype=I32)
    got = K.token_logprobs(wide.to(dev)[:, offset:offset + v], tokens.to(dev), top)
    _check(x, tokens, top, 1.0, got)
    # the same row wherever it lies: the same bits
    ref = K.token_logprobs(x.to(dev), tokens.to(dev), top)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("v", [100, 8192, 30000])
@pytest.mark.parametrize("top", [1, 8, 32])
def test_ties_go_to_the_lowest_index(dev, v, top):
    rows = torch.stack([
        torch.zeros(v), torch.full((v,), -5.0), (torch.arange(v) % 7).float(), (torch.arange(v) % 2).float() * 0.0 - 0.0,
        torch.where(torch.arange(v) % 3 == 0, -0.0, 0.0), torch.arange(v).float().flip(0), torch.arange(v).float(),
        torch.where(torch.arange(v) >= v - 40, 4.0, 1.0)]).to(BF16)
    tokens = torch.zeros(rows.shape[0], dtype=I32)
    _check(rows, tokens, top, 1.0, K.token_logprobs(rows.to(dev), tokens.to(dev), top))


def test_peaked_flat_and_large_scores(dev):
    v = 20000
    x = _scores(5, v, 6)
    x[0, 17777] = 3e38      # one token has it all: ln p = 0, entropy 0
    x[1] *= 1e4             # far apart
    x[2] = -3e38            # the type's lowest values, all alike
    x[3, :] = -3.3e38
    x[3, 5] = 0.0
    tokens = torch.tensor([17777, 3, 4, 5, 6], dtype=I32)
    got = K.token_logprobs(x.to(dev), tokens.to(dev), 4)
    _check(x, tokens, 4, 1.0, got)
    assert got[0][0] == 0 and got[1][0] == 0 and got[0][3] == 0


def test_banned_tokens_and_whole_slices_of_them(dev):
    v = 40000
    x = _scores(4, v, 7)
    x[0, ::2] = float("-inf")
    x[1, 8192:32768] = float("-inf")  # whole slices
    x[2, :] = float("-inf")
    x[2, 39999] = -4.0               # one token left
    x[3, 100:] = float("-inf")
    tokens = torch.tensor([4, 9000, 39999, 3], dtype=I32)
    got = K.token_logprobs(x.to(dev), tokens.to(dev), 32)
    _check(x, tokens, 32, 1.0, got)
    assert got[0][0] == float("-inf") and got[0][2] == 0 and got[1][2] == 0


def test_rows_without_a_distribution(dev):
    """NaN, +inf or nothing but -inf: NaN numbers; alternatives still in order, NaN scores last; the rows beside them are right."""
    v = 9000
    x = _scores(5, v, 8)
    x[1, 8500] = float("nan")
    x[2, 3] = float("inf")
    x[3] = float("-inf")
    tokens = torch.tensor([1, 1, 1, 1, 2], dtype=I32)
    lp, ent, ids, alt = (t.cpu() for t in K.token_logprobs(x.to(dev), tokens.to(dev), 6))
    assert torch.isnan(lp[1:4]).all() and torch.isnan(ent[1:4]).all() and torch.isnan(alt[1:4]).all()
    keep = [0, 4]
    _check(x[keep], tokens[keep], 6, 1.0, (lp[keep], ent[keep], ids[keep], alt[keep]))
    y = x.float()
    y[1, 8500] = float("-inf")
    assert torch.equal(ids[1].long(), torch.sort(y[1], dim=-1, descending=True, stable=True).indices[:6])
    assert ids[2, 0] == 3 and ids[3].tolist() == list(range(6))
    # fewer numbers than alternatives: every index once, the NaN ones last, by index
    z = torch.full((1, 10), float("nan"), dtype=BF16)
    z[0, 7], z[0, 2] = 1.0, float("-inf")
    assert K.token_logprobs(z.to(dev), tokens[:1].to(dev), 10)[2][0].tolist() == [7, 2, 0, 1, 3, 4, 5, 6, 8, 9]


def test_tokens_outside_the_vocabulary(dev):
    x = _scores(4, 500, 9)
    tokens = torch.tensor([-1, 500, 2 ** 31 - 1, -2 ** 31], dtype=I32)
    lp, ent, ids, alt = K.token_logprobs(x.to(dev), tokens.to(dev), 2)
    assert (lp == float("-inf")).all() and torch.isfinite(ent).all() and torch.isfinite(alt).all()


def test_rows_do_not_depend_on_their_batch(dev):
    x = _scores(300, 50001, 10).to(dev)
    tokens = torch.randint(0, 50001, (300,), dtype=I32).to(dev)
    both = K.token_logprobs(x, tokens, 7)
    for r in (0, 1, 150, 299):
        one = K.token_logprobs(x[r:r + 1], tokens[r:r + 1], 7)
        assert all(torch.equal(a[r:r + 1], b) for a, b in zip(both, one)), r


def test_no_rows(dev):
    got = K.token_logprobs(torch.zeros((0, 10), dtype=BF16, device=dev), torch.zeros(0, dtype=I32, device=dev), 3)
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0, 3), (0, 3)]


def test_captured_and_replayed(dev):
    x = _scores(6, 30001, 11).to(dev)
    tokens = torch.arange(6, dtype=I32, device=dev)
    buf = x.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = K.token_logprobs(buf, tokens, 5)
    for i in range(4):
        y = torch.roll(x, i * 1001, 1)
        buf.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        ref = K.token_logprobs(y, tokens, 5)
        assert all(torch.equal(a, b) for a, b in zip(outs, ref)), i


def test_wrapper_refuses(dev):
    x = _scores(2, 100, 12).to(dev)
    tok = torch.zeros(2, dtype=I32, device=dev)
    for match, args in (("logits", (x.float(), tok)), ("logits", (x.t(), tok)), ("tokens", (x, tok.long())), ("tokens", (x, tok[:1])),
                        ("tokens", (x, tok.cpu())), ("top=101", (x, tok, 101)), ("top=-1", (x, tok, -1)), ("top=33", (x, tok, 33)),
                        ("temperature", (x, tok, 1, 0.0)), ("temperature", (x, tok, 1, float("nan"))),
                        ("temperature", (x, tok, 1, float("inf"))), ("overlap", (x[:1].expand(2, -1), tok))):
        with pytest.raises(ValueError, match=match):
            K.token_logprobs(*args)
    wide = torch.zeros((1, 524289), dtype=BF16, device=dev)
    with pytest.raises(ValueError, match="V=524289"):
        K.token_logprobs(wide, tok[:1])


@pytest.mark.parametrize("v", [151936, 524288])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_equal_scores_in_many_slices(dev, v, top):
    """More candidates of one score than a row's join can list: still the lowest indices first."""
    rows = torch.stack([torch.full((v,), 2.0), torch.where(torch.arange(v) % 997 == 5, 7.0, -1.0),
                        torch.where(torch.arange(v) >= v - 9000, 3.0, 0.5)]).to(BF16)
    tokens = torch.tensor([0, 5, v - 1], dtype=I32)
    _check(rows, tokens, top, 1.0, K.token_logprobs(rows.to(dev), tokens.to(dev), top), f"{v} {top}")


def test_the_most_rows(dev):
    x = _scores(65535, 40, 13)
    tokens = torch.arange(65535, dtype=I32) % 40
    _check(x, tokens, 3, 1.0, K.token_logprobs(x.to(dev), tokens.to(dev), 3))


def test_calls_on_two_streams_at_once(dev):
    x = _scores(16, 100003, 14).to(dev)
    tokens = torch.arange(16, dtype=I32, device=dev)
    ref = K.token_logprobs(x, tokens, 5)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(K.token_logprobs(x, tokens, 5))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, ref))


@pytest.mark.parametrize("T", [1e-3, 0.05, 30.0])
def test_cold_and_hot_temperatures(dev, T):
    x = _scores(4, 20001, 15)
    tokens = torch.tensor([0, 1, 2, 20000], dtype=I32)
    tokens[0] = int(x[0].float().argmax())
    _check(x, tokens, 6, T, K.token_logprobs(x.to(dev), tokens.to(dev), 6, T))


@pytest.mark.parametrize("v", [9000, 40000, 151936])
@pytest.mark.parametrize("top", [2, 7, 32])
def test_plateaus_below_and_beside_the_largest(dev, v, top):
    """Rows whose top-th score is one of many equal ones: few above them, in other places; more of them than can be ranked, in few
    threads' parts or in many; all of them late in the row."""
    g = torch.Generator().manual_seed(v + top)
    x = torch.randn((6, v), generator=g).to(BF16).clamp(-4, 2.5)
    x[0, 100:1700] = 3.0
    x[1, 100:1700] = 3.0
    x[1, [5, 1699, v - 1, v // 2]] = torch.tensor([4.0, 5.0, 4.0, 6.0], dtype=BF16)
    x[2, ::9] = 3.0
    x[2, -3:] = 3.5
    x[3, v - 2000:] = 3.0
    x[3, 7] = 8.0
    x[4, :2048] = torch.linspace(3.0, 60.0, 2048).to(BF16)  # many above any thread's, ascending
    x[5] = float("-inf")
    x[5, [1, v - 1, v // 3]] = torch.tensor([1.0, 1.0, -2.0], dtype=BF16)
    tokens = torch.tensor([0, v - 1, 3, 7, 2047, 1], dtype=I32)
    _check(x, tokens, top, 1.0, K.token_logprobs(x.to(dev), tokens.to(dev), top), f"{v} {top}")


def test_few_numbers_among_nan(dev):
    v = 30000
    x = torch.full((1, v), float("nan"), dtype=BF16)
    x[0, [29999, 12000, 4]] = torch.tensor([2.0, float("-inf"), 1.0], dtype=BF16)
    lp, ent, ids, alt = K.token_logprobs(x.to(dev), torch.zeros(1, dtype=I32, device=dev), 32)
    rest = [i for i in range(40) if i != 4][:29]
    assert ids[0].tolist() == [29999, 4, 12000] + rest
    assert torch.isnan(lp).all() and torch.isnan(ent).all() and torch.isnan(alt).all()
