"""Operators of a served batch of hybrid decoders as timed cases: the causal conv of the Gated-DeltaNet
mixers over several sequences (kernels.gdn_conv_silu_batch), their gated delta rule, token by token for a
decode step and in chunks for prompts (kernels.gdn_recurrence_batch), and the attention of sequences that
begin with one long prefix, whose keys are read once for all of them (kernels.paged_attention_shared).

Head layouts are those of the package's decoders (model.PRESETS), with one small generic layout of 64-dim
heads beside them. Token counts go from the one token of a decode step over the few of a verify step to a
prompt's, ragged inside a batch; prefixes from a page's worth to 65536 tokens.

listed() and draw(rng) give cases as plain dicts; prepare(case, seed) what a program holds before the
call; run(state) is one pass: with `own` the package's kernels, without it the same operators by
elementary torch operations; exact(case, seed) the same outputs in 64 bits.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "skinny-mlx_amd"))

own = False

DEV = "cuda:0"
BF16 = torch.bfloat16
DIM = 128  # dims of a Gated-DeltaNet key and value head
KW = 4     # taps of its conv

# Gated-DeltaNet layers: (value heads, key heads)
MIXERS = {"hybrid": (16, 16), "qwen35": (32, 16), "tiny": (4, 2)}
# attention layers: (query heads, kv heads, head dim, output gate)
LAYOUTS = {"dense": (32, 8, 128, False), "qwen35": (16, 4, 256, True), "tiny": (4, 1, 128, False),
           "heads64": (8, 8, 64, False)}
MAX_TOKENS = 16 * 1501 * 32           # tokens x value heads of the largest recurrence
MAX_SCORES = 64 * 32 * 128 * 32768    # rows x query heads x dims x prefix of the largest attention


def listed():
    return [
        # the new token of a lone sequence: a launch's latency
        dict(name="conv_b1", op="conv", mixer="qwen35", batch=1, tokens=1, ragged=False, start="own"),
        # the prompts of three sequences, one state for each
        dict(name="conv_prompt", op="conv", mixer="qwen35", batch=3, tokens=1501, ragged=True, start="own"),
        # the new token of a lone sequence
        dict(name="gdn_b1", op="gdn", mixer="hybrid", batch=1, tokens=1, ragged=False, start="own"),
        # a decode step of 64 sequences: their states, read and written
        dict(name="gdn_b64", op="gdn", mixer="qwen35", batch=64, tokens=1, ragged=False, start="own"),
        # a verify step: up to 8 drafted tokens each
        dict(name="gdn_verify", op="gdn", mixer="qwen35", batch=16, tokens=8, ragged=True, start="own"),
        # one prompt from nothing: the sequence's length is all there is
        dict(name="gdn_prompt", op="gdn", mixer="hybrid", batch=1, tokens=2039, ragged=False, start="none"),
        # the prompts of 16 sequences that go on from one shared prefix's state
        dict(name="gdn_prompts", op="gdn", mixer="qwen35", batch=16, tokens=1501, ragged=True, start="shared"),
        # two sequences at the start of their answers, behind a short prefix
        dict(name="shared_b2", op="shared", layout="dense", batch=2, tokens=1, prefix=200, past=50, page=16, ragged=False),
        # an ordinary decode step behind a system prompt
        dict(name="shared_b32", op="shared", layout="dense", batch=32, tokens=1, prefix=4099, past=500, page=64, ragged=True),
        # a large batch over one long document
        dict(name="shared_long", op="shared", layout="dense", batch=64, tokens=1, prefix=32768, past=1000, page=256, ragged=True),
        # a verify step in the gated layout with 256-dim heads
        dict(name="shared_verify", op="shared", layout="qwen35", batch=12, tokens=4, prefix=5003, past=700, page=32, ragged=True),
        # heads of their own keys: each is read for one query head alone
        dict(name="shared_heads64", op="shared", layout="heads64", batch=24, tokens=1, prefix=8191, past=300, page=64, ragged=True),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["conv", "gdn", "gdn", "shared", "shared"])
    if op != "shared":
        mixer = rng.choice(sorted(MIXERS))
        heads = MIXERS[mixer][0]
        tokens = rng.choice([1, _log_int(rng, 1, 16), _log_int(rng, 1, 4096)])
        batch = _log_int(rng, 1, max(1, min(2048 // heads, MAX_TOKENS // (heads * tokens))))
        return dict(op=op, mixer=mixer, batch=batch, tokens=tokens, ragged=rng.random() < 0.7,
                    start=rng.choice(["own", "shared", "none"]))
    layout = rng.choice(sorted(LAYOUTS))
    hq, hkv, d, _ = LAYOUTS[layout]
    tokens = 1 if rng.random() < 0.6 else _log_int(rng, 2, min(16, 64 // (hq // hkv)))
    batch = _log_int(rng, 2, 128)
    prefix = _log_int(rng, 16, min(65536, MAX_SCORES // (batch * tokens * hq * d)))
    past = _log_int(rng, 1, max(1, min(2000, 64000 // batch)))
    return dict(op=op, layout=layout, batch=batch, tokens=tokens, prefix=prefix, past=past,
                page=rng.choice([16, 32, 64, 128, 256]), ragged=rng.random() < 0.7)


# --- inputs -------------------------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)


def _rows(shape, g, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(BF16)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _counts(rng: random.Random, case):
    """New tokens of each sequence: all of them, or ragged, now and then none."""
    b, t = case["batch"], case["tokens"]
    if not case["ragged"]:
        return [t] * b
    return [t if i == b // 2 else rng.randint(0 if i % 5 == 4 else min(t, max(1, t // 2)), t) for i in range(b)]


def _slots(rng: random.Random, case):
    """Which states of a pool the sequences read and write: each its own, in place; all the one that a shared
    prefix left, and each its own from then on; or none (-1: from zeros)."""
    b = case["batch"]
    order = list(range(b + 3))
    rng.shuffle(order)
    if case["start"] == "own":
        return order[:b], None
    return [order[b] if case["start"] == "shared" else -1] * b, order[:b]


def _mixer_inputs(case, seed):
    rng, g = random.Random(int(seed)), _gen(seed)
    heads, key_heads = MIXERS[case["mixer"]]
    rows, c = case["batch"] * case["tokens"], (2 * key_heads + heads) * DIM
    counts = _counts(rng, case)
    read, written = _slots(rng, case)
    s = dict(counts=_ints(counts) if case["ragged"] else None, slots=_ints(read),
             slots_out=None if written is None else _ints(written), host=(counts, read, written))
    # the fused projection's rows: q | k | v, then the output gate, then the two gates' columns
    wide = _rows((rows, c + heads * DIM + 2 * heads), g)
    if case["op"] == "conv":
        return dict(s, x=wide[:, :c], taps=_rows((c, KW), g, 0.5), pool=_rows((case["batch"] + 3, KW - 1, c), g))
    x = wide[:, :c].float()
    return dict(s, qkv=(x / (1 + torch.exp(-x))).to(BF16),  # what the conv's SiLU leaves
                b=wide[:, -2 * heads:-heads], a=wide[:, -heads:],
                a_log=torch.log(torch.rand((heads,), generator=g, device=DEV) * 15 + 1),
                dt=torch.rand((heads,), generator=g, device=DEV) * 2 - 1,
                pool=torch.randn((case["batch"] + 3, heads, DIM, DIM), generator=g, device=DEV) * 0.1)


def _shared_inputs(case, seed):
    """Pages dealt in no order to the prefix and the sequences; entries that no token needs are -1."""
    rng, g = random.Random(int(seed)), _gen(seed)
    hq, hkv, d, gate = LAYOUTS[case["layout"]]
    b, t, past, page = case["batch"], case["tokens"], case["past"], case["page"]
    counts = _counts(rng, case)
    lengths = [past if i == b // 2 or not case["ragged"] else rng.randint(0, past) for i in range(b)]
    need = [-(-(n + c) // page) for n, c in zip(lengths, counts)]
    width, front = -(-(past + t) // page), -(-case["prefix"] // page)
    total = front + b * width
    order = list(range(total))
    rng.shuffle(order)
    table, at = [], front
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    rows = b * t
    # queries of normalised heads with a gain, so that a few keys stand out; the gate as q_proj's rows hold it
    wide = _rows((rows, hq, 2 * d), g) if gate else None
    return dict(q=_rows((rows, hq, d), g, 2.0), gate=None if wide is None else wide[..., d:],
                k=_rows((total, hkv, page, d), g), vt=_rows((total, hkv, d, page), g),
                prefix=_ints([case["prefix"]]), prefix_pages=_ints(order[:front]), lengths=_ints(lengths),
                pages=_ints(table), counts=_ints(counts) if case["ragged"] else None, host=(lengths, counts))


def prepare(case, seed):
    if case["op"] == "shared":
        return dict(_shared_inputs(case, seed), case=case)
    return dict(_mixer_inputs(case, seed), case=case)


# --- one pass -----------------------------------------------------------------------------------

def run(state):
    s, case = state, state["case"]
    if case["op"] == "conv":
        if own:
            from skinny_mlx import kernels as K

            y = K.gdn_conv_silu_batch(s["x"], s["pool"], s["taps"], s["slots"], counts=s["counts"],
                                      slots_out=s["slots_out"])
        else:
            y = _plain_conv(s, case)
        return [y, s["pool"]]
    if case["op"] == "gdn":
        heads, key_heads = MIXERS[case["mixer"]]
        if own:
            from skinny_mlx import kernels as K

            y = K.gdn_recurrence_batch(s["qkv"], s["b"], s["a"], s["a_log"], s["dt"], s["pool"], s["slots"], heads, DIM,
                                       DIM, counts=s["counts"], slots_out=s["slots_out"], n_key_heads=key_heads)
        else:
            y = _plain_gdn(s, case, heads, key_heads)
        return [y, s["pool"]]
    hq, hkv, d, _ = LAYOUTS[case["layout"]]
    if own:
        from skinny_mlx import kernels as K

        return K.paged_attention_shared(s["q"], s["prefix"], s["prefix_pages"], s["lengths"], s["pages"], s["k"], s["vt"],
                                        d ** -0.5, counts=s["counts"], gate=s["gate"], prefix_keys=case["prefix"],
                                        keys=case["past"] + case["tokens"])
    return _plain_shared(s, case, hkv, d)


def _there(s, case):
    """[B, T]: which rows are tokens (the others pad their sequence)."""
    t = torch.arange(case["tokens"], device=DEV)
    there = t < (case["tokens"] if s["counts"] is None else s["counts"][:, None])
    return there.expand(case["batch"], case["tokens"])


def _read(s):
    """The states that the sequences begin with, in 32 bits."""
    slots = s["slots"].long()
    first = s["pool"][slots.clamp(min=0)].float()
    return torch.where((slots >= 0).view(-1, *[1] * (first.dim() - 1)), first, 0)


def _written(s):
    return (s["slots"] if s["slots_out"] is None else s["slots_out"]).long()


def _plain_conv(s, case):
    b, t = case["batch"], case["tokens"]
    x = torch.cat([_read(s), s["x"].view(b, t, -1).float()], 1)  # the state's rows, then the tokens'
    w = s["taps"].float()
    y = sum(x[:, j:j + t] * w[:, j] for j in range(KW))
    y = y / (1 + torch.exp(-y))
    count = torch.full((b,), t, device=DEV) if s["counts"] is None else s["counts"].long()
    last = count[:, None] + torch.arange(KW - 1, device=DEV)
    s["pool"][_written(s)] = x.gather(1, last[..., None].expand(-1, -1, x.shape[2])).to(BF16)
    return torch.where(_there(s, case)[..., None], y, 0).to(BF16).view(b * t, -1)


def _plain_gdn(s, case, heads, key_heads):
    b, t = case["batch"], case["tokens"]
    x = s["qkv"].float().view(b, t, -1)
    q, k, v = x.split([key_heads * DIM, key_heads * DIM, heads * DIM], -1)

    def unit(h):
        h = h.reshape(b, t, key_heads, DIM)
        return (h * torch.rsqrt(h.square().sum(-1, keepdim=True) + 1e-6)).repeat_interleave(heads // key_heads, 2)

    q, k, v = unit(q) * DIM ** -0.5, unit(k), v.reshape(b, t, heads, DIM)
    there = _there(s, case)[..., None]
    a = s["a"].float().view(b, t, heads) + s["dt"]
    step = torch.clamp(a, min=0) + torch.log1p(torch.exp(-a.abs()))
    decay = torch.where(there, torch.exp(-torch.exp(s["a_log"]) * step), 1)
    beta = torch.where(there, 1 / (1 + torch.exp(-s["b"].float().view(b, t, heads))), 0)
    state = _read(s)
    y = torch.empty((b, t, heads, DIM), dtype=torch.float32, device=DEV)
    for i in range(t):
        state = state * decay[:, i, :, None, None]
        key = k[:, i, :, None, :]
        delta = beta[:, i, :, None] * (v[:, i] - (state * key).sum(-1))
        state = state + delta[..., None] * key
        y[:, i] = (state * q[:, i, :, None, :]).sum(-1)
    s["pool"][_written(s)] = state
    return torch.where(there[..., None], y, 0).view(b * t, heads, DIM)


def _plain_shared(s, case, hkv, d):
    b, t, page, n0 = case["batch"], case["tokens"], case["page"], case["prefix"]
    hq = s["q"].shape[1]
    g = hq // hkv
    front = s["prefix_pages"].long()
    k0 = s["k"][front].permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :n0].float()
    v0 = s["vt"][front].permute(1, 0, 3, 2).reshape(hkv, -1, d)[:, :n0].float()
    ids = s["pages"].clamp(min=0).long()
    n = ids.shape[1] * page
    k = s["k"][ids].permute(0, 2, 1, 3, 4).reshape(b, hkv, n, d).float()
    v = s["vt"][ids].permute(0, 2, 1, 4, 3).reshape(b, hkv, n, d).float()
    q = s["q"].float().reshape(b, t, hkv, g, d).permute(2, 0, 1, 3, 4)  # [Hkv, B, T, G, D]
    far = torch.matmul(q.reshape(hkv, -1, d), k0.transpose(1, 2).contiguous()).reshape(hkv, b, t * g, n0) * d ** -0.5
    near = torch.matmul(q.transpose(0, 1).reshape(b, hkv, t * g, d), k.transpose(2, 3).contiguous()) * d ** -0.5
    there = _there(s, case)
    last = s["lengths"][:, None] + torch.arange(t, device=DEV)
    seen = (torch.arange(n, device=DEV) <= last[..., None]).repeat_interleave(g, 1)[:, None]
    near = near.masked_fill(~seen, float("-inf")).transpose(0, 1)  # [Hkv, B, T*G, n]
    top = torch.maximum(far.amax(-1, keepdim=True), near.amax(-1, keepdim=True))
    far, near = torch.exp(far - top), torch.exp(near - top)
    o = torch.matmul(far.reshape(hkv, -1, n0), v0).reshape(hkv, b, t * g, d)
    o = o + torch.matmul(near.transpose(0, 1), v).transpose(0, 1)
    o = o / (far.sum(-1, keepdim=True) + near.sum(-1, keepdim=True))
    o = o.reshape(hkv, b, t, g, d).permute(1, 2, 0, 3, 4).reshape(b * t, hq, d)
    if s["gate"] is not None:
        o = o / (1 + torch.exp(-s["gate"].float()))
    return torch.where(there.reshape(-1)[:, None, None], o, 0).to(BF16).reshape(b * t, hq * d)


# --- what a pass cannot do without ---------------------------------------------------------------

def _tokens(case):
    """Tokens of the batch: a ragged one's are three in four of its rows where there are several."""
    b, t = case["batch"], case["tokens"]
    return b * t if not case["ragged"] or t == 1 else t + (b - 1) * max(1, (3 * t) // 4)


def work(case):
    n, b = _tokens(case), case["batch"]
    if case["op"] != "shared":
        heads, key_heads = MIXERS[case["mixer"]]
        c = (2 * key_heads + heads) * DIM
        first = {"own": b, "shared": 1, "none": 0}[case["start"]]  # states read
        if case["op"] == "conv":
            return dict(bytes=4 * n * c + 2 * (KW - 1) * c * (b + first) + 2 * KW * c, flops=n * c * (2 * KW + 4))
        return dict(bytes=n * (2 * c + 4 * heads + 4 * heads * DIM) + 4 * heads * DIM * DIM * (b + first),
                    flops=7 * n * heads * DIM * DIM)
    hq, hkv, d, gate = LAYOUTS[case["layout"]]
    t, past = case["tokens"], case["past"]
    keys = b * (past + t) if not case["ragged"] else past + t + (b - 1) * (past // 2 + max(1, (3 * t) // 4))
    return dict(bytes=4 * (case["prefix"] + keys) * hkv * d + 2 * n * hq * d * (3 if gate else 2),
                flops=4 * hq * d * (n * case["prefix"] + keys * n // b))


# --- the same in 64 bits --------------------------------------------------------------------------

def exact(case, seed):
    b, t = case["batch"], case["tokens"]
    if case["op"] == "conv":
        s = _mixer_inputs(case, seed)
        counts, read, written = s["host"]
        pool = s["pool"].double()
        c = pool.shape[2]
        x = s["x"].double().view(b, t, c)
        y = torch.zeros((b, t, c), dtype=torch.float64, device=DEV)
        left = pool.clone()
        for i in range(b):
            line = torch.cat([pool[read[i]] if read[i] >= 0 else torch.zeros_like(pool[0]), x[i, :counts[i]]])
            if counts[i]:
                z = torch.nn.functional.conv1d(line.t()[None], s["taps"].double()[:, None], groups=c)[0].t()
                y[i, :counts[i]] = z * torch.sigmoid(z)
            left[(written or read)[i]] = line[-(KW - 1):]
        return [y.view(b * t, c), left]
    if case["op"] == "gdn":
        return _exact_gdn(case, seed)
    s = _shared_inputs(case, seed)
    hq, hkv, d, gate = LAYOUTS[case["layout"]]
    page, n0, g = case["page"], case["prefix"], LAYOUTS[case["layout"]][0] // LAYOUTS[case["layout"]][1]
    lengths, counts = s["host"]
    front = s["prefix_pages"].long()
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device=DEV)
    q = s["q"].double().view(b, t, hkv, g, d)
    for h in range(hkv):
        k0 = s["k"][front, h].reshape(-1, d)[:n0].double()
        v0 = s["vt"][front, h].transpose(1, 2).reshape(-1, d)[:n0].double()
        for i in range(b):
            n, c = lengths[i] + counts[i], counts[i]
            if not c:
                continue
            ids = s["pages"][i, :-(-n // page)].long()
            keys = torch.cat([k0, s["k"][ids, h].reshape(-1, d)[:n].double()])
            vals = torch.cat([v0, s["vt"][ids, h].transpose(1, 2).reshape(-1, d)[:n].double()])
            sc = q[i, :c, h].reshape(-1, d) @ keys.t() / math.sqrt(d)
            last = n0 + lengths[i] + torch.arange(c, device=DEV).repeat_interleave(g)
            sc = torch.where(torch.arange(n0 + n, device=DEV) > last[:, None], float("-inf"), sc)
            out[i, :c, h * g:(h + 1) * g] = (torch.softmax(sc, -1) @ vals).view(c, g, d)
    if gate:
        out = out * torch.sigmoid(s["gate"].double()).view(b, t, hq, d)
    return out.view(b * t, hq * d)


def _exact_gdn(case, seed):
    """Sixteen tokens at a time: the token's corrections d_i = beta_i (v_i - k_i . S_i-) solve a unit lower
    triangular system, the state is then the old one, decayed, and the sum of k_j d_j, decayed."""
    s = _mixer_inputs(case, seed)
    heads, key_heads = MIXERS[case["mixer"]]
    b, t = case["batch"], case["tokens"]
    counts, read, written = s["host"]
    x = s["qkv"].double().view(b, t, 2 * key_heads + heads, DIM).transpose(1, 2)  # [B, heads, T, 128]
    rep = heads // key_heads
    norm = lambda h: (h / torch.sqrt(torch.sum(h * h, -1, keepdim=True) + 1e-6)).repeat_interleave(rep, 1)  # noqa: E731
    q, k, v = norm(x[:, :key_heads]) / math.sqrt(DIM), norm(x[:, key_heads:2 * key_heads]), x[:, 2 * key_heads:]
    there = torch.arange(t, device=DEV) < torch.tensor(counts, device=DEV)[:, None, None]
    log_decay = -s["a_log"].double().exp()[:, None] * torch.nn.functional.softplus(
        s["a"].double().view(b, t, heads).transpose(1, 2) + s["dt"].double()[:, None])
    log_decay = torch.where(there, log_decay, 0.0)
    beta = torch.where(there, torch.sigmoid(s["b"].double().view(b, t, heads).transpose(1, 2)), 0.0)
    pool = s["pool"].double()
    state = torch.stack([pool[i].transpose(1, 2) if i >= 0 else torch.zeros_like(pool[0]) for i in read])  # [.., Dk, Dv]
    y = torch.zeros((b, heads, t, DIM), dtype=torch.float64, device=DEV)
    for lo in range(0, t, 16):
        at = slice(lo, min(lo + 16, t))
        kk, qq, bb = k[:, :, at], q[:, :, at], beta[:, :, at, None]
        total = torch.cumsum(log_decay[:, :, at], -1)
        between = torch.exp(total[..., :, None] - total[..., None, :]).tril()
        system = torch.matmul(kk, kk.transpose(2, 3).contiguous()) * between * bb
        system = system.tril(-1) + torch.eye(kk.shape[2], dtype=torch.float64, device=DEV)
        since = total.exp()[..., None]
        d = torch.linalg.solve_triangular(system, bb * (v[:, :, at] - since * torch.matmul(kk, state)), upper=False,
                                          unitriangular=True)
        y[:, :, at] = since * torch.matmul(qq, state)
        y[:, :, at] += torch.matmul(torch.matmul(qq, kk.transpose(2, 3).contiguous()) * between, d)
        until = torch.exp(total[..., -1:] - total)[..., None]
        state = state * since[:, :, -1:] + torch.matmul((kk * until).transpose(2, 3).contiguous(), d)
    left = pool.clone()
    for i in range(b):
        left[(written or read)[i]] = state[i].transpose(1, 2)
    return [torch.where(there.transpose(1, 2)[..., None], y.transpose(1, 2), 0.0).reshape(b * t, heads, DIM), left]
