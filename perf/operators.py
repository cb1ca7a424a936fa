"""The operators of batched serving as timed cases: new keys and values into a paged cache with the
head norms and the rotation on the way (kernels.paged_store), the attention of each sequence's new
tokens over its pages (kernels.paged_attention), and the log-probabilities, entropy and top
alternatives of the tokens that were answered (kernels.token_logprobs).

Head layouts and vocabularies are those of the package's decoders (model.PRESETS), with one small
generic layout of 64-dim heads beside them. Token counts go from the one token of a decode step over
the few of a verify step to a prompt's; cached lengths from none to 65536, ragged inside a batch.

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
EPS = 1e-6

# (query heads, kv heads, head dim, rotary dim, output gate, RoPE base)
LAYOUTS = {
    "dense": (32, 8, 128, 128, False, 1e6),
    "qwen35": (16, 4, 256, 64, True, 1e7),
    "tiny": (4, 1, 128, 128, False, 1e6),
    "heads64": (8, 8, 64, 64, False, 1e4),
}
VOCABS = [1024, 32768, 151936, 248320]
MAX_CACHE = 4 * 65536 * 8 * 128  # keys x kv heads x dims of the largest attention case


def listed():
    return [
        # the new token of a lone sequence: a launch's latency and nothing else
        dict(name="store_b1", op="store", layout="dense", batch=1, tokens=1, past=300, page=64, ragged=False),
        # a decode step of 64 sequences at their own lengths
        dict(name="store_b64", op="store", layout="dense", batch=64, tokens=1, past=500, page=16, ragged=True),
        # a verify step: up to 8 drafted tokens a sequence, in the gated 256-dim layout with a quarter rotated
        dict(name="store_verify", op="store", layout="qwen35", batch=16, tokens=8, past=700, page=32, ragged=True),
        # two prompts' keys and values, the pages' edges met at odd places
        dict(name="store_prompt", op="store", layout="dense", batch=2, tokens=1501, past=90, page=64, ragged=True),
        # one sequence at the start of its answer
        dict(name="attn_b1_short", op="attn", layout="dense", batch=1, tokens=1, past=100, page=16, ragged=False),
        # an ordinary decode step: 32 sequences of up to 2048 tokens
        dict(name="attn_b32", op="attn", layout="dense", batch=32, tokens=1, past=2048, page=64, ragged=True),
        # few sequences over long caches: the cache's length is all the parallel work there is
        dict(name="attn_long", op="attn", layout="dense", batch=4, tokens=1, past=65535, page=256, ragged=False),
        # a verify step over small pages
        dict(name="attn_verify", op="attn", layout="dense", batch=12, tokens=8, past=4000, page=32, ragged=True),
        # the gated layout with 256-dim heads, a few drafts each
        dict(name="attn_qwen35", op="attn", layout="qwen35", batch=9, tokens=3, past=5003, page=64, ragged=True),
        # the answered token's log-probability after a decode step
        dict(name="logprobs_m1", op="logprobs", rows=1, vocab=151936, top=0, temp=1.0),
        # a batch's, with alternatives, over the largest vocabulary
        dict(name="logprobs_m16", op="logprobs", rows=16, vocab=248320, top=8, temp=1.0),
        # a prompt's tokens scored
        dict(name="logprobs_prompt", op="logprobs", rows=1021, vocab=151936, top=5, temp=1.0),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["store", "attn", "attn", "logprobs"])
    if op == "logprobs":
        # a decoder's own vocabulary, or any other (odd ones shift the rows off the 16-byte grid)
        vocab = rng.choice(VOCABS) if rng.random() < 0.5 else _log_int(rng, 1000, 248320)
        rows = _log_int(rng, 1, max(1, min(1021, 1021 * 151936 // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, top=rng.choice([0, 1, 2, 5, 8, 13, 20, 32]),
                    temp=rng.choice([1.0, 1.0, 0.7, 1.5]))
    layout = rng.choice(sorted(LAYOUTS))
    hq, hkv, d = LAYOUTS[layout][:3]
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "store":
        tokens = rng.choice([1, _log_int(rng, 1, 16), _log_int(rng, 1, 1500)])
        batch = _log_int(rng, 1, max(1, min(256, 3002 // tokens)))
        past = _log_int(rng, 1, max(1, min(2000, 40000 // batch)))
        return dict(op=op, layout=layout, batch=batch, tokens=tokens, past=past, page=page, ragged=rng.random() < 0.7)
    tokens = 1 if rng.random() < 0.6 else _log_int(rng, 2, min(16, 64 // (hq // hkv)))
    batch = _log_int(rng, 1, 64)
    past = _log_int(rng, 1, max(1, min(65535, MAX_CACHE // (batch * hkv * d) - tokens)))
    return dict(op=op, layout=layout, batch=batch, tokens=tokens, past=past, page=page, ragged=rng.random() < 0.7)


# --- inputs -------------------------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed) & 0x7FFFFFFF)


def _rows(shape, g, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(BF16)


def _sequences(case, seed):
    """Cached lengths, new tokens and page tables of a batch. A ragged batch has lengths from none to `past`
    and, for several tokens, counts from none to `tokens`; pages are dealt in no order, entries that no token
    needs yet are -1."""
    rng = random.Random(int(seed))
    b, t, past, page = case["batch"], case["tokens"], case["past"], case["page"]
    lengths, counts = [past] * b, [t] * b
    if case["ragged"]:
        lengths = [past if i == b // 2 else rng.randint(0, past) for i in range(b)]
        counts = [t if i == b // 2 else rng.randint(0 if i % 5 == 4 else min(t, max(1, t // 2)), t) for i in range(b)]
    need = [-(-(n + c) // page) for n, c in zip(lengths, counts)]
    width = -(-(past + t) // page)
    total = b * width  # the pool holds the whole batch at its longest
    order = list(range(total))
    rng.shuffle(order)
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    put = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    live = [i * t + j for i, c in enumerate(counts) for j in range(c)]
    return dict(lengths=put(lengths), counts=put(counts) if case["ragged"] else None, pages=put(table), total=total,
                live=torch.tensor(live, dtype=torch.int64, device=DEV), host=(lengths, counts))


def _rope_angles(positions, rd, base):
    """float64 [positions, rd / 2]: position * base^(-2i / rd)."""
    freq = base ** (-2.0 * torch.arange(rd // 2, dtype=torch.float64, device=DEV) / rd)
    return torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * freq


def _store_inputs(case, seed):
    g = _gen(seed)
    hq, hkv, d, rd, gate, base = LAYOUTS[case["layout"]]
    s = _sequences(case, seed)
    qs = 2 * d if gate else d
    angles = _rope_angles(s["pages"].shape[1] * case["page"], rd, base)
    return dict(s, qkv=_rows((case["batch"] * case["tokens"], hq * qs + 2 * hkv * d), g), qs=qs,
                qn=(torch.randn(d, generator=g, device=DEV) * 0.1 + 1).to(BF16),
                kn=(torch.randn(d, generator=g, device=DEV) * 0.1 + 1).to(BF16),
                table=torch.stack([angles.cos(), angles.sin()], -1).float().contiguous(),
                k=_rows((s["total"], hkv, case["page"], d), g), vt=_rows((s["total"], hkv, d, case["page"]), g))


def _attn_inputs(case, seed):
    g = _gen(seed)
    hq, hkv, d, rd, gate, base = LAYOUTS[case["layout"]]
    s = _sequences(case, seed)
    rows = case["batch"] * case["tokens"]
    # queries of normalised heads with a gain, so that a few keys stand out; the gate as q_proj's rows hold it,
    # beside the query of its head
    wide = _rows((rows, hq, 2 * d), g) if gate else None
    return dict(s, q=_rows((rows, hq, d), g, 2.0), gate=None if wide is None else wide[..., d:],
                k=_rows((s["total"], hkv, case["page"], d), g), vt=_rows((s["total"], hkv, d, case["page"]), g))


def _logits_inputs(case, seed):
    """A head's bf16 scores, one in 50 tokens banned (-inf) in every row, and the tokens that were answered:
    a frequent one mostly, any other now and then, none of them banned."""
    g = _gen(seed)
    rows, v = case["rows"], case["vocab"]
    logits = torch.randn((rows, v), generator=g, device=DEV).mul_(3.0).to(BF16)
    banned = torch.rand((v,), generator=g, device=DEV) < 0.02
    banned[0] = False
    logits[:, banned] = float("-inf")
    tokens = torch.randint(0, v, (rows,), generator=g, device=DEV)
    often = torch.rand((rows,), generator=g, device=DEV) < 0.7
    tokens = torch.where(often, logits.argmax(-1), tokens)
    tokens = torch.where(banned[tokens], 0, tokens)
    return logits, tokens.to(torch.int32)


def prepare(case, seed):
    op = case["op"]
    if op == "logprobs":
        logits, tokens = _logits_inputs(case, seed)
        return dict(case=case, logits=logits, tokens=tokens)
    return dict(_store_inputs(case, seed) if op == "store" else _attn_inputs(case, seed), case=case,
                keys=case["past"] + case["tokens"])


# --- one pass -----------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    op = case["op"]
    if op == "logprobs":
        if own:
            from skinny_mlx import kernels as K

            return K.token_logprobs(state["logits"], state["tokens"], case["top"], case["temp"])
        return _plain_logprobs(state["logits"], state["tokens"], case["top"], case["temp"])
    hq, hkv, d, rd, gate, base = LAYOUTS[case["layout"]]
    s = state
    if op == "store":
        koff = hq * s["qs"]
        if own:
            from skinny_mlx import kernels as K

            q = K.paged_store(s["qkv"], hq, hkv, d, s["qs"], koff, koff + hkv * d, s["qn"], s["kn"], EPS, rd, s["table"],
                              s["lengths"], s["pages"], s["k"], s["vt"], counts=s["counts"])
        else:
            q = _plain_store(s, case, hq, hkv, d, rd)
        return [q, s["k"], s["vt"]]
    if own:
        from skinny_mlx import kernels as K

        return K.paged_attention(s["q"], s["lengths"], s["pages"], s["k"], s["vt"], d ** -0.5, counts=s["counts"],
                                 gate=s["gate"], keys=s["keys"])
    return _plain_attention(s, case, hkv, d)


def _positions(s, case):
    """[B, T] position of every row, and which rows are tokens (the others pad their sequence)."""
    t = torch.arange(case["tokens"], device=DEV)
    counts = s["counts"]
    there = t < (case["tokens"] if counts is None else counts[:, None])
    return s["lengths"][:, None] + t, there.expand(case["batch"], case["tokens"])


def _plain_store(s, case, hq, hkv, d, rd):
    page, half = case["page"], rd // 2
    rows = s["qkv"].shape[0]
    x = s["qkv"].float()
    q = x[:, :hq * s["qs"]].view(rows, hq, s["qs"])[..., :d]
    k, v = x[:, hq * s["qs"]:].view(rows, 2, hkv, d).unbind(1)
    heads = torch.cat([q, k], 1)
    weight = torch.cat([s["qn"].float().expand(hq, d), s["kn"].float().expand(hkv, d)])
    heads = heads * torch.rsqrt(heads.square().mean(-1, keepdim=True) + EPS) * weight
    pos, there = _positions(s, case)
    pos, there = pos.reshape(-1).long(), there.reshape(-1)
    turn = s["table"][pos]
    c, sn = turn[:, None, :, 0], turn[:, None, :, 1]
    a, b = heads[..., :half], heads[..., half:rd]
    heads = torch.cat([a * c - b * sn, b * c + a * sn, heads[..., rd:]], -1).to(BF16)
    i = s["live"]
    at = s["pages"][i // case["tokens"], pos[i] // page].long()
    s["k"][at, :, pos[i] % page] = heads[i, hq:]
    s["vt"][at, :, :, pos[i] % page] = v[i].to(BF16)
    return torch.where(there[:, None, None], heads[:, :hq], 0)


def _plain_attention(s, case, hkv, d):
    b, t, page = case["batch"], case["tokens"], case["page"]
    hq = s["q"].shape[1]
    ids = s["pages"].clamp(min=0).long()
    n = ids.shape[1] * page
    k = s["k"][ids].permute(0, 2, 1, 3, 4).reshape(b, hkv, n, d).float()
    v = s["vt"][ids].permute(0, 2, 1, 4, 3).reshape(b, hkv, n, d).float()
    q = s["q"].float().view(b, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    score = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    pos, there = _positions(s, case)
    seen = torch.arange(n, device=DEV) <= pos[..., None]
    seen = seen.repeat_interleave(hq // hkv, 1)[:, None]
    score = score.masked_fill(~seen, float("-inf"))
    e = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    o = o.view(b, hkv, t, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b * t, hq, d)
    if s["gate"] is not None:
        o = o / (1 + torch.exp(-s["gate"].float()))
    return torch.where(there.reshape(-1)[:, None, None], o, 0).to(BF16).view(b * t, hq * d)


def _plain_logprobs(logits, tokens, top, temp):
    x = logits.float()
    order = None
    if top:  # decreasing, ties by index: the value's bits as an ordered integer, then the index
        bits = x.view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * x.shape[1] - torch.arange(x.shape[1], device=DEV)
        order = key.topk(top, -1).indices
    x = x / temp
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x)
    z = e.sum(-1, keepdim=True)
    log_z = z.log()
    entropy = log_z[:, 0] - torch.where(e > 0, e * x, 0).sum(-1) / z[:, 0]
    logprob = x.gather(1, tokens.long()[:, None])[:, 0] - log_z[:, 0]
    if not top:
        return logprob, entropy, logits.new_empty((x.shape[0], 0), dtype=torch.int32), x.new_empty((x.shape[0], 0))
    return logprob, entropy, order.to(torch.int32), x.gather(1, order) - log_z


# --- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    if case["op"] == "logprobs":
        rows, v, top = case["rows"], case["vocab"], case["top"]
        return dict(bytes=rows * (2 * v + 4 + 8 + 8 * top), flops=6 * rows * v)
    hq, hkv, d, rd, gate, base = LAYOUTS[case["layout"]]
    b, t, past = case["batch"], case["tokens"], case["past"]
    # a ragged batch's lengths are even over 0 .. past; three in four of its rows are tokens where there are several
    keys = b * (past + t) if not case["ragged"] else past + t + (b - 1) * (past // 2 + max(1, (3 * t) // 4))
    rows = b * t if not case["ragged"] or t == 1 else t + (b - 1) * max(1, (3 * t) // 4)
    if case["op"] == "store":
        return dict(bytes=2 * rows * (2 * hq + 4 * hkv) * d + rows * 4 * rd + 4 * d, flops=rows * (hq + hkv) * (4 * d + 3 * rd))
    return dict(bytes=2 * 2 * keys * hkv * d + 2 * rows * hq * d * (3 if gate else 2),
                flops=4 * hq * d * (keys * rows // b))


# --- the same in 64 bits --------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "logprobs":
        logits, tokens = _logits_inputs(case, seed)
        rows, v, top = case["rows"], case["vocab"], case["top"]
        lp, ent, alt = [], [], []
        for lo in range(0, rows, 64):
            y = torch.log_softmax(logits[lo:lo + 64].double() / case["temp"], -1)
            lp.append(y[torch.arange(y.shape[0], device=DEV), tokens[lo:lo + 64].long()])
            ent.append(-(y.exp() * y.clamp(min=-1e4)).sum(-1))
            alt.append(y.topk(top, -1).values)
        return torch.cat(lp), torch.cat(ent), None, torch.cat(alt)
    hq, hkv, d, rd, gate, base = LAYOUTS[case["layout"]]
    b, t, page = case["batch"], case["tokens"], case["page"]
    if case["op"] == "store":
        s = _store_inputs(case, seed)
        lengths, counts = s["host"]
        q_out = torch.zeros((b, t, hq, d), dtype=torch.float64, device=DEV)
        k_out, vt_out = s["k"].double(), s["vt"].double()
        x = s["qkv"].double().view(b, t, -1)
        cos, sin = s["table"].double().unbind(-1)

        def turned(h, w, pos):
            h = h / torch.sqrt((h * h).sum(-1, keepdim=True) / d + EPS) * w.double()
            z = torch.complex(h[..., :rd // 2], h[..., rd // 2:rd]) * torch.complex(cos[pos], sin[pos])[:, None]
            return torch.cat([z.real, z.imag, h[..., rd:]], -1)

        for i in range(b):
            c = counts[i]
            pos = torch.arange(lengths[i], lengths[i] + c, device=DEV)
            heads = x[i, :c, :hq * s["qs"]].view(c, hq, s["qs"])[..., :d]
            q_out[i, :c] = turned(heads, s["qn"], pos)
            kv = x[i, :c, hq * s["qs"]:]
            at = s["pages"][i].long()[pos // page]
            k_out[at, :, pos % page] = turned(kv[:, :hkv * d].reshape(c, hkv, d), s["kn"], pos)
            vt_out[at, :, :, pos % page] = kv[:, hkv * d:].reshape(c, hkv, d)
        return [q_out.view(b * t, hq, d), k_out, vt_out]
    s = _attn_inputs(case, seed)
    lengths, counts = s["host"]
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device=DEV)
    q = s["q"].double().view(b, t, hkv, hq // hkv, d)
    for i in range(b):
        n, c = lengths[i] + counts[i], counts[i]
        if not c:
            continue
        ids = s["pages"][i, :-(-n // page)].long()
        for h in range(hkv):
            keys = s["k"][ids, h].reshape(-1, d)[:n].double()
            vals = s["vt"][ids, h].transpose(1, 2).reshape(-1, d)[:n].double()
            sc = q[i, :c, h].reshape(-1, d) @ keys.t() / math.sqrt(d)
            last = lengths[i] + torch.arange(c, device=DEV).repeat_interleave(hq // hkv)
            sc = torch.where(torch.arange(n, device=DEV) > last[:, None], float("-inf"), sc)
            out[i, :c, h * (hq // hkv):(h + 1) * (hq // hkv)] = (torch.softmax(sc, -1) @ vals).view(c, -1, d)
    if gate:
        out = out * torch.sigmoid(s["gate"].double()).view(b, t, hq, d)
    return out.view(b * t, hq * d)
