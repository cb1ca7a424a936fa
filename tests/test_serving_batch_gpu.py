"""The operators of a served batch of hybrid decoders together, on the small presets: a prompt that all sequences begin with is
run once (its states and pages kept), each sequence's own tokens are run behind it, then all are decoded token by token."""

import numpy as np
import pytest
import torch

from skinny_mlx import kernels as K

pytestmark = pytest.mark.gpu

BF16, I32 = torch.bfloat16, torch.int32
NAN = float("nan")
PAGE, WIDTH = 16, 6


def _ints(v, dev):
    return torch.tensor(v, dtype=I32, device=dev)


class Served:
    """A model's layers over rows of several sequences, from its own modules and the batch calls."""

    def __init__(self, model, dev, prefix, batch):
        a = self.a = model.args
        self.model, self.dev, self.prefix = model, dev, prefix
        front = -(-prefix // PAGE)
        n = front + batch * WIDTH
        self.front = torch.arange(front, dtype=I32, device=dev).flip(0).contiguous()
        self.pages = (front + torch.arange(batch * WIDTH, dtype=I32, device=dev)).view(WIDTH, batch).t().contiguous()
        self.length = _ints([prefix], dev)
        self.table = K.rope_table_dim(a.rope_theta, a.rotary_dim, prefix + WIDTH * PAGE, dev)
        hkv, d = a.num_key_value_heads, a.head_dim
        self.caches = []
        for layer in model.layers:
            at = getattr(layer, "linear_attn", None)
            if at is None:
                self.caches.append((torch.full((n, hkv, PAGE, d), NAN, dtype=BF16, device=dev),
                                    torch.full((n, hkv, d, PAGE), NAN, dtype=BF16, device=dev)))
            else:
                self.caches.append((torch.full((batch + 1, a.linear_num_heads, 128, 128), NAN, device=dev),
                                    torch.full((batch + 1, a.linear_conv_kernel_dim - 1, at.conv_dim), NAN, dtype=BF16, device=dev)))

    def _attention(self, at, y, cache, ln, counts, T, front):
        """In steps of eight tokens: of the prefix itself (`front`) over its pages, of the sequences behind it."""
        a = self.a
        hq, hkv, d = a.num_attention_heads, a.num_key_value_heads, a.head_dim
        qs = 2 * d if a.attn_output_gate else d
        qkv = torch.cat([at.q_proj(y), at.k_proj(y), at.v_proj(y)], -1)
        b = ln.numel()
        out = torch.empty((b, T, hq * d), dtype=BF16, device=self.dev)
        rows = qkv.view(b, T, -1)
        for t0 in range(0, T, 8):
            t = min(8, T - t0)
            part = rows[:, t0:t0 + t].reshape(b * t, -1)
            some, at_len = (counts - t0).clamp(0, t), ln + torch.minimum(counts, _ints(t0, self.dev))
            pages = self.front.view(1, -1) if front else self.pages
            q = K.paged_store(part, hq, hkv, d, qs, hq * qs, hq * qs + hkv * d, at.q_norm, at.k_norm, a.rms_norm_eps, a.rotary_dim,
                              self.table if front else self.table[self.prefix:], at_len, pages, *cache, counts=some)
            gate = part[:, :hq * qs].view(b * t, hq, 2, d)[:, :, 1] if a.attn_output_gate else None
            if front:
                o = K.paged_attention(q, at_len, pages, *cache, d ** -0.5, counts=some, gate=gate)
            else:
                o = K.paged_attention_shared(q, self.length, self.front, at_len, pages, *cache, d ** -0.5, counts=some, gate=gate)
            out[:, t0:t0 + t] = o.view(b, t, -1)
        return at.o_proj(out.view(b * T, -1))

    def _mixer(self, at, y, cache, counts, slots, slots_out):
        a = self.a
        state, conv = cache
        xc = K.gdn_conv_silu_batch(at.in_proj_qkv(y), conv, at.conv1d_weight, slots, counts, slots_out)
        ys = K.gdn_recurrence_batch(xc, at.in_proj_b(y).contiguous(), at.in_proj_a(y).contiguous(), at.A_log, at.dt_bias, state,
                                    slots, a.linear_num_heads, 128, 128, counts, slots_out, a.gdn_key_heads)
        return at.out_proj(K.gated_rmsnorm(ys, at.in_proj_z(y), at.norm_weight, a.rms_norm_eps))

    def run(self, ids, ln, counts, slots, slots_out, front=False):
        """ids int32 [B, T] -> the last layer's normed rows [B, T, hidden]."""
        model, a = self.model, self.a
        b, T = ids.shape
        h = K.embed(ids.reshape(-1), model.embed_tokens)
        for layer, cache in zip(model.layers, self.caches):
            y = K.rmsnorm(h, layer.input_layernorm, a.rms_norm_eps)
            at = getattr(layer, "linear_attn", None)
            if at is None:
                o = self._attention(layer.self_attn, y, cache, ln, counts, T, front)
            else:
                o = self._mixer(at, y, cache, counts, slots, slots_out)
            h = h + o
            y = K.rmsnorm(h, layer.post_attention_layernorm, a.rms_norm_eps)
            h = h + layer.mlp.down_proj(K.silu_mul(torch.cat([layer.mlp.gate_proj(y), layer.mlp.up_proj(y)], -1)))
        return K.rmsnorm(h, model.norm, a.rms_norm_eps).view(b, T, -1)


@pytest.mark.parametrize("preset", ["tiny-hybrid", "tiny-qwen35"])
def test_a_shared_prompt_then_own_tokens_then_decode(dev, preset):
    """Own parts of 33, 1 and 12 tokens (chunks, and steps) behind a prompt of 75, eight tokens answered: the logits are the model's
    own over its contiguous cache and states, as near as its oracle tests ask. The prompt's state and pages keep their bits."""
    from skinny_mlx.cache import make_prompt_cache
    from skinny_mlx.model import build_model
    from skinny_mlx.patch import patch_model
    from skinny_mlx.spec import forward

    model = build_model(preset, device=dev)
    patch_model(model, fuse=False)
    rng = np.random.default_rng(1)
    prompt = rng.integers(0, model.args.vocab_size, 75).tolist()
    own = [rng.integers(0, model.args.vocab_size, n).tolist() for n in (33, 1, 12)]
    b, T = 3, 33
    s = Served(model, dev, len(prompt), b)
    s.run(_ints([prompt], dev), _ints([0], dev), _ints([75], dev), _ints([-1], dev), _ints([0], dev), front=True)
    kept = [(x[:s.front.numel()].clone(), y[:s.front.numel()].clone()) if x.dtype == BF16 else (x[0].clone(), y[0].clone())
            for x, y in s.caches]
    counts = _ints([len(p) for p in own], dev)
    slots = _ints([3, 1, 2], dev)
    h = s.run(_ints([p + [0] * (T - len(p)) for p in own], dev), _ints([0] * 3, dev), counts, _ints([0] * 3, dev), slots)
    last = torch.stack([h[i, len(p) - 1] for i, p in enumerate(own)])
    logits, tokens, ln = [], [], counts.clone()
    one = _ints([1] * 3, dev)
    for _ in range(8):
        logits.append(model.lm_head(last))
        tokens.append(K.argmax_rows(logits[-1]).clone())
        last = s.run(tokens[-1].view(b, 1), ln, one, slots, None)[:, 0]
        ln += 1
    for i, p in enumerate(own):
        answered = [int(t[i]) for t in tokens]
        _, ref = forward(model, prompt + p + answered[:-1], make_prompt_cache(model))
        ref = ref[len(prompt) + len(p) - 1:].float()
        got = torch.stack([x[i] for x in logits]).float()
        assert (got - ref).norm() <= 2e-2 * ref.norm()
    for (x, y), (kx, ky) in zip(s.caches, kept):
        now = (x[:s.front.numel()], y[:s.front.numel()]) if x.dtype == BF16 else (x[0], y[0])
        for m, n in zip(now, (kx, ky)):
            assert torch.equal(m.contiguous().view(I32), n.contiguous().view(I32))
