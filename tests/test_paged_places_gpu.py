"""Where the paged calls read and write (csrc/paged.hip): pages far into a pool, rows and weights at odd addresses, and one
workspace for calls of several sizes."""

import pytest
import torch

from skinny_mlx import kernels as K

pytestmark = pytest.mark.gpu

BF16, I32 = torch.bfloat16, torch.int32
EPS = 1e-6


def _ints(v, dev):
    return torch.tensor(v, dtype=I32, device=dev)


def _bits(t):
    return t.contiguous().view(torch.int16)


@pytest.mark.parametrize("n,stride,used", [((1 << 16) + 40, 1 << 16, [(1 << 16) + 39, 3, (1 << 16) + 38]),  # pages next to each other
                                           (19, 1 << 28, [17, 3, 18])])                                     # and far apart
def test_pages_past_32_bits_lie_where_the_table_says(dev, n, stride, used):
    """New tokens in pages past 2^32 elements: there, and not in the pages that the low 32 bits of their places name."""
    hq, hkv, d, page, tokens = 2, 1, 256, 256, 700
    assert max(used) * stride >= 1 << 32
    aliases = [(p * stride & 0xFFFFFFFF) // stride for p in used if p * stride >> 32]
    assert len(aliases) == 2 and not set(aliases) & set(used)
    room = (n - 1) * stride + hkv * page * d
    k = torch.empty(room, dtype=BF16, device=dev).as_strided((n, hkv, page, d), (stride, page * d, d, 1))
    vt = torch.empty(room, dtype=BF16, device=dev).as_strided((n, hkv, d, page), (stride, page * d, page, 1))
    for p in aliases + used:
        k[p], vt[p] = 3.0, 5.0
    ks = torch.full((3, hkv, page, d), 3.0, dtype=BF16, device=dev)
    vs = torch.full((3, hkv, d, page), 5.0, dtype=BF16, device=dev)
    table = K.rope_table_dim(1e7, 64, 3 * page, dev)
    rows = torch.randn((tokens, 4 * d), generator=torch.Generator().manual_seed(1)).to(BF16).to(dev)
    outs = []
    for p, kk, vv in ((used, k, vt), ([0, 1, 2], ks, vs)):
        q = K.paged_store(rows, hq, hkv, d, d, 2 * d, 3 * d, None, None, EPS, 64, table, _ints([0], dev), _ints([p], dev), kk, vv)
        outs.append(K.paged_attention(q[-1:], _ints([tokens - 1], dev), _ints([p], dev), kk, vv, 0.06))
    for i, p in enumerate(used):
        assert torch.equal(_bits(k[p]), _bits(ks[i])) and torch.equal(_bits(vt[p]), _bits(vs[i])), p
    # what the pages must hold: keys whose first 64 dims are turned, values as they are
    for i in range(3):
        m = min(page, tokens - i * page)
        part = rows[i * page:i * page + m]
        assert torch.equal(_bits(ks[i, 0, :m, 64:]), _bits(part[:, 2 * d + 64:3 * d]))
        assert torch.equal(_bits(vs[i, 0, :, :m].t()), _bits(part[:, 3 * d:]))
        assert (ks[i, 0, m:] == 3).all() and (vs[i, 0, :, m:] == 5).all()
    for p in aliases:
        assert (k[p] == 3).all() and (vt[p] == 5).all(), p
    assert torch.isfinite(outs[0]).all() and torch.equal(_bits(outs[0]), _bits(outs[1]))
    # the attention reads them there: the same rows with the pages that the low bits name full of NaN
    for p in aliases:
        k[p], vt[p] = float("nan"), float("nan")
    q = outs[1].view(1, hq, d)
    far = K.paged_attention(q, _ints([tokens - 1], dev), _ints([used], dev), k, vt, 0.06)
    near = K.paged_attention(q, _ints([tokens - 1], dev), _ints([[0, 1, 2]], dev), ks, vs, 0.06)
    assert torch.equal(_bits(far), _bits(near))


@pytest.mark.parametrize("d,rd", [(64, 64), (64, 50), (128, 128), (256, 64)])
@pytest.mark.parametrize("T", [1, 5, 37])
@pytest.mark.parametrize("shift,q_gap,k_gap,v_gap,tail", [(1, 0, 0, 0, 0), (0, 1, 0, 0, 0), (0, 0, 1, 0, 0), (0, 0, 0, 1, 0),
                                                          (0, 0, 0, 0, 1), (3, 1, 3, 5, 7)])
def test_store_of_rows_at_odd_addresses(dev, d, rd, T, shift, q_gap, k_gap, v_gap, tail):
    """Rows, heads and norm weights at any even byte address: the bits of the call with all of them on 16 bytes."""
    hq, hkv, page, b = 4, 2, 16, 2
    g = torch.Generator().manual_seed(d + T)
    heads = torch.randn((b * T, hq + 2 * hkv, d), generator=g).to(BF16)
    norms = (1 + 0.1 * torch.randn((2, d), generator=g)).to(BF16).to(dev)
    ln = _ints([9, 30], dev)
    pages = _ints([[3, 1, 7, 5, 9], [0, 8, 2, 4, 6]], dev)
    table = K.rope_table_dim(1e4, rd, 5 * page, dev)

    def store(shift, q_gap, k_gap, v_gap, tail, qn, kn):
        qs = d + q_gap
        koff = hq * qs + k_gap
        voff = koff + hkv * d + v_gap
        cols = voff + hkv * d
        wide = torch.full((b * T, shift + cols + tail), float("nan"), dtype=BF16)
        rows = wide[:, shift:shift + cols]
        for h in range(hq):
            rows[:, h * qs:h * qs + d] = heads[:, h]
        rows[:, koff:koff + hkv * d] = heads[:, hq:hq + hkv].flatten(1)
        rows[:, voff:] = heads[:, hq + hkv:].flatten(1)
        k = torch.full((10, hkv, page, d), 7.0, dtype=BF16, device=dev)
        vt = torch.full((10, hkv, d, page), 7.0, dtype=BF16, device=dev)
        q = K.paged_store(wide.to(dev)[:, shift:shift + cols], hq, hkv, d, qs, koff, voff, qn, kn, EPS, rd, table, ln, pages, k, vt)
        return q, k, vt

    odd = torch.zeros(2 * d + 3, dtype=BF16, device=dev)
    odd[1:1 + d], odd[2 + d:2 + 2 * d] = norms[0], norms[1]
    got = store(shift, q_gap, k_gap, v_gap, tail, odd[1:1 + d], odd[2 + d:2 + 2 * d])
    ref = store(0, 0, 0, 0, 0, norms[0], norms[1])
    assert torch.isfinite(ref[0]).all()
    assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip(got, ref))


def test_one_workspace_for_all_of_a_programs_sizes(dev):
    """Fewer sequences or a lower bound can need more than the largest call does; the largest of the sizes serves them all."""
    hq, hkv, d, page = 8, 2, 128, 64
    sizes = [(b, keys) for b in (1, 3, 17, 64) for keys in (128, 1000, 1024, 4096)]
    need = {s: K.paged_attn_workspace(s[0], 1, hq, hkv, d, s[1], dev).numel() for s in sizes}
    ws = torch.empty(max(need.values()), dtype=torch.uint8, device=dev)
    g = torch.Generator(dev).manual_seed(2)
    k = torch.randn((64 * 64, hkv, page, d), device=dev, generator=g).to(BF16)
    vt = torch.randn((64 * 64, hkv, d, page), device=dev, generator=g).to(BF16)
    pages = torch.randperm(64 * 64, device=dev, generator=g).to(I32).view(64, 64)
    q = torch.randn((64, hq, d), device=dev, generator=g).to(BF16)
    for b, keys in sizes:
        ln = torch.randint(0, keys, (b,), device=dev, generator=g).to(I32)
        ref = K.paged_attention(q[:b], ln, pages[:b], k, vt, d ** -0.5, keys=keys)
        ws.fill_(255)
        got = K.paged_attention(q[:b], ln, pages[:b], k, vt, d ** -0.5, keys=keys, workspace=ws)
        assert torch.isfinite(ref).all() and torch.equal(_bits(got), _bits(ref)), (b, keys)
