"""The batched-serving entry points (pages, token log-probabilities) refuse bad arguments on the host, before
any launch; no GPU needed."""

import ctypes

import pytest
import torch

from skinny_mlx import _lib
from skinny_mlx import kernels as K

DUMMY = ctypes.c_void_p(4096)  # never dereferenced: validation fails before any launch


def _expect_einval(rc, fragment):
    assert rc == -1
    assert fragment in _lib.lib().skinny_last_error().decode()


def _kv(**change):
    f = dict(lengths=4096, counts=None, pages=4096, ld_pages=8, max_pages=8, k_pages=4096, vt_pages=4096,
             k_stride=8 * 64 * 128, vt_stride=8 * 64 * 128, n_pages=20, page=64, n_kv=8, head_dim=128)
    f.update(change)
    return _lib.PagedKV(*(f[n] for n, _ in _lib.PagedKV._fields_))


BAD_CACHES = [
    (dict(lengths=None), "null"), (dict(pages=None), "null"), (dict(k_pages=None), "null"), (dict(vt_pages=None), "null"),
    (dict(head_dim=96), "head dim 96"), (dict(n_kv=0), "multiple of Hkv"), (dict(n_kv=5), "multiple of Hkv"),
    (dict(page=8), "page=8"), (dict(page=48), "page=48"), (dict(page=512), "page=512"), (dict(n_pages=0), "n_pages=0"),
    (dict(max_pages=0), "max_pages=0"), (dict(ld_pages=7), "ld_pages=7"),
    (dict(max_pages=1 << 25, ld_pages=1 << 25), "max_pages"), (dict(k_stride=8 * 64 * 128 - 8), "page strides"),
    (dict(vt_stride=8 * 64 * 128 + 4), "page strides"), (dict(k_pages=4104), "misaligned"), (dict(lengths=4098), "misaligned"),
    (dict(counts=4097), "misaligned"),
]


def _store(kv=None, qkv=DUMMY, ldq=48 * 128, b=2, t=3, hq=32, qs=128, koff=4096, voff=5120, rd=128, table=DUMMY, positions=512,
           out=DUMMY):
    kv = _kv() if kv is None else kv
    return _lib.lib().skinny_paged_store_bf16(qkv, ldq, b, t, hq, qs, koff, voff, None, None, 1e-6, rd, table, positions, kv,
                                              out, None)


def _attend(kv=None, q=DUMMY, b=2, t=3, hq=32, keys=512, gate=None, ldg=0, gs=0, ws=DUMMY, nbytes=1 << 40, out=DUMMY):
    kv = _kv() if kv is None else kv
    return _lib.lib().skinny_paged_attention_bf16(q, b, t, hq, kv, keys, 0.1, gate, ldg, gs, ws, nbytes, out, None)


@pytest.mark.parametrize("change,fragment", BAD_CACHES)
def test_bad_caches_are_refused(change, fragment):
    _expect_einval(_store(_kv(**change)), fragment)
    _expect_einval(_attend(_kv(**change)), fragment)


@pytest.mark.parametrize("args,fragment", [
    (dict(qkv=None), "null"), (dict(table=None), "null"), (dict(out=None), "null"), (dict(b=0), "B=0"), (dict(t=0), "T=0"),
    (dict(b=65536), "B=65536"), (dict(t=65536), "T=65536"), (dict(hq=31), "multiple of Hkv"), (dict(rd=63), "rotary_dim=63"),
    (dict(rd=0), "rotary_dim=0"), (dict(rd=130), "rotary_dim=130"), (dict(ldq=6143), "do not fit"), (dict(qs=127), "do not fit"),
    (dict(koff=-1), "do not fit"), (dict(voff=5121), "do not fit"), (dict(positions=511), "RoPE table"),
    (dict(qkv=ctypes.c_void_p(4097)), "misaligned"), (dict(out=ctypes.c_void_p(4104)), "misaligned"),
])
def test_paged_store_refuses(args, fragment):
    _expect_einval(_store(**args), fragment)


@pytest.mark.parametrize("args,fragment", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(t=17), "68 query rows"), (dict(t=65535), "query rows"),
    (dict(keys=0), "keys=0"), (dict(keys=513), "keys=513"), (dict(gate=DUMMY, ldg=-1), "gate strides"),
    (dict(gate=DUMMY, gs=-1), "gate strides"), (dict(q=ctypes.c_void_p(4104)), "misaligned"),
    (dict(ws=ctypes.c_void_p(4104)), "misaligned"), (dict(gate=ctypes.c_void_p(4097)), "misaligned"),
    (dict(nbytes=16), "workspace of 16"), (dict(ws=None), "workspace of 0"),
])
def test_paged_attention_refuses(args, fragment):
    _expect_einval(_attend(**args), fragment)


def test_paged_attention_workspace_sizes():
    size = _lib.lib().skinny_paged_attn_workspace_bytes
    assert size(1, 1, 32, 8, 128, 100) == 0       # one block of keys: nothing to join
    assert size(2, 3, 32, 8, 128, 512) > 0
    assert size(4, 3, 32, 8, 128, 512) == 2 * size(2, 3, 32, 8, 128, 512)
    assert size(64, 16, 32, 8, 128, 1 << 20) > 1 << 32  # past 32 bits
    for bad in ((0, 1, 32, 8, 128, 1000), (1, 0, 32, 8, 128, 1000), (1, 1, 30, 8, 128, 1000), (1, 1, 32, 8, 100, 1000),
                (1, 1, 32, 8, 128, 0), (1, 17, 32, 8, 128, 1000), (1, 1 << 30, 32, 8, 128, 1000)):
        assert size(*bad) == 0, bad


@pytest.mark.parametrize("args,fragment", [
    (dict(logits=None), "null"), (dict(tokens=None), "null"), (dict(ws=None), "null"), (dict(lp=None), "null"),
    (dict(ent=None), "null"), (dict(top=3, ids=None), "null"), (dict(top=3, alt=None), "null"), (dict(rows=0), "rows=0"),
    (dict(rows=65536), "rows=65536"), (dict(v=0, ld=8), "V=0"), (dict(v=524289, ld=524289), "V=524289"), (dict(ld=999), "ld=999"),
    (dict(top=-1), "top=-1"), (dict(top=33), "top=33"), (dict(v=5, ld=5, top=6), "top=6"), (dict(it=0.0), "temperature"),
    (dict(it=float("inf")), "temperature"), (dict(it=float("nan")), "temperature"), (dict(nbytes=8), "workspace of 8"),
    (dict(logits=ctypes.c_void_p(4097)), "misaligned"), (dict(ws=ctypes.c_void_p(4098)), "misaligned"),
])
def test_token_logprobs_refuses(args, fragment):
    a = dict(logits=DUMMY, rows=4, v=1000, ld=1000, tokens=DUMMY, it=1.0, top=0, ws=DUMMY, nbytes=1 << 30, lp=DUMMY, ent=DUMMY,
             ids=DUMMY, alt=DUMMY)
    a.update(args)
    _expect_einval(_lib.lib().skinny_token_logprobs_bf16(a["logits"], a["rows"], a["v"], a["ld"], a["tokens"], a["it"], a["top"],
                                                         a["ws"], a["nbytes"], a["lp"], a["ent"], a["ids"], a["alt"], None),
                   fragment)


def test_token_logprobs_workspace_sizes():
    size = _lib.lib().skinny_token_logprobs_workspace_bytes
    assert size(1, 1, 0) > 0 and size(10, 151936, 8) == 10 * size(1, 151936, 8)
    for bad in ((0, 10, 0), (1, 0, 0), (1, 524289, 0), (1, 10, -1), (1, 100, 33)):
        assert size(*bad) == 0, bad


def test_wrappers_refuse_host_tensors():
    b16, i32 = torch.bfloat16, torch.int32
    kp, vp = torch.zeros((2, 1, 16, 64), dtype=b16), torch.zeros((2, 1, 64, 16), dtype=b16)
    ln, pages = torch.zeros(1, dtype=i32), torch.zeros((1, 2), dtype=i32)
    with pytest.raises(ValueError, match="GPU"):
        K.paged_store(torch.zeros((1, 192), dtype=b16), 1, 1, 64, 64, 64, 128, None, None, 1e-6, 64, torch.zeros((32, 32, 2)), ln,
                      pages, kp, vp)
    with pytest.raises(ValueError, match="GPU"):
        K.paged_attention(torch.zeros((1, 1, 64), dtype=b16), ln, pages, kp, vp, 1.0)
    with pytest.raises(ValueError, match="GPU"):
        K.token_logprobs(torch.zeros((1, 64), dtype=b16), torch.zeros(1, dtype=i32))


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("inf"), 2e38])
def test_paged_attention_refuses_scales(scale):
    rc = _lib.lib().skinny_paged_attention_bf16(DUMMY, 2, 3, 32, _kv(), 512, scale, None, 0, 0, DUMMY, 1 << 40, DUMMY, None)
    _expect_einval(rc, "scale=")


def test_sequences_past_the_grid_are_refused():
    kv = _kv(max_pages=1 << 22, ld_pages=1 << 22, page=256, k_stride=8 * 256 * 128, vt_stride=8 * 256 * 128)
    _expect_einval(_attend(kv, keys=65535 * 8 * 128 + 1, nbytes=1 << 60), "at most 67107840")


def test_temperatures_whose_inverse_is_no_number_are_refused():
    rc = _lib.lib().skinny_token_logprobs_bf16(DUMMY, 4, 1000, 1000, DUMMY, 2e38, 0, DUMMY, 1 << 30, DUMMY, DUMMY, None, None, None)
    _expect_einval(rc, "temperature")
