"""The entry points of a batch of hybrid sequences (the mixer's conv and recurrence over a pool of states, attention behind a
shared prefix) refuse bad arguments on the host, before any launch; no GPU needed."""

import ctypes

import pytest
import torch

from skinny_mlx import _lib
from skinny_mlx import kernels as K
from test_serving_abi import BAD_CACHES, _kv

DUMMY = ctypes.c_void_p(4096)  # never dereferenced: validation fails before any launch
ODD = ctypes.c_void_p(4097)
STATE = 16 * 128 * 128


def _expect_einval(rc, fragment):
    assert rc == -1
    assert fragment in _lib.lib().skinny_last_error().decode()


def _pool(**change):
    f = dict(slots=4096, slots_out=None, counts=None, n_slots=9, stride=STATE)
    f.update(change)
    return _lib.StatePool(*(f[n] for n, _ in _lib.StatePool._fields_))


def _conv(pool=None, x=DUMMY, ldx=6144, b=2, t=3, c=6144, kw=4, state=DUMMY, w=DUMMY, out=DUMMY, ldo=6144):
    return _lib.lib().skinny_gdn_conv_silu_batch(x, ldx, b, t, c, kw, pool or _pool(), state, w, out, ldo, None)


def _gdn(pool=None, qkv=DUMMY, ldq=6144, bb=DUMMY, a=DUMMY, ldab=16, al=DUMMY, dt=DUMMY, b=2, t=3, state=DUMMY, y=DUMMY, h=16, hk=16,
         dk=128, dv=128):
    return _lib.lib().skinny_gdn_recurrence_batch(qkv, ldq, bb, a, ldab, al, dt, b, t, pool or _pool(), state, y, h, hk, dk, dv, None)


@pytest.mark.parametrize("change,fragment", [
    (dict(slots=None), "null"), (dict(n_slots=0), "n_slots=0"), (dict(stride=-1), "stride=-1"), (dict(stride=100), "stride=100"),
    (dict(slots=4097), "misaligned"), (dict(slots_out=4098), "misaligned"), (dict(counts=4097), "misaligned"),
])
def test_bad_pools_are_refused(change, fragment):
    _expect_einval(_conv(_pool(**change)), fragment)
    _expect_einval(_gdn(_pool(**change)), fragment)


@pytest.mark.parametrize("args,fragment", [
    (dict(x=None), "null"), (dict(state=None), "null"), (dict(w=None), "null"), (dict(out=None), "null"), (dict(kw=3), "width 3"),
    (dict(c=0), "C=0"), (dict(ldx=6143), "ldx=6143"), (dict(ldo=6143), "ldo=6143"), (dict(b=0), "B=0"), (dict(t=0), "T=0"),
    (dict(b=65536), "B=65536"), (dict(t=65536), "T=65536"), (dict(x=ODD), "misaligned"), (dict(out=ODD), "misaligned"),
    (dict(state=ODD), "misaligned"), (dict(w=ODD), "misaligned"),
])
def test_the_conv_refuses(args, fragment):
    _expect_einval(_conv(**args), fragment)


@pytest.mark.parametrize("args,fragment", [
    (dict(qkv=None), "null"), (dict(bb=None), "null"), (dict(a=None), "null"), (dict(al=None), "null"), (dict(dt=None), "null"),
    (dict(state=None), "null"), (dict(y=None), "null"), (dict(dk=64), "64x128"), (dict(dv=256), "128x256"), (dict(h=0), "H=0"),
    (dict(hk=3), "Hk=3"), (dict(hk=0), "Hk=0"), (dict(ldq=6143), "ldq=6143"), (dict(ldab=15), "ldab=15"), (dict(b=0), "B=0"),
    (dict(t=0), "T=0"), (dict(b=65536), "B=65536"), (dict(t=65536), "T=65536"), (dict(qkv=ctypes.c_void_p(4104)), "16-byte"),
    (dict(ldq=6148), "16-byte"), (dict(state=ctypes.c_void_p(4104)), "16-byte"), (dict(pool=_pool(stride=STATE + 2)), "16-byte"),
    (dict(y=ctypes.c_void_p(4104)), "misaligned"), (dict(a=ODD), "misaligned"), (dict(al=ctypes.c_void_p(4098)), "misaligned"),
    (dict(ldq=1 << 25), "too far apart"), (dict(ldab=1 << 25), "too far apart"),
])
def test_the_recurrence_refuses(args, fragment):
    _expect_einval(_gdn(**args), fragment)


def _shared(kv=None, q=DUMMY, b=2, t=3, hq=32, prefix=DUMMY, front=DUMMY, n_front=6, prefix_keys=384, keys=512, scale=0.1, gate=None,
            ldg=0, gs=0, ws=DUMMY, nbytes=1 << 40, out=DUMMY):
    return _lib.lib().skinny_paged_attention_shared_bf16(q, b, t, hq, kv or _kv(), prefix, front, n_front, prefix_keys, keys, scale,
                                                         gate, ldg, gs, ws, nbytes, out, None)


@pytest.mark.parametrize("change,fragment", BAD_CACHES)
def test_bad_caches_behind_a_prefix_are_refused(change, fragment):
    _expect_einval(_shared(_kv(**change)), fragment)


@pytest.mark.parametrize("args,fragment", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(prefix=None), "null"), (dict(front=None), "null"),
    (dict(t=17), "68 query rows"), (dict(keys=0), "keys=0"), (dict(keys=513), "keys=513"), (dict(n_front=0), "prefix_keys=384"),
    (dict(prefix_keys=0), "prefix_keys=0"), (dict(prefix_keys=385), "prefix_keys=385"), (dict(prefix_keys=-1), "prefix_keys=-1"),
    (dict(n_front=1 << 30), "pages of a prefix"), (dict(gate=DUMMY, ldg=-1), "gate strides"), (dict(gate=DUMMY, gs=-1), "gate strides"),
    (dict(q=ctypes.c_void_p(4104)), "misaligned"), (dict(ws=ctypes.c_void_p(4104)), "misaligned"), (dict(prefix=ODD), "misaligned"),
    (dict(front=ctypes.c_void_p(4098)), "misaligned"), (dict(gate=DUMMY, out=ctypes.c_void_p(4104)), "misaligned"),
    (dict(nbytes=16), "workspace of 16"), (dict(ws=None), "workspace of 0"), (dict(scale=0.0), "scale="),
    (dict(scale=float("nan")), "scale="), (dict(scale=float("inf")), "scale="), (dict(b=65536), "B=65536"),
])
def test_attention_behind_a_prefix_refuses(args, fragment):
    _expect_einval(_shared(**args), fragment)


def test_workspace_sizes_behind_a_prefix():
    size = _lib.lib().skinny_paged_attn_shared_workspace_bytes
    assert size(1, 1, 32, 8, 128, 1, 1) > 0
    assert size(64, 2, 32, 8, 128, 100000, 1 << 20) > size(64, 2, 32, 8, 128, 100000, 100)
    for bad in ((0, 1, 32, 8, 128, 10, 10), (65536, 1, 32, 8, 128, 10, 10), (1, 0, 32, 8, 128, 10, 10), (1, 1, 30, 8, 128, 10, 10),
                (1, 1, 32, 8, 100, 10, 10), (1, 1, 32, 8, 128, 0, 10), (1, 1, 32, 8, 128, 10, 0), (1, 17, 32, 8, 128, 10, 10),
                (1, 1, 32, 8, 128, (1 << 30) + 1, 10), (1, 1, 32, 0, 128, 10, 10), (1, 1 << 30, 32, 8, 128, 10, 10)):
        assert size(*bad) == 0, bad


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (16, 4, 256), (8, 8, 64), (64, 1, 128), (1, 1, 64)])
def test_workspaces_grow_with_what_is_bounded(hq, hkv, d):
    """The cut of a call is a rule on its sizes: any sizes within the limits have a workspace, of the rows' one part each at least and
    of no more than a part for every 64 keys of the prefix and every 32 of the own."""
    size = _lib.lib().skinny_paged_attn_shared_workspace_bytes
    for b in (1, 2, 7, 64, 1000, 65535):
        for t in {1, min(3, 64 * hkv // hq), 64 * hkv // hq}:
            for prefix in (1, 63, 64, 65, 4096, 100001, 1 << 30):
                for keys in (1, 31, 32, 33, 5000, 1 << 30):
                    n = size(b, t, hq, hkv, d, prefix, keys) // (b * t * hq * (d + 2) * 4)
                    assert 2 <= n <= -(-prefix // 64) + -(-keys // 32), (b, t, prefix, keys)


def test_wrappers_refuse_host_tensors():
    b16, i32 = torch.bfloat16, torch.int32
    one = torch.zeros(1, dtype=i32)
    with pytest.raises(ValueError, match="GPU"):
        K.gdn_conv_silu_batch(torch.zeros((1, 64), dtype=b16), torch.zeros((2, 3, 64), dtype=b16), torch.zeros((64, 4), dtype=b16), one)
    with pytest.raises(ValueError, match="GPU"):
        K.gdn_recurrence_batch(torch.zeros((1, 384), dtype=b16), torch.zeros((1, 1), dtype=b16), torch.zeros((1, 1), dtype=b16),
                               torch.zeros(1), torch.zeros(1), torch.zeros((2, 1, 128, 128)), one, 1, 128, 128)
    with pytest.raises(ValueError, match="GPU"):
        K.paged_attention_shared(torch.zeros((1, 1, 64), dtype=b16), one, one, one, torch.zeros((1, 2), dtype=i32),
                                 torch.zeros((2, 1, 16, 64), dtype=b16), torch.zeros((2, 1, 64, 16), dtype=b16), 1.0)
