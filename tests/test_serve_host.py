"""CPU tests of the serving operators: what they refuse (before anything that
touches a GPU), the C entries' own checks, and the oracle's format."""
import ctypes

import numpy as np
import pytest
import torch

import bfloat16x_amd as bx
from bfloat16x_amd import _lib, kv4, sampling
from oracle import serve

BF, I32 = torch.bfloat16, torch.int32


def _cache(batch=2, kv=2, max_len=16, dim=64):
    return kv4.Kv4Cache.zeros(batch, kv, max_len, dim)


def _kv(batch=2, tokens=3, kv=2, dim=64, dtype=BF):
    return torch.zeros(batch, tokens, kv, dim, dtype=dtype)


POS = torch.zeros(2, dtype=I32)


def test_cache_sizes():
    c = _cache(dim=128)
    assert c.k.shape == (2, 2, 16, 64) and c.k_scale.shape == (2, 2, 16, 4, 2) and c.max_len == 16
    assert c.nbytes() == 2 * 2 * 2 * 16 * 80
    for bad in (dict(dim=96), dict(kv=0), dict(max_len=0), dict(batch=-1)):
        with pytest.raises(ValueError):
            _cache(**bad)
    assert bx.kv4 is kv4 and bx.sampling is sampling


def test_packed_words_follow_the_format():
    codes = np.tile(np.arange(16, dtype=np.uint8), 2).reshape(1, 32)             # one group
    p = serve.pack(codes)
    w = p.view(np.uint32)[0]
    assert w[0] == sum((2 * i) << (4 * i) | (2 * i + 1) << (16 + 4 * i) for i in range(4))
    v = serve.values(p, np.array([[[2.0, -1.0]]], np.float16))
    assert np.array_equal(v, codes * 2.0 - 1.0)


@pytest.mark.parametrize("change,kind,what", [
    (dict(k=None), TypeError, "k must be a tensor"),
    (dict(k=_kv(dtype=torch.float64)), TypeError, "k must be bf16"),
    (dict(v=_kv(dtype=torch.float16)), TypeError, "v must have k's type"),
    (dict(k=_kv(batch=1)), ValueError, "k must be"),
    (dict(k=_kv(kv=4)), ValueError, "k must be"),
    (dict(k=_kv(dim=128)), ValueError, "k must be"),
    (dict(k=_kv()[0]), ValueError, "k must be"),
    (dict(v=_kv(tokens=2)), ValueError, "v must be"),
    (dict(pos=POS.long()), TypeError, "pos must be"),
    (dict(pos=POS[:1]), ValueError, "pos must be"),
    (dict(pos=torch.zeros(4, dtype=I32)[::2]), ValueError, "pos must be"),
    (dict(q=_kv()), ValueError, "needs cos_sin"),
    (dict(q=_kv(tokens=2), cos_sin=torch.zeros(8, 32, 2)), ValueError, "q must be"),
    (dict(q=_kv(dtype=torch.float16), cos_sin=torch.zeros(8, 32, 2)), TypeError, "q must have"),
    (dict(cos_sin=torch.zeros(8, 64, 2)), ValueError, "cos_sin must be"),
    (dict(cos_sin=torch.zeros(0, 32, 2)), ValueError, "cos_sin must be"),
    (dict(cos_sin=torch.zeros(8, 32, 2, dtype=BF)), TypeError, "cos_sin must be"),
    (dict(cache=_cache()[:3]), TypeError, "cache must be"),
    (dict(cache=torch.zeros(4)), TypeError, "cache must be"),
    (dict(cache=7), TypeError, "cache must be"),
    (dict(cache=_cache()._replace(k=torch.zeros(2, 2, 16, 32))), TypeError, "cache k must be"),
    (dict(cache=_cache()._replace(v=torch.zeros(2, 2, 8, 32, dtype=torch.uint8))), ValueError, "cache v must"),
    (dict(cache=_cache()._replace(v_scale=torch.zeros(2, 2, 16, 2, dtype=torch.float16))), ValueError, "scale"),
    (dict(cache=_cache()._replace(k=torch.zeros(2, 16, 2, 32, dtype=torch.uint8).transpose(1, 2))), ValueError,
     "contiguous"),
    (dict(cache=kv4.Kv4Cache(*(t[:, :, :0] for t in _cache()))), ValueError, "no rows"),
    (dict(), ValueError, "GPU tensor"),
])
def test_append_refuses(change, kind, what):
    a = dict(k=_kv(), v=_kv(), cache=_cache(), pos=POS, q=None, cos_sin=None) | change
    with pytest.raises(kind, match=what):
        kv4.append(a["k"], a["v"], a["cache"], a["pos"], q=a["q"], cos_sin=a["cos_sin"])


@pytest.mark.parametrize("change,kind,what", [
    (dict(q=torch.zeros(2, 1, 4, 64)), TypeError, "q must be bf16 or fp16"),
    (dict(q=torch.zeros(2, 4, 64, dtype=BF)), ValueError, "q must be"),
    (dict(q=torch.zeros(2, 1, 3, 64, dtype=BF)), ValueError, "must divide"),
    (dict(q=torch.zeros(2, 1, 0, 64, dtype=BF)), ValueError, "must divide"),
    (dict(q=torch.zeros(1, 1, 4, 64, dtype=BF)), ValueError, "q must be"),
    (dict(start=POS.float()), TypeError, "start must be"),
    (dict(start=POS[:1]), ValueError, "start must be"),
    (dict(window=-1), ValueError, "window"),
    (dict(window=1.5), TypeError, None),
    (dict(scale="x"), TypeError, None),
    (dict(out=torch.zeros(2, 1, 4, 64, dtype=torch.float16)), TypeError, "out must be"),
    (dict(out=torch.zeros(2, 2, 4, 64, dtype=BF)), ValueError, "out must be"),
    (dict(), ValueError, "GPU tensor"),
])
def test_attention_refuses(change, kind, what):
    a = dict(q=torch.zeros(2, 1, 4, 64, dtype=BF), start=None, window=0, scale=None, out=None) | change
    with pytest.raises(kind, match=what):
        kv4.attention(a["q"], _cache(), POS, start=a["start"], window=a["window"], scale=a["scale"], out=a["out"])


def test_read_refuses():
    for args, kind in (((_cache(), POS, -1), ValueError), ((_cache(), POS, 2, torch.int8), TypeError),
                       ((_cache(), POS.long(), 2), TypeError), ((_cache(), POS, 2), ValueError)):
        with pytest.raises(kind):
            kv4.read(*args)


@pytest.mark.parametrize("change,kind,what", [
    (dict(logits=torch.zeros(3, 9, dtype=torch.float64)), TypeError, "logits must be"),
    (dict(logits=torch.zeros(3, 0)), ValueError, "logits must have"),
    (dict(logits=torch.zeros(1, 3, 9)), ValueError, "logits must be"),
    (dict(logits=torch.zeros(1).expand(3, (1 << 20) + 1)), ValueError, "logits must have"),
    (dict(u=torch.zeros(3, dtype=torch.float64)), TypeError, "u must be"),
    (dict(u=torch.zeros(2)), ValueError, "u must hold"),
    (dict(u=torch.zeros(6)[::2]), ValueError, "u must be contiguous"),
    (dict(temperature="a"), TypeError, None),
    (dict(temperature=torch.ones(2)), ValueError, "temperature must be"),
    (dict(temperature=torch.ones(3, dtype=BF)), TypeError, "temperature must be"),
    (dict(top_k=1.5), TypeError, None),
    (dict(top_k=torch.ones(3)), TypeError, "top_k must be"),
    (dict(token=torch.zeros(3, dtype=I32)), TypeError, "token must be"),
    (dict(token=torch.zeros(2, dtype=torch.int64)), ValueError, "token must be"),
    (dict(state=torch.zeros(2, dtype=I32)), ValueError, "state goes with one row"),
    (dict(history=torch.zeros(2, dtype=I32)), ValueError, "history"),
    (dict(), ValueError, "GPU tensor"),
])
def test_sample_refuses(change, kind, what):
    a = dict(logits=torch.zeros(3, 9), u=torch.zeros(3)) | change
    with pytest.raises(kind, match=what):
        sampling.sample(a.pop("logits"), a.pop("u"), **a)


def test_entries_validate_before_launch():
    """Every call is refused by the host-side checks; `p` is a 16-byte aligned host address, never read."""
    keep = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(keep) + (-ctypes.addressof(keep)) % 16
    L = _lib.lib()

    def append(q=None, q_out=None, k=p, cos=None, cos_rows=0, typ=0, batch=1, tokens=1, heads=0, kv=1, dim=64,
               max_len=8, pos=p, st=64):
        return L.bf16x_kv4_append(q, st, st, st, k, st, st, st, p, st, st, st, typ, batch, tokens, heads, kv, dim,
                                  max_len, pos, cos, cos_rows, q_out, p, p, p, p, None)

    assert append(k=None) == _lib.EARG and append(pos=None) == _lib.EARG
    assert append(q=p, q_out=p, heads=1) == _lib.EARG                           # q without a table
    assert append(q=p, cos=p, cos_rows=1, heads=1) == _lib.EARG                 # q without q_out
    assert append(cos=p) == _lib.EARG                                           # an empty table
    assert append(typ=3) == _lib.EDTYPE and append(dim=96) == _lib.ESHAPE and append(kv=0) == _lib.ESHAPE
    assert append(batch=-1) == _lib.EARG and append(max_len=0) == _lib.ESHAPE
    assert append(k=p + 2) == _lib.EARG and append(st=60) == _lib.EARG
    assert append(batch=0) == _lib.OK and append(tokens=0) == _lib.OK           # nothing to do, no launch

    def read(typ=0, dim=64, out=p, tokens=1):
        return L.bf16x_kv4_read(p, p, p, p, 1, tokens, 1, dim, 8, p, typ, out, p, None)

    assert read(typ=5) == _lib.EDTYPE and read(dim=32) == _lib.ESHAPE and read(out=p + 4) == _lib.EARG
    assert read(out=None) == _lib.EARG and read(tokens=0) == _lib.OK

    def attend(q=p, typ=0, heads=2, kv=1, dim=64, window=0, ws=p, n=1 << 40, tokens=1, out=p, max_len=4096):
        return L.bf16x_kv4_attention(q, 64, 64, 64, typ, 1, tokens, heads, kv, dim, max_len, p, p, p, p, p, None,
                                     window, 1.0, out, ws, n, None)

    assert attend(q=None) == _lib.EARG and attend(typ=2) == _lib.EDTYPE and attend(heads=3, kv=2) == _lib.ESHAPE
    assert attend(window=-1) == _lib.EARG and attend(dim=256) == _lib.ESHAPE and attend(q=p + 8) == _lib.EARG
    need = L.bf16x_kv4_attention_workspace(1, 1, 2, 1, 64, 4096)
    assert need > 0 and attend(n=need - 1) == _lib.ECAPACITY and attend(ws=None) == _lib.ECAPACITY
    assert attend(tokens=0) == _lib.OK
    assert L.bf16x_kv4_attention_workspace(1, 1, 3, 2, 64, 4096) == -1
    assert L.bf16x_kv4_attention_workspace(1, 1, 2, 1, 80, 4096) == -1

    settings = ctypes.create_string_buffer(64)
    s = ctypes.addressof(settings)

    def draw(x=p, typ=0, rows=1, vocab=100, n_u=1, state=None, hist=None, ws=p, n=1 << 40, set_=s, token=p):
        return L.bf16x_sample(x, typ, vocab, rows, vocab, p, n_u, set_, token, None, state, hist, 0, ws, n, None)

    assert draw(x=None) == _lib.EARG and draw(set_=None) == _lib.EARG and draw(ws=None) == _lib.EARG
    assert draw(typ=4) == _lib.EDTYPE and draw(vocab=0) == _lib.ESHAPE and draw(vocab=(1 << 20) + 1) == _lib.ESHAPE
    assert draw(rows=2, n_u=1) == _lib.ESHAPE and draw(rows=2, n_u=2, state=p) == _lib.ESHAPE
    assert draw(hist=p) == _lib.EARG and draw(token=p + 4) == _lib.EARG
    assert draw(n=L.bf16x_sample_workspace(1, 100) - 1) == _lib.ECAPACITY
    assert draw(rows=0, n_u=0) == _lib.OK
    assert L.bf16x_sample_workspace(1, 0) == -1 and L.bf16x_sample_workspace(70000, 100) == -1


@pytest.mark.parametrize("batch,tokens,heads,kv", [(1, 1, 32, 8), (1, 5, 32, 8), (2, 16, 8, 2), (1, 17, 32, 8),
                                                   (3, 100, 12, 4), (1, 700, 32, 8), (16, 1, 32, 8), (90, 1, 8, 8)])
def test_workspace_never_shrinks(batch, tokens, heads, kv):
    """A window makes a call see fewer keys, and its workspace is sized without it: fewer keys may need no more."""
    f = _lib.lib().bf16x_kv4_attention_workspace
    lengths = sorted({n + d for n in (1, 256, 512, 1024, 1536, 4096, 8192, 10000, 16384, 40000, 1 << 20)
                      for d in (-1, 0, 1, 300) if n + d > 0})
    sizes = [f(batch, tokens, heads, kv, 128, n) for n in lengths]
    assert sizes == sorted(sizes)
