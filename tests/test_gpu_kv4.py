"""The 4-bit KV cache on the GPU against the numpy oracle: codes bit for bit,
attention within what fp16 values and weights may change (oracle.serve.attention
gives that bound) and the output's own rounding."""
import numpy as np
import pytest
import torch

from bfloat16x_amd import kv4
from oracle import serve

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _rand(*shape, seed=0, dtype=BF, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _table(n, dim):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 5e5 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    return torch.stack([a.cos(), a.sin()], -1).float()


def _cache(k, v):
    """Kv4Cache on the GPU of k, v [B, KV, L, D] (fp32), and the values it stands for."""
    out, vals = [], []
    for x in (k, v):
        c, s, m = serve.quantise(x.numpy())
        sc = np.stack([s, m], -1)
        out += [torch.from_numpy(serve.pack(c)).to(DEV), torch.from_numpy(sc).to(DEV)]
        vals.append(serve.values(serve.pack(c), sc))
    return kv4.Kv4Cache(*out), vals


def _np(t):
    return t.float().cpu().numpy()


def _check_attention(q, cache, vals, pos, got, **kw):
    want, bound = serve.attention(q.double().numpy(), *vals, pos, **kw)
    eps = torch.finfo(q.dtype).eps / 2
    err = np.abs(got.double().cpu().numpy() - want)
    tol = bound * (1 + eps) + eps * np.abs(want) + 1e-7
    assert np.isfinite(got.float().cpu().numpy()).all()
    worst = (err / tol).max() if err.size else 0.0
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,tokens,kv", [(1, 1, 1), (2, 3, 8), (5, 37, 3)])
def test_append_codes_are_the_oracles(dtype, dim, batch, tokens, kv):
    L = tokens + 20
    k, v = (_rand(batch, tokens, kv, dim, seed=s, dtype=dtype, scale=2.0) for s in (1, 2))
    pos = [(3 * b) % 20 for b in range(batch)]
    c = kv4.Kv4Cache.zeros(batch, kv, L, dim, device=DEV)
    assert kv4.append(k.to(DEV), v.to(DEV), c, _i32(pos)) is None
    for x, codes, scales in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        n, s, m = serve.quantise(x.float().numpy())
        want_c = np.zeros(codes.shape, np.uint8)
        want_s = np.zeros(scales.shape, np.float16)
        for b in range(batch):
            want_c[b, :, pos[b]:pos[b] + tokens] = serve.pack(n)[b].swapaxes(0, 1)
            want_s[b, :, pos[b]:pos[b] + tokens] = np.stack([s, m], -1)[b].swapaxes(0, 1)
        assert np.array_equal(codes.cpu().numpy(), want_c)
        assert np.array_equal(scales.cpu().numpy().view(np.uint16), want_s.view(np.uint16))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_append_rotates_k_and_q(dim, dtype):
    B, T, H, KV, L = 2, 9, 6, 2, 64
    qkv = _rand(B, T, H + 2 * KV, dim, seed=3, dtype=dtype)
    t = _table(L, dim)
    pos = [0, 50]
    c = kv4.Kv4Cache.zeros(B, KV, L, dim, device=DEV)
    q, k, v = qkv.to(DEV).split([H, KV, KV], dim=2)            # strided views of one projection
    qr = kv4.append(k, v, c, _i32(pos), q=q, cos_sin=t.to(DEV))
    at = np.array(pos)[:, None] + np.arange(T)
    x = qkv.float().numpy()
    kr = serve.rotate(x[:, :, H:H + KV], t.numpy(), at)
    want_q = torch.from_numpy(serve.rotate(x[:, :, :H], t.numpy(), at)).to(dtype)
    assert torch.equal(qr.cpu(), want_q)
    kk, vv = kv4.read(c, _i32(pos), T, dtype=FP)
    for got, src in ((kk, kr), (vv, x[:, :, H + KV:])):
        n, s, m = serve.quantise(src)
        want = serve.values(serve.pack(n), np.stack([s, m], -1)).astype(np.float32)
        assert np.array_equal(got.cpu().numpy(), want)


def test_many_fp32_rows():
    """Enough rows for values at the borders of a scale's and a code's rounding."""
    B, T, KV, D = 1, 3000, 4, 128
    k, v = (_rand(B, T, KV, D, seed=s, dtype=FP) for s in (50, 51))
    t = _table(T, D)
    c = kv4.Kv4Cache.zeros(B, KV, T, D, device=DEV)
    kv4.append(k.to(DEV), v.to(DEV), c, _i32([0]), cos_sin=t.to(DEV))
    kr = serve.rotate(k.numpy(), t.numpy(), np.arange(T)[None])
    for src, codes, scales in ((kr, c.k, c.k_scale), (v.numpy(), c.v, c.v_scale)):
        n, s, m = serve.quantise(src)
        assert np.array_equal(scales.cpu().numpy(), np.stack([s, m], -1).swapaxes(1, 2))
        assert np.array_equal(codes.cpu().numpy(), serve.pack(n).swapaxes(1, 2))


def test_quantiser_edges():
    """Constant groups, zeros, an outlier, tiny and huge values, infinities and NaN."""
    x = torch.zeros(1, 8, 1, 64)
    x[0, 1] = 3.0
    x[0, 2] = torch.linspace(-1, 1, 64)
    x[0, 2, 0, 5] = 1e4
    x[0, 3] = torch.linspace(-1, 1, 64) * 1e-6
    x[0, 4] = torch.linspace(-1, 1, 64) * 3e38
    x[0, 5, 0, ::3] = float("inf")
    x[0, 5, 0, 1::3] = -float("inf")
    x[0, 6, 0, 7] = float("nan")
    x[0, 7] = torch.linspace(9.999, 10.001, 64)
    c = kv4.Kv4Cache.zeros(1, 1, 8, 64, device=DEV)
    kv4.append(x.to(DEV), -x.to(DEV), c, _i32([0]))
    for src, codes, scales in ((x, c.k, c.k_scale), (-x, c.v, c.v_scale)):
        n, s, m = serve.quantise(src.numpy())
        assert np.array_equal(codes.cpu().numpy()[0, 0], serve.pack(n)[0, :, 0])
        assert np.array_equal(scales.cpu().numpy()[0, 0], np.stack([s, m], -1)[0, :, 0])
        assert np.isfinite(scales.cpu().numpy()).all()
    k, _ = kv4.read(c, _i32([0]), 8, dtype=HF)
    assert torch.isfinite(k).all()


def test_rows_outside_the_cache():
    """Rows before 0 and from max_len on are dropped by append and zero in read; the neighbours' rows stay."""
    B, T, KV, D, L = 3, 6, 2, 64, 10
    k, v = (_rand(B, T, KV, D, seed=s, dtype=FP) for s in (1, 2))
    c = kv4.Kv4Cache.zeros(B, KV, L, D, device=DEV)
    pos = [-2, 7, 2 ** 31 - 1]
    kv4.append(k.to(DEV), v.to(DEV), c, _i32(pos))
    n, s, m = serve.quantise(k.numpy())
    want = np.zeros((B, KV, L, D // 2), np.uint8)
    want[0, :, 0:4] = serve.pack(n)[0, 2:].swapaxes(0, 1)
    want[1, :, 7:10] = serve.pack(n)[1, :3].swapaxes(0, 1)
    assert np.array_equal(c.k.cpu().numpy(), want)
    kk, vv = kv4.read(c, _i32(pos), T, dtype=FP)
    assert (kk[0, :2] == 0).all() and (kk[1, 3:] == 0).all() and (kk[2] == 0).all() and (vv[2] == 0).all()
    assert (kk[0, 2:] != 0).any()
    kv4.append(k.to(DEV)[:, :0], v.to(DEV)[:, :0], c, _i32(pos))
    assert kv4.read(c, _i32(pos), 0)[0].shape == (B, 0, KV, D)


def test_append_copies_what_is_not_aligned():
    B, T, KV, D, L = 1, 4, 2, 64, 8
    flat = _rand(B * T * KV * D + 3, seed=4).to(DEV)
    k = flat[3:].view(B, T, KV, D)                             # starts at an odd element
    v = _rand(B, T, D, KV, seed=5).to(DEV).transpose(2, 3)     # heads not contiguous
    c, d = (kv4.Kv4Cache.zeros(B, KV, L, D, device=DEV) for _ in range(2))
    kv4.append(k, v, c, _i32([2]))
    kv4.append(k.clone(), v.contiguous(), d, _i32([2]))
    assert all(torch.equal(a, b) for a, b in zip(c, d))


# (batch, tokens, heads, kv heads, dim, max_len): one key, ends inside and at the borders of 16 and 32 keys, several
# splits, query rows below, at and above the tiles of 16 and 128
SHAPES = [(1, 1, 1, 1, 64, 1), (1, 1, 4, 1, 128, 17), (2, 1, 8, 2, 128, 32), (1, 1, 32, 8, 128, 640),
          (3, 1, 6, 2, 64, 333), (1, 1, 32, 1, 128, 200), (2, 5, 12, 4, 64, 131), (1, 16, 4, 4, 128, 16),
          (1, 33, 3, 1, 128, 97), (1, 70, 4, 2, 64, 70), (2, 128, 2, 1, 128, 129), (1, 150, 4, 1, 128, 300),
          (1, 257, 1, 1, 64, 1000), (1, 1, 8, 8, 128, 2500)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention(shape, dtype):
    B, T, H, KV, D, L = shape
    q = _rand(B, T, H, D, seed=6, dtype=dtype)
    cache, vals = _cache(_rand(B, KV, L, D, seed=7, dtype=FP), _rand(B, KV, L, D, seed=8, dtype=FP))
    pos = [max(L - T - 5 * b, 0) for b in range(B)]
    got = kv4.attention(q.to(DEV), cache, _i32(pos))
    _check_attention(q, cache, vals, pos, got)


@pytest.mark.parametrize("tile", [16, 64, 128])
@pytest.mark.parametrize("split", [1, 2, 3, 7, 128])
@pytest.mark.parametrize("shape", [(1, 1, 4, 2, 128, 333), (2, 9, 6, 2, 64, 130), (2, 75, 4, 2, 128, 700)], ids=str)
def test_every_tile_and_split(shape, tile, split, tune):
    """Each kernel on each kind of call, the keys cut into more ranges than there are steps among it."""
    B, T, H, KV, D, L = shape
    tune(kv4_tile=tile, kv4_split=split)
    q = _rand(B, T, H, D, seed=60)
    cache, vals = _cache(_rand(B, KV, L, D, seed=61, dtype=FP), _rand(B, KV, L, D, seed=62, dtype=FP))
    pos, start = [L - T, 37][:B], [3, 50][:B]
    got = kv4.attention(q.to(DEV), cache, _i32(pos), start=_i32(start))
    _check_attention(q, cache, vals, pos, got, start=start)


def test_batch_of_many_lengths():
    """More sequences than a wave has lanes, from one key to thousands: each gets its own steps."""
    B, H, KV, D, L = 70, 4, 2, 64, 4096
    q = _rand(B, 1, H, D, seed=63)
    cache, vals = _cache(_rand(B, KV, L, D, seed=64, dtype=FP), _rand(B, KV, L, D, seed=65, dtype=FP))
    pos = [(L - 1) * i * i // (B - 1) ** 2 for i in range(B)]
    pos[5] = -1
    got = kv4.attention(q.to(DEV), cache, _i32(pos))
    _check_attention(q, cache, vals, pos, got)
    assert (got[5] == 0).all()


@pytest.mark.parametrize("shape", [(4, 1, 8, 2, 128, 300), (4, 6, 6, 2, 64, 300), (4, 90, 4, 1, 128, 300)], ids=str)
@pytest.mark.parametrize("window", [0, 1, 7, 64, 1000])
def test_masks(shape, window):
    """start inside, at and beyond the position (rows without a key), windows shorter and longer than the context,
    positions before 0 and past the cache's end."""
    B, T, H, KV, D, L = shape
    q = _rand(B, T, H, D, seed=9)
    cache, vals = _cache(_rand(B, KV, L, D, seed=10, dtype=FP), _rand(B, KV, L, D, seed=11, dtype=FP))
    pos, start = [L - 1, 150, 40, -3], [0, 100, 44, 0]
    got = kv4.attention(q.to(DEV), cache, _i32(pos), start=_i32(start), window=window)
    _check_attention(q, cache, vals, pos, got, start=start, window=window)
    none = [(b, t) for b in range(B) for t in range(T)
            if max(start[b], pos[b] + t - window + 1 if window else 0, 0) > min(pos[b] + t, L - 1)]
    assert none and all((got[b, t] == 0).all() for b, t in none)


@pytest.mark.parametrize("tokens", [1, 20, 140])
def test_hidden_rows_do_not_matter(tokens):
    """Rows that no query sees may hold anything, NaN scales and infinite minima among it."""
    B, H, KV, D, L = 2, 4, 2, 128, 400
    q = _rand(B, tokens, H, D, seed=12).to(DEV)
    cache, _ = _cache(_rand(B, KV, L, D, seed=13, dtype=FP), _rand(B, KV, L, D, seed=14, dtype=FP))
    pos, start = [100, 211], [9, 0]
    want = kv4.attention(q, cache, _i32(pos), start=_i32(start))
    for s in (cache.k_scale, cache.v_scale):
        for b in range(B):
            s[b, :, pos[b] + tokens:] = float("nan")
            s[b, :, pos[b] + tokens + 1::2] = float("inf")
            s[b, :, :start[b]] = float("nan")
    assert torch.equal(kv4.attention(q, cache, _i32(pos), start=_i32(start)), want)


@pytest.mark.parametrize("tokens", [1, 150])
@pytest.mark.parametrize("scale", [1e-30, 1e-3, 300.0, 1e30])
def test_query_range(tokens, scale):
    """bf16 queries of any size: a power of two moves them into fp16's range."""
    q = (_rand(1, tokens, 2, 64, seed=15).float() * scale).to(BF)
    cache, vals = _cache(_rand(1, 1, 200, 64, seed=16, dtype=FP), _rand(1, 1, 200, 64, seed=17, dtype=FP))
    pos = [200 - tokens]
    got = kv4.attention(q.to(DEV), cache, _i32(pos), scale=0.125 / scale)
    _check_attention(q, cache, vals, pos, got, scale=0.125 / scale)


@pytest.mark.parametrize("tokens", [1, 140])
def test_small_values_keep_their_steps(tokens):
    """Groups whose scale is near fp16's smallest normal number."""
    q = _rand(1, tokens, 2, 128, seed=18)
    cache, vals = _cache(_rand(1, 1, 200, 128, seed=19, dtype=FP), _rand(1, 1, 200, 128, seed=20, dtype=FP) * 1e-3)
    got = kv4.attention(q.float().to(HF).to(DEV), cache, _i32([200 - tokens]))
    _check_attention(q.float().to(HF), cache, vals, [200 - tokens], got)


def test_attention_takes_strides_out_and_streams():
    B, T, H, KV, D, L = 2, 3, 8, 2, 128, 90
    qkv = _rand(B, T, H + 2 * KV, D, seed=21).to(DEV)
    q = qkv[:, :, :H]
    cache, _ = _cache(_rand(B, KV, L, D, seed=22, dtype=FP), _rand(B, KV, L, D, seed=23, dtype=FP))
    pos = _i32([87, 30])
    want = kv4.attention(q.contiguous(), cache, pos)
    assert torch.equal(kv4.attention(q, cache, pos), want)
    swapped = q.transpose(1, 2).contiguous().transpose(1, 2)   # [batch, heads, tokens] in memory
    assert torch.equal(kv4.attention(swapped, tuple(cache), pos), want)
    out = torch.empty_like(want)
    assert kv4.attention(q, cache, pos, out=out).data_ptr() == out.data_ptr() and torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = kv4.attention(q, cache, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)


def test_step_in_a_graph():
    """append + attention captured once and replayed at other positions, with eager work between."""
    B, H, KV, D, L = 2, 8, 2, 128, 600
    cache, ref = (kv4.Kv4Cache.zeros(B, KV, L, D, device=DEV) for _ in range(2))
    qkv = torch.zeros(B, 1, H + 2 * KV, D, dtype=BF, device=DEV)
    pos, t = _i32([0, 300]), _table(L, D).to(DEV)
    q, k, v = qkv.split([H, KV, KV], dim=2)

    def step(c):
        return kv4.attention(kv4.append(k, v, c, pos, q=q, cos_sin=t), c, pos)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(cache)
    for i in range(4):
        qkv.copy_(_rand(*qkv.shape, seed=30 + i))
        pos.copy_(_i32([i, 300 + i]))
        g.replay()
        want = step(ref)
        if i:
            assert torch.equal(out, want)
    assert all(torch.equal(a[1, :, 301:], b[1, :, 301:]) for a, b in zip(cache, ref))


def test_long_cache_offsets():
    """A cache of more than 2^32 bytes of codes: the last sequence's rows are its own."""
    B, KV, D, L = 9, 8, 128, 1 << 20
    cache = kv4.Kv4Cache.zeros(B, KV, L, D, device=DEV)
    assert cache.k.numel() > 1 << 32
    q = _rand(B, 1, 8, D, seed=40).to(DEV)
    k, v = (_rand(B, 40, KV, D, seed=s).to(DEV) for s in (41, 42))
    pos = _i32([L - 40] * B)
    kv4.append(k, v, cache, pos)
    got = kv4.attention(q, cache, _i32([L - 1] * B), start=pos)
    kk, vv = kv4.read(cache, pos, 40, dtype=FP)
    small = kv4.Kv4Cache.zeros(B, KV, 40, D, device=DEV)
    kv4.append(k, v, small, _i32([0] * B))
    assert torch.equal(kk, kv4.read(small, _i32([0] * B), 40, dtype=FP)[0])
    vals = [x.permute(0, 2, 1, 3).double().cpu().numpy() for x in (kk, vv)]
    _check_attention(q.cpu(), cache, vals, [39] * B, got)


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("window", [1000, 1025, 8100, 8191, 8200])
def test_windows_in_a_long_cache(window, tokens):
    """Windows a little shorter than the cache, at lengths where the split of the keys changes."""
    L, D, KV, G = 8300, 64, 1, 4
    k, v = (_rand(1, KV, L, D, seed=s, dtype=FP) for s in (51, 52))
    cache, vals = _cache(k, v)
    q = _rand(1, tokens, KV * G, D, seed=53)
    got = kv4.attention(q.to(DEV), cache, _i32([L - tokens]), window=window)
    _check_attention(q, cache, vals, [L - tokens], got, window=window)
