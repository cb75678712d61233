"""Token sampling on the GPU against the numpy oracle: the same tokens, and their
log-probabilities within fp32's rounding and the masses' steps of 2^-44."""
import math

import numpy as np
import pytest
import torch

from bfloat16x_amd import sampling
from oracle import serve

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _logits(rows, vocab, seed, dtype, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * spread
    x[:, : max(1, vocab // 50)] += 3.0
    return x.to(dtype), torch.rand(rows, generator=g)


def _check(x, u, got, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    tokens, logp = got[0].tolist(), got[1].tolist()
    assert got[0].dtype == torch.int64 and got[1].dtype == torch.float32
    pick = lambda v, r: v[r].item() if isinstance(v, torch.Tensor) else v
    xs = x.float().numpy() if x.dtype != torch.float32 else x.numpy()
    for r in range(len(tokens)):
        t, lp = serve.sample(xs[r], u[r].item(), pick(temperature, r), pick(top_k, r), pick(top_p, r), pick(min_p, r))
        assert tokens[r] == t, (r, tokens[r], t)
        if math.isinf(lp):
            assert logp[r] == lp
        else:
            # the mass's step against the token's weight (>= its probability), the sum's steps, fp32's rounding
            tol = 2.0 ** -45 / math.exp(lp) + x.shape[1] * 2.0 ** -45 + 2.0 ** -23 * abs(lp) + 1e-12
            assert abs(logp[r] - lp) <= tol, (r, logp[r], lp)


FILTERS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=40), dict(top_p=0.9), dict(min_p=0.05),
           dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.02), dict(temperature=1.5, top_k=1000, top_p=0.5),
           dict(top_k=1), dict(top_p=0.0), dict(top_p=1e-6), dict(min_p=1.0), dict(temperature=0.01),
           dict(temperature=50.0, top_p=0.99), dict(temperature=30.0, top_k=3000, top_p=0.9)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kw", FILTERS, ids=str)
def test_filters(kw, dtype):
    x, u = _logits(24, 5003, 1, dtype)
    _check(x, u, sampling.sample(x.to(DEV), u.to(DEV), **kw), **kw)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 7), (5, 63), (1, 4096), (2, 4097), (70, 1000), (1, 128256),
                                        (65, 32003), (1, 1 << 20)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_sizes(rows, vocab, dtype):
    x, u = _logits(rows, vocab, 2, dtype)
    for kw in (dict(temperature=0.9), dict(temperature=1.1, top_k=30, top_p=0.9, min_p=0.01)):
        _check(x, u, sampling.sample(x.to(DEV), u.to(DEV), **kw), **kw)


def test_settings_per_row():
    rows = 40
    x, u = _logits(rows, 3001, 3, torch.bfloat16)
    g = torch.Generator().manual_seed(4)
    pick = lambda vals, dt: torch.tensor(vals, dtype=dt)[torch.randint(0, len(vals), (rows,), generator=g)]
    kw = dict(temperature=pick([0.0, 0.5, 1.0, 2.0], torch.float32), top_k=pick([0, 1, 20, 5000, -3], torch.int32),
              top_p=pick([1.0, 0.9, 0.3], torch.float32), min_p=pick([0.0, 0.1], torch.float32))
    got = sampling.sample(x.to(DEV), u.to(DEV), **{k: v.to(DEV) for k, v in kw.items()})
    _check(x, u, got, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=300), dict(top_p=0.6), dict(top_k=6000, top_p=0.5),
                                dict(top_k=17, top_p=0.5, min_p=0.5)], ids=str)
@pytest.mark.parametrize("levels", [1, 2, 3])
def test_ties(kw, levels):
    """Rows of one, two or three values: more equal logits than the sorted list holds; ties go to the lowest index."""
    vocab = 20011
    g = torch.Generator().manual_seed(5)
    x = torch.randint(0, levels, (6, vocab), generator=g).to(torch.bfloat16)
    u = torch.tensor([0.0, 0.1, 0.37, 0.5, 0.93, 1.0 - 2.0 ** -24])
    _check(x, u, sampling.sample(x.to(DEV), u.to(DEV), **kw), **kw)


@pytest.mark.parametrize("kw", [dict(top_k=700), dict(top_p=0.4), dict(top_k=1500, top_p=0.9), dict(top_k=5, min_p=0.9),
                                dict(min_p=0.999)], ids=str)
@pytest.mark.parametrize("vocab", [300, 513, 1000, 2047, 4096, 4097])
def test_ties_of_every_list_length(kw, vocab):
    """Rows of one value, and of one value and a few larger ones: lists sorted by counting, bitonically, and too long."""
    x = torch.zeros(5, vocab)
    x[1, ::97] = 0.5
    x[2] = -7.25
    x[3, vocab // 2:] = -30.0
    x[4, 3] = 9.0
    u = torch.tensor([0.0, 0.3, 0.999, 0.5, 0.77])
    for dtype in (torch.bfloat16, torch.float32):
        _check(x.to(dtype), u, sampling.sample(x.to(DEV, dtype), u.to(DEV), **kw), **kw)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("center", [0.0, 5.0, -3.0, -20.0])
def test_long_lists(center, dtype):
    """Hundreds to thousands of tokens in a threshold's bins, many of them equal or a rounding step apart; the last row
    has its larger logits at the later tokens."""
    x, u = _logits(6, 50021, 21, torch.float32, spread=1.0)
    x[:, : 50021 // 50] -= 3.0
    x[5] = torch.sort(x[5]).values
    x = (x + center).to(dtype)
    for kw in (dict(top_p=0.7), dict(temperature=1.3, top_p=0.95), dict(top_k=20000), dict(top_k=9000, top_p=0.8),
               dict(temperature=0.9, top_k=12000, top_p=0.9, min_p=0.01), dict(temperature=3.0, top_k=30, top_p=0.99)):
        _check(x, u, sampling.sample(x.to(DEV), u.to(DEV), **kw), **kw)


@pytest.mark.parametrize("spread", [0.01, 0.3, 12.0, 100.0])
def test_spreads(spread):
    """Flat rows (few bins), steep ones (most tokens below all bins)."""
    for dtype in TYPES:
        x, u = _logits(8, 9001, 11, dtype, spread=spread)
        for kw in (dict(), dict(top_k=64), dict(top_p=0.97), dict(temperature=0.05, top_k=5000, top_p=0.99),
                   dict(temperature=20.0, top_p=0.9, min_p=0.3), dict(min_p=1e-5)):
            _check(x, u, sampling.sample(x.to(DEV), u.to(DEV), **kw), **kw)


def test_masked_and_special_rows():
    vocab = 1031
    x, _ = _logits(10, vocab, 6, torch.float32)
    x[0] = -math.inf                                            # nothing to draw
    x[1] = math.nan
    x[2, 5:] = -math.inf
    x[3] = -math.inf
    x[3, 700] = -3e38                                           # one token left
    x[4] = torch.finfo(torch.float32).min
    x[4, 9] = 2.0
    x[5, ::2] = math.nan
    x[6, 100] = x[6, 900] = math.inf                            # only these two
    x[7] = 0.0
    x[7, ::2] = -0.0
    x[8] = torch.finfo(torch.float32).min                       # all masked the finite way: all alike
    x[9, 3:] = torch.finfo(torch.float32).max
    u = torch.tensor([0.5, 0.5, 0.99, 0.5, 0.999, 0.7, 0.6, 0.25, 0.5, 0.5])
    for kw in (dict(), dict(temperature=0.7, top_k=5, top_p=0.9, min_p=0.01), dict(temperature=0.0),
               dict(top_p=0.5), dict(temperature=math.inf), dict(temperature=1e-30, top_k=3)):
        _check(x, u, sampling.sample(x.to(DEV), u.to(DEV), **kw), **kw)


def test_uniform_numbers_at_their_ends():
    x, _ = _logits(6, 500, 7, torch.float16)
    u = torch.tensor([0.0, -1.0, 1.0 - 2.0 ** -24, 1.0, 7.0, math.nan])
    want = u.clone()
    want[5] = 0.0
    for kw in (dict(), dict(top_k=9)):
        _check(x, want, sampling.sample(x.to(DEV), u.to(DEV), **kw), **kw)


def test_strides_vectors_and_outputs():
    x, u = _logits(7, 2003, 8, torch.bfloat16)
    want = sampling.sample(x.to(DEV), u.to(DEV), top_k=50)
    wide = torch.zeros(7, 2051, dtype=torch.bfloat16, device=DEV)
    wide[:, 5:2008] = x.to(DEV)
    got = sampling.sample(wide[:, 5:2008], u.to(DEV), top_k=50)
    cols = sampling.sample(x.t().contiguous().t().to(DEV), u.to(DEV), top_k=50)
    for g in (got, cols):
        assert torch.equal(g[0], want[0]) and torch.equal(g[1], want[1])
    one = sampling.sample(x[3].to(DEV), u[3:4].to(DEV), top_k=50)
    assert one[0].item() == want[0][3].item() and one[1].item() == want[1][3].item()
    token = torch.zeros(7, dtype=torch.int64, device=DEV)
    sampling.sample(x.to(DEV), u.to(DEV), top_k=50, token=token)
    assert torch.equal(token, want[0])
    assert sampling.sample(x.to(DEV)[:0], u.to(DEV)[:0])[0].shape == (0,)
    again = [sampling.sample(x.to(DEV), u.to(DEV), top_k=50)[1] for _ in range(3)]
    assert all(torch.equal(a, want[1]) for a in again)


def test_state_in_a_graph():
    """A captured step draws with u[state[1]], appends to the history and counts, at every replay."""
    vocab, n = 4001, 6
    g = torch.Generator().manual_seed(9)
    u = torch.rand(n, generator=g)
    ud = u.to(DEV)
    x = torch.zeros(vocab, dtype=torch.bfloat16, device=DEV)
    state = torch.tensor([10, 0], dtype=torch.int32, device=DEV)
    history = torch.full((4,), -7, dtype=torch.int32, device=DEV)
    token = torch.zeros(1, dtype=torch.int64, device=DEV)
    kw = dict(temperature=0.9, top_k=200, top_p=0.95)
    step = lambda: sampling.sample(x, ud, token=token, state=state, history=history, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, logp = step()
    state.copy_(torch.tensor([10, 0], dtype=torch.int32))
    want = []
    for i in range(6):
        row, _ = _logits(1, vocab, 20 + i, torch.bfloat16)
        x.copy_(row[0])
        graph.replay()
        t, lp = serve.sample(row[0].float().numpy(), u[i].item(), 0.9, 200, 0.95, 0.0)
        want.append(t)
        assert token.item() == t and abs(logp.item() - lp) < 1e-5
        assert state.tolist() == [11 + i, 1 + i]
    assert history.tolist() == want[:4]
