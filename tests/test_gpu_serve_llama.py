"""The decoder stack over the 4-bit cache, with sampled tokens: prompt and
single-token paths agree, graph and eager steps agree, drawn tokens are the
oracle's."""
import pytest
import torch

from bfloat16x_amd import kv4, llama
from bfloat16x_amd.nn import deploy_bf16x_fused
from oracle import serve

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CFG = llama.LlamaConfig(n_layers=3, hidden=1024, ffn=2048, n_heads=8, n_kv_heads=2, vocab=2000)


def _stack(packed):
    m = llama.LlamaStack(CFG, device=DEV, seed=3)
    if packed:
        deploy_bf16x_fused(m)
    return m


def _ids(n, seed=1):
    return torch.randint(0, CFG.vocab, (n,), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("n", [2, 40, 200])
def test_prompt_and_steps_agree(packed, n):
    """The logits after n tokens, all as a prompt or the last as a step.  The products differ in their order of
    summation: about ten bf16 roundings (2^-9 rms) a layer, so 2^-9 sqrt(30) = 1 % of the logits' norm, and a code of
    the cache that such a difference moves by one step; 5 % allows for both."""
    m = _stack(packed)
    ids = _ids(n)
    a = llama.LlamaRunner(m, 256, 8, kv_bits=4)
    a.prefill(ids)
    want = a.logits.clone()
    b = llama.LlamaRunner(m, 256, 8, kv_bits=4)
    b.prefill(ids[:-1])
    b.token.copy_(ids[-1:])
    b.step()
    assert _rel(b.logits, want) < 0.05
    # a cache row holds the same positions in both
    for ca, cb in zip(a.kv4_caches, b.kv4_caches):
        ka, kb = (kv4.read(c, a.zero_pos, n)[0] for c in (ca, cb))
        assert _rel(ka, kb) < 0.05
        assert (ca.k[:, :, n:] == 0).all()


def test_close_to_the_16_bit_cache():
    """4-bit rows of normal values: steps of about 4.2 sigma / 15, so 8 % of a value's size in K and V (0.28 sigma /
    sqrt(12)); three layers of attention, beside the residual stream, leave less than that in the logits."""
    m = _stack(False)
    ids = _ids(100)
    a, b = (llama.LlamaRunner(m, 256, 4, kv_bits=bits) for bits in (16, 4))
    a.prefill(ids)
    b.prefill(ids)
    assert _rel(b.logits, a.logits) < 0.15
    assert b.kv_bytes_per_step() * 256 == a.kv_bytes_per_step() * 80


@pytest.mark.parametrize("packed", [False, True])
def test_graph_and_eager_steps_agree(packed):
    m = _stack(packed)
    ids = _ids(50)
    kw = dict(kv_bits=4, sample=dict(temperature=0.9, top_k=100, top_p=0.95, min_p=0.01), seed=7)
    a = llama.LlamaRunner(m, 128, 20, **kw)
    want = a.generate(ids, 20, graph=False)
    a.prefill(ids)
    a.capture()
    assert a.generate(ids, 20) == want
    assert a.generate(ids, 20) == want


@pytest.mark.parametrize("bits", [16, 4])
def test_drawn_tokens_are_the_oracles(bits):
    m = _stack(False)
    s = dict(temperature=1.2, top_k=300, top_p=0.9, min_p=0.001)
    r = llama.LlamaRunner(m, 128, 12, kv_bits=bits, sample=s)
    u = torch.rand(12, generator=torch.Generator().manual_seed(5))
    r.uniform.copy_(u)
    r.prefill(_ids(30))
    for i in range(12):
        want, _ = serve.sample(r.logits.float().cpu().numpy(), u[i].item(), s["temperature"], s["top_k"], s["top_p"],
                               s["min_p"])
        assert r.token.item() == want and r.history[i].item() == want
        assert r.state.tolist() == [30 + i, i + 1]
        if i < 11:
            r.step()


def test_temperature_zero_is_greedy():
    m = _stack(True)
    ids = _ids(20)
    want = llama.LlamaRunner(m, 64, 10).generate(ids, 10, graph=False)
    assert llama.LlamaRunner(m, 64, 10, sample=dict(temperature=0.0)).generate(ids, 10, graph=False) == want


def test_runner_refuses():
    m = _stack(False)
    for bad in (dict(kv_bits=8), dict(sample=dict(beams=2)), dict(max_len=20000)):
        with pytest.raises(ValueError):
            llama.LlamaRunner(m, **(dict(max_len=64, max_new=4) | bad))
    llama.LlamaRunner(m, 20000, 4, max_prompt=16, kv_bits=4)
