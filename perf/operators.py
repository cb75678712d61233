"""Cases of the serving operators: the 4-bit KV cache (append, read back, attention over it) and token sampling.

Formats and formulas, as include/bf16x_llama.h has them:

  cache    codes uint8 [batch, kv_heads, max_len, D / 2], scales fp16 [batch, kv_heads, max_len, D / 32, 2] = (scale,
           minimum) of each group of 32 values of a row; value = minimum + scale * code.  The 8 codes of values 8w ..
           8w + 7 are the 4-byte word w of a row: value 8w + 2i at bits 4i, value 8w + 2i + 1 at bits 16 + 4i.
  append   minimum = fp16(min x), scale = fp16(max(0, max x - minimum) / 15), code = round((x - minimum) / scale) cut to
           0 .. 15 (0 where the scale is 0), x the row after the rotary embedding where one is given
  attend   out = softmax(scale q . K) V over keys j with start <= j, p - window < j <= p for the query at position p; a
           query with no key gives zeros
  sample   w = exp((x - max x) / T); keep the first top_k by (x, then lower index), of those the shortest prefix with
           top_p of their weight, of those w >= min_p; the token is the first kept one, by index, at which the running
           weight passes u times the kept weight; T = 0 takes the maximum
"""
import math

import torch

own = False
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

LISTED = [
    # one new token of one conversation: rotary embedding, K and V of 8 heads into the cache; all launch and host time
    dict(name="append 1 token", kind="append", batch=1, tokens=1, heads=32, kv=8, dim=128, max_len=640, rope=True,
         type="bf16"),
    # a long prompt's K and V, the queries rotated with them
    dict(name="append prompt 2048", kind="append", batch=1, tokens=2048, heads=32, kv=8, dim=128, max_len=4096,
         rope=True, type="bf16"),
    # continued prompts of a batch, rows rotated elsewhere, half-size heads
    dict(name="append 16x37 dim 64", kind="append", batch=16, tokens=37, heads=16, kv=4, dim=64, max_len=1000,
         rope=False, type="fp16"),
    # a decode step of the 512 + 128 token generation
    dict(name="attend 1x1 at 640", kind="attend", batch=1, tokens=1, heads=32, kv=8, dim=128, max_len=640, window=0,
         padded=False, type="bf16"),
    # a decode step at the longest cache of the decoder stack
    dict(name="attend 1x1 at 16384", kind="attend", batch=1, tokens=1, heads=32, kv=8, dim=128, max_len=16384,
         window=0, padded=False, type="bf16"),
    # a decode batch of conversations of many lengths, left-padded
    dict(name="attend 32x1 at 8192", kind="attend", batch=32, tokens=1, heads=32, kv=8, dim=128, max_len=8192,
         window=0, padded=True, type="fp16"),
    # a few drafted tokens per sequence checked at once, three query heads to a KV head, sliding window
    dict(name="attend 7x5 at 1531 dim 64", kind="attend", batch=7, tokens=5, heads=12, kv=4, dim=64, max_len=1531,
         window=1000, padded=False, type="bf16"),
    # the 512-token prompt
    dict(name="attend prompt 512", kind="attend", batch=1, tokens=512, heads=32, kv=8, dim=128, max_len=512, window=0,
         padded=False, type="bf16"),
    # a 2011-token chunk of a long prompt that is in the cache already
    dict(name="attend chunk 2011 at 8192", kind="attend", batch=1, tokens=2011, heads=32, kv=8, dim=128, max_len=8192,
         window=0, padded=False, type="bf16"),
    # the sampled token of one conversation
    dict(name="sample 1 row", kind="sample", rows=1, vocab=128256, type="bf16", filters="all"),
    # a small batch over an odd vocabulary, temperature and min-p only
    dict(name="sample 9x32003", kind="sample", rows=9, vocab=32003, type="fp16", filters="min_p"),
    # a large batch, each row with its own settings
    dict(name="sample 128 rows fp32", kind="sample", rows=128, vocab=128256, type="fp32", filters="mixed"),
]


def listed():
    return [dict(c) for c in LISTED]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "sample", "sample"])
    if kind == "sample":
        vocab = _log(rng, 1000, 128256)
        rows = min(_log(rng, 1, 128), 128 * 128256 // vocab)
        return dict(kind=kind, rows=rows, vocab=vocab, type=rng.choice(["bf16", "fp16", "fp32"]),
                    filters=rng.choice(["all", "min_p", "mixed", "top_k", "top_p"]))
    dim = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    type_ = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "append":
        batch = _log(rng, 1, 32)
        tokens = rng.choice([1, _log(rng, 1, max(2, 2048 // batch))])
        return dict(kind=kind, batch=batch, tokens=tokens, heads=heads, kv=kv, dim=dim,
                    max_len=tokens + _log(rng, 1, 2048), rope=rng.random() < 0.7, type=type_)
    if rng.random() < 0.6:                                      # single tokens, or a few
        tokens, batch, max_len = rng.choice([1, 1, rng.randrange(2, 9)]), _log(rng, 1, 32), _log(rng, 16, 8192)
    else:                                                       # a prompt or a chunk of one
        tokens, batch = _log(rng, 9, 1500), rng.choice([1, 1, 2])
        max_len = tokens + rng.choice([0, _log(rng, 1, 4096)])
    max_len = max(max_len, tokens)
    return dict(kind=kind, batch=batch, tokens=tokens, heads=heads, kv=kv, dim=dim, max_len=max_len,
                window=rng.choice([0, 0, 0, _log(rng, 8, 4096)]), padded=rng.random() < 0.3, type=type_)


def _gen(seed, k):
    return torch.Generator(device=DEV).manual_seed(1_000_003 * (seed + 1) + k)


def _lengths(case):
    """Position of the first new token of each sequence: the cache's end for one, spread evenly below it for a batch
    (short conversations, then longer ones)."""
    last = case["max_len"] - case["tokens"]
    return [last * (i + 1) // case["batch"] for i in range(case["batch"])]


def _starts(case, lengths):
    return [n * (i % 4) // 8 if case["padded"] else 0 for i, n in enumerate(lengths)]


def _kv(shape, g):
    """Keys: channels of their own offset and spread, a few of them large; values: plain normal."""
    kv, dim = shape[-2], shape[-1]
    off = torch.randn(kv, dim, generator=g, device=DEV)
    spread = torch.exp(0.5 * torch.randn(kv, dim, generator=g, device=DEV))
    big = torch.rand(kv, dim, generator=g, device=DEV) < 0.03
    off = torch.where(big, off * 4.0, off * 0.5)
    k = torch.randn(shape, generator=g, device=DEV) * spread + off
    return k, torch.randn(shape, generator=g, device=DEV) * 0.7


def _table(max_len, dim):
    inv = 5e5 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim)
    a = torch.arange(max_len, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], dim=-1).to(torch.float32)


# value 8w + e of a row: bits _SHIFT[e] of word w
_SHIFT = [0, 16, 4, 20, 8, 24, 12, 28]


def _pack(code):
    """Codes [..., D] (int32) as bytes [..., D / 2]."""
    w = code.to(torch.int32).reshape(*code.shape[:-1], -1, 8) << torch.tensor(_SHIFT, dtype=torch.int32, device=DEV)
    return w.sum(-1, dtype=torch.int32).view(torch.uint8)


def _quantised(x):
    """Codes (int32 [..., D]) and (scale, minimum) pairs (fp16 [..., D / 32, 2]) of x (fp32 [..., D])."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    low = g.amin(-1, keepdim=True).to(torch.float16)
    scale = ((g.amax(-1, keepdim=True) - low.float()).clamp_min(0.0) / 15.0).to(torch.float16)
    code = torch.round((g - low.float()) / scale.float()).clamp(0, 15)
    code = torch.where(scale > 0, code, torch.zeros_like(code)).to(torch.int32).reshape(x.shape)
    return code, torch.cat([scale, low], dim=-1)


def _values(packed, scales):
    """Values (fp32 [..., D]) of packed codes and their scales."""
    word = packed.view(torch.int32)[..., None]
    code = (word >> torch.tensor(_SHIFT, dtype=torch.int32, device=DEV)) & 15
    s = scales.float()
    g = code.float().reshape(*scales.shape[:-1], 32)
    return (g * s[..., 0:1] + s[..., 1:2]).reshape(*packed.shape[:-1], -1)


def _settings(case, g):
    """(temperature, top_k, top_p, min_p) of the rows: numbers, or with "mixed" tensors."""
    kind, rows = case["filters"], case["rows"]
    if kind == "all":
        return 0.8, 50, 0.95, 0.02
    if kind == "min_p":
        return 1.0, 0, 1.0, 0.05
    if kind == "top_k":
        return 0.7, 40, 1.0, 0.0
    if kind == "top_p":
        return 1.0, 0, 0.9, 0.0

    def pick(values, dtype):
        at = torch.randint(0, len(values), (rows,), generator=g, device=DEV)
        return torch.tensor(values, dtype=dtype, device=DEV)[at]

    return (pick([0.0, 0.6, 0.8, 1.0, 1.3], torch.float32), pick([0, 0, 20, 50, 1000], torch.int32),
            pick([1.0, 1.0, 0.95, 0.9, 0.5], torch.float32), pick([0.0, 0.0, 0.02, 0.1], torch.float32))


@torch.no_grad()
def prepare(case, seed):
    g = _gen(seed, 1)
    s = dict(case=case, kind=case["kind"])
    t = TYPES[case["type"]]
    if case["kind"] == "sample":
        x = torch.randn(case["rows"], case["vocab"], generator=g, device=DEV) * 2.5
        peak = torch.rand(x.shape, generator=g, device=DEV) < 8.0 / case["vocab"]     # a few likely continuations
        s["logits"] = torch.where(peak, x.abs() + 9.0, x).to(t)
        s["u"] = torch.rand(case["rows"], generator=g, device=DEV)
        s["settings"] = _settings(case, g)
        return s
    B, T, KV, D = case["batch"], case["tokens"], case["kv"], case["dim"]
    order = torch.randperm(B, generator=g, device=DEV)
    lengths = _lengths(case)
    s["pos"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)[order].contiguous()
    s["q"] = torch.randn(B, T, case["heads"], D, generator=g, device=DEV).to(t)
    if case["kind"] == "append":
        k, v = _kv((B, T, KV, D), g)
        # one projection's rows [q heads | k heads | v heads], as a model hands them over
        s["qkv"] = torch.cat([s["q"], k.to(t), v.to(t)], dim=2).contiguous()
        s["cache"] = tuple(torch.zeros(B, KV, case["max_len"], *tail, dtype=d, device=DEV) for tail, d in
                           (((D // 2,), torch.uint8), ((D // 32, 2), torch.float16)) * 2)
        s["table"] = _table(case["max_len"], D) if case["rope"] else None
        return s
    s["start"] = torch.tensor(_starts(case, lengths), dtype=torch.int32, device=DEV)[order].contiguous() \
        if case["padded"] else None
    k, v = _kv((B, case["max_len"], KV, D), g)
    cache = []
    for x in (k, v):
        code, scales = _quantised(x.to(t).float().transpose(1, 2).contiguous())
        cache += [_pack(code), scales]
    s["cache"] = tuple(cache)
    return s


def _rotated(x, table, rows):
    """x [B, T, heads, D] (fp32) at the positions `rows` [B, T]: pairs (i, i + D / 2)."""
    c, n = table[rows][:, :, None, :, 0], table[rows][:, :, None, :, 1]
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * c - b * n, b * c + a * n], dim=-1)


def _append(s):
    case, t = s["case"], s["q"].dtype
    H, KV = case["heads"], case["kv"]
    rows = s["pos"].long()[:, None] + torch.arange(case["tokens"], device=DEV)
    q, k, v = (x.float() for x in s["qkv"].split([H, KV, KV], dim=2))
    if s["table"] is not None:
        q, k = _rotated(q, s["table"], rows), _rotated(k, s["table"], rows)
    at = (torch.arange(case["batch"], device=DEV)[:, None], slice(None), rows)
    got = []
    for x, codes, scales in ((k, *s["cache"][:2]), (v, *s["cache"][2:])):
        code, sc = _quantised(x)
        codes[at], scales[at] = _pack(code), sc
        got.append(_values(codes[at], scales[at]).to(t))
    return (*got, q.to(t))


def _attend(s):
    case, q, pos = s["case"], s["q"], s["pos"].long()
    B, T, H, D = q.shape
    KV, L = case["kv"], case["max_len"]
    k, v = _values(*s["cache"][:2]), _values(*s["cache"][2:])                         # [B, KV, L, D]
    p = pos[:, None] + torch.arange(T, device=DEV)                                    # [B, T]
    j = torch.arange(L, device=DEV)
    ok = j <= p[..., None]
    if case["window"]:
        ok &= j > p[..., None] - case["window"]
    if s["start"] is not None:
        ok &= j >= s["start"][:, None, None]
    qg = q.float().reshape(B, T, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(B, KV, -1, D)
    x = (qg @ k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    x = x.reshape(B, KV, H // KV, T, L).masked_fill(~ok[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m > -math.inf, m, torch.zeros_like(m)))
    n = e.sum(-1, keepdim=True)
    o = (e.reshape(B, KV, -1, L) @ v).reshape(B, KV, H // KV, T, D) / torch.where(n > 0, n, torch.ones_like(n))
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(q.dtype)


def _column(value, rows, dtype):
    return value.to(dtype)[:, None] if isinstance(value, torch.Tensor) else \
        torch.full((rows, 1), value, dtype=dtype, device=DEV)


def _sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    temp, top_k, top_p, min_p = (_column(v, rows, torch.int64 if i == 1 else torch.float32)
                                 for i, v in enumerate(s["settings"]))
    top_k = torch.where(top_k > 0, top_k, torch.full_like(top_k, vocab))
    top_k = torch.where(temp > 0, top_k, torch.ones_like(top_k))                      # T = 0: the maximum alone
    m = x.amax(-1, keepdim=True)
    w = torch.exp((x - m) / torch.where(temp > 0, temp, torch.ones_like(temp)).double())
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    kept = torch.where(torch.arange(vocab, device=DEV) < top_k, ws, torch.zeros_like(ws))
    c = kept.cumsum(-1)
    before = torch.nn.functional.pad(c[:, :-1], (1, 0))
    ok = (kept > 0) & ((before < top_p.double() * c[:, -1:]) | (top_p >= 1.0)) & (ws >= min_p.double())
    kept = torch.zeros_like(w).scatter(1, order, torch.where(ok, kept, torch.zeros_like(kept)))
    c = kept.cumsum(-1)
    total = c[:, -1:]
    token = (c <= s["u"].double()[:, None] * total).sum(-1, keepdim=True).clamp_max(vocab - 1)
    return token[:, 0], torch.log(kept.gather(1, token) / total)[:, 0].float()


@torch.no_grad()
def run(s):
    if own:
        from bfloat16x_amd import kv4, sampling
        if s["kind"] == "append":
            H, KV = s["case"]["heads"], s["case"]["kv"]
            q, k, v = s["qkv"].split([H, KV, KV], dim=2)
            q = kv4.append(k, v, s["cache"], s["pos"], q=q, cos_sin=s["table"]) if s["table"] is not None else \
                kv4.append(k, v, s["cache"], s["pos"]) or q
            return (*kv4.read(s["cache"], s["pos"], s["case"]["tokens"], dtype=k.dtype), q)
        if s["kind"] == "attend":
            return kv4.attention(s["q"], s["cache"], s["pos"], start=s["start"], window=s["case"]["window"])
        temp, top_k, top_p, min_p = s["settings"]
        return sampling.sample(s["logits"], s["u"], temperature=temp, top_k=top_k, top_p=top_p, min_p=min_p)
    return {"append": _append, "attend": _attend, "sample": _sample}[s["kind"]](s)


def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": n * size + case["rows"] * 32, "flops": 4 * n}
    B, T, H, KV, D = (case[k] for k in ("batch", "tokens", "heads", "kv", "dim"))
    row = KV * (D // 2 + D // 32 * 4)                           # a token's K (or V) codes and scales
    if case["kind"] == "append":
        # q, k and v read, the rotated q, the cache rows and (read back) the values they stand for written
        q = B * T * H * D * 2 * 2 if case["rope"] else 0
        return {"bytes": q + B * T * (2 * KV * D * 2 * 2 + 2 * row),
                "flops": B * T * D * (KV * 12 + (3 * (H + KV) if case["rope"] else 0))}
    rows = pairs = 0
    lengths = _lengths(case)
    for n, start in zip(lengths, _starts(case, lengths)):
        first = [max(start, n + t + 1 - case["window"] if case["window"] else 0) for t in range(T)]
        rows += max(0, n + T - first[0])
        pairs += sum(max(0, n + t + 1 - first[t]) for t in range(T))
    return {"bytes": 2 * B * T * H * D * 2 + 2 * rows * row, "flops": 4 * D * H * pairs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits

def _exact_values(packed, scales):
    """Byte i of a word holds, low nibble then high, values (0, 2), (4, 6), (1, 3), (5, 7)."""
    b = packed.reshape(*packed.shape[:-1], -1, 4).to(torch.int64)
    lo, hi = b % 16, b // 16
    code = torch.stack([lo[..., 0], lo[..., 2], hi[..., 0], hi[..., 2], lo[..., 1], lo[..., 3], hi[..., 1], hi[..., 3]],
                       dim=-1).reshape(*packed.shape[:-1], -1)
    s = scales.double().repeat_interleave(32, dim=-2)
    return s[..., 1] + s[..., 0] * code.double()


def _exact_quantised(x):
    """The values that the codes of x (fp64 [B, T, heads, D]) stand for."""
    parts = torch.stack(x.split(32, dim=-1), dim=-2)
    low = parts.min(-1, keepdim=True).values.half().double()
    step = ((parts.max(-1, keepdim=True).values - low).clamp(min=0) / 15).half().double()
    n = torch.where(step > 0, ((parts - low) / torch.where(step > 0, step, torch.ones_like(step))).round(),
                    torch.zeros_like(parts)).clamp(0, 15)
    return (low + step * n).flatten(-2)


def _exact_append(s):
    H, KV, D = s["case"]["heads"], s["case"]["kv"], s["case"]["dim"]
    x = s["qkv"].double()
    q, k, v = x[:, :, :H], x[:, :, H:H + KV], x[:, :, H + KV:]
    if s["table"] is not None:
        t = torch.stack([s["table"][p:p + s["case"]["tokens"]] for p in s["pos"].tolist()]).double()[:, :, None]
        turn = torch.view_as_complex(t.contiguous())

        def rotate(y):
            z = torch.complex(y[..., :D // 2].contiguous(), y[..., D // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], dim=-1)

        q, k = rotate(q), rotate(k)
    return _exact_quantised(k), _exact_quantised(v), q


def _exact_attend(s):
    case = s["case"]
    B, T, H, D = s["q"].shape
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device=DEV)
    starts = s["start"].tolist() if s["start"] is not None else [0] * B
    for b, (n, first) in enumerate(zip(s["pos"].tolist(), starts)):
        at = torch.arange(n, n + T, device=DEV)[:, None]
        key = torch.arange(n + T, device=DEV)[None]
        hidden = (key > at) | (key < first)
        if case["window"]:
            hidden |= at - key >= case["window"]
        for h in range(H):
            kh = h // (H // case["kv"])
            k, v = (_exact_values(c[b, kh, :n + T], z[b, kh, :n + T]) for c, z in (s["cache"][:2], s["cache"][2:]))
            x = torch.mm(s["q"][b, :, h].double(), k.t()) / math.sqrt(D)
            x[hidden] = -math.inf
            out[b, :, h] = torch.nan_to_num(torch.softmax(x, dim=-1), nan=0.0) @ v
    return out


def _exact_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    settings = [v.tolist() if isinstance(v, torch.Tensor) else [float(torch.tensor(v, dtype=torch.float32))] * rows
                for v in s["settings"]]
    tokens, logp = [], []
    for r, (u, temp, top_k, top_p, min_p) in enumerate(zip(s["u"].tolist(), *settings)):
        value, index = torch.sort(x[r], descending=True, stable=True)
        n = vocab if top_k <= 0 else min(int(top_k), vocab)
        if temp <= 0:
            n, temp = 1, 1.0
        weight = ((value[:n] - value[0]) / temp).exp()
        if top_p < 1:
            run_ = torch.cumsum(weight, 0)
            n = min(n, int((run_ < top_p * run_[-1]).sum()) + 1)
        n = min(n, int((weight >= min_p).sum()))
        index, place = torch.sort(index[:n])
        weight = weight[place]
        run_ = torch.cumsum(weight, 0)
        at = min(int(torch.searchsorted(run_, u * run_[-1], right=True)), n - 1)
        tokens.append(int(index[at]))
        logp.append(float(torch.log(weight[at] / run_[-1])))
    return torch.tensor(tokens, device=DEV), torch.tensor(logp, dtype=torch.float64, device=DEV)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](s)
