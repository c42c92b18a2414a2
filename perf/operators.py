"""What is timed when the operators of a decoder that drafts tokens and bounds its cache are measured.

Three operators that a serving step uses one after the other:

* ``verify``: tokens that somebody drafted (a small model, or a search in the prompt) are held against the target's
  probabilities, with given random numbers: how many of a request's drafts stand, and the token behind them.
* ``weights``: the attention weights that the step's query rows put on every cached key are added to what each key has
  gathered so far, for the rows that the verification let stand.
* ``evict``: of a cache that has grown beyond its budget, the entries that gathered the most stay, next to the first and the
  latest ones; those that lie beyond the budget move into the places of those that go.

``run`` is one call of one of them, on what a serving program holds: float32 logits in the order of the step's wanted
places, the paged cache with its block tables, the gathered weights and the positions of every cached entry.  The
gathered weights are read from one tensor and written to another, and an eviction only reads cache places behind the
budget and only writes places before it, so that a pass can be made again on the same state.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DEVICE = "cuda:0"
_DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases -------------------------------------------------------------------------------------------------------

def _verify(name, requests, drafts, vocab, proposals="model", top_k=0, greedy=0.0, ragged=False):
    """``proposals``: "model" (a draft model's logits are given) or "lookup" (the drafts alone); ``top_k``: of every second
    request; ``greedy``: the share of requests with temperature 0; ``ragged``: 0 to ``drafts`` drafts a request."""
    c = dict(op="verify", requests=requests, drafts=drafts, vocab=vocab, proposals=proposals, top_k=top_k, greedy=greedy, ragged=ragged)
    return dict(c, name=name) if name else c


def _weights(name, requests, tokens, context, heads, kv_heads, head_dim, page, dtype="bfloat16", ragged=False, counted=False,
             window=0, softcap=0.0, sinks=False, slopes=False):
    """``requests`` bring ``tokens`` rows each behind ``context`` cached tokens (``ragged``: up to so many); ``counted``: only
    the first rows of a request count, as a verification leaves them."""
    c = dict(op="weights", requests=requests, tokens=tokens, context=context, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
             dtype=dtype, ragged=ragged, counted=counted, window=window, softcap=softcap, sinks=sinks, slopes=slopes)
    return dict(c, name=name) if name else c


def _evict(name, layers, requests, length, keep, first, recent, kv_heads, head_dim, page, dtype="bfloat16", ragged=False):
    """``layers`` layers of ``requests`` caches of ``length`` entries (``ragged``: 1 to so many) go down to ``keep``, of which those at
    the ``first`` positions and at the ``recent`` latest are not up for choice."""
    c = dict(op="evict", layers=layers, requests=requests, length=length, keep=keep, first=first, recent=recent, kv_heads=kv_heads,
             head_dim=head_dim, page=page, dtype=dtype, ragged=ragged)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's answer streaming, four drafted tokens a step: all latency
        _verify("verify-1x4", 1, 4, 151936),
        # a few users whose drafts were found in their prompts, some greedy, every second one with a top-k, an odd vocabulary
        _verify("verify-lookup-8", 8, 7, 32003, proposals="lookup", top_k=50, greedy=0.25, ragged=True),
        # a loaded server with a draft model: every logit of the step is read once
        _verify("verify-64x5", 64, 5, 151936, top_k=20),
        # one user's decoded token over a short context: all latency
        _weights("weights-1x1-1k", 1, 1, 1024, 16, 8, 128, 16),
        # a loaded server's verification step: five rows a request, contexts of every length
        _weights("weights-32x5-8k", 32, 5, 8200, 32, 8, 128, 16, ragged=True, counted=True),
        # a few very long contexts, one token each
        _weights("weights-4x1-128k", 4, 1, 131071, 32, 8, 128, 16),
        # a long prompt in one portion
        _weights("weights-prompt-4096", 1, 4096, 0, 32, 8, 128, 16),
        # prompt portions of odd lengths behind what is cached, a window and a sink, heads of 64 channels
        _weights("weights-portions-window", 3, 517, 1500, 16, 4, 64, 32, ragged=True, window=700, sinks=True),
        # the 32-bit path, as one checks a model: bent scores, odd sizes
        _weights("weights-float32", 3, 37, 411, 6, 2, 80, 16, dtype="float32", ragged=True, softcap=20.0),
        # one token too many in every layer of a small model: the eviction of a step at the budget
        _evict("evict-28x1-1025", 28, 1, 1025, 1024, 4, 64, 8, 128, 16),
        # four long prompts go down to an eighth
        _evict("evict-4x4-32k", 4, 4, 32768, 4096, 4, 256, 8, 128, 16),
        # the 32-bit cache, lengths on both sides of the budget, odd sizes
        _evict("evict-float32", 2, 7, 2011, 333, 3, 21, 3, 80, 24, dtype="float32", ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_one(rng):
    op = rng.choice(["verify", "weights", "weights", "evict"])
    if op == "verify":
        return _verify(None, _log_int(rng, 1, 64), rng.randint(0, 8), _log_int(rng, 300, 152064), rng.choice(["model", "lookup"]),
                       rng.choice([0, 0, 1, 20, 50, 1000]), rng.choice([0.0, 0.0, 0.5]), rng.random() < 0.5)
    if op == "weights":
        heads, kv_heads, head_dim = rng.choice([(16, 8, 128), (32, 8, 128), (6, 2, 80), (8, 8, 64), (12, 1, 96), (5, 5, 48), (8, 1, 192)])
        many = rng.random() < 0.4                     # prompt portions, or a few rows a request
        tokens = _log_int(rng, 17, 4096) if many else rng.randint(1, 8)
        requests = rng.randint(1, 4) if many else _log_int(rng, 1, 48)
        context = rng.choice([0, _log_int(rng, 1, 131071), _log_int(rng, 1, 131071)])
        bias = rng.choice(["", "", "softcap", "sinks", "slopes"])
        return _weights(None, requests, tokens, context, heads, kv_heads, head_dim, rng.choice([16, 16, 32, 64, 24]),
                        rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]), rng.random() < 0.6, rng.random() < 0.4,
                        rng.choice([0, 0, _log_int(rng, 5, 4000)]), 30.0 if bias == "softcap" else 0.0, bias == "sinks", bias == "slopes")
    length = _log_int(rng, 2, 60000)
    keep = max(1, min(length, _log_int(rng, 1, 8192)))
    if rng.random() < 0.3:
        keep = max(1, length - rng.randint(1, 8))
    first = rng.randint(0, min(4, keep))
    return _evict(None, rng.randint(1, 8), _log_int(rng, 1, 16), length, keep, first, rng.randint(0, keep - first) // rng.choice([1, 8]),
                  rng.choice([1, 2, 3, 8]), rng.choice([64, 80, 128]), rng.choice([16, 16, 32, 24]), rng.choice(["bfloat16", "bfloat16", "float32"]),
                  rng.random() < 0.5)


def draw(rng):
    """A case of the listed ones' ranges that costs no more than the largest of its operator's (and of its type's: the
    32-bit products have no tensor cores)."""
    limits = {"verify": (3.9e8, 1e13), "weights": (1.1e9, 6.9e10), "float32": (3e8, 1e10), "evict": (4e8, 1e13)}
    while True:
        c = _draw_one(rng)
        w = work(c)
        most = limits["float32"] if c["op"] == "weights" and c["dtype"] == "float32" else limits[c["op"]]
        held = c["requests"] * (c["tokens"] + c["context"]) * c["kv_heads"] * c["head_dim"] if c["op"] == "weights" else 0
        scores = c["requests"] * c["heads"] * c["tokens"] * (c["tokens"] + c["context"]) if c["op"] == "weights" else 0
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and held <= 540e6 and scores <= 540e6:
            return c


# ---- what a serving program has in hand -----------------------------------------------------------------------------------

def _lengths(case, most, least):
    """A request's number of drafts, tokens or cached tokens: ``most``, or where the case is ragged any number from ``least``;
    the same ones for every seed, so that what comes back has one shape."""
    n = case["requests"]
    if not case["ragged"]:
        return [most] * n
    got = torch.randint(least, most + 1, (n,), generator=torch.Generator().manual_seed(17 * n + most)).tolist()
    got[0] = most
    return got


def _tables(lens, page, gen, max_extra=0):
    """Block tables over pages in an order of no kind, -1 behind a request's last page."""
    blocks = [max(1, -(-n // page)) for n in lens]
    pages = sum(blocks) + max_extra
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(lens), max(blocks)), -1, dtype=torch.int32)
    at = 0
    for r, b in enumerate(blocks):
        table[r, :b] = torch.tensor(order[at:at + b], dtype=torch.int32)
        at += b
    return table, pages


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEVICE)


def _cumulated(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"verify": _prepare_verify, "weights": _prepare_weights, "evict": _prepare_evict}[case["op"]](case, host, dev)


def _prepare_verify(case, host, dev):
    R, V = case["requests"], case["vocab"]
    drafts = _lengths(case, case["drafts"], 0)
    starts = _cumulated([n + 1 for n in drafts])
    N = starts[-1]
    D = N - R
    logits = torch.randn(N, V, generator=dev, device=DEVICE) * 2.5
    logits.scatter_add_(1, torch.randint(0, V, (N, 8), generator=dev, device=DEVICE), 6 * torch.rand(N, 8, generator=dev, device=DEVICE))
    greedy = torch.rand(R, generator=host) < case["greedy"]
    temperature = torch.where(greedy, torch.zeros(R), 0.5 + 0.7 * torch.rand(R, generator=host))
    top_k = torch.tensor([min(case["top_k"], V) if r % 2 == 0 else 0 for r in range(R)], dtype=torch.int32)
    # the rows of the step that a draft follows, and each one's request
    rows = [starts[r] + i for r in range(R) for i in range(drafts[r])]
    owner = [r for r in range(R) for _ in range(drafts[r])]
    s = SimpleNamespace(logits=logits, draft_logits=None, row_starts=_i32(starts), temperature=temperature.to(DEVICE),
                        top_k=top_k.to(DEVICE), uniform=torch.rand(N, generator=host).to(DEVICE), num_requests=R,
                        tokens=torch.full((N,), -1, dtype=torch.int32, device=DEVICE), counts=torch.zeros(R, dtype=torch.int32, device=DEVICE))
    if D == 0:
        s.draft_tokens = torch.zeros(0, dtype=torch.int32, device=DEVICE)
        s.draft_logits = torch.zeros(0, V, device=DEVICE) if case["proposals"] == "model" else None
        return s
    target = logits[torch.tensor(rows, device=DEVICE)]
    if case["proposals"] == "model":
        s.draft_logits = target + 0.7 * torch.randn(D, V, generator=dev, device=DEVICE)
        # drawn as the draft model's sampler draws: the largest of logit / temperature plus Gumbel noise
        t = temperature.clamp_min(1e-3).to(DEVICE)[torch.tensor(owner, device=DEVICE)][:, None]
        noise = -torch.log(-torch.log(torch.rand(D, V, generator=dev, device=DEVICE).clamp(1e-9, 1 - 1e-7)))
        s.draft_tokens = (s.draft_logits / t + noise).argmax(1).to(torch.int32)
    else:
        found = target.argmax(1)
        other = torch.randint(0, V, (D,), generator=dev, device=DEVICE)
        s.draft_tokens = torch.where(torch.rand(D, generator=dev, device=DEVICE) < 0.7, found, other).to(torch.int32)
    return s


def _prepare_weights(case, host, dev):
    R, Hq, Hkv, D, P = case["requests"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    dt = _DTYPES[case["dtype"]]
    q_lens = _lengths(case, case["tokens"], 1)
    ctx_lens = _lengths(case, case["context"], min(1, case["context"]))
    totals = [q + c for q, c in zip(q_lens, ctx_lens)]
    table, pages = _tables(totals, P, host, 1)
    T, cap, slots = sum(q_lens), max(totals) + 5, R + 2
    kv = torch.randn(pages, 2, Hkv, P, D, generator=dev, device=DEVICE, dtype=dt)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=dev, device=DEVICE, dtype=dt) * 1.5
    slot_ids = torch.randperm(slots, generator=host)[:R].to(torch.int32)
    positions = [c + i for q, c in zip(q_lens, ctx_lens) for i in range(q)]
    counted = [int(torch.randint(1, q + 1, (1,), generator=host)) for q in q_lens] if case["counted"] else None
    weights = torch.rand(slots, Hkv, cap, generator=dev, device=DEVICE) * 3
    ctx = SimpleNamespace(num_tokens=T, num_reqs=R, dtype=dt, page_size=P, positions=_i32(positions), cu_q=_i32(_cumulated(q_lens)),
                          ctx_lens=_i32(ctx_lens), slot_ids=slot_ids.to(DEVICE), q_lens_host=q_lens, ctx_lens_host=ctx_lens,
                          max_q_len=max(q_lens))
    return SimpleNamespace(
        ctx=ctx, qkv=qkv, kv_pages=kv, block_tables=table.to(DEVICE), weights=weights, out=torch.zeros_like(weights),
        positions=torch.full((slots, Hkv, cap), -1, dtype=torch.int32, device=DEVICE), counted=_i32(counted) if counted else None,
        sinks=torch.randn(Hq, generator=host).to(DEVICE) if case["sinks"] else None,
        slopes=(2.0 ** (-8.0 * torch.arange(1, Hq + 1) / Hq)).to(torch.float32).to(DEVICE) if case["slopes"] else None,
        scale=D ** -0.5, window=case["window"], softcap=case["softcap"], heads=Hq, kv_heads=Hkv, head_dim=D)


def _prepare_evict(case, host, dev):
    S, R, Hkv, D, P = case["layers"], case["requests"], case["kv_heads"], case["head_dim"], case["page"]
    dt = _DTYPES[case["dtype"]]
    lens = _lengths(case, case["length"], 1)
    table, pages = _tables(lens, P, host, 1)
    cap, slots = max(max(lens), case["keep"]) + 3, R + 1
    # what entries gather is spread over some orders of magnitude, with ties: entries that no query ever looked at
    weights = torch.exp(1.5 * torch.randn(S, slots, Hkv, cap, generator=dev, device=DEVICE))
    weights = weights * (torch.rand(S, slots, Hkv, cap, generator=dev, device=DEVICE) > 0.03)
    # entries that an earlier eviction moved do not lie in the order of their positions
    positions = torch.argsort(torch.rand(S, slots, Hkv, cap, generator=dev, device=DEVICE), dim=-1).to(torch.int32)
    return SimpleNamespace(
        cache=torch.randn(S, pages, 2, Hkv, P, D, generator=dev, device=DEVICE, dtype=dt), block_tables=table.to(DEVICE),
        slot_ids=torch.randperm(slots, generator=host)[:R].to(torch.int32).to(DEVICE), lens=_i32(lens), lens_host=lens, weights=weights,
        positions=positions, weights_out=torch.zeros_like(weights), positions_out=torch.zeros_like(positions),
        keep=case["keep"], first=case["first"], recent=case["recent"])


# ---- one pass -----------------------------------------------------------------------------------------------------------

def run(s):
    if hasattr(s, "logits"):
        return _verify_own(s) if own else _verify_plain(s)
    if hasattr(s, "qkv"):
        return _weights_own(s) if own else _weights_plain(s)
    return _evict_own(s) if own else _evict_plain(s)


def _scratch(shape, dtype):
    return torch.empty(shape, dtype=dtype, device=DEVICE)


def _verify_own(s):
    from qwen_engine_b200 import ops
    ops.verify_drafts(s.logits, s.draft_tokens, s.draft_logits, s.row_starts, s.temperature, s.top_k, s.uniform, s.tokens, s.counts, _scratch)
    return {"tokens": s.tokens, "counts": s.counts}


def _weights_own(s):
    from qwen_engine_b200 import ops
    ops.accumulate_attention(s.qkv, s.kv_pages, s.block_tables, s.ctx, s.weights, s.out, s.scale, s.window, s.heads, s.kv_heads,
                             s.head_dim, _scratch, positions=s.positions, counted=s.counted, slopes=s.slopes, softcap=s.softcap, sinks=s.sinks)
    return {"weights": s.out, "positions": s.positions}


def _evict_own(s):
    from qwen_engine_b200 import ops
    ops.evict_tokens(s.cache, s.block_tables, s.slot_ids, s.lens, s.weights, s.positions, s.weights_out, s.positions_out, s.keep,
                     s.first, s.recent, _scratch)
    return {"cache": s.cache, "weights": s.weights_out, "positions": s.positions_out}


def _probabilities(logits, temperature, top_k):
    """softmax of the logits at or above the row's top_k-th largest, divided by the row's temperature; one-hot at the first
    largest logit where the temperature is 0.  In 64 bits: a token is where a running sum over the vocabulary crosses a given
    number, and the sums of 32-bit terms put that border elsewhere for one row in some thousands."""
    V = logits.shape[1]
    k = torch.where((top_k > 0) & (top_k < V), top_k, torch.full_like(top_k, V))
    ranked = logits.sort(dim=1, descending=True).values
    least = ranked.gather(1, (k - 1)[:, None])
    x = logits.double()
    t = torch.where(temperature > 0, temperature, torch.ones_like(temperature)).double()[:, None]
    e = torch.exp((x - x.amax(1, keepdim=True)) / t) * (logits >= least)
    p = e / e.sum(1, keepdim=True)
    greedy = torch.zeros_like(p).scatter_(1, logits.argmax(1, keepdim=True), 1.0)
    return torch.where((temperature > 0)[:, None], p, greedy)


def _verify_plain(s):
    N, V = s.logits.shape
    R, D = s.num_requests, N - s.num_requests
    starts = s.row_starts.long()
    row = torch.arange(N, device=s.logits.device)
    owner = torch.searchsorted(starts[1:], row, right=True)
    last = torch.zeros(N, dtype=torch.bool, device=row.device)
    last[starts[1:] - 1] = True
    p = _probabilities(s.logits, s.temperature[owner], s.top_k[owner].long())
    draft_of = row - owner                                        # the index of the draft behind a row, where there is one
    rows = row[~last]
    q = torch.zeros_like(p)
    if s.draft_logits is not None:
        q[rows] = _probabilities(s.draft_logits, s.temperature[owner[rows]], s.top_k[owner[rows]].long())
    elif D > 0:
        q[rows] = q[rows].scatter(1, s.draft_tokens.long()[:, None], 1.0)
    hot = s.temperature[owner] <= 0
    token = torch.zeros(N, dtype=torch.long, device=row.device)
    token[rows] = s.draft_tokens.long()
    q = torch.where((hot & ~last)[:, None], torch.zeros_like(q).scatter(1, token[:, None], 1.0), q)
    at = token[:, None]
    stands = (s.uniform.double() * q.gather(1, at)[:, 0] < p.gather(1, at)[:, 0]) & ~last
    # the drafts in front of a request's first that does not stand
    before = torch.cumsum((~stands).long(), 0)
    failed = before - torch.where(starts[owner] > 0, before[(starts[owner] - 1).clamp_min(0)], torch.zeros_like(before))
    accepted = torch.zeros(R, dtype=torch.long, device=row.device).scatter_add_(0, owner, (failed == 0).long())
    # the token behind them, from what the target gives beyond the draft
    here = starts[:-1] + accepted
    left = (p[here] - q[here]).clamp_min(0)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, p[here])
    sums = torch.cumsum(left, 1)
    u = s.uniform.double()[starts[1:] - 1]
    crossed = sums > (u * left.sum(1))[:, None]
    drawn = torch.where(crossed.any(1), crossed.to(torch.int8).argmax(1), p[here].argmax(1))
    out = torch.where(failed == 0, token, torch.full_like(token, -1))
    out[here] = drawn
    s.tokens.copy_(out)
    s.counts.copy_(accepted + 1)
    return {"tokens": s.tokens, "counts": s.counts}


def _weights_plain(s):
    ctx, Hq, Hkv, D, P = s.ctx, s.heads, s.kv_heads, s.head_dim, s.ctx.page_size
    R, G, dev = ctx.num_reqs, s.heads // s.kv_heads, s.qkv.device
    q_lens = (ctx.cu_q[1:] - ctx.cu_q[:-1]).long()
    cached = ctx.ctx_lens.long()
    Tm, Lm = ctx.max_q_len, max(a + b for a, b in zip(ctx.q_lens_host, ctx.ctx_lens_host))
    j, i = torch.arange(Lm, device=dev), torch.arange(Tm, device=dev)
    page = s.block_tables.long()[:, j // P].clamp_min(0)
    k = s.kv_pages[page, 0, :, (j % P).expand(R, -1)].float()                                       # [R, L, Hkv, D]
    row = (ctx.cu_q[:-1].long()[:, None] + i).clamp_max(s.qkv.shape[0] - 1)
    q = s.qkv[row][:, :, :Hq * D].float().view(R, Tm, Hkv, G, D)
    x = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(R, Hkv, G * Tm, D), k.permute(0, 2, 3, 1)) * s.scale
    x = x.view(R, Hkv, G, Tm, Lm)
    if s.softcap > 0:
        x = s.softcap * torch.tanh(x / s.softcap)
    at = cached[:, None] + i                                                                          # a row's place [R, T]
    if s.slopes is not None:
        x = x - s.slopes.view(1, Hkv, G, 1, 1) * (at[:, None, None, :, None] - j).float()
    seen = j <= at[..., None]
    if s.window > 0:
        seen = seen & (j > at[..., None] - s.window)
    x = x.masked_fill(~seen[:, None, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    if s.sinks is not None:
        z = z + torch.exp(s.sinks.view(1, Hkv, G, 1, 1) - m)
    counted = q_lens if s.counted is None else s.counted.long()
    e = e / z * (i < counted[:, None])[:, None, None, :, None]
    gained = e.sum((2, 3))                                                                             # [R, Hkv, L]
    slots = ctx.slot_ids.long()
    old = s.weights[slots][:, :, :Lm]
    new = torch.where(j < cached[:, None, None], old, torch.zeros_like(old)) + gained
    held = (j < (cached + q_lens)[:, None])[:, None]
    s.out[slots, :, :Lm] = torch.where(held, new, s.out[slots][:, :, :Lm])
    note = (j >= cached[:, None]) & (j < (cached + q_lens)[:, None])
    place = (ctx.cu_q[:-1].long()[:, None] + j - cached[:, None]).clamp(0, ctx.num_tokens - 1)
    s.positions[slots, :, :Lm] = torch.where(note[:, None], ctx.positions[place][:, None], s.positions[slots][:, :, :Lm])
    return {"weights": s.out, "positions": s.positions}


def _evict_plain(s):
    L, P, keep = max(s.lens_host), s.cache.shape[4], s.keep
    slots, dev = s.slot_ids.long(), s.cache.device
    w, pos = s.weights[:, slots][..., :L], s.positions[:, slots][..., :L]                             # [S, R, Hkv, L]
    j = torch.arange(L, device=dev)
    held = (j < s.lens.long()[:, None])[None, :, None].expand_as(w)
    latest = torch.where(held, pos, torch.full_like(pos, -1)).amax(-1, keepdim=True)
    safe = held & ((pos < s.first) | (pos > latest - s.recent))
    # those first, then the heaviest of the others, the lowest place among equals
    value = torch.where(safe, torch.full_like(w, float("inf")), torch.where(held, w, torch.full_like(w, -1.0)))
    by = torch.argsort(value, dim=-1, descending=True, stable=True)
    place = torch.empty_like(by).scatter_(-1, by, j.expand_as(by))
    stays = held & (place < keep)
    over = (s.lens.long() > keep)[None, :, None, None]
    stays = torch.where(over, stays, held)
    src = (stays & (j >= keep)).nonzero()                                                              # [moves, (layer, request, head, place)]
    dst = (~stays & held & (j < keep)).nonzero()
    kept = (j < s.lens.clamp_max(keep).long()[:, None])[None, :, None].expand_as(w)
    new_w, new_pos = w.clone(), pos.clone()
    new_w[tuple(dst.unbind(1))] = w[tuple(src.unbind(1))]
    new_pos[tuple(dst.unbind(1))] = pos[tuple(src.unbind(1))]
    s.weights_out[:, slots, :, :L] = torch.where(kept, new_w, s.weights_out[:, slots][..., :L])
    s.positions_out[:, slots, :, :L] = torch.where(kept, new_pos, s.positions_out[:, slots][..., :L])
    table = s.block_tables.long()
    from_page, to_page = table[src[:, 1], src[:, 3] // P], table[dst[:, 1], dst[:, 3] // P]
    s.cache[dst[:, 0], to_page, :, dst[:, 2], dst[:, 3] % P] = s.cache[src[:, 0], from_page, :, src[:, 2], src[:, 3] % P]
    return {"cache": s.cache, "weights": s.weights_out, "positions": s.positions_out}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "verify":
        return _exact_verified(s)
    if case["op"] == "weights":
        return {"weights": _exact_weights(s), "positions": None}
    return {"cache": None, "weights": _exact_evicted(s), "positions": None}


def _exact_verified(s):
    """Request by request and draft by draft, up to the first that does not stand."""
    def chances(x, t, k):
        if t <= 0:
            return torch.nn.functional.one_hot((x == x.max()).nonzero()[0, 0], x.numel()).double()
        x = x.double() / t
        if 0 < k < x.numel():
            x = x.masked_fill(x < x.topk(k).values[-1], -math.inf)
        return torch.softmax(x, 0)

    tokens, counts = torch.full_like(s.tokens, -1), torch.zeros_like(s.counts)
    starts = s.row_starts.tolist()
    for r in range(s.num_requests):
        t, k, n = float(s.temperature[r].double()), int(s.top_k[r]), starts[r + 1] - starts[r] - 1
        for i in range(n + 1):
            p = chances(s.logits[starts[r] + i], t, k)
            if i == n:
                break
            at = starts[r] - r + i
            d = int(s.draft_tokens[at])
            if t > 0 and s.draft_logits is not None:
                q = chances(s.draft_logits[at], t, k)
            else:
                q = torch.nn.functional.one_hot(torch.tensor(d, device=p.device), p.numel()).double()
            if not float(s.uniform[starts[r] + i]) < float(p[d] / q[d]):
                p = torch.relu(p - q) if float(torch.relu(p - q).sum()) > 0 else p
                break
            tokens[starts[r] + i] = d
        counts[r] = i + 1
        total = torch.cumsum(p, 0)
        tokens[starts[r] + i] = int((total > float(s.uniform[starts[r + 1] - 1]) * total[-1]).nonzero()[0, 0])
    return {"tokens": tokens, "counts": counts}


def _exact_weights(s):
    """Request by request and head by head: the softmax's weights, column by column."""
    ctx, P, G = s.ctx, s.ctx.page_size, s.heads // s.kv_heads
    out = s.out.double()
    start = 0
    for r in range(ctx.num_reqs):
        n, c = ctx.q_lens_host[r], ctx.ctx_lens_host[r]
        L, slot = n + c, int(ctx.slot_ids[r])
        rows = n if s.counted is None else int(s.counted[r])
        blocks = s.block_tables[r, :-(-L // P)].long()
        for h in range(s.kv_heads):
            keys = s.kv_pages[blocks, 0, h].reshape(-1, s.head_dim)[:L].double()
            total = torch.zeros(L, dtype=torch.float64, device=keys.device)
            total[:c] = s.weights[slot, h, :c].double()
            for g in range(G):
                head = h * G + g
                for a in range(0, rows, 1024):
                    b = min(rows, a + 1024)
                    queries = s.qkv[start + a:start + b, head * s.head_dim:(head + 1) * s.head_dim].double()
                    score = (queries @ keys.T) * s.scale
                    if s.softcap > 0:
                        score = s.softcap * torch.tanh(score / s.softcap)
                    place = torch.arange(c + a, c + b, device=keys.device)[:, None]
                    key = torch.arange(L, device=keys.device)[None]
                    if s.slopes is not None:
                        score -= s.slopes[head].double() * (place - key)
                    gone = key > place
                    if s.window > 0:
                        gone = gone | (key <= place - s.window)
                    score[gone] = -math.inf
                    if s.sinks is not None:
                        score = torch.cat([score, s.sinks[head].double().expand(b - a, 1)], 1)
                    total += torch.softmax(score, 1)[:, :L].sum(0)
            out[slot, h, :L] = total
        start += n
    return out


def _exact_evicted(s):
    """Row by row, by sorting (weight, place) pairs on the host."""
    out = s.weights_out.double().cpu()
    w, pos = s.weights.double().cpu(), s.positions.cpu()
    for layer in range(w.shape[0]):
        for r, n in enumerate(s.lens_host):
            slot = int(s.slot_ids[r])
            for h in range(w.shape[2]):
                row, at = w[layer, slot, h, :n].tolist(), pos[layer, slot, h, :n].tolist()
                stays = set(range(n))
                if n > s.keep:
                    latest = max(at)
                    stays = {i for i in range(n) if at[i] < s.first or at[i] > latest - s.recent}
                    for i in sorted((i for i in range(n) if i not in stays), key=lambda i: (-row[i], i))[:s.keep - len(stays)]:
                        stays.add(i)
                end = min(n, s.keep)
                holes = [i for i in range(end) if i not in stays]
                for hole, i in zip(holes, sorted(i for i in stays if i >= s.keep)):
                    row[hole] = row[i]
                out[layer, slot, h, :end] = torch.tensor(row[:end], dtype=torch.float64)
    return out.to(s.weights.device)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------

def work(case):
    mean = 0.5 if case["ragged"] else 1.0
    if case["op"] == "verify":
        drafts = case["requests"] * case["drafts"] * mean
        rows = drafts + case["requests"] + (drafts if case["proposals"] == "model" else 0)
        return {"bytes": int(rows * case["vocab"] * 4), "flops": int(rows * case["vocab"] * 4)}
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "weights":
        R, D, Hq, Hkv = case["requests"], case["head_dim"], case["heads"], case["kv_heads"]
        n, c = max(1.0, case["tokens"] * mean), case["context"] * mean
        reach = min(n + c, case["window"] + n) if case["window"] else n + c      # keys that some row sees
        seen = min(c + (n + 1) / 2, case["window"] or c + n)                      # keys that a row sees, on average
        rows = n * (0.5 if case["counted"] else 1.0)
        return {"bytes": int(R * (reach * Hkv * D * size + n * Hq * D * size + (n + c) * Hkv * 8 + n * Hkv * 4)),
                "flops": int(R * rows * Hq * seen * (2 * D + 4))}
    S, R, Hkv, D = case["layers"], case["requests"], case["kv_heads"], case["head_dim"]
    length, keep = case["length"] * mean, case["keep"]
    kept = min(length, keep)
    moves = kept * max(0.0, length - keep) / max(1.0, length)                     # kept entries that lie beyond the budget
    return {"bytes": int(S * R * Hkv * (length * 8 + kept * 8 + moves * 2 * D * size * 2)), "flops": int(S * R * Hkv * length * 4)}
