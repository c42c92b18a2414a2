"""Verification of drafted tokens, gathered attention weights and eviction against their definitions in 64 bits
(tests/plain_drafts.py): types, head layouts, lengths from none and one to long ones, odd sizes, strides, masks, ties."""
import math
import random
from types import SimpleNamespace

import pytest
import torch

import plain_drafts
from qwen_engine_b200 import ops
from qwen_engine_b200.sampling import Sampler, SamplingParams

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _alloc(shape, dtype):
    return torch.empty(shape, dtype=dtype, device=DEV)


# ---- verification ----------------------------------------------------------------------------------------------------------

def _verify_case(R, drafts, V, seed, model=True, top_ks=(0,), temps=(0.8,), scale=2.0):
    g = torch.Generator().manual_seed(seed)
    rnd = random.Random(seed)
    ns = [rnd.choice(drafts) for _ in range(R)]
    starts = [0]
    for n in ns:
        starts.append(starts[-1] + n + 1)
    N = starts[-1]
    logits = torch.randn(N, V, generator=g) * scale
    rows = [starts[r] + i for r in range(R) for i in range(ns[r])]
    draft_logits = logits[rows] + 0.5 * torch.randn(len(rows), V, generator=g) if model else None
    tokens = (draft_logits if model else logits[rows]).add(2 * torch.randn(len(rows), V, generator=g)).argmax(1).to(torch.int32)
    return dict(logits=logits, draft_tokens=tokens, draft_logits=draft_logits, row_starts=torch.tensor(starts, dtype=torch.int32),
                temperature=torch.tensor([rnd.choice(temps) for _ in range(R)]), top_k=torch.tensor([rnd.choice(top_ks) for _ in range(R)], dtype=torch.int32),
                uniform=torch.rand(N, generator=g))


def _verify(c, **other):
    d = {k: (v.to(DEV) if isinstance(v, torch.Tensor) else v) for k, v in {**c, **other}.items()}
    N, R = d["logits"].shape[0], d["temperature"].numel()
    tokens = torch.full((N,), -7, dtype=torch.int32, device=DEV)
    counts = torch.full((R,), -7, dtype=torch.int32, device=DEV)
    ops.verify_drafts(d["logits"], d["draft_tokens"], d["draft_logits"], d["row_starts"], d["temperature"], d["top_k"], d["uniform"],
                      tokens, counts, _alloc)
    return tokens.cpu(), counts.cpu()


def _same(got, want):
    assert torch.equal(got[1], want[1]), (got[1].tolist(), want[1].tolist())
    assert torch.equal(got[0], want[0]), [(i, a, b) for i, (a, b) in enumerate(zip(got[0].tolist(), want[0].tolist())) if a != b][:5]


@pytest.mark.parametrize("model", [True, False])
@pytest.mark.parametrize("R,drafts,V", [(1, [4], 151936), (7, [0, 1, 2, 5], 1001), (33, [3], 130), (3, [0], 389), (2, [40, 1], 77), (5, [2], 1), (9, [1, 3], 2),
                                        (4, [2, 6], 32003)])
def test_verify_drafts(model, R, drafts, V):
    for seed in range(3):
        c = _verify_case(R, drafts, V, 10 * seed + R, model)
        _same(_verify(c), plain_drafts.verify(**c))


@pytest.mark.parametrize("model", [True, False])
@pytest.mark.parametrize("V", [97, 4099, 70001])
def test_verify_drafts_with_top_k_and_greedy_requests(model, V):
    for seed in range(3):
        c = _verify_case(12, [0, 1, 4], V, 77 + seed, model, top_ks=(0, 1, 2, 50, 1000, V, V + 3), temps=(0.0, 0.3, 1.0, 2.5))
        _same(_verify(c), plain_drafts.verify(**c))


def test_verify_drafts_with_ties_at_the_threshold_and_coarse_logits():
    """Logits in steps of a half: many equal the top_k-th largest (all are kept) and many the largest (the lowest place is the argmax)."""
    for seed in range(3):
        c = _verify_case(8, [3], 515, 200 + seed, True, top_ks=(1, 5, 40), temps=(0.0, 0.7))
        c["logits"], c["draft_logits"] = (c["logits"] * 2).round() / 2, (c["draft_logits"] * 2).round() / 2
        c["logits"][:, ::7] *= -0.0
        _same(_verify(c), plain_drafts.verify(**c))


def test_verify_drafts_with_masked_logits():
    """-inf, NaN and the type's lowest value in masked places, rows without any finite logit, +inf, drafts that are masked or outside the vocabulary."""
    low = torch.finfo(torch.float32).min
    for seed in range(4):
        for model in (True, False):
            c = _verify_case(10, [2, 4], 333, 300 + seed, model, top_ks=(0, 3, 30), temps=(0.0, 0.6, 1.0))
            g = torch.Generator().manual_seed(seed)
            N = c["logits"].shape[0]
            for x in [c["logits"]] + ([c["draft_logits"]] if model else []):
                m = torch.rand(x.shape, generator=g)
                x[m < 0.3] = -math.inf
                x[(m >= 0.3) & (m < 0.35)] = math.nan
                x[(m >= 0.35) & (m < 0.5)] = low
            c["logits"][1] = -math.inf
            c["logits"][4] = math.nan
            c["logits"][6] = low
            c["logits"][8, 5] = c["logits"][8, 100] = math.inf
            if model:
                c["draft_logits"][2] = -math.inf
            c["draft_tokens"][3], c["draft_tokens"][5] = 333, -1
            _same(_verify(c), plain_drafts.verify(**c))


def test_verify_drafts_at_the_ends_of_the_uniform_numbers():
    c = _verify_case(6, [3], 501, 5, True)
    for u in (0.0, 1.0 - 2.0 ** -24):
        c["uniform"][:] = u
        _same(_verify(c), plain_drafts.verify(**c))
    # the draft's distribution is the target's: every draft stands, whatever the number
    starts = c["row_starts"].tolist()
    c["draft_logits"] = c["logits"][[starts[r] + i for r in range(6) for i in range(3)]].clone()
    c["uniform"][:] = 1.0 - 2.0 ** -24
    got = _verify(c)
    assert got[1].tolist() == [4] * 6
    _same(got, plain_drafts.verify(**c))


def test_verify_drafts_off_a_16_byte_boundary():
    c = _verify_case(4, [2], 1003, 6, True, top_ks=(0, 9))
    want = plain_drafts.verify(**c)
    for shift in (1, 2, 3):
        def moved(x):
            room = torch.zeros(x.numel() + 4, device=DEV)
            v = room[shift:shift + x.numel()].view(x.shape)
            v.copy_(x)
            return v
        _same(_verify(c, logits=moved(c["logits"]), draft_logits=moved(c["draft_logits"])), want)


@pytest.mark.parametrize("model", [True, False])
def test_verified_tokens_are_distributed_as_the_targets(model):
    """Many requests with one target: the first token each gains (the draft, or the one in its place) has the target's
    probabilities.  A count of n trials is off by 5 standard deviations, sqrt(n p (1 - p)), once in millions."""
    R, V = 20000, 7
    g = torch.Generator().manual_seed(3)
    target, other = torch.randn(V, generator=g) * 1.5, torch.randn(V, generator=g) * 1.5
    q = torch.softmax(other, 0)
    drafts = torch.multinomial(q, R, replacement=True, generator=g).to(torch.int32) if model else torch.full((R,), 2, dtype=torch.int32)
    c = dict(logits=target.expand(2 * R, V).contiguous(), draft_tokens=drafts, draft_logits=other.expand(R, V).contiguous() if model else None,
             row_starts=torch.arange(0, 2 * R + 1, 2, dtype=torch.int32), temperature=torch.ones(R), top_k=torch.zeros(R, dtype=torch.int32),
             uniform=torch.rand(2 * R, generator=g))
    tokens, counts = _verify(c)
    p = torch.softmax(target.double(), 0)
    seen = torch.bincount(tokens[::2].long(), minlength=V).double()
    assert (torch.abs(seen - R * p) <= 5 * torch.sqrt(R * p * (1 - p))).all(), (seen / R, p)
    assert int(tokens[::2].min()) >= 0 and 0.1 < float((counts == 2).double().mean()) < 0.99


def test_verify_drafts_of_very_many_requests():
    """More rows than a grid's second dimension holds: every request is the same one, and so is what it gains."""
    R, V = 40000, 6
    c = _verify_case(1, [1], V, 14, True)
    want = plain_drafts.verify(**c)
    many = dict(logits=c["logits"].repeat(R, 1), draft_tokens=c["draft_tokens"].repeat(R), draft_logits=c["draft_logits"].repeat(R, 1),
                row_starts=torch.arange(0, 2 * R + 1, 2, dtype=torch.int32), temperature=c["temperature"].repeat(R), top_k=c["top_k"].repeat(R),
                uniform=c["uniform"].repeat(R))
    tokens, counts = _verify(many)
    assert (counts == want[1]).all() and (tokens.view(R, 2) == want[0]).all()


def test_verify_drafts_with_extreme_temperatures():
    """Temperatures at which nothing but the largest logits, or all of them alike, have weight; large logits and close ones."""
    c = _verify_case(12, [2], 257, 15, True)
    c["temperature"] = torch.tensor([1e-30, 1e-6, 1e-3, 1e3, 1e6, 1e20, 3e38, 1.0, 0.5, -1.0, 1e-38, 2.0])
    for scale, shift in ((1.0, 0.0), (1e-3, 1e4), (1e6, 0.0), (1e30, 0.0)):
        d = dict(c, logits=c["logits"] * scale + shift, draft_logits=c["draft_logits"] * scale + shift)
        _same(_verify(d), plain_drafts.verify(**d))


def test_verify_drafts_of_a_request_without_rows():
    """It gets no tokens, and the requests in front of it theirs."""
    c = _verify_case(2, [2], 50, 9, True)
    want = plain_drafts.verify(**c)
    c["row_starts"] = torch.tensor([0, 3, 6, 6], dtype=torch.int32)
    c["temperature"], c["top_k"] = torch.cat([c["temperature"], torch.ones(1)]), torch.cat([c["top_k"], torch.zeros(1, dtype=torch.int32)])
    c["draft_tokens"], c["draft_logits"] = c["draft_tokens"][:3], c["draft_logits"][:3]      # (N - R of them)
    tokens, counts = _verify(c)
    assert counts[2] == 0 and counts[0] == want[1][0] and torch.equal(tokens[:3], want[0][:3])


def test_the_sampler_verifies():
    V = 301
    c = _verify_case(4, [0, 2, 3], V, 12, True, top_ks=(0, 20), temps=(0.0, 0.9))
    starts = c["row_starts"].tolist()
    params = [SamplingParams(temperature=float(t), top_k=int(k)) for t, k in zip(c["temperature"], c["top_k"])]
    drafts = [c["draft_tokens"][starts[r] - r:starts[r + 1] - r - 1].tolist() for r in range(4)]
    uniforms = [c["uniform"][starts[r]:starts[r + 1]].tolist() for r in range(4)]
    for model in (True, False):
        dl = c["draft_logits"] if model else None
        tokens, counts = plain_drafts.verify(**{**c, "draft_logits": dl})
        got = Sampler(DEV).verify(c["logits"].to(DEV), params, drafts, uniforms, dl.to(DEV) if model else None)
        assert got == [tokens[starts[r]:starts[r] + counts[r]].tolist() for r in range(4)]
    # no drafts: what the sampler draws
    rows = c["logits"][:4].contiguous().to(DEV)
    got = Sampler(DEV).verify(rows, params, [[]] * 4, [[u] for u in (0.1, 0.4, 0.6, 0.9)])
    assert [t[0] for t in got] == Sampler(DEV).sample(rows, params, [0.1, 0.4, 0.6, 0.9])


# ---- gathered attention weights -------------------------------------------------------------------------------------------------

def _weights_case(dtype, Hq, Hkv, D, P, q_lens, ctx_lens, seed, planes=2, counted=None, extra=3, std=1.0):
    g = torch.Generator().manual_seed(seed)
    R, T = len(q_lens), sum(q_lens)
    totals = [a + b for a, b in zip(q_lens, ctx_lens)]
    blocks = [-(-t // P) for t in totals]
    pages = sum(blocks) + 2
    order = iter(torch.randperm(pages, generator=g).tolist())
    table = torch.full((R, max(blocks) + 1), -1, dtype=torch.int32)
    for r, nb in enumerate(blocks):
        for b in range(nb):
            table[r, b] = next(order)
    cap, slots = max(totals) + extra, R + 2
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    return dict(qkv=(torch.randn(T, (Hq + 2 * Hkv) * D, generator=g) * std).to(dtype), pages=torch.randn(pages, planes, Hkv, P, D, generator=g).to(dtype),
                table=table, cu=torch.tensor(cu, dtype=torch.int32), ctx=torch.tensor(ctx_lens, dtype=torch.int32),
                slots=torch.randperm(slots, generator=g)[:R].to(torch.int32), weights=torch.rand(slots, Hkv, cap, generator=g),
                step_positions=torch.randint(0, 10 ** 6, (T,), generator=g, dtype=torch.int32), q_lens=list(q_lens), ctx_lens=list(ctx_lens),
                counted=None if counted is None else torch.tensor(counted, dtype=torch.int32), heads=(Hq, Hkv, D))


def _context(c, dev=DEV):
    return SimpleNamespace(num_reqs=len(c["q_lens"]), cu_q=c["cu"].to(dev), ctx_lens=c["ctx"].to(dev), slot_ids=c["slots"].to(dev),
                           positions=c["step_positions"].to(dev), q_lens_host=c["q_lens"], ctx_lens_host=c["ctx_lens"],
                           max_q_len=max(c["q_lens"]))


def _rows_on_device(x):
    """The rows on the device with the stride they have here."""
    wide = torch.zeros(x.shape[0], x.stride(0), dtype=x.dtype, device=DEV)
    wide[:, :x.shape[1]] = x.to(DEV)
    return wide[:, :x.shape[1]]


def _gather(c, window=0, in_place=False, **options):
    Hq, Hkv, D = c["heads"]
    w = c["weights"].to(DEV)
    out = w if in_place else torch.full_like(w, -5.0)
    positions = torch.full(w.shape, -9, dtype=torch.int32, device=DEV)
    opts = {k: (v.to(DEV) if isinstance(v, torch.Tensor) else v) for k, v in options.items()}
    ops.accumulate_attention(_rows_on_device(c["qkv"]), c["pages"].to(DEV), c["table"].to(DEV), _context(c), w, out, c.get("scale", D ** -0.5), window,
                             Hq, Hkv, D, _alloc, positions=positions, counted=None if c["counted"] is None else c["counted"].to(DEV), **opts)
    torch.cuda.synchronize()
    return out.cpu(), positions.cpu()


def _check_weights(c, window=0, in_place=False, **options):
    Hq, Hkv, D = c["heads"]
    got, noted = _gather(c, window, in_place, **options)
    before = c["weights"] if in_place else torch.full_like(c["weights"], -5.0)
    want, tol = plain_drafts.gathered(c["qkv"], c["pages"], c["table"], c["cu"], c["ctx"], c["slots"], c["weights"], before,
                                      c.get("scale", D ** -0.5), window, Hq, Hkv, D, c["counted"], **options)
    assert torch.isfinite(got).all()
    over = (got.double() - want).abs() - tol
    assert float(over.max()) <= 0.0, f"{int((over > 0).sum())} of {over.numel()} entries are off, by {float((got.double() - want).abs().max()):.3e}"
    for r in range(len(c["q_lens"])):
        n, k, s = c["q_lens"][r], c["ctx_lens"][r], int(c["slots"][r])
        a = int(c["cu"][r])
        assert (noted[s, :, k:k + n] == c["step_positions"][a:a + n]).all()
        assert (noted[s, :, :k] == -9).all() and (noted[s, :, k + n:] == -9).all()
    return got


LAYOUTS = [(torch.float32, 4, 2, 16, 8), (torch.float32, 6, 2, 80, 24), (torch.bfloat16, 16, 8, 128, 16), (torch.bfloat16, 32, 8, 128, 16),
           (torch.bfloat16, 12, 1, 96, 32), (torch.bfloat16, 5, 5, 48, 16), (torch.bfloat16, 8, 8, 64, 7), (torch.bfloat16, 7, 1, 20, 16),
           (torch.bfloat16, 4, 4, 192, 64), (torch.float32, 3, 1, 33, 5), (torch.bfloat16, 40, 2, 256, 16)]
BATCHES = [([1], [0]), ([1], [77]), ([1, 1, 1], [5, 530, 33]), ([7, 1, 2, 1], [9, 40, 0, 63]), ([40], [25]), ([130, 5], [300, 127]), ([5, 5, 5], [0, 256, 1000])]


@pytest.mark.parametrize("q_lens,ctx_lens", BATCHES)
@pytest.mark.parametrize("dtype,Hq,Hkv,D,P", LAYOUTS)
def test_accumulate_attention(dtype, Hq, Hkv, D, P, q_lens, ctx_lens):
    _check_weights(_weights_case(dtype, Hq, Hkv, D, P, q_lens, ctx_lens, Hq + D))


@pytest.mark.parametrize("dtype,Hq,Hkv,D,P", [(torch.float32, 4, 2, 32, 8), (torch.bfloat16, 16, 4, 128, 16), (torch.bfloat16, 6, 2, 80, 16)])
@pytest.mark.parametrize("q_lens,ctx_lens", [([1, 3, 1], [700, 65, 1]), ([150, 9], [40, 200])])
@pytest.mark.parametrize("option", ["window", "window1", "sinks", "softcap", "slopes", "counted", "counted0", "all"])
def test_accumulate_attention_options(dtype, Hq, Hkv, D, P, q_lens, ctx_lens, option):
    counted = None
    if option == "counted":
        counted = [max(1, n // 2) for n in q_lens]
    if option in ("counted0", "all"):
        counted = [0 if i == 1 else n + 5 for i, n in enumerate(q_lens)]
    c = _weights_case(dtype, Hq, Hkv, D, P, q_lens, ctx_lens, 17, counted=counted)
    g = torch.Generator().manual_seed(4)
    options = {}
    if option in ("sinks", "all"):
        options["sinks"] = torch.randn(Hq, generator=g) * 2
    if option in ("softcap", "all"):
        options["softcap"] = 3.0
    if option in ("slopes", "all"):
        options["slopes"] = torch.rand(Hq, generator=g) * 0.2
    window = {"window": 50, "window1": 1, "all": 33}.get(option, 0)
    _check_weights(c, window=window, **options)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_accumulate_attention_over_a_latent_cache_and_more_planes(dtype):
    for planes, Hq, Hkv, D in ((1, 16, 1, 64), (3, 4, 2, 128), (1, 24, 1, 256)):
        for q_lens, ctx_lens in (([1, 1], [300, 5]), ([60], [100])):
            _check_weights(_weights_case(dtype, Hq, Hkv, D, 16, q_lens, ctx_lens, planes, planes=planes))


def test_accumulate_attention_in_place_and_twice_the_same_bits():
    for q_lens, ctx_lens in (([1, 1], [600, 90]), ([200], [33])):
        c = _weights_case(torch.bfloat16, 8, 2, 128, 16, q_lens, ctx_lens, 8)
        a = _check_weights(c, in_place=True)
        assert torch.equal(a, _check_weights(c, in_place=True))
        apart = _check_weights(c)
        for r in range(len(q_lens)):
            L, s = q_lens[r] + ctx_lens[r], int(c["slots"][r])
            assert torch.equal(apart[s, :, :L], a[s, :, :L])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_lens,ctx_lens", [([1], [200]), ([100], [60])])
def test_accumulate_attention_where_a_page_is_missing_and_garbage_behind_the_end(dtype, q_lens, ctx_lens):
    """Keys that lie in no page get no weight; NaN in places that no row may see (behind the end, in the future of the rows that count) stays there."""
    c = _weights_case(dtype, 4, 2, 128, 16, q_lens, ctx_lens, 21)
    total = q_lens[0] + ctx_lens[0]
    last = int(c["table"][0, (total - 1) // 16])
    if total % 16:
        c["pages"][last, 0, :, total % 16:] = math.nan
    c["table"][0, 3] = -1
    _check_weights(c)


def test_accumulate_attention_takes_strided_rows_and_large_scores():
    for q_lens, ctx_lens in (([1, 2], [100, 30]), ([129], [64])):
        c = _weights_case(torch.bfloat16, 4, 2, 128, 16, q_lens, ctx_lens, 31, std=12.0)
        wide = torch.zeros(c["qkv"].shape[0], c["qkv"].shape[1] + 24, dtype=torch.bfloat16)
        wide[:, :c["qkv"].shape[1]] = c["qkv"]
        c["qkv"] = wide[:, :c["qkv"].shape[1]]
        _check_weights(c)
        odd = torch.zeros(c["qkv"].shape[0], c["qkv"].shape[1] + 3, dtype=torch.bfloat16)     # rows off a 16-byte boundary
        odd[:, :c["qkv"].shape[1]] = c["qkv"]
        c["qkv"] = odd[:, :c["qkv"].shape[1]]
        _check_weights(c)


def test_accumulate_attention_of_a_long_context():
    c = _weights_case(torch.bfloat16, 8, 2, 128, 16, [1, 3], [40000, 1], 41)
    _check_weights(c)
    c = _weights_case(torch.bfloat16, 4, 1, 128, 64, [700], [3000], 42)
    _check_weights(c)


# ---- eviction ------------------------------------------------------------------------------------------------------------------

def _evict_case(dtype, S, Hkv, D, P, lens, seed, planes=2, coarse=False, ordered=False, extra=2):
    g = torch.Generator().manual_seed(seed)
    R = len(lens)
    blocks = [max(1, -(-n // P)) for n in lens]
    pages = sum(blocks) + 1
    order = iter(torch.randperm(pages, generator=g).tolist())
    table = torch.full((R, max(blocks)), -1, dtype=torch.int32)
    for r, nb in enumerate(blocks):
        for b in range(nb):
            table[r, b] = next(order)
    cap, slots = max(lens) + extra, R + 1
    w = torch.exp(1.5 * torch.randn(S, slots, Hkv, cap, generator=g))
    if coarse:
        w = w.round()
    pos = torch.argsort(torch.rand(S, slots, Hkv, cap, generator=g), dim=-1).to(torch.int32)
    if ordered:
        pos = torch.arange(cap, dtype=torch.int32).expand(S, slots, Hkv, cap).contiguous()
    return dict(cache=torch.randn(S, pages, planes, Hkv, P, D, generator=g).to(dtype), table=table,
                slot_ids=torch.randperm(slots, generator=g)[:R].to(torch.int32), lens=torch.tensor(lens, dtype=torch.int32), weights=w, positions=pos)


def _check_evict(c, keep, first, recent, in_place=False):
    d = {k: v.to(DEV) for k, v in c.items()}
    wo = d["weights"] if in_place else torch.full_like(d["weights"], -3.0)
    po = d["positions"] if in_place else torch.full_like(d["positions"], -3)
    want = plain_drafts.evict(c["cache"], c["table"], c["slot_ids"], c["lens"], c["weights"], c["positions"],
                              c["weights"] if in_place else wo.cpu(), c["positions"] if in_place else po.cpu(), keep, first, recent)
    ops.evict_tokens(d["cache"], d["table"], d["slot_ids"], d["lens"], d["weights"], d["positions"], wo, po, keep, first, recent, _alloc)
    torch.cuda.synchronize()
    assert torch.equal(po.cpu(), want[2])
    assert torch.equal(wo.cpu().view(torch.int32), want[1].view(torch.int32))
    assert torch.equal(d["cache"].cpu().contiguous().view(torch.uint8), want[0].contiguous().view(torch.uint8))
    return d, wo, po


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype,S,Hkv,D,P,planes", [(torch.bfloat16, 2, 2, 128, 16, 2), (torch.float32, 1, 3, 80, 24, 2), (torch.bfloat16, 2, 1, 33, 5, 1),
                                                    (torch.bfloat16, 1, 2, 6, 16, 3)])
@pytest.mark.parametrize("lens,keep,first,recent", [([65], 64, 2, 8), ([300, 17, 64, 63, 1, 0, 65], 64, 3, 20), ([40, 41], 1, 0, 0), ([40, 9], 1, 0, 1),
                                                    ([100], 33, 0, 33), ([513, 1030], 512, 4, 0), ([700, 3], 1000, 1, 1)])
def test_evict_tokens(dtype, S, Hkv, D, P, planes, lens, keep, first, recent, in_place):
    _check_evict(_evict_case(dtype, S, Hkv, D, P, lens, keep + len(lens), planes), keep, first, recent, in_place)


def test_evict_tokens_with_equal_weights():
    _check_evict(_evict_case(torch.bfloat16, 1, 2, 64, 16, [500, 90], 3, coarse=True), 77, 2, 9)
    c = _evict_case(torch.bfloat16, 1, 2, 64, 16, [500, 90], 4)
    c["weights"][:] = 0.25
    _check_evict(c, 77, 2, 9)


def test_evict_tokens_with_infinities_and_nan():
    c = _evict_case(torch.float32, 1, 2, 16, 16, [200, 130], 5)
    g = torch.Generator().manual_seed(1)
    m = torch.rand(c["weights"].shape, generator=g)
    c["weights"][m < 0.2] = math.nan
    c["weights"][(m >= 0.2) & (m < 0.3)] = math.inf
    c["weights"][(m >= 0.3) & (m < 0.4)] = -math.inf
    c["weights"][(m >= 0.4) & (m < 0.5)] = -0.0
    c["weights"][(m >= 0.5) & (m < 0.6)] = 0.0
    for keep in (20, 80, 120):
        d = {k: v.clone() for k, v in c.items()}
        _check_evict(d, keep, 1, 5)


@pytest.mark.parametrize("lens,keep,first,recent", [([9001, 4097, 20], 1000, 4, 100), ([33000], 32999, 4, 64), ([20000, 20000], 15000, 0, 0), ([70001], 128, 2, 32)])
def test_evict_tokens_from_long_caches(lens, keep, first, recent):
    for in_place in (False, True):
        _check_evict(_evict_case(torch.bfloat16, 1, 1, 16, 16, lens, 6, ordered=keep == 1000), keep, first, recent, in_place)


def test_evict_tokens_from_a_cache_whose_keys_do_not_fit_on_the_chip():
    for keep in (300, 409999):
        _check_evict(_evict_case(torch.bfloat16, 1, 1, 8, 64, [410000], 7, planes=1), keep, 3, 50)


def test_evicting_twice_is_evicting_from_what_is_left():
    c = _evict_case(torch.bfloat16, 2, 2, 64, 16, [300, 200], 9)
    d, w, p = _check_evict(c, 150, 2, 20, in_place=True)
    again = dict(cache=d["cache"].cpu(), table=c["table"], slot_ids=c["slot_ids"], lens=torch.tensor([150, 150], dtype=torch.int32),
                 weights=w.cpu(), positions=p.cpu())
    _check_evict(again, 40, 2, 20, in_place=True)


def test_a_slot_or_a_page_that_is_not_there_is_left_alone():
    """A slot outside the rows: the request is passed over.  A place without a page: its entry is not moved, the others are."""
    c = _evict_case(torch.bfloat16, 1, 1, 16, 16, [64, 64], 11)
    c["slot_ids"][0] = 99
    d = {k: v.to(DEV) for k, v in c.items()}
    wo, po = torch.zeros_like(d["weights"]), torch.zeros_like(d["positions"])
    ops.evict_tokens(d["cache"], d["table"], d["slot_ids"], d["lens"], d["weights"], d["positions"], wo, po, 30, 1, 2, _alloc)
    mine = c["table"][0].long()
    assert torch.equal(d["cache"].cpu()[:, mine], c["cache"][:, mine])
    want = plain_drafts.evict(c["cache"], c["table"][1:], c["slot_ids"][1:], c["lens"][1:], c["weights"], c["positions"], wo.cpu() * 0, po.cpu() * 0, 30, 1, 2)
    assert torch.equal(po.cpu(), want[2]) and torch.equal(d["cache"].cpu(), want[0])


# ---- all three, as a serving program calls them -----------------------------------------------------------------------------------

def test_a_step_that_verifies_gathers_and_evicts():
    """The counts of the verification say which rows' weights are gathered and how long the caches are; the evicted cache, read by the attention
    kernel, gives the attention over exactly the entries that stayed."""
    Hq, Hkv, D, P, keep, first, recent = 4, 2, 128, 16, 100, 2, 10
    q_lens, ctx_lens = [4, 1, 3, 4], [130, 99, 100, 20]
    c = _weights_case(torch.bfloat16, Hq, Hkv, D, P, q_lens, ctx_lens, 51)
    c["positions"] = torch.arange(c["weights"].shape[2], dtype=torch.int32).expand(c["weights"].shape).contiguous()
    c["step_positions"] = torch.tensor([k + i for n, k in zip(q_lens, ctx_lens) for i in range(n)], dtype=torch.int32)
    g = torch.Generator().manual_seed(5)
    N, R, V = sum(q_lens), 4, 300
    logits = torch.randn(N, V, generator=g) * 2
    rows = [int(c["cu"][r]) + i for r in range(R) for i in range(q_lens[r] - 1)]
    dl = logits[rows] + 0.3 * torch.randn(len(rows), V, generator=g)
    v = dict(logits=logits, draft_tokens=dl.argmax(1).to(torch.int32), draft_logits=dl, row_starts=c["cu"], temperature=torch.tensor([0.7, 0.0, 1.0, 0.9]),
             top_k=torch.tensor([0, 0, 40, 5], dtype=torch.int32), uniform=torch.rand(N, generator=g))
    d = {k: x.to(DEV) for k, x in v.items()}
    tokens, counts = torch.zeros(N, dtype=torch.int32, device=DEV), torch.zeros(R, dtype=torch.int32, device=DEV)
    ops.verify_drafts(d["logits"], d["draft_tokens"], d["draft_logits"], d["row_starts"], d["temperature"], d["top_k"], d["uniform"], tokens, counts, _alloc)
    w, pos, cache, ctx = c["weights"].to(DEV), c["positions"].to(DEV), c["pages"].to(DEV)[None], _context(c)
    want_tokens, want_counts = plain_drafts.verify(**v)
    assert torch.equal(tokens.cpu(), want_tokens) and torch.equal(counts.cpu(), want_counts)
    ops.accumulate_attention(c["qkv"].to(DEV), cache[0], c["table"].to(DEV), ctx, w, w, D ** -0.5, 0, Hq, Hkv, D, _alloc, positions=pos, counted=counts)
    want, tol = plain_drafts.gathered(c["qkv"], c["pages"], c["table"], c["cu"], c["ctx"], c["slots"], c["weights"], c["weights"], D ** -0.5, 0, Hq, Hkv, D, want_counts)
    assert float(((w.cpu().double() - want).abs() - tol).max()) <= 0
    lens = ctx.ctx_lens + counts
    gathered, noted = w.cpu(), pos.cpu()
    ops.evict_tokens(cache, c["table"].to(DEV), ctx.slot_ids, lens, w[None], pos[None], w[None], pos[None], keep, first, recent, _alloc)
    left = plain_drafts.evict(c["pages"][None], c["table"], c["slots"], lens.cpu(), gathered[None], noted[None], gathered[None], noted[None], keep, first, recent)
    assert torch.equal(cache.cpu(), left[0]) and torch.equal(w[None].cpu(), left[1]) and torch.equal(pos[None].cpu(), left[2])
    # attention of the next token over what is left, against attention over the entries that stayed, in the order of their positions
    q = torch.randn(R, (Hq + 2 * Hkv) * D, generator=g).to(torch.bfloat16)
    after = [min(int(n), keep) for n in lens]
    actx = SimpleNamespace(cu_q=torch.arange(R + 1, dtype=torch.int32, device=DEV), ctx_lens=torch.tensor([n - 1 for n in after], dtype=torch.int32, device=DEV),
                           attn_plan=None, q_lens_host=[1] * R, ctx_lens_host=[n - 1 for n in after], arena=None, max_q_len=1)
    plan = ops.plan_attention([1] * R, actx.ctx_lens_host, P, (), torch.bfloat16)
    actx.attn_plan = {"tiles": torch.tensor(plan["tiles"], dtype=torch.int32, device=DEV)}
    out = torch.zeros(R, Hq * D, dtype=torch.bfloat16, device=DEV)
    ops.paged_attention(q.to(DEV), cache[0], c["table"].to(DEV), actx, out, D ** -0.5, 0, Hq, Hkv, D)
    for r in range(R):
        s = int(c["slots"][r])
        for h in range(Hq):
            kv = h // (Hq // Hkv)
            stayed = sorted(noted_of for noted_of in left[2][0, s, kv, :after[r]].tolist())
            blocks = c["table"][r].long()
            k = torch.stack([c["pages"][blocks[j // P], 0, kv, j % P] for j in stayed]).double()
            val = torch.stack([c["pages"][blocks[j // P], 1, kv, j % P] for j in stayed]).double()
            o = torch.softmax((k @ q[r, h * D:(h + 1) * D].double()) * D ** -0.5, 0) @ val
            # the output is rounded to bfloat16 (half a step), as are the softmax's weights in the kernel
            assert float((out[r, h * D:(h + 1) * D].cpu().double() - o).abs().max()) <= 2.0 ** -8 * (float(o.abs().max()) + float(val.abs().max()))


def test_captured_and_replayed_with_other_inputs():
    """All three in one graph: the second replay, on other logits, caches and lengths in the same buffers, gives what eager calls give."""
    Hq, Hkv, D, P, keep = 8, 2, 128, 16, 60
    q_lens = [3, 3]
    cases = [_weights_case(torch.bfloat16, Hq, Hkv, D, P, q_lens, ctx, 60 + i, extra=40) for i, ctx in enumerate(([90, 100], [100, 40]))]
    rnd = [_verify_case(2, [2], 1000, 70 + i, True) for i in range(2)]
    cap = 143

    def buffers(c, v):
        t = {k: x.to(DEV) for k, x in v.items()}
        wide = torch.full((2, 9), -1, dtype=torch.int32)
        wide[:, :c["table"].shape[1]] = c["table"][:, :9]
        t.update(qkv=c["qkv"].to(DEV), pages=torch.zeros(20, 2, Hkv, P, D, dtype=torch.bfloat16, device=DEV), table=wide.to(DEV), ctx=c["ctx"].to(DEV),
                 slots=c["slots"].to(DEV), w=c["weights"][..., :cap].contiguous().to(DEV) if c["weights"].shape[2] >= cap else
                 torch.nn.functional.pad(c["weights"], (0, cap - c["weights"].shape[2])).to(DEV),
                 pos=torch.arange(cap, dtype=torch.int32, device=DEV).expand(4, Hkv, cap).contiguous(), at=c["step_positions"].to(DEV))
        t["pages"][:c["pages"].shape[0]] = c["pages"].to(DEV)
        t.update(tokens=torch.zeros(6, dtype=torch.int32, device=DEV), counts=torch.zeros(2, dtype=torch.int32, device=DEV), lens=torch.zeros(2, dtype=torch.int32, device=DEV))
        return t

    def step(t, scratch):
        it = iter(scratch)

        def alloc(shape, dtype):
            key = next(it)
            if scratch[key] is None:
                scratch[key] = torch.empty(shape, dtype=dtype, device=DEV)
            return scratch[key]
        ctx = SimpleNamespace(num_reqs=2, cu_q=cases[0]["cu"].to(DEV) if t.get("cu") is None else t["cu"], ctx_lens=t["ctx"], slot_ids=t["slots"],
                              positions=t["at"], q_lens_host=q_lens, ctx_lens_host=[90, 100], max_q_len=3)
        ops.verify_drafts(t["logits"], t["draft_tokens"], t["draft_logits"], t["row_starts"], t["temperature"], t["top_k"], t["uniform"], t["tokens"], t["counts"], alloc)
        ops.accumulate_attention(t["qkv"], t["pages"], t["table"], ctx, t["w"], t["w"], D ** -0.5, 0, Hq, Hkv, D, alloc, positions=t["pos"], counted=t["counts"])
        torch.add(t["ctx"], t["counts"], out=t["lens"])
        ops.evict_tokens(t["pages"][None], t["table"], t["slots"], t["lens"], t["w"][None], t["pos"][None], t["w"][None], t["pos"][None], keep, 2, 9, alloc)

    keys = ("pages", "w", "pos", "tokens", "counts")
    want = []
    for c, v in zip(cases, rnd):
        t = buffers(c, v)
        step(t, {i: None for i in range(8)})
        want.append({k: t[k].clone() for k in keys})
    live, scratch = buffers(cases[0], rnd[0]), {i: None for i in range(8)}
    live["cu"] = cases[0]["cu"].to(DEV)
    step(live, scratch)                           # sizes the scratch memory
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(live, scratch)
    for i in (0, 1, 0):
        fresh = buffers(cases[i], rnd[i])
        for k, x in fresh.items():
            live[k].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for k in keys:
            assert torch.equal(live[k], want[i][k]), k


def test_on_another_stream_and_two_calls_at_once():
    """Two calls on two streams, each with scratch memory of its own, and the same on the default stream."""
    c = [_weights_case(torch.bfloat16, 8, 2, 128, 16, q, k, 80 + i) for i, (q, k) in enumerate((([1, 1], [500, 900]), ([300], [20])))]
    want = [_gather(x)[0] for x in c]
    streams = [torch.cuda.Stream() for _ in c]
    got = []
    for x, s in zip(c, streams):
        Hq, Hkv, D = x["heads"]
        w = x["weights"].to(DEV)
        out = torch.full_like(w, -5.0)
        args = (x["qkv"].to(DEV), x["pages"].to(DEV), x["table"].to(DEV), _context(x))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            ops.accumulate_attention(*args, w, out, D ** -0.5, 0, Hq, Hkv, D, _alloc)
        got.append(out)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


def test_another_device_is_refused(monkeypatch):
    monkeypatch.setattr(ops, "_current_device", lambda: 1)
    c = _verify_case(2, [1], 10, 1)
    with pytest.raises(ops.KernelRefused, match="current device"):
        _verify(c)


# ---- which kernels served ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("Hq,Hkv,D,P", [(32, 8, 128, 16), (5, 5, 48, 16), (12, 1, 96, 24), (4, 4, 192, 64), (6, 3, 256, 8), (128, 1, 64, 128), (7, 1, 8, 16)])
@pytest.mark.parametrize("q_lens,ctx_lens", [([33], [0]), ([129, 1, 700], [1, 300, 257]), ([1100, 260], [900, 0])])
def test_accumulate_attention_on_the_tensor_cores_and_without(Hq, Hkv, D, P, q_lens, ctx_lens, monkeypatch):
    """Portions of many rows through both kernels that take them, units of one to four tiles, odd numbers of tiles, several parts; no wait ran out."""
    c = _weights_case(torch.bfloat16, Hq, Hkv, D, P, q_lens, ctx_lens, 90)
    before = ops.launch_count
    a = _check_weights(c)
    assert ops.device_status() == {}
    assert torch.equal(a, _check_weights(c))
    monkeypatch.setattr(ops, "ATTENTION_WEIGHTS_TC", False)
    _check_weights(c)
    assert ops.launch_count > before


def test_accumulate_attention_on_the_tensor_cores_with_every_option():
    for q_lens, ctx_lens in (([300, 90], [500, 3]), ([64], [0])):
        for Hq, Hkv in ((8, 2), (6, 2), (3, 3)):
            c = _weights_case(torch.bfloat16, Hq, Hkv, 64, 16, q_lens, ctx_lens, 91, counted=[q_lens[0] - 7] + [0] * (len(q_lens) - 1))
            _check_weights(c, window=100, sinks=torch.randn(Hq), softcap=4.0, slopes=torch.rand(Hq) * 0.1)
            _check_weights(c, window=1, sinks=torch.randn(Hq))
            _check_weights(c, window=129, in_place=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_accumulate_attention_of_requests_without_tokens(dtype):
    """A request that brings nothing keeps what its keys have gathered, beside others and alone."""
    for q_lens, ctx_lens in (([0, 2], [70, 9]), ([0, 90], [300, 5]), ([0], [40])):
        c = _weights_case(dtype, 4, 2, 64, 16, q_lens, ctx_lens, 95)
        c["qkv"] = c["qkv"] if sum(q_lens) else torch.zeros(0, 8 * 64, dtype=dtype)
        _check_weights(c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_lens,ctx_lens", [([1, 1], [700, 20]), ([2], [5000]), ([40], [30])])
def test_accumulate_attention_over_wide_latents(dtype, q_lens, ctx_lens):
    """Heads of 576 channels over one plane and one kv head: beyond what the tensor cores' tiles take for many rows."""
    _check_weights(_weights_case(dtype, 16, 1, 576, 16, q_lens, ctx_lens, 97, planes=1, std=0.3))


def test_with_the_steps_arena():
    """Scratch memory from a step's arena, too small at first (it falls back, grows at the reset) and then of the right size: the same bits."""
    from qwen_engine_b200.parts.base import Arena
    arena = Arena(DEV, capacity=1 << 12)
    for q_lens, ctx_lens in (([1, 2], [700, 5000]), ([150], [40])):
        c = _weights_case(torch.bfloat16, 8, 2, 128, 16, q_lens, ctx_lens, 98)
        want = _gather(c)[0]
        Hq, Hkv, D = c["heads"]
        for _ in range(3):
            arena.reset()
            w = c["weights"].to(DEV)
            out = torch.full_like(w, -5.0)
            ops.accumulate_attention(c["qkv"].to(DEV), c["pages"].to(DEV), c["table"].to(DEV), _context(c), w, out, D ** -0.5, 0, Hq, Hkv, D, arena.alloc)
            assert torch.equal(out.cpu(), want)
    v = _verify_case(3, [2], 501, 16, True)
    want = plain_drafts.verify(**v)
    d = {k: x.to(DEV) for k, x in v.items()}
    for _ in range(2):
        arena.reset()
        tokens, counts = torch.zeros(9, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
        ops.verify_drafts(d["logits"], d["draft_tokens"], d["draft_logits"], d["row_starts"], d["temperature"], d["top_k"], d["uniform"], tokens, counts, arena.alloc)
        _same((tokens.cpu(), counts.cpu()), want)


def test_drafts_through_the_step_function():
    """A model's own step with a request's newest token and its drafts, every place wanted: greedy requests gain exactly the tokens that decoding one by
    one gives, drafts that stand and the first that does not."""
    from qwen_engine_b200.cache.manager import CacheManager
    from qwen_engine_b200.config import preset_config_dict
    from qwen_engine_b200.engine.loading import load_model
    from qwen_engine_b200.engine.runner import StepEntry
    from qwen_engine_b200.registry import config_from_dict
    loaded = load_model(None, torch.float32, DEV, 16, 64, 4, False, config=config_from_dict(preset_config_dict("tiny-b")), random_seed=3)
    runner, cache = loaded.runner, loaded.cache
    assert isinstance(cache, CacheManager)
    prompt = [5, 6, 7, 8, 9]
    rc = cache.open("one by one")
    logits = runner.step([StepEntry(rc, prompt, [len(prompt) - 1])])
    truth = [int(logits[0].argmax())]
    for _ in range(4):
        logits = runner.step([StepEntry(rc, [truth[-1]], [0])])
        truth.append(int(logits[0].argmax()))
    cache.close(rc)
    greedy = [SamplingParams(temperature=0.0)]
    for wrong in (None, 0, 2):
        drafts = list(truth[1:4])
        if wrong is not None:
            drafts[wrong] = (drafts[wrong] + 1) % 389
        rc = cache.open(f"drafted {wrong}")
        runner.step([StepEntry(rc, prompt, [len(prompt) - 1])])
        logits = runner.step([StepEntry(rc, [truth[0]] + drafts, range(4))])
        got = Sampler(DEV).verify(logits, greedy, [drafts], [[0.5] * 4])
        assert got == [truth[1:5] if wrong is None else truth[1:wrong + 2]]
        cache.close(rc)


@pytest.mark.parametrize("dtype,n", [(torch.float32, 40), (torch.bfloat16, 3), (torch.bfloat16, 70)])
def test_rows_that_are_one_row_in_memory(dtype, n):
    """A row given n times over by a stride of 0 gathers what n equal rows gather."""
    c = _weights_case(dtype, 8, 2, 128, 16, [n], [50], 23)
    c["qkv"] = c["qkv"][:1].repeat(n, 1)
    Hq, Hkv, D = c["heads"]
    w = c["weights"].to(DEV)
    out = w.clone()
    ops.accumulate_attention(c["qkv"][:1].to(DEV).expand(n, -1), c["pages"].to(DEV), c["table"].to(DEV), _context(c), w, out, D ** -0.5, 0, Hq, Hkv, D, _alloc)
    want, tol = plain_drafts.gathered(c["qkv"], c["pages"], c["table"], c["cu"], c["ctx"], c["slots"], c["weights"], c["weights"],
                                      D ** -0.5, 0, Hq, Hkv, D, None)
    assert ((out.cpu().double() - want).abs() <= tol).all()


# ---- rows with little or nothing in them -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("V", [97, 4099, 40001])
def test_verify_drafts_whose_own_draft_logit_is_nan(V):
    """A NaN counts as -inf: the draft's probability is 0, and so it stands wherever the target gives it any."""
    for top_k in (0, 5):
        c = _verify_case(12, [1, 3], V, 500 + top_k, True, top_ks=(top_k,), temps=(0.7, 1.3))
        for j, d in enumerate(c["draft_tokens"].tolist()):
            c["draft_logits"][j, d] = math.nan if j % 2 else -math.inf
        _same(_verify(c), plain_drafts.verify(**c))


@pytest.mark.parametrize("model", [True, False])
@pytest.mark.parametrize("V", [5, 333, 9001])
def test_verify_drafts_of_token_0_where_a_greedy_row_has_nothing(V, model):
    """A row without any logit above -inf lets no draft stand, not the draft of token 0 either, and gives token 0."""
    c = _verify_case(8, [1, 3], V, 600 + V, model, temps=(0.0, 0.0, 0.8))
    starts = c["row_starts"].tolist()
    c["draft_tokens"][:] = c["logits"][[starts[r] + i for r in range(8) for i in range(starts[r + 1] - starts[r] - 1)]].argmax(1).to(torch.int32)
    for r in range(8):
        row = starts[r] + (r % 2) * (starts[r + 1] - starts[r] - 2)              # the request's first or last drafted place
        c["logits"][row] = math.nan if r % 3 == 0 else -math.inf
        c["draft_tokens"][row - r] = 0
    want = plain_drafts.verify(**c)
    for r in range(8):
        assert int(want[1][r]) <= 1 + (r % 2) * (starts[r + 1] - starts[r] - 2)
    _same(_verify(c), want)


@pytest.mark.parametrize("top_k", [3, 50, 1000])
@pytest.mark.parametrize("V", [333, 4099, 32003, 151936])
def test_verify_drafts_with_fewer_finite_logits_than_top_k(V, top_k):
    """Rows of which 1 to top_k - 1 logits are above -inf (all of those are kept), of the target's and of the draft model's, among rows that are whole:
    nothing of one row's top_k-th logit shows in another's, and equal calls give equal tokens."""
    rnd = random.Random(V + top_k)
    for seed, model in ((0, True), (1, True), (2, False)):
        c = _verify_case(7, [2, 4], V, 400 + seed, model, top_ks=(0, top_k, top_k), temps=(0.6, 1.0))
        starts = c["row_starts"].tolist()
        draft_of = {starts[r] + i: starts[r] + i - r for r in range(7) for i in range(starts[r + 1] - starts[r] - 1)}      # row -> draft

        def thin(x, draft):
            """All but a few of the row's logits go; the draft's own mostly stays."""
            n = rnd.randint(1, min(top_k, V) - 1)
            stay = rnd.sample(range(V), n)
            if draft is not None and rnd.random() < 0.8:
                stay[0] = int(c["draft_tokens"][draft])
            kept = x[stay].clone()
            x[:] = -math.inf
            x[::5] = math.nan
            x[stay] = kept
        for row in range(c["logits"].shape[0]):
            if row % 3 != 2:
                thin(c["logits"][row], draft_of.get(row))
        if model:
            for j in range(c["draft_logits"].shape[0]):
                if j % 3 != 1:
                    thin(c["draft_logits"][j], j)
        got = _verify(c)
        _same(got, plain_drafts.verify(**c))
        _same(_verify(c), got)


# ---- NaN in what a row sees ----------------------------------------------------------------------------------------------------------

NAN_BATCHES = [(torch.float32, [2, 3], [70, 9], {}), (torch.bfloat16, [2, 3], [70, 9], {}), (torch.bfloat16, [3, 2], [5000, 40], {}),
               (torch.bfloat16, [150, 40], [40, 7], {}), (torch.bfloat16, [150, 40], [40, 7], {"tc": False}), (torch.bfloat16, [150, 40], [40, 7], {"softcap": 3.0}),
               (torch.bfloat16, [90, 40], [300, 7], {"window": 100}), (torch.float32, [90, 40], [300, 7], {"window": 100})]


def _check_nan(c, clean, row, head, seen, monkeypatch, options):
    """Request 0's kv head of ``head``: the keys ``seen`` are NaN.  Every other head and request: as without the NaN."""
    Hq, Hkv, D = c["heads"]
    opts = dict(options)
    monkeypatch.setattr(ops, "ATTENTION_WEIGHTS_TC", opts.pop("tc", True))
    got, _ = _gather(c, opts.pop("window", 0), **opts)
    kv, s0 = head // (Hq // Hkv), int(c["slots"][0])
    assert torch.isnan(got[s0, kv, :len(seen)][seen]).all(), (row, head, (~torch.isnan(got[s0, kv, :len(seen)]) & seen).nonzero().flatten().tolist()[:5])
    other = torch.ones(got.shape, dtype=torch.bool)
    other[s0, kv, :len(seen)] = False
    assert torch.equal(got[other], clean[other])


@pytest.mark.parametrize("dtype,q_lens,ctx_lens,options", NAN_BATCHES)
def test_accumulate_attention_of_a_query_that_is_nan(dtype, q_lens, ctx_lens, options, monkeypatch):
    """Every key that the row sees becomes NaN, whatever the row's place in its tile and whichever kernel serves."""
    Hq, Hkv, D = 4, 2, 128
    c = _weights_case(dtype, Hq, Hkv, D, 16, q_lens, ctx_lens, 700)
    window = options.get("window", 0)
    clean = _gather(c, window, **{k: v for k, v in options.items() if k == "softcap"})[0] if options.get("tc", True) else None
    if clean is None:
        monkeypatch.setattr(ops, "ATTENTION_WEIGHTS_TC", False)
        clean = _gather(c)[0]
    total = q_lens[0] + ctx_lens[0]
    key = torch.arange(total)
    for row in range(0, q_lens[0], 1 if q_lens[0] < 8 else 9):
        for head in (0, 1, 3):
            d = dict(c, qkv=c["qkv"].clone())
            d["qkv"][row, head * D + 5] = math.nan
            pos = ctx_lens[0] + row
            seen = (key <= pos) & ((key > pos - window) if window else torch.ones(total, dtype=torch.bool))
            _check_nan(d, clean, row, head, seen, monkeypatch, options)


@pytest.mark.parametrize("dtype,q_lens,ctx_lens,options", NAN_BATCHES)
def test_accumulate_attention_over_a_key_that_is_nan(dtype, q_lens, ctx_lens, options, monkeypatch):
    """Every key of the rows that see it becomes NaN: their softmax's sum is."""
    Hq, Hkv, D = 4, 2, 128
    c = _weights_case(dtype, Hq, Hkv, D, 16, q_lens, ctx_lens, 701)
    window = options.get("window", 0)
    monkeypatch.setattr(ops, "ATTENTION_WEIGHTS_TC", options.get("tc", True))
    clean = _gather(c, window, **{k: v for k, v in options.items() if k == "softcap"})[0]
    total, ctx0 = q_lens[0] + ctx_lens[0], ctx_lens[0]
    key = torch.arange(total)
    for j in list(range(0, min(total, 19))) + [ctx0, total - 1]:
        d = dict(c, pages=c["pages"].clone())
        d["pages"][int(c["table"][0, j // 16]), 0, 1, j % 16, 9] = math.nan
        seen = torch.zeros(total, dtype=torch.bool)
        for i in range(q_lens[0]):
            pos = ctx0 + i
            if j <= pos and (not window or j > pos - window):
                seen |= (key <= pos) & ((key > pos - window) if window else torch.ones(total, dtype=torch.bool))
        _check_nan(d, clean, j, 2, seen, monkeypatch, options)


# ---- scratch memory ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("lens,keep", [([65, 60], 64), ([500, 130], 120), ([40], 400)])
def test_evict_tokens_asks_for_scratch_memory_by_what_may_move(lens, keep):
    """Two numbers for every entry that can move, min(keep, places - keep) a head at most, and one for how many do."""
    c = _evict_case(torch.bfloat16, 2, 3, 16, 16, lens, 12)
    d = {k: v.to(DEV) for k, v in c.items()}
    asked = []

    def alloc(shape, dtype):
        asked.append(math.prod(shape))
        return _alloc(shape, dtype)
    wo, po = torch.zeros_like(d["weights"]), torch.zeros_like(d["positions"])
    want = plain_drafts.evict(c["cache"], c["table"], c["slot_ids"], c["lens"], c["weights"], c["positions"], wo.cpu(), po.cpu(), keep, 2, 9)
    ops.evict_tokens(d["cache"], d["table"], d["slot_ids"], d["lens"], d["weights"], d["positions"], wo, po, keep, 2, 9, alloc)
    assert torch.equal(po.cpu(), want[2]) and torch.equal(wo.cpu(), want[1]) and torch.equal(d["cache"].cpu(), want[0])
    places = min(c["weights"].shape[3], c["table"].shape[1] * 16)
    assert sum(asked) <= 2 * len(lens) * 3 * (1 + 2 * max(0, min(keep, places - keep)))


def _record(monkeypatch):
    """The bytes that the calls from here on ask for as scratch memory, one number a piece."""
    asked, plain = [], _alloc

    def alloc(shape, dtype):
        asked.append(math.prod(shape) * dtype.itemsize)
        return plain(shape, dtype)
    monkeypatch.setitem(globals(), "_alloc", alloc)
    return asked


def _widen(c, places, P):
    """The same case in slots and block tables of so many places."""
    table = torch.full((c["table"].shape[0], places // P), -1, dtype=torch.int32)
    table[:, :c["table"].shape[1]] = c["table"]
    return dict(c, table=table, weights=torch.nn.functional.pad(c["weights"], (0, places - c["weights"].shape[2])))


def test_accumulate_attention_in_wide_tables_asks_for_bounded_scratch_memory(monkeypatch):
    """One long request among many short ones in tables of 131 072 places: the scores of all would be 805 MB."""
    q_lens = [4] * 23 + [3]
    c = _widen(_weights_case(torch.bfloat16, 16, 2, 64, 16, q_lens, [3 + 11 * r for r in range(23)] + [9000], 800), 131072, 16)
    asked = _record(monkeypatch)
    _check_weights(c)
    assert asked and max(asked) <= ops.ATTENTION_WEIGHTS_SCRATCH and sum(asked) <= 1.1 * ops.ATTENTION_WEIGHTS_SCRATCH
    # ... and where more is held than that: what is held, up to a limit
    c["q_lens"] = [4] * 24
    c["ctx_lens"] = [131000] * 24
    meta = lambda shape, dtype: asked.append(math.prod(shape) * dtype.itemsize) or torch.empty(4, dtype=dtype, device=DEV)
    del asked[:]
    monkeypatch.setattr(ops, "_entry", lambda name: lambda *a: 0)          # (asked for, not launched)
    monkeypatch.setitem(globals(), "_alloc", meta)
    c["cu"], c["qkv"] = torch.arange(0, 97, 4, dtype=torch.int32), torch.zeros(96, c["qkv"].shape[1], dtype=torch.bfloat16)
    c["step_positions"] = torch.zeros(96, dtype=torch.int32)
    _gather(c)
    assert 0.9 * 4 * 24 * 2 * 32 * 131000 <= sum(asked) <= 1.1 * ops.ATTENTION_WEIGHTS_SCRATCH_MOST


@pytest.mark.parametrize("q_lens,ctx_lens", [([4, 1, 3, 4, 2], [600, 9, 5000, 40, 77]), ([4, 150, 0, 2, 90, 1], [600, 9, 50, 4000, 5, 0])])
@pytest.mark.parametrize("Hq,D", [(12, 64), (24, 200)])
@pytest.mark.parametrize("option", ["", "window", "sinks", "slopes"])
def test_accumulate_attention_where_some_requests_scores_find_no_room(q_lens, ctx_lens, Hq, D, option, monkeypatch):
    """Scratch memory for the scores of none, of some and of all requests: those that find no room are formed twice, with the same bits.  (Portions of more rows are cut into fewer parts
    where their sums do not fit, and added up in another order: those are held against the definition alone.)"""
    c = _weights_case(torch.bfloat16, Hq, 3, D, 16, q_lens, ctx_lens, 801, counted=[max(0, n - 1) for n in q_lens])
    kw = {"window": dict(window=70), "sinks": dict(sinks=torch.randn(Hq)), "slopes": dict(slopes=torch.rand(Hq) * 0.1)}.get(option, {})
    want = _check_weights(c, **kw)
    longest = max(a + b for a, b in zip(q_lens, ctx_lens)) + 64
    for heads in (0, 2, 3, 7, 10):
        for name in ("ATTENTION_WEIGHTS_SCRATCH", "ATTENTION_WEIGHTS_SCRATCH_MOST"):
            monkeypatch.setattr(ops, name, max(1, heads * 4 * 16 * longest))
        got = _check_weights(c, **kw)
        for n, slot in zip(q_lens, c["slots"].tolist()):
            assert n * (Hq // 3) > ops.ATTENTION_WEIGHTS_FEW_ROWS or torch.equal(got[slot], want[slot])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_accumulate_attention_of_prompts_in_wide_tables_asks_for_bounded_scratch_memory(dtype, monkeypatch):
    """A portion among requests of a few rows: parts of the keys' sums for the portion's own range of requests, and no parts where they would not fit."""
    c = _widen(_weights_case(dtype, 8, 2, 64, 16, [1, 300, 1, 60] + [1] * 8, [50, 40, 700, 20] + [30] * 8, 802), 65536, 16)
    asked = _record(monkeypatch)
    _check_weights(c)
    assert sum(asked) <= 2 * ops.ATTENTION_WEIGHTS_SCRATCH
    del asked[:]
    monkeypatch.setattr(ops, "ATTENTION_WEIGHTS_SCRATCH", 1 << 16)
    _check_weights(c)
    assert sum(asked) <= 6 << 20                  # (the rows' statistics)


def test_evict_tokens_from_a_cache_that_was_shared():
    """A request whose first pages another one holds too: made private (copies as at the beginning of a step) and evicted, it gives what an unshared
    one gives, the other's pages stay as they are, and a third with the same tokens finds the other's alone."""
    from qwen_engine_b200.cache import CacheManager, PagedKVSpec
    Hkv, D, P, n, keep = 2, 64, 16, 150, 40
    cm = CacheManager([PagedKVSpec(Hkv, D)] * 2, P, 40, 4, torch.bfloat16, DEV)
    prompt = list(range(200, 200 + n))

    def opened(name, tokens):
        rc = cm.open(name, tokens, len(tokens))
        cm.append(rc, tokens[rc.num_tokens:])
        cm.commit(rc)
        return rc
    a, b = opened("a", prompt), opened("b", prompt[:100])
    assert b.shared_tokens == 96
    g = torch.Generator().manual_seed(900)
    cache = cm.groups[0].tensor
    cache.copy_(torch.randn(cache.shape, generator=g).to(torch.bfloat16))
    before, table = cache.cpu(), torch.tensor([a.tables[0]], dtype=torch.int32)
    cm.make_private(a, 0)
    ops.copy_pages(cache, torch.tensor(cm.page_copies_by_group()[0], dtype=torch.int32, device=DEV))
    mine = torch.tensor([a.tables[0]], dtype=torch.int32)
    w, pos = torch.rand(2, 1, Hkv, n, generator=g), torch.arange(n, dtype=torch.int32).expand(2, 1, Hkv, n).contiguous()
    slot, lens = torch.zeros(1, dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
    want = plain_drafts.evict(before, table, slot, lens, w, pos, w, pos, keep, 2, 8)
    dw, dp = w.to(DEV), pos.to(DEV)
    ops.evict_tokens(cache, mine.to(DEV), slot.to(DEV), lens.to(DEV), dw, dp, dw, dp, keep, 2, 8, _alloc)
    after = cache.cpu()
    assert torch.equal(after[:, mine[0].long()], want[0][:, table[0].long()]) and torch.equal(dw.cpu(), want[1]) and torch.equal(dp.cpu(), want[2])
    theirs = torch.tensor(b.tables[0])
    assert torch.equal(after[:, theirs], before[:, theirs])
    c = cm.open("c", prompt, n)
    assert c.shared_tokens == 96 and c.tables[0] == b.tables[0][:6]
    cm.check_invariants()


@pytest.mark.parametrize("dtype,q_lens,tc,want", [(torch.bfloat16, [33, 200], True, {"qe_attention_weights_tc"}), (torch.bfloat16, [33, 200], False, {"qe_attention_weights"}),
                                                  (torch.bfloat16, [1, 8], True, {"qe_attention_weights_few"}), (torch.float32, [1, 200], True, {"qe_attention_weights"}),
                                                  (torch.bfloat16, [1, 200], True, {"qe_attention_weights_few", "qe_attention_weights_tc"}),
                                                  (torch.bfloat16, [1, 200], False, {"qe_attention_weights_few", "qe_attention_weights"})])
def test_which_kernels_gather_attention_weights(dtype, q_lens, tc, want, monkeypatch):
    called, entry = set(), ops._entry
    monkeypatch.setattr(ops, "_entry", lambda name: called.add(name) or entry(name))
    monkeypatch.setattr(ops, "ATTENTION_WEIGHTS_TC", tc)
    _check_weights(_weights_case(dtype, 8, 2, 128, 16, q_lens, [40, 7], 92))
    assert called == want


@pytest.mark.parametrize("V", [7, 1001, 32003, 151935])
def test_verify_drafts_that_fall_where_both_distributions_are_one(V):
    """Drafts that can only fall (outside the vocabulary, or masked in both models) where the draft model's logits are the target's, rows on every boundary:
    nothing is left of max(p - q, 0), not a rounding either, and the token comes from p."""
    for seed, top_ks in ((0, (0,)), (1, (0, 5))):
        c = _verify_case(6, [1, 3], V, 950 + seed, True, top_ks=top_ks, temps=(0.7, 1.0, 1.3))
        starts = c["row_starts"].tolist()
        rows = [starts[r] + i for r in range(6) for i in range(starts[r + 1] - starts[r] - 1)]
        for j, row in enumerate(rows):
            if j % 2:
                c["draft_tokens"][j] = V
            else:
                c["draft_tokens"][j] = j % V
                c["logits"][row, j % V] = -math.inf
        c["draft_logits"] = c["logits"][rows].clone()
        want = plain_drafts.verify(**c)
        assert (want[1] == 1).all()
        for u in (0.05, 0.3, 0.5, 0.8, 0.99):
            c["uniform"][:] = u
            _same(_verify(c), plain_drafts.verify(**c))


def test_replayed_with_longer_contexts_than_scratch_memory_was_asked_for(monkeypatch):
    """A captured call whose scratch memory goes by the lengths at its capture: replayed with longer ones, it gives what eager calls give."""
    for name in ("ATTENTION_WEIGHTS_SCRATCH", "ATTENTION_WEIGHTS_SCRATCH_MOST"):
        monkeypatch.setattr(ops, name, 1 << 16)
    Hq, Hkv, D, q_lens = 8, 2, 64, [4, 1, 3, 2, 4, 1, 1, 2, 3]
    cases = [_weights_case(torch.bfloat16, Hq, Hkv, D, 16, q_lens, ctx, 960 + i, extra=0) for i, ctx in enumerate(([20 * r for r in range(9)], [1200 - 130 * r for r in range(9)]))]
    places = 1600
    cases = [_widen(dict(c, pages=torch.cat([c["pages"], torch.zeros(600 - c["pages"].shape[0], *c["pages"].shape[1:], dtype=c["pages"].dtype)])), places, 16) for c in cases]
    want = [_check_weights(c) for c in cases]
    live = {k: cases[0][k].to(DEV) for k in ("qkv", "pages", "table", "weights", "ctx", "slots", "cu", "step_positions")}
    out = torch.full_like(live["weights"], -5.0)
    ctx = SimpleNamespace(num_reqs=9, cu_q=live["cu"], ctx_lens=live["ctx"], slot_ids=live["slots"], positions=live["step_positions"], q_lens_host=q_lens,
                          ctx_lens_host=cases[0]["ctx_lens"], max_q_len=4)

    def call():
        ops.accumulate_attention(live["qkv"], live["pages"], live["table"], ctx, live["weights"], out, D ** -0.5, 0, Hq, Hkv, D, _alloc)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        call()
    for i in (1, 0, 1):
        for k, x in live.items():
            x.copy_(cases[i][k])
        out.fill_(-5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), want[i])


@pytest.mark.parametrize("dtype,q_lens", [(torch.float32, [3, 40]), (torch.bfloat16, [3, 1]), (torch.bfloat16, [3, 140])])
def test_accumulate_attention_of_rows_in_a_larger_buffer(dtype, q_lens):
    """Rows behind the step's tokens (NaN here) are not looked at, with positions for them and without."""
    c = _weights_case(dtype, 8, 2, 64, 16, q_lens, [50, 9], 970)
    want = _check_weights(c)
    c["qkv"] = torch.cat([c["qkv"], torch.full((5, c["qkv"].shape[1]), math.nan, dtype=dtype)])
    assert torch.equal(_check_weights_of_tokens(c, q_lens), want)
    c["step_positions"] = torch.cat([c["step_positions"], torch.full((5,), -4, dtype=torch.int32)])
    assert torch.equal(_check_weights_of_tokens(c, q_lens), want)


def _check_weights_of_tokens(c, q_lens):
    got, noted = _gather(c)
    for r, n in enumerate(q_lens):
        k, a = c["ctx_lens"][r], int(c["cu"][r])
        assert (noted[int(c["slots"][r]), :, k:k + n] == c["step_positions"][a:a + n]).all()
    return got
