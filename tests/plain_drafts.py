"""The verification of drafted tokens, the gathered attention weights and the eviction, from their definitions in 64 bits: one
request, head and row at a time, on the host."""
from __future__ import annotations

import math

import torch


def distribution(x, temperature, top_k):
    """What a row is drawn from: softmax of the logits at or above the top_k-th largest, divided by the temperature; None where
    no logit is above -inf."""
    x = torch.nan_to_num(x.double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    top = x.max()
    if top == -math.inf:
        return None
    if not temperature > 0:
        p = torch.zeros_like(x)
        p[int((x == top).nonzero()[0])] = 1.0
        return p
    kept = x >= x.sort(descending=True).values[top_k - 1] if 0 < top_k < x.numel() else torch.ones_like(x, dtype=torch.bool)
    e = torch.where(x == top, torch.ones_like(x), torch.exp((x - top) / float(temperature))) * kept
    return e / e.sum()


def draw(p, u):
    run = torch.cumsum(p, 0)
    return int((run > u * run[-1]).nonzero()[0])


def verify(logits, draft_tokens, draft_logits, row_starts, temperature, top_k, uniform):
    """(tokens [N], counts [R]) as ``ops.verify_drafts`` leaves them."""
    N, V = logits.shape
    starts = row_starts.tolist()
    tokens, counts = [-1] * N, []
    for r in range(len(starts) - 1):
        a, n = starts[r], starts[r + 1] - starts[r] - 1
        t, k = float(temperature[r]), int(top_k[r])
        end = n
        for i in range(n):
            d = int(draft_tokens[a - r + i])
            p = distribution(logits[a + i], t, k)
            if not 0 <= d < V or p is None:
                end = i
                break
            if t > 0 and draft_logits is not None:
                q = distribution(draft_logits[a - r + i], t, k)
                qd = math.nan if q is None else float(q[d])
            else:
                qd = 1.0
            if not float(uniform[a + i]) * qd < float(p[d]):
                end = i
                break
            tokens[a + i] = d
        counts.append(end + 1)
        p = distribution(logits[a + end], t, k)
        if p is None:
            tokens[a + end] = 0
            continue
        w = p
        if end < n and t > 0:
            d = int(draft_tokens[a - r + end])
            if draft_logits is not None:
                q = distribution(draft_logits[a - r + end], t, k)
            else:
                q = torch.zeros_like(p)
                if 0 <= d < V:
                    q[d] = 1.0
            if q is not None:
                w = (p - q).clamp_min(0)
            if not float(w.sum()) > 0:
                w = p
        tokens[a + end] = draw(w, float(uniform[starts[r + 1] - 1]))
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32)


def gathered(q, pages, table, cu_q, ctx_lens, slot_ids, weights, out, scale, window, Hq, Hkv, D, counted=None, slopes=None,
             softcap=0.0, sinks=None):
    """(out float64 [slots, Hkv, capacity], how far float32 arithmetic may be off per entry).

    The second: a raw score is a sum of D products, off by at most (D + 2) 2^-24 of the sum of the products' magnitudes
    whatever the order of the sum; the scale, the cap's tanh (2 ulp, times the cap), the distance bias and the change of base
    are a rounding each, of what they give.  A weight exp(s - m) / z is then off by e = 2 x the row's largest such error (s
    against m), and 32 roundings (two exponentials of 2 ulp and their arguments, a sum that is merged from parts, a
    quotient); z is a sum of weights that are off by as much each, and up to 2^-24 times the number of summands of a
    thread, at most 64 + 32; so a weight is off by 2 e relative to itself.  Adding rows up costs half an ulp of the running sum each."""
    u = 2.0 ** -24
    P = pages.shape[3]
    res, tol = out.double().clone(), torch.zeros_like(out, dtype=torch.float64)
    G = Hq // Hkv
    for r in range(len(ctx_lens)):
        n, c, row0, slot = int(cu_q[r + 1] - cu_q[r]), int(ctx_lens[r]), int(cu_q[r]), int(slot_ids[r])
        L = n + c
        rows = n if counted is None else min(n, int(counted[r]))
        blocks = table[r, :-(-L // P)].long()
        key = torch.arange(L)
        held = (blocks >= 0)[key // P]
        for h in range(Hkv):
            keys = pages[blocks.clamp_min(0), 0, h].reshape(-1, D)[:L].double()
            keys = torch.where(held[:, None], keys, torch.zeros_like(keys))
            total, off = torch.zeros(L, dtype=torch.float64), torch.zeros(L, dtype=torch.float64)
            for g in range(G):
                head = h * G + g
                x = q[row0:row0 + rows, head * D:(head + 1) * D].double()
                place = c + torch.arange(rows)[:, None]
                gone = (key[None] > place) | ~held[None]
                if window > 0:
                    gone = gone | (key[None] <= place - window)
                keys_here = torch.where(torch.isfinite(keys), keys, torch.zeros_like(keys))
                s = (x @ keys_here.T) * scale
                err = (D + 6) * u * (x.abs() @ keys_here.abs().T) * scale
                if softcap > 0:
                    s = softcap * torch.tanh(s / softcap)
                    err = err + 8 * u * softcap
                if slopes is not None:
                    s = s - float(slopes[head]) * (place - key[None])
                    err = err + 4 * u * float(slopes[head]) * (place - key[None]).abs()
                err = err + 4 * u * s.abs()
                s = s.masked_fill(gone, -math.inf)
                err = err.masked_fill(gone, 0.0)
                if sinks is not None:
                    s = torch.cat([s, sinks[head].double().expand(rows, 1)], 1)
                empty = gone.all(1)
                p = torch.softmax(s, 1)[:, :L]
                p = torch.where(empty[:, None], torch.zeros_like(p), p)
                e = 2 * (2 * err.amax(1, keepdim=True) + (32 + 96) * u) if rows else torch.zeros(0, 1, dtype=torch.float64)
                total += p.sum(0)
                off += (p * e).sum(0)
            old = torch.zeros(L, dtype=torch.float64)
            old[:c] = weights[slot, h, :c].double()
            res[slot, h, :L] = old + total
            tol[slot, h, :L] = off + (rows * G + 2) * u * (old.abs() + total) + 1e-37
    return res, tol


def evict(cache, table, slot_ids, lens, weights, positions, weights_out, positions_out, keep, first, recent):
    """The three outputs of ``ops.evict_tokens`` on copies of its operands."""
    cache, wo, po = cache.clone(), weights_out.clone(), positions_out.clone()
    P = cache.shape[4]
    for layer in range(cache.shape[0]):
        for r in range(len(lens)):
            n, slot = int(lens[r]), int(slot_ids[r])
            for h in range(cache.shape[3]):
                w, at = weights[layer, slot, h, :n].tolist(), positions[layer, slot, h, :n].tolist()
                stays = set(range(n))
                if n > keep:
                    latest = max(at)

                    def rank(i):
                        if at[i] < first or at[i] > latest - recent:
                            return (0, 0.0, i)
                        return (1, math.inf if math.isnan(w[i]) else -w[i], i)
                    stays = set(sorted(range(n), key=rank)[:keep])
                end = min(n, keep)
                holes = [i for i in range(end) if i not in stays]
                movers = sorted(i for i in stays if i >= keep)
                assert len(holes) == len(movers)
                for i in range(end):
                    wo[layer, slot, h, i], po[layer, slot, h, i] = weights[layer, slot, h, i], positions[layer, slot, h, i]
                for to, frm in zip(holes, movers):
                    wo[layer, slot, h, to], po[layer, slot, h, to] = weights[layer, slot, h, frm], positions[layer, slot, h, frm]
                    cache[layer, int(table[r, to // P]), :, h, to % P] = cache[layer, int(table[r, frm // P]), :, h, frm % P]
    return cache, wo, po
