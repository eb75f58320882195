"""Plain float64 forms of the generation operators, on the CPU, one element after the other."""
import math

import torch

NONE = float("-inf")
BLOCK = 64


def log_probabilities(row):
    """log softmax of a list of floats; NaN counts as -inf, +inf share everything; None where nothing is left."""
    row = [NONE if x != x else x for x in row]
    top = max(row)
    if top == NONE:
        return None
    if top == math.inf:
        n = sum(x == math.inf for x in row)
        return [-math.log(n) if x == math.inf else NONE for x in row]
    total = math.fsum(math.exp(x - top) for x in row)
    lse = top + math.log(total)
    return [x - lse for x in row]


def step(logits, scores, pool_scores, pool_steps, pool_beams, done, pos, eos=1, pad=0, length_penalty=1.0, early=False):
    """Lists in, lists out, for a whole batch: (tokens, parents, scores, pool scores, steps, beams, done)."""
    B, K = len(scores), len(scores[0])
    out = []
    for b in range(B):
        if done[b]:
            out.append(([pad] * K, list(range(K)), scores[b], pool_scores[b], pool_steps[b], pool_beams[b], True))
            continue
        ranked = []
        for k in range(K):
            row = [NONE if x != x else x for x in logits[b * K + k]]
            run = scores[b][k] if scores[b][k] == scores[b][k] else NONE
            logp = log_probabilities(row) if run > NONE else None
            for t, x in enumerate(row):
                value = NONE if logp is None else run + logp[t]
                ranked.append((-(value if value == value else NONE), k, -x, t))
        ranked = sorted(ranked)[:2 * K]
        length = float(pos + 1) ** length_penalty
        pool = [(s if s == s else NONE, st, be) for s, st, be in zip(pool_scores[b], pool_steps[b], pool_beams[b])]
        for value, k, _, t in ranked[:K]:
            if t == eos and -value > NONE:
                pool.append((torch.tensor(-value / length, dtype=torch.float64).float().item(), pos, k))
        pool = sorted(pool, key=lambda e: -e[0])[:K]
        on = [(k, t, -value) for value, k, _, t in ranked if t != eos][:K]
        places, free = {}, sorted(set(range(K)) - {k for k, _, _ in on})
        for k, t, value in on:
            places[k if k not in places else free.pop(0)] = (t, k, value)
        tokens, parents, new = zip(*(places[j] for j in range(K)))
        highest = max(torch.tensor(v, dtype=torch.float64).float().item() for v in new)
        full = pool[-1][0] > NONE and (early or pool[-1][0] >= highest / length)
        out.append((list(tokens), list(parents), list(new), *[list(c) for c in zip(*pool)], full or highest == NONE))
    return [list(c) for c in zip(*out)]


def sequences(tokens, parents, scores, pool_scores, pool_steps, pool_beams, done, R, eos=1, pad=0, length_penalty=1.0):
    T, B, K = len(tokens), len(tokens[0]), len(tokens[0][0])
    every, values = [], []
    for b in range(B):
        cand = [(pool_scores[b][j], pool_steps[b][j] - 1, pool_beams[b][j], [eos]) for j in range(K)]
        cand += [(NONE if done[b] else scores[b][j] / T ** length_penalty, T - 1, j, []) for j in range(K)]
        cand = sorted(cand, key=lambda c: -c[0])[:R]
        values.append([c[0] for c in cand])
        rows = []
        for value, t, beam, tail in cand:
            words = []
            if value > NONE:
                while t >= 0:
                    words.append(tokens[t][b][beam])
                    beam = parents[t][b][beam]
                    t -= 1
                words = words[::-1] + tail
            rows.append(words + [pad] * (T - len(words)))
        every.append(rows)
    return every, values


def scale_of(values):
    """The block scale of a float64 tensor's finite elements: the smallest power of two that fits the largest."""
    finite = values[torch.isfinite(values)].abs()
    most = finite.max().item() if finite.numel() else 0.0
    e = -100
    while e < 120 and most > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def round_e4m3(y):
    """float64 -> nearest e4m3 number (ties to even), saturating; NaN stays."""
    a = y.abs().clamp(max=1e30)
    e = torch.floor(torch.log2(a.clamp(min=2.0 ** -30)))
    e = torch.where(a >= 2.0 ** (e + 1), e + 1, torch.where(a < 2.0 ** e, e - 1, e)).clamp(min=-6)
    step = 2.0 ** (e - 3)
    r = (torch.round(a / step) * step).clamp(max=448.0)
    return torch.where(y != y, y, torch.copysign(r, y))


def fill(x, cache, scale, start, counts):
    """x (B,H,M,D) into cache values (B,H,cap,D) and scales (B,H,cap/64), all float64; new tensors."""
    cache, scale = cache.clone(), scale.clone()
    B, H, M, D = x.shape
    cap = cache.shape[2]
    for b in range(B):
        end = min(start + min(max(counts[b], 0), M), cap)
        for h in range(H):
            t = start
            while t < end:
                blk = t // BLOCK
                hi = min(end, (blk + 1) * BLOCK)
                fresh = x[b, h, t - start:hi - start]
                s = scale_of(fresh)
                if t > blk * BLOCK:
                    was = scale[b, h, blk].item()
                    s = max(s, was)
                    cache[b, h, blk * BLOCK:t] = round_e4m3(cache[b, h, blk * BLOCK:t] * (was / s))
                cache[b, h, t:hi] = round_e4m3(fresh / s)
                scale[b, h, blk] = s
                t = hi
    return cache, scale


def bucket(delta, nb, md, bidirectional):
    """T5's bucket of key position - query position, in whole numbers."""
    side, base = (nb // 2, nb // 2 if delta > 0 else 0) if bidirectional else (nb, 0)
    d = abs(delta) if bidirectional else max(-delta, 0)
    half = side // 2
    if d < half:
        return base + d
    rest, j = side - half, 0
    while j + 1 < rest and d ** rest * half ** (j + 1) >= half ** rest * md ** (j + 1):
        j += 1
    return base + half + j


def attend(q, k, v, table, lengths, causal, scale, nb=32, md=128, q_pos_offset=None):
    """(out, error scale): attention in float64 of q (B,H,M,D) over the first lengths[b] keys, and for every output the sum
    of |weight * value| and the largest sum |q k| * scale of its row, which rounding errors are relative to."""
    B, H, M, D = q.shape
    out, mass, size = torch.zeros(B, H, M, D, dtype=torch.float64), torch.zeros(B, H, M, D, dtype=torch.float64), torch.zeros(B, H, M, 1, dtype=torch.float64)
    for b, n in enumerate(lengths):
        off = n - M if q_pos_offset is None else q_pos_offset
        for m in range(M):
            seen = min(n, max(off + m + 1, 0)) if causal else n
            if seen == 0:
                continue
            kk, vv = k[b, :, :seen].double(), v[b, :, :seen].double()
            s = torch.einsum("hd,hnd->hn", q[b, :, m].double(), kk) * scale
            size[b, :, m, 0] = (torch.einsum("hd,hnd->hn", q[b, :, m].double().abs(), kk.abs()) * abs(scale)).amax(-1)
            if table is not None:
                idx = torch.tensor([bucket(j - off - m, nb, md, not causal) for j in range(seen)])
                s = s + table.double()[idx].t()
                size[b, :, m, 0] += table.double().abs().amax(0)
            p = torch.softmax(s, -1)
            out[b, :, m] = torch.einsum("hn,hnd->hd", p, vv)
            mass[b, :, m] = torch.einsum("hn,hnd->hd", p, vv.abs())
    return out, mass, size
