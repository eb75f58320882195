"""The operators of beam search over a cache, as they are timed and compared: five calls of one generation step.

A case is a dict of plain values with a `kind`:

* `step`       `beam_search_step`: log-probabilities, the best continuations over beams and vocabulary, the pool of
               finished sentences
* `sequences`  `beam_search_sequences`: the best sentences read back from the tokens and parents of every step
* `reorder`    `reorder_beam_cache`: the cached keys and values of every layer follow their beams, in place
* `quantize`   `quantize_into_cache`: keys and values into a cache of 8-bit floats with a scale per 64 tokens and head
* `attend`     `flash_decoding_quantized_with_fusing_bias`: a few query rows against such a cache

`run` computes a case with elementary tensor operations where `own` is false and with the framework's operators where
it is true; `exact` is the operators' definition in 64 bits.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}
_FP8 = torch.float8_e4m3fn
_BLOCK = 64                        # tokens that share a scale
_BUCKETS, _MAX_DISTANCE = 32, 128
_LOWEST, _HIGHEST = -100, 120      # exponents of a scale
_EOS, _PAD = 1, 0
_NONE = float("-inf")


def listed():
    return [
        # One sentence translated with four beams: the smallest step of a generation, all latency.
        dict(name="step_one_sentence", kind="step", B=1, K=4, V=32128, pos=17, dtype="bf16", first=False, masked=0.0,
             length_penalty=1.0, early_stopping=False),
        # A full serving batch of summaries with the usual four beams.
        dict(name="step_batch", kind="step", B=64, K=4, V=32128, pos=60, dtype="bf16", first=False, masked=0.0,
             length_penalty=2.0, early_stopping=True),
        # A wide search over a large vocabulary of odd size, logits in float32 after a processor that masks tokens.
        dict(name="step_wide_fp32", kind="step", B=8, K=16, V=65537, pos=5, dtype="fp32", first=False, masked=0.3,
             length_penalty=0.6, early_stopping=False),
        # The answer of one short generation.
        dict(name="sequences_one", kind="sequences", B=1, K=4, T=32, returned=1, ended=1),
        # Every hypothesis of a batch of long generations.
        dict(name="sequences_batch", kind="sequences", B=64, K=8, T=512, returned=8, ended=2),
        # The 16-bit cache of a twelve-layer decoder early in the generation of one sentence.
        dict(name="reorder_one_sentence", kind="reorder", layers=12, B=1, K=4, H=12, D=64, cap=128, used=41, dtype="bf16",
             slots=False, pattern=3),
        # The 8-bit cache of a deep decoder late in the generation of a batch, parents as the step leaves them.
        dict(name="reorder_batch_8bit", kind="reorder", layers=24, B=8, K=4, H=16, D=64, cap=512, used=500, dtype="fp8",
             slots=True, pattern=4),
        # One layer's cross-attention keys and values of a batch of prompts of every length.
        dict(name="quantize_prompts", kind="quantize", B=16, H=12, D=64, M=1024, cap=1024, start=0, dtype="bf16", lengths=5),
        # The newest token of a batch of beams, in the middle of a block of tokens.
        dict(name="quantize_token", kind="quantize", B=64, H=16, D=64, M=1, cap=512, start=203, dtype="fp16", lengths=0),
        # Self-attention of one sentence's beams, a few hundred cached keys.
        dict(name="attend_self_beams", kind="attend", B=4, M=1, H=12, D=64, cap=512, used=200, lengths=0, causal=True,
             dtype="bf16"),
        # Cross attention of a batch: the four beams of a sentence read its keys together, prompts of every length.
        dict(name="attend_cross_beams", kind="attend", B=16, M=4, H=12, D=64, cap=2048, used=2000, lengths=7, causal=False,
             dtype="fp16"),
        # Cross attention of one large-shaped decoder layer for a full serving batch: the K/V stream.
        dict(name="attend_serving_batch", kind="attend", B=64, M=1, H=16, D=64, cap=8192, used=8192, lengths=0, causal=False,
             dtype="bf16"),
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random):
    kind = rng.choice(("step", "step", "step", "sequences", "reorder", "quantize", "quantize", "attend", "attend", "attend"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    half = rng.choice(("bf16", "fp16"))
    D = rng.choice((64, 64, 64, 128, 32, 16))
    if kind == "step":
        K = rng.choice((1, 2, 3, 4, 4, 5, 8, 10, 16))
        V = rng.choice((32128, _between(rng, 100, 200000), _between(rng, 1000, 70000)))
        B = max(1, min(_between(rng, 1, 128), int(8 * 16 * 65537 / (K * V))))
        return dict(kind=kind, B=B, K=K, V=V, pos=rng.randrange(128), dtype=dtype, first=rng.random() < 0.15,
                    masked=rng.choice((0.0, 0.0, 0.3, 0.9)), length_penalty=rng.choice((0.0, 0.6, 1.0, 1.0, 2.0)),
                    early_stopping=rng.random() < 0.5)
    if kind == "sequences":
        K = rng.choice((1, 2, 4, 5, 8, 16))
        return dict(kind=kind, B=_between(rng, 1, 64), K=K, T=_between(rng, 1, 512), returned=rng.randint(1, K),
                    ended=rng.randrange(1 << 20))
    if kind == "reorder":
        K, cap = rng.choice((2, 3, 4, 4, 5, 8, 16)), _between(rng, 16, 1024)
        stored = rng.choice(("fp8", "bf16", "fp32"))
        if stored == "fp8":
            cap = -(-cap // _BLOCK) * _BLOCK
        H = rng.choice((8, 12, 16))
        row = K * H * cap * D * 2 * _BYTES[stored]
        layers = max(1, min(rng.choice((1, 6, 12, 24)), int(8e8 / row)))
        row *= layers
        return dict(kind=kind, layers=layers, B=max(1, min(_between(rng, 1, 32), int(8e8 / row))), K=K, H=H, D=D, cap=cap,
                    used=rng.randint(1, cap), dtype=stored, slots=rng.random() < 0.6, pattern=rng.randrange(1 << 20))
    H = rng.choice((8, 12, 16))
    if kind == "quantize":
        if rng.random() < 0.5:
            cap = _BLOCK * _between(rng, 1, 32)
            return dict(kind=kind, B=_between(rng, 1, 128), H=H, D=D, M=1, cap=cap, start=rng.randrange(cap), dtype=dtype,
                        lengths=0)
        M = _between(rng, 2, 8192)
        start = rng.choice((0, 0, _between(rng, 1, 200)))
        return dict(kind=kind, B=max(1, min(_between(rng, 1, 32), int(2e8 / (H * M * D)))), H=H, D=D, M=M,
                    cap=-(-(start + M + rng.randrange(100)) // _BLOCK) * _BLOCK, start=start, dtype=dtype,
                    lengths=rng.choice((0, rng.randrange(1, 1 << 20))))
    causal = rng.random() < 0.5
    used = _between(rng, 1, 2048 if causal else 16384)
    M = min(used, rng.choice((1, 1, 2, 3, 4, 5, 8, 16)))
    cap = -(-(used + rng.randrange(200)) // _BLOCK) * _BLOCK
    return dict(kind=kind, B=max(1, min(_between(rng, 1, 128), int(5e8 / (H * cap * D)))), M=M, H=H, D=D, cap=cap, used=used,
                lengths=rng.choice((0, rng.randrange(1, 1 << 20))), causal=causal, dtype=half)


# ---- what follows from a case

def _lengths(case):
    """Cached keys (new tokens) of every batch row: all of them, or between an eighth and all."""
    most = case["used"] if case["kind"] == "attend" else case["M"]
    if not case["lengths"]:
        return [most] * case["B"]
    r = random.Random(case["lengths"])
    least = case.get("M", 1) if case["kind"] == "attend" and case["causal"] else 1
    return [r.randint(min(most, max(least, most // 8)), most) for _ in range(case["B"])]


def _parents(case):
    """The beam that each beam of a sentence continues, one list per sentence.  The best beams have the most
    continuations; with `slots` a beam that goes on stays where it is and only further continuations move."""
    r = random.Random(case["pattern"])
    K, every = case["K"], []
    for _ in range(case["B"]):
        ranked = [min(K - 1, int(r.expovariate(1.0) * K / 3)) for _ in range(K)]
        if case["slots"]:
            goes_on = set(ranked)
            free = [j for j in range(K) if j not in goes_on]
            again = [p for i, p in enumerate(ranked) if p in ranked[:i]]
            ranked = [j if j in goes_on else again[free.index(j)] for j in range(K)]
        every.append(ranked)
    return every


def work(case):
    kind = case["kind"]
    if kind == "step":
        # Every logit read once, a maximum, a difference, an exponential and a sum for each; a few numbers per beam.
        n = case["B"] * case["K"] * case["V"]
        return {"bytes": n * _BYTES[case["dtype"]] + case["B"] * case["K"] * 48, "flops": 4 * n}
    if kind == "sequences":
        # A token and a parent read and a token written for every position of every sentence that is returned.
        return {"bytes": case["B"] * case["returned"] * (case["T"] * (4 + 4 + 8) + 4), "flops": 0}
    if kind == "reorder":
        # The beams that change are written; the ones that they continue are read.
        moved = 0
        for parents in _parents(case):
            changed = [j for j, p in enumerate(parents) if p != j]
            moved += len(changed) + len({parents[j] for j in changed})
        per = case["used"] * case["D"] * _BYTES[case["dtype"]]
        if case["dtype"] == "fp8":
            per += -(-case["used"] // _BLOCK) * 4
        return {"bytes": max(1, moved) * case["layers"] * 2 * case["H"] * per + case["B"] * case["K"] * 4, "flops": 0}
    if kind == "quantize":
        tokens = sum(_lengths(case))
        blocks = sum(-(-(case["start"] % _BLOCK + n) // _BLOCK) for n in _lengths(case))
        per_head = tokens * case["D"] * (_BYTES[case["dtype"]] + 1) + blocks * 4
        return {"bytes": 2 * case["H"] * per_head, "flops": 4 * case["H"] * tokens * case["D"]}
    keys = sum(_lengths(case))
    scales = sum(-(-n // _BLOCK) for n in _lengths(case))
    rows = case["B"] * case["H"] * case["M"] * case["D"]
    return {"bytes": 2 * case["H"] * (keys * case["D"] + scales * 4) + 2 * rows * _BYTES[case["dtype"]],
            "flops": 4 * case["H"] * case["M"] * case["D"] * keys}


# ---- inputs

def _normal(g, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _ints(g, high, shape, dtype):
    return torch.randint(0, high, shape, generator=g, device="cuda").to(dtype)


def _eight_bit(g, shape):
    """A cache (..., cap, D) of 8-bit values with their scales (..., cap / 64), as keys of N(0, 1) leave it, with rows
    and heads of different magnitude."""
    *lead, cap, D = shape
    scale = torch.exp2(torch.randint(-8, -5, (*lead, cap // _BLOCK), generator=g, device="cuda").float())
    return (_normal(g, shape, std=64.0).clamp_(-448, 448)).to(_FP8), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, s = case["kind"], dict(case=case)
    if kind == "step":
        B, K, V, pos = case["B"], case["K"], case["V"], case["pos"]
        logits = _normal(g, (B * K, V), std=2.5)
        # some beams are about to end: the end token is among their best
        logits[:, _EOS] += torch.where(torch.rand(B * K, generator=g, device="cuda") < 0.3, 10.0, 0.0)
        if case["masked"]:
            logits.masked_fill_(torch.rand(V, generator=g, device="cuda") < case["masked"], _NONE)
        s["logits"] = logits.to(_DTYPES[case["dtype"]])
        scores = -_normal(g, (B, K)).abs() * 2 - 1.3 * (pos + 1)
        if case["first"]:
            scores = torch.full((B, K), _NONE, device="cuda")
            scores[:, 0] = 0.0
        s["scores"] = scores
        # a pool with a few ended sentences, best first
        ended = torch.rand((B, K), generator=g, device="cuda") < 0.3
        ended &= pos > 0 and not case["first"]
        pool = torch.where(ended, (scores - 1.5 * _normal(g, (B, K)).abs()) / (pos + 1) ** case["length_penalty"], _NONE)
        s["finished_scores"] = pool.sort(-1, descending=True)[0]
        s["finished_steps"] = _ints(g, pos + 1, (B, K), torch.int32)
        s["finished_beams"] = _ints(g, K, (B, K), torch.int32)
        s["done"] = torch.zeros(B, dtype=torch.bool, device="cuda")
        s["pos"] = torch.full((1,), pos, dtype=torch.long, device="cuda")
        s["out"] = (torch.empty((B, K), dtype=torch.long, device="cuda"),
                    torch.empty((B, K), dtype=torch.int32, device="cuda"),
                    *(torch.empty_like(s[n]) for n in ("scores", "finished_scores", "finished_steps", "finished_beams", "done")))
    elif kind == "sequences":
        B, K, T = case["B"], case["K"], case["T"]
        s["tokens"] = _ints(g, 32000, (T, B, K), torch.int32) + 2
        s["parents"] = _ints(g, K, (T, B, K), torch.int32)
        s["scores"] = -_normal(g, (B, K)).abs() * 2 - T
        share = random.Random(case["ended"]).random()
        ended = torch.rand((B, K), generator=g, device="cuda") < share
        s["finished_scores"] = torch.where(ended, -1 - _normal(g, (B, K)).abs(), _NONE).sort(-1, descending=True)[0]
        s["finished_steps"] = _ints(g, T, (B, K), torch.int32)
        s["finished_beams"] = _ints(g, K, (B, K), torch.int32)
        s["done"] = torch.rand(B, generator=g, device="cuda") < 0.5 * share
    elif kind == "reorder":
        B, K, H, cap, D, n = case["B"], case["K"], case["H"], case["cap"], case["D"], case["layers"]
        shape = (n, 2, B * K, H, cap, D)
        s["scales"] = None
        if case["dtype"] == "fp8":
            s["cache"], s["scales"] = _eight_bit(g, shape)
        else:
            s["cache"] = _normal(g, shape, _DTYPES[case["dtype"]])
        order = torch.randperm(B, generator=g, device="cuda")
        s["parents"] = torch.tensor(_parents(case), dtype=torch.int32, device="cuda")[order].contiguous()
        s["seqlens"] = torch.full((B * K,), case["used"], dtype=torch.int32, device="cuda")
        s["layers"] = list(s["cache"].unbind(0))
        s["layer_scales"] = [] if s["scales"] is None else list(s["scales"].unbind(0))
    elif kind == "quantize":
        B, H, M, D, cap = case["B"], case["H"], case["M"], case["D"], case["cap"]
        dtype = _DTYPES[case["dtype"]]
        # a view of token-major rows, as the stacked projection gives it; one token in fifty is an outlier
        kv = _normal(g, (B, M, 2, H, D))
        kv *= torch.where(torch.rand((B, M, 1, 1, 1), generator=g, device="cuda") < 0.02, 16.0, 1.0)
        s["k"], s["v"] = (t.transpose(1, 2) for t in kv.to(dtype).unbind(2))
        s["k_cache"], s["k_scale"] = _eight_bit(g, (B, H, cap, D))
        s["v_cache"], s["v_scale"] = _eight_bit(g, (B, H, cap, D))
        s["start"] = torch.full((1,), case["start"], dtype=torch.long, device="cuda") if M == 1 else case["start"]
        s["seqlens"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["lengths"] else None
    else:
        B, M, H, D, cap = case["B"], case["M"], case["H"], case["D"], case["cap"]
        dtype = _DTYPES[case["dtype"]]
        s["q"] = _normal(g, (B, M, H, D), dtype, std=D ** -0.5 * 2).transpose(1, 2)
        s["k"], s["k_scale"] = _eight_bit(g, (B, H, cap, D))
        s["v"], s["v_scale"] = _eight_bit(g, (B, H, cap, D))
        s["table"] = _normal(g, (_BUCKETS, H), dtype, 0.5) if case["causal"] else None
        s["seqlens"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    return s


# ---- one pass

def run(s):
    return _own(s) if own else _PLAIN[s["case"]["kind"]](s)


def _own(s):
    import turbot5_b200 as t5b
    c = s["case"]
    kind = c["kind"]
    if kind == "step":
        return t5b.beam_search_step(s["logits"], s["scores"], s["finished_scores"], s["finished_steps"], s["finished_beams"],
                                    s["done"], s["pos"], eos_token_id=_EOS, pad_token_id=_PAD,
                                    length_penalty=c["length_penalty"], early_stopping=c["early_stopping"], out=s["out"])
    if kind == "sequences":
        return t5b.beam_search_sequences(s["tokens"], s["parents"], s["scores"], s["finished_scores"], s["finished_steps"],
                                         s["finished_beams"], s["done"], num_return_sequences=c["returned"],
                                         pad_token_id=_PAD, length_penalty=1.0)
    if kind == "reorder":
        t5b.reorder_beam_cache(s["layers"], s["parents"], seqlens=s["seqlens"], scales=s["layer_scales"])
        return (s["cache"],) if s["scales"] is None else (s["cache"], s["scales"])
    if kind == "quantize":
        t5b.quantize_into_cache(s["k"], s["v"], s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"], s["start"],
                                seqlens=s["seqlens"])
        return s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"]
    return t5b.flash_decoding_quantized_with_fusing_bias(s["q"], s["k"], s["k_scale"], s["v"], s["v_scale"], s["table"],
                                                         causal=c["causal"], sm_scale=1.0, NUM_BUCKETS=_BUCKETS,
                                                         MAX_DISTANCE=_MAX_DISTANCE, seqlens_k=s["seqlens"])


def _plain_step(s):
    """The order of candidates is decided by sums of numbers that differ in their last bits: in 64 bits."""
    c = s["case"]
    B, K, V = c["B"], c["K"], c["V"]
    n, taken = 2 * K, min(2 * K, V)
    x = s["logits"].view(B, K, V).double()
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    # within a beam by the logit, lowest token first; then over the beams, lowest beam first
    best, token = x.sort(dim=-1, descending=True, stable=True)
    total = (s["scores"].double()[..., None] + (best - lse)[..., :taken]).flatten(1)
    total, at = total.sort(dim=-1, descending=True, stable=True)
    total, at = total[:, :n], at[:, :n]
    beam, token = at // taken, token[..., :taken].flatten(1).gather(1, at)
    ends = token == _EOS
    length = (s["pos"] + 1).double() ** c["length_penalty"]
    # ended sentences among the K best candidates join the pool
    joins = ends & (torch.arange(n, device=x.device) < K) & (total > _NONE)
    pool = torch.cat([s["finished_scores"], torch.where(joins, total / length, _NONE).float()], 1)
    pool, keep = pool.sort(dim=-1, descending=True, stable=True)
    pool, keep = pool[:, :K].contiguous(), keep[:, :K]
    steps = torch.cat([s["finished_steps"], s["pos"].int().expand(B, n)], 1).gather(1, keep)
    beams = torch.cat([s["finished_beams"], beam.int()], 1).gather(1, keep)
    # the K best that go on; one that continues a beam stays in its place, further ones take the free places in order
    on = ends.int().argsort(dim=-1, stable=True)[:, :K]
    beam, token, total = beam.gather(1, on), token.gather(1, on), total.gather(1, on)
    earlier = torch.ones((K, K), dtype=torch.bool, device=x.device).tril(-1)
    further = ((beam[:, :, None] == beam[:, None, :]) & earlier).any(-1)
    used = torch.zeros((B, K), dtype=torch.int32, device=x.device).scatter_(1, beam, 1)
    free = used.argsort(dim=-1, stable=True)
    place = torch.where(further, free.gather(1, (further.cumsum(-1) - 1).clamp(min=0)), beam)
    token, parent, scores = (torch.empty_like(t).scatter_(1, place, t) for t in (token, beam.int(), total.float()))
    full = pool[:, -1] > _NONE
    highest = scores.amax(-1)
    if not c["early_stopping"]:
        full &= pool[:, -1].double() >= highest.double() / length
    return token, parent, scores, pool, steps, beams, full | (highest == _NONE) | s["done"]


def _plain_sequences(s):
    c = s["case"]
    T, K, R = c["T"], c["K"], c["returned"]
    tokens, parents = s["tokens"].long(), s["parents"].long()
    running = torch.where(s["done"][:, None], _NONE, s["scores"] / T)
    scores, at = torch.cat([s["finished_scores"], running], 1).sort(dim=-1, descending=True, stable=True)
    scores, at = scores[:, :R].contiguous(), at[:, :R]
    ended = at < K
    slot = at.clamp(max=K - 1)
    last = torch.where(ended, s["finished_steps"].long().gather(1, slot), T - 1)
    # the beam of every step as a function of the next step's: a constant at a sentence's last beam, the parent
    # before it; composed with twice as many steps each time
    start = torch.where(ended, s["finished_beams"].long().gather(1, slot), (at - K).clamp(min=0))
    at_last = torch.where(ended, last - 1, last)
    step = torch.arange(T, device=tokens.device).view(T, 1, 1, 1)
    follow = torch.cat([parents[1:], parents[:1]])[:, :, None, :].expand(T, -1, R, K)
    beam = torch.where(step >= at_last[..., None], start[..., None], follow)
    ahead = 1
    while ahead < T:
        beam = torch.cat([beam[:-ahead].gather(-1, beam[ahead:]), beam[-ahead:]])
        ahead *= 2
    words = tokens.gather(-1, beam[..., 0]).permute(1, 2, 0)
    t = torch.arange(T, device=tokens.device)
    words = torch.where(t <= at_last[..., None], words, _PAD)
    words = torch.where((t == last[..., None]) & ended[..., None], _EOS, words)
    return torch.where((scores == _NONE)[..., None], _PAD, words), scores


def _plain_reorder(s):
    c = s["case"]
    B, K, n = c["B"], c["K"], c["used"]
    rows = (s["parents"].long() + torch.arange(B, device="cuda")[:, None] * K).flatten()
    cache = s["cache"].view(torch.uint8) if s["scales"] is not None else s["cache"]
    cache[..., :n, :] = cache[..., :n, :].index_select(2, rows)
    if s["scales"] is None:
        return (s["cache"],)
    blocks = -(-n // _BLOCK)
    s["scales"][..., :blocks] = s["scales"][..., :blocks].index_select(2, rows)
    return s["cache"], s["scales"]


def _exponent(largest):
    """The smallest e with largest <= 448 * 2^e, between the lowest and the highest."""
    m, e = torch.frexp(largest.double() / 448.0)
    return torch.where(largest > 0, torch.where(m > 0.5, e, e - 1), _LOWEST).clamp(_LOWEST, _HIGHEST)


def _plain_fill(x, cache, scale, case, seqlens):
    M, start = case["M"], case["start"]
    first, last = start // _BLOCK, -(-(start + M) // _BLOCK)
    span = slice(first * _BLOCK, last * _BLOCK)
    shape = (*cache.shape[:2], last - first, _BLOCK, cache.shape[-1])
    old = cache[:, :, span].float().reshape(shape)
    new = torch.nn.functional.pad(x.float(), (0, 0, start % _BLOCK, last * _BLOCK - start - M)).reshape(shape)
    at = torch.arange(first * _BLOCK, last * _BLOCK, device=x.device).view(1, 1, -1, _BLOCK, 1)
    count = torch.full((x.shape[0],), M, device=x.device) if seqlens is None else seqlens.long()
    written = (at >= start) & (at < start + count.view(-1, 1, 1, 1, 1))
    kept = (at < start) & torch.ones_like(written)
    was = scale[:, :, first:last]
    e = _exponent(torch.where(written, new.abs(), 0.0).amax((-1, -2)))
    before = kept.any(-2).squeeze(-1)
    e = torch.where(before, torch.maximum(e, torch.log2(was).round().int()), e)
    now = torch.where(written.any(-2).squeeze(-1), torch.exp2(e.float()), was)
    value = torch.where(written, new / now[..., None, None], old)
    value = torch.where(kept, old * (was / now)[..., None, None], value)
    cache[:, :, span] = value.clamp(-448, 448).to(_FP8).reshape(cache[:, :, span].shape)
    scale[:, :, first:last] = now


def _plain_quantize(s):
    _plain_fill(s["k"], s["k_cache"], s["k_scale"], s["case"], s["seqlens"])
    _plain_fill(s["v"], s["v_cache"], s["v_scale"], s["case"], s["seqlens"])
    return s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"]


def _bias(table, delta):
    """T5's bias of keys at or before the query: table rows by the distance, logarithmic from half of the buckets on."""
    distance = (-delta).clamp(min=0)
    half = _BUCKETS // 2
    far = half + (torch.log(distance.clamp(min=1).float() / half) / math.log(_MAX_DISTANCE / half) * (_BUCKETS - half)).long()
    return table.float()[torch.where(distance < half, distance, far.clamp(max=_BUCKETS - 1))]


def _plain_attend(s):
    c = s["case"]
    n = c["used"]
    k = s["k"][:, :, :n].float() * s["k_scale"].repeat_interleave(_BLOCK, -1)[:, :, :n, None]
    v = s["v"][:, :, :n].float() * s["v_scale"].repeat_interleave(_BLOCK, -1)[:, :, :n, None]
    scores = s["q"].float() @ k.transpose(-1, -2)
    at = torch.arange(n, device=k.device)
    lengths = s["seqlens"].long()
    visible = (at < lengths[:, None])[:, None, None, :]
    if c["causal"]:
        query = lengths[:, None] - c["M"] + torch.arange(c["M"], device=k.device)
        delta = at - query[..., None]
        scores += _bias(s["table"], delta).permute(0, 3, 1, 2)
        visible = visible & (delta <= 0)[:, None]
    scores = torch.where(visible, scores, _NONE)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return (p @ v / p.sum(-1, keepdim=True)).to(s["q"].dtype)


_PLAIN = {"step": _plain_step, "sequences": _plain_sequences, "reorder": _plain_reorder, "quantize": _plain_quantize,
          "attend": _plain_attend}


# ---- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s)


def _exact_step(s):
    c = s["case"]
    B, K, V = c["B"], c["K"], c["V"]
    logits = s["logits"].to(torch.float64).reshape(B, K, V)
    flat = (s["scores"].to(torch.float64)[:, :, None] + logits - torch.logsumexp(logits, -1, keepdim=True)).reshape(B, K * V)
    every, index = torch.topk(flat, min(4 * K + 64, K * V), dim=-1)
    every, index, L = every.tolist(), index.tolist(), float(c["pos"] + 1) ** c["length_penalty"]
    fs, fp, fb = (s[n].tolist() for n in ("finished_scores", "finished_steps", "finished_beams"))
    result = []
    for b in range(B):
        # equal values: lowest beam and token first
        ranked = sorted(zip(every[b], index[b]), key=lambda t: (-t[0], t[1]))[:2 * K]
        pool = list(zip(fs[b], fp[b], fb[b]))
        pool += [(v / L, c["pos"], i // V) for v, i in ranked[:K] if i % V == _EOS and v > _NONE]
        pool = sorted(pool, key=lambda t: -t[0])[:K]
        on = [(v, i // V, i % V) for v, i in ranked if i % V != _EOS][:K]
        places, free = {}, sorted(set(range(K)) - {p for _, p, _ in on})
        for hyp in on:
            places[hyp[1] if hyp[1] not in places else free.pop(0)] = hyp
        # (a place that is handed to a later continuation is never the parent of another: those keep their own)
        beams = [places[j] for j in range(K)]
        highest = max(v for v, _, _ in beams)
        full = pool[-1][0] > _NONE and (c["early_stopping"] or pool[-1][0] >= highest / L)
        result.append(([t for _, _, t in beams], [p for _, p, _ in beams], [v for v, _, _ in beams], [t[0] for t in pool],
                       [t[1] for t in pool], [t[2] for t in pool], full or highest == _NONE))
    types = (torch.int64, torch.int32, torch.float64, torch.float64, torch.int32, torch.int32, torch.bool)
    return tuple(torch.tensor(list(column), dtype=t) for column, t in zip(zip(*result), types))


def _exact_sequences(s):
    c = s["case"]
    T, K, R = c["T"], c["K"], c["returned"]
    tokens, parents = s["tokens"].tolist(), s["parents"].tolist()
    run, fs, fp, fb = (s[n].tolist() for n in ("scores", "finished_scores", "finished_steps", "finished_beams"))
    done, rows, values = s["done"].tolist(), [], []
    for b in range(c["B"]):
        pool = [(fs[b][j], fp[b][j] - 1, fb[b][j], [_EOS]) for j in range(K)]
        pool += [(_NONE if done[b] else run[b][j] / T, T - 1, j, []) for j in range(K)]
        pool = sorted(pool, key=lambda t: -t[0])[:R]
        values.append([t[0] for t in pool])
        rows.append([])
        for value, t, beam, tail in pool:
            words = []
            while t >= 0 and value > _NONE:
                words.append(tokens[t][b][beam])
                beam = parents[t][b][beam]
                t -= 1
            words = words[::-1] + (tail if value > _NONE else [])
            rows[-1].append(words + [_PAD] * (T - len(words)))
    return torch.tensor(rows, dtype=torch.int64), torch.tensor(values, dtype=torch.float64)


def _exact_reorder(s):
    c = s["case"]
    n, K = c["used"], c["K"]
    shape = s["cache"].shape
    values = s["cache"].view(torch.uint8) if s["scales"] is not None else s["cache"]
    by_beam = values.unflatten(2, (-1, K))
    index = s["parents"].long()[None, None, :, :, None, None, None].expand(*by_beam.shape[:5], n, shape[-1])
    moved = torch.cat([torch.gather(by_beam[..., :n, :], 3, index), by_beam[..., n:, :]], -2).flatten(2, 3)
    if s["scales"] is None:
        return (moved.double(),)
    blocks = -(-n // _BLOCK)
    scales = s["scales"].unflatten(2, (-1, K))
    index = s["parents"].long()[None, None, :, :, None, None].expand(*scales.shape[:5], blocks)
    scales = torch.cat([torch.gather(scales[..., :blocks], 3, index), scales[..., blocks:]], -1).flatten(2, 3)
    return moved.contiguous().view(_FP8).double(), scales.double()


def _to_eight_bits(y):
    """The nearest number with three bits after the leading one and exponents from -6 on, ties to even."""
    exponent = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    exponent += (y.abs() >= torch.exp2(exponent + 1)).double() - (y.abs() < torch.exp2(exponent)).double() * (exponent > -6)
    step = torch.exp2(exponent - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def _exact_fill(x, cache, scale, case, counts):
    cache, scale, start = cache.double(), scale.double(), case["start"]
    for b, count in enumerate(counts):
        if not count:
            continue
        for block in range(start // _BLOCK, (start + count - 1) // _BLOCK + 1):
            lo, hi = max(start, block * _BLOCK), min(start + count, (block + 1) * _BLOCK)
            fresh = x[b, :, lo - start:hi - start].double()
            largest = fresh.abs().flatten(1).amax(1)
            e = torch.ceil(torch.log2((largest / 448).clamp(min=2.0 ** _LOWEST)))
            e = torch.where(largest > 448 * torch.exp2(e), e + 1, e)
            now = torch.exp2(torch.where(largest <= 448 * torch.exp2(e - 1), e - 1, e).clamp(_LOWEST, _HIGHEST))
            if lo > block * _BLOCK:
                was = scale[b, :, block]
                now = torch.maximum(now, was)
                earlier = cache[b, :, block * _BLOCK:lo]
                cache[b, :, block * _BLOCK:lo] = _to_eight_bits(earlier * (was / now)[:, None, None])
            cache[b, :, lo:hi] = _to_eight_bits(fresh / now[:, None, None])
            scale[b, :, block] = now
    return cache, scale


def _exact_quantize(s):
    c = s["case"]
    if c["B"] * c["M"] > 200000:
        return None                       # a block at a time takes too long
    counts = _lengths(c)
    return (*_exact_fill(s["k"], s["k_cache"], s["k_scale"], c, counts),
            *_exact_fill(s["v"], s["v_cache"], s["v_scale"], c, counts))


def _exact_attend(s):
    c = s["case"]
    half, rest, out = _BUCKETS // 2, _BUCKETS - _BUCKETS // 2, []
    # the first distance of each logarithmic bucket, in whole numbers: d^rest * half^j >= half^rest * MAX^j
    first = [next(d for d in range(half, _MAX_DISTANCE + 1) if d ** rest * half ** j >= half ** rest * _MAX_DISTANCE ** j)
             for j in range(1, rest)]
    for b, n in enumerate(_lengths(c)):
        blocks = torch.arange(n, device="cuda") // _BLOCK
        k = s["k"][b, :, :n].double() * s["k_scale"][b].double()[:, blocks, None]
        v = s["v"][b, :, :n].double() * s["v_scale"][b].double()[:, blocks, None]
        w = torch.einsum("hmd,hnd->hmn", s["q"][b].double(), k)
        if c["causal"]:
            delta = torch.arange(n)[None, :] - (n - c["M"] + torch.arange(c["M"]))[:, None]
            distance = (-delta).clamp(min=0)
            bucket = torch.where(distance < half, distance, half + sum((distance >= d).long() for d in first))
            w = w + s["table"].double()[bucket.to(w.device)].permute(2, 0, 1)
            w = w.masked_fill((delta > 0).to(w.device), _NONE)
        out.append(torch.softmax(w, -1) @ v)
    return torch.stack(out)


_EXACT = {"step": _exact_step, "sequences": _exact_sequences, "reorder": _exact_reorder, "quantize": _exact_quantize,
          "attend": _exact_attend}
