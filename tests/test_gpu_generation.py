"""The generation operators against their plain float64 forms, at the sizes and masks where they can go wrong."""
import math

import pytest
import torch

from tests import generation_plain as plain

pytestmark = pytest.mark.gpu
NONE = float("-inf")
FP8 = torch.float8_e4m3fn


# ---------------------------------------------------------------- the step

def _search(B, K, seed, pos, first=False, ended=0.3):
    g = torch.Generator().manual_seed(seed)
    scores = -torch.rand((B, K), generator=g) * 4 - pos
    if first:
        scores[:, 1:] = NONE
        scores[:, 0] = 0.0
    pool = torch.where(torch.rand((B, K), generator=g) < ended, -torch.rand((B, K), generator=g) * 3 - 0.5, NONE)
    return dict(scores=scores, pool=pool.sort(-1, descending=True)[0].contiguous(),
                steps=torch.randint(0, pos + 1, (B, K), generator=g).int(),
                beams=torch.randint(0, K, (B, K), generator=g).int(), done=torch.zeros(B, dtype=torch.bool), pos=pos)


def _logits(B, K, V, dtype, seed, std=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((B * K, V), generator=g) * std
    x[:, 1] += torch.where(torch.rand(B * K, generator=g) < 0.3, 8.0, 0.0)
    return x.to(dtype)


def _run_step(logits, s, out=None, history=None, **kw):
    import turbot5_b200 as t5b
    dev = [t.cuda() for t in (s["scores"], s["pool"], s["steps"], s["beams"], s["done"])]
    pos = torch.tensor([s["pos"]], device="cuda")
    got = t5b.beam_search_step(logits, *dev, pos, out=dev_out(dev, out), history=history, **kw)
    torch.cuda.synchronize()
    return got


def dev_out(dev, out):
    if out != "inputs":
        return out
    B, K = dev[0].shape
    return [torch.empty((B, K), dtype=torch.long, device="cuda"), torch.empty((B, K), dtype=torch.int32, device="cuda"), *dev]


def _check_step(got, logits, s, eos=1, **kw):
    B, K = s["scores"].shape
    want = plain.step(logits.double().cpu().view(B * K, -1).tolist(), *(s[n].tolist() for n in ("scores", "pool", "steps", "beams", "done")),
                      s["pos"], eos=-1 if eos is None else eos, **kw)
    for i, name in ((0, "tokens"), (1, "parents"), (4, "steps"), (5, "beams"), (6, "done")):
        assert got[i].cpu().tolist() == want[i], name
    for i in (2, 3):
        w, g = torch.tensor(want[i], dtype=torch.float64), got[i].cpu().double()
        # float32 rounding of the result, and of the sum of exponentials: 2^-22 for each exponential, its argument's
        # rounding (up to 15 * ln 2 * 2^-23) and 64 float32 additions
        tol = w.abs().clamp(max=1e30) * 2.0 ** -23 + 6e-6
        fine = torch.isfinite(w)
        assert torch.equal(fine, torch.isfinite(g)) and torch.equal(w[~fine], g[~fine]), (w, g)
        assert ((w - g).abs()[fine] <= tol[fine]).all(), (w - g).abs()[fine].max()


SIZES = [(1, 1, 2), (3, 1, 5), (2, 2, 3), (2, 4, 37), (1, 16, 33), (2, 16, 100), (5, 3, 1001), (1, 4, 32128), (2, 5, 4099),
         (40, 4, 300), (80, 2, 777), (150, 10, 64), (310, 1, 130), (300, 16, 40)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,K,V", SIZES)
def test_step(B, K, V, dtype):
    logits, s = _logits(B, K, V, dtype, 1 + V), _search(B, K, V, 7)
    _check_step(_run_step(logits.cuda(), s), logits, s)


@pytest.mark.parametrize("length_penalty,early,eos", [(0.0, False, 1), (2.0, True, 1), (-0.7, False, 1), (1.3, True, 3), (1.0, False, None)])
def test_step_options(length_penalty, early, eos):
    logits, s = _logits(6, 4, 200, torch.float32, 5), _search(6, 4, 6, 11, ended=0.8)
    got = _run_step(logits.cuda(), s, length_penalty=length_penalty, early_stopping=early, eos_token_id=eos)
    _check_step(got, logits, s, eos=eos, length_penalty=length_penalty, early=early)


@pytest.mark.parametrize("K", [1, 4, 8, 16])
def test_first_step_has_one_running_beam(K):
    logits, s = _logits(3, K, 500, torch.bfloat16, 8), _search(3, K, 9, 0, first=True, ended=0.0)
    _check_step(_run_step(logits.cuda(), s), logits, s)


def _special(kind, B, K, V, dtype):
    x = _logits(B, K, V, dtype, 21)
    g = torch.Generator().manual_seed(3)
    if kind == "equal":
        x.fill_(0.5)
    elif kind == "zeros of both signs":
        x = torch.where(torch.rand(x.shape, generator=g) < 0.5, 0.0, -0.0).to(dtype)
    elif kind == "few left":
        x[:, 5:] = NONE
    elif kind == "lowest":
        x[:, 3:] = torch.finfo(dtype).min
    elif kind == "all lowest":
        x.fill_(torch.finfo(dtype).min)
    elif kind == "empty rows":
        x[::2] = NONE
    elif kind == "nothing":
        x.fill_(NONE)
    elif kind == "nan":
        x[torch.rand(x.shape, generator=g) < 0.2] = float("nan")
        x[1] = float("nan")
    elif kind == "inf":
        x[0, 7] = math.inf
        x[1, :4] = math.inf
        x[2, 2] = math.nan
        x[2, 3] = math.inf
    elif kind == "same beams":
        x[:] = x[:1]
    elif kind == "one token":
        x.fill_(-30000.0)
        x[:, V - 1] = 30000.0
    return x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K,V", [(2, 4, 100), (1, 16, 70), (3, 3, 2049), (160, 4, 30)])
@pytest.mark.parametrize("kind", ["equal", "zeros of both signs", "few left", "lowest", "all lowest", "empty rows", "nothing", "nan", "inf",
                                  "same beams", "one token"])
def test_step_masks_and_ties(kind, B, K, V, dtype):
    logits, s = _special(kind, B, K, V, dtype), _search(B, K, 4, 3)
    if kind == "same beams":
        s["scores"].fill_(-2.5)
    _check_step(_run_step(logits.cuda(), s), logits, s)


def test_step_scores_that_are_not_finite():
    logits, s = _logits(3, 4, 90, torch.float32, 2), _search(3, 4, 3, 3)
    s["scores"][0, 1] = float("nan")
    s["scores"][1] = NONE
    s["scores"][2, :3] = NONE
    s["pool"][0, 1] = float("nan")
    _check_step(_run_step(logits.cuda(), s), logits, s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset,pad,V", [(0, 0, 513), (1, 3, 509), (3, 0, 1027), (5, 11, 31), (7, 1, 3)])
def test_step_rows_anywhere(offset, pad, V, dtype):
    """Rows that start on any element, with gaps (NaN) between them."""
    B, K = 3, 4
    logits, s = _logits(B, K, V, dtype, 31), _search(B, K, 14, 3)
    buf = torch.full((offset + B * K * (V + pad) + 8,), float("nan"), dtype=dtype, device="cuda")
    view = buf[offset:offset + B * K * (V + pad)].view(B * K, V + pad)[:, :V]
    view.copy_(logits)
    _check_step(_run_step(view, s), logits, s)
    _check_step(_run_step(view.unsqueeze(1), s), logits, s)                    # (rows, 1, vocab), as a decoder gives them
    turned = logits.cuda().t().contiguous().t()                                # last dim not contiguous
    _check_step(_run_step(turned, s), logits, s)


def test_step_done_sentences_stay():
    B, K = 4, 3
    logits, s = _logits(B, K, 50, torch.float32, 3), _search(B, K, 3, 6)
    s["done"][1] = s["done"][3] = True
    logits[3 * K:] = float("nan")
    got = _run_step(logits.cuda(), s, pad_token_id=9)
    _check_step(got, logits, s, pad=9)


def test_step_in_place_and_history():
    B, K, T = 5, 4, 6
    logits, s = _logits(B, K, 333, torch.bfloat16, 13), _search(B, K, 12, 4)
    s["done"][2] = True
    history = [torch.full((T, B, K), -7, dtype=torch.int32, device="cuda") for _ in range(2)]
    got = _run_step(logits.cuda(), s, out="inputs", history=history)
    _check_step(got, logits, s)
    assert torch.equal(history[0][4], got[0].int()) and torch.equal(history[1][4], got[1])
    for h in history:
        assert (h[:4] == -7).all() and (h[5:] == -7).all()
    s["pos"] = T                                       # behind the history: nothing is written to it
    before = [h.clone() for h in history]
    _check_step(_run_step(logits.cuda(), s, history=history), logits, s)
    assert all(torch.equal(a, b) for a, b in zip(before, history))


def test_step_twice_gives_the_same_bits():
    logits, s = _logits(16, 8, 5000, torch.bfloat16, 13).cuda(), _search(16, 8, 12, 4)
    a, b = _run_step(logits, s), _run_step(logits, s)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---------------------------------------------------------------- sentences

@pytest.mark.parametrize("T,B,K,R", [(1, 1, 1, 1), (1, 3, 4, 4), (2, 2, 16, 16), (31, 2, 3, 2), (32, 1, 4, 1), (33, 5, 5, 5), (512, 2, 8, 8),
                                     (1024, 1, 2, 2), (1025, 2, 16, 3), (2500, 1, 4, 4)])
def test_sequences(T, B, K, R):
    import turbot5_b200 as t5b
    g = torch.Generator().manual_seed(T)
    tokens = torch.randint(2, 30000, (T, B, K), generator=g).int()
    parents = torch.randint(0, K, (T, B, K), generator=g).int()
    s = _search(B, K, T, T - 1, ended=0.5)
    s["done"][::2] = True
    want, values = plain.sequences(tokens.tolist(), parents.tolist(), *(s[n].tolist() for n in ("scores", "pool", "steps", "beams", "done")), R,
                                   pad=77, length_penalty=0.8)
    got, scores = t5b.beam_search_sequences(tokens.cuda(), parents.cuda(), *(s[n].cuda() for n in ("scores", "pool", "steps", "beams", "done")),
                                            num_return_sequences=R, pad_token_id=77, length_penalty=0.8)
    assert got.cpu().tolist() == want
    values = torch.tensor(values, dtype=torch.float64)
    fine = torch.isfinite(values)
    assert torch.equal(fine, torch.isfinite(scores.cpu()))
    # one float32 rounding of a float64 quotient
    assert ((scores.cpu().double() - values).abs()[fine] <= values.abs()[fine] * 2.0 ** -23).all()


def test_sequences_of_bad_histories_stay_in_bounds():
    import turbot5_b200 as t5b
    B, K, T = 2, 4, 40
    tokens = torch.ones((T, B, K), dtype=torch.int32, device="cuda")
    parents = torch.full((T, B, K), 1 << 30, dtype=torch.int32, device="cuda")
    parents[::2] = -5
    s = _search(B, K, 1, 3, ended=1.0)
    s["steps"].fill_(1 << 20)
    s["beams"].fill_(-9)
    got, _ = t5b.beam_search_sequences(tokens, parents, *(s[n].cuda() for n in ("scores", "pool", "steps", "beams", "done")))
    assert got.shape == (B, 1, T) and (got == 1).all()


def test_whole_search_matches_plain():
    """Steps, history and sentences together on a small Markov model, against the plain form of all of them."""
    import turbot5_b200 as t5b
    B, K, V, T = 3, 4, 40, 12
    g = torch.Generator().manual_seed(11)
    chain = torch.randn((B, V, V), generator=g) * 3
    chain[:, :, 1] += 1.5
    s = _search(B, K, 1, 0, first=True, ended=0.0)
    state = [s[n].cuda() for n in ("scores", "pool", "steps", "beams", "done")]
    history = [torch.zeros((T, B, K), dtype=torch.int32, device="cuda") for _ in range(2)]
    pos, cur = torch.zeros(1, dtype=torch.long, device="cuda"), torch.zeros((B, K), dtype=torch.long, device="cuda")
    parents = torch.empty((B, K), dtype=torch.int32, device="cuda")
    device_chain = chain.cuda()
    plain_state = [s[n].tolist() for n in ("scores", "pool", "steps", "beams", "done")]
    plain_cur, plain_history = [[0] * K for _ in range(B)], ([], [])
    for t in range(T):
        rows = torch.stack([device_chain[b, cur[b]] for b in range(B)]).view(B * K, V)
        t5b.beam_search_step(rows, *state, pos, out=[cur, parents, *state], history=history)
        pos += 1
        flat = [chain[b, w].tolist() for b in range(B) for w in plain_cur[b]]
        out = plain.step(flat, *plain_state, t)
        plain_cur, plain_state = out[0], [[[torch.tensor(x).item() for x in r] for r in out[2]], *out[3:]]
        plain_history[0].append(out[0])
        plain_history[1].append(out[1])
        assert cur.tolist() == out[0] and parents.tolist() == out[1] and state[4].tolist() == out[6], t
    want, values = plain.sequences(*plain_history, *plain_state, K)
    got, scores = t5b.beam_search_sequences(*history, *state, num_return_sequences=K)
    assert got.tolist() == want
    assert torch.allclose(scores.cpu().double(), torch.tensor(values, dtype=torch.float64), atol=1e-4)


# ---------------------------------------------------------------- reordering

def _parents(B, K, seed, kind="any"):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, K, (B, K), generator=g).int()
    if kind == "same":
        p[:] = torch.arange(K)
    elif kind == "turned":
        p[:] = torch.arange(K).roll(1)
    elif kind == "one":
        p.fill_(K - 1)
    elif kind == "outside":
        p[:, 0], p[:, -1] = -1, K
    return p


def _reordered(t, parents, used):
    """t (rows, heads, tokens, ...) with the first used[b] tokens of every sentence's beams following their parents."""
    B, K = parents.shape
    out = t.clone()
    for b in range(B):
        for j in range(K):
            p = int(parents[b, j])
            if 0 <= p < K:
                out[b * K + j, :, :used[b]] = t[b * K + p, :, :used[b]]
    return out


@pytest.mark.parametrize("kind", ["any", "same", "turned", "one", "outside"])
@pytest.mark.parametrize("B,K,H,cap,D,dtype", [(2, 4, 3, 10, 64, torch.bfloat16), (3, 5, 2, 7, 3, torch.float16), (1, 16, 2, 65, 16, torch.float32),
                                               (2, 2, 1, 1, 1, torch.uint8), (4, 8, 2, 130, 6, torch.bfloat16), (1, 1, 2, 4, 8, torch.float32)])
def test_reorder(B, K, H, cap, D, dtype, kind):
    import turbot5_b200 as t5b
    g = torch.Generator().manual_seed(cap)
    caches = [torch.randint(0, 200, (2, B * K, H, cap, D), generator=g).to(dtype) for _ in range(3)]
    parents = _parents(B, K, 5, kind)
    lens = torch.randint(0, cap + 1, (B * K,), generator=g).int()
    used = lens.view(B, K).amax(1).tolist()
    for seqlens, use in ((lens, used), (None, [cap] * B)):
        got = [c.cuda() for c in caches]
        t5b.reorder_beam_cache(got, parents.cuda(), seqlens=None if seqlens is None else seqlens.cuda())
        want = [torch.stack([_reordered(c[i], parents, use) for i in range(2)]) for c in caches]
        for a, w in zip(got, want):
            assert torch.equal(a.cpu(), w)
    got = caches[0][0].cuda()                          # keys alone: one dimension less
    t5b.reorder_beam_cache([got], parents.cuda())
    assert torch.equal(got.cpu(), want[0][0])


def test_reorder_views_many_tensors_and_scales():
    import turbot5_b200 as t5b
    B, K, H, cap, D = 2, 3, 2, 130, 16
    g = torch.Generator().manual_seed(3)
    parents = _parents(B, K, 7)
    lens = torch.full((B * K,), 70, dtype=torch.int32)
    # heads in front of the rows, 70 tensors: two launches
    base = torch.randint(0, 255, (70, 2, H, B * K, cap, D), generator=g).to(torch.uint8).cuda()
    scale = torch.rand((70, 2, H, B * K, 3), generator=g).cuda()
    caches, scales = [t.transpose(1, 2) for t in base.clone()], [t.transpose(1, 2) for t in scale.clone()]
    t5b.reorder_beam_cache([c.view(FP8) for c in caches], parents.cuda(), seqlens=lens.cuda(), scales=scales)
    rows = (parents.long() + torch.arange(B)[:, None] * K).flatten().cuda()
    for c, s, c0, s0 in zip(caches, scales, base, scale):
        c0, s0 = c0.transpose(1, 2), s0.transpose(1, 2)
        assert torch.equal(c[..., :70, :], c0[:, rows][..., :70, :]) and torch.equal(c[..., 70:, :], c0[..., 70:, :])
        assert torch.equal(s[..., :2], s0[:, rows][..., :2]) and torch.equal(s[..., 2:], s0[..., 2:])


def test_reorder_single_tokens_and_numbers():
    """Dimensions of size one may have any stride."""
    import turbot5_b200 as t5b
    parents = torch.tensor([[1, 0, 0]], dtype=torch.int32, device="cuda")
    for shape, order in (((3, 2, 1, 8), (0, 1, 3, 2)), ((3, 2, 5, 1), (0, 1, 2, 3))):
        base = torch.arange(48, device="cuda", dtype=torch.float32)[:math.prod(shape)]
        cache = base.view(*(shape[i] for i in order)).permute(*(order.index(i) for i in range(4)))
        want = cache[[1, 0, 0]].clone()
        t5b.reorder_beam_cache([cache], parents)
        assert torch.equal(cache, want)


def test_reorder_lengths_outside_the_cache():
    import turbot5_b200 as t5b
    cache = torch.arange(2 * 4 * 8, device="cuda", dtype=torch.float32).view(2, 1, 4, 8).contiguous()
    parents = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    for n in (-3, 0):
        got = cache.clone()
        t5b.reorder_beam_cache([got], parents, seqlens=torch.full((2,), n, dtype=torch.int32, device="cuda"))
        assert torch.equal(got, cache)
    got = cache.clone()
    t5b.reorder_beam_cache([got], parents, seqlens=torch.full((2,), 1 << 30, dtype=torch.int32, device="cuda"))
    assert torch.equal(got, cache.flip(0))


# ---------------------------------------------------------------- 8-bit caches

def _cache(B, H, cap, D, seed):
    g = torch.Generator().manual_seed(seed)
    values = (torch.randn((B, H, cap, D), generator=g) * 60).clamp(-448, 448).to(FP8)
    scale = torch.exp2(torch.randint(-9, -3, (B, H, cap // 64), generator=g).float())
    return values, scale


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("M,start,cap", [(1, 0, 64), (1, 63, 64), (1, 70, 128), (2, 63, 128), (64, 0, 64), (65, 1, 128), (130, 60, 256), (3, 125, 128)])
def test_quantize(M, start, cap, D, dtype):
    import turbot5_b200 as t5b
    B, H = 3, 2
    g = torch.Generator().manual_seed(M + start)
    kv = torch.randn((B, M, 2, H, D), generator=g).to(dtype)
    kv[0] *= 30                                        # larger than what the block holds: its tokens move
    kv[1, :, :, 1] = 0
    k, v = (t.transpose(1, 2) for t in kv.cuda().unbind(2))
    counts = [M, max(M - 1, 0), M // 2]
    for seqlens in (None, torch.tensor(counts, dtype=torch.int32)):
        for place in (start, torch.tensor([start], device="cuda")):
            (kc, ks), (vc, vs) = _cache(B, H, cap, D, 1), _cache(B, H, cap, D, 2)
            dev = [t.cuda() for t in (kc, ks, vc, vs)]
            t5b.quantize_into_cache(k, v, *dev, place, seqlens=None if seqlens is None else seqlens.cuda())
            for x, c, s, gc, gs in ((k, kc, ks, *dev[:2]), (v, vc, vs, *dev[2:])):
                wc, ws = plain.fill(x.double().cpu(), c.double(), s.double(), start, [M] * B if seqlens is None else counts)
                assert torch.equal(gs.cpu().double(), ws)
                assert torch.equal(gc.cpu().double(), wc)


def test_quantize_extreme_values():
    import turbot5_b200 as t5b
    D, cap = 16, 64
    rows = torch.zeros((8, 1, 2, D))
    rows[0, 0, 0, 0] = 448.0                           # exactly the largest number: scale 1
    rows[1, 0, 0, 0] = 448.0 * (1 + 2.0 ** -23)        # the next float: scale 2
    rows[2, 0, 0, 0] = 3.0e38
    rows[3, 0, 0, 0] = 1e-42                           # below the smallest scale
    rows[4, 0, 0, 0], rows[4, 0, 0, 1] = math.inf, 5.0
    rows[5, 0, 0, 0], rows[5, 0, 0, 1] = math.nan, 5.0
    rows[6, 0, 0, 0], rows[6, 0, 0, 1] = -math.inf, -0.0
    rows[7, 0, 0, 0], rows[7, 0, 0, 1] = 1.0, 2.0 ** -30
    kc, vc = (torch.zeros((8, 1, cap, D), device="cuda").to(FP8) for _ in range(2))
    ks, vs = (torch.ones((8, 1, 1), device="cuda") for _ in range(2))
    t5b.quantize_into_cache(rows.cuda(), rows.cuda(), kc, ks, vc, vs)
    wc, ws = plain.fill(rows.double(), torch.zeros((8, 1, cap, D), dtype=torch.float64), torch.ones((8, 1, 1), dtype=torch.float64), 0, [2] * 8)
    for c, s in ((kc, ks), (vc, vs)):
        assert torch.equal(s.cpu().double(), ws)
        assert torch.equal(torch.nan_to_num(c.cpu().double(), nan=1e9), torch.nan_to_num(wc, nan=1e9))
    assert ks[0].item() == 1.0 and ks[1].item() == 2.0 and ks[3].item() == 2.0 ** -100
    assert torch.equal(kc[4, 0, 0, :1].float().cpu(), torch.tensor([448.0])) and torch.isnan(kc[5, 0, 0, 0].float())


def test_quantize_past_the_capacity_and_misaligned():
    import turbot5_b200 as t5b
    B, H, D, cap = 2, 2, 64, 64
    g = torch.Generator().manual_seed(1)
    for dtype in (torch.bfloat16, torch.float32):
        raw = torch.randn((B * H * 5 * (D + 1) + 1,), generator=g).to(dtype).cuda()
        x = raw[1:].view(B, H, 5, D + 1)[..., :D]      # rows on any element
        for start in (62, 64, 1000, -1):
            (c, s), (c2, s2) = _cache(B, H, cap, D, 3), _cache(B, H, cap, D, 4)
            dev = [t.cuda() for t in (c, s, c2, s2)]
            t5b.quantize_into_cache(x, x, *dev, torch.tensor([start], device="cuda"))
            wc, ws = plain.fill(x.double().cpu(), c.double(), s.double(), start, [5] * B) if 0 <= start < cap else (c.double(), s.double())
            assert torch.equal(dev[0].cpu().double(), wc) and torch.equal(dev[1].cpu().double(), ws)


# ---------------------------------------------------------------- attention over them

def _check_attention(q, kv, table, lengths, causal, scale, nb=32, md=128, offset=None, poison=True, **kw):
    import turbot5_b200 as t5b
    (k, ks), (v, vs) = kv
    B, H, M, D = q.shape
    kd, vd = (c.double() * s.double().repeat_interleave(64, -1)[..., None] for c, s in kv)
    want, mass, size = plain.attend(q, kd, vd, table, lengths, causal, scale, nb, md, offset)
    k, v, ks, vs = k.clone(), v.clone(), ks.clone(), vs.clone()
    if poison:                                         # what lies behind the keys in use is never data
        for b, n in enumerate(lengths):
            k.view(torch.uint8)[b, :, n:] = 0x7f
            v.view(torch.uint8)[b, :, n:] = 0xff
            ks[b, :, (n + 63) // 64:] = float("nan")
            vs[b, :, (n + 63) // 64:] = float("nan")
    got = t5b.flash_decoding_quantized_with_fusing_bias(
        q.cuda(), k.cuda(), ks.cuda(), v.cuda(), vs.cuda(), None if table is None else table.cuda(), causal=causal, sm_scale=scale,
        NUM_BUCKETS=nb, MAX_DISTANCE=md, seqlens_k=torch.tensor(lengths, dtype=torch.int32).cuda(), q_pos_offset=offset, **kw)
    got = got.double().cpu()
    # float32 sums of D products and a few roundings of the score (base 2), twice in weight / sum of weights; 2^-20 for the
    # exponential, the weight's two halves and the float32 sums; the result's own rounding
    rel = 2 * (D + 8) * 2.0 ** -24 * 1.5 * (size + 1) + 2.0 ** -20 + max(lengths) * 2.0 ** -24
    tol = want.abs() * torch.finfo(q.dtype).eps / 2 * (1 + 2.0 ** -8) + mass * rel + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("M,lengths,causal", [
    (1, [0, 1, 63], False), (1, [64, 65, 200], True), (2, [2, 64, 129], True), (3, [0, 5, 130], False), (4, [4, 66, 300], True),
    (5, [5, 64, 257], True), (8, [8, 9, 190], True), (8, [1, 70, 512], False), (9, [9, 100, 64], True), (16, [16, 65, 333], True),
    (19, [19, 500, 64], False)])
def test_attention(M, lengths, causal, D, dtype):
    B, H = len(lengths), 2
    g = torch.Generator().manual_seed(M * 100 + D)
    q = (torch.randn((B, M, H, D), generator=g) * 2 * D ** -0.5).to(dtype).transpose(1, 2)
    table = torch.randn((32, H), generator=g).to(dtype)
    kv = _cache(B, H, 512, D, 5), _cache(B, H, 512, D, 6)
    _check_attention(q, kv, table, lengths, causal, 1.0)
    _check_attention(q.contiguous(), kv, None, lengths, causal, 0.3)


@pytest.mark.parametrize("nb,md,causal", [(8, 20, True), (64, 300, False), (32, 128, False), (16, 2048, True)])
@pytest.mark.parametrize("offset", [None, 0, 37, 400])
def test_attention_bias_and_positions(nb, md, causal, offset):
    g = torch.Generator().manual_seed(nb)
    M, H, lengths = 3, 3, [64, 400, 450]
    q = (torch.randn((3, H, M, 64), generator=g) * 0.2).to(torch.float16)
    table = torch.randn((nb, H), generator=g) * 2      # float32 table
    _check_attention(q, (_cache(3, H, 512, 64, 5), _cache(3, H, 512, 64, 6)), table, lengths, causal, 1.0, nb, md, offset)


def test_attention_long_cache_and_splits():
    """Caches that several blocks of a cluster share; every block's part is merged."""
    g = torch.Generator().manual_seed(2)
    for H, n, M in ((1, 4096, 1), (2, 3001, 4), (1, 2500, 7)):
        q = (torch.randn((1, H, M, 64), generator=g) * 0.5).to(torch.bfloat16)
        _check_attention(q, (_cache(1, H, 4096, 64, 7), _cache(1, H, 4096, 64, 8)), None, [n], False, 1.0)


def test_attention_scales_of_every_size():
    """Blocks whose scales are 2^60 apart, queries far from one."""
    g = torch.Generator().manual_seed(2)
    (k, ks), (v, vs) = _cache(2, 2, 256, 64, 7), _cache(2, 2, 256, 64, 8)
    vs = torch.exp2(torch.randint(-60, 20, vs.shape, generator=g).float())
    ks[:, 0] = torch.exp2(torch.randint(-60, -8, ks[:, 0].shape, generator=g).float())
    for size in (1e-3, 1e-30, 1.0):
        q = (torch.randn((2, 2, 2, 64), generator=g) * size).to(torch.bfloat16)
        _check_attention(q, ((k, ks), (v, vs)), None, [256, 200], False, 1.0)
    q = torch.zeros((2, 2, 1, 64), dtype=torch.bfloat16)
    q[:, :, :, 5] = 2.0 ** 100
    _check_attention(q, ((k, ks * 2.0 ** -103), (v, vs)), None, [256, 200], False, 1.0)


def test_attention_nan_of_a_visible_key_shows():
    import turbot5_b200 as t5b
    (k, ks), (v, vs) = _cache(1, 2, 128, 64, 7), _cache(1, 2, 128, 64, 8)
    k.view(torch.uint8)[0, 0, 70, 3] = 0x7f
    q = torch.ones((1, 2, 1, 64), dtype=torch.float16)
    for n, bad in ((70, False), (71, True)):
        out = t5b.flash_decoding_quantized_with_fusing_bias(q.cuda(), k.cuda(), ks.cuda(), v.cuda(), vs.cuda(), None, kv_len=n)
        assert bool(torch.isnan(out[0, 0]).any()) == bad and not torch.isnan(out[0, 1]).any()


def test_attention_offsets_beyond_32_bits():
    """The last rows of a cache of more than 2^32 bytes."""
    import turbot5_b200 as t5b
    B, H, cap, D = 36, 8, 131072, 128
    k = torch.empty((B, H, cap, D), dtype=torch.uint8, device="cuda")
    assert k.numel() > 1 << 32
    scale = torch.ones((B, H, cap // 64), device="cuda")
    (kv, _) = _cache(1, H, 128, D, 9)
    for b in (0, B - 1):
        k[b, :, :128] = kv[0].view(torch.uint8).cuda()
    q = (torch.randn((B, H, 1, D), generator=torch.Generator().manual_seed(1)) * 0.01).to(torch.bfloat16)
    q[B - 1] = q[0]
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    lens[0] = lens[B - 1] = 100
    out = t5b.flash_decoding_quantized_with_fusing_bias(q.cuda(), k.view(FP8), scale, k.view(FP8), scale, None, seqlens_k=lens)
    assert torch.equal(out[0], out[B - 1]) and out[0].abs().sum() > 0 and (out[1:B - 1] == 0).all()
    x = torch.randn((B, H, 1, D), device="cuda", dtype=torch.bfloat16)
    k2, scale2 = k[:, :, :, :64].contiguous().view(FP8), scale.clone()          # (k is D = 128: a second cache of half its size)
    t5b.quantize_into_cache(x[..., :64].contiguous(), x[..., 64:].contiguous(), k2, scale, k.view(FP8)[..., :64].contiguous(), scale2, cap - 1)
    back = k2[B - 1, :, cap - 1].float() * scale[B - 1, :, -1, None]
    # e4m3: half a step is 2^-4 of the value, or of the smallest normal number, 2^-6 of a scale that holds older tokens
    assert ((back - x[B - 1, :, 0, :64].float()).abs() <= x[B - 1, :, 0, :64].float().abs() * 2.0 ** -4 + scale[B - 1, :, -1, None] * 2.0 ** -10).all()


# ---------------------------------------------------------------- together

def _pipeline(state, k_new, logits, q):
    """One generation step of one layer: append, attend, choose, reorder, advance."""
    import turbot5_b200 as t5b
    c = state
    t5b.quantize_into_cache(k_new, k_new, c["kv"][0], c["scale"][0], c["kv"][1], c["scale"][1], c["pos"])
    out = t5b.flash_decoding_quantized_with_fusing_bias(q, c["kv"][0], c["scale"][0], c["kv"][1], c["scale"][1], c["table"], causal=True,
                                                        sm_scale=1.0, seqlens_k=c["seqlens"])
    t5b.beam_search_step(logits, *c["search"], c["pos"], out=[c["tokens"], c["parents"], *c["search"]], history=c["history"])
    t5b.reorder_beam_cache([c["kv"]], c["parents"], seqlens=c["seqlens"], scales=[c["scale"]])
    c["pos"] += 1
    c["seqlens"] += 1
    return out


def _new_state(B, K, H, D, cap, T):
    s = _search(B, K, 1, 0, first=True, ended=0.0)
    return dict(kv=torch.zeros((2, B * K, H, cap, D), device="cuda").to(FP8), scale=torch.ones((2, B * K, H, cap // 64), device="cuda"),
                pos=torch.zeros(1, dtype=torch.long, device="cuda"), seqlens=torch.ones(B * K, dtype=torch.int32, device="cuda"),
                table=torch.randn((32, H), generator=torch.Generator().manual_seed(5)).cuda(),
                search=[s[n].cuda() for n in ("scores", "pool", "steps", "beams", "done")],
                tokens=torch.zeros((B, K), dtype=torch.long, device="cuda"), parents=torch.zeros((B, K), dtype=torch.int32, device="cuda"),
                history=[torch.zeros((T, B, K), dtype=torch.int32, device="cuda") for _ in range(2)])


def _steps(B, K, H, D, V, T):
    g = torch.Generator().manual_seed(9)
    for _ in range(T):
        yield (torch.randn((B * K, H, 1, D), generator=g).to(torch.bfloat16).cuda(),
               (torch.randn((B * K, V), generator=g) * 3).to(torch.bfloat16).cuda(),
               (torch.randn((B * K, H, 1, D), generator=g) * 0.2).to(torch.bfloat16).cuda())


def test_the_operators_together_captured_and_on_other_streams():
    B, K, H, D, V, T, cap = 2, 4, 3, 64, 500, 70, 128
    inputs = list(_steps(B, K, H, D, V, T))
    eager = _new_state(B, K, H, D, cap, T)
    outs = [_pipeline(eager, *x) for x in inputs]
    # the same in a graph that is replayed: positions and lengths live on the device
    graphed = _new_state(B, K, H, D, cap, T)
    static = [t.clone() for t in inputs[0]]
    warm = _new_state(B, K, H, D, cap, T)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                      # a stream of its own, concurrently with the eager one's last steps
        _pipeline(warm, *static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _pipeline(graphed, *static)
    for x, want in zip(inputs, outs):
        for a, b in zip(static, x):
            a.copy_(b)
        graph.replay()
        assert torch.equal(out, want)
    for name in ("kv", "scale", "pos", "seqlens", "tokens", "parents"):
        a, b = eager[name], graphed[name]
        assert torch.equal(a.view(torch.uint8) if a.dtype == FP8 else a, b.view(torch.uint8) if b.dtype == FP8 else b), name
    assert all(torch.equal(a, b) for a, b in zip(eager["search"] + eager["history"], graphed["search"] + graphed["history"]))


def test_two_calls_at_once_do_not_touch_each_other():
    """No operator keeps state or scratch: calls on two streams give what they give alone."""
    import turbot5_b200 as t5b
    g = torch.Generator().manual_seed(4)
    cases = []
    for i in range(2):
        kv = _cache(2, 4, 4096, 64, 20 + i), _cache(2, 4, 4096, 64, 30 + i)
        q = torch.randn((2, 4, 3, 64), generator=g).to(torch.float16).cuda()
        cases.append(([t.cuda() for t in (*kv[0], *kv[1])], q, _logits(4, 4, 30000, torch.bfloat16, i).cuda(), _search(4, 4, i, 5)))
    def call(c):
        (k, ks, v, vs), q, logits, s = c
        dev = [t.cuda() for t in (s["scores"], s["pool"], s["steps"], s["beams"], s["done"])]
        pos = torch.tensor([5], device="cuda")
        torch.cuda.current_stream().synchronize()
        return [r for _ in range(20) for r in (t5b.flash_decoding_quantized_with_fusing_bias(q, k, ks, v, vs, None),
                                               *t5b.beam_search_step(logits, *dev, pos))]
    alone = [call(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    both = []
    for c, st in zip(cases, streams):
        with torch.cuda.stream(st):
            both.append(call(c))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x, y in zip(alone, both) for a, b in zip(x, y))


# ---------------------------------------------------------------- refusals

def test_refusals_on_the_device():
    import turbot5_b200 as t5b
    s = _search(2, 4, 1, 0)
    dev = [s[n].cuda() for n in ("scores", "pool", "steps", "beams", "done")]
    pos, logits = torch.zeros(1, dtype=torch.long, device="cuda"), torch.zeros((8, 50), device="cuda")
    step = lambda *a, **k: t5b.beam_search_step(*a, **k)
    for bad, error in (((logits[:7], *dev, pos), ValueError), ((logits[:, :1], *dev, pos), ValueError), ((logits.double(), *dev, pos), TypeError),
                       ((logits, dev[0].double(), *dev[1:], pos), TypeError), ((logits, *dev[:4], dev[4].int(), pos), TypeError),
                       ((logits, *dev, pos.int()), TypeError), ((logits, *dev, pos.cpu()), RuntimeError),
                       ((logits, dev[0].t().contiguous().t(), *dev[1:], pos), ValueError),
                       ((torch.zeros((34, 50), device="cuda"), torch.zeros((2, 17), device="cuda"), *dev[1:], pos), ValueError)):
        with pytest.raises(error):
            step(*bad)
    with pytest.raises(ValueError):
        step(logits, *dev, pos, length_penalty=float("nan"))
    with pytest.raises(ValueError):
        step(logits, *dev, pos, out=dev)
    twice = [torch.empty((2, 4), dtype=torch.long, device="cuda"), dev[2], *dev]
    with pytest.raises(ValueError, match="same"):
        step(logits, *dev, pos, out=twice)
    with pytest.raises((TypeError, ValueError)):
        step(logits, *dev, pos, history=[torch.zeros((3, 2, 4), device="cuda")] * 2)
    hist = torch.zeros((3, 2, 4), dtype=torch.int32, device="cuda")
    for kw in (dict(num_return_sequences=0), dict(num_return_sequences=5), dict(length_penalty=float("inf"))):
        with pytest.raises(ValueError):
            t5b.beam_search_sequences(hist, hist, *dev, **kw)
    with pytest.raises(ValueError):
        t5b.beam_search_sequences(hist[:0], hist[:0], *dev)
    parents = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    cache = torch.zeros((2, 8, 3, 10, 16), device="cuda")
    for bad in ([cache, cache], [cache[:, :7]], [cache, cache[..., :8]], [cache[..., ::2]], [cache.transpose(-1, -2)],
                [cache[:1].expand(2, 8, 3, 10, 16)]):
        with pytest.raises(ValueError):
            t5b.reorder_beam_cache(bad, parents)
    with pytest.raises(TypeError):
        t5b.reorder_beam_cache([cache], parents.long())
    with pytest.raises(ValueError):
        t5b.reorder_beam_cache([cache], parents, scales=[torch.zeros((2, 8, 3, 2), device="cuda")])
    (k, ks), (v, vs) = ([t.cuda() for t in _cache(2, 3, 128, 64, i)] for i in (1, 2))
    x = torch.zeros((2, 3, 5, 64), device="cuda", dtype=torch.bfloat16)
    fill = lambda *a, **kw: t5b.quantize_into_cache(*a, **kw)
    for bad, error in (((x, x, k, ks, v, vs, 124), ValueError), ((x, x, k, ks, v, vs, -1), ValueError), ((x, x.float(), k, ks, v, vs), TypeError),
                       ((x[..., :48], x[..., :48], k, ks, v, vs), ValueError), ((x, x, k.view(torch.uint8), ks, v, vs), TypeError),
                       ((x, x, k, ks[..., :1], v, vs), ValueError), ((x, x, k[:, :, :100], ks, v, vs), ValueError),
                       ((x, x, k, ks, k, ks), ValueError), ((x, x, k[:1].expand(2, 3, 128, 64), ks, v, vs), ValueError),
                       ((x, x, k, ks, v, vs, torch.zeros(1, device="cuda")), TypeError)):
        with pytest.raises(error):
            fill(*bad)
    att = lambda q, *a, **kw: t5b.flash_decoding_quantized_with_fusing_bias(q, *a, **kw)
    q, table = x[:, :, :1], torch.zeros((32, 3), device="cuda")
    for bad, error in (((q.float(), k, ks, v, vs, None), TypeError), ((q[:, :2], k, ks, v, vs, None), ValueError),
                       ((q, k, ks, v[:, :, :64], vs[..., :1], None), ValueError), ((q, k, ks, v, vs, table[:, :2]), ValueError),
                       ((q, k, ks, v, vs, table[:20]), ValueError), ((q, k.float(), ks, v, vs, None), TypeError)):
        with pytest.raises(error):
            att(*bad)
    with pytest.raises(RuntimeError):
        att(q, k, ks, v, vs, None, q_pos_offset=0x7fffffff - 100)
    for kw in (dict(kv_len=129), dict(kv_len=-1), dict(seqlens_k=torch.zeros(3, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            att(q, k, ks, v, vs, None, **kw)
    with pytest.raises(RuntimeError):
        att(q, k, ks, v, vs, torch.zeros((3000, 3), device="cuda"), NUM_BUCKETS=1024)
    # empty problems are no errors
    assert att(q[:0], k[:0], ks[:0], v[:0], vs[:0], None).shape == (0, 3, 1, 64)
    assert att(x[:, :, :0], k, ks, v, vs, None).shape == (2, 3, 0, 64)
    assert (att(q, k, ks, v, vs, None, kv_len=0) == 0).all()
    fill(x[:, :, :0], x[:, :, :0], k, ks, v, vs, 128)
    t5b.reorder_beam_cache([], parents)
    t5b.beam_search_step(logits[:0], *(t[:0] for t in dev), pos)


def test_written_tensors_that_overlap_or_have_gradients_are_refused():
    """Tensors that a call writes overlap one another, or an input that they do not replace: no order of the threads is
    promised, so there is no right result."""
    import turbot5_b200 as t5b
    s = _search(2, 4, 1, 0)
    scores, pool, steps, beams, done = (s[n].cuda() for n in ("scores", "pool", "steps", "beams", "done"))
    pos, logits = torch.zeros(1, dtype=torch.long, device="cuda"), torch.zeros((8, 50), device="cuda")
    step = lambda out, history=None: t5b.beam_search_step(logits, scores, pool, steps, beams, done, pos, out=out, history=history)
    fresh = lambda: [torch.empty((2, 4), dtype=d, device="cuda") for d in (torch.long, torch.int32, torch.float32, torch.float32, torch.int32, torch.int32)] + [
        torch.empty(2, dtype=torch.bool, device="cuda")]
    shifted = torch.zeros(9, device="cuda")
    hist = torch.zeros((3, 2, 4), dtype=torch.int32, device="cuda")
    for change in ({2: pool, 3: scores}, {1: steps}, {2: shifted[:8].view(2, 4), 3: shifted[1:].view(2, 4)}, {3: logits.view(-1)[:8].view(2, 4)}):
        out = fresh()
        for i, t in change.items():
            out[i] = t
        with pytest.raises(ValueError, match="overlap"):
            step(out)
    out = fresh()
    with pytest.raises(ValueError, match="overlap"):
        step(out, [hist, hist])
    with pytest.raises(ValueError, match="overlap"):
        step([out[0], hist[1], *out[2:]], [hist, torch.zeros_like(hist)])
    out[2].requires_grad_()
    with pytest.raises(ValueError, match="gradients"):
        step(out)
    before = scores._version
    step([*out[:2], scores, pool, steps, beams, done])
    assert scores._version == before + 1

    parents = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    both = torch.zeros((9, 3, 10, 16), device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        t5b.reorder_beam_cache([both[:8], both[1:]], parents)
    between = torch.zeros((8, 2, 3, 10, 16), device="cuda")
    t5b.reorder_beam_cache([between[:, 0], between[:, 1]], parents)         # one between the other's rows
    with pytest.raises(ValueError, match="gradients"):
        t5b.reorder_beam_cache([both[:8].clone().requires_grad_()], parents)
    x = torch.zeros((2, 3, 5, 64), device="cuda", dtype=torch.bfloat16)
    cache, scale = torch.zeros((3, 3, 128, 64), device="cuda").to(FP8), torch.ones((2, 2, 3, 2), device="cuda")
    with pytest.raises(ValueError, match="own"):
        t5b.quantize_into_cache(x, x, cache[:2], scale[0], cache[1:], scale[1])
    with pytest.raises(ValueError, match="own"):
        t5b.quantize_into_cache(x, x, cache[:2], scale[0], cache[:2].clone(), scale.view(-1)[6:18].view(2, 3, 2))
    version = cache._version
    t5b.quantize_into_cache(x, x, cache[:2], scale[0], cache[:2].clone(), scale[1])
    assert cache._version == version + 1


def test_lengths_of_other_layouts():
    """Lengths as a column of a larger tensor, or (B, 1)."""
    import turbot5_b200 as t5b
    (k, ks), (v, vs) = ([t.cuda() for t in _cache(2, 3, 128, 64, i)] for i in (1, 2))
    x = torch.randn((2, 3, 5, 64), device="cuda").bfloat16()
    lens = torch.tensor([[2, 9], [5, 9]], dtype=torch.int32, device="cuda")
    want = t5b.flash_decoding_quantized_with_fusing_bias(x, k, ks, v, vs, None, seqlens_k=lens[:, 0].contiguous())
    assert torch.equal(want, t5b.flash_decoding_quantized_with_fusing_bias(x, k, ks, v, vs, None, seqlens_k=lens[:, :1]))
    a, b = [[t.clone() for t in (k, ks, v, vs)] for _ in range(2)]
    t5b.quantize_into_cache(x, x, *a, 64, seqlens=lens[:, 0].contiguous())
    t5b.quantize_into_cache(x, x, *b, 64, seqlens=lens[:, 0])
    assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a, b))


@pytest.mark.parametrize("value", [1 << 40, (1 << 63) - 1, -1, -(1 << 63)])
def test_quantize_starts_far_outside_the_cache(value):
    import turbot5_b200 as t5b
    (k, ks), (v, vs) = ([t.cuda() for t in _cache(2, 3, 128, 64, i)] for i in (1, 2))
    before = [t.clone() for t in (k, ks, v, vs)]
    for M in (1, 70):
        x = torch.ones((2, 3, M, 64), device="cuda", dtype=torch.bfloat16)
        t5b.quantize_into_cache(x, x, k, ks, v, vs, torch.tensor([value], device="cuda"))
    torch.cuda.synchronize()
    assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(before, (k, ks, v, vs)))


@pytest.mark.parametrize("D", [16, 128])
def test_attention_over_more_than_2_31_numbers_of_a_head(D):
    """The first and the last key of a head whose keys fill more than 2^31 bytes; all others are zero and far below."""
    import turbot5_b200 as t5b
    N = (1 << 31) // D + 100
    cap = -(-N // 64) * 64
    k, v = (torch.zeros((1, 1, cap, D), dtype=torch.uint8, device="cuda") for _ in range(2))
    scale = torch.ones((1, 1, cap // 64), device="cuda")
    q = torch.full((1, 1, 1, D), 4.0, dtype=torch.bfloat16, device="cuda")
    values = torch.randn((2, D), generator=torch.Generator().manual_seed(1)).cuda().to(FP8)
    for n, i in ((0, 0), (N - 1, 1)):
        k[0, 0, n] = torch.full((D,), 4.0, device="cuda").to(FP8).view(torch.uint8)
        v[0, 0, n] = values[i].view(torch.uint8)
    out = t5b.flash_decoding_quantized_with_fusing_bias(q, k.view(FP8), scale, v.view(FP8), scale, None, sm_scale=1.0, kv_len=N)
    # weights 1/2 each and exp(-256) for the others; one bf16 rounding, and float32 ones that are far smaller
    want = values.double().mean(0)
    assert ((out[0, 0, 0].double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.01 + 1e-30).all()
    k[0, 0, 0] = 0
    out = t5b.flash_decoding_quantized_with_fusing_bias(q, k.view(FP8), scale, v.view(FP8), scale, None, sm_scale=1.0, kv_len=N)
    assert torch.equal(out[0, 0, 0], values[1].to(torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,K,V", [(3, 4, 384), (2, 10, 384), (1, 16, 384), (40, 10, 126), (1, 1, 15), (2, 8, 65), (1, 4, 4097), (1, 4, 4300), (9, 5, 1000)])
def test_step_of_small_vocabularies(B, K, V, dtype):
    """Slices of a few vectors, whose elements the lanes share, with rows that start anywhere and masked and special numbers."""
    for offset, special in ((0, False), (3, True)):
        x = _logits(B, K, V, torch.float32, 41 + offset)
        if special:
            x[0, ::3] = NONE
            x[-1, 1::5] = float("nan")
        x = x.to(dtype)
        flat = torch.zeros(offset + B * K * (V + offset), dtype=dtype)
        rows = flat[offset:].view(B * K, V + offset)[:, :V] if offset else x
        if offset:
            rows.copy_(x)
            flat = flat.cuda()
            rows = flat[offset:].view(B * K, V + offset)[:, :V]
        s = _search(B, K, 42, 3)
        _check_step(_run_step(rows if offset else rows.cuda(), s), x, s)


def test_step_of_many_short_launches_gives_the_same_bits():
    """Launches one behind the other whose pass is next to nothing, so that a cluster's blocks start and write at almost the
    same time."""
    logits, s = _logits(60, 4, 40, torch.bfloat16, 13), _search(60, 4, 12, 4)
    want = _run_step(logits.cuda(), s)
    _check_step(want, logits, s)
    import turbot5_b200 as t5b
    dev, pos, x = [s[n].cuda() for n in ("scores", "pool", "steps", "beams", "done")], torch.tensor([s["pos"]], device="cuda"), logits.cuda()
    every = [t5b.beam_search_step(x, *dev, pos) for _ in range(400)]
    assert all(torch.equal(a, b) for got in every for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,M,N", [(64, 1, 2000), (64, 4, 16384), (64, 7, 2000), (16, 2, 5000), (32, 8, 3000), (128, 1, 16384), (128, 5, 2000),
                                   (64, 1, 100000), (128, 3, 40)])
@pytest.mark.parametrize("nats", [10.12, 17.5, 22.0])
def test_attention_faint_tail_behind_a_leading_key(nats, D, M, N, dtype):
    """One key that takes nearly all of the weight, with values of 0: the result is that of the others, e^-nats each."""
    import turbot5_b200 as t5b
    cap = -(-N // 64) * 64
    g = torch.Generator().manual_seed(N)
    for lead in {0, N // 2, N - 1}:
        k, v = torch.zeros((1, 1, cap, D)), torch.rand((1, 1, cap, D), generator=g).add(1).mul(200).to(FP8).float()
        k[0, 0, lead, 0] = 1.0
        v[0, 0, lead] = 0
        # rows of their own: 16 / 16, 15 / 16, ... of the leading key's score; the first row's result is about 1
        q = torch.zeros((1, 1, M, D))
        q[0, 0, :, 0] = 1 - torch.arange(M) / 16
        v_scale = 2.0 ** round(math.log2(math.exp(nats) / N / 300))
        ks, vs = torch.ones((1, 1, cap // 64)), torch.full((1, 1, cap // 64), v_scale)
        got = t5b.flash_decoding_quantized_with_fusing_bias(q.to(dtype).cuda(), k.to(FP8).cuda(), ks.cuda(), v.to(FP8).cuda(), vs.cuda(), None,
                                                            sm_scale=nats, kv_len=N)[0, 0].double().cpu()
        tail = v[0, 0, :N].double().sum(0) * v_scale
        for m in range(M):
            faint = math.exp(-nats * (1 - m / 16))
            total = 1 + faint * (N - 1)
            want = tail * faint / total
            # per weight: its two halves 2^-22, two exponentials of 2^-22 (its own, its item's), their arguments (up to
            # 1.5 nats + 14 each, rounded twice); sums of an item, of a warp's items and of the warps in float32; keys that
            # share the leading key's item: half of 2^-38 of its weight (rounding of hi and of lo, at 2^14: 2^-25 each)
            steps = N / (32 * 8) + 2 + 64 + 64
            rel = 3 * 2.0 ** -22 + 4 * (1.5 * nats + 14) * 2.0 ** -24 + 2 * steps * 2.0 ** -23
            tol = want * (torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -8) + rel) + 63 * 2.0 ** -38 * 400 * v_scale / total
            off = (got[m] - want).abs()
            assert (off <= tol).all(), (lead, m, (off / want).max(), (tol / want).min())


@pytest.mark.parametrize("D,M", [(64, 1), (64, 6), (128, 2)])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_equal_scores_of_any_size(D, M, sign):
    """Equal scores give the mean of the values, however large they are (their last place may be wider than the 14 that
    weights are kept above 1); a second group of keys far below takes no part."""
    import turbot5_b200 as t5b
    N = 150
    (k, _), (v, vs) = _cache(1, 2, 192, D, 3), _cache(1, 2, 192, D, 4)
    k = torch.zeros_like(k.float())
    k[..., 0] = sign
    k[:, :, 64:100, 0] = -2
    q = torch.zeros((1, 2, M, D))
    q[..., 0] = 1
    kept = [n for n in range(N) if not 64 <= n < 100]
    want = (v.double() * vs.double().repeat_interleave(64, -1)[..., None])[:, :, kept]
    want, size = want.mean(2, keepdim=True), want.abs().mean(2, keepdim=True)
    for power in (9, 18, 19, 20, 21, 24, 25, 26, 27, 30, 60, 100):
        got = t5b.flash_decoding_quantized_with_fusing_bias(q.half().cuda(), k.to(FP8).cuda(), torch.ones((1, 2, 3), device="cuda"), v.cuda(), vs.cuda(),
                                                            None, sm_scale=2.0 ** power, kv_len=N).double().cpu()
        # float32 sums of 150 numbers (each half of a weight exact), a quotient, the result's rounding
        tol = want.abs() * 2.0 ** -11 * (1 + 2.0 ** -8) + size * 200 * 2.0 ** -23 + 2.0 ** -25
        assert ((got - want).abs() <= tol).all(), power


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,M", [(16, 1), (64, 4), (64, 8), (128, 1)])
def test_attention_small_elements_of_a_query_beside_a_large_one(D, M, dtype):
    """The keys are 0 where the query is large: its small elements alone make the scores."""
    B, H, n = 2, 2, 130
    g = torch.Generator().manual_seed(D + M)
    for power in (-12, -20, -24):                      # (held exactly down to 2^-31 of the row's largest element)
        q = torch.randn((B, H, M, D), generator=g) * 2.0 ** power
        q[..., 3] = 1.0
        (k, ks), kv_v = _cache(B, H, 192, D, 3), _cache(B, H, 192, D, 4)
        kf = k.float()
        kf[..., 3] = 0
        # scores of a few units; float16 holds no elements below 2^-24: the large one is then 2^14
        lift = 2.0 ** 14 if dtype == torch.float16 else 1.0
        _check_attention((q * lift).to(dtype), ((kf.to(FP8), torch.full_like(ks, 2.0 ** -6)), kv_v), None, [n, 60], False,
                         2.0 ** -power / lift * D ** -0.5)


@pytest.mark.parametrize("power", [-133, -126, -112, 100, 124, 126])
def test_attention_queries_of_any_size(power):
    """From subnormal numbers to the largest ones, with scales and a factor that make ordinary scores of them."""
    B, H, M, D, n = 1, 2, 3, 64, 100
    g = torch.Generator().manual_seed(5)
    q = (torch.randn((B, H, M, D), generator=g).clamp(-1.9, 1.9).double() * 2.0 ** power).to(torch.bfloat16)
    (k, ks), kv_v = _cache(B, H, 128, D, 3), _cache(B, H, 128, D, 4)
    half = 2.0 ** (-power // 2)
    _check_attention(q, ((k, torch.full_like(ks, 2.0 ** -8 * half)), kv_v), None, [n], False, 2.0 ** -power / half)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K,V,std", [(100, 16, 128256, 6.0), (16, 4, 32128, 2.5), (40, 16, 32128, 1.0)])
def test_step_log_sums(B, K, V, std, dtype):
    """Running scores that cancel the log-probability of each row's best token: what is left is the error of the log-sum, not
    hidden by the rounding of the result."""
    import turbot5_b200 as t5b
    g = torch.Generator(device="cuda").manual_seed(V)
    logits = (torch.randn((B * K, V), generator=g, device="cuda") * std).to(dtype)
    lse = torch.cat([torch.logsumexp(rows.double(), -1) for rows in logits.split(64)])
    scores = (lse - logits.max(-1)[0].double()).float()
    none = torch.zeros((B, K), dtype=torch.int32, device="cuda")
    tokens, parents, out, *_ = t5b.beam_search_step(logits, scores.view(B, K), torch.full((B, K), NONE, device="cuda"), none, none,
                                                    torch.zeros(B, dtype=torch.bool, device="cuda"), torch.zeros(1, dtype=torch.long, device="cuda"),
                                                    eos_token_id=None)
    rows = (torch.arange(B, device="cuda")[:, None] * K + parents.long()).flatten()
    want = scores[rows].double() + (logits[rows, tokens.flatten()].double() - lse[rows])
    off = (out.flatten().double() - want)[want.abs() < 1e-3]           # (float32 of 1e-3: 2^-34)
    assert off.numel() >= B * K // 2
    # at most: four exponentials in a row (a term's, those to its lane's, its warp's and the row's maximum) of 2^-22, their
    # arguments (up to 40 in base 2, three roundings), 12 float32 additions
    assert off.abs().max() <= 4 * 2.0 ** -22 + 3 * 40 * 2.0 ** -24 * math.log(2) + 12 * 2.0 ** -24
    # on average the roundings cancel.  What remains: an exponential is 5.1e-8 too small (three of them), and log2(e) in
    # float32 1.4e-8 of the distance from the maximum (3 on the weighted average)
    assert off.mean().abs() <= 3 * 5.1e-8 + 3 * 1.4e-8


@pytest.mark.parametrize("V", [5000, 140001])
def test_step_logarithms(V):
    """Rows of n equal logits: their sum of exponentials is n exactly, and running scores that cancel the logarithm leave
    its error."""
    import turbot5_b200 as t5b
    B, K = 8, 8
    g = torch.Generator().manual_seed(V)
    counts = [2, 3, 5, 7, 11, 16, 45, 46, 63, 64, 65, 90, 91, 1448, 1449, 4096] + torch.randint(2, V + 1, (B * K - 16,), generator=g).tolist()
    logits = torch.full((B * K, V), NONE)
    for row, n in zip(logits, counts):
        row[:n] = 1.5
    logs = torch.tensor([math.log(n) for n in counts], dtype=torch.float64)
    scores = logs.float()
    none = torch.zeros((B, K), dtype=torch.int32, device="cuda")
    _, parents, out, *_ = t5b.beam_search_step(logits.cuda(), scores.view(B, K).cuda(), torch.full((B, K), NONE, device="cuda"), none, none,
                                               torch.zeros(B, dtype=torch.bool, device="cuda"), torch.zeros(1, dtype=torch.long, device="cuda"),
                                               eos_token_id=None)
    rows = (torch.arange(B)[:, None] * K + parents.long().cpu()).flatten()
    want = scores[rows].double() - logs[rows]
    # the series' first missing term 2 / 17 * 0.172^17 = 1e-14, a reciprocal of 48 bits, float64 roundings of numbers up to
    # 12; the result's own, of 2^-21 at most
    assert ((out.flatten().double().cpu() - want).abs() <= 1e-13 + want.abs() * 2.0 ** -24).all()
    assert len(set(rows.tolist())) >= B                # (the best row of each sentence at least)


def test_caches_between_and_over_one_another_rows():
    """Views with gaps: refused where two of them share bytes, wherever that is, and taken where they lie between one
    another's rows, heads or tokens."""
    import turbot5_b200 as t5b
    parents = torch.tensor([[1, 0], [0, 0]], dtype=torch.int32, device="cuda")
    base = torch.arange(4 * 3 * 128 * 16, device="cuda").view(4, 3, 128, 16) % 251
    rows = [1, 0, 2, 2]
    for a, b in ((slice(0, 64), slice(32, 96)), (slice(0, 64), slice(63, 127)), (slice(5, 8), slice(6, 9))):
        got = base.to(torch.uint8)
        with pytest.raises(ValueError, match="overlap"):
            t5b.reorder_beam_cache([got[:, :, a], got[:, :, b]], parents)
        assert torch.equal(got, base.to(torch.uint8))
    got = base.to(torch.uint8)
    with pytest.raises(ValueError, match="overlap"):
        t5b.reorder_beam_cache([got[:, :, :32], got[:, :, 64:96], got[:, :, 90:122]], parents)
    with pytest.raises(ValueError, match="overlap"):
        t5b.reorder_beam_cache([got[:, :2], got[:, 1:]], parents)
    t5b.reorder_beam_cache([got[:, :, :64], got[:, :, 64:]], parents)
    assert torch.equal(got, base.to(torch.uint8)[rows])
    got = base.to(torch.uint8)
    t5b.reorder_beam_cache([got[:, h:h + 1] for h in (2, 0, 1)], parents)
    assert torch.equal(got, base.to(torch.uint8)[rows])
    x = torch.ones((4, 1, 5, 16), device="cuda", dtype=torch.bfloat16)
    cache, scale = torch.zeros((4, 3, 192, 16), device="cuda").to(FP8), torch.ones((4, 3, 2, 2), device="cuda")
    with pytest.raises(ValueError, match="own"):
        t5b.quantize_into_cache(x, x, cache[:, :1, :128], scale[:, :1, 0], cache[:, :1, 64:], scale[:, :1, 1])
    with pytest.raises(ValueError, match="own"):
        t5b.quantize_into_cache(x, x, cache[:, :1, :64], scale[:, :1, 0, :1], cache[:, :1, 64:128], scale[:, :1, 0, :1])
    t5b.quantize_into_cache(x, x * 2, cache[:, :1, :64], scale[:, :1, 0, :1], cache[:, :1, 64:128], scale[:, :1, 1, 1:])
    back = lambda c, s: (c[:, :, :5].float() * s[..., None]).unique().tolist()
    assert back(cache[:, :1, :64], scale[:, :1, 0, :1]) == [1.0] and back(cache[:, :1, 64:128], scale[:, :1, 1, 1:]) == [2.0]


def test_caches_that_overlap_themselves_are_refused():
    import turbot5_b200 as t5b
    parents = torch.tensor([[1, 0], [0, 0]], dtype=torch.int32, device="cuda")
    base = torch.zeros(4 * 3 * 128 * 16, device="cuda", dtype=torch.uint8)
    x = torch.ones((4, 1, 5, 16), device="cuda", dtype=torch.bfloat16)
    scale = [torch.ones((4, 1, 2), device="cuda") for _ in range(2)]
    # rows that begin inside of one another, heads that do, one row for all
    for sizes, strides in (((4, 1, 128, 16), (1024, 2048, 16, 1)), ((4, 3, 128, 16), (6144, 2032, 16, 1)), ((4, 1, 128, 16), (0, 2048, 16, 1))):
        windows = base.as_strided(sizes, strides)
        with pytest.raises(ValueError, match="itself"):
            t5b.reorder_beam_cache([windows], parents)
        if sizes[1] == 1:
            with pytest.raises(ValueError, match="itself"):
                t5b.quantize_into_cache(x, x, windows.view(FP8), scale[0], torch.zeros((4, 1, 128, 16), device="cuda").to(FP8), scale[1])
    # any order of dims, steps over rows, and sizes of one with any stride are none of that
    t5b.reorder_beam_cache([base.view(3, 4, 128, 16).transpose(0, 1)], parents)
    t5b.reorder_beam_cache([base.view(8, 3, 64, 16)[::2]], parents)
    t5b.reorder_beam_cache([base.as_strided((4, 1, 128, 16), (2048, 1, 16, 1))], parents)


@pytest.mark.parametrize("B,K,V", [(100, 16, 128256), (300, 4, 32128), (64, 10, 50001), (148, 8, 20000), (700, 2, 9001)])
def test_step_of_large_batches(B, K, V):
    """Batches whose sentences have few blocks each, wide vocabularies: the best continuations against float64 sorting."""
    import turbot5_b200 as t5b
    g = torch.Generator(device="cuda").manual_seed(V)
    logits = torch.randn((B * K, V), generator=g, device="cuda") * 2.5
    scores = -torch.rand((B, K), generator=g, device="cuda") * 4
    none = torch.zeros((B, K), dtype=torch.int32, device="cuda")
    tokens, parents, out, *_ = t5b.beam_search_step(logits, scores, torch.full((B, K), NONE, device="cuda"), none, none,
                                                    torch.zeros(B, dtype=torch.bool, device="cuda"), torch.zeros(1, dtype=torch.long, device="cuda"),
                                                    eos_token_id=None)
    compared = 0
    for b in range(B):
        every = scores[b].double()[:, None] + logits[b * K:(b + 1) * K].double().log_softmax(-1)
        best = every.flatten().topk(K + 1)
        values = best.values.tolist()
        # what log-sums are off by (1e-6 covers the bound, both ways) may turn the last place around, in a few sentences
        if values[K - 1] - values[K] < 2e-6:
            continue
        compared += 1
        assert sorted(best.indices[:K].tolist()) == sorted((parents[b].long() * V + tokens[b]).tolist()), b
        got = out[b].double().sort(descending=True)[0]
        assert ((got - best.values[:K]).abs() <= best.values[:K].abs() * 2.0 ** -24 + 1e-6).all()
        for j in range(K):                             # a beam that goes on keeps its place once
            assert int(parents[b, j]) == j or j not in parents[b].tolist()
    assert compared >= B * 0.99 - 1
