"""Beam search and 8-bit caches through the model: `T5ForConditionalGeneration.beam_search` / `generate`."""
import pytest
import torch

from tests import generation_plain as plain
from tests.helpers import TINY_T5, seed_named_parameters

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def _model(dtype=torch.float32, **kw):
    from turbot5_b200.t5 import T5ForConditionalGeneration, T5StackConfig
    model = T5ForConditionalGeneration(T5StackConfig(**{**TINY_T5, **kw}))
    return seed_named_parameters(model, seed=3).to(dtype).cuda().eval()


def _states(B, L, dtype=torch.float32, d_model=TINY_T5["d_model"]):
    return torch.randn((B, L, d_model), generator=torch.Generator().manual_seed(L)).to(dtype).cuda()


def _recorded(model, states, steps, beams, **kw):
    """A search launched step by step, with the logits of every step."""
    from turbot5_b200.t5 import BeamDecoding
    seen, logits = [], type(model).logits
    model.logits = lambda hidden: seen.append(logits(model, hidden)) or seen[-1]
    try:
        search = BeamDecoding(model, states, steps, beams, use_cuda_graph=False, **kw)
        for _ in range(steps):
            search.step()
    finally:
        del model.logits
    return search, [x.double().cpu().view(-1, x.shape[-1]) for x in seen]


def _plain_search(logits, B, K, eos=1, pad=0, **kw):
    none = float("-inf")
    state = [[[0.0] + [none] * (K - 1) for _ in range(B)], [[none] * K for _ in range(B)], [[0] * K for _ in range(B)], [[0] * K for _ in range(B)],
             [False] * B]
    history = ([], [])
    for t, x in enumerate(logits):
        out = plain.step(x.tolist(), *state, t, eos=eos, pad=pad, **kw)
        state = [[torch.tensor(r, dtype=torch.float64).float().tolist() for r in out[2]], *out[3:]]
        history[0].append(out[0])
        history[1].append(out[1])
    return state, history


@pytest.mark.parametrize("B,K,length_penalty,early", [(1, 1, 1.0, False), (3, 4, 1.0, False), (2, 5, 2.0, True), (1, 16, 0.0, False)])
def test_search_over_the_model_is_the_plain_search_over_its_logits(B, K, length_penalty, early):
    model, states, steps = _model(), _states(B, 23), 12
    search, logits = _recorded(model, states, steps, K, length_penalty=length_penalty, early_stopping=early)
    state, history = _plain_search(logits, B, K, length_penalty=length_penalty, early=early)
    assert search.history[0].tolist() == history[0] and search.history[1].tolist() == history[1]
    assert search.done.tolist() == state[4] and search.finished_steps.tolist() == state[2]
    want, values = plain.sequences(*history, *state, K, length_penalty=length_penalty)
    got, scores = search.sequences(K)
    assert got.tolist() == want
    fine = torch.isfinite(scores.cpu())
    # twelve float32 sums of step scores, each with the bound of one step's (6e-6 and half a step of the sum)
    assert ((scores.cpu().double() - torch.tensor(values, dtype=torch.float64)).abs()[fine] <= 1e-4).all()


def test_cached_logits_are_those_of_the_sentences_so_far():
    """The reordered caches hold what their beams have seen: every step's logits against an uncached pass over the beams'
    tokens."""
    B, K, steps = 2, 4, 9
    model, states = _model(), _states(B, 31)
    search, logits = _recorded(model, states, steps, K)
    tokens, parents = (h.cpu() for h in search.history)
    with torch.no_grad():
        for t in range(steps):
            rows = []
            for b in range(B):
                for j in range(K):
                    words, beam = [], j
                    for s in range(t - 1, -1, -1):
                        words.append(int(tokens[s, b, beam]))
                        beam = int(parents[s, b, beam])
                    rows.append([0] + words[::-1])
            ids = torch.tensor(rows, device="cuda")
            want = model.logits(model.decoder(ids, encoder_hidden_states=states.repeat_interleave(K, 0)))[:, -1].double().cpu()
            # float32 on both sides, two layers: the tolerance of the module tests
            assert (logits[t] - want).abs().max().item() <= 1e-3, t


@pytest.mark.parametrize("dtype,cache", [(torch.float32, None), (torch.bfloat16, None), (torch.bfloat16, FP8), (torch.float16, FP8)])
def test_graph_and_eager_searches_are_the_same(dtype, cache):
    from turbot5_b200.t5 import BeamDecoding
    B, K, steps = 3, 4, 70                             # more than a block of cached tokens
    model, states = _model(dtype), _states(B, 40, dtype)
    lens = torch.tensor([40, 17, 1], dtype=torch.int32, device="cuda")
    a = BeamDecoding(model, states, steps, K, lens, cache_dtype=cache)
    b = BeamDecoding(model, states, steps, K, lens, cache_dtype=cache, use_cuda_graph=False)
    for turn in range(2):                              # again after going back to the start
        for _ in range(steps):
            a.step()
            b.step()
        for x, y in zip(a.sequences(K) + (a.scores, *a.history), b.sequences(K) + (b.scores, *b.history)):
            assert torch.equal(x, y)
        with pytest.raises(RuntimeError, match="full"):
            a.step()
        a.rewind()
        b.rewind()


def test_two_captured_searches_replayed_at_once():
    from turbot5_b200.t5 import BeamDecoding
    K, steps = 4, 20
    model = _model(torch.bfloat16)
    for cache in (None, FP8):
        searches = [BeamDecoding(model, _states(4, n, torch.bfloat16), steps, K, cache_dtype=cache) for n in (700, 1500)]
        alone = []
        for s in searches:
            for _ in range(steps):
                s.step()
            alone.append([t.clone() for t in s.sequences(K)])
            s.rewind()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in searches]
        for _ in range(steps):
            for s, st in zip(searches, streams):
                with torch.cuda.stream(st):
                    s.step()
        torch.cuda.synchronize()
        for s, want in zip(searches, alone):
            assert all(torch.equal(x, y) for x, y in zip(s.sequences(K), want))


def test_one_beam_is_greedy():
    """A search with one beam that nothing ends makes the greedy choices."""
    model, states, steps = _model(torch.bfloat16, eos_token_id=-1), _states(3, 50, torch.bfloat16), 24
    search, logits = _recorded(model, states, steps, 1)
    assert search.history[0][:, :, 0].t().tolist() == torch.stack([x.argmax(-1) for x in logits], 1).tolist()


def test_eight_bit_cache_attends_over_what_it_holds():
    """A layer-by-layer step over an 8-bit cache against the same step over a 16-bit cache of the numbers that the 8-bit one
    stands for (a power of two times three mantissa bits: exact in bfloat16)."""
    B, N, steps = 3, 90, 6
    model, states = _model(torch.bfloat16), _states(B, N, torch.bfloat16)
    dec = model.decoder
    with torch.no_grad():
        eight, sixteen = dec.new_cache(states, 80, cache_dtype=FP8), dec.new_cache(states, 80)
        for i in range(len(dec.block)):
            back = [c[:, :, :N].float() * s.repeat_interleave(64, -1)[:, :, :N, None] for c, s in
                    ((eight.cross_k[i], eight.cross_scales[i][0]), (eight.cross_v[i], eight.cross_scales[i][1]))]
            sixteen.set_cross(i, *(t.to(torch.bfloat16) for t in back))
        for t in range(steps):
            ids = torch.randint(2, 100, (B, 1), generator=torch.Generator().manual_seed(t)).cuda()
            a = dec.decode_step(ids, eight)
            b = dec.decode_step(ids, sixteen)
            # the newest key and value are rounded in one of them: 2^-4 of each at most, and a self-attention output with
            # them; what they are added to is of the same size or larger, and there are two layers of it
            assert (a.float() - b.float()).norm() <= 2 * 2.0 ** -3 * b.float().norm()
            for i in range(len(dec.block)):            # from now on the 16-bit cache holds what the 8-bit one does
                for half in range(2):
                    got = eight.self_kv[i][half][:, :, :t + 1].float() * eight.scales[i][half].repeat_interleave(64, -1)[:, :, :t + 1, None]
                    kept = sixteen.self_kv[i][half][:, :, :t + 1]
                    # the first layer's input is the same in both: half a step of e4m3, 2^-4 of the number or 2^-10 of the
                    # scale below the normal numbers (a later layer's input has moved with the one before it, so that no
                    # bound by the element holds there)
                    if i == 0:
                        scale = eight.scales[i][half][:, :, :1, None]
                        assert ((got - kept.float()).abs() <= kept.float().abs() * 2.0 ** -4 + 2.0 ** -10 * scale).all()
                    kept.copy_(got)


@pytest.mark.parametrize("cache", [None, FP8])
def test_generate_with_beams_and_8_bit_caches(cache):
    model = _model(torch.bfloat16)
    ids = torch.randint(2, 100, (3, 40), generator=torch.Generator().manual_seed(1)).cuda()
    mask = torch.ones((3, 40), dtype=torch.long, device="cuda")
    mask[1, 25:] = 0
    out = model.generate(ids, attention_mask=mask, max_new_tokens=20, num_beams=4, cache_dtype=cache)
    more = model.generate(ids, attention_mask=mask, max_new_tokens=20, num_beams=4, num_return_sequences=3, cache_dtype=cache, use_cuda_graph=False)
    assert out.shape == (3, 20) and more.shape == (3, 3, 20) and torch.equal(out, more[:, 0])
    for row in more.flatten(0, 1).tolist():            # nothing but padding behind the end
        if 1 in row:
            assert set(row[row.index(1) + 1:]) <= {0}
    greedy = model.generate(ids, attention_mask=mask, max_new_tokens=20, cache_dtype=cache)
    assert torch.equal(greedy, model.generate(ids, attention_mask=mask, max_new_tokens=20, cache_dtype=cache, use_cuda_graph=False))


def test_search_ends_early():
    """When every search is done, the rest is padding and the steps end."""
    from turbot5_b200.t5 import BeamDecoding
    model, states = _model(), _states(2, 12)
    with torch.no_grad():
        model.lm_head.weight[1] = 0                    # the end token: as likely as it can be made
        hidden = model.decoder(torch.zeros((2, 1), dtype=torch.long, device="cuda"), encoder_hidden_states=states)
        model.lm_head.weight[1] = 50 * hidden.mean((0, 1))
    calls, step = [], BeamDecoding.step
    BeamDecoding.step = lambda self: (calls.append(1), step(self))
    try:
        ids, scores = model.beam_search(states, 64, 2, early_stopping=True, num_return_sequences=2)
    finally:
        BeamDecoding.step = step
    assert ids.shape == (2, 2, 64) and torch.isfinite(scores).all()
    assert len(calls) < 64 and (ids[:, :, len(calls):] == 0).all()


def test_refusals():
    from turbot5_b200.t5 import BeamDecoding
    model, states = _model(), _states(2, 12)
    for beams in (0, 17):
        with pytest.raises(ValueError):
            model.beam_search(states, 4, beams)
    with pytest.raises(ValueError):
        model.beam_search(states, 0, 2)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        model.beam_search(states, 4, 2, cache_dtype=FP8)
    with pytest.raises(ValueError, match="cache_dtype"):
        model.beam_search(states, 4, 2, cache_dtype=torch.int8)
    with pytest.raises(ValueError):
        model.beam_search(states, 4, 2, num_return_sequences=3)
    with pytest.raises(ValueError):
        model.generate(torch.zeros((1, 4), dtype=torch.long, device="cuda"), num_return_sequences=2)
    with pytest.raises(RuntimeError, match="no step"):
        BeamDecoding(model, states, 4, 2, use_cuda_graph=False).sequences()
    with pytest.raises(ValueError, match="decode_step_static"):
        model.decoder.decode_step(torch.zeros((4, 1), dtype=torch.long, device="cuda"), model.decoder.new_cache(states, 4, beams=2))


def test_more_refusals_before_any_step():
    model, states = _model(), _states(2, 12)
    with pytest.raises(ValueError, match="sentences"):
        model.beam_search(states, 4, 2, num_return_sequences=0)
    with pytest.raises(ValueError, match="beams"):
        model.generate(torch.zeros((1, 4), dtype=torch.long, device="cuda"), num_beams=0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K,steps", [(6, 70), (12, 9), (16, 9)])
def test_wide_searches_from_8_bit_caches(K, steps, dtype):
    """More beams than rows of one pass over the encoder's keys: the choices are the plain search's over the logits, and the
    logits those of each beam's sentence fed through a cache of its own, which nothing reorders."""
    B = 2
    model, states = _model(dtype), _states(B, 150, dtype)
    search, logits = _recorded(model, states, steps, K, cache_dtype=FP8)
    state, history = _plain_search(logits, B, K)
    assert search.history[0].tolist() == history[0] and search.history[1].tolist() == history[1]
    got, _ = search.sequences(K)
    assert got.tolist() == plain.sequences(*history, *state, K)[0]
    tokens, parents = (h.cpu() for h in search.history)
    last, lines = steps - 1, []
    for b in range(B):
        for j in range(K):
            words, beam = [], j
            for s in range(last - 1, -1, -1):
                words.append(int(tokens[s, b, beam]))
                beam = int(parents[s, b, beam])
            lines.append([0] + words[::-1])
    ids = torch.tensor(lines, device="cuda")
    with torch.no_grad():
        cache = model.decoder.new_cache(states.repeat_interleave(K, 0), steps, cache_dtype=FP8)
        for t in range(steps):
            pos, lens = torch.tensor([t], device="cuda"), torch.full((B * K,), t + 1, dtype=torch.int32, device="cuda")
            hidden = model.decoder.decode_step_static(ids[:, t:t + 1], cache, pos, lens)
        want = model.logits(hidden)[:, -1].double().cpu()
    running = [b * K + j for b in range(B) for j in range(K) if not bool(search.done[b])]
    assert running
    # the same arithmetic but for the rows that share a product: 16-bit roundings may fall the other way, and with them
    # those of the cached keys and values, half a step of e4m3 (2^-4) of some numbers, in two layers
    assert (logits[last] - want)[running].norm() <= 2 * 2.0 ** -4 * want[running].norm()
