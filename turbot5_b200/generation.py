"""Operators of generation: beam search and the caches that it works on.

TurboT5 inherits its generation loop (src/turbot5/heads/t5_heads.py:100-130 prepares the inputs of a step) and keeps
its cache in the model's type (src/turbot5/model/attentions.py:198,229-234).  Here a step of beam search is one launch on
the logits, the history is kept as tokens and parents and read back once at the end, the caches of all layers follow
their beams in place with one launch, and a cache can be held in 8 bits.  Nothing is read back from the device and no
operator keeps state of its own, so every call can be captured; no gradients are recorded.  The loop around them is
`T5ForConditionalGeneration.beam_search`.
"""
from . import _native as nat

_host = nat.host

CACHE_BLOCK = 64        # tokens of an 8-bit cache that share a scale
MAX_BEAMS = 16


def beam_search_step(logits, scores, finished_scores, finished_steps, finished_beams, done, pos, *, eos_token_id=1,
                     pad_token_id=0, length_penalty=1.0, early_stopping=False, out=None, history=None):
    """One step of beam search: returns (tokens, parents, scores, finished_scores, finished_steps, finished_beams, done).

    `logits` (batch * num_beams, vocab) in float32, float16 or bfloat16 are those of the running beams, whose summed
    log-probabilities are `scores` (batch, num_beams) float32 (start with 0 for one beam of a sentence and -inf for the
    others).  The candidates are the 2 * num_beams best continuations by score + log_softmax(logits), compared in float64 (a
    row's log-sum comes from float32 exponentials and is good to about 1.4e-7); among equal scores the lowest beam, within a beam the largest logit, then the lowest token.
    A candidate that is `eos_token_id` (None: there is no such token) and among the num_beams best joins the pool of
    finished sentences with score / (pos + 1) ** length_penalty; `finished_scores` (float32, best first, -inf where
    empty), `finished_steps` and `finished_beams` (int32: step and parent beam of the end token) hold the num_beams
    best of them.  The best other candidates go on: `tokens` (int64, the next input ids) and `parents` (int32, the beam
    that each one continues).  The first continuation of a beam keeps its place, so a cache has to move for further
    ones only; the running beams are not sorted.

    A sentence is `done` (bool) when its pool is full and either `early_stopping` is set or no running beam's score /
    (pos + 1) ** length_penalty is above the pool's worst, or when nothing can go on (all running scores -inf).  From then
    on its scores and pool stay, its tokens are `pad_token_id` and its parents itself.

    `pos` is the step's number from 0, one int64 on the device.  `out`: seven tensors to write to, each of them the
    matching input if wanted.  `history`: two int32 (steps, batch, num_beams) tensors whose row `pos` gets tokens and parents.
    NaN logits count as -inf; where a row has +inf, those tokens share the whole probability.  num_beams is at most 16."""
    return _host.beam_step(logits, scores, finished_scores, finished_steps, finished_beams, done, pos, eos_token_id,
                           pad_token_id, length_penalty, early_stopping, out, history)


def beam_search_sequences(tokens, parents, scores, finished_scores, finished_steps, finished_beams, done, *,
                          num_return_sequences=1, eos_token_id=1, pad_token_id=0, length_penalty=1.0):
    """The best sentences after the steps in `tokens` and `parents` (the history, int32 (steps, batch, num_beams)):
    (sequences (batch, num_return_sequences, steps) int64, their scores float32).

    The finished sentences compete with the running beams of searches that are not done, whose scores are divided by
    steps ** length_penalty; best first, finished ones first among equals.  `pad_token_id` stands behind the end, and
    everywhere where there is no such sentence (score -inf).  Sentences end with `eos_token_id` where they finished."""
    return _host.beam_sequences(tokens, parents, scores, finished_scores, finished_steps, finished_beams, done,
                                num_return_sequences, eos_token_id, pad_token_id, length_penalty)


def reorder_beam_cache(caches, parents, *, seqlens=None, scales=()):
    """Let cached keys and values follow their beams, in place: row b * num_beams + j of every tensor becomes what row
    b * num_beams + parents[b, j] was.

    `caches` are alike: (batch * num_beams, heads, capacity, head dim) of any type, or with one more dimension in front
    (`DecoderCache.self_kv`: keys and values in one tensor); `scales` are those of 8-bit caches, one per cache,
    (..., heads, capacity / 64) float32.  Only the first `seqlens` tokens (int32 (batch * num_beams,) on the device, the
    longest of a sentence's beams counts; None: all) of beams that change are moved; nothing else is touched.  One
    launch for up to 64 tensors."""
    _host.reorder_caches(caches, parents, seqlens, scales)


def quantize_into_cache(k, v, k_cache, k_scale, v_cache, v_scale, start=0, *, seqlens=None):
    """Write keys and values (B, H, M, D) in float32, float16 or bfloat16 into an 8-bit cache, at tokens start ..
    start + M.

    `k_cache` and `v_cache` are float8_e4m3fn (B, H, capacity, D), the capacity a multiple of 64, `k_scale` and `v_scale`
    float32 (B, H, capacity / 64): the smallest power of two with which the block's largest element fits 448 (from 2^-100
    to 2^120).  Tokens that join a block with a larger scale move the older ones to it, exactly unless they fall below
    the format's normal numbers.  Infinities saturate, NaN stays NaN, neither sets a scale.
    `start` is a number, or one int64 on the device (then tokens past the capacity are dropped).  With `seqlens`
    (int32 (B,)) only the first seqlens[b] of the M tokens are written and count for the scales.  What lies behind the
    written tokens counts as empty and is left as it is."""
    _host.cache_quantize(k, v, k_cache, k_scale, v_cache, v_scale, start, seqlens)
