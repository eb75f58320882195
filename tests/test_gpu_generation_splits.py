"""The launches of the generation operators that large batches and long caches take: every rule that splits their work."""
import math

import pytest
import torch

from tests import generation_plain as plain
from tests.test_gpu_generation import FP8, _parents, _reordered

pytestmark = pytest.mark.gpu


def _device_cache(B, H, cap, D, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    values = torch.empty((B, H, cap, D), dtype=FP8, device="cuda")
    for b in range(B):
        values[b] = (torch.randn((H, cap, D), generator=g, device="cuda") * 60).clamp(-448, 448).to(FP8)
    return values, torch.exp2(torch.randint(-9, -3, (B, H, cap // 64), generator=g, device="cuda").float())


# heads x keys: which rule a call meets is said by `way`; 148 multiprocessors
WAYS = [
    # more than 512 heads of at most 16 items: two warps a head
    ("two warps", 32, 16, 1, 512, 64, False), ("two warps", 64, 12, 1, 500, 64, True), ("two warps", 64, 12, 4, 300, 64, False),
    ("two warps", 40, 16, 8, 512, 128, False), ("two warps", 32, 16, 2, 1024, 32, True), ("two warps", 43, 12, 1, 1000, 16, False),
    # somewhat more heads than blocks of four warps are resident: two warps, any length
    ("two warps", 32, 16, 1, 1100, 128, False), ("two warps", 34, 16, 3, 700, 128, True),
    # 401 to 1199 heads over 256 items and more: two blocks of four warps a head, merged in a cluster
    ("clusters of two", 28, 16, 1, 8192, 64, False), ("clusters of two", 34, 12, 4, 8200, 64, True), ("clusters of two", 28, 16, 1, 8192, 128, False),
    ("clusters of two", 34, 12, 7, 8500, 64, False), ("clusters of two", 70, 16, 1, 16400, 16, False),
    # else four warps a head, one block
    ("four warps", 20, 16, 1, 700, 64, False), ("four warps", 100, 16, 1, 640, 64, True), ("four warps", 80, 16, 5, 1400, 64, False),
    ("four warps", 16, 16, 2, 2048, 128, False),
    # few heads: eight warps, one block or a cluster of up to 16
    ("eight warps", 16, 13, 1, 2048, 64, False), ("eight warps", 2, 4, 1, 9000, 64, True), ("eight warps", 1, 2, 1, 40000, 128, False),
    ("eight warps", 9, 12, 8, 3000, 64, False),
]


@pytest.mark.parametrize("way,B,H,M,N,D,causal", WAYS)
def test_attention_of_every_split(way, B, H, M, N, D, causal):
    import turbot5_b200 as t5b
    cap = -(-N // 64) * 64
    (k, ks), (v, vs) = _device_cache(B, H, cap, D, 1), _device_cache(B, H, cap, D, 2)
    g = torch.Generator().manual_seed(N)
    q = (torch.randn((B, M, H, D), generator=g) * 2 * D ** -0.5).to(torch.bfloat16).transpose(1, 2)
    table = torch.randn((32, H), generator=g) if causal else None
    lengths = torch.randint(N // 3, N + 1, (B,), generator=g)
    lengths[0], lengths[B // 2], lengths[-1] = N, 0, N
    if B > 3:
        lengths[1], lengths[2] = 1, 65
    device_lengths = lengths.int().cuda()
    call = lambda rows: t5b.flash_decoding_quantized_with_fusing_bias(
        q[rows].cuda(), k[rows], ks[rows], v[rows], vs[rows], None if table is None else table.cuda(), causal=causal, sm_scale=1.0, kv_len=N,
        seqlens_k=device_lengths[rows])
    got = call(slice(None))
    # some heads against the plain form: float32 sums and roundings of scores and weights as in the other attention tests
    # (an item's sum of 64 and a warp's of its items in place of the whole length)
    steps = 64 + 64 + N / 32 / 2
    for b, h in {(0, 0), (0, H - 1), (B - 1, H // 2), (B // 3, H - 1), (min(2, B - 1), 0)}:
        n = int(lengths[b])
        heads = [(c[b:b + 1, h:h + 1].double() * s[b:b + 1, h:h + 1].double().repeat_interleave(64, -1)[..., None]).cpu() for c, s in ((k, ks), (v, vs))]
        want, mass, size = plain.attend(q[b:b + 1, h:h + 1], *heads, None if table is None else table[:, h:h + 1], [n], causal, 1.0)
        rel = 2 * (D + 8) * 2.0 ** -24 * 1.5 * (size + 1) + 2.0 ** -20 + 2 * steps * 2.0 ** -23
        tol = want.abs() * 2.0 ** -8 * (1 + 2.0 ** -8) + mass * rel + 1e-30
        off = (got[b:b + 1, h:h + 1].double().cpu() - want).abs()
        assert (off <= tol).all(), (b, h, (off / tol).max())
    # all of them against calls of one sentence each, which go another way: both are within half a step of the exact one,
    # and what float32 leaves of the largest value
    most = (v.float().abs().amax(dim=(2, 3)) * vs.amax(-1)).view(B, H, 1, 1)
    alone = torch.cat([call(slice(b, b + 1)) for b in range(B)])
    off = (got.float() - alone.float()).abs()
    assert (off <= alone.float().abs() * 2.0 ** -7 * (1 + 2.0 ** -7) + most * 2.0 ** -13).all()
    assert (got[lengths == 0] == 0).all()


@pytest.mark.parametrize("K", [2, 4, 7, 8, 11, 16])
@pytest.mark.parametrize("layers,B,H,cap,D,dtype", [(12, 2, 4, 512, 64, torch.bfloat16), (3, 5, 16, 700, 32, torch.uint8), (24, 3, 8, 200, 64, torch.float32)])
def test_reorder_blocks_that_take_many_pieces(K, layers, B, H, cap, D, dtype):
    """As many heads as there are blocks to share, so that each takes piece after piece of its head."""
    import turbot5_b200 as t5b
    g = torch.Generator().manual_seed(K)
    caches = [torch.randint(0, 200, (2, B * K, H, cap, D), generator=g).to(dtype) for _ in range(layers)]
    scales = [torch.rand((2, B * K, H, -(-cap // 64)), generator=g) for _ in range(layers)]
    parents = _parents(B, K, 5)
    lens = torch.randint(1, cap + 1, (B * K,), generator=g).int()
    lens[0] = cap
    got, got_scales = [c.cuda() for c in caches], [s.cuda() for s in scales]
    t5b.reorder_beam_cache(got, parents.cuda(), seqlens=lens.cuda(), scales=got_scales)
    used = lens.view(B, K).amax(1).tolist()
    for a, s, c, cs in zip(got, got_scales, caches, scales):
        for half in range(2):
            assert torch.equal(a[half].cpu(), _reordered(c[half], parents, used))
            assert torch.equal(s[half].cpu(), _reordered(cs[half], parents, [math.ceil(u / 64) for u in used]))
