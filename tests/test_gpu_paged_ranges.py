"""Attention over a paged cache where numbers are large, odd or 0: caps and scales over their whole range, infinities in work that is cut into splits."""
import math

import pytest
import torch

from optimus_dl_amd import native
from optimus_dl_amd.modules.paged import append_kv, paged_attention
from tests.paged_helpers import BF16, E4M3, Case, assert_near, bits
from tests.paged_oracle import attention_rows

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")


def attend(c, rows=None, scale=None, **kwargs):
    """Against the definition, in the given rows (all)."""
    scale, rows = c.dim ** -0.5 if scale is None else scale, list(range(c.rows)) if rows is None else rows
    want, far = attention_rows(c, rows, scale, kwargs.get("window", 0), kwargs.get("softcap", 0.0))
    c.to(CUDA)
    got = paged_attention(c.q, c.keys, c.values, *c.batch(), scale=scale, **kwargs, **c.scales())
    assert_near(got[rows], want, far)
    return got


FEW, MANY = ([1, 4], [300, 70]), ([70, 2], [200, 33])


@pytest.mark.parametrize("cap", [0.5, 3.0, 30.0, 256.0, 257.0, 1e3, 1e4, 1e5, 1e6])
@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("new,lengths", [FEW, MANY])
def test_caps_of_every_size(cap, cache, new, lengths):
    attend(Case(new, lengths, 4, 2, 64, 16, cache, seed=1), softcap=cap)
    attend(Case(new, lengths, 4, 2, 96, 16, cache, seed=2, q_scale=6.0), softcap=cap)


@pytest.mark.parametrize("cap", [1e3, 1e6])
@pytest.mark.parametrize("new,lengths", [FEW, MANY])
def test_scores_near_a_large_cap_beside_small_ones(cap, new, lengths):
    """Heads whose scores reach the cap in the same tile as heads whose scores are of size 1."""
    c = Case(new, lengths, 4, 1, 64, 16, seed=3)
    c.q[:, 1] *= cap / 10
    c.q[:, 3] *= cap / 200
    attend(c, softcap=cap)


@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("new,lengths", [FEW, MANY])
def test_scales_of_0_and_below(softcap, new, lengths):
    """A code stands for code * scale, whatever the scale: keys of 0 answer the mean of the values that are seen."""
    c = Case(new, lengths, 6, 3, 64, 16, E4M3, seed=4)
    c.key_scale[0], c.key_scale[1], c.value_scale[2] = 0.0, -c.key_scale[1], -c.value_scale[2]
    attend(c, softcap=softcap)
    c = Case(new, lengths, 4, 2, 128, 16, E4M3, seed=5)
    c.key_scale[1], c.value_scale[0] = 0.0, 0.0
    got = attend(c, softcap=softcap, window=50)
    assert (got[:, :2] == 0).all()


@pytest.mark.parametrize("new,lengths", [FEW, MANY])
def test_scales_that_are_none(new, lengths):
    """A scale of NaN is that head's answer, and that head's alone."""
    c = Case(new, lengths, 4, 2, 64, 16, E4M3, seed=6)
    c.key_scale[0] = math.nan
    c.to(CUDA)
    got = paged_attention(c.q, c.keys, c.values, *c.batch(), **c.scales())
    assert got[:, :2].isnan().all() and got[:, 2:].isfinite().all()


def test_nothing_is_kept_of_a_head_whose_scale_is_0():
    """Every code stands for 0 there; 0 / 0 is no code."""
    c = Case([3, 1], [20, 9], 4, 2, 64, 16, E4M3, seed=14)
    c.key_scale[0], c.value_scale[1] = 0.0, 0.0
    c.k[1, 0], c.v[2, 1] = 0.0, 0.0
    c.to(CUDA)
    q = append_kv(c.q, c.k, c.v, c.keys, c.values, *c.batch(), **c.scales())
    for t, dead in ((c.keys, 0), (c.values, 1)):
        for s, p in ((0, 17), (0, 18), (0, 19), (1, 8)):
            page = int(c.pages[s, p // 16])
            assert (bits(t)[page, dead, p % 16] == 0).all() and (bits(t)[page, 1 - dead, p % 16] != 0).any()
    assert paged_attention(q, c.keys, c.values, *c.batch(), **c.scales()).isfinite().all()
    c.k[0, 0, 3], c.k[0, 0, 5] = math.nan, math.inf
    append_kv(c.q, c.k, c.v, c.keys, c.values, *c.batch(), **c.scales())
    assert c.keys[int(c.pages[0, 1]), 0, 1].float().isnan().tolist() == [i == 3 for i in range(64)]


# Contexts that are cut into splits: (new tokens, tokens, heads, key heads)
CUT = [([1, 1], [3000, 40], 4, 1), ([40, 1], [5000, 70], 2, 1)]


@pytest.mark.parametrize("new,lengths,heads,kv", CUT)
def test_infinities_of_little_weight_in_a_split(new, lengths, heads, kv):
    """A seen infinity comes through whatever its weight, some e^-160 here, in whichever split or wave it lies."""
    for place in (5, 700, lengths[0] - new[0] - 60):
        c = Case(new, lengths, heads, kv, 64, 16, seed=7)
        c.q.fill_(1.0)
        c.keys.mul_(0.01)
        last = lengths[0] - new[0] - 10            # keys from here on score 20 * 64 / 8 more
        for p in range(last, lengths[0]):
            c.keys[int(c.pages[0, p // 16]), :, p % 16] += 20.0
        at = int(c.pages[0, place // 16]), 0, place % 16
        c.values[at + (3,)], c.values[at + (4,)], c.values[at + (5,)] = math.inf, -math.inf, math.nan
        got = attend(c, rows=list(range(sum(new))))[0]
        assert (got[:, 3] == math.inf).all() and (got[:, 4] == -math.inf).all() and got[:, 5].isnan().all() and got[:, 6:].isfinite().all()


@pytest.mark.parametrize("new,lengths", [([2], [40]), ([60], [200]), ([1], [3000])])
def test_rows_without_a_score_above_minus_infinity_answer_0_beside_odd_values(new, lengths):
    c = Case(new, lengths, 2, 1, 64, 16, seed=8)
    c.q.fill_(1.0)
    c.keys[..., 7] = -math.inf
    c.values[..., 3], c.values[..., 4] = math.inf, math.nan
    c.to(CUDA)
    assert (paged_attention(c.q, c.keys, c.values, *c.batch()) == 0).all()


@pytest.mark.parametrize("new,lengths", [FEW, MANY])
def test_rows_in_front_of_the_first_sequence_answer_0(new, lengths):
    """Offsets that begin behind row 0: those rows belong to nobody, as those behind the last sequence do."""
    c = Case(new, lengths, 4, 2, 64, 16, pad=3, seed=9)
    c.offsets = c.offsets + 2
    want, far = attention_rows(c, list(range(c.rows)), 0.125)
    c.to(CUDA)
    for _ in range(3):                             # (memory that the answer is likely to get)
        torch.full_like(c.q, math.nan)
        got = paged_attention(c.q, c.keys, c.values, *c.batch())
        assert (got[:2] == 0).all() and (got[-1:] == 0).all()
        assert_near(got, want, far)
    assert (append_kv(c.q, c.k, c.v, c.keys, c.values, *c.batch())[:2] == 0).all()


@pytest.mark.parametrize("length", [1, 129, 257, 511, 512, 700, 2048, 2049])
@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("dim,heads,kv", [(64, 12, 12), (128, 8, 2)])
def test_tables_of_any_width(length, cache, dim, heads, kv):
    """Which work is cut, and how, changes nothing: as wide as the context, one page wider, and much wider than it."""
    need = -(-length // 16)
    for width in (need, need + 1, 32, 33, 64, 65, 300):
        if width >= need:
            attend(Case([1], [length], heads, kv, dim, 16, cache, seed=length, width=width), max_new=1)


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_norms_with_bf16_weights_take_the_short_way(cache):
    """A model in bf16 has bf16 weights: widened by the kernel, bit by bit what fp32 copies of them give; weights of two types, or spread in memory, the long way."""
    def run(q_weight, k_weight, plain):
        c = Case([1, 3, 17], [1, 40, 33], 6, 2, 96, 16, cache, seed=15).to(CUDA)
        args = c.q, c.k, c.v, c.keys, c.values, *c.batch()
        if plain:
            out = native.plain_append_kv(*args, None, None, True, q_weight, k_weight, 1e-5, c.key_scale, c.value_scale)
            assert out is not None
        else:
            out = append_kv(*args, q_weight=q_weight, k_weight=k_weight, eps=1e-5, **c.scales())
        return [bits(t) for t in (out, c.keys, c.values)]

    g = torch.Generator().manual_seed(16)
    wide = [(1 + 0.2 * torch.randn(97, generator=g)).bfloat16().cuda() for _ in range(2)]
    for first in (0, 1):                                                             # (aligned to 16 bytes, and to 2)
        wq, wk = (w[first:first + 96] for w in wide)
        want = run(wq.float(), wk.float(), True)
        spread = torch.stack((wq, wq), 1)[:, 0]
        for a, b, plain in ((wq, wk, True), (wq.float(), wk, False), (wq, wk, False), (spread, wk, False)):
            assert all(torch.equal(x, y) for x, y in zip(run(a, b, plain), want))
    only = run(wq, None, True), run(wq.float(), None, True)
    assert all(torch.equal(x, y) for x, y in zip(*only))


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("dim,heads,kv", [(64, 16, 2), (128, 16, 2), (96, 16, 2)])
def test_splits_of_more_than_64_tiles(cache, dim, heads, kv):
    """A prompt whose splits have more tiles than are looked up at a time (64 of 64 keys), some of its pages none."""
    c = Case([2048], [9000], heads, kv, dim, 16, cache, seed=10)
    c.pages[0, 270], c.pages[0, 300] = -1, c.keys.shape[0]
    attend(c, rows=[0, 1, 31, 255, 256, 700, 1300, 1791, 1792, 2000, 2046, 2047])


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("heads,dim", [(1, 128), (2, 64)])
def test_tiles_of_more_than_64_splits(cache, heads, dim):
    """Forty tokens of one key head behind 20000: a tile in more splits than weights are kept of at a time."""
    attend(Case([40], [20040], heads, 1, dim, 16, cache, seed=11))


@pytest.mark.parametrize("new,lengths,heads,kv", CUT + [([1, 4], [300, 70], 4, 2), ([70, 2], [200, 33], 4, 2)])
def test_odd_values_and_codes(new, lengths, heads, kv):
    """NaN among codes of keys and values, infinities in bf16: in tokens that all rows of a sequence see, that some see, and that none does; uncut and cut."""
    n, length = new[0], lengths[0]
    for cache in (BF16, E4M3):
        c = Case(new, lengths, heads, kv, 64, 16, cache, seed=12)
        put = lambda t, p, h, d, x: t.view(torch.uint8 if cache == E4M3 else BF16)[int(c.pages[0, p // 16]), h, p % 16].__setitem__(d, x)
        nan = 0x7f if cache == E4M3 else math.nan
        put(c.values, 100, 0, 3, nan)                                                 # all rows of one key head
        put(c.values, length - 1, kv - 1, 5, nan)                                     # the last token's row alone
        if cache == BF16:
            put(c.values, 130, 0, 7, math.inf)
            put(c.values, length - 1, 0, 9, -math.inf)
        got = attend(c)
        assert got[0, 0, 3].isnan() and got[n - 1, heads - 1, 5].isnan()
        assert n == 1 or got[n - 2, heads - 1, 5].isfinite()
        c = Case(new, lengths, heads, kv, 64, 16, cache, seed=13)
        put(c.keys, length - 1, 0, 2, nan)                                            # a score of NaN, in the last token's row of a key head
        c.to(CUDA)
        got = paged_attention(c.q, c.keys, c.values, *c.batch()) if cache == BF16 else paged_attention(c.q, c.keys, c.values, *c.batch(), **c.scales())
        assert got[n - 1, :heads // kv].isnan().all() and got[:n - 1].isfinite().all() and got[n:].isfinite().all() and got[n - 1, heads // kv:].isfinite().all()
