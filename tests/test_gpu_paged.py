"""A paged cache on the GPU: what goes into it, bit by bit, and attention over it against its definition in 64 bits."""
import math

import pytest
import torch

from optimus_dl_amd import native
from optimus_dl_amd.modules.paged import append_kv, paged_attention
from tests.paged_helpers import BF16, E4M3, Case, angles, append32, assert_near, attention64, bits

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")


def attend(c, scale=None, window=0, softcap=0.0, max_new=None):
    scale = c.dim ** -0.5 if scale is None else scale
    want, far = attention64(c, scale, window, softcap)
    c.to(CUDA)
    got = paged_attention(c.q, c.keys, c.values, *c.batch(), scale=scale, window=window, softcap=softcap, max_new=max_new, **c.scales())
    assert got.dtype == BF16 and got.is_contiguous()
    assert_near(got, want, far)
    return got


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("dim,half,norm", [(128, 64, False), (128, 64, True), (64, 16, False), (96, 48, True), (16, 8, False), (80, 40, False), (48, 0, True), (112, 0, False)])
def test_append_bits(interleaved, cache, dim, half, norm):
    c = Case([1, 3, 0, 17, 1], [1, 40, 9, 17, 33], 6, 2, dim, 16, cache, pad=2, seed=dim)
    cos, sin = angles(c.width * c.page, half) if half else (None, None)
    weights = [1 + 0.2 * torch.randn(dim) for _ in range(2)] if norm else [None, None]
    want = append32(c, cos, sin, interleaved, *weights)
    c.to(CUDA)
    on = [None if t is None else t.to(CUDA) for t in (cos, sin, *weights)]
    q = append_kv(c.q, c.k, c.v, c.keys, c.values, *c.batch(), cos=on[0], sin=on[1], interleaved=interleaved, q_weight=on[2], k_weight=on[3], **c.scales())
    for got, w, name in zip((q, c.keys, c.values), want, ("q", "keys", "values")):
        assert torch.equal(bits(got.cpu()), bits(w)), name


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("dim,heads,kv", [(128, 8, 2), (64, 12, 12), (96, 3, 1), (16, 8, 1)])
def test_attention_of_single_tokens(cache, dim, heads, kv):
    attend(Case([1] * 5, [1, 31, 32, 129, 700], heads, kv, dim, 16, cache, seed=1), max_new=1)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("dim,heads,kv,page", [(128, 8, 2, 16), (64, 3, 3, 64), (112, 4, 1, 4)])
def test_attention_of_prompts_and_chunks(cache, dim, heads, kv, page):
    attend(Case([100, 1, 33, 0, 70], [100, 200, 65, 12, 300], heads, kv, dim, page, cache, pad=5, seed=2))
