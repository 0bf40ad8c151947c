"""The paged cache on the CPU where numbers are odd or 0."""
import torch

from optimus_dl_amd.modules.paged import append_kv, paged_attention
from tests.paged_helpers import E4M3, Case, bits


def test_nothing_is_kept_of_a_head_whose_scale_is_0():
    """Every code stands for 0 there; 0 / 0 is no code."""
    c = Case([3], [20], 4, 2, 16, 4, E4M3, seed=1)
    c.key_scale[0], c.value_scale[1] = 0.0, 0.0
    c.k[1, 0], c.v[2, 1] = 0.0, 0.0
    q = append_kv(c.q, c.k, c.v, c.keys, c.values, *c.batch(), **c.scales())
    for p in (17, 18, 19):
        page = int(c.pages[0, p // 4])
        for t, dead in ((c.keys, 0), (c.values, 1)):
            assert (bits(t)[page, dead, p % 4] == 0).all() and (bits(t)[page, 1 - dead, p % 4] != 0).any()
    assert paged_attention(q, c.keys, c.values, *c.batch(), **c.scales()).isfinite().all()
    c.k[0, 0, 3] = float("nan")
    append_kv(c.q, c.k, c.v, c.keys, c.values, *c.batch(), **c.scales())
    assert c.keys[int(c.pages[0, 4]), 0, 1].float().isnan().tolist() == [i == 3 for i in range(16)]
