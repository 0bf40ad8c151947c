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


def test_rows_without_a_score_above_minus_infinity_answer_0_beside_odd_values():
    c = Case([2, 1], [30, 5], 4, 2, 16, 4, seed=2)
    c.q.fill_(1.0)
    c.values[..., 3], c.values[..., 4] = float("inf"), float("nan")
    c.keys[..., 7] = -torch.inf
    c.keys[int(c.pages[1, 1])] = 0.0             # the second sequence's last token
    y = paged_attention(c.q, c.keys, c.values, *c.batch())
    assert (y[:2] == 0).all() and (y[2, :, 3] == torch.inf).all() and y[2, :, 4].isnan().all() and y[2, :, 5:].isfinite().all()
