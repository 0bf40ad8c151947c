"""The paged cache on the CPU where numbers are odd or 0."""
import ctypes

import pytest
import torch

from optimus_dl_amd import native
from optimus_dl_amd.modules.model import GPT2, GPT2Config
from optimus_dl_amd.modules.paged import PagedBatch, PagedKVCache, append_kv, paged_attention
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


def test_a_batch_looks_at_new_pages_alone(monkeypatch):
    """A decode step of long sequences: what is built in Python is the new pages, an offset and a length each, and not the whole table; the table says the same."""
    cache = PagedKVCache(1, 1, 16, pages=700, page_size=4, max_tokens=128, device="cpu", dtype=torch.float32)
    s = [cache.add() for _ in range(20)]
    lengths = [100 + i for i in range(20)]
    cache.batch(s, lengths)
    built, made = [], torch.tensor
    monkeypatch.setattr(torch, "tensor", lambda v, *a, **k: built.append(len(v)) or made(v, *a, **k))
    for step in range(6):
        if step == 3:
            cache.shorten(s[4], 3)
            cache.remove(s[7])
            s[7] = cache.add()
            lengths[4], lengths[7] = 3, 0
        built.clear()
        batch = cache.batch(s, [1] * 20)
        lengths = [n + 1 for n in lengths]
        assert sum(built) <= 20 + 41
        assert batch.lengths.tolist() == lengths and batch.offsets.tolist() == list(range(21))
        for row, i in zip(batch.pages.tolist(), s):
            assert row == cache._pages[i] + [0] * (32 - len(cache._pages[i])) and len(cache._pages[i]) == -(-cache.length(i) // 4)
    held = [p for i in s for p in cache._pages[i]]
    assert len(set(held)) == len(held) == 700 - cache.free_pages
    before = batch.pages.clone()
    cache.shorten(s[0], 0)
    assert torch.equal(batch.pages, before)              # (a batch that was made stays as it is)
    empty = cache.batch([], [])
    assert empty.pages.shape == (0, 32) and empty.offsets.tolist() == [0] and empty.lengths.shape == (0,) and empty.max_new == 0


def test_angles_belong_to_the_function_that_makes_them():
    cache = PagedKVCache(1, 1, 16, pages=2, page_size=4, device="cpu")
    made = []

    def first(dim, positions, theta, device):
        made.append(1)
        return torch.ones(positions, dim // 2), torch.zeros(positions, dim // 2)

    def second(dim, positions, theta, device):
        return torch.zeros(positions, dim // 2), torch.ones(positions, dim // 2)

    for _ in range(2):
        assert (cache.angles(first, 16, 1e4)[0] == 1).all() and (cache.angles(second, 16, 1e4)[0] == 0).all()
    assert len(made) == 1


@pytest.mark.parametrize("rows,heads,seqs,append_fits,attention_fits", [((1 << 24) - 1, 2, 3, True, True), (1 << 24, 2, 3, False, True), (1 << 20, 32, 1 << 20, True, False)])
def test_entries_refuse_more_blocks_than_a_launch_has(rows, heads, seqs, append_fits, attention_fits):
    """Pointers that nothing follows: what is refused is refused in front of a launch.  What fits goes on to the checks behind, and to an address that is refused."""
    if not native.is_built():
        pytest.skip("library not built")
    L = native.load()
    kv = heads // 2
    cache = native._PagedCache(4096, 4096, None, None, 10, kv, 16, 64)
    cache.key_strides[:] = cache.value_strides[:] = (1024 * kv, 1024, 64)
    batch = native._PagedBatch(4096, 4096, 4096, seqs, rows, 5, 5)
    refs, q, k = (ctypes.byref(cache), ctypes.byref(batch)), (ctypes.c_int64 * 2)(heads * 64, 64), (ctypes.c_int64 * 2)(kv * 64, 64)
    code = L.odl_fp8_append_kv(4096, q, 4096, k, 4096, k, heads, *refs, 4096, 4096, 80, 16, 1, None, None, 1e-6, 4104 if append_fits else 4096, None)
    assert code in (1, 2) and (b"aligned" if append_fits else b"blocks") in L.odl_fp8_last_error()
    code = L.odl_fp8_paged_attention(4096, q, heads, 1, *refs, 1.0, 0, 0.0, 4104 if attention_fits else 4096, 4096, 1 << 40, None)
    assert code in (1, 2) and (b"aligned" if attention_fits else b"blocks") in L.odl_fp8_last_error()


def test_positions_take_few_operations():
    """Every step of a model with learned positions makes them: each operation is a launch."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Count(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            self.made = getattr(self, "made", 0) + (not func.is_view and "empty" not in str(func))
            return out

    ints = lambda v: torch.tensor(v, dtype=torch.int32)
    for offsets, lengths in (([0, 3, 3, 4, 9], [10, 7, 1, 5]), ([0], []), ([0, 0], [5]), ([0, 2], [1]), ([0, 1, 2, 3], [2 ** 30, 1, 2 ** 30])):
        batch = PagedBatch(ints([[0]] * len(lengths)), ints(offsets), ints(lengths))
        with Count() as count:
            got = batch.positions(offsets[-1] + 3)
        want = [max(n - (offsets[s + 1] - r), 0) for s, n in enumerate(lengths) for r in range(offsets[s], offsets[s + 1])] + [0] * 3
        assert got.dtype == torch.int64 and got.tolist() == want and count.made <= 9
    assert batch.positions(0).shape == (0,)


def test_caches_without_heads_or_of_empty_heads_are_refused():
    ints = lambda v: torch.tensor(v, dtype=torch.int32)
    for heads, dim in ((0, 16), (1, 0)):
        q, cache = torch.zeros(1, 2, dim), torch.zeros(1, heads, 4, dim)
        batch = ints([[0]]), ints([0, 1]), ints([1])
        for call in (lambda: paged_attention(q, cache, cache, *batch), lambda: append_kv(q, q[:, :heads], q[:, :heads], cache, cache, *batch)):
            with pytest.raises(ValueError, match="kv heads"):
                call()


def test_tokens_of_a_step_that_raised_are_taken_out_again():
    model = GPT2(GPT2Config(vocab_size=32, n_embd=32, n_head=2, n_layer=1, block_size=16)).eval()
    cache = model.new_cache(pages=4, page_size=4)
    s, ids = cache.add(), torch.arange(9)
    model.step(ids[:5], cache, cache.batch([s], [5]))
    batch = cache.batch([s], [2])
    with pytest.raises(IndexError):
        model.step(ids[5:7] + 100, cache, batch)
    cache.shorten(s, cache.length(s) - 2)
    got = model.step(ids[5:9], cache, cache.batch([s], [4]))["logits"]
    assert torch.allclose(got, model(ids[None])["logits"][0, 5:].detach(), atol=1e-5)
