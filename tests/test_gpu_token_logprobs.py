"""Log probabilities, entropy, top alternatives and their gradient against the definition in 64 bits.

Bounds.  u = 2^-24.  An exponential is off by u (|d| + 2) of itself, d its argument (the product that makes its exponent, and one last place
of the exponential).  A lane adds 8 logits of every 2048 columns, the lanes of a block 8 times more: C = 8 ceil(V / 2048) + 32 additions;
the sum s is off by (C + 4) u of itself plus u times the mean of |d| under the distribution, which is at most ln V + 2 for what is
drawn here.  So
  logprob   u (C + 8 (|logprob| + ln V + 4))
  entropy   u (3 C + 64) (1 + entropy)                    (q / s: both sums; entropy = ln s - q / s, both of one sign)
  gradient  half a step + u (C + 64 + 8 |ln p|) p (|A| + |B| (|ln p| + H + 1)) / T + 2 u (|A at the target| + sum |C|) / T"""
import math

import pytest
import torch

from optimus_dl_amd.modules.logprobs import token_logprobs

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def logits_of(rows, cols, dtype, seed=0, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    l = (torch.randn((rows, cols), device="cuda", generator=g) * spread).to(dtype)
    t = torch.randint(0, cols, (rows,), device="cuda", generator=g)
    return l, t, [torch.randn(s, device="cuda", generator=g) for s in ((rows,), (rows,), (rows, 64))]


def check(logits, targets, grads, n_vocab=None, top_k=0, temperature=1.0, entropy_grad=True, top_grad=True, spread=2.0):
    V = logits.shape[1] if n_vocab is None else n_vocab
    rows = logits.shape[0]
    C, lnv = 8 * math.ceil(V / 2048) + 32, math.log(V) + spread
    live = logits.detach().requires_grad_(True)
    r = token_logprobs(live, targets, n_vocab=n_vocab, top_k=top_k, temperature=temperature)
    exact = logits.detach().double().requires_grad_(True)
    logp = torch.log_softmax(exact[:, :V] / temperature, 1)
    lp = logp.gather(1, targets.unsqueeze(1)).squeeze(1)
    H = -(logp.exp() * logp).sum(1)
    assert r.logprobs.dtype == r.entropy.dtype == F32
    assert bool(((r.logprobs - lp).abs() <= U * (C + 8 * (lp.abs() + lnv + 4))).all())
    assert bool(((r.entropy - H).abs() <= U * (3 * C + 64) * (1 + H)).all())
    A, B, T = grads[0], grads[1] if entropy_grad else torch.zeros(rows, device="cuda"), grads[2][:, :top_k] if top_grad else torch.zeros((rows, top_k), device="cuda")
    outs, given = [r.logprobs], [A]
    if entropy_grad:
        outs.append(r.entropy), given.append(B)
    loss = (lp * A.double()).sum() + (H * B.double()).sum()
    if top_k:
        order = logits.detach()[:, :V].double().sort(dim=1, descending=True, stable=True).indices[:, :top_k]      # ties to the lowest index
        assert torch.equal(r.top_ids, order)
        top = logp.gather(1, order)
        assert bool(((r.top_logprobs - top).abs() <= U * (C + 8 * (top.abs() + lnv + 4))).all())
        if top_grad:
            outs.append(r.top_logprobs), given.append(T)
            loss = loss + (top * T.double()).sum()
    (got,) = torch.autograd.grad(outs, live, given)
    (want,) = torch.autograd.grad(loss, exact)
    with torch.no_grad():
        p = logp.exp()
        a = A.double().abs().unsqueeze(1) + T.double().abs().sum(1, keepdim=True)
        bound = U * (C + 64 + 8 * logp.abs()) * p * (a + B.double().abs().unsqueeze(1) * (logp.abs() + H.unsqueeze(1) + 1)) / temperature
        bound += 2 * U * a / temperature * torch.zeros_like(p).scatter_(1, targets.unsqueeze(1), 1.0)
        if top_k:
            bound += 2 * U * a / temperature * torch.zeros_like(p).scatter_(1, order, 1.0)
        assert got.shape == logits.shape and got.dtype == logits.dtype
        off = (got[:, :V].double() - want[:, :V]).abs() - HALF[got.dtype] * want[:, :V].abs() - bound
        assert bool((off <= 1e-38).all()), off.max().item()
        assert not got[:, V:].any()
    return r, got


# one column, less than a chunk, chunk ends, one section and several, odd sizes, vocabularies of real heads
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cols", [1, 5, 8, 9, 63, 64, 257, 1000, 2047, 2048, 2049, 4100, 32000, 50257])
@pytest.mark.parametrize("rows", [1, 3, 67])
def test_sizes(rows, cols, dtype):
    l, t, g = logits_of(rows, cols, dtype, seed=cols)
    check(l, t, g, top_k=min(5, cols))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0])
@pytest.mark.parametrize("top_k", [0, 1, 20, 64])
def test_temperatures_and_counts_of_alternatives(dtype, temperature, top_k):
    l, t, g = logits_of(33, 5003, dtype, seed=top_k)
    check(l, t, g, top_k=top_k, temperature=temperature)
    check(l, t, g, top_k=top_k, temperature=temperature, entropy_grad=False, top_grad=False)


def test_more_rows_than_blocks_of_the_backward():
    l, t, g = logits_of(1500, 1003, BF16)
    check(l, t, g, top_k=3)
    l, t, g = logits_of(20, 131072, BF16)                  # many sections a row
    check(l, t, g, top_k=64)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_columns_behind_the_vocabulary_are_never_read(dtype):
    for cols, V in ((1024, 1000), (50304, 50257), (72, 65), (100, 3)):
        l, t, g = logits_of(6, cols, dtype)
        l[:, V:] = float("nan")
        check(l, t % V, g, n_vocab=V, top_k=2)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_at_any_distance_and_alignment(dtype):
    l, t, g = logits_of(9, 1003, dtype)
    want, grad = check(l, t, g, top_k=4)
    wide = torch.full((9, 2011), float("nan"), dtype=dtype, device="cuda")
    for at in (0, 1, 3, 8):
        wide[:, at:at + 1003] = l
        r, got = check(wide[:, at:at + 1003], t, g, top_k=4)
        assert torch.equal(r.logprobs, want.logprobs) and torch.equal(got, grad)
    r, got = check(l.t().contiguous().t(), t, g, top_k=4)                               # columns apart: copied
    assert torch.equal(got, grad)
    one = l[:1].expand(9, -1)                                                           # one row for all
    assert torch.equal(token_logprobs(one, t).entropy, want.entropy[:1].expand(9))
    shaped = token_logprobs(l.reshape(3, 3, 1003), t.reshape(3, 3), top_k=4)
    assert torch.equal(shaped.logprobs.flatten(), want.logprobs) and shaped.top_ids.shape == (3, 3, 4)


def test_ties_go_to_the_lowest_index_also_where_thousands_share_a_value():
    g = torch.Generator(device="cuda").manual_seed(1)
    for cols in (3000, 40000):
        few = torch.randint(0, 3, (7, cols), device="cuda", generator=g).to(BF16)       # a third of the columns share the maximum
        few[1] = 0.0                                                                    # all equal
        few[2] = -0.0
        few[2, 5::7] = 0.0                                                              # zeros of both signs are equal
        few[3] = float("-inf")
        few[3, [17, 2500, 99]] = torch.tensor([1.0, 2.0, 1.0], device="cuda", dtype=BF16)   # all but three masked
        few[4] = torch.finfo(BF16).min                                                  # masked by the lowest value: uniform
        r = token_logprobs(few, torch.full((7,), 17, device="cuda"), top_k=64)
        assert torch.equal(r.top_ids, few.float().sort(dim=1, descending=True, stable=True).indices[:, :64])
        assert r.top_logprobs[3, :3].isfinite().all() and (r.top_logprobs[3, 3:] == float("-inf")).all()
        assert abs(r.entropy[4].item() - math.log(cols)) < 1e-4 and abs(r.logprobs[1].item() + math.log(cols)) < 1e-4


@pytest.mark.parametrize("rows", [8, 1100])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_ignored_empty_and_unsound_rows(rows, dtype):
    l, t, g = logits_of(rows, 6007, dtype)
    clean, grad = check(l, t, g, top_k=3)
    l = l.clone()
    l[0] = float("nan")
    t[0] = -100                                            # ignored: never looked at
    l[1] = float("-inf")                                   # nothing left
    l[2, ::2] = float("-inf")                              # half masked
    l[3, 77] = float("nan")
    l[4, 78] = float("inf")
    t[5], t[6] = 6007, -1                                  # no tokens
    live = l.requires_grad_(True)
    r = token_logprobs(live, t, top_k=3)
    (got,) = torch.autograd.grad((r.logprobs, r.entropy, r.top_logprobs), live, (g[0], g[1], g[2][:, :3].contiguous()))
    assert r.logprobs[0] == 0 and r.entropy[0] == 0 and not got[0].any() and (r.top_ids[0] == -1).all() and not r.top_logprobs[0].any()
    assert r.logprobs[1] == float("-inf") and r.entropy[1] == 0 and not got[1].any() and r.top_ids[1].tolist() == [0, 1, 2]
    for i in (3, 4):
        assert r.logprobs[i].isnan() and r.entropy[i].isnan() and r.top_logprobs[i].isnan().all() and (r.top_ids[i] == -1).all() and got[i].isnan().all()
    for i in (5, 6):
        assert r.logprobs[i].isnan() and got[i].isnan().all() and torch.equal(r.entropy[i], clean.entropy[i]) and torch.equal(r.top_ids[i], clean.top_ids[i])
    assert torch.equal(r.logprobs[7:], clean.logprobs[7:]) and torch.equal(got[7:], grad[7:])
    half = l.detach()[2:3, 1::2].contiguous()
    at = t[2] // 2 if t[2] % 2 else None
    alone = token_logprobs(half, torch.zeros(1, dtype=torch.int64, device="cuda") if at is None else at.reshape(1))
    assert abs((alone.entropy - r.entropy[2]).item()) < U * 400 * (1 + r.entropy[2].item()) and not got[2, ::2].float().sub(0).isnan().any()
    # the same as the torch operations that CPU tensors take
    c = l.detach().cpu().requires_grad_(True)
    from optimus_dl_amd.modules.logprobs import _plain

    p = _plain(c, t.cpu(), 6007, 3, 1.0, -100)
    assert torch.equal(p.top_ids, r.top_ids.cpu()) and torch.allclose(p.entropy, r.entropy.cpu().detach(), rtol=1e-4, atol=1e-4, equal_nan=True)
    assert torch.allclose(p.logprobs, r.logprobs.cpu().detach(), rtol=1e-4, atol=1e-4, equal_nan=True)


def test_extreme_values():
    """The largest differences of a type: exponents that run out at both ends."""
    for dtype in (BF16, F32):
        top, low = torch.finfo(dtype).max, torch.finfo(dtype).min
        l = torch.full((3, 4000), low, dtype=dtype, device="cuda")
        l[0, 3000] = top
        l[1, :2] = 5.0
        l[2, 1] = -1e30
        r = token_logprobs(l.requires_grad_(True), torch.tensor([3000, 1, 1], device="cuda"), top_k=2)
        (got,) = torch.autograd.grad((r.logprobs.sum() + r.entropy.sum()), l)
        assert r.logprobs.tolist()[0] == 0 and r.logprobs[2] == 0 and abs(r.logprobs[1].item() + math.log(2)) < 1e-6
        assert r.entropy[0] == 0 and abs(r.entropy[1].item() - math.log(2)) < 1e-6 and got.isfinite().all()
        assert r.top_ids.tolist() == [[3000, 0], [0, 1], [1, 0]]


def test_gradient_against_differences():
    l, t, g = logits_of(4, 700, F32)
    v = torch.randn(l.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))
    f = lambda x: sum((o.double() * w).sum() for o, w in zip(token_logprobs(x, t, top_k=2)[:3], (g[0], g[1], g[2][:, :2]))).item()
    live = l.clone().requires_grad_(True)
    r = token_logprobs(live, t, top_k=2)
    (got,) = torch.autograd.grad((r.logprobs, r.entropy, r.top_logprobs), live, (g[0], g[1], g[2][:, :2].contiguous()))
    h = 2.0 ** -7
    # value errors of 4e-6 each over 2 h, third derivatives of a mean of |v|^3 under a distribution times |ln p|, twenty at most, h^2 / 6
    assert abs((f(l + h * v) - f(l - h * v)) / (2 * h) - (got.double() * v).sum().item()) < 16 * 4e-6 / h + 40 * h * h


def test_parts_streams_and_captured_passes():
    from optimus_dl_amd import native as N

    for rows, dtype in ((5, BF16), (700, BF16), (5, F32)):
        l, t, g = logits_of(rows, 3001, dtype)
        lp, H, stats, top, ids = N.token_logprobs(l, t, 3001, 4, 1.0, -100, True)
        dl, parts = N.token_logprobs_bwd(l, t, 3001, 4, 1.0, -100, ids, stats, H, g[0], g[1], g[2][:, :4].contiguous())
        assert parts.shape == (N.AMAX_PARTS,) and parts.max().item() == dl.float().abs().max().item()
    l, t, g = logits_of(6, 9000, BF16)
    d_top = g[2][:, :4].contiguous()

    def step():
        lp, H, stats, top, ids = N.token_logprobs(l, t, 9000, 4, 1.0, -100, True)
        return lp, H, top, ids, *N.token_logprobs_bwd(l, t, 9000, 4, 1.0, -100, ids, stats, H, g[0], g[1], d_top)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    held = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(step())
    for seed in (3, 4, 5):
        nl, nt, _ = logits_of(6, 9000, BF16, seed)
        l.copy_(nl), t.copy_(nt)
        for graph in graphs:
            graph.replay()
        eager = step()
        torch.cuda.synchronize()
        for h in held:
            assert all(torch.equal(a, b) for a, b in zip(h, eager))


def test_no_rows():
    r = token_logprobs(torch.zeros((0, 100), device="cuda", requires_grad=True), torch.zeros(0, dtype=torch.int64, device="cuda"), top_k=3)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 3)
    r.logprobs.sum().backward()


@pytest.mark.parametrize("lead", [(), (6,), (2, 3), (2, 1, 3), (2, 0)])
@pytest.mark.parametrize("top_k", [0, 4])
def test_any_number_of_axes_with_and_without_a_graph(lead, top_k):
    rows = math.prod(lead)
    l, t, _ = logits_of(max(rows, 1), 300, BF16)
    l, t = l[:rows].reshape(*lead, 300), t[:rows].reshape(lead)
    with torch.no_grad():
        r = token_logprobs(l, t, top_k=top_k)
    live = token_logprobs(l.clone().requires_grad_(True), t, top_k=top_k)
    assert r.logprobs.shape == r.entropy.shape == lead and torch.equal(r.logprobs, live.logprobs) and torch.equal(r.entropy, live.entropy)
    if top_k:
        assert r.top_ids.shape == r.top_logprobs.shape == (*lead, top_k)
        assert torch.equal(r.top_ids, live.top_ids) and torch.equal(r.top_logprobs, live.top_logprobs)
    else:
        assert r.top_ids is None and r.top_logprobs is None


@pytest.mark.parametrize("temperature", [1.0, 1e-10, 1e-25, 1e10])
@pytest.mark.parametrize("log2_size", [-20, 0, 10, 20, 27, 29, 34, 50, 80, 95, 97, 120])
def test_logits_of_any_size(log2_size, temperature):
    """Bounds as above, C = 48: the exponents of what is drawn here are off by u (4 |d| + 2), d = (l - max) / T, whose product is rounded before or behind the
    subtraction.  What lies beyond the range of fp32 is -inf.  Rows of one sign, around a number by its last places, and with a step up for every lane."""
    g = torch.Generator(device="cuda").manual_seed(log2_size + 100)
    l = torch.randn((5, 3000), device="cuda", generator=g) * 2.0 ** log2_size
    l[1] = l[1].abs()
    l[2] = -l[2].abs()
    l[3] = l[3].abs().max() * (1 + torch.randint(0, 9, (3000,), device="cuda", generator=g) * 2.0 ** -23)      # the last places of one number
    l[4] = torch.sort(l[4]).values
    t = torch.randint(0, 3000, (5,), device="cuda", generator=g)
    live = l.clone().requires_grad_(True)
    r = token_logprobs(live, t, top_k=3, temperature=temperature)
    logp = torch.log_softmax(l.double() / temperature, 1)
    want = logp.gather(1, t.unsqueeze(1)).squeeze(1)
    fits = want > -2e38
    assert not r.logprobs.isnan().any() and bool(((r.logprobs - want).abs()[fits] <= (U * (8 * want.abs() + 250))[fits]).all())
    assert (r.logprobs[~fits] < -1e38).all()
    H = -(logp.exp() * logp.clamp_min(-1e300)).sum(1)
    assert bool(((r.entropy - H).abs() <= U * 250 * (1 + H)).all())
    assert torch.equal(r.top_ids, l.sort(dim=1, descending=True, stable=True).indices[:, :3])
    r.logprobs.sum().backward()
    p = logp.exp()
    want = -p / temperature
    want[torch.arange(5), t] += 1 / temperature
    assert bool(((live.grad * temperature - want * temperature).abs() <= U * (200 + 16 * logp.abs().clamp_max(1e3)) * p + 4 * U).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cols", [64, 100, 4097, 50257])
def test_many_alternatives_wherever_the_logits_lie(dtype, cols):
    """The ids are those of a stable sort, for values of one sign, of both, around zero (of either sign, subnormal too), with infinities below and with ties."""
    l, t, _ = logits_of(9, cols, dtype, seed=cols)
    l[1] = l[1].abs() + 1
    l[2] = -l[2].abs() - 1
    l[3] *= 1e-39
    l[4] = torch.where(l[4] > 0, 0.0, -0.0).to(dtype)
    l[5, 40:] = float("-inf")
    l[6] = (l[6] * 4).round() / 4
    l[7] *= 1e30
    l[8] = -3.0 - torch.arange(cols, device="cuda").flip(0).to(dtype) / cols
    want = l.float().sort(dim=1, descending=True, stable=True).indices
    for top_k in (31, 32, 33, 48, 64):
        r = token_logprobs(l, t, top_k=top_k)
        assert torch.equal(r.top_ids, want[:, :top_k])
        assert bool((r.top_logprobs[:, 1:] <= r.top_logprobs[:, :-1]).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 3, 64, 127, 129])
@pytest.mark.parametrize("cols", [98303, 98304, 131077, 151936])
def test_rows_that_several_blocks_share(rows, cols, dtype):
    l, t, grads = logits_of(rows, cols, dtype, seed=rows)
    for top_k in (0, 1, 20, 64):
        check(l, t, grads, top_k=top_k)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_what_parts_of_a_row_may_hold(dtype):
    V = 131077                                              # eight parts of 16392, the last one shorter
    l, t, _ = logits_of(10, V, dtype, seed=4)
    l[0] = float("-inf")                                    # nothing
    l[1, :100000] = float("-inf")                           # parts with nothing
    l[2] = float("-inf")
    l[2, [5, 40000, 131076]] = torch.tensor([1.0, 2.0, 1.0], device="cuda", dtype=dtype)
    l[3, 70000] = float("nan")
    l[4, 131076] = float("inf")
    l[5] = 0.25                                             # all equal: thousands of candidates in each part
    l[6] = torch.finfo(dtype).min
    l[6, 100000:] = torch.randint(0, 5, (V - 100000,), device="cuda").to(dtype)        # ties within and across parts
    l[7] = torch.randint(0, 3, (V,), device="cuda").to(dtype)
    l[8] = torch.arange(V, device="cuda").to(dtype) / 1000  # all of the best in the last part
    t[9] = -100
    for top_k in (0, 5, 64):
        live = l.clone().requires_grad_(True)
        r = token_logprobs(live, t, top_k=top_k)
        exact = l.double()
        logp = torch.log_softmax(exact[[1, 2, 5, 6, 7, 8]], 1)
        want = logp.gather(1, t[[1, 2, 5, 6, 7, 8], None]).squeeze(1)
        got = r.logprobs[[1, 2, 5, 6, 7, 8]].double()
        assert torch.equal(got == -math.inf, want == -math.inf)
        ok = want > -1e30
        assert bool(((got - want).abs()[ok] <= 2e-6 * (20 + want.abs()[ok])).all())
        assert r.logprobs[0] == -math.inf and r.entropy[0] == 0 and r.logprobs[3].isnan() and r.logprobs[4].isnan() and r.logprobs[9] == 0 == r.entropy[9]
        assert abs(r.entropy[5].item() - math.log(V)) < 1e-4 and r.entropy[[3, 4]].isnan().all()
        if top_k:
            order = l.float().sort(dim=1, descending=True, stable=True).indices[:, :top_k]
            sound = [0, 1, 2, 5, 6, 7, 8]
            assert torch.equal(r.top_ids[sound], order[sound]) and (r.top_ids[[3, 4, 9]] == -1).all()
            assert r.top_logprobs[[3, 4]].isnan().all() and (r.top_logprobs[9] == 0).all() and (r.top_logprobs[0] == -math.inf).all()
        (r.logprobs[[1, 5, 6, 7, 8, 9]].nan_to_num(neginf=0.0).sum() + r.entropy[[0, 1, 2, 5, 6, 7, 8, 9]].sum()).backward()
        assert live.grad[[0, 9]].abs().max() == 0 and live.grad[[1, 2, 5, 6, 7, 8]].isfinite().all()
