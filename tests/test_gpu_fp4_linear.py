"""Products with 4-bit weights and the cast that makes them.

Bound of a product: half a step of bf16 (2^-8) and, of the sum of |x| |w|, 2^-24 for every addition on the longest way: those of a wave (a group of K / 256 / 8
trips, each at most 8), its lanes and the waves of a block: K / 256 + 64.  Sums of small whole numbers are exact."""
from fractions import Fraction

import pytest
import torch

from optimus_dl_amd.modules.fp4_linear import E2M1, FP4Linear, dequantise_fp4, fp4_linear, quantise_fp4

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def weight_of(n, k, group, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.int64).to(torch.uint8)
    scales = (torch.rand((n, k // group), device="cuda", generator=g) * 0.02 + 1e-3).bfloat16()
    return codes, scales, g


def check(x, codes, scales, bias=None):
    got = fp4_linear(x, codes, scales, bias)
    w = dequantise_fp4(codes, scales).double()
    x2 = x.double().reshape(-1, x.shape[-1])
    want, mag = x2 @ w.t(), x2.abs() @ w.abs().t()
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    off = (got.double().reshape(want.shape) - want).abs() - 2.0 ** -8 * want.abs() - U * (x.shape[-1] / 256 + 64) * mag
    assert got.dtype == torch.bfloat16 and got.shape == (*x.shape[:-1], codes.shape[0]) and bool((off <= 0).all()), off.max().item()
    return got


# every nibble of every position: the order of k, and the value of each code
@pytest.mark.parametrize("group", [32, 64, 128])
def test_each_code_at_each_position(group):
    k = 384
    codes = torch.arange(256, device="cuda", dtype=torch.int64).to(torch.uint8).repeat(3)[:576].reshape(3, 192)
    scales = torch.tensor([1.0, 2.0, 0.5], device="cuda", dtype=torch.bfloat16).reshape(3, 1).expand(3, k // group).contiguous()
    got = fp4_linear(torch.eye(k, device="cuda", dtype=torch.bfloat16), codes, scales)
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device="cuda")
    nibbles = torch.stack((codes & 15, codes >> 4), -1).reshape(3, k).long()
    assert torch.equal(got.float(), (table[nibbles] * scales[:, :1].float()).t())
    assert torch.equal(dequantise_fp4(codes, scales), table[nibbles] * scales[:, :1].float())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 32, 33, 63, 64, 65, 120, 200])
def test_rows(rows, group):
    codes, scales, g = weight_of(300, 1024, group, rows)
    x = torch.randn((rows, 1024), device="cuda", generator=g).bfloat16()
    got = check(x, codes, scales)
    assert torch.equal(got, fp4_linear(x, codes, scales))


@pytest.mark.parametrize("rows", [1, 20, 70])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 100, 2304])
@pytest.mark.parametrize("k,group", [(32, 32), (64, 64), (128, 128), (96, 32), (160, 32), (192, 64), (384, 128), (768, 32), (2080, 32), (4096, 128)])
def test_sizes(rows, n, k, group):
    codes, scales, g = weight_of(n, k, group, n + k)
    x = torch.randn((rows, k), device="cuda", generator=g).bfloat16()
    check(x, codes, scales, torch.randn(n, device="cuda", generator=g))


@pytest.mark.parametrize("n,k,group", [(4096, 14336, 32), (14336, 4096, 128), (1024, 8192, 64)])
def test_layers_of_models(n, k, group):
    codes, scales, g = weight_of(n, k, group)
    for rows in (1, 32, 100):
        check(torch.randn((rows, k), device="cuda", generator=g).bfloat16(), codes, scales)


# blocks of 16, 32, 64 and 128 rows, of 128 and 256 columns, K in one run and in several, the last ones ragged
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,k", [(33, 4100, 1664), (63, 8200, 1664), (257, 4100, 1664), (200, 8200, 1664), (33, 4100, 2176), (257, 100, 4224),
                                      (13, 1030, 8320), (31, 8200, 3200), (17, 8200, 6272), (130, 4100, 2176), (50, 4100, 3200), (65, 8200, 4224),
                                      (65, 4100, 6272), (257, 8200, 1664), (530, 8200, 1664), (530, 2050, 3200)])
def test_ways_of_cutting_a_product(rows, n, k, group):
    codes, scales, g = weight_of(n, k, group, rows)
    x = torch.randn((rows, k), device="cuda", generator=g).bfloat16()
    bias = torch.randn(n, device="cuda", generator=g)
    assert torch.equal(check(x, codes, scales, bias), fp4_linear(x, codes, scales, bias))


def test_whole_numbers_are_exact_and_every_group_has_its_own_scale():
    for group in (32, 64, 128):
        codes, _, g = weight_of(70, 1280, group)
        scales = (2.0 ** torch.randint(-1, 3, (70, 1280 // group), device="cuda", generator=g).float()).bfloat16()
        x = torch.zeros((40, 1280), device="cuda")
        at = torch.randint(0, 1280, (40, 4), device="cuda", generator=g)
        x.scatter_(1, at, 1.0)
        want = x @ dequantise_fp4(codes, scales).t()
        assert torch.equal(fp4_linear(x.bfloat16(), codes, scales).float(), want.bfloat16().float()) and want.abs().max() <= 96


def test_strides_leading_dimensions_biases_and_rows_left_alone():
    codes, scales, g = weight_of(200, 512, 64)
    x = torch.randn((12, 512), device="cuda", generator=g).bfloat16()
    bias = torch.randn(200, device="cuda", generator=g)
    want = check(x, codes, scales, bias)
    check(x, codes, scales, bias.bfloat16())
    wide = torch.full((12, 1024), float("nan"), device="cuda", dtype=torch.bfloat16)
    for at in (0, 8, 3):                                   # rows apart; off the 16-byte grid: copied
        wide[:, at:at + 512] = x
        assert torch.equal(fp4_linear(wide[:, at:at + 512], codes, scales, bias), want)
    assert torch.equal(fp4_linear(x.reshape(3, 4, 512), codes, scales, bias).reshape(12, 200), want)
    assert torch.equal(fp4_linear(x[5], codes, scales, bias), want[5])
    assert torch.equal(fp4_linear(x.t().contiguous().t(), codes, scales, bias), want)
    assert fp4_linear(x[:0], codes, scales).shape == (0, 200)
    odd = torch.empty(codes.numel() + 3, device="cuda", dtype=torch.uint8)[3:].view_as(codes).copy_(codes)
    assert torch.equal(fp4_linear(x, odd, scales, bias), want)
    x[3, 100], x[7, 5] = float("nan"), float("inf")        # one row's values are no other row's
    got = fp4_linear(x, codes, scales, bias)
    kept = [i for i in range(12) if i not in (3, 7)]
    assert torch.equal(got[kept], want[kept]) and got[3].isnan().all() and not got[7].isfinite().any()


def nearest_bf16(q: Fraction) -> float:
    """The bf16 nearest to a positive number, ties to even, from whole numbers."""
    e = 0
    while q >= 2 ** (e + 1):
        e += 1
    while q < Fraction(2) ** e:
        e -= 1
    step = Fraction(2) ** (max(e, -126) - 7)
    return float(round(q / step) * step)                   # (round: half to even)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantise(dtype, group):
    g = torch.Generator(device="cuda").manual_seed(group)
    n, k = 40, 512
    w = (torch.randn((n, k), device="cuda", generator=g) * torch.rand((n, 1), device="cuda", generator=g)).to(dtype)
    w[0], w[1] = 0.0, -0.0
    w[2, :group] = torch.linspace(-6, 6, group, device="cuda").to(dtype)
    middles = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], device="cuda")
    w[3, :8], w[3, 8:16], w[3, 16:group] = middles.to(dtype), -middles.to(dtype), 0.0                     # ties, scale 1
    if dtype == torch.float32:
        w[4, :group] = 0.0
        w[4, 3] = 6.0 * (1 + 2.0 ** -8)                                    # the ratio lies between two bf16: to the even one
        w[5, :group] = 0.0
        w[5, 3] = torch.tensor(6.0 * (1 + 2.0 ** -8), device="cuda") * (1 + 2.0 ** -23)      # a last place above: up
        w[6, :group] = 1e-41                                               # subnormal: the scale rounds to zero
        w[7, :group] = 3e38
    codes, scales = quantise_fp4(w, group)
    assert codes.shape == (n, k // 2) and scales.shape == (n, k // group)
    wd = w.double().cpu().reshape(n, k // group, group)
    am = wd.abs().amax(-1)
    for i in range(n):
        for j in range(k // group):
            want = nearest_bf16(Fraction(am[i, j].item()) / 6) if am[i, j] > 0 else 0.0
            assert scales[i, j].item() == want, (i, j, am[i, j].item())
    s = scales.double().cpu().unsqueeze(-1)
    nib = torch.stack((codes & 15, codes >> 4), -1).reshape(n, k // group, group).cpu().long()
    values, ratio = torch.tensor(E2M1, dtype=torch.float64), wd.abs() / torch.where(s == 0, torch.ones_like(s), s)
    mids = (values[1:] + values[:-1]) / 2
    code = torch.zeros_like(nib)
    for c, m in enumerate(mids.tolist()):
        edge = m * s                                                       # exact: 8 bits times 3
        code += ((wd.abs() > edge) | ((wd.abs() == edge) & (c % 2 == 1))) & (s > 0)
    assert torch.equal(nib & 7, code) and torch.equal(nib >> 3, torch.signbit(w).cpu().reshape(nib.shape).long())
    assert bool(((values[nib & 7] * s - wd.abs()).abs() <= s * 1.0 + 6 * s * 2.0 ** -8 + (s == 0) * 1e-40).all()) and ratio.max() < 6.1


def test_quantise_refusals_and_module():
    w = torch.randn(64, 256, device="cuda")
    w[3, 7] = float("nan")
    with pytest.raises(ValueError, match="finite"):
        quantise_fp4(w)
    lin = torch.nn.Linear(256, 96, device="cuda")
    m = FP4Linear.from_linear(lin, 64).eval()
    x = torch.randn(5, 256, device="cuda")
    with torch.no_grad():
        y = m(x)
        assert y.dtype == torch.float32 and m(x.bfloat16()).dtype == torch.bfloat16 and torch.equal(m(x.bfloat16()).float(), y)
        with torch.autocast("cuda", torch.bfloat16):
            assert m(x).dtype == torch.bfloat16
        check(x.bfloat16(), m.codes, m.scales, m.bias)
        whole = FP4Linear(256, 96, group_size=64, device="cuda")
        whole.load_state_dict(m.state_dict())
        assert torch.equal(whole.half().float()(x), y) or whole.bias.dtype == torch.float32     # a cast of the model: the bias alone is rounded
        assert torch.equal(whole.scale_bits, m.scale_bits) and torch.equal(whole.codes, m.codes)
    with pytest.raises(RuntimeError, match="no backward"):
        m(x.requires_grad_(True))


def test_streams_and_captured_products():
    codes, scales, g = weight_of(512, 1024, 32)
    x = torch.randn((4, 1024), device="cuda", generator=g).bfloat16()
    want = fp4_linear(x, codes, scales)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(fp4_linear(x, codes, scales), want)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    held = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            held.append(fp4_linear(x, codes, scales))
    for _ in range(3):
        x.copy_(torch.randn((4, 1024), device="cuda", generator=g).bfloat16())
        for graph in graphs:
            graph.replay()
        eager = fp4_linear(x, codes, scales)
        torch.cuda.synchronize()
        assert torch.equal(held[0], eager) and torch.equal(held[1], eager)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,n,k", [(7, 100, 384), (20, 1030, 8320), (50, 4100, 3200), (130, 1030, 4224), (65, 8200, 4224)])
def test_nan_and_infinity_stay_in_their_rows_and_what_is_behind_k_is_nothing(rows, n, k, group):
    """With codes of zero among the weights an infinity makes infinities and NaN, each where the definition has them; x beyond K, here NaN, is not looked at."""
    codes, scales, g = weight_of(n, k, group, rows)
    wide = torch.full((rows, k + 128), float("nan"), device="cuda", dtype=torch.bfloat16)
    x = wide[:, :k]
    x.copy_(torch.randn((rows, k), device="cuda", generator=g))
    want = check(x, codes, scales)
    x[1, k - 1], x[3, 0], x[rows - 2, k // 2], x[rows - 1, k - 33] = float("inf"), -float("inf"), float("nan"), float("inf")
    got = fp4_linear(x, codes, scales)
    whole = [i for i in range(rows) if i not in (1, 3, rows - 2, rows - 1)]
    assert torch.equal(got[whole], want[whole])
    w = dequantise_fp4(codes, scales)
    for i, at in ((1, k - 1), (3, 0), (rows - 1, k - 33)):
        line = torch.where(w[:, at] == 0, float("nan"), w[:, at] * x[i, at].float())
        assert torch.equal(got[i].isnan(), line.isnan()) and torch.equal(got[i][~line.isnan()].float(), line[~line.isnan()])
    assert got[rows - 2].isnan().all()


def test_captured_products_of_several_runs_on_two_streams():
    """Each capture has a workspace of its own: replayed in turn, and at the same time."""
    rows, n, k = 50, 4100, 3200
    made = []
    for seed in range(2):
        codes, scales, g = weight_of(n, k, 64, seed)
        x = torch.randn((rows, k), device="cuda", generator=g).bfloat16()
        want = check(x, codes, scales)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp4_linear(x, codes, scales)
        made.append((graph, torch.cuda.Stream(), x, codes, scales, want, y))
    for trip in range(4):
        for graph, stream, *_, y in made:
            y.zero_()
        torch.cuda.synchronize()
        for graph, stream, *_ in made:
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [fp4_linear(x, codes, scales) for _, _, x, codes, scales, *_ in made]
        torch.cuda.synchronize()
        for (*_, want, y), e in zip(made, eager):
            assert torch.equal(y, want) and torch.equal(e, want)


@pytest.mark.parametrize("rows,n,k,group", [(70001, 100, 64, 32), (66000, 770, 256, 64), (65537, 300, 1024, 128)])
def test_rows_of_a_long_batch(rows, n, k, group):
    codes, scales, g = weight_of(n, k, group)
    x = torch.randn((rows, k), device="cuda", generator=g).bfloat16()
    check(x, codes, scales, torch.randn(n, device="cuda", generator=g))
