"""Products with 4-bit weights in the forms that a few rows of a long K take, and a module after a cast of the whole model.

Bound: half a step of bf16 (2^-8), and 2^-24 of the sum of |x| |w| for every addition on the longest way.  Groups of 32: a wave of the thin kernel adds K / 32 / 8
groups one behind the other, the eight or sixteen waves then, and the 32 products inside of an instruction before; the wide one K / 32 / 2 over its runs, 24 to 32 of
which are added up behind.  K / 256 + 96 is no less for any of them: K / 256 + 8 + 32 with eight waves, K / 512 + 16 + 32 with sixteen, and K / 64 / runs + 32 + 1 + runs with
24 or 32 runs.  Groups of 64 and 128 add half and a quarter as often."""
import pytest
import torch

from optimus_dl_amd.modules.fp4_linear import FP4Linear, dequantise_fp4, fp4_linear

pytestmark = pytest.mark.gpu


def check(rows, n, k, group, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=g, dtype=torch.int64).to(torch.uint8)
    scales = (torch.rand((n, k // group), device="cuda", generator=g) * 0.02 + 1e-3).bfloat16()
    # rows of x apart, with what must not be looked at between them; columns and rows of codes are left to the allocator's neighbours
    wide = torch.full((rows, k + 256), float("nan"), device="cuda", dtype=torch.bfloat16)
    x = wide[:, :k]
    x.copy_(torch.randn((rows, k), device="cuda", generator=g))
    bias = torch.randn(n, device="cuda", generator=g)
    got = fp4_linear(x, codes, scales, bias)
    w = dequantise_fp4(codes, scales).double()
    want, mag = x.double() @ w.t() + bias.double(), x.double().abs() @ w.abs().t() + bias.double().abs()
    off = (got.double() - want).abs() - 2.0 ** -8 * want.abs() - 2.0 ** -24 * (k / 256 + 96) * mag
    assert bool((off <= 0).all()), off.max().item()
    assert torch.equal(got, fp4_linear(x, codes, scales, bias))
    alone = fp4_linear(x.contiguous(), codes, scales, bias)
    assert torch.equal(got, alone)


# x from memory: more than LDS holds beside the scales.  K ends inside of a chunk, columns inside of a block.
@pytest.mark.parametrize("n", [1000, 4100])
@pytest.mark.parametrize("rows,k,group", [(16, 5152, 32), (16, 5184, 64), (16, 5248, 128), (11, 7200, 32), (11, 7232, 64), (11, 7296, 128)])
def test_up_to_16_rows_from_memory(rows, n, k, group):
    check(rows, n, k, group)


# x through LDS, up to 150 KB of it, eight waves and (K of 8192 and more) sixteen
@pytest.mark.parametrize("n", [100, 1030])
@pytest.mark.parametrize("rows,k,group", [(16, 2048, 64), (16, 4128, 32), (16, 4160, 64), (16, 4224, 128), (13, 5088, 32), (2, 8352, 32), (7, 8256, 64), (5, 9344, 128),
                                          (4, 14336, 32), (4, 14400, 64), (4, 14464, 128), (1, 16512, 128)])
def test_up_to_16_rows_through_lds(rows, n, k, group):
    check(rows, n, k, group)


# K in many runs of the wide kernel, from 65 568 inputs on (groups of 32) however few the rows: scales of whole rows do not fit into LDS
@pytest.mark.parametrize("rows,n,k,group", [(1, 100, 28736, 64), (1, 40, 65568, 32), (3, 40, 67616, 32), (2, 300, 131392, 64), (1, 17, 262528, 128), (5, 40, 262528, 128), (20, 40, 67616, 32)])
def test_a_few_rows_of_a_very_long_k(rows, n, k, group):
    check(rows, n, k, group)


@pytest.mark.parametrize("n,k,group", [(3001, 32800, 32), (4099, 41024, 64)])
def test_one_row_of_a_long_k_and_many_columns(n, k, group):
    check(1, n, k, group)


def test_a_module_after_a_cast_of_the_model_rounds_its_bias_alone():
    lin = torch.nn.Linear(256, 96, device="cuda")
    m = FP4Linear.from_linear(lin, 64).eval()
    bits, x = m.scale_bits.clone(), torch.randn(5, 256, device="cuda")
    with torch.no_grad():
        for cast in (torch.float16, torch.bfloat16):
            whole = FP4Linear(256, 96, group_size=64, device="cuda")
            whole.load_state_dict(m.state_dict())
            whole.to(cast).float()
            bias = lin.bias.to(cast).float()
            assert torch.equal(whole.bias, bias) and torch.equal(whole.scale_bits, bits) and torch.equal(whole.codes, m.codes)
            assert torch.equal(whole(x), fp4_linear(x.bfloat16(), m.codes, m.scales, bias).float())
            half = whole.to(torch.bfloat16)
            assert half.bias.dtype == torch.bfloat16 and torch.equal(half(x.bfloat16()), fp4_linear(x.bfloat16(), m.codes, m.scales, half.bias))
