"""The residual stream's step between two blocks against its definition in 64 bits.

Bounds, element by element.  An fp32 operation is off by u = 2^-24 of its result.  A sum over a row goes through at most 16 additions of a lane,
6 of a wave, 7 of a block: 32 u of the sum of magnitudes.  With Y = (|a x| + |g u|) / rms(y), the magnitude behind y / rms(y):
  y   32 u (|a x| + |g u|)                  (half a row sum in 1 / rms(h), some products; then its own rounding)
  z   half a step + 64 u Y |weight|
  E = |dy| + (|t| + Y mean(|t| Y)) / rms(y), the magnitude behind the whole gradient of y; dx 128 u |a| E (+ half a step)
  dh  128 u / rms(h) (|b| E + |hh| mean(|b hh| E)) (+ half a step);  weights 128 u of the sum over rows of their magnitudes
(128: three row sums of 32 u one behind the other, and up to 32 roundings on the way; a column is added up over at most 2 rows a lane here,
then 32 additions of slabs, 16 of groups.)  A half step: 2^-8 for bf16, 2^-24 for fp32."""
import pytest
import torch

from optimus_dl_amd.modules.fused import residual_norm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
BF16, F32 = torch.bfloat16, torch.float32
EPS = 1e-6


def case(rows, cols, stream, branch, post, gate, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s, scale=1.0, shift=0.0: torch.randn(s, device="cuda", generator=g) * scale + shift
    t = {"x": n(rows, cols).to(stream), "h": n(rows, cols, scale=0.3).to(branch), "weight": n(cols, scale=0.1, shift=1.0),
         "post_weight": n(cols, scale=0.1, shift=1.0) if post else None,
         "gate": {"none": None, "scalar": n(1, shift=0.5), "channel": n(cols, scale=0.2, shift=0.5)}[gate]}
    return t, n(rows, cols, scale=1e-2).to(stream), n(rows, cols, scale=1e-2).to(BF16)


def definition(t, dy, dz, a, eps, post_eps):
    """Outputs, gradients and the magnitudes of the bounds, in 64 bits."""
    d = {k: None if v is None else v.detach().double().requires_grad_(True) for k, v in t.items()}
    x, h, wn, wp, g = (d[k] for k in ("x", "h", "weight", "post_weight", "gate"))
    rms = lambda v, e: (v * v).mean(-1, keepdim=True).add(e).sqrt()
    hh = h / rms(h, post_eps) if wp is not None else h
    b = (1.0 if g is None else g) * (1.0 if wp is None else wp) * torch.ones_like(wn)
    y = a * x + b * hh
    z = y / rms(y, eps) * wn
    leaves = {k: v for k, v in d.items() if v is not None}
    pairs = [(o, gr.double()) for o, gr in ((y, dy), (z, dz)) if gr is not None]
    grads = dict(zip(leaves, torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [gr for _, gr in pairs], allow_unused=True)))
    with torch.no_grad():
        big = (a * x).abs() + (b * hh).abs()
        ry, rh = 1 / rms(y, eps), 1 / rms(h, post_eps) if wp is not None else torch.ones_like(h[..., :1])
        Y = big * ry
        t_ = torch.zeros_like(Y) if dz is None else (dz.double() * wn).abs()
        E = (0.0 if dy is None else dy.double().abs()) + ry * (t_ + Y * (t_ * Y).mean(-1, keepdim=True))
        D = (E * hh.abs()).flatten(0, -2).sum(0)
        mag = {"y": big, "z": Y * wn.abs(), "x": abs(a) * E,
               "h": rh * (b.abs() * E + (hh.abs() * ((b * hh).abs() * E).mean(-1, keepdim=True) if wp is not None else 0.0)),
               "weight": (t_ / wn.abs() * Y).flatten(0, -2).sum(0)}
        if wp is not None:
            mag["post_weight"] = D * (1.0 if g is None else g.abs())
        if g is not None:
            dg = D * (1.0 if wp is None else wp.abs())
            mag["gate"] = dg if g.numel() > 1 else dg.sum().reshape(1)
    return y.detach(), z.detach(), grads, mag


def check(got, want, mag, u, what):
    half = HALF[got.dtype]
    off = (got.double() - want).abs() - (half * want.abs() + u * U * mag)
    assert got.shape == want.shape and bool((off <= 1e-30).all()), (what, off.max().item())


def run(t, dy, dz, a=1.0, eps=EPS, post_eps=None, fn=residual_norm):
    live = {k: None if v is None else v.detach().clone().requires_grad_(True) for k, v in t.items()}
    y, z = fn(live["x"], live["h"], live["weight"], eps, post_weight=live["post_weight"], post_eps=post_eps, gate=live["gate"], residual_scale=a,
              out_dtype=BF16)
    pairs = [(o, g) for o, g in ((y, dy), (z, dz)) if g is not None]
    torch.autograd.backward([o for o, _ in pairs], [g for _, g in pairs])
    return y.detach(), z.detach(), {k: v.grad for k, v in live.items() if v is not None}


def check_all(t, dy, dz, a=1.0, eps=EPS, post_eps=None):
    y, z, grads = run(t, dy, dz, a, eps, post_eps)
    wy, wz, wgrads, mag = definition(t, dy, dz, a, eps, eps if post_eps is None else post_eps)
    assert y.dtype == t["x"].dtype and z.dtype == BF16
    check(y, wy, mag["y"], 32, "y")
    check(z, wz, mag["z"], 64, "z")
    for k, w in wgrads.items():
        if w is not None:
            assert grads[k].dtype == t[k].dtype
            check(grads[k], w, mag[k], 128, "d" + k)
    return grads


@pytest.mark.parametrize("post,gate", [(True, "channel"), (True, "none"), (False, "scalar"), (True, "scalar"), (False, "channel"), (False, "none")])
@pytest.mark.parametrize("stream,branch", [(F32, BF16), (BF16, BF16), (F32, F32)])
def test_every_form_and_type(post, gate, stream, branch):
    check_all(*case(37, 1024, stream, branch, post, gate), a=0.5)


# one chunk, both sides of every row width that has a layout of its own, odd numbers of chunks, the widest
@pytest.mark.parametrize("cols", [8, 72, 128, 136, 256, 264, 512, 520, 1000, 1024, 1032, 2048, 2056, 4096, 4104, 8184, 8192])
@pytest.mark.parametrize("rows", [1, 5, 600])
def test_row_widths(rows, cols):
    for stream, branch in ((F32, BF16), (BF16, BF16), (F32, F32)):
        check_all(*case(rows, cols, stream, branch, True, "channel", seed=cols))


def test_many_rows_and_leading_dimensions():
    t, dy, dz = case(2100, 256, F32, BF16, True, "scalar")
    wide = {k: v.reshape(3, 700, 256) if k in ("x", "h") else v for k, v in t.items()}
    y, z, grads = run(wide, dy.reshape(3, 700, 256), dz.reshape(3, 700, 256))
    flat = run(t, dy, dz)
    assert torch.equal(y.reshape(2100, 256), flat[0]) and torch.equal(z.reshape(2100, 256), flat[1])
    assert all(torch.equal(grads[k].reshape(flat[2][k].shape), flat[2][k]) for k in grads)
    again = run(t, dy, dz)
    assert torch.equal(again[2]["weight"], flat[2]["weight"]) and torch.equal(again[2]["gate"], flat[2]["gate"])


def test_gradients_of_one_output_only():
    t, dy, dz = case(19, 768, F32, BF16, True, "channel")
    check_all(t, dy, None)
    check_all(t, None, dz)


def test_two_epsilons_zero_rows_and_a_stream_that_cancels():
    t, dy, dz = case(12, 512, F32, F32, True, "none")
    check_all(t, dy, dz, eps=1e-3, post_eps=1e-2)
    t["x"][3] = 0.0
    t["h"][3] = 0.0                                        # rms of zeros: sqrt(eps)
    check_all(t, dy, dz, eps=1e-3)
    t, dy, dz = case(12, 512, F32, F32, False, "none")
    t["h"] = -t["x"] + 1e-2 * t["h"]                       # y is a hundredth of what it is the sum of: its own squares are summed
    check_all(t, dy, dz)


def test_nan_and_infinity_stay_in_their_rows():
    t, dy, dz = case(9, 1024, F32, BF16, True, "channel")
    clean = run(t, dy, dz)
    t["x"][2, 5], t["h"][6, 7] = float("nan"), float("inf")
    y, z, grads = run(t, dy, dz)
    kept = [i for i in range(9) if i not in (2, 6)]
    assert z[2].isnan().all() and y[6].isnan().any() and z[6].isnan().all()
    assert torch.equal(y[kept], clean[0][kept]) and torch.equal(z[kept], clean[1][kept])
    assert torch.equal(grads["x"][kept], clean[2]["x"][kept]) and torch.equal(grads["h"][kept], clean[2]["h"][kept])


def test_strides_offsets_and_broadcast_gradients():
    t, dy, dz = case(16, 512, F32, BF16, True, "channel")
    want = run(t, dy, dz)
    odd = dict(t)
    odd["x"] = torch.cat([t["x"], t["x"]], 1)[:, :512]                                  # rows apart
    odd["h"] = torch.cat([t["h"].new_zeros(3), t["h"].flatten()])[3:].view(16, 512)     # off the 16-byte grid
    odd["weight"] = torch.stack([t["weight"], t["weight"]], 1)[:, 0]
    for fn in (residual_norm,):
        x, h, w = (odd[k].requires_grad_(True) for k in ("x", "h", "weight"))
        y, z = fn(x, h, w, EPS, post_weight=t["post_weight"], gate=t["gate"], out_dtype=BF16)
        gx, gh, gw = torch.autograd.grad((y, z), (x, h, w), (dy.t().contiguous().t(), dz))
        assert torch.equal(y, want[0]) and torch.equal(z, want[1])
        assert torch.equal(gx, want[2]["x"]) and torch.equal(gh, want[2]["h"]) and torch.equal(gw, want[2]["weight"])
    x = t["x"].clone().requires_grad_(True)
    y, z = residual_norm(x, t["h"], t["weight"], EPS, out_dtype=BF16)
    (y.sum() + z.float().sum()).backward()                                              # gradients of stride 0
    _, _, grads, mag = definition({**t, "post_weight": None, "gate": None}, torch.ones_like(dy), torch.ones_like(dz), 1.0, EPS, EPS)
    check(x.grad, grads["x"], mag["x"], 128, "dx")


def test_parts_are_the_maxima_and_weights_in_bf16_get_their_gradients():
    from optimus_dl_amd import native as N

    for stream, branch in ((F32, BF16), (BF16, BF16), (F32, F32)):
        for rows in (1, 700):
            t, dy, dz = case(rows, 1024, stream, branch, True, "channel")
            y, z, stats, parts = N.residual_norm(t["x"], t["h"], t["weight"], EPS, t["post_weight"], None, t["gate"], 1.0)
            assert parts.shape == (N.AMAX_PARTS,) and parts.max().item() == z.float().abs().max().item()
            bare = N.residual_norm(t["x"], t["h"], t["weight"], EPS, t["post_weight"], None, t["gate"], 1.0, keep=False)
            assert torch.equal(bare[0], y) and torch.equal(bare[1], z) and bare[2:] == (None, None)
            dx, dh, parts, dw, dpost, dgate = N.residual_norm_bwd(dy, dz, t["x"], t["h"], t["weight"], t["post_weight"], t["gate"], 1.0, stats)
            assert parts.max().item() == dh.float().abs().max().item()
            frozen = N.residual_norm_bwd(dy, dz, t["x"], t["h"], t["weight"], t["post_weight"], t["gate"], 1.0, stats, want_weights=False)
            assert torch.equal(frozen[0], dx) and torch.equal(frozen[1], dh) and frozen[3:] == (None, None, None)
    t, dy, dz = case(33, 512, BF16, BF16, True, "scalar")
    t = {k: v.bfloat16() for k, v in t.items()}
    check_all(t, dy, dz)


def test_no_gradient_asked_for_none_computed():
    t, dy, dz = case(4, 64, F32, BF16, True, "channel")
    with torch.no_grad():
        y, z = residual_norm(t["x"], t["h"], t["weight"], EPS, post_weight=t["post_weight"], gate=t["gate"], out_dtype=BF16)
    assert y.grad_fn is None and z.grad_fn is None
    h = t["h"].clone().requires_grad_(True)
    y, z = residual_norm(t["x"], h, t["weight"], EPS, out_dtype=BF16)
    z.backward(dz)
    assert h.grad is not None
    (g,) = torch.autograd.grad(residual_norm(t["x"], h, t["weight"], EPS, out_dtype=BF16)[0].sum(), h, create_graph=True)
    with pytest.raises(RuntimeError):                      # once differentiable: says so, where a constant would be wrong
        g.sum().backward()


def test_another_stream_and_a_captured_step():
    t, dy, dz = case(64, 1024, F32, BF16, True, "channel")
    want = run(t, dy, dz)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(t, dy, dz)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2]["h"], want[2]["h"])

    from optimus_dl_amd import native as N

    def step():
        y, z, stats, parts = N.residual_norm(t["x"], t["h"], t["weight"], EPS, t["post_weight"], None, t["gate"], 1.0)
        return y, z, parts, *N.residual_norm_bwd(dy, dz, t["x"], t["h"], t["weight"], t["post_weight"], t["gate"], 1.0, stats)

    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.cuda.graph(other):
        held2 = step()
    for seed in (5, 6, 7):
        new, ndy, ndz = case(64, 1024, F32, BF16, True, "channel", seed)
        for k in t:
            t[k].copy_(new[k])
        dy.copy_(ndy), dz.copy_(ndz)
        graph.replay()
        other.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager)) and all(torch.equal(a, b) for a, b in zip(held2, eager))


def test_calls_that_the_kernels_do_not_take_run_as_torch_operations():
    t, dy, dz = case(6, 1024, F32, F32, True, "channel")
    y, z = residual_norm(t["x"], t["h"], t["weight"], EPS, post_weight=t["post_weight"], gate=t["gate"])
    assert z.dtype == F32                                  # no recipe, no autocast: the type of the stream
    wy, wz, _, mag = definition(t, dy, dz, 1.0, EPS, EPS)
    check(y, wy, mag["y"], 64 * 32, "y")                   # (torch's order of a row sum: 1024 additions at most, 32 times 32)
    check(z, wz, mag["z"], 64 * 64, "z")
    with torch.autocast("cuda", torch.bfloat16):
        assert residual_norm(t["x"], t["h"], t["weight"], EPS)[1].dtype == BF16
    odd = t["x"][:, :1003].contiguous(), t["h"][:, :1003].contiguous(), t["weight"][:1003].contiguous()
    assert residual_norm(*odd, EPS, out_dtype=BF16)[1].shape == (6, 1003)
    empty = residual_norm(t["x"][:0], t["h"][:0], t["weight"], EPS, out_dtype=BF16)
    assert empty[0].shape == (0, 1024) and empty[1].dtype == BF16
