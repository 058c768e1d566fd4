"""Layer norm forward and backward against the definition in 64 bits (bounds: tests/train_ref.py)."""
import pytest
import torch

import train_ref as R
from diffphore_amd import layers

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}


def _inputs(rows, width, dtype, wdtype, seed=0, affine=True):
    g = torch.Generator().manual_seed(seed + rows * 31 + width)
    x = (torch.randn(rows, width, generator=g) * 2 + 0.5).to(dtype).cuda()
    dy = torch.randn(rows, width, generator=g).to(dtype).cuda()
    w = (torch.randn(width, generator=g) * 0.3 + 1).to(wdtype).cuda() if affine else None
    b = torch.randn(width, generator=g).to(wdtype).cuda() if affine else None
    return x, dy, w, b


def _check(x, dy, w, b, eps=1e-5):
    width = x.shape[-1]
    (y, by), (m, bm), (r, br) = R.layer_norm(x, w, b, eps, x.dtype)
    gy, gm, gr = layers.layer_norm_forward(x, w, b, eps)
    R.within(gy, y, by, "y")
    R.within(gm, m.reshape(-1), bm.reshape(-1), "mean")
    R.within(gr, r.reshape(-1), br.reshape(-1), "rstd")
    wtype = w.dtype if w is not None else x.dtype
    (dx, bdx), (dw, bdw), (db, bdb) = R.layer_norm_backward(dy, x, w, eps, x.dtype, wtype)
    gx, gw, gb = layers.layer_norm_backward(dy, x, gm, gr, w)
    assert gx.dtype == x.dtype and gw.dtype == gb.dtype == wtype and gw.shape == (width,)
    R.within(gx, dx, bdx, "dx")
    R.within(gw, dw, bdw, "dweight")
    R.within(gb, db, bdb, "dbias")


# widths around every change of lanes per row; rows from one to several per group; odd widths (no 16-byte rows)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows, width", [(1, 1), (3, 2), (5, 3), (800, 20), (1, 32), (33, 33), (257, 60), (17, 64), (19, 65), (4, 256), (9, 257), (130, 1000),
                                         (5, 1024), (6, 1025), (700, 2048), (3, 4096), (2, 4097), (5, 8192), (3, 8193), (2, 16383), (4, 16384), (5000, 40)])
def test_matches_the_definition(rows, width, dtype):
    x, dy, w, b = _inputs(rows, width, T[dtype], T[dtype])
    _check(x, dy, w, b)


@pytest.mark.parametrize("width", [24, 60, 520])
def test_bf16_rows_with_fp32_parameters_and_without_parameters(width):
    x, dy, w, b = _inputs(70, width, torch.bfloat16, torch.float32)
    _check(x, dy, w, b)
    x, dy, w, b = _inputs(70, width, torch.bfloat16, torch.bfloat16, affine=False)
    _check(x, dy, None, None)
    y1, _, _ = layers.layer_norm_forward(x, None, torch.ones(width, device="cuda"))
    y0, _, _ = layers.layer_norm_forward(x.float())
    assert torch.equal(y1, (y0 + 1).bfloat16())


def test_rows_close_together_and_far_from_zero():
    """entries that differ in their last bits only: the mean's own rounding must not show"""
    g = torch.Generator().manual_seed(1)
    x = (1000.0 + torch.randn(64, 48, generator=g) * 1e-3).cuda()
    dy = torch.randn(64, 48, generator=g).cuda()
    _check(x, dy, None, None, eps=1e-12)
    x = torch.full((5, 48), 3.7).cuda()                      # constant rows: y = bias exactly
    y, m, r = layers.layer_norm_forward(x, torch.ones(48).cuda(), torch.full((48,), 0.25).cuda())
    assert torch.equal(y, torch.full_like(y, 0.25)) and torch.allclose(r, torch.full_like(r, 1e-5 ** -0.5))


def test_strided_and_expanded_rows_and_leading_dimensions():
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(40, 3, 100, generator=g).cuda()
    x, dy = wide[:, 1, 3:67], torch.randn(1, 64, generator=g).cuda().expand(40, 64)          # misaligned rows, one gradient row for all
    assert not x.is_contiguous()
    w = torch.randn(64, generator=g).cuda()
    _check(x, dy, w, w)
    x4 = torch.randn(2, 3, 4, 64, generator=g).cuda()
    y, m, _ = layers.layer_norm_forward(x4, w, w)
    y2, _, _ = layers.layer_norm_forward(x4.reshape(24, 64), w, w)
    assert y.shape == x4.shape and m.shape == (24,) and torch.equal(y.reshape(24, 64), y2)
    yt, _, _ = layers.layer_norm_forward(x4.reshape(24, 64).t().contiguous().t(), w, w)      # unit stride along the rows: copied
    assert torch.equal(yt, y2)


def test_nonfinite_rows_stay_alone():
    x, dy, w, b = _inputs(9, 80, torch.float32, torch.float32)
    clean, _, _ = layers.layer_norm_forward(x, w, b)
    x[3, 7], x[5, 2] = float("nan"), float("inf")
    y, m, r = layers.layer_norm_forward(x, w, b)
    keep = [0, 1, 2, 4, 6, 7, 8]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[3]).all() and torch.isnan(y[5]).any()
    dx, _, _ = layers.layer_norm_backward(dy, x, m, r, w)
    assert torch.isfinite(dx[keep]).all()


def test_no_rows():
    w = torch.ones(12, device="cuda")
    y, m, r = layers.layer_norm_forward(torch.empty(0, 12, device="cuda"), w, w)
    assert y.shape == (0, 12) and m.numel() == r.numel() == 0
    dx, dw, db = layers.layer_norm_backward(y, y, m, r, w)
    assert dx.shape == (0, 12) and not dw.any() and not db.any()


def test_same_bits_every_time_and_on_another_stream():
    x, dy, w, b = _inputs(5000, 200, torch.bfloat16, torch.bfloat16)
    _, m, r = layers.layer_norm_forward(x, w, b)
    ref = layers.layer_norm_backward(dy, x, m, r, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = layers.layer_norm_backward(dy, x, m, r, w)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, c) for a, c in zip(ref, other))


def test_autograd():
    x, dy, w, b = _inputs(50, 36, torch.float32, torch.float32)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    layers.layer_norm(x, w, b).backward(dy)
    (dx, bdx), (dw, bdw), (db, bdb) = R.layer_norm_backward(dy, x.detach(), w.detach(), 1e-5, torch.float32, torch.float32)
    for t, ref, bound in ((x, dx, bdx), (w, dw, bdw), (b, db, bdb)):
        R.within(t.grad, ref, bound, "grad")
    xs = x.detach().clone().requires_grad_()
    layers.layer_norm(xs).sum().backward()                   # an expanded gradient, no parameters
    assert xs.grad.abs().max() < 1e-4 and w.grad is not None
    x2 = x.detach().requires_grad_()
    (g,) = torch.autograd.grad(layers.layer_norm(x2, w.detach()), x2, dy, create_graph=False)
    R.within(g, dx, bdx, "grad of x alone")


def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    for bad in (x.half(), x.double(), torch.zeros(4, 0, device="cuda"), torch.zeros((), device="cuda"), torch.zeros(1, 16385, device="cuda")):
        with pytest.raises((TypeError, ValueError)):
            layers.layer_norm_forward(bad)
    for kw in (dict(weight=torch.zeros(7, device="cuda")), dict(weight=torch.zeros(8)), dict(weight=torch.zeros(8, device="cuda").bfloat16()),
               dict(weight=torch.zeros(16, device="cuda")[::2]), dict(eps=-1.0), dict(eps=float("nan")),
               dict(weight=torch.zeros(8, device="cuda"), bias=torch.zeros(8, device="cuda").bfloat16())):
        with pytest.raises((TypeError, ValueError)):
            layers.layer_norm_forward(x, **kw)
    y, m, r = layers.layer_norm_forward(x)
    for args in ((y[:3], x, m, r), (y.bfloat16(), x, m, r), (y, x, m[:3], r), (y, x, m.double(), r)):
        with pytest.raises((TypeError, ValueError)):
            layers.layer_norm_backward(*args)
    with pytest.raises(TypeError):
        layers.layer_norm_backward(y, x, m, r, param_dtype=torch.bfloat16)
