"""AdamW over many tensors against the formula in 64 bits (bounds: tests/train_ref.py); 8-bit codes have to be the nearest ones exactly."""
import pytest
import torch

import train_ref as R
from diffphore_amd import optim

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZES = [(3,), (256,), (0,), (20, 20), (1,), (7, 61), (513,), (1000, 40)]
LR, B1, B2, EPS, WD, D = 1e-2, 0.9, 0.99, 1e-8, 0.1, 0.95


def _setup(dtype, bits, ema, grad_dtype=None, sizes=SIZES, seed=0, **kw):
    g = torch.Generator().manual_seed(seed)
    params = [torch.randn(s, generator=g).to(T[dtype]).cuda() for s in sizes]
    opt = optim.AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, no_decay=[0, 4], state_bits=bits, ema_decay=D if ema else None, **kw)

    def grads(scale=1.0):
        return [(torch.randn(s, generator=g) * scale * 10.0 ** (i % 4 - 2)).to(grad_dtype or T[dtype]).cuda() for i, s in enumerate(sizes)]
    return params, opt, grads


def _cut(opt, flat):
    return [x.detach().double().cpu().reshape(-1) for x in opt.views(flat)]


@pytest.mark.parametrize("ema", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype, grad_dtype", [("f32", None), ("bf16", None), ("bf16", torch.float32)])
def test_steps_match_the_formula(dtype, grad_dtype, bits, ema):
    params, opt, grads = _setup(dtype, bits, ema, grad_dtype)
    for t in range(1, 5):
        before = [x.double().cpu().reshape(-1) for x in (opt.views(opt.master) if dtype == "bf16" else [p.clone() for p in params])]
        m0, v0 = (_cut(opt, f.clone()) for f in opt.moments())
        codes0 = (opt.exp_avg.cpu(), opt.exp_avg_scale.cpu(), opt.exp_avg_sq.cpu(), opt.exp_avg_sq_scale.cpu()) if bits == 8 else None
        e0 = _cut(opt, opt.ema.clone()) if ema else None
        if bits == 8:                            # what the codes stand for, in 64 bits
            exact = [R.decode(codes0[0], codes0[1], 2), R.decode(codes0[2], codes0[3], 4)]
            m0, v0 = ([f[b * 256:b * 256 + n] for b, n in zip(opt.first_block, opt._numel)] for f in exact)
        gs = grads()
        opt.step(gs)
        m1, v1 = (_cut(opt, f) for f in opt.moments())
        for i, p in enumerate(params):
            g = gs[i].double().cpu().reshape(-1)
            (pr, bp), (mr, bm), (vr, bv) = R.adamw(before[i], g, m0[i], v0[i], t, LR, B1, B2, EPS, 0.0 if i in (0, 4) else WD)
            new = (opt.views(opt.master)[i] if dtype == "bf16" else p).double().cpu().reshape(-1)
            R.within(new, pr, bp, f"p{i} step {t}")
            if dtype == "bf16":
                assert torch.equal(p.reshape(-1), opt.views(opt.master)[i].bfloat16().reshape(-1))
            if ema:
                R.within(opt.views(opt.ema)[i].reshape(-1), D * e0[i] + (1 - D) * new, 4 * R.F32 * (e0[i].abs() + new.abs()), "ema")
            if bits == 32:
                R.within(m1[i], mr, bm, "m")
                R.within(v1[i], vr, bv, "v")
            else:
                pad = -len(mr) % 256
                for x, power, code, scale in ((mr, 2, opt.exp_avg, opt.exp_avg_scale), (vr, 4, opt.exp_avg_sq, opt.exp_avg_sq_scale)):
                    if not len(x):
                        continue
                    c, s = R.encode(torch.nn.functional.pad(x, (0, pad)), power)
                    lo, hi = opt.first_block[i], opt.first_block[i + 1]
                    assert torch.equal(code[lo * 256:hi * 256].cpu(), c), f"codes of power {power}, tensor {i}, step {t}"
                    # the scale is the 64-bit maximum rounded once: an ulp where the kernel's 64-bit sum differs in its last bit
                    assert torch.allclose(scale[lo:hi].cpu(), s, rtol=2.0 ** -23, atol=0)
    assert opt.state_dict()["step"] == 4


def test_many_tensors_take_several_launches():
    sizes = [(i % 5 + 1,) for i in range(900)]
    params, opt, grads = _setup("f32", 32, True, sizes=sizes)
    one, opt1, grads1 = _setup("f32", 32, True, sizes=sizes)
    gs = grads()
    flat = torch.cat([g.reshape(-1) for g in gs])
    opt.step(gs)
    single = optim.AdamW([torch.cat([p.reshape(-1) for p in one])], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=0.0)
    single.step([flat])
    no_wd = optim.AdamW(one, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=0.0)
    no_wd.step(gs)
    assert torch.equal(torch.cat([p.reshape(-1) for p in one]), single.params[0])
    assert opt.state_dict()["step"] == no_wd.state_dict()["step"] == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_views_at_odd_addresses_and_padding(bits):
    """parameters and gradients that start off a 16-byte border; nothing beside them is written; the padding of the state stays 0"""
    base = torch.randn(4000, device="cuda")
    gbase = torch.randn(4000, device="cuda")
    cuts = [(1, 1000), (1003, 259), (1263, 512), (1777, 2000)]
    copy = base.clone()
    params = [base[a:a + n] for a, n in cuts]
    plain = [copy[a:a + n].clone() for a, n in cuts]
    opt, ref = (optim.AdamW(p, lr=LR, betas=(B1, B2), weight_decay=WD, state_bits=bits) for p in (params, plain))
    for _ in range(3):
        gbase = torch.randn(4000, device="cuda")
        opt.step([gbase[a:a + n] for a, n in cuts])
        ref.step([gbase[a:a + n].clone() for a, n in cuts])
    assert all(torch.equal(p, r) for p, r in zip(params, plain))
    inside = torch.zeros(4000, dtype=torch.bool)
    for a, n in cuts:
        inside[a:a + n] = True
    assert torch.equal(base.cpu()[~inside], copy.cpu()[~inside])
    m, v = opt.moments()
    for a, b, n in zip(opt.first_block, opt.first_block[1:], opt._numel):
        assert not m[a * 256 + n:b * 256].any() and not v[a * 256 + n:b * 256].any()


def test_none_gradients_grad_scale_lr_and_dicts():
    p = {"a": torch.ones(300, device="cuda"), "b": torch.ones(5, device="cuda"), "c": torch.ones(2, 2, device="cuda")}
    opt = optim.AdamW(p, lr=0.5, weight_decay=0.0, no_decay=["b"], ema_decay=0.0)
    opt.step({"a": torch.full((300,), 2.0, device="cuda"), "c": torch.ones(2, 2, device="cuda")}, lr=torch.tensor(0.25, device="cuda"),
             grad_scale=torch.tensor(0.5, device="cuda"))
    assert torch.equal(p["b"], torch.ones(5, device="cuda")) and not opt.views(opt.exp_avg)["b"].any()
    # the first step moves every entry by lr (m / c1) / sqrt(v / c2) = lr
    assert torch.allclose(p["a"], torch.full_like(p["a"], 0.75), atol=1e-5) and torch.allclose(p["c"], torch.full_like(p["c"], 0.75), atol=1e-5)
    assert torch.allclose(opt.views(opt.exp_avg)["a"], torch.full((300,), 0.1, device="cuda"))
    assert torch.equal(opt.ema_parameters()["a"], p["a"])
    for q in p.values():
        q.requires_grad_()
    (p["a"].sum() * 3).backward()
    opt.step()                                   # .grad, and None for the others
    opt.zero_grad()
    assert p["a"].grad is None and opt.state_dict()["step"] == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(bits):
    params, opt, grads = _setup("bf16", bits, True)
    for _ in range(3):
        opt.step(grads())
    clones = [p.clone() for p in params]
    again = optim.AdamW(clones, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, no_decay=[0, 4], state_bits=bits, ema_decay=D)
    again.load_state_dict(opt.state_dict())
    g = grads()
    opt.step(g)
    again.step(g)
    assert all(torch.equal(a, b) for a, b in zip(params, clones)) and torch.equal(opt.exp_avg, again.exp_avg) and torch.equal(opt.ema, again.ema)
    wrong = optim.AdamW(clones, state_bits=40 - bits, ema_decay=D)
    with pytest.raises(ValueError):
        wrong.load_state_dict(opt.state_dict())
    with pytest.raises(ValueError):
        optim.AdamW(clones, state_bits=bits).load_state_dict(opt.state_dict())


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite_and_extreme_sizes(bits):
    p = torch.ones(1024, device="cuda")
    opt = optim.AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=bits)
    g = torch.zeros(1024, device="cuda")
    g[300], g[600] = float("nan"), 1e-30
    g[700:720] = torch.logspace(-18, 15, 20, device="cuda")
    opt.step([g])
    m, v = opt.moments()
    bad = torch.isnan(p)
    assert bad[300] and bad.sum() == 1
    where = torch.zeros(1024, dtype=torch.bool, device="cuda")
    where[300 if bits == 32 else slice(256, 512)] = True
    assert torch.equal(torch.isnan(m), where) and torch.equal(torch.isnan(v), where)
    if bits == 8:
        assert opt.exp_avg_sq[700:720].min() >= 1                       # never 0 for a positive second moment
    opt.step([torch.zeros(1024, device="cuda")])
    assert torch.isnan(p[256:512]).any() and torch.isfinite(p[512:]).all() and torch.isfinite(p[:256]).all()


def test_eight_bits_move_parameters_as_32_do():
    """400 steps on a quadratic from one start: the 8-bit run stays within a tenth of the way that the parameters travel"""
    g = torch.Generator().manual_seed(2)
    start, goal = torch.randn(2000, generator=g).cuda(), torch.randn(2000, generator=g).cuda()
    ends = []
    for bits in (32, 8):
        p = start.clone()
        opt = optim.AdamW([p], lr=3e-3, weight_decay=0.0, state_bits=bits)
        for _ in range(400):
            opt.step([p - goal])
        ends.append(p)
    assert (ends[0] - ends[1]).norm() < 0.1 * (ends[0] - start).norm()


def test_refusals():
    a = torch.ones(8, device="cuda")
    for params in ([a.half()], [a, a.bfloat16()], [a, a], [a, a[4:]], [torch.ones(4, 4, device="cuda").t()], [a.cpu()], []):
        with pytest.raises((TypeError, ValueError)):
            optim.AdamW(params)
    for kw in (dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)), dict(weight_decay=-1.0), dict(state_bits=16), dict(ema_decay=1.5), dict(no_decay=[1]),
               dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            optim.AdamW([a], **kw)
    opt = optim.AdamW([a])
    for g in ([], [a, a], [a.half()], [a.bfloat16()], [a[:4]], [torch.ones(16, device="cuda")[::2]], [a.cpu()], {"x": a}):
        with pytest.raises((TypeError, ValueError)):
            opt.step(g)
    for kw in (dict(lr=torch.tensor(0.1)), dict(lr=torch.ones(2, device="cuda")), dict(grad_scale=torch.ones(1, device="cuda").double())):
        with pytest.raises(ValueError):
            opt.step([torch.zeros(8, device="cuda")], **kw)
    with pytest.raises(ValueError):
        opt.ema_parameters()
    assert torch.equal(a, torch.ones(8, device="cuda"))


def test_loading_bf16_state_refreshes_the_parameters():
    params, opt, grads = _setup("bf16", 32, False)
    opt.step(grads())
    saved = opt.state_dict()
    want = [p.clone() for p in params]
    opt.step(grads())
    opt.load_state_dict(saved)
    assert all(torch.equal(p, w) for p, w in zip(params, want)) and opt.state_dict()["step"] == 1
    with pytest.raises(TypeError):
        opt.step([1.0] * len(params))
    with pytest.raises(ValueError):
        opt.load_state_dict({**saved, "step": -1})


def test_parameters_pointed_elsewhere_are_not_written_through():
    """the optimiser writes to the memory that the tensors had, which it keeps alive"""
    p = torch.ones(300, device="cuda")
    old = p.data
    opt = optim.AdamW([p], lr=0.1)
    p.data = torch.zeros(300, device="cuda")
    opt.step([torch.ones(300, device="cuda")])
    assert not p.any() and (old < 1).all()


def test_small_and_absent_eps_with_moments_next_to_underflow():
    """sqrt(v) of second moments below 2^-126 still counts when eps does not cover it"""
    p = torch.zeros(6, device="cuda")
    opt = optim.AdamW([p], lr=1.0, betas=(0.0, 0.5), eps=0.0, weight_decay=0.0)
    opt.step([torch.tensor([1e-15, 1e-18, 3e-20, 1e3, 1e15, -1e-18], device="cuda")])
    # m / sqrt(v / (1 - b2)) = 1; 9e-40 / 2 in fp32 has 18 bits left
    assert torch.allclose(p.cpu(), torch.tensor([-1.0, -1, -1, -1, -1, 1]), rtol=1e-5)


def test_scales_of_blocks_whose_largest_moment_is_a_tie():
    """b1 = 0.9 and bf16 gradients: the largest new moment of a block is often exactly between two 32-bit numbers.  Its rounding is that of the formula evaluated
    operation by operation in 64 bits - and so is every code of every block, over a million of them"""
    g = torch.Generator().manual_seed(12)
    n = 1 << 20
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    opt = optim.AdamW([p], lr=1e-3, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8)
    for step in range(3):
        mc, ms, vc, vs = (t.cpu() for t in (opt.exp_avg, opt.exp_avg_scale, opt.exp_avg_sq, opt.exp_avg_sq_scale))
        grad = (torch.randn(n, generator=g) * 1e-3).bfloat16()
        opt.step([grad.cuda()])
        x, c, u = grad.double(), mc.double(), vc.double() / 255.0
        u = u * u
        m = c * c.abs() / 127.0 ** 2 * ms.double().repeat_interleave(256) * 0.9 + x * (1.0 - 0.9)
        v = u * u * vs.double().repeat_interleave(256) * 0.999 + x * x * (1.0 - 0.999)
        for val, power, code, scale in ((m, 2, opt.exp_avg, opt.exp_avg_scale), (v, 4, opt.exp_avg_sq, opt.exp_avg_sq_scale)):
            want, s = R.encode(val, power)
            assert torch.equal(scale.cpu(), s), (step, power, "scales")
            assert torch.equal(code.cpu(), want), (step, power, "codes")


@pytest.mark.parametrize("bits", [32, 8])
def test_lists_of_empty_tensors(bits):
    """nothing but empty tensors, and a launch of the list whose tensors are all empty: the step counts, nothing is read"""
    empty = optim.AdamW([torch.empty(0, 3, device="cuda")], state_bits=bits, ema_decay=0.9)
    empty.step([torch.empty(0, 3, device="cuda")])
    assert empty.state_dict()["step"] == 1
    params = [torch.ones(7, device="cuda")] + [torch.empty(0, device="cuda") for _ in range(900)]
    opt = optim.AdamW(params, lr=0.5, weight_decay=0.0, state_bits=bits)
    opt.step([torch.ones_like(p) for p in params])
    opt.step([torch.ones_like(p) for p in params])
    assert opt.state_dict()["step"] == 2 and torch.allclose(params[0], torch.zeros(7, device="cuda"), atol=0.02)


def test_a_transposed_gradient_is_refused():
    p = [torch.zeros(4, 6, device="cuda"), torch.zeros(5, device="cuda")]
    opt = optim.AdamW(p)
    for bad in ([torch.ones(6, 4, device="cuda"), torch.ones(5, device="cuda")], [torch.ones(6, 4, device="cuda"), None], [torch.ones(4, 6, device="cuda"), torch.ones(4, device="cuda")]):
        with pytest.raises(ValueError):
            opt.step(bad)
    assert not p[0].any() and not p[1].any() and opt.state_dict()["step"] == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_an_optimiser_dropped_while_another_stream_still_works(bits):
    """its state and records are its own memory: what is allocated after it is gone is not written over"""
    params, opt, grads = _setup("bf16", bits, True)
    again, opt2, _ = _setup("bf16", bits, True)
    gs = grads()
    opt.step(gs)
    sizes = [t.numel() * t.element_size() for t in (opt._blocks, opt._counter, *(getattr(opt, n) for n in opt._STATE)) if t is not None]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        opt2.step(gs)
    del opt2
    junk = [torch.zeros(n, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(params, again)) and not any(j.any() for j in junk)


def test_settings_that_the_launches_hold_cannot_be_set():
    """a setting or a state buffer put in place of the optimiser's own would be ignored (or leave the launches with the address of freed memory); lr is used"""
    opt = optim.AdamW([torch.zeros(8, device="cuda")], lr=0.5, weight_decay=0.0, ema_decay=0.5)
    for name in ("betas", "eps", "weight_decay", "ema_decay", "state_bits", "master", "ema", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
        with pytest.raises(AttributeError):
            setattr(opt, name, torch.zeros(256, device="cuda"))
    assert opt.betas == (0.9, 0.999) and opt.eps == 1e-8 and opt.weight_decay == 0.0 and opt.ema_decay == 0.5 and opt.state_bits == 32 and opt.master is None
    for lr in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            opt.lr = lr
        with pytest.raises(ValueError):
            opt.step([torch.ones(8, device="cuda")], lr=lr)
    assert opt.lr == 0.5 and not opt.params[0].any() and opt.state_dict()["step"] == 0
    opt.lr = 0.25
    opt.step([torch.ones(8, device="cuda")])
    assert torch.allclose(opt.params[0], torch.full((8,), -0.25, device="cuda"), rtol=1e-5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_backward_pass_over_changed_parameters_raises(dtype):
    """a step is an in-place change that autograd sees: old activations and new weights do not meet.  A parameter without a gradient is not changed"""
    from diffphore_amd import layers
    w, b = (torch.ones(8, dtype=T[dtype], device="cuda").requires_grad_() for _ in range(2))
    x = torch.arange(24.0, device="cuda").view(3, 8).to(T[dtype])
    opt = optim.AdamW([w, b], lr=0.1, ema_decay=0.5)
    y, kept = layers.layer_norm(x, w, b), (x * b).sum()
    opt.step([torch.ones_like(w), None])
    assert w._version == 1 and b._version == 0 and opt.ema._version > 0
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    kept.backward()
    assert torch.equal(b.grad, x.sum(0))
    layers.layer_norm(x, w, b).sum().backward()                 # the new weights' own graph
    assert w.grad is not None
    opt.step()
    assert w._version == 2 and b._version == 1


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_padding_stays_zero_whatever_the_factors(dtype, bits):
    """what fills a tensor's last block up is 0 in every flat buffer: also without eps (0 / 0 there) and with a gradient scale or a learning rate of infinity"""
    inf = torch.tensor(float("inf"), device="cuda")
    for eps, kw in ((0.0, {}), (1e-8, dict(grad_scale=inf)), (1e-8, dict(lr=inf)), (0.0, dict(grad_scale=torch.zeros_like(inf)))):
        params, _, grads = _setup(dtype, bits, False)
        opt = optim.AdamW(params, lr=LR, eps=eps, state_bits=bits, ema_decay=D)
        gs = grads()
        gs[3] = None                                                     # a tensor that is left alone
        opt.step(gs, **kw)
        flats = [f for f in (opt.master, opt.ema, opt.exp_avg, opt.exp_avg_sq) if f is not None]
        assert len(flats) == (4 if dtype == "bf16" else 3)
        for f in flats:
            for lo, hi, n in zip(opt.first_block, opt.first_block[1:], opt._numel):
                assert not f[lo * 256 + n:hi * 256].float().ne(0).any(), (eps, kw)
        if not kw:
            assert all(torch.isfinite(p).all() for p in params) and torch.isfinite(opt.ema).all()


@pytest.mark.parametrize("top", [4e20, 2.9e20, 2e20, 3e19])
def test_codes_of_the_largest_second_moments(top):
    """v up to the last values before overflow, where 1 / v is below the normal 32-bit numbers: the codes are those of the formula in 64 bits there, too"""
    g = torch.Generator().manual_seed(3)
    grad = torch.randn(1000, generator=g) * (top / 4)
    grad[5] = top
    grad[300:] *= 1e-3                                                   # blocks of ordinary scales beside it
    p = torch.zeros(1000, device="cuda")
    opt = optim.AdamW([p], lr=1e-3, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8)
    opt.step([grad.cuda()])
    x = torch.nn.functional.pad(grad.double(), (0, 24))
    for val, power, code, scale in ((x * (1 - 0.9), 2, opt.exp_avg, opt.exp_avg_scale), (x * x * (1 - 0.999), 4, opt.exp_avg_sq, opt.exp_avg_sq_scale)):
        want, s = R.encode(val, power)
        assert torch.equal(scale.cpu(), s) and torch.equal(code.cpu(), want), power


@pytest.mark.parametrize("bits", [32, 8])
def test_updates_of_the_largest_second_moments(bits):
    """v / (1 - b2^t) = g^2 passes the 32-bit numbers at g = 1.8e19, v itself only at 5.8e20: the first step is lr in every direction up to there"""
    grad = torch.tensor([1.0, 1e10, -1e15, 1e19, 2e19, 1e20, -4e20, 5e20])
    p = torch.zeros(8, device="cuda")
    opt = optim.AdamW([p], lr=1.0, betas=(0.9, 0.999), weight_decay=0.0, state_bits=bits)
    opt.step([grad.cuda()])
    # m / c1 and v / c2 are g and g^2 to a few roundings
    assert torch.allclose(p.cpu(), -grad.sign(), rtol=1e-5)
    if bits == 32:
        opt.step([torch.zeros(8, device="cuda")])
        m, v = 0.9 * 0.1 / (1 - 0.81), 0.999 * 0.001 / (1 - 0.999 ** 2)
        assert torch.allclose(p.cpu(), -grad.sign() * (1 + m / v ** 0.5), rtol=1e-5)


def test_gradients_have_their_parameters_shapes():
    """one rule, whether or not some gradients are None"""
    p = [torch.zeros(4, 6, device="cuda"), torch.zeros(5, device="cuda"), torch.zeros((), device="cuda")]
    opt = optim.AdamW(p)
    good = [torch.ones_like(t) for t in p]
    for i, shape in ((0, (24,)), (0, (6, 4)), (1, (5, 1)), (1, (1, 5)), (2, (1,))):
        for rest in (good, [None] * 3):
            with pytest.raises(ValueError, match=f"gradient {i}"):
                opt.step([torch.ones(shape, device="cuda") if j == i else g for j, g in enumerate(rest)])
    assert opt.state_dict()["step"] == 0 and not any(t.any() for t in p)
    opt.step(good)
    opt.step([None, good[1], None])
    assert opt.state_dict()["step"] == 2 and all(t.any() for t in p)


def test_a_state_of_other_tensors_is_refused():
    """buffers of the same length whose tensors lie in another order, have other shapes or other names"""
    make = lambda **kw: optim.AdamW({n: torch.zeros(s, device="cuda") for n, s in kw.items()})                             # noqa: E731
    opt = make(a=(300,), b=(20, 20))
    opt.step({"a": torch.ones(300, device="cuda"), "b": torch.full((20, 20), 2.0, device="cuda")})
    state = opt.state_dict()
    for other in (make(b=(20, 20), a=(300,)), make(a=(300,), b=(400,)), make(a=(300,), c=(20, 20)), make(a=(301,), b=(20, 20)), make(a=(512,), b=(512,))):
        with pytest.raises(ValueError):
            other.load_state_dict(state)
        assert not other.exp_avg.any() and other.state_dict()["step"] == 0
    for same in (make(a=(300,), b=(20, 20)), optim.AdamW([torch.zeros(300, device="cuda"), torch.zeros(20, 20, device="cuda")])):
        same.load_state_dict(state)
        assert torch.equal(same.exp_avg, opt.exp_avg) and same.state_dict()["step"] == 1
    again = make(a=(300,), b=(20, 20))
    again.load_state_dict({n: t for n, t in state.items() if n not in ("names", "sizes")})
    assert torch.equal(again.exp_avg_sq, opt.exp_avg_sq)


@pytest.mark.parametrize("dtype, bits", [("f32", 32), ("bf16", 8)])
def test_every_launch_of_a_long_list_follows_the_formula(dtype, bits):
    """900 tensors take three launches: parameters, moments and averages of each, and the tensors without decay, against the formula"""
    sizes = [(i % 5 + 1,) if i % 90 else (300 + i,) for i in range(900)]
    free = (0, 4, 399, 400, 450, 801, 899)
    g = torch.Generator().manual_seed(6)
    params = [torch.randn(s, generator=g).to(T[dtype]).cuda() for s in sizes]
    grads = [(torch.randn(s, generator=g) * 10.0 ** (i % 4 - 2)).to(T[dtype]).cuda() for i, s in enumerate(sizes)]
    before = [p.double().cpu() for p in params]
    opt = optim.AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, no_decay=free, state_bits=bits, ema_decay=D)
    opt.step(grads)
    for i, p in enumerate(params):
        z = torch.zeros(sizes[i], dtype=torch.float64)
        (pr, bp), (mr, bm), (vr, bv) = R.adamw(before[i], grads[i], z, z, 1, LR, B1, B2, EPS, 0.0 if i in free else WD)
        new = (opt.views(opt.master)[i] if dtype == "bf16" else p).double().cpu()
        R.within(new, pr, bp, f"p{i}")
        assert torch.equal(p.cpu(), new.to(T[dtype]))
        R.within(opt.views(opt.ema)[i], D * before[i] + (1 - D) * new, 4 * R.F32 * (before[i].abs() + new.abs()), f"ema{i}")
        if bits == 32:
            R.within(opt.views(opt.exp_avg)[i], mr, bm, f"m{i}")
            R.within(opt.views(opt.exp_avg_sq)[i], vr, bv, f"v{i}")
        else:
            for x, power, code, scale in ((mr, 2, opt.exp_avg, opt.exp_avg_scale), (vr, 4, opt.exp_avg_sq, opt.exp_avg_sq_scale)):
                c, s = R.encode(torch.nn.functional.pad(x, (0, -len(x) % 256)), power)
                lo, hi = opt.first_block[i], opt.first_block[i + 1]
                assert torch.equal(code[lo * 256:hi * 256].cpu(), c) and torch.allclose(scale[lo:hi].cpu(), s, rtol=2.0 ** -23, atol=0), (i, power)


def test_saving_and_loading_on_another_stream_tells_the_allocator():
    """the copies that state_dict leaves under way read the optimiser's own memory, on whatever stream is current"""
    params, opt, grads = _setup("bf16", 32, True)
    opt.step(grads())
    torch.cuda.synchronize()
    save, load = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(save):
        state = opt.state_dict()
    save.synchronize()
    _, again, _ = _setup("bf16", 32, True)
    torch.cuda.synchronize()
    with torch.cuda.stream(load):
        again.load_state_dict(state)
    torch.cuda.synchronize()
    assert save.cuda_stream in opt._streams._known and load.cuda_stream in again._streams._known
    assert torch.equal(opt.exp_avg, again.exp_avg) and all(torch.equal(a, b) for a, b in zip(params, again.params))
