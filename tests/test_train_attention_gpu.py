"""Attention over packed complexes, forward and backward, against the definition in 64 bits (bounds: tests/train_ref.py)."""
import math

import pytest
import torch

import train_ref as R
from diffphore_amd import layers

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}


def ptr(n):
    out = [0]
    for x in n:
        out.append(out[-1] + x)
    return out


def make(nq, nk, heads, kv_heads, dim, dtype, bias=False, seed=0):
    g = torch.Generator().manual_seed(seed + dim + 7 * heads)
    q = torch.randn(sum(nq), heads, dim, generator=g).to(T[dtype]).cuda()
    k = torch.randn(sum(nk), kv_heads, dim, generator=g).to(T[dtype]).cuda()
    v = torch.randn(sum(nk), kv_heads, dim, generator=g).to(T[dtype]).cuda()
    do = torch.randn(sum(nq), heads, dim, generator=g).to(T[dtype]).cuda()
    b = torch.randn(heads, sum(a * c for a, c in zip(nq, nk)), generator=g).to(T[dtype]).cuda() if bias else None
    return q, k, v, do, b, layers.PairPlan(ptr(nq), ptr(nk))


def check(q, k, v, do, b, plan, causal=False, scale=None):
    qp, kp = plan.q_ptr.tolist(), plan.k_ptr.tolist()
    out, stats = layers.attention_forward(q, k, v, plan, bias=b, causal=causal, scale=scale)
    (o, bo), (m, bm), (l, bl) = R.attention(q, k, v, qp, kp, b, causal, scale)
    R.within(out, o, bo, "out")
    R.within(stats[0], m, bm, "m")
    R.within(stats[1], l, bl, "l")
    if do is None:
        return
    got = layers.attention_backward(do, q, k, v, out, stats, plan, bias=b, causal=causal, scale=scale)
    for g, ref, name in zip(got, R.attention(q, k, v, qp, kp, b, causal, scale, dout=do), ("dq", "dk", "dv", "dbias")):
        assert (g is None) == (ref is None)
        if g is not None:
            R.within(g, *ref, name)


RAGGED = ([5, 0, 33, 64, 1, 17, 130, 3], [7, 9, 0, 65, 1, 128, 63, 200])


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads, kv_heads, dim", [(4, 4, 20), (6, 2, 32), (2, 1, 5), (4, 4, 64), (8, 2, 128), (3, 1, 97), (2, 2, 40)])
def test_ragged_batches_with_empty_complexes(heads, kv_heads, dim, dtype, bias, causal):
    nq, nk = RAGGED
    check(*make(nq, nk, heads, kv_heads, dim, dtype, bias), causal=causal)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq, nk", [([1], [1]), ([20] * 6, [79] * 6), ([31, 32, 33], [33, 32, 31]), ([15, 45, 20], [16, 48, 30]), ([127, 129], [128, 130])])
def test_small_complexes(nq, nk, dtype):
    check(*make(nq, nk, 4, 4, 20, dtype, True))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq", [1, 2, 5])
def test_single_tokens_against_long_caches(nq, dtype):
    """few rows, many keys: the keys are split over workgroups and joined"""
    nk = [1, 700, 2500, 257]
    check(*make([nq] * 4, nk, 8, 2, 64, dtype), causal=True)
    check(*make([nq] * 4, nk, 4, 4, 33, dtype, True))
    check(*make([nq] * 2, [4000, 0], 16, 2, 128, dtype), causal=nq > 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long(dtype):
    check(*make([600, 300], [600, 513], 4, 2, 64, dtype), causal=True)
    check(*make([513], [640], 2, 2, 128, dtype))


def test_forced_splits_change_nothing_but_roundings():
    """DptAttnArgs.splits through the C ABI: 1, 3 and 64 ranges (more than there are key tiles) hold the same bounds"""
    import ctypes as C
    from diffphore_amd import _trainlib
    q, k, v, _, b, plan = make([40, 3], [300, 70], 4, 2, 32, "f32", True)
    (o, bo), (m, bm), (l, bl) = R.attention(q, k, v, plan.q_ptr.tolist(), plan.k_ptr.tolist(), b, False)
    L = _trainlib.lib()
    for splits in (1, 3, 64):
        a = layers._attn_args(q, k, v, plan, b, False, 1 / math.sqrt(32))
        out, stats = torch.empty_like(q), torch.empty(2, 4, q.shape[0], device="cuda")
        a.splits, a.out, a.stats = splits, out.data_ptr(), stats.data_ptr()
        ws = torch.empty(max(16, L.dpt_attn_ws_bytes(C.byref(a), 0)), dtype=torch.uint8, device="cuda")
        a.ws, a.ws_bytes = ws.data_ptr(), ws.numel()
        assert L.dpt_attn_fwd(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
        R.within(out, o, bo, f"out, {splits} splits")
        R.within(stats[0], m, bm, "m")
        R.within(stats[1], l, bl, "l")
        if splits == 3:
            a.ws_bytes = 16
            assert L.dpt_attn_fwd(C.byref(a), torch.cuda.current_stream().cuda_stream) == -1


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masks_by_bias(dtype):
    """-inf takes a pair out (also one whose score is not finite), whole rows too; the type's lowest value leaves a row its softmax over equals"""
    q, k, v, do, b, plan = make([4, 3], [40, 5], 2, 2, 16, dtype, True)
    b[:, :160].view(2, 4, 40)[:, 1, :] = -math.inf                       # a row without keys
    b[:, :160].view(2, 4, 40)[:, 2, 1:] = -math.inf                      # a row with one key
    b[:, :160].view(2, 4, 40)[:, :, 7] = -math.inf                       # a key that nothing sees
    check(q, k, v, do, b, plan)
    out, stats = layers.attention_forward(q, k, v, plan, bias=b)
    assert not out[1].any() and (stats[0, :, 1] == -math.inf).all() and (stats[1, :, 1] == 0).all()
    grads = layers.attention_backward(do, q, k, v, out, stats, plan, bias=b)
    assert all(torch.isfinite(g).all() for g in grads) and not grads[0][1].any() and not grads[1][7].any() and not grads[2][7].any()
    k2 = k.clone()
    k2[7] = math.nan                                                     # only in the key: its scores are taken out before they count
    out2, _ = layers.attention_forward(q, k2, v, plan, bias=b)
    assert torch.equal(out, out2)
    b = torch.zeros_like(b)
    b[:, :160].view(2, 4, 40)[:, 1, :] = torch.finfo(b.dtype).min
    out, stats = layers.attention_forward(q, k, v, plan, bias=b)
    assert torch.allclose(out[1].float(), v[:40].float().mean(0), atol=2.0 ** -7) and torch.allclose(stats[1, :, 1], torch.full((2,), 40.0, device="cuda"))
    dq, dk, dv, db = layers.attention_backward(do, q, k, v, out, stats, plan, bias=b)
    assert all(torch.isfinite(g).all() for g in (dq, dk, dv, db))
    # p = 1/40 for every key of that row: its share of dv is do / 40
    do1 = torch.zeros_like(do)
    do1[1] = 1.0
    _, _, dv, _ = layers.attention_backward(do1, q, k, v, out, stats, plan, bias=b)
    assert torch.allclose(dv[:40].float(), torch.full_like(dv[:40].float(), 1 / 40), rtol=2.0 ** -7)


def test_nan_and_inf_reach_their_own_rows():
    q, k, v, do, b, plan = make([50, 20], [60, 30], 2, 2, 32, "bf16")
    clean, _ = layers.attention_forward(q, k, v, plan)
    q[5, 0, 3] = math.nan
    k[70, 1, 0] = math.inf                                               # second complex, head 1
    out, _ = layers.attention_forward(q, k, v, plan)
    assert torch.isnan(out[5, 0]).all() and torch.equal(out[5, 1], clean[5, 1])
    rest = [i for i in range(50) if i != 5]
    assert torch.equal(out[rest], clean[rest]) and torch.equal(out[50:, 0], clean[50:, 0])


def test_causal_rows_before_the_first_key_are_empty():
    q, k, v, do, b, plan = make([10], [4], 1, 1, 16, "f32")              # queries 0..5 see nothing
    out, stats = layers.attention_forward(q, k, v, plan, causal=True)
    assert not out[:6].any() and (stats[1, :, :6] == 0).all() and (stats[1, :, 6] == 1).all()
    check(q, k, v, do, b, plan, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(dtype):
    """packed q k v, a head-major bias as a view of a pair-major one, shared over heads, misaligned rows, expanded gradients"""
    g = torch.Generator().manual_seed(11)
    nq, H, D = [20, 37, 5], 4, 24
    qkv = torch.randn(sum(nq), 3, H, D, generator=g).to(T[dtype]).cuda()
    plan = layers.PairPlan(ptr(nq), ptr(nq))
    pair = torch.randn(plan.n_pairs, H, generator=g).to(T[dtype]).cuda()
    q, k, v = qkv.unbind(1)
    do = torch.randn(sum(nq), H, D, generator=g).to(T[dtype]).cuda()
    check(q, k, v, do, pair.t(), plan)
    check(q, k, v, do[:1].expand_as(do), pair[:, :1].t().expand(H, -1), plan)
    odd = torch.randn(sum(nq), H * D + 3, generator=g).to(T[dtype]).cuda()[:, 3:].view(sum(nq), H, D)
    check(odd, k, v, do, None, plan)
    last = torch.randn(sum(nq), H, D, 2, generator=g).to(T[dtype]).cuda()[..., 1]               # no unit stride: copied
    check(last, k, last, last, None, plan)


def test_gradients_against_differences():
    q, k, v, do, b, plan = make([9, 4], [11, 6], 2, 1, 16, "f32", True)
    qp, kp = plan.q_ptr.tolist(), plan.k_ptr.tolist()
    out, stats = layers.attention_forward(q, k, v, plan, bias=b)
    grads = layers.attention_backward(do, q, k, v, out, stats, plan, bias=b)
    R.U[torch.float64] = 2.0 ** -53
    args = [t.double().cpu() for t in (q, k, v, b)]
    g = torch.Generator().manual_seed(3)
    for i, gr in enumerate(grads):
        step, h = torch.randn(args[i].shape, generator=g, dtype=torch.float64), 2.0 ** -10

        def value(s):
            a = [t + s * h * step if j == i else t for j, t in enumerate(args)]
            return (R.attention(*a[:3], qp, kp, a[3])[0][0] * do.double().cpu()).sum()
        diff = (value(1) - value(-1)) / (2 * h)
        # h^2 times a third derivative of order 10 |step|^3, against a sum over |step| n entries
        assert abs(diff - (gr.double().cpu() * step).sum()) < 1e-3 * (1.0 + abs(diff))


def test_autograd_shared_bias_and_partial_gradients():
    q, k, v, do, _, plan = make([12, 7], [9, 30], 4, 2, 20, "f32")
    g = torch.Generator().manual_seed(1)
    shared = torch.randn(1, plan.n_pairs, generator=g).cuda().requires_grad_()
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    out = layers.attention(q, k, v, plan, bias=shared.expand(4, -1))
    out.backward(do)
    ref = R.attention(q.detach(), k.detach(), v.detach(), plan.q_ptr.tolist(), plan.k_ptr.tolist(), shared.detach().expand(4, -1), dout=do)
    for t, (r, bound) in zip((q, k, v), ref[:3]):
        R.within(t.grad, r, bound, "grad")
    R.within(shared.grad, ref[3][0].sum(0, keepdim=True), ref[3][1].sum(0, keepdim=True) + 8 * R.F32 * ref[3][0].abs().sum(0, keepdim=True), "shared bias")
    k2 = k.detach().requires_grad_()
    (gk,) = torch.autograd.grad(layers.attention(q.detach(), k2, v.detach(), plan, bias=shared.detach().expand(4, -1)), k2, do)
    assert torch.equal(gk, k.grad)


def test_same_bits_every_time_on_any_stream_and_in_any_company():
    q, k, v, do, b, plan = make([200, 31], [333, 64], 8, 2, 64, "bf16")
    out, stats = layers.attention_forward(q, k, v, plan, causal=True)
    ref = layers.attention_backward(do, q, k, v, out, stats, plan, causal=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out2, stats2 = layers.attention_forward(q, k, v, plan, causal=True)
        other = layers.attention_backward(do, q, k, v, out2, stats2, plan, causal=True)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, out2) and all(torch.equal(a, c) for a, c in zip(ref[:3], other[:3]))
    # one complex alone gives the bits it has in the batch
    alone = layers.PairPlan([0, 31], [0, 64])
    o3, s3 = layers.attention_forward(q[200:], k[333:], v[333:], alone, causal=True)
    R.within(o3, out[200:], 2 * R.U[torch.bfloat16] * out[200:].abs() + 2.0 ** -8 * v.abs().max(), "alone")


def test_no_rows():
    for nq, nk in (([0], [5]), ([3], [0]), ([0, 0], [0, 0])):
        q, k, v, do, b, plan = make(nq, nk, 2, 1, 8, "f32", True)
        out, stats = layers.attention_forward(q, k, v, plan, bias=b)
        assert not out.any() and (stats[0] == -math.inf).all()
        dq, dk, dv, db = layers.attention_backward(do, q, k, v, out, stats, plan, bias=b)
        assert not dq.any() and not dk.any() and not dv.any() and db.shape == b.shape
    plan = layers.PairPlan([0], [0])
    e = torch.empty(0, 2, 8, device="cuda")
    out, _ = layers.attention_forward(e, e, e, plan)
    assert out.shape == (0, 2, 8)


def test_refusals():
    q, k, v, do, b, plan = make([4], [5], 4, 2, 16, "f32", True)
    z = lambda *s, **kw: torch.zeros(*s, device="cuda", **kw)          # noqa: E731
    for args in ((q.half(), k.half(), v.half(), plan), (q.bfloat16(), k, v, plan), (q[:3], k, v, plan), (q, k[:4], v[:4], plan), (q, k, v[..., :8], plan),
                 (q[:, :3], k, v, plan), (q.flatten(1), k, v, plan), (q.cpu(), k, v, plan), (z(4, 4, 129), z(5, 2, 129), z(5, 2, 129), plan),
                 (z(4, 4, 0), z(5, 2, 0), z(5, 2, 0), plan)):
        with pytest.raises((TypeError, ValueError)):
            layers.attention_forward(*args)
    for kw in (dict(bias=b[:, :-1]), dict(bias=b[:2]), dict(bias=b.bfloat16()), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan)):
        with pytest.raises((TypeError, ValueError)):
            layers.attention_forward(q, k, v, plan, **kw)
    out, stats = layers.attention_forward(q, k, v, plan)
    for args in ((do[:3], q, k, v, out, stats, plan), (do.bfloat16(), q, k, v, out, stats, plan), (do, q, k, v, out, stats[0], plan),
                 (do, q, k, v, out[:, :2], stats, plan), (do, q, k, v, out, stats.double(), plan)):
        with pytest.raises((TypeError, ValueError)):
            layers.attention_backward(*args)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads, kv_heads, dim", [(1, 1, 1), (40, 1, 8), (12, 2, 64), (3, 3, 2)])
def test_one_dimension_and_many_heads_on_one_key_head(heads, kv_heads, dim, dtype):
    check(*make([3, 40, 1], [5, 70, 33], heads, kv_heads, dim, dtype, True), causal=True)
    check(*make([90], [200], heads, kv_heads, dim, dtype), causal=True)


@pytest.mark.parametrize("scale", [1e-3, 1.0, 30.0])
def test_scales(scale):
    """from almost uniform rows to rows that one key decides; the running base follows maxima that move far"""
    check(*make([70, 5], [300, 90], 2, 2, 32, "f32"), scale=scale)
    q, k, v, do, b, plan = make([64], [256], 2, 1, 64, "bf16")
    k = (k.float() * torch.linspace(0.01, 3, 256, device="cuda")[:, None, None]).bfloat16()    # scores grow along the keys
    out, stats = layers.attention_forward(q, k, v, plan, scale=scale)
    (o, bo), (m, bm), (l, bl) = R.attention(q, k, v, [0, 64], [0, 256], None, False, scale)
    # exp2(fma(x, c, -m c)): the product m c is rounded once, a relative error of |m| 2^-24 (times log 2) in every term
    extra = 2 * R.F32 * m.abs()
    R.within(stats[0], m, bm + extra, "m")
    R.within(stats[1], l, bl + l * extra, "l")
    R.within(out, o, bo + 2 * extra.t()[:, :, None] * v.abs().max().double().cpu(), "out")


def test_two_captured_graphs_with_workspaces_of_their_own():
    q, k, v, do, b, plan = make([2, 1], [3000, 900], 8, 2, 64, "bf16")
    inputs = [[t.clone() for t in (q, k, v)] for _ in range(2)]
    inputs[1][0].mul_(2.0)
    layers.attention_forward(*inputs[0], plan, causal=True)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layers.attention_forward(*a, plan, causal=True))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for i in range(3):
        for a in inputs:
            a[2].add_(0.5)
        for s, g in zip(streams, graphs):                      # side by side
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for a, (o, st) in zip(inputs, outs):
            oe, ste = layers.attention_forward(*a, plan, causal=True)
            torch.cuda.synchronize()
            assert torch.equal(o, oe) and torch.equal(st, ste), i


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_backward_of_few_workgroups_is_split_and_joined(causal, dtype):
    """one complex, one key head: key ranges of the rows' gradient and row ranges of the keys' are summed; the same bits every time"""
    for args in (([783], [674], 2, 1, 42, dtype), ([600, 0, 70], [900, 40, 513], 2, 2, 64, dtype, True), ([1], [2000], 4, 1, 128, dtype), ([1500], [3], 1, 1, 20, dtype, True)):
        q, k, v, do, b, plan = make(*args)
        check(q, k, v, do, b, plan, causal=causal)
        out, stats = layers.attention_forward(q, k, v, plan, bias=b, causal=causal)
        one, two = (layers.attention_backward(do, q, k, v, out, stats, plan, bias=b, causal=causal) for _ in range(2))
        assert all(x is None or torch.equal(x, y) for x, y in zip(one, two))


def test_forced_splits_of_the_backward_pass():
    """DptAttnArgs.splits through the C ABI: more ranges than there are tiles, empty complexes among them"""
    import ctypes as C
    from diffphore_amd import _trainlib
    q, k, v, do, b, plan = make([40, 0, 3], [300, 9, 0], 4, 2, 32, "f32", True)
    out, stats = layers.attention_forward(q, k, v, plan, bias=b)
    ref = R.attention(q, k, v, plan.q_ptr.tolist(), plan.k_ptr.tolist(), b, dout=do)
    L = _trainlib.lib()
    for splits in (1, 2, 5, 64):
        a = layers._attn_args(q, k, v, plan, b, False, 1 / math.sqrt(32))
        a.dout_row, a.dout_head, _ = do.stride()
        got = [torch.full_like(t, math.nan) for t in (q, k, v, b)]
        a.splits, (a.out, a.stats, a.dout, a.dq, a.dk, a.dv, a.dbias) = splits, (t.data_ptr() for t in (out, stats, do, *got))
        ws = torch.empty(L.dpt_attn_ws_bytes(C.byref(a), 1), dtype=torch.uint8, device="cuda")
        a.ws, a.ws_bytes = ws.data_ptr(), ws.numel()
        assert L.dpt_attn_bwd(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
        for g, r, name in zip(got, ref, ("dq", "dk", "dv", "dbias")):
            R.within(g, *r, f"{name}, {splits} splits")
        a.ws_bytes = 16
        assert L.dpt_attn_bwd(C.byref(a), torch.cuda.current_stream().cuda_stream) == -1


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_row_that_is_nan_leaves_the_values_that_it_does_not_see(dtype, bias):
    """causal: query 3 is NaN, so are its statistics; dv of the keys behind it, and dbias of the other rows, are those of the rows that see them"""
    q, k, v, do, b, plan = make([40], [40], 1, 1, 32, dtype, bias)
    out, stats = layers.attention_forward(q, k, v, plan, bias=b, causal=True)
    _, _, dv, db = layers.attention_backward(do, q, k, v, out, stats, plan, bias=b, causal=True)
    q[3] = math.nan
    out, stats = layers.attention_forward(q, k, v, plan, bias=b, causal=True)
    assert torch.isnan(out[3]).all() and torch.isfinite(out[4:]).all()
    _, _, dv2, db2 = layers.attention_backward(do, q, k, v, out, stats, plan, bias=b, causal=True)
    assert torch.equal(dv2[4:], dv[4:]) and torch.isnan(dv2[:4]).all()
    if bias:
        rest = [i for i in range(40) if i != 3]
        assert torch.equal(db2.view(1, 40, 40)[:, rest], db.view(1, 40, 40)[:, rest])


def test_offsets_beyond_32_bits():
    """keys and values of more than 2^31 elements: a small complex behind a very long one, and the long one's last keys"""
    n, tail, H, D = 1_060_000, 70, 16, 128
    assert n * H * D > 1 << 31
    g = torch.Generator().manual_seed(2)
    k, v = (torch.zeros(n + tail, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k[-tail - 1:], v[-tail - 1:] = (torch.randn(tail + 1, H, D, generator=g).bfloat16().cuda() for _ in range(2))      # the long one's last key too
    q, do = (torch.randn(4, H, D, generator=g).bfloat16().cuda() for _ in range(2))
    plan = layers.PairPlan([0, 1, 4], [0, n, n + tail])
    out, stats = layers.attention_forward(q, k, v, plan)
    (o, bo), _, _ = R.attention(q[1:], k[n:], v[n:], [0, 3], [0, tail])
    R.within(out[1:], o, bo, "out")
    # the long complex: n - 1 scores of 0 with values 0, and one of s.  A sum of n terms in 32 bits is good to n 2^-24 (6 %), p and the output to half a step each
    s = (q[0].double() * k[n - 1].double()).sum(-1) / D ** 0.5
    top, wide = s.clamp(min=0), n * R.F32 + 3 * R.U[torch.bfloat16]
    total = torch.exp(s - top) + (n - 1) * torch.exp(-top)
    p = torch.exp(s - top) / total
    R.within(stats[1, :, 0], total, n * R.F32 * total, "l")
    want = p[:, None] * v[n - 1].double()
    R.within(out[0], want, wide * want.abs(), "out of the long complex")
    dq, dk, dv, _ = layers.attention_backward(do, q, k, v, out, stats, plan)
    for got, ref, name in zip((dq[1:], dk[n:], dv[n:]), R.attention(q[1:], k[n:], v[n:], [0, 3], [0, tail], dout=do[1:]), ("dq", "dk", "dv")):
        R.within(got, *ref, name)
    want = p[:, None] * do[0].double()
    R.within(dv[n - 1], want, wide * want.abs(), "dv of the last key")


@pytest.mark.parametrize("long_keys", [False, True])
def test_more_workgroups_than_one_launch_takes(long_keys):
    """one long complex among a thousand short ones: the blocks of the largest complex times the complexes are more than 2^24 workgroups of 256 lanes, whose
    lanes do not fit the 32 bits of one launch.  A short complex has one query and one key: out = v, dv = dout, dq = dk = 0"""
    short, long, H, D = 1030, 32768, 64, 4
    assert (long // 128) * (short + 1) * H > 1 << 24
    nq, nk = [1] * short + [3 if long_keys else long], [1] * short + [long if long_keys else 3]
    q, k, v, do, _, plan = make(nq, nk, H, H, D, "f32")
    out, stats = layers.attention_forward(q, k, v, plan)
    dq, dk, dv, _ = layers.attention_backward(do, q, k, v, out, stats, plan)
    assert torch.equal(out[:short], v[:short]) and torch.equal(dv[:short], do[:short]) and not dq[:short].any() and not dk[:short].any()
    assert torch.equal(stats[1, :, :short], torch.ones_like(stats[1, :, :short]))
    for h in (0, H - 1):
        args = [t[short:, h:h + 1] for t in (q, k, v)]
        (o, bo), (m, bm), (l, bl) = R.attention(*args, [0, nq[-1]], [0, nk[-1]])
        R.within(out[short:, h:h + 1], o, bo, "out")
        R.within(stats[0, h:h + 1, short:], m, bm, "m")
        R.within(stats[1, h:h + 1, short:], l, bl, "l")
        refs = R.attention(*args, [0, nq[-1]], [0, nk[-1]], dout=do[short:, h:h + 1])
        for got, ref, name in zip((dq, dk, dv), refs, ("dq", "dk", "dv")):
            R.within(got[short:, h:h + 1], *ref, name)


def test_a_plan_dropped_while_another_stream_still_reads_it():
    """the plan's offsets are the plan's own memory: what is allocated after it is gone does not overwrite what a launch under way reads (zeros there would leave
    every complex empty)"""
    q, k, v, do, _, plan = make([5, 40, 7], [9, 70, 3], 2, 2, 16, "f32")
    out, stats = layers.attention_forward(q, k, v, plan)
    ref = layers.attention_backward(do, q, k, v, out, stats, plan)
    n, side = plan._dev.numel(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        out2, stats2 = layers.attention_forward(q, k, v, plan)
        got = layers.attention_backward(do, q, k, v, out2, stats2, plan)
    del plan
    junk = [torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(64)]
    torch.cuda.synchronize()
    assert torch.equal(out, out2) and all(torch.equal(a, b) for a, b in zip(ref[:3], got[:3])) and len(junk) == 64


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_smallest_and_largest_scales(dtype):
    """scales whose exponent factor is no normal number are refused; at the ends of the range equal scores still weigh equally"""
    v = torch.randn(4, 1, 8, generator=torch.Generator().manual_seed(1)).to(T[dtype]).cuda()
    plan = layers.PairPlan([0, 4], [0, 4])
    for scale in (1e-50, 1e-39, 1e38, 2.9e38, 1e300):
        with pytest.raises(ValueError, match="scale"):
            layers.attention_forward(v, v, v, plan, scale=scale)
    for scale, q in ((2.0 ** -126, v), (2.0 ** 126, torch.zeros_like(v))):
        out, stats = layers.attention_forward(q, q, v, plan, scale=scale)
        (o, bo), _, (l, bl) = R.attention(q, q, v, [0, 4], [0, 4], scale=scale)
        R.within(out, o, bo, "out")
        R.within(stats[1], l, bl, "l")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nk", [40, 3000])
def test_rows_without_keys_are_zero_beside_values_that_are_not_finite(nk, dtype):
    """out and dq of a row that sees nothing are 0 whatever k and v hold; a row that is NaN itself is no such row, and its statistics say so"""
    q, k, v, do, _, plan = make([nk + 3], [nk], 1, 1, 32, dtype)                         # causal: the first 3 rows see nothing
    q[8, 0, 1] = math.nan
    k[0], v[0] = math.nan, math.inf                                                      # in the tile of the first rows
    out, stats = layers.attention_forward(q, k, v, plan, causal=True)
    assert not out[:3].any() and (stats[0, 0, :3] == -math.inf).all() and not stats[1, 0, :3].any()
    assert torch.isnan(out[8]).all() and torch.isnan(stats[1, 0, 8])
    dq = layers.attention_backward(do, q, k, v, out, stats, plan, causal=True)[0]
    assert not dq[:3].any() and torch.isnan(dq[8]).all()
    q, k, v, do, b, plan = make([3], [nk], 1, 1, 32, dtype, True)                        # (3000 keys: ranges that are joined)
    b.view(1, 3, nk)[:, 1] = -math.inf
    k[nk - 1], v[nk - 1] = math.inf, math.nan
    out, stats = layers.attention_forward(q, k, v, plan, bias=b)
    assert not out[1].any() and not stats[1, 0, 1] and torch.isnan(out[0]).all()
    dq, _, _, db = layers.attention_backward(do, q, k, v, out, stats, plan, bias=b)
    assert not dq[1].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_a_complex_alone_holds_the_same_bounds(causal, dtype):
    """alone or in a batch, a complex's rows are those of the definition; their bits may differ, since the number of joined ranges goes by the batch"""
    q, k, v, do, b, plan = make([200, 31], [333, 64], 4, 2, 64, dtype, True)
    check(q, k, v, do, b, plan, causal=causal)
    check(q[200:], k[333:], v[333:], do[200:], b[:, 200 * 333:], layers.PairPlan([0, 31], [0, 64]), causal=causal)


def test_copies_of_a_plan_have_memory_of_their_own():
    import copy
    import pickle
    q, k, v, _, _, plan = make([5, 40, 7], [9, 70, 3], 2, 2, 16, "f32")
    out, _ = layers.attention_forward(q, k, v, plan)
    copies = [copy.copy(plan), copy.deepcopy(plan), pickle.loads(pickle.dumps(plan))]
    assert len({c._ptrs for c in copies} | {plan._ptrs}) == 4 and all(c._ptrs[2] == c._dev.data_ptr() for c in copies)
    n = plan._dev.numel()
    del plan
    junk = [torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(16)]
    for c in copies:
        assert torch.equal(layers.attention_forward(q, k, v, c)[0], out) and c.n_pairs == 5 * 9 + 40 * 70 + 7 * 3
    assert len(junk) == 16
