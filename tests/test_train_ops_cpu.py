"""Training operators without a GPU: the library loads and exports what its header declares, struct mirrors fit, every refusal is an exception, and the
64-bit references agree with differences."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import train_ref as R
from diffphore_amd import _trainlib, layers, optim, weights

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_declared_symbol_and_nothing_else():
    hdr = open(os.path.join(ROOT, "include", "train", "diffphore_train.h")).read()
    names = set(re.findall(r"^\s*(?:int|size_t)\s+(dpt_\w+)\s*\(", hdr, flags=re.M))
    out = subprocess.run(["nm", "-D", "--defined-only", _trainlib.LIB_PATH], capture_output=True, text=True, check=True).stdout
    exported = {ln.split()[-1] for ln in out.splitlines() if len(ln.split()) >= 3 and ln.split()[-2] in "TtDdBbRrWwVv"}
    assert exported == names and {"dpt_attn_fwd", "dpt_attn_bwd", "dpt_layer_norm_fwd", "dpt_layer_norm_bwd", "dpt_adamw_step"} <= names
    assert _trainlib.lib().dpt_layer_norm_max_width() == layers._LN_MAX_WIDTH


def _attn_args(**kw):
    a = _trainlib.DptAttnArgs()
    a.type, a.B, a.heads, a.kv_heads, a.dim, a.n_q, a.n_k, a.max_nq, a.max_nk, a.n_pairs, a.scale = 0, 1, 4, 2, 32, 8, 8, 8, 8, 64, 0.1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, rc", [({}, -1), (dict(type=7), -1), (dict(heads=3), -1), (dict(dim=129), -3), (dict(dim=0), -1), (dict(scale=0.0), -1),
                                    (dict(scale=float("nan")), -1), (dict(max_nq=9), -1), (dict(B=-1), -1), (dict(n_q=2 ** 31 - 1, max_nq=2 ** 31 - 1), -3)])
def test_c_entry_points_refuse_before_any_gpu_call(kw, rc):
    """the default arguments are refused for their NULL pointers"""
    L = _trainlib.lib()
    a = _attn_args(**kw)
    assert L.dpt_attn_fwd(C.byref(a), None) == rc and L.dpt_attn_bwd(C.byref(a), None) == rc
    assert L.dpt_attn_fwd(None, None) == -1 and L.dpt_attn_bwd(None, None) == -1


def test_c_entry_points_of_norm_and_adamw_refuse():
    L = _trainlib.lib()
    n = None
    assert L.dpt_layer_norm_fwd(0, 0, 4, 8, n, 8, n, n, 1e-5, n, 8, n, n, n) == -1
    assert L.dpt_layer_norm_fwd(0, 0, 4, 16385, n, 8, n, n, 1e-5, n, 8, n, n, n) == -3
    assert L.dpt_layer_norm_fwd(0, 1, 4, 8, n, 8, n, n, 1e-5, n, 8, n, n, n) == -1          # bf16 weights of fp32 rows
    assert L.dpt_layer_norm_fwd(0, 0, 4, 8, n, 8, n, n, -1.0, n, 8, n, n, n) == -1
    assert L.dpt_layer_norm_fwd(0, 0, 0, 8, n, 8, n, n, 1e-5, n, 8, n, n, n) == 0
    assert L.dpt_layer_norm_bwd(0, 0, 4, 8, n, 8, n, 8, n, n, n, n, 8, n, n, n, 0, n) == -1
    assert L.dpt_layer_norm_ws_bytes(4, 8) > 0 and L.dpt_layer_norm_ws_bytes(4, 0) == 0
    a = _trainlib.DptAdamWArgs()
    assert L.dpt_adamw_step(C.byref(a), None, None) == -1 and L.dpt_adamw_step(None, None, None) == -1
    a.state_bits, a.n_tensors = 8, 401
    assert L.dpt_adamw_step(C.byref(a), None, None) == -1
    assert L.dpt_adamw_moments(n, n, n, n, 3, n, n, n) == -1 and L.dpt_adamw_moments(n, n, n, n, 0, n, n, n) == 0


@pytest.mark.parametrize("q, k", [([1, 2], [0, 2]), ([0, 3, 2], [0, 1, 2]), ([0, 2], [0, 1, 2]), ([], []), ([0.0, 1.0], [0, 1]), ([[0, 1]], [0, 1]),
                                  ([0, 1 << 31], [0, 1])])
def test_plan_refuses_offsets(q, k):
    with pytest.raises(ValueError):
        layers.PairPlan(q, k)


def test_cpu_tensors_and_other_types_are_refused():
    x = torch.zeros(3, 4)
    with pytest.raises(ValueError, match="GPU only"):
        layers.layer_norm(x)
    with pytest.raises(ValueError, match="GPU only"):
        optim.AdamW([x])
    with pytest.raises(ValueError):
        optim.AdamW([])
    with pytest.raises(ValueError, match="GPU only"):
        layers.attention_forward(torch.zeros(2, 1, 4), torch.zeros(2, 1, 4), torch.zeros(2, 1, 4), None)
    with pytest.raises(ValueError, match="GPU only"):
        layers.PairPlan([0, 1], [0, 1], "cpu")
    with pytest.raises(TypeError):
        layers.layer_norm("x")


def test_trainable_parameters_are_the_state_dict_without_its_buffers():
    sd = weights.init_state_dict(3)
    named = weights.trainable_parameters(sd, "cpu")
    assert len(named) == 228 and all(p.is_leaf and p.requires_grad for p in named.values())
    assert not any(n.endswith(("running_mean", "running_var", "offset")) for n in named)
    again = weights.clean_state_dict({**sd, **named})
    assert all(torch.equal(again[n], sd[n]) for n in sd)
    with torch.no_grad():
        named["final_conv.fc.0.bias"] += 1.0
    assert not torch.equal(named["final_conv.fc.0.bias"], sd["final_conv.fc.0.bias"])     # copies, not the dict's own tensors


@pytest.mark.parametrize("causal", [False, True])
def test_reference_gradients_agree_with_differences(causal):
    """the formulas the GPU tests hold the kernels to, against central differences of the forward formula in 64 bits"""
    g = torch.Generator().manual_seed(5)
    qp, kp = [0, 3, 3, 8], [0, 4, 6, 9]
    q, k, v, do = (torch.randn(n, h, 6, generator=g, dtype=torch.float32) for n, h in ((8, 4), (9, 2), (9, 2), (8, 4)))
    bias = torch.randn(4, 3 * 4 + 5 * 3, generator=g)
    grads = R.attention(q, k, v, qp, kp, bias, causal, dout=do)
    args = [q, k, v, bias]
    for i, (gr, _) in enumerate(grads):
        step = torch.randn(args[i].shape, generator=g)
        h = 2.0 ** -8

        def value(s):
            a = list(args)
            a[i] = a[i].double() + s * h * step.double()
            qd, kd, vd, bd = a
            (o, _), _, _ = _forward64(qd, kd, vd, qp, kp, bd, causal)
            return (o * do.double()).sum()
        diff = (value(1) - value(-1)) / (2 * h)
        assert abs(diff - (gr * step.double()).sum()) < 1e-3 * (1 + abs(diff))
    x, w, b, dy = (torch.randn(s, generator=g) for s in ((4, 7), (7,), (7,), (4, 7)))
    (dx, _), (dw, _), (dbb, _) = R.layer_norm_backward(dy, x, w, 1e-5, torch.float32, torch.float32)
    for arg, gr in ((0, dx), (1, dw), (2, dbb)):
        step = torch.randn(gr.shape, generator=g).double()

        def ln(s):
            a = [x.double(), w.double(), b.double()]
            a[arg] = a[arg] + s * 2.0 ** -10 * step
            return (R.layer_norm(*a, 1e-5, torch.float32)[0][0] * dy.double()).sum()
        diff = (ln(1) - ln(-1)) / 2.0 ** -9
        assert abs(diff - (gr * step).sum()) < 1e-3 * (1 + abs(diff))


def _forward64(q, k, v, qp, kp, bias, causal):
    R.U[torch.float64] = 2.0 ** -53
    return R.attention(q, k, v, qp, kp, bias, causal)


@pytest.mark.parametrize("power", [2, 4])
def test_codes_are_nearest_and_keep_small_second_moments(power):
    g = torch.Generator().manual_seed(power)
    x = torch.randn(4 * 256, generator=g, dtype=torch.float64) * torch.exp(4 * torch.randn(4 * 256, generator=g, dtype=torch.float64))
    x = x.abs() if power == 4 else x
    x[256:512] = 0
    code, scale = R.encode(x, power)
    y = R.decode(code, scale, power)
    top = 127 if power == 2 else 255
    # on the curve's axis a code is off by half a step at most, but for the second moments that would become 0
    root = lambda t: (t.abs().view(-1, 256) / scale.double()[:, None].clamp(min=1e-300)) ** (1 / power)      # noqa: E731
    off = (root(x) - root(y)).abs() * top
    small = (root(x) * top < 0.5) & (root(x) > 0) if power == 4 else torch.zeros_like(off, dtype=torch.bool)
    assert off[~small].max() <= 0.5 + 1e-5 and torch.equal(y == 0, x == 0) if power == 4 else off.max() <= 0.5 + 1e-5
    assert np.isfinite(y.numpy()).all() and code[256:512].abs().max() == 0 if power == 2 else True


@pytest.mark.parametrize("kw", [dict(n_k=2 ** 31 - 1, max_nk=2 ** 31 - 1), dict(n_k=2 ** 31 - 1024, max_nk=8), dict(n_q=2 ** 31 - 1024, max_nq=8),
                                dict(n_q=2 ** 31 - 1025, max_nq=2 ** 31 - 1025), dict(heads=2 ** 31 - 1, kv_heads=1, n_q=2 ** 30, max_nq=2 ** 30),
                                dict(B=2 ** 31 - 1, heads=2 ** 31 - 1, kv_heads=2 ** 31 - 1, n_k=2 ** 30, max_nk=2 ** 30)])
def test_lengths_and_counts_whose_arithmetic_would_wrap_are_too_large(kw):
    """row numbers of a last block that pass 2^31, and products of sizes that pass 2^63: refused on the host (the pointers are NULL, so -1 follows otherwise)"""
    L = _trainlib.lib()
    a = _attn_args(**kw)
    assert L.dpt_attn_fwd(C.byref(a), None) == -3 and L.dpt_attn_bwd(C.byref(a), None) == -3 and L.dpt_attn_ws_bytes(C.byref(a), 1) == 0
    a = _attn_args(heads=1, kv_heads=1, n_k=2 ** 31 - 1025, max_nk=2 ** 31 - 1025)
    assert L.dpt_attn_fwd(C.byref(a), None) == -1
    with pytest.raises(ValueError, match="rows"):
        layers.PairPlan([0, 1], [0, 2 ** 31 - 1024])


@pytest.mark.parametrize("scale", [1e-39, -1.0, 2.9e38, float("inf"), 2.0 ** 126])
def test_scales_without_a_normal_exponent_factor_are_refused(scale):
    """the kernels form scale log2 e: 0 or infinite, it made rows of equal scores NaN (the pointers are NULL and valid scales end at those: both -1)"""
    L = _trainlib.lib()
    ok = scale == 2.0 ** 126
    a = _attn_args(scale=scale)
    assert (L.dpt_attn_ws_bytes(C.byref(a), 1) > 0) == ok and L.dpt_attn_fwd(C.byref(a), None) == -1


@pytest.mark.parametrize("power", [2, 4])
def test_decoded_codes_are_finite_and_a_block_of_zeros_stays_zero(power):
    g = torch.Generator().manual_seed(power)
    x = torch.randn(4 * 256, generator=g, dtype=torch.float64) * torch.exp(4 * torch.randn(4 * 256, generator=g, dtype=torch.float64))
    x = x.abs() if power == 4 else x
    x[256:512] = 0
    code, scale = R.encode(x, power)
    y = R.decode(code, scale, power)
    assert torch.isfinite(y).all() and not code[256:512].any() and not y[256:512].any()
    # off by half a step of the curve's axis, or by less than a step where a second moment is kept from becoming 0
    top = 127 if power == 2 else 255
    root = lambda t: (t.abs().view(-1, 256) / scale.double()[:, None].clamp(min=1e-300)) ** (1 / power) * top              # noqa: E731
    off = (root(x) - root(y)).abs()
    kept = (root(x) < 0.5) & (root(x) > 0)
    if power == 4:
        assert (code.view(-1, 256)[kept] == 1).all() and off[kept].max() < 1
        off = off[~kept]
    assert off.max() <= 0.5 + 1e-5
