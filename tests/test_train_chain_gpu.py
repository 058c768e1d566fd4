"""The training operators together: an attention layer on a packed batch of complexes (layer norm, attention of the atoms over the pharmacophore with a bias
per pair, layer norm) trained with AdamW - against autograd in 64 bits, as one captured graph - and AdamW's averaged weights in the score model."""
import pytest
import torch

import train_ref as R
from diffphore_amd import config, layers, optim, synthetic, weights
from diffphore_amd.engine import PackedBatch

pytestmark = pytest.mark.gpu


def _layer(plan, dtype=torch.float32, H=4, C=20, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0, mean=0.0: (torch.randn(*s, generator=g) * std + mean)          # noqa: E731
    x = {"lig": r(plan.n_q, C), "ph": r(plan.n_k, C), "pair": r(plan.n_pairs, 9)}
    p = {"n1.w": r(C, std=0.1, mean=1), "n1.b": r(C, std=0.1), "n2.w": r(C, std=0.1, mean=1), "n2.b": r(C, std=0.1), "q": r(C, C, std=0.3),
         "k": r(C, C, std=0.3), "v": r(C, C, std=0.3), "bias": r(9, H, std=0.3)}
    return {n: t.to(dtype).cuda() for n, t in x.items()}, {n: t.to(dtype).cuda() for n, t in p.items()}


def _forward(x, p, plan, H=4):
    n = lambda t: t.view(t.shape[0], H, -1)                                                # noqa: E731
    a = layers.layer_norm(x["lig"], p["n1.w"], p["n1.b"])
    o = layers.attention(n(a @ p["q"]), n(x["ph"] @ p["k"]), n(x["ph"] @ p["v"]), plan, bias=(x["pair"] @ p["bias"]).t())
    return layers.layer_norm(x["lig"] + o.flatten(1), p["n2.w"], p["n2.b"])


def _forward64(x, p, plan, H=4):
    ln = lambda t, w, b: torch.nn.functional.layer_norm(t, t.shape[-1:], w, b)             # noqa: E731
    a = ln(x["lig"], p["n1.w"], p["n1.b"])
    q, k, v, bias = a @ p["q"], x["ph"] @ p["k"], x["ph"] @ p["v"], x["pair"] @ p["bias"]
    out = []
    for b in range(plan.B):
        i, j, c = (slice(int(t[b]), int(t[b + 1])) for t in (plan.q_ptr, plan.k_ptr, plan.pair_ptr))
        n = lambda t: t.view(t.shape[0], H, -1).transpose(0, 1)                            # noqa: E731
        s = n(q[i]) @ n(k[j]).transpose(1, 2) / (q.shape[1] // H) ** 0.5
        s = s + bias[c].t().view(H, s.shape[1], s.shape[2])
        out.append((s.softmax(-1) @ n(v[j])).transpose(0, 1).flatten(1))
    return ln(x["lig"] + torch.cat(out), p["n2.w"], p["n2.b"])


@pytest.fixture(scope="module")
def plan():
    batch = PackedBatch(synthetic.synthetic_pairs(7, 5, 20, 3, 17), "cuda")
    plan = layers.PairPlan.from_batch(batch)
    assert plan.B == 5 and plan.n_q == int(sum(batch.nl)) and plan.n_k == int(sum(batch.np_)) and plan.n_pairs == batch.struct.n_x
    return plan


def test_gradients_of_an_attention_layer_match_64_bits(plan):
    x, p = _layer(plan)
    p = {n: t.requires_grad_() for n, t in p.items()}
    g = torch.Generator().manual_seed(4)
    dy = torch.randn(plan.n_q, 20, generator=g)
    y = _forward(x, p, plan)
    y.backward(dy.cuda())
    xd = {n: t.double().cpu() for n, t in x.items()}
    pd = {n: t.detach().double().cpu().requires_grad_() for n, t in p.items()}
    yd = _forward64(xd, pd, plan)
    yd.backward(dy.double())
    # a chain of about ten 32-bit operators with sums of up to 100 terms: 1e-5 of the largest entry is about 170 roundings
    assert (y.detach().cpu().double() - yd.detach()).abs().max() < 1e-5 * yd.abs().max()
    for n in p:
        assert (p[n].grad.cpu().double() - pd[n].grad).abs().max() < 1e-5 * pd[n].grad.abs().max(), n


def test_training_steps_follow_64_bits(plan):
    x, p = _layer(plan, seed=1)
    p = {n: t.requires_grad_() for n, t in p.items()}
    kw = dict(lr=1e-3, betas=(0.9, 0.99), weight_decay=0.05)
    opt = optim.AdamW(p, no_decay=["n1.w", "n1.b", "n2.w", "n2.b"], ema_decay=0.9, **kw)
    xd = {n: t.double().cpu() for n, t in x.items()}
    pd = {n: t.detach().double().cpu().requires_grad_() for n, t in p.items()}
    ref = torch.optim.AdamW([{"params": [t for n, t in pd.items() if n[0] == "n"], "weight_decay": 0.0}, {"params": [t for n, t in pd.items() if n[0] != "n"]}], **kw)
    ema = {n: t.detach().clone() for n, t in pd.items()}
    goal = torch.randn(plan.n_q, 20, generator=torch.Generator().manual_seed(9))
    for _ in range(5):
        opt.zero_grad()
        ((_forward(x, p, plan) - goal.cuda()) ** 2).mean().backward()
        opt.step()
        ref.zero_grad()
        ((_forward64(xd, pd, plan) - goal.double()) ** 2).mean().backward()
        ref.step()
        ema = {n: 0.9 * e + 0.1 * pd[n].detach() for n, e in ema.items()}
    for n in p:
        # a step is lr g / |g| early on: a gradient's relative error of 1e-4 (small entries among large) is 1e-7 of a parameter per step
        assert (p[n].detach().cpu().double() - pd[n].detach()).abs().max() < 5e-6, n
        assert (opt.ema_parameters()[n].cpu().double() - ema[n]).abs().max() < 5e-6, n


def _step(x, p, opt, plan, dy):
    """one training step by the explicit functions: nothing of autograd is captured"""
    H, n = 4, lambda t: t.view(t.shape[0], 4, -1)                                          # noqa: E731
    a, m1, r1 = layers.layer_norm_forward(x["lig"], p["n1.w"], p["n1.b"])
    q, k, v = n(a @ p["q"]), n(x["ph"] @ p["k"]), n(x["ph"] @ p["v"])
    bias = (x["pair"] @ p["bias"]).t()
    o, st = layers.attention_forward(q, k, v, plan, bias=bias)
    h = x["lig"] + o.flatten(1)
    y, m2, r2 = layers.layer_norm_forward(h, p["n2.w"], p["n2.b"])
    dh, dw2, db2 = layers.layer_norm_backward(dy, h, m2, r2, p["n2.w"])
    dq, dk, dv, dbias = layers.attention_backward(n(dh), q, k, v, o, st, plan, bias=bias)
    da = dq.flatten(1) @ p["q"].t()
    _, dw1, db1 = layers.layer_norm_backward(da, x["lig"], m1, r1, p["n1.w"])
    grads = {"n1.w": dw1, "n1.b": db1, "n2.w": dw2, "n2.b": db2, "q": a.t() @ dq.flatten(1), "k": x["ph"].t() @ dk.flatten(1), "v": x["ph"].t() @ dv.flatten(1),
             "bias": x["pair"].t() @ dbias.t()}
    opt.step(grads)
    return y


@pytest.mark.parametrize("dtype, bits", [(torch.float32, 32), (torch.bfloat16, 8)])
def test_a_captured_step_replays_as_the_eager_one(plan, dtype, bits):
    make = lambda: _layer(plan, dtype, seed=3)                                             # noqa: E731
    x, p = make()
    _, pe = make()
    opt, ope = (optim.AdamW(t, lr=1e-3, state_bits=bits, ema_decay=0.9) for t in (p, pe))
    dy = torch.randn(plan.n_q, 20, generator=torch.Generator().manual_seed(6)).to(dtype).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):                                                            # warm up on the capture's stream
        _step(x, p, opt, plan, dy)
    torch.cuda.current_stream().wait_stream(s)
    _step(x, pe, ope, plan, dy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _step(x, p, opt, plan, dy)
    for i in range(4):
        x["lig"].add_(0.125)                                                              # new inputs in the captured buffers
        dy.mul_(-1.0)
        graph.replay()
        ye = _step(x, pe, ope, plan, dy)                                                  # the program's own work between the replays
        torch.cuda.synchronize()
        assert torch.equal(y, ye), i
        for n in p:
            assert torch.equal(p[n], pe[n]), (i, n)
        assert torch.equal(opt.exp_avg, ope.exp_avg) and torch.equal(opt.exp_avg_sq, ope.exp_avg_sq) and torch.equal(opt.ema, ope.ema)
    assert opt.state_dict()["step"] == ope.state_dict()["step"] == 5                      # a warm-up, a capture that runs nothing, 4 replays


def test_averaged_weights_drive_the_score_model():
    """the score model's 228 parameters under AdamW with a running average; the average loaded into the score model gives the oracle's scores"""
    from diffphore_amd.score_model import TensorProductScoreModel
    from oracle.model import OracleScoreModel
    from oracle.tables import load_tables
    from oracle.sampler import set_time_phore
    from diffphore_amd.hetero import Batch
    sd = weights.init_state_dict(11)
    named = weights.trainable_parameters(sd)
    opt = optim.AdamW(named, lr=1e-3, no_decay=[n for n, t in named.items() if t.dim() < 2], ema_decay=0.5)
    g = torch.Generator().manual_seed(8)
    want = {n: t.detach().double().cpu().clone() for n, t in named.items()}
    ema = {n: t.clone() for n, t in want.items()}
    m, v = ({n: torch.zeros_like(t) for n, t in want.items()} for _ in range(2))
    for t in (1, 2):
        grads = {n: torch.randn(p.shape, generator=g).cuda() for n, p in named.items()}
        opt.step(grads)
        for n in want:
            (want[n], _), (m[n], _), (v[n], _) = R.adamw(want[n], grads[n], m[n], v[n], t, 1e-3, 0.9, 0.999, 1e-8, 0.01 if want[n].dim() > 1 else 0.0)
            ema[n] = 0.5 * ema[n] + 0.5 * want[n]
    averaged = {**sd, **{n: t.cpu() for n, t in opt.ema_parameters().items()}}
    for n in ema:
        assert ema[n].numel() == 0 or (averaged[n].double() - ema[n]).abs().max() < 1e-6, n
    cfg = config.ModelConfig()
    graphs = synthetic.synthetic_pairs(5, 3, 16, 3, 12)
    batch = Batch.from_data_list(graphs)
    set_time_phore(batch, 0.65, 0.65, 0.65, batch.num_graphs)
    ref = OracleScoreModel(averaged, cfg, dtype=torch.float64, tables=load_tables())(batch)
    model = TensorProductScoreModel(device="cuda:0").load_state_dict(averaged)
    for a, b in zip(model(batch), ref):                                                    # the score model's own bound (test_forward_gpu.py)
        assert (a.double().cpu() - b.double().cpu()).abs().max() < 1e-5 * b.abs().max()


def test_what_is_no_tensor_or_plan_is_a_type_error():
    x = torch.zeros(2, 8, device="cuda")
    q = torch.zeros(2, 1, 8, device="cuda")
    plan = layers.PairPlan([0, 2], [0, 2])
    _, mean, rstd = layers.layer_norm_forward(x)
    out, stats = layers.attention_forward(q, q, q, plan)
    opt = optim.AdamW([x.clone()])
    for call in (lambda: layers.layer_norm_backward(x, x, None, rstd), lambda: layers.layer_norm_backward(x, x, mean, 1.0), lambda: layers.layer_norm_backward(None, x, mean, rstd),
                 lambda: layers.attention_backward(q, q, q, q, out, None, plan), lambda: layers.attention_backward(q, q, q, q, None, stats, plan),
                 lambda: layers.attention_forward(q, q, q, None), lambda: layers.attention_forward(q, q, q, ([0, 2], [0, 2])), lambda: opt.step([x], grad_scale=0.5)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: layers.layer_norm_backward(x, x, mean.cpu(), rstd), lambda: layers.attention_backward(q, q, q, q, out, stats.cpu(), plan)):
        with pytest.raises(ValueError):
            call()
    assert opt.state_dict()["step"] == 0
