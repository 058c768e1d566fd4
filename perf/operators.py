"""Cases for timing the training operators: layer norm, attention over packed complexes, AdamW - each in plain torch and through the framework.

`own` selects the side: False computes the operators with elementary torch operations in 32 bits (64 where the 8-bit code of a value next to a border
depends on it) and rounds once at the end; True makes the calls a program makes of `diffphore_amd.layers` and `diffphore_amd.optim`.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
LN_EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, WEIGHT_DECAY, EMA_DECAY, STEPS_DONE = 1e-3, 0.9, 0.999, 1e-8, 0.01, 0.999, 100
BLOCK = 256                                  # elements that share one scale of an 8-bit state; every tensor's slot is a multiple of it


# ----------------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # node features of the 40 samples of one 20-atom complex, ns = 20 channels: the smallest call, latency counts
        dict(name="ln_fwd_nodes", op="ln_fwd", rows=800, width=20, dtype="f32"),
        # token rows of a wide layer
        dict(name="ln_fwd_wide", op="ln_fwd", rows=16384, width=4096, dtype="bf16"),
        # 512 complexes of 30 atoms, the 3 ns = 60 hidden units of a radial network
        dict(name="ln_bwd_nodes", op="ln_bwd", rows=15360, width=60, dtype="f32"),
        # an odd number of rows of a wide layer in training
        dict(name="ln_bwd_wide", op="ln_bwd", rows=32749, width=2048, dtype="bf16"),
        # 40 samples of a 20-atom ligand against a pharmacophore of 79 nodes, a bias per pair: a small call of the sampler's shape
        dict(name="attn_fwd_complex", op="attn_fwd", dtype="f32", graphs=40, nq_lo=20, nq_hi=20, nk_lo=79, nk_hi=79, heads=4, kv_heads=4, dim=20,
             bias=True, causal=False, lens=1),
        # one new token of 24 requests against caches of up to 16384 positions, heads shared in fours
        dict(name="attn_fwd_token", op="attn_fwd", dtype="bf16", graphs=24, nq_lo=1, nq_hi=1, nk_lo=1500, nk_hi=16384, heads=32, kv_heads=8, dim=128,
             bias=False, causal=True, lens=2),
        # two long sequences, causal, heads shared in fours
        dict(name="attn_fwd_long", op="attn_fwd", dtype="bf16", graphs=2, nq_lo=4096, nq_hi=4096, nk_lo=4096, nk_hi=4096, heads=16, kv_heads=4, dim=128,
             bias=False, causal=True, lens=3),
        # a training batch of 512 complexes of 15 to 45 atoms against 16 to 48 pharmacophore nodes, a bias per pair and its gradient
        dict(name="attn_bwd_complex", op="attn_bwd", dtype="f32", graphs=512, nq_lo=15, nq_hi=45, nk_lo=16, nk_hi=48, heads=4, kv_heads=4, dim=20,
             bias=True, causal=False, lens=4),
        # ragged sequences of ordinary length, one key head for four query heads
        dict(name="attn_bwd_ragged", op="attn_bwd", dtype="bf16", graphs=48, nq_lo=33, nq_hi=700, nk_lo=1, nk_hi=900, heads=8, kv_heads=2, dim=64,
             bias=False, causal=False, lens=5),
        # the long sequences in training
        dict(name="attn_bwd_long", op="attn_bwd", dtype="bf16", graphs=2, nq_lo=4096, nq_hi=4096, nk_lo=4096, nk_hi=4096, heads=16, kv_heads=16, dim=128,
             bias=False, causal=True, lens=6),
        # the score model's own parameter list: 228 tensors, many of them a few numbers, with the running average of the weights
        dict(name="adamw_score_model", op="adamw", dtype="f32", state_bits=32, tensors=0, numel=0, ema=True, lens=7),
        # layers of a large model: bf16 parameters with 32-bit masters, states in 8 bits
        dict(name="adamw_wide_8bit", op="adamw", dtype="bf16", state_bits=8, tensors=48, numel=120_000_000, ema=False, lens=8),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "attn_fwd", "attn_bwd", "adamw"])
    dtype = rng.choice(["f32", "bf16"])
    if op in ("ln_fwd", "ln_bwd"):
        width = _log(rng, 4, 16384)                             # two entries have no direction left that the gradient could take
        return dict(op=op, rows=_log(rng, 1, max(1, min(100_000, 33_000_000 // width))), width=width, dtype=dtype)
    if op == "adamw":
        tensors = rng.choice([0, _log(rng, 1, 60)])
        return dict(op=op, dtype=dtype, state_bits=rng.choice([8, 32]), tensors=tensors, numel=_log(rng, max(1, 100 * tensors), 60_000_000) if tensors else 0,
                    ema=rng.random() < 0.5, lens=rng.randrange(1 << 20))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    dim = rng.choice([_log(rng, 5, 128), 16, 20, 32, 64, 128])
    shape = rng.choice(["complex", "ragged", "long", "token"])
    bias = rng.random() < {"complex": 0.8, "ragged": 0.3, "long": 0.1, "token": 0.2}[shape]
    if shape == "complex":
        graphs, nq, nk = _log(rng, 1, 512), _log(rng, 5, 80), _log(rng, 5, 96)
    elif shape == "ragged":
        graphs, nq, nk = _log(rng, 1, 48), _log(rng, 64, 1000), _log(rng, 64, 1000)
    elif shape == "long":
        graphs, nq = rng.choice([1, 2]), _log(rng, 1000, 4096)
        nk = nq if rng.random() < 0.6 else _log(rng, 1000, 4096)
    else:
        graphs, nq, nk = _log(rng, 1, 24), rng.choice([1, 1, 2, 5]), _log(rng, 100, 16384)
    if dtype == "f32" or bias:                                  # no drawn case costs more than the largest listed one
        while graphs * heads * nq * nk > 60_000_000 and (nk > 64 or graphs > 1):
            graphs, nq, nk = max(1, graphs // 2), max(1, nq * 2 // 3), max(1, nk * 2 // 3)
    whole = rng.random() < 0.3
    return dict(op=op, dtype=dtype, graphs=graphs, nq_lo=nq if whole else max(1, nq // 3), nq_hi=nq, nk_lo=nk if whole else max(1, nk // 3), nk_hi=nk,
                heads=heads, kv_heads=kv_heads, dim=dim, bias=bias, causal=rng.random() < 0.4, lens=rng.randrange(1 << 20))


def _lengths(case):
    r = random.Random(case["lens"])
    nq = [r.randint(case["nq_lo"], case["nq_hi"]) for _ in range(case["graphs"])]
    nk = [r.randint(case["nk_lo"], case["nk_hi"]) for _ in range(case["graphs"])]
    return nq, nk


def _score_model_sizes():
    """Element counts of the released score model's parameters: ns = 20, nv = 10, 4 layers, 6 convolution families, the embeddings and the heads."""
    ns, sizes = 20, []
    numel, bn = (600, 1100, 1600, 2200), ((30, 20), (40, 20), (60, 20), (60, 20))
    for width in (119, 4, 12, 12, 8, 10, 6, 6, 2, 8, 2, 2, 2, 2, 2, 2) + (11, 2, 2) + (2,) * 5:
        sizes.append(width * ns)                                                              # categorical embeddings
    for fan_in, fan_out in ((20, 20), (22, 20), (1, 20), (44, 20), (20, 20), (40, 20), (20, 20), (73, 20), (20, 20), (40, 20), (20, 20), (20, 20), (20, 20),
                            (20, 10), (10, 1), (1, 11), (11, 1), (33, 11), (11, 1), (21, 20), (20, 1), (21, 20), (20, 1)):
        sizes += [fan_in * fan_out, fan_out]
    for layer in range(4):
        for _ in range(6):
            sizes += [60 * 60, 60, 60 * numel[layer], numel[layer], bn[layer][0], bn[layer][1]]
    sizes += [40 * 40, 40, 40 * 200, 200, 4, 0, 60 * 60, 60, 60 * 1600, 1600, 40, 20, 800, 20]   # an empty one among them
    return sizes


def _sizes(case):
    if case["tensors"] == 0:
        return _score_model_sizes()
    r = random.Random(case["lens"])
    share = [math.exp(r.uniform(0.0, 5.0)) for _ in range(case["tensors"])]
    return [max(1, int(case["numel"] * s / sum(share))) for s in share]


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "ln_fwd":
        n = case["rows"] * case["width"]
        return {"bytes": 2 * n * e + 8 * case["rows"] + 2 * case["width"] * e, "flops": 8 * n}
    if case["op"] == "ln_bwd":
        n = case["rows"] * case["width"]
        return {"bytes": 3 * n * e + 8 * case["rows"] + 3 * case["width"] * e, "flops": 14 * n}
    if case["op"] == "adamw":
        n, states = sum(_sizes(case)), 16 if case["state_bits"] == 32 else 4 + 16 / BLOCK
        params = 8 if case["dtype"] == "f32" else 2 + 8                                        # bf16: the value is written, its 32-bit master read and written
        return {"bytes": n * (e + params + states + (8 if case["ema"] else 0)), "flops": 16 * n}
    nq, nk = _lengths(case)
    pairs = 0
    for a, b in zip(nq, nk):
        if not case["causal"]:
            pairs += a * b
        elif b >= a:
            pairs += a * (b - a) + a * (a + 1) // 2
        else:
            pairs += b * (b + 1) // 2
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    rows = (sum(nq) * h * 2 + sum(nk) * g * 2) * d * e + 8 * sum(nq) * h
    bias = sum(a * b for a, b in zip(nq, nk)) * h * e if case["bias"] else 0
    if case["op"] == "attn_fwd":
        return {"bytes": rows + bias, "flops": 4 * pairs * h * d}
    return {"bytes": rows + (sum(nq) * h * 2 + sum(nk) * g * 2) * d * e + 2 * bias, "flops": 10 * pairs * h * d}


# ----------------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------------
def _randn(gen, dtype, *shape, mean=0.0, std=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * std + mean).to(dtype)


def _offsets(n):
    out = [0]
    for x in n:
        out.append(out[-1] + x)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(op=case["op"], case=case)
    if case["op"] in ("ln_fwd", "ln_bwd"):
        rows, width = case["rows"], case["width"]
        s["x"] = _randn(gen, dtype, rows, width, mean=0.5, std=2.0)
        s["w"] = _randn(gen, dtype, width, mean=1.0, std=0.2)
        s["b"] = _randn(gen, dtype, width, std=0.2)
        if case["op"] == "ln_bwd":
            s["dy"] = _randn(gen, dtype, rows, width, std=0.1)
            s["mean"], s["rstd"] = _plain_stats(s["x"].float())
        return s
    if case["op"] == "adamw":
        return _prepare_adamw(case, gen, s)
    nq, nk = _lengths(case)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    s["q"] = _randn(gen, dtype, sum(nq), h, d)
    s["k"] = _randn(gen, dtype, sum(nk), g, d)
    s["v"] = _randn(gen, dtype, sum(nk), g, d)
    s["bias"] = _randn(gen, dtype, h, sum(a * b for a, b in zip(nq, nk))) if case["bias"] else None
    s["max_nq"], s["max_nk"] = max(nq), max(nk)
    s["nq"], s["nk"] = (torch.tensor(x, device="cuda") for x in (nq, nk))
    s["q_ptr"], s["k_ptr"] = (torch.tensor(_offsets(x), device="cuda") for x in (nq, nk))
    s["pair_ptr"] = torch.tensor(_offsets([a * b for a, b in zip(nq, nk)]), device="cuda")
    if case["op"] == "attn_bwd":
        s["dout"] = _randn(gen, dtype, sum(nq), h, d, std=0.1)
        s["out"], s["stats"] = _plain_attention(s)
    if own:
        from diffphore_amd.layers import PairPlan
        s["plan"] = PairPlan(_offsets(nq), _offsets(nk), "cuda")
    return s


def _prepare_adamw(case, gen, s):
    """Parameters of a run that is STEPS_DONE steps old.  The tensors are views of flat buffers, each slot rounded up to BLOCK elements; nothing in the
    padding is ever anything but 0."""
    sizes, dtype = _sizes(case), DTYPES[case["dtype"]]
    slots = [-(-n // BLOCK) * BLOCK for n in sizes]
    total, at = sum(slots), _offsets(slots)
    which = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"), torch.tensor(slots, device="cuda"), output_size=total)
    at_d, n_d = torch.tensor(at[:-1], device="cuda"), torch.tensor(sizes, device="cuda")
    live = (torch.arange(total, device="cuda") - at_d[which]) < n_d[which]
    level = torch.exp(torch.randn(len(sizes), generator=gen, device="cuda"))[which] * 1e-3       # gradients differ in size from tensor to tensor

    def values(std):
        return torch.where(live, torch.randn(total, generator=gen, device="cuda") * std, 0.0)
    s["master"] = values(0.05).to(dtype).float()
    s["param"] = s["master"].to(dtype) if case["dtype"] == "bf16" else s["master"]
    s["grad"] = values(level).to(dtype)
    s["m"], s["v"] = values(0.3 * level), values(level).square()
    s["ema"] = s["master"] + values(1e-4) if case["ema"] else None
    # one-dimensional parameters take no weight decay: here every third tensor
    s["decay"] = torch.where((which % 3 != 2)[::BLOCK], WEIGHT_DECAY, 0.0)
    s["step"] = STEPS_DONE
    if case["state_bits"] == 8:
        (s["m"], s["m_scale"]), (s["v"], s["v_scale"]) = _encode(s["m"].double(), 2), _encode(s["v"].double(), 4)
    if own:
        from diffphore_amd.optim import AdamW

        def tensors(flat):
            return [flat[a:a + n] for a, n in zip(at, sizes)]
        opt = AdamW(tensors(s["param"]), lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=WEIGHT_DECAY, no_decay=range(2, len(sizes), 3),
                    state_bits=case["state_bits"], ema_decay=EMA_DECAY if case["ema"] else None)
        opt.load_state_dict({"step": STEPS_DONE, "state_bits": case["state_bits"], "master": s["master"] if case["dtype"] == "bf16" else None, "ema": s["ema"], "exp_avg": s["m"],
                             "exp_avg_sq": s["v"], "exp_avg_scale": s.get("m_scale"), "exp_avg_sq_scale": s.get("v_scale")})
        s["opt"], s["grads"] = opt, tensors(s["grad"])
    return s


# ----------------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["op"]
    if own:
        from diffphore_amd import layers
        if op == "ln_fwd":
            return layers.layer_norm_forward(s["x"], s["w"], s["b"], LN_EPS)
        if op == "ln_bwd":
            return layers.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["w"])
        if op == "attn_fwd":
            return layers.attention_forward(s["q"], s["k"], s["v"], s["plan"], bias=s["bias"], causal=s["case"]["causal"])
        if op == "attn_bwd":
            return layers.attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["stats"], s["plan"], bias=s["bias"], causal=s["case"]["causal"])
        opt = s["opt"]
        opt.step(s["grads"])
        m, v = opt.moments()
        return s["param"], opt.master, m, v, opt.ema
    if op == "ln_fwd":
        x = s["x"].float()
        mean, rstd = _plain_stats(x)
        y = _centred(x, mean) * rstd[:, None] * s["w"].float() + s["b"].float()
        return y.to(s["x"].dtype), mean, rstd
    if op == "ln_bwd":
        dy, xh = s["dy"].float(), _centred(s["x"].float(), s["mean"]) * s["rstd"][:, None]
        g = dy * s["w"].float()
        dx = (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True)) * s["rstd"][:, None]
        return dx.to(s["x"].dtype), (dy * xh).sum(0).to(s["w"].dtype), dy.sum(0).to(s["w"].dtype)
    if op == "attn_fwd":
        return _plain_attention(s)
    if op == "attn_bwd":
        return _plain_attention_backward(s)
    return _plain_adamw(s)


def _centred(x, mean):
    """x - mean, less what the mean's own rounding leaves (rows whose entries are close together would show it)."""
    d = x - mean[:, None]
    return d - d.mean(1, keepdim=True)


def _plain_stats(x):
    mean = x.mean(1)
    mean = mean + (x - mean[:, None]).mean(1)
    return mean, (_centred(x, mean).square().mean(1) + LN_EPS).rsqrt()


def _padded(x, ptr, n, most):
    """Rows of a packed [N, heads, dim] tensor as [graphs, heads, most, dim] in 32 bits, 0 behind each graph's last row."""
    i = torch.arange(most, device=x.device)
    live = i < n[:, None]
    at = torch.where(live, ptr[:-1, None] + i, 0)
    return (x.float()[at] * live[:, :, None, None]).transpose(1, 2)


def _packed(x, ptr, n, total):
    """The inverse of _padded."""
    b = torch.repeat_interleave(torch.arange(len(n), device=x.device), n, output_size=total)
    return x[b, :, torch.arange(total, device=x.device) - ptr[b]]


def _pairs(s, total):
    """(graph, query, key) of every pair."""
    b = torch.repeat_interleave(torch.arange(len(s["nq"]), device="cuda"), s["nq"] * s["nk"], output_size=total)
    at = torch.arange(total, device="cuda") - s["pair_ptr"][b]
    return b, at // s["nk"][b], at % s["nk"][b]


def _scores(s, q, k):
    """Masked logits [graphs, key heads, heads per key head, queries, keys]."""
    c = s["case"]
    x = (q.flatten(2, 3) @ k.transpose(2, 3)).unflatten(2, q.shape[2:4]) * (1.0 / math.sqrt(c["dim"]))
    if s["bias"] is not None:
        b, i, j = _pairs(s, s["bias"].shape[1])
        full = torch.zeros(c["graphs"], s["max_nq"], s["max_nk"], c["heads"], device="cuda")
        full[b, i, j] = s["bias"].float().t()
        x = x + full.permute(0, 3, 1, 2).reshape(x.shape)
    j, i = torch.arange(s["max_nk"], device="cuda"), torch.arange(s["max_nq"], device="cuda")
    seen = (j < s["nk"][:, None])[:, None]
    if c["causal"]:
        seen = seen & (j <= i[:, None] + (s["nk"] - s["nq"])[:, None, None])
    return torch.where(seen[:, None, None], x, -math.inf)


def _plain_attention(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    q = _padded(s["q"], s["q_ptr"], s["nq"], s["max_nq"]).unflatten(1, (c["kv_heads"], group))
    k, v = (_padded(s[n], s["k_ptr"], s["nk"], s["max_nk"]) for n in "kv")
    x = _scores(s, q, k)
    m = x.amax(-1)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m)[..., None])
    total = p.sum(-1)
    o = (p.flatten(2, 3) @ v).unflatten(2, (group, s["max_nq"])) / torch.where(total == 0, 1.0, total)[..., None]
    n = s["q"].shape[0]
    stats = _packed(torch.stack((m, total), -1).flatten(1, 2), s["q_ptr"], s["nq"], n)
    return _packed(o.flatten(1, 2), s["q_ptr"], s["nq"], n).to(s["q"].dtype), stats.permute(2, 1, 0).contiguous()


def _plain_attention_backward(s):
    c = s["case"]
    group, scale = c["heads"] // c["kv_heads"], 1.0 / math.sqrt(c["dim"])
    q, do = (_padded(s[n], s["q_ptr"], s["nq"], s["max_nq"]).unflatten(1, (c["kv_heads"], group)) for n in ("q", "dout"))
    k, v = (_padded(s[n], s["k_ptr"], s["nk"], s["max_nk"]) for n in "kv")
    stats = _padded(s["stats"].permute(2, 1, 0), s["q_ptr"], s["nq"], s["max_nq"]).unflatten(1, (c["kv_heads"], group))
    m, total = stats[..., 0], stats[..., 1]
    p = torch.exp(_scores(s, q, k) - torch.where(m == -math.inf, 0.0, m)[..., None]) / torch.where(total == 0, 1.0, total)[..., None]
    p, do2, q2 = p.flatten(2, 3), do.flatten(2, 3), q.flatten(2, 3)
    dv = p.transpose(2, 3) @ do2
    ds = do2 @ v.transpose(2, 3)
    ds = p * (ds - (p * ds).sum(-1, keepdim=True))
    dq = (ds @ k).unflatten(2, q.shape[2:4]).flatten(1, 2) * scale
    dk = (ds.transpose(2, 3) @ q2) * scale
    dbias = None
    if s["bias"] is not None:
        b, i, j = _pairs(s, s["bias"].shape[1])
        dbias = ds.unflatten(2, (group, s["max_nq"])).flatten(1, 2)[b, :, i, j].t().contiguous().to(s["bias"].dtype)
    dtype, nq, nk = s["q"].dtype, s["q"].shape[0], s["k"].shape[0]
    return (_packed(dq, s["q_ptr"], s["nq"], nq).to(dtype), _packed(dk, s["k_ptr"], s["nk"], nk).to(dtype),
            _packed(dv, s["k_ptr"], s["nk"], nk).to(dtype), dbias)


def _decode(code, scale, power):
    """Values (64 bits) of 8-bit codes: scale (c/127)|c/127| for power 2, scale (c/255)^4 for power 4."""
    c = code.double().view(-1, BLOCK)
    x = c * c.abs() / 127.0 ** 2 if power == 2 else (c / 255.0).square().square()
    return (x * scale.double()[:, None]).view(-1)


def _encode(x, power):
    """Nearest codes on the curve's own axis, one 32-bit scale (the largest magnitude) per block; a positive second moment never becomes 0."""
    x = x.view(-1, BLOCK)
    scale = x.abs().amax(1).float()
    u = torch.where(scale[:, None] > 0, x.abs() / scale.double()[:, None], 0.0)
    if power == 2:
        return (torch.floor(u.sqrt() * 127.0 + 0.5).clamp(max=127.0) * x.sign()).to(torch.int8).view(-1), scale
    c = torch.floor(u.sqrt().sqrt() * 255.0 + 0.5).clamp(max=255.0)
    return torch.where((u > 0) & (c < 1), 1.0, c).to(torch.uint8).view(-1), scale


def _plain_adamw(s):
    s["step"] += 1
    small = s["case"]["state_bits"] == 8
    g, m, v = s["grad"].float(), s["m"], s["v"]
    if small:                                  # 64 bits: the new codes are taken next to the borders between them
        g, m, v = g.double(), _decode(m, s["m_scale"], 2), _decode(v, s["v_scale"], 4)
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + g * g * (1.0 - BETA2)
    c1, c2 = 1.0 - BETA1 ** s["step"], 1.0 - BETA2 ** s["step"]
    p = s["master"].view(-1, BLOCK)
    step = (m / c1 / ((v / c2).sqrt() + ADAM_EPS) * LR).view(-1, BLOCK)
    s["master"] = (p * (1.0 - LR * s["decay"])[:, None] - step).float().view(-1)
    s["param"] = s["master"].to(s["param"].dtype)
    if s["ema"] is not None:
        s["ema"] = s["ema"] * EMA_DECAY + s["master"] * (1.0 - EMA_DECAY)
    if small:
        (s["m"], s["m_scale"]), (s["v"], s["v_scale"]) = _encode(m, 2), _encode(v, 4)
        m, v = _decode(s["m"], s["m_scale"], 2).float(), _decode(s["v"], s["v_scale"], 4).float()
    else:
        s["m"], s["v"] = m, v
    return s["param"], s["master"] if s["case"]["dtype"] == "bf16" else None, m, v, s["ema"]


# ----------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, graph by graph
# ----------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("ln_fwd", "ln_bwd"):
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = 1.0 / (var + LN_EPS).sqrt()
        if case["op"] == "ln_fwd":
            return torch.addcmul(s["b"].double(), (x - mean[:, None]) * rstd[:, None], s["w"].double()), mean, rstd
        dy, w, n = s["dy"].double(), s["w"].double(), case["width"]
        r = rstd[:, None]
        centred = x - mean[:, None]
        dx = r * w * dy - r / n * (dy @ w)[:, None] - r ** 3 / n * centred * ((dy * centred) @ w)[:, None]
        return dx, torch.einsum("rc,rc->c", dy, centred * r), dy.sum(0)
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    nq, nk = _lengths(case)
    if case["heads"] * sum(a * b for a, b in zip(nq, nk)) * case["dim"] > 3e11:
        return None
    q, k, v = (s[n].double() for n in "qkv")
    group, back = case["heads"] // case["kv_heads"], case["op"] == "attn_bwd"
    do = s["dout"].double() if back else None
    out, stats = torch.zeros_like(q), torch.zeros(2, case["heads"], q.shape[0], dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v))
    dbias = torch.zeros(s["bias"].shape, dtype=torch.float64, device="cuda") if case["bias"] else None
    for b, (a, n) in enumerate(zip(nq, nk)):
        i0, j0, p0 = (int(s[name][b]) for name in ("q_ptr", "k_ptr", "pair_ptr"))
        rows, cols = slice(i0, i0 + a), slice(j0, j0 + n)
        heads = range(0, case["heads"], group) if a * n > 1 << 20 else [None]
        for h0 in heads:
            hs = slice(None) if h0 is None else slice(h0, h0 + group)
            gs = slice(None) if h0 is None else slice(h0 // group, h0 // group + 1)
            qb = q[rows, hs].permute(1, 0, 2).contiguous()
            kb, vb = (x[cols, gs].permute(1, 0, 2).repeat_interleave(group, 0).contiguous() for x in (k, v))
            x = torch.matmul(qb, kb.mT.contiguous()) / math.sqrt(case["dim"])
            if case["bias"]:
                x += s["bias"][hs, p0:p0 + a * n].double().view(-1, a, n)
            if case["causal"]:
                x.masked_fill_(torch.ones(a, n, dtype=torch.bool, device="cuda").triu(n - a + 1), -math.inf)
            top = x.max(-1).values
            e = torch.exp(x - top.clamp(min=-1e300)[..., None])
            stats[0, hs, rows], stats[1, hs, rows] = top, e.sum(-1)
            e /= e.sum(-1, keepdim=True).clamp(min=1e-300)
            if not back:
                out[rows, hs] = torch.matmul(e, vb).permute(1, 0, 2)
                continue
            dob = do[rows, hs].permute(1, 0, 2).contiguous()
            de = torch.matmul(dob, vb.mT.contiguous())
            dx = e * (de - (dob * torch.matmul(e, vb)).sum(-1, keepdim=True))
            dq[rows, hs] = torch.matmul(dx, kb).permute(1, 0, 2) / math.sqrt(case["dim"])
            for total, part in ((dk, torch.matmul(dx.mT.contiguous(), qb) / math.sqrt(case["dim"])), (dv, torch.matmul(e.mT.contiguous(), dob))):
                total[cols, gs] = part.view(-1, group, n, case["dim"]).sum(1).permute(1, 0, 2)
            if case["bias"]:
                dbias[hs, p0:p0 + a * n] = dx.reshape(-1, a * n)
    return (dq, dk, dv, dbias) if back else (out, stats)


def _exact_adamw(case, s):
    g, p, t = s["grad"].double(), s["master"].double(), STEPS_DONE + 1
    small = case["state_bits"] == 8
    m, v = (_decode(s["m"], s["m_scale"], 2), _decode(s["v"], s["v_scale"], 4)) if small else (s["m"].double(), s["v"].double())
    m, v = torch.lerp(g, m, BETA1), torch.lerp(g ** 2, v, BETA2)
    decay = torch.repeat_interleave(s["decay"].double(), BLOCK)
    new = p - LR * decay * p - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + ADAM_EPS)
    ema = None if s["ema"] is None else torch.lerp(new, s["ema"].double(), EMA_DECAY)
    if small:
        m, v = _nearest(m, 127, 2), _nearest(v, 255, 4)
    return new, new if case["dtype"] == "bf16" else None, m, v, ema


def _nearest(x, top, power):
    """The value that stands for each entry: the table's entry whose root is nearest to the root of the entry's share of its block's largest."""
    x = x.view(-1, BLOCK)
    scale = x.abs().max(1).values.float().double()[:, None]
    table = torch.arange(top + 1, dtype=torch.float64, device="cuda") / top
    between = ((torch.arange(top, dtype=torch.float64, device="cuda") + 0.5) / top) ** power
    share = torch.where(scale > 0, x.abs() / scale, torch.zeros_like(x))
    at = torch.bucketize(share, between, right=True)
    if power == 4:
        at = torch.where((share > 0) & (at == 0), 1, at)
    return (torch.sign(x) * table[at] ** power * scale).view(-1)
