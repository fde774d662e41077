"""Operators of language models whose performance is followed: the fully connected layer with its epilogue, the norms
around a block with its gate and residual sum, and the clipped policy loss, forward and backward.

``run`` computes them in their plain form, in elementary torch operations, or - where ``own`` is true - through
portdnn_b200.api.  ``listed()`` names the cases that are followed, ``draw()`` gives further ones of the same ranges.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # serving: one token through the down projection of a block, where latency and the weight's bytes are all
        {"name": "linear_one_token", "kind": "linear", "m": 1, "k": 4096, "n": 4096, "weight": "out_in", "act": "silu",
         "bias": True, "residual": True, "save": False, "scale": 1.0, "dtype": "bf16"},
        # the fully connected layer at the end of the classifiers here: 250 images, 2048 features, 1000 classes
        {"name": "linear_classifier_head", "kind": "linear", "m": 250, "k": 2048, "n": 1000, "weight": "in_out",
         "act": "none", "bias": True, "residual": False, "save": False, "scale": 1.0, "dtype": "f16"},
        # training: the up projection of a block over 8192 tokens, which keeps its pre-activation for the backward pass
        {"name": "linear_up_train", "kind": "linear", "m": 8192, "k": 2048, "n": 8192, "weight": "in_out", "act": "gelu",
         "bias": True, "residual": False, "save": True, "scale": 1.0, "dtype": "bf16"},
        # single precision, nothing a multiple of anything
        {"name": "linear_ragged_f32", "kind": "linear", "m": 1003, "k": 515, "n": 777, "weight": "in_out", "act": "tanh",
         "bias": True, "residual": True, "save": True, "scale": 0.5, "dtype": "f32"},
        # gradients of the up projection: a ragged number of tokens, all three gradients
        {"name": "linear_grad_up", "kind": "linear_grad", "m": 4101, "k": 2048, "n": 8192, "weight": "in_out", "act": "gelu",
         "input_act": "none", "scale": 1.0, "dtype": "bf16"},
        # gradients of the down projection, the one with respect to its input through the activation before it
        {"name": "linear_grad_down", "kind": "linear_grad", "m": 2000, "k": 4096, "n": 1024, "weight": "out_in", "act": "none",
         "input_act": "relu", "scale": 0.7, "dtype": "f16"},
        # serving: the norms around a block for a handful of tokens
        {"name": "norm_few_tokens", "kind": "norm", "rows": 4, "channels": 4096, "post": "rms", "pre": "rms", "gate": 1,
         "gate_act": "none", "scale": 1.0, "dtype": "bf16"},
        # training: both norms, a gate to each of eight sequences
        {"name": "norm_train", "kind": "norm", "rows": 16384, "channels": 4096, "post": "rms", "pre": "rms", "gate": 8,
         "gate_act": "tanh", "scale": 1.0, "dtype": "bf16"},
        # their gradients
        {"name": "norm_grad_train", "kind": "norm_grad", "rows": 8192, "channels": 2048, "post": "rms", "pre": "rms", "gate": 8,
         "gate_act": "tanh", "scale": 1.0, "dtype": "bf16"},
        # layer norms in single precision on an odd width, a scale to each channel
        {"name": "norm_grad_ragged_f32", "kind": "norm_grad", "rows": 1999, "channels": 1003, "post": "layer", "pre": "layer",
         "gate": 1, "gate_act": "none", "scale": 0.3, "dtype": "f32"},
        # the loss of a short answer over a small vocabulary, in single precision
        {"name": "loss_short_f32", "kind": "loss", "rows": 61, "vocab": 1000, "pitch": 1000, "masked": 0.25, "kl": 0.05,
         "temperature": 1.0, "dtype": "f32"},
        # the loss of a training step: answers behind masked prompts, an odd vocabulary in rows of whole packets
        {"name": "loss_train", "kind": "loss", "rows": 6000, "vocab": 50001, "pitch": 50048, "masked": 0.25, "kl": 0.02,
         "temperature": 1.2, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: the kind first, then its sizes over the logarithm of their range."""
    kind = rng.choice(["linear", "linear", "linear_grad", "linear_grad", "norm", "norm_grad", "loss"])
    half = rng.choice(["f16", "bf16", "bf16"])
    acts = ["none", "relu", "gelu", "silu", "tanh", "relu6"]
    if kind in ("linear", "linear_grad"):
        dtype = rng.choice([half, half, half, "f32"])
        k, n = _log(rng, 64, 8192), _log(rng, 64, 8192)
        if rng.random() < 0.6:  # widths as models mostly have them
            k, n = (k + 63) // 64 * 64, (n + 63) // 64 * 64
        most = (1.2e11 if kind == "linear" else 6e10) / (k * n) / (8 if dtype == "f32" else 1)
        case = {"kind": kind, "m": _log(rng, 1, max(1, min(8192, int(most)))), "k": k, "n": n,
                "weight": rng.choice(["in_out", "out_in"]), "act": rng.choice(acts), "scale": rng.choice([1.0, 1.0, 0.5]),
                "dtype": dtype}
        if kind == "linear":
            case.update(bias=rng.random() < 0.7, residual=rng.random() < 0.5, save=rng.random() < 0.4)
        else:
            case.update(input_act=rng.choice(["none", "relu", "gelu", "silu"]))
        return case
    if kind in ("norm", "norm_grad"):
        dtype = rng.choice([half, half, "f32"])
        channels = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            channels = (channels + 31) // 32 * 32
        most = (5e7 if kind == "norm" else 1.5e7) / channels
        gates = rng.choice([0, 1, 1, 4, 8])
        rows = _log(rng, 1, max(2, min(20000, int(most))))
        rows = max(rows // max(gates, 1), 1) * max(gates, 1)
        return {"kind": kind, "rows": rows, "channels": channels, "post": rng.choice(["rms", "layer", "none"]),
                "pre": rng.choice(["rms", "layer"]), "gate": gates, "gate_act": rng.choice(["none", "tanh", "sigmoid"]),
                "scale": rng.choice([1.0, 0.5]), "dtype": dtype}
    dtype = rng.choice([half, half, "f32"])
    vocab = _log(rng, 100, 130000)
    pitch = vocab if rng.random() < 0.4 else (vocab + 63) // 64 * 64
    return {"kind": "loss", "rows": _log(rng, 1, max(2, min(8000, int(1.4e8 / vocab)))), "vocab": vocab, "pitch": pitch,
            "masked": rng.choice([0.0, 0.25, 0.5]), "kl": rng.choice([0.0, 0.02, 0.1]),
            "temperature": rng.choice([1.0, 0.8]), "dtype": dtype}


# ---- inputs --------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dt)

    s = {"case": case}
    if case["kind"] in ("linear", "linear_grad"):
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = normal(m, k)
        s["w"] = normal(*((n, k) if case["weight"] == "out_in" else (k, n)), std=k ** -0.5)
        if case["kind"] == "linear":
            s["bias"] = normal(n, std=0.3) if case["bias"] else None
            s["residual"] = normal(m, n) if case["residual"] else None
        else:
            s["dy"] = normal(m, n, std=0.5)
            s["pre"] = normal(m, n) if case["act"] != "none" else None
            s["input_pre"] = None
            if case["input_act"] != "none":  # the layer's input is what the activation made of it
                s["input_pre"] = normal(m, k)
                s["x"] = _act(case["input_act"], s["input_pre"].float()).to(dt)
        return s
    if case["kind"] in ("norm", "norm_grad"):
        rows, c = case["rows"], case["channels"]
        # branches come out of projections at any size; the residual stream is several times as large
        s["branch"] = normal(rows, c, std=0.8, mean=0.1)
        s["residual"] = normal(rows, c, std=3.0)
        s["gate"] = normal(case["gate"], c, std=0.5, mean=0.5) if case["gate"] else None
        for which in ("post", "pre"):
            kind = case[which]
            s[which + "_gamma"] = normal(c, std=0.2, mean=1.0) if kind != "none" else None
            s[which + "_beta"] = normal(c, std=0.1) if kind == "layer" else None
        if case["kind"] == "norm_grad":
            s["d_sum"], s["d_out"] = normal(rows, c, std=0.5), normal(rows, c, std=0.5)
            total, _, statistics = _norm_plain(s)
            s["sum"], s["statistics"] = total, statistics
        return s
    rows, vocab, pitch = case["rows"], case["vocab"], case["pitch"]
    whole = torch.randn((rows, pitch), generator=g, device="cuda").mul_(2.0).to(dt)
    s["logits"] = whole[:, :vocab]
    s["targets"] = torch.randint(vocab, (rows,), generator=g, device="cuda")
    at = torch.arange(rows, device="cuda")
    # most sampled tokens are likely ones
    s["logits"][at, s["targets"]] += (torch.rand(rows, generator=g, device="cuda") * 12).to(dt)
    x = s["logits"].float() / case["temperature"]
    lp = x[at, s["targets"]] - torch.logsumexp(x, 1)
    s["old"] = lp + 0.15 * torch.randn(rows, generator=g, device="cuda")
    s["ref"] = lp + 0.3 * torch.randn(rows, generator=g, device="cuda") if case["kl"] else None
    s["advantages"] = torch.randn(rows, generator=g, device="cuda")
    keep = (torch.rand(rows, generator=g, device="cuda") >= case["masked"]).float()
    s["weights"] = keep / keep.sum().clamp(min=1.0)
    return s


# ---- the plain form ------------------------------------------------------------------------------


def _act(name, z):
    if name == "relu":
        return z.clamp(min=0)
    if name == "relu6":
        return z.clamp(min=0, max=6)
    if name == "tanh":
        return torch.tanh(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z


def _act_grad(name, z):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "relu6":
        return ((z > 0) & (z < 6)).to(z.dtype)
    if name == "tanh":
        return 1 - torch.tanh(z) ** 2
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if name == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 - s)
    return torch.ones_like(z)


def _f(t):
    return None if t is None else t.float()


def _linear_plain(s):
    c, dt = s["case"], s["x"].dtype
    w = s["w"].float()
    z = s["x"].float() @ (w.t() if c["weight"] == "out_in" else w)
    if s["bias"] is not None:
        z = z + s["bias"].float()
    out = c["scale"] * _act(c["act"], z)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return {"out": out.to(dt), "pre": z.to(dt)} if c["save"] else {"out": out.to(dt)}


def _linear_grad_plain(s):
    c, dt = s["case"], s["x"].dtype
    dz = c["scale"] * s["dy"].float()
    if s["pre"] is not None:
        dz = dz * _act_grad(c["act"], s["pre"].float())
    w, x = s["w"].float(), s["x"].float()
    if c["weight"] == "out_in":
        dx, dw = dz @ w, dz.t() @ x
    else:
        dx, dw = dz @ w.t(), x.t() @ dz
    if s["input_pre"] is not None:
        dx = dx * _act_grad(c["input_act"], s["input_pre"].float())
    return {"dx": dx.to(dt), "dw": dw.to(dt), "db": dz.sum(0).to(dt)}


EPSILON = 1e-5


def _normalise(kind, v, gamma, beta):
    """(result, mean, reciprocal deviation)"""
    rows = v.shape[0]
    if kind == "none":
        return v, torch.zeros(rows, device=v.device), torch.ones(rows, device=v.device)
    mean = v.mean(1) if kind == "layer" else torch.zeros(rows, device=v.device)
    centred = v - mean[:, None]
    r = 1 / torch.sqrt((centred * centred).mean(1) + EPSILON)
    out = centred * r[:, None] * gamma
    return (out + beta if beta is not None else out), mean, r


def _norm_plain(s):
    c, dt = s["case"], s["branch"].dtype
    n, mean1, r1 = _normalise(c["post"], s["branch"].float(), _f(s["post_gamma"]), _f(s["post_beta"]))
    if s["gate"] is not None:
        a = _act(c["gate_act"], s["gate"].float())
        n = (n.view(a.shape[0], -1, a.shape[1]) * a[:, None]).view(n.shape)
    total = s["residual"].float() + c["scale"] * n
    out, mean2, r2 = _normalise(c["pre"], total, _f(s["pre_gamma"]), _f(s["pre_beta"]))
    return total.to(dt), out.to(dt), torch.stack([mean1, r1, mean2, r2])


def _normalise_grad(kind, v, mean, r, gamma, g):
    """(dv, dgamma, dbeta)"""
    if kind == "none":
        return g, None, None
    hat = (v - mean[:, None]) * r[:, None]
    u = g * gamma
    inner = u - hat * (u * hat).mean(1, keepdim=True)
    if kind == "layer":
        inner = inner - u.mean(1, keepdim=True)
    return inner * r[:, None], (g * hat).sum(0), g.sum(0) if kind == "layer" else None


def _norm_grad_plain(s):
    c, dt = s["case"], s["branch"].dtype
    mean1, r1, mean2, r2 = s["statistics"]
    dv, d_pre_gamma, d_pre_beta = _normalise_grad(c["pre"], s["sum"].float(), mean2, r2, _f(s["pre_gamma"]), s["d_out"].float())
    d_sum = s["d_sum"].float() + dv
    d_normed, d_gate = c["scale"] * d_sum, None
    f = s["branch"].float()
    if s["gate"] is not None:
        gate = s["gate"].float()
        n = f
        if c["post"] != "none":
            n = (f - mean1[:, None]) * r1[:, None] * s["post_gamma"].float()
            n = n + s["post_beta"].float() if s["post_beta"] is not None else n
        groups = (gate.shape[0], -1, gate.shape[1])
        d_gate = (d_normed * n).view(groups).sum(1) * _act_grad(c["gate_act"], gate)
        d_normed = (d_normed.view(groups) * _act(c["gate_act"], gate)[:, None]).view(f.shape)
    df, d_post_gamma, d_post_beta = _normalise_grad(c["post"], f, mean1, r1, _f(s["post_gamma"]), d_normed)
    named = {"branch": df, "residual": d_sum, "post_gamma": d_post_gamma, "post_beta": d_post_beta, "gate": d_gate,
             "pre_gamma": d_pre_gamma, "pre_beta": d_pre_beta}
    return {k: v.to(dt) for k, v in named.items() if v is not None}


CLIP_LOW, CLIP_HIGH, GRAD_SCALE = 0.2, 0.28, 1.0


def _loss_plain(s):
    c = s["case"]
    x = s["logits"].float() / c["temperature"]
    rows = torch.arange(x.shape[0], device=x.device)
    top = x.max(1, keepdim=True).values
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    live = s["weights"] != 0
    lp = torch.where(live, (x[rows, s["targets"]] - top[:, 0]) - torch.log(total[:, 0]), 0.0)
    ratio, a = torch.exp(lp - s["old"]), s["advantages"]
    free, clipped = ratio * a, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a
    loss = -torch.minimum(free, clipped)
    slope = torch.where(free <= clipped, -free, 0.0)
    if s["ref"] is not None:
        d = s["ref"] - lp
        loss = loss + c["kl"] * (torch.exp(d) - d - 1)
        slope = slope + c["kl"] * (1 - torch.exp(d))
    token_loss = torch.where(live, s["weights"] * loss, 0.0)
    slope = torch.where(live, s["weights"] * slope, 0.0) * (GRAD_SCALE / c["temperature"])
    grad = e.div_(total).mul_(-slope[:, None])
    grad[rows, s["targets"]] += slope
    return {"loss": token_loss.sum(), "token_loss": token_loss, "logp": lp, "grad": grad.to(s["logits"].dtype)}


# ---- one pass ------------------------------------------------------------------------------------


def run(state):
    c = state["case"]
    if not own:
        if c["kind"] == "linear":
            return _linear_plain(state)
        if c["kind"] == "linear_grad":
            return _linear_grad_plain(state)
        if c["kind"] == "norm":
            total, out, statistics = _norm_plain(state)
            return {"sum": total, "out": out, "statistics": statistics}
        return _norm_grad_plain(state) if c["kind"] == "norm_grad" else _loss_plain(state)

    from portdnn_b200 import api
    acts = {"none": api.ACT_NONE, "relu": api.ACT_RELU, "tanh": api.ACT_TANH, "relu6": api.ACT_RELU6}
    if c["kind"] == "linear":
        acts.update(gelu=api.ACT_GELU, silu=api.ACT_SILU)
        pre = torch.empty((c["m"], c["n"]), dtype=state["x"].dtype, device="cuda") if c["save"] else None
        out = api.matmul_fused(state["x"], state["w"], transpose_rhs=c["weight"] == "out_in", bias=state["bias"],
                               activation=acts[c["act"]], residual=state["residual"], scale=c["scale"], pre_activation=pre)
        return {"out": out, "pre": pre} if c["save"] else {"out": out}
    if c["kind"] == "linear_grad":
        acts.update(gelu=api.ACT_GELU, silu=api.ACT_SILU)
        dx, dw, db = api.matmul_fused_grad(state["dy"], state["x"], state["w"], transpose_rhs=c["weight"] == "out_in",
                                           activation=acts[c["act"]], pre_activation=state["pre"], scale=c["scale"],
                                           input_activation=acts[c["input_act"]], input_pre_activation=state["input_pre"])
        return {"dx": dx, "dw": dw, "db": db}
    if c["kind"] in ("norm", "norm_grad"):
        acts.update(sigmoid=api.ACT_SIGMOID)
        kinds = {"none": api.NORM_NONE, "rms": api.NORM_RMS, "layer": api.NORM_LAYER}
        p = api.residual_norm_params(c["rows"], c["channels"], post_norm=kinds[c["post"]], pre_norm=kinds[c["pre"]],
                                     gate_groups=c["gate"], gate_activation=acts[c["gate_act"]], scale=c["scale"],
                                     epsilon=EPSILON)
        if c["kind"] == "norm":
            total, out, statistics = api.residual_norm(
                state["branch"], state["residual"], p, post_gamma=state["post_gamma"], post_beta=state["post_beta"],
                gate=state["gate"], pre_gamma=state["pre_gamma"], pre_beta=state["pre_beta"])
            return {"sum": total, "out": out, "statistics": statistics}
        grads = api.residual_norm_grad(
            state["d_sum"], state["d_out"], state["branch"], state["sum"], state["statistics"], p,
            post_gamma=state["post_gamma"], post_beta=state["post_beta"], gate=state["gate"], pre_gamma=state["pre_gamma"],
            pre_beta=state["pre_beta"])
        names = ("branch", "residual", "post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta")
        return {k: v for k, v in zip(names, grads) if v is not None}
    loss, token_loss, logp, grad = api.policy_loss(
        state["logits"], state["targets"], state["advantages"], old_logp=state["old"], ref_logp=state["ref"],
        weights=state["weights"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl=c["kl"], temperature=c["temperature"],
        grad_scale=GRAD_SCALE)
    return {"loss": loss, "token_loss": token_loss, "logp": logp, "grad": grad}


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        tensors = 1 + bool(case["residual"]) + bool(case["save"])
        return {"bytes": es * (m * k + k * n + tensors * m * n + (n if case["bias"] else 0)), "flops": 2 * m * k * n}
    if case["kind"] == "linear_grad":
        m, k, n = case["m"], case["k"], case["n"]
        rows = n * (1 + (case["act"] != "none")) + k * (2 + (case["input_act"] != "none"))
        return {"bytes": es * (m * rows + 2 * k * n + n), "flops": 4 * m * k * n}
    if case["kind"] in ("norm", "norm_grad"):
        rows, c = case["rows"], case["channels"]
        vectors = case["gate"] + sum({"none": 0, "rms": 1, "layer": 2}[case[w]] for w in ("post", "pre"))
        if case["kind"] == "norm":
            return {"bytes": es * (4 * rows * c + vectors * c) + 16 * rows, "flops": 12 * rows * c}
        return {"bytes": es * (6 * rows * c + 2 * vectors * c) + 16 * rows, "flops": 30 * rows * c}
    rows, vocab = case["rows"], case["vocab"]
    live = round(rows * (1 - case["masked"]))  # a row of weight 0 needs no logit
    return {"bytes": es * vocab * (live + rows) + 36 * rows, "flops": 8 * vocab * live}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def _exact_activation(name, z):
    """(value, derivative)"""
    zero, one = torch.zeros_like(z), torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, zero), torch.where(z > 0, one, zero)
    if name == "relu6":
        return torch.where(z > 0, torch.where(z < 6, z, 6 * one), zero), torch.where((z > 0) & (z < 6), one, zero)
    if name == "tanh":
        t = 1 - 2 / (torch.exp(2 * z) + 1)
        return t, (1 - t) * (1 + t)
    if name == "sigmoid":
        e = torch.exp(-z)
        return 1 / (1 + e), e / (1 + e) ** 2
    if name == "silu":
        e = torch.exp(-z)
        return z / (1 + e), (1 + e + z * e) / (1 + e) ** 2
    if name == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, one


def exact(case, seed):
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in prepare(case, seed).items()}
    if case["kind"] == "linear":
        w = s["w"] if case["weight"] == "in_out" else s["w"].t()
        z = torch.mm(s["x"], w)
        z = z if s["bias"] is None else z + s["bias"]
        out = _exact_activation(case["act"], z)[0] * case["scale"]
        out = out if s["residual"] is None else out + s["residual"]
        return {"out": out, "pre": z} if case["save"] else {"out": out}
    if case["kind"] == "linear_grad":
        dz = s["dy"] * case["scale"]
        if s["pre"] is not None:
            dz *= _exact_activation(case["act"], s["pre"])[1]
        w = s["w"] if case["weight"] == "in_out" else s["w"].t()
        dx, dw = torch.mm(dz, w.t()), torch.mm(s["x"].t(), dz)
        if s["input_pre"] is not None:
            dx *= _exact_activation(case["input_act"], s["input_pre"])[1]
        return {"dx": dx, "dw": (dw if case["weight"] == "in_out" else dw.t()).contiguous(), "db": dz.sum(0)}
    if case["kind"] == "norm":
        return _exact_norm(case, s)
    return _exact_norm_grad(case, s) if case["kind"] == "norm_grad" else _exact_loss(case, s)


def _exact_norm(case, s):
    rows = case["rows"]
    total, statistics = s["branch"], []
    for which in ("post", "pre"):
        kind, v = case[which], total
        mean = v.mean(1, keepdim=True) if kind == "layer" else v.new_zeros(rows, 1)
        r = (((v - mean) ** 2).mean(1, keepdim=True) + EPSILON) ** -0.5 if kind != "none" else v.new_ones(rows, 1)
        statistics += [mean[:, 0], r[:, 0]]
        v = (v - mean) * r
        v = v * s[which + "_gamma"] if s[which + "_gamma"] is not None else v
        v = v + s[which + "_beta"] if s[which + "_beta"] is not None else v
        if which == "post":
            if s["gate"] is not None:
                v = v * _exact_activation(case["gate_act"], s["gate"])[0].repeat_interleave(rows // case["gate"], 0)
            total = s["residual"] + case["scale"] * v
        else:
            out = v
    return {"sum": total, "out": out, "statistics": torch.stack(statistics)}


def _exact_norm_grad(case, s):
    rows, c = case["rows"], case["channels"]
    mean1, r1, mean2, r2 = (t[:, None] for t in s["statistics"])
    # back through the norm before the next block
    hat = (s["sum"] - mean2) * r2
    out = {"pre_gamma": (s["d_out"] * hat).sum(0)}
    u = s["d_out"] * s["pre_gamma"]
    back = u - hat * (u * hat).sum(1, keepdim=True) / c
    if case["pre"] == "layer":
        out["pre_beta"] = s["d_out"].sum(0)
        back = back - u.sum(1, keepdim=True) / c
    out["residual"] = s["d_sum"] + r2 * back
    # the gate
    hat = s["branch"] if case["post"] == "none" else (s["branch"] - mean1) * r1
    g = out["residual"] * case["scale"]
    if s["gate"] is not None:
        n = hat if s["post_gamma"] is None else hat * s["post_gamma"]
        n = n if s["post_beta"] is None else n + s["post_beta"]
        value, slope = _exact_activation(case["gate_act"], s["gate"])
        out["gate"] = (g * n).reshape(case["gate"], rows // case["gate"], c).sum(1) * slope
        g = g * value.repeat_interleave(rows // case["gate"], 0)
    # the norm behind the block
    if case["post"] == "none":
        out["branch"] = g
        return out
    out["post_gamma"] = (g * hat).sum(0)
    u = g * s["post_gamma"]
    back = u - hat * (u * hat).sum(1, keepdim=True) / c
    if case["post"] == "layer":
        out["post_beta"] = g.sum(0)
        back = back - u.sum(1, keepdim=True) / c
    out["branch"] = r1 * back
    return out


def _exact_loss(case, s):
    tau, rows = case["temperature"], case["rows"]
    grad = torch.empty((rows, case["vocab"]), dtype=torch.float64, device="cuda")
    token_loss, logp = (torch.zeros(rows, dtype=torch.float64, device="cuda") for _ in range(2))
    for lo in range(0, rows, 1024):  # slices: the whole would take several times its size
        at = slice(lo, min(rows, lo + 1024))
        x = s["logits"][at] / tau
        t, w, a = s["targets"][at, None], s["weights"][at], s["advantages"][at]
        lse = torch.logsumexp(x, 1)
        lp = x.gather(1, t)[:, 0] - lse
        ratio = torch.exp(lp - s["old"][at])
        bound = torch.where(a >= 0, ratio.clamp(max=1 + CLIP_HIGH), ratio.clamp(min=1 - CLIP_LOW))
        value, slope = -a * bound, torch.where(bound == ratio, -a * ratio, torch.zeros_like(a))
        if s["ref"] is not None:
            q = torch.exp(s["ref"][at] - lp)
            value, slope = value + case["kl"] * (q - 1 - (s["ref"][at] - lp)), slope + case["kl"] * (1 - q)
        slope = slope * w * GRAD_SCALE / tau
        token_loss[at] = torch.where(w != 0, value * w, torch.zeros_like(w))
        logp[at] = torch.where(w != 0, lp, torch.zeros_like(w))
        grad[at] = -slope[:, None] * torch.exp(x - lse[:, None])
        grad[at].scatter_add_(1, t, slope[:, None])
    return {"loss": token_loss.sum(), "token_loss": token_loss, "logp": logp, "grad": grad}
