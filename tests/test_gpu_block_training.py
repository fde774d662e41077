"""A run of the operators around a block's matrix products as a model uses them: norm, two fused products, norms with gate and
residual sum, a third product, the policy loss, and the way back, against float64 with torch's own differentiation.

Tolerances, of whole tensors (norm of the difference over the norm of the result).  No value is rounded more than 14 times on its
way there and back; each rounding is off by half a step at most (2^-8 in bf16, 2^-11 in fp16), and the norms - the only
steps that divide - at most double what arrives: 28 half steps.  In fp32 each of the 14 steps is off by 2^-17 of its terms' sizes
(the operators' own tests), which exceed the results four times at most: 14 * 2^-15."""
import pytest
import torch

import portdnn_b200 as pd

pytestmark = pytest.mark.gpu
TOLERANCE = {torch.float32: 14 * 2.0 ** -15, torch.bfloat16: 28 * 2.0 ** -8, torch.float16: 28 * 2.0 ** -11}
EPS = 1e-5


def _model(dt, tokens, width, hidden, vocab, groups):
    g = torch.Generator(device="cuda").manual_seed(3)
    n = lambda *s, std=1.0, mean=0.0: (torch.randn(s, generator=g, device="cuda") * std + mean).to(dt)  # noqa: E731
    return {"x": n(tokens, width), "g0": n(width, std=0.2, mean=1.0), "w1": n(width, hidden, std=width ** -0.5),
            "b1": n(hidden, std=0.2), "w2": n(width, hidden, std=hidden ** -0.5), "b2": n(width, std=0.2),
            "g1": n(width, std=0.2, mean=1.0), "gate": n(groups, width, std=0.5, mean=0.5), "g2": n(width, std=0.2, mean=1.0),
            "w3": n(vocab, width, std=2 * width ** -0.5)}


def _step(p, tokens, loss_inputs):
    """Loss and gradients of every tensor, as a program calls the library."""
    width, groups = p["x"].shape[1], p["gate"].shape[0]
    first = pd.residual_norm_params(tokens, width, pd.NORM_NONE, pd.NORM_RMS, epsilon=EPS)
    second = pd.residual_norm_params(tokens, width, pd.NORM_RMS, pd.NORM_RMS, groups, pd.ACT_SIGMOID, 0.8, EPS)
    x, h0, st0 = pd.residual_norm(p["x"], None, first, pre_gamma=p["g0"])
    z1 = torch.empty((tokens, p["w1"].shape[1]), dtype=p["x"].dtype, device="cuda")
    a1 = pd.matmul_fused(h0, p["w1"], bias=p["b1"], activation=pd.ACT_GELU, pre_activation=z1)
    y = pd.matmul_fused(a1, p["w2"], transpose_rhs=True, bias=p["b2"])
    s, h, st = pd.residual_norm(y, x, second, post_gamma=p["g1"], gate=p["gate"], pre_gamma=p["g2"])
    logits = pd.matmul_fused(h, p["w3"], transpose_rhs=True)
    loss, _, logp, dlogits = pd.policy_loss(logits, kl=0.1, clip_low=0.2, clip_high=0.2, **loss_inputs)
    dh, dw3, _ = pd.matmul_fused_grad(dlogits, h, p["w3"], transpose_rhs=True, want_bias_grad=False)
    dy, dx, dg1, _, dgate, dg2, _ = pd.residual_norm_grad(None, dh, y, s, st, second, post_gamma=p["g1"], gate=p["gate"], pre_gamma=p["g2"])
    dz1, dw2, db2 = pd.matmul_fused_grad(dy, a1, p["w2"], transpose_rhs=True, input_activation=pd.ACT_GELU, input_pre_activation=z1)
    dh0, dw1, db1 = pd.matmul_fused_grad(dz1, h0, p["w1"])
    d0, _, _, _, _, dg0, _ = pd.residual_norm_grad(dx, dh0, p["x"], x, st0, first, pre_gamma=p["g0"])
    return loss, logp, {"x": d0, "g0": dg0, "w1": dw1, "b1": db1, "w2": dw2, "b2": db2, "g1": dg1, "gate": dgate, "g2": dg2, "w3": dw3}


def _rms(v, gamma):
    return v * (v.square().mean(1, keepdim=True) + EPS).rsqrt() * gamma


def _exact(p, tokens, loss_inputs):
    q = {k: v.double().requires_grad_() for k, v in p.items()}
    h0 = _rms(q["x"], q["g0"])
    a1 = torch.nn.functional.gelu(h0 @ q["w1"] + q["b1"])
    y = a1 @ q["w2"].t() + q["b2"]
    gate = torch.sigmoid(q["gate"]).repeat_interleave(tokens // q["gate"].shape[0], 0)
    s = q["x"] + 0.8 * gate * _rms(y, q["g1"])
    logits = _rms(s, q["g2"]) @ q["w3"].t()
    lp = torch.log_softmax(logits, 1).gather(1, loss_inputs["targets"][:, None])[:, 0]
    ratio, a = torch.exp(lp - loss_inputs["old_logp"]), loss_inputs["advantages"].double()
    d = loss_inputs["ref_logp"] - lp
    t = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a) + 0.1 * (torch.exp(d) - d - 1)
    loss = (loss_inputs["weights"] * t).sum()
    loss.backward()
    return loss.detach(), lp.detach(), {k: v.grad for k, v in q.items()}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens,width,hidden,vocab", [(48, 64, 160, 200), (250, 136, 520, 1003), (600, 512, 2048, 4096)])
def test_step(dtype, tokens, width, hidden, vocab):
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    p = _model(dt, tokens, width, hidden, vocab, 2)
    g = torch.Generator(device="cuda").manual_seed(4)
    targets = torch.randint(vocab, (tokens,), generator=g, device="cuda")
    weights = (torch.rand(tokens, generator=g, device="cuda") < 0.8).float() / tokens
    inputs = {"targets": targets, "advantages": torch.randn(tokens, generator=g, device="cuda"), "weights": weights}
    # old and reference log-probabilities near the model's own, the ratio well inside the clip's borders or well outside them (a
    # rounding that crosses a border switches a token's gradient on or off, which no bound on roundings covers)
    zero = torch.zeros(tokens, device="cuda")
    lp = _exact(p, tokens, {**inputs, "old_logp": zero, "ref_logp": zero})[1].float()
    side = torch.randint(3, (tokens,), generator=g, device="cuda")
    inputs["old_logp"] = lp + torch.tensor([0.02, 0.9, -0.9], device="cuda")[side]
    inputs["ref_logp"] = lp + 0.2 * torch.randn(tokens, generator=g, device="cuda")
    loss, logp, grads = _step(p, tokens, inputs)
    want_loss, want_logp, want = _exact(p, tokens, inputs)
    tol = TOLERANCE[dt]
    live = weights != 0
    assert (logp.double() - want_logp)[live].norm() <= tol * want_logp[live].norm()
    terms = (weights.double() * (inputs["advantages"].double().abs() * 2.5 + 0.1)).sum()  # (the loss' own terms may cancel)
    assert (loss.double() - want_loss).abs() <= tol * terms
    for k, v in want.items():
        off = float((grads[k].double() - v).norm() / v.norm())
        assert off <= tol, (k, off, tol)


def test_step_is_repeatable_and_replays_from_a_graph():
    """The same bits called twice, captured and replayed, and with two captured steps replayed in turn."""
    sets = []
    for seed in (1, 2):
        p = _model(torch.bfloat16, 250, 136, 520, 1003, 2)
        g = torch.Generator(device="cuda").manual_seed(seed)
        p["x"] = torch.randn((250, 136), generator=g, device="cuda").bfloat16()
        n = lambda: torch.randn(250, generator=g, device="cuda")  # noqa: E731
        inputs = {"targets": torch.randint(1003, (250,), generator=g, device="cuda"), "advantages": n(), "old_logp": n() - 7,
                  "ref_logp": n() - 7, "weights": torch.full((250,), 0.004, device="cuda")}
        sets.append((p, inputs))
    want = [_step(p, 250, i) for p, i in sets]
    again = [_step(p, 250, i) for p, i in sets]
    torch.cuda.synchronize()
    graphs, got = [], []
    for p, i in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(_step(p, 250, i))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, again, got):
        for other in (b, c):
            assert torch.equal(a[0], other[0]) and torch.equal(a[1], other[1])
            assert all(torch.equal(a[2][k], other[2][k]) for k in a[2])
