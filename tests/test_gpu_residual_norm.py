"""The norms around a block with its gate and residual sum, and their gradients, against the formulas in 64 bits.

Tolerances.  A team's sums over a row have at most 64 additions in a chain, so that statistics are off by 2^-18 of the values'
size; a result is off by that of the largest entry of its row, where the sum's entries count as large as the terms that it
is made of (residual and branch may cancel).  A gradient is the difference r (u - hat mean(u hat) - mean(u)) of
terms that may all but cancel (a row of one channel: u (1 - hat^2), where hat^2 is 1 but for epsilon), and each term is rounded by
its own size: it is off by 2^-16 of the largest sum of the terms' sizes in its row (hat is off by 2^-18, and twice in a term).
Sums over rows are off by 2^-15 of the sum of their terms' sizes (terms off by 2^-16, at most 2^8 additions in a chain), hat
itself being off by 2^-18 of its row's size, not of its own; a gate's slope by 2^-20 of 1."""
import itertools

import pytest
import torch

import portdnn_b200 as pd
from block_operators import ACTS, DTYPES, act, close, slope

pytestmark = pytest.mark.gpu
KINDS = {"none": pd.NORM_NONE, "rms": pd.NORM_RMS, "layer": pd.NORM_LAYER}
EPS = 1e-5


def _normal(g, *shape, std=1.0, mean=0.0):
    return torch.randn(shape, generator=g, device="cuda") * std + mean


def _inputs(rows, c, post, pre, groups, dtype, seed=0, residual=True, vectors=True):
    g, dt = torch.Generator(device="cuda").manual_seed(seed), DTYPES[dtype]
    s = {"branch": _normal(g, rows, c, std=0.8, mean=0.1).to(dt), "residual": _normal(g, rows, c, std=3.0).to(dt) if residual else None,
         "gate": _normal(g, groups, c, std=0.7, mean=0.3).to(dt) if groups else None}
    for which, kind in (("post", post), ("pre", pre)):
        s[which + "_gamma"] = _normal(g, c, std=0.3, mean=1.0).to(dt) if vectors and kind != "none" else None
        s[which + "_beta"] = _normal(g, c, std=0.2).to(dt) if vectors and kind == "layer" else None
    s["sum_grad"], s["out_grad"] = _normal(g, rows, c).to(dt), _normal(g, rows, c).to(dt)
    return s


def _norm(kind, v, gamma, beta):
    mean = v.mean(1) if kind == "layer" else v.new_zeros(v.shape[0])
    r = ((v - mean[:, None]) ** 2).mean(1).add(EPS).rsqrt() if kind != "none" else v.new_ones(v.shape[0])
    out = (v - mean[:, None]) * r[:, None]
    out = out if gamma is None else out * gamma.double()
    return out if beta is None else out + beta.double(), mean, r


def _spread(gate, rows):
    return gate.repeat_interleave(rows // gate.shape[0], 0)


def _row_max(v):
    return v.abs().max(1, keepdim=True).values if v.numel() else v.abs()


def _check_forward(s, post, pre, gate_act, scale, got):
    rows = s["branch"].shape[0]
    n, m1, r1 = _norm(post, s["branch"].double(), s["post_gamma"], s["post_beta"])
    k = scale * (1 if s["gate"] is None else _spread(act(gate_act, s["gate"].double()), rows))
    want = (0 if s["residual"] is None else s["residual"].double()) + k * n
    size = (k * n).abs() + (0 if s["residual"] is None else s["residual"].double().abs())
    out, m2, r2 = _norm(pre, want, s["pre_gamma"], s["pre_beta"])
    close(got[0], want, 2.0 ** -18 * _row_max(size), "sum")
    gamma = 1 if s["pre_gamma"] is None else s["pre_gamma"].double().abs()
    close(got[1], out, 2.0 ** -17 * _row_max(out.abs() + size * r2[:, None] * gamma), "out")
    most = size.abs().max(1).values
    for i, v in enumerate((m1, r1, m2, r2)):
        close(got[2][i], v, 2.0 ** -17 * ((v.abs() * (1 + most * r2) if i == 3 else v.abs()) + (1 + most if i % 2 == 0 else 0)), "statistics")


def _norm_back(kind, v, mean, r, gamma, g):
    """(gradient of v, hat, the terms' sizes)"""
    u = g if gamma is None else g * gamma.double()
    if kind == "none":
        return u, v, u.abs()
    hat = (v - mean[:, None]) * r[:, None]
    inner = (u * hat).mean(1, keepdim=True)
    back = u - hat * inner - (u.mean(1, keepdim=True) if kind == "layer" else 0)
    size = u.abs() + hat.abs() * (u * hat).abs().mean(1, keepdim=True) + u.abs().mean(1, keepdim=True)
    return back * r[:, None], hat, size * r[:, None]


def _check_gradients(s, post, pre, gate_act, scale, total, statistics, got, sum_grad=True):
    rows, c = s["branch"].shape
    m1, r1, m2, r2 = statistics.double()
    do = s["out_grad"].double()
    back, hat, size = _norm_back(pre, total.double(), m2, r2, s["pre_gamma"], do)
    d_sum = back + (s["sum_grad"].double() if sum_grad else 0)
    size = size + d_sum.abs()
    g = scale * d_sum
    f = s["branch"].double()
    fhat = f if post == "none" else (f - m1[:, None]) * r1[:, None]
    n = fhat if s["post_gamma"] is None else fhat * s["post_gamma"].double()
    n = n if s["post_beta"] is None else n + s["post_beta"].double()
    dn = g if s["gate"] is None else g * _spread(act(gate_act, s["gate"].double()), rows)
    k = abs(scale) * (1 if s["gate"] is None else _spread(act(gate_act, s["gate"].double()).abs(), rows))
    df, _, df_size = _norm_back(post, f, m1, r1, s["post_gamma"], dn.abs() + k * size)  # (what arrives is off by its terms' sizes, too)
    df = _norm_back(post, f, m1, r1, s["post_gamma"], dn)[0]
    close(got[1], d_sum, 2.0 ** -16 * _row_max(size), "residual")
    close(got[0], df, 2.0 ** -16 * _row_max(df_size), "branch")

    def sums(t, terms, size, what):
        if t is not None:
            close(t, terms.sum(0), 2.0 ** -15 * _row_max(size.sum(0)[None])[0], what)

    sums(got[2], dn * fhat, k * size * (fhat.abs() + 1), "post_gamma")
    sums(got[3], dn, k * size, "post_beta")
    sums(got[5], do * hat, do.abs() * (hat.abs() + 1), "pre_gamma")
    sums(got[6], do, do.abs(), "pre_beta")
    assert [t is None for t in got[2:]] == [s[k] is None for k in ("post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta")]
    if s["gate"] is not None:
        groups = s["gate"].shape[0]
        terms = (g * n).view(groups, rows // groups, c)
        d = slope(gate_act, s["gate"].double())
        off = (abs(scale) * size * (n.abs() + 1)).view(groups, rows // groups, c).sum(1)
        close(got[4], terms.sum(1) * d, 2.0 ** -15 * off * (d.abs() + 2.0 ** -5), "gate")


def _both(rows, c, post, pre, groups, gate_act, scale, dtype, **more):
    s = _inputs(rows, c, post, pre, groups, dtype, **more)
    p = pd.residual_norm_params(rows, c, KINDS[post], KINDS[pre], groups, ACTS[gate_act], scale, EPS)
    vectors = {k: s[k] for k in ("post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta")}
    got = pd.residual_norm(s["branch"], s["residual"], p, **vectors)
    _check_forward(s, post, pre, gate_act, scale, got)
    grads = pd.residual_norm_grad(s["sum_grad"], s["out_grad"], s["branch"], got[0], got[2], p, **vectors)
    _check_gradients(s, post, pre, gate_act, scale, got[0], got[2], grads)
    return s, p, vectors, got, grads


# every shape of a team, whole packets and single elements, and rows too long for any
@pytest.mark.parametrize("channels", [1, 3, 8, 32, 100, 129, 256, 504, 512, 1000, 1003, 1024, 2040, 2048, 3001, 4096, 4104, 8192, 16392, 20000])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_widths(channels, dtype):
    _both(37, channels, "rms", "rms", 1, "none", 1.0, dtype)
    _both(5, channels, "layer", "layer", 5, "sigmoid", 0.5, dtype)


@pytest.mark.parametrize("post,pre", list(itertools.product(KINDS, repeat=2)))
@pytest.mark.parametrize("groups,gate_act", [(0, "none"), (1, "tanh"), (6, "sigmoid"), (300, "none")])
def test_norms_and_gates(post, pre, groups, gate_act):
    _both(300, 264, post, pre, groups, gate_act, 0.7, "bf16")
    _both(300, 77, post, pre, groups, gate_act, -1.0, "f32")


@pytest.mark.parametrize("rows", [1, 2, 3, 147, 149, 1000, 5000])
@pytest.mark.parametrize("channels", [64, 640, 2056])
def test_rows(rows, channels):
    _both(rows, channels, "rms", "layer", 1, "none", 1.0, "bf16")
    _both(rows, channels, "layer", "rms", 0, "none", 1.0, "f16", residual=False)


# rows that no team keeps: more rows than blocks, groups cut into stretches, more groups than blocks walk at once
@pytest.mark.parametrize("post,pre", [("rms", "rms"), ("layer", "rms"), ("none", "layer"), ("none", "none")])
@pytest.mark.parametrize("rows,channels,groups,dtype", [(700, 8200, 0, "bf16"), (700, 8200, 7, "f16"), (320, 9001, 1, "bf16"),
                                                        (400, 8200, 400, "bf16"), (200, 8196, 2, "f32")])
def test_long_rows(rows, channels, groups, dtype, post, pre):
    _both(rows, channels, post, pre, groups, "sigmoid" if groups else "none", 0.7, dtype)


@pytest.mark.parametrize("activation", sorted(ACTS))
def test_gate_activations(activation):
    _both(64, 128, "rms", "rms", 4, activation, 1.0, "f32")


def test_without_gammas():
    _both(40, 136, "rms", "layer", 2, "none", 1.0, "bf16", vectors=False)
    _both(40, 20000, "layer", "rms", 2, "none", 1.0, "f32", vectors=False)


def test_gradient_of_the_first_norm_alone():
    """Nothing arrives by the residual stream."""
    s, p, vectors, got, _ = _both(50, 256, "rms", "rms", 0, "none", 1.0, "bf16")
    grads = pd.residual_norm_grad(None, s["out_grad"], s["branch"], got[0], got[2], p, **vectors)
    _check_gradients(s, "rms", "rms", "none", 1.0, got[0], got[2], grads, sum_grad=False)


@pytest.mark.parametrize("channels", [256, 1003, 4096, 40000])
def test_in_place_and_repeatable(channels):
    s, p, vectors, got, grads = _both(150, channels, "rms", "rms", 1, "none", 1.0, "bf16")
    again = pd.residual_norm_grad(s["sum_grad"], s["out_grad"], s["branch"], got[0], got[2], p, **vectors)
    assert all(a is b or torch.equal(a, b) for a, b in zip(grads, again))
    total, out, statistics = pd.residual_norm(s["branch"].clone(), s["residual"], p, sum_out=s["residual"], out=(b := s["branch"].clone()), **vectors)
    assert torch.equal(total, got[0]) and torch.equal(out, got[1]) and torch.equal(statistics, got[2])
    total, out, statistics = pd.residual_norm(b.copy_(s["branch"]), total.copy_(got[0]), p, out=b, **vectors)
    want = pd.residual_norm(s["branch"], got[0], p, **vectors)
    assert out.data_ptr() == b.data_ptr() and torch.equal(out, want[1])
    grads2 = pd.residual_norm_grad(s["sum_grad"], s["out_grad"], s["branch"], got[0], got[2], p, branch_grad=s["out_grad"],
                                   residual_grad=s["sum_grad"], **vectors)
    assert all(a is b or torch.equal(a, b) for a, b in zip(grads, grads2))


def test_off_a_packet_boundary():
    """The same values where no tensor starts on 16 bytes: the same sums to a rounding."""
    s, p, vectors, got, grads = _both(33, 512, "rms", "layer", 3, "tanh", 1.0, "bf16")

    def shifted(t):
        if t is None:
            return None
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:]
        return flat.copy_(t.flatten()).view(t.shape)

    s = {k: shifted(v) for k, v in s.items()}
    vectors = {k: s[k] for k in vectors}
    got = pd.residual_norm(s["branch"], s["residual"], p, **vectors)
    _check_forward(s, "rms", "layer", "tanh", 1.0, got)
    grads = pd.residual_norm_grad(s["sum_grad"], s["out_grad"], s["branch"], got[0], got[2], p, **vectors)
    _check_gradients(s, "rms", "layer", "tanh", 1.0, got[0], got[2], grads)


def test_no_rows():
    for groups in (0, 1):
        p = pd.residual_norm_params(0, 64, gate_groups=groups)
        e, v = torch.empty((0, 64), device="cuda"), torch.ones(64, device="cuda")
        gate = torch.ones((1, 64), device="cuda") if groups else None
        total, out, statistics = pd.residual_norm(e, e, p, post_gamma=v, pre_gamma=v, gate=gate)
        assert total.shape == out.shape == (0, 64)
        grads = pd.residual_norm_grad(e, e, e, total, statistics, p, post_gamma=v, pre_gamma=v, gate=gate)
        assert all((t == 0).all() for t in grads if t is not None and t.numel())


def test_infinities_and_nan_stay_in_their_rows():
    for channels in (256, 1003, 4096):
        s = _inputs(12, channels, "rms", "layer", 1, "bf16")
        p = pd.residual_norm_params(12, channels, pd.NORM_RMS, pd.NORM_LAYER, 1, epsilon=EPS)
        vectors = {k: s[k] for k in ("post_gamma", "gate", "pre_gamma", "pre_beta")}
        want = pd.residual_norm(s["branch"], s["residual"], p, **vectors)
        s["branch"][3, 1], s["residual"][7, 2] = float("nan"), float("inf")
        got = pd.residual_norm(s["branch"], s["residual"], p, **vectors)
        keep = [i for i in range(12) if i not in (3, 7)]
        assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1][keep], want[1][keep])
        assert torch.isnan(got[1][3]).all() and torch.isnan(got[1][7]).any()


def test_constant_and_zero_rows():
    """Rows without variance, or of zeros: epsilon alone is under the root."""
    x = torch.zeros((4, 96), device="cuda")
    x[2:] = 5.0
    p = pd.residual_norm_params(4, 96, pd.NORM_NONE, pd.NORM_LAYER, epsilon=EPS)
    total, out, statistics = pd.residual_norm(x, None, p)
    assert torch.equal(total, x) and (out == 0).all()
    close(statistics[3], torch.full((4,), EPS, device="cuda").double().rsqrt(), 2.0 ** -20 * EPS ** -0.5, "r")


def test_gradients_against_differences():
    rows, c, h = 6, 40, 2.0 ** -5
    for post, pre in (("rms", "layer"), ("layer", "rms")):
        s = _inputs(rows, c, post, pre, 2, "f32")
        p = pd.residual_norm_params(rows, c, KINDS[post], KINDS[pre], 2, pd.ACT_SIGMOID, 0.8, EPS)
        names = [k for k in ("branch", "residual", "post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta") if s[k] is not None]

        def loss(s):
            total, out, _ = pd.residual_norm(s["branch"], s["residual"], p, **{k: s[k] for k in names[2:]})
            return (total.double() * s["sum_grad"]).sum() + (out.double() * s["out_grad"]).sum()

        got = pd.residual_norm(s["branch"], s["residual"], p, **{k: s[k] for k in names[2:]})
        grads = pd.residual_norm_grad(s["sum_grad"], s["out_grad"], s["branch"], got[0], got[2], p, **{k: s[k] for k in names[2:]})
        named = dict(zip(("branch", "residual", "post_gamma", "post_beta", "gate", "pre_gamma", "pre_beta"), grads))
        for i, k in enumerate(names):
            d = _normal(torch.Generator(device="cuda").manual_seed(50 + i), *s[k].shape)
            # differences over h and h / 2: their own distance bounds what either leaves of the third derivative
            slopes = [(loss({**s, k: s[k] + e * d}) - loss({**s, k: s[k] - e * d})) / (2 * e) for e in (h, h / 2)]
            rounding = 2.0 ** -20 / h * (got[0].double().abs() * s["sum_grad"].abs() + got[1].double().abs() * s["out_grad"].abs()).sum()
            want = (named[k].double() * d).sum()
            assert (slopes[1] - want).abs() <= 2 * (slopes[0] - slopes[1]).abs() + rounding, (post, k)


def test_refusals():
    x, v = torch.ones((8, 64), device="cuda"), torch.ones(64, device="cuda")
    params = pd.residual_norm_params
    for p, more, error in (
            (params(8, 63), {}, ValueError), (params(7, 64), {}, ValueError), (params(8, 64), dict(post_gamma=v[:63]), ValueError),
            (params(8, 64), dict(pre_gamma=v.half()), ValueError), (params(8, 64, gate_groups=3), dict(gate=torch.ones((3, 64), device="cuda")), pd.PortDNNError),
            (params(8, 64, gate_groups=2), {}, pd.PortDNNError), (params(8, 64, post_norm=3), {}, pd.PortDNNError),
            (params(8, 64, gate_activation=4), {}, pd.PortDNNError), (params(8, 64, epsilon=-1.0), {}, pd.PortDNNError),
            (params(8, 64, epsilon=float("nan")), {}, pd.PortDNNError), (params(8, 64), dict(gate=torch.ones((1, 64), device="cuda")), ValueError),
            (params(8, 64), dict(out=torch.empty((8, 128), device="cuda")[:, :64]), ValueError)):
        with pytest.raises(error):
            pd.residual_norm(x, x, p, **more)
    with pytest.raises(ValueError):
        pd.residual_norm(x.t(), x, params(8, 64))
    with pytest.raises(ValueError):
        pd.residual_norm_grad(x, x, x, x, torch.ones(31, device="cuda"), params(8, 64))
    with pytest.raises(TypeError):
        pd.residual_norm(x, x, pd.pool_params(1, 4, 4, 1, 2, 2))


def test_results_across_inputs_are_refused():
    x = torch.ones((9, 64), device="cuda")
    p = pd.residual_norm_params(8, 64)
    a, b = x[:8], x[1:]
    for bad in (dict(sum_out=b), dict(out=b), dict(sum_out=a, out=a)):
        with pytest.raises(pd.PortDNNError):
            pd.residual_norm(a, a.clone(), p, **bad)
    total, out, statistics = pd.residual_norm(a.clone(), a.clone(), p)
    for bad in (dict(branch_grad=b), dict(residual_grad=b), dict(branch_grad=total, residual_grad=total)):
        with pytest.raises(pd.PortDNNError):
            pd.residual_norm_grad(a, a, a, total, statistics, p, **bad)


def test_results_in_any_input_s_place():
    for channels in (72, 1003, 4096, 40000):
        s, p, vectors, got, grads = _both(30, channels, "rms", "layer", 1, "none", 1.0, "bf16")
        b, r = s["branch"].clone(), s["residual"].clone()
        total, out, _ = pd.residual_norm(b, r, p, sum_out=b, out=r, **vectors)
        assert torch.equal(total, got[0]) and torch.equal(out, got[1])
        b, total = s["branch"].clone(), got[0].clone()
        again = pd.residual_norm_grad(s["sum_grad"], s["out_grad"], b, total, got[2], p, branch_grad=total, residual_grad=b, **vectors)
        assert all(u is v or torch.equal(u, v) for u, v in zip(grads, again))
