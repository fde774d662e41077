"""The clipped policy loss and its gradient against the formulas in 64 bits.

Tolerances.  The sum over a row is off by at most 2^-16 of itself: a chain of at most 100 additions to a thread, and terms
2^((x - top) c) off by 2^-22 and by 2^-24 of an exponent of at most 60.  That is what logp is off by, beside 2^-22 of the logits' size;
ratio and exp(ref - logp) are off by it relative to themselves, and the gradient's p too, twice."""
import pytest
import torch

import portdnn_b200 as pd
from block_operators import DTYPES, close

pytestmark = pytest.mark.gpu
LOW, HIGH = 0.2, 0.3


def _inputs(rows, vocab, dtype, pitch=None, seed=0, masked=0.3, std=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    whole = (torch.randn((rows, pitch or vocab), generator=g, device="cuda") * std).to(DTYPES[dtype])
    x = whole[:, :vocab]
    t = torch.randint(vocab, (rows,), generator=g, device="cuda")
    lp = torch.log_softmax(x.float(), 1)[torch.arange(rows, device="cuda"), t]
    noise = [torch.randn(rows, generator=g, device="cuda") for _ in range(3)]
    w = (torch.rand(rows, generator=g, device="cuda") >= masked).float() * (0.5 + torch.rand(rows, generator=g, device="cuda"))
    return {"logits": x, "targets": t, "advantages": noise[0], "old_logp": lp + 0.3 * noise[1], "ref_logp": lp + 0.3 * noise[2], "weights": w}


def _check(s, got, kl=0.0, temperature=1.0, grad_scale=1.0, grad=True):
    x, t = s["logits"].double() / temperature, s["targets"].long()
    rows, vocab = x.shape
    w = torch.ones(rows, device="cuda") if s.get("weights") is None else s["weights"]
    counts = (w != 0) & (t >= 0) & (t < vocab) & (x > -float("inf")).any(1)
    x = torch.where(counts[:, None], x, 0.0)
    t = torch.where(counts, t, 0)
    lse = torch.logsumexp(x, 1)
    lp = x.gather(1, t[:, None])[:, 0] - lse
    a = s["advantages"].double()
    ratio = torch.exp(lp - (s["old_logp"].double() if s.get("old_logp") is not None else lp))
    free, clipped = ratio * a, ratio.clamp(1 - float(torch.tensor(LOW)), 1 + float(torch.tensor(HIGH))) * a
    loss, slope, size = -torch.minimum(free, clipped), torch.where(free <= clipped, -free, 0.0), free.abs()
    if s.get("ref_logp") is not None:
        q = torch.exp(s["ref_logp"].double() - lp)
        d = s["ref_logp"].double() - lp
        loss, slope, size = loss + kl * (q - d - 1), slope + kl * (1 - q), size + kl * (q + d.abs() + 1)
    off = 2.0 ** -16 + 2.0 ** -22 * (x.abs().max(1).values + lp.abs())  # of logp
    zero = torch.zeros_like(lp)
    keep = lambda v: torch.where(counts, v, zero)  # noqa: E731
    close(got[2], keep(lp), keep(off), "logp")
    close(got[1], keep(w * loss), keep(w * size * 4 * off), "token_loss")
    close(got[0], keep(w * loss).sum(), keep(w * size * 4 * off).sum() + (rows + 8) * 2.0 ** -23 * keep(w * loss).abs().sum(), "loss")
    if not grad:
        assert got[3] is None
        return
    k = keep(w * slope) * grad_scale / temperature
    p = torch.exp(x - lse[:, None])
    one = torch.zeros_like(p).scatter_(1, t[:, None], 1.0)
    want = k[:, None] * (one - p)
    allowed = (keep(w * size) * abs(grad_scale) / temperature * 4 * off)[:, None] * (one + p) + k.abs()[:, None] * (one + p) * 2 * off[:, None]
    close(got[3], want, allowed, "grad")
    assert (got[3][~counts] == 0).all()


# one element, less than a packet, single walks, clusters of CTAs over few long rows, and many rows
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 5), (3, 100), (7, 1000), (1, 130000), (5, 50001), (40, 32000), (200, 4099), (700, 513), (2000, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_sizes(rows, vocab, dtype):
    s = _inputs(rows, vocab, dtype)
    _check(s, pd.policy_loss(**s, clip_low=LOW, clip_high=HIGH, kl=0.1), kl=0.1)


@pytest.mark.parametrize("vocab,pitch", [(1000, 1024), (1003, 1024), (1003, 1007), (50001, 50048), (9, 16)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_of_wider_tensors(vocab, pitch, dtype):
    s = _inputs(30, vocab, dtype, pitch=pitch)
    _check(s, pd.policy_loss(**s, clip_low=LOW, clip_high=HIGH, kl=0.1, temperature=0.7, grad_scale=128.0), 0.1, 0.7, 128.0)


@pytest.mark.parametrize("without", [("old_logp",), ("ref_logp",), ("weights",), ("old_logp", "ref_logp", "weights")])
def test_parts(without):
    for rows, vocab in ((20, 777), (3, 40000)):
        s = _inputs(rows, vocab, "bf16")
        for k in without:
            s[k] = None
        _check(s, pd.policy_loss(**s, clip_low=LOW, clip_high=HIGH, kl=0.1), kl=0.1)
        _check(s, pd.policy_loss(**s, clip_low=LOW, clip_high=HIGH, kl=0.1, want_grad=False), kl=0.1, grad=False)


def test_targets_of_32_bits_and_outside_the_vocabulary():
    s = _inputs(50, 321, "f16", masked=0.0)
    s["targets"][::7] = -100
    s["targets"][1::7] = 321
    s["targets"][2] = 2 ** 40  # (64 bits only)
    _check(s, pd.policy_loss(**s, clip_low=LOW, clip_high=HIGH, kl=0.1), kl=0.1)
    s["targets"][2] = -1
    wide = pd.policy_loss(**s, clip_low=LOW, clip_high=HIGH, kl=0.1)
    narrow = pd.policy_loss(**{**s, "targets": s["targets"].int()}, clip_low=LOW, clip_high=HIGH, kl=0.1)
    assert all(torch.equal(a, b) for a, b in zip(wide, narrow))


@pytest.mark.parametrize("rows,vocab", [(12, 1000), (4, 60000)])
def test_masked_logits(rows, vocab):
    """Minus infinity and the type's lowest value as masks, a row of nothing else; what stands in rows that do not count."""
    s = _inputs(rows, vocab, "bf16", masked=0.0)
    keep = s["targets"].clone()
    x = s["logits"]
    at = torch.arange(rows, device="cuda")
    chosen = x[at, keep].clone()
    x[0, ::2] = -float("inf")
    x[1, 1::2] = torch.finfo(torch.bfloat16).min
    x[at, keep] = chosen
    x[2] = -float("inf")
    x[3] = float("nan")
    s["weights"][3] = 0.0
    got = pd.policy_loss(**s, clip_low=LOW, clip_high=HIGH, kl=0.1)
    x[3] = 0.0
    _check(s, got, kl=0.1)
    assert (got[3][0, ::2][torch.arange(0, vocab, 2, device="cuda") != keep[0]] == 0).all()


@pytest.mark.parametrize("rows,vocab", [(8, 1000), (3, 60000)])
def test_nan_and_infinities_stay_in_their_rows(rows, vocab):
    s = _inputs(rows, vocab, "f32", masked=0.0)
    want = pd.policy_loss(**s, kl=0.1)
    s["logits"][1, vocab // 2] = float("nan")
    s["logits"][2, vocab // 3] = float("inf")
    got = pd.policy_loss(**s, kl=0.1)
    keep = [i for i in range(rows) if i not in (1, 2)]
    for i in (1, 2, 3):
        assert torch.equal(got[i][keep], want[i][keep])
        assert torch.isnan(got[i][1]).any() and torch.isnan(got[i][2]).any()


@pytest.mark.parametrize("rows,vocab,pitch", [(300, 1003, 1024), (4, 70000, 70000), (6, 999, 999)])
def test_in_place_repeatable_and_beside(rows, vocab, pitch):
    """The gradient in the logits' place; the same bits every time; columns behind the vocabulary are left alone."""
    s = _inputs(rows, vocab, "bf16", pitch=pitch)
    want = pd.policy_loss(**s, kl=0.1)
    again = pd.policy_loss(**s, kl=0.1)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    whole = torch.full((rows + 1, pitch), 3.0, dtype=torch.bfloat16, device="cuda")
    pd.policy_loss(**s, kl=0.1, grad=whole[:rows, :vocab])
    assert torch.equal(whole[:rows, :vocab], want[3]) and (whole[rows:] == 3).all() and (whole[:, vocab:] == 3).all()
    got = pd.policy_loss(**s, kl=0.1, grad=s["logits"])
    assert got[3].data_ptr() == s["logits"].data_ptr() and all(torch.equal(a, b) for a, b in zip(want, got))


def test_clipping_on_both_sides():
    """Ratios far on either side with advantages of both signs: where the clipped value is the smaller one no gradient is left."""
    s = _inputs(4, 500, "f32", masked=0.0)
    lp = pd.policy_loss(**s)[2]
    s["old_logp"] = lp - torch.tensor([1.0, 1.0, -1.0, -1.0], device="cuda")
    s["advantages"] = torch.tensor([2.0, -2.0, 2.0, -2.0], device="cuda")
    s["ref_logp"], s["weights"] = None, None
    got = pd.policy_loss(**s, clip_low=LOW, clip_high=HIGH)
    _check(s, got)
    assert [bool((g != 0).any()) for g in got[3]] == [False, True, True, False]


def test_gradient_against_differences():
    s = _inputs(6, 40, "f32", masked=0.0)
    # away from the clip's borders, where the loss has a kink
    lp = pd.policy_loss(**s)[2]
    s["old_logp"] = lp + torch.tensor([0.05, -0.1, 0.1, -0.05, 0.0, 0.08], device="cuda")
    got = pd.policy_loss(**s, clip_low=LOW, clip_high=HIGH, kl=0.2, temperature=0.9)
    d = torch.randn((6, 40), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    h = 2.0 ** -6
    slopes = []
    for e in (h, h / 2):
        ends = [pd.policy_loss(**{**s, "logits": s["logits"] + sign * e * d}, clip_low=LOW, clip_high=HIGH, kl=0.2, temperature=0.9,
                               want_grad=False)[1].double().sum() for sign in (1, -1)]
        slopes.append((ends[0] - ends[1]) / (2 * e))
    want = (got[3].double() * d).sum()
    rounding = 2.0 ** -18 / h * (1 + s["advantages"].double().abs()).sum() * float(s["weights"].max())
    assert (slopes[1] - want).abs() <= 2 * (slopes[0] - slopes[1]).abs() + rounding


def test_no_rows():
    e = torch.empty(0, device="cuda")
    got = pd.policy_loss(torch.empty((0, 50), device="cuda"), torch.empty(0, dtype=torch.long, device="cuda"), e)
    assert got[0] == 0 and got[3].shape == (0, 50)


def test_graph_replay():
    s = _inputs(90, 2000, "bf16")
    want = [t.clone() for t in pd.policy_loss(**s, kl=0.1)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = pd.policy_loss(**s, kl=0.1)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals():
    s = _inputs(6, 100, "f32")
    for bad in (dict(targets=s["targets"][:5]), dict(targets=s["targets"].float()), dict(advantages=s["advantages"].half()),
                dict(weights=s["weights"].cpu()), dict(advantages=None), dict(logits=s["logits"].t()), dict(logits=s["logits"][0]),
                dict(grad=torch.empty((6, 101), device="cuda"))):
        with pytest.raises(ValueError):
            pd.policy_loss(**{**s, **bad})
    wide = torch.zeros((6, 150), device="cuda")
    with pytest.raises(pd.PortDNNError):  # the gradient across the logits
        pd.policy_loss(**{**s, "logits": wide[:, :100]}, grad=wide[:, 50:])
    for bad in (dict(temperature=0.0), dict(temperature=float("nan")), dict(clip_low=-0.1), dict(clip_high=float("nan"))):
        with pytest.raises(pd.PortDNNError):
            pd.policy_loss(**s, **bad)
