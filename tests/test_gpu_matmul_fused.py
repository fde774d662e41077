"""The matrix product with bias, activation and residual, and its gradients, against the formulas in 64 bits.

Tolerances.  A sum of k products in 32 bits is off by at most (k + 8) 2^-23 of the sum of the products' sizes (a step of the
accumulator to each addition), and fp32 operands, which are multiplied in three parts, by 2^-19 of it more (two parts of 11
bits each, the product of the smaller ones left out).  Activations change by at most 1.2 times what their argument does, and are
computed to 2^-20 of 1 + |z|.  Each 16-bit rounding adds half a step: of the result, and in gradients of dz, which the tensor
cores multiply in the tensors' type."""
import itertools
import re

import pytest
import torch

import portdnn_b200 as pd
from block_operators import ACTS, DTYPES, act, close, half_step, slope
from gpu_util import assert_no_device_error
from launched import launched

pytestmark = pytest.mark.gpu


def _normal(seed, *shape, std=1.0):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * std


def _sum_error(a, b, dtype):
    k = a.shape[1]
    return ((k + 8) * 2.0 ** -23 + (2.0 ** -19 if dtype == torch.float32 else 0)) * (a.double().abs() @ b.double().abs())


def _pitched(t, extra):
    """The same values as a slice of a wider tensor."""
    wide = torch.full((t.shape[0], t.shape[1] + extra), 7.0, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _forward(m, k, n, tr, dtype, activation, bias, residual, scale, save, extra=0, seed=0):
    dt = DTYPES[dtype]
    x, w = _normal(seed, m, k).to(dt), _normal(seed + 1, *((n, k) if tr else (k, n)), std=k ** -0.5).to(dt)
    b = _normal(seed + 2, n, std=0.3).to(dt) if bias else None
    r = _normal(seed + 3, m, n).to(dt) if residual else None
    if extra:
        x, w, r = _pitched(x, extra), _pitched(w, extra), None if r is None else _pitched(r, extra)
    pre = torch.empty((m, n), dtype=dt, device="cuda") if save else None
    got = pd.matmul_fused(x, w, transpose_rhs=tr, bias=b, activation=ACTS[activation], residual=r, scale=scale, pre_activation=pre)
    assert_no_device_error()
    wd = w.double().t() if tr else w.double()
    z = x.double() @ wd + (0 if b is None else b.double())
    off = _sum_error(x, wd, dt) + 2.0 ** -23 * z.abs()
    want = scale * act(activation, z) + (0 if r is None else r.double())
    allowed = abs(scale) * (1.2 * off + (0 if activation == "none" else 2.0 ** -20 * (1 + z.abs()))) + 2.0 ** -23 * want.abs()
    close(got, want, allowed, "out")
    if save:
        close(pre, z, off, "pre")


SHAPES = [(1, 64, 64), (1, 1, 1), (3, 7, 5), (2, 4096, 1024), (16, 512, 640), (17, 520, 200), (33, 129, 65), (64, 64, 8),
          (128, 256, 128), (129, 72, 264), (250, 512, 1000), (511, 515, 257), (1000, 96, 136), (2304, 320, 2056), (4500, 136, 520)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tr", [False, True])
def test_forward(m, k, n, dtype, tr):
    _forward(m, k, n, tr, dtype, "gelu", True, True, 0.5, True)


# on both sides of the numbers of rows from which fp32 products leave the CUDA cores
@pytest.mark.parametrize("tr", [False, True])
@pytest.mark.parametrize("m", [15, 16, 17, 23, 24, 25])
def test_few_rows_in_single_precision(m, tr):
    _forward(m, 300, 203, tr, "f32", "tanh", True, True, 0.7, True)
    _forward(m, 1024, 512, tr, "f32", "none", False, False, 1.0, False)
    _gradients(m, 300, 203, tr, "f32", "silu", "none", 1.0)


# few tiles and long sums: clusters of every size, rings of stages that take all of an SM's shared memory or half
@pytest.mark.parametrize("m,k,n", [(128, 4096, 2048), (256, 2048, 1000), (60, 6000, 1000), (100, 8000, 104), (700, 4160, 64), (1, 8192, 72)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tr", [False, True])
def test_long_sums(m, k, n, dtype, tr):
    _forward(m, k, n, tr, dtype, "silu", True, False, 1.0, True)


@pytest.mark.parametrize("activation", sorted(ACTS))
@pytest.mark.parametrize("m", [5, 300, 2500])
def test_activations(activation, m):
    _forward(m, 192, 2048, False, "bf16", activation, True, False, 1.0, True)
    _forward(m, 192, 2048, True, "f16", activation, False, True, -2.0, False)


@pytest.mark.parametrize("bias,residual,save", list(itertools.product([False, True], repeat=3)))
@pytest.mark.parametrize("m,n", [(9, 320), (200, 320), (2500, 2304)])
def test_parts_of_the_epilogue(bias, residual, save, m, n):
    _forward(m, 128, n, False, "bf16", "relu", bias, residual, 1.0, save)


@pytest.mark.parametrize("extra", [1, 8, 24])
@pytest.mark.parametrize("m,k,n", [(5, 128, 256), (300, 136, 264), (2400, 128, 2304), (2400, 131, 2309)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_of_wider_tensors(m, k, n, extra, dtype):
    for tr in (False, True):
        _forward(m, k, n, tr, dtype, "silu", True, True, 1.0, True, extra=extra)


@pytest.mark.parametrize("m,n", [(6, 200), (300, 264), (2400, 2312)])
def test_results_in_slices_leave_the_rest_alone(m, n):
    """out and pre_activation as column slices, off a 16-byte boundary or not."""
    dt = torch.bfloat16
    x, w, b = _normal(1, m, 64).to(dt), _normal(2, 64, n).to(dt), _normal(3, n).to(dt)
    want_pre = torch.empty((m, n), dtype=dt, device="cuda")
    want = pd.matmul_fused(x, w, bias=b, activation=pd.ACT_RELU, pre_activation=want_pre)
    for left, right in ((8, 16), (3, 2), (8, 1)):
        wide, wide_pre = (torch.full((m + 1, n + left + right), 9.0, dtype=dt, device="cuda") for _ in range(2))
        out, pre = wide[:m, left:left + n], wide_pre[:m, left:left + n]
        pd.matmul_fused(x, w, bias=b, activation=pd.ACT_RELU, pre_activation=pre, out=out)
        assert torch.equal(out, want) and torch.equal(pre, want_pre)
        for t in (wide, wide_pre):
            assert (t[m:] == 9).all() and (t[:, :left] == 9).all() and (t[:, left + n:] == 9).all()


@pytest.mark.parametrize("m", [4, 300, 2400])
def test_residual_in_place_and_repeatable(m):
    dt = torch.float16
    x, w, r = _normal(1, m, 512).to(dt), _normal(2, 512, 2048, std=0.05).to(dt), _normal(3, m, 2048).to(dt)
    want = pd.matmul_fused(x, w, activation=pd.ACT_SILU, residual=r)
    for _ in range(3):
        assert torch.equal(pd.matmul_fused(x, w, activation=pd.ACT_SILU, residual=r), want)
    got = pd.matmul_fused(x, w, activation=pd.ACT_SILU, residual=r, out=r)
    assert got.data_ptr() == r.data_ptr() and torch.equal(r, want)


def _gradients(m, k, n, tr, dtype, activation, input_activation, scale, extra=0, seed=0):
    dt = DTYPES[dtype]
    dy, w = _normal(seed, m, n).to(dt), _normal(seed + 1, *((n, k) if tr else (k, n)), std=n ** -0.5).to(dt)
    x = _normal(seed + 2, m, k).to(dt)
    pre = _normal(seed + 3, m, n).to(dt) if activation != "none" else None
    input_pre = _normal(seed + 4, m, k).to(dt) if input_activation != "none" else None
    if extra:
        dy, w, x = (_pitched(t, extra) for t in (dy, w, x))
        pre, input_pre = (None if t is None else _pitched(t, extra) for t in (pre, input_pre))
    dx, dw, db = pd.matmul_fused_grad(dy, x, w, transpose_rhs=tr, activation=ACTS[activation], pre_activation=pre, scale=scale,
                                      input_activation=ACTS[input_activation], input_pre_activation=input_pre)
    assert_no_device_error()
    dz = scale * dy.double() * (1 if pre is None else slope(activation, pre.double()))
    # dz as it is multiplied: a rounding of its type (none where dz is dy), and the slope's own error
    rounding = 0.0 if activation == "none" and scale == 1 else half_step(dt)
    dz_off = rounding * dz.abs() + (0 if pre is None else 2.0 ** -20 * abs(scale) * dy.double().abs() * (1 + pre.double().abs()))
    wd, xd = (w.double().t() if tr else w.double()), x.double()
    big = dz.abs() + dz_off
    off = dz_off @ wd.abs().t() + _sum_error(big, wd.t(), dt)
    want = dz @ wd.t()
    if input_pre is not None:
        s = slope(input_activation, input_pre.double())
        off = off * s.abs() + 2.0 ** -20 * (want.abs() + off) * (1 + input_pre.double().abs())
        want = want * s
    close(dx, want, off + 2.0 ** -23 * want.abs(), "dx")
    want, off = xd.t() @ dz, xd.abs().t() @ dz_off + _sum_error(xd.t(), big, dt)
    close(dw, want.t() if tr else want, off.t() if tr else off, "dw")
    close(db, dz.sum(0), (dz_off + (m + 8) * 2.0 ** -23 * big).sum(0), "db")


@pytest.mark.parametrize("m,k,n", [(1, 64, 64), (1, 1, 1), (3, 7, 5), (17, 520, 200), (61, 128, 1000), (250, 512, 264),
                                   (515, 257, 131), (2100, 320, 2304), (4200, 1024, 136)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tr", [False, True])
def test_gradients(m, k, n, dtype, tr):
    _gradients(m, k, n, tr, dtype, "gelu", "none", 1.0)
    _gradients(m, k, n, tr, dtype, "none", "silu", 0.7)


@pytest.mark.parametrize("activation", sorted(ACTS))
def test_gradients_of_activations(activation):
    _gradients(300, 136, 264, False, "bf16", activation, "none", 1.0)
    _gradients(300, 136, 264, True, "f16", "none", activation, 1.0)
    _gradients(2400, 2304, 64, True, "bf16", activation, activation, -1.5)


@pytest.mark.parametrize("extra", [1, 8])
def test_gradients_of_rows_of_wider_tensors(extra):
    for tr in (False, True):
        _gradients(300, 136, 264, tr, "bf16", "relu", "gelu", 1.0, extra=extra)
        _gradients(130, 36, 64, tr, "f32", "relu", "gelu", 1.0, extra=extra)


def test_gradients_that_are_not_wanted():
    dt = torch.bfloat16
    dy, x, w = _normal(1, 40, 64).to(dt), _normal(2, 40, 96).to(dt), _normal(3, 96, 64).to(dt)
    every = pd.matmul_fused_grad(dy, x, w, scale=0.5)
    for i in range(3):
        want = [j == i for j in range(3)]
        some = pd.matmul_fused_grad(dy, x, w, scale=0.5, want_lhs_grad=want[0], want_rhs_grad=want[1], want_bias_grad=want[2])
        assert [t is not None for t in some] == want and torch.equal(some[i], every[i])


def test_gradients_against_differences():
    """The forward call's own differences, in fp32: the loss sum(out * dy) along a random direction."""
    m, k, n = 24, 40, 36
    x, w, b, dy = _normal(1, m, k), _normal(2, k, n, std=0.2), _normal(3, n), _normal(4, m, n)
    for activation in ("gelu", "silu", "tanh", "sigmoid"):
        pre = torch.empty((m, n), device="cuda")
        pd.matmul_fused(x, w, bias=b, activation=ACTS[activation], scale=0.7, pre_activation=pre)
        grads = pd.matmul_fused_grad(dy, x, w, activation=ACTS[activation], pre_activation=pre, scale=0.7)
        for i, t in enumerate((x, w, b)):
            d = _normal(10 + i, *t.shape)
            h = 2.0 ** -6
            ends = []
            for sign in (1, -1):
                args = [x, w, b]
                args[i] = t + sign * h * d
                ends.append((pd.matmul_fused(args[0], args[1], bias=args[2], activation=ACTS[activation], scale=0.7).double() * dy).sum())
            want = (grads[i].double() * d).sum()
            # third derivatives of the activations are below 2, and of the order of h^2 / 6 of them is left: summed over the
            # outputs' |dy| |dz|^3.  The ends are off by 2^-19 of the terms' sizes, divided by 2 h.
            dz = (d @ w if i == 0 else x @ d if i == 1 else d.expand(m, n)).double()
            allowed = 0.7 * 2 * h * h / 6 * (dy.double().abs() * dz.abs() ** 3).sum() + 2.0 ** -19 / h * \
                (dy.double().abs() * (1 + x.double().abs() @ w.double().abs())).sum() * 0.7
            assert (((ends[0] - ends[1]) / (2 * h)) - want).abs() <= allowed, (activation, i)


def test_no_rows():
    dt = torch.float16
    x, w = torch.empty((0, 64), dtype=dt, device="cuda"), _normal(1, 64, 32).to(dt)
    assert pd.matmul_fused(x, w).shape == (0, 32)
    dx, dw, db = pd.matmul_fused_grad(torch.empty((0, 32), dtype=dt, device="cuda"), x, w)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all() and dw.shape == (64, 32)


def test_infinities_and_nan_stay_in_their_rows():
    dt = torch.bfloat16
    for m in (6, 300, 2400):
        x, w = _normal(1, m, 128).to(dt), _normal(2, 128, 2304, std=0.1).to(dt)
        want = pd.matmul_fused(x, w, activation=pd.ACT_RELU)
        x[3, 5] = float("nan")
        x[4, 7] = float("inf")
        got = pd.matmul_fused(x, w, activation=pd.ACT_RELU)
        assert torch.isnan(got[3]).all()
        keep = [i for i in range(m) if i not in (3, 4)]
        assert torch.equal(got[keep], want[keep])
        z = torch.where(w[7] > 0, float("inf"), 0.0)
        assert torch.equal(got[4][w[7] != 0].float(), z[w[7] != 0])


def test_streams_and_graphs():
    """Calls on two streams at once, and two captured graphs replayed side by side, give what calls alone give."""
    dt = torch.bfloat16
    sets = []
    for i in range(2):
        x, w = _normal(i, 300, 520).to(dt), _normal(5 + i, 515, 520).to(dt)
        dy, pre = _normal(7 + i, 300, 515).to(dt), _normal(9 + i, 300, 515).to(dt)
        sets.append((x, w, dy, pre))

    def call(x, w, dy, pre):
        return [pd.matmul_fused(x, w, transpose_rhs=True, activation=pd.ACT_GELU)] + \
            list(pd.matmul_fused_grad(dy, x, w, transpose_rhs=True, activation=pd.ACT_GELU, pre_activation=pre))

    want = [call(*s) for s in sets]
    torch.cuda.synchronize()
    streams, graphs, got = [torch.cuda.Stream() for _ in sets], [], []
    for s, stream in zip(sets, streams):
        with torch.cuda.stream(stream):
            call(*s)
    torch.cuda.synchronize()
    for s, stream in zip(sets, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            got.append(call(*s))
        graphs.append(g)
    for _ in range(5):
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    assert_no_device_error()


def test_refusals():
    dt = torch.bfloat16
    x, w, b = _normal(1, 8, 16).to(dt), _normal(2, 16, 24).to(dt), _normal(3, 24).to(dt)
    for bad in (dict(rhs=w.t().contiguous()), dict(bias=b[:23]), dict(bias=b.float()), dict(residual=x), dict(rhs=w.float()),
                dict(lhs=x.t()), dict(out=torch.empty((8, 25), dtype=dt, device="cuda")), dict(lhs=x.cpu()), dict(lhs=x.flatten()),
                dict(residual=torch.empty((1, 24), dtype=dt, device="cuda").expand(8, 24))):
        args = dict(lhs=x, rhs=w, bias=b)
        args.update(bad)
        with pytest.raises(ValueError):
            pd.matmul_fused(**args)
    with pytest.raises(pd.PortDNNError):
        pd.matmul_fused(x, w, activation=5)
    with pytest.raises(pd.PortDNNError):  # the slope of an activation needs its argument
        pd.matmul_fused_grad(_normal(4, 8, 24).to(dt), x, w, activation=pd.ACT_GELU)
    with pytest.raises(KeyError):
        pd.matmul_fused(x.double(), w.double())
    for f in (lambda: pd.pointwise(pd.ACT_GELU, x), lambda: pd.bias_add(x, b[:16].contiguous(), 16, activation=pd.ACT_SILU)):
        with pytest.raises(pd.PortDNNError):
            f()


@pytest.mark.parametrize("m,k,n,dtype,kernel", [
    (8192, 256, 2048, "bf16", r"pair_gemm_kernelI13__nv_bfloat16Li256ELb0"), (4000, 128, 512, "f16", r"pair_gemm_kernelI6__halfLi128ELb0"),
    (1, 4096, 4096, "bf16", r"solo_gemm_kernelI13__nv_bfloat16Lb0"), (250, 2048, 1000, "f16", r"solo_gemm_kernelI6__halfLb0"),
    (4096, 128, 1024, "f32", r"pair_gemm_kernelIfLi128ELb1"), (300, 520, 515, "f32", r"solo_gemm_kernelIfLb1"),
    (1, 512, 512, "f32", r"rows_product_kernelILi1E"), (16, 512, 511, "f32", r"rows_product_kernelILi8ELi1E")])
def test_every_kernel_is_reached(m, k, n, dtype, kernel):
    """The kernels that the other tests' shapes run on, by the names in a captured call."""
    dt = DTYPES[dtype]
    x, w = _normal(1, m, k).to(dt), _normal(2, k, n).to(dt)
    names = [launch.name for launch in launched(lambda: pd.matmul_fused(x, w, activation=pd.ACT_RELU))]
    assert re.search(kernel, names[-1]), names
    _forward(m, k, n, False, dtype, "silu", True, True, 1.0, True)
    _forward(m, k, n, True, dtype, "relu", False, False, 1.0, False)


def test_long_sums_in_single_precision():
    """Where the accumulator's own rounding would show: the error does not grow with the number of terms."""
    for m, n in ((300, 200), (2300, 1100)):
        x, w = _normal(1, m, 8192), _normal(2, 8192, n)
        got, want = pd.matmul_fused(x, w).double(), x.double() @ w.double()
        # chains of 64 terms in the accumulator (12 additions to a step of two, 24 in all, each off by 2^-23 of the chain's sum at
        # most), 128 chains added with 2^-24 each: norm-wise, for sums of terms of random signs, 24 2^-23 + sqrt(128) 2^-24
        assert (got - want).norm() <= (24 * 2.0 ** -23 + 12 * 2.0 ** -24) * want.norm()


def test_calls_follow_their_tensors_device_and_stream():
    """On a stream that waits for the one that makes its inputs; the tensors' device is the current one already on a box of one GPU."""
    dt = torch.bfloat16
    x, w = _normal(1, 2000, 2048).to(dt), _normal(2, 2048, 2048, std=0.02).to(dt)
    want = pd.matmul_fused(pd.matmul_fused(x, w), w)
    side = torch.cuda.Stream()
    for _ in range(3):
        y = pd.matmul_fused(x, w)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = pd.matmul_fused(y, w)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
    if torch.cuda.device_count() > 1:
        there = [t.to("cuda:1") for t in (x, w)]
        assert torch.equal(pd.matmul_fused(pd.matmul_fused(*there), there[1]).to("cuda:0"), want)


def test_results_on_operands_are_refused_and_slices_beside_them_are_not():
    dt = torch.bfloat16
    wide = _normal(1, 300, 512).to(dt)
    w, r = _normal(2, 128, 128).to(dt), _normal(3, 300, 128).to(dt)
    x = wide[:, :128]
    want = pd.matmul_fused(x, w, residual=r)
    got = pd.matmul_fused(x, w, residual=r, out=wide[:, 256:384])  # beside the operand, in the same rows
    assert torch.equal(got, want)
    pre = torch.empty_like(want)
    for bad in (dict(out=x), dict(out=wide[:, 64:192]),
                dict(out=pre, pre_activation=pre), dict(pre_activation=r), dict(pre_activation=x)):
        with pytest.raises((pd.PortDNNError, ValueError)):
            pd.matmul_fused(x, w, residual=r, **bad)
    # the residual shifted by a row is not the residual in place
    tall = torch.cat([r, r[:1]])
    with pytest.raises(pd.PortDNNError):
        pd.matmul_fused(x, w, residual=tall[:-1], out=tall[1:])
    dy = _normal(4, 300, 128).to(dt)
    for bad in (dict(lhs_grad=dy), dict(rhs_grad=w), dict(lhs_grad=x), dict(bias_grad=w[5])):
        with pytest.raises(pd.PortDNNError):
            pd.matmul_fused_grad(dy, x.contiguous() if "lhs_grad" not in bad else x, w, **bad)
