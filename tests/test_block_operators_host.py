"""Refusals of the operators around a block's matrix products that need no GPU: parameters the C ABI checks before it looks for
a device, tensors that are not on one, and the sizes of the mirrored structures."""
import ctypes

import pytest
import torch

import portdnn_b200 as pd

INVALID, INDEX = 5, 2


class MatmulParams(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("m", "k", "n", "transpose_rhs")] + \
        [(n, ctypes.c_longlong) for n in ("lhs_pitch", "rhs_pitch", "output_pitch")]


class MatmulEpilogue(ctypes.Structure):
    _fields_ = [("bias", ctypes.c_void_p), ("activation", ctypes.c_int), ("scale", ctypes.c_float), ("residual", ctypes.c_void_p),
                ("residual_pitch", ctypes.c_longlong), ("pre_activation", ctypes.c_void_p), ("pre_activation_pitch", ctypes.c_longlong)]


class PolicyLossParams(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("rows", "vocab", "target_bytes")] + \
        [(n, ctypes.c_float) for n in ("clip_low", "clip_high", "kl", "temperature", "grad_scale")] + \
        [(n, ctypes.c_longlong) for n in ("logits_pitch", "grad_pitch")]


def _fused(dtype=0, activation=-1, params=(8, 16, 24, 0, 0, 0, 0), null=False):
    p, e = MatmulParams(*params), MatmulEpilogue(None, activation, 1.0, None, 0, None, 0)
    return pd.lib().pdnn_matmul_fused(dtype, None, None, None, None if null else ctypes.byref(p), ctypes.byref(e), None)


def test_matmul_fused_parameters():
    assert _fused(null=True) == INVALID
    for bad in (dict(dtype=3), dict(dtype=-1), dict(activation=3), dict(activation=10), dict(activation=-2),
                dict(params=(-1, 16, 24, 0, 0, 0, 0)), dict(params=(8, 0, 24, 0, 0, 0, 0)), dict(params=(8, 16, -3, 0, 0, 0, 0)),
                dict(params=(8, 16, 24, 0, 15, 0, 0)), dict(params=(8, 16, 24, 0, 0, 23, 0)), dict(params=(8, 16, 24, 1, 0, 15, 0)),
                dict(params=(8, 16, 24, 0, 0, 0, -24))):
        assert _fused(**bad) == INVALID, bad
        assert pd.lib().pdnn_last_error()


@pytest.mark.parametrize("sizes", [(2 ** 31 - 1, 1, 1), (1, 2 ** 31 - 1, 1), (1, 1, 2 ** 31 - 1)])
def test_matmul_fused_counts_past_its_sizes(sizes):
    assert _fused(params=sizes + (0, 0, 0, 0)) == INVALID
    assert b"too large" in pd.lib().pdnn_last_error()


def _norm(rows=8, channels=64, post=1, pre=1, groups=0, act=-1, epsilon=1e-6, dtype=0):
    p = pd.ResidualNormParams(rows, channels, post, pre, groups, act, 1.0, epsilon)
    tensors, gradients = (ctypes.c_void_p * 10)(), (ctypes.c_void_p * 9)()
    forward = pd.lib().pdnn_residual_norm(dtype, ctypes.byref(p), tensors, None)
    assert pd.lib().pdnn_residual_norm_gradient(dtype, ctypes.byref(p), tensors, gradients, None) == forward
    return forward


def test_residual_norm_parameters():
    for bad in (dict(rows=-1), dict(channels=0), dict(post=3), dict(pre=-1), dict(groups=-1), dict(groups=3), dict(act=5),
                dict(epsilon=-1.0), dict(epsilon=float("nan")), dict(dtype=7), dict(groups=2), dict()):  # (the last two: null tensors)
        assert _norm(**bad) == INVALID, bad
    assert pd.lib().pdnn_residual_norm(0, None, None, None) == INVALID


@pytest.mark.parametrize("sizes", [dict(rows=2 ** 31 - 1, channels=1), dict(rows=1, channels=2 ** 31 - 1)])
def test_residual_norm_counts_past_its_sizes(sizes):
    assert _norm(**sizes) == INVALID
    assert b"too many" in pd.lib().pdnn_last_error()


def test_norm_results_on_vectors():
    p = pd.ResidualNormParams(8, 64, 1, 1, 0, -1, 1.0, 1e-6)
    far = [0x10000000 * (i + 1) for i in range(10)]  # (addresses that nothing reads: branch, residual, five vectors, sum, output, statistics)
    far[4] = None
    for result in (7, 8):
        for vector in (2, 3, 5, 6):
            at = list(far)
            at[result] = far[vector] - 8 * 64 * 4 + 16
            assert pd.lib().pdnn_residual_norm(0, ctypes.byref(p), (ctypes.c_void_p * 10)(*at), None) == INVALID
            assert b"vector" in pd.lib().pdnn_last_error()
            gradients = (ctypes.c_void_p * 9)(0xB0000000, 0xC0000000, *((at[result], None) if result == 7 else (None, at[result])))
            assert pd.lib().pdnn_residual_norm_gradient(0, ctypes.byref(p), (ctypes.c_void_p * 10)(*far), gradients, None) == INVALID
            assert b"vector" in pd.lib().pdnn_last_error()


def test_policy_loss_parameters():
    def run(rows=4, vocab=100, target_bytes=8, low=0.2, high=0.2, temperature=1.0, pitch=100, grad_pitch=100, dtype=0):
        p = PolicyLossParams(rows, vocab, target_bytes, low, high, 0.1, temperature, 1.0, pitch, grad_pitch)
        tensors = (ctypes.c_void_p * 10)()
        return pd.lib().pdnn_policy_loss(dtype, ctypes.byref(p), tensors, None)

    for bad in (dict(rows=-1), dict(vocab=0), dict(target_bytes=2), dict(low=-0.1), dict(high=float("nan")), dict(temperature=0.0),
                dict(temperature=-1.0), dict(temperature=float("inf")), dict(temperature=float("nan")), dict(pitch=99), dict(dtype=3), dict()):
        assert run(**bad) == INVALID, bad
    assert run(vocab=2 ** 30 + 1, pitch=2 ** 31) == INDEX
    assert pd.lib().pdnn_policy_loss(0, None, None, None) == INVALID


def test_tensors_have_to_be_on_a_gpu():
    x, v = torch.ones((4, 8)), torch.ones(8)
    for call in (lambda: pd.matmul_fused(x, x.t().contiguous()), lambda: pd.matmul_fused_grad(x, x, x),
                 lambda: pd.residual_norm(x, x, pd.residual_norm_params(4, 8), post_gamma=v),
                 lambda: pd.residual_norm_grad(x, x, x, x, x, pd.residual_norm_params(4, 8)),
                 lambda: pd.policy_loss(x, torch.zeros(4, dtype=torch.long), torch.ones(4)),
                 lambda: pd.matmul_fused(None, x), lambda: pd.policy_loss(None, x, x)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: pd.matmul_fused("x", x), lambda: pd.residual_norm(x, x, None)):
        with pytest.raises((TypeError, ValueError)):
            call()


def test_new_activations_are_for_the_new_operators_only():
    class Epilogue(ctypes.Structure):
        _fields_ = [("bias", ctypes.c_void_p), ("activation", ctypes.c_int), ("alpha", ctypes.c_float), ("beta", ctypes.c_float),
                    ("relu_bitmask", ctypes.c_void_p), ("constant_filter", ctypes.c_int), ("any_order", ctypes.c_int)]

    p, e = pd.conv_params(1, 8, 8, 16, 16, 3, 1), Epilogue(None, pd.ACT_GELU, 1.0, 0.0, None, 0, 0)
    assert pd.lib().pdnn_conv2d_fused(1, None, None, None, ctypes.byref(p), pd.ALGO_IM2COL, ctypes.byref(e), None, 0, None) == INVALID
