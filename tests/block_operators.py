"""Shared by the tests of the operators around a block's matrix products: activations and their slopes in 64 bits, tolerances."""
import math

import torch

import portdnn_b200 as pd

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTS = {"none": pd.ACT_NONE, "relu": pd.ACT_RELU, "tanh": pd.ACT_TANH, "relu6": pd.ACT_RELU6, "gelu": pd.ACT_GELU,
        "silu": pd.ACT_SILU, "sigmoid": pd.ACT_SIGMOID}


def act(name, z):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "tanh": lambda: torch.tanh(z),
            "relu6": lambda: z.clamp(min=0, max=6), "gelu": lambda: 0.5 * z * torch.erfc(-z / math.sqrt(2)),
            "silu": lambda: z * torch.sigmoid(z), "sigmoid": lambda: torch.sigmoid(z)}[name]()


def slope(name, z):
    s = torch.sigmoid(z)
    return {"none": lambda: torch.ones_like(z), "relu": lambda: (z > 0).double(), "tanh": lambda: 1 - torch.tanh(z) ** 2,
            "relu6": lambda: ((z > 0) & (z < 6)).double(),
            "gelu": lambda: 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
            "silu": lambda: s * (1 + z * (1 - s)), "sigmoid": lambda: s * (1 - s)}[name]()


def half_step(dtype):
    """How far one rounding to the type is off at most, relative to the value."""
    return torch.finfo(dtype).eps / 2


def close(got, want, allowed, what):
    """|got - want| <= half a step of got's type times |want|, plus `allowed`; below the type's normal numbers half of its
    smallest step."""
    want, allowed = want.double(), torch.as_tensor(allowed, dtype=torch.float64, device=got.device)
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    limit = half_step(got.dtype) * (want.abs() + allowed) + allowed + tiny
    off = (got.double() - want).abs()
    assert not torch.isnan(off).any(), "%s: NaN" % what
    bad = off > limit
    assert not bad.any(), "%s: %d of %d off, the worst %.3g of what is allowed" % (
        what, int(bad.sum()), bad.numel(), float((off / limit).max()))
