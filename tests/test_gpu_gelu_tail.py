"""The fused product's activations of f32 outputs hold their value to f32's accuracy far out on the left too, where an
absolute bound says nothing.

Every output is one bf16 value y (one entry of x is 1, the others 0). Tolerance relative to the value: eight roundings of
2^-24 for the polynomial, reciprocal, exponential and products, another eight for the polynomial's own error, and the
exponent, y^2 / 2 or the gate's argument z in powers of two: two roundings of it, at most 2^-23 of y^2 / 2 and of z. Where a
sigmoid is below f32's smallest normal number it counts as 0: off by at most |y| 2^-126."""
import math

import pytest
import torch

from glm53f_forward import ffi

import harness as hs
from harness import ptr

pytestmark = pytest.mark.gpu
DEV = hs.DEV


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "sigmoid"])
@pytest.mark.parametrize("rows", [1, 300])
def test_values_of_the_left_tail(act, rows):
    n, k = 1024, 64
    y = -torch.exp(torch.linspace(math.log(1e-3), math.log(12.0), n)).bfloat16()
    y[::4] = -y[::4]
    w = torch.zeros(n, k, dtype=torch.bfloat16)
    w[:, 5] = y
    x = torch.zeros(rows, k, dtype=torch.bfloat16)
    x[:, 5] = 1.0
    d_x, d_w, out = x.to(DEV), w.to(DEV), torch.zeros(rows, n, device=DEV)
    code = ("none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid").index(act)
    assert ffi.glm53f_fwd_gemm_bf16_fused(ptr(d_x), k, 0, ptr(d_w), k, 0, 1, rows, n, k, None, 0, code, None, 0, 0, ptr(out), 1, n, 0, None) == 0
    hs.sync()
    y = y.double()
    z = 2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3) if act == "gelu_tanh" else y
    want = {"silu": y * torch.sigmoid(y), "gelu": 0.5 * y * torch.special.erfc(-y / math.sqrt(2)), "gelu_tanh": y * torch.sigmoid(z),
            "sigmoid": torch.sigmoid(y)}[act]
    tol = (16 * 2.0 ** -24 + 2.0 ** -23 * (y * y / 2 if act == "gelu" else z.abs())) * want.abs() + 2.0 ** -126 * (1 + y.abs())
    err = (out.cpu().double() - want).abs()
    at = int((err / tol).argmax()) % n
    assert bool((err <= tol).all()), f"{float((err / tol).max()):.2f} of the tolerance at {float(y[at])}"
