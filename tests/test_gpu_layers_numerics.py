"""How exact the 16-bit layers are where 16 bits could cost more than the one rounding of each result, against the
formulas in 64 bits.

u = half a step of the element type (bf16 2^-8, fp16 2^-11), relative to a value.  Activations and their derivatives are
computed in fp32 with the hardware's exp2 and reciprocal: an argument of exp2 of magnitude A is off by 2^-24 A times two
roundings, so a derivative that is 2^-A is off by at most 2^-23 A + 2^-20 of itself, below 2^-15 for all A up to 150."""
import math

import pytest
import torch

from test_gpu_layers import HALF, TINY, TYPES, act64, gpu, rand, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layers():
    from bnp_vae_amd import layers as module
    return module


# ------------------------------------------------------------------------------------------------ derivatives far out
@pytest.mark.parametrize("act,most", [("softsign", 3e4), ("tanh", 40.0), ("silu", 80.0)])
@pytest.mark.parametrize("M", [8, 96])
def test_small_derivatives_keep_their_bits(layers, act, most, M):
    """bf16 holds the derivative far from 0 (softsign' is 1e-8 at 1e4), so the gradient has it too: relative to itself,
    not to 1.  z = x[:, 0] exactly, dx[:, 0] = dy act'(z), rounded to 16 bits where it is dz and where it is dx."""
    T = torch.bfloat16
    z = (torch.linspace(1.0, math.log2(most), M) ** 2 / math.log2(most)).exp2().to(T)
    z[::2] = -z[::2]
    if act == "silu":
        z = -z.abs()                              # towards + infinity its derivative is 1
    x = torch.zeros((M, 16), dtype=T)
    x[:, 0] = z
    w = torch.zeros((8, 16), dtype=T)
    w[0, 0] = 1
    X = gpu(x).requires_grad_(True)
    y = layers.dense(X, gpu(w), activation=act)
    dy = torch.zeros((M, 8), dtype=T)
    dy[:, 0] = rand((M,), T, 3)
    dx, = torch.autograd.grad(y, X, gpu(dy))
    want = dy[:, 0].double() * act64(act, z.double())[1]
    within(dx[:, 0], want, (2 * 2.0 ** -8 + 2.0 ** -14) * want.abs() + TINY[T])
