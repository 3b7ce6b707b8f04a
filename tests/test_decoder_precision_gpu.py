"""How closely the activations of ``linear`` and their derivatives follow the formulas far out, relative to their own
size: saturated units have small derivatives, not none, whatever kernel their layer's sizes select.

With the identity as weight z is x itself and a gradient of ones comes back as the derivative: every other term of the
sums is an exact zero.  So all error is the activation's evaluation in 32 bits, and one rounding to the tensors' type.

The evaluation, counted in e = 2^-24 of what is added up (to first order; the sums below leave half as much again):
exp(-|z|) has its argument rounded twice (2 |z| e) and its own result (2 e for an instruction good to one unit in the
last place); a reciprocal has 2 e and the sum in it e; each further product e: sigmoid and its derivative stay within
(2 |z| + 9) e.  exp(-z^2 / 2) has its argument rounded three times (1.5 z^2 e); a polynomial of positive total with ten
coefficients adds 2 e for each, its variable 3 e, what it approximates 1 e: Phi and the density stay within
(1.5 z^2 + 30) e."""
import math

import pytest
import torch

import decoder_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F = torch.float64
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# rows, width: few rows; rows streaming past the weight; tiles straight into shared memory, whole and cut along the
# reduction; tiles through registers
FORMS = {"few": (48, 64), "streamed": (300, 128), "tiles": (300, 512), "cut": (100, 1024), "registers": (200, 301)}
# how far z goes
RANGES = {"silu": (-24.0, 24.0), "sigmoid": (-24.0, 24.0), "gelu": (-12.0, 12.0)}


def exact(z, act):
    """-> value, derivative, and what the terms that the derivative adds up come to, in 64 bits"""
    if act == "gelu":
        # (torch's ndtr is a sum about 1 on this device, and zero below -8.3)
        phi, pdf = torch.erfc(-z / math.sqrt(2)) / 2, torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * phi, phi + z * pdf, phi + z.abs() * pdf
    up, down = torch.sigmoid(z), torch.sigmoid(-z)
    if act == "silu":
        return z * up, up + z * up * down, up + z.abs() * up * down
    return up, up * down, up * down


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("act", sorted(RANGES))
@pytest.mark.parametrize("form", sorted(FORMS))
def test_activations_keep_their_size(form, act, dtype):
    from neuralgaussiansplatting_amd import decoder_ops as ops
    rows, width = FORMS[form]
    g = torch.Generator(device=DEV).manual_seed(width)
    z = torch.linspace(*RANGES[act], rows * width, device=DEV)
    x = z[torch.randperm(rows * width, generator=g, device=DEV)].view(rows, width).to(dtype).requires_grad_()
    eye = torch.eye(width, device=DEV, dtype=dtype)
    y = ops.linear(x, eye, activation=act)
    (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    z = x.detach().to(F)
    value, slope, terms = exact(z, act)
    rel = 1.5 * (1.5 * z * z + 30 if act == "gelu" else 2 * z.abs() + 9) * ref.E
    ref.assert_within(y, (value, ref.rounded(value, rel * value.abs(), dtype)), "y")
    ref.assert_within(dx, (slope, ref.rounded(slope, rel * terms, dtype)), "dx")
