"""How far the activations of group norm are from their values in 64 bits, as ops.group_norm states it.

With a group for each channel of one row h is 0, so z = bias and y = act(bias) exactly as the kernels compute it, and db = dy act'(bias).  u = 2^-24.
  silu   z s, s = 1 / (1 + e^-z): e^-z = 2^(-z log2 e) has its exponent rounded (|z| u relative) and takes log2 e as a float32, which is off by 0.224 u of
         itself (0.224 |z| u relative); then an u or two of its own, the sum, the reciprocal and the product one each: (1.25 |z| + 4) u of the value.  Its
         slope s (1 + z (1 - s)) has 1 - s off by u and a relative error of s: (2 |z| + 8) u.
  gelu   z Phi(z): the polynomial is off by 7.5e-8, the six roundings of t p e / 2 (at most 1/2) by 1.8e-7 at most, the rest by an u: 3.2e-7 |z| in all.
         Its slope Phi(z) + z pdf(z): the same and six roundings of z pdf(z), which is at most 0.242: 4e-7.
So float32 results of gelu have lost digits far on the negative side, where the value itself is small."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_distance_from_64_bits(act):
    import ogl_amd  # noqa: F401
    from ogl_amd import ops
    n = 1 << 20
    z = torch.linspace(-16, 16, n, device="cuda")
    x, w, b = torch.randn(1, n, device="cuda"), torch.ones(n, device="cuda"), z.clone().requires_grad_()
    y = ops.group_norm(x, n, w, b, activation=act)
    (slope,) = torch.autograd.grad(y, b, torch.ones_like(y))
    zd = z.double()
    if act == "silu":
        s = torch.sigmoid(zd)
        want, want_slope = zd * s, s * (1 + zd * (1 - s))
        bound, bound_slope = (1.25 * zd.abs() + 4) * U * want.abs(), (2 * zd.abs() + 8) * U
    else:
        phi = 0.5 * torch.special.erfc(-zd / 2 ** 0.5)
        want, want_slope = zd * phi, phi + zd * torch.exp(-0.5 * zd * zd) / (2 * torch.pi) ** 0.5
        bound, bound_slope = 3.2e-7 * zd.abs(), 4e-7
    assert ((y.detach()[0].double() - want).abs() <= bound).all()
    assert ((slope.double() - want_slope).abs() <= bound_slope).all()
