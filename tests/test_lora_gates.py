"""strasgpt_k_lora's SwiGLU where silu(g) u is far from its usual sizes: gates of -30 to
-95, for which silu is 1e-12 to 1e-39, gates that no exponential holds, infinite ones, ups
of up to 1e30. Few tokens and many (512 are the most of the few) give the same values.

Tolerance, relative to the result, with h = 2^-24 and b = 2^-8 (half a step of bf16). For a
gate below -2 an error d of the gate, 0.3 at most, makes silu(g + d) / silu(g) at most
e^d (1 + d / 2), which is below 1 + 2 d; else silu's slope is at most 1.1. An up that is off
by e adds |silu| e. bf16: exp2 of g log2(e), whose rounding and constant are off by
1.5 h |g log2(e)|, which moves the result by 1.5 h |g| (95 at most: 2^-16.9), a few
approximate operations of 2^-22 each: 2^-16 in all, and b. fp32: 8 h for exp, division and
products; 1 / (1 + e^-g) is below the normal numbers for gates below -87, and 0 below -88.7
(as in the framework's other SwiGLUs): 2^-126 |g u| there.
"""
import pytest
import test_lora as lora

F32, BF16, SWIGLU = lora.F32, lora.BF16, lora.SWIGLU
H, B = lora.H, lora.B


def inputs(torch, m, type_, seed, n=200):
    x, a, b, adapter, scale, base = lora.inputs(torch, m, 64, n, 8, 3, type_, seed)
    adapter[m // 3:m // 3 + 70] = 1     # runs as well
    return x, a, b, adapter, scale, base


def expected(torch, x, a, b, adapter, scale, base, type_):
    """Float64 result and the bound on its error."""
    v, err = lora.reference(torch, x, a, b, adapter, scale, base, None, lora.STORE, F32)
    if type_ == BF16:    # A x in two parts
        err = lora.reference(torch, x, a, b, adapter, scale, base, None, lora.STORE, BF16)[1]
        err = err - B * (v.abs() + err) / (1 + B)
    err[adapter < 0] = 0.0    # v is base
    g, u, dg, du = v[:, 0::2], v[:, 1::2], err[:, 0::2], err[:, 1::2]
    s = g * torch.sigmoid(g)
    ds = torch.where(g < -2, 2 * dg * s.abs(), 1.1 * dg)
    tol = u.abs() * ds + (s.abs() + ds) * du
    y = s * u
    if type_ == BF16:
        tol = tol + 2.0 ** -16 * y.abs()
        tol = tol + B * (y.abs() + tol)
    else:
        tol = tol + 8 * H * y.abs() + torch.where(g < -87, 2.0 ** -126 * (g * u).abs(), 0.0)
    return y, tol


def call(torch, x, a, b, adapter, scale, base, type_):
    out = torch.full((x.shape[0], base.shape[1] // 2), 7.0, device="cuda", dtype=x.dtype)
    assert lora.call(torch, x, a, b, adapter, scale, base, out, SWIGLU, type_) == 0
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("m", [40, 512, 513, 1000])
def test_gates_far_below_zero(cuda, type_, m):
    torch = cuda
    x, a, b, adapter, scale, base = inputs(torch, m, type_, m)
    base[:, 0::2] = torch.linspace(-95, 5, base[:, 0::2].numel(), device="cuda").view(
        m, -1)[torch.randperm(m, device="cuda")].to(base)
    base[:, 1::2] *= 1e6
    base[1::3, 1::2] *= 1e24
    want, tol = expected(torch, x, a, b, adapter, scale, base, type_)
    got = call(torch, x, a, b, adapter, scale, base, type_).double()
    assert ((got - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("m", [40, 512, 513, 1000])
def test_gates_beyond_any_exponential(cuda, type_, m):
    """Far gates times large ups are 0, infinite and NaN ones what silu makes of them, and
    none of them reaches its neighbours."""
    torch = cuda
    x, a, b, adapter, scale, base = inputs(torch, m, type_, m + 1)
    base[:, 0::2] = 3 * torch.randn(m, base.shape[1] // 2, device="cuda").to(base)
    clean = base.clone()
    far = [(-1e3, 1e30), (-1e20, 1e20), (-3e38, -3e38), (float("-inf"), 1.0), (float("inf"), -2.0),
           (float("nan"), 1.0), (1.0, float("nan")), (2.0, float("inf"))]
    which = torch.arange(m * base.shape[1] // 2, device="cuda").view(m, -1) * 5 % 37
    for i, (g, u) in enumerate(far):
        base[:, 0::2][which == i], base[:, 1::2][which == i] = g, u
    want, tol = expected(torch, x, a, b, adapter, scale, clean, type_)
    got = call(torch, x, a, b, adapter, scale, base, type_).double()
    usual = which >= len(far)
    assert ((got - want).abs() <= tol)[usual].all()
    # (An adapter adds to gate and up, so an infinity's sign is the formula's.)
    v = lora.reference(torch, x, a, b, adapter, scale, base, None, lora.STORE, F32)[0]
    value = v[:, 0::2] * torch.sigmoid(v[:, 0::2]) * v[:, 1::2]
    for i, pair in enumerate(far):
        of = which == i
        assert ((got == value) | (got.isnan() & value.isnan()))[of].all(), pair
    assert (got[which < 3] == 0).all()
