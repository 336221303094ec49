"""strasgpt_k_rope_axes (include/strasgpt_kernels.h): rotary positions with
several axes, against a float64 restatement of its definition.

Tolerance, as strasgpt_k_rope's, with h = 2^-24 (half a step of fp32) and
b = 2^-8 (of bf16): the angle's rounding pi h, its fp32 sine 4 h, the
magnitude's and the product's roundings 2 h, the sum of two products 2 h more:
below 16 h (|a| + |b|) magnitude. bf16 adds b |y|. The float64 reference's
angle is itself off by pos f 2^-53 with f's own 2^-52: at positions below 2^21
less than 2^-30.
"""
import ctypes

import numpy as np
import pytest

from strasgpt_b200 import runtime

F32, BF16 = runtime.F32, runtime.BF16
RUNS, DEALT = runtime.AXES_RUNS, runtime.AXES_DEALT
H, B = 2.0 ** -24, 2.0 ** -8
FAKE = 1 << 20  # aligned, never dereferenced


def dtype(torch, type_):
    return torch.float32 if type_ == F32 else torch.bfloat16


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


def shared_out(sections, order):
    """[(axis, number among the axis's pairs)] of every pair."""
    if order == RUNS:
        return [(a, m) for a, s in enumerate(sections) for m in range(s)]
    return [(a, m) for m in range(max(sections)) for a, s in enumerate(sections) if m < s]


def angles(torch, pos, r, sections, order, separate):
    """[t][dim / 2] in 64 bits; pos [axes][t]."""
    out = []
    for j, (a, m) in enumerate(shared_out(sections, order)):
        f = r.theta ** (-m / sections[a] if separate else -2 * j / r.dim)
        if r.scaling == runtime.ROPE_LINEAR:
            f /= r.factor
        if r.scaling == runtime.ROPE_BANDS:
            keep = np.clip((r.original * f / (2 * np.pi) - r.low) / (r.high - r.low), 0, 1)
            f *= keep + (1 - keep) / r.factor
        out.append(pos[a].double() * f)
    return torch.stack(out, 1)


def check(torch, got, x, pos, r, sections, order, separate, type_):
    x = x.double()
    angle = angles(torch, pos, r, sections, order, separate)[:, None]
    c, s = torch.cos(angle) * r.magnitude, torch.sin(angle) * r.magnitude
    want, size = x.clone(), torch.zeros_like(x)
    half = r.dim // 2
    a, b = ((slice(0, r.dim, 2), slice(1, r.dim, 2)) if r.interleaved
            else (slice(0, half), slice(half, r.dim)))
    want[..., a] = x[..., a] * c - x[..., b] * s
    want[..., b] = x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    tol = 16 * H * size * abs(r.magnitude)
    if type_ == BF16:
        tol = tol + B * want.abs()
    assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(got[..., r.dim:].double(), x[..., r.dim:])


def turn(torch, x, y, type_, pos, pa, pt, r, axes):
    t, heads, hd = x.shape
    return runtime.lib().strasgpt_k_rope_axes(
        x.data_ptr(), x.stride(0), x.stride(1), y.data_ptr(), y.stride(0), y.stride(1), type_, t,
        heads, hd, pos.data_ptr(), pa, pt, r, axes, stream(torch))


KINDS = {
    "plain": dict(theta=500000.0),
    "linear": dict(theta=10000.0, scaling=runtime.ROPE_LINEAR, factor=4.0),
    "bands": dict(theta=500000.0, scaling=runtime.ROPE_BANDS, factor=8.0, magnitude=1.25),
}


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("order", [RUNS, DEALT])
@pytest.mark.parametrize("separate", [0, 1])
@pytest.mark.parametrize("t,heads,hd,sections", [
    (1, 40, 128, [24, 20, 20]), (7, 3, 80, [20, 20]), (33, 5, 96, [7, 1, 9, 6]),
    (257, 2, 128, [16, 24, 24]), (5, 1, 6, [0, 3]), (3, 2, 513, [100, 0, 156]),
    (2, 4, 2, [1]), (600, 12, 64, [0, 0, 0, 32])])
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_axes(cuda, type_, order, separate, t, heads, hd, sections, kind):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(t + heads * hd)
    x = torch.randn(t, heads, hd, device="cuda", generator=g).to(dtype(torch, type_))
    pos = torch.randint(-5, 1 << 21, (len(sections), t), device="cuda", generator=g,
                        dtype=torch.int32)
    for interleaved in (0, 1):
        y = torch.full_like(x, float("nan"))
        r = runtime.Rope(2 * sum(sections), interleaved=interleaved, **KINDS[kind])
        axes = runtime.RopeAxes(sections, order, separate)
        assert turn(torch, x, y, type_, pos, t, 1, r, axes) == 0
        check(torch, y, x, pos, r, sections, order, separate, type_)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_one_position_on_all_axes_is_rope_bit_for_bit(cuda, type_):
    """Text: every axis has the token's position (axis stride 0)."""
    torch = cuda
    t, heads, hd = 65, 6, 128
    x = torch.randn(t, heads, hd, device="cuda").to(dtype(torch, type_))
    pos = torch.randint(0, 1 << 30, (t,), device="cuda", dtype=torch.int32)
    r = runtime.Rope(hd, **KINDS["bands"])
    y, z = torch.empty_like(x), torch.empty_like(x)
    assert runtime.lib().strasgpt_k_rope(x.data_ptr(), heads * hd, hd, y.data_ptr(), heads * hd,
                                         hd, type_, t, heads, hd, pos.data_ptr(), r,
                                         stream(torch)) == 0
    for sections, order in (([24, 20, 20], DEALT), ([16, 24, 24], RUNS), ([64], RUNS)):
        z.fill_(float("nan"))
        assert turn(torch, x, z, type_, pos, 0, 1, r, runtime.RopeAxes(sections, order)) == 0
        assert torch.equal(y, z)
    # One axis of its own is the whole head.
    assert turn(torch, x, z, type_, pos, 0, 1, r, runtime.RopeAxes([64], RUNS, 1)) == 0
    assert torch.equal(y, z)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("odd", [0, 1])
def test_in_place_into_a_cache_with_positions_per_token(cuda, type_, odd):
    """q heads in place within wider rows, k heads into cache rows, positions
    stored token by token; everything around them as it was. odd: rows that
    start off 16 bytes."""
    torch = cuda
    t, qh, kh, hd, ctx, n = 21, 6, 2, 64, 100, 57
    dt = dtype(torch, type_)
    rows = torch.randn(t, (qh + 2 * kh) * hd + odd, device="cuda").to(dt)
    before = rows.clone()
    cache = torch.randn(kh, ctx, hd, device="cuda").to(dt)
    old = cache.clone()
    pos = torch.randint(0, 4000, (t, 3), device="cuda", dtype=torch.int32)
    sections = [12, 11, 9]
    r, axes = runtime.Rope(hd, theta=10000.0), runtime.RopeAxes(sections, DEALT)
    k = rows[:, qh * hd:(qh + kh) * hd].unflatten(1, (kh, hd))
    into = cache[:, n:n + t].transpose(0, 1)
    assert turn(torch, k, into, type_, pos, 1, 3, r, axes) == 0
    q = rows[:, :qh * hd].unflatten(1, (qh, hd))
    assert turn(torch, q, q, type_, pos, 1, 3, r, axes) == 0
    for got, a in ((into, slice(qh * hd, (qh + kh) * hd)), (q, slice(0, qh * hd))):
        check(torch, got, before[:, a].unflatten(1, (-1, hd)), pos.T, r, sections, DEALT, 0, type_)
    assert torch.equal(rows[:, qh * hd:], before[:, qh * hd:])
    assert torch.equal(cache[:, :n], old[:, :n]) and torch.equal(cache[:, n + t:], old[:, n + t:])


@pytest.mark.gpu
def test_captured_call_reads_positions_anew(cuda):
    torch = cuda
    t, heads, hd, sections = 9, 2, 128, [24, 20, 20]
    x, y = torch.randn(t, heads, hd, device="cuda"), torch.empty(t, heads, hd, device="cuda")
    pos = torch.randint(0, 5000, (3, t), device="cuda", dtype=torch.int32)
    r, axes = runtime.Rope(hd, theta=500000.0), runtime.RopeAxes(sections)
    turn(torch, x, y, F32, pos, t, 1, r, axes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turn(torch, x, y, F32, pos, t, 1, r, axes)
    for _ in range(2):
        pos.copy_(torch.randint(0, 5000, (3, t), device="cuda", dtype=torch.int32))
        y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        check(torch, y, x, pos, r, sections, RUNS, 0, F32)


@pytest.mark.parametrize("change,words", [
    (dict(axes=None), "null axes"), (dict(sections=[64], n=0), "1 to 4 axes"),
    (dict(sections=[64], n=5), "1 to 4 axes"), (dict(order=2), "unknown order"),
    (dict(sections=[65, -1]), "fewer than 0"), (dict(sections=[30, 30]), "add up"),
    (dict(sections=[32, 33]), "add up"), (dict(sections=[2 ** 31 - 1, 2 ** 31 - 1, 66]), "add up"),
    (dict(pa=-1), "stride of pos"), (dict(pt=-1), "stride of pos"),
    (dict(type_=2), "unknown type"), (dict(t=-1), "empty shape"), (dict(rope=None), "null param"),
    (dict(rope=dict(dim=7)), "turned part"), (dict(rope=dict(theta=0.0)), "theta"),
    (dict(rope=dict(theta=5e-324), separate=1), "beyond 64 bits"),
    (dict(x=None), "null buffer"), (dict(pos=None), "null buffer"), (dict(xt=-1), "negative"),
    (dict(yt=100), "overlap"), (dict(xt=512, x=2 * FAKE), "in place"),
    (dict(x=FAKE + 2), "aligned"), (dict(pos=FAKE + 2), "aligned"), (dict(), ""),
])
def test_refuses(capfd, change, words):
    a = dict(type_=F32, t=4, heads=3, hd=128, x=FAKE, xt=384, xh=128, y=2 * FAKE, yt=384, yh=128,
             pos=FAKE, pa=4, pt=1, rope={}, sections=[24, 20, 20], order=RUNS, separate=0)
    a.update(change)
    if a["rope"] is not None:
        a["rope"] = runtime.Rope(**{**dict(dim=128, theta=1e4), **a["rope"]})
    axes = None if "axes" in a else runtime.RopeAxes(a["sections"], a["order"], a["separate"])
    if "n" in a:
        axes.axes = a["n"]
    status = runtime.lib().strasgpt_k_rope_axes(
        a["x"], a["xt"], a["xh"], a["y"], a["yt"], a["yh"], a["type_"], a["t"], a["heads"],
        a["hd"], a["pos"], a["pa"], a["pt"], a["rope"], axes, None)
    err = capfd.readouterr().err
    assert status == -1 and "[StrasGPT] Error" in err and words in err, (status, err)


def test_no_tokens_are_no_error():
    r, axes = runtime.Rope(64, theta=1e4), runtime.RopeAxes([16, 16])
    assert runtime.lib().strasgpt_k_rope_axes(None, 0, 0, None, 64, 64, F32, 0, 1, 64, None, 0, 1,
                                              r, axes, None) == 0
    assert ctypes.sizeof(runtime.RopeAxes) == 28
    with pytest.raises(ValueError):
        runtime.RopeAxes([1] * 5)
