"""The three entry points of a step over drafted tokens
(include/strasgpt_kernels.h): strasgpt_k_rope, strasgpt_k_attn_tree and
strasgpt_k_sample, against float64 restatements of their definitions.

Tolerances, with h = 2^-24 (half a step of fp32) and b = 2^-8 (of bf16):

rope: the fp32 sine of an angle of at most half a turn: the angle's own
rounding gives pi h, sincospif at most 2 steps (4 h), the magnitude's and the
product's roundings 2 h; a turned entry is the sum of two products, 2 h more:
below 16 h (|a| + |b|) magnitude. bf16 adds b |y|.

attn_tree: a score errs by E = scale sum |q k| e, with e = 2^-19 of the tf32
parts (both operands cut at 2^-21, lo.lo below 2^-20 left out; 0 for bf16,
whose products are exact) plus the sum's roundings, 3 head_dim / 8 + 8 MMA
steps of 2 h. An error E of every score moves a softmax by a factor of at most
e^(2E), so an output by 2E max|v| (1 + E); the output's own products and sums
add (2^-19 + (n / 8 + 64) 2 h) max|v| (n / 8 MMA steps, the joins of the
splits), bf16 probabilities in two parts 2^-16 max|v|, the bf16 result b |o|.

sample: whole numbers are equal; a probability has one rounding, and its
weights are held to 2^-42: 4 h relative.
"""
import ctypes
import math

import numpy as np
import pytest

from strasgpt_b200 import runtime

F32, BF16 = runtime.F32, runtime.BF16
H, B = 2.0 ** -24, 2.0 ** -8


def dtype(torch, type_):
    return torch.float32 if type_ == F32 else torch.bfloat16


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


# --------------------------------------------------------------------------
# rope
# --------------------------------------------------------------------------
def frequencies(r):
    j = np.arange(0, r.dim, 2, dtype=np.float64)
    f = r.theta ** (-j / r.dim)
    if r.scaling == runtime.ROPE_LINEAR:
        f = f / r.factor
    if r.scaling == runtime.ROPE_BANDS:
        turns = r.original * f / (2 * math.pi)
        keep = np.clip((turns - r.low) / (r.high - r.low), 0, 1)
        f = f * (keep + (1 - keep) / r.factor)
    return f


def rope_reference(torch, x, pos, r):
    """x [t][heads][hd] -> float64 result and the entries' bound |a| + |b|."""
    x = x.double()
    f = torch.from_numpy(frequencies(r)).to(x.device)
    angle = pos.double()[:, None, None] * f
    c, s = torch.cos(angle) * r.magnitude, torch.sin(angle) * r.magnitude
    y, size = x.clone(), torch.zeros_like(x)
    half = r.dim // 2
    a, b = ((slice(0, r.dim, 2), slice(1, r.dim, 2)) if r.interleaved
            else (slice(0, half), slice(half, r.dim)))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def check_rope(torch, got, x, pos, r, type_):
    want, size = rope_reference(torch, x, pos, r)
    tol = 16 * H * size * abs(r.magnitude)
    if type_ == BF16:
        tol = tol + B * want.abs()
    assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(got[..., r.dim:], x[..., r.dim:])


ROPES = {
    "plain": dict(theta=500000.0),
    "linear": dict(theta=10000.0, scaling=runtime.ROPE_LINEAR, factor=4.0),
    "bands": dict(theta=500000.0, scaling=runtime.ROPE_BANDS, factor=8.0, low=1.0, high=4.0,
                  original=8192, magnitude=1.25),
}


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("t,heads,hd,dim", [
    (1, 1, 2, 2), (1, 40, 128, 128), (7, 3, 80, 80), (5, 8, 64, 32), (33, 5, 96, 46),
    (257, 2, 128, 64), (3, 2, 513, 512), (2, 4, 30, 16), (1000, 12, 128, 128)])
@pytest.mark.parametrize("kind", sorted(ROPES))
def test_rope(cuda, type_, interleaved, t, heads, hd, dim, kind):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(t + heads * hd + dim)
    x = torch.randn(t, heads, hd, device="cuda", generator=g).to(dtype(torch, type_))
    pos = torch.randint(0, 1 << 21, (t,), device="cuda", generator=g, dtype=torch.int32)
    y = torch.full_like(x, float("nan"))
    r = runtime.Rope(dim, interleaved=interleaved, **ROPES[kind])
    assert runtime.lib().strasgpt_k_rope(
        x.data_ptr(), x.stride(0), x.stride(1), y.data_ptr(), y.stride(0), y.stride(1), type_,
        t, heads, hd, pos.data_ptr(), r, stream(torch)) == 0
    check_rope(torch, y, x, pos, r, type_)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("odd", [0, 1])
def test_rope_in_place_into_a_cache_and_nothing_else(cuda, type_, odd):
    """q heads turned in place within wider rows; k heads into cache rows;
    everything around them as it was. odd: rows that start off 16 bytes."""
    torch = cuda
    t, qh, kh, hd, ctx, n = 21, 6, 2, 64, 100, 57
    dt = dtype(torch, type_)
    rows = torch.randn(t, (qh + 2 * kh) * hd + odd, device="cuda").to(dt)
    before = rows.clone()
    cache = torch.randn(kh, ctx, hd, device="cuda").to(dt)
    old = cache.clone()
    pos = torch.randint(-5, 4000, (t,), device="cuda", dtype=torch.int32)
    r = runtime.Rope(hd, theta=10000.0)
    L, ld = runtime.lib(), rows.stride(0)
    k = rows[:, qh * hd:]
    assert L.strasgpt_k_rope(k.data_ptr(), ld, hd, cache[:, n:].data_ptr(), hd, ctx * hd, type_,
                             t, kh, hd, pos.data_ptr(), r, stream(torch)) == 0
    assert L.strasgpt_k_rope(rows.data_ptr(), ld, hd, rows.data_ptr(), ld, hd, type_, t, qh, hd,
                             pos.data_ptr(), r, stream(torch)) == 0
    check_rope(torch, cache[:, n:n + t].transpose(0, 1),
               before[:, qh * hd:(qh + kh) * hd].view(t, kh, hd), pos, r, type_)
    check_rope(torch, rows[:, :qh * hd].view(t, qh, hd), before[:, :qh * hd].view(t, qh, hd),
               pos, r, type_)
    assert torch.equal(rows[:, qh * hd:], before[:, qh * hd:])
    assert torch.equal(cache[:, :n], old[:, :n]) and torch.equal(cache[:, n + t:], old[:, n + t:])


@pytest.mark.gpu
def test_rope_turns_back_and_broadcasts(cuda):
    """A negative position undoes a positive one; a stride of 0 on the input
    gives one head's entries to all."""
    torch = cuda
    t, heads, hd = 9, 4, 128
    x = torch.randn(t, 1, hd, device="cuda")
    y, z = torch.empty(t, heads, hd, device="cuda"), torch.empty(t, heads, hd, device="cuda")
    pos = torch.randint(0, 100000, (t,), device="cuda", dtype=torch.int32)
    r = runtime.Rope(hd, theta=500000.0)
    L = runtime.lib()
    assert L.strasgpt_k_rope(x.data_ptr(), hd, 0, y.data_ptr(), heads * hd, hd, F32, t, heads, hd,
                             pos.data_ptr(), r, stream(torch)) == 0
    check_rope(torch, y, x.expand(t, heads, hd), pos, r, F32)
    back = -pos
    assert L.strasgpt_k_rope(y.data_ptr(), heads * hd, hd, z.data_ptr(), heads * hd, hd, F32, t,
                             heads, hd, back.data_ptr(), r, stream(torch)) == 0
    # Two turns, each within 16 h of (|a| + |b|), the second of entries up to
    # |a| + |b| in size: 48 h (|a| + |b|).
    size = x.abs() + torch.roll(x.abs(), hd // 2, dims=-1)
    assert ((z - x).abs() <= 48 * H * size).all()


# --------------------------------------------------------------------------
# attn_tree
# --------------------------------------------------------------------------
def tree_mask(t, seed):
    """Ancestors (self included) of a random tree: bool [t][t]."""
    rng = np.random.RandomState(seed)
    m = np.zeros((t, t), dtype=bool)
    for i in range(t):
        parent = int(rng.randint(-1, i)) if i else -1
        if parent >= 0:
            m[i] = m[parent]
        m[i, i] = True
    return m


def mask_words(torch, m):
    t = m.shape[0]
    words = np.zeros((t, (t + 63) // 64), dtype=np.uint64)
    for i, j in zip(*np.nonzero(m)):
        words[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return torch.from_numpy(words.view(np.int64)).cuda()


def tree_reference(torch, q, k, v, n, m):
    """Float64 attention of q [t][kh * g][hd]; rows that see nothing: zeros.
    Also the bound sum |q k| / sqrt(hd) of each row and max |v|, over what the
    row sees."""
    t, qh, hd = q.shape
    kh = k.shape[0]
    g = qh // kh
    see = torch.cat([torch.ones(t, n, dtype=torch.bool), torch.from_numpy(m)], 1).cuda()
    out = torch.zeros(t, qh, hd, dtype=torch.float64, device="cuda")
    reach, top = 0.0, 0.0
    for h in range(qh):
        for i in range(t):
            kk, vv = k[h // g, :n + t][see[i]].double(), v[h // g, :n + t][see[i]].double()
            if not len(kk):
                continue
            s = kk @ q[i, h].double() / hd ** 0.5
            out[i, h] = torch.softmax(s, 0) @ vv
            reach = max(reach, ((kk.abs() @ q[i, h].double().abs()).max() / hd ** 0.5).item())
            top = max(top, vv.abs().max().item())
    return out, reach, top


def run_tree(torch, q, k, v, n, m, type_, att=None, workspace=None):
    L = runtime.lib()
    t, qh, hd = q.shape
    kh, ctx = k.shape[:2]
    cached = torch.tensor([n], dtype=torch.int32, device="cuda")
    words = mask_words(torch, m)
    size = L.strasgpt_k_attn_tree_workspace(t, kh, qh // kh, hd)
    if workspace is None:
        workspace = torch.full((size // 4 + 1,), float("nan"), device="cuda")
    if att is None:
        att = torch.full_like(q, float("nan"))
    assert L.strasgpt_k_attn_tree(q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), type_, t,
                                  kh, qh // kh, hd, ctx, cached.data_ptr(), words.data_ptr(),
                                  att.data_ptr(), att.stride(0), workspace.data_ptr(), size,
                                  stream(torch)) == 0
    torch.cuda.synchronize()
    return att


def tree_tolerance(want, reach, top, n, hd, type_):
    e = (2.0 ** -19 if type_ == F32 else 0.0) + (3 * hd / 8 + 8) * 2 * H
    E = reach * e
    tol = 2 * E * top * (1 + E) + (2.0 ** -19 + (n / 8 + 64) * 2 * H) * top
    if type_ == F32:
        return tol
    return tol + 2.0 ** -16 * top + B * want.abs()


def inputs(torch, t, kh, g, hd, ctx, type_, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = dtype(torch, type_)
    make = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(dt)  # noqa: E731
    return 2 * make(t, kh * g, hd), make(kh, ctx, hd), make(kh, ctx, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("t,kh,g,n", [
    (1, 1, 1, 0), (1, 2, 4, 1), (1, 2, 8, 333), (2, 1, 5, 31), (5, 2, 3, 32), (4, 1, 4, 33),
    (6, 2, 4, 63), (8, 1, 4, 64), (9, 1, 4, 65), (16, 1, 4, 127), (17, 2, 4, 128),
    (11, 1, 7, 129), (64, 1, 2, 700), (33, 1, 8, 255), (70, 1, 1, 40), (130, 1, 3, 0),
    (3, 1, 2, 5000), (40, 1, 4, 1500), (33, 8, 4, 2999), (256, 2, 1, 77), (257, 2, 1, 130)])
def test_tree_matches_float64(cuda, type_, hd, t, kh, g, n):
    torch = cuda
    q, k, v = inputs(torch, t, kh, g, hd, n + t + 13, type_, t * 131 + n)
    m = tree_mask(t, n + t)
    want, reach, top = tree_reference(torch, q, k, v, n, m)
    got = run_tree(torch, q, k, v, n, m, type_)
    err = (got.double() - want).abs()
    assert (err <= tree_tolerance(want, reach, top, n + t, hd, type_)).all(), err.max().item()
    # The same in the mean: independent errors of scores and products stay
    # near the parts' own 2^-21 (fp32); a rounding to bf16 is 2^-8 / sqrt(3)
    # at most in the root mean square.
    rel = (err.norm() / want.norm()).item()
    assert rel <= (2.0 ** -18 if type_ == F32 else B / 3 ** 0.5 + 2.0 ** -15), rel


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_tree_one_split_per_head_and_wide_rows(cuda, type_):
    """So many kv heads that the keys are not split (the result is written by
    the first kernel), and q and att as parts of wider rows."""
    torch = cuda
    t, kh, g, hd, n = 3, 320, 2, 32, 45
    q0, k, v = inputs(torch, t, kh, g, hd, 64, type_, 5)
    wide = torch.zeros(t, kh * g * hd + 64, device="cuda", dtype=q0.dtype)
    wide[:, 32:-32] = q0.view(t, -1)
    q = wide[:, 32:-32].view(t, kh * g, hd)
    out = torch.full((t, kh * g * hd + 48), 7.0, device="cuda").to(q0.dtype)
    att = out[:, 16:-32].view(t, kh * g, hd)
    m = tree_mask(t, 1)
    assert runtime.lib().strasgpt_k_attn_tree_workspace(t, kh, g, hd) == 0
    run_tree(torch, q, k, v, n, m, type_, att=att)
    want, reach, top = tree_reference(torch, q, k, v, n, m)
    err = (att.double() - want).abs()
    assert (err <= tree_tolerance(want, reach, top, n + t, hd, type_)).all()
    assert (out[:, :16] == 7).all() and (out[:, -32:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("t,g,n", [(6, 1, 0), (6, 1, 40), (20, 4, 0), (70, 4, 300), (80, 1, 0)])
def test_tree_hidden_rows_may_hold_anything(cuda, type_, t, g, n):
    """NaN and infinities in drafted rows that some tokens do not see, and
    behind the last row, reach none of the others; a token that sees nothing
    gets zeros, one that sees a NaN value gets NaN."""
    torch = cuda
    hd, kh = 64, 2
    q, k, v = inputs(torch, t, kh, g, hd, n + t + 20, type_, 3)
    m = tree_mask(t, 2)
    bad = [1, t // 2, t - 1]
    for b in bad:
        m[:, b] = False
    if n == 0:
        m[3] = False                       # sees nothing at all
    clean = [x.clone() for x in (k, v)]
    for i, b in enumerate(bad):
        k[:, n + b] = [float("nan"), float("inf"), -float("inf")][i]
        v[:, n + b] = [float("inf"), float("nan"), -float("inf")][i]
    k[:, n + t:] = float("nan")
    v[:, n + t:] = float("nan")
    got = run_tree(torch, q, k, v, n, m, type_)
    want, reach, top = tree_reference(torch, q, *clean, n, m)
    err = (got.double() - want).abs()
    assert (err <= tree_tolerance(want, reach, top, n + t, hd, type_)).all(), err.max().item()
    if n == 0:
        assert (got[3] == 0).all()
    # Now token 0 sees the row whose values are NaN; the others stay.
    m2 = m.copy()
    m2[0, t // 2] = True
    k[:, n + t // 2] = clean[0][:, n + t // 2]
    got2 = run_tree(torch, q, k, v, n, m2, type_)
    assert got2[0].isnan().all()
    assert torch.equal(got2[1:], got[1:]) or (
        (got2[1:].double() - want[1:]).abs()
        <= (tree_tolerance(want, reach, top, n + t, hd, type_) if type_ == F32
            else tree_tolerance(want, reach, top, n + t, hd, type_)[1:])).all()


@pytest.mark.gpu
def test_tree_length_is_read_on_the_device(cuda):
    """A captured call serves later lengths and a length outside the cache is
    cut to it; two graphs with a workspace each run side by side."""
    torch = cuda
    L = runtime.lib()
    t, kh, g, hd, ctx = 12, 2, 4, 64, 2048
    m = tree_mask(t, 4)
    words = mask_words(torch, m)
    size = L.strasgpt_k_attn_tree_workspace(t, kh, g, hd)
    assert size > 0
    sides = []
    for seed in (1, 2):
        q, k, v = inputs(torch, t, kh, g, hd, ctx, F32, seed)
        s = dict(q=q, k=k, v=v, att=torch.empty_like(q), stream=torch.cuda.Stream(),
                 work=torch.full((size // 4,), float("nan"), device="cuda"),
                 cached=torch.zeros(1, dtype=torch.int32, device="cuda"),
                 graph=torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(s["graph"], stream=s["stream"]):
            assert L.strasgpt_k_attn_tree(
                q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), F32, t, kh, g, hd, ctx,
                s["cached"].data_ptr(), words.data_ptr(), s["att"].data_ptr(),
                s["att"].stride(0), s["work"].data_ptr(), size,
                torch.cuda.current_stream().cuda_stream) == 0
        sides.append(s)
    for n in (0, 5, 900, ctx - t, ctx + 77, -3):
        for s in sides:
            s["cached"].fill_(n)
            s["att"].fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(3):
            for s in sides:
                with torch.cuda.stream(s["stream"]):
                    s["graph"].replay()
        torch.cuda.synchronize()
        cut = min(max(n, 0), ctx - t)
        for s in sides:
            want, reach, top = tree_reference(torch, s["q"], s["k"], s["v"], cut, m)
            err = (s["att"].double() - want).abs()
            assert (err <= tree_tolerance(want, reach, top, cut + t, hd, F32)).all()


@pytest.mark.gpu
def test_tree_offsets_beyond_32_bits(cuda):
    """A cache of more than 2^31 entries: heads far apart, and keys far into
    one head. Keys and values are zeros but for the last rows, so every other
    score is 0 and every other value adds nothing."""
    torch = cuda
    t, g, hd = 4, 4, 128
    for kh, ctx, n in ((5, 3_500_000, 90), (1, 17_000_016, 17_000_000)):
        k = torch.zeros(kh, ctx, hd, device="cuda", dtype=torch.bfloat16)
        v = torch.zeros_like(k)
        q, k2, v2 = inputs(torch, t, kh, g, hd, 64, BF16, 11)
        k[:, n + t - 64:n + t] = k2
        v[:, n + t - 64:n + t] = 1000 * v2
        m = tree_mask(t, 6)
        got = run_tree(torch, q, k, v, n, m, BF16).double()
        zeros = n + t - 64
        want = torch.zeros(t, kh * g, hd, dtype=torch.float64, device="cuda")
        for h in range(kh * g):
            for i in range(t):
                see = torch.cat([torch.ones(64 - t, dtype=torch.bool),
                                 torch.from_numpy(m[i])]).cuda()
                s = k2[h // g][see].double() @ q[i, h].double() / hd ** 0.5
                w = torch.exp(s)
                want[i, h] = w @ (1000 * v2)[h // g][see].double() / (w.sum() + zeros)
        # Relative to the largest output: a dropped or doubled row is off by
        # far more than the roundings (scores up to 2^5, b of the result).
        scale = want.abs().max()
        assert scale > 0
        assert ((got - want).abs() <= B * want.abs() + 2.0 ** -12 * scale).all()
        del k, v


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("t,kh,g", [(4, 1, 1), (3, 2, 1), (2, 3, 2), (1, 8, 3), (1, 1, 4),
                                    (4, 320, 1), (5, 2, 1)])
@pytest.mark.parametrize("n", [0, 7, 31, 33, 500, 4097])
def test_tree_few_rows(cuda, type_, t, kh, g, n):
    """Up to four rows per kv head (and five), some drafted rows hidden from
    all and not finite; the last token sees nothing where nothing is cached."""
    torch = cuda
    hd = 128
    if kh > 100:
        n = min(n, 500)
    q, k, v = inputs(torch, t, kh, g, hd, n + t + 9, type_, 7 * t + n)
    m = tree_mask(t, n)
    clean = k.clone(), v.clone()
    if t > 1:
        m[:, 0] = False
        m[-1] = False
        k[:, n], v[:, n] = float("nan"), float("inf")
    k[:, n + t:], v[:, n + t:] = float("inf"), float("nan")
    want, reach, top = tree_reference(torch, q, *clean, n, m)
    got = run_tree(torch, q, k, v, n, m, type_)
    err = (got.double() - want).abs()
    assert (err <= tree_tolerance(want, reach, top, n + t, hd, type_)).all(), err.max().item()
    if n == 0 and t > 1:
        assert (got[-1] == 0).all()
    if t > 1:
        m[1, 0] = True                     # now the second token sees it
        got = run_tree(torch, q, k, v, n, m, type_)
        assert got[1].isnan().all() and not got[2:].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128])
def test_tree_many_rows_one_split_and_wide_rows(cuda, type_, hd):
    """As above where the cached keys have a kernel of their own: one split per
    kv head, q and att as parts of wider rows."""
    torch = cuda
    t, kh, g, n = 40, 160, 1, 200
    q0, k, v = inputs(torch, t, kh, g, hd, 250, type_, 6)
    wide = torch.full((t, kh * g * hd + 64), float("nan"), device="cuda", dtype=q0.dtype)
    wide[:, 32:-32] = q0.view(t, -1)
    q = wide[:, 32:-32].view(t, kh * g, hd)
    out = torch.full((t, kh * g * hd + 48), 7.0, device="cuda").to(q0.dtype)
    att = out[:, 16:-32].view(t, kh * g, hd)
    m = tree_mask(t, 1)
    run_tree(torch, q, k, v, n, m, type_, att=att)
    want, reach, top = tree_reference(torch, q, k, v, n, m)
    err = (att.double() - want).abs()
    assert (err <= tree_tolerance(want, reach, top, n + t, hd, type_)).all()
    assert (out[:, :16] == 7).all() and (out[:, -32:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_tree_many_rows_with_offsets_beyond_32_bits(cuda, type_):
    """The same caches of more than 2^31 entries as above, for more rows per kv
    head."""
    torch = cuda
    t, g, hd = 5, 4, 128
    for kh, ctx, n in ((5, 3_500_000, 90), (1, 17_000_016, 17_000_000)):
        k = torch.zeros(kh, ctx, hd, device="cuda", dtype=dtype(torch, type_))
        v = torch.zeros_like(k)
        q, k2, v2 = inputs(torch, t, kh, g, hd, 64, type_, 11)
        k[:, n + t - 64:n + t] = k2
        v[:, n + t - 64:n + t] = 1000 * v2
        m = tree_mask(t, 6)
        got = run_tree(torch, q, k, v, n, m, type_).double()
        zeros = n + t - 64
        want = torch.zeros(t, kh * g, hd, dtype=torch.float64, device="cuda")
        for h in range(kh * g):
            for i in range(t):
                see = torch.cat([torch.ones(64 - t, dtype=torch.bool),
                                 torch.from_numpy(m[i])]).cuda()
                s = k2[h // g][see].double() @ q[i, h].double() / hd ** 0.5
                w = torch.exp(s)
                want[i, h] = w @ (1000 * v2)[h // g][see].double() / (w.sum() + zeros)
        scale = want.abs().max()
        assert scale > 0
        assert ((got - want).abs() <= B * want.abs() + 2.0 ** -12 * scale).all()
        del k, v


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("scale", [1e-12, 1e12])
@pytest.mark.parametrize("t", [3, 24])
def test_tree_large_and_small_numbers(cuda, type_, t, scale):
    """Keys and values far from 1, queries that bring the scores back: nothing
    overflows or vanishes on the way."""
    torch = cuda
    q, k, v = inputs(torch, t, 2, 4, 128, 700, type_, 9)
    q, k, v = q / scale, k * scale, v * scale ** 2
    m = tree_mask(t, 3)
    want, reach, top = tree_reference(torch, q, k, v, 600, m)
    got = run_tree(torch, q, k, v, 600, m, type_)
    err = (got.double() - want).abs()
    assert (err <= tree_tolerance(want, reach, top, 600 + t, 128, type_)).all(), err.max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("t,g,hd", [(9, 4, 128), (17, 1, 128), (33, 1, 64), (256, 1, 64),
                                    (2, 128, 128), (1, 128, 32)])
def test_tree_caches_that_end_with_the_tree(cuda, type_, t, g, hd):
    """No row behind the drafted ones, few or none before them: caches shorter
    than a tile of keys, and the length cut to what the cache holds."""
    torch = cuda
    for n in (0, 1, 62, 64):
        q, k, v = inputs(torch, t, 2, g, hd, n + t, type_, t + n)
        m = tree_mask(t, 4)
        want, reach, top = tree_reference(torch, q, k, v, n, m)
        got = run_tree(torch, q, k, v, n, m, type_)
        err = (got.double() - want).abs()
        assert (err <= tree_tolerance(want, reach, top, n + t, hd, type_)).all()
        cut = run_tree(torch, q, k, v, 2 ** 31 - 1, m, type_)
        assert torch.equal(cut, got)
        if n == 0:
            assert torch.equal(run_tree(torch, q, k, v, -5, m, type_), got)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("t,hd", [(24, 128), (20, 64), (3, 128)])
def test_tree_two_graphs_at_once(cuda, type_, t, hd):
    """Two captured calls with workspaces of their own, replayed on two streams
    at the same time, the lengths changed between replays."""
    torch = cuda
    L, kh, g, ctx = runtime.lib(), 2, 4, 4000
    sides = []
    for seed in (1, 2):
        q, k, v = inputs(torch, t, kh, g, hd, ctx, type_, seed)
        m = tree_mask(t, seed)
        size = L.strasgpt_k_attn_tree_workspace(t, kh, g, hd)
        x = dict(q=q, k=k, v=v, m=m, words=mask_words(torch, m), att=torch.zeros_like(q),
                 n=torch.zeros(1, dtype=torch.int32, device="cuda"),
                 work=torch.full((size // 4 + 1,), float("nan"), device="cuda"),
                 stream=torch.cuda.Stream(), graph=torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(x["graph"], stream=x["stream"]):
            assert L.strasgpt_k_attn_tree(
                q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), type_, t, kh, g, hd, ctx,
                x["n"].data_ptr(), x["words"].data_ptr(), x["att"].data_ptr(), q.stride(0),
                x["work"].data_ptr(), size, torch.cuda.current_stream().cuda_stream) == 0
        sides.append(x)
    for lengths in ((3900, 1), (0, 3333), (640, 641)):
        for x, n in zip(sides, lengths):
            x["n"].fill_(n)
        torch.cuda.synchronize()
        for _ in range(10):
            for x in sides:
                with torch.cuda.stream(x["stream"]):
                    x["graph"].replay()
        torch.cuda.synchronize()
        for x, n in zip(sides, lengths):
            assert torch.equal(x["att"], run_tree(torch, x["q"], x["k"], x["v"], n, x["m"], type_))


# --------------------------------------------------------------------------
# sample
# --------------------------------------------------------------------------
def sample_row(x, heat, top_k, top_p, min_p, u):
    """The definition, in float64, for one row of float64 logits."""
    x = np.where(np.isnan(x), -np.inf, x)
    real = np.nonzero(x > -np.inf)[0]
    if not len(real):
        return -1, 0.0, 0
    order = real[np.argsort(-x[real], kind="stable")]
    if not heat > 0:
        return int(order[0]), 1.0, 1
    top = x[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / heat))
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    if top_p < 1:
        before = np.cumsum(w) - w
        keep = before < top_p * w.sum()
        keep[0] = True
        order, w = order[keep], w[keep]
    if min_p > 0:
        keep = w >= min(min_p, 1.0)
        order, w = order[keep], w[keep]
    by = np.argsort(order)
    order, w = order[by], w[by]
    sums = np.cumsum(w)
    some = np.nonzero(w > 0)[0]
    at = np.searchsorted(sums, max(u, 0.0) * sums[-1], side="right") if u > 0 else some[0]
    at = min(at, some[-1])
    return int(order[at]), w[at] / sums[-1], len(order)


def run_sample(torch, x, heat=None, top_k=None, top_p=None, min_p=None, u=None, ld=None,
               prob=True):
    rows, vocab = x.shape
    row = lambda v, dt: None if v is None else torch.as_tensor(  # noqa: E731
        np.broadcast_to(np.asarray(v), (rows,)).copy(), dtype=dt).cuda()
    a = dict(heat=row(heat, torch.float32), k=row(top_k, torch.int32),
             p=row(top_p, torch.float32), m=row(min_p, torch.float32), u=row(u, torch.float32))
    token = torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda")
    out = torch.full((rows + 1,), -7.0, device="cuda")
    kept = torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda")
    ptr = lambda v: None if v is None else v.data_ptr()  # noqa: E731
    assert runtime.lib().strasgpt_k_sample(
        x.data_ptr(), F32 if x.dtype == torch.float32 else BF16, x.stride(0) if ld is None else ld,
        rows, vocab, ptr(a["heat"]), ptr(a["k"]), ptr(a["p"]), ptr(a["m"]), ptr(a["u"]),
        token.data_ptr(), out.data_ptr() if prob else None, kept.data_ptr() if prob else None,
        stream(torch)) == 0
    torch.cuda.synchronize()
    assert token[-1] == -7 and out[-1] == -7 and kept[-1] == -7
    return token[:-1].cpu().numpy(), out[:-1].cpu().numpy(), kept[:-1].cpu().numpy()


def check_sample(torch, x, heat=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.5, **kw):
    rows = x.shape[0]
    full = lambda v, dt: np.broadcast_to(np.asarray(v, dtype=dt), (rows,))  # noqa: E731
    heat, top_p, min_p, u = (full(v, np.float32) for v in (heat, top_p, min_p, u))
    top_k = full(top_k, np.int32)
    token, prob, kept = run_sample(torch, x, heat, top_k, top_p, min_p, u, **kw)
    xs = x.double().cpu().numpy()
    for r in range(rows):
        want = sample_row(xs[r], float(heat[r]), int(top_k[r]), float(top_p[r]),
                          float(min_p[r]), float(u[r]))
        assert (token[r], kept[r]) == (want[0], want[2]), (r, token[r], kept[r], want)
        assert abs(prob[r] - want[1]) <= 4 * H * want[1], (r, prob[r], want[1])
    return token, prob, kept


def logits(torch, rows, vocab, type_, seed, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = spread * torch.randn(rows, vocab, device="cuda", generator=g)
    return x.to(dtype(torch, type_))


FILTERS = [dict(), dict(top_k=1), dict(top_k=5), dict(top_k=40, top_p=0.9), dict(top_p=0.95),
           dict(top_p=0.3, min_p=0.1), dict(min_p=0.05), dict(top_k=1000, top_p=0.99, min_p=0.01),
           dict(top_p=0.9999), dict(top_k=7777)]


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(3, 1), (3, 2), (5, 7), (9, 33), (4, 511), (6, 1024),
                                        (6, 4097), (3, 16384), (4, 50001), (9, 128256),
                                        (2, 201088), (2, 360448)])
def test_sample_matches_float64(cuda, type_, rows, vocab):
    torch = cuda
    rng = np.random.RandomState(vocab)
    for i, f in enumerate(FILTERS):
        x = logits(torch, rows, vocab, type_, i)
        check_sample(torch, x, heat=rng.uniform(0.3, 1.6, rows).astype(np.float32),
                     u=rng.uniform(0, 1, rows).astype(np.float32), **f)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("vocab", [50, 3001, 40000, 128256])
def test_sample_equal_logits_rank_by_index(cuda, type_, vocab):
    """Whole-number logits: thousands of equal ones at every border, first in
    one bin of the histogram, then spread by a temperature."""
    torch = cuda
    rng = np.random.RandomState(7)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randint(-3, 4, (7, vocab), device="cuda", generator=g).to(dtype(torch, type_))
    x[1] = 2.5                                   # all equal
    x[2] = torch.where(torch.arange(vocab, device="cuda") % 3 == 0, 0.0, -0.0)
    x[3, vocab // 2:] = 4.0
    for f in FILTERS + [dict(top_k=vocab // 2), dict(top_k=vocab - 1, top_p=0.7)]:
        for heat in (0.2, 1.0, 50.0):
            check_sample(torch, x, heat=heat, u=rng.uniform(0, 1, 7).astype(np.float32), **f)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_sample_borders_within_one_bin(cuda, type_):
    """Nearly all logits within a hair of each other, one far above and one
    far below: the border's bin holds thousands of entries and is divided by
    key, more than once."""
    torch = cuda
    vocab = 100000
    g = torch.Generator(device="cuda").manual_seed(1)
    x = 1 + 2.0 ** -9 * torch.rand(4, vocab, device="cuda", generator=g)
    x[0, 5], x[0, 6] = 9.0, -20.0
    x[1, 7], x[1, 8] = 2.0, -3.0e38
    x[2, 9] = 25.0
    x = x.to(dtype(torch, type_))
    rng = np.random.RandomState(3)
    for f in [dict(top_k=50), dict(top_k=30000), dict(top_p=0.5), dict(top_k=60000, top_p=0.9),
              dict(top_p=0.999999), dict(top_k=99999)]:
        check_sample(torch, x, u=rng.uniform(0, 1, 4).astype(np.float32), **f)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_sample_masked_and_odd_values(cuda, type_):
    torch = cuda
    vocab, inf, nan = 9001, float("inf"), float("nan")
    x = logits(torch, 12, vocab, type_, 3)
    low = torch.finfo(x.dtype).min
    x[0] = -inf                                  # nothing left
    x[1] = nan
    x[2] = -inf
    x[2, 1234] = low                             # one entry, the lowest value
    x[3, ::2] = -inf
    x[4, 1::2] = low
    x[5, :] = low                                # all the lowest value
    x[6, 17] = inf
    x[6, 4000:4003] = inf                        # four equal infinities
    x[7, ::3] = nan
    x[8, :-1] = -inf                             # the last only
    x[9, 1:] = -inf                              # the first only
    x[10] *= 1e-38 if type_ == F32 else 1.0      # denormals
    rng = np.random.RandomState(5)
    for f in FILTERS:
        for heat in (1.0, 1e-3, 1e-30, 1e30):
            check_sample(torch, x, heat=heat, u=rng.uniform(0, 1, 12).astype(np.float32), **f)
    token, prob, kept = run_sample(torch, x, u=0.3, heat=float("inf"))
    assert token[0] == -1 and prob[0] == 0 and kept[0] == 0
    # An infinite temperature draws evenly from what is not masked.
    assert kept[3] == vocab // 2 and abs(prob[3] * (vocab // 2) - 1) < 1e-6


@pytest.mark.gpu
def test_sample_edges_of_the_parameters(cuda):
    torch = cuda
    vocab, nan = 5000, float("nan")
    x = logits(torch, 8, vocab, F32, 9)
    best = x.argmax(1).cpu().numpy()
    for kw in (dict(heat=0.0), dict(heat=-1.0), dict(heat=nan), dict(top_k=1), dict(top_p=0.0),
               dict(top_p=-1.0), dict(min_p=1.0), dict(min_p=7.0), dict(heat=1e-30)):
        token, prob, kept = run_sample(torch, x, u=0.999, **kw)
        assert (token == best).all() and (prob == 1).all() and (
            (kept == 1).all() or "heat" in kw), kw
    # No filter: parameters that say so, and none given.
    plain = run_sample(torch, x, u=0.6)
    for kw in (dict(top_k=0), dict(top_k=-3), dict(top_k=vocab), dict(top_k=2 ** 31 - 1),
               dict(top_p=1.0), dict(top_p=2.0), dict(top_p=nan), dict(min_p=0.0),
               dict(min_p=-1.0), dict(min_p=nan), dict(heat=1.0)):
        for a, b in zip(run_sample(torch, x, u=0.6, **kw), plain):
            assert (a == b).all(), kw
    assert (run_sample(torch, x, u=0.6, prob=False)[0] == plain[0]).all()
    # u at and beyond its ends: the first and the last entry.
    first = run_sample(torch, x, u=0.0, top_k=20)[0]
    last = run_sample(torch, x, u=1.0, top_k=20)[0]
    inside = torch.sort(torch.topk(x, 20, dim=1).indices, dim=1).values.cpu().numpy()
    assert (first == inside[:, 0]).all() and (last == inside[:, -1]).all()
    assert (run_sample(torch, x, u=nan, top_k=20)[0] == first).all()
    assert (run_sample(torch, x, u=-4.0, top_k=20)[0] == first).all()
    assert (run_sample(torch, x, u=3.0, top_k=20)[0] == last).all()
    for u in (2.0 ** -30, 1 - 2.0 ** -24):
        check_sample(torch, x, u=np.float32(u), top_k=20)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_sample_rows_of_a_wider_matrix(cuda, type_):
    """Rows apart, not 16-byte aligned, with other values between them."""
    torch = cuda
    for start, vocab, ld in ((1, 4099, 4111), (8, 4096, 4120), (3, 129, 1000)):
        big = torch.full((6 * ld + 8,), float("inf"), device="cuda", dtype=dtype(torch, type_))
        x = logits(torch, 6, vocab, type_, ld)
        view = big[start:start + 6 * ld].view(6, ld)[:, :vocab]
        view.copy_(x)
        check_sample(torch, view, top_k=30, top_p=0.9, u=0.77, ld=ld)


@pytest.mark.gpu
def test_sample_parameters_differ_by_row_and_replays_agree(cuda):
    """Every row with filters of its own, captured and replayed on another
    stream: the same bits every time."""
    torch = cuda
    L, rows, vocab = runtime.lib(), 40, 32003
    x = logits(torch, rows, vocab, F32, 21)
    rng = np.random.RandomState(2)
    heat = rng.choice([0.0, 0.4, 1.0, 1.3], rows).astype(np.float32)
    k = rng.choice([0, 1, 10, 400], rows).astype(np.int32)
    p = rng.choice([1.0, 0.95, 0.4], rows).astype(np.float32)
    m = rng.choice([0.0, 0.02], rows).astype(np.float32)
    u = rng.uniform(0, 1, rows).astype(np.float32)
    want = check_sample(torch, x, heat, k, p, m, u)
    dev = [torch.from_numpy(v).cuda() for v in (heat, k, p, m, u)]
    token = torch.zeros(rows, dtype=torch.int32, device="cuda")
    prob = torch.zeros(rows, device="cuda")
    kept = torch.zeros(rows, dtype=torch.int32, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        assert L.strasgpt_k_sample(x.data_ptr(), F32, vocab, rows, vocab,
                                   *[v.data_ptr() for v in dev], token.data_ptr(),
                                   prob.data_ptr(), kept.data_ptr(),
                                   torch.cuda.current_stream().cuda_stream) == 0
    for _ in range(5):
        for v in (token, prob, kept):
            v.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        for got, w in zip((token, prob, kept), want):
            assert (got.cpu().numpy() == w).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(300, 1), (301, 60), (330, 700), (299, 5003),
                                        (150, 40001), (40, 201088), (40, 700)])
def test_sample_many_rows_under_top_k(cuda, type_, rows, vocab):
    """More rows than the GPU holds clusters: a top-k row may be a block's own;
    here with rows among them that are not (no top-k, one above 512, one of the
    whole vocabulary)."""
    torch = cuda
    rng = np.random.RandomState(rows)
    ks = [0, 1, 2, 50, 300, 511, 512, 513, 2000, vocab - 1, vocab, -4]
    for i, f in enumerate([dict(), dict(top_p=0.9), dict(min_p=0.02),
                           dict(top_p=0.99, min_p=0.001)]):
        x = logits(torch, rows, vocab, type_, 40 + i)
        check_sample(torch, x, heat=rng.choice([0.0, 0.3, 1.0, 1.6], rows).astype(np.float32),
                     top_k=rng.choice(ks, rows).astype(np.int32),
                     u=rng.uniform(0, 1, rows).astype(np.float32), **f)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("vocab", [600, 9001])
def test_sample_many_rows_masked_and_odd_values(cuda, type_, vocab):
    torch = cuda
    inf, nan = float("inf"), float("nan")
    x = logits(torch, 36, vocab, type_, 6)
    low, high = torch.finfo(x.dtype).min, torch.finfo(x.dtype).max
    x[0] = -inf
    x[1] = nan
    x[2] = -inf
    x[2, 123] = low
    x[3, ::2] = -inf
    x[4, 1::2] = low
    x[5] = low
    x[6, 17] = inf
    x[6, 400:403] = inf
    x[7, ::3] = nan
    x[8, :-1] = -inf
    x[9, 1:] = -inf
    x[10] = 1.25                                 # all equal: more than a block holds
    x[11, 100:] = -inf                           # fewer entries than some k
    x[12] = -inf                                 # the widest range there is, and masked ones
    x[12, 5], x[12, 50:60], x[12, 70] = high, 1.0, low
    x[13] = 0.0
    x[13, ::2] = -0.0
    x[14, 1:] = x[14, 1:] * 2.0 ** -20 + 1       # all but one nearly equal
    x[15, 0] = high                              # far above the others
    x[16] = -inf
    x[16, 3] = inf                               # one infinity, nothing else
    x = x[:20].repeat(15, 1)                     # more rows than clusters at once
    rng = np.random.RandomState(8)
    for k in (1, 2, 40, 300, 512):
        for heat in (1.0, 1e-3, 1e30):
            for f in (dict(), dict(top_p=0.7), dict(min_p=0.3)):
                check_sample(torch, x, heat=heat, top_k=k,
                             u=rng.uniform(0, 1, 300).astype(np.float32), **f)
    token, prob, kept = run_sample(torch, x, u=0.3, heat=float("inf"), top_k=300)
    assert token[1] == -1 and kept[11] == 100 and abs(prob[11] - 0.01) < 1e-8
    assert kept[12] == 12 and abs(prob[12] * 12 - 1) < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_sample_many_rows_of_a_wider_matrix(cuda, type_):
    torch = cuda
    for start, vocab, ld in ((1, 4099, 4111), (8, 4096, 4120), (3, 129, 1000)):
        big = torch.full((300 * ld + 8,), float("inf"), device="cuda", dtype=dtype(torch, type_))
        x = logits(torch, 300, vocab, type_, ld)
        view = big[start:start + 300 * ld].view(300, ld)[:, :vocab]
        view.copy_(x)
        check_sample(torch, view, top_k=30, top_p=0.9, u=0.77, ld=ld)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(160, 2050), (40, 8200), (80, 16500), (160, 16500),
                                        (150, 39900), (150, 39945), (75, 80001)])
def test_sample_rows_that_fill_the_gpu(cuda, type_, rows, vocab):
    """Rows of one, two, four and eight CTAs, slices up to the longest that
    two CTAs on an SM leave room for."""
    torch = cuda
    rng = np.random.RandomState(rows + vocab)
    for i, f in enumerate([dict(top_p=0.95), dict(top_p=0.6, min_p=0.01), dict()]):
        x = logits(torch, rows, vocab, type_, i)
        check_sample(torch, x, heat=rng.uniform(0.3, 1.6, rows).astype(np.float32),
                     u=rng.uniform(0, 1, rows).astype(np.float32), **f)


@pytest.mark.gpu
def test_sample_calls_at_once(cuda):
    """Many rows with a block each on one stream, a few rows on another, at
    the same time: what each gives alone."""
    torch = cuda
    a, b = logits(torch, 150, 50000, BF16, 1), logits(torch, 9, 128256, F32, 2)
    ka = dict(top_k=50, top_p=0.9, u=0.35)
    kb = dict(top_p=0.9, u=0.8)
    one, two = check_sample(torch, a, **ka), check_sample(torch, b, **kb)
    L = runtime.lib()

    def prepare(x, k, p, u):
        n = x.shape[0]
        full = lambda v, dt: torch.full((n,), v, dtype=dt, device="cuda")  # noqa: E731
        out = (full(-7, torch.int32), full(0, torch.float32), full(-7, torch.int32))
        keep = (full(k, torch.int32), full(p, torch.float32), full(u, torch.float32))
        call = lambda s: L.strasgpt_k_sample(  # noqa: E731
            x.data_ptr(), F32 if x.dtype == torch.float32 else BF16, x.shape[1], n, x.shape[1],
            None, keep[0].data_ptr(), keep[1].data_ptr(), None, keep[2].data_ptr(),
            *[o.data_ptr() for o in out], s.cuda_stream)
        return call, out, keep

    ca, oa, _ka = prepare(a, 50, 0.9, 0.35)
    cb, ob, _kb = prepare(b, 0, 0.9, 0.8)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        assert ca(sa) == 0 and cb(sb) == 0
    torch.cuda.synchronize()
    for out, want in ((oa, one), (ob, two)):
        for got, w in zip(out, want):
            assert (got.cpu().numpy() == w).all()


# --------------------------------------------------------------------------
# together
# --------------------------------------------------------------------------
@pytest.mark.gpu
def test_a_step_over_drafted_tokens(cuda):
    """A layer's projections of a drafted tree: q turned in place, k turned
    into the cache, attention over both, a head's logits, a token for every
    drafted one; all on one stream, against the same in float64. Each row's u
    is the middle of its likeliest token's interval, so the choice survives
    fp32 logits."""
    torch = cuda
    L = runtime.lib()
    t, kh, g, hd, n, ctx, vocab = 19, 2, 4, 64, 333, 512, 2048
    qh, d = kh * g, kh * g * hd
    gen = torch.Generator(device="cuda").manual_seed(99)
    rows = torch.randn(t, (qh + 2 * kh) * hd, device="cuda", generator=gen)
    k, v = (torch.randn(kh, ctx, hd, device="cuda", generator=gen) for _ in range(2))
    w = (torch.randn(vocab, d, device="cuda", generator=gen) * 0.8).to(torch.bfloat16)
    m = tree_mask(t, 13)
    pos = torch.from_numpy(n + m.sum(1) - 1).to(torch.int32).cuda()
    r = runtime.Rope(hd, theta=500000.0)
    heat, top_k, top_p = 0.8, 50, 0.9

    x = rows.view(t, qh + 2 * kh, hd)
    q64 = rope_reference(torch, x[:, :qh], pos, r)[0]
    k64, v64 = k.double(), v.double()
    k64[:, n:n + t] = rope_reference(torch, x[:, qh:qh + kh], pos, r)[0].transpose(0, 1)
    v64[:, n:n + t] = x[:, qh + kh:].double().transpose(0, 1)
    att64 = tree_reference(torch, q64, k64, v64, n, m)[0]
    logits64 = (att64.view(t, d) @ w.double().T).cpu().numpy()
    u, want = [], []
    for i in range(t):
        likely = int(np.argmax(logits64[i]))
        # Bisect for the interval of u that draws it.
        lo = [0.0, 1.0]
        draw = lambda u: sample_row(logits64[i], heat, top_k, top_p, 0.0, u)[0]  # noqa: E731
        for _ in range(40):
            mid = sum(lo) / 2
            lo[draw(mid) >= likely] = mid
        hi = [lo[0], 1.0]
        for _ in range(40):
            mid = sum(hi) / 2
            hi[draw(mid) > likely] = mid
        u.append((lo[0] + hi[0]) / 2)
        want.append(sample_row(logits64[i], heat, top_k, top_p, 0.0, np.float32(u[-1])))
        assert want[-1][0] == likely

    full = lambda v, dt: torch.full((t,), v, dtype=dt, device="cuda")  # noqa: E731
    temps, ks, ps = full(heat, torch.float32), full(top_k, torch.int32), full(top_p, torch.float32)
    us = torch.tensor(u, dtype=torch.float32, device="cuda")
    cached = torch.tensor([n], dtype=torch.int32, device="cuda")
    words, att = mask_words(torch, m), torch.empty(t, qh, hd, device="cuda")
    size = L.strasgpt_k_attn_tree_workspace(t, kh, g, hd)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    out = torch.empty(t, vocab, device="cuda")
    token, prob = full(0, torch.int32), full(0.0, torch.float32)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        s, ld = stream(torch), rows.stride(0)
        assert L.strasgpt_k_rope(x[:, qh:].data_ptr(), ld, hd, k[:, n:].data_ptr(), hd, ctx * hd,
                                 F32, t, kh, hd, pos.data_ptr(), r, s) == 0
        v[:, n:n + t] = x[:, qh + kh:].transpose(0, 1)
        assert L.strasgpt_k_rope(x.data_ptr(), ld, hd, x.data_ptr(), ld, hd, F32, t, qh, hd,
                                 pos.data_ptr(), r, s) == 0
        assert L.strasgpt_k_attn_tree(x.data_ptr(), ld, k.data_ptr(), v.data_ptr(), F32, t, kh,
                                      g, hd, ctx, cached.data_ptr(), words.data_ptr(),
                                      att.data_ptr(), d, work.data_ptr(), size, s) == 0
        assert L.strasgpt_k_gemm_simt(att.data_ptr(), d, w.data_ptr(), d, t, vocab,
                                      out.data_ptr(), vocab, 0, s) == 0
        assert L.strasgpt_k_sample(out.data_ptr(), F32, vocab, t, vocab, temps.data_ptr(),
                                   ks.data_ptr(), ps.data_ptr(), None, us.data_ptr(),
                                   token.data_ptr(), prob.data_ptr(), None, s) == 0
    torch.cuda.synchronize()
    assert token.tolist() == [x[0] for x in want]
    # Logits up to 2^7 with relative errors of 2^-17 move a probability by
    # less than 2^-8 of itself at this temperature.
    for a, b in zip(prob.tolist(), want):
        assert abs(a - b[1]) <= 2.0 ** -8 * b[1]


# --------------------------------------------------------------------------
# refusals: host-side checks, no device work
# --------------------------------------------------------------------------
FAKE = 1 << 20  # aligned, never dereferenced


def refused(capfd, status, words):
    err = capfd.readouterr().err
    assert status == -1 and "[StrasGPT] Error" in err and words in err, (status, err)


@pytest.mark.parametrize("change,words", [
    (dict(type_=2), "unknown type"), (dict(t=-1), "empty shape"), (dict(heads=0), "empty shape"),
    (dict(hd=0), "empty shape"), (dict(rope=None), "null parameters"),
    (dict(rope=dict(dim=7)), "turned part"), (dict(rope=dict(dim=0)), "turned part"),
    (dict(rope=dict(dim=130)), "turned part"), (dict(rope=dict(theta=0.0)), "theta"),
    (dict(rope=dict(theta=float("nan"))), "theta"),
    (dict(rope=dict(magnitude=float("inf"))), "magnitude"),
    (dict(rope=dict(magnitude=1e300)), "magnitude"),
    (dict(rope=dict(scaling=3)), "unknown scaling"),
    (dict(rope=dict(scaling=1, factor=0.0)), "factor"),
    (dict(rope=dict(scaling=2, factor=2.0, low=4.0, high=4.0)), "bands"),
    (dict(rope=dict(scaling=2, factor=2.0, original=0)), "bands"),
    (dict(x=None), "null buffer"), (dict(y=None), "null buffer"), (dict(pos=None), "null buffer"),
    (dict(xt=-1), "negative stride"), (dict(yt=100), "overlap"), (dict(yh=100), "overlap"),
    (dict(yh=0), "overlap"), (dict(yt=300), "overlap"), (dict(xt=512, x=2 * FAKE), "in place"),
    (dict(x=FAKE + 2), "aligned"), (dict(pos=FAKE + 2), "aligned"), (dict(hd=70000), "too many"),
    (dict(), ""),
])
def test_rope_refuses(capfd, change, words):
    a = dict(type_=F32, t=4, heads=3, hd=128, x=FAKE, xt=384, xh=128, y=2 * FAKE, yt=384, yh=128,
             pos=FAKE, rope={})
    a.update(change)
    if a["rope"] is not None:
        a["rope"] = runtime.Rope(**{**dict(dim=128, theta=1e4), **a["rope"]})
    # A call that passes the checks of its arguments is refused for its
    # buffers, or for want of a GPU: these are no device memory.
    refused(capfd, runtime.lib().strasgpt_k_rope(
        a["x"], a["xt"], a["xh"], a["y"], a["yt"], a["yh"], a["type_"], a["t"], a["heads"],
        a["hd"], a["pos"], a["rope"], None), words)


@pytest.mark.parametrize("change,words", [
    (dict(type_=5), "unknown type"), (dict(t=-1), "empty shape"), (dict(kh=0), "empty shape"),
    (dict(g=0), "empty shape"), (dict(t=1025, ctx=4000), "more than 1024"),
    (dict(g=129, ld=1 << 20), "more than 128"), (dict(hd=96), "head_dim"), (dict(hd=256), "head_dim"),
    (dict(ctx=7), "fewer rows"), (dict(ldq=1023), "overlap"), (dict(ldo=512), "overlap"),
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"),
    (dict(cached=None), "null"), (dict(mask=None), "null"), (dict(att=None), "null"),
    (dict(q=FAKE + 4), "16-byte"), (dict(k=FAKE + 8), "16-byte"), (dict(ldq=1026), "16-byte"),
    (dict(att=FAKE + 8), "16-byte"), (dict(cached=FAKE + 2), "aligned"),
    (dict(mask=FAKE + 4), "aligned"),
    (dict(t=1024, kh=65535, g=128, ctx=4000, ld=1 << 30), "rows of q heads"), (dict(), ""),
])
def test_tree_refuses(capfd, change, words):
    a = dict(type_=F32, t=8, kh=2, g=4, hd=128, ctx=64, ldq=1024, ldo=1024, q=FAKE, k=FAKE, v=FAKE,
             cached=FAKE, mask=FAKE, att=FAKE)
    ld = change.pop("ld", None)
    a.update(change)
    if ld:
        a["ldq"] = a["ldo"] = ld
    refused(capfd, runtime.lib().strasgpt_k_attn_tree(
        a["q"], a["ldq"], a["k"], a["v"], a["type_"], a["t"], a["kh"], a["g"], a["hd"], a["ctx"],
        a["cached"], a["mask"], a["att"], a["ldo"], FAKE, 1 << 40, None), words)


def test_tree_workspace_refuses(capfd):
    f = runtime.lib().strasgpt_k_attn_tree_workspace
    for shape in ((-1, 1, 1, 64), (1, 0, 1, 64), (1, 1, 200, 64), (1, 1, 1, 65), (2000, 1, 1, 64),
                  (1024, 65535, 128, 32)):
        assert f(*shape) == 0
        assert "[StrasGPT] Error" in capfd.readouterr().err


@pytest.mark.parametrize("change,words", [
    (dict(type_=-1), "unknown type"), (dict(rows=-1), "empty shape"), (dict(vocab=0), "empty"),
    (dict(vocab=360449, ld=400000), "360448"), (dict(ld=999), "overlap"), (dict(x=None), "null"),
    (dict(u=None), "null"), (dict(token=None), "null"), (dict(x=FAKE + 1), "aligned"),
    (dict(u=FAKE + 2), "aligned"), (dict(prob=FAKE + 1), "aligned"),
    (dict(rows=1 << 25), "too many"), (dict(), ""),
])
def test_sample_refuses(capfd, change, words):
    a = dict(type_=BF16, rows=2, vocab=1000, ld=1000, x=FAKE, u=FAKE, token=FAKE, prob=FAKE)
    a.update(change)
    refused(capfd, runtime.lib().strasgpt_k_sample(
        a["x"], a["type_"], a["ld"], a["rows"], a["vocab"], None, None, None, None, a["u"],
        a["token"], a["prob"], None, None), words)


def test_nothing_to_do_is_no_error():
    L, r = runtime.lib(), runtime.Rope(64, theta=1e4)
    assert L.strasgpt_k_rope(None, 0, 0, None, 64, 64, F32, 0, 1, 64, None, r, None) == 0
    assert L.strasgpt_k_attn_tree(None, 0, None, None, F32, 0, 1, 1, 64, 8, None, None, None, 0,
                                  None, 0, None) == 0
    assert L.strasgpt_k_sample(None, F32, 8, 0, 8, None, None, None, None, None, None, None, None,
                               None) == 0


@pytest.mark.gpu
def test_buffers_that_are_not_this_device_s_are_refused(cuda, capfd):
    torch = cuda
    L, r = runtime.lib(), runtime.Rope(64, theta=1e4)
    x = torch.randn(2, 1, 64, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    host = torch.zeros(4096).pin_memory()
    call = lambda a, b, c: L.strasgpt_k_rope(a, 64, 64, b, 64, 64, F32, 2, 1, 64, c, r,  # noqa: E731
                                             None)
    for args in ((host.data_ptr(), x.data_ptr(), pos.data_ptr()),
                 (x.data_ptr(), host.data_ptr(), pos.data_ptr()),
                 (x.data_ptr(), x.data_ptr(), host.data_ptr())):
        refused(capfd, call(*args), "not device memory")
    if torch.cuda.device_count() > 1:
        far = torch.zeros(2, 1, 64, device="cuda:1")
        refused(capfd, call(far.data_ptr(), x.data_ptr(), pos.data_ptr()), "another device")
    size = L.strasgpt_k_attn_tree_workspace(1, 1, 1, 64)
    assert size > 0
    k, m = torch.zeros(1, 8, 64, device="cuda"), torch.ones(1, dtype=torch.int64, device="cuda")
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    w = torch.zeros(size // 4 + 4, device="cuda")
    tree = lambda p, b: L.strasgpt_k_attn_tree(  # noqa: E731
        x.data_ptr(), 64, k.data_ptr(), k.data_ptr(), F32, 1, 1, 1, 64, 8, n.data_ptr(),
        m.data_ptr(), x.data_ptr(), 64, p, b, None)
    refused(capfd, tree(w.data_ptr(), size - 1), "workspace")
    refused(capfd, tree(None, size), "workspace")
    refused(capfd, tree(w.data_ptr() + 4, size), "workspace must be")
    refused(capfd, tree(host.data_ptr(), size), "not device memory")
    assert ctypes.sizeof(runtime.Rope) == 56
