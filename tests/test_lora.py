"""strasgpt_k_lora (include/strasgpt_kernels.h): low-rank adapters of a batch's
tokens beside a shared projection, against float64.

Tolerance, with h = 2^-24 (half a step of fp32) and b = 2^-8 (of bf16). A matrix
instruction cuts its sums: 2 h of the sum of the products' sizes each. For a
token, |A||x| (of a rank) and |B||s| stand for those sums.

A x. fp32 rows: products are exact (three parts of 8 bits). Up to 512 tokens, 32
entries take six instructions from zero, 12 h; a warp's steps, at most k / 1024 + 1,
are added with roundings of h. More tokens: two instructions per 32 entries in one sum
of the large parts over at most k / 16 + 64 entries, 4 h (k / 512 + 2), and the small
parts' (2^-7 of them, twice as many): 5 h (k / 512 + 2) in all. Then up to 8 warps' and
8 CTAs' sums, and the scale, 17 h: below (12 + 5 (k / 512 + 2) + 17) h. bf16 rows:
products as they are, four instructions per 64 entries in one sum, 4 h (k / 512 + 2)
as well: the same bound.
B s. s as three parts (fp32; exact) or two (2^-17): rank / 16 steps, three
instructions each: 6 (rank / 16 + 1) h, and 2^-16 for two parts.
Then big and small sums, base and ADD's old value are added: 3 h of their sizes.
SwiGLU: silu has a slope of at most 1.1, so y = silu(g) u errs by
1.1 |u| dg + |silu(g)| du, and its own exp, divide and products by 8 h |y|.
bf16 results add b |y|.
"""
import pytest

from strasgpt_b200 import runtime

F32, BF16 = runtime.F32, runtime.BF16
STORE, ADD, SWIGLU = 0, 1, 2
H, B = 2.0 ** -24, 2.0 ** -8
FAKE = 1 << 20  # aligned, never dereferenced


def dtype(torch, type_):
    return torch.float32 if type_ == F32 else torch.bfloat16


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


def reference(torch, x, a, b, adapter, scale, base, out, epi, type_):
    """Float64 result and the bound on its error."""
    m, k = x.shape
    d, n, r = b.shape
    v = torch.zeros(m, n, dtype=torch.float64, device="cuda") if base is None else base.double()
    size, err = v.abs(), torch.zeros_like(v)
    first = (12 + 5 * (k / 512 + 2) + 17) * H
    second = 6 * (r / 16 + 1) * H + (2.0 ** -16 if type_ == BF16 else 0)
    for i in range(d):
        of = torch.nonzero(adapter == i)[:, 0]
        if not len(of):
            continue
        c = 1.0 if scale is None else scale[i].double()
        w, z = a[i].double(), b[i].double()
        low, reach = c * (x[of].double() @ w.T), abs(c) * (x[of].double().abs() @ w.abs().T)
        v[of] += low @ z.T
        err[of] = (first * reach + second * (low.abs() + first * reach)) @ z.abs().T
        size[of] += low.abs() @ z.abs().T
    err += 3 * H * size
    if epi == SWIGLU:
        g, u, dg, du = v[:, 0::2], v[:, 1::2], err[:, 0::2], err[:, 1::2]
        s = g * torch.sigmoid(g)
        v = s * u
        err = 1.1 * u.abs() * dg + (s.abs() + 1.1 * dg) * du + 8 * H * v.abs()
    elif epi == ADD:
        v = v + out.double()
        err += 3 * H * (out.double().abs() + v.abs())
    if type_ == BF16:
        err = err + B * (v.abs() + err)
    return v, err


def call(torch, x, a, b, adapter, scale, base, out, epi, type_, m=None):
    return runtime.lib().strasgpt_k_lora(
        x.data_ptr(), x.stride(0), a.data_ptr(), b.data_ptr(), type_,
        x.shape[0] if m is None else m, x.shape[1], b.shape[1], a.shape[1], a.shape[0],
        adapter.data_ptr(), None if scale is None else scale.data_ptr(),
        None if base is None else base.data_ptr(), 0 if base is None else base.stride(0),
        out.data_ptr(), out.stride(0), epi, stream(torch))


def inputs(torch, m, k, n, r, d, type_, seed, none=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    dt = dtype(torch, type_)
    adapter = torch.randint(0, d, (m,), device="cuda", generator=g, dtype=torch.int32)
    adapter[torch.rand(m, device="cuda", generator=g) < none] = -1
    return (rand(m, k).to(dt), (rand(d, r, k) / k ** 0.5).bfloat16(),
            (rand(d, n, r) / r ** 0.5).bfloat16(), adapter, 0.5 + rand(d).abs(),
            rand(m, n).to(dt))


SHAPES = [(1, 8, 1, 8, 1), (1, 2048, 2048, 8, 4), (2, 40, 33, 16, 2), (3, 264, 31, 24, 1),
          (15, 1000, 70, 40, 3), (16, 512, 256, 64, 16), (17, 4096, 300, 32, 5),
          (64, 1024, 514, 16, 64), (75, 320, 129, 128, 7), (149, 96, 200, 104, 4),
          (300, 640, 96, 64, 3), (600, 72, 1026, 48, 9), (1200, 136, 66, 88, 4),
          (2500, 256, 130, 16, 6), (1, 16384, 40, 128, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("epi", [STORE, ADD, SWIGLU])
@pytest.mark.parametrize("m,k,n,r,d", SHAPES)
def test_matches_float64(cuda, type_, epi, m, k, n, r, d):
    torch = cuda
    n += n % 2 if epi == SWIGLU else 0
    x, a, b, adapter, scale, base = inputs(torch, m, k, n, r, d, type_, m + k + n)
    out = torch.randn(m, n // 2 if epi == SWIGLU else n, device="cuda").to(x.dtype)
    want, err = reference(torch, x, a, b, adapter, scale, base, out, epi, type_)
    assert call(torch, x, a, b, adapter, scale, base, out, epi, type_) == 0
    assert ((out.double() - want).abs() <= err).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_runs_of_tokens_have_one_adapter(cuda, type_):
    """Prompts: runs whose borders lie inside tiles, and one without an adapter."""
    torch = cuda
    x, a, b, adapter, scale, base = inputs(torch, 700, 512, 384, 32, 4, type_, 3)
    at = 0
    for length, d in ((1, 3), (130, 0), (5, 9), (300, 2), (200, -1), (64, 1)):
        adapter[at:at + length] = d      # 9: none, as any number outside
        at += length
    out = torch.empty_like(base)
    want, err = reference(torch, x, a, b, adapter, scale, base, None, STORE, type_)
    assert call(torch, x, a, b, adapter, scale, base, out, STORE, type_) == 0
    assert ((out.double() - want).abs() <= err).all()
    assert torch.equal(out[136 + 300:136 + 500], base[136 + 300:136 + 500])
    assert torch.equal(out[131:136], base[131:136])


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("m,d,n", [(256, 1, 96), (256, 256, 40), (512, 300, 40), (513, 600, 40), (300, 1, 96), (65, 2, 8200),
                                   (64, 70, 40), (256, 1, 8200)])
def test_one_adapter_for_all_and_one_for_each(cuda, type_, m, d, n):
    torch = cuda
    x, a, b, adapter, scale, base = inputs(torch, m, 104, n, 8, d, type_, m + d, none=0)
    if d >= m:
        adapter = torch.randperm(d, device="cuda")[:m].int()
    out = torch.full_like(base, float("nan"))
    want, err = reference(torch, x, a, b, adapter, scale, base, None, STORE, type_)
    assert call(torch, x, a, b, adapter, scale, base, out, STORE, type_) == 0
    assert ((out.double() - want).abs() <= err).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("odd", [0, 1])
def test_strides_no_base_no_scale_in_place(cuda, type_, odd):
    """Rows within wider ones, whose other entries stay as they are; odd: base
    and out rows off 16 bytes."""
    torch = cuda
    m, k, n, r, d = 37, 256, 90, 16, 3
    x, a, b, adapter, _, base = inputs(torch, m, k, n, r, d, type_, 5)
    wide_x = torch.full((m, k + 64), float("nan"), device="cuda").to(x.dtype)
    wide_x[:, 32:32 + k] = x
    wide = torch.randn(m, n + 38 + odd, device="cuda").to(x.dtype)
    wide[:, 16 + odd:16 + odd + n] = base
    before, part = wide.clone(), wide[:, 16 + odd:16 + odd + n]
    want, err = reference(torch, x, a, b, adapter, None, base, None, STORE, type_)
    assert call(torch, wide_x[:, 32:32 + k], a, b, adapter, None, part, part, STORE, type_) == 0
    assert ((part.double() - want).abs() <= err).all()
    part.copy_(base)
    assert torch.equal(wide, before)
    for epi in (STORE, ADD, SWIGLU):
        out = torch.randn(m, n // 2 if epi == SWIGLU else n, device="cuda").to(x.dtype)
        want, err = reference(torch, x, a, b, adapter, None, None, out, epi, type_)
        assert call(torch, x, a, b, adapter, None, None, out, epi, type_) == 0
        assert ((out.double() - want).abs() <= err).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("m,k,n,r", [(257, 72, 65, 8), (600, 72, 65, 8), (1000, 200, 190, 72), (9000, 64, 34, 8)])
@pytest.mark.parametrize("epi", [STORE, ADD, SWIGLU])
def test_many_tokens_within_wider_rows(cuda, type_, m, k, n, r, epi):
    """Many tokens, whose rows of base and out are off 16 bytes and lie in wider ones;
    runs of adapters, and more tokens than one look at the adapters takes."""
    torch = cuda
    n += n % 2 if epi == SWIGLU else 0
    x, a, b, adapter, scale, base = inputs(torch, m, k, n, r, 5, type_, m)
    adapter[m // 4:m // 2] = 3
    adapter[m // 2:m // 2 + 130] = -1
    wide_x = torch.full((m, k + 48), float("nan"), device="cuda").to(x.dtype)
    wide_x[:, 16:16 + k] = x
    wide_b = torch.full((m, n + 11), float("nan"), device="cuda").to(x.dtype)
    wide_b[:, 5:5 + n] = base
    outs = n // 2 if epi == SWIGLU else n
    wide = torch.randn(m, outs + 9, device="cuda").to(x.dtype)
    before = wide.clone()
    want, err = reference(torch, x, a, b, adapter, scale, base, wide[:, 3:3 + outs], epi, type_)
    assert call(torch, wide_x[:, 16:16 + k], a, b, adapter, scale, wide_b[:, 5:5 + n],
                wide[:, 3:3 + outs], epi, type_) == 0
    assert ((wide[:, 3:3 + outs].double() - want).abs() <= err).all()
    assert torch.equal(wide[:, :3], before[:, :3])
    assert torch.equal(wide[:, 3 + outs:], before[:, 3 + outs:])


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("m", [5, 200, 900])
def test_other_tokens_rows_and_adapters_stay_out(cuda, type_, m):
    """Infinities and NaN in one token's row, in an adapter that others do not
    have and in rows without one reach nobody else; x rows of tokens without an
    adapter are not even read."""
    torch = cuda
    x, a, b, adapter, scale, base = inputs(torch, m, 320, 130, 24, 3, type_, 8)
    adapter[:5] = torch.tensor([0, 1, -1, 2, 0])
    want, err = reference(torch, x, a, b, adapter, scale, base, None, STORE, type_)
    bad = (adapter == 1) | (torch.arange(m, device="cuda") == 0)
    x[0, 7], a[1, 3, 5], b[1, 4], scale[1] = float("inf"), float("nan"), float("inf"), float("inf")
    x[adapter < 0] = float("nan")
    out = torch.full_like(base, float("nan"))
    assert call(torch, x, a, b, adapter, scale, base, out, STORE, type_) == 0
    assert ((out.double() - want).abs() <= err)[~bad].all()
    assert not torch.isfinite(out[0]).any()


@pytest.mark.gpu
def test_rows_behind_the_last_and_far_adapters(cuda):
    """Rows from m on stay as they are; adapters beyond 2^31 entries."""
    torch = cuda
    m, k, n, r = 20, 8192, 64, 128
    d = (1 << 31) // (r * k) + 3
    x = torch.randn(m + 9, k, device="cuda")
    a = torch.empty(d, r, k, device="cuda", dtype=torch.bfloat16)
    b = (torch.randn(d, n, r, device="cuda") / r ** 0.5).bfloat16()
    a[0] = a[d - 1] = torch.nan
    a[d - 1].normal_().div_(k ** 0.5)
    adapter = torch.full((m + 9,), d - 1, dtype=torch.int32, device="cuda")
    base = torch.randn(m + 9, n, device="cuda")
    out = torch.full_like(base, 7.0)
    assert call(torch, x, a, b, adapter, None, base, out, STORE, F32, m=m) == 0
    few = lambda w: w[d - 1:]  # noqa: E731
    want, err = reference(torch, x, few(a), few(b), adapter - (d - 1), None, base, None, STORE, F32)
    assert ((out.double() - want).abs() <= err)[:m].all()
    assert (out[m:] == 7.0).all()


@pytest.mark.gpu
def test_same_bits_again_on_two_streams_and_from_a_graph(cuda):
    torch = cuda
    x, a, b, adapter, scale, base = inputs(torch, 90, 2048, 512, 16, 30, F32, 4)
    first = torch.empty_like(base)
    assert call(torch, x, a, b, adapter, scale, base, first, STORE, F32) == 0
    torch.cuda.synchronize()
    outs, streams = [torch.empty_like(base) for _ in range(4)], [torch.cuda.Stream() for _ in
                                                                 range(2)]
    for i, out in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            assert call(torch, x, a, b, adapter, scale, base, out, STORE, F32) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(out, first) for out in outs)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(base)
    with torch.cuda.graph(graph):
        call(torch, x, a, b, adapter, scale, base, out, STORE, F32)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    adapter.copy_(adapter.flip(0))         # read anew at each replay
    graph.replay()
    want, err = reference(torch, x, a, b, adapter, scale, base, None, STORE, F32)
    assert ((out.double() - want).abs() <= err).all()


@pytest.mark.parametrize("change,words", [
    (dict(type_=2), "unknown type"), (dict(m=-1), "empty shape"), (dict(k=0), "empty shape"),
    (dict(n=0), "empty shape"), (dict(adapters=0), "empty shape"), (dict(rank=0), "rank"),
    (dict(rank=12), "rank"), (dict(rank=136), "rank"), (dict(k=68), "k must"),
    (dict(epi=3), "epilogue"), (dict(epi=SWIGLU, n=33), "odd"), (dict(ldx=56), "overlap"),
    (dict(ldb=31), "overlap"), (dict(ldo=31), "overlap"), (dict(epi=SWIGLU, ldo=15), "overlap"),
    (dict(x=None), "null"), (dict(a=None), "null"), (dict(b=None), "null"),
    (dict(adapter=None), "null"), (dict(out=None), "null"), (dict(x=FAKE + 8), "16-byte"),
    (dict(a=FAKE + 8), "16-byte"), (dict(b=FAKE + 2), "16-byte"), (dict(ldx=66), "16-byte"),
    (dict(base=FAKE + 2), "aligned"), (dict(out=2 * FAKE + 2), "aligned"),
    (dict(scale=FAKE + 2), "aligned"), (dict(adapter=FAKE + 1), "aligned"),
    (dict(out=FAKE), "x cannot"), (dict(base=2 * FAKE, ldb=36), "base can"),
    (dict(base=2 * FAKE, epi=ADD), "base can"), (dict(base=2 * FAKE, epi=SWIGLU), "base can"),
    (dict(), ""),
])
def test_refuses(capfd, change, words):
    p = dict(type_=F32, m=4, k=64, n=32, rank=8, adapters=2, x=FAKE, ldx=64, a=FAKE, b=FAKE,
             adapter=FAKE, scale=None, base=3 * FAKE, ldb=32, out=2 * FAKE, ldo=32, epi=STORE)
    p.update(change)
    status = runtime.lib().strasgpt_k_lora(
        p["x"], p["ldx"], p["a"], p["b"], p["type_"], p["m"], p["k"], p["n"], p["rank"],
        p["adapters"], p["adapter"], p["scale"], p["base"], p["ldb"], p["out"], p["ldo"], p["epi"],
        None)
    err = capfd.readouterr().err
    assert status == -1 and "[StrasGPT] Error" in err and words in err, (status, err)


def test_no_tokens_are_no_error():
    assert runtime.lib().strasgpt_k_lora(None, 64, None, None, F32, 0, 64, 32, 8, 1, None, None,
                                         None, 0, None, 32, STORE, None) == 0
