"""strasgpt_k_lora above 512 tokens, whose kernel is another one than the few tokens': the
forms of a call that test_lora.py makes with few. Tolerances are test_lora's.
"""
import pytest
import test_batch_step as batch
import test_lora as lora

F32, BF16 = lora.F32, lora.BF16
STORE, ADD, SWIGLU = lora.STORE, lora.ADD, lora.SWIGLU


def inputs(torch, m, k, n, r, d, type_, seed):
    """Mixed adapters at both ends; runs between them, whose borders lie inside tiles."""
    x, a, b, adapter, scale, base = lora.inputs(torch, m, k, n, r, d, type_, seed)
    at = 40
    for length, of in ((130, 0), (1, d - 1), (31, -1), (200, 1), (33, 0), (150, d - 1)):
        adapter[at:at + length] = of
        at += length
    return x, a, b, adapter, scale, base


def fits(got, want_err):
    want, err = want_err
    return ((got.double() - want).abs() <= err).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("epi", [STORE, ADD, SWIGLU])
@pytest.mark.parametrize("m,r,n", [(700, 16, 178), (700, 16, 182), (700, 72, 18), (1300, 72, 194),
                                   (2500, 64, 190), (700, 8, 192), (600, 8, 2)])
def test_entries_behind_the_rows_stay(cuda, type_, epi, m, r, n):
    """Rows of out on 16 bytes within wider ones and before other memory, which end
    anywhere within 16 bytes: all around them stays as it is, behind the last row too."""
    torch = cuda
    x, a, b, adapter, scale, base = inputs(torch, m, 264, n, r, 3, type_, m + n)
    outs = n // 2 if epi == SWIGLU else n
    ld = (outs + 7) // 8 * 8
    for wider in (ld, ld + 24):
        flat = torch.randn(m * wider + 64, device="cuda").to(x.dtype)
        before, part = flat.clone(), flat[:m * wider].view(m, wider)[:, :outs]
        want = lora.reference(torch, x, a, b, adapter, scale, base, part, epi, type_)
        assert lora.call(torch, x, a, b, adapter, scale, base, part, epi, type_) == 0
        assert fits(part, want)
        part.copy_(before[:m * wider].view(m, wider)[:, :outs])
        assert torch.equal(flat, before)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("m,r", [(700, 16), (1300, 72), (2500, 64)])
@pytest.mark.parametrize("epi", [STORE, ADD, SWIGLU])
@pytest.mark.parametrize("odd", [0, 1])
def test_no_base_no_scale(cuda, type_, m, r, epi, odd):
    """Without a base (ADD reads out alone) and without scales; odd: out's rows off 16
    bytes. Entries around the rows stay as they are."""
    torch = cuda
    x, a, b, adapter, _, _ = inputs(torch, m, 264, 90, r, 3, type_, m + epi)
    outs = 45 if epi == SWIGLU else 90
    wide = torch.randn(m, 112 + odd, device="cuda").to(x.dtype)
    before, part = wide.clone(), wide[:, 16 + odd:16 + odd + outs]
    want = lora.reference(torch, x, a, b, adapter, None, None, part, epi, type_)
    assert lora.call(torch, x, a, b, adapter, None, None, part, epi, type_) == 0
    assert fits(part, want)
    part.copy_(before[:, 16 + odd:16 + odd + outs])
    assert torch.equal(wide, before)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("m,r", [(700, 16), (1300, 72), (2500, 64)])
@pytest.mark.parametrize("odd", [0, 1])
def test_in_place(cuda, type_, m, r, odd):
    """base is out: runs' neighbours, which other clusters store to, are read in the same
    boxes. The same bits as apart, call after call."""
    torch = cuda
    x, a, b, adapter, scale, base = inputs(torch, m, 264, 90, r, 3, type_, m)
    wide = torch.randn(m, 128 + odd, device="cuda").to(x.dtype)
    part = wide[:, 16 + odd:16 + odd + 90]
    part.copy_(base)
    before = wide.clone()
    apart = torch.full((m, 112 + odd), 7.0, device="cuda").to(x.dtype)[:, odd:odd + 90]
    assert lora.call(torch, x, a, b, adapter, scale, part, apart, STORE, type_) == 0
    assert fits(apart, lora.reference(torch, x, a, b, adapter, scale, base, None, STORE, type_))
    for _ in range(5):
        part.copy_(base)
        assert lora.call(torch, x, a, b, adapter, scale, part, part, STORE, type_) == 0
        assert torch.equal(part, apart)
    part.copy_(base)
    assert torch.equal(wide, before)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_far_adapters_and_rows_behind_the_last(cuda, type_):
    """Adapters beyond 2^31 entries; rows from m on stay as they are."""
    torch = cuda
    m, k, n, r = 600, 8192, 64, 128
    d = (1 << 31) // (r * k) + 3
    x = torch.randn(m + 40, k, device="cuda").to(lora.dtype(torch, type_))
    a = torch.empty(d, r, k, device="cuda", dtype=torch.bfloat16)
    b = torch.full((d, n, r), float("nan"), device="cuda", dtype=torch.bfloat16)
    a[0] = a[1] = torch.nan
    for i in (d - 2, d - 1):
        a[i].normal_().div_(k ** 0.5)
        b[i].normal_().div_(r ** 0.5)
    adapter = torch.full((m + 40,), d - 1, dtype=torch.int32, device="cuda")
    adapter[100:333], adapter[400:450] = d - 2, d
    base = torch.randn(m + 40, n, device="cuda").to(x.dtype)
    out = torch.full_like(base, 7.0)
    assert lora.call(torch, x, a, b, adapter, None, base, out, STORE, type_, m=m) == 0
    want, err = lora.reference(torch, x, a[d - 2:], b[d - 2:], adapter - (d - 2), None, base, None,
                               STORE, type_)
    assert ((out.double() - want).abs() <= err)[:m].all()
    assert (out[m:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("epi", [STORE, ADD, SWIGLU])
def test_same_bits_on_two_streams_and_from_a_graph(cuda, type_, epi):
    """Two calls at once, and a captured one whose adapters are others at each replay."""
    torch = cuda
    x, a, b, adapter, scale, base = inputs(torch, 900, 520, 258, 24, 5, type_, 4)
    old = torch.randn(900, 129 if epi == SWIGLU else 258, device="cuda").to(x.dtype)

    def run(out):
        out.copy_(old)
        assert lora.call(torch, x, a, b, adapter, scale, base, out, epi, type_) == 0
        return out

    first = run(torch.empty_like(old))
    torch.cuda.synchronize()
    outs, streams = ([torch.empty_like(old) for _ in range(6)],
                     [torch.cuda.Stream() for _ in range(2)])
    for i, out in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            run(out)
    torch.cuda.synchronize()
    assert all(torch.equal(out, first) for out in outs)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(old)
    with torch.cuda.graph(graph):
        run(out)
    graph.replay()
    assert torch.equal(out, first)
    order = torch.arange(900, device="cuda")
    for now in (adapter.flip(0), order.int() % 7 - 1, torch.full_like(adapter, 2),
                (order // 300).int(), torch.full_like(adapter, -1)):
        adapter.copy_(now)
        graph.replay()
        assert fits(out, lora.reference(torch, x, a, b, adapter, scale, base, old, epi, type_))


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_a_batch_s_step_above_512_tokens(cuda, type_):
    """The operators one after the other, eager and captured, with prompts of up to 100
    tokens of six requests."""
    torch, most, requests, ctx = cuda, 100, 6, 160
    step = batch.Step(torch, type_, requests=requests, most=most, ctx=ctx)
    assert step.tokens > 512
    step.requests_are([1] * requests, [9] * requests, [0] * requests)
    step.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step.run()
    for i in range(3):
        new = [(most * (r + 1) // requests + 17 * i) % (most + 1) for r in range(requests)]
        rows = [min(ctx - 1, c + 13 * (r + i)) for r, c in enumerate(new)]
        step.requests_are(new, rows, [(r + i) % 6 - 1 for r in range(requests)])
        graph.replay()
        torch.cuda.synchronize()
        got, att, u = out.clone(), step.att.clone(), step.used
        again = step.run(step.check)
        assert torch.equal(step.att[:u], att[:u]) and torch.equal(again[:u], got[:u])
