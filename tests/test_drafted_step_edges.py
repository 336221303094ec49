"""Calls at the edges of what include/strasgpt_kernels.h allows of a step over
drafted tokens: threads, captured and replayed steps, values at the ends of
their ranges, buffers that are shared.
"""
import os
import subprocess
import sys

import numpy as np
import pytest
from strasgpt_b200 import runtime
from test_drafted_step import (BF16, F32, FAKE, H, check_rope, check_sample, dtype, inputs,
                               mask_words, run_sample, run_tree, sample_row, tree_mask,
                               tree_reference, tree_tolerance)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
def test_first_calls_from_two_threads(cuda):
    """In a process of its own: the first calls of two host threads, with
    vocabularies whose rows need 100 and 200 KB of shared memory, are served,
    and so are all later ones."""
    program = """
import threading, torch
from strasgpt_b200 import runtime
L = runtime.lib()
u = torch.full((1,), 0.5, device="cuda")
xs = [torch.randn(1, v, device="cuda") for v in (160000, 320000)]
out = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in xs]
torch.cuda.synchronize()
ready, status = threading.Barrier(2), []
def calls(i):
    ready.wait()
    for _ in range(200):
        status.append(L.strasgpt_k_sample(
            xs[i].data_ptr(), 0, xs[i].shape[1], 1, xs[i].shape[1], None, None, None, None,
            u.data_ptr(), out[i].data_ptr(), None, None, None))
threads = [threading.Thread(target=calls, args=(i,)) for i in (0, 1)]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
assert status == [0] * 400, status
"""
    for _ in range(2):
        subprocess.run([sys.executable, "-c", program], cwd=ROOT, check=True, timeout=300,
                       env=dict(os.environ, PYTHONPATH=ROOT))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("dim,theta,scaling", [(512, 1e4, "none"), (512, 2.0, "none"),
                                               (256, 5e5, "linear"), (512, 1e3, "bands"),
                                               (128, 1e4, "none")])
def test_rope_far_positions(cuda, interleaved, dim, theta, scaling):
    """Positions up to the largest int, against angles with 64-bit mantissas.
    The turns per position are off by 2^-54 of themselves (a running product)
    and rounded to 64 bits, as is their product with the position, 2^-53 each:
    1.25 2^-52 |pos| f radians on top of the bound for near positions."""
    torch = cuda
    ld = np.longdouble
    kind = dict(none=dict(), linear=dict(scaling=runtime.ROPE_LINEAR, factor=3.0),
                bands=dict(scaling=runtime.ROPE_BANDS, factor=8.0, original=8192))[scaling]
    r = runtime.Rope(dim, theta=theta, interleaved=interleaved, **kind)
    pos = np.array([2 ** 31 - 1, -2 ** 31, 2 ** 30 + 12345, 2 ** 29 - 7, 100000007, 2 ** 24 + 1, 1])
    f = ld(theta) ** (-ld(2) * np.arange(dim // 2, dtype=ld) / ld(dim))
    two_pi = 8 * np.arctan(ld(1))
    if scaling == "linear":
        f = f / ld(3)
    if scaling == "bands":
        keep = np.clip((8192 * f / two_pi - 1) / ld(3), 0, 1)
        f = f * (keep + (1 - keep) / ld(8))
    turns = pos.astype(ld)[:, None] * (f / two_pi)
    angle = ((turns - np.rint(turns)) * two_pi).astype(np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    gen = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn(len(pos), 3, dim, device="cuda", generator=gen)
    y = torch.full_like(x, float("nan"))
    where = torch.from_numpy(pos).to(torch.int32).cuda()
    assert runtime.lib().strasgpt_k_rope(
        x.data_ptr(), 3 * dim, dim, y.data_ptr(), 3 * dim, dim, F32, len(pos), 3, dim,
        where.data_ptr(), r, torch.cuda.current_stream().cuda_stream) == 0
    one, two = ((slice(0, dim, 2), slice(1, dim, 2)) if interleaved
                else (slice(0, dim // 2), slice(dim // 2, dim)))
    a, b = (x.double().cpu().numpy()[..., i] for i in (one, two))
    got = y.double().cpu().numpy()
    tol = (16 * H + 1.25 * 2.0 ** -52 * np.abs(pos)[:, None] * f.astype(np.float64))[:, None]
    tol = tol * (np.abs(a) + np.abs(b))
    assert (np.abs(got[..., one] - (a * c - b * s)) <= tol).all()
    assert (np.abs(got[..., two] - (a * s + b * c)) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("theta,dim", [(1e4, 128), (5e5, 64), (1e4, 6)])
def test_rope_sines_keep_their_bits(cuda, theta, dim):
    """Pairs (1, 0) become (cosine, sine). Near whole and half turns the sine
    is small, near quarters the cosine, and each is right relative to itself:
    sincospif to 2 steps (4 h), the correction's sum and the products (by 1, 0
    and the magnitude 1) to half a step each (2 h), the correction itself to
    2^-23 steps; and to the 64-bit angle's own error, 1.25 2^-52 |pos| f."""
    torch = cuda
    t = 4096
    rng = np.random.RandomState(dim)
    pos = np.concatenate([np.arange(t // 2), rng.randint(-2 ** 21, 2 ** 21, t - t // 2)])
    ld = np.longdouble
    two_pi = 8 * np.arctan(ld(1))
    f = ld(theta) ** (-ld(2) * np.arange(dim // 2, dtype=ld) / ld(dim))
    turns = pos.astype(ld)[:, None] * (f / two_pi)
    angle = (turns - np.rint(turns)) * two_pi
    x = torch.zeros(t, 1, dim, device="cuda")
    x[..., :dim // 2] = 1.0
    y = torch.full_like(x, float("nan"))
    where = torch.from_numpy(pos).to(torch.int32).cuda()
    assert runtime.lib().strasgpt_k_rope(
        x.data_ptr(), dim, dim, y.data_ptr(), dim, dim, F32, t, 1, dim, where.data_ptr(),
        runtime.Rope(dim, theta=theta), torch.cuda.current_stream().cuda_stream) == 0
    got = y[:, 0].double().cpu().numpy()
    for part, want in ((got[:, :dim // 2], np.cos(angle)), (got[:, dim // 2:], np.sin(angle))):
        err = np.abs(part - want)
        tol = ((6 + 2.0 ** -20) * H * np.abs(want) + 2.0 ** -46 * H
               + 1.25 * 2.0 ** -52 * np.abs(pos)[:, None] * f)
        assert (err <= tol).all(), float((err - tol).max())


def check_tiny(torch, x, period, u, heat=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """check_sample where probabilities may be below what fp32 holds: half a
    step of fp32 is 2^-150 there, whatever the value. Rows of x repeat after
    `period`."""
    f32 = lambda v: float(np.float32(v))  # noqa: E731
    token, prob, kept = run_sample(torch, x, u=u, heat=heat, top_k=top_k, top_p=top_p, min_p=min_p)
    wants = [sample_row(row, f32(heat), top_k, f32(top_p), f32(min_p), f32(u))
             for row in x[:period].double().cpu().numpy()]
    for r in range(x.shape[0]):
        want = wants[r % period]
        assert (token[r], kept[r]) == (want[0], want[2]), (r, token[r], kept[r], want)
        assert abs(prob[r] - want[1]) <= 4 * H * want[1] + 2.0 ** -150


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("vocab", [70, 3001, 40000])
@pytest.mark.parametrize("rows", [7, 300])
def test_sample_distances_beyond_fp32(cuda, type_, vocab, rows):
    """Logits whose distance from the largest overflows fp32, at temperatures
    that give them a weight all the same: the largest and the lowest value of
    the type; masks of the lowest value under ordinary logits. With few rows
    (clusters) and with many (under top-k, a block each)."""
    torch = cuda
    inf = float("inf")
    x = torch.full((7, vocab), -inf, device="cuda", dtype=dtype(torch, type_))
    low, high = torch.finfo(x.dtype).min, torch.finfo(x.dtype).max
    x[0, 5], x[0, 50:60], x[0, 69] = high, 1.0, low
    x[1, 0:3] = torch.tensor([low, 1.0, high])
    x[2] = low
    x[2, 11:40] = torch.arange(29, device="cuda") / 4
    x[3] = 2e38
    x[3, ::2] = -2e38
    x[4, ::3] = high
    x[4, 1::3] = low
    x[5] = torch.linspace(low / 2, high / 2, vocab, device="cuda")   # the difference just fits
    x[6] = torch.linspace(float(low) * 0.9, float(high) * 0.9, vocab, device="cuda",
                          dtype=torch.float64).to(x.dtype)
    x = x.repeat((rows + 6) // 7, 1)[:rows]
    rng = np.random.RandomState(vocab)
    for heat in (inf, 1e38, 3e38, 2e37, 1e36, 1.0):
        for f in (dict(), dict(top_k=2), dict(top_k=40, top_p=0.97), dict(top_p=0.7),
                  dict(min_p=0.01), dict(top_k=300, min_p=0.3)):
            check_sample(torch, x, heat=heat, u=rng.uniform(0.01, 0.99, rows).astype(np.float32),
                         **f)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("rows", [6, 312])
@pytest.mark.parametrize("vocab", [600, 9001, 128256])
def test_sample_ends_of_u_take_the_smallest_weights(cuda, type_, rows, vocab):
    """u of 0 takes the first entry that remains and u of 1 the last, however
    little they weigh beside the largest one (2^-100 to 2^-900), under each
    filter, with few rows and many."""
    torch = cuda
    if rows > 6 and vocab > 9001:
        rows = 60                                # more than the GPU holds clusters
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    x = -300 + 60 * torch.randn(6, vocab, device="cuda", generator=gen).clamp(-4, 4)
    x[0] = -600.0                                # thousands of equal tiny weights
    x[1, : vocab // 2] = -72.5                   # 2^-104.6
    x[2] = -float("inf")
    x[2, ::7] = -100.0
    x[3, vocab - 1], x[3, 0] = -620.0, -620.0
    x[4, 1:40] = torch.arange(39, device="cuda") / -2
    x[:, vocab // 2] = 0.0
    x[:, vocab // 2 + 3] = -0.25
    x = x.to(dtype(torch, type_)).repeat((rows + 5) // 6, 1)[:rows]
    for f in (dict(), dict(top_k=30), dict(top_k=vocab // 2), dict(top_k=513), dict(min_p=1e-35),
              dict(top_k=vocab - 1), dict(top_p=0.9), dict(top_k=520, top_p=0.9999999)):
        for u in (0.0, -1.0, 1e-38, 1e-28, 1e-20, 0.4, 1 - 2.0 ** -24, 1.0, 2.0):
            check_tiny(torch, x, 6, u, **f)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("rows", [5, 320])
def test_sample_smallest_weights(cuda, type_, rows):
    """Weights down to the smallest number that 64 bits hold (2^-1074, at 744.4
    below the largest logit) can be drawn: u of 0 takes the first entry that
    has one."""
    torch = cuda
    vocab = 5000
    x = torch.full((5, vocab), -900.0, device="cuda", dtype=dtype(torch, type_))
    x[:, 4321] = 0.0
    x[0, 77], x[0, 4400] = -700.0, -1.0          # 2^-1010
    x[1, 40:60] = -740.0                         # 2^-1068
    x[2, 1000] = -744.0                          # 2^-1074 times 1.4
    x[2, 999] = -748.0                           # rounds to 0
    x[3, ::5] = -720.0
    x[4, 4990] = -743.0                          # behind the largest
    x = x.repeat((rows + 4) // 5, 1)[:rows]
    for f in (dict(), dict(top_k=30), dict(top_k=2000), dict(min_p=1e-40), dict(top_p=0.9)):
        for u in (0.0, 1e-30, 0.5, 1.0):
            check_tiny(torch, x, 5, u, **f)


@pytest.mark.parametrize("one,other,apart,shared", [
    ("token", "k", 0, True), ("token", "u", 4, True), ("prob", "u", 0, True),
    ("kept", "token", -4, True), ("prob", "heat", 8, True), ("kept", "p", -8, True),
    ("token", "m", 12, False), ("prob", "kept", -12, False), ("heat", "u", 0, False)])
def test_sample_refuses_shared_outputs(capfd, one, other, apart, shared):
    """The outputs of three rows, a few bytes before or behind another array.
    (Inputs may be one array; what passes is refused as no device memory.)"""
    names = ("heat", "k", "p", "m", "u", "token", "prob", "kept")
    at = {n: (2 + i) * FAKE for i, n in enumerate(names)}
    at[one] = at[other] + apart
    status = runtime.lib().strasgpt_k_sample(FAKE, F32, 100, 3, 100, *[at[n] for n in names], None)
    err = capfd.readouterr().err
    assert status == -1 and ("share memory" in err) == shared, err


@pytest.mark.parametrize("kind,far", [
    (dict(dim=512, theta=5e-324), True),
    (dict(dim=64, theta=1e-300, scaling=1, factor=1e-100), True),
    (dict(dim=64, theta=1e4, scaling=1, factor=5e-324), True),
    (dict(dim=64, theta=1e4, scaling=2, factor=1e-300, original=10), True),
    (dict(dim=512, theta=1e-290), False), (dict(dim=512, theta=1.7e308), False),
    (dict(dim=2, theta=5e-324), False), (dict(dim=64, theta=1e4, scaling=1, factor=1e300), False)])
def test_rope_refuses_frequencies_beyond_64_bits(capfd, kind, far):
    """Parameters whose angles would not be finite numbers at every position.
    (What passes is refused as no device memory.)"""
    status = runtime.lib().strasgpt_k_rope(FAKE, 512, 512, 2 * FAKE, 512, 512, F32, 4, 1, 512,
                                           FAKE, runtime.Rope(**kind), None)
    err = capfd.readouterr().err
    assert status == -1 and ("beyond 64 bits" in err) == far, err


# (t, kv heads, q heads on each, head_dim, cached) -> every kernel of the
# attention, with and without splits of the keys.
SHAPES = [(1, 2, 4, 128, 700), (4, 320, 1, 128, 100), (3, 2, 5, 128, 700), (6, 2, 4, 64, 1000),
          (20, 320, 1, 64, 90), (9, 2, 8, 32, 500), (3, 320, 2, 32, 45), (70, 2, 1, 32, 300),
          (24, 2, 4, 128, 900), (40, 160, 1, 64, 200), (260, 1, 1, 128, 400)]


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("t,kh,g,hd,n", SHAPES)
def test_tree_in_place(cuda, type_, t, kh, g, hd, n):
    """The outputs over the queries: what another buffer gets."""
    torch = cuda
    q, k, v = inputs(torch, t, kh, g, hd, n + t + 3, type_, t)
    m = tree_mask(t, n)
    want = run_tree(torch, q, k, v, n, m, type_)
    same = q.clone()
    assert torch.equal(run_tree(torch, same, k, v, n, m, type_, att=same), want)


@pytest.mark.parametrize("ldo,words", [(1024, "device"), (1536, "in place")])
def test_tree_refuses_other_strides_in_place(capfd, ldo, words):
    status = runtime.lib().strasgpt_k_attn_tree(
        FAKE, 1024, 2 * FAKE, 3 * FAKE, F32, 8, 2, 4, 128, 64, FAKE, FAKE, FAKE, ldo, FAKE,
        1 << 40, None)
    err = capfd.readouterr().err
    assert status == -1 and words in err.lower(), err


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("t,kh,g,hd,n", SHAPES)
def test_tree_infinite_cached_rows_stay_in_their_head(cuda, type_, t, kh, g, hd, n):
    """Infinities and NaN in rows that all tokens see: nothing is said of the q
    heads on that kv head, all others have the same bits."""
    torch = cuda
    kh = max(kh, 2)
    q, k, v = inputs(torch, t, kh, g, hd, n + t + 3, type_, t)
    m = tree_mask(t, n)
    want = run_tree(torch, q, k, v, n, m, type_).view(t, kh, g, hd)
    k[1, 5], k[1, n - 1, 3] = float("inf"), -float("inf")
    v[1, 17], v[1, n // 2, 0] = float("nan"), float("inf")
    got = run_tree(torch, q, k, v, n, m, type_).view(t, kh, g, hd)
    others = [h for h in range(kh) if h != 1]
    assert torch.equal(got[:, others], want[:, others])


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("t,kh,g,hd,n", SHAPES)
def test_tree_repeats_itself(cuda, type_, t, kh, g, hd, n):
    """The same call, the same bits."""
    torch = cuda
    q, k, v = inputs(torch, t, kh, g, hd, n + t + 3, type_, t)
    m = tree_mask(t, n)
    want = run_tree(torch, q, k, v, n, m, type_)
    for _ in range(3):
        assert torch.equal(run_tree(torch, q, k, v, n, m, type_), want)


# --------------------------------------------------------------------------
# captured steps
# --------------------------------------------------------------------------
class Step:
    """A step over drafted tokens on buffers of its own: q turned in place, k
    and v rows into the caches, attention, a head's logits, a token each."""
    T, KH, G, HD, CTX, VOCAB = 19, 2, 4, 64, 512, 2048

    def __init__(self, torch):
        self.torch, self.L = torch, runtime.lib()
        t, kh, hd, ctx, qh = self.T, self.KH, self.HD, self.CTX, self.KH * self.G
        self.gen = torch.Generator(device="cuda").manual_seed(5)
        self.rows = torch.zeros(t, qh + 2 * kh, hd, device="cuda")
        self.turned = torch.zeros(t, kh, hd, device="cuda")
        self.k, self.v = (torch.randn(kh, ctx, hd, device="cuda", generator=self.gen)
                          for _ in range(2))
        self.w = torch.randn(self.VOCAB, qh * hd, device="cuda",
                             generator=self.gen).to(torch.bfloat16)
        self.cached = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.pos = torch.zeros(t, dtype=torch.int32, device="cuda")
        self.mask = tree_mask(t, 13)
        self.words = mask_words(torch, self.mask)
        self.att = torch.zeros(t, qh, hd, device="cuda")
        self.logits = torch.zeros(t, self.VOCAB, device="cuda")
        self.u = torch.zeros(t, device="cuda")
        self.token = torch.zeros(t, dtype=torch.int32, device="cuda")
        self.size = self.L.strasgpt_k_attn_tree_workspace(t, kh, self.G, hd)
        self.work = torch.zeros(self.size, dtype=torch.uint8, device="cuda")
        self.rope = runtime.Rope(hd, theta=500000.0)
        self.side = torch.cuda.Stream()

    def turn(self, n):
        """q in place, k into the cache rows from n on (None: a buffer)."""
        s, qh, t = self.torch.cuda.current_stream().cuda_stream, self.KH * self.G, self.T
        ld, hd = self.rows.stride(0), self.HD
        to, yt, yh = ((self.turned, self.turned.stride(0), hd) if n is None
                      else (self.k[:, n:], hd, self.CTX * hd))
        assert self.L.strasgpt_k_rope(self.rows[:, qh:].data_ptr(), ld, hd, to.data_ptr(), yt, yh,
                                      F32, t, self.KH, hd, self.pos.data_ptr(), self.rope, s) == 0
        assert self.L.strasgpt_k_rope(self.rows.data_ptr(), ld, hd, self.rows.data_ptr(), ld, hd,
                                      F32, t, qh, hd, self.pos.data_ptr(), self.rope, s) == 0

    def values(self, n):
        self.v[:, n:n + self.T].copy_(self.rows[:, -self.KH:].transpose(0, 1))

    def answer(self):
        s, d = self.torch.cuda.current_stream().cuda_stream, self.att.stride(0)
        assert self.L.strasgpt_k_attn_tree(
            self.rows.data_ptr(), self.rows.stride(0), self.k.data_ptr(), self.v.data_ptr(), F32,
            self.T, self.KH, self.G, self.HD, self.CTX, self.cached.data_ptr(),
            self.words.data_ptr(), self.att.data_ptr(), d, self.work.data_ptr(), self.size, s) == 0
        assert self.L.strasgpt_k_gemm_simt(self.att.data_ptr(), d, self.w.data_ptr(), d, self.T,
                                           self.VOCAB, self.logits.data_ptr(), self.VOCAB, 0,
                                           s) == 0
        assert self.L.strasgpt_k_sample(self.logits.data_ptr(), F32, self.VOCAB, self.T,
                                        self.VOCAB, None, None, None, None, self.u.data_ptr(),
                                        self.token.data_ptr(), None, None, s) == 0

    def capture(self, *parts):
        graph = self.torch.cuda.CUDAGraph()
        self.torch.cuda.synchronize()
        with self.torch.cuda.graph(graph, stream=self.side):
            for part in parts:
                part()
        return graph

    def new_inputs(self, n):
        """On the side stream, for a step at length n; a copy for check()."""
        self.rows.normal_(generator=self.gen)
        self.u.uniform_(generator=self.gen)
        self.cached.fill_(n)
        self.pos.copy_(self.torch.from_numpy(n + self.mask.sum(1) - 1))
        self.token.fill_(-7)
        self.att.fill_(float("nan"))
        self.before = [x.clone() for x in (self.rows, self.k, self.v)]

    def check(self, n):
        self.torch.cuda.synchronize()
        torch, t, qh, kh = self.torch, self.T, self.KH * self.G, self.KH
        rows, k, v = self.before
        check_rope(torch, self.rows[:, :qh], rows[:, :qh], self.pos, self.rope, F32)
        check_rope(torch, self.k[:, n:n + t].transpose(0, 1), rows[:, qh:qh + kh], self.pos,
                   self.rope, F32)
        v[:, n:n + t] = rows[:, qh + kh:].transpose(0, 1)
        k[:, n:n + t] = self.k[:, n:n + t]
        assert torch.equal(self.k, k) and torch.equal(self.v, v)   # and nothing else
        want, reach, top = tree_reference(torch, self.rows[:, :qh], k, v, n, self.mask)
        err = (self.att.double() - want).abs()
        assert (err <= tree_tolerance(want, reach, top, n + t, self.HD, F32)).all()
        for i, row in enumerate(self.logits.double().cpu().numpy()):
            assert self.token[i] == sample_row(row, 1.0, 0, 1.0, 0.0, float(self.u[i]))[0]


@pytest.mark.gpu
def test_a_captured_step_is_replayed(cuda):
    """The whole step in one graph, replayed for other inputs of the same
    length; captured again for another length, whose rows it then writes."""
    torch = cuda
    step = Step(torch)
    for n in (333, 40):
        graph = step.capture(lambda: step.turn(n), lambda: step.values(n), step.answer)
        for _ in range(3):
            with torch.cuda.stream(step.side):
                step.new_inputs(n)
                graph.replay()
            step.check(n)


@pytest.mark.gpu
def test_captured_parts_serve_every_length(cuda):
    """Rotation into a buffer is one graph, attention to token another; between
    their replays the keys and values go to the rows behind the cached ones by
    copies that are not captured. The length moves on, back and to the end."""
    torch = cuda
    step = Step(torch)
    turn, answer = step.capture(lambda: step.turn(None)), step.capture(step.answer)
    for n in (333, 338, 0, 7, step.CTX - step.T):
        with torch.cuda.stream(step.side):
            step.new_inputs(n)
            turn.replay()
            step.k[:, n:n + step.T].copy_(step.turned.transpose(0, 1))
            step.values(n)
            answer.replay()
        step.check(n)
