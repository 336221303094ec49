"""strasgpt_k_attn_shared (include/strasgpt_kernels.h): attention of a batch of
requests behind one prefix, against float64.

Tolerance as strasgpt_k_attn_tree's, whose kernels and parts it shares, with
h = 2^-24 (half a step of fp32) and b = 2^-8 (of bf16). A score errs by
E = scale sum |q k| e, with e = 2^-19 of the tf32 parts (both operands cut at
2^-21, lo.lo below 2^-20 left out; 0 for bf16, whose products are exact) plus
the sum's roundings, 3 head_dim / 8 + 8 MMA steps of 2 h. An error E of every
score moves a softmax by a factor of at most e^(2E), so an output by
2E max|v| (1 + E); the output's own products and sums add
(2^-19 + (n / 8 + 64) 2 h) max|v| (n / 8 MMA steps, the joins of the parts),
bf16 probabilities in two parts 2^-16 max|v|, the bf16 result b |o|.
"""
import math

import numpy as np
import pytest

from strasgpt_b200 import runtime

F32, BF16 = runtime.F32, runtime.BF16
H, B = 2.0 ** -24, 2.0 ** -8
FAKE = 1 << 20  # aligned, never dereferenced


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


class Batch:
    """new: tokens of each request; rows: of its cache, those included."""

    def __init__(self, torch, kh, g, hd, prefix, new, rows, type_, seed, ctx=None, pad=(0, 0),
                 most=None):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        dt = torch.float32 if type_ == F32 else torch.bfloat16
        make = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(dt)  # noqa: E731
        self.torch, self.type_, self.kh, self.g, self.hd = torch, type_, kh, g, hd
        self.new, self.rows, self.n = list(new), list(rows), prefix
        self.most = most or max(1, *new)
        self.tokens = sum(new) + sum(pad)
        ctx = ctx or max(1, *rows) + 5
        self.q = 2 * make(self.tokens, kh * g, hd)
        self.kp, self.vp = make(kh, prefix + 11, hd), make(kh, prefix + 11, hd)
        self.k, self.v = make(len(new), kh, ctx, hd), make(len(new), kh, ctx, hd)
        self.first = np.concatenate([[0], np.cumsum(new)]) + pad[0]
        i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
        self.d_first, self.d_rows, self.d_prefix = i32(self.first), i32(rows), i32([prefix])
        self.att = torch.full_like(self.q, float("nan"))
        size = self.size()
        self.work = torch.full((size // 4 + 1,), float("nan"), device="cuda")

    def size(self):
        return runtime.lib().strasgpt_k_attn_shared_workspace(
            self.type_, len(self.new), self.most, self.tokens, self.kh, self.g, self.hd)

    def run(self, att=None, first=True, work=None):
        att = self.att if att is None else att
        work = self.work if work is None else work
        assert runtime.lib().strasgpt_k_attn_shared(
            self.q.data_ptr(), self.q.stride(0), self.kp.data_ptr(), self.vp.data_ptr(),
            self.kp.shape[1], self.d_prefix.data_ptr(), self.k.data_ptr(), self.v.data_ptr(),
            self.k.stride(0), self.k.shape[2], self.d_rows.data_ptr(),
            self.d_first.data_ptr() if first else None, self.type_, len(self.new), self.most,
            self.tokens, self.kh, self.g, self.hd, att.data_ptr(), att.stride(0), work.data_ptr(),
            self.size(), stream(self.torch)) == 0
        return att

    def check(self, got=None):
        """Every row of every request within the tolerance."""
        torch, hd = self.torch, self.hd
        got = self.att if got is None else got
        for r, c in enumerate(self.new):
            n, a = self.rows[r], int(self.first[r])
            for j in range(c):
                own = max(0, min(n, n - c + j + 1))
                k = torch.cat([self.kp[:, :self.n], self.k[r, :, :own]], 1).double()
                v = torch.cat([self.vp[:, :self.n], self.v[r, :, :own]], 1).double()
                q = self.q[a + j].double().view(self.kh, self.g, hd)
                if not k.shape[1]:
                    assert (got[a + j] == 0).all()
                    continue
                s = q @ k.transpose(1, 2) / math.sqrt(hd)
                want = (torch.softmax(s, -1) @ v).view(-1, hd)
                reach = (q.abs() @ k.abs().transpose(1, 2)).max().item() / math.sqrt(hd)
                top = v.abs().max().item()
                e = (2.0 ** -19 if self.type_ == F32 else 0.0) + (3 * hd / 8 + 8) * 2 * H
                E = reach * e
                tol = (2 * E * top * (1 + E)
                       + (2.0 ** -19 + (k.shape[1] / 8 + 64) * 2 * H) * top)
                if self.type_ == BF16:
                    tol = tol + 2.0 ** -16 * top + B * want.abs()
                assert ((got[a + j].double() - want).abs() <= tol).all(), (r, j)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("kh,g,prefix,new,rows", [
    (1, 1, 1, [1], [1]), (2, 2, 613, [1, 1], [40, 1]), (1, 4, 0, [1, 1, 1], [5, 1, 70]),
    (2, 5, 64, [1] * 7, [3, 64, 65, 128, 129, 1, 300]), (1, 8, 127, [2, 1, 5], [2, 1, 200]),
    (8, 4, 1000, [1] * 40, list(range(1, 400, 10))), (1, 3, 33, [17, 0, 4], [17, 9, 90]),
    (2, 1, 129, [70, 3, 64, 1], [70, 3, 200, 33]), (1, 2, 300, [130, 260], [131, 700]),
    (1, 16, 65, [9, 2], [40, 2]), (1, 7, 2, [3, 3], [0, 2]), (2, 4, 0, [4, 2], [0, 1])])
def test_matches_float64(cuda, type_, hd, kh, g, prefix, new, rows):
    b = Batch(cuda, kh, g, hd, prefix, new, rows, type_, prefix + sum(rows))
    b.run()
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("hd,g,requests", [(64, 1, 40), (128, 2, 12), (128, 1, 3), (32, 3, 2),
                                           (64, 8, 600)])
def test_one_kv_head_and_a_long_prefix(cuda, type_, hd, g, requests):
    """As many parts of a row as there are CTAs; one request's rows over many of them."""
    torch = cuda
    b = Batch(torch, 1, g, hd, 20000, [1] * requests, [9000] + [3] * (requests - 1), type_, hd,
              ctx=9000 if requests < 100 else 9001)
    b.run()
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("new", [[1] * 6, [3, 1, 0, 2]])
def test_rows_of_no_request_stay_as_they_are(cuda, type_, new):
    """Padding before the first and behind the last request's tokens (q there
    may hold anything), and wider rows around both."""
    torch = cuda
    b = Batch(torch, 2, 4, 64, 200, new, [20 + i for i in range(len(new))], type_, 3, pad=(2, 5))
    out = torch.full((b.tokens, 8 + 16, 64), 7.0, device="cuda", dtype=b.q.dtype)
    part = out[:, 8:16]
    b.q[0], b.q[-1] = float("nan"), float("inf")
    b.run(part)
    b.check(part)
    a, z = int(b.first[0]), int(b.first[-1])
    assert (out[:a] == 7).all() and (out[z:] == 7).all()
    assert (out[:, :8] == 7).all() and (out[:, 16:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("g,most", [(1, 1), (4, 1), (4, 3), (8, 20)])
def test_rows_nobody_sees_may_hold_anything(cuda, type_, g, most):
    """NaN and infinities behind the prefix, behind each request's rows and in
    new rows that earlier tokens do not see."""
    torch = cuda
    b = Batch(torch, 2, g, 128, 150, [most, 1, most], [most + 70, 9, most], type_, 5)
    b.run()
    last, clean, k, v = most - 1, b.att.clone(), b.k.clone(), b.v.clone()
    b.kp[:, b.n:], b.vp[:, b.n:] = float("nan"), float("inf")
    for r, n in enumerate(b.rows):
        b.k[r, :, n:], b.v[r, :, n:] = float("inf"), float("nan")
    b.run()
    assert torch.equal(b.att, clean)
    # Request 0's last new row: only its last token sees it. (Its other tokens'
    # sums may be taken in another order then.)
    b.k[0, :, b.rows[0] - 1], b.v[0, :, b.rows[0] - 1] = float("nan"), float("inf")
    b.run()
    assert torch.equal(b.att[most:], clean[most:])
    b.k, b.v = k, v
    b.att[last] = clean[last]
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("g,most", [(1, 8), (8, 1), (5, 3), (16, 2), (8, 6), (3, 21), (1, 130)])
def test_hidden_new_rows_may_hold_anything(cuda, type_, hd, g, most):
    """Every size of a request's rows: NaN and infinities in all new rows but the first
    token's, which alone is looked at then, and behind the rows."""
    torch = cuda
    b = Batch(torch, 2, g, hd, 40, [most] * 3, [most, most + 64, most + 131], type_, hd + g)
    b.run()
    b.check()
    clean = b.att.clone()
    for r, n in enumerate(b.rows):
        b.k[r, :, n:], b.v[r, :, n:] = float("nan"), float("inf")
    b.run()
    assert torch.equal(b.att, clean)
    for r, n in enumerate(b.rows):
        b.v[r, :, n - most + 1:] = torch.tensor([float("inf"), float("nan")] * (hd // 2)).to(b.v)
        b.k[r, :, n - most + 1:] = float("nan")
    b.run()
    b.v[:] = torch.nan_to_num(b.v, 0.0, 0.0, 0.0)
    got = b.att[0::most].clone()
    b.att.copy_(clean)
    b.att[0::most] = got
    for r, n in enumerate(b.rows):     # what the first tokens see is as it was
        own = n - most + 1
        for x in (b.k, b.v):
            assert torch.isfinite(x[r, :, :own]).all()
    b.new, first = [1] * 3, b.first
    b.first, b.rows = first[:-1], [n - most + 1 for n in b.rows]
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("g,most", [(4, 1), (8, 1), (4, 4), (8, 6), (4, 20)])
@pytest.mark.parametrize("way", [1, -1])
def test_scores_that_rise_and_fall(cuda, type_, hd, g, most, way):
    """Scores that climb (or fall) along the keys, slowly and by more than any weight's
    range: maxima that move all the time, and such as never do."""
    torch = cuda
    b = Batch(torch, 2, g, hd, 333, [most] * 4, [most + 500, most + 37, most, most + 200], type_, 6)
    q = torch.randn(hd, device="cuda")
    b.q[:] = (q + 0.1 * torch.randn_like(b.q.float())).to(b.q)
    def slope(n):
        return way * torch.linspace(-4, 4, n, device="cuda")[:, None]
    unit = q / q.norm() ** 2 * math.sqrt(hd) * 12
    b.kp[:] = (slope(b.kp.shape[1]) * unit + 0.05 * torch.randn_like(b.kp.float())).to(b.kp)
    b.k[:] = (slope(b.k.shape[2]) * unit + 0.05 * torch.randn_like(b.k.float())).to(b.k)
    b.run()
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_equal_counts_need_no_first_in_place(cuda, type_):
    torch = cuda
    b = Batch(torch, 2, 4, 128, 500, [3] * 9, [3, 4, 100, 65, 64, 63, 7, 30, 300], type_, 7)
    b.run()
    b.check()
    q, want = b.q.clone(), b.att.clone()
    b.run(b.q, first=False)
    assert torch.equal(b.q, want)
    b.q = q


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_captured_call_serves_other_lengths(cuda, type_):
    """Prefix, rows and counts are read at each replay, and cut to the buffers;
    what is out of range reaches no memory outside."""
    torch = cuda
    b = Batch(torch, 2, 4, 64, 300, [2, 2, 2, 2], [70, 2, 5, 60], type_, 9, ctx=96, pad=(0, 4),
              most=6)
    b.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run()
    for n, new, rows in ((0, [1, 6, 0, 3], [96, 6, 0, 3]), (311, [6, 1, 1, 1], [8, 1, 90, 33])):
        b.n, b.new, b.rows = n, new, rows
        b.first = np.concatenate([[0], np.cumsum(new)])
        for to, v in ((b.d_prefix, [n]), (b.d_rows, rows), (b.d_first, b.first)):
            to.copy_(torch.tensor(np.asarray(v), dtype=torch.int32))
        b.att.fill_(float("nan"))
        graph.replay()
        b.check()
    # Cut: the prefix to its cache, rows to theirs.
    for v, n in ((1 << 30, 311), (-5, 0)):
        b.d_prefix.fill_(v)
        b.n = n
        graph.replay()
        b.check()
    b.d_rows.copy_(torch.tensor([1 << 30, -3, 90, 1 << 30], dtype=torch.int32))
    b.rows = [96, 0, 90, 96]
    graph.replay()
    b.check()
    # Tokens that are not there: nothing outside is written.
    guard = b.work.clone()
    for first in ([0, 1 << 30, 5, 6, 7], [-9, 2, 1, 40, 1 << 30], [9, 3, 1, 0, -1]):
        b.d_first.copy_(torch.tensor(first, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
    assert math.isnan(b.work[-1].item()) and math.isnan(guard[-1].item())


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
def test_far_rows_two_calls_at_once_same_bits(cuda, type_):
    """A request's rows beyond 2^31 bytes; calls on two streams, a workspace
    each."""
    torch = cuda
    kh, g, hd = 1, 2, 128
    ctx = (1 << 31) // (hd * 2) + 64
    b = Batch(torch, kh, g, hd, 70, [1, 1], [50, 90], type_, 2)
    k = torch.empty(2, kh, ctx, hd, device="cuda", dtype=b.q.dtype)
    v = torch.empty_like(k)
    k[:, :, :b.k.shape[2]], v[:, :, :b.v.shape[2]] = b.k, b.v
    b.k, b.v = k, v
    b.run()
    b.check()
    torch.cuda.synchronize()
    works = [torch.full_like(b.work, float("nan")) for _ in range(2)]
    atts = [torch.empty_like(b.att) for _ in range(2)]
    for s, w, a in zip([torch.cuda.Stream() for _ in range(2)], works, atts):
        with torch.cuda.stream(s):
            for _ in range(3):
                b.run(a, work=w)
    torch.cuda.synchronize()
    assert torch.equal(atts[0], b.att) and torch.equal(atts[1], b.att)


@pytest.mark.gpu
def test_one_prefix_for_all_is_one_tree_for_each(cuda):
    """A request alone is strasgpt_k_attn_tree over prefix and own rows in one
    cache, within both tolerances (their sums are split elsewhere)."""
    torch = cuda
    b = Batch(torch, 2, 4, 128, 700, [5], [60], F32, 4)
    b.run()
    L = runtime.lib()
    k = torch.cat([b.kp[:, :700], b.k[0, :, :60]], 1).contiguous()
    v = torch.cat([b.vp[:, :700], b.v[0, :, :60]], 1).contiguous()
    n = torch.tensor([755], dtype=torch.int32, device="cuda")
    mask = torch.tensor([(2 << i) - 1 for i in range(5)], dtype=torch.int64, device="cuda")
    size = L.strasgpt_k_attn_tree_workspace(5, 2, 4, 128)
    work, att = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty_like(b.q)
    assert L.strasgpt_k_attn_tree(
        b.q.data_ptr(), b.q.stride(0), k.data_ptr(), v.data_ptr(), F32, 5, 2, 4, 128, 760,
        n.data_ptr(), mask.data_ptr(), att.data_ptr(), att.stride(0), work.data_ptr(), size,
        stream(torch)) == 0
    b.check()
    b.check(att)


GOOD = dict(type_=F32, requests=3, t=2, tokens=6, kh=2, g=4, hd=128, pctx=64, ctx=32, ldq=1024,
            ldo=1024, stride=2 * 32 * 128, q=FAKE, kp=FAKE, vp=FAKE, prefix=FAKE, k=FAKE, v=FAKE,
            rows=FAKE, first=FAKE, att=FAKE, work=FAKE)


@pytest.mark.parametrize("change,words", [
    (dict(type_=7), "unknown type"), (dict(requests=-1), "empty shape"), (dict(t=0), "empty"),
    (dict(tokens=-1), "empty shape"), (dict(kh=0), "empty shape"), (dict(g=0), "empty shape"),
    (dict(t=1025), "1024 new"), (dict(g=129, ldq=1 << 20, ldo=1 << 20), "more than 128"),
    (dict(hd=96), "head_dim"), (dict(pctx=0), "without rows"), (dict(ctx=0), "without rows"),
    (dict(tokens=1 << 29), "2^31"), (dict(tokens=1 << 20, g=4, kh=1, t=1024), "4194240"),
    (dict(requests=1 << 30), "2^30"),
    (dict(ldq=1023), "overlap"), (dict(ldo=512), "overlap"), (dict(stride=-8), "negative"),
    *[({name: None}, "null") for name in ("q", "kp", "vp", "prefix", "k", "v", "rows", "att")],
    *[({name: FAKE + 8}, "16-byte") for name in ("q", "kp", "vp", "k", "v", "att")],
    (dict(ldq=1026), "16-byte"), (dict(stride=8194), "16-byte"), (dict(prefix=FAKE + 2), "aligned"),
    (dict(rows=FAKE + 1), "aligned"), (dict(first=FAKE + 2), "aligned"),
    (dict(ldo=1028), "same strides"), (dict(), ""),
])
def test_refuses(capfd, change, words):
    a = {**GOOD, **change}
    status = runtime.lib().strasgpt_k_attn_shared(
        a["q"], a["ldq"], a["kp"], a["vp"], a["pctx"], a["prefix"], a["k"], a["v"], a["stride"],
        a["ctx"], a["rows"], a["first"], a["type_"], a["requests"], a["t"], a["tokens"], a["kh"],
        a["g"], a["hd"], a["att"], a["ldo"], a["work"], 1 << 40, None)
    err = capfd.readouterr().err
    assert status == -1 and "[StrasGPT] Error" in err and words in err, (status, err)


def test_workspace_refuses_and_nothing_is_no_error(capfd):
    L = runtime.lib()
    for shape in ((9, 1, 1, 1, 1, 1, 64), (F32, -1, 1, 1, 1, 1, 64), (F32, 1, 0, 1, 1, 1, 64),
                  (F32, 1, 1, 1, 1, 1, 65), (F32, 1, 2000, 1, 1, 1, 64)):
        assert L.strasgpt_k_attn_shared_workspace(*shape) == 0
        assert "[StrasGPT] Error" in capfd.readouterr().err
    for requests, tokens in ((0, 5), (5, 0)):
        assert L.strasgpt_k_attn_shared(
            None, 512, None, None, 8, None, None, None, 0, 8, None, None, F32, requests, 1, tokens,
            1, 1, 64, None, 512, None, 0, None) == 0


@pytest.mark.gpu
def test_buffers_that_are_not_this_device_s_are_refused(cuda, capfd):
    torch = cuda
    b = Batch(torch, 1, 2, 64, 10, [1, 1], [4, 5], F32, 1)
    host = torch.zeros(1 << 16).pin_memory()
    args = [b.q.data_ptr(), b.q.stride(0), b.kp.data_ptr(), b.vp.data_ptr(), b.kp.shape[1],
            b.d_prefix.data_ptr(), b.k.data_ptr(), b.v.data_ptr(), b.k.stride(0), b.k.shape[2],
            b.d_rows.data_ptr(), b.d_first.data_ptr(), F32, 2, 1, 2, 1, 2, 64, b.att.data_ptr(),
            b.att.stride(0), b.work.data_ptr(), b.size(), None]
    for i in (0, 2, 3, 5, 6, 7, 10, 11, 19, 21):
        assert runtime.lib().strasgpt_k_attn_shared(*args[:i], host.data_ptr(), *args[i + 1:]) == -1
        assert "not device memory" in capfd.readouterr().err
    for i, v, words in ((22, b.size() - 1, "workspace is smaller"), (21, None, "workspace is smaller"),
                        (21, b.work.data_ptr() + 4, "workspace must be")):
        assert runtime.lib().strasgpt_k_attn_shared(*args[:i], v, *args[i + 1:]) == -1
        assert words in capfd.readouterr().err
