"""A layer's attention for a batch of requests, as the entry points of
include/strasgpt_kernels.h make it up: adapters beside the fused q, k, v projection,
positions on several axes, keys and values into each request's cache, attention behind
the shared prefix, adapters beside the output projection onto the residual, and beside
the gated feed-forward one. Each operator is checked against float64 on what the one
before it left, within the tolerances of its own tests; then all of it from a graph,
for other requests, against the same calls made one by one, bit for bit.
"""
import pytest
import test_attn_shared as shared
import test_lora as lora
import test_rope_axes as rope

from strasgpt_b200 import runtime

F32, BF16 = runtime.F32, runtime.BF16
STORE, ADD, SWIGLU = lora.STORE, lora.ADD, lora.SWIGLU
AXES = [10, 12, 10]


class Step:
    """Buffers for up to `most` new tokens of each of `requests` requests."""

    def __init__(self, torch, type_, requests=7, most=5, kh=2, g=4, hd=64, width=256, ctx=96,
                 prefix=300, adapters=4, rank=16, seed=1):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        dt = torch.float32 if type_ == F32 else torch.bfloat16
        rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
        i32 = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)  # noqa: E731
        self.torch, self.type_, self.requests, self.most = torch, type_, requests, most
        self.kh, self.g, self.hd, self.width, self.ctx = kh, g, hd, width, ctx
        self.tokens, self.qkv = requests * most, (g + 2) * kh * hd
        self.dt, self.gen, self.n, self.rank, self.adapters = dt, gen, prefix, rank, adapters
        m = self.tokens
        self.x, self.w = rand(m, width).to(dt), (rand(self.qkv, width) / width ** 0.5).to(dt)
        self.wo = (rand(width, g * kh * hd) / (g * kh * hd) ** 0.5).to(dt)
        self.wg = (rand(2 * width, width) / width ** 0.5).to(dt)
        low = lambda k, n: ((rand(adapters, rank, k) / k ** 0.5).bfloat16(),  # noqa: E731
                            (rand(adapters, n, rank) / rank ** 0.5).bfloat16())
        self.lq, self.lo, self.lg = (low(width, self.qkv), low(g * kh * hd, width),
                                     low(width, 2 * width))
        self.scale = 0.5 + torch.rand(adapters, device="cuda", generator=gen)
        self.kp, self.vp = rand(kh, prefix, hd).to(dt), rand(kh, prefix, hd).to(dt)
        self.k, self.v = (rand(requests, kh, ctx, hd).to(dt) for _ in range(2))
        self.adapter, self.d_first = i32(m), i32(requests + 1)
        self.d_rows, self.d_prefix = i32(requests), i32(1) + prefix
        self.pos, self.place = i32(3, m), torch.zeros(m, device="cuda", dtype=torch.int64)
        self.att = torch.zeros(m, g * kh * hd, device="cuda", dtype=dt)
        self.rope = runtime.Rope(2 * sum(AXES), theta=10000.0)
        self.axes = runtime.RopeAxes(AXES, runtime.AXES_DEALT)
        size = runtime.lib().strasgpt_k_attn_shared_workspace(type_, requests, most, m, kh, g, hd)
        self.work, self.size = torch.empty(size, dtype=torch.uint8, device="cuda"), size

    def requests_are(self, new, rows, adapters):
        """`rows` of each request with its new tokens; the other tokens are padding."""
        torch, first = self.torch, [0]
        place = torch.zeros(self.tokens, dtype=torch.int64)
        of = torch.full((self.tokens,), -1, dtype=torch.int32)
        pos = torch.zeros(3, self.tokens, dtype=torch.int32)
        for r, c in enumerate(new):
            a = first[-1]
            first.append(a + c)
            of[a:a + c] = adapters[r]
            at = torch.arange(rows[r] - c, rows[r])
            place[a:a + c] = r * self.kh * self.ctx + at
            pos[:, a:a + c] = torch.stack([at + self.n, at % 5 + 3 * r, at // 5]).int()
        self.new, self.rows, self.first, self.used = new, rows, first, first[-1]
        # Padding writes to a row of its own cache that no request has.
        place[self.used:] = (self.requests - 1) * self.kh * self.ctx + self.ctx - 1
        for to, v in ((self.place, place), (self.adapter, of), (self.pos, pos),
                      (self.d_first, torch.tensor(first)), (self.d_rows, torch.tensor(rows))):
            to.copy_(v)

    def lora(self, x, pair, base, out, epi):
        assert lora.call(self.torch, x, *pair, self.adapter, self.scale, base, out, epi,
                         self.type_) == 0

    def run(self, see=None):
        """All on the current stream; `see` gets (operator, what it had, what it left)."""
        torch, L, kh, g, hd = self.torch, runtime.lib(), self.kh, self.g, self.hd
        m, heads = self.tokens, self.g * self.kh
        see = see or (lambda *_: None)
        s = torch.cuda.current_stream().cuda_stream
        base = self.x @ self.w.T
        qkv = base.clone()
        self.lora(self.x, self.lq, qkv, qkv, STORE)
        see("lora", self.x, self.lq, base, None, qkv, STORE)
        rows = qkv.view(m, heads + 2 * kh, hd)
        # q and k turn where they are, in one call: k's heads stand behind q's.
        before = rows.clone()
        turned = rows[:, :heads + kh]
        assert L.strasgpt_k_rope_axes(
            turned.data_ptr(), rows.stride(0), hd, turned.data_ptr(), rows.stride(0), hd,
            self.type_, m, heads + kh, hd, self.pos.data_ptr(), m, 1, self.rope, self.axes, s) == 0
        see("rope", before[:, :heads + kh], turned)
        for cache, part in ((self.k, rows[:, heads:heads + kh]), (self.v, rows[:, heads + kh:])):
            head = torch.arange(kh, device="cuda") * self.ctx
            cache.view(-1, hd)[self.place[:, None] + head] = part
        q = rows[:, :heads]
        assert L.strasgpt_k_attn_shared(
            q.data_ptr(), rows.stride(0), self.kp.data_ptr(), self.vp.data_ptr(),
            self.kp.shape[1], self.d_prefix.data_ptr(), self.k.data_ptr(), self.v.data_ptr(),
            self.k.stride(0), self.ctx, self.d_rows.data_ptr(), self.d_first.data_ptr(),
            self.type_, self.requests, self.most, m, kh, g, hd, self.att.data_ptr(),
            self.att.stride(0), self.work.data_ptr(), self.size, s) == 0
        see("attn", q.contiguous(), self.att)
        x, base = self.x.clone(), self.att @ self.wo.T
        self.lora(self.att, self.lo, base, x, ADD)
        see("lora", self.att, self.lo, base, self.x, x, ADD)
        base, y = x @ self.wg.T, torch.empty_like(x)
        self.lora(x, self.lg, base, y, SWIGLU)
        see("lora", x, self.lg, base, None, y, SWIGLU)
        return y

    def check(self, what, *v):
        torch, u = self.torch, self.used
        if what == "lora":
            x, pair, base, old, got, epi = v
            want, err = lora.reference(torch, x, *pair, self.adapter, self.scale, base, old, epi,
                                       self.type_)
            assert ((got.double() - want).abs() <= err)[:u].all()
        elif what == "rope":
            rope.check(torch, v[1], v[0], self.pos, self.rope, AXES, runtime.AXES_DEALT, 0,
                       self.type_)
        else:
            b = shared.Batch.__new__(shared.Batch)
            b.torch, b.type_, b.kh, b.g, b.hd, b.n = (torch, self.type_, self.kh, self.g, self.hd,
                                                      self.n)
            b.new, b.rows, b.first, b.q = self.new, self.rows, self.first, v[0]
            b.kp, b.vp, b.k, b.v = self.kp, self.vp, self.k, self.v
            b.check(v[1].view(-1, self.g * self.kh, self.hd))


BATCHES = [([1, 1, 1, 1, 1, 1, 1], [1, 30, 64, 65, 90, 7, 2], [0, 1, 2, 3, -1, 0, 9]),
           ([5, 1, 0, 3, 5, 2, 1], [5, 80, 3, 64, 95, 2, 66], [3, -1, 2, 1, 1, 0, 3]),
           ([0, 0, 0, 1, 0, 0, 0], [1, 2, 3, 95, 4, 5, 6], [-1, 0, 0, 2, 0, 0, 0])]


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("new,rows,adapters", BATCHES)
def test_a_step_of_a_batch(cuda, type_, new, rows, adapters):
    step = Step(cuda, type_)
    step.requests_are(new, rows, adapters)
    step.run(step.check)


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("most,requests", [(5, 7), (60, 6)])
def test_captured_step_serves_other_batches(cuda, type_, most, requests):
    """Captured once; then other requests, lengths and adapters, two graphs with a
    workspace each at once among them. Prompts of up to 60 tokens as well, which go to
    other kernels."""
    torch = cuda
    steps = [Step(torch, type_, requests=requests, most=most, seed=s) for s in (1, 2)]
    graphs, outs = [], []
    for step in steps:
        step.requests_are([1] * requests, [9] * requests, [0] * requests)
        step.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step.run())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in steps]
    for i in range(3):
        for j, step in enumerate(steps):
            new = [(most * (r + 1) // requests + i + j) % (most + 1) for r in range(requests)]
            rows = [min(95, c + 13 * (r + i)) for r, c in enumerate(new)]
            step.requests_are(new, rows, [(r + i) % 6 - 1 for r in range(requests)])
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for step, out in zip(steps, outs):
            got, att = out.clone(), step.att.clone()
            again = step.run(step.check)
            u = step.used
            assert torch.equal(step.att[:u], att[:u]) and torch.equal(again[:u], got[:u])
