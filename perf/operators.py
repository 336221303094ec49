"""The operators of a step over drafted tokens, case by case: what each case
stands for in use, its inputs, its plain form and its exact value.

Three operators of include/strasgpt_kernels.h:

  rope        rotary positions given per token, both pair layouts, part of the
              head, stretched for long contexts (strasgpt_k_rope)
  attn_tree   attention of a tree of drafted tokens over the key/value cache
              that ends with the tree's own rows (strasgpt_k_attn_tree)
  sample      a token per row of logits under a temperature, top-k, top-p and
              min-p, from given random numbers (strasgpt_k_sample)

`run` computes the plain form with elementary torch operations, or, where
`own` is true, makes the library's calls.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "bf16": 2}
_CODES = {"fp32": 0, "bf16": 1}      # STRASGPT_F32, STRASGPT_BF16
_SCALINGS = {"none": 0, "linear": 1, "bands": 2}
_WORD = 64                           # drafted tokens per mask word


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def _rope(t, heads, head_dim, dim, type_, interleaved, scaling, far, to_cache):
    return {"op": "rope", "t": t, "heads": heads, "head_dim": head_dim, "dim": dim,
            "type": type_, "interleaved": interleaved, "scaling": scaling, "far": far,
            "to_cache": to_cache}


def _tree(t, kv_heads, group, head_dim, cached, type_):
    return {"op": "attn_tree", "t": t, "kv_heads": kv_heads, "group": group,
            "head_dim": head_dim, "cached": cached, "type": type_}


def _sample(rows, vocab, type_, top_k, top_p, min_p, masked):
    return {"op": "sample", "rows": rows, "vocab": vocab, "type": type_, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "masked": masked}


def listed():
    named = {
        # One new token: the 32 q and 8 k heads of a projection's row.
        "rope_token": _rope(1, 40, 128, 128, "fp32", False, "none", 8192, False),
        # The keys of a 2048-token chunk, rotated on their way from the
        # projection's rows into a layer's cache, wavelengths stretched.
        "rope_chunk_keys": _rope(2048, 8, 128, 128, "fp32", False, "bands", 131072, True),
        # A long bf16 chunk, adjacent pairs, half of the head turned, positions
        # close to a million.
        "rope_part_bf16": _rope(8191, 40, 128, 64, "bf16", True, "linear", 1000000, False),
        # A single token over a short cache (16 q heads on 8 kv heads).
        "tree_token": _tree(1, 8, 2, 128, 613, "fp32"),
        # A 24-token draft after a prompt of usual length.
        "tree_draft": _tree(24, 8, 4, 128, 2291, "fp32"),
        # A few tokens over a long cache: the cache's bytes are what counts.
        "tree_long_bf16": _tree(5, 8, 4, 128, 130021, "bf16"),
        # 64 wide heads on 8, head dimension 64, a chain of 16 drafted tokens.
        "tree_wide_bf16": _tree(16, 8, 8, 64, 32801, "bf16"),
        # A full tree of 64 over a long cache, in both types.
        "tree_full_fp32": _tree(64, 8, 4, 128, 32768, "fp32"),
        "tree_full_bf16": _tree(64, 8, 4, 128, 65500, "bf16"),
        # One row of an ordinary request.
        "sample_token": _sample(1, 128256, "fp32", 50, 0.9, 0.0, 0.0),
        # The rows of a full tree, one choice for each drafted token.
        "sample_tree": _sample(64, 151936, "fp32", 0, 0.95, 0.0, 0.0),
        # A large batch of bf16 rows (many equal values), a third of the
        # vocabulary ruled out by a grammar.
        "sample_batch_bf16": _sample(256, 201088, "bf16", 200, 0.98, 0.02, 0.33),
    }
    return [dict(case, name=name) for name, case in named.items()]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "attn_tree", "attn_tree", "sample"])
    type_ = rng.choice(["fp32", "bf16"])
    if op == "rope":
        head_dim = rng.choice([32, 64, 80, 96, 128])
        dim = rng.choice([head_dim, head_dim // 2, 2 * rng.randint(1, head_dim // 2)])
        return _rope(_log_int(rng, 1, 8191), rng.randint(1, 40), head_dim, dim, type_,
                     rng.random() < 0.5, rng.choice(sorted(_SCALINGS)),
                     _log_int(rng, 1000, 2000000), rng.random() < 0.5)
    if op == "attn_tree":
        head_dim = rng.choice([32, 64, 128])
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8])
        t = _log_int(rng, 1, 96)
        most = 65536 * 64 * 32 // (t * kv_heads * group)
        cached = _log_int(rng, 1, min(131072, most)) - 1
        return _tree(t, kv_heads, group, head_dim, cached, type_)
    vocab = _log_int(rng, 500, 260000)
    rows = _log_int(rng, 1, min(256, 256 * 201088 // vocab))
    return _sample(rows, vocab, type_, rng.choice([0, 1, 20, 50, 1000]),
                   rng.choice([1.0, 0.99, 0.9, 0.5]), rng.choice([0.0, 0.0, 0.05, 0.3]),
                   rng.choice([0.0, 0.0, 0.5, 0.99]))


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _prepare_rope(c, gen):
    type_ = _TYPES[c["type"]]
    t, heads, hd = c["t"], c["heads"], c["head_dim"]
    # The rows of a fused projection: these heads and as many entries again
    # that another call reads.
    rows = torch.randn(t, 2 * heads * hd, device="cuda", generator=gen).to(type_)
    x = rows[:, :heads * hd].view(t, heads, hd)
    if c["to_cache"]:
        ctx = (t + 63) // 64 * 64 + 64
        cache = torch.zeros(heads, ctx, hd, device="cuda", dtype=type_)
        y = cache[:, ctx - t:].transpose(0, 1)      # [t][heads][hd] of the cache's rows
    else:
        y = torch.empty(t, heads, hd, device="cuda", dtype=type_)
    start = torch.randint(0, max(1, c["far"] - t), (1,), device="cuda", generator=gen)
    # Neighbours in a drafted tree share a position.
    step = torch.randint(0, 2, (t,), device="cuda", generator=gen)
    pos = (start + torch.cumsum(step, 0)).to(torch.int32)
    turn = {"dim": c["dim"], "interleaved": int(c["interleaved"]), "theta": 500000.0,
            "scaling": _SCALINGS[c["scaling"]], "factor": 8.0, "low": 1.0, "high": 4.0,
            "original": 8192, "magnitude": 1.0 if c["scaling"] == "none" else 1.2}
    return {"x": x, "y": y, "pos": pos, "turn": turn}


def _prepare_tree(c, gen, seed):
    type_ = _TYPES[c["type"]]
    t, kh, g, hd, n = c["t"], c["kv_heads"], c["group"], c["head_dim"], c["cached"]
    ctx = (n + t + 63) // 64 * 64
    # Scores of a standard deviation of about 2: a few keys carry most of a row.
    q = (2 * torch.randn(t, kh * g, hd, device="cuda", generator=gen)).to(type_)
    k = torch.randn(kh, ctx, hd, device="cuda", generator=gen).to(type_)
    v = torch.randn(kh, ctx, hd, device="cuda", generator=gen).to(type_)
    # A random tree: every drafted token follows an earlier one or the cache,
    # and attends to itself and to those on its way to the root.
    rng = np.random.RandomState(seed % (1 << 32))
    words = (t + _WORD - 1) // _WORD
    mask = np.zeros((t, words), dtype=np.uint64)
    for i in range(t):
        parent = int(rng.randint(max(-1, i - 8), i)) if i else -1
        if parent >= 0:
            mask[i] = mask[parent]
        mask[i, i // _WORD] |= np.uint64(1 << (i % _WORD))
    mask = torch.from_numpy(mask.view(np.int64)).cuda()
    cached = torch.tensor([n], dtype=torch.int32, device="cuda")
    return {"q": q, "k": k, "v": v, "mask": mask, "cached": cached, "n": n,
            "att": torch.empty_like(q)}


def _prepare_sample(c, gen):
    rows, vocab = c["rows"], c["vocab"]
    x = 2 * torch.randn(rows, vocab, device="cuda", generator=gen)
    # A model's likely next tokens stand out of the rest.
    likely = torch.randint(0, vocab, (rows, 48), device="cuda", generator=gen)
    x.scatter_add_(1, likely, 4 + 9 * torch.rand(rows, 48, device="cuda", generator=gen))
    if c["masked"]:
        out = torch.rand(rows, vocab, device="cuda", generator=gen) < c["masked"]
        x.masked_fill_(out, float("-inf"))
    x = x.to(_TYPES[c["type"]])
    spread = torch.rand(rows, device="cuda", generator=gen)
    temperature = 0.4 + 1.1 * spread
    if rows > 4:
        temperature[3] = 0.0                 # one greedy request among the others
    full = lambda v, dt: torch.full((rows,), v, device="cuda", dtype=dt)  # noqa: E731
    return {"logits": x, "temperature": temperature, "top_k": full(c["top_k"], torch.int32),
            "top_p": full(c["top_p"], torch.float32), "min_p": full(c["min_p"], torch.float32),
            "u": torch.rand(rows, device="cuda", generator=gen),
            "token": full(0, torch.int32), "prob": full(0.0, torch.float32),
            "kept": full(0, torch.int32)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["op"] == "rope":
        state = _prepare_rope(case, gen)
    elif case["op"] == "attn_tree":
        state = _prepare_tree(case, gen, int(seed))
    else:
        state = _prepare_sample(case, gen)
    return {**state, "case": dict(case)}


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def _frequencies(turn, device):
    """Radians per position of every pair, in 64 bits."""
    dim = turn["dim"]
    j = torch.arange(0, dim, 2, device=device, dtype=torch.float64)
    f = torch.exp(-j / dim * math.log(turn["theta"]))
    if turn["scaling"] == 1:
        f = f / turn["factor"]
    elif turn["scaling"] == 2:
        turns = turn["original"] * f / (2 * math.pi)
        keep = ((turns - turn["low"]) / (turn["high"] - turn["low"])).clamp(0, 1)
        f = f * (keep + (1 - keep) / turn["factor"])
    return f


def _plain_rope(s):
    turn, x, y = s["turn"], s["x"], s["y"]
    dim = turn["dim"]
    # Angles of far positions need 64 bits.
    angle = s["pos"].double()[:, None] * _frequencies(turn, x.device)
    cos = (torch.cos(angle) * turn["magnitude"]).float()[:, None]
    sin = (torch.sin(angle) * turn["magnitude"]).float()[:, None]
    f = x.float()
    out = f.clone()
    if turn["interleaved"]:
        a, b = f[..., 0:dim:2], f[..., 1:dim:2]
        out[..., 0:dim:2], out[..., 1:dim:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = f[..., :dim // 2], f[..., dim // 2:dim]
        out[..., :dim // 2], out[..., dim // 2:dim] = a * cos - b * sin, a * sin + b * cos
    y.copy_(out)
    return y


def _allowed(mask, t):
    """[t][t]: which drafted tokens a drafted token attends to."""
    j = torch.arange(t, device=mask.device)
    return ((mask[:, j // _WORD] >> (j % _WORD)) & 1).bool()


def _plain_tree(s):
    c, n = s["case"], s["n"]
    t, kh, g, hd = c["t"], c["kv_heads"], c["group"], c["head_dim"]
    q = s["q"].float().view(t, kh, g, hd).permute(1, 0, 2, 3).reshape(kh, t * g, hd)
    k, v = s["k"][:, :n + t].float(), s["v"][:, :n + t].float()
    score = torch.matmul(q, k.transpose(1, 2)).view(kh, t, g, n + t) / math.sqrt(hd)
    score[..., n:].masked_fill_(~_allowed(s["mask"], t)[None, :, None], float("-inf"))
    score = score.view(kh, t * g, n + t)
    score.sub_(score.max(-1, keepdim=True).values).exp_()
    out = torch.matmul(score, v) / score.sum(-1, keepdim=True)
    return out.view(kh, t, g, hd).permute(1, 0, 2, 3).reshape(t, kh * g, hd).to(s["q"].dtype)


def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    greedy = s["temperature"] <= 0
    heat = torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    # From the largest logit down, equal ones by index.
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    # Sums over a vocabulary and their borders need 64 bits.
    w = torch.exp((x - x[:, :1]) / heat)
    rank = torch.arange(vocab, device=x.device)
    k = torch.where(greedy, 1, torch.where(s["top_k"] > 0, s["top_k"], vocab))[:, None]
    keep = (rank < k) & (w > 0)
    w = w * keep
    before = torch.cumsum(w, 1) - w
    top_p = s["top_p"].double()[:, None]
    keep &= (before < top_p * w.sum(1, keepdim=True)) | (top_p >= 1) | (rank == 0)
    keep &= w >= s["min_p"].double()[:, None]
    w = w * keep
    # The choice goes by index: back to the vocabulary's order.
    mass = torch.zeros_like(w).scatter_(1, order, w)
    total = mass.sum(1, keepdim=True)
    below = torch.cumsum(mass, 1) <= s["u"].double()[:, None] * total
    token = below.sum(1, keepdim=True).clamp(max=vocab - 1)
    prob = mass.gather(1, token) / total
    return (token[:, 0].to(torch.int32), prob[:, 0].float(), keep.sum(1).to(torch.int32))


def _own_rope(s):
    from strasgpt_b200 import runtime
    c, x, y, lib = s["case"], s["x"], s["y"], runtime.lib()
    if "params" not in s:
        s["params"] = runtime.Rope(**s["turn"])
    lib.strasgpt_k_rope(x.data_ptr(), x.stride(0), x.stride(1), y.data_ptr(), y.stride(0),
                        y.stride(1), _CODES[c["type"]], c["t"], c["heads"], c["head_dim"],
                        s["pos"].data_ptr(), s["params"],
                        torch.cuda.current_stream().cuda_stream)
    return y


def _own_tree(s):
    from strasgpt_b200 import runtime
    c, q, k, lib = s["case"], s["q"], s["k"], runtime.lib()
    if "workspace" not in s:
        size = lib.strasgpt_k_attn_tree_workspace(c["t"], c["kv_heads"], c["group"],
                                                  c["head_dim"])
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    work = s["workspace"]
    lib.strasgpt_k_attn_tree(q.data_ptr(), q.stride(0), k.data_ptr(), s["v"].data_ptr(),
                             _CODES[c["type"]], c["t"], c["kv_heads"], c["group"],
                             c["head_dim"], k.shape[1], s["cached"].data_ptr(),
                             s["mask"].data_ptr(), s["att"].data_ptr(), s["att"].stride(0),
                             work.data_ptr(), work.numel(),
                             torch.cuda.current_stream().cuda_stream)
    return s["att"]


def _own_sample(s):
    from strasgpt_b200 import runtime
    c, x, lib = s["case"], s["logits"], runtime.lib()
    lib.strasgpt_k_sample(x.data_ptr(), _CODES[c["type"]], x.stride(0), c["rows"], c["vocab"],
                          s["temperature"].data_ptr(), s["top_k"].data_ptr(),
                          s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["u"].data_ptr(),
                          s["token"].data_ptr(), s["prob"].data_ptr(), s["kept"].data_ptr(),
                          torch.cuda.current_stream().cuda_stream)
    return s["token"], s["prob"], s["kept"]


def run(state):
    op = state["case"]["op"]
    if own:
        if op == "rope":
            return _own_rope(state)
        return _own_tree(state) if op == "attn_tree" else _own_sample(state)
    if op == "rope":
        return _plain_rope(state)
    return _plain_tree(state) if op == "attn_tree" else _plain_sample(state)


# --------------------------------------------------------------------------
# what a pass cannot do without, and its exact value
# --------------------------------------------------------------------------
def work(case):
    c, size = case, _BYTES[case["type"]]
    if c["op"] == "rope":
        every = c["t"] * c["heads"] * c["head_dim"]
        return {"bytes": 2 * every * size + 4 * c["t"],
                "flops": 3 * c["t"] * c["heads"] * c["dim"]}
    if c["op"] == "attn_tree":
        t, kh, g, hd, n = c["t"], c["kv_heads"], c["group"], c["head_dim"], c["cached"]
        words = (t + _WORD - 1) // _WORD
        return {"bytes": 2 * kh * (n + t) * hd * size + 2 * t * kh * g * hd * size + 8 * t * words,
                "flops": 4 * t * kh * g * hd * (n + 1)}
    every = c["rows"] * c["vocab"]
    return {"bytes": every * size + 32 * c["rows"], "flops": 4 * every}


def _exact_rope(s):
    """Pairs as complex numbers, turned by e^(i angle)."""
    turn = s["turn"]
    dim, half = turn["dim"], turn["dim"] // 2
    x, pos = s["x"].double(), s["pos"].double()
    turned = []
    for j in range(half):
        f = turn["theta"] ** (-2.0 * j / dim)
        if turn["scaling"] == 1:
            f /= turn["factor"]
        elif turn["scaling"] == 2:
            wave = 2 * math.pi / f
            keep = (turn["original"] / wave - turn["low"]) / (turn["high"] - turn["low"])
            keep = min(1.0, max(0.0, keep))
            f = (1 - keep) * f / turn["factor"] + keep * f
        a, b = (2 * j, 2 * j + 1) if turn["interleaved"] else (j, j + half)
        z = torch.complex(x[..., a], x[..., b])
        e = torch.polar(torch.full_like(pos, turn["magnitude"]), pos * f)
        turned.append((a, b, z * e[:, None]))
    for a, b, z in turned:
        x[..., a], x[..., b] = z.real, z.imag
    return x


def _exact_tree(s):
    """One kv head at a time; the tree's own rows joined to the cache's by
    their sums."""
    c, n = s["case"], s["n"]
    t, kh, g, hd = c["t"], c["kv_heads"], c["group"], c["head_dim"]
    bits = s["mask"].cpu().numpy().view(np.uint64)
    allowed = torch.tensor([[bool((int(bits[i, j // _WORD]) >> (j % _WORD)) & 1)
                             for j in range(t)] for i in range(t)], device="cuda")
    out = torch.empty(t, kh * g, hd, dtype=torch.float64, device="cuda")
    for h in range(kh):
        k, v = s["k"][h].double(), s["v"][h].double()
        for a in range(h * g, (h + 1) * g):
            q = s["q"][:, a].double() / math.sqrt(hd)
            old = q @ k[:n].T
            new = torch.where(allowed, q @ k[n:n + t].T, -math.inf)
            top = new.amax(1, keepdim=True)
            if n:
                top = torch.maximum(top, old.amax(1, keepdim=True))
            old, new = torch.exp(old - top), torch.exp(new - top)
            out[:, a] = ((old @ v[:n] + new @ v[n:n + t])
                         / (old.sum(1, keepdim=True) + new.sum(1, keepdim=True)))
    return out


def _exact_sample(s):
    """A row at a time on the host, from the definition."""
    x = s["logits"].float().cpu().numpy().astype(np.float64)
    get = lambda name: s[name].cpu().numpy().astype(np.float64)  # noqa: E731
    heat, top_k, top_p, min_p, u = (get(n) for n in
                                    ("temperature", "top_k", "top_p", "min_p", "u"))
    rows, vocab = x.shape
    token, prob, kept = [], [], []
    for r in range(rows):
        row = x[r]
        if heat[r] <= 0:
            token.append(int(np.argmax(row)))
            prob.append(1.0)
            kept.append(1)
            continue
        order = np.argsort(-row, kind="stable")
        order = order[:int(top_k[r])] if top_k[r] > 0 else order
        weight = np.exp((row[order] - row[order[0]]) / heat[r])
        order, weight = order[weight > 0], weight[weight > 0]
        if top_p[r] < 1:
            sums = np.cumsum(weight)
            last = int(np.searchsorted(sums, top_p[r] * sums[-1]))
            order, weight = order[:last + 1], weight[:last + 1]
        order, weight = order[weight >= min_p[r]], weight[weight >= min_p[r]]
        by_index = np.argsort(order)
        order, weight = order[by_index], weight[by_index]
        sums = np.cumsum(weight)
        at = min(int(np.searchsorted(sums, u[r] * sums[-1], side="right")), len(order) - 1)
        token.append(int(order[at]))
        prob.append(weight[at] / sums[-1])
        kept.append(len(order))
    return (torch.tensor(token, dtype=torch.int32), torch.tensor(prob, dtype=torch.float64),
            torch.tensor(kept, dtype=torch.int32))


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(state)
    return _exact_tree(state) if case["op"] == "attn_tree" else _exact_sample(state)
