"""The operators of a step of a batch of requests, case by case: what each
case stands for in use, its inputs, its plain form and its exact value.

Three operators of include/strasgpt_kernels.h:

  rope_axes    rotary positions with several axes (time, height, width), the
               pairs of a head shared out among them (strasgpt_k_rope_axes)
  lora         low-rank adapters of many requests at once, beside a projection
               that all of them share (strasgpt_k_lora)
  attn_shared  attention of a batch of requests behind one prefix, each with
               cache rows of its own (strasgpt_k_attn_shared)

`run` computes the plain form with elementary torch operations, or, where
`own` is true, makes the library's calls.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "bf16": 2}
_CODES = {"fp32": 0, "bf16": 1}            # STRASGPT_F32, STRASGPT_BF16
_SCALINGS = {"none": 0, "linear": 1, "bands": 2}
_ORDERS = {"runs": 0, "dealt": 1}          # STRASGPT_AXES_RUNS, STRASGPT_AXES_DEALT
_EPILOGUES = {"store": 0, "swiglu": 2}     # STRASGPT_EPI_*


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def _axes(t, heads, head_dim, sections, type_, order, separate, scaling, far, to_cache):
    """sections: the pairs of each axis, "24 20 20"; separate: each axis has
    frequencies of its own; far: positions lie below it."""
    return {"op": "rope_axes", "t": t, "heads": heads, "head_dim": head_dim,
            "sections": sections, "type": type_, "order": order, "separate": separate,
            "scaling": scaling, "far": far, "to_cache": to_cache}


def _lora(m, k, n, rank, adapters, type_, mixed, epilogue):
    """mixed: any token may have any adapter; else a run of tokens has one."""
    return {"op": "lora", "m": m, "k": k, "n": n, "rank": rank, "adapters": adapters,
            "type": type_, "mixed": mixed, "epilogue": epilogue}


def _shared(requests, most, kv_heads, group, head_dim, prefix, behind, type_):
    """most: new tokens of a request, at most; behind: a request's own rows, at
    most, new ones included."""
    return {"op": "attn_shared", "requests": requests, "most": most, "kv_heads": kv_heads,
            "group": group, "head_dim": head_dim, "prefix": prefix, "behind": behind,
            "type": type_}


def listed():
    named = {
        # One new token of text after images: the 32 q and 8 k heads of a row.
        "axes_token": _axes(1, 40, 128, "24 20 20", "fp32", "dealt", False, "none", 8192, False),
        # The keys of a 2048-token chunk with images in it on their way into a
        # layer's cache, wavelengths stretched.
        "axes_chunk_keys": _axes(2048, 8, 128, "16 24 24", "fp32", "runs", False, "bands",
                                 131072, True),
        # The patches of a large image, height and width, q and k heads.
        "axes_image_bf16": _axes(8191, 32, 80, "20 20", "bf16", "runs", True, "none", 1000,
                                 False),
        # One request's token on a projection of 2048 x 2048.
        "lora_token": _lora(1, 2048, 2048, 8, 4, "fp32", True, "store"),
        # A batch of single tokens, most with an adapter of their own, on a
        # fused q, k, v projection.
        "lora_batch": _lora(61, 4096, 6144, 16, 48, "fp32", True, "store"),
        # Some requests' prompts at once, an adapter each.
        "lora_prompts": _lora(2047, 4096, 4096, 32, 6, "fp32", False, "store"),
        # A longer chunk on a gated feed-forward projection, bf16.
        "lora_gated_bf16": _lora(4001, 4096, 28672, 64, 5, "bf16", False, "swiglu"),
        # Two requests that have just begun (16 q heads on 8 kv heads).
        "shared_few": _shared(2, 1, 8, 2, 128, 613, 40, "fp32"),
        # A full batch behind a long system prompt, each some hundred tokens on.
        "shared_batch_bf16": _shared(64, 1, 8, 4, 128, 32768, 1021, "bf16"),
        "shared_batch_fp32": _shared(48, 1, 8, 4, 128, 8191, 700, "fp32"),
        # Drafted tokens of each request, 64 wide heads on 8, head dimension 64.
        "shared_drafts_bf16": _shared(31, 6, 8, 8, 64, 16001, 2000, "bf16"),
        # The questions of a batch about one document, all of them new.
        "shared_prompts_bf16": _shared(16, 96, 8, 4, 128, 8192, 96, "bf16"),
    }
    return [dict(case, name=name) for name, case in named.items()]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_axes(rng, type_):
    head_dim = rng.choice([32, 64, 80, 96, 128])
    axes = rng.choice([2, 3, 3, 4])
    pairs = rng.choice([head_dim // 2, head_dim // 4, rng.randint(axes, head_dim // 2)])
    cuts = sorted(rng.sample(range(1, pairs), axes - 1))
    sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
    return _axes(_log_int(rng, 1, 8191), rng.randint(1, 32), head_dim,
                 " ".join(str(s) for s in sections), type_, rng.choice(sorted(_ORDERS)),
                 rng.random() < 0.4, rng.choice(sorted(_SCALINGS)), _log_int(rng, 1000, 2000000),
                 rng.random() < 0.5)


def _draw_lora(rng, type_):
    m = _log_int(rng, 1, 4096)
    k, rank = 8 * _log_int(rng, 64, 1024), 8 * _log_int(rng, 1, 16)
    n = _log_int(rng, 64, min(28672, max(256, 190000000 // (m * _BYTES[type_]) - k)))
    mixed = m <= 256
    adapters = rng.randint(1, 64 if mixed else 8)
    epilogue = rng.choice(["store", "swiglu"])
    return _lora(m, k, n + n % 2 if epilogue == "swiglu" else n, rank, adapters, type_, mixed,
                 epilogue)


def _draw_shared(rng, type_):
    head_dim = rng.choice([32, 64, 128])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8])
    requests = _log_int(rng, 1, 96)
    most = rng.choice([1, 1, 1, 2, 5, _log_int(rng, 2, 96)])
    # Pairs of a row and a key, and rows of the caches, that no listed case is over.
    pairs, keys = 1 << (27 if type_ == "bf16" else 25), (1 << 20) // _BYTES[type_]
    rows = requests * most * kv_heads * group
    prefix = _log_int(rng, 1, min(131072, pairs // rows, keys // kv_heads))
    behind = most + _log_int(rng, 1, max(2, min(4096, pairs // rows // 4,
                                                keys // (requests * kv_heads)))) - 1
    return _shared(requests, most, kv_heads, group, head_dim, prefix, behind, type_)


def draw(rng):
    op = rng.choice([_draw_axes, _draw_lora, _draw_shared, _draw_shared])
    return op(rng, rng.choice(["fp32", "bf16"]))


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _prepare_axes(c, gen):
    type_ = _TYPES[c["type"]]
    t, heads, hd = c["t"], c["heads"], c["head_dim"]
    sections = [int(s) for s in c["sections"].split()]
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
    # Patches row by row behind a text: the last axis runs fastest, and what
    # is left over is the first one's.
    start = torch.randint(0, max(1, c["far"] - t), (1,), device="cuda", generator=gen)
    i, pos = torch.arange(t, device="cuda"), []
    for width in [23, 37, 64][:len(sections) - 1]:
        pos.insert(0, i % width)
        i = i // width
    pos = (torch.stack([i] + pos) + start).to(torch.int32)
    turn = {"dim": 2 * sum(sections), "interleaved": 0, "theta": 500000.0,
            "scaling": _SCALINGS[c["scaling"]], "factor": 8.0, "low": 1.0, "high": 4.0,
            "original": 8192, "magnitude": 1.0 if c["scaling"] == "none" else 1.2}
    return {"x": x, "y": y, "pos": pos, "turn": turn, "sections": sections}


def _token_adapters(c):
    """Which adapter each token has, -1: none."""
    i, m, d = np.arange(c["m"]), c["m"], c["adapters"]
    if c["mixed"]:
        return np.where(i % 16 == 15, -1, (i * 7 + i // 5) % d)
    # Uneven runs, one without an adapter if there are several.
    run = np.minimum((np.sqrt((i + 1) / m) * (d + 1)).astype(np.int64), d)
    return np.where(run == d, d - 1 if d == 1 else -1, run)


def _prepare_lora(c, gen):
    type_ = _TYPES[c["type"]]
    m, k, n, r, d = c["m"], c["k"], c["n"], c["rank"], c["adapters"]
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    out = torch.empty(m, n // 2 if c["epilogue"] == "swiglu" else n, device="cuda", dtype=type_)
    return {"x": rand(m, k).to(type_), "base": rand(m, n).to(type_),
            "a": (rand(d, r, k) / math.sqrt(k)).to(torch.bfloat16),
            "b": (rand(d, n, r) / math.sqrt(r)).to(torch.bfloat16),
            "scale": 0.25 + 0.5 * torch.rand(d, device="cuda", generator=gen),
            "adapter": torch.from_numpy(_token_adapters(c).astype(np.int32)).cuda(), "out": out}


def _counts(c):
    """New tokens of each request, and its own rows with them."""
    r = np.arange(c["requests"])
    new = c["most"] - r * 5 % c["most"] if c["most"] > 1 else np.ones_like(r)
    rows = c["behind"] - r * 7919 % (c["behind"] // 2 + 1)
    return new, np.maximum(rows, new)


def _prepare_shared(c, gen):
    type_ = _TYPES[c["type"]]
    kh, g, hd = c["kv_heads"], c["group"], c["head_dim"]
    new, rows = _counts(c)
    tokens, ctx = int(new.sum()), (c["behind"] + 63) // 64 * 64
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    # Scores of a standard deviation of about 2: a few keys carry most of a row.
    q = (2 * rand(tokens, kh * g, hd)).to(type_)
    i32 = lambda v: torch.from_numpy(np.asarray(v, dtype=np.int32)).cuda()  # noqa: E731
    return {"q": q, "kp": rand(kh, c["prefix"], hd).to(type_),
            "vp": rand(kh, c["prefix"], hd).to(type_),
            "k": rand(c["requests"], kh, ctx, hd).to(type_),
            "v": rand(c["requests"], kh, ctx, hd).to(type_),
            "prefix": i32([c["prefix"]]), "rows": i32(rows),
            "first": i32(np.concatenate([[0], np.cumsum(new)])), "att": torch.empty_like(q)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    make = {"rope_axes": _prepare_axes, "lora": _prepare_lora, "attn_shared": _prepare_shared}
    return {**make[case["op"]](case, gen), "case": dict(case)}


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def _axis_of_pairs(sections, order):
    """Each pair's axis, and its number among that axis's pairs."""
    if order == "runs":
        return ([a for a, s in enumerate(sections) for _ in range(s)],
                [j for s in sections for j in range(s)])
    axis = [a for j in range(max(sections)) for a, s in enumerate(sections) if j < s]
    return axis, [j for j in range(max(sections)) for s in sections if j < s]


def _plain_axes(s):
    c, turn, x, y = s["case"], s["turn"], s["x"], s["y"]
    dim, sections = turn["dim"], s["sections"]
    if "of_pairs" not in s:  # a table that such a program keeps
        axis, number = _axis_of_pairs(sections, c["order"])
        power = ([j / sections[a] for a, j in zip(axis, number)] if c["separate"]
                 else [2 * j / dim for j in range(dim // 2)])
        s["of_pairs"] = (torch.tensor(axis, device=x.device),
                         torch.tensor(power, device=x.device, dtype=torch.float64))
    axis, power = s["of_pairs"]
    f = torch.exp(-power * math.log(turn["theta"]))
    if c["scaling"] == "linear":
        f = f / turn["factor"]
    elif c["scaling"] == "bands":
        turns = turn["original"] * f / (2 * math.pi)
        keep = ((turns - turn["low"]) / (turn["high"] - turn["low"])).clamp(0, 1)
        f = f * (keep + (1 - keep) / turn["factor"])
    # Angles of far positions need 64 bits.
    angle = s["pos"].double()[axis].T * f
    cos = (torch.cos(angle) * turn["magnitude"]).float()[:, None]
    sin = (torch.sin(angle) * turn["magnitude"]).float()[:, None]
    f = x.float()
    out = f.clone()
    a, b = f[..., :dim // 2], f[..., dim // 2:dim]
    out[..., :dim // 2], out[..., dim // 2:dim] = a * cos - b * sin, a * sin + b * cos
    y.copy_(out)
    return y


def _plain_lora(s):
    c, out = s["case"], s["out"]
    m, k, n, r, d = c["m"], c["k"], c["n"], c["rank"], c["adapters"]
    # All adapters' entries of every token; each keeps its own adapter's.
    low = torch.matmul(s["x"].float(), s["a"].float().view(d * r, k).T).view(m, d, r)
    mine = s["adapter"][:, None] == torch.arange(d, device=out.device)
    low = torch.where(mine[..., None], low * s["scale"][:, None], 0.0).view(m, d * r)
    y = torch.matmul(low, s["b"].float().permute(0, 2, 1).reshape(d * r, n)) + s["base"].float()
    if c["epilogue"] == "swiglu":
        gate, up = y[:, 0::2], y[:, 1::2]
        y = gate / (1 + torch.exp(-gate)) * up
    out.copy_(y)
    return out


def _plain_shared(s):
    c, q, first = s["case"], s["q"], s["first"].long()
    kh, g, hd, prefix, most = c["kv_heads"], c["group"], c["head_dim"], c["prefix"], c["most"]
    requests, tokens, ctx = c["requests"], q.shape[0], s["k"].shape[2]
    # [requests][kh][most * g][hd], requests with fewer new tokens padded.
    j = torch.arange(most, device=q.device)
    at = (first[:-1, None] + j).clamp(max=tokens - 1)
    rows = q.float()[at].view(requests, most, kh, g, hd).permute(0, 2, 1, 3, 4)
    rows = rows.reshape(requests, kh, most * g, hd) / math.sqrt(hd)
    # The prefix in one product for all requests: [kh][requests * most * g].
    one = lambda x: x.transpose(0, 1).reshape(kh, requests * most * g, -1)  # noqa: E731
    each = lambda x: x.view(kh, requests, most * g, -1).transpose(0, 1)     # noqa: E731
    old = each(torch.matmul(one(rows), s["kp"].float().transpose(1, 2)))
    new = torch.matmul(rows, s["k"].float().transpose(2, 3)).view(requests, kh, most, g, ctx)
    # Token j of a request sees its rows up to its own.
    last = s["rows"][:, None] - (first[1:] - first[:-1])[:, None] + j
    hidden = torch.arange(ctx, device=q.device) > last[..., None]
    new = new.masked_fill(hidden[:, None, :, None], -math.inf).view(requests, kh, most * g, ctx)
    top = old.amax(-1, keepdim=True).maximum(new.amax(-1, keepdim=True))
    old, new = old.sub_(top).exp_(), new.sub_(top).exp_()
    total = old.sum(-1, keepdim=True) + new.sum(-1, keepdim=True)
    v = s["v"].float().masked_fill_(
        (torch.arange(ctx, device=q.device) >= s["rows"][:, None])[:, None, :, None], 0.0)
    out = (each(torch.matmul(one(old), s["vp"].float())) + torch.matmul(new, v)) / total
    out = out.view(requests, kh, most, g, hd).permute(0, 2, 1, 3, 4).reshape(
        requests, most, kh * g, hd)
    # Back to the tokens' rows.
    i = torch.arange(tokens, device=q.device)
    request = torch.searchsorted(first[1:], i, right=True)
    return out[request, i - first[request]].to(q.dtype)


def _own_axes(s):
    from strasgpt_b200 import runtime
    c, x, y, pos = s["case"], s["x"], s["y"], s["pos"]
    if "params" not in s:
        s["params"] = (runtime.Rope(**s["turn"]),
                       runtime.RopeAxes(s["sections"], order=_ORDERS[c["order"]],
                                        separate=int(c["separate"])))
    rope, axes = s["params"]
    runtime.lib().strasgpt_k_rope_axes(
        x.data_ptr(), x.stride(0), x.stride(1), y.data_ptr(), y.stride(0), y.stride(1),
        _CODES[c["type"]], c["t"], c["heads"], c["head_dim"], pos.data_ptr(), pos.stride(0),
        pos.stride(1), rope, axes, torch.cuda.current_stream().cuda_stream)
    return y


def _own_lora(s):
    from strasgpt_b200 import runtime
    c, x, base, out = s["case"], s["x"], s["base"], s["out"]
    runtime.lib().strasgpt_k_lora(
        x.data_ptr(), x.stride(0), s["a"].data_ptr(), s["b"].data_ptr(), _CODES[c["type"]],
        c["m"], c["k"], c["n"], c["rank"], c["adapters"], s["adapter"].data_ptr(),
        s["scale"].data_ptr(), base.data_ptr(), base.stride(0), out.data_ptr(), out.stride(0),
        _EPILOGUES[c["epilogue"]], torch.cuda.current_stream().cuda_stream)
    return out


def _own_shared(s):
    from strasgpt_b200 import runtime
    c, q, k, att, lib = s["case"], s["q"], s["k"], s["att"], runtime.lib()
    shape = (c["requests"], c["most"], q.shape[0], c["kv_heads"], c["group"], c["head_dim"])
    if "workspace" not in s:
        size = lib.strasgpt_k_attn_shared_workspace(_CODES[c["type"]], *shape)
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    work = s["workspace"]
    lib.strasgpt_k_attn_shared(
        q.data_ptr(), q.stride(0), s["kp"].data_ptr(), s["vp"].data_ptr(), c["prefix"],
        s["prefix"].data_ptr(), k.data_ptr(), s["v"].data_ptr(), k.stride(0), k.shape[2],
        s["rows"].data_ptr(), s["first"].data_ptr(), _CODES[c["type"]], *shape, att.data_ptr(),
        att.stride(0), work.data_ptr(), work.numel(), torch.cuda.current_stream().cuda_stream)
    return att


def run(state):
    op = state["case"]["op"]
    if own:
        if op == "rope_axes":
            return _own_axes(state)
        return _own_lora(state) if op == "lora" else _own_shared(state)
    if op == "rope_axes":
        return _plain_axes(state)
    return _plain_lora(state) if op == "lora" else _plain_shared(state)


# --------------------------------------------------------------------------
# what a pass cannot do without, and its exact value
# --------------------------------------------------------------------------
def work(case):
    c, size = case, _BYTES[case["type"]]
    if c["op"] == "rope_axes":
        sections = [int(s) for s in c["sections"].split()]
        every = c["t"] * c["heads"] * c["head_dim"]
        return {"bytes": 2 * every * size + 4 * c["t"] * len(sections),
                "flops": 6 * c["t"] * c["heads"] * sum(sections)}
    if c["op"] == "lora":
        m, k, n, r = c["m"], c["k"], c["n"], c["rank"]
        met = _token_adapters(c)
        met = met[met >= 0]
        outs = n // 2 if c["epilogue"] == "swiglu" else n
        return {"bytes": m * (k + n + outs) * size + 2 * len(set(met.tolist())) * r * (k + n)
                + 4 * m + 4 * c["adapters"], "flops": 2 * len(met) * r * (k + n)}
    kh, g, hd = c["kv_heads"], c["group"], c["head_dim"]
    new, rows = _counts(c)
    tokens = int(new.sum())
    seen = tokens * c["prefix"] + int((new * (rows - new) + new * (new + 1) // 2).sum())
    return {"bytes": 2 * kh * (c["prefix"] + int(rows.sum())) * hd * size
            + 2 * tokens * kh * g * hd * size + 8 * c["requests"] + 8,
            "flops": 4 * hd * kh * g * seen}


def _exact_axes(s):
    """Pairs as complex numbers, turned by e^(i angle)."""
    c, turn, sections = s["case"], s["turn"], s["sections"]
    dim, half = turn["dim"], turn["dim"] // 2
    x, pos = s["x"].double(), s["pos"].double()
    left, axis, turned = list(sections), -1, []
    for j in range(half):
        # The next axis in turn, or the present one's run, with pairs left.
        if c["order"] == "dealt":
            axis = (axis + 1) % len(sections)
        axis = max(axis, 0)
        while not left[axis]:
            axis = (axis + 1) % len(sections)
        number = sections[axis] - left[axis]
        left[axis] -= 1
        f = turn["theta"] ** (-number / sections[axis] if c["separate"] else -2.0 * j / dim)
        if c["scaling"] == "linear":
            f /= turn["factor"]
        elif c["scaling"] == "bands":
            wave = 2 * math.pi / f
            keep = (turn["original"] / wave - turn["low"]) / (turn["high"] - turn["low"])
            keep = min(1.0, max(0.0, keep))
            f = (1 - keep) * f / turn["factor"] + keep * f
        z = torch.complex(x[..., j], x[..., j + half])
        e = torch.polar(torch.full_like(pos[axis], turn["magnitude"]), pos[axis] * f)
        turned.append((j, z * e[:, None]))
    for j, z in turned:
        x[..., j], x[..., j + half] = z.real, z.imag
    return x


def _exact_lora(s):
    """One adapter's tokens at a time."""
    c, y = s["case"], s["base"].double()
    for d in range(c["adapters"]):
        of = torch.nonzero(s["adapter"] == d)[:, 0]
        if len(of):
            low = s["x"][of].double() @ s["a"][d].double().T
            y[of] += s["scale"][d].double() * (low @ s["b"][d].double().T)
    if c["epilogue"] == "swiglu":
        pair = y.view(c["m"], c["n"] // 2, 2)
        y = pair[..., 0] * torch.sigmoid(pair[..., 0]) * pair[..., 1]
    return y


def _exact_shared(s):
    """One request and kv head at a time, prefix and own rows in one."""
    c, first = s["case"], s["first"].tolist()
    kh, g, hd, q = c["kv_heads"], c["group"], c["head_dim"], s["q"]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for h in range(kh):
        kp, vp = s["kp"][h].double(), s["vp"][h].double()
        for r, n in enumerate(s["rows"].tolist()):
            a, b = first[r], first[r + 1]
            k = torch.cat([kp, s["k"][r, h, :n].double()])
            v = torch.cat([vp, s["v"][r, h, :n].double()])
            row = q[a:b, h * g:(h + 1) * g].double().transpose(0, 1)      # [g][new][hd]
            score = row @ k.T / math.sqrt(hd)
            seen = torch.ones(b - a, len(k), dtype=torch.bool, device=q.device)
            score = score.masked_fill(~seen.tril(len(k) - (b - a)), -math.inf)
            out[a:b, h * g:(h + 1) * g] = (torch.softmax(score, -1) @ v).transpose(0, 1)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rope_axes":
        return _exact_axes(state)
    return _exact_lora(state) if case["op"] == "lora" else _exact_shared(state)
