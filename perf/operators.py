"""The operators of a windowed-attention transformer block, in training and in serving, and the cases they are timed on.

Four operators:

* `window`: causal attention in which a query sees its last `window` positions and the first `sinks`
  tokens of the sequence, key/value heads shared by groups of query heads; forward, or forward and
  backward;
* `paged`: attention of each sequence's newest tokens (one token, or a chunk) over keys and values
  that lie in the pages of a cache, with or without window and sinks;
* `append`: the keys and values of new tokens written into the pages of that cache;
* `norm`: what stands between two blocks of a transformer,
  `y = residual_scale * residual + gate * rms_norm(input) * post_weight` and
  `h = rms_norm(y) * pre_weight`, with rms_norm(x) = x / (sqrt(mean(x^2)) + eps); forward, or forward
  and backward.

`run` computes a case with elementary torch operations in 32 bits, or, where `own` is set, with the
framework's functions; `exact` gives the same values in 64 bits.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# ------------------------------------------------------------------------------------- cases
def _window(name, dtype, B, kv_heads, group, S, D, window, sinks, train):
    case = {"op": "window", "dtype": dtype, "B": B, "kv_heads": kv_heads, "group": group, "S": S, "D": D,
            "window": window, "sinks": sinks, "train": train}
    return dict(case, name=name) if name else case


def _paged(name, dtype, n, kv_heads, group, D, page, context, chunk, window, sinks):
    case = {"op": "paged", "dtype": dtype, "n": n, "kv_heads": kv_heads, "group": group, "D": D, "page": page,
            "context": context, "chunk": chunk, "window": window, "sinks": sinks}
    return dict(case, name=name) if name else case


def _append(name, dtype, n, kv_heads, D, page, context, chunk):
    case = {"op": "append", "dtype": dtype, "n": n, "kv_heads": kv_heads, "D": D, "page": page, "context": context,
            "chunk": chunk}
    return dict(case, name=name) if name else case


def _norm(name, dtype, batch, rows, cols, gate, scale, train):
    case = {"op": "norm", "dtype": dtype, "batch": batch, "rows": rows, "cols": cols, "gate": gate, "scale": scale,
            "train": train}
    return dict(case, name=name) if name else case


def listed():
    return [
        # a short prompt of a small model: latency
        _window("window_fwd_bf16_S200", "bf16", 1, 2, 4, 200, 64, 64, 4, False),
        # a training step at the attention benchmark's heads, length and head size, with a window of 1024
        _window("window_train_bf16_S4096", "bf16", 2, 8, 4, 4096, 128, 1024, 4, True),
        # odd length, window, sink and group sizes, half precision
        _window("window_train_fp16_S1111", "fp16", 3, 2, 3, 1111, 64, 300, 7, True),
        # single precision, no sinks, one key head per query head
        _window("window_train_fp32_S1024", "fp32", 1, 8, 1, 1024, 64, 256, 0, True),
        # a batch of 64 sequences that each add one token, contexts of 512 to 8192
        _paged("paged_decode_bf16_n64", "bf16", 64, 8, 4, 128, 16, 8192, 1, 0, 0),
        # a single user's next token over a short context: latency
        _paged("paged_decode_fp16_n1", "fp16", 1, 4, 2, 64, 32, 700, 1, 0, 0),
        # chunks of up to 512 prompt tokens over long contexts, with the window and sinks of the training step
        _paged("paged_chunk_bf16_n4", "bf16", 4, 8, 4, 128, 64, 16384, 512, 1024, 4),
        # the cache write of the batch of 64 single tokens
        _append("append_decode_bf16_n64", "bf16", 64, 8, 128, 16, 8192, 1),
        # the cache write of 4 prompts of up to 4096 tokens
        _append("append_prompt_bf16_n4", "bf16", 4, 8, 128, 64, 4096, 4096),
        # a training step at the RMSNorm benchmark's size, one gate per feature
        _norm("norm_train_bf16_8192x4096", "bf16", 1, 8192, 4096, "feature", 1.0, True),
        # odd rows and width, one gate vector per sequence, a scaled residual
        _norm("norm_train_fp32_5x333x1021", "fp32", 5, 333, 1021, "sequence", 0.75, True),
        # a batch of 16 new tokens in serving: latency
        _norm("norm_fwd_fp16_16x4096", "fp16", 1, 16, 4096, "feature", 1.0, False),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["window", "window", "paged", "paged", "norm", "norm", "append"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8])
    D = rng.choice([32, 64, 64, 128, 128])
    if op == "window":
        # with one visible key per query the score gradients are zero: training starts above that
        train = rng.random() < 0.6
        S, window = _log(rng, 16 if train else 1, 4096), _log(rng, 4 if train else 1, 2048)
        B = rng.randint(1, 4)
        while B * kv_heads * group * S * S > (2 * 32 if dtype != "fp32" else 8) * 4096 * 4096 // (1 if dtype != "fp32" else 4):
            S = S * 2 // 3
        return _window(None, dtype, B, kv_heads, group, S, D, window, rng.choice([0, 1, 4, 16, _log(rng, 1, 200)]), train)
    if op == "paged":
        n, context = _log(rng, 1, 64), _log(rng, 1, 16384)
        chunk = min(context, rng.choice([1, _log(rng, 1, 512)]))
        most = 1 if dtype != "fp32" else 8
        while n > 1 and (n * kv_heads * group * chunk * context * most > 4 * 32 * 512 * 16384 or n * context * kv_heads * D * most > 64 * 8192 * 8 * 128):
            n = n // 2
        return _paged(None, dtype, n, kv_heads, group, D, rng.choice([8, 16, 24, 32, 64, 128, 256]), context, chunk,
                      rng.choice([0, _log(rng, 1, 4096)]), rng.choice([0, 4, _log(rng, 1, 200)]))
    if op == "append":
        context = _log(rng, 1, 4096)
        return _append(None, dtype, _log(rng, 1, 16), kv_heads, D, rng.choice([8, 16, 24, 32, 64, 128, 256]), context,
                       rng.choice([1, _log(rng, 1, context)]))
    batch = _log(rng, 1, 16)
    cols = 8 * _log(rng, 8, 1024) if rng.random() < 0.7 else _log(rng, 64, 4096)
    rows = max(1, min(_log(rng, 1, 8192), 8192 * 4096 // cols) // batch)
    return _norm(None, dtype, batch, rows, cols, rng.choice(["none", "feature", "sequence", "element"]), rng.choice([1.0, 0.5, 1.25]), rng.random() < 0.6)


def _lengths(case):
    """(new tokens, context length) of every sequence: contexts from 1/16 of the longest up to the longest,
    chunks from half of the longest up to the longest, in an order that is not sorted."""
    n, longest, chunk = case["n"], case["context"], case["chunk"]
    new, context = [], []
    for i in range(n):
        f = 1.0 if n == 1 else ((i * 37) % n) / (n - 1) if math.gcd(37, n) == 1 else i / (n - 1)
        context.append(max(1, round(longest * (1 + 15 * f) / 16)))
        g = 1.0 if n == 1 else (n - 1 - i) / (n - 1)
        new.append(min(context[-1], max(1, round(chunk * (1 + g) / 2))))
    return new, context


# ----------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32)


def prepare(case, seed):
    g, dtype, op = _generator(seed), DTYPES[case["dtype"]], case["op"]
    state = {"case": case}
    if op == "window":
        B, KV, G, S, D = (case[k] for k in ("B", "kv_heads", "group", "S", "D"))
        # queries and the first keys share a direction: the first tokens draw weight, as they do in trained models
        u = _randn(g, D)
        state["q"] = (_randn(g, B, KV * G, S, D) + 0.3 * u).to(dtype)
        k = _randn(g, B, KV, S, D)
        k[:, :, : case["sinks"]] += 0.6 * u
        state["k"] = k.to(dtype)
        state["v"] = _randn(g, B, KV, S, D).to(dtype)
        if case["train"]:
            state["dout"] = _randn(g, B, KV * G, S, D).to(dtype)
            for name in ("q", "k", "v"):
                state[name].requires_grad_(True)
    elif op in ("paged", "append"):
        KV, D, page = case["kv_heads"], case["D"], case["page"]
        new, context = _lengths(case)
        blocks = [-(-length // page) for length in context]
        pages = sum(blocks) + 3
        order = torch.randperm(pages, generator=g, device=DEVICE)
        # every sequence's pages lie anywhere in the pool; unused entries of the table are 0
        row_of = torch.tensor([r for r, b in enumerate(blocks) for _ in range(b)], device=DEVICE)
        col_of = torch.tensor([c for b in blocks for c in range(b)], device=DEVICE)
        table = torch.zeros(len(blocks), max(blocks), dtype=torch.int32, device=DEVICE)
        table[row_of, col_of] = order[: sum(blocks)].to(torch.int32)
        state["table"] = table
        state["context"] = torch.tensor(context, dtype=torch.int32, device=DEVICE)
        starts = [0]
        for t in new:
            starts.append(starts[-1] + t)
        state["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE) if case["chunk"] > 1 else None
        state["tokens"], state["max_new"], state["max_context"] = starts[-1], max(new), max(context)
        state["key_cache"] = _randn(g, pages, page, KV, D).to(dtype)
        state["value_cache"] = _randn(g, pages, page, KV, D).to(dtype)
        if op == "paged":
            state["q"] = _randn(g, starts[-1], KV * case["group"], D).to(dtype)
        else:
            state["k"] = _randn(g, starts[-1], KV, D).to(dtype)
            state["v"] = _randn(g, starts[-1], KV, D).to(dtype)
    else:
        batch, rows, cols = case["batch"], case["rows"], case["cols"]
        state["x"] = (_randn(g, batch, rows, cols) * (0.5 + torch.rand((batch, rows, 1), generator=g, device=DEVICE))).to(dtype)
        state["residual"] = (2 * _randn(g, batch, rows, cols)).to(dtype)
        state["post_weight"] = (1 + 0.1 * _randn(g, cols)).to(dtype)
        state["pre_weight"] = (1 + 0.1 * _randn(g, cols)).to(dtype)
        shape = {"none": None, "feature": (cols,), "sequence": (batch, 1, cols), "element": (batch, rows, cols)}[case["gate"]]
        state["gate"] = None if shape is None else (0.5 + 0.3 * _randn(g, *shape)).to(dtype)
        if case["train"]:
            state["dy"] = _randn(g, batch, rows, cols).to(dtype)
            state["dh"] = _randn(g, batch, rows, cols).to(dtype)
            for name in ("x", "residual", "post_weight", "pre_weight", "gate"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
    return state


# --------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"window": _own_window, "paged": _own_paged, "append": _own_append, "norm": _own_norm}[op](state)
    with torch.no_grad():
        return {"window": _plain_window, "paged": _plain_paged, "append": _plain_append, "norm": _plain_norm}[op](state)


def _own_window(state):
    import trident_b200 as trident

    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    out = trident.function.sliding_window_attention(q, k, v, case["window"], case["sinks"])
    if not case["train"]:
        return {"out": out}
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), state["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


def _own_paged(state):
    import trident_b200 as trident

    case = state["case"]
    return trident.function.paged_attention(
        state["q"], state["key_cache"], state["value_cache"], state["table"], state["context"], state["starts"],
        max_query_length=state["max_new"], max_context_length=state["max_context"],
        window_size=case["window"] or None, num_sinks=case["sinks"] if case["window"] else 0,
    )


def _own_append(state):
    import trident_b200 as trident

    trident.function.paged_cache_append(
        state["k"], state["v"], state["key_cache"], state["value_cache"], state["table"], state["context"], state["starts"],
    )
    return {"key_cache": state["key_cache"], "value_cache": state["value_cache"]}


def _own_norm(state):
    import trident_b200 as trident

    case = state["case"]
    h, y = trident.function.gated_residual_rms_norm(
        state["x"], state["residual"], state["post_weight"], state["pre_weight"], state["gate"], case["scale"], EPS
    )
    if not case["train"]:
        return {"h": h, "y": y}
    names = [n for n in ("x", "residual", "post_weight", "pre_weight", "gate") if state[n] is not None]
    grads = torch.autograd.grad((h, y), [state[n] for n in names], (state["dh"], state["dy"]))
    return {"h": h.detach(), "y": y.detach(), **{"d" + n: d for n, d in zip(names, grads)}}


def _visible(q_pos, k_pos, window, sinks):
    """Whether the query at position q_pos sees the key at position k_pos; window 0: all earlier ones."""
    seen = k_pos <= q_pos
    if window:
        seen = seen & ((q_pos - k_pos < window) | (k_pos < sinks))
    return seen


def _softmax(scores, seen):
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.clamp_min(torch.finfo(scores.dtype).min))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, 1.0)


def _plain_window(state):
    case, dtype = state["case"], state["q"].dtype
    B, KV, G, S, D = (case[k] for k in ("B", "kv_heads", "group", "S", "D"))
    q = state["q"].float().view(B, KV, G * S, D)
    k, v = state["k"].float(), state["v"].float()
    at = torch.arange(S, device=q.device)
    seen = _visible(at[:, None], at[None, :], case["window"], case["sinks"]).repeat(G, 1)
    p = _softmax(q @ k.transpose(-1, -2) * D ** -0.5, seen)
    out = p @ v
    result = {"out": out.view(B, KV * G, S, D).to(dtype)}
    if case["train"]:
        dout = state["dout"].float().view(B, KV, G * S, D)
        result["dv"] = (p.transpose(-1, -2) @ dout).to(dtype)
        ds = dout @ v.transpose(-1, -2)
        ds = ds.sub_((dout * out).sum(-1, keepdim=True)).mul_(p).mul_(D ** -0.5)
        result["dq"] = (ds @ k).view(B, KV * G, S, D).to(dtype)
        result["dk"] = (ds.transpose(-1, -2) @ q).to(dtype)
    return result


def _positions(state):
    """For every new token its sequence, its place among that sequence's new tokens and its position."""
    context = state["context"].long()
    token = torch.arange(state["tokens"], device=context.device)
    starts = torch.arange(len(context) + 1, device=context.device) if state["starts"] is None else state["starts"].long()
    seq = torch.searchsorted(starts, token, right=True) - 1
    place = token - starts[seq]
    return seq, place, context[seq] - (starts[seq + 1] - starts[seq]) + place


def _plain_paged(state):
    case, q, page = state["case"], state["q"], state["case"]["page"]
    n, KV, G, D = (case[k] for k in ("n", "kv_heads", "group", "D"))
    seq, place, position = _positions(state)
    at = torch.arange(state["max_context"], device=q.device)
    pages = state["table"].long()[:, at // page]
    k = state["key_cache"][pages, at % page].float().permute(0, 2, 3, 1)  # [n, KV, D, keys]
    v = state["value_cache"][pages, at % page].float().permute(0, 2, 1, 3)  # [n, KV, keys, D]
    width = state["max_new"]
    padded = torch.zeros(n, width, KV * G, D, device=q.device)
    padded[seq, place] = q.float()
    q_pos = torch.full((n, width), -1, device=q.device)
    q_pos[seq, place] = position
    seen = _visible(q_pos[:, :, None], at, case["window"], case["sinks"])
    rows = padded.view(n, width, KV, G, D).permute(0, 2, 3, 1, 4).reshape(n, KV, G * width, D)
    p = _softmax((rows @ k * D ** -0.5).view(n, KV, G, width, -1), seen[:, None, None])
    out = (p.view(n, KV, G * width, -1) @ v).view(n, KV * G, width, D)
    return out[seq, :, place].to(q.dtype)


def _plain_append(state):
    page = state["case"]["page"]
    seq, _, position = _positions(state)
    at = (state["table"].long()[seq, position // page], position % page)
    state["key_cache"].index_put_(at, state["k"])
    state["value_cache"].index_put_(at, state["v"])
    return {"key_cache": state["key_cache"], "value_cache": state["value_cache"]}


def _rms(x):
    return x.square().mean(-1, keepdim=True).sqrt()


def _rms_norm_gradient(dn, x, rms):
    """Gradient of x / (rms(x) + EPS) given that of its result."""
    along = (dn * x).mean(-1, keepdim=True) / torch.where(rms > 0, rms, 1.0)
    return (dn - x * along / (rms + EPS)) / (rms + EPS)


def _to_shape(t, shape):
    """The sum of t over the dimensions that a tensor of `shape` is broadcast over."""
    t = t.sum(0) if len(shape) < t.dim() and t.shape[0] == 1 else t
    return t.sum_to_size(shape)


def _plain_norm(state):
    case, dtype = state["case"], state["x"].dtype
    x, residual, w1, w2 = (state[n].float() for n in ("x", "residual", "post_weight", "pre_weight"))
    gate = torch.ones((), device=x.device) if state["gate"] is None else state["gate"].float()
    r1 = _rms(x)
    normed = x / (r1 + EPS)
    y = case["scale"] * residual + gate * (normed * w1)
    r2 = _rms(y)
    h = y / (r2 + EPS) * w2
    result = {"h": h.to(dtype), "y": y.to(dtype)}
    if case["train"]:
        dh, dy = state["dh"].float(), state["dy"].float()
        dy = dy + _rms_norm_gradient(dh * w2, y, r2)
        result["dresidual"] = (case["scale"] * dy).to(dtype)
        result["dx"] = _rms_norm_gradient(dy * gate * w1, x, r1).to(dtype)
        result["dpost_weight"] = _to_shape(dy * gate * normed, w1.shape).to(dtype)
        result["dpre_weight"] = _to_shape(dh * (y / (r2 + EPS)), w2.shape).to(dtype)
        if state["gate"] is not None:
            result["dgate"] = _to_shape(dy * normed * w1, gate.shape).to(dtype)
    return result


# ------------------------------------------------------------------------------ work of a pass
def _pairs(first, last, window, sinks):
    """Keys seen by the queries at positions first..last, summed."""
    total = 0
    for i in range(first, last + 1):
        seen = i + 1
        if window and window < seen:
            seen = window + min(sinks, i + 1 - window)
        total += seen
    return total


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "window":
        B, KV, G, S, D = (case[k] for k in ("B", "kv_heads", "group", "S", "D"))
        pairs = B * KV * G * _pairs(0, S - 1, case["window"], case["sinks"])
        q, kv = B * KV * G * S * D, B * KV * S * D
        if case["train"]:  # q, dout, out, dq; k, v, dk, dv; two products forward, five backward
            return {"bytes": size * (4 * q + 4 * kv), "flops": 14 * D * pairs}
        return {"bytes": size * (2 * q + 2 * kv), "flops": 4 * D * pairs}
    if case["op"] in ("paged", "append"):
        new, context = _lengths(case)
        KV, D = case["kv_heads"], case["D"]
        if case["op"] == "append":
            return {"bytes": 4 * size * KV * D * sum(new), "flops": 0}
        H, W, K = KV * case["group"], case["window"], case["sinks"]
        keys = pairs = 0
        for t, c in zip(new, context):
            first = max(0, c - t - W + 1) if W else 0
            keys += c - first + min(first, K if W else 0)
            pairs += H * _pairs(c - t, c - 1, W, K)
        return {"bytes": size * (2 * KV * D * keys + 2 * H * D * sum(new)), "flops": 4 * D * pairs}
    n, cols = case["batch"] * case["rows"] * case["cols"], case["cols"]
    gates = {"none": 0, "feature": cols, "sequence": case["batch"] * cols, "element": n}[case["gate"]]
    if case["train"]:  # x, residual, dy, dh read; y, h, dx, dresidual written; weights and gates and their gradients
        return {"bytes": size * (8 * n + 4 * cols + 2 * gates), "flops": 40 * n}
    return {"bytes": size * (4 * n + 2 * cols + gates), "flops": 10 * n}


# ---------------------------------------------------------------------------- 64-bit values
def _exact_attention(q, k, v, q_pos, window, sinks, scale):
    """[heads, queries, D] of one sequence; q [H, T, D], k and v [KV, L, D], in 64 bits."""
    group = q.shape[0] // k.shape[0]
    k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    j = torch.arange(k.shape[1], device=q.device)
    hidden = j > q_pos[:, None]
    if window:
        hidden = hidden | ((j <= q_pos[:, None] - window) & (j >= sinks))
    scores = torch.einsum("htd,hld->htl", q, k) * scale
    return torch.einsum("htl,hld->htd", torch.softmax(scores.masked_fill(hidden, float("-inf")), -1), v)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "window":
        outs = {"out": [], "dq": [], "dk": [], "dv": []}
        at = torch.arange(case["S"], device=DEVICE)
        for b in range(case["B"]):
            per_kv = {"out": [], "dq": [], "dk": [], "dv": []}
            for h in range(case["kv_heads"]):
                G = case["group"]
                q, k, v = (t.detach().double().requires_grad_(case["train"]) for t in (
                    state["q"][b, h * G:(h + 1) * G], state["k"][b, h:h + 1], state["v"][b, h:h + 1]))
                o = _exact_attention(q, k, v, at, case["window"], case["sinks"], 1 / math.sqrt(case["D"]))
                per_kv["out"].append(o.detach())
                if case["train"]:
                    grads = torch.autograd.grad(o, (q, k, v), state["dout"][b, h * G:(h + 1) * G].double())
                    for name, t in zip(("dq", "dk", "dv"), grads):
                        per_kv[name].append(t)
            for name, t in per_kv.items():
                if t:
                    outs[name].append(torch.cat(t))
        return {name: torch.stack(t) for name, t in outs.items() if t}
    if case["op"] == "paged":
        new, context = _lengths(case)
        out, at = [], 0
        for s, (t, c) in enumerate(zip(new, context)):
            pages = state["table"][s, : -(-c // case["page"])].long()
            k, v = (state[name][pages].flatten(0, 1)[:c].double().transpose(0, 1) for name in ("key_cache", "value_cache"))
            q = state["q"][at:at + t].double().transpose(0, 1)
            o = _exact_attention(q, k, v, torch.arange(c - t, c, device=DEVICE), case["window"], case["sinks"], 1 / math.sqrt(case["D"]))
            out.append(o.transpose(0, 1))
            at += t
        return torch.cat(out)
    if case["op"] == "append":
        new, context = _lengths(case)
        caches, at = {n: state[n].double() for n in ("key_cache", "value_cache")}, 0
        for s, (t, c) in enumerate(zip(new, context)):
            where = torch.arange(c - t, c, device=DEVICE)
            pages = state["table"][s].long()[torch.div(where, case["page"], rounding_mode="floor")]
            caches["key_cache"][pages, where % case["page"]] = state["k"][at:at + t].double()
            caches["value_cache"][pages, where % case["page"]] = state["v"][at:at + t].double()
            at += t
        return caches
    names = [n for n in ("x", "residual", "post_weight", "pre_weight", "gate") if state[n] is not None]
    leaf = {n: state[n].detach().double().requires_grad_(case["train"]) for n in names}

    def unit(t):
        return t / (torch.sqrt((t * t).sum(-1, keepdim=True) / t.shape[-1]) + EPS)

    branch = unit(leaf["x"]) * leaf["post_weight"]
    y = leaf["residual"] * case["scale"] + (branch * leaf["gate"] if "gate" in leaf else branch)
    h = unit(y) * leaf["pre_weight"]
    result = {"h": h.detach(), "y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad((h, y), [leaf[n] for n in names], (state["dh"].double(), state["dy"].double()))
        result.update({"d" + n: t for n, t in zip(names, grads)})
    return result
