"""Window attention in 64 bits, with a bound on the error of a kernel that computes it.

Roundings. u is half a step of the operands' type (`torch.finfo(t).eps / 2`), e = 2^-24 that of fp32.

* A score is a sum of D products in fp32, scaled: off by at most (D + 8) e times its terms' magnitudes;
  the exponent adds a few e of its own value. `ds` bounds both, for a row's largest.
* A probability p is off by the factor 1 +- (2 ds + c e) (the row's sum carries the same), and, where the
  product with the values runs on 16-bit operands, by its rounding u. c = 64 covers the exponential (2^-22),
  the sums' order and the divisions.
* The output is sum p v: the same factors times sum p |v|, and its own rounding u.
* dv = sum p do likewise; the score gradient g = p (do . v - delta) has in addition the errors of do . v
  (D e of its terms) and of delta = do . out (u of out's rounding, and out's own error), and, as a 16-bit
  operand, its rounding u, taken from a p that may have been rounded: 2 u. dq, dk: sums of g with k, q.
* fp16 probabilities and score gradients below 2^-14 are rounded to multiples of 2^-24: half of that for
  each visible key (values are relative to the row's maximum, which is at least 1 before division).
"""

import torch

E = 2.0 ** -24
C = 64.0


def visible(q_pos, n_keys, window, sinks):
    j = torch.arange(n_keys, device=q_pos.device)
    i = q_pos[:, None]
    seen = j <= i
    if window:
        seen = seen & ((i - j < window) | (j < sinks))
    return seen


def attention(q, k, v, q_pos, window, sinks, scale, dtype, dout=None):
    """One key head: q [G, T, D], k, v [L, D] in 64 bits, query positions q_pos [T]. Returns
    {name: (value, bound)}; rows without keys give zeros."""
    u = torch.finfo(dtype).eps / 2
    up = 0.0 if dtype == torch.float32 else u
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    G, T, D = q.shape
    if k.shape[0] == 0:  # no keys at all
        return {"out": (torch.zeros_like(q), torch.zeros_like(q))}
    seen = visible(q_pos, k.shape[0], window, sinks)
    s = (q @ k.T) * scale
    s_mag = (q.abs() @ k.abs().T) * abs(scale)
    s = s.masked_fill(~seen, float("-inf"))
    some = seen.any(-1)
    p = torch.where(some[:, None], torch.softmax(torch.where(some[:, None], s, 0.0), -1), 0.0)
    ds = ((D + 8) * E * s_mag + 4 * E * s_mag).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    f = 3 * ds + C * E  # relative error of a probability in fp32
    keys = seen.sum(-1, keepdim=True)
    v_max = v.abs().amax() if v.numel() else torch.zeros((), dtype=torch.float64)
    out = p @ v
    pv = p @ v.abs()
    out_err = (up + f) * pv + tiny * keys * v_max
    result = {"out": (out, out_err + u * (out.abs() + out_err) + tiny)}
    if dout is None:
        return result
    dv = torch.einsum("gtl,gtd->ld", p, dout)
    dv_err = torch.einsum("gtl,gtd->ld", (up + f) * p + tiny, dout.abs() * some[:, None])
    result["dv"] = (dv, dv_err + u * (dv.abs() + dv_err) + tiny)
    dp, dp_mag = dout @ v.T, dout.abs() @ v.abs().T
    delta = (dout * out).sum(-1, keepdim=True)
    delta_err = (dout.abs() * (out_err + u * out.abs())).sum(-1, keepdim=True) + (D + 8) * E * (dout * out).abs().sum(-1, keepdim=True)
    g = p * (dp - delta)
    g_err = (2 * up + f) * g.abs() + (1 + up) * p * ((D + 8) * E * dp_mag + delta_err) + C * E * p * (dp.abs() + delta.abs())
    if tiny:
        g_err = g_err + tiny * (1 + (dp - delta).abs()) * seen
    # (the sums over keys and queries in fp32 are within c e of their terms' magnitudes)
    g_sum = g_err + C * E * g.abs()
    dq, dq_err = (g @ k) * scale, (g_sum @ k.abs()) * abs(scale)
    dk, dk_err = torch.einsum("gtl,gtd->ld", g, q) * scale, torch.einsum("gtl,gtd->ld", g_sum, q.abs()) * abs(scale)
    result["dq"] = (dq, dq_err + u * (dq.abs() + dq_err) + tiny)
    result["dk"] = (dk, dk_err + u * (dk.abs() + dk_err) + tiny)
    return result


def batched(q, k, v, window, sinks, scale, dtype, dout=None):
    """The training form: q [B, H, S, D], k, v [B, KV, S, D]; values and bounds in the same shapes."""
    B, H, S, D = q.shape
    KV = k.shape[1]
    G = H // KV
    parts = {}
    at = torch.arange(S)
    for b in range(B):
        for h in range(KV):
            heads = slice(h * G, (h + 1) * G)
            one = attention(q[b, heads].double(), k[b, h].double(), v[b, h].double(), at, window, sinks, scale, dtype,
                            None if dout is None else dout[b, heads].double())
            for name, pair in one.items():
                parts.setdefault(name, []).append(pair)
    shapes = {"out": (B, H, S, D), "dq": (B, H, S, D), "dk": (B, KV, S, D), "dv": (B, KV, S, D)}
    return {n: tuple(torch.stack([p[i] for p in pairs]).reshape(shapes[n]) for i in range(2)) for n, pairs in parts.items()}


def check(got, want, what):
    value, bound = (t.cpu() for t in want)
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    excess = ((got - value).abs() - bound).max().item()
    assert excess <= 0, f"{what}: {excess:.3e} beyond the bound (largest error {(got - value).abs().max():.3e})"
