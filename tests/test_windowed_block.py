"""A transformer's blocks built from the windowed operators, as they are used together: trained on whole
sequences, and served from a paged cache, prompt in chunks and then token by token.

Tolerance. The blocks run in fp32 and are compared with the same formulas in 64 bits. Each of the at most
eight operators that a value passes through adds an error below 2^-16 of its terms' magnitudes (bounds in the
operators' own tests: C = 256 roundings of 2^-24), and the next ones pass it on with a condition below 32 here
(scores below 10, norms of vectors far from zero): 8 * 32 * 2^-16 = 4e-3 of the largest value of a tensor.
The operators' mistakes (a wrong key, head, row or gate) show as errors of the order of the value itself.
"""

import pytest
import torch

import trident_b200 as trident
from tests import local_reference as ref
from tests import util

HEADS, KV, SIZE, WINDOW, SINKS, SCALE, EPS, LAYERS = 4, 2, 32, 20, 3, 0.8, 1e-6, 2
WIDTH = HEADS * SIZE


def _weights(seed=0):
    make = lambda i, *shape, std=1.0, mean=0.0: util.randn(*shape, seed=seed + i, std=std, mean=mean)  # noqa: E731
    return [
        {
            "qkv": make(10 * layer, (HEADS + 2 * KV) * SIZE, WIDTH, std=WIDTH ** -0.5),
            "out": make(10 * layer + 1, WIDTH, WIDTH, std=WIDTH ** -0.5),
            "post": make(10 * layer + 2, WIDTH, std=0.1, mean=1.0),
            "pre": make(10 * layer + 3, WIDTH, std=0.1, mean=1.0),
            "gate": make(10 * layer + 4, WIDTH, std=0.3, mean=0.5),
        }
        for layer in range(LAYERS)
    ]


def _blocks(x, weights, attention, norm):
    """`attention(layer, q, k, v)` over [..., tokens, heads, size]."""
    residual, h = x, x
    for layer, w in enumerate(weights):
        qkv = (h @ w["qkv"].t()).unflatten(-1, (HEADS + 2 * KV, SIZE))
        a = attention(layer, *qkv.split([HEADS, KV, KV], -2))
        h, residual = norm(a.flatten(-2) @ w["out"].t(), residual, w["post"], w["pre"], w["gate"], SCALE, EPS)
    return h, residual


def _plain_attention(layer, q, k, v):
    q, k, v = (t.transpose(-2, -3) for t in (q, k, v))
    k, v = (t.repeat_interleave(HEADS // KV, -3) for t in (k, v))
    seen = ref.visible(torch.arange(q.shape[-2]), q.shape[-2], WINDOW, SINKS)
    s = (q @ k.transpose(-1, -2) * SIZE ** -0.5).masked_fill(~seen, float("-inf"))
    return (torch.softmax(s, -1) @ v).transpose(-2, -3)


def _plain_norm(x, residual, post, pre, gate, scale, eps):
    rms = lambda t, w: t * w / (t.square().mean(-1, keepdim=True).sqrt() + eps)  # noqa: E731
    y = scale * residual + gate * rms(x, post)
    return rms(y, pre), y


def _close(got, want, what):
    error = (got.detach().double().cpu() - want.detach()).abs().max().item()
    assert error <= 4e-3 * want.abs().max().item(), f"{what}: {error:.3e} of {want.abs().max().item():.3e}"


@pytest.mark.gpu
def test_training(device):
    x, target = util.randn(2, 75, WIDTH, seed=100), util.randn(2, 75, WIDTH, seed=101)
    weights = _weights()

    def window(layer, q, k, v):
        return trident.function.sliding_window_attention(
            *(t.transpose(-2, -3) for t in (q, k, v)), WINDOW, SINKS
        ).transpose(-2, -3)

    def run(kind, dev, attention, norm):
        leaves = [{n: t.to(dev, kind).requires_grad_(True) for n, t in w.items()} for w in weights]
        h, residual = _blocks(x.to(dev, kind), leaves, attention, norm)
        loss = (h * target.to(dev, kind)).sum() + residual.square().sum()
        loss.backward()
        return loss, leaves

    got_loss, got = run(torch.float32, device, window, trident.function.gated_residual_rms_norm)
    want_loss, want = run(torch.float64, "cpu", _plain_attention, _plain_norm)
    _close(got_loss, want_loss, "loss")
    for layer in range(LAYERS):
        for name in want[layer]:
            _close(got[layer][name].grad, want[layer][name].grad, f"{name} of layer {layer}")


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [1, 7, 16, 50])
def test_serving(chunk, device):
    """Two sequences of different lengths: prompts in chunks, then single tokens, against the whole sequences."""
    page, lengths, prompts = 8, [61, 45], [50, 33]
    weights = _weights()
    sequences = [util.randn(n, WIDTH, seed=110 + i) for i, n in enumerate(lengths)]
    on_device = [{n: t.to(device) for n, t in w.items()} for w in weights]
    blocks = -(-max(lengths) // page)
    table = torch.randperm(2 * blocks, generator=util.seeded(112)).view(2, blocks).to(torch.int32).to(device)
    caches = [[torch.full((2 * blocks, page, KV, SIZE), float("nan"), device=device) for _ in range(2)] for _ in weights]
    done, rows = [0, 0], [[], []]
    while done != lengths:
        new = [min(chunk, p - d) if d < p else min(1, n - d) for d, p, n in zip(done, prompts, lengths)]
        context = torch.tensor([d + t for d, t in zip(done, new)], dtype=torch.int32, device=device)
        offsets = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=device)
        x = torch.cat([s[d:d + t] for s, d, t in zip(sequences, done, new)]).to(device)

        def paged(layer, q, k, v):
            place = (*caches[layer], table, context, offsets)
            trident.function.paged_cache_append(k, v, *place)
            return trident.function.paged_attention(q, *place, max(new), max(lengths), WINDOW, SINKS)

        h, _ = _blocks(x, on_device, paged, trident.function.gated_residual_rms_norm)
        for s, part in enumerate(h.split(new)):
            rows[s].append(part)
        done = [d + t for d, t in zip(done, new)]
    for s, x in enumerate(sequences):
        want, _ = _blocks(x.double(), [{n: t.double() for n, t in w.items()} for w in weights], _plain_attention, _plain_norm)
        _close(torch.cat(rows[s]), want, f"sequence {s}")


@pytest.mark.gpu
def test_on_a_second_device(device):
    """Tensors of another device than the current one; refused when they are on two."""
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two visible GPUs")
    q, k = (util.randn(1, h, 60, 64, seed=120 + h).to(torch.bfloat16) for h in (4, 2))
    here = trident.function.sliding_window_attention(*(t.to("cuda:0") for t in (q, k, k)), 20, 2)
    there = trident.function.sliding_window_attention(*(t.to("cuda:1") for t in (q, k, k)), 20, 2)
    assert there.device.index == 1 and torch.equal(here.cpu(), there.cpu())
    with pytest.raises(ValueError, match="device"):
        trident.function.sliding_window_attention(q.to("cuda:0"), k.to("cuda:1"), k.to("cuda:1"), 20, 2)


@pytest.mark.gpu
def test_without_gradients_nothing_is_kept_and_nothing_changes(device, dtype):
    """Calls that autograd does not record keep no statistics and give the same bits."""
    q, k, v = (util.randn(2, h, 90, 64, seed=130 + h).to(dtype).to(device) for h in (4, 2, 2))
    for D in (64, 32):
        plain = trident.function.sliding_window_attention(*(t[..., :D] for t in (q, k, v)), 30, 2)
        recorded = trident.function.sliding_window_attention(q[..., :D].detach().requires_grad_(True), k[..., :D], v[..., :D], 30, 2)
        assert recorded.requires_grad and not plain.requires_grad and torch.equal(plain, recorded)
    for cols in (64, 63, 4500, 9001):
        x, r, w = (util.randn(*s, seed=140 + i).to(dtype).to(device) for i, s in enumerate(((7, cols), (7, cols), (cols,))))
        plain = trident.function.gated_residual_rms_norm(x, r, w, w, w, 0.5, EPS)
        recorded = trident.function.gated_residual_rms_norm(x.clone().requires_grad_(True), r, w, w, w, 0.5, EPS)
        assert all(torch.equal(a, b) for a, b in zip(plain, recorded))
