"""Window attention with sinks against its formula in 64 bits, forward and backward."""

import pytest
import torch

import trident_b200 as trident
from tests import local_reference as ref
from tests import util
from trident_b200 import _lib

F = trident.function.sliding_window_attention


def _problem(B, KV, G, S, D, dtype, seed=0, q_std=1.0):
    q, dout = (util.randn(B, KV * G, S, D, seed=seed + i, std=s).to(dtype) for i, s in ((0, q_std), (1, 1.0)))
    k, v = (util.randn(B, KV, S, D, seed=seed + 2 + i).to(dtype) for i in range(2))
    return q, k, v, dout


def _run(problem, window, sinks, device, scale=None):
    q, k, v = (t.to(device).requires_grad_(True) for t in problem[:3])
    out = F(q, k, v, window, sinks, scale)
    out.backward(problem[3].to(device))
    return {"out": out, "dq": q.grad, "dk": k.grad, "dv": v.grad}


def _compare(problem, window, sinks, device, scale=None):
    q, k, v, dout = problem
    want = ref.batched(q, k, v, window, sinks, q.shape[-1] ** -0.5 if scale is None else scale, q.dtype, dout)
    got = _run(problem, window, sinks, device, scale)
    for name in ("out", "dv", "dq", "dk"):
        ref.check(got[name], want[name], name)
    assert _lib.device_status() == 0


# ------------------------------------------------------------------------------------ no GPU
def test_the_reference_agrees_with_autograd():
    q, k, v, dout = (t.double() for t in _problem(1, 2, 3, 23, 16, torch.float64))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    seen = ref.visible(torch.arange(23), 23, 5, 2)
    s = leaves[0] @ leaves[1].repeat_interleave(3, 1).transpose(-1, -2) * 0.25
    out = torch.softmax(s.masked_fill(~seen, float("-inf")), -1) @ leaves[2].repeat_interleave(3, 1)
    grads = torch.autograd.grad(out, leaves, dout)
    want = ref.batched(q, k, v, 5, 2, 0.25, torch.float32, dout)
    for name, value in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert torch.allclose(want[name][0], value, rtol=1e-10, atol=1e-12), name


def test_refusals():
    q, k = torch.randn(1, 4, 8, 16), torch.randn(1, 2, 8, 16)
    for args, match in (
        ((q[0], k, k, 4), "dimension"),
        ((q, k, k[:, :1], 4), "key and value"),
        ((q, k[:, :, :4], k[:, :, :4], 4), "same batch, length"),
        ((q[:, :3], k, k, 4), "multiple"),
        ((q[:, :0], k, k, 4), "1 to 64"),
        ((q, k[:, :0], k[:, :0], 4), "multiple"),
        ((q[..., :12], k[..., :12], k[..., :12], 4), "head size"),
        ((q, k, k, 0), "window_size"),
        ((q, k, k, 2.0), "window_size"),
        ((q, k, k, True), "window_size"),
        ((q, k, k, 4, -1), "num_sinks"),
        ((q, k.half(), k.half(), 4), "same dtype"),
        ((q.double(), k.double(), k.double(), 4), "Unable to convert"),
        ((torch.randn(1, 65, 2, 16), k[:, :1, :2], k[:, :1, :2], 4), "1 to 64"),
    ):
        with pytest.raises(ValueError, match=match):
            F(*args)
    with pytest.raises(_lib.Tb200Error, match="CUDA tensors only"):
        F(q, k, k, 4)


def test_library_refuses_before_launch():
    import ctypes

    lib = _lib.load()
    s = (ctypes.c_int64 * 4)(1, 1, 1, 1)
    call = lambda *a: lib.tb200_window_attention_fwd(*a)  # noqa: E731
    assert call(None, None, None, None, None, 1, 1, 1, 8, 16, s, s, s, s, 4, 0, 1.0, 0, None) == -1
    assert call(8, 8, 8, 8, 8, 1, 3, 2, 8, 16, s, s, s, s, 4, 0, 1.0, 0, None) == -1
    assert call(8, 8, 8, 8, 8, 1, 2, 2, 8, 24, s, s, s, s, 4, 0, 1.0, 0, None) == -2
    assert call(8, 8, 8, 8, 8, 1, 2, 2, 8, 16, s, s, s, s, 0, 0, 1.0, 0, None) == -1
    assert call(8, 8, 8, 8, 8, 1, 2, 2, 8, 16, s, s, s, None, 4, 0, 1.0, 0, None) == -1


# ------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize(
    "S, window, sinks", [(1, 1, 0), (2, 1, 1), (65, 16, 3), (130, 500, 0), (300, 100, 70), (257, 1, 0), (400, 129, 1)]
)
def test_lengths(S, window, sinks, D, dtype, device):
    _compare(_problem(1, 2, 2, S, D, dtype), window, sinks, device)


@pytest.mark.gpu
@pytest.mark.parametrize("B, KV, G", [(1, 1, 1), (3, 1, 3), (2, 3, 5), (1, 1, 8), (1, 2, 16), (1, 1, 7), (1, 1, 64), (1, 1, 33)])
@pytest.mark.parametrize("D", [64, 128])
def test_head_groups(B, KV, G, D, device, dtype):
    _compare(_problem(B, KV, G, 150, D, dtype, seed=10), 40, 2, device)


@pytest.mark.gpu
@pytest.mark.parametrize("S, window, sinks", [(1000, 200, 4), (1000, 64, 200), (640, 640, 5), (777, 128, 128), (513, 255, 0), (900, 1000, 0)])
@pytest.mark.parametrize("D", [64, 128])
def test_many_tiles(S, window, sinks, D, dtype, device):
    _compare(_problem(1, 1, 2, S, D, dtype, seed=20), window, sinks, device)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_large_scores(D, device, dtype):
    """Scores of hundreds: one key takes almost all the weight, the running maximum moves by large steps."""
    _compare(_problem(1, 1, 2, 400, D, dtype, seed=30, q_std=25.0), 150, 3, device)


@pytest.mark.gpu
def test_scale_is_taken(device):
    _compare(_problem(1, 1, 2, 100, 64, torch.bfloat16, seed=40), 30, 1, device, scale=0.5)
    _compare(_problem(1, 1, 2, 100, 64, torch.bfloat16, seed=40), 30, 1, device, scale=-0.25)
    _compare(_problem(1, 1, 2, 100, 64, torch.float32, seed=40), 30, 1, device, scale=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_strides(D, device, dtype):
    """[batch, length, heads, size] projections, one joint projection, odd offsets, expanded gradients."""
    q, k, v, dout = _problem(2, 2, 2, 140, D, dtype, seed=50)
    want = ref.batched(q, k, v, 50, 3, D ** -0.5, dtype, dout)
    names = ("out", "dq", "dk", "dv")

    def run(q, k, v, dout):
        q, k, v = (t.requires_grad_(True) for t in (q, k, v))
        out = F(q, k, v, 50, 3)
        return dict(zip(names, (out, *torch.autograd.grad(out, (q, k, v), dout))))

    swapped = [t.to(device).transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, dout)]
    got = run(*swapped)
    assert got["out"].stride() == swapped[0].stride()  # laid out as the query is
    joint = torch.cat([t.to(device).transpose(1, 2) for t in (q, k, v)], 2)
    slices = [joint[:, :, a:b].transpose(1, 2) for a, b in ((0, 4), (4, 6), (6, 8))]
    got_joint = run(*slices, dout.to(device))

    def off(t):
        base = torch.empty(t.numel() + 1, dtype=dtype, device=device)[1:]
        return base.view(t.shape).copy_(t)

    got_off = run(*(off(t) for t in (q, k, v, dout)))
    wide = [torch.stack([t, t + 1], -1).to(device)[..., 0] for t in (q, k, v, dout)]  # feature stride 2
    got_wide = run(*wide)
    for g in (got, got_joint, got_off, got_wide):
        for name in names:
            ref.check(g[name], want[name], name)
    one = torch.ones_like(dout)
    want = ref.batched(q, k, v, 50, 3, D ** -0.5, dtype, one)
    got = run(*(t.to(device) for t in (q, k, v)), torch.ones((), dtype=dtype, device=device).expand(one.shape))
    for name in names:
        ref.check(got[name], want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
def test_same_bits_every_time_and_on_another_stream(D, device, dtype):
    problem = _problem(2, 2, 3, 700, D, dtype, seed=60)
    first = _run(problem, 130, 4, device)
    for _ in range(3):
        again = _run(problem, 130, 4, device)
        assert all(torch.equal(first[n], again[n]) for n in first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = _run(problem, 130, 4, device)
    stream.synchronize()
    assert all(torch.equal(first[n], again[n]) for n in first)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_whole_window_is_causal_attention(D, device):
    """With a window as long as the sequence the result is that of the dense causal attention."""
    dt = torch.bfloat16
    q, k, v, _ = _problem(1, 4, 1, 512, D, dt, seed=70)
    dense = trident.function.scaled_dot_product_attention(*(t.to(device) for t in (q, k, v)), is_causal=True)
    want = ref.batched(q, k, v, 512, 0, D ** -0.5, dt)["out"]
    ref.check(dense, want, "dense")
    ref.check(F(*(t.to(device) for t in (q, k, v)), 512), want, "window")
    assert torch.equal(F(*(t.to(device) for t in (q, k, v)), 512), F(*(t.to(device) for t in (q, k, v)), 10 ** 30, 10 ** 30))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_a_window_forgets(D, device, dtype):
    """What lies outside window and sinks has no influence, to the last bit."""
    q, k, v, _ = (t.to(device) for t in _problem(1, 1, 2, 600, D, dtype, seed=80))
    before = F(q, k, v, 100, 4)
    k2, v2 = k.clone(), v.clone()
    k2[:, :, 4:300], v2[:, :, 4:300] = 7.0, -3.0
    after = F(q, k2, v2, 100, 4)
    assert torch.equal(before[:, :, 400:], after[:, :, 400:])
    assert not torch.equal(before[:, :, 300:399], after[:, :, 300:399])


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_guarded_buffers(D, device, dtype):
    """Nothing is written outside the outputs: the library is called on slices of one poisoned buffer."""
    B, KV, G, S = 1, 2, 3, 131
    q, k, v, dout = (t.to(device) for t in _problem(B, KV, G, S, D, dtype, seed=90))
    pad = 4096

    def guarded(t, dt=None):
        dt = t.dtype if dt is None else dt
        buf = torch.full((t.numel() + 2 * pad,), 123.0, dtype=dt, device=device)
        return buf, buf[pad:-pad].view(t.shape)

    bufs, views = zip(*(guarded(t, dt) for t, dt in ((q, None), (q[..., 0], torch.float32), (q, None), (k, None), (v, None))))
    out, lse, dq, dk, dv = views
    _lib.window_attention_fwd(out, lse, q, k, v, 40, 3, D ** -0.5)
    size = _lib.window_attention_bwd_workspace(q, k, 40, 3)
    ws = torch.full((size + 2 * pad,), 77, dtype=torch.uint8, device=device)
    _lib.window_attention_bwd(dq, dk, dv, dout, q, k, v, out, lse, ws[pad:-pad], 40, 3, D ** -0.5)
    torch.cuda.synchronize()
    for buf in bufs:
        assert torch.all(buf[:pad] == 123.0) and torch.all(buf[-pad:] == 123.0)
    assert torch.all(ws[:pad] == 77) and torch.all(ws[-pad:] == 77)
    want = ref.batched(*(t.cpu() for t in (q, k, v)), 40, 3, D ** -0.5, dtype, dout.cpu())
    for name, got in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        ref.check(got, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_captured_step(dt, device):
    """Forward and backward captured into a CUDA graph, replayed on new values."""
    problem = [t.to(device) for t in _problem(1, 2, 2, 300, 64, dt, seed=100)]
    leaves = [t.clone().requires_grad_(True) for t in problem[:3]]

    def step():
        out = F(*leaves, 90, 2)
        return (out, *torch.autograd.grad(out, leaves, problem[3]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    fresh = _problem(1, 2, 2, 300, 64, dt, seed=110)
    with torch.no_grad():
        for dst, src in zip(leaves + [problem[3]], fresh):
            dst.copy_(src)
    graph.replay()
    torch.cuda.synchronize()
    want = ref.batched(*fresh[:3], 90, 2, 0.125, dt, fresh[3])
    for name, got in zip(("out", "dq", "dk", "dv"), outs):
        ref.check(got, want[name], name)


@pytest.mark.gpu
def test_gradients_against_differences(device):
    q, k, v, dout = (t.to(device) for t in _problem(1, 1, 2, 40, 16, torch.float32, seed=120))
    grads = _run((q, k, v, dout), 9, 2, device)
    step = 2.0 ** -6
    for i, name in enumerate(("dq", "dk", "dv")):
        direction = util.randn(*(q, k, v)[i].shape, seed=130 + i, device=device)
        up, down = [q, k, v], [q, k, v]
        up[i], down[i] = up[i] + step * direction, down[i] - step * direction
        slope = ((F(*up, 9, 2) - F(*down, 9, 2)).double() * dout.double()).sum() / (2 * step)
        want = (grads[name].double() * direction.double()).sum()
        # third-order term of the difference (step^2 = 2.4e-4 of the terms) and fp32 noise
        assert abs(slope - want) <= 5e-3 * (grads[name].double() * direction.double()).abs().sum(), name


@pytest.mark.gpu
def test_empty(device):
    q, k = torch.empty(2, 4, 0, 64, device=device, requires_grad=True), torch.empty(2, 2, 0, 64, device=device)
    out = F(q, k, k, 5, 1)
    out.sum().backward()
    assert out.shape == q.shape and q.grad.shape == q.shape
    assert F(torch.empty(0, 4, 7, 64, device=device), torch.empty(0, 2, 7, 64, device=device), torch.empty(0, 2, 7, 64, device=device), 5).shape == (0, 4, 7, 64)


@pytest.mark.gpu
def test_module(device, dtype):
    m = trident.SlidingWindowAttention(16, 2)
    q, k, v, dout = (t.to(device) for t in _problem(1, 2, 2, 50, 64, dtype, seed=140))
    assert torch.equal(m(q, k, v), F(q, k, v, 16, 2))
    assert "backend=Trident" in repr(m)


@pytest.mark.gpu
@pytest.mark.parametrize("B, KV, G, S, window, sinks", [(7, 5, 2, 400, 90, 3), (40, 4, 4, 65, 20, 0), (3, 2, 1, 1300, 300, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_many_tiles_per_sm(B, KV, G, S, window, sinks, D, dtype, device):
    """Several times more tiles than SMs, walks of unequal lengths."""
    _compare(_problem(B, KV, G, S, D, dtype, seed=150), window, sinks, device)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_heads_and_batches_that_share_keys(D, dtype, device):
    """Keys expanded over the batch, values over the heads: their gradients are sums over what shares them."""
    q, k, v, dout = _problem(3, 2, 2, 90, D, dtype, seed=160)
    k, v = k[:1], v[:, :1]
    want = ref.batched(q, k.expand(3, -1, -1, -1), v.expand(-1, 2, -1, -1), 30, 2, D ** -0.5, dtype, dout)
    leaves = [t.to(device).requires_grad_(True) for t in (q, k, v)]
    out = F(leaves[0], leaves[1].expand(3, -1, -1, -1), leaves[2].expand(-1, 2, -1, -1), 30, 2)
    dq, dk, dv = torch.autograd.grad(out, leaves, dout.to(device))
    ref.check(out, want["out"], "out")
    ref.check(dq, want["dq"], "dq")
    # the sum of the parts' bounds, and the roundings of the parts' sum (at most three, in the operands' type)
    u = torch.finfo(dtype).eps / 2
    for name, got, dim in (("dk", dk, 0), ("dv", dv, 1)):
        value, bound = (t.sum(dim, keepdim=True) for t in want[name])
        ref.check(got, (value, bound + 3 * u * (want[name][0].abs().sum(dim, keepdim=True) + bound)), name)


@pytest.mark.gpu
@pytest.mark.parametrize("needs", [(True, False, False), (False, True, False), (False, False, True)])
def test_only_one_needs_a_gradient(needs, device):
    problem = _problem(1, 2, 2, 100, 64, torch.bfloat16, seed=170)
    full = _run(problem, 40, 2, device)
    leaves = [t.to(device).requires_grad_(n) for t, n in zip(problem[:3], needs)]
    out = F(*leaves, 40, 2)
    out.backward(problem[3].to(device))
    assert torch.equal(out, full["out"])
    for leaf, name, need in zip(leaves, ("dq", "dk", "dv"), needs):
        assert torch.equal(leaf.grad, full[name]) if need else leaf.grad is None


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_more_than_32_bit_offsets(D, device):
    """The last rows of a sequence whose queries are more than 2^31 elements: they see the last keys and the sinks."""
    G, window, sinks, tail = 64, 60, 3, 40
    S = 2 ** 31 // (G * D) + 77
    dt = torch.bfloat16
    generator = torch.Generator(device=device).manual_seed(180)
    q, dout = (torch.randn(1, S, G, D, dtype=dt, device=device, generator=generator).transpose(1, 2) for _ in range(2))
    k, v = (torch.randn(1, 1, S, D, dtype=dt, device=device, generator=generator) for _ in range(2))
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    out = F(q, k, v, window, sinks)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    # tokens that the last ones (and their keys' other queries) see, sinks first, at positions that keep who sees whom
    near = tail + 2 * window
    keep = torch.cat([torch.arange(sinks), torch.arange(S - near, S)])
    cut = [t.detach()[:, :, keep.to(device)].cpu() for t in (q, k, v, dout)]
    want = ref.batched(*cut[:3], window, sinks, D ** -0.5, dt, cut[3])
    for name, got in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        value, bound = (t[:, :, -tail:] for t in want[name])
        ref.check(got.detach()[:, :, -tail:], (value, bound), name)


@pytest.mark.gpu
@pytest.mark.parametrize("B, KV, G, S, window, sinks", [(12, 2, 64, 988, 116, 55), (40, 3, 33, 200, 1, 0), (30, 1, 64, 600, 20, 4)])
@pytest.mark.parametrize("D", [64, 128])
def test_many_short_walks(B, KV, G, S, window, sinks, D, device):
    """Tiles of two or three tokens, dozens of them one after the other on every SM (the formula on the device, in
    64 bits too)."""
    dt = torch.bfloat16
    q, k, v, _ = (t.to(device) for t in _problem(B, KV, G, S, D, dt, seed=190))
    out = F(q, k, v, window, sinks)
    assert _lib.device_status() == 0
    at = torch.arange(S, device=device)
    for b in range(B):
        for h in range(KV):
            heads = slice(h * G, (h + 1) * G)
            want = ref.attention(q[b, heads].double(), k[b, h].double(), v[b, h].double(), at, window, sinks, D ** -0.5, dt)["out"]
            ref.check(out[b, heads], want, f"sequence {b}, key head {h}")


def test_workspace_of_many_sinks():
    """The parts of the sinks' gradients: at most eight far pieces an SM in all, or one of each tile, and its window part."""
    bytes_of = _lib.load().tb200_window_attention_bwd_workspace
    for B, H, KV, S, D, window, sinks in ((1, 32, 8, 65536, 128, 1024, 8192), (4, 8, 8, 100000, 64, 128, 50000), (1, 8, 1, 65536, 128, 1024, 4)):
        tiles = B * KV * -(-sinks // 64)  # (of the CUDA-core kernels; those of the tensor cores are twice as long)
        rows = 2 * B * KV * -(-S // (96 // (H // KV))) * 96 * 4 + 256
        assert bytes_of(B, H, KV, S, D, window, sinks, 2) <= rows + (8 * 148 + 2 * tiles) * 2 * 128 * D * 4
    assert bytes_of(1, 32, 8, 65536, 128, 1024, 8192, 2) < 600e6  # (dk and dv are 270 MB)


@pytest.mark.gpu
@pytest.mark.parametrize("dt, D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)], ids=["bf16", "fp16", "fp32"])
def test_many_sinks(dt, D, device):
    """More tiles with sinks than the far pieces are cut for."""
    _compare(_problem(8, 4, 1, 1600, D, dt, seed=80), 60, 1100, device)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [16, 64])
def test_error_of_long_sums(D, device):
    """dq of the last tokens where the score gradients of the first half of the keys have one sign and those of the
    second half the other: the partial sums rise to P and fall. As in the test of paged attention, a sum per 64 keys is
    off by about sqrt(n / 64) e / 3 of P, one running sum by sqrt(n) e / 3. The weights are exp(-log n), the same for
    all keys: their error, 20 e with the sums' last roundings, is doubled for the two halves."""
    n, last = 2 ** 16, 64
    sign = torch.where(torch.arange(n) < n // 2, 1.0, -1.0)
    k = util.randn(n, D, seed=90) + 6.0
    v = sign[:, None] * (1.0 + 0.1 * util.randn(n, D, seed=91).abs())
    dout = torch.zeros(n, D)
    dout[-last:] = 1.0
    q = torch.zeros(n, D)
    leaves = [t[None, None].to(device).requires_grad_(True) for t in (q, k, v)]
    F(*leaves, n, 0, 1.0).backward(dout[None, None].to(device))
    got = leaves[0].grad[0, 0, -last:].double()
    k, v = k.double().to(device), v.double().to(device)
    i = torch.arange(n - last, n, device=device)[:, None]
    p = (torch.arange(n, device=device) <= i).double() / (i + 1.0)
    dp = v.sum(-1)
    g = p * (dp - (p * dp).sum(-1, keepdim=True))
    most = (g.clamp(min=0) @ k)  # P
    off = ((got - g @ k) / most).square().mean().sqrt().item() / 2.0 ** -24
    assert off < (n / 64) ** 0.5 + 40, off


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("KV, G", [(4, 1), (2, 3), (2, 4)])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_error_of_short_windows(D, KV, G, dt, device):
    """The score gradients of a row sum to zero: what delta = sum out dout is off by goes to dq as a common part of them
    times the sum of p k, the more the shorter the window is. With delta of the unrounded output the roundings of the
    score gradients (an operand of the tensor cores: not at D = 32) and of dq itself remain. A rounding is off by at most
    half a step of 2 u of its value, spread over it evenly by 2 u / sqrt(12) in the mean, and less for mantissas
    above 1; the two of them by sqrt(2) times that. (delta of the rounded output: 0.0038 at a window of 2 in bf16.)"""
    u = torch.finfo(dt).eps / 2
    bound = 2 * u / 12 ** 0.5 * (2 ** 0.5 if D >= 64 else 1.0)
    for window in (2, 3):
        problem = _problem(2, KV, G, 900, D, dt, seed=95)
        want = ref.batched(*problem[:3], window, 0, D ** -0.5, dt, problem[3])
        got = _run(problem, window, 0, device)
        for name in ("dq", "dk"):
            value = want[name][0]
            off = ((got[name].double().cpu() - value).norm() / value.norm()).item()
            assert off < bound, (window, name, off, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dt, D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 32), (torch.float32, 64)], ids=str)
def test_entry_points_without_the_rest_of_the_output(dt, D, device):
    """The C entry points that keep nothing of what the output's rounding leaves: the same output, gradients in bounds."""
    q, k, v, dout = problem = _problem(2, 2, 2, 500, D, dt, seed=97)
    q, k, v, dout = (t.to(device) for t in problem)
    window, sinks, scale = 40, 3, D ** -0.5
    out, dq, dk, dv = (torch.empty_like(t) for t in (q, q, k, v))
    lse = torch.empty(2, 4, 500, device=device)
    code = _lib.dtype_code(dt)
    sizes, strides = (2, 4, 2, 500, D), [t.stride() for t in (q, k, v, out)]
    _lib._call("tb200_window_attention_fwd", q, *(t.data_ptr() for t in (out, lse, q, k, v)), *sizes, *strides, window, sinks, scale, code)
    work = torch.empty(_lib.window_attention_bwd_workspace(q, k, window, sinks), dtype=torch.uint8, device=device)
    _lib._call("tb200_window_attention_bwd", q, *(t.data_ptr() for t in (dq, dk, dv, dout, q, k, v, out, lse, work)), work.numel(),
               *sizes, *strides, *(t.stride() for t in (dout, dq, dk, dv)), window, sinks, scale, code)
    assert torch.equal(out, F(q, k, v, window, sinks))
    want = ref.batched(*problem[:3], window, sinks, scale, dt, problem[3])
    for name, got in (("out", out), ("dv", dv), ("dq", dq), ("dk", dk)):
        ref.check(got, want[name], name)


def test_entry_points_with_the_rest_of_the_output_refuse():
    strides = (1, 1, 1, 1)
    forward, backward = (_lib._entry(f"tb200_window_attention_{name}_low") for name in ("fwd", "bwd"))
    assert forward(8, 8, 8, 8, 8, 8, 1, 3, 2, 8, 16, *[strides] * 4, 4, 0, 1.0, 0, 0) == -1  # heads
    assert forward(None, 8, 8, 8, 8, 8, 1, 2, 2, 8, 16, *[strides] * 4, 4, 0, 1.0, 0, 0) == -1
    assert backward(*[8] * 11, 0, 1, 2, 2, 8, 16, *[strides] * 8, 4, 0, 1.0, 0, 0) == -3  # no workspace
    assert backward(*[8] * 7, None, *[8] * 3, 1 << 20, 1, 2, 2, 8, 16, *[strides] * 8, 4, 0, 1.0, 0, 0) == -1
