"""Gated residual RMSNorm against its formula in 64 bits, forward and backward.

Tolerances. Every output is one rounding of an fp32 value: half a step of its type. The fp32 value's
own error is bounded by C * 2^-24 times the formula's value with all terms taken absolutely: a sum of k
terms is off by at most (chain length) * 2^-24 times the sum of their magnitudes, and the chains here
are at most ceil(cols / 256) + 13 in a row statistic (<= 45 at 8192 columns), rows / parts + parts / 32 + 36
in a column sum (<= 160 at the sizes below), with under 20 roundings around them: C = 256.
"""

import pytest
import torch

import trident_b200 as trident
from tests import util
from trident_b200.operation.gated_residual_rms_norm import rows_per_gate

C = 256.0
EPS = 1e-6


def _formula(x, r, w1, w2, g, a, eps, dh, dy):
    """All outputs in 64 bits, and their magnitudes (every term taken absolutely)."""

    def rms(v):
        return v.square().mean(-1, keepdim=True).sqrt()

    def ratio(num, den):
        return torch.where(den > 0, num / torch.where(den > 0, den, 1.0), 0.0)

    n_cols = x.shape[-1]
    one = torch.ones((), dtype=torch.float64)
    G = one if g is None else g
    W1 = one if w1 is None else w1
    m1 = rms(x)
    i1 = one if w1 is None else 1 / (m1 + eps)
    n = x * i1 * W1
    y = a * r + G * n
    ym = (a * r).abs() + (G * n).abs()
    m2 = rms(y)
    i2 = 1 / (m2 + eps)
    # the statistic of y carries y's own error: its magnitude relative to y is folded into every user
    loss = (rms(ym) / torch.where(m2 > 0, m2, 1.0)).clamp_min(1.0)
    out = {"h": (y * i2 * w2, ym * i2 * w2.abs() * loss), "y": (y, ym)}
    if dh is None:
        return out
    k2 = ratio((dh * w2 * y).sum(-1, keepdim=True) * i2 ** 2 / n_cols, m2)
    k2m = ratio((dh * w2 * ym).abs().sum(-1, keepdim=True) * i2 ** 2 / n_cols, m2) * loss ** 3
    dY = dy + dh * w2 * i2 - y * k2
    dYm = dy.abs() + (dh * w2 * i2).abs() * loss + ym * k2m
    out["residual"] = (a * dY, abs(a) * dYm)
    t, tm = dY * G * W1, dYm * (G * W1).abs()
    if w1 is None:
        k1 = k1m = 0.0
    else:
        k1 = ratio((t * x).sum(-1, keepdim=True) * i1 ** 2 / n_cols, m1)
        k1m = ratio((tm * x.abs()).sum(-1, keepdim=True) * i1 ** 2 / n_cols, m1)
    out["input"] = (t * i1 - x * k1, tm * i1 + x.abs() * k1m)

    def to(v, like):
        v = v.reshape(-1, n_cols).sum(0) if like.dim() == 1 else v.sum_to_size(like.shape)
        return v

    if w1 is not None:
        out["post_weight"] = (to(dY * G * x * i1, w1), to((dYm * G * x * i1).abs(), w1))
    out["pre_weight"] = (to(dh * y * i2, w2), to((dh * ym * i2).abs() * loss, w2))
    if g is not None:
        out["gate"] = (to(dY * n, g), to((dYm * n).abs(), g))
    return out


def _check(got, want, dtype, what):
    value, magnitude = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    tiny = {torch.float16: 2.0 ** -25}.get(dtype, 0.0)  # half of the smallest step: subnormal results
    slack = C * 2.0 ** -24 * magnitude
    bound = slack + torch.finfo(dtype).eps / 2 * (value.abs() + slack) + tiny
    excess = ((got - value).abs() - bound).max().item()
    assert excess <= 0, f"{what}: {excess:.3e} beyond the bound"


def _problem(shape, gate, post, dtype, seed=0):
    x = util.randn(*shape, seed=seed, std=1.3).to(dtype)
    r = util.randn(*shape, seed=seed + 1, std=2.0).to(dtype)
    cols = shape[-1]
    w1 = util.randn(cols, seed=seed + 2, std=0.1, mean=1.0).to(dtype) if post else None
    w2 = util.randn(cols, seed=seed + 3, std=0.1, mean=1.0).to(dtype)
    gshape = {"none": None, "feature": (cols,), "sequence": (shape[0],) + (1,) * (len(shape) - 2) + (cols,),
              "element": shape}[gate]
    g = None if gshape is None else util.randn(*gshape, seed=seed + 4, std=0.5, mean=0.3).to(dtype)
    dh, dy = (util.randn(*shape, seed=seed + 5 + i).to(dtype) for i in range(2))
    return x, r, w1, w2, g, dh, dy


def _run(problem, a, device, eps=EPS):
    x, r, w1, w2, g, dh, dy = (None if t is None else t.to(device) for t in problem)
    leaves = {"input": x, "residual": r, "post_weight": w1, "pre_weight": w2, "gate": g}
    leaves = {n: t.clone().requires_grad_(True) for n, t in leaves.items() if t is not None}
    h, y = trident.function.gated_residual_rms_norm(
        leaves["input"], leaves["residual"], leaves.get("post_weight"), leaves["pre_weight"], leaves.get("gate"), a, eps
    )
    torch.autograd.backward([h, y], [dh, dy])
    return {"h": h, "y": y, **{n: t.grad for n, t in leaves.items()}}


def _want(problem, a, eps=EPS):
    x, r, w1, w2, g, dh, dy = (None if t is None else t.double() for t in problem)
    return _formula(x, r, w1, w2, g, a, eps, dh, dy)


def _compare(problem, a, device, dtype, eps=EPS):
    got, want = _run(problem, a, device, eps), _want(problem, a, eps)
    assert set(got) == set(want)
    for name in want:
        _check(got[name], want[name], dtype, name)


def test_the_formula_agrees_with_autograd():
    problem = tuple(None if t is None else t.double() for t in _problem((3, 5, 24), "sequence", True, torch.float64))
    x, r, w1, w2, g, dh, dy = problem
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w1, w2, g)]

    def f(x, r, w1, w2, g):
        n = x / (x.square().mean(-1, keepdim=True).sqrt() + EPS) * w1
        y = 0.75 * r + g * n
        return y / (y.square().mean(-1, keepdim=True).sqrt() + EPS) * w2, y

    grads = torch.autograd.grad(f(*leaves), leaves, (dh, dy))
    want = _formula(x, r, w1, w2, g, 0.75, EPS, dh, dy)
    for name, grad in zip(("input", "residual", "post_weight", "pre_weight", "gate"), grads):
        assert torch.allclose(want[name][0], grad, rtol=1e-9, atol=1e-11), name


def test_gate_shapes():
    x = torch.empty(4, 6, 8)
    assert rows_per_gate(x, torch.empty(8)) == 0
    assert rows_per_gate(x, torch.empty(1, 1, 8)) == 0
    assert rows_per_gate(x, torch.empty(4, 1, 8)) == 6
    assert rows_per_gate(x, torch.empty(4, 6, 8)) == 1
    for shape in ((7,), (1, 6, 8), (6, 8), (4, 8), (1, 4, 6, 8), (2, 1, 8)):
        with pytest.raises(ValueError, match="does not fit"):
            rows_per_gate(x, torch.empty(*shape))


def test_refusals():
    f = trident.function.gated_residual_rms_norm
    x, w = torch.randn(4, 8), torch.ones(8)
    with pytest.raises(ValueError, match="same shape"):
        f(x, x[:2], w, w)
    with pytest.raises(ValueError, match="pre_weight"):
        f(x, x, w)
    with pytest.raises(ValueError, match="shape"):
        f(x, x, torch.ones(7), w)
    with pytest.raises(ValueError, match="does not fit"):
        f(x, x, w, w, torch.ones(3, 8))
    with pytest.raises(ValueError, match="same dtype"):
        f(x, x.half(), w, w)
    with pytest.raises(ValueError, match="Unable to convert"):
        f(x.double(), x.double(), w.double(), w.double())
    with pytest.raises(trident._lib.Tb200Error, match="CUDA tensors only"):
        f(x, x, w, w)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "feature", "sequence", "element"])
@pytest.mark.parametrize("post", [True, False], ids=["post", "nopost"])
@pytest.mark.parametrize("shape", [(3, 5, 24), (7, 13, 1021), (4, 40, 1024)], ids=str)
def test_against_the_formula(shape, post, gate, dtype, device):
    _compare(_problem(shape, gate, post, dtype), 0.75, device, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize(
    "shape",
    [(1, 1), (1, 8), (2, 3), (1, 4096), (600, 64), (5, 8200), (3, 16392), (2, 40000), (301, 2048), (9, 8192), (1500, 520)],
    ids=str,
)
def test_widths(shape, dtype, device):
    _compare(_problem(shape, "feature", True, dtype, seed=20), 1.0, device, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("batch, rows", [(1, 700), (700, 1), (2, 333), (37, 19), (350, 2), (3, 1)])
def test_gate_per_sequence(batch, rows, device):
    _compare(_problem((batch, rows, 256), "sequence", True, torch.bfloat16, seed=40), 1.25, device, torch.bfloat16)


@pytest.mark.gpu
def test_rows_of_zeros(device):
    """rms is 0 there: outputs and gradients are finite, dx is dn / eps. eps is large so that 16 bits hold it."""
    problem = list(_problem((6, 64), "feature", True, torch.float32, seed=60))
    problem[0][2] = 0.0
    problem[0][4], problem[1][4] = 0.0, 0.0
    _compare(tuple(problem), 1.0, device, torch.float32, eps=0.125)


@pytest.mark.gpu
def test_one_gradient_only(device):
    """Only one of the two outputs is used: the other's gradient counts as zero."""
    x, r, w1, w2, g, dh, dy = _problem((5, 96), "feature", True, torch.float32, seed=70)
    for use in (0, 1):
        leaves = [t.to(device).requires_grad_(True) for t in (x, r, w1, w2, g)]
        outs = trident.function.gated_residual_rms_norm(*leaves[:2], leaves[2], leaves[3], leaves[4], 1.0, EPS)
        outs[use].backward((dh, dy)[use].to(device))
        zero = torch.zeros_like(dh).double()
        want = _formula(*(t.double() for t in (x, r, w1, w2, g)), 1.0, EPS, dh.double() if use == 0 else zero,
                        dy.double() if use == 1 else zero)
        for name, leaf in zip(("input", "residual", "post_weight", "pre_weight", "gate"), leaves):
            _check(leaf.grad, want[name], torch.float32, name)


@pytest.mark.gpu
def test_only_what_needs_a_gradient(device):
    x, r, w1, w2, g, dh, dy = (t.to(device) for t in _problem((5, 96), "element", True, torch.float16, seed=80))
    full = _run((x, r, w1, w2, g, dh, dy), 1.0, device)
    for wanted in ("input", "post_weight", "gate"):
        leaves = {"input": x, "residual": r, "post_weight": w1, "pre_weight": w2, "gate": g}
        leaves = {n: t.clone().requires_grad_(n == wanted) for n, t in leaves.items()}
        outs = trident.function.gated_residual_rms_norm(*leaves.values(), 1.0, EPS)
        torch.autograd.backward(outs, [dh, dy])
        assert torch.equal(leaves[wanted].grad, full[wanted])
        assert all(t.grad is None for n, t in leaves.items() if n != wanted)


@pytest.mark.gpu
def test_gradients_against_differences(device):
    """Directional differences of the forward pass, fp32: (f(+e) - f(-e)) / 2e against the gradients."""
    x, r, w1, w2, g, dh, dy = (t.to(device) for t in _problem((4, 3, 32), "sequence", True, torch.float32, seed=90))
    grads = _run((x, r, w1, w2, g, dh, dy), 0.5, device)
    step = 2.0 ** -7

    def loss(args):
        h, y = trident.function.gated_residual_rms_norm(*args, 0.5, EPS)
        return (h.double() * dh.double()).sum() + (y.double() * dy.double()).sum()

    for i, name in enumerate(("input", "residual", "post_weight", "pre_weight", "gate")):
        args = [x, r, w1, w2, g]
        direction = util.randn(*args[i].shape, seed=100 + i, device=device)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step * direction, args[i] - step * direction
        slope = (loss(up) - loss(down)) / (2 * step)
        want = (grads[name].double() * direction.double()).sum()
        # third-order term of the difference: step^2 ~ 6e-5 of the sum of term magnitudes
        scale = (grads[name].double().abs() * direction.double().abs()).sum()
        assert abs(slope - want) <= 2e-3 * scale, name


@pytest.mark.gpu
def test_strided_inputs_unaligned_views_streams_and_repeats(device):
    dt = torch.bfloat16
    x, r, w1, w2, g, dh, dy = _problem((12, 128), "feature", True, dt, seed=110)
    want = _want((x, r, w1, w2, g, dh, dy), 1.0)
    first = _run((x, r, w1, w2, g, dh, dy), 1.0, device)
    again = _run((x, r, w1, w2, g, dh, dy), 1.0, device)
    for name in first:
        assert torch.equal(first[name], again[name]), name
    # a transposed input, and weights that start 2 bytes off a 16-byte boundary
    base = torch.empty(129, dtype=dt, device=device)
    w_odd = base[1:].copy_(w1)
    h, y = trident.function.gated_residual_rms_norm(
        x.t().contiguous().t().to(device), r.to(device), w_odd, w2.to(device), g.to(device), 1.0, EPS
    )
    _check(h, want["h"], dt, "h strided")
    _check(y, want["y"], dt, "y strided")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = _run((x, r, w1, w2, g, dh, dy), 1.0, device)
    stream.synchronize()
    for name in first:
        assert torch.equal(first[name], other[name]), name


@pytest.mark.gpu
def test_captured_step(device):
    """Forward and backward captured into a CUDA graph and replayed on new values."""
    dt = torch.bfloat16
    problem = [t.to(device) for t in _problem((64, 512), "feature", True, dt, seed=120)]
    leaves = [t.clone().requires_grad_(True) for t in problem[:5]]

    def step():
        h, y = trident.function.gated_residual_rms_norm(*leaves, 1.0, EPS)
        return (h, y, *torch.autograd.grad((h, y), leaves, problem[5:]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    fresh = _problem((64, 512), "feature", True, dt, seed=130)
    with torch.no_grad():
        for dst, src in zip(leaves + problem[5:], fresh):
            dst.copy_(src)
    graph.replay()
    torch.cuda.synchronize()
    want = _want(fresh, 1.0)
    for name, got in zip(("h", "y", "input", "residual", "post_weight", "pre_weight", "gate"), outs):
        _check(got, want[name], dt, name)


@pytest.mark.gpu
def test_module(device, dtype):
    m = trident.GatedResidualRMSNorm(64, device=device, dtype=dtype)
    x, r = (util.randn(2, 3, 64, seed=s, dtype=dtype, device=device).requires_grad_(True) for s in (1, 2))
    h, y = m(x, r)
    (h.float().sum() + y.float().sum()).backward()
    for t in (x, r, m.post_weight, m.pre_weight, m.gate):
        assert t.grad is not None and t.grad.dtype == dtype and torch.isfinite(t.grad).all()
    assert "backend=Trident" in repr(m)
    bare = trident.GatedResidualRMSNorm(64, post_norm=False, gate=False, device=device, dtype=dtype)
    assert set(dict(bare.named_parameters())) == {"pre_weight"}
    assert bare(x, r, torch.ones(2, 1, 64, device=device, dtype=dtype))[0].shape == x.shape


@pytest.mark.gpu
def test_no_rows(device):
    w = torch.ones(16, device=device, requires_grad=True)
    g = torch.ones(3, 1, 16, device=device, requires_grad=True)
    x = torch.empty(3, 0, 16, device=device, requires_grad=True)
    h, y = trident.function.gated_residual_rms_norm(x, x, w, w, g)
    (h.sum() + y.sum()).backward()
    assert h.shape == x.shape and torch.all(w.grad == 0) and torch.all(g.grad == 0)


@pytest.mark.gpu
def test_more_than_32_bit_offsets(device):
    """The last rows of more than 2^31 elements."""
    cols, dt = 4096, torch.bfloat16
    rows = 2 ** 31 // cols + 5
    generator = torch.Generator(device=device).manual_seed(400)
    x, r, dh, dy = (torch.randn(rows, cols, dtype=dt, device=device, generator=generator) for _ in range(4))
    w1, w2, g = (torch.randn(cols, dtype=dt, device=device, generator=generator) for _ in range(3))
    x.requires_grad_(True)
    r.requires_grad_(True)
    h, y = trident.function.gated_residual_rms_norm(x, r, w1, w2, g, 0.9, EPS)
    dx, dr = torch.autograd.grad((h, y), (x, r), (dh, dy))
    tail = tuple(t.detach()[-6:].cpu() for t in (x, r)) + tuple(t.cpu() for t in (w1, w2, g)) + tuple(t[-6:].cpu() for t in (dh, dy))
    want = _want(tail, 0.9)
    for name, got in (("h", h), ("y", y), ("input", dx), ("residual", dr)):
        _check(got[-6:], want[name], dt, name)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "feature", "sequence", "element"])
@pytest.mark.parametrize("shape", [(40, 9, 1), (3, 50, 257), (35, 8, 1025), (2, 33, 2049), (5, 7, 4095), (2, 9, 4097)], ids=str)
def test_odd_widths(shape, gate, dtype, device):
    """The widths at which the kernels for rows of any alignment change, one and many gate vectors."""
    _compare(_problem(shape, gate, gate != "feature", dtype, seed=420), 0.9, device, dtype)


def test_library_refuses_before_launch():
    from trident_b200 import _lib

    call = _lib.load().tb200_gated_residual_rms_norm_fwd

    def fwd(out=8, x=8, post=None, pre=8, gate=None, rows=2, cols=16, group=0, dtype=0):
        return call(out, 8, 8, 8, x, 8, post, pre, gate, rows, cols, group, 1.0, 1e-6, dtype, None)

    assert fwd(out=None) < 0 and fwd(x=None) < 0 and fwd(pre=None) < 0 and fwd(rows=-1) < 0 and fwd(cols=0) < 0
    assert fwd(gate=8, group=-1) < 0 and fwd(dtype=9) < 0 and fwd(rows=0) == 0
