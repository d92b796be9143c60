"""A bounded wait that runs out: the abort path of the tensor-core kernels, executed once.

Every mbarrier wait of those kernels has a time limit; when one expires the CTA raises an abort
flag, records a code in the device status word, lets its roles run to their end, drains what
they have in flight and frees its tensor memory. The test hook `tb200_test_wait_fault(1)` makes
exactly that happen in the attention forward: the limit shrinks to about a millisecond and the
producer of one CTA leaves out the copy of one key tile (it touches no memory a normal launch
would not touch), so the MMA issuer waits for a tile that never arrives. Nothing faults and
nothing hangs: the launch ends by itself, the status word is non-zero, and the next normal call
on the same context is correct.
"""

import math

import pytest
import torch

import trident_b200 as trident
from oracle import torch_oracle
from tests import util
from trident_b200 import _lib

pytestmark = pytest.mark.gpu


def test_expired_wait_sets_the_status_word_and_the_context_stays_usable(device):
    dt = torch.bfloat16
    B, H, S, D = 1, 2, 256, 64
    q, k, v = (util.randn(B, H, S, D, seed=s, dtype=dt, device=device) for s in (1, 2, 3))
    _lib.device_status(reset=True)
    assert _lib.device_status() == 0
    out = torch.empty_like(q)
    lse = torch.empty(B, H, S, device=device, dtype=torch.float32)
    old = _lib.test_wait_fault(1)
    try:
        _lib.attention_fwd(out, lse, q, k, v, None, False, 1.0 / math.sqrt(D))
        assert _lib.last_kernel() == "attn_tcgen05"
        torch.cuda.synchronize()  # returns: the kernel ended by itself
    finally:
        _lib.test_wait_fault(old)
    code = _lib.device_status(reset=True)
    assert code != 0, "the expired wait was not recorded"
    assert _lib.device_status() == 0
    # the same context, the same kernel, without the hook: correct result and a clean status
    got = trident.function.scaled_dot_product_attention(q, k, v)
    want = torch_oracle.scaled_dot_product_attention(q.float().cpu(), k.float().cpu(), v.float().cpu())
    util.assert_half_close(got, want, dt, atol=1e-2, ulps=1.0, what="forward after the aborted launch")
    assert _lib.device_status() == 0


# ------------------------------------------------------------------ window and paged attention, norms between blocks
# (the hook's mode 1 means the kernel of a call, of the window attention backward that of dQ, mode 2 that of dK, dV)
def _expires(call, outputs, mode, kernel):
    """`call` fills `outputs`: right, then with a wait that runs out, then right again, to the bit."""
    _lib.device_status(reset=True)
    call()
    torch.cuda.synchronize()
    assert _lib.device_status() == 0 and _lib.last_kernel() == kernel
    want = [t.clone() for t in outputs]
    old = _lib.test_wait_fault(mode)
    try:
        call()
        torch.cuda.synchronize()  # returns: the kernels ended by themselves
    finally:
        _lib.test_wait_fault(old)
    assert _lib.device_status(reset=True) != 0, "the expired wait was not recorded"
    for t in outputs:
        t.fill_(float("nan"))
    call()
    assert _lib.device_status() == 0
    for got, value in zip(outputs, want):
        assert torch.equal(got, value)


# one piece of work of the first CTA, several of them (most of which follow the expired wait)
@pytest.mark.parametrize("H, S", [(2, 512), (64, 2000)])
@pytest.mark.parametrize("D", [64, 128])
def test_window_attention_ends_after_an_expired_wait(D, H, S, device):
    dt = torch.bfloat16
    q, dout = (util.randn(2, H, S, D, seed=s, dtype=dt, device=device) for s in (1, 2))
    k, v = (util.randn(2, H // 2, S, D, seed=s, dtype=dt, device=device) for s in (3, 4))
    out, dq, dk, dv = (torch.empty_like(t) for t in (q, q, k, v))
    lse = torch.empty(2, H, S, device=device, dtype=torch.float32)
    _expires(lambda: _lib.window_attention_fwd(out, lse, q, k, v, 400, 3, 0.1), [out, lse], 1, "local_tcgen05")
    workspace = torch.empty(_lib.window_attention_bwd_workspace(q, k, 400, 3), dtype=torch.uint8, device=device)
    for mode in (1, 2):
        _expires(lambda: _lib.window_attention_bwd(dq, dk, dv, dout, q, k, v, out, lse, workspace, 400, 3, 0.1),
                 [dq, dk, dv], mode, "local_tcgen05")


@pytest.mark.parametrize("n, new", [(1, 1), (40, 1), (1, 300), (40, 200)])
@pytest.mark.parametrize("D", [64, 128])
def test_paged_attention_ends_after_an_expired_wait(D, n, new, device):
    """Single tokens (the kernel for few rows) and chunks, whose last pages are not full."""
    dt, KV, page, context = torch.bfloat16, 2, 16, 1003
    blocks = -(-context // page)
    kc, vc = (util.randn(n * blocks, page, KV, D, seed=s, dtype=dt, device=device) for s in (5, 6))
    table = torch.arange(n * blocks, dtype=torch.int32, device=device).view(n, blocks)
    lengths = torch.full((n,), context, dtype=torch.int32, device=device)
    offsets = torch.arange(0, n * new + 1, new, dtype=torch.int32, device=device)
    q = util.randn(n * new, 4 * KV, D, seed=7, dtype=dt, device=device)
    out = torch.empty_like(q)

    def call():
        trident.function.paged_attention(q, kc, vc, table, lengths, offsets, new, context, output=out)

    _expires(call, [out], 1, "local_tcgen05")


@pytest.mark.parametrize("cols", [256, 4096, 16384])
def test_norm_backward_ends_after_an_expired_wait(cols, device):
    dt, rows = torch.bfloat16, 1500
    x, r, dh, dy = (util.randn(rows, cols, seed=s, dtype=dt, device=device) for s in range(4))
    w1, w2, gate = (util.randn(cols, seed=4 + s, dtype=dt, device=device) for s in range(3))
    h, y, dx, dr = (torch.empty_like(x) for _ in range(4))
    dw1, dw2, dgate = (torch.empty_like(w1) for _ in range(3))
    rms = torch.empty(2, rows, device=device, dtype=torch.float32)
    _lib.gated_residual_rms_norm_fwd(h, y, rms, x, r, w1, w2, gate, rows, cols, 0, 0.5, 1e-5)
    workspace = torch.empty(_lib.gated_residual_rms_norm_bwd_workspace(x, rows, cols, 0), dtype=torch.uint8, device=device)

    def call():
        _lib.gated_residual_rms_norm_bwd(dx, dr, dw1, dw2, dgate, dh, dy, x, r, w1, w2, gate, rms, workspace, rows, cols, 0, 0.5, 1e-5)

    _expires(call, [dx, dr, dw1, dw2, dgate], 1, "row_vec")
