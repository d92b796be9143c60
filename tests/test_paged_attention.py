"""Attention over a paged cache and the write into it, against the formula in 64 bits."""

import pytest
import torch

import trident_b200 as trident
from tests import local_reference as ref
from tests import util
from trident_b200 import _lib

attend = trident.function.paged_attention
append = trident.function.paged_cache_append


class Cache:
    """A pool of pages in random order, with the sequences' keys and values in it; everything else in the
    pool (the rest of last pages, spare pages) is NaN, and unused table entries are -1."""

    def __init__(self, context, KV, D, page, dtype, device, seed=0, poison=float("nan")):
        self.context, self.page = context, page
        g = util.seeded(seed)
        blocks = [-(-c // page) for c in context]
        pages = sum(blocks) + 2
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((len(context), max(blocks + [1]) + 1), -1, dtype=torch.int32)
        self.keys, self.values = [], []
        kc, vc = (torch.full((pages, page, KV, D), poison) for _ in range(2))
        at = 0
        for s, (c, b) in enumerate(zip(context, blocks)):
            self.table[s, :b] = order[at:at + b].to(torch.int32)
            at += b
            k, v = (torch.randn(c, KV, D, generator=g).to(dtype) for _ in range(2))
            self.keys.append(k)
            self.values.append(v)
            for cache, rows in ((kc, k), (vc, v)):
                x = torch.arange(c)
                cache[self.table[s, (x // page)].long(), x % page] = rows.float()
        self.key_cache, self.value_cache = kc.to(dtype).to(device), vc.to(dtype).to(device)
        self.table_dev = self.table.to(device)
        self.context_dev = torch.tensor(context, dtype=torch.int32, device=device)


def _offsets(new, device):
    return torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device=device)


def _want(q, cache, new, window, sinks, scale, dtype):
    """Values and bounds [T, H, D]."""
    T, H, D = q.shape
    KV = cache.key_cache.shape[2]
    G = H // KV
    value, bound = (torch.zeros(T, H, D, dtype=torch.float64) for _ in range(2))
    at = 0
    for s, t in enumerate(new):
        c = cache.context[s]
        pos = torch.arange(c - t, c)
        for h in range(KV):
            one = ref.attention(q[at:at + t, h * G:(h + 1) * G].double().transpose(0, 1), cache.keys[s][:, h].double(),
                                cache.values[s][:, h].double(), pos, window, sinks, scale, dtype)["out"]
            value[at:at + t, h * G:(h + 1) * G] = one[0].transpose(0, 1)
            bound[at:at + t, h * G:(h + 1) * G] = one[1].transpose(0, 1)
        at += t
    return value, bound


def _compare(context, new, KV, G, D, page, dtype, device, window=None, sinks=0, seed=0, decode=False, **more):
    cache = Cache(context, KV, D, page, dtype, device, seed)
    q = util.randn(sum(new), KV * G, D, seed=seed + 1000).to(dtype)
    got = attend(q.to(device), cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev,
                 None if decode else _offsets(new, device), window_size=window, num_sinks=sinks, **more)
    ref.check(got, _want(q, cache, new, window or 0, sinks, D ** -0.5, dtype), "out")
    assert _lib.device_status() == 0
    return got


# ------------------------------------------------------------------------------------ no GPU
def _cpu_call(**change):
    args = dict(query=torch.randn(3, 4, 16), key_cache=torch.randn(5, 8, 2, 16), value_cache=torch.randn(5, 8, 2, 16),
                block_table=torch.zeros(2, 3, dtype=torch.int32), context_lengths=torch.ones(2, dtype=torch.int32),
                query_offsets=torch.tensor([0, 1, 3], dtype=torch.int32))
    args.update(change)
    return args


@pytest.mark.parametrize("change, match", [
    (dict(query=torch.randn(3, 64)), "dimension of query"),
    (dict(key_cache=torch.randn(5, 8, 32)), "dimension of key_cache"),
    (dict(value_cache=torch.randn(5, 4, 2, 16)), "same shape"),
    (dict(key_cache=torch.randn(5, 0, 2, 16), value_cache=torch.randn(5, 0, 2, 16)), "at least one token"),
    (dict(query=torch.randn(3, 4, 32)), "same head size"),
    (dict(query=torch.randn(3, 3, 16)), "multiple"),
    (dict(block_table=torch.zeros(2, 3)), "torch.int32"),
    (dict(context_lengths=torch.ones(2, dtype=torch.int64)), "torch.int32"),
    (dict(context_lengths=torch.ones(3, dtype=torch.int32)), r"\[sequences\]"),
    (dict(query_offsets=torch.tensor([0, 3], dtype=torch.int32)), r"sequences \+ 1"),
    (dict(query_offsets=None), "one new token per sequence"),
    (dict(query=torch.randn(3, 4, 16).half()), "same dtype"),
    (dict(window_size=0), "window_size"),
    (dict(num_sinks=2), "needs a window_size"),
    (dict(window_size=4, num_sinks=-1), "num_sinks"),
    (dict(max_query_length=-1), "max_query_length"),
    (dict(max_context_length=-1), "max_context_length"),
    (dict(output=torch.empty(2, 4, 16)), "output and query"),
    (dict(query=torch.randn(3, 4, 16, requires_grad=True)), "no backward"),
])
def test_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        attend(**_cpu_call(**change))


def test_append_refusals():
    args = _cpu_call()
    del args["query"]
    k = torch.randn(3, 2, 16)
    for key, value, match in ((k, k[:2], "same shape"), (k[0], k[0], "same shape"), (k[:, :1], k[:, :1], "same heads"),
                              (k.half(), k.half(), "same dtype")):
        with pytest.raises(ValueError, match=match):
            append(key, value, **args)
    with pytest.raises(_lib.Tb200Error, match="CUDA tensors only"):
        append(k, k, **args)
    with pytest.raises(_lib.Tb200Error, match="CUDA tensors only"):
        attend(**_cpu_call())


# ------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("page", [1, 8, 16, 24, 64, 100, 256])
def test_single_tokens(page, D, dtype, device):
    _compare([1, 7, 64, 129, 500], [1] * 5, 2, 4, D, page, dtype, device, decode=True)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 24, 128, 37])
@pytest.mark.parametrize("window, sinks", [(None, 0), (50, 3), (1, 0), (200, 140)])
@pytest.mark.parametrize("D", [64, 128])
def test_chunks(D, window, sinks, page, dtype, device):
    _compare([300, 33, 513, 1], [40, 33, 130, 1], 2, 3, D, page, dtype, device, window, sinks, seed=1)


@pytest.mark.gpu
@pytest.mark.parametrize("KV, G", [(1, 1), (3, 1), (1, 8), (2, 16), (1, 7), (1, 64), (1, 40)])
@pytest.mark.parametrize("D", [64, 128])
def test_head_groups(KV, G, D, dtype, device):
    _compare([200, 90], [1, 1], KV, G, D, 16, dtype, device, decode=True, seed=2)
    _compare([200, 90], [30, 20], KV, G, D, 16, dtype, device, 60, 2, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("G, t", [(1, 1), (4, 1), (4, 9), (8, 40)])
@pytest.mark.parametrize("window, sinks", [(None, 0), (3000, 5), (700, 600)])
@pytest.mark.parametrize("D", [64, 128])
def test_long_contexts_of_few_sequences(D, window, sinks, G, t, dtype, device):
    """Few rows and many keys: the walk along the keys is cut and joined."""
    _compare([5000], [t], 1, G, D, 32, dtype, device, window, sinks, seed=4)
    _compare([4100, 70], [t, t], 2, G, D, 16, dtype, device, window, sinks, seed=5)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_announced_lengths_only_change_the_speed(D, device):
    """Contexts longer than announced are still right, and so is every announced number."""
    for announced in (None, 1, 300, 3000, 10 ** 6):
        _compare([2500, 40], [1, 1], 1, 4, D, 16, torch.bfloat16, device, decode=True, seed=6, max_context_length=announced)
        _compare([2500, 40], [3, 7], 1, 4, D, 16, torch.bfloat16, device, seed=6, max_query_length=7, max_context_length=announced)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
def test_sequences_without_tokens_or_keys(D, dtype, device):
    """No new tokens, no keys, more new tokens than keys (positions below zero see nothing)."""
    cache = Cache([50, 0, 20, 3], 2, D, 16, dtype, device, seed=7)
    new = [0, 2, 5, 6]
    q = util.randn(13, 4, D, seed=8).to(dtype)
    got = attend(q.to(device), cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev, _offsets(new, device))
    want = _want(q, cache, new, 0, 0, D ** -0.5, dtype)
    ref.check(got, want, "out")
    assert torch.all(got[:2] == 0) and torch.all(got[7:10] == 0)  # the second sequence, and the last one's first three


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
def test_rows_behind_the_last_sequence(D, dtype, device):
    cache = Cache([30, 45], 1, D, 8, dtype, device, seed=9)
    q = util.randn(300, 2, D, seed=10).to(dtype)
    offsets = _offsets([4, 6], device)
    got = attend(q.to(device), cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev, offsets)
    ref.check(got[:10], _want(q[:10], cache, [4, 6], 0, 0, D ** -0.5, dtype), "out")
    assert torch.all(got[10:] == 0)
    mine = torch.full_like(got, 5.0)
    back = attend(q.to(device), cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev, offsets, output=mine)
    assert back is mine and torch.equal(mine[:10], got[:10]) and torch.all(mine[10:] == 5.0)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_released_pages_are_not_read(D, dtype, device):
    """Blocks that lie wholly outside window and sinks may carry any table entry and any content."""
    context, window, sinks, page = [900], 100, 20, 16
    for t in (1, 30):
        cache = Cache(context, 2, D, page, dtype, device, seed=11)
        q = util.randn(t, 4, D, seed=12).to(dtype)
        first = context[0] - t - window + 1
        gone = [b for b in range(-(-context[0] // page)) if b * page >= sinks and (b + 1) * page <= first]
        assert len(gone) > 40
        for mode in ("poisoned", "missing"):
            table = cache.table_dev.clone()
            kc, vc = cache.key_cache.clone(), cache.value_cache.clone()
            for b in gone:
                if mode == "missing":
                    table[0, b] = (-1, 10 ** 9)[b % 2]
                else:
                    kc[table[0, b].long()] = float("nan")
                    vc[table[0, b].long()] = float("inf")
            got = attend(q.to(device), kc, vc, table, cache.context_dev, _offsets([t], device), window_size=window, num_sinks=sinks)
            ref.check(got, _want(q, cache, [t], window, sinks, D ** -0.5, dtype), mode)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_bad_pages_and_offsets_touch_nothing_else(D, dtype, device):
    """Table entries outside the pool that a token sees read as zeros; offsets and contexts out of range are cut."""
    cache = Cache([64], 1, D, 16, dtype, device, seed=13)
    q = util.randn(2, 2, D, seed=14).to(dtype)
    table = cache.table_dev.clone()
    table[0, 1], table[0, 2] = -5, 2 ** 31 - 1
    cache.keys[0][16:48], cache.values[0][16:48] = 0.0, 0.0
    got = attend(q.to(device), cache.key_cache, cache.value_cache, table, cache.context_dev, _offsets([2], device))
    ref.check(got, _want(q, cache, [2], 0, 0, D ** -0.5, dtype), "bad pages")
    wild = torch.tensor([-7, 10 ** 9], dtype=torch.int32, device=device)
    got = attend(q.to(device), cache.key_cache, cache.value_cache, table, cache.context_dev, wild)
    ref.check(got, _want(q, cache, [2], 0, 0, D ** -0.5, dtype), "wild offsets")
    # a context beyond the table counts as what the table holds (here 5 blocks, the last of which is missing)
    long = attend(q.to(device), cache.key_cache, cache.value_cache, table, torch.full_like(cache.context_dev, 10 ** 9), wild)
    assert torch.isfinite(long.float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_layouts(D, dtype, device):
    """A pool that keeps heads before positions, a strided query, a table that is a slice."""
    cache = Cache([100, 260], 2, D, 32, dtype, device, seed=15)
    q = util.randn(2, 8, D, seed=16).to(dtype)
    want = _want(q, cache, [1, 1], 0, 0, D ** -0.5, dtype)
    kc, vc = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (cache.key_cache, cache.value_cache))
    wide = torch.stack([q, q], 2).to(device)[:, :, 0]
    table = torch.cat([cache.table_dev, cache.table_dev], 1)[:, : cache.table_dev.shape[1]]
    ref.check(attend(wide, kc, vc, table, cache.context_dev), want, "layouts")
    both = torch.stack([cache.key_cache, cache.value_cache], 1)  # [pages, 2, page, KV, D]
    ref.check(attend(q.to(device), both[:, 0], both[:, 1], cache.table_dev.t().contiguous().t(), cache.context_dev), want, "joint pool")
    out = torch.empty(8, 2, D, dtype=dtype, device=device).transpose(0, 1)
    ref.check(attend(q.to(device), cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev, output=out), want, "strided output")
    odd_k, odd_v = (torch.empty(t.numel() + 1, dtype=dtype, device=device)[1:].view(t.shape).copy_(t) for t in (cache.key_cache, cache.value_cache))
    ref.check(attend(q.to(device), odd_k, odd_v, cache.table_dev, cache.context_dev), want, "unaligned pool")


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 16, 24, 64])
@pytest.mark.parametrize("D", [16, 64, 128])
def test_append(D, page, dtype, device):
    context, new = [20, 70, 3, 0, 9], [20, 5, 1, 0, 12]
    cache = Cache(context, 2, D, page, dtype, device, seed=17)
    k, v = (util.randn(sum(new) + 4, 2, D, seed=18 + i).to(dtype).to(device) for i in range(2))
    kc, vc = cache.key_cache.clone(), cache.value_cache.clone()
    append(k, v, kc, vc, cache.table_dev, cache.context_dev, _offsets(new, device))
    want_k, want_v = cache.key_cache.clone(), cache.value_cache.clone()
    at = 0
    for s, t in enumerate(new):
        for i in range(t):
            pos = context[s] - t + i
            if pos >= 0:
                where = cache.table[s, pos // page].long().item(), pos % page
                want_k[where], want_v[where] = k[at + i], v[at + i]
        at += t
    assert torch.equal(kc.view(torch.uint8 if dtype != torch.float32 else torch.int32), want_k.view(torch.uint8 if dtype != torch.float32 else torch.int32))
    assert torch.equal(torch.nan_to_num(vc), torch.nan_to_num(want_v))
    # one token each, strided rows, and pages outside the pool left out
    table = cache.table_dev.clone()
    table[0] = torch.tensor([-1, 2 ** 31 - 1], dtype=torch.int32, device=device)[torch.arange(table.shape[1], device=device) % 2]
    kc, vc = cache.key_cache.clone(), cache.value_cache.clone()
    joint = torch.cat([k, v], 1)[:5]
    append(joint[:, :2], joint[:, 2:], kc, vc, table, cache.context_dev)
    want_k = cache.key_cache.clone()
    for s, c in enumerate(context):
        if s > 0 and c > 0:
            want_k[cache.table[s, (c - 1) // page].long(), (c - 1) % page] = k[s]
    assert torch.equal(torch.nan_to_num(kc), torch.nan_to_num(want_k))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_captured_decode_grows(dt, device):
    """One captured step (write, attend) replayed while the contexts grow; two graphs live side by side."""
    D, KV, G, page = 64, 2, 2, 16
    cache = Cache([300, 40], KV, D, page, dt, device, seed=20)
    spare = [int(p) for p in range(cache.key_cache.shape[0]) if p not in set(cache.table[cache.table >= 0].tolist())]
    for s, c in enumerate(cache.context):  # room for the next tokens
        if cache.table[s, c // page] < 0:
            cache.table[s, c // page] = spare.pop()
    cache.table_dev.copy_(cache.table)
    q = torch.zeros(2, KV * G, D, dtype=dt, device=device)
    k, v = (torch.zeros(2, KV, D, dtype=dt, device=device) for _ in range(2))

    def step():
        append(k, v, cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev)
        return attend(q, cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev, max_context_length=320)

    cache.context_dev += 1
    step()
    torch.cuda.synchronize()
    cache.context_dev -= 1
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step())
    for i in range(4):
        fresh = [util.randn(*t.shape, seed=30 + 3 * i + j).to(dt) for j, t in enumerate((q, k, v))]
        for dst, src in zip((q, k, v), fresh):
            dst.copy_(src)
        cache.context_dev += 1
        for s in range(2):
            cache.context[s] += 1
            cache.keys[s] = torch.cat([cache.keys[s], fresh[1][s:s + 1]])
            cache.values[s] = torch.cat([cache.values[s], fresh[2][s:s + 1]])
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        ref.check(outs[i % 2], _want(fresh[0], cache, [1, 1], 0, 0, D ** -0.5, dt), f"step {i}")


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_same_bits_every_time_and_two_streams(D, dtype, device):
    cache = Cache([3000, 900], 1, D, 16, dtype, device, seed=40)
    q = util.randn(2, 4, D, seed=41).to(dtype).to(device)

    def call():
        return attend(q, cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev, max_context_length=3000)

    first = call()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(call())
    for s in streams:
        s.synchronize()
    assert all(torch.equal(first, r) for r in results)


@pytest.mark.gpu
def test_module(device, dtype):
    D = 64
    cache = Cache([40, 12], 2, D, 16, dtype, device, seed=50, poison=0.0)
    q, k, v = (util.randn(2, h, D, seed=51 + h).to(dtype).to(device) for h in (4, 2, 2))
    m = trident.PagedAttention(window_size=20, num_sinks=2)
    with torch.no_grad():
        got = m(q, k, v, cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev)
    for s in range(2):
        cache.keys[s][-1], cache.values[s][-1] = k[s].cpu(), v[s].cpu()
    ref.check(got, _want(q.cpu(), cache, [1, 1], 20, 2, D ** -0.5, dtype), "module")
    assert "backend=Trident" in repr(m)


@pytest.mark.gpu
def test_nothing_to_do(device):
    kc = torch.zeros(2, 8, 1, 64, device=device)
    table = torch.zeros(0, 1, dtype=torch.int32, device=device)
    none = torch.zeros(0, dtype=torch.int32, device=device)
    assert attend(torch.zeros(0, 2, 64, device=device), kc, kc, table, none).shape == (0, 2, 64)
    out = attend(torch.ones(3, 2, 64, device=device), kc, kc, table, none, torch.zeros(1, dtype=torch.int32, device=device))
    assert torch.all(out == 0)
    append(torch.zeros(0, 1, 64, device=device), torch.zeros(0, 1, 64, device=device), kc, kc, table, none)


def _random(low, high, count, seed):
    return torch.randint(low, high, (count,), generator=util.seeded(seed)).tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("window, sinks", [(None, 0), (70, 5)])
@pytest.mark.parametrize("D", [64, 128])
def test_many_sequences(D, window, sinks, dtype, device):
    """Many more pieces of work than SMs, of very unequal lengths, some of them empty: chunks and single tokens."""
    n, KV = 90, 6
    new = _random(0, 40, n, 60)
    context = [t + c if i % 7 else t for i, (t, c) in enumerate(zip(new, _random(0, 400, n, 61)))]
    for _ in range(2):
        _compare(context, new, KV, 2, D, 16, dtype, device, window, sinks, seed=62)
    _compare([1 + c for c in _random(0, 700, n, 63)], [1] * n, KV, 4, D, 16, dtype, device, window, sinks, seed=64, decode=True)


@pytest.mark.gpu
@pytest.mark.parametrize("G, t", [(1, 17), (4, 6), (16, 2), (1, 64), (8, 8), (5, 9), (64, 1), (33, 1)])
@pytest.mark.parametrize("window, sinks", [(None, 0), (500, 3)])
@pytest.mark.parametrize("D", [64, 128])
def test_up_to_64_rows(D, window, sinks, G, t, dtype, device):
    """Every width of the kernel for few rows, with the walk whole and cut."""
    _compare([1500, t, 3], [t, t, 0], 2, G, D, 16, dtype, device, window, sinks, seed=65, max_query_length=t)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
def test_no_announced_lengths(D, dtype, device):
    """Hundreds of ragged chunks in one call whose longest is not given: almost all planned pieces of work are empty,
    and the roles of a kernel wait for one another while they pass over them."""
    n, KV = 400, 2
    new = _random(0, 60, n, 80)
    context = [t + c for t, c in zip(new, _random(0, 90, n, 81))]
    for _ in range(3):
        _compare(context, new, KV, 4, D, 16, dtype, device, None, 0, seed=82)


@pytest.mark.gpu
@pytest.mark.parametrize("G, KV", [(16, 3), (4, 2), (64, 1)])
@pytest.mark.parametrize("window, sinks", [(None, 0), (4, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_more_new_tokens_than_keys(D, window, sinks, G, KV, dtype, device):
    """Long chunks over short contexts: most rows lie at positions below zero, whole tiles of them next to tiles
    with keys."""
    n = 100
    _compare(_random(0, 30, n, 90), _random(0, 130, n, 91), KV, G, D, 16, dtype, device, window, sinks, seed=92)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 0.7])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_scales(D, scale, dtype, device):
    cache = Cache([700, 150], 1, D, 16, dtype, device, seed=66)
    for new, decode in (([1, 1], True), ([90, 150], False)):
        q = util.randn(sum(new), 4, D, seed=67).to(dtype)
        got = attend(q.to(device), cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev,
                     None if decode else _offsets(new, device), softmax_scale=scale)
        ref.check(got, _want(q, cache, new, 0, 0, scale, dtype), f"{new}")


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_large_scores(D, dtype, device):
    """Scores of hundreds: one key takes almost all the weight, the running maximum moves by large steps."""
    cache = Cache([1700, 300], 2, D, 16, dtype, device, seed=68)
    for new in ([1, 1], [100, 77]):
        q = util.randn(sum(new), 4, D, seed=69, std=25.0).to(dtype)
        got = attend(q.to(device), cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev, _offsets(new, device))
        ref.check(got, _want(q, cache, new, 0, 0, D ** -0.5, dtype), f"{new}")


@pytest.mark.gpu
def test_offsets_and_contexts_out_of_order(device, dtype):
    """Offsets that fall and negative contexts count as no tokens and no keys; other sequences keep their results."""
    D = 64
    cache = Cache([60, 33, 20], 2, D, 16, dtype, device, seed=70)
    q = util.randn(9, 4, D, seed=71).to(dtype)
    offsets = torch.tensor([0, 5, 3, 9], dtype=torch.int32, device=device)  # 5 tokens, none, tokens 3 to 8
    context = cache.context_dev.clone()
    context[0] = -(2 ** 31)
    got = attend(q.to(device), cache.key_cache, cache.value_cache, cache.table_dev, context, offsets, window_size=10, num_sinks=2)
    cache.context[0], cache.keys[0], cache.values[0] = 0, cache.keys[0][:0], cache.values[0][:0]
    assert torch.all(got[:3] == 0) and torch.isfinite(got.float()).all()
    mine = torch.empty_like(q)
    mine[3:] = q[3:]
    want = _want(mine[3:], Third(cache, 2), [6], 10, 2, D ** -0.5, dtype)
    ref.check(got[5:], tuple(t[2:] for t in want), "third sequence")  # (rows 3 and 4 belong to two sequences)
    kc = cache.key_cache.clone()
    k = util.randn(9, 2, D, seed=72).to(dtype).to(device)
    append(k, k, kc, kc.clone(), cache.table_dev, context, offsets)
    changed = (kc != cache.key_cache) & ~(torch.isnan(kc.float()) & torch.isnan(cache.key_cache.float()))
    assert changed.flatten(2).any(-1).sum() == 6  # the third sequence's six tokens


class Third:
    """One sequence of a cache, as _want sees a cache."""

    def __init__(self, cache, s):
        self.context, self.keys, self.values = [cache.context[s]], [cache.keys[s]], [cache.values[s]]
        self.key_cache = cache.key_cache


@pytest.mark.gpu
def test_shared_pages(device, dtype):
    """Sequences may share the pages of a common beginning."""
    D, page = 128, 16
    cache = Cache([200], 2, D, page, dtype, device, seed=73)
    q = util.randn(3, 4, D, seed=74).to(dtype)
    table = cache.table_dev.expand(3, -1)  # (a stride of zero: one row for all)
    lengths = [200, 64, 7]
    got = attend(q.to(device), cache.key_cache, cache.value_cache, table, torch.tensor(lengths, dtype=torch.int32, device=device))
    for s, c in enumerate(lengths):
        one = type("One", (), dict(context=[c], keys=[cache.keys[0][:c]], values=[cache.values[0][:c]], key_cache=cache.key_cache))
        ref.check(got[s:s + 1], _want(q[s:s + 1], one, [1], 0, 0, D ** -0.5, dtype), f"sequence {s}")


@pytest.mark.gpu
@pytest.mark.parametrize("dt, D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)], ids=["bf16", "fp16", "fp32"])
def test_pool_of_more_than_32_bit_offsets(dt, D, device):
    """Pages whose elements lie beyond 2^31 and 2^32 elements (bytes, in fp32) from the start of the pool."""
    KV, page = 8, 16
    row = KV * page * D
    beyond = (2 ** 32 if dt != torch.float32 else 2 ** 31) // row
    pages = beyond + 64
    kc, vc = (torch.empty(pages, page, KV, D, dtype=dt, device=device) for _ in range(2))
    numbers = [pages - 1, 3, beyond // 2 + 5, beyond, pages - 7, beyond - 1, beyond // 2 - 1]
    table = torch.tensor([numbers, numbers[4:] + numbers[:4]], dtype=torch.int32, device=device)
    context = [55, 40]  # the first four pages, and the other three
    k, v = (util.randn(95, KV, D, seed=75 + i).to(dt) for i in range(2))
    args = (kc, vc, table, torch.tensor(context, dtype=torch.int32, device=device))
    append(k.to(device), v.to(device), *args, _offsets(context, device))
    for s, (b, c) in enumerate(((0, 55), (55, 40))):
        for x in (0, c // 2, c - 1):
            assert torch.equal(kc[table[s, x // page].long(), x % page].cpu(), k[b + x])
            assert torch.equal(vc[table[s, x // page].long(), x % page].cpu(), v[b + x])
    cache = type("Both", (), dict(context=context, keys=[k[:55], k[55:]], values=[v[:55], v[55:]], key_cache=kc))
    for tokens in ([1, 1], [30, 40]):
        q = util.randn(sum(tokens), 2 * KV, D, seed=77).to(dt)
        got = attend(q.to(device), *args, _offsets(tokens, device))
        ref.check(got, _want(q, cache, tokens, 0, 0, D ** -0.5, dt), f"{tokens}")


@pytest.mark.gpu
def test_no_room_is_refused(device):
    q, k = torch.zeros(2, 4, 64, device=device), torch.zeros(2, 2, 64, device=device)
    lengths = torch.zeros(2, dtype=torch.int32, device=device)
    for pages, blocks in ((0, 3), (3, 0)):
        cache = torch.zeros(pages, 16, 2, 64, device=device)
        table = torch.zeros(2, blocks, dtype=torch.int32, device=device)
        with pytest.raises(ValueError, match="at least one page"):
            attend(q, cache, cache, table, lengths)
        with pytest.raises(ValueError, match="at least one page"):
            append(k, k, cache, cache, table, lengths)


def test_direct_entry_points_check_their_arguments():
    """The extension module behind the calls: numbers, kinds and lengths of its arguments, before the library."""
    from trident_b200 import _fastcall

    for name in ("tb200_window_attention_fwd", "tb200_paged_attention", "tb200_paged_cache_append", "tb200_gated_residual_rms_norm_fwd"):
        entry = getattr(_fastcall, name)
        count = len(_lib.SIGNATURES[name][1])
        for args in ((), (0,) * (count - 1), (0,) * (count + 1), ("x",) * count, (2 ** 70,) * count):
            with pytest.raises((TypeError, OverflowError)):
                entry(*args)
    strides = (1, 1, 1, 1)
    window = _fastcall.tb200_window_attention_fwd
    for bad in ((1, 1, 1), [1, 1, 1, 1], None, (1, 1, 1, "x"), (1, 1, 1, 2 ** 70)):
        with pytest.raises((TypeError, OverflowError)):
            window(8, 8, 8, 8, 8, 1, 2, 2, 8, 16, strides, bad, strides, strides, 4, 0, 1.0, 0, 0)
    assert window(8, 8, 8, 8, 8, 1, 3, 2, 8, 16, strides, strides, strides, strides, 4, 0, 1.0, 0, 0) == -1


def test_library_refuses_before_launch():
    import ctypes

    lib = _lib.load()
    s = (ctypes.c_int64 * 4)(1, 1, 1, 1)

    def call(T=2, n=2, H=4, KV=2, D=64, page=16, max_q=1, max_ctx=10, sinks=0, starts=8, strides=s, ws=0, where=None):
        return lib.tb200_paged_attention(8, 8, 8, 8, 8, 8, starts, where, ws, T, n, H, KV, D, page, 4, 3, 3, strides, s, s, s,
                                         max_q, max_ctx, 0, sinks, 1.0, 0, 0, None)

    assert call(H=3) == -1 and call(D=24) == -2 and call(H=130) == -2 and call(page=0) == -1 and call(max_q=0) == -1
    assert call(max_ctx=-1) == -1 and call(sinks=-1) == -1 and call(T=3, starts=None) == -1 and call(strides=None) == -1
    assert call(n=70000, T=70000) == -2 and call(T=0) == 0
    append_call = lib.tb200_paged_cache_append
    assert append_call(8, 8, 8, 8, 8, 8, 8, 2, 2, 2, 24, 16, 4, 3, 3, s, s, s, s, 0, None) == -2
    assert append_call(8, 8, 8, 8, 8, 8, None, 3, 2, 2, 64, 16, 4, 3, 3, s, s, s, s, 0, None) == -1
    assert append_call(None, 8, 8, 8, 8, 8, 8, 2, 2, 2, 64, 16, 4, 3, 3, s, s, s, s, 0, None) == -1
    assert append_call(8, 8, 8, 8, 8, 8, 8, 2, 2, 2, 64, 16, 4, 3, 3, s, s, None, s, 0, None) == -1


# ------------------------------------------------------------------------------------ contexts beyond the table
def _full(room, beyond, KV, D, page, dtype, device, seed):
    """A sequence whose table is full, its context `beyond` tokens longer, next to one with room left."""
    cache = Cache([room, 50], KV, D, page, dtype, device, seed)
    cache.table = cache.table[:, : room // page].contiguous()
    cache.table_dev = cache.table.to(device)
    cache.context = [room + beyond, 50]
    cache.context_dev = torch.tensor(cache.context, dtype=torch.int32, device=device)
    return cache


@pytest.mark.gpu
@pytest.mark.parametrize("beyond", [0, 1, 30, 500, 2 ** 31 - 97])
@pytest.mark.parametrize("window, sinks", [(None, 0), (40, 3), (5, 0), (200, 130)])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_contexts_beyond_the_table(D, window, sinks, beyond, dtype, device):
    """Tokens keep their positions: they see the keys that the table holds, as far as window and sinks reach."""
    cache = _full(96, beyond, 2, D, 16, dtype, device, 110)
    for new in ([1, 1], [3, 1], [70, 50], [150, 10]):
        q = util.randn(sum(new), 4, D, seed=111).to(dtype)
        got = attend(q.to(device), cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev, _offsets(new, device),
                     max_query_length=max(new), window_size=window, num_sinks=sinks)
        ref.check(got, _want(q, cache, new, window or 0, sinks, D ** -0.5, dtype), f"{new}")
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_long_contexts_beyond_the_table(D, dtype, device):
    """The same where the walk along the keys is cut."""
    cache = _full(4000, 150, 1, D, 16, dtype, device, 112)
    for new in ([1, 1], [200, 5]):
        for window, sinks in ((None, 0), (3000, 5), (160, 1500)):
            q = util.randn(sum(new), 4, D, seed=113).to(dtype)
            got = attend(q.to(device), cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev, _offsets(new, device),
                         max_query_length=max(new), window_size=window, num_sinks=sinks)
            ref.check(got, _want(q, cache, new, window or 0, sinks, D ** -0.5, dtype), f"{new} {window}")


@pytest.mark.gpu
@pytest.mark.parametrize("beyond", [1, 2, 6, 500, 2 ** 31 - 65])
@pytest.mark.parametrize("D", [16, 64])
def test_append_beyond_the_table(D, beyond, dtype, device):
    """Tokens behind the table's last place are left out, and nothing else in the pool changes."""
    cache = _full(64, beyond, 2, D, 16, dtype, device, 114)
    new = [4, 3]
    k, v = (util.randn(7, 2, D, seed=115 + i).to(dtype).to(device) for i in range(2))
    kc, vc = cache.key_cache.clone(), cache.value_cache.clone()
    append(k, v, kc, vc, cache.table_dev, cache.context_dev, _offsets(new, device))
    for got, before, rows in ((kc, cache.key_cache, k), (vc, cache.value_cache, v)):
        want = before.clone()
        at = 0
        for s, t in enumerate(new):
            for i in range(t):
                pos = cache.context[s] - t + i
                if pos < 64:
                    want[cache.table[s, pos // 16].long(), pos % 16] = rows[at + i]
            at += t
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


# ------------------------------------------------------------------------------------ rows that are not computed
def _poisoned(call, shape, dtype, device):
    """`call`, with NaN in the memory that its output is most likely made from."""
    block = torch.full(shape, float("nan"), dtype=dtype, device=device)
    torch.cuda.synchronize()
    del block
    return call()


@pytest.mark.gpu
@pytest.mark.parametrize("new, at, tokens", [([4, 6], 9, 40), ([1, 1], 5, 8), ([1, 1], 300, 302), ([150, 70], 1, 600), ([0, 3], 200, 203)])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_rows_before_the_first_sequence(D, new, at, tokens, dtype, device):
    cache = Cache([160, 75], 2, D, 16, dtype, device, seed=120)
    q = util.randn(tokens, 4, D, seed=121).to(dtype).to(device)
    offsets = _offsets(new, device) + at
    last = at + sum(new)
    want = _want(q[at:last].cpu(), cache, new, 20, 2, D ** -0.5, dtype)

    def call(**more):
        return attend(q, cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev, offsets,
                      max_query_length=max(new), window_size=20, num_sinks=2, **more)

    got = _poisoned(call, q.shape, dtype, device)
    ref.check(got[at:last], want, "rows of the sequences")
    assert torch.all(got[:at] == 0) and torch.all(got[last:] == 0)
    mine = torch.full_like(q, 5.0)
    call(output=mine)
    assert torch.equal(mine[at:last], got[at:last]) and torch.all(mine[:at] == 5.0) and torch.all(mine[last:] == 5.0)


@pytest.mark.gpu
@pytest.mark.parametrize("longest", [1, 5, 40, 100])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_rows_beyond_max_query_length(D, longest, dtype, device):
    """A sequence's first max_query_length tokens are computed, at their positions among all of its tokens."""
    new = [3, 60, 1, 200, 0, 41] * 8
    cache = Cache([t + 30 for t in new], 1, D, 16, dtype, device, seed=122)
    q = util.randn(sum(new) + 3, 4, D, seed=123).to(dtype)
    kept = torch.cat([torch.arange(t) < longest for t in new] + [torch.zeros(3, dtype=torch.bool)])
    value, bound = _want(q[:-3], cache, new, 50, 1, D ** -0.5, dtype)

    def call(**more):
        return attend(q.to(device), cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev, _offsets(new, device),
                      max_query_length=longest, window_size=50, num_sinks=1, **more)

    got = _poisoned(call, q.shape, dtype, device).cpu()
    ref.check(got[kept], (value[kept[:-3]], bound[kept[:-3]]), "rows that are computed")
    assert torch.all(got[~kept] == 0)
    mine = torch.full_like(q.to(device), 5.0)
    call(output=mine)
    assert torch.equal(mine.cpu()[kept], got[kept]) and torch.all(mine.cpu()[~kept] == 5.0)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [16, 64, 128])
def test_error_of_long_sums(D, device):
    """fp32 values of one sign with equal weights, walks of 2^16 keys that are not cut (many sequences on the same pages):
    partial sums grow along the walk. Each addition is off by e / sqrt(3) of the sum at most in the mean (e = 2^-24), so
    a sum per 64 keys and their sum are off by about sqrt(n / 64) e / 3, one running sum by sqrt(n) e / 3. The
    bound is between the two: sqrt(n / 64) e, and 4 e for the division and the last rounding."""
    n, sequences, page = 2 ** 16, 600, 256
    v = util.randn(n, D, seed=130) + 6.0
    vc = v.view(n // page, page, 1, D).to(device)
    table = torch.arange(n // page, dtype=torch.int32, device=device).expand(sequences, -1)
    lengths = torch.full((sequences,), n, dtype=torch.int32, device=device)
    got = attend(torch.zeros(sequences, 1, D, device=device), torch.ones_like(vc), vc, table, lengths)
    want = v.double().mean(0)
    off = (got[0, 0].double().cpu() / want - 1).square().mean().sqrt() / 2.0 ** -24
    assert off < (n / 64) ** 0.5 + 4, off


# ------------------------------------------------------------------------------------ listed pieces of work
def _tokens_of_few(new, KV, G, D, dtype, device, seed):
    """Many sequences on the pages of a small pool: (arguments of the call, longest, one that checks given sequences)."""
    n, page, pages = len(new), 8, 64
    blocks = 5
    g = util.seeded(seed)
    kc, vc = (torch.randn(pages, page, KV, D, generator=g).to(dtype) for _ in range(2))
    table = torch.randint(0, pages, (n, blocks), generator=g, dtype=torch.int32)
    context = torch.randint(0, blocks * page + 1, (n,), generator=g, dtype=torch.int32)
    q = torch.randn(sum(new), KV * G, D, generator=g).to(dtype)
    offsets = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)

    def check(got, sequences, window, sinks):
        for s in sequences:
            c, (a, b) = int(context[s]), offsets[s:s + 2].tolist()
            if a == b:
                continue
            rows = [t[table[s].long()].flatten(0, 1)[:c] for t in (kc, vc)]
            one = type("One", (), dict(context=[c], keys=[rows[0]], values=[rows[1]], key_cache=kc))
            ref.check(got[a:b], _want(q[a:b], one, [b - a], window, sinks, D ** -0.5, dtype), f"sequence {s}")

    return [t.to(device) for t in (q, kc, vc, table, context, offsets)], max(new), check


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 300, 1025, 5000])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_one_long_chunk_among_many_sequences(D, n, dtype, device):
    """Most pieces of work that the longest chunk plans for every sequence are empty: they are listed first. The same
    results as announced exactly; rows of no sequence and beyond the longest length as ever."""
    new = _random(0, 4, n, 140)
    new[-1] = 0
    new[n // 2] = 3000
    args, longest, check = _tokens_of_few(new, 2, 4, D, dtype, device, 141)
    got = attend(*args, window_size=30, num_sinks=2)
    check(got, sorted({0, 1 % n, n // 2, max(n - 2, 0), n - 1}), 30, 2)
    assert torch.equal(got, attend(*args, max_query_length=longest, window_size=30, num_sinks=2))
    short = _poisoned(lambda: attend(*args, max_query_length=1000, window_size=30, num_sinks=2), got.shape, dtype, device)
    at = sum(new[: n // 2])
    assert torch.equal(short[: at + 1000], got[: at + 1000]) and torch.equal(short[at + 3000:], got[at + 3000:])
    assert torch.all(short[at + 1000: at + 3000] == 0)
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_more_planned_pieces_than_31_bits(dt, device):
    """60000 sequences of 0 to 6 tokens whose longest is not announced."""
    new = _random(0, 7, 60000, 142)
    new[7] = 0
    args, longest, check = _tokens_of_few(new, 1, 64 if dt == torch.bfloat16 else 16, 64, dt, device, 143)
    args[0] = args[0].contiguous()
    got = attend(*args)
    check(got, (0, 1, 7, 30011, 59998, 59999), 0, 0)
    assert torch.equal(got, attend(*args, max_query_length=longest))
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_listed_pieces_in_a_graph(device):
    """The list is made anew at every replay: offsets and contexts may change."""
    dt = torch.bfloat16
    args, _, check = _tokens_of_few([1500] + [1] * 300, 2, 4, 64, dt, device, 144)
    attend(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend(*args)
    for new in ([1] * 300 + [1500], [6] * 300 + [0], [0] * 300 + [1800]):
        args[5].copy_(_offsets(new, device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[: sum(new)], attend(*args)[: sum(new)])
    assert _lib.device_status() == 0


# ------------------------------------------------------------------------------------ what is written
def test_expanded_tensors_are_not_written():
    args = _cpu_call()
    one = torch.randn(3, 1, 16)
    with pytest.raises(ValueError, match="output should not be expanded"):
        attend(**args, output=one.expand(3, 4, 16))
    del args["query"]
    k = torch.randn(3, 2, 16)
    for name in ("key_cache", "value_cache"):
        for shape in ((1, 8, 2, 16), (5, 8, 1, 16)):
            with pytest.raises(ValueError, match=f"{name} should not be expanded"):
                append(k, k, **{**args, name: torch.zeros(shape).expand(5, 8, 2, 16)})
    with pytest.raises(_lib.Tb200Error, match="CUDA tensors only"):  # (a dimension of one may have any stride)
        append(k[:, :1], k[:, :1], **{**args, "key_cache": torch.zeros(5, 8, 16).unsqueeze(2).as_strided((5, 8, 1, 16), (128, 16, 0, 1)),
                                     "value_cache": torch.zeros(5, 8, 1, 16)})


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
def test_output_may_be_the_query(D, dtype, device):
    """Each row is read by the pieces of work that write it, before they do."""
    for new in ([1, 1], [3, 200]):
        cache = Cache([2500, 300], 2, D, 16, dtype, device, seed=150)
        q = util.randn(sum(new), 8, D, seed=151).to(dtype)
        mine = q.to(device)
        attend(mine, cache.key_cache, cache.value_cache, cache.table_dev, cache.context_dev, _offsets(new, device),
               max_query_length=max(new), output=mine)
        ref.check(mine, _want(q, cache, new, 0, 0, D ** -0.5, dtype), f"{new}")
