"""Dense attention over paged caches, append and eviction on the GPU against their 64-bit definitions."""

import itertools
import math

import pytest
import torch

import paged_ref as ref
from paged_ref import D, Cache
from pqhsa_release_b200 import PagedAttention

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def layer(cache, G, T=1, **kw):
    att = PagedAttention(num_query_heads=cache.H * G, num_kv_heads=cache.H, max_requests=len(cache.lens), token_capacity=cache.cap,
                         dtype=cache.dtype, device="cuda", max_query_len=T, **kw)
    att.bind_kv_paged(cache.kv, cache.table)
    return att


def queries(cache, G, T, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(len(cache.lens), T, cache.H * G, D, generator=g).to(cache.dtype).cuda()


def check(out, lse, want, what=""):
    o, z, _, tol, ds = want
    bad = ~((out.double() - o).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((out.double() - o).abs() / tol).nan_to_num(9e9).max()):.3g} x tolerance"
    if lse is not None:
        empty = torch.isinf(z)
        assert torch.equal(torch.isneginf(lse), empty), f"{what}: empty rows"
        off = (lse.double() - z).abs()[~empty]
        assert (off <= ds[~empty] * 2 + 2.0**-21 + 2.0**-22 * z[~empty].abs()).all(), f"{what}: lse off by {float(off.max()):.3g}"


def run(cache, G, T, seed=1, first=None, key_pos=None, query_pos=None, mass=False, **kw):
    """One call against the definition; returns what the call gave."""
    q = queries(cache, G, T, seed)
    slopes = kw.get("alibi_slopes")
    att = layer(cache, G, T, **kw)
    B = len(cache.lens)
    lse = torch.full((B, T, cache.H * G), 7.0, device="cuda")
    m = torch.rand(B, cache.H, cache.cap, device="cuda") if mass else None
    m0 = m.clone() if mass else None
    ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")
    out = att.forward(q, cache.seq_lens, lse=lse, first_key=ints(first), key_pos=key_pos, query_pos=ints(query_pos), mass=m)
    want = ref.attend(cache, q, kw.get("scale"), kw.get("softcap", 0.0), slopes, kw.get("window", 0), kw.get("sink_tokens", 0), first,
                      key_pos, query_pos)
    check(out, lse, want)
    if mass:
        for r, n in enumerate(cache.lens):
            n = max(n, 0)
            for h in range(cache.H):
                w = want[2][r][h]
                # a weight is off by its score's error and its exponential, the sum by half a step of fp32 per row
                ds = float(want[4][r, :, h * G : (h + 1) * G].max())
                tol = w * (2 * ds + 2.0**-20) + (m0[r, h, :n].double() + w) * 2.0**-24 * (G * T + 1) + 1e-30
                off = (m[r, h, :n].double() - m0[r, h, :n].double() - w).abs()
                assert (off <= tol).all(), f"mass of request {r}, head {h}: off by {float((off / tol).max()):.3g} x tolerance"
                assert torch.equal(m[r, h, :n][w == 0], m0[r, h, :n][w == 0])
                assert torch.equal(m[r, h, n:], m0[r, h, n:])
    return att, q, out, lse, m


LENS = [[1], [2, 17, 0, 16], [513, 100, 1029], [3000]]


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout,block", [("rows", 16), ("heads", 16), ("heads", 7), ("rows", 1), ("heads", 128)])
@pytest.mark.parametrize("lens", LENS, ids=["one", "tiny", "ragged", "long"])
def test_plain(dtype, layout, block, lens):
    run(Cache(lens, 2, dtype, block, layout), 4, 1)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("G,T,H", [(1, 1, 3), (3, 1, 2), (5, 2, 1), (8, 1, 1), (8, 2, 2), (7, 3, 1), (4, 8, 2), (8, 8, 1), (5, 8, 2),
                                   (16, 4, 1), (13, 1, 1), (6, 6, 1)])
def test_groups_and_tokens(dtype, G, T, H):
    run(Cache([300, 5, 700], H, dtype, 16, "heads", seed=G), G, T, mass=True)


FEATURES = {
    "cap": dict(softcap=20.0), "alibi": dict(alibi=True), "window": dict(window=100), "window_sinks": dict(window=50, sink_tokens=4),
    "window_one": dict(window=1), "documents": dict(first=True), "documents_window": dict(first=True, window=33, sink_tokens=20),
    "all": dict(softcap=5.0, alibi=True, window=200, sink_tokens=3, first=True), "scale": dict(scale=-0.3), "scale0": dict(scale=0.0),
}


@pytest.mark.parametrize("name", FEATURES)
@pytest.mark.parametrize("dtype,T", [(BF, 1), (HF, 4), (F32, 1), (F32, 3), (BF, 8)], ids=["bf16", "fp16x4", "fp32", "fp32x3", "bf16x8"])
def test_features(name, dtype, T):
    kw = dict(FEATURES[name])
    lens = [1, 40, 1000, 333, 0]
    first = [0, 39, 500, 400, 2] if kw.pop("first", False) else None
    if kw.pop("alibi", False):
        kw["alibi_slopes"] = torch.exp2(-torch.arange(1, 9, device="cuda").float())
    run(Cache(lens, 2, dtype, 16, "rows"), 4, T, first=first, mass=True, **kw)


def shuffled_positions(cache, seed=5, stride=3):
    g = torch.Generator().manual_seed(seed)
    pos = torch.empty(len(cache.lens), cache.H, cache.cap, dtype=torch.int32)
    for r, h in itertools.product(range(len(cache.lens)), range(cache.H)):
        pos[r, h] = stride * torch.randperm(cache.cap, generator=g).int() + torch.randint(0, stride, (cache.cap,), generator=g).int()
    return pos.cuda()


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("kw", [{}, dict(window=700, sink_tokens=9), dict(alibi=True)], ids=["plain", "window", "alibi"])
def test_stored_positions(dtype, T, kw):
    kw = dict(kw)
    cache = Cache([900, 33, 1, 0, 400], 2, dtype, 13, "heads")
    pos = shuffled_positions(cache)
    pos[0, 0, 5] = -1  # a hole is never seen
    if kw.pop("alibi", False):
        kw["alibi_slopes"] = torch.exp2(-torch.arange(1, 7, device="cuda").float()) * 0.1
    # some keys lie behind the query's position
    run(cache, 3, T, key_pos=pos, query_pos=[2500, 60, 10000, 5, 1200], first=[0, 7, 0, 0, 300], mass=True, **kw)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T", [1, 4])
@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf])
def test_what_no_token_sees_stays_out(dtype, T, junk):
    """Slots behind the end, before the document, outside the window, and keys behind an early token of the step."""
    lens, first, window, sinks = [400, 77, 20], [100, 0, 19], 64, 3
    cache = Cache(lens, 2, dtype, 16, "heads")
    clean = cache.kv.clone()
    q = queries(cache, 4, T)
    args = dict(window=window, sinks=sinks, first=first)
    want = ref.attend(cache, q, **args)
    for r, n in enumerate(lens):
        seen = torch.zeros(cache.cap, dtype=torch.bool)
        for t in range(T):
            seen[:n] |= ref.visible(torch.arange(n), n - T + t, first[r], window, sinks)
        for h, i in itertools.product(range(2), (~seen).nonzero().view(-1).tolist()):
            row = torch.full((D,), junk)
            cache.put(r, h, i, row, row)
    assert not torch.equal(cache.kv, clean)
    att = layer(cache, 4, T, window=window, sink_tokens=sinks)
    lse = torch.empty(q.shape[:-1], device="cuda")
    out = att.forward(q, cache.seq_lens, lse=lse, first_key=torch.tensor(first, dtype=torch.int32, device="cuda"))
    check(out, lse, want)


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("window", [0, 40])
def test_a_later_tokens_row_does_not_reach_an_earlier_one(dtype, window):
    """Speculative tokens: infinite values at the last key reach the last token alone; with a window, those at the
    first key of the first token's window reach the first token alone."""
    T, n = 4, 200
    cache = Cache([n], 1, dtype, 16, "rows")
    q = queries(cache, 2, T)
    want = ref.attend(cache, q, window=window)
    _, v = cache.views()
    blk = lambda i: int(cache.table[0, i // 16])
    v[blk(n - 1), (n - 1) % 16, 0] = math.inf
    if window:
        low = n - T - window + 1
        v[blk(low), low % 16, 0] = math.nan
    out = layer(cache, 2, T, window=window).forward(q, cache.seq_lens)
    lo = 1 if window else 0
    check(out[:, lo : T - 1], None, tuple(x[:, lo : T - 1] if torch.is_tensor(x) else x for x in want))
    assert bool((out[:, T - 1] == math.inf).all())
    if window:
        assert bool(out[:, 0].isnan().all())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_nan_in_a_seen_key_shows(dtype):
    cache = Cache([100, 100], 1, dtype, 16, "rows")
    k, _ = cache.views()
    k[int(cache.table[0, 3]), 5, 0, 0] = math.nan
    q = queries(cache, 4, 1)
    mass = torch.zeros(2, 1, cache.cap, device="cuda")
    out = layer(cache, 4).forward(q, cache.seq_lens, mass=mass)
    assert bool(out[0].isnan().all()) and bool(torch.isfinite(out[1].float()).all())
    assert bool(mass[0, 0, :100].isnan().all()) and bool((mass[0, 0, 100:] == 0).all())


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_missing_pages_and_lengths_past_the_end(dtype):
    cache = Cache([100, 60], 2, dtype, 16, "heads")
    q = queries(cache, 4, 1)
    before = ref.attend(cache, q)
    cache.table[0, 2], cache.table[0, 4] = -1, 1 << 30
    att = layer(cache, 4)
    mass = torch.zeros(2, 2, cache.cap, device="cuda")
    out = att.forward(q, cache.seq_lens, mass=mass)
    pos = torch.arange(cache.cap, dtype=torch.int32, device="cuda").repeat(2, 2, 1)
    pos[0, :, 32:48] = pos[0, :, 64:80] = -1
    cache.table[0, 2] = cache.table[0, 4] = 0
    want = ref.attend(cache, q, key_pos=pos, query_pos=[99, 59])
    check(out, None, want)
    check(out[1:], None, tuple(x[1:] for x in before))
    assert bool((mass[0, :, 32:48] == 0).all()) and bool((mass[0, :, 64:80] == 0).all())
    # a length past the block table is clamped to it, a negative one is idle
    lens = torch.tensor([1 << 30, -5], dtype=torch.int32, device="cuda")
    cache.lens = [cache.cap, 0]
    out = att.forward(q, lens)
    check(out, None, ref.attend(cache, q))
    assert bool((out[1] == 0).all())


def test_strided_rows_and_contiguous_cache():
    g = torch.Generator(device="cuda").manual_seed(3)
    B, H, G, T, S = 3, 2, 4, 2, 150
    qkv = torch.randn(B, T, H * (G + 2), D, generator=g, device="cuda").to(BF)  # q is a slice of a fused projection
    keys, values = torch.randn(2, B, S, H, D, generator=g, device="cuda").to(BF).permute(0, 1, 3, 2, 4)
    att = PagedAttention(num_query_heads=H * G, num_kv_heads=H, max_requests=B, token_capacity=S, dtype=BF, device="cuda", max_query_len=T)
    att.bind_kv_contiguous(keys, values)
    cache = Cache([S, 3, 77], H, BF, S, "rows", room=S)
    cache.kv = torch.stack([keys.transpose(1, 2), values.transpose(1, 2)])
    cache.table = torch.arange(B, dtype=torch.int32, device="cuda").view(B, 1)
    q = qkv[:, :, : H * G]
    big = torch.full((B, T, 2 * H * G, D), 5.0, dtype=BF, device="cuda")
    out = att.forward(q, cache.seq_lens, out=big[:, :, H * G :])
    check(out, None, ref.attend(cache, q))
    assert bool((big[:, :, : H * G] == 5).all())
    one = att.forward(q[:, 1], cache.seq_lens)
    check(one[:, None], None, ref.attend(cache, q[:, 1:2]))


def test_offsets_past_32_bits():
    """Pages at the far end of a cache of more than 2^32 elements."""
    H, bs = 8, 16
    per = bs * H * 2 * D
    blocks = (1 << 32) // per + 64
    kv = torch.empty(blocks, H, bs, 2 * D, dtype=BF, device="cuda")
    small = Cache([600, 40], H, BF, bs, "heads")
    far = torch.arange(blocks - small.kv.shape[0], blocks, device="cuda")
    kv[far] = small.kv
    q = queries(small, 4, 1)
    want = ref.attend(small, q)
    att = PagedAttention(num_query_heads=4 * H, num_kv_heads=H, max_requests=2, token_capacity=small.cap, dtype=BF, device="cuda")
    table = (small.table + (blocks - small.kv.shape[0])).int()
    att.bind_kv_paged(kv, table)
    check(att.forward(q, small.seq_lens), None, want)
    k = torch.randn(2, H, D, device="cuda").to(BF)
    att.append(k, k, small.seq_lens)
    assert torch.equal(kv[table[0, 600 // bs].long(), :, 600 % bs, D:], k[0])
    del kv


def test_many_requests_share_the_grid():
    lens = [(37 * i) % 91 for i in range(300)]
    run(Cache(lens, 2, BF, 16, "heads", room=96), 4, 1, mass=True)
    run(Cache(lens[:70], 1, F32, 16, "heads", room=96), 8, 1)


def test_same_bits_every_run():
    cache = Cache([4000, 10, 2500], 2, BF, 16, "heads")
    q = queries(cache, 4, 1)
    att = layer(cache, 4)
    got = []
    for _ in range(5):
        mass = torch.zeros(3, 2, cache.cap, device="cuda")
        got.append((att.forward(q, cache.seq_lens, mass=mass), mass))
    for o, m in got[1:]:
        assert torch.equal(o, got[0][0]) and torch.equal(m, got[0][1])


def test_two_streams_and_captured_calls():
    cache = Cache([3000, 500], 2, BF, 16, "heads")
    q1, q2 = queries(cache, 4, 1, 1), queries(cache, 4, 1, 2)
    att = layer(cache, 4)
    w1, w2 = ref.attend(cache, q1), ref.attend(cache, q2)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(s1):
            o1 = att.forward(q1, cache.seq_lens)
        with torch.cuda.stream(s2):
            o2 = att.forward(q2, cache.seq_lens)
    torch.cuda.synchronize()
    check(o1, None, w1)
    check(o2, None, w2)
    # two graphs of one layer, replayed at the same time; lengths change between replays
    outs, graphs = [], []
    for q in (q1, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(att.forward(q, cache.seq_lens, mass=None))
        graphs.append(g)
    for _ in range(20):
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
    torch.cuda.synchronize()
    check(outs[0], None, w1)
    check(outs[1], None, w2)
    cache.lens = [77, 2]
    cache.seq_lens.copy_(torch.tensor(cache.lens, dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    check(outs[0], None, ref.attend(cache, q1))


# ---- append ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF, HF, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout,block,T", [("rows", 16, 1), ("heads", 7, 3), ("rows", 1, 8)])
def test_append(dtype, layout, block, T):
    lens = [0, 15, -1, 40]
    cache = Cache([max(n, 0) for n in lens], 3, dtype, block, layout)
    cache.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    att = layer(cache, 2, T)
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(4, T, 3, D, generator=g).to(dtype).cuda() for _ in range(2))
    pos = torch.full((4, 3, cache.cap), -7, dtype=torch.int32, device="cuda")
    mass = torch.full((4, 3, cache.cap), 9.0, device="cuda")
    qp = torch.tensor([100, 200, 300, 400], dtype=torch.int32, device="cuda")
    want, wpos, wmass = cache.kv.clone(), pos.clone(), mass.clone()
    shadow = Cache(cache.lens, 3, dtype, block, layout)
    shadow.kv, shadow.table = want, cache.table
    for r, n in enumerate(lens):
        for t in range(T if n >= 0 else 0):
            wpos[r, :, n + t], wmass[r, :, n + t] = int(qp[r]) - (T - 1) + t, 0.0
            for h in range(3):
                shadow.put(r, h, n + t, k[r, t, h], v[r, t, h])
    new = torch.empty(4, dtype=torch.int32, device="cuda")
    att.append(k, v, cache.seq_lens, new_lens=new, key_pos=pos, query_pos=qp, mass=mass)
    assert torch.equal(cache.kv, want) and torch.equal(pos, wpos) and torch.equal(mass, wmass)
    assert new.tolist() == [n + T if n >= 0 else n for n in lens] and cache.seq_lens.tolist() == lens
    att.append(k, v, cache.seq_lens, key_pos=pos)  # in place; without query_pos a slot is its position
    assert cache.seq_lens.tolist() == new.tolist()
    assert pos[1, 0, 15 : 15 + T].tolist() == list(range(15, 15 + T))
    assert torch.equal(cache.kv, want)


def test_append_past_the_end_is_dropped():
    cache = Cache([30], 1, BF, 16, "rows", room=32)
    att = layer(cache, 1, 4)
    before = cache.kv.clone()
    k = torch.ones(1, 4, 1, D, dtype=BF, device="cuda")
    att.append(k, k, cache.seq_lens)
    assert cache.seq_lens.tolist() == [32]
    kc, _ = cache.rows(0, 0, 32)
    assert bool((kc[30:] == 1).all())
    changed = (cache.kv != before).any(-1)
    assert int(changed.sum()) == 4  # two key and two value rows
    att.append(k, k, cache.seq_lens)
    assert cache.seq_lens.tolist() == [32] and int((cache.kv != before).any(-1).sum()) == 4


# ---- eviction ----------------------------------------------------------------------------------------------


def evict_case(lens, H, dtype, block, layout, budget, recent, sinks, mass, pos, last, inplace, room=None):
    cache = Cache(lens, H, dtype, block, layout, room=room)
    att = layer(cache, 2, sink_tokens=sinks)
    B = len(lens)
    qp = torch.tensor(last, dtype=torch.int32, device="cuda")
    source = torch.full((B, H, budget), -9, dtype=torch.int32, device="cuda")
    kv0, m0, p0 = cache.kv.clone(), mass.clone(), pos.clone()
    extra = {} if inplace else dict(new_lens=torch.empty_like(qp), new_mass=torch.full_like(mass, 3.0), new_pos=torch.full_like(pos, 3))
    lens_t = cache.seq_lens.clone()
    new = att.evict(lens_t, mass=mass, key_pos=pos, query_pos=qp, budget=budget, recent=recent, source=source, **extra)
    nm, npos = (mass, pos) if inplace else (extra["new_mass"], extra["new_pos"])
    if not inplace:
        assert torch.equal(mass.nan_to_num(-3), m0.nan_to_num(-3)) and torch.equal(pos, p0) and lens_t.tolist() == list(lens)
    assert new.tolist() == [min(n, budget) for n in lens]
    shadow = Cache(lens, H, dtype, block, layout, room=room)
    shadow.kv, shadow.table = kv0.clone(), cache.table
    old = Cache(lens, H, dtype, block, layout, room=room)
    old.kv, old.table = kv0, cache.table
    wm, wp = (m0.clone(), p0.clone()) if inplace else (torch.full_like(m0, 3.0), torch.full_like(p0, 3))
    for r, n in enumerate(lens):
        n = max(min(n, cache.cap), 0)
        for h in range(H):
            src = ref.evict(m0[r, h].tolist(), p0[r, h].tolist(), n, budget, sinks, recent, last[r])
            assert source[r, h].tolist() == src + [-1] * (budget - len(src))
            k, v = old.rows(r, h, n)
            at = torch.tensor(src, dtype=torch.long, device="cuda")
            wm[r, h, : len(src)], wp[r, h, : len(src)] = m0[r, h][at], p0[r, h][at]
            for i, j in enumerate(src):
                if i != j:
                    shadow.put(r, h, i, k[j], v[j])
    assert torch.equal(cache.kv, shadow.kv)
    assert torch.equal(nm.nan_to_num(-3), wm.nan_to_num(-3)) and torch.equal(npos, wp)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("layout,block", [("rows", 16), ("heads", 7)])
@pytest.mark.parametrize("inplace", [True, False], ids=["inplace", "apart"])
@pytest.mark.parametrize("budget,recent,sinks", [(64, 10, 4), (1, 0, 0), (40, 36, 4), (500, 100, 0), (2000, 3, 3)])
def test_evict(dtype, layout, block, inplace, budget, recent, sinks):
    lens = [700, 64, 0, 1, 41, 501, -3]
    g = torch.Generator().manual_seed(budget)
    cap = Cache(lens, 2, dtype, block, layout).cap
    mass = torch.rand(7, 2, cap, generator=g)
    mass[torch.rand(7, 2, cap, generator=g) < 0.3] = 0.0
    mass[0, 0, ::7] = 0.25
    mass[0, 1, 3], mass[0, 1, 5], mass[0, 1, 9], mass[0, 1, 600] = math.nan, -0.0, math.inf, math.nan
    mass[5, 0] = 0.5  # all alike: the lowest slots stay
    pos = torch.arange(cap, dtype=torch.int32).repeat(7, 2, 1)
    pos[5, 1, :501] = torch.randperm(501, generator=g).int()
    evict_case(lens, 2, dtype, block, layout, budget, recent, sinks, mass.cuda(), pos.cuda(), [n - 1 for n in lens], inplace)


def test_evict_negative_and_infinite_masses():
    cap = Cache([300], 1, BF, 16, "rows").cap
    for fill in (math.nan, math.inf, -math.inf, -1.0):
        mass = torch.full((1, 1, cap), fill)
        mass[0, 0, 100:200] = torch.linspace(-5, 5, 100)
        evict_case([300], 1, BF, 16, "rows", 128, 5, 2, mass.cuda(), torch.arange(cap, dtype=torch.int32).repeat(1, 1, 1).cuda(), [299], True)


@pytest.mark.parametrize("n,budget", [(20000, 5000), (70001, 69999), (130000, 1000)])
def test_evict_long(n, budget):
    g = torch.Generator().manual_seed(n)
    cap = Cache([n, n // 2], 1, BF, 64, "heads").cap
    mass = torch.exp(torch.randn(2, 1, cap, generator=g))
    mass[torch.rand(2, 1, cap, generator=g) < 0.5] = 0.125
    pos = torch.arange(cap, dtype=torch.int32).repeat(2, 1, 1)
    evict_case([n, n // 2], 1, BF, 64, "heads", budget, 64, 4, mass.cuda(), pos.cuda(), [n - 1, n // 2 - 1], True)


def test_evict_past_what_shared_memory_holds():
    """More slots than the eight CTAs of a cluster keep: every sweep makes the keys again."""
    n, budget = 400_001, 300
    g = torch.Generator().manual_seed(1)
    cap = Cache([n], 1, BF, 64, "heads").cap
    mass = torch.exp(torch.randn(1, 1, cap, generator=g))
    mass[0, 0, ::3] = 20.0
    pos = torch.arange(cap, dtype=torch.int32).repeat(1, 1, 1)
    evict_case([n], 1, BF, 64, "heads", budget, 16, 4, mass.cuda(), pos.cuda(), [n - 1], True)


# ---- extremes and refusals --------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_extreme_windows_and_positions(dtype):
    top = 2**31 - 1
    cache = Cache([50, 20], 1, dtype, 16, "heads")
    pos = torch.full((2, 1, cache.cap), top, dtype=torch.int32, device="cuda")
    pos[:, :, ::2] = torch.arange(cache.cap // 2, dtype=torch.int32, device="cuda") * 3
    pos[0, 0, 1], pos[0, 0, 3] = -(2**31), top - 1
    for window, sinks in ((top, 0), (1, 7), (2, top), (0, 0)):
        run(cache, 2, 3, key_pos=pos, query_pos=[top, 30], window=window, sink_tokens=sinks)
    run(cache, 2, 2, window=top, sink_tokens=top)
    run(cache, 2, 1, first=[top, -5])
    run(cache, 2, 2, key_pos=pos, query_pos=[-(2**31), -1])


def test_forward_refusals():
    cache = Cache([10, 10], 2, BF, 16, "rows")
    att = layer(cache, 4, 2)
    q = torch.zeros(2, 8, D, dtype=BF, device="cuda")
    lens = cache.seq_lens
    pos = torch.zeros(2, 2, cache.cap, dtype=torch.int32, device="cuda")
    mass = torch.zeros(2, 2, cache.cap, device="cuda")
    ok = dict(q=q, seq_lens=lens)
    bad = [
        dict(q=q.float()), dict(q=q.cpu()), dict(q=q[:, :7]), dict(q=q[..., :64]), dict(q=torch.zeros(3, 8, D, dtype=BF, device="cuda")),
        dict(q=torch.zeros(2, 3, 8, D, dtype=BF, device="cuda")), dict(q=torch.zeros(2, 8, D + 4, dtype=BF, device="cuda")[..., 4:]),
        dict(q=torch.zeros(2, 8, 2 * D, dtype=BF, device="cuda")[..., ::2]), dict(q=q[0]),
        dict(seq_lens=lens.long()), dict(seq_lens=lens[:1]), dict(seq_lens=lens.cpu()), dict(out=torch.empty(2, 8, D, device="cuda")),
        dict(out=torch.empty(2, 4, D, dtype=BF, device="cuda")), dict(lse=torch.empty(2, 4, device="cuda")),
        dict(lse=torch.empty(2, 8, dtype=BF, device="cuda")), dict(first_key=lens.long()), dict(key_pos=pos), dict(key_pos=pos.long(), query_pos=lens),
        dict(key_pos=pos[:, :, :-1], query_pos=lens), dict(mass=mass.double()), dict(mass=mass[:1]), dict(mass=mass[:, :1]),
    ]
    att.forward(**ok)
    for kw in bad:
        with pytest.raises(ValueError):
            att.forward(**{**ok, **kw})
    free = PagedAttention(num_query_heads=8, num_kv_heads=2, max_requests=2, token_capacity=16, dtype=BF, device="cuda")
    with pytest.raises(RuntimeError, match="bind"):
        free.forward(q, lens)
    for kv, table in [(cache.kv.float(), cache.table), (cache.kv, cache.table.long()), (cache.kv[:1], cache.table), (cache.kv[..., :64], cache.table),
                      (cache.kv[0, 0], cache.table), (cache.kv, cache.table[:, :0]), (cache.kv[:, :, :, :1], cache.table)]:
        with pytest.raises(ValueError):
            free.bind_kv_paged(kv, table)
    with pytest.raises(ValueError):
        free.bind_kv_contiguous(cache.kv[0], cache.kv[0])
    k = torch.zeros(2, 2, D, dtype=BF, device="cuda")
    for kw in (dict(keys=k.float()), dict(values=k[:1]), dict(keys=k[:, :1], values=k[:, :1]), dict(new_lens=lens.long()), dict(mass=mass[:1])):
        with pytest.raises(ValueError):
            att.append(**{**dict(keys=k, values=k, seq_lens=lens), **kw})
    ev = dict(seq_lens=lens, mass=mass, key_pos=pos, query_pos=lens, budget=8)
    for kw in (dict(budget=0), dict(recent=9), dict(recent=-1), dict(mass=mass.double()), dict(key_pos=pos[:1]), dict(query_pos=lens.long()),
               dict(source=torch.zeros(2, 2, 7, dtype=torch.int32, device="cuda")), dict(new_mass=mass[:1]), dict(new_lens=lens[:1])):
        with pytest.raises(ValueError):
            att.evict(**{**ev, **kw})
    torch.cuda.synchronize()


def test_no_requests_and_fewer_than_the_layer_was_made_for():
    cache = Cache([100, 200, 30], 2, BF, 16, "rows")
    att = layer(cache, 4)
    q = queries(cache, 4, 1)
    assert att.forward(q[:0], cache.seq_lens[:0]).shape == (0, 1, 8, D)
    want = ref.attend(cache, q)
    for b in (3, 1, 2, 3):  # workspaces of different sizes in turn
        mass = torch.zeros(3, 2, cache.cap, device="cuda")
        out = att.forward(q[:b], cache.seq_lens[:b], mass=mass if b % 2 else None)
        check(out, None, tuple(x[:b] for x in want))


def test_two_graphs_with_weights_at_once():
    cache = Cache([2000, 700], 2, BF, 16, "heads")
    att = layer(cache, 4)
    qs = [queries(cache, 4, 1, s) for s in (1, 2)]
    masses = [torch.zeros(2, 2, cache.cap, device="cuda") for _ in qs]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in qs]
    for q, m in zip(qs, masses):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(att.forward(q, cache.seq_lens, mass=m))
        graphs.append(g)
    for m in masses:
        m.zero_()
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for q, m, o in zip(qs, masses, outs):
        check(o, None, ref.attend(cache, q))
        one = torch.zeros_like(m)
        att.forward(q, cache.seq_lens, mass=one)
        ten = torch.zeros_like(m)
        for _ in range(10):
            ten += one
        assert torch.equal(m, ten)


@pytest.mark.parametrize("dtype,T", [(BF, 1), (HF, 4), (F32, 1)], ids=["bf16", "fp16x4", "fp32"])
@pytest.mark.parametrize("softcap", [0.02, 1.0, 300.0, 1e5, 1e9, 3e38])
def test_caps_small_and_large_against_the_scores(dtype, T, softcap):
    run(Cache([300, 5, 700], 2, dtype, 16, "heads"), 4, T, softcap=softcap, mass=True)


def test_a_refused_call_leaves_the_next_one_alone():
    cache = Cache([60, 33, 90], 2, BF, 16, "heads")
    q = queries(cache, 4, 1).squeeze(1)
    att = layer(cache, 4, 1)
    want = att.forward(q, cache.seq_lens)
    odd = torch.zeros(1, 8, 2 * D, dtype=BF, device="cuda")[:, :, ::2]  # elements of a row apart
    with pytest.raises(ValueError, match="contiguous"):
        att.forward(odd, cache.seq_lens[:1])
    assert torch.equal(att.forward(q, cache.seq_lens), want)
    k = torch.randn(3, 2, D, device="cuda").to(BF)
    lens = cache.seq_lens - 1  # the last rows are written again
    kept = cache.kv.clone()
    att.append(k, k, lens.clone())
    first = cache.kv.clone()
    cache.kv.copy_(kept)
    with pytest.raises(ValueError, match="contiguous"):
        att.append(odd[:, :2], odd[:, :2], lens[:1].clone())
    att.append(k, k, lens.clone())
    assert torch.equal(cache.kv, first)
