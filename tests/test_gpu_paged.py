"""Paged decode attention on the GPU against 64-bit attention over the decoded pages."""
import math

import pytest
import torch

from paged_util import assert_attention, attention64, make_pool, make_tables, planes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def F():
    import bitcache_amd
    from bitcache_amd import functional
    bitcache_amd._require_extension()
    return functional


@pytest.fixture(autouse=True)
def shared_kernel(monkeypatch):
    """The shared prefix's kernel at the tests' sizes too."""
    monkeypatch.setenv("BITCACHE_SHARED", "1")


def rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def setup(seed, lens, H, Hkv, d, page, residual, dtype, shared=0, extra=0, std=1.0, q_std=1.0):
    g = rng(seed)
    tables, n_pages = make_tables(g, lens, page, shared // page, extra)
    blobs = make_pool(g, n_pages, page, Hkv, d, residual, std)
    q = (torch.randn((len(lens), H, d), generator=g, device="cuda") * q_std).to(dtype)
    return q, blobs, tables, torch.tensor(lens, dtype=torch.int32, device="cuda")


def check(F, q, blobs, tables, lens, page, hkv, max_len, shared=0, what=""):
    got = F.paged_attention(q, *blobs, tables, lens, max_len, page, n_kv_heads=hkv, shared_len=shared)
    assert got.shape == q.shape and got.dtype == q.dtype
    ref, size = attention64(q, blobs, tables, lens, page, hkv)
    assert_attention(got, ref, size, what)
    return got


LENS = [0, 1, 63, 64, 65, 127, 128, 129, 700]


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,Hkv,d,page", [(8, 2, 128, 64), (4, 4, 128, 128), (8, 1, 64, 64), (2, 1, 256, 192),
                                          (3, 1, 96, 64), (6, 2, 32, 64), (16, 1, 128, 64), (4, 1, 160, 64),
                                          (4, 2, 192, 128), (5, 5, 224, 64), (8, 4, 256, 64), (8, 8, 64, 256)])
def test_ragged(F, H, Hkv, d, page, residual, dtype):
    q, blobs, tables, lens = setup(d + H, LENS, H, Hkv, d, page, residual, dtype, extra=2)
    got = check(F, q, blobs, tables, lens, page, Hkv, 700)
    assert bool((got[0] == 0).all())
    # a larger bound plans another launch for the same sequences
    check(F, q, blobs, tables, lens, page, Hkv, tables.shape[1] * page)


@pytest.mark.parametrize("B,lo,hi,H,Hkv,d,page,residual", [
    (1, 30011, 30011, 8, 2, 128, 64, True), (1, 1, 1, 8, 8, 128, 64, True), (3, 5000, 20000, 4, 1, 64, 256, True),
    (40, 1, 3000, 8, 2, 128, 64, True), (200, 0, 300, 4, 4, 64, 64, False), (70, 64, 2000, 8, 1, 256, 64, True),
    (5, 9000, 9100, 8, 8, 128, 128, False), (300, 1, 70, 2, 2, 128, 64, True)])
def test_lengths_and_batches(F, B, lo, hi, H, Hkv, d, page, residual):
    r = torch.Generator().manual_seed(B)
    lens = torch.randint(lo, hi + 1, (B,), generator=r).tolist()
    q, blobs, tables, lens = setup(B, lens, H, Hkv, d, page, residual, torch.float16)
    check(F, q, blobs, tables, lens, page, Hkv, hi)


def test_sharp_scores(F):
    """Queries whose softmax rests on a few keys, the largest far above the others."""
    q, blobs, tables, lens = setup(4, [5000, 64, 321, 1500], 8, 2, 128, 64, True, torch.float16, q_std=6.0)
    check(F, q, blobs, tables, lens, 64, 2, 5000)


def test_stale_slots_and_junk_tables(F):
    """Slots behind a sequence's last key hold NaN scales, table entries behind its last page
    are junk: neither is read into a result."""
    q, blobs, tables, lens = setup(6, [65, 1, 100, 0, 64], 8, 2, 128, 64, True, torch.float16, extra=3)
    want = F.paged_attention(q, *blobs, tables, lens, 320, 64, n_kv_heads=2)
    live = torch.zeros(blobs[0].numel() // 36, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens.tolist()):
        s = torch.arange(n, device="cuda")
        for h in range(2):
            live[(tables[b].long()[s // 64] * 2 + h) * 64 + s % 64] = True
    for blob, r in zip(blobs, (False, True, False, True)):
        by, sc = planes(blob, 128, r)
        sc[~live] = float("nan")
        by[~live] = 255
    got = F.paged_attention(q, *blobs, tables, lens, 320, 64, n_kv_heads=2)
    assert torch.equal(got, want)


def test_bad_pages_and_lengths(F):
    """A page outside the pool among a sequence's keys, or a length above the bound or the
    table, gives NaN for that sequence and leaves the others as they are."""
    lens = [200, 300, 70, 128, 0, 900]
    q, blobs, tables, lens = setup(7, lens, 8, 2, 128, 64, True, torch.float16)
    want = F.paged_attention(q, *blobs, tables, lens, 900, 64, n_kv_heads=2)
    n_pages = blobs[0].numel() // 36 // 128
    t2 = tables.clone()
    t2[0, 3] = n_pages            # holds keys 192..199
    t2[1, 0] = -1
    t2[2, 1] = 2 ** 31 - 1
    t2[3, 2] = -7                 # behind its last page
    got = F.paged_attention(q, *blobs, t2, lens, 900, 64, n_kv_heads=2)
    assert bool(torch.isnan(got[:3]).all())
    assert torch.equal(got[3:], want[3:])
    l2 = lens.clone()
    l2[1], l2[2], l2[4] = 901, 2 ** 31 - 1, -5
    got = F.paged_attention(q, *blobs, tables, l2, 900, 64, n_kv_heads=2)
    assert bool(torch.isnan(got[1:3]).all()) and bool((got[4] == 0).all())
    keep = torch.tensor([0, 3, 5], device="cuda")
    assert torch.equal(got[keep], want[keep])
    # a bound above what the table holds
    got = F.paged_attention(q, *blobs, tables[:, :2].contiguous(), lens, 900, 64, n_kv_heads=2)
    assert bool(torch.isnan(got[torch.tensor([0, 1, 5], device="cuda")]).all())
    assert bool(torch.isfinite(got[2:5]).all())


def test_nan_scales_stay_with_their_sequence(F):
    q, blobs, tables, lens = setup(8, [200, 300, 70], 8, 2, 128, 64, True, torch.float16)
    want = F.paged_attention(q, *blobs, tables, lens, 300, 64, n_kv_heads=2)
    _, sc = planes(blobs[2], 128, False)
    sc[(int(tables[1, 2]) * 2 + 1) * 64 + 5] = float("nan")     # a value of head 1
    got = F.paged_attention(q, *blobs, tables, lens, 300, 64, n_kv_heads=2)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    assert torch.equal(got[1, :4], want[1, :4]) and bool(torch.isnan(got[1, 4:]).all())


SHARED = [
    # B, H, Hkv, d, page, prefix, own lengths, residual, dtype
    (4, 8, 2, 128, 64, 640, (1, 200), True, torch.float16),
    (33, 8, 2, 128, 64, 1024, (0, 90), True, torch.float16),
    (17, 4, 4, 128, 128, 2048, (1, 300), True, torch.bfloat16),
    (70, 16, 2, 64, 64, 512, (1, 100), True, torch.float16),
    (20, 8, 1, 256, 64, 512, (5, 80), True, torch.float16),
    (9, 6, 2, 96, 64, 320, (1, 80), True, torch.float16),
    (16, 8, 2, 128, 64, 8192, (1, 40), False, torch.bfloat16),
    (64, 4, 1, 128, 256, 5120, (1, 500), True, torch.float16),
    (2, 2, 2, 128, 64, 64, (1, 10), True, torch.float16),
    (40, 12, 4, 160, 64, 448, (1, 64), True, torch.float16),
    (130, 8, 2, 64, 64, 4096, (1, 20), False, torch.float16),
]


@pytest.mark.parametrize("B,H,Hkv,d,page,prefix,own,residual,dtype", SHARED)
def test_shared_prefix(F, B, H, Hkv, d, page, prefix, own, residual, dtype):
    r = torch.Generator().manual_seed(B)
    lens = (torch.randint(own[0], own[1] + 1, (B,), generator=r) + prefix).tolist()
    lens[0] = prefix              # a sequence of the prefix alone
    q, blobs, tables, lens = setup(B + d, lens, H, Hkv, d, page, residual, dtype, shared=prefix)
    check(F, q, blobs, tables, lens, page, Hkv, max(lens.tolist()), prefix)


def test_shared_prefix_with_shorter_sequences(F):
    """Sequences that end inside the prefix, or hold nothing, beside whole ones; the prefix is
    read from the first row whatever its own length."""
    lens = [0, 1, 64, 500, 1023, 1024, 1025, 1500, 3, 77, 0, 1200, 900, 1024, 65, 2, 1300, 1024]
    for residual in (True, False):
        q, blobs, tables, lens_t = setup(10, lens, 8, 2, 128, 64, residual, torch.float16, shared=1024)
        got = check(F, q, blobs, tables, lens_t, 64, 2, 1500, 1024)
        assert bool((got[0] == 0).all()) and bool((got[10] == 0).all())


def test_shared_prefix_bad_pages(F):
    """A bad page of the prefix spoils every sequence that reads it, one of a sequence's own
    pages that sequence; a length above the bound its own."""
    lens = [1024 + 5 * i for i in range(20)]
    lens[3] = 100
    q, blobs, tables, lens = setup(12, lens, 8, 2, 128, 64, True, torch.float16, shared=1024)
    want = F.paged_attention(q, *blobs, tables, lens, 1200, 64, n_kv_heads=2, shared_len=1024)
    t2 = tables.clone()
    t2[7, 16] = -1
    l2 = lens.clone()
    l2[9] = 1201
    got = F.paged_attention(q, *blobs, t2, l2, 1200, 64, n_kv_heads=2, shared_len=1024)
    bad = torch.zeros(20, dtype=torch.bool, device="cuda")
    bad[7] = bad[9] = True
    assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[~bad], want[~bad])
    t2 = tables.clone()
    t2[:, 5] = 10 ** 6            # keys 320..383
    got = F.paged_attention(q, *blobs, t2, lens, 1200, 64, n_kv_heads=2, shared_len=1024)
    bad[:] = True
    bad[3] = False                # ends before them
    assert bool(torch.isnan(got[bad]).all())
    ref, size = attention64(q[3:4], blobs, tables[3:4], lens[3:4], 64, 2)
    assert_attention(got[3:4], ref, size)


def test_repeatable(F):
    for shared in (0, 1024):
        q, blobs, tables, lens = setup(13, [1024 + 37 * i for i in range(24)], 8, 2, 128, 64, True, torch.float16,
                                       shared=shared)
        a = F.paged_attention(q, *blobs, tables, lens, 2000, 64, n_kv_heads=2, shared_len=shared)
        for _ in range(3):
            assert torch.equal(a, F.paged_attention(q, *blobs, tables, lens, 2000, 64, n_kv_heads=2, shared_len=shared))


@pytest.mark.parametrize("shared", [0, 512])
def test_captured_call_follows_lengths_and_tables(F, shared):
    """Two captured calls in turn with eager ones, lengths and tables moving between replays."""
    lens0 = [512 + 30 * i for i in range(18)]
    q, blobs, tables, lens = setup(14, lens0, 8, 2, 128, 64, True, torch.float16, shared=shared)
    call = lambda x: F.paged_attention(x, *blobs, tables, lens, 1100, 64, n_kv_heads=2, shared_len=shared)  # noqa: E731
    q2 = q.flip(0).contiguous()
    call(q)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in (q, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(x))
        graphs.append(g)
    n_pages = blobs[0].numel() // 36 // 128
    for i in range(4):
        lens.copy_(torch.tensor([max(0, n - 97 * i * (k % 3)) for k, n in enumerate(lens0)], dtype=torch.int32))
        tables[:, shared // 64:] = (tables[:, shared // 64:].clamp(min=0) + i) % n_pages
        for g in graphs:
            g.replay()
        for g in reversed(graphs):
            g.replay()
        torch.cuda.synchronize()
        for x, o in zip((q, q2), outs):
            assert torch.equal(o, call(x))
    ref, size = attention64(q, blobs, tables, lens, 64, 2)
    assert_attention(outs[0], ref, size)


def test_two_streams_at_once(F):
    a = setup(15, [900 + i for i in range(30)], 8, 2, 128, 64, True, torch.float16, shared=512)
    b = setup(16, [1400 - i for i in range(50)], 8, 2, 128, 64, True, torch.float16, shared=512)
    call = lambda s: F.paged_attention(s[0], *s[1], s[2], s[3], 1500, 64, n_kv_heads=2, shared_len=512)  # noqa: E731
    want = [call(a), call(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for st, s in zip(streams, (a, b)):
            with torch.cuda.stream(st):
                got.append(call(s))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])


def test_planes_past_four_gib(F):
    """A pool whose code planes pass 2^32 bytes: keys in its last pages."""
    d, page, n_pages = 256, 256, (1 << 25) // 256 + 64
    n = n_pages * page
    bins = torch.zeros(n * 36, dtype=torch.uint8, device="cuda")
    res = torch.zeros(n * 130, dtype=torch.uint8, device="cuda")
    blobs = [bins, res, bins, res]      # keys and values share a pool
    g = rng(17)
    T = 700
    x = torch.randn((T, 1, d), generator=g, device="cuda").half()
    table = torch.tensor([[n_pages - 1, n_pages // 2 + 7, n_pages - 3]], dtype=torch.int32, device="cuda")
    s = torch.arange(T, device="cuda")
    slots = table[0].long()[s // page] * page + s % page
    F.paged_append(x, x, slots, *blobs, page)
    q = torch.randn((1, 4, d), generator=g, device="cuda").half()
    check(F, q, blobs, table, torch.tensor([T], dtype=torch.int32, device="cuda"), page, 1, T)
    # the same bytes as in a pool of three pages
    small = [torch.zeros(768 * w, dtype=torch.uint8, device="cuda") for w in (36, 130)]
    F.paged_append(x, x, s, small[0], small[1], small[0], small[1], page)
    for b, m, r in ((bins, small[0], False), (res, small[1], True)):
        for p, q2 in zip(planes(b, d, r), planes(m, d, r)):
            assert torch.equal(p[slots], q2[s])


def test_decode_loop_together(F):
    """A served batch: prompts of different lengths appended with rotation, then decode steps
    (norm, rotation, append, attention) over pages, against rings with the same rows."""
    from bitcache_amd import BitCache, PagedBitCache
    B, H, Hkv, d, page, steps, pre = 5, 8, 2, 128, 64, 4, 192
    g = rng(18)
    prompts = [pre + n for n in (0, 1, 63, 64, 200)]
    per = 7
    pool = PagedBitCache(3 + B * per, page, H, d, n_kv_heads=Hkv)
    perm = torch.randperm(3 + B * per, generator=g, device="cuda").to(torch.int32)
    tables = torch.cat([perm[:3].expand(B, 3), perm[3:].view(B, per)], 1).contiguous()
    ang = torch.arange(2000, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
        1e4, -torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
    w = [(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).half() for _ in range(2)]
    qkv = lambda T: torch.randn((T, H + 2 * Hkv, d), generator=g, device="cuda").half()  # noqa: E731
    cut = lambda x: (x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:])  # noqa: E731
    common = qkv(pre)
    rings = []
    for b in range(B):
        own = qkv(prompts[b] - pre)
        x = torch.cat([common, own])
        pos = torch.arange(len(x), device="cuda")
        # the common part goes into the shared pages once, with the first sequence
        s = slice(0 if b == 0 else pre, len(x))
        slots = tables[b].long()[pos // page] * page + pos % page
        q, k, v = cut(x)
        pool.append_rotary(q[s], k[s], v[s], pos[s], slots[s].contiguous(), cos, sin, q_weight=w[0], k_weight=w[1])
        ring = BitCache(1, H, d, 512, n_kv_heads=Hkv)
        _, kr = F.norm_rotary(q, k, pos, cos, sin, q_weight=w[0], k_weight=w[1])
        ring.prefill(kr[None].contiguous(), v[None].contiguous(), layout="bshd")
        rings.append(ring)
    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    for _ in range(steps):
        x = qkv(B)
        q, k, v = cut(x)
        pos = lens.long()
        q1 = pool.append_rotary(q, k, v, pos, pool.slots(tables, pos), cos, sin, q_weight=w[0], k_weight=w[1])
        lens += 1
        out = pool.attend(q1, tables, lens, 512, shared_len=pre)
        apart = pool.attend(q1, tables, lens, 512)
        q2, k2 = F.norm_rotary(q, k, pos, cos, sin, q_weight=w[0], k_weight=w[1])
        assert torch.equal(q1, q2)
        blobs = [pool._k_bin, pool._k_res, pool._v_bin, pool._v_res]
        ref, size = attention64(q1, blobs, tables, lens, page, Hkv)
        assert_attention(out, ref, size)
        assert_attention(apart, ref, size)
        for b in range(B):
            ringed = rings[b].append_attend(k2[b:b + 1].contiguous(), v[b:b + 1].contiguous(), q2[b:b + 1].contiguous())
            assert_attention(ringed, ref[b:b + 1], size[b:b + 1], "ring")


def test_refusals(F):
    q, blobs, tables, lens = setup(19, [100, 200], 8, 2, 128, 64, True, torch.float16)

    def bad(*a, page=64, n_kv_heads=2, shared_len=0, max_len=256, blobs=blobs):
        with pytest.raises(RuntimeError):
            F.paged_attention(a[0], *blobs, a[1], a[2], max_len, page, n_kv_heads=n_kv_heads, shared_len=shared_len)

    bad(q.float(), tables, lens)
    bad(q[:, :, ::2], tables, lens)
    bad(q.transpose(0, 1).contiguous().transpose(0, 1), tables, lens)
    bad(q, tables.long(), lens)
    bad(q, tables, lens.long())
    bad(q, tables[:1], lens)
    bad(q, tables, lens[:1])
    bad(q, tables.t().contiguous().t(), lens)
    bad(q, tables.cpu(), lens)
    bad(q, tables, lens, n_kv_heads=3)
    bad(q, tables, lens, page=32)
    bad(q, tables, lens, page=0)
    bad(q, tables, lens, shared_len=32)
    bad(q, tables, lens, shared_len=-64)
    bad(q, tables, lens, shared_len=320)
    bad(q, tables, lens, max_len=-1)
    bad(q, tables, lens, max_len=2 ** 31)
    bad(q, tables, lens, max_len=64, shared_len=128)
    bad(q, tables, lens, blobs=[blobs[0], None, blobs[2], blobs[3]])
    bad(q, tables, lens, blobs=[blobs[0].cpu()] + blobs[1:])
    bad(q, tables, lens, blobs=[blobs[0][:-36].clone()] + blobs[1:])
    bad(q.clone().requires_grad_(), tables, lens)
    e = F.paged_attention(q[:0], *blobs, tables[:0], lens[:0], 256, 64, n_kv_heads=2)
    assert e.shape == (0, 8, 128)


@pytest.mark.parametrize("residual,B", [(True, 24), (False, 2), (True, 2)])
def test_shared_prefix_by_its_size(F, monkeypatch, residual, B):
    """The rule's own choice, and both ways by force: each within the bound."""
    own = [1 + 37 * i for i in range(B)]
    lens = [2560 + n for n in own]
    q, blobs, tables, lens_t = setup(40 + B, lens, 16, 16, 256, 64, residual, torch.bfloat16, shared=2560)
    for choice in (None, "0", "1"):
        monkeypatch.delenv("BITCACHE_SHARED") if choice is None else monkeypatch.setenv("BITCACHE_SHARED", choice)
        check(F, q, blobs, tables, lens_t, 64, 16, max(lens), shared=2560, what=f"choice {choice}")


def test_slots_outside_the_tables(F):
    """Positions and pages that do not exist are padding, not an index error on the device."""
    import bitcache_amd
    pool = bitcache_amd.PagedBitCache(4, 64, 2, 64)
    tables = torch.tensor([[2, 0], [-1, 3], [1, 9], [3, 1], [0, 1]], dtype=torch.int32, device="cuda")
    at = torch.tensor([65, 3, 64, -1, 128], device="cuda")
    assert pool.slots(tables, at).tolist() == [1, -1, -1, -1, -1]
    assert pool.slots(tables[:, :0], at).tolist() == [-1] * 5
    assert pool.slots(tables, torch.tensor([127, 64, 0, 63, 0], dtype=torch.int32, device="cuda")).tolist() == \
        [63, 192, 64, 255, 0]


@pytest.mark.parametrize("shared", [0, 640])
def test_queries_at_odd_elements(F, shared):
    """Contiguous queries that start at any element of their storage."""
    lens = [641 + 50 * i for i in range(6)]
    q, blobs, tables, lens_t = setup(50, lens, 8, 2, 128, 64, True, torch.float16, shared=shared)
    odd = torch.empty(q.numel() + 3, dtype=q.dtype, device="cuda")[3:].view(q.shape)
    odd.copy_(q)
    check(F, odd, blobs, tables, lens_t, 64, 2, max(lens), shared=shared)
    with pytest.raises(RuntimeError, match="aligned"):
        moved = torch.empty(blobs[0].numel() + 4, dtype=torch.uint8, device="cuda")[4:]
        F.paged_attention(q, moved, *blobs[1:], tables, lens_t, max(lens), 64, n_kv_heads=2, shared_len=shared)


def test_two_streams_merging_units(F):
    """Calls on two streams, each with its own workspace, and the same calls alone."""
    calls = []
    for seed in (60, 61):
        lens = [100 + 333 * i for i in range(20)]
        q, blobs, tables, lens_t = setup(seed, lens, 8, 2, 128, 64, True, torch.float16)
        calls.append(lambda q=q, b=blobs, t=tables, n=lens_t: F.paged_attention(q, *b, t, n, 7000, 64, n_kv_heads=2))
    alone = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        got = []
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(c())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, got))


@pytest.mark.parametrize("B,H,Hkv,d,residual", [(700, 2, 1, 64, True), (641, 2, 2, 32, False), (300, 8, 8, 64, True)])
def test_large_batches(F, B, H, Hkv, d, residual):
    """Batches whose units are equal ones of every sequence, several of long sequences; a bad
    page, and a length over the bound, give NaN there alone; with a shared prefix too."""
    lens = [(37 * i) % 400 for i in range(B)]
    lens[3], lens[B - 1], lens[64] = 16385, 20000, 33000
    q, blobs, tables, lens_t = setup(B, lens, H, Hkv, d, 64, residual, torch.float16)
    want = check(F, q, blobs, tables, lens_t, 64, Hkv, 40000)
    tables[3, 200], lens_t[65] = -7, 40001
    got = F.paged_attention(q, *blobs, tables, lens_t, 40000, 64, n_kv_heads=Hkv)
    assert bool(torch.isnan(got[3]).all()) and bool(torch.isnan(got[65]).all())
    rest = torch.ones(B, dtype=torch.bool, device="cuda")
    rest[3] = rest[65] = False
    assert torch.equal(got[rest], want[rest])
    lens = [64 + n for n in lens[:400]]
    if d == 64:
        q, blobs, tables, lens_t = setup(B + 1, lens, H, Hkv, d, 64, residual, torch.float16, shared=64)
        check(F, q, blobs, tables, lens_t, 64, Hkv, 40000, shared=64)
