"""norm_rotary and the paged append on the GPU against 64-bit restatements."""
import numpy as np
import pytest
import torch

from paged_util import half_step, online_encode, planes, rotate64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def F():
    import bitcache_amd
    from bitcache_amd import functional
    bitcache_amd._require_extension()
    return functional


def rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def inputs(seed, T, H, Hkv, d, rot, dtype, norm, layout="fused", table=5000):
    g = rng(seed)
    x = (torch.randn((T, H + 2 * Hkv, d), generator=g, device="cuda") *
         torch.exp(0.5 * torch.randn((T, H + 2 * Hkv, 1), generator=g, device="cuda"))).to(dtype)
    if layout == "fused":
        q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    elif layout == "whole":
        q, k, v = (y.contiguous() for y in (x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]))
    elif layout == "odd":    # rows at odd elements: no 16-byte alignment
        buf = torch.empty((T, H + 2 * Hkv, d + 3), dtype=dtype, device="cuda")
        buf[..., 1:d + 1] = x
        x = buf[..., 1:d + 1]
        q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    else:                    # heads outermost
        y = x.transpose(0, 1).contiguous().transpose(0, 1)
        q, k, v = y[:, :H], y[:, H:H + Hkv], y[:, H + Hkv:]
    pos = torch.randint(0, table, (T,), generator=g, device="cuda")
    ang = torch.arange(table, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
        1e4, -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dtype) for _ in range(2))
    return dict(q=q, k=k, v=v, pos=pos, cos=torch.cos(ang).float(), sin=torch.sin(ang).float(),
                wq=wq if norm else None, wk=wk if norm else None)


def reference(x, s, w, eps, inter):
    n = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    return rotate64(n(x), s["pos"].cpu().numpy(), n(s["cos"]), n(s["sin"]), n(w), eps, inter)


def assert_rows(got, ref):
    """Once rounded: half a step (its double rounding through fp32 adds 2^-13 of one)."""
    h = half_step(got.dtype)
    off = np.abs(got.double().cpu().numpy() - ref)
    assert (off <= h * (1 + 2.0 ** -10) * np.abs(ref) + 2.0 ** -25).all(), off.max()


CASES = [
    # T, H, Hkv, d, rot, interleaved, dtype, norm, layout
    (1, 4, 1, 128, 128, False, torch.float16, True, "fused"),
    (7, 8, 2, 128, 128, True, torch.bfloat16, True, "whole"),
    (9, 3, 3, 128, 64, False, torch.float16, True, "odd"),
    (65, 8, 8, 64, 64, False, torch.bfloat16, False, "fused"),
    (300, 12, 4, 96, 96, False, torch.float16, True, "heads"),
    (33, 5, 5, 96, 32, True, torch.float16, False, "fused"),
    (40, 2, 1, 32, 16, False, torch.float16, True, "odd"),
    (17, 4, 2, 256, 256, False, torch.bfloat16, True, "fused"),
    (17, 4, 2, 256, 48, False, torch.float16, True, "heads"),
    (20, 4, 4, 160, 160, False, torch.float16, True, "fused"),
    (20, 4, 4, 192, 128, True, torch.bfloat16, True, "whole"),
    (20, 4, 4, 224, 224, False, torch.bfloat16, True, "fused"),
    (20, 4, 4, 128, 128, False, torch.float16, False, "odd"),
    (2100, 4, 2, 128, 128, False, torch.float16, True, "fused"),
]
IDS = ["-".join(str(x).replace("torch.", "") for x in c) for c in CASES]


@pytest.mark.parametrize("T,H,Hkv,d,rot,inter,dtype,norm,layout", CASES, ids=IDS)
def test_norm_rotary(F, T, H, Hkv, d, rot, inter, dtype, norm, layout):
    s = inputs(T + d, T, H, Hkv, d, rot, dtype, norm, layout)
    before = s["q"].clone()
    q, k = F.norm_rotary(s["q"], s["k"], s["pos"], s["cos"], s["sin"], q_weight=s["wq"], k_weight=s["wk"],
                         eps=1e-5, interleaved=inter)
    assert q.shape == s["q"].shape and k.shape == s["k"].shape and q.is_contiguous() and q.dtype == dtype
    assert_rows(q, reference(s["q"], s, s["wq"], 1e-5, inter))
    assert_rows(k, reference(s["k"], s, s["wk"], 1e-5, inter))
    assert torch.equal(before, s["q"])


def test_parts_of_the_pass(F):
    """Queries alone, norms alone, a norm on one side only, no tokens."""
    s = inputs(3, 21, 6, 2, 128, 128, torch.float16, True)
    q, k = F.norm_rotary(s["q"], None, s["pos"], s["cos"], s["sin"], q_weight=s["wq"])
    assert k is None
    assert_rows(q, reference(s["q"], s, s["wq"], 1e-6, False))
    q, k = F.norm_rotary(s["q"], s["k"], None, None, None, q_weight=s["wq"], k_weight=s["wk"])
    for got, x, w in ((q, s["q"], s["wq"]), (k, s["k"], s["wk"])):
        assert_rows(got, rotate64(x.double().cpu().numpy(), None, None, None, w.double().cpu().numpy(), 1e-6, False))
    q, k = F.norm_rotary(s["q"], s["k"], s["pos"], s["cos"], s["sin"], k_weight=s["wk"])
    assert_rows(q, reference(s["q"], s, None, 1e-6, False))
    assert_rows(k, reference(s["k"], s, s["wk"], 1e-6, False))
    q, k = F.norm_rotary(s["q"][:0], s["k"][:0], s["pos"][:0], s["cos"], s["sin"])
    assert q.shape == (0, 6, 128) and k.shape == (0, 2, 128)


@pytest.mark.parametrize("d,rot,inter", [(128, 128, False), (128, 64, False), (64, 64, True), (96, 96, False)])
def test_unknown_positions_and_extremes(F, d, rot, inter):
    """Positions outside the table give NaN in their token's turned elements and nothing
    else; infinities stay with their row; a zero row and one of the smallest and largest
    values come out as the formula has them."""
    s = inputs(5, 40, 4, 2, d, rot, torch.float16, True)
    for t, p in ((0, -1), (3, 5000), (39, 2 ** 40), (20, -2 ** 40)):
        s["pos"][t] = p
    q = s["q"].clone()
    q[10, 0], q[11, 1], q[12, 2] = 0.0, 6e-8, 65504.0
    q[13, 3, 1] = float("inf")
    got, _ = F.norm_rotary(q, None, s["pos"], s["cos"], s["sin"], q_weight=s["wq"], interleaved=inter)
    bad = torch.tensor([0, 3, 39, 20], device="cuda")
    assert bool(torch.isnan(got[bad][..., :rot]).all())
    rest = torch.ones(40, dtype=torch.bool, device="cuda")
    rest[bad] = False
    s["pos"][bad] = 0
    ref = reference(q, s, s["wq"], 1e-6, inter)
    r = rest.cpu().numpy()
    r[13] = False
    assert_rows(got[torch.from_numpy(r).cuda()], ref[r])
    assert bool(torch.isfinite(got[13, :3]).all()) and not bool(torch.isfinite(got[13, 3]).all())


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("T,H,Hkv,d,rot,inter,dtype,norm,layout", CASES, ids=IDS)
def test_rotary_append(F, T, H, Hkv, d, rot, inter, dtype, norm, layout, residual):
    """The pool's bytes are the encodings of norm_rotary's keys and of the values, in their
    slots; padding goes nowhere; every other byte stays as it was."""
    page, n_pages = 64, T // 64 + 5
    s = inputs(7 * T + d, T, H, Hkv, d, rot, dtype, norm, layout)
    slots = torch.randperm(n_pages * page, generator=rng(T), device="cuda")[:T].contiguous()
    if T > 5:
        slots[2], slots[5], slots[4] = -1, n_pages * page, 2 ** 40
    n = n_pages * page * Hkv
    blobs = [torch.randint(0, 256, (n * w,), generator=rng(d), device="cuda", dtype=torch.uint8)
             if w == 36 or residual else None for w in (36, 130, 36, 130)]
    want = [None if b is None else b.clone() for b in blobs]
    args = (s["pos"], s["cos"], s["sin"])
    kw = dict(q_weight=s["wq"], k_weight=s["wk"], eps=1e-5, interleaved=inter)
    q2, k2 = F.norm_rotary(s["q"], s["k"], *args, **kw)
    q = F.rotary_append(s["q"], s["k"], s["v"], s["pos"], slots, s["cos"], s["sin"], *blobs, page, **kw)
    assert torch.equal(q, q2)
    live = [t for t in range(T) if 0 <= int(slots[t]) < n_pages * page]
    at = torch.tensor([((int(slots[t]) // page) * Hkv + h) * page + int(slots[t]) % page
                       for t in live for h in range(Hkv)], device="cuda")
    for rows, b, r in ((k2, want[0], want[1]), (s["v"], want[2], want[3])):
        enc = online_encode(rows[torch.tensor(live, device="cuda")].reshape(-1, d).float().cpu().numpy())
        by, sc = planes(b, d, False)
        by[at], sc[at] = torch.from_numpy(enc[0]).cuda(), torch.from_numpy(enc[1]).cuda()
        if residual:
            by, sc = planes(r, d, True)
            by[at], sc[at] = torch.from_numpy(enc[2]).cuda(), torch.from_numpy(enc[3]).cuda()
    for g, w in zip(blobs, want):
        assert g is None or torch.equal(g, w)


def test_append_without_rotation_is_the_ring_append(F):
    """paged_append of rows = the ring cache's append of the same rows, byte for byte."""
    from bitcache_amd import BitCache, PagedBitCache
    B, H, Hkv, d, page = 3, 8, 2, 128, 64
    g = rng(1)
    ring = BitCache(B, H, d, 128, n_kv_heads=Hkv)
    pool = PagedBitCache(2 * B, page, H, d, n_kv_heads=Hkv)
    tables = torch.randperm(2 * B, generator=g, device="cuda").to(torch.int32).view(B, 2)
    for t in range(70):
        k, v = (torch.randn((B, Hkv, d), generator=g, device="cuda").half() for _ in range(2))
        ring.append(k, v)
        pool.append(k, v, pool.slots(tables, torch.full((B,), t, device="cuda")))
    s = torch.arange(70, device="cuda")
    for b in range(B):
        for h in range(Hkv):
            mine = (tables[b].long()[s // page] * Hkv + h) * page + s % page
            ringed = (b * Hkv + h) * 128 + s
            for x, y, r in ((pool._k_bin, ring._k_bin, False), (pool._v_bin, ring._v_bin, False),
                            (pool._k_res, ring._k_res, True), (pool._v_res, ring._v_res, True)):
                for p, q in zip(planes(x, d, r), planes(y, d, r)):
                    assert torch.equal(p[mine], q[ringed])


def test_capture_and_streams(F):
    """A captured append follows its inputs over replays, beside eager calls; a call on
    another stream runs there."""
    page, n_pages, T, H, Hkv, d = 64, 4, 13, 8, 2, 128
    s = inputs(9, T, H, Hkv, d, d, torch.float16, True, "whole")
    n = n_pages * page * Hkv
    blobs = [torch.zeros(n * w, dtype=torch.uint8, device="cuda") for w in (36, 130, 36, 130)]
    eager = [b.clone() for b in blobs]
    slots = torch.arange(T, device="cuda")
    call = lambda bl: F.rotary_append(s["q"], s["k"], s["v"], s["pos"], slots, s["cos"], s["sin"], *bl, page,  # noqa: E731
                                      q_weight=s["wq"], k_weight=s["wk"])
    call(blobs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = call(blobs)
    for i in range(3):
        s["k"].copy_(torch.randn((T, Hkv, d), generator=rng(i), device="cuda"))
        s["q"].mul_(1.5)
        s["pos"].add_(7)
        slots.add_(17)
        graph.replay()
        torch.cuda.synchronize()
        q2 = call(eager)
        assert torch.equal(q, q2)
    # (the capture's first eager call wrote slots 0..12 of its own pool only)
    for a, b, r in zip(blobs, eager, (False, True, False, True)):
        for x, y in zip(planes(a, d, r), planes(b, d, r)):
            x, y = x.view(n_pages, Hkv, page, -1), y.view(n_pages, Hkv, page, -1)
            assert torch.equal(x[0, :, 17:], y[0, :, 17:]) and torch.equal(x[1:], y[1:])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q3 = call([b.clone() for b in eager])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(q3, q2)


def test_refusals(F):
    s = inputs(11, 6, 4, 2, 128, 128, torch.float16, True)
    q, k, v, pos, cos, sin = (s[x] for x in ("q", "k", "v", "pos", "cos", "sin"))
    n = 2 * 64 * 2
    blobs = [torch.zeros(n * w, dtype=torch.uint8, device="cuda") for w in (36, 130, 36, 130)]
    slots = torch.arange(6, device="cuda")

    def bad(f, *a, **kw):
        with pytest.raises(RuntimeError):
            f(*a, **kw)

    nr, ra, pa = F.norm_rotary, F.rotary_append, F.paged_append
    bad(nr, q.float(), k.float(), pos, cos, sin)                       # fp32 rows
    bad(nr, q, k.to(torch.bfloat16), pos, cos, sin)                    # mixed types
    bad(nr, q, k, pos.int(), cos, sin)                                 # int32 positions
    bad(nr, q, k, pos[:5], cos, sin)                                   # too few positions
    bad(nr, q, k, pos, cos.double(), sin.double())
    bad(nr, q, k, pos, cos[:, :63].contiguous(), sin[:, :63].contiguous())   # rot 126
    bad(nr, q[..., :64], k[..., :64], pos, cos, sin)                   # rot above d
    bad(nr, q, k, pos, cos, sin[:10])
    bad(nr, q, k, pos, cos, None)
    bad(nr, q, k, pos, cos[:0], sin[:0])
    bad(nr, q, k, pos, cos, sin, q_weight=s["wq"].float())
    bad(nr, q, None, pos, cos, sin, k_weight=s["wk"])
    bad(nr, q, k[:5], pos, cos, sin)
    bad(nr, q[..., ::2], None, pos, cos, sin)                          # stride 2 in the last dim
    bad(nr, q[..., :48], None, None, None, None)                       # head dim
    bad(nr, q.reshape(6, -1), None, pos, cos, sin)
    bad(nr, q.cpu(), None, pos.cpu(), cos.cpu(), sin.cpu())
    bad(nr, q, k, pos.cpu(), cos, sin)
    bad(nr, q.detach().clone().requires_grad_(), k, pos, cos, sin)
    bad(nr, q, k, pos, cos, sin, q_weight=s["wq"].clone().requires_grad_())
    with torch.no_grad():
        nr(q.detach().clone().requires_grad_(), k, pos, cos, sin)
    bad(ra, q, k, v[:, :1], pos, slots, cos, sin, *blobs, 64)
    bad(ra, q, k, v, pos, slots.int(), cos, sin, *blobs, 64)
    bad(ra, q, k, v, pos, slots[:5], cos, sin, *blobs, 64)
    bad(pa, k, v, slots, *blobs, 48)                                   # page size
    bad(pa, k, v, slots, *blobs, 192)                                  # not whole pages
    bad(pa, k, v, slots, blobs[0], blobs[1], blobs[2], None, 64)
    bad(pa, k, v, slots, blobs[0], torch.zeros(130 * 64, dtype=torch.uint8, device="cuda"), blobs[2], blobs[3], 64)
    bad(pa, k, v, slots, blobs[0].cpu(), blobs[1], blobs[2], blobs[3], 64)


LANES = [(d, rot, dtype) for d, dtype in ((32, torch.float16), (64, torch.bfloat16), (96, torch.float16),
                                          (128, torch.bfloat16), (160, torch.float16), (224, torch.bfloat16),
                                          (256, torch.float16))
         for rot in (16, 32, 64) if rot <= d]


@pytest.mark.parametrize("d,rot,dtype", LANES, ids=[f"{d}-{r}" for d, r, _ in LANES])
def test_few_turned_dims(F, d, rot, dtype):
    """Half pairs within the first 64 elements, with norms and without; the elements past
    them, infinities and signs of zero among them, stay where there is no norm."""
    s = inputs(d + rot, 11, 3, 2, d, rot, dtype, True)
    q, k = F.norm_rotary(s["q"], s["k"], s["pos"], s["cos"], s["sin"], k_weight=s["wk"])
    assert_rows(q, reference(s["q"], s, None, 1e-6, False))
    assert_rows(k, reference(s["k"], s, s["wk"], 1e-6, False))
    if rot < d:
        x = s["q"].clone()
        x[0, 0, rot], x[1, 0, d - 1], x[2, 1, rot] = float("inf"), float("-inf"), -0.0
        q, _ = F.norm_rotary(x, None, s["pos"], s["cos"], s["sin"])
        assert torch.equal(q[..., rot:].contiguous().view(torch.int16), x[..., rot:].contiguous().view(torch.int16))


@pytest.mark.parametrize("d,inter,layout", [(128, False, "fused"), (96, True, "whole"), (96, False, "odd")])
def test_long_prompt_is_its_parts(F, d, inter, layout):
    """Rows past what the caches hold are read by other loads: the same rows."""
    T = 45000
    s = inputs(2, T, 9, 1, d, d, torch.bfloat16, True, layout)
    s["pos"] = torch.arange(T, device="cuda") % s["cos"].shape[0]
    call = lambda a, b: F.norm_rotary(s["q"][a:b], s["k"][a:b], s["pos"][a:b], s["cos"], s["sin"], q_weight=s["wq"],
                                      k_weight=s["wk"], interleaved=inter)
    q, k = call(0, T)
    for a, b in ((0, 9001), (9001, 20000), (20000, 31111), (31111, T)):
        qp, kp = call(a, b)
        assert torch.equal(q[a:b], qp) and torch.equal(k[a:b], kp)
