"""The paged serving path over the compressed cache, and its measured cases.

  rotary   norms of queries and keys per head, with the position rotation (``functional.norm_rotary``)
  append   rotation and encoding of new keys and values into a paged cache (``functional.rotary_append``)
  attend   decode attention over pages, a length per sequence (``functional.paged_attention``)
  shared   the same for a batch whose sequences share a long prefix (``shared_len=``)

``run`` computes them in elementary torch operations, or through the framework's entry
points where ``own`` is set.  A paged cache is a binary and a residual blob (planes of
signs / codes, then of fp16 scales) whose vector ``(page * kv_heads + head) *
page_size + offset`` is a key or a value; a slot is ``page * page_size + offset``.

A case is a dict of plain values:
  op              rotary, append, attend or shared
  dtype           fp16 or bf16: queries, keys, values and outputs
  heads, kv_heads, dim
  tokens          (rotary, append) new tokens, one row of positions each
  rot             rotated dims (the first `rot` of a head); interleaved: pairs
                  (2i, 2i + 1), else (i, i + rot / 2)
  norm            RMS norms of query and key heads with learned weights
  page            slots of a page
  residual        the cache holds INT4 residuals, else signs only
  batch           (attend, shared) sequences; their lengths run from `shortest` to
                  `longest` on a logarithmic scale (shared: own keys, after the prefix)
  prefix          (shared) keys that all sequences share, whole pages
"""
from __future__ import annotations

import math

import torch

own = False

_EPS = 1e-6
# Bytes and products of a drawn case at most (the largest listed ones: 0.5 GB of
# keys and values, 3.7e10 operations)
_DRAWN_BYTES, _DRAWN_KEYS = 3e8, 6e6


def _new(op, heads, kv_heads, dim, tokens, rot, interleaved=False, norm=True, dtype="fp16",
         page=64, residual=True):
    return dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, tokens=tokens, rot=rot,
                interleaved=interleaved, norm=norm, dtype=dtype, page=page, residual=residual)


def _read(op, batch, heads, kv_heads, dim, shortest, longest, prefix=0, dtype="fp16", page=64,
          residual=True):
    return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, shortest=shortest,
                longest=longest, prefix=prefix, dtype=dtype, page=page, residual=residual)


def listed():
    return [
        # one decode step of a small served batch: the smallest calls, all latency
        dict(name="rotary_step", **_new("rotary", 32, 8, 128, 4, 128)),
        # a 16K-token prompt through the same layer
        dict(name="rotary_prompt", **_new("rotary", 32, 8, 128, 16384, 128, dtype="bf16")),
        # rotation alone, of part of each head in adjacent pairs, odd token count
        dict(name="rotary_part", **_new("rotary", 32, 32, 96, 5001, 32, interleaved=True, norm=False)),
        # a decode step of 32 sequences: each token goes to a page of its own
        dict(name="append_step", **_new("append", 32, 8, 128, 32, 128)),
        # a prompt of four 4K-token sequences, one token short of whole pages
        dict(name="append_prompt", **_new("append", 32, 8, 128, 16383, 128, dtype="bf16")),
        # signs only (the memory-saving mode), d = 64, no norms
        dict(name="append_binary", **_new("append", 32, 32, 64, 4096, 64, norm=False, residual=False)),
        # one sequence at the start of a chat (latency and launches)
        dict(name="attend_short", **_read("attend", 1, 32, 8, 128, 301, 301)),
        # a served batch in the middle of its work: 64 sequences of 128 to 32K tokens
        dict(name="attend_ragged", **_read("attend", 64, 32, 8, 128, 128, 32768)),
        # binary attention of single heads, large pages, near-equal long sequences
        dict(name="attend_binary", **_read("attend", 8, 32, 32, 128, 28001, 32768, page=256,
                                           residual=False)),
        # wide heads, bf16 activations
        dict(name="attend_d256", **_read("attend", 16, 16, 8, 256, 999, 12345, dtype="bf16", page=128)),
        # a chat service: 32 users behind one 4K-token system prompt, short turns
        dict(name="shared_chat", **_read("shared", 32, 32, 8, 128, 17, 700, prefix=4096)),
        # 64 questions about one 32K-token document
        dict(name="shared_document", **_read("shared", 64, 32, 8, 128, 64, 2000, prefix=32768)),
    ]


def draw(rng):
    """One more case of the same ranges: head dims 64 to 256 (now and then any multiple
    of 32), 1 to 16 query heads per KV head, 1 to 16,384 new tokens, 1 to 128
    sequences of 1 to 32,768 keys, prefixes of 128 to 32,768."""
    op = rng.choice(["rotary", "append", "attend", "attend", "shared", "shared"])
    dim = rng.choice([128, 128, 128, 128, 64, 64, 256, 256, 96, rng.choice([32, 160, 192, 224])])
    group = rng.choice([1, 1, 2, 4, 4, 4, 8, 8, 3, 16])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 8, 16, 32])
    while kv_heads * group > 64:
        kv_heads //= 2
    heads = kv_heads * group
    dtype = rng.choice(["fp16", "fp16", "bf16"])
    page = rng.choice([64, 64, 128, 192, 256])
    residual = rng.random() < 0.75

    def log(lo, hi):
        return max(lo, min(hi, int(round(2.0 ** rng.uniform(math.log2(lo), math.log2(hi))))))

    if op in ("rotary", "append"):
        most = int(_DRAWN_BYTES / (4 * dim * (heads + 2 * kv_heads)))
        rot = dim if rng.random() < 0.7 else 16 * rng.randint(1, dim // 16)
        return _new(op, heads, kv_heads, dim, log(1, min(16384, most)), rot, rng.random() < 0.3,
                    rng.random() < 0.6, dtype, page, residual)
    batch = log(1, 128)
    # the plain forms hold [batch, kv_heads, keys, dim] tensors in 32 bits
    most = int(min(_DRAWN_BYTES / (2 * _vec_bytes(dim, residual) * kv_heads * batch),
                   _DRAWN_KEYS * 256 / (batch * kv_heads * dim)))
    if op == "attend":
        longest = log(16, max(16, min(32768, most)))
        return _read(op, batch, heads, kv_heads, dim, log(1, longest), longest, 0, dtype, page, residual)
    prefix = log(128, max(128, min(32768, most)))
    prefix = max(1, prefix // page) * page
    longest = log(1, max(1, min(2000, most - prefix)))
    return _read(op, batch, heads, kv_heads, dim, log(1, longest), longest, prefix, dtype, page, residual)


# ---------------------------------------------------------------- sizes
def _vec_bytes(dim, residual):
    """Bytes of one encoded vector: sign bits and scale, INT4 codes and their scale."""
    return dim // 8 + 2 + ((dim // 2 + 2) if residual else 0)


def _lengths(case):
    """Keys of each sequence (without the prefix): log-spaced, the same for every seed."""
    B, lo, hi = case["batch"], case["shortest"], case["longest"]
    if B == 1:
        return [hi]
    return [min(hi, int(round(lo * (hi / lo) ** (b / (B - 1))))) for b in range(B)]


def work(case):
    H, Hkv, d = case["heads"], case["kv_heads"], case["dim"]
    vec = _vec_bytes(d, case["residual"])
    if case["op"] in ("rotary", "append"):
        T = case["tokens"]
        rows = T * (H + Hkv)
        moved = T * H * d * 4 + T * case["rot"] * 4 + T * 8
        if case["op"] == "rotary":
            return {"bytes": moved + T * Hkv * d * 4, "flops": rows * d * (8 if case["norm"] else 3)}
        return {"bytes": moved + T * 8 + T * Hkv * d * 4 + 2 * T * Hkv * vec,
                "flops": rows * d * (8 if case["norm"] else 3) + 2 * T * Hkv * d * 8}
    B, keys, P = case["batch"], sum(_lengths(case)), case["prefix"]
    # the prefix is read once for all, and multiplied with every query
    return {"bytes": (keys + P) * Hkv * 2 * vec + B * H * d * 4,
            "flops": 4.0 * H * d * (keys + B * P)}


# ---------------------------------------------------------------- the format, in 32 bits
def _mean_abs(x):
    """Mean |x| of rows [n, d] fp32 in the format's order: thread t of 128 adds |x_t| and
    |x_(t+128)|, then halves fold onto each other."""
    n, d = x.shape
    p = torch.zeros((n, 256), device=x.device)
    p[:, :d] = x.abs()
    for half in (128, 64, 32, 16, 8, 4, 2, 1):
        p = p[:, :half] + p[:, half:]
    return p / torch.full_like(p, float(d))


def _encode(x):
    """Rows [n, d] fp32 -> (sign bytes [n, d/8], fp16 scale [n], code bytes [n, d/2], fp16 scale
    [n]): the online encode, codes against the 32-bit mean."""
    n, d = x.shape
    mean = _mean_abs(x)
    positive = x >= 0
    r = x - torch.where(positive, mean, -mean)
    top = r.abs().amax(-1, keepdim=True)
    inv = torch.where(top > 0, torch.full_like(top, 7.0) / top, torch.zeros_like(top))
    codes = torch.round(r * inv).clamp_(-7, 7).to(torch.int16) & 15
    bit = torch.tensor([1, 2, 4, 8, 16, 32, 64, 128], device=x.device, dtype=torch.int16)
    signs = (positive.view(n, d // 8, 8).to(torch.int16) * bit).sum(-1).to(torch.uint8)
    nibbles = (codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8)
    return signs, mean.half().view(n), nibbles, top.half().view(n)


def _planes(case, blob, residual):
    """(bytes [n, d/8 or d/2], fp16 scales [n]) of a blob."""
    n = blob.numel() // (130 if residual else 36)
    w = case["dim"] // 2 if residual else case["dim"] // 8
    return blob[:n * w].view(n, w), blob[n * w:n * (w + 2)].view(torch.float16)


def _decode_signs(planes):
    """sign * scale of vectors [n, d], 32 bits, and the signs (+-1)."""
    signs, scale = planes
    bits = (signs[:, :, None] >> torch.arange(8, device=signs.device, dtype=torch.uint8)) & 1
    s = bits.view(signs.shape[0], -1).float() * 2 - 1
    return s, scale.float()


def _decode_codes(planes):
    """code / 7 * scale of vectors [n, d], 32 bits."""
    codes, scale = planes
    n = torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1).to(torch.int8)
    n = torch.where(n > 7, n - 16, n)
    return n.float() * (scale.float() / 7.0)[:, None]


# ---------------------------------------------------------------- inputs
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(gen, shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _blobs(case, pages):
    """Empty (k_bin, k_res, v_bin, v_res) of a pool of pages."""
    n = pages * case["kv_heads"] * case["page"]
    sizes = (36, 130, 36, 130) if case["residual"] else (36, None, 36, None)
    return [None if s is None else torch.zeros(n * s, dtype=torch.uint8, device="cuda") for s in sizes]


def _fill(case, gen, blobs):
    """Keys and values of normal elements, the rows' magnitudes spread log-normally, in every
    slot of the pool: those behind a sequence's last key too, as pages that were in use hold."""
    d = case["dim"]
    n = blobs[0].numel() // 36
    for i in (0, 2):
        for at in range(0, n, 1 << 20):
            m = min(1 << 20, n - at)
            x = _randn(gen, (m, d)) * torch.exp(0.25 * _randn(gen, (m, 1)))
            signs, scale, codes, rscale = _encode(x.half().float())
            p, s = _planes(case, blobs[i], False)
            p[at:at + m], s[at:at + m] = signs, scale
            if case["residual"]:
                p, s = _planes(case, blobs[i + 1], True)
                p[at:at + m], s[at:at + m] = codes, rscale


def prepare(case, seed):
    gen, t = _gen(seed), _dtype(case)
    H, Hkv, d, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    s = dict(case=case)
    if case["op"] in ("rotary", "append"):
        T, R = case["tokens"], case["rot"]
        # one projection holds queries, keys and values side by side
        qkv = (_randn(gen, (T, H + 2 * Hkv, d)) * torch.exp(0.25 * _randn(gen, (T, H + 2 * Hkv, 1)))).to(t)
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        # tokens of a decode step sit anywhere in their sequences, a prompt's follow each other
        start = torch.randint(0, 32768, (T,), generator=gen, device="cuda")
        s["positions"] = start if T < 256 else (torch.arange(T, device="cuda") + start[0] % 1024) % 32768
        angle = torch.arange(32768, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
            1e6, -torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
        s["cos"], s["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        s["q_weight"] = (1 + 0.2 * _randn(gen, (d,))).to(t) if case["norm"] else None
        s["k_weight"] = (1 + 0.2 * _randn(gen, (d,))).to(t) if case["norm"] else None
        if case["op"] == "append":
            # a decode step's tokens go to a page each, a prompt's fill pages in scattered order
            per = 1 if T < 256 else page
            pages = -(-T // per) + 2
            table = torch.randperm(pages, generator=gen, device="cuda")
            i = torch.arange(T, device="cuda")
            offset = i % page if per == page else start % page
            s["slots"] = table[i // per] * page + offset
            s["blobs"] = _blobs(case, pages)
        return s
    B, P = case["batch"], case["prefix"] // page
    lens = torch.tensor(_lengths(case))[torch.randperm(case["batch"], generator=torch.Generator().manual_seed(int(seed)))]
    need = [-(-n // page) for n in lens.tolist()]
    pages = P + sum(need) + 1
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu()
    table = torch.zeros((B, P + max(need)), dtype=torch.int32)
    at = P
    for b in range(B):
        table[b, :P] = order[:P]
        table[b, P:P + need[b]] = order[at:at + need[b]]
        at += need[b]
    s["tables"] = table.cuda()
    s["lens"] = (lens + P * page).to(torch.int32).cuda()
    s["longest"] = case["longest"] + P * page
    s["q"] = _randn(gen, (B, H, d)).to(t)
    s["blobs"] = _blobs(case, pages)
    _fill(case, gen, s["blobs"])
    return s


# ---------------------------------------------------------------- the plain forms
def _rotate(case, x, s, weight):
    """Norm and rotation of rows [T, h, d], in 64 bits (the encoder's borders follow)."""
    R, t = case["rot"], x.dtype
    x = x.double()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight.double()
    c = s["cos"][s["positions"]].double()[:, None]
    n = s["sin"][s["positions"]].double()[:, None]
    y = x.clone()
    if case["interleaved"]:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y[..., 0:R:2], y[..., 1:R:2] = a * c - b * n, b * c + a * n
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        y[..., :R // 2], y[..., R // 2:R] = a * c - b * n, b * c + a * n
    return y.float().to(t)


def _store(case, rows, slots, binary, residual):
    """Encode rows [T, kv_heads, d] into the slots of a pool."""
    T, Hkv, d = rows.shape
    page = case["page"]
    head = torch.arange(Hkv, device=rows.device)
    at = ((slots[:, None] // page * Hkv + head) * page + slots[:, None] % page).reshape(-1)
    signs, scale, codes, rscale = _encode(rows.reshape(-1, d).float())
    p, q = _planes(case, binary, False)
    p[at], q[at] = signs, scale
    if residual is not None:
        p, q = _planes(case, residual, True)
        p[at], q[at] = codes, rscale


def _attend(case, s):
    """Attention over the gathered, decoded pages of every sequence, in 32 bits."""
    B, H = s["q"].shape[:2]
    Hkv, d, page = case["kv_heads"], case["dim"], case["page"]
    k_bin, k_res, v_bin, v_res = s["blobs"]

    def gather(rows):   # [vectors, ...] -> [B, kv_heads, keys, ...]
        x = rows.view(-1, Hkv, page, *rows.shape[1:])[s["tables"].long()]
        return x.transpose(1, 2).reshape(B, Hkv, -1, *rows.shape[1:])

    q = s["q"].float().view(B, Hkv, H // Hkv, d)
    match, scale = _decode_signs(_planes(case, k_bin, False))
    score = torch.where(q >= 0, 1.0, -1.0) @ gather(match).transpose(2, 3)
    score = score * q.abs().mean(-1, keepdim=True) * gather(scale)[:, :, None]
    if k_res is not None:
        score += q @ gather(_decode_codes(_planes(case, k_res, True))).transpose(2, 3)
    outside = torch.arange(score.shape[-1], device=q.device) >= s["lens"][:, None]
    score = (score / math.sqrt(d)).masked_fill_(outside[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    match, scale = _decode_signs(_planes(case, v_bin, False))
    value = match.mul_(scale[:, None])
    if v_res is not None:
        value += _decode_codes(_planes(case, v_res, True))
    return (p @ gather(value)).view(B, H, d).to(s["q"].dtype)


def _written(case, s):
    """The planes of the pool: signs and codes as the bytes that they are, scales as fp16."""
    return [x for b, r in zip(s["blobs"], (False, True, False, True)) if b is not None
            for x in _planes(case, b, r)]


def run(s):
    case = s["case"]
    op = case["op"]
    norms = dict(q_weight=s.get("q_weight"), k_weight=s.get("k_weight"), eps=_EPS,
                 interleaved=case.get("interleaved", False))
    if own:
        from bitcache_amd import functional as F
        if op == "rotary":
            return F.norm_rotary(s["q"], s["k"], s["positions"], s["cos"], s["sin"], **norms)
        if op == "append":
            q = F.rotary_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["cos"], s["sin"],
                                *s["blobs"], case["page"], **norms)
            return [q] + _written(case, s)
        return F.paged_attention(s["q"], *s["blobs"], s["tables"], s["lens"], s["longest"], case["page"],
                                 n_kv_heads=case["kv_heads"], shared_len=case["prefix"])
    if op == "rotary":
        return _rotate(case, s["q"], s, s["q_weight"]), _rotate(case, s["k"], s, s["k_weight"])
    if op == "append":
        q = _rotate(case, s["q"], s, s["q_weight"])
        k_bin, k_res, v_bin, v_res = s["blobs"]
        _store(case, _rotate(case, s["k"], s, s["k_weight"]), s["slots"], k_bin, k_res)
        _store(case, s["v"], s["slots"], v_bin, v_res)
        return [q] + _written(case, s)
    return _attend(case, s)


# ---------------------------------------------------------------- from the definition, in 64 bits
def _exact_rotary(case, s, x, weight):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + _EPS) * weight.double()
    R = case["rot"]
    i = torch.arange(0, R, 2, device=x.device)
    first, second = (i, i + 1) if case["interleaved"] else (i // 2, i // 2 + R // 2)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, None]
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _exact_rows(case, binary, residual, rows):
    """(signs, scale, residual) in 64 bits of the pool's vectors `rows`."""
    d = case["dim"]
    e = torch.arange(d, device=binary.device)
    signs, scale = _planes(case, binary, False)
    s = ((signs[rows][:, e // 8].long() >> (e % 8)) & 1).double() * 2 - 1
    r = None
    if residual is not None:
        codes, top = _planes(case, residual, True)
        n = (codes[rows][:, e // 2].long() >> (4 * (e % 2))) & 15
        r = (n - 16 * (n > 7).long()).double() / 7 * top[rows].double()[:, None]
    return s, scale[rows].double()[:, None], r


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("rotary", "append"):
        q = _exact_rotary(case, s, s["q"], s["q_weight"])
        if case["op"] == "append":
            return [q] + [None] * len(_written(case, s))
        return q, _exact_rotary(case, s, s["k"], s["k_weight"])
    H, Hkv, d, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
    k_bin, k_res, v_bin, v_res = s["blobs"]
    out = torch.zeros((case["batch"], H, d), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        at = torch.arange(n, device="cuda")
        pages, offset = s["tables"][b].long()[at // page], at % page
        for h in range(Hkv):
            rows = (pages * Hkv + h) * page + offset
            mine = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
            q = s["q"][b, mine].double()
            ks, kscale, kr = _exact_rows(case, k_bin, k_res, rows)
            vs, vscale, vr = _exact_rows(case, v_bin, v_res, rows)
            score = torch.where(q >= 0, 1.0, -1.0).double() @ ks.T * kscale.T * q.abs().mean(-1, keepdim=True)
            if kr is not None:
                score = score + q @ kr.T
            p = torch.softmax(score / math.sqrt(d), -1)
            out[b, mine] = p @ (vs * vscale if vr is None else vs * vscale + vr)
    return out
