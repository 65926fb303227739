"""Plain restatements, in 64 bits, of the rotation, the paged cache and its attention."""
from __future__ import annotations

import math

import numpy as np
import torch


def rotate64(x, positions, cos, sin, weight, eps, interleaved):
    """Norm and rotation of rows [T, h, d] (float64 numpy), unrounded."""
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    if positions is None:
        return x
    R = 2 * cos.shape[1]
    i = np.arange(R // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    c, s = cos.astype(np.float64)[positions][:, None], sin.astype(np.float64)[positions][:, None]
    y = x.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def half_step(dtype):
    return float(torch.finfo(dtype).eps) / 2


def online_encode(x):
    """Rows [n, d] float32 -> sign bytes, fp16 scale, code bytes, fp16 scale: the online
    encode, in the format's order of summation."""
    x = np.asarray(x, np.float32)
    n, d = x.shape
    p = np.zeros((n, 256), np.float32)
    p[:, :d] = np.abs(x)
    w = 128
    while w:
        p = p[:, :w] + p[:, w:2 * w]
        w //= 2
    mean = p / np.float32(d)
    pos = x >= 0
    r = x - np.where(pos, mean, -mean)
    top = np.abs(r).max(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        inv = np.where(top > 0, np.float32(7) / top, np.float32(0)).astype(np.float32)
    codes = np.clip(np.rint(r * inv), -7, 7).astype(np.int64) & 15
    signs = np.packbits(pos.reshape(n, d // 8, 8), axis=-1, bitorder="little")[..., 0]
    return (signs, mean[:, 0].astype(np.float16), (codes[:, 0::2] | codes[:, 1::2] << 4).astype(np.uint8),
            top[:, 0].astype(np.float16))


def planes(blob, d, residual):
    """(bytes [n, d/8 or d/2], fp16 scales [n]) of a blob, as views."""
    n = blob.numel() // (130 if residual else 36)
    w = d // 2 if residual else d // 8
    return blob[:n * w].view(n, w), blob[n * w:n * (w + 2)].view(torch.float16)


def decode64(bin_blob, res_blob, d, rows):
    """(signs, scales, residual values or None) of vectors `rows`, float64 on the device."""
    e = torch.arange(d, device=bin_blob.device)
    by, sc = planes(bin_blob, d, False)
    s = ((by[rows][:, e // 8].long() >> (e % 8)) & 1).double() * 2 - 1
    r = None
    if res_blob is not None:
        cb, rs = planes(res_blob, d, True)
        c = (cb[rows][:, e // 2].long() >> (4 * (e % 2))) & 15
        r = torch.where(c > 7, c - 16, c).double() / 7 * rs[rows].double()[:, None]
    return s, sc[rows].double(), r


def attention64(q, blobs, tables, lens, page, hkv):
    """(out [B, H, d], bound [B, H, d]) in 64 bits: bound is sum p |v|, what errors of the
    weights are relative to."""
    k_bin, k_res, v_bin, v_res = blobs
    B, H, d = q.shape
    out = torch.zeros((B, H, d), dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for b, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        at = torch.arange(n, device=q.device)
        pages, off = tables[b].long()[at // page], at % page
        for h in range(hkv):
            rows = (pages * hkv + h) * page + off
            mine = slice(h * (H // hkv), (h + 1) * (H // hkv))
            x = q[b, mine].double()
            ks, ksc, kr = decode64(k_bin, k_res, d, rows)
            vs, vsc, vr = decode64(v_bin, v_res, d, rows)
            s = torch.where(x >= 0, 1.0, -1.0).double() @ ks.T * ksc * x.abs().mean(-1, keepdim=True)
            v = vs * vsc[:, None]
            if kr is not None:
                s = s + x @ kr.T
                v = v + vr
            p = torch.softmax(s / math.sqrt(d), -1)
            out[b, mine] = p @ v
            size[b, mine] = p @ v.abs()
    return out, size


def assert_attention(got, ref, size, what=""):
    """Half a step of the output's type, and of the weights: scores are right to 2^-11 nats
    (the query's fixed point), which moves a weight and the sum it is divided by, and
    weights may be rounded to fp16 (half a step 2^-11): 3 * 2^-11 of sum p |v|."""
    tol = half_step(got.dtype) * ref.abs() + 3 * 2.0 ** -11 * size + 2.0 ** -25
    off = (got.double() - ref).abs()
    assert bool(torch.isfinite(got).all()), f"not finite {what}"
    worst = float((off - tol).max())
    assert worst <= 0, f"off by {float(off.max()):.3e}, {worst:.3e} over the tolerance {what}"


def make_pool(gen, n_pages, page, hkv, d, residual, std=1.0):
    """(k_bin, k_res, v_bin, v_res), every slot holding a vector."""
    from bitcache_amd import functional as F
    blobs = []
    for _ in range(2):
        x = torch.randn((n_pages * hkv * page, d), generator=gen, device="cuda") * std
        x = (x * torch.exp(0.25 * torch.randn((x.shape[0], 1), generator=gen, device="cuda"))).half()
        b, r = F.encode_fused(x, True)
        blobs += [b, r if residual else None]
    return blobs


def make_tables(gen, lens, page, shared_pages=0, width_extra=0, n_spare=1):
    """(tables int32 [B, width], n_pages): scattered pages; entries behind a sequence's last
    page are junk numbers."""
    need = [max(-(-max(n, 0) // page), 0) for n in lens]
    width = max(max(need), shared_pages) + width_extra
    own = [max(k - shared_pages, 0) for k in need]
    n_pages = shared_pages + sum(own) + n_spare
    perm = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32).cpu()
    t = torch.full((len(lens), width), -12345, dtype=torch.int32)
    at = shared_pages
    for b, k in enumerate(own):
        t[b, :shared_pages] = perm[:shared_pages]
        t[b, shared_pages:shared_pages + k] = perm[at:at + k]
        at += k
    return t.cuda(), n_pages
