"""CPU checks of the paged entry points: bad arguments are refused before any launch."""
import ctypes

import pytest

from test_abi import (BC_ERR_INVALID_ARGUMENT, BC_ERR_UNSUPPORTED, BC_ERR_WORKSPACE, BC_OK, lib, no_gpu)  # noqa: F401

P, I, L, D, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_double, ctypes.c_size_t
X = P(0x1000)


def test_rotary_argument_errors(lib, no_gpu):  # noqa: F811
    f = lib.bc_norm_rotary
    f.argtypes = [P, L, L, P, L, L, P, P, P, L, P, P, D, P, P, L, I, I, I, I, I, I, P]

    def call(q=X, k=X, pos=X, cos=X, table=10, qo=X, ko=X, T=3, H=4, Hkv=2, d=128, rot=128, dtype=0):
        return f(q, 512, 128, k, 512, 128, pos, cos, X if cos else None, table, None, None, 1e-6, qo, ko, T, H, Hkv,
                 d, rot, 0, dtype, None)

    assert call(d=48) == BC_ERR_UNSUPPORTED
    assert call(d=288) == BC_ERR_UNSUPPORTED
    assert call(rot=24) == BC_ERR_UNSUPPORTED
    assert call(rot=144) == BC_ERR_UNSUPPORTED
    assert call(rot=0) == BC_ERR_UNSUPPORTED
    assert call(dtype=2) == BC_ERR_UNSUPPORTED
    assert call(pos=None) == BC_ERR_INVALID_ARGUMENT
    assert call(cos=None) == BC_ERR_INVALID_ARGUMENT
    assert call(table=0) == BC_ERR_INVALID_ARGUMENT
    assert call(T=-1) == BC_ERR_INVALID_ARGUMENT
    assert call(T=2 ** 31) == BC_ERR_INVALID_ARGUMENT
    assert call(H=-1) == BC_ERR_INVALID_ARGUMENT
    assert call(q=None) == BC_ERR_INVALID_ARGUMENT
    assert call(ko=None) == BC_ERR_INVALID_ARGUMENT
    assert call(ko=P(0x1002)) == BC_ERR_INVALID_ARGUMENT
    assert call(Hkv=65536) == BC_ERR_UNSUPPORTED
    assert call(T=0, q=None, k=None, qo=None, ko=None) == BC_OK
    assert call(H=0, Hkv=0, q=None, k=None, qo=None, ko=None) == BC_OK


def test_append_argument_errors(lib, no_gpu):  # noqa: F811
    f = lib.bc_paged_append
    f.argtypes = [P, L, L, P, L, L, P, L, L, P, P, P, L, P, P, D, P, P, P, P, P, P, I, I, L, I, I, I, I, I, I, P]

    def call(q=X, k=X, v=X, qw=None, qo=X, slots=X, kb=X, kr=X, vr=X, pages=4, page=64, T=3, H=4, d=128, rot=128,
             dtype=1):
        return f(q, 512, 128, k, 512, 128, v, 512, 128, X, X, X, 10, qw, None, 1e-6, qo, slots, kb, kr, X, vr, pages,
                 page, T, H, 2, d, rot, 0, dtype, None)

    assert call(d=100) == BC_ERR_UNSUPPORTED
    assert call(rot=8) == BC_ERR_UNSUPPORTED
    assert call(dtype=-1) == BC_ERR_UNSUPPORTED
    assert call(pages=1 << 20, page=1 << 12) == BC_ERR_UNSUPPORTED
    assert call(page=96) == BC_ERR_INVALID_ARGUMENT
    assert call(page=0) == BC_ERR_INVALID_ARGUMENT
    assert call(pages=-1) == BC_ERR_INVALID_ARGUMENT
    assert call(kr=None) == BC_ERR_INVALID_ARGUMENT
    assert call(kb=None) == BC_ERR_INVALID_ARGUMENT
    assert call(k=None) == BC_ERR_INVALID_ARGUMENT
    assert call(slots=None) == BC_ERR_INVALID_ARGUMENT
    assert call(qo=None) == BC_ERR_INVALID_ARGUMENT
    assert call(H=0, q=None, qo=None, qw=X) == BC_ERR_INVALID_ARGUMENT
    assert call(H=65536) == BC_ERR_UNSUPPORTED
    assert call(qo=P(0x1008)) == BC_ERR_INVALID_ARGUMENT
    assert call(kb=P(0x1004)) == BC_ERR_INVALID_ARGUMENT
    assert call(vr=P(0x1002)) == BC_ERR_INVALID_ARGUMENT
    assert call(T=0, q=None, k=None, v=None, slots=None) == BC_OK


def test_paged_attention_argument_errors(lib, no_gpu):  # noqa: F811
    w = lib.bc_paged_attention_workspace_size
    w.argtypes = [I] * 6 + [ctypes.POINTER(Z)]
    f = lib.bc_paged_attention
    f.argtypes = [P] * 6 + [I, P, P] + [I] * 9 + [P, Z, P]
    n = Z(0)
    assert w(4, 8, 2, 1000, 0, 128, ctypes.byref(n)) == BC_OK
    assert w(4, 8, 2, 1000, 0, 128, None) == BC_ERR_INVALID_ARGUMENT
    assert w(4, 8, 3, 1000, 0, 128, ctypes.byref(n)) == BC_ERR_INVALID_ARGUMENT
    assert w(4, 8, 2, 1000, 0, 80, ctypes.byref(n)) == BC_ERR_UNSUPPORTED
    assert w(-1, 8, 2, 1000, 0, 128, ctypes.byref(n)) == BC_ERR_INVALID_ARGUMENT
    assert w(4, 8, 2, 1000, 1024, 128, ctypes.byref(n)) == BC_ERR_INVALID_ARGUMENT
    assert w(4, 8, 2, 1000, 32, 128, ctypes.byref(n)) == BC_ERR_INVALID_ARGUMENT
    # every shape has a plan, and a shared prefix's partials are in it
    for B in (1, 2, 3, 17, 64, 500, 65535):
        for H, Hkv in ((1, 1), (8, 2), (24, 8), (64, 1), (32, 32)):
            for longest in (0, 1, 64, 65, 1000, 131072):
                for shared in (0, 64, 640, 65536):
                    for d in (32, 64, 96, 128, 160, 192, 224, 256):
                        if shared <= longest and B * (longest // 64 + 1) < 2 ** 31:
                            assert w(B, H, Hkv, longest, shared, d, ctypes.byref(n)) == BC_OK
    assert w(64, 32, 8, 34816, 0, 128, ctypes.byref(n)) == BC_OK
    alone = n.value
    assert w(64, 32, 8, 34816, 32768, 128, ctypes.byref(n)) == BC_OK and n.value > 64 * 32 * 130 * 4 and alone > 0

    def call(q=X, kb=X, kr=X, vr=X, tables=X, width=20, lens=X, out=X, B=4, H=8, Hkv=2, pages=50, page=64, longest=1000,
             shared=0, d=128, dtype=0, ws=P(0x10000), size=1 << 40):
        return f(q, kb, kr, X, vr, tables, width, lens, out, B, H, Hkv, pages, page, longest, shared, d, dtype, ws,
                 size, None)

    assert call(d=72) == BC_ERR_UNSUPPORTED
    assert call(dtype=3) == BC_ERR_UNSUPPORTED
    assert call(B=70000) == BC_ERR_UNSUPPORTED
    assert call(pages=1 << 20, page=1 << 12) == BC_ERR_UNSUPPORTED
    assert call(H=7) == BC_ERR_INVALID_ARGUMENT
    assert call(page=100) == BC_ERR_INVALID_ARGUMENT
    assert call(width=-1) == BC_ERR_INVALID_ARGUMENT
    assert call(shared=32) == BC_ERR_INVALID_ARGUMENT
    assert call(shared=1024, longest=2000, width=10) == BC_ERR_INVALID_ARGUMENT
    assert call(kr=None) == BC_ERR_INVALID_ARGUMENT
    assert call(q=None) == BC_ERR_INVALID_ARGUMENT
    assert call(out=None) == BC_ERR_INVALID_ARGUMENT
    assert call(lens=None) == BC_ERR_INVALID_ARGUMENT
    assert call(tables=None) == BC_ERR_INVALID_ARGUMENT
    assert call(kb=None) == BC_ERR_INVALID_ARGUMENT
    assert call(kr=P(0x1008)) == BC_ERR_INVALID_ARGUMENT
    assert call(ws=P(0x10008)) == BC_ERR_INVALID_ARGUMENT
    assert call(B=0, q=None, out=None) == BC_OK


def test_paged_operators_reject_cpu_tensors():
    import torch
    import bitcache_amd
    if not bitcache_amd._HAS_EXTENSION:
        pytest.skip("extension not built")
    from bitcache_amd import functional as F
    q = torch.zeros((2, 4, 128), dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int64)
    blob = torch.zeros(36 * 64, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="ROCm"):
        F.norm_rotary(q, None, None, None, None)
    with pytest.raises(RuntimeError, match="ROCm"):
        F.paged_append(q, q, i, blob, None, blob, None, 64)
    with pytest.raises(RuntimeError, match="ROCm"):
        F.paged_attention(q, blob, None, blob, None, i.int()[:, None], i.int(), 64, 64)
    with pytest.raises(RuntimeError, match="ROCm"):
        bitcache_amd.PagedBitCache(4, 64, 4, 128, device="cpu")
