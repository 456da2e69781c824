"""The C entries of drafted decoding and the 8-bit products reject bad arguments with an
error code and message, before any CUDA call. No GPU needed."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib(built_lib):
    from lizard_cuda import _lib
    return _lib.load()


def _fake(n=1):
    # never dereferenced: validation rejects the calls first
    return [ctypes.c_void_p(0x1000 * (i + 1)) for i in range(n)]


def _msg(lib):
    return lib.lz_last_error_string()


def test_gla_decode_block_validates(lib):
    p = _fake(12)

    def call(B=2, H=8, Hkv=2, Hs=2, T=4, Tp=4, F=64, D=64, gph=0, **swap):
        a = dict(enumerate(p))
        a.update({int(k[1:]): v for k, v in swap.items()})
        return lib.lz_gla_decode_block(a[0], a[1], a[2], a[3], gph, a[4], a[5], a[6], a[7], a[8],
                                       a[9], a[10], B, H, Hkv, Hs, T, Tp, F, D, None)

    assert call(B=0) == 1
    assert call(T=0, Tp=0) == 1 and b"no tokens" in _msg(lib)
    assert call(T=-1) == 1
    assert call(H=7) == 1 and b"divide" in _msg(lib)
    assert call(gph=1) == 1 and b"state heads" in _msg(lib)
    assert call(T=65) == 2 and b"at most 64" in _msg(lib)
    assert call(Tp=65) == 2
    assert call(F=257) == 2 and call(D=66) == 2 and call(D=260) == 2
    assert call(_0=None) == 1 and b"null" in _msg(lib)
    assert call(_4=None) == 1 and b"previous block" in _msg(lib)
    assert call(_8=ctypes.c_void_p(0x1004)) == 1 and b"aligned" in _msg(lib)


def test_swa_decode_block_validates(lib):
    p = _fake(16)
    st = (ctypes.c_longlong * 12)(*[0, 0, 0, 1] * 3)
    stp = (ctypes.c_longlong * 8)(*[0, 0, 0, 1] * 2)
    bad = (ctypes.c_longlong * 12)(*[0, 0, 0, 1, 0, 0, 0, 2, 0, 0, 0, 1])

    def call(B=2, H=8, Hkv=2, T=4, Tp=4, W=64, D=64, x=0, cs=0, n_meta=4, meta=p[13], strides=st,
             q=p[0], kp=p[5], ws=p[15], n=1 << 30):
        return lib.lz_swa_decode_block(q, p[1], p[2], x, strides, p[3], p[4], cs, 0, kp, p[6], stp,
                                       p[7], p[8], 0, p[9], p[10], p[11], p[12], meta, n_meta,
                                       p[14], ws, n, B, H, Hkv, T, Tp, W, D, None)

    assert call(W=0) == 1
    assert call(T=0, Tp=0) == 1 and b"no tokens" in _msg(lib)
    assert call(H=7) == 1 and b"divide" in _msg(lib)
    assert call(D=63) == 1 and b"even" in _msg(lib)
    assert call(T=65) == 2 and call(W=1025) == 2 and call(D=258) == 2
    assert call(n_meta=33) == 1 and call(meta=None) == 1 and b"n_meta" in _msg(lib)
    assert call(x=2) == 1 and call(cs=7) == 1 and b"dtypes" in _msg(lib)
    assert call(q=None) == 1 and call(strides=None) == 1
    assert call(strides=bad) == 1 and b"contiguous" in _msg(lib)
    assert call(kp=None) == 1 and b"previous block" in _msg(lib)
    need = lib.lz_swa_decode_block_workspace_bytes(2, 8, 2, 4, 64)
    assert need >= 4 * (16 * 64 * 4 + 2 * 16 * 64 * 4)
    assert call(n=need - 1) == 4 and b"workspace" in _msg(lib)
    assert call(ws=ctypes.c_void_p(0x1008)) == 1 and b"aligned" in _msg(lib)
    assert lib.lz_swa_decode_block_workspace_bytes(2, 8, 2, 0, 64) == 0
    assert lib.lz_swa_decode_block_workspace_bytes(2, 8, 3, 4, 64) == 0


def test_verify_drafts_validates(lib):
    p = _fake(10)
    size = lib.lz_verify_drafts_workspace_bytes(4, 3, 1000)
    assert size > 0 and lib.lz_verify_drafts_workspace_bytes(4, 65, 1000) == 0
    assert lib.lz_verify_drafts_workspace_bytes(0, 3, 1000) == 0
    assert lib.lz_verify_drafts_workspace_bytes(65535, 0, 1000) > 0
    assert lib.lz_verify_drafts_workspace_bytes(65535, 1, 1000) == 0

    def call(B=4, K=3, V=1000, dt=0, ws=p[8], n=size, draft=p[1], noise=p[4]):
        return lib.lz_verify_drafts(p[0], 0, 0, draft, 0, 0, dt, p[2], 1, p[3], noise, 0, None,
                                    1.0, None, p[6], p[7], ws, n, B, K, V, None)

    assert call(V=0) == 1 and call(K=-1) == 1
    assert call(K=65) == 2 and b"at most 64" in _msg(lib)
    assert call(B=40000) == 2
    assert call(dt=3) == 1 and b"logits" in _msg(lib)
    assert call(draft=None) == 1 and b"draft" in _msg(lib)
    assert call(noise=None) == 1
    assert call(n=size - 1) == 4 and b"workspace" in _msg(lib)
    assert call(ws=ctypes.c_void_p(0x1008)) == 1 and b"aligned" in _msg(lib)


def test_int8_entries_validate(lib):
    p = _fake(8)

    def mm(M=4, N=8, K=32, ld=32, ydt=0, bdt=0, bias=None, a=p[0], b=p[2], ws=None, n=0):
        return lib.lz_int8_matmul(a, ld, p[1], b, ld, p[3], bias, bdt, p[4], ydt, ws, n, M, N, K,
                                  None)

    assert mm(M=0) == 1
    assert mm(K=131072, ld=131072) == 2 and b"131071" in _msg(lib)
    assert mm(ydt=2) == 1 and mm(bias=p[5], bdt=5) == 1 and b"bias" in _msg(lib)
    assert mm(ld=31) == 1 and b"overlap" in _msg(lib)
    assert mm(ld=40) == 4 and b"workspace" in _msg(lib)  # rows off 16 bytes need one
    assert mm(a=ctypes.c_void_p(0x1001)) == 4
    assert mm(b=None) == 1
    need = lib.lz_int8_workspace_bytes(4, 8, 33)
    assert need >= (4 + 8) * 48 and mm(K=33, ld=33, ws=p[6], n=need - 1) == 4
    assert lib.lz_int8_linear_workspace_bytes(20, 8, 33) >= 20 * 48 + 80
    assert lib.lz_int8_linear_workspace_bytes(4, 8, 33) == 0  # a few tokens need none
    rc = lib.lz_int8_linear(p[0], 0, 32, p[1], 32, p[2], None, 0, p[3], 0, None, 0, 20, 8, 32, None)
    assert rc == 4 and b"workspace" in _msg(lib)
    rc = lib.lz_int8_linear(p[0], 9, 32, p[1], 32, p[2], None, 0, p[3], 0, p[4], 1 << 20, 4, 8, 32,
                            None)
    assert rc == 1 and b"x must be" in _msg(lib)
    assert lib.lz_int8_quantize(p[0], 0, 32, p[1], 33, p[2], 4, 33, None) == 1
    assert b"16-byte" in _msg(lib)
    assert lib.lz_int8_quantize(p[0], 0, 32, p[1], 32, None, 4, 32, None) == 1
    assert lib.lz_int8_set_path(3) == -1 and b"path" in _msg(lib)
    assert lib.lz_int8_set_path(1) == 0 and lib.lz_int8_set_path(0) == 1


def test_cpu_tensors_are_rejected_not_computed(built_lib):
    import lizard_cuda
    from lizard_cuda.decode import gla_decode_block, swa_decode_block
    x = torch.rand(1, 1, 4, 8)
    one = torch.ones(1)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        lizard_cuda.int8_linear(x, torch.zeros(3, 8, dtype=torch.int8), torch.ones(3))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        lizard_cuda.Int8Linear(torch.nn.Linear(8, 3))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        lizard_cuda.verify_drafts(x[0], x[0], torch.zeros(1, 3), one, one)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        gla_decode_block(x, x, x, one, x, one)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        swa_decode_block(x, x, x, one, one, one, x, x, one)


def test_a_cache_starts_token_by_token():
    from lizard_cuda.decode import LizardCache
    cache = LizardCache()
    assert not cache.drafting
    assert cache.draft() is cache and cache.drafting and cache.accepted is None
    cache.settle(None)
    assert not cache.drafting


def test_arguments_as_words(lib):
    """lz_call: the entry's own errors, and those of the words."""
    import struct

    def call(entry, *words, n=None):
        w = struct.pack(f"{len(words)}q", *words)
        return lib.lz_call(entry, w, len(words) if n is None else n)

    assert lib.lz_call(1, None, 21) == 1 and b"null" in _msg(lib)
    assert call(0, *range(32)) == 1 and b"unknown entry" in _msg(lib)
    assert call(6, *range(32)) == 1
    p = 0x1000
    gla = [p, p, p, p, 0, 0, 0, 0, 0, p, p, p, 2, 8, 2, 2, 4, 0, 64, 64, 0]
    assert call(1, *gla[:20]) == 1 and b"too few words" in _msg(lib)
    assert call(1, *gla[:13], 7, *gla[14:]) == 1 and b"divide" in _msg(lib)
    assert call(1, *gla[:12], 1 << 32, *gla[13:]) == 1 and b"does not fit" in _msg(lib)
    assert call(1, 0, *gla[1:]) == 1 and b"null" in _msg(lib)
    swa = [p, p, p, 0, 32, p, p, 0, 0, 0, 0, 0, 0, 0, 0, 0, p, p, p, p, 4, p, p, 1 << 30, 2, 8, 2, 4,
           0, 64, 64, 0]
    bad = [0, 0, 0, 1, 0, 0, 0, 2, 0, 0, 0, 1]
    assert len(swa) == 32
    assert call(2, *swa, *bad, *[0] * 8) == 1 and b"contiguous" in _msg(lib)
    assert call(2, *swa[:4], 60, *swa[5:], *bad, *[0] * 8) == 1 and b"does not fit" in _msg(lib)
    assert call(2, *swa[:4], 0, *swa[5:], *bad, *[0] * 8) == 1 and b"null" in _msg(lib)
    verify = struct.pack("13qd9q", p, 0, 0, p, 0, 0, 0, p, 1, p, p, 0, 0, 1.0, 0, p, p, p, 0, 2, 65, 9,
                         0)
    assert lib.lz_call(3, verify, 23) == 2 and b"at most 64" in _msg(lib)
    assert call(4, p, 16, p, p, 16, p, 0, 0, p, 0, 0, 0, 4, 4, 1 << 20, 0) == 2
    assert call(5, p, 0, 16, p, 8, p, 0, 0, p, 0, 0, 0, 4, 4, 16, 0) == 1
