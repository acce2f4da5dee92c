"""Host argument checks of the page, shared-prefix attention and 8-bit product entry points (no GPU needed: every
call below is rejected before any CUDA call)."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from estudiocanciones_b200 import _lib, build
    build.build()
    return _lib.lib()


def state(**kw):
    from estudiocanciones_b200._lib import PageState
    a = dict(table=16, table_ld=8, lens=16, refs=16, err=None, n_seqs=4, max_pages=8, n_pages=16, page=64)
    a.update(kw)
    return C.byref(PageState(**a))


def pool(**kw):
    from estudiocanciones_b200._lib import PagePoolDesc
    a = dict(k=16, v=16, layers=2, n_pages=16, Hk=2, page=64, row_bytes=256)
    a.update(kw)
    return C.byref(PagePoolDesc(**a))


BAD_STATES = [dict(table=None), dict(lens=None), dict(refs=None), dict(n_seqs=0), dict(max_pages=0), dict(table_ld=7),
              dict(n_pages=0), dict(n_pages=(1 << 30) + 1), dict(page=0), dict(page=1025)]
BAD_POOLS = [dict(k=None), dict(v=None), dict(k=24), dict(layers=0), dict(Hk=0), dict(n_pages=15), dict(page=32),
             dict(row_bytes=8), dict(row_bytes=24)]


def test_page_calls(lib):
    for kw in BAD_STATES:
        assert lib.hm_pages_grow(state(**kw), 16, 1, 1, None) == -1
        assert lib.hm_pages_free(state(**kw), 16, 1, None) == -1
        assert lib.hm_pages_fork(state(**kw), pool(), 16, 16, 1, 16, 1 << 20, None) == -1
        if "lens" not in kw:
            assert lib.hm_pages_compact(state(**kw), pool(), 16, 16, 1 << 20, None) == -1
    for kw in BAD_POOLS:
        assert lib.hm_pages_fork(state(), pool(**kw), 16, 16, 1, 16, 1 << 20, None) == -1
        assert lib.hm_pages_compact(state(), pool(**kw), 16, 16, 1 << 20, None) == -1
        if "n_pages" not in kw and "page" not in kw:
            assert lib.hm_pages_copy(pool(**kw), 16, 16, 1, 16, 1 << 20, None, None) == -1
    for n in (0, -1, 1025):
        assert lib.hm_pages_grow(state(), 16, n, 1, None) == -1
        assert lib.hm_pages_free(state(), 16, n, None) == -1
        assert lib.hm_pages_fork(state(), pool(), 16, 16, n, 16, 1 << 20, None) == -1
        assert lib.hm_pages_copy(pool(), 16, 16, n, 16, 1 << 20, None, None) == -1
    assert lib.hm_pages_grow(state(), 16, 1, -1, None) == -1
    assert lib.hm_pages_grow(state(), None, 1, 1, None) == -1
    # scratch: missing, misaligned, too small
    need = lib.hm_pages_workspace_bytes(3, 0)
    for ws, n in ((None, need), (24, need), (16, need - 1)):
        assert lib.hm_pages_fork(state(), pool(), 16, 16, 3, ws, n, None) == -1
        assert lib.hm_pages_copy(pool(), 16, 16, 3, ws, n, None, None) == -1
    assert lib.hm_pages_compact(state(), pool(), 16, 16, lib.hm_pages_workspace_bytes(8, 16) - 1, None) == -1
    assert lib.hm_pages_compact(state(), pool(), None, 16, 1 << 20, None) == -1


def test_rope_pages(lib):
    good = dict(qkv=16, ldq=1536, rope=16, rows=64, pos=16, q=16, ld=1024, k=16, v=16, dt=2, table=16, tld=8, seqs=None,
                nt=4, mp=8, np=16, page=64, R=4, S=1, Hq=8, Hk=2, hd=128, err=None, st=None)
    for kw in (dict(qkv=None), dict(qkv=24), dict(rope=None), dict(pos=None), dict(q=24), dict(k=None), dict(v=18),
               dict(table=None), dict(dt=0), dict(ldq=1535), dict(ldq=1540), dict(ld=1016), dict(tld=7), dict(nt=3),
               dict(R=0), dict(S=0), dict(hd=12), dict(hd=0), dict(page=0), dict(np=0), dict(mp=0), dict(rows=0),
               dict(Hq=0), dict(Hk=0)):
        assert lib.hm_rope_pages(*{**good, **kw}.values()) == -1, kw


def test_prefix_attn(lib):
    from estudiocanciones_b200._lib import PrefixAttnDesc
    good = dict(q=16, ld_q=1024, o=16, ld_o=1024, k=16, v=16, pos=16, table=16, table_ld=8, seqs=None, gstart=16, owner=16,
                plen=16, ws=16, ws_bytes=1 << 40, err=None, dtype=2, R=4, S=1, Hq=8, Hk=2, hd=128, n_table=4, max_pages=8,
                n_pages=16, page=64, n_groups=1, scale=0.1)
    for kw in (dict(q=None), dict(q=24), dict(o=None), dict(k=24), dict(v=None), dict(pos=None), dict(table=None),
               dict(ws=None), dict(ws=24), dict(gstart=None), dict(owner=None), dict(plen=None), dict(ld_q=1020),
               dict(ld_q=1000), dict(ld_o=1016), dict(dtype=0), dict(R=0), dict(S=0), dict(S=3), dict(Hq=7), dict(Hk=0),
               dict(Hk=16), dict(hd=96), dict(n_table=3), dict(max_pages=0), dict(table_ld=7), dict(n_pages=0),
               dict(page=8), dict(page=24), dict(page=96), dict(n_groups=-1), dict(n_groups=1025), dict(R=1025, n_table=2000),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(n_pages=1 << 26), dict(max_pages=1 << 26, table_ld=1 << 26), dict(max_pages=1 << 22, table_ld=1 << 22)):
        assert lib.hm_prefix_attn(C.byref(PrefixAttnDesc(**{**good, **kw})), None) == -1, kw
    assert lib.hm_prefix_attn(None, None) == -1
    ws = lib.hm_prefix_attn_workspace_bytes
    assert ws(4, 1, 8, 2, 128, 1, 148) > 0 and ws(4, 1, 8, 2, 96, 1, 148) == 0 and ws(4, 3, 8, 2, 128, 1, 148) == 0
    assert ws(8, 1, 65 * 2, 2, 128, 1, 148) == 0


def test_integer_product(lib):
    quant = dict(x=16, ldx=128, dt=2, M=4, K=128, q=16, ldq=128, sx=16, st=None)
    for kw in (dict(x=None), dict(x=24), dict(ldx=120), dict(ldx=132), dict(dt=0), dict(M=0), dict(K=0), dict(K=120),
               dict(K=131088, ldx=131088, ldq=131088), dict(q=None), dict(q=24), dict(ldq=120), dict(ldq=130), dict(sx=None),
               dict(sx=18)):
        assert lib.hm_quant_tokens(*{**quant, **kw}.values()) == -1, kw
    gemm = dict(q=16, ldq=128, sx=16, dt=2, w=16, s=16, res=None, ldr=0, c=16, ldc=64, M=4, N=64, K=128, epi=0, err=None,
                st=None)
    for kw in (dict(q=None), dict(q=24), dict(ldq=120), dict(ldq=136), dict(sx=None), dict(dt=0), dict(w=24), dict(w=None),
               dict(s=None), dict(s=17), dict(res=16, ldr=63), dict(res=17, ldr=64), dict(c=None), dict(c=17), dict(ldc=63),
               dict(M=0), dict(N=0), dict(K=8), dict(K=100), dict(K=131088), dict(epi=1), dict(epi=2, N=63),
               dict(epi=2, res=16, ldr=64)):
        assert lib.hm_gemm_i8a8(*{**gemm, **kw}.values()) == -1, kw
    mm = dict(x=16, ldx=128, dt=2, w=16, s=16, res=None, ldr=0, c=16, ldc=64, M=4, N=64, K=128, epi=0, ws=16, wsb=1 << 20,
              err=None, st=None)
    for kw in (dict(x=None), dict(ldx=120), dict(dt=0), dict(w=None), dict(c=17), dict(ldc=10), dict(K=24, ldx=24), dict(M=0),
               dict(ws=None), dict(ws=24), dict(wsb=lib.hm_int8_mm_a8_workspace_bytes(4, 128) - 1), dict(epi=2, N=7)):
        assert lib.hm_int8_mm_a8(*{**mm, **kw}.values()) == -1, kw
    assert lib.hm_int8_mm_a8_workspace_bytes(0, 128) == 0
    assert lib.hm_int8_mm_a8_workspace_bytes(65, 128) == 512 + 65 * 128


def test_cpu_tensors_are_refused():
    """There is no CPU path: the Python calls raise before they reach the library."""
    import torch
    from estudiocanciones_b200 import kernels as K
    from estudiocanciones_b200._lib import HMError
    k = torch.zeros(2, 4, 1, 16, 64, dtype=torch.float16)
    table, lens, refs = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)
    ids = torch.zeros(1, dtype=torch.int32)
    q, pos = torch.zeros(1, 64, dtype=torch.float16), torch.zeros(1, dtype=torch.int64)
    x, w = torch.zeros(1, 64, dtype=torch.float16), torch.zeros(8, 64, dtype=torch.int8)
    s = torch.ones(8, dtype=torch.float16)
    for f in (lambda: K.pages_grow(table, lens, refs, 16, ids), lambda: K.pages_free(table, lens, refs, ids),
              lambda: K.pages_fork(k, k, table, lens, refs, ids, ids), lambda: K.pages_copy(k, k, ids, ids),
              lambda: K.pages_compact(k, k, table, refs), lambda: K.prefix_attn(q, k[0], k[0], table, pos),
              lambda: K.rope_pages(q, torch.zeros(4, 32, 2), pos, q, k[0], k[0], table, 1, 1, 1),
              lambda: K.quant_tokens(x), lambda: K.int8_mm_a8(x, w, s),
              lambda: K.gemm_i8a8(w, torch.ones(8), w, s)):
        with pytest.raises(HMError):
            f()


def test_pool_sizes_that_no_call_takes():
    """Refused when the pool is made, not at the first call."""
    import torch
    from estudiocanciones_b200._lib import HMError
    from estudiocanciones_b200.pages import PagePool
    PagePool(1, 2, 1, 8, 1, 1024, 1024, torch.float16, "cpu")
    for kw in (dict(page=1025), dict(hd=4), dict(hd=12), dict(hd=100), dict(page=0), dict(n_pages=0), dict(dtype=torch.float32)):
        a = dict(layers=1, n_pages=2, kv_heads=1, hd=64, max_seqs=1, max_len=64, page=16, dtype=torch.float16)
        with pytest.raises(HMError):
            PagePool(**{**a, **kw}, device="cpu")


def test_descriptor_layouts(lib):
    from estudiocanciones_b200 import _lib
    assert _lib.abi_mismatches() == []
