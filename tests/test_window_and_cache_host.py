"""What the sliding-window and paged-cache entry points decide on the host, without a
GPU: statuses of bad arguments (no pointer is touched), workspace sizes, and which
pages a cache gives its sequences."""
import ctypes

import pytest
import torch

import hba_amd
from hba_amd import _lib, ops

FAKE = ctypes.c_void_p(16)
OFF = ctypes.c_void_p(24)                # not on 16 bytes
S2, S3 = (ctypes.c_int64 * 2)(64, 64), (ctypes.c_int64 * 3)(64, 64, 64)


def size(fn, *args):
    n = ctypes.c_size_t(0)
    return fn(*args, ctypes.byref(n)), n.value


def swa(B=1, n=5, Hq=4, Hkv=2, d=64, W=3, S=1, scale=0.1, dtype=1, q=FAKE, k=FAKE, out=FAKE, st=S3,
        kst=S3):
    return _lib.lib().hba_swa_fwd(dtype, q, st, k, kst, FAKE, S3, None, B, n, Hq, Hkv, d, W, S, scale, out, None,
                                  None)


@pytest.mark.parametrize("bad,status", [
    (dict(B=0), -1), (dict(n=0), -1), (dict(Hq=3), -1), (dict(Hkv=0), -1), (dict(W=0), -1), (dict(S=-1), -1),
    (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1),
    (dict(q=None), -1), (dict(out=None), -1), (dict(dtype=7), -2), (dict(d=96), -2), (dict(d=32), -2),
    (dict(q=OFF), -2), (dict(k=OFF), -2), (dict(st=(ctypes.c_int64 * 3)(64, 64, 63)), -2),
    (dict(kst=(ctypes.c_int64 * 3)(64, -64, 64)), -2), (dict(kst=(ctypes.c_int64 * 3)(64, 1 << 24, 64)), -2)])
def test_swa_refuses(bad, status):
    assert swa(**bad) == status


def test_swa_backward_refuses_a_short_workspace():
    L = _lib.lib()
    st, need = size(L.hba_swa_bwd_workspace_bytes, 1, 1, 500, 4, 2, 64, 100, 4)
    assert st == 0 and need >= 500 * 4 * 4

    def bwd(ws, nbytes):
        return L.hba_swa_bwd(1, FAKE, S3, FAKE, S3, FAKE, S3, FAKE, FAKE, FAKE, S3, None, 1, 500, 4, 2, 64, 100, 4, 0.1,
                             ws, nbytes, FAKE, FAKE, FAKE, None)

    assert bwd(FAKE, need - 1) == -1 and bwd(None, need) == -1 and bwd(OFF, need) == -2


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 63, 1000, 8192, 100000])
def test_swa_backward_workspace(n, d, dtype):
    """Every row's <dout, out>; of parts no more than four rounds of sink tiles' (768
    workgroups of 128 keys at most), one for every such tile and 32 for every other."""
    for W, S in ((1, 0), (64, 4), (1024, 8), (1, n), (64, n // 2), (1024, 4096), (n, 0), (n, n)):
        W, S = min(W, n), min(S, n)
        st, need = size(_lib.lib().hba_swa_bwd_workspace_bytes, dtype, 2, n, 8, 2, d, W, S)
        tiles, sinks = -(-n // 128), -(-S // 128)
        parts = 4 * 768 + 2 * sinks * 4 + 32 * (tiles - sinks) * 4
        assert st == 0 and 2 * 8 * n * 4 <= need <= 2 * 8 * n * 4 + parts * (128 * 2 * d * 4 + 16) + 1024


def paged(T=2, Bd=2, Hq=4, Hkv=2, d=64, Bk=64, W=0, S=0, shared=0, max_len=1000, maxp=16, pages=40, dtype=1, q=FAKE,
          st=S2, cu=None, cos=None, sin=None, n_tab=0, ws=FAKE, nbytes=1 << 30, out=FAKE):
    return _lib.lib().hba_paged_attn(dtype, q, st, None, 1e-6, cos, sin, n_tab, FAKE, FAKE, pages, FAKE, maxp, FAKE,
                                     FAKE, cu, T, Bd, Hq, Hkv, d, Bk, W, S, shared, max_len, ws, nbytes, out, None)


@pytest.mark.parametrize("bad,status", [
    (dict(T=0), -1), (dict(Bd=0, T=0), -1), (dict(T=3), -1), (dict(Hq=5), -1), (dict(W=-1), -1), (dict(S=-1), -1),
    (dict(shared=-1), -1), (dict(shared=1, W=5), -1), (dict(max_len=0), -1), (dict(pages=0), -1), (dict(q=None), -1),
    (dict(out=None), -1), (dict(cos=FAKE), -1), (dict(cos=FAKE, sin=FAKE), -1), (dict(d=96), -2), (dict(Bk=32), -2),
    (dict(shared=17), -2), (dict(max_len=1 << 31), -2), (dict(q=OFF), -2), (dict(out=OFF), -2),
    (dict(st=(ctypes.c_int64 * 2)(64, 60)), -2), (dict(max_len=9000, maxp=200, ws=None), -1),
    (dict(max_len=9000, maxp=200, nbytes=64), -1), (dict(max_len=9000, maxp=200, ws=OFF), -2)])
def test_paged_attention_refuses(bad, status):
    assert paged(**bad) == status


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("Bd", [1, 3, 64, 700])
def test_paged_attention_workspace(Bd, d):
    """None where nothing is cut; never more than a part for every page of a row, and
    for long decodes as much as the card's 256 workgroups leave at their ends."""
    L = _lib.lib()
    for max_len in (1, 64, 2048, 2049, 30000, 500000):
        for W, S in ((0, 0), (1000, 4), (4000, 100)):
            st, one = size(L.hba_paged_attn_workspace_bytes, Bd, Bd, 8, 2, d, W, S, 0, 1, max_len)
            assert st == 0 and one <= 256 * 32 * (d + 2) * 4
            if max_len <= 1920:
                assert one == 0
            st, many = size(L.hba_paged_attn_workspace_bytes, 5 * Bd, Bd, 8, 2, d, W, S, 0, 0, max_len)
            assert st == 0 and many <= 5 * Bd * 8 * (max_len // 64 + 4) * (d + 2) * 4
    st, pre = size(L.hba_paged_attn_workspace_bytes, Bd, Bd, 8, 2, d, 0, 0, 16, 1, 2000)
    assert st == 0 and pre >= 2 * Bd * 8 * (d + 2) * 4
    assert size(L.hba_paged_attn_workspace_bytes, Bd, Bd, 8, 3, d, 0, 0, 0, 1, 100)[0] == -1


def append(T=2, Bd=2, Hkv=2, d=64, Bk=64, m=4, pages=4, maxp=2, n_tab=128, dtype=1, k=FAKE, st=S2, kc=FAKE, kr=FAKE,
           probes=FAKE, proj=FAKE, summ=FAKE):
    return _lib.lib().hba_kv_append_ragged(dtype, k, st, FAKE, S2, FAKE, T, None, 1e-6, FAKE, FAKE, n_tab, FAKE, maxp,
                                           FAKE, Bd, Hkv, d, Bk, pages, kc, kr, FAKE, probes, proj, m, summ, None)


@pytest.mark.parametrize("bad,status", [
    (dict(T=-1), -1), (dict(Bd=-1), -1), (dict(Hkv=0), -1), (dict(pages=0), -1), (dict(k=None), -1), (dict(kr=None), -1),
    (dict(kc=None), -1), (dict(probes=None), -1), (dict(proj=None), -1), (dict(d=96), -2), (dict(Bk=16), -2),
    (dict(m=9), -2), (dict(k=OFF), -2), (dict(st=(ctypes.c_int64 * 2)(64, 60)), -2)])
def test_ragged_append_refuses(bad, status):
    assert append(**bad) == status


def test_there_is_no_cpu_path():
    q, k = torch.zeros(1, 8, 2, 64), torch.zeros(1, 8, 1, 64)
    with pytest.raises((RuntimeError, NotImplementedError)):
        hba_amd.sliding_attention(q, k, k, 4)
    with pytest.raises((RuntimeError, NotImplementedError)):
        hba_amd.sliding_attention(q.requires_grad_(), k, k, 4)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises((RuntimeError, NotImplementedError)):
        ops.paged_attn(torch.zeros(1, 2, 64), None, 1e-6, torch.zeros(1, 1, 4096), torch.zeros(1, 1, 4096),
                       i[:1].view(1, 1), i[:1], None, None, torch.ones(1), 1)
    with pytest.raises((RuntimeError, NotImplementedError)):
        ops.kv_append_ragged(torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), i, None, 1e-6, torch.zeros(64, 64),
                             torch.zeros(64, 64), i[:1].view(1, 1), i[:1], None, torch.zeros(1, 1, 4096),
                             torch.zeros(1, 1, 4096), None, None, None)


def test_shared_pages_belong_to_nobody_else():
    """share names the same pages; loading over them is refused; what follows gets its own."""
    cfg = hba_amd.HBAConfig(n_heads=4, n_kv=2, head_dim=64)
    cache = hba_amd.PagedKVCache(cfg, 4, 512, torch.float32, "cpu")
    cache._ensure_pages(1, 200)
    cache.lens[1] = 200
    with pytest.raises(ValueError):
        cache.share(1, 100, [0])                # not whole pages
    with pytest.raises(ValueError):
        cache.share(1, 256, [0])                # more than it holds
    with pytest.raises(ValueError):
        cache.share(1, 128, [0, 0])
    with pytest.raises(ValueError):
        cache.share(1, 128, [1])
    cache.share(1, 128, (s for s in (0, 3)))
    assert cache.lens == [128, 200, 0, 128] and cache.seq_lens.tolist() == cache.lens
    assert cache._table[0] == cache._table[3] == cache._table[1][:2]
    assert cache.page_table[0, :2].tolist() == cache.page_table[1, :2].tolist()
    with pytest.raises(ValueError):
        cache.share(2, 0, [3])                  # it is not empty any more
    for s in (0, 1, 3):
        with pytest.raises(ValueError):
            cache.load(s, *(torch.zeros(10, 2, 64) for _ in range(3)), None)
    for s in range(4):
        cache._ensure_pages(s, 300)
    own = [p for s in range(4) for p in (cache._table[s][2:] if s != 2 else cache._table[s])]
    assert len(set(own)) == len(own) and not set(own) & set(cache._table[0][:2])
