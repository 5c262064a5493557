"""The cache in 4 and 8 bits on the host: its format, what the entry points refuse, and
the cache object's bookkeeping.  Nothing here needs a GPU."""
import ctypes

import pytest
import torch

import hba_amd
import mx64
from hba_amd import _lib, ops
from hba_amd.build import overlaps

FAKE, OFF = 0x10000, 0x10008
S2 = (ctypes.c_int64 * 2)(128, 64)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128])
def test_every_code_and_scale_has_its_place(d, bits):
    assert ops.mx_page_bytes(d, bits) == mx64.page_bytes(d, bits)
    for keys in (True, False):
        at, high, sc = mx64.places(d, bits, keys)
        half = at * 2 + high.int() if bits == 4 else at
        assert half.unique().numel() == 64 * d and int(half.max()) == 64 * d - 1
        assert sc.unique().numel() == 2 * d and int(sc.min()) == 64 * d * bits // 8
        assert int(sc.max()) == ops.mx_page_bytes(d, bits) - 1


@pytest.mark.parametrize("bits", [4, 8])
def test_what_a_page_holds(bits):
    """The definition against itself: values of codes are their own codes, the largest
    magnitude decides the scale, and nothing is further off than half a step of its size."""
    torch.manual_seed(0)
    x = torch.randn(500, 64) * torch.exp2(torch.randint(-20, 20, (500, 1)).float())
    c, b = mx64.quantise(x, bits)
    y = mx64.values(c, b, bits)
    again = mx64.values(*mx64.quantise(y, bits), bits)
    assert torch.equal(y, again)
    big = x.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).double()
    # the step at the top is 2 of at most 7 (e2m1), 32 of at most 448; e2m1 cuts 7 to 6
    assert bool(((y - x).unflatten(-1, (-1, 32)).abs() <= big * (1 / 3.5 if bits == 4 else 1 / 14)).all())
    if bits == 8:
        import numpy as np
        f8 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
        mine = mx64.values(torch.arange(256, dtype=torch.uint8)[None].expand(1, 256),
                           torch.full((1, 8), 127, dtype=torch.uint8), 8)[0]
        assert np.array_equal(f8.numpy(), mine.numpy(), equal_nan=True)
    assert mx64.quantise(torch.tensor([[7.0] + [0.0] * 31]), 4)[1].item() == 127
    assert mx64.quantise(torch.tensor([[7.0001] + [0.0] * 31]), 4)[1].item() == 128
    assert mx64.quantise(torch.tensor([[float("inf")] + [1.0] * 31]), 4)[1].item() == 255


def append(T=2, Bd=2, Hkv=2, d=64, Bk=64, bits=4, pages=4, maxp=2, n_tab=128, dtype=1, k=FAKE, st=S2, cu=FAKE, cos=FAKE,
           sin=FAKE, kp=FAKE, vp=FAKE):
    return _lib.lib().hba_kv_append_mx(dtype, k, st, FAKE, S2, cu, T, None, 1e-6, cos, sin, n_tab, FAKE, maxp, FAKE, Bd,
                                       Hkv, d, Bk, bits, pages, kp, vp, None)


@pytest.mark.parametrize("bad,status", [
    (dict(T=-1), -1), (dict(Bd=0), -1), (dict(Hkv=0), -1), (dict(pages=0), -1), (dict(maxp=0), -1), (dict(k=None), -1),
    (dict(kp=None), -1), (dict(vp=None), -1), (dict(cos=None), -1), (dict(n_tab=0), -1), (dict(cu=None, T=3), -1),
    (dict(d=96), -2), (dict(Bk=16), -2), (dict(bits=6), -2), (dict(k=OFF), -2), (dict(kp=OFF), -2), (dict(dtype=2), -2),
    (dict(st=(ctypes.c_int64 * 2)(64, 60)), -2), (dict(T=1 << 31), -2), (dict(T=1 << 24, Bd=1 << 24), -2)])
def test_append_refuses(bad, status):
    assert append(**bad) == status


def read(T=2, Bd=2, Hkv=2, d=64, Bk=64, bits=4, pages=4, maxp=2, dtype=1, cu=FAKE, kp=FAKE, k=FAKE, v=FAKE):
    return _lib.lib().hba_kv_read_mx(dtype, kp, FAKE, pages, FAKE, maxp, FAKE, cu, T, Bd, Hkv, d, Bk, bits, k, v, None)


@pytest.mark.parametrize("bad,status", [
    (dict(T=-1), -1), (dict(Bd=0), -1), (dict(Hkv=0), -1), (dict(pages=0), -1), (dict(k=None), -1), (dict(kp=None), -1),
    (dict(cu=None, T=3), -1), (dict(d=32), -2), (dict(Bk=16), -2), (dict(bits=16), -2), (dict(k=OFF), -2),
    (dict(v=OFF), -2), (dict(kp=OFF), -2), (dict(T=1 << 31), -2), (dict(T=1 << 30, Bd=1 << 24), -2)])
def test_read_refuses(bad, status):
    assert read(**bad) == status


def attend(T=2, Bd=2, Hq=4, Hkv=2, d=64, Bk=64, bits=4, W=0, S=0, shared=0, max_len=1000, maxp=16, pages=40, dtype=1,
           q=FAKE, st=S2, cu=None, cos=None, sin=None, n_tab=0, ws=FAKE, nbytes=1 << 30, out=FAKE):
    return _lib.lib().hba_paged_attn_mx(dtype, q, st, None, 1e-6, cos, sin, n_tab, bits, FAKE, FAKE, pages, FAKE, maxp,
                                        FAKE, FAKE, cu, T, Bd, Hq, Hkv, d, Bk, W, S, shared, max_len, ws, nbytes, out, None)


@pytest.mark.parametrize("bad,status", [
    (dict(bits=2), -2), (dict(T=0), -1), (dict(T=3), -1), (dict(Hq=5), -1), (dict(W=-1), -1), (dict(S=-1), -1),
    (dict(shared=1, W=5), -1), (dict(max_len=0), -1), (dict(pages=0), -1), (dict(q=None), -1), (dict(out=None), -1),
    (dict(cos=FAKE), -1), (dict(cos=FAKE, sin=FAKE), -1), (dict(d=96), -2), (dict(Bk=32), -2), (dict(shared=17), -2),
    (dict(max_len=1 << 31), -2), (dict(q=OFF), -2), (dict(out=OFF), -2), (dict(st=(ctypes.c_int64 * 2)(64, 60)), -2),
    (dict(max_len=9000, maxp=200, ws=None), -1), (dict(max_len=9000, maxp=200, nbytes=64), -1),
    (dict(max_len=9000, maxp=200, ws=OFF), -2)])
def test_attention_refuses(bad, status):
    assert attend(**bad) == status


def test_there_is_no_cpu_path():
    i = torch.zeros(2, dtype=torch.int32)
    p = torch.zeros(1, 1, ops.mx_page_bytes(64, 4), dtype=torch.uint8)
    x = torch.zeros(1, 1, 64)
    for f in (lambda: ops.kv_append_mx(x, x, i, None, 1e-6, None, None, i[:1].view(1, 1), i[:1], p, p),
              lambda: ops.kv_read_mx(p, p, i[:1].view(1, 1), i[:1], i, 1, 64, torch.float32),
              lambda: ops.paged_attn_mx(x, None, 1e-6, p, p, i[:1].view(1, 1), i[:1], None, None, torch.ones(1), 1)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            f()


def make(batch=3, **kw):
    cfg = hba_amd.HBAConfig(n_heads=4, n_kv=2, head_dim=64)
    return cfg, hba_amd.MXKVCache(cfg, batch, 512, torch.float32, "cpu", **kw)


def test_the_cache_has_as_many_bits_as_asked_for():
    for bits, nbytes in ((4, 2176), (8, 4224)):
        c = make(bits=bits)[1]
        assert c.k_pages.shape == c.v_pages.shape == (24, 2, nbytes) and c.k_pages.dtype == torch.uint8
    with pytest.raises(ValueError):
        make(bits=6)


def test_a_refused_append_leaves_the_cache_as_it_was():
    """The append itself refuses (here: no GPU) after lengths and pages are planned."""
    cfg, c = make()
    qkn = hba_amd.QKNorm(cfg)
    cos, sin = hba_amd.rope_tables(512, 64, 1e4, "cpu")
    c._ensure_pages(1, 64)
    c.lens[1] = 64
    c._sync_table()
    free, table = list(c._free), [list(t) for t in c._table]
    k = torch.zeros(200, 2, 64)
    for f in (lambda: c.extend(k, k, [130, 70, 0], qkn, cos, sin), lambda: c.append(k[:3], k[:3], qkn, cos, sin),
              lambda: c.load(0, k, k), lambda: c.read([0, 65, 0]), lambda: c.read([0, 64])):
        with pytest.raises((RuntimeError, ValueError)):
            f()
        assert c.lens == c.seq_lens.tolist() == [0, 64, 0]
        assert c._free == free and c._table == table
    for bad in (dict(counts=[1, 1, -2]), dict(counts=[600, 0, 0]), dict(counts=[200, 0])):
        with pytest.raises(ValueError):
            c.extend(torch.zeros(max(0, sum(bad["counts"])), 2, 64), torch.zeros(max(0, sum(bad["counts"])), 2, 64),
                     bad["counts"], qkn, cos, sin)


def test_sharing_is_the_paged_caches():
    cfg, c = make(4)
    c._ensure_pages(1, 200)
    c.lens[1] = 200
    c.share(1, 128, [0, 3])
    assert c.lens == [128, 200, 0, 128] and c._table[0] == c._table[3] == c._table[1][:2]
    with pytest.raises(ValueError):
        c.load(0, *(torch.zeros(10, 2, 64) for _ in range(2)))


def test_the_selection_needs_the_other_cache():
    cfg, c = make()
    qkn, summ = hba_amd.QKNorm(cfg), hba_amd.SlotSummarizer(cfg)
    cos, sin = hba_amd.rope_tables(512, 64, 1e4, "cpu")
    with pytest.raises(TypeError, match="MXKVCache"):
        hba_amd.hba_decode_step(torch.zeros(3, 4, 64), c, cfg, qkn, cos, sin)
    with pytest.raises(TypeError, match="MXKVCache"):
        hba_amd.DecodeLoop(c, cfg, qkn, summ, cos, sin)
    with pytest.raises(ValueError):
        c.key_rows(0, rotated=False)


def test_conversions_that_write_over_their_operands_are_found():
    good = """
\tv_cvt_scalef32_2xpk16_fp6_f32 v[66:71], v[50:65], v[34:49], v72
\tv_cvt_scalef32_pk32_f32_fp6 v[2:33], v[66:71], v72
\tv_cvt_scalef32_pk_bf16_fp4 v3, v3, v4 op_sel:[1,0,0]
"""
    assert not overlaps(good)
    bad = ["\tv_cvt_scalef32_2xpk16_fp6_f32 v[2:7], v[50:65], v[34:49], v2",
           "\tv_cvt_scalef32_2xpk16_fp6_f32 v[50:55], v[50:65], v[34:49], v72",
           "\tv_cvt_scalef32_pk32_f32_fp6 v[2:33], v[28:33], v72", "\tv_cvt_scalef32_pk32_f32_fp6 v[2:33], v[66:71], v9"]
    assert [s for _, s in overlaps(good + "\n".join(bad))] == [b.strip() for b in bad]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("Bd", [1, 3, 64, 700, 1500])
def test_attention_workspace(Bd, d):
    """Parts of 256 workgroups at most where the lists are shared out evenly (two of 128 rows
    each, and 16 bytes a row tile), or of every page of a row at most, whichever of 4 and 8 bits
    needs more; none for short single tokens."""
    L = _lib.lib()

    def need(T, W, S, shared, single, max_len, Hq=8, Hkv=2):
        n = ctypes.c_size_t(0)
        st = L.hba_paged_attn_mx_workspace_bytes(T, Bd, Hq, Hkv, d, W, S, shared, single, max_len, ctypes.byref(n))
        return st, n.value

    for max_len in (1, 64, 2048, 2049, 30000, 500000):
        for W, S in ((0, 0), (1000, 4), (4000, 100)):
            st, one = need(Bd, W, S, 0, 1, max_len)
            assert st == 0 and one <= 256 * 32 * (d + 2) * 4 + Bd * 2 * 8
            if max_len <= 1920:
                assert one == 0
            st, many = need(5 * Bd, W, S, 0, 0, max_len)
            tiles = -(-5 * Bd * 4 // 128) + Bd
            even = 256 * 2 * 128 * (d + 2) * 4 + (1 + 2 * tiles) * 16
            assert st == 0 and many <= max(even if Bd <= 1024 and tiles <= 2048 else 0, 5 * Bd * 8 * (max_len // 64 + 4) * (d + 2) * 4)
    st, pre = need(Bd, 0, 0, 16, 1, 2000)
    assert st == 0 and pre >= 2 * Bd * 8 * (d + 2) * 4
    assert need(Bd, 0, 0, 0, 1, 100, Hkv=3)[0] == -1
