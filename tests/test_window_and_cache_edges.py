"""Calls of the window and cache operators at the edges of what their documentation
allows: state after an error, lengths of any type, launches of any size, pages with
anything behind their sequences, and every form that the gradients' kernels take."""
import pytest
import torch

import hba_amd
import test_gpu_append_ragged as ragged
from test_gpu_append_ragged import append


@pytest.mark.gpu
def test_autograd_sees_the_append():
    """A loss that saved the pages refuses its backward pass once they have changed."""
    s = ragged.setup(torch.float32, 64, 2, [3, 4], [2, 2])
    for name in ("kc", "kr", "vp", "summ"):
        w = torch.ones_like(s[name], requires_grad=True)
        loss = (w * s[name]).sum()
        append(s)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    with torch.inference_mode():
        t = {n: s[n].clone() for n in ("kc", "kr", "vp", "summ")}
    append(s, **t)
    append(s, summ=None)
    append(s, kc=None, summ=None)


def test_a_refused_extend_leaves_the_cache_as_it_was():
    """The append itself refuses (here: no GPU) after lengths and pages are planned."""
    cfg = hba_amd.HBAConfig(n_heads=4, n_kv=2, head_dim=64)
    qkn, summ = hba_amd.QKNorm(cfg), hba_amd.SlotSummarizer(cfg)
    cos, sin = hba_amd.rope_tables(512, 64, 1e4, "cpu")
    c = hba_amd.PagedKVCache(cfg, 3, 512, torch.float32, "cpu")
    c._ensure_pages(1, 70)
    c.lens[1] = 70
    c._sync_table()
    free, table = list(c._free), [list(t) for t in c._table]
    k = torch.zeros(200, 2, 64)
    with pytest.raises(RuntimeError):
        c.extend(k, k, [130, 70, 0], qkn, summ, cos, sin)
    assert c.lens == c.seq_lens.tolist() == [0, 70, 0]
    assert c._free == free and c._table == table


@pytest.mark.gpu
def test_extend_goes_on_after_a_refusal():
    x = ragged.Knobs()
    a, b = x.cache(), x.cache()
    k, v = x.kv(100)
    k2, v2 = x.kv(300)
    for c in (a, b):
        c.extend(k, v, [60, 0, 40], x.qkn, x.summ, x.cos, x.sin)
    wrong = hba_amd.SlotSummarizer(hba_amd.HBAConfig(n_heads=4, n_kv=2, head_dim=64, slots=9)).cuda()
    for args in ((x.summ, x.cos, x.sin[:400]), (x.summ, x.cos[:, :32], x.sin[:, :32]), (wrong, x.cos, x.sin)):
        with pytest.raises((ValueError, RuntimeError)):
            a.extend(k2, v2, [100, 150, 50], x.qkn, *args)
        assert a.lens == a.seq_lens.tolist() == [60, 0, 40] and not a._table[1]
    for c in (a, b):
        c.extend(k2, v2, [100, 150, 50], x.qkn, x.summ, x.cos, x.sin)
    k, v = x.kv(3)
    for c in (a, b):
        c.append(k, v, x.qkn, x.summ, x.cos, x.sin)
    assert a.lens == a.seq_lens.tolist() == b.lens and a._table == b._table
    for n in ("kc_pages", "kr_pages", "v_pages", "summ_pages", "page_table"):
        assert torch.equal(getattr(a, n), getattr(b, n))
