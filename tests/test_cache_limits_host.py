"""The paged caches at their limits, on the host: what attention plans for the largest windows,
sinks and sizes, and what the cache objects refuse.  Nothing here needs a GPU."""
import ctypes

import pytest
import torch

import hba_amd
from hba_amd import _lib

LARGEST = 2 ** 63 - 1


def workspace(mx, T, Bd, Hq, Hkv, d, W, S, shared, single, max_len):
    """(status, bytes): the most that 4 and 8 bits need, or (mx false) the cache of rows."""
    n, L = ctypes.c_size_t(0), _lib.lib()
    f = L.hba_paged_attn_mx_workspace_bytes if mx else L.hba_paged_attn_workspace_bytes
    return f(T, Bd, Hq, Hkv, d, W, S, shared, single, max_len, ctypes.byref(n)), n.value


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("single", [0, 1])
@pytest.mark.parametrize("max_len", [1, 64, 1000, 2000, 8000, 30000, 1 << 30])
def test_windows_and_sinks_past_every_length(max_len, single, mx):
    """They mean every key: the same plan as a window, or sinks, of the longest length."""
    T = 3 if single else 15

    def need(W, S):
        return workspace(mx, T, 3, 14, 2, 64, W, S, 0, single, max_len)

    every = need(max_len, 0)
    assert every[0] == 0 and every == need(0, 0)
    for W in (max_len + 1, 2 ** 31, 2 ** 62, LARGEST - 64, LARGEST):
        assert need(W, 0) == every and need(W, LARGEST) == need(max_len, max_len)
    for W in (1, 100, max_len):
        for S in (max_len + 1, 2 ** 31, LARGEST - 62, LARGEST):
            assert need(W, S) == need(W, max_len)


def caches(max_len, num_pages=None, batch=2):
    cfg = hba_amd.HBAConfig(n_heads=4, n_kv=2, head_dim=64)
    return [hba_amd.PagedKVCache(cfg, batch, max_len, torch.float32, "cpu", num_pages=num_pages),
            *(hba_amd.MXKVCache(cfg, batch, max_len, torch.float32, "cpu", bits=b, num_pages=num_pages) for b in (4, 8))]


def load(c, s, n, v=None):
    """n tokens into sequence s; their keys, or (v) other values."""
    x = torch.zeros(n, 2, 64)
    v = x if v is None else v
    c.load(s, x, v) if isinstance(c, hba_amd.MXKVCache) else c.load(s, x, x, v, None)


def test_a_load_past_the_longest_length_is_refused():
    """The last page holds more tokens than max_len allows: a length there has no scale."""
    for c in caches(50):
        with pytest.raises(ValueError, match="exceeds max_len"):
            load(c, 1, 60)
        assert c.lens == c.seq_lens.tolist() == [0, 0] and c._table == [[], []] and len(c._free) == 2
        c.scales()


def test_what_a_refused_call_took_is_given_back():
    """Pages that only the host's table names would be written as page 0 by the next append."""
    for c in caches(512, num_pages=3):
        assert c.max_pages == 8
        load_zeros = lambda: load(c, 0, 300)   # noqa: E731  five pages of three
        for f in (load_zeros, lambda: c.reserve(128), lambda: c.reserve(), lambda: c.reserve(600)):
            with pytest.raises((RuntimeError, ValueError)):
                f()
            assert c._table == [[], []] and sorted(c._free) == [0, 1, 2] and c.lens == [0, 0]
        for bad in (torch.zeros(70, 3, 64), torch.zeros(69, 2, 64)):   # refused once the pages are there
            with pytest.raises((RuntimeError, ValueError)):
                load(c, 1, 70, bad)
            assert c._table == [[], []] and sorted(c._free) == [0, 1, 2] and c.lens == [0, 0]
        c.reserve(64)
        assert [len(t) for t in c._table] == [1, 1] and c.page_table[:, 0].tolist() == [t[0] for t in c._table]


@pytest.mark.parametrize("pages", [16, -17, [0, 16], torch.tensor([3, -17]), torch.tensor([[2], [99]])])
def test_rows_of_pages_that_there_are_none_of(pages):
    """As of any tensor's index."""
    for c in caches(512):
        for f in (lambda: c.key_rows(pages, rotated=True), lambda: c.value_rows(pages)):
            with pytest.raises(IndexError):
                f()


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("T,Bd,Hq,Hkv", [(1, 2 ** 62, 8, 4), (1, 2 ** 60, 16, 16), (2 ** 62, 1, 4, 1), (2 ** 32, 1, 2 ** 32, 1),
                                         (2 ** 34, 2 ** 34, 2 ** 30, 2 ** 15), (5, 2 ** 58, 32, 2), (2 ** 63 - 1, 3, 2, 1)])
def test_sizes_whose_products_overflow(T, Bd, Hq, Hkv, mx):
    assert workspace(mx, T, Bd, Hq, Hkv, 64, 0, 0, 0, int(T == Bd), 1000) == (-2, 0)
