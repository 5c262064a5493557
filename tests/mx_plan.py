"""How attention over the cache in 4 and 8 bits shares its keys out: the rule restated, the
workspace of each form, and batches that reach them.

A 128-row tile of a KV head's queries (token, head) has a list of keys, a decoded sequence a
list of pages for each KV head's 16 query heads (a group).  Lists are worked on whole, in runs
of pages, or as one list of all that the workgroups take even shares of.
"""
import ctypes

import torch

import hba_amd
import mx64
from hba_amd import _lib

FAKE, OFF = 0x10000, 0x10008
CUS, MOST, TILES = 256, 1024, 2048   # workgroups; sequences, row tiles that are shared out at most


def ceil(a, b):
    return -(-a // b)


def pages_of(T, Bd, Hq, Hkv, W, S, single, max_len):
    """Pages of the longest list, an upper bound."""
    keys = max_len
    if W and single:
        keys = min(W, max_len)
    elif W:
        keys = min(W + 128 // (Hq // Hkv) + 1, max_len)
    return max(1, min(ceil(keys, 64) + 1 + (ceil(min(S, max_len), 64) if W else 0), ceil(max_len, 64)))


def runs(pages, base, most, least):
    """(parts of a list, pages of one)."""
    parts = max(1, min(max(min(most // base, pages // least), CUS // base), pages))
    per = ceil(pages, parts)
    return ceil(pages, per), per


def workspace(bits, T, Bd, Hq, Hkv, d, W, S, single, max_len):
    """(form, bytes) without shared pages."""
    G, pages = Hq // Hkv, pages_of(T, Bd, Hq, Hkv, W, S, single, max_len)
    if single:
        groups = Bd * Hkv * ceil(G, 16)
        if pages > 32 and groups < 1024:
            shares = min(CUS, groups * pages // 8 + 1)
            return "shares", shares * 32 * (d + 2) * 4 + groups * 8
        return "whole", 0
    tiles = ceil(T * G, 128) + Bd
    every = tiles * Hkv * pages
    enough = every >= 512 if bits == 8 and d == 128 else pages > 32 and every >= 2048
    if enough and Bd <= MOST and tiles <= TILES and tiles * Hkv <= 1 << 19 and every < 1 << 29:
        return "shares", min(CUS, every // 2 + 1) * 2 * 128 * (d + 2) * 4 + (1 + tiles * Hkv) * 16
    n = runs(pages, ceil(T * G, 128) * Hkv, 1024, 8)[0]
    return ("runs", T * Hq * n * (d + 2) * 4) if n > 1 else ("whole", 0)


def asked(bits, T, Bd, Hq, Hkv, d, W, S, single, max_len):
    """The bytes that the call itself asks for with so many bits: the fewest that it does not
    refuse as too few.  (Their place is refused next, so nothing is launched; a call that
    needs none would be, so this is for machines without a GPU.)"""
    assert not torch.cuda.is_available()
    cu, st = None if single else FAKE, (ctypes.c_int64 * 2)(Hq * d, d)

    def status(n):
        return _lib.lib().hba_paged_attn_mx(1, FAKE, st, None, 1e-6, None, None, 0, bits, FAKE, FAKE, 9, FAKE, 1 << 24, FAKE,
                                            FAKE, cu, T, Bd, Hq, Hkv, d, 64, W, S, 0, max_len, OFF, n, FAKE, None)

    n = ctypes.c_size_t(0)
    assert _lib.lib().hba_paged_attn_mx_workspace_bytes(T, Bd, Hq, Hkv, d, W, S, 0, single, max_len, ctypes.byref(n)) == 0
    lo, hi = -1, n.value                 # too few, enough
    assert status(hi) != -1
    while hi - lo > 1:
        mid = (lo + hi) // 2
        lo, hi = (mid, hi) if status(mid) == -1 else (lo, mid)
    return hi


def decode_shares(bits, d, Hq, Hkv, lens, W, S, max_len):
    """Of single tokens that are shared out: (whether every workgroup has one part of a list at
    most, else it takes what comes next whatever lists that belongs to; the most shares that a
    list lies in)."""
    groups = Hkv * ceil(Hq // Hkv, 16)
    pages = []
    for n in lens:
        lo = max(0, n - W) if W else 0
        first = lo // 64
        pages.append(max(1, min(ceil(min(S, n), 64) if W else 0, first) + ceil(n, 64) - first))
    shares = min(CUS, len(lens) * groups * pages_of(1, len(lens), Hq, Hkv, W, S, 1, max_len) // 8 + 1)
    per = max(8, ceil(sum(pages) * groups, shares))
    for c in range(16):
        if sum(ceil(n, per + c) for n in pages) * groups <= shares:
            return True, max(ceil(n, per + c) for n in pages)
    at, most = 0, 0
    for n in pages:
        for _ in range(groups):
            most = max(most, (at + n - 1) // per - at // per + 1)
            at += n
    return False, most


class _Rows:
    """Rows of each sequence, from pages that several may have."""

    def __init__(self, held, table):
        self.held, self.table = held, table

    def __getitem__(self, s):
        Hkv, d = self.held[0].shape[1], self.held[0].shape[3]
        return [x[self.table[s].long()].transpose(0, 1).reshape(Hkv, -1, d) for x in self.held]


def pooled(dt, d, bits, Hq, Hkv, lens, new=None, max_len=None, pool=24, seed=0):
    """A batch as test_gpu_mx_cache.setup makes it, of long sequences: their pages are drawn
    from a few.  max_len: also the page table's width."""
    g = torch.Generator().manual_seed(seed)
    Bd, T = len(lens), len(lens) if new is None else sum(new)
    max_len = max_len or max(1, max(lens))
    maxp = ceil(max_len, 64)
    table = torch.randint(0, pool, (Bd, maxp), generator=g).int()
    pages, held = [], []
    for keys in (True, False):
        p = torch.zeros(pool, Hkv, mx64.page_bytes(d, bits), dtype=torch.uint8)
        c, b = mx64.quantise(torch.randn(pool, Hkv, 64, d, generator=g) * (d ** 0.25 if keys else 1.0), bits)
        for i in range(pool):
            for h in range(Hkv):
                mx64.write(p[i, h], torch.arange(64), c[i, h], b[i, h], bits, keys)
        pages.append(p)
        held.append(mx64.values(c, b, bits))
    short = ceil(max(1, max(lens)), 64)
    cos, sin = hba_amd.rope_tables(maxp * 64, d, 1e4, "cpu")
    return dict(q=torch.randn(T, Hq, d, generator=g).to(dt), gain=1.2 + 0.1 * torch.randn(Hq, generator=g), kp=pages[0],
                vp=pages[1], table=table, lens=torch.tensor(lens, dtype=torch.int32), cos=cos, sin=sin,
                scales=(0.5 + torch.rand(Bd, generator=g)) / d, rows=_Rows(held, table[:, :short]), new=new, shared=0,
                bits=bits, cu=None if new is None else torch.tensor([0] + new).cumsum(0).int(), max_len=max_len)


# Parts of prompts: name -> (lengths, new tokens, Hq, Hkv, max_len).  All are shared out with
# W = 0 and W = 2100 but those named "over".
PARTS = {
    "a share crosses heads": ([300, 9, 0, 1500, 64], [300, 0, 0, 700, 64], 3, 3, 6000),
    "a tile in many shares": ([2000], [1], 32, 2, 40000),
    "pieces of one tile": ([65] * 200, [1] * 200, 2, 2, 4000),
    "tokens behind the cache": ([3, 10, 0, 700], [5, 12, 4, 300], 6, 2, 20000),
    "more sequences than a scan takes at once": ([1 + 7 * i % 130 for i in range(600)], [i % 3 for i in range(600)], 2, 1, 4000),
    "most sequences": ([1 + 7 * i % 60 for i in range(MOST)], [i % 2 for i in range(MOST)], 2, 1, 4000),
    "over most sequences": ([1 + 7 * i % 60 for i in range(MOST + 1)], [i % 2 for i in range(MOST + 1)], 2, 1, 4000),
    "most row tiles": ([40] * 32, [16] * 24 + [15] * 8, 512, 1, 4000),
    "over most row tiles": ([40] * 32, [16] * 25 + [15] * 7, 512, 1, 4000),
}
# Single tokens: name -> (lengths, Hq, Hkv, W, S, one part a workgroup, the most shares of a list)
DECODE = {
    "alike": ([2100] * 9, 6, 3, 0, 0),
    "uneven": ([300 + 37 * i for i in range(30)] + [9000, 8000, 0, 1, 5200], 8, 8, 0, 0),
    "very uneven": ([64 + i for i in range(120)] + [9000, 4000, 9000], 4, 2, 0, 0),
    "many heads of a group": ([300 + 37 * i for i in range(60)] + [6000, 1, 7000], 34, 2, 0, 0),
    "windows": ([2000 + 99 * i for i in range(50)], 6, 6, 2200, 70),
    "long windows": ([100 + 31 * i for i in range(60)] + [9000] * 4, 8, 4, 6000, 130),
}
