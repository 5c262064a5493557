"""The ragged append (ops.kv_append_ragged, PagedKVCache.extend): the bits of appending
token by token, what it leaves alone, and what it refuses."""
import pytest
import torch

import hba_amd
from attn64 import assert_within, norm_rotate, unit
from hba_amd import ops
from hba_amd.decode import key_offsets, value_offsets

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


def setup(dt, d, Hkv, old, new, m=4, maxp=6, extra=3, seed=0):
    g = torch.Generator().manual_seed(seed)
    Bd, T = len(old), sum(new)
    P = Bd * maxp + extra
    s = dict(k=torch.randn(T, Hkv, d, generator=g).to(dt).cuda(), v=torch.randn(T, Hkv, d, generator=g).to(dt).cuda(),
             gain=(1.5 + 0.1 * torch.randn(Hkv, generator=g)).cuda(),
             table=torch.randperm(P, generator=g)[:Bd * maxp].view(Bd, maxp).int().cuda(),
             lens=torch.tensor([a + b for a, b in zip(old, new)], dtype=torch.int32).cuda(),
             cu=torch.tensor([0] + new).cumsum(0).int().cuda(),
             probes=(torch.randn(Hkv, m, d, generator=g) * d ** -0.5).cuda(),
             proj=(torch.eye(d) + 0.02 * torch.randn(Hkv, d, d, generator=g)).cuda())
    s["cos"], s["sin"] = hba_amd.rope_tables(maxp * 64, d, 1e4, "cpu")
    s["cos"], s["sin"] = s["cos"].cuda(), s["sin"].cuda()
    for name, w in (("kc", 64 * d), ("kr", 64 * d), ("vp", 64 * d), ("summ", m * d)):
        s[name] = torch.randn(P, Hkv, w, generator=g).to(dt).cuda()
    s["summ"] = s["summ"].view(P, Hkv, m, d)
    return s


def append(s, **kw):
    a = {**s, **kw}
    ops.kv_append_ragged(a["k"], a["v"], a["cu"], a["gain"], EPS, a["cos"], a["sin"], a["table"], a["lens"], a["kc"],
                         a["kr"], a["vp"], a["probes"], a["proj"], a["summ"])


def bits(t):
    return t.view(torch.int16 if t.element_size() == 2 else torch.int32)


def one_by_one(s, old, new):
    """The same tokens through hba_kv_append, and the filled pages' summaries."""
    c = {n: s[n].clone() for n in ("kc", "kr", "vp", "summ")}
    cu = s["cu"].tolist()
    for b in range(len(old)):
        for i in range(new[b]):
            n = old[b] + i + 1
            ops.kv_append(s["k"][cu[b] + i][None], s["v"][cu[b] + i][None], s["gain"], EPS, s["cos"], s["sin"],
                          s["table"][b:b + 1].contiguous(), torch.tensor([n], dtype=torch.int32).cuda(), c["kc"],
                          c["kr"], c["vp"])
        full = s["table"][b, old[b] // 64:(old[b] + new[b]) // 64]
        if full.numel():
            ops.summarize_pages(c["kc"], full, s["probes"], s["proj"], c["summ"])
    return c


CASES = [([0], [1]), ([0], [64]), ([63], [1]), ([62], [3]), ([0], [65]), ([1], [127]), ([0, 5, 64], [0, 0, 1]),
         ([10, 0, 100, 63], [7, 200, 28, 130]), ([0] * 5, [1, 2, 3, 0, 4]), ([5, 300], [300, 0])]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("old,new", CASES)
def test_bits_of_single_appends(old, new, dt, d):
    s = setup(DT[dt], d, 2, old, new, seed=len(old) + new[0])
    want = one_by_one(s, old, new)
    before = s["kr"].clone()
    append(s)
    for name in ("kc", "vp", "summ"):       # pages that nothing is appended to among them
        assert torch.equal(bits(s[name]), bits(want[name])), name
    if dt == "f32":
        assert torch.equal(bits(s["kr"]), bits(want["kr"]))
    off, cu = key_offsets(d), s["cu"].tolist()
    wr, bound = before.double().cpu(), torch.zeros(before.shape, dtype=torch.float64)
    for b in range(len(old)):
        pos = torch.arange(old[b], old[b] + new[b])
        _, y, e = norm_rotate(s["k"][cu[b]:cu[b + 1]].cpu(), s["gain"].cpu(), EPS, s["cos"].cpu()[pos],
                              s["sin"].cpu()[pos], unit(DT[dt]))
        for i, p in enumerate(pos.tolist()):
            page = int(s["table"][b, p // 64])
            wr[page][:, off[p % 64]], bound[page][:, off[p % 64]] = y[i], e[i]
    assert_within(s["kr"], wr, bound, "kr")
    first = [s[n].clone() for n in ("kc", "kr", "vp", "summ")]
    append(s)                               # nothing is advanced: the same again
    assert all(torch.equal(bits(a), bits(s[n])) for a, n in zip(first, ("kc", "kr", "vp", "summ")))


@pytest.mark.parametrize("m", [1, 3, 8])
def test_slots_heads_and_no_norm(m):
    old, new = [30, 0], [100, 64]
    s = setup(torch.bfloat16, 64, 5, old, new, m=m)
    s["gain"] = None
    want = one_by_one(s, old, new)
    append(s)
    for name in ("kc", "vp", "summ"):
        assert torch.equal(bits(s[name]), bits(want[name])), name


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_strides_and_optional_pages(dt):
    old, new = [50, 3], [90, 61]
    s = setup(DT[dt], 64, 2, old, new)
    both = {n: s[n].clone() for n in ("kc", "kr", "vp", "summ")}
    append(s)
    T = sum(new)
    kv = torch.stack((s["k"], s["v"]), 1)                                # [T, 2, H, d]
    odd = torch.nn.functional.pad(s["k"], (1, 2))[..., 1:-2]             # rows off 16 bytes
    heads = s["v"].transpose(0, 1).contiguous().transpose(0, 1)
    assert kv.shape[0] == T
    for k, v in ((kv[:, 0], kv[:, 1]), (odd, heads)):
        c = {n: t.clone() for n, t in both.items()}
        append(s, k=k, v=v, **c)
        assert all(torch.equal(bits(c[n]), bits(s[n])) for n in c)
    c = {n: t.clone() for n, t in both.items()}
    append(s, **{**c, "summ": None})
    assert torch.equal(bits(c["kc"]), bits(s["kc"])) and torch.equal(bits(c["kr"]), bits(s["kr"]))
    c = {n: t.clone() for n, t in both.items()}
    append(s, **{**c, "kc": None, "summ": None})
    assert torch.equal(bits(c["kr"]), bits(s["kr"])) and torch.equal(bits(c["vp"]), bits(s["vp"]))


def test_many_sequences():
    """More sequences than a workgroup has threads, most of them without tokens."""
    g = torch.Generator().manual_seed(3)
    old = torch.randint(0, 120, (700,), generator=g).tolist()
    new = (torch.randint(0, 4, (700,), generator=g) * (torch.rand(700, generator=g) < 0.3)).tolist()
    s = setup(torch.bfloat16, 64, 1, old, new, maxp=2)
    want = one_by_one(s, old, new)
    append(s)
    for name in ("kc", "vp", "summ"):
        assert torch.equal(bits(s[name]), bits(want[name])), name


def test_places_that_are_not_there():
    """Tokens past the page table or the rotation tables, below position 0, or on a page
    outside the cache are left out; the others arrive."""
    old, new = [370, 10, 10], [30, 40, 20]
    s = setup(torch.float32, 64, 1, old, new)
    ref = {n: s[n].clone() for n in ("kc", "kr", "vp", "summ")}
    c = {n: t.clone() for n, t in ref.items()}
    short = s["cos"][:380].contiguous(), s["sin"][:380].contiguous()
    lens = s["lens"].clone()
    lens[1] = 15                    # 40 tokens end at position 14: the first 25 have no place
    table = s["table"].clone()
    table[2, 0] = 10 ** 6
    append(s, cos=short[0], sin=short[1], lens=lens, table=table, **c)
    want = {n: t.clone() for n, t in ref.items()}
    cu = s["cu"].tolist()
    for b, toks, first in ((0, range(cu[0], cu[0] + 10), 370), (1, range(cu[1] + 25, cu[1] + 40), 0)):
        for i, t in enumerate(toks):
            ops.kv_append(s["k"][t][None], s["v"][t][None], s["gain"], EPS, s["cos"], s["sin"],
                          s["table"][b:b + 1].contiguous(), torch.tensor([first + i + 1], dtype=torch.int32).cuda(),
                          want["kc"], want["kr"], want["vp"])
    assert all(torch.equal(bits(c[n]), bits(want[n])) for n in c)
    append(s, lens=torch.full_like(lens, -3), **c)
    assert all(torch.equal(bits(c[n]), bits(want[n])) for n in c)
    c2 = {n: t.clone() for n, t in want.items()}
    append(s, table=torch.full_like(table, -1), **c2)
    assert all(torch.equal(bits(c2[n]), bits(want[n])) for n in c2)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_padded_batch(dt):
    """Tokens behind the last sequence go nowhere."""
    s = setup(dt, 64, 2, [10, 60], [50, 5])
    want = {n: s[n].clone() for n in ("kc", "kr", "vp", "summ")}
    append(s, **want)
    got = {n: s[n].clone() for n in want}
    pad = torch.full((77, *s["k"].shape[1:]), float("nan"), dtype=dt, device="cuda")
    append(s, k=torch.cat([s["k"], pad]), v=torch.cat([s["v"], pad]), **got)
    assert all(torch.equal(bits(got[n]), bits(want[n])) for n in got)


def test_pages_far_apart():
    """The same pages at the end of a cache of over 4 GiB."""
    s = setup(torch.bfloat16, 64, 2, [10, 60], [150, 5])
    near = {n: s[n].clone() for n in ("kc", "kr", "vp", "summ")}
    append(s, **near)
    extra = 270000
    far = {}
    for n in near:
        far[n] = torch.empty(extra + s[n].shape[0], *s[n].shape[1:], dtype=torch.bfloat16, device="cuda")
        far[n][extra:] = s[n]
    append(s, table=s["table"] + extra, **far)
    assert all(torch.equal(bits(far[n][extra:]), bits(near[n])) for n in near)


def test_graph_replays():
    old, new = [50, 3], [90, 61]
    s = setup(torch.bfloat16, 64, 2, old, new)
    append(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        append(s)
    for seed in range(3):
        t = setup(torch.bfloat16, 64, 2, old, new, seed=10 + seed)
        for n in ("k", "v", "kc", "kr", "vp", "summ", "table"):
            s[n].copy_(t[n])
        t["gain"] = s["gain"]
        for n in ("probes", "proj"):
            t[n] = s[n]
        append(t)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(bits(s[n]), bits(t[n])) for n in ("kc", "kr", "vp", "summ"))


def test_refusals():
    s = setup(torch.float32, 64, 2, [3, 4], [2, 2])
    bad = [dict(k=s["k"][:1]), dict(v=s["v"].bfloat16()), dict(cu=s["cu"].long()), dict(cu=s["cu"][:-1]),
           dict(lens=s["lens"].long()), dict(lens=s["lens"][:1]), dict(table=s["table"].long()), dict(table=s["table"][0]),
           dict(kc=s["kc"][:-1]), dict(kr=s["kr"].bfloat16()), dict(vp=s["vp"][:, :1]), dict(kc=None),
           dict(probes=None), dict(summ=s["summ"][..., :32]), dict(gain=torch.ones(3).cuda()),
           dict(cos=s["cos"][:, :32]), dict(cu=s["cu"].cpu()), dict(v=s["v"].cpu())]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            append(s, **kw)
    append(s, k=s["k"][:0], v=s["v"][:0])


class Knobs:
    """A config, gains and a summarizer for PagedKVCache."""

    def __init__(self, dt=torch.bfloat16, batch=3, max_len=512, seed=0):
        torch.manual_seed(seed)
        self.cfg = hba_amd.HBAConfig(n_heads=4, n_kv=2, head_dim=64, window=100, sinks=4, k_blocks=2)
        self.qkn, self.summ = hba_amd.QKNorm(self.cfg).cuda(), hba_amd.SlotSummarizer(self.cfg).cuda()
        self.cos, self.sin = hba_amd.rope_tables(max_len, 64, 1e6, "cuda")
        self.dt, self.batch, self.max_len = dt, batch, max_len

    def cache(self, num_pages=None):
        return hba_amd.PagedKVCache(self.cfg, self.batch, self.max_len, self.dt, "cuda", num_pages)

    def kv(self, n):
        return [torch.randn(n, 2, 64).to(self.dt).cuda() for _ in range(2)]


def test_extend_is_appending():
    """A prompt in parts and single appends between them: the same caches and lengths as
    token by token, and the decode step goes on from either."""
    x = Knobs()
    a, b = x.cache(), x.cache()
    for counts in ([70, 0, 130], [1, 1, 1], [58, 65, 0], [0, 0, 0], [200, 3, 7]):
        k, v = x.kv(sum(counts))
        cu = a.extend(k, v, counts, x.qkn, x.summ, x.cos, x.sin)
        assert cu.tolist() == [sum(counts[:i]) for i in range(4)]
        at = cu.tolist()
        for i in range(max(counts)):
            # one by one, the sequences that have an i-th token
            for s in range(3):
                if i < counts[s]:
                    n = b.lens[s] + 1
                    for j, p in enumerate(b._ensure_pages(s, n)):
                        b.page_table[s, len(b._table[s]) - 1 + j] = p
                    ln = torch.tensor([n], dtype=torch.int32).cuda()
                    row = b.page_table[s:s + 1].contiguous()
                    ops.kv_append(k[at[s] + i][None], v[at[s] + i][None], x.qkn.k.gain, x.qkn.k.eps, x.cos, x.sin,
                                  row, ln, b.kc_pages, b.kr_pages, b.v_pages)
                    ops.summarize_filled(b.kc_pages, row, ln, x.summ.probes, x.summ.proj, b.summ_pages)
                    b.lens[s] = n
                    b.seq_lens[s] = n
        assert a.lens == b.lens and a.seq_lens.tolist() == a.lens
        for s in range(3):
            n = a.lens[s]
            pa, pb = a._table[s], b._table[s]
            assert a.page_table[s, :len(pa)].tolist() == pa
            for f in (lambda c, p: c.key_rows(p), lambda c, p: c.value_rows(p)):
                ra, rb = (f(c, torch.tensor(p, dtype=torch.long).cuda()).transpose(1, 2).reshape(-1, 2, 64)[:n]
                          for c, p in ((a, pa), (b, pb)))
                assert torch.equal(ra, rb)
            full = n // 64
            assert torch.equal(a.summ_pages[pa[:full]], b.summ_pages[pb[:full]])
    q = torch.randn(3, 4, 64).to(x.dt).cuda()
    oa, sa, _ = hba_amd.hba_decode_step(q, a, x.cfg, x.qkn, x.cos, x.sin)
    ob, sb, _ = hba_amd.hba_decode_step(q, b, x.cfg, x.qkn, x.cos, x.sin)
    assert torch.equal(sa, sb)
    # the caches' kr differ by up to 5 roundings (2^-8) a key; a logit by their sum at most
    assert float((oa - ob).abs().max()) <= 0.1


def test_extend_refusals():
    x = Knobs()
    c = x.cache(num_pages=5)
    k, v = x.kv(10)
    for counts in ([10, 0], [5, 5, 1], [11, -1, 0]):
        with pytest.raises(ValueError):
            c.extend(k, v, counts, x.qkn, x.summ, x.cos, x.sin)
    with pytest.raises(ValueError):
        c.extend(k.float(), v, [10, 0, 0], x.qkn, x.summ, x.cos, x.sin)
    with pytest.raises(ValueError):
        c.extend(k, v, [10, 0, 0], x.qkn, x.summ, x.cos[:9], x.sin[:9])
    k, v = x.kv(513)
    with pytest.raises(ValueError):
        c.extend(k, v, [513, 0, 0], x.qkn, x.summ, x.cos, x.sin)
    with pytest.raises(RuntimeError):
        c.extend(k[:500], v[:500], [500, 0, 0], x.qkn, x.summ, x.cos, x.sin)
    assert c.lens == [0, 0, 0] and c.seq_lens.tolist() == [0, 0, 0] and len(c._free) == 5
    c.extend(k[:300], v[:300], [300, 0, 0], x.qkn, x.summ, x.cos, x.sin)
    with pytest.raises(ValueError):
        c.share(0, 100, [1])
    with pytest.raises(ValueError):
        c.share(0, 320, [1])
    with pytest.raises(ValueError):
        c.share(0, 64, [0])
    with pytest.raises(ValueError):
        c.share(0, 64, [1, 1])
    c.share(0, 128, [1, 2])
    with pytest.raises(ValueError):
        c.share(0, 128, [1])
    with pytest.raises(ValueError):
        c.load(1, k[:64], k[:64], v[:64], x.summ)
    assert c.lens == [300, 128, 128] and c.seq_lens.tolist() == [300, 128, 128]
    assert c.page_table[1, :2].tolist() == c._table[0][:2]
    assert value_offsets(64).numel() == 64 * 64
