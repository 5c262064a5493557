"""Attention over the paged cache (ops.paged_attn, hba_amd.cache_attention) against
64-bit results: one token a sequence, ragged parts of prompts, windows with sinks, and
shared first pages; what lies behind the lengths, and what it refuses."""
import pytest
import torch

import hba_amd
from attn64 import assert_within, attend, norm_rotate, unit, visible
from hba_amd import ops
from hba_amd.decode import key_offsets, value_offsets

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


def setup(dt, d, Hq, Hkv, lens, new=None, shared=0, maxp=None, seed=0, gain=True):
    """Random rows in permuted pages; everything behind a sequence's length is NaN."""
    g = torch.Generator().manual_seed(seed)
    Bd, T = len(lens), len(lens) if new is None else sum(new)
    maxp = maxp or max(1, max((n + 63) // 64 for n in lens), shared // 64)
    P = Bd * maxp + 2
    table = torch.randperm(P, generator=g)[:Bd * maxp].view(Bd, maxp).int()
    table[:, :shared // 64] = table[0, :shared // 64]
    ko, vo = key_offsets(d), value_offsets(d)
    rows, kp, vp = [], torch.full((P, Hkv, 64 * d), float("nan")), torch.full((P, Hkv, 64 * d), float("nan"))
    keys, vals = (torch.randn(P, Hkv, 64, d, generator=g).to(dt) for _ in range(2))
    keys = (keys.float() * d ** 0.25).to(dt)
    for b, n in enumerate(lens):
        for p in range((min(n, 64 * maxp) + 63) // 64):
            at, m = int(table[b, p]), min(64, n - 64 * p)
            if p < shared // 64:
                m = 64          # another sequence may be longer
            for h in range(Hkv):
                kp[at, h][ko[:m]] = keys[at, h, :m].float()
                vp[at, h][vo[:m]] = vals[at, h, :m].float()
        pages = table[b].long()
        rows.append((keys[pages].transpose(0, 1).reshape(Hkv, -1, d), vals[pages].transpose(0, 1).reshape(Hkv, -1, d)))
    cos, sin = hba_amd.rope_tables(maxp * 64, d, 1e4, "cpu")
    return dict(q=torch.randn(T, Hq, d, generator=g).to(dt), gain=1.2 + 0.1 * torch.randn(Hq, generator=g) if gain else None,
                kr=kp.to(dt), vp=vp.to(dt), table=table, lens=torch.tensor(lens, dtype=torch.int32), cos=cos, sin=sin,
                scales=(0.5 + torch.rand(Bd, generator=g)) / d, rows=rows, new=new, shared=shared,
                cu=None if new is None else torch.tensor([0] + new).cumsum(0).int(), max_len=max(1, max(lens)))


def call(s, W=0, S=0, **kw):
    a = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in {**s, **kw}.items()}
    return ops.paged_attn(a["q"], a["gain"], EPS, a["kr"], a["vp"], a["table"], a["lens"], a["cos"], a["sin"],
                          a["scales"], a["max_len"], W, S, a["cu"], a["shared"])


def expect(s, W=0, S=0):
    dt, (T, Hq, d) = s["q"].dtype, s["q"].shape
    Hkv = s["kr"].shape[1]
    G, u = Hq // Hkv, unit(dt)
    out, bound = torch.zeros(T, Hq, d, dtype=torch.float64), torch.zeros(T, Hq, d, dtype=torch.float64)
    t = 0
    for b, n in enumerate(s["lens"].tolist()):
        n = min(n, s["max_len"], 64 * s["table"].shape[1])
        c = 1 if s["new"] is None else s["new"][b]
        pos = torch.arange(n - c, n)
        at = pos.clamp(0, s["cos"].shape[0] - 1) if s["cos"] is not None else None
        cs, sn = (None, None) if at is None else (s["cos"][at], s["sin"][at])
        # two bf16 parts of a query leave u of the second, u of the first at most: u * u
        _, q, qe = norm_rotate(s["q"][t:t + c], s["gain"], EPS, cs, sn, u * u if dt == torch.bfloat16 else 0.0)
        see = visible(pos, torch.arange(max(n, 0)), W or None, S)
        for h in range(Hkv):
            if n > 0 and c > 0:
                k, v = (r[h, :n] for r in s["rows"][b])
                out[t:t + c, h * G:h * G + G], bound[t:t + c, h * G:h * G + G] = attend(
                    q[:, h * G:h * G + G], k, v, see, float(s["scales"][b]), u, qerr=qe[:, h * G:h * G + G])
        t += c
    return out, bound


def check(s, W=0, S=0, **kw):
    got = call(s, W, S, **kw)
    assert got.dtype == s["q"].dtype and got.shape == s["q"].shape
    assert_within(got, *expect({**s, **kw}, W, S), "out")


LENS = [[1], [0, 1, 63], [64, 65, 128, 200], [700, 3, 0, 129], [1500]]
WINDOWS = [(0, 0), (1, 0), (1, 3), (64, 0), (70, 4), (63, 65), (500, 130), (5000, 2)]


@pytest.mark.parametrize("dt,d", [("f32", 64), ("f32", 128), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("W,S", WINDOWS)
@pytest.mark.parametrize("lens", LENS)
def test_decode(lens, W, S, dt, d):
    check(setup(DT[dt], d, 4, 2, lens, seed=len(lens)), W, S)


@pytest.mark.parametrize("dt,d", [("f32", 64), ("f32", 128), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("W,S", [(0, 0), (2100, 0), (2200, 70)])
@pytest.mark.parametrize("lens,Hq,Hkv", [([2049], 2, 1), ([0, 4000, 1, 63, 2600], 6, 2), ([0, 0, 2200, 0], 17, 1),
                                         ([2100] * 9, 3, 3)])
def test_long_sequences_in_even_shares(lens, Hq, Hkv, W, S, dt, d):
    """More than 32 pages: all sequences' pages are cut evenly, shares begin and end inside sequences."""
    check(setup(DT[dt], d, Hq, Hkv, lens, seed=len(lens)), W, S)


@pytest.mark.parametrize("bd", [300, 1100])
def test_many_sequences_under_a_long_bound(bd):
    """More sequences than the scan has threads for a run each; the bound is far above every length."""
    s = setup(torch.bfloat16, 64, 2, 1, [(37 * i) % 130 for i in range(bd)], seed=3)
    s["cos"], s["sin"] = hba_amd.rope_tables(4000, 64, 1e4, "cpu")
    check({**s, "table": torch.cat([s["table"], torch.zeros(bd, 60, dtype=torch.int32)], 1), "max_len": 4000})


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (7, 1), (14, 2), (16, 1), (17, 1), (40, 2), (6, 6)])
def test_groups(Hq, Hkv, dt):
    check(setup(DT[dt], 64, Hq, Hkv, [300, 65, 1], seed=Hq))
    check(setup(DT[dt], 64, Hq, Hkv, [300, 65, 1], [40, 65, 1], seed=Hq), 50, 2)
    check(setup(DT[dt], 64, Hq, Hkv, [300, 165, 129], shared=128, seed=Hq))


@pytest.mark.parametrize("dt,d", [("f32", 64), ("f32", 128), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("W,S", WINDOWS)
@pytest.mark.parametrize("lens,new", [([1], [1]), ([5, 70, 0, 300], [5, 3, 0, 299]), ([64, 640], [64, 65]),
                                      ([129, 900, 66], [0, 130, 1]), ([3, 10], [5, 12])])
def test_parts_of_prompts(lens, new, W, S, dt, d):
    """The last case: more tokens than the cache holds, the first ones see nothing."""
    check(setup(DT[dt], d, 6, 2, lens, new, seed=sum(new)), W, S)


@pytest.mark.parametrize("dt,d", [("f32", 64), ("f32", 128), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("shared,lens", [(64, [65, 64, 100]), (128, [129, 700, 130, 300]), (640, [641] * 20),
                                         (1024, [1100, 1024, 1500]), (128, [0, 5, 128, 200])])
def test_shared_prefix(shared, lens, dt, d):
    """The last case: sequences that end within the shared pages."""
    check(setup(DT[dt], d, 4, 2, lens, shared=shared, seed=shared))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_shared_prefix_with_parts(dt):
    check(setup(DT[dt], 64, 4, 2, [200, 300, 128, 129], [10, 150, 0, 129], shared=128))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shared,lens,new", [(0, [40, 20], [30, 1]), (0, [900, 700], [60, 65]), (0, [5, 0], [0, 0]),
                                             (64, [200, 130], [9, 66])])
def test_padded_batch(shared, lens, new, dt):
    """Tokens behind the last sequence give 0, whatever they hold."""
    s = setup(DT[dt], 64, 6, 2, lens, new, shared=shared, seed=3)
    T = sum(new)
    s["q"] = torch.cat([s["q"], torch.full((300, 6, 64), float("nan"), dtype=DT[dt])])
    torch.full((T + 300, 6, 64), float("nan"), dtype=DT[dt], device="cuda")   # the output's memory, perhaps
    got = call(s)
    assert not got[T:].any() and got.shape[0] == T + 300
    if T:
        want, bound = expect({**s, "q": s["q"][:T]})
        assert_within(got[:T], want, bound, "out")


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("new", [None, [3, 60]])
def test_no_norm_no_rotation_and_sharp_logits(new, dt):
    s = setup(DT[dt], 64, 4, 2, [200, 90], new, gain=False)
    check(s, cos=None, sin=None)
    check({**s, "scales": s["scales"] * 40}, cos=None, sin=None)
    check({**s, "scales": s["scales"] * 0})


def test_max_len_and_long_tables():
    s = setup(torch.bfloat16, 64, 4, 2, [300, 64], maxp=9)
    check({**s, "max_len": 576})
    check({**s, "max_len": 200}, 70, 1)         # a longer length is read as max_len
    s = setup(torch.bfloat16, 64, 4, 2, [300, 64])
    s["lens"] = torch.tensor([10 ** 6, -5], dtype=torch.int32)      # past the page table, below 0
    s["max_len"] = 10 ** 6
    n = 64 * s["table"].shape[1]
    cos, sin = hba_amd.rope_tables(n, 64, 1e4, "cpu")
    s.update(cos=cos, sin=sin)
    kp, vp = s["kr"].clone(), s["vp"].clone()
    kp[kp != kp] = 0.5
    vp[vp != vp] = 0.5
    out = call({**s, "kr": kp, "vp": vp})
    assert bool(torch.isfinite(out.float()).all()) and bool((out[1] == 0).all())
    bad = s["table"].clone()
    bad[0, 1], bad[0, 2] = 10 ** 8, -7          # clamped into the cache
    assert bool(torch.isfinite(call({**s, "kr": kp, "vp": vp, "table": bad}).float()).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_masked_values_have_no_effect(dt):
    """NaN in a key and value that only some tokens of a part see."""
    W, S, n = 40, 2, 200
    s = setup(DT[dt], 64, 4, 2, [n], [100])
    clean = call(s, W, S).float().cpu()
    ko, vo = key_offsets(64), value_offsets(64)
    for which, off in (("kr", ko), ("vp", vo)):
        for bad in (float("nan"), float("inf")):
            d = {**s, which: s[which].clone()}
            d[which][int(s["table"][0, 130 // 64])][:, off[130 % 64]] = bad
            got = call(d, W, S).float().cpu()
            pos = torch.arange(100, 200)
            sees = (pos >= 130) & (pos < 130 + W)
            assert bool(torch.isfinite(got[~sees]).all())
            # computed again key by key: the same up to the order of the sums and P's rounding
            assert float((got - clean)[~sees].abs().max()) <= (2e-2 if dt == "bf16" else 1e-5)
            if which == "vp":
                assert not bool(torch.isfinite(got[sees]).any())


@pytest.mark.parametrize("new", [None, [70, 3]])
def test_pages_far_apart(new):
    """The same pages at the end of a cache of over 4 GiB."""
    s = setup(torch.bfloat16, 64, 4, 2, [2300, 190], new)
    near = call(s)
    P, extra = s["kr"].shape[0], 270000
    far = {**s, "table": s["table"] + extra}
    for n in ("kr", "vp"):
        far[n] = torch.empty(P + extra, *s[n].shape[1:], dtype=torch.bfloat16, device="cuda")
        far[n][extra:] = s[n].cuda()
    assert far["kr"].numel() * 2 > 2 ** 32
    assert torch.equal(call(far), near)


def test_strides_streams_and_graphs():
    s = setup(torch.bfloat16, 64, 4, 2, [300, 65, 700, 1])
    want = call(s)
    q = torch.randn(4, 3, 4, 64).to(torch.bfloat16)
    q[:, 1] = s["q"]
    assert torch.equal(call({**s, "q": q.cuda()[:, 1]}), want)
    assert torch.equal(call({**s, "q": torch.nn.functional.pad(s["q"], (1, 2)).cuda()[..., 1:-2]}), want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = call(s)
    stream.synchronize()
    assert torch.equal(got, want)
    a = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in s.items()}
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = call(a)
    with torch.cuda.graph(g2):
        o2 = call(a, 70, 4)
    for seed in range(3):
        a["q"].copy_(torch.randn(4, 4, 64, generator=torch.Generator().manual_seed(seed)))
        a["lens"].copy_(torch.tensor([300 - seed, 65, 700 - 10 * seed, min(seed, 1)]))   # what the pages hold
        g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        x, y = o1.clone(), o2.clone()
        assert torch.equal(x, call(a)) and torch.equal(y, call(a, 70, 4))


def test_custom_op():
    s = setup(torch.bfloat16, 64, 4, 2, [300, 65])
    a = {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in s.items()}
    got = torch.ops.hba.paged_attn(a["q"], a["gain"], EPS, a["kr"], a["vp"], a["table"], a["lens"], a["cos"], a["sin"],
                                   a["scales"], a["max_len"], 70, 4)
    assert torch.equal(got, call(s, 70, 4))


def test_refusals():
    s = setup(torch.float32, 64, 4, 2, [100, 65])
    bad = [(0, 1, {}), (-1, 0, {}), (4, -1, {}), (5, 0, dict(shared=64)), (0, 0, dict(shared=63)),
           (0, 0, dict(shared=64 * 100)), (0, 0, dict(shared=-64)), (0, 0, dict(q=s["q"][:1])),
           (0, 0, dict(q=s["q"][:, :3])), (0, 0, dict(q=s["q"].bfloat16())), (0, 0, dict(kr=s["kr"][:-1])),
           (0, 0, dict(vp=s["vp"].bfloat16())), (0, 0, dict(table=s["table"].long())),
           (0, 0, dict(lens=s["lens"][:1])), (0, 0, dict(cu=torch.tensor([0, 1], dtype=torch.int32))),
           (0, 0, dict(scales=s["scales"][:1])), (0, 0, dict(gain=s["gain"][:1])), (0, 0, dict(max_len=0)),
           (0, 0, dict(cos=None)), (0, 0, dict(cos=s["cos"][:10], sin=s["sin"][:10])),
           (0, 0, dict(q=s["q"][0]))]
    for W, S, kw in bad:
        with pytest.raises((ValueError, TypeError)):
            call(s, W, S, **kw)
    assert call(s, q=s["q"][:0], table=s["table"][:0], lens=s["lens"][:0], scales=s["scales"][:0]).shape == (0, 4, 64)


class TestTogether:
    """Prompts in parts, a shared beginning, decode steps: the cache against
    sliding_attention on the same rotated rows."""

    def rotated(self, x, pos, gain, eps, cos, sin):
        return norm_rotate(x.cpu(), gain.detach().cpu(), eps, cos.cpu()[pos], sin.cpu()[pos], 0.0)[1]

    @pytest.mark.parametrize("window,sinks", [(None, 0), (70, 4)])
    def test_prompt_then_decode(self, window, sinks):
        torch.manual_seed(0)
        cfg = hba_amd.HBAConfig(n_heads=4, n_kv=2, head_dim=64, temp_c=0.0)
        qkn, summ = hba_amd.QKNorm(cfg).cuda(), hba_amd.SlotSummarizer(cfg).cuda()
        n, dt = 333, torch.float32
        cos, sin = hba_amd.rope_tables(512, 64, 1e4, "cuda")
        cache = hba_amd.PagedKVCache(cfg, 2, 512, dt, "cuda")
        q, k, v = (torch.randn(2, n, h, 64, device="cuda") for h in (4, 2, 2))
        got = torch.empty(2, n, 4, 64, device="cuda")
        at = [0, 0]
        for counts in ([100, 64], [1, 1], [120, 3], [50, 200], [62, 65]):
            part = lambda x: torch.cat([x[s, at[s]:at[s] + counts[s]] for s in range(2)])  # noqa: E731
            if counts == [1, 1]:
                cache.append(part(k), part(v), qkn, summ, cos, sin)
                cu = None
            else:
                cu = cache.extend(part(k), part(v), counts, qkn, summ, cos, sin)
            out = hba_amd.cache_attention(part(q), cache, cfg, qkn, cos, sin, window, sinks, cu)
            for s in range(2):
                got[s, at[s]:at[s] + counts[s]] = out[sum(counts[:s]):][:counts[s]]
                at[s] += counts[s]
        assert at == [n, n]
        pos = torch.arange(n)
        qr, kr = (torch.stack([self.rotated(x[s], pos, m.gain, m.eps, cos, sin) for s in range(2)]).float().cuda()
                  for x, m in ((q, qkn.q), (k, qkn.k)))
        want = hba_amd.sliding_attention(qr, kr, v, window or n, sinks, scale=1 / 64)
        # both in fp32: the sums' orders and a rounding of q and k, 64 elements of about 1
        assert float((got - want).abs().max()) <= 64 * 2.0 ** -20

    def test_shared_beginning(self):
        """Sequences that begin with another's pages, and a cache that holds copies."""
        torch.manual_seed(1)
        cfg = hba_amd.HBAConfig(n_heads=4, n_kv=2, head_dim=64)
        qkn, summ = hba_amd.QKNorm(cfg).cuda(), hba_amd.SlotSummarizer(cfg).cuda()
        dt = torch.bfloat16
        cos, sin = hba_amd.rope_tables(512, 64, 1e4, "cuda")
        a, b = (hba_amd.PagedKVCache(cfg, 3, 512, dt, "cuda") for _ in range(2))
        k, v = (torch.randn(200, 2, 64, device="cuda").to(dt) for _ in range(2))
        a.extend(k, v, [200, 0, 0], qkn, summ, cos, sin)
        a.share(0, 192, [1, 2])
        b.extend(torch.cat((k, k[:192], k[:192])), torch.cat((v, v[:192], v[:192])), [200, 192, 192], qkn, summ, cos,
                 sin)
        assert len(a._free) == len(b._free) + 6
        k, v = (torch.randn(150, 2, 64, device="cuda").to(dt) for _ in range(2))
        for c in (a, b):
            cu = c.extend(k, v, [20, 0, 130], qkn, summ, cos, sin)
        q = torch.randn(150, 4, 64, device="cuda").to(dt)
        x = hba_amd.cache_attention(q, a, cfg, qkn, cos, sin, cu=cu, shared=192)
        y = hba_amd.cache_attention(q, b, cfg, qkn, cos, sin, cu=cu)
        assert float((x.float() - y.float()).abs().max()) <= 2e-2
        k, v = (torch.randn(3, 2, 64, device="cuda").to(dt) for _ in range(2))
        for c in (a, b):
            c.append(k, v, qkn, summ, cos, sin)
        q = torch.randn(3, 4, 64, device="cuda").to(dt)
        x = hba_amd.cache_attention(q, a, cfg, qkn, cos, sin, shared=192)
        y = hba_amd.cache_attention(q, b, cfg, qkn, cos, sin)
        assert float((x.float() - y.float()).abs().max()) <= 2e-2
        ox, sx, _ = hba_amd.hba_decode_step(q, a, cfg, qkn, cos, sin)
        oy, sy, _ = hba_amd.hba_decode_step(q, b, cfg, qkn, cos, sin)
        assert torch.equal(ox, oy)
        with pytest.raises(ValueError):
            hba_amd.cache_attention(q, b, cfg, qkn, cos, sin, shared=192)
        with pytest.raises(ValueError):
            hba_amd.cache_attention(q, a, cfg, qkn, cos, sin, shared=256)
        with pytest.raises(ValueError):
            hba_amd.cache_attention(q, a, cfg, qkn, cos, sin, window=0)
        with pytest.raises(ValueError):
            hba_amd.cache_attention(q, a, cfg, qkn, cos, sin, max_len=100)
