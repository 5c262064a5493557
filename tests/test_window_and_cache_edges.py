"""Calls of the window and cache operators at the edges of what their documentation
allows: state after an error, lengths of any type, launches of any size, pages with
anything behind their sequences, and every form that the gradients' kernels take."""
import ctypes

import pytest
import torch

import hba_amd
import test_gpu_paged_attn as paged
import test_gpu_swa as swa
import test_window_and_cache_host as host
import test_gpu_append_ragged as ragged
from attn64 import E, assert_within, attend, norm_rotate, sliding, unit, visible
from hba_amd.decode import key_offsets, value_offsets
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


def test_launches_of_too_many_threads_are_refused():
    """A launch has fewer than 2^32 threads; what needs more is refused before any of its work."""
    s3 = (ctypes.c_int64 * 3)(64, 64, 64)
    assert host.swa(B=1 << 24, n=1, Hq=1, Hkv=1, st=s3, kst=s3) == -2
    assert host.paged(T=1 << 23, Bd=1 << 23, Hq=1, Hkv=1, max_len=64, maxp=1) == -2
    assert host.paged(T=1 << 27, Bd=1, Hq=8, Hkv=8, max_len=128, shared=1, maxp=2, cu=host.FAKE, nbytes=1 << 62) == -2
    assert host.append(T=1 << 24, Bd=1 << 24, Hkv=1) == -2


@pytest.mark.parametrize("B,n,Hq,Hkv,d,W,S,parts", [
    (8, 8192, 28, 4, 128, 1024, 8, 7 * 32),         # a tile of sinks in 7 parts, the others whole
    (4, 32768, 56, 8, 128, 1024, 8, 28 * 32),
    (1, 8192, 28, 4, 128, 1024, 8, None),           # every tile in parts
    (600, 130, 4, 2, 64, 40, 3, 0)])
def test_gradients_workspace_has_room_for_what_is_written(B, n, Hq, Hkv, d, W, S, parts):
    """Each row's <dout, out>, a mark a wave, and the sums of those key tiles that are cut."""
    st, need = host.size(host._lib.lib().hba_swa_bwd_workspace_bytes, 1, B, n, Hq, Hkv, d, W, S)
    rows = 4 * B * Hq * n
    assert st == 0 and need >= rows
    tiles = B * Hkv * -(-n // 128)
    if parts is not None:
        marks = 16 * (tiles + parts)
        assert parts * 128 * 2 * d * 4 <= need - rows <= marks + 512 + parts * 128 * 2 * d * 4
    else:
        assert need - rows >= 2 * tiles * 128 * 2 * d * 4


@pytest.mark.gpu
@pytest.mark.parametrize("dt,d,Hkv", [("bf16", 64, 16), ("f32", 128, 8)])
def test_gradients_of_a_million_heads(dt, d, Hkv):
    """More key tiles than one launch joins; the keys that a NaN of another token's query
    spoils, which only the join computes, are those of the first and the last launch."""
    B, n = 65536, 3
    q, k, v, do = swa.make(swa.DT[dt], 4, n, Hkv, Hkv, d)
    x = [torch.empty(B, n, Hkv, d, dtype=swa.DT[dt], device="cuda") for _ in range(4)]
    at = torch.tensor([0, 1, B // 2, B - 1])
    for t, rows in zip(x, (q, k, v, do)):
        t[:] = rows[1].cuda()
        t[at] = rows.cuda()
    clean = [t.clone() for t in (q, k, v, do)]
    for b in range(4):
        x[0][at[b], 0] = float("nan")
    got = swa.run(*x[:3], 1, 0, dout=x[3])
    want, bound = sliding(*clean[:3], 1, 0, d ** -0.5, None, unit(swa.DT[dt]), clean[3])
    for name, a, w, c in zip(("out", "dq", "dk", "dv"), got, want, bound):
        assert_within(a[at][:, 1:].cpu(), w[:, 1:], c[:, 1:], name)
        assert torch.equal(a[2:100], a[2:3].expand(98, -1, -1, -1)), name


@pytest.mark.gpu
def test_lengths_of_every_type():
    """Lengths are taken as the numbers they are, past 32 bits too."""
    q, k, v, do = swa.make(torch.bfloat16, 4, 200, 4, 2, 64, seed=3)
    x = [t.cuda().requires_grad_() for t in (q, k, v)]

    def run(lens):
        o = hba_amd.sliding_attention(*x, 70, 5, lens=lens)
        return (o.detach(), *torch.autograd.grad(o, x, do.cuda()))

    want = run(torch.tensor([200, 0, 130, 200], dtype=torch.int32).cuda())
    big = torch.tensor([2 ** 32 + 7, -2 ** 32 + 50, 130, 2 ** 31])
    for lens in (big.cuda(), big):
        assert all(torch.equal(a, b) for a, b in zip(run(lens), want))
    for dt in (torch.uint8, torch.int16, torch.int64):
        lens = torch.tensor([200, 0, 130, 200], dtype=dt).cuda()
        assert all(torch.equal(a, b) for a, b in zip(run(lens), want))
    with pytest.raises(ValueError):
        run(torch.ones(4, dtype=torch.complex64).cuda())


@pytest.mark.gpu
def test_no_query_heads():
    """Keys without a query have gradients of 0."""
    q, k = torch.empty(2, 50, 0, 64, device="cuda"), torch.randn(2, 50, 2, 64, device="cuda").requires_grad_()
    torch.full((4, 50, 2, 64), float("nan"), device="cuda")       # the gradients' memory, perhaps
    out = hba_amd.sliding_attention(q, k, k * 2, 5)
    assert out.shape == q.shape
    out.sum().backward()
    assert not k.grad.any()


# Batches whose key tiles are cut into (parts of a tile with sinks, parts of the others):
# every form that swa_dkv and swa_join take beside the one of small grids, several and several
CUTS = [("f32", 64, "one, one", 600, 130, 4, 2, 40, 3), ("f32", 128, "one, one", 600, 130, 4, 2, 40, 3),
        ("bf16", 64, "one, one", 600, 130, 4, 2, 40, 3), ("bf16", 128, "one, one", 600, 130, 4, 2, 40, 3),
        ("f32", 64, "several, one", 150, 200, 2, 2, 1, 4), ("f32", 128, "several, one", 150, 200, 2, 2, 1, 4),
        ("bf16", 64, "several, one", 150, 200, 2, 2, 1, 4), ("bf16", 128, "several, one", 150, 200, 2, 2, 1, 4),
        ("f32", 64, "no sinks, one", 150, 200, 2, 2, 1, 0), ("bf16", 128, "no sinks, one", 150, 200, 2, 2, 1, 0),
        ("f32", 64, "one, several", 105, 2131, 2, 2, 1, 2000), ("bf16", 128, "one, several", 63, 2125, 6, 3, 2125, 2000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt,d,parts,B,n,Hq,Hkv,W,S", CUTS)
def test_gradients_of_every_cut(dt, d, parts, B, n, Hq, Hkv, W, S):
    """Whole, short and empty sequences against 64 bits; in the last one two queries are
    NaN, which spoils what they see and nothing else."""
    dtype = swa.DT[dt]
    g = torch.Generator(device="cuda").manual_seed(n)
    q, k, v, do = (torch.randn(B, n, h, d, generator=g, device="cuda").to(dtype) for h in (Hq, Hkv, Hkv, Hq))
    lens = torch.tensor([(n, 0, 7, n // 2, n - 1, 129)[b % 6] for b in range(B)])
    lens[-1] = n
    bad = [5, 100]
    dirty = q.clone()
    dirty[-1, bad] = float("nan")
    leaves = [t.requires_grad_() for t in (dirty, k.clone(), v.clone())]
    out = hba_amd.sliding_attention(*leaves, W, S, lens=lens)
    got = (out.detach(), *torch.autograd.grad(out, leaves, do))
    i = torch.arange(n, device="cuda")
    for b in (0, 1, 2, 3, B - 1):
        m = int(lens[b])
        assert not any(t[b, m:].any() for t in got)
        if not m:
            continue
        see = visible(i[:m], i[:m], W, S)
        rows, keys = torch.ones(m, dtype=torch.bool, device="cuda"), torch.ones(m, dtype=torch.bool, device="cuda")
        if b == B - 1:
            rows[bad] = False
            keys = ~see[bad].any(0)
        G = Hq // Hkv
        for h in range(Hkv):
            hs = slice(h * G, h * G + G)
            with torch.device("cuda"):
                want, bound = attend(q[b, :m, hs], k[b, :m, h], v[b, :m, h], see, d ** -0.5, unit(dtype), do[b, :m, hs])
            for name, x, w, c in zip(("out", "dq", "dk", "dv"), got, want, bound):
                x, keep = (x[b, :m, hs], rows) if name in ("out", "dq") else (x[b, :m, h], keys)
                assert_within(x[keep], w[keep].cpu(), c[keep].cpu(), f"{name} of {b}, {h}")


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("B,n,Hq,Hkv", [(1, 200, 2, 1), (2, 900, 14, 2), (8, 700, 14, 2)])
def test_log_sum_exps(B, n, Hq, Hkv, dt, d):
    """Of the probabilities, not of their roundings, in every form of the forward: off by
    the largest error of a logit (d + 4 roundings of its products), the roundings of the
    sum and the logarithm, and one of the result."""
    q, k, v, _ = swa.make(swa.DT[dt], B, n, Hq, Hkv, d, seed=n)
    _, lse = hba_amd.ops.swa_fwd(q.cuda(), k.cuda(), v.cuda(), None, 300, 2, d ** -0.5)
    x, K = q[-1].double().transpose(0, 1), k[-1].double().repeat_interleave(Hq // Hkv, 1).transpose(0, 1)
    i = torch.arange(n)
    see = visible(i, i, 300, 2)
    c = d ** -0.5 / torch.log(torch.tensor(2.0, dtype=torch.float64))
    logits = (x @ K.transpose(1, 2) * c).masked_fill(~see, float("-inf"))
    want = torch.logsumexp(logits / c * d ** -0.5, -1) * c / d ** -0.5
    size = (x.abs() @ K.abs().transpose(1, 2) * c).masked_fill(~see, 0.0).amax(-1)
    bound = E * ((d + 4) * size + 1.4427 * n + 8 + 4 * want.abs())
    assert_within(lse[-1].cpu(), want, bound, "lse")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("which", range(4))
def test_masked_places_at_head_dim_128(which, bad, dt):
    """A non-finite query, key, value or cotangent spoils only what sees it."""
    W, S, n, at, d = 40, 3, 200, 100, 128
    x = swa.make(swa.DT[dt], 1, n, 4, 2, d, seed=7)
    want, bound = sliding(*x[:3], W, S, d ** -0.5, None, unit(swa.DT[dt]), x[3])
    dirty = [t.clone() for t in x]
    dirty[which][:, at] = bad
    i = torch.arange(n)
    see = visible(i, i, W, S)
    rows = see[:, at] if which in (1, 2) else i == at
    keys = see[rows].any(0)
    got = swa.run(*dirty[:3], W, S, dout=dirty[3])
    for name, a, w, c in zip(("out", "dq", "dk", "dv"), got, want, bound):
        keep = ~(rows if name in ("out", "dq") else keys)
        assert_within(a.detach().cpu()[:, keep], w[:, keep], c[:, keep], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("at", [5, 300, 590])
def test_few_rows_spoiled_at_head_dim_128(at, bad, dt):
    q, k, v, _ = swa.make(swa.DT[dt], 1, 600, 2, 1, 128, seed=at)
    want, bound = sliding(q, k, v, 300, 2, 128 ** -0.5, None, unit(q.dtype))
    k[0, at], v[0, at] = bad, bad
    got = swa.run(q, k, v, 300, 2).cpu()
    i = torch.arange(600)
    sees = (i >= at) & (i < at + 300)
    assert not got[0, sees].isfinite().any()
    assert_within(got[:, ~sees], want[:, ~sees], bound[:, ~sees], "out")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("name", ["kr", "vp"])
def test_masked_keys_of_a_cache_at_head_dim_128(name, bad, dt):
    W, S, n, at = 40, 2, 200, 130
    s = paged.setup(swa.DT[dt], 128, 4, 2, [n], [100])
    want, bound = paged.expect(s, W, S)
    off = (key_offsets if name == "kr" else value_offsets)(128)
    s[name][int(s["table"][0, at // 64])][:, off[at % 64]] = bad
    got = paged.call(s, W, S).cpu()
    pos = torch.arange(100, 200)
    sees = (pos >= at) & (pos < at + W)
    assert_within(got[~sees], want[~sees], bound[~sees], "out")
    if name == "vp":
        assert not got[sees].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt,d", [("f32", 64), ("f32", 128), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("W,S", [(0, 0), (70, 4)])
@pytest.mark.parametrize("lens,new,shared", [([1], [1], 0), ([40, 70, 129, 350], [40, 3, 128, 1], 0),
                                             ([65, 96, 31, 959], [1, 33, 31, 300], 0), ([135, 200], [7, 20], 128)])
def test_what_lies_behind_a_sequence_changes_no_bit(lens, new, shared, W, S, dt, d):
    """Parts of prompts: the rest of a last page may be anything, and no row takes
    another way for it."""
    if shared and W:
        W, S = 0, 0
    s = paged.setup(swa.DT[dt], d, 6, 2, lens, new, shared=shared, seed=len(lens))
    want = paged.call({**s, "kr": s["kr"].nan_to_num(), "vp": s["vp"].nan_to_num()}, W, S)
    assert s["vp"].isnan().any()
    for fill in (float("nan"), float("inf"), torch.finfo(swa.DT[dt]).max):
        kr, vp = (torch.where(s[n].isnan(), fill, s[n]) for n in ("kr", "vp"))
        assert torch.equal(paged.call({**s, "kr": kr, "vp": vp}, W, S), want), fill


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_how_far_extend_and_append_are_apart(dt):
    """The rotated keys of both ways into the cache, and what a decode makes of the
    difference.  In bf16 append rounds the key, the table, both products and their sum (4
    roundings of the products' magnitudes, and what they make of one another), extend the
    sum alone; in fp32 both do the same.  A logit moves by the keys' differences times
    |q|, its probability by at most twice that relative to it."""
    x = ragged.Knobs(dt, batch=1)
    a, b = x.cache(), x.cache()
    n, d = 200, 64
    k, v = x.kv(n)
    a.extend(k, v, [n], x.qkn, x.summ, x.cos, x.sin)
    for i in range(n):
        b.append(k[i:i + 1], v[i:i + 1], x.qkn, x.summ, x.cos, x.sin)
    ra, rb = (c.key_rows(torch.tensor(c._table[0]).cuda(), rotated=True).transpose(1, 2).reshape(-1, 2, d)[:n]
              .double().cpu() for c in (a, b))
    gain, eps = x.qkn.k.gain.detach().cpu(), x.qkn.k.eps
    cos, sin = x.cos.cpu()[:n], x.sin.cpu()[:n]
    y, want, _ = norm_rotate(k.cpu(), gain, eps, cos, sin, 0.0)
    other = torch.cat((y[..., d // 2:], y[..., :d // 2]), -1)
    size = y.abs() * cos.double()[:, None].abs() + other.abs() * sin.double()[:, None].abs()
    u = unit(dt)
    one = (d / 2 + 12) * E * size
    ea, eb = (one + u * size, one + (4.1 * u if dt == torch.bfloat16 else u) * size)
    assert_within(ra, want, ea, "extend's kr")
    assert_within(rb, want, eb, "append's kr")
    q = torch.randn(1, 4, d).to(dt).cuda()
    oa, ob = (hba_amd.cache_attention(q, c, x.cfg, x.qkn, x.cos, x.sin).detach().cpu() for c in (a, b))
    _, qr, qe = norm_rotate(q.cpu(), x.qkn.q.gain.detach().cpu(), x.qkn.q.eps, cos[-1:], sin[-1:],
                            u * u if dt == torch.bfloat16 else 0.0)
    scale = float(a.scales()[0])
    see = torch.ones(1, n, dtype=torch.bool)
    for h in range(2):
        hs, vals = slice(2 * h, 2 * h + 2), v[:, h].cpu()
        move = 2 * scale * (qr[:, hs].abs() @ (ea + eb)[:, h].T).amax(-1, keepdim=True)
        middle, bound = attend(qr[:, hs], want[:, h], vals, see, scale, u, qerr=qe[:, hs])
        weight, _ = attend(qr[:, hs], want[:, h], vals.abs(), see, scale, u)
        assert_within(oa[:, hs], middle, bound + move * weight, "over extend's keys")
        assert_within(ob[:, hs], middle, bound + move * weight, "over append's keys")
