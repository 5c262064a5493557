"""Calls at the ends of what the paged caches' operators take, against 64-bit results."""
import pytest
import torch

import hba_amd
import mx64
import test_gpu_mx_cache as mxc
import test_gpu_paged_attn as rows
from hba_amd import ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dt,d", [("f32", 64), ("bf16", 128)])
@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("new", [None, [40, 3]])
def test_windows_and_sinks_past_every_length(new, bits, dt, d):
    """They mean every key, however large the number."""
    lens, heads = [2200, 70], (6, 2)
    m = rows if bits == 16 else mxc
    s = m.setup(DT[dt], d, *heads, lens, new) if bits == 16 else m.setup(DT[dt], d, bits, *heads, lens, new)
    want = m.expect(s)
    for W in (2 ** 31, 2 ** 63 - 1, 2 ** 64 + 5):
        for S in (0, 2 ** 63 - 1, 2 ** 64 + 5):
            m.assert_within(m.call(s, W, S), *want, "out")
    part = m.expect(s, 100, 2200)
    m.assert_within(m.call(s, 100, 2 ** 63 - 1), *part, "out")


@pytest.mark.parametrize("dt,d,bits", mxc.FORMS)
@pytest.mark.parametrize("turn", [False, True])
def test_keys_at_the_edges_with_the_norm(turn, dt, d, bits):
    """Keys that are tiny, huge or not finite, normalised: a NaN makes the whole key NaN, an
    infinity all others 0 and itself (and what it is rotated with) NaN."""
    s = mxc.new_tokens(DT[dt], d, bits, 2, [120], [120], seed=8, gain=True, turn=turn)
    k = s["k"]
    k[1], k[2] = 0.0, -0.0
    k[3] *= 2.0 ** -120
    k[4] *= 2.0 ** -132
    k[5] *= 2.0 ** 120
    k[6, :, 5] = float("nan")
    k[7, :, d - 1] = float("nan")
    k[8, 1, 40] = float("nan")
    k[9, :, 33] = float("inf")
    k[10, :, 63], k[10, 0, 2] = float("-inf"), float("nan")
    k[11] = torch.finfo(k.dtype).max
    k[12] = float("nan")
    got = mxc.append(s)
    mxc.same(got, mxc.appended(s))
    a = mxc.dev(s)
    back = ops.kv_read_mx(got[0].cuda(), got[1].cuda(), a["table"], a["lens"], a["cu"], 120, d, torch.float32)[0].cpu()
    assert back[[6, 7, 10, 12], 0].isnan().all() and back[8, 1].isnan().all() and not back[8, 0].isnan().any()
    assert bool((back[9].isnan().sum(-1) == (64 if turn else 32)).all())


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_of_pages_by_any_index(bits):
    """What the whole cache's key_rows and value_rows take: numbers from either end, lists,
    slices, masks, tensors on either side; within a captured graph tensors on the device."""
    cfg = hba_amd.HBAConfig(n_heads=4, n_kv=2, head_dim=64)
    c = hba_amd.MXKVCache(cfg, 2, 200, torch.float32, "cuda", bits=bits)
    for s in range(2):
        c.load(s, *(torch.randn(200, 2, 64, device="cuda") for _ in range(2)))
    mask = torch.zeros(8, dtype=torch.bool)
    mask[[1, 6]] = True
    for rows_of, pages in ((c.key_rows, c.k_pages), (c.value_rows, c.v_pages)):
        held = mx64.rows(pages.cpu(), bits, 64, pages is c.k_pages).float().cuda()
        for i in (3, -1, [0, -8], slice(2, 7, 2), mask, mask.cuda(), torch.tensor([[7, -2]]), torch.tensor([5, 5, 0]).cuda(),
                  torch.tensor(4).cuda(), torch.zeros(0, dtype=torch.long)):
            assert torch.equal(rows_of(i), held[i]), i
        i = torch.tensor([[-1, 2], [0, -8]], device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = rows_of(i)
        for j in (i.clone(), torch.tensor([[4, -3], [7, 1]], device="cuda")):
            i.copy_(j)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, held[j])


def anywhere(t, by):
    """t in memory that begins `by` elements behind a 16-byte boundary."""
    flat = torch.empty(t.numel() + by, dtype=t.dtype, device="cuda")
    assert flat.data_ptr() % 16 == 0
    flat[by:] = t.cuda().flatten()
    return flat[by:].view(t.shape)


@pytest.mark.parametrize("by", [1, 2, 3])
@pytest.mark.parametrize("dt,d,bits", mxc.FORMS)
def test_tables_that_begin_anywhere(dt, d, bits, by):
    """cos and sin are read in 16 bytes wherever they begin: append, single tokens, parts."""
    s = mxc.new_tokens(DT[dt], d, bits, 2, [70, 9], [33, 2])
    mxc.same(mxc.append(s, cos=anywhere(s["cos"], by), sin=anywhere(s["sin"], (by + 1) % 4)), mxc.append(s))
    for new, shared in ((None, 0), ([40, 3], 0), (None, 64)):
        s = mxc.setup(DT[dt], d, bits, 4, 2, [200, 65], new, shared=shared)
        got = mxc.call(s, cos=anywhere(s["cos"], by), sin=anywhere(s["sin"], (by + 1) % 4))
        assert torch.equal(got, mxc.call(s))


@pytest.mark.parametrize("dt,d,bits", [*mxc.FORMS, ("f32", 64, 16), ("bf16", 128, 16)])
def test_pages_outside_the_cache_are_read_as_the_nearest(dt, d, bits):
    """Attention clamps page numbers: the same results as with the first and the last page there."""
    whole = bits == 16
    m = rows if whole else mxc
    for lens, new, shared in (([300, 65], None, 0), ([300, 65], [40, 3], 0), ([300, 200], None, 128), ([3000], None, 0),
                              ([3000, 700], [600, 7], 0)):
        s = m.setup(DT[dt], d, *(() if whole else (bits,)), 6, 3, lens, new, shared=shared)
        for name in ("kr", "vp") if whole else ("kp", "vp"):   # the first and the last page: whole, and unlike the others
            s[name][0], s[name][-1] = s[name][int(s["table"][0, 1])], s[name][int(s["table"][0, 2])]
        far, near = s["table"].clone(), s["table"].clone()
        for at, page, there in (((0, 0), -7, 0), ((0, 3), 10 ** 8, -1), ((-1, 1), 2 ** 31 - 1, -1), ((-1, 0), -2 ** 31, 0)):
            if at[1] < shared // 64:
                far[:, at[1]], near[:, at[1]] = page, there % len(s["vp"])
            else:
                far[at], near[at] = page, there % len(s["vp"])
        got, want = m.call(s, table=far), m.call(s, table=near)
        assert torch.isfinite(want).all() and torch.equal(got, want) and not torch.equal(want, m.call(s))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128])
def test_read_at_the_smallest_scales(d, bits):
    """fp32 rows are the values; bf16 rows too, but for 8 bits at 2^-126 and 2^-125, whose smallest
    codes lie below bf16's last step: those are the nearest, ties to even."""
    g = torch.Generator().manual_seed(bits)
    pages = torch.randint(0, 256, (20, 1, mx64.page_bytes(d, bits)), generator=g).to(torch.uint8)
    if bits == 8:
        pages[(pages & 127) == 127] = 3                       # no NaN
    for b in range(20):
        pages[b, :, 64 * d * bits // 8:] = b + 1
    a = [torch.arange(20, dtype=torch.int32).view(1, 20).cuda(), torch.tensor([1280], dtype=torch.int32).cuda(),
         torch.tensor([0, 1280], dtype=torch.int32).cuda()]
    for dt in (torch.float32, torch.bfloat16):
        out = ops.kv_read_mx(pages.cuda(), pages.cuda(), *a, 1280, d, dt)
        for x, keys in zip(out, (True, False)):
            want = mx64.rows(pages, bits, d, keys).float()    # [20, 1, 64, d]
            got = x.cpu().view(20, 64, 1, d).transpose(1, 2)
            assert torch.equal(got, want.to(dt))
            exact = got.float() == want
            assert exact[2:].all() and (exact.all() or (bits == 8 and dt == torch.bfloat16))


@pytest.mark.parametrize("dt,d,bits", mxc.FORMS)
def test_calls_repeat_themselves(dt, d, bits):
    """Bit for bit: no sum's order depends on which workgroup is first."""
    for lens, new, shared in (([300, 65], None, 0), ([5000, 700, 2100], None, 0), ([3000, 700], [600, 7], 0),
                              ([300, 200, 1500], None, 128), ([300, 65], [40, 3], 0)):
        a = mxc.dev(mxc.setup(DT[dt], d, bits, 6, 3, lens, new, shared=shared))
        want = mxc.call(a)
        for _ in range(4):
            assert torch.equal(mxc.call(a), want)
