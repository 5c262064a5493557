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
