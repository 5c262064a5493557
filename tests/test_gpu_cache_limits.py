"""Calls at the ends of what the paged caches' operators take, against 64-bit results."""
import pytest
import torch

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
