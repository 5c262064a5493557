"""Calls at the ends of what the paged caches' operators take, against 64-bit results."""
import pytest
import torch

import test_gpu_mx_cache as mxc
import test_gpu_paged_attn as rows

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
