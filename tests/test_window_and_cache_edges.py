"""Calls of the window and cache operators at the edges of what their documentation
allows: state after an error, lengths of any type, launches of any size, pages with
anything behind their sequences, and every form that the gradients' kernels take."""
import pytest
import torch

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
