"""Index arrays of other dimensions than one are refused with the package's error."""
import types

import pytest
import torch

from jasnamacos_amd import _lib
from jasnamacos_amd import frame_attention as fa
from jasnamacos_amd.deform_conv import INVALID_SHAPE, DeformConvError


@pytest.mark.parametrize("which", ["cu_q", "cu_kv"])
@pytest.mark.parametrize("shape", [(), (2, 2)])
def test_dimensions(which, shape):
    op = fa.FrameAttention(types.SimpleNamespace(ctx=None, device=0, _lib=_lib.load()), 4, 2, 64)
    q, k = torch.zeros(8, 4, 64), torch.zeros(8, 2, 64)
    with pytest.raises(DeformConvError) as e:
        op.forward_dev(q, k, k, q, **{which: torch.zeros(shape, dtype=torch.int32)})
    assert e.value.status == INVALID_SHAPE
