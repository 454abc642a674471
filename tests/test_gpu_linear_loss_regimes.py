"""The C entry points of the loss from hidden states with a gradient of no rows."""

import pytest
import torch

from conftest import announce, load_pkg
from test_gpu_linear_loss import BOTH, DEV

pytestmark = pytest.mark.gpu
pkg = load_pkg()


@pytest.mark.parametrize("dtype", BOTH)
def test_no_rows_at_any_element(dtype):
    announce("linear loss, no rows, any alignment", dtype)
    native, stream = pkg._native, torch.cuda.current_stream().cuda_stream
    vocab, c = 33, 65
    for off in (0, 1, 3):
        flat = torch.full((vocab * c + 9,), 7.0, dtype=dtype, device=DEV)
        native.call("rwkv_linear_loss_backward", None, None, None, None, None, None, None, 0.0, 0, vocab, c,
                    pkg.neighbors._code(dtype), -100, None, flat[off:].data_ptr(), None, 0, stream)
        torch.cuda.synchronize()
        assert not flat[off:off + vocab * c].any()
        assert (flat[:off] == 7).all() and (flat[off + vocab * c:] == 7).all()
