"""How the paged entry points take [tokens, heads, head_dim] arguments: address and token stride, or a refusal (host tensors: nothing is
launched)."""
from types import SimpleNamespace

import pytest
import torch

from runtherder_b200._lib import RhError
from runtherder_b200.kernels import _token_rows

HOST = SimpleNamespace(device_index=-1)


def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_what_is_taken():
    fused = bf(9, 8 + 2 + 2, 64)
    flat = fused.view(9, -1)
    for t, n, heads, want in (
            (bf(9, 8, 64), 9, 8, (0, 512)), (bf(20, 8, 64), 9, 8, (0, 512)), (bf(9, 512), 9, 8, (0, 512)), (bf(72, 64), 9, 8, (0, 512)),
            (bf(3, 3, 512), 9, 8, (0, 512)), (bf(9 * 512), 9, 8, (0, 512)), (bf(3, 3, 8, 64), 9, 8, (0, 512)), (fused[:, :8], 9, 8, (0, 768)),
            (fused[:, 8:10], 9, 2, (512, 768)), (flat[:, 640:], 9, 2, (640, 768)), (fused[:1], 1, 8, (0, 512)), (fused[3:4, 8:10], 1, 2, (3 * 768 + 512, None))):
        at, stride = _token_rows(HOST, t, n, heads, 64, "q")
        assert (at - (t.untyped_storage().data_ptr())) // 2 == want[0]
        assert want[1] is None or stride == want[1]


@pytest.mark.parametrize("t,n,heads", [
    (bf(9, 12, 64), 9, 8),            # a whole fused projection in place of its slice: tokens would be read 512 values apart
    (bf(9, 12, 64), 2, 8), (bf(18, 4, 64), 9, 8), (bf(8, 8, 64), 9, 8), (bf(9, 8, 64).float(), 9, 8), (bf(9, 8, 64).transpose(0, 1), 8, 9),
    (bf(9, 64, 8).transpose(1, 2), 9, 8), (bf(9, 12, 64)[:, ::2], 9, 6), (bf(9, 12, 64)[:, :4], 9, 8),
])
def test_what_is_refused(t, n, heads):
    with pytest.raises(RhError):
        _token_rows(HOST, t, n, heads, 64, "q")
