"""Calls of the packed, 4-bit and page operators at the edges of what their documentation allows."""
import pytest
import torch

import b200_llama as B

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("order", [(0, 1), (1, 0), (1,)])
def test_compact_with_a_pool_that_holds_nothing(order):
    full = torch.arange(6, device=DEV).float().view(1, 6, 1, 1, 1).expand(2, 6, 2, 4, 8).contiguous()
    empty = torch.zeros(0, 6, 2, 4, 8, device=DEV)
    table = torch.tensor([[5, 4, 2, -1]], dtype=torch.int32, device=DEV)
    B.compact_pages([(full, empty)[i] for i in order], [5, 4], [0, 1], table, [0, 1, 2, 3, 1, 0])
    assert B.device_status() == 0 and table.tolist() == [[0, 1, 2, -1]]
    if 0 in order:
        assert full[0, :, 0, 0, 0].tolist() == [5, 4, 2, 3, 4, 5]
