"""Tables with more rows than a gradient can have: looked up without one, refused by the forward pass with one."""
import pytest
import torch

from deep_ep.ops.embedding import embedding_lookup


@pytest.mark.gpu
def test_more_rows_than_a_gradient_takes():
    import deep_ep
    row = torch.arange(8.0, device='cuda')
    table = row.expand(2 ** 30, 8)          # (one row in memory)
    ids = torch.tensor([2 ** 30 - 1, 2 ** 30, -1, 0], device='cuda')
    want = torch.stack([row, row * 0, row * 0, row])
    assert torch.equal(embedding_lookup(table, ids), want)
    row.requires_grad_()
    with pytest.raises(deep_ep.EPException, match='2\\^30'):
        embedding_lookup(row.expand(2 ** 30, 8), ids)
    with torch.no_grad():
        assert torch.equal(embedding_lookup(row.expand(2 ** 30, 8), ids), want)
