"""How the distillation's Python side turns its arguments into the library's, on CPU tensors."""

import torch

from alphafly_b200 import distill


def test_lists_without_entries_are_lists():
    """The library takes two NULLs for "all moves": a list of width 0, whose tensors have no address, must not become that."""
    logits = torch.zeros(3, 50)
    moves, valid, listed = distill._legal((torch.zeros(3, 0, dtype=torch.int64), torch.zeros(3, 0, dtype=torch.bool)), logits)
    assert moves.data_ptr() and valid.data_ptr() and listed == moves.shape[1] == valid.shape[1] >= 1
    assert moves.shape[0] == 3 and moves.dtype == torch.int64 and valid.dtype == torch.bool and not valid.any()
    assert distill._legal(None, logits) == (None, None, 0)
