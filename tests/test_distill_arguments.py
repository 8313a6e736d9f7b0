"""How the distillation's Python side turns its arguments into the library's, on CPU tensors."""

import pytest
import torch

from alphafly_b200 import distill


def test_lists_without_entries_are_lists():
    """The library takes two NULLs for "all moves": a list of width 0, whose tensors have no address, must not become that."""
    logits = torch.zeros(3, 50)
    moves, valid, listed = distill._legal((torch.zeros(3, 0, dtype=torch.int64), torch.zeros(3, 0, dtype=torch.bool)), logits)
    assert moves.data_ptr() and valid.data_ptr() and listed == moves.shape[1] == valid.shape[1] >= 1
    assert moves.shape[0] == 3 and moves.dtype == torch.int64 and valid.dtype == torch.bool and not valid.any()
    assert distill._legal(None, logits) == (None, None, 0)


def test_a_teacher_keeps_the_modes_of_its_parts(monkeypatch):
    """A part that is frozen in its evaluation mode stays so, whatever the whole's mode, and also after a failure."""
    class Teacher(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.frozen, self.other, self.fails, self.seen = torch.nn.Linear(2, 2), torch.nn.Linear(2, 2), False, None

        def forward(self, x):
            self.seen = [m.training for m in self.modules()]
            if self.fails:
                raise RuntimeError("planted")
            return x, x

    monkeypatch.setattr(distill, "top_logits", lambda logits, *args: logits)
    teacher, x = Teacher().train(), torch.ones(1, 2)
    teacher.frozen.eval()
    assert distill.teacher_targets(teacher, x, 1) is x and teacher.seen == [False, False, False]
    assert teacher.training and teacher.other.training and not teacher.frozen.training
    teacher.fails = True
    with pytest.raises(RuntimeError, match="planted"):
        distill.teacher_targets(teacher, x, 1)
    assert teacher.training and teacher.other.training and not teacher.frozen.training
