"""What the Python calls on the paged cache take for positions and sequences, without a
device."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import qllama_b200 as qb
from qllama_b200 import model as qm

# (tensors of the CPU have device -1 for get_device)
KV = SimpleNamespace(ctx=SimpleNamespace(device=-1))


def args(start_pos, seq_ids=None, batch=3):
    qm._L or qm._start()
    q, out = torch.zeros(batch, 2, 4, 32), torch.zeros(batch, 2, 128)
    a, _ = qm._appended_args(KV, 0, q, start_pos, 4, 2, 32, 1e4, seq_ids, out, None)
    return [a.start_pos[b] for b in range(batch)], [a.seq_ids[b] for b in range(batch)]


@pytest.mark.parametrize("start_pos", [5, np.int64(5), [5], (5,), np.array(5), np.array([5]), [5] * 3, [5.0] * 3,
                                       torch.tensor(5), torch.tensor([5]), torch.tensor([5, 5, 5])])
def test_one_position_stands_for_all(start_pos):
    assert args(start_pos) == ([5, 5, 5], [0, 1, 2])


@pytest.mark.parametrize("seq_ids", [[4, 0, 2], (4, 0, 2), np.array([4, 0, 2], np.int32),
                                     torch.tensor([4, 0, 2])])
def test_positions_and_sequences_of_a_batch(seq_ids):
    assert args(np.array([7, 8, 1 << 40]), seq_ids) == ([7, 8, 1 << 40], [4, 0, 2])
    assert args(range(7, 10), seq_ids) == ([7, 8, 9], [4, 0, 2])


def test_one_sequence_may_be_a_number():
    for seq in (3, np.int32(3), np.array(3), [3]):
        assert args(9, seq, batch=1) == ([9], [3])


@pytest.mark.parametrize("start_pos, seq_ids", [([1, 2], None), ([], None), ([1] * 4, None),
                                                (0, [0, 1]), (0, []), (0, range(4))])
def test_other_numbers_of_them_are_refused(start_pos, seq_ids):
    with pytest.raises(qb.QllamaError, match="one position and one sequence"):
        args(start_pos, seq_ids)
