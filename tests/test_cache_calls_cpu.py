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


def test_plan_of_too_many_tiles_or_jobs():
    """The Q4_0 kernel's quotients stay below 2^22 and its list below 2^30 places."""
    plan = getattr(qb.load(), "_ZN2ql10attn4_planEiiPKiiiPNS_9Attn4ArgsEPmS4_")
    args = ctypes.create_string_buffer(1 << 14)
    a, b = ctypes.c_size_t(), ctypes.c_size_t()

    def run(tiles, jobs, hd=128):
        t = (ctypes.c_int32 * len(tiles))(*tiles)
        return plan(hd, 148, t, len(tiles), jobs, args, ctypes.byref(a), ctypes.byref(b))

    for hd in (64, 128):
        assert run([1], (1 << 22) - 1, hd) == 0 and a.value > 0 and b.value > 0
        assert run([1, 1], 1 << 22, hd) == 1
        assert run([1 << 20], 1 << 10, hd) == 0
        assert run([1 << 20], (1 << 10) + 1, hd) == 1


def test_reading_changes_nothing_of_the_cache():
    """ql_kv_read takes the cache as const: two threads may read it at once."""
    from tests.test_cache_ops_cpu import P, Cache, i32, i64, refused

    c = Cache(lens=(100, 50, 0, 0))
    before = ctypes.string_at(ctypes.addressof(c.kv), ctypes.sizeof(c.kv))
    L = qb.load()
    assert L.ql_kv_read(*c.args(), 0, 2, i32(0, 1), i64(100, 50), i32(0, 0), qb.F32, None, None) == qb.OK
    refused(L.ql_kv_read(*c.args(), 0, 2, i32(0, 0), i64(0, 99), i32(9, 2), qb.F32, P, P + 32768),
            "beyond the written prefix")
    assert list(c.marks) == [0] * 4
    assert ctypes.string_at(ctypes.addressof(c.kv), ctypes.sizeof(c.kv)) == before
