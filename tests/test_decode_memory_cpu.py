"""The addresses that a cache, a batch and a plan keep are those of memory that they hold."""
import torch

from tts_amd import ops


def _given():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return [torch.zeros(2, 1, 4, 8) for _ in range(2)], [i32(0, 1).view(1, 2), i32(3), i32(0, 1)]


def test_given_tensors_that_move_leave_theirs_behind():
    """A tensor whose data is exchanged (as by a module's .to) takes its name to other memory: the cache and the batch stay where they were."""
    (k, v), (table, lens, starts) = _given()
    cache, batch = ops.PagedKV(k, v), ops.PagedBatch(table, lens, starts, 1)
    was = [t.data_ptr() for t in (k, v, table, lens, starts)]
    for t in (k, v, table, lens, starts):
        t.data = torch.ones_like(t)
    held = (cache.k, cache.v, batch.block_table, batch.seq_lens, batch.q_starts)
    assert [t.data_ptr() for t in held] == was
    assert [cache._c.k, cache._c.v, batch._c.block_table, batch._c.seq_lens, batch._c.q_starts] == was
    assert bool((cache.k == 0).all()) and int(batch.seq_lens) == 3


def test_given_tensors_are_written_through():
    (k, v), (table, lens, starts) = _given()
    cache, batch = ops.PagedKV(k, v), ops.PagedBatch(table, lens, starts, 1)
    k[1, 0, 2] = 5.0
    lens += 1
    assert bool((cache.k[1, 0, 2] == 5).all()) and int(batch.seq_lens) == 4
    cache.v.fill_(2.0)
    assert bool((v == 2).all())
