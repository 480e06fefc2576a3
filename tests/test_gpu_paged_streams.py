"""The paged cache's calls on a stream that its tensors were not made on."""
import pytest
import torch

from test_gpu_paged import BF, F32, Batch, ints, rope_table, step_buffers
from vireo_amd import paged as P

pytestmark = pytest.mark.gpu


class Busy:
    """A stream that has work for some milliseconds, and new tensors of the current stream that are filled at once: a
    stream that does not share its hardware queue with the current one, if there is one (else all is in order anyway)."""

    def __init__(self, dev):
        self.dev, self.x, self.y = dev, torch.zeros((4096, 4096), device=dev), torch.zeros((4096, 4096), device=dev)
        warm = [torch.zeros(1 << 17, device=dev) for _ in range(32)]  # memory that needs no new allocation below
        del warm
        for _ in range(8):
            self.s = torch.cuda.Stream()
            torch.cuda.synchronize()
            with self as s:
                torch.zeros(8, device=dev)
                torch.cuda.current_stream().synchronize()
                apart = not s.query()
            torch.cuda.synchronize()
            if apart:
                break

    def __enter__(self):
        with torch.cuda.stream(self.s):
            for _ in range(20):
                torch.mm(self.x, self.x, out=self.y)
        return self.s

    def __exit__(self, *_):
        pass

    def fill(self, like, value):
        """Memory of tensors of this size that were dropped is taken again and written while the other stream is busy."""
        kept = [torch.full_like(like, value) for _ in range(16)]
        torch.cuda.synchronize()
        return kept


def test_bookkeeping_with_dropped_tensors(cuda):
    t = P.PagedTable.create(50, 40, 400, 16, device=cuda)
    busy = Busy(cuda)
    with busy as s:
        bufs = step_buffers(50, 2000, cuda)
        s.wait_stream(torch.cuda.current_stream())
        ids, n_new = ints(list(range(49, -1, -1)), cuda), ints([7 + i for i in range(50)], cuda)
        t.extend(n_new, *bufs, ids=ids, stream=s)
        like = n_new.clone()
        del ids, n_new
        busy.fill(like, 1)
    assert t.len.tolist() == [56 - i for i in range(50)]
    with busy as s:
        t.truncate(ints([5] * 50, cuda), stream=s)
        busy.fill(like, 1)
    assert t.len.tolist() == [5] * 50
    # two updates in a row: the first one's ids are still to be read
    lens = [40 * i for i in range(50)]
    b = Batch(cuda, lens, 4, 2, 64, 16, BF, BF, seed=50)
    plan = P.PagedPlan(b.table, b.cache, 50, 4)
    out = torch.zeros_like(b.q)
    torch.cuda.synchronize()
    with busy as s:
        plan.update(ids=b.tids.clone(), stream=s)
        b.cache.attend(b.q, out, plan, stream=s)
        plan.update(ids=ints([0] * 50, cuda), stream=s)
        busy.fill(b.tids, 1)
    b.check(out)


def test_rows_and_queries_dropped(cuda):
    b = Batch(cuda, [100, 33], 4, 2, 64, 16, BF, F32, seed=51)
    rope = rope_table(64, 50, cuda)
    pos, slots = ints([3, 4], cuda), ints([1, 17], cuda)
    x = torch.randn((2, 8, 64), device=cuda)
    k0, v0 = b.k.clone(), b.v.clone()
    want_q = torch.zeros((2, 4, 64), device=cuda)
    b.cache.append(x[:, :4], x[:, 4:6], x[:, 6:], pos, slots, want_q, rope)
    want_k, want_v = b.k.clone(), b.v.clone()
    want = b.attend()
    b.k.copy_(k0), b.v.copy_(v0)
    plan = P.PagedPlan(b.table, b.cache, 2, 4)
    out, q_out = torch.zeros_like(b.q), torch.zeros_like(want_q)
    busy = Busy(cuda)
    with busy as s:
        y, p, o = x.clone(), pos.clone(), slots.clone()
        s.wait_stream(torch.cuda.current_stream())
        b.cache.append(y[:, :4], y[:, 4:6], y[:, 6:], p, o, q_out, rope, stream=s)
        plan.update(ids=b.tids, stream=s)
        b.cache.attend(b.q.clone(), out, plan, stream=s)
        del y, p, o
        mem = plan.mem.clone()
        del plan  # and its memory, which the enqueued calls use
        kept = [torch.ones_like(x) for _ in range(8)], [torch.ones_like(mem) for _ in range(8)], [torch.ones_like(b.q) for _ in range(8)]
        busy.fill(pos, 9)
    bits = lambda t: t.view(torch.int16)  # noqa: E731  (unwritten slots hold NaN)
    assert torch.equal(bits(b.k), bits(want_k)) and torch.equal(bits(b.v), bits(want_v)) and torch.equal(q_out, want_q)
    assert torch.equal(out, want) and len(kept) == 3


def test_a_handle_records_its_tensors_on_every_stream(cuda):
    b = Batch(cuda, [100], 4, 2, 64, 16, BF, BF, seed=52)
    plan = P.PagedPlan(b.table, b.cache, 1, 4)
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = torch.zeros_like(b.q)
    torch.cuda.synchronize()
    for s in streams:
        plan.update(ids=b.tids, stream=s)
        b.cache.attend(b.q, out, plan, stream=s)
        torch.cuda.synchronize()
    for h in (plan, b.table, b.cache):
        assert h.streams == {s.cuda_stream for s in streams}


def test_counts_past_32_bits_are_refused(cuda):
    """A C int would hold their low bits, which are counts that the library takes."""
    b = Batch(cuda, [100], 4, 2, 64, 16, BF, BF, seed=53)
    more = 2 ** 32
    with pytest.raises(ValueError):
        P.PagedTable(b.table.blocks, b.table.len, b.table.free_blocks, b.table.n_free, more + 16)
    for n, heads, lists in ((more + 1, 4, 0), (1, more + 4, 0), (1, 4, more)):
        with pytest.raises(ValueError):
            P.PagedPlan(b.table, b.cache, n, heads, lists)
    cache = P.PagedCache(b.k, b.v, torch.zeros((b.cache.n_blocks, 2, 64), dtype=BF, device=cuda))
    plan = P.PagedPlan(b.table, cache, 1, 4, 5)
    plan.update(ids=b.tids)
    lists = torch.zeros((1, 2, 5), dtype=torch.int32, device=cuda)
    for sinks, window in ((more, 1), (1, more + 1), (-more, 1)):
        with pytest.raises(ValueError):
            cache.select(b.q, plan, lists, sinks=sinks, window=window)
    cache.select(b.q, plan, lists, sinks=1, window=1)
    assert lists[0, 0].tolist()[0] == 0
