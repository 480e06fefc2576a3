"""The paged cache's operators (include/vireo_paged.h) against plain forms: the bookkeeping entry for entry, the
arithmetic against fp64 with bounds that count each rounding (tests/paged_ref.py)."""
import ctypes as C
import math
import random

import pytest
import torch

from paged_ref import E2BIG, EINVAL, ENOSPC, RefTable, attend64, attend_bound, half_step, heads64
from vireo_amd import _lib
from vireo_amd import paged as P

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def randn(shape, dtype, dev, seed):
    return torch.randn(shape, generator=gen(dev, seed), device=dev).to(dtype)


def rope_table(rotary, max_pos, dev):
    t = torch.empty((max_pos, rotary), device=dev)
    _lib.check(_lib.load().vireo_rope_table(C.c_float(10000.0), rotary, max_pos, C.c_void_p(t.data_ptr())),
               "vireo_rope_table")
    return t


# ---- block tables ---------------------------------------------------------------------------------------------------

def same(table, ref):
    assert table.blocks.tolist() == ref.blocks
    assert table.len.tolist() == ref.len
    assert table.n_free.item() == ref.n_free
    assert table.free_blocks.tolist() == ref.free


def step_buffers(n, max_rows, dev):
    return (torch.full((n + 1,), 77, dtype=torch.int32, device=dev),
            torch.full((max_rows,), 77, dtype=torch.int32, device=dev),
            torch.full((max_rows,), 77, dtype=torch.int32, device=dev), torch.full((n,), 77, dtype=torch.int32, device=dev))


# (sequences of the table, blocks a sequence may have, blocks, block tokens, batch, largest growth, row buffer):
# one sequence; blocks that run out; a table too narrow; rows in a second launch; more sequences than threads; LDS
# beyond 64 KB
TABLES = [(1, 8, 8, 16, 1, 5, 8), (7, 9, 9, 16, 5, 60, 400), (9, 3, 100, 32, 9, 60, 500), (50, 300, 120, 16, 40, 200, 9000),
          (40, 16, 400, 64, 33, 90, 700), (1500, 6, 1100, 16, 1400, 9, 8000), (4096, 2, 6000, 16, 4000, 3, 2048),
          (20, 10, 100, 128, 20, 300, 2048)]


@pytest.mark.parametrize("seqs,width,n_blocks,G,batch,most,max_rows", TABLES)
def test_tables_step_by_step(cuda, seqs, width, n_blocks, G, batch, most, max_rows):
    """Steps of extensions and cuts with sequences in any order, some named twice or out of range, negative counts,
    tables and pools that run out: every array equal to the plain form's after every call."""
    rng = random.Random(seqs + most)
    t, ref = P.PagedTable.create(seqs, width, n_blocks, G, device=cuda), RefTable(seqs, width, n_blocks, G)
    same(t, ref)
    seen = set()
    for step in range(8):
        ids = rng.sample(range(seqs), min(batch, seqs))
        if step % 2 and len(ids) > 2:  # not a sequence, or not again
            ids[rng.randrange(len(ids))] = ids[0]
            ids[rng.randrange(1, len(ids))] = rng.choice([-1, seqs, 2 ** 31 - 1, -2 ** 31])
        new = [rng.choice([0, 1, 1, rng.randint(0, most)]) for _ in ids]
        if step == 3:
            new[-1] = -3
        bufs = step_buffers(len(ids), max_rows, cuda)
        t.extend(ints(new, cuda), *bufs, ids=ints(ids, cuda))
        want = ref.extend(ids, new, max_rows)
        for got, w in zip(bufs, want):
            assert got.tolist() == w
        seen |= set(want[3])
        same(t, ref)
        ids = rng.sample(range(seqs), min(batch, seqs))
        if step % 2:
            ids[-1] = rng.choice([-5, seqs, ids[0]])
        cut = [rng.choice([-1, 0, 10 ** 6, 10 ** 6, 10 ** 6,
                           rng.randint(0, max(1, ref.len[i] if 0 <= i < seqs else 1))]) for i in ids]
        t.truncate(ints(cut, cuda), ids=ints(ids, cuda))
        ref.truncate(ids, cut)
        same(t, ref)
    assert 0 in seen
    if seqs in (7, 50, 1500):
        assert ENOSPC in seen
    if seqs in (9, 4096):
        assert E2BIG in seen
    if len(ids) > 2:
        assert EINVAL in seen
    t.truncate()  # every sequence ends
    ref.truncate(range(seqs), [0] * seqs)
    same(t, ref)
    assert t.n_free.item() == n_blocks


def test_extend_by_one_and_empty_batches(cuda):
    """n_new None is a token each, ids None the first rows; a batch of no sequences and a step of no rows."""
    t, ref = P.PagedTable.create(6, 4, 12, 16, device=cuda), RefTable(6, 4, 12, 16)
    for _ in range(18):
        bufs = step_buffers(4, 7, cuda)
        t.extend(None, *bufs)
        for got, w in zip(bufs, ref.extend(range(4), [1] * 4, 7)):
            assert got.tolist() == w
    same(t, ref)
    bufs = step_buffers(0, 3, cuda)
    t.extend(None, *bufs)
    assert bufs[0].tolist() == [0] and bufs[2].tolist() == [-1] * 3
    bufs = step_buffers(2, 0, cuda)
    t.extend(ints([0, 1], cuda), *bufs)  # the second one's row does not fit
    assert bufs[3].tolist() == [0, E2BIG] and bufs[0].tolist() == [0, 0, 1]
    same(t, ref)


def test_cut_and_extend_again_takes_the_same_blocks(cuda):
    t = P.PagedTable.create(5, 40, 150, 16, device=cuda)
    bufs = step_buffers(5, 900, cuda)
    t.extend(ints([100, 17, 300, 16, 1], cuda), *bufs)
    base = t.len.clone()
    t.extend(ints([30, 0, 64, 1, 16], cuda), *bufs)
    before = [x.clone() for x in (t.blocks, t.len, t.free_blocks, t.n_free, *bufs)]
    for _ in range(3):
        t.truncate(base)
        t.extend(ints([30, 0, 64, 1, 16], cuda), *bufs)
        for a, b in zip(before, (t.blocks, t.len, t.free_blocks, t.n_free, *bufs)):
            assert torch.equal(a, b)


# ---- rows into the cache --------------------------------------------------------------------------------------------

# (head size, heads, kv heads, block tokens, input, cache, q_out, rotary, norms, biases, rows)
ROWS = [(128, 32, 4, 32, F32, BF, F32, 128, True, False, 1), (128, 8, 2, 16, BF, BF, BF, 128, True, True, 77),
        (64, 6, 2, 16, HF, HF, HF, 32, False, True, 33), (64, 1, 1, 128, F32, HF, HF, 64, True, True, 130),
        (256, 8, 1, 64, BF, HF, F32, 256, True, False, 65), (256, 3, 3, 16, F32, BF, BF, 16, False, False, 18),
        (128, 4, 4, 16, HF, BF, F32, 0, True, True, 9), (64, 16, 16, 32, BF, BF, BF, 48, True, False, 300)]


@pytest.mark.parametrize("d,H,KV,G,tin,tc,tq,rotary,norms,biases,T", ROWS)
def test_append(cuda, d, H, KV, G, tin, tc, tq, rotary, norms, biases, T):
    """Rows of one projection's output (strided views) against fp64. Each result is rounded once, by half a step of
    its type; the fp32 arithmetic before it is a bias, a norm (a sum of d squares: d / 16 + 4 additions in line; a root, a division,
    three products) and a rotation (two products, a sum): under 24 + d / 16 half steps of fp32, of the largest value that a
    rotated pair may take. Rows without a slot leave everything as it was, a position outside the table rotates nothing."""
    dev, max_pos, eps = cuda, 300, 1e-5
    n_blocks = T // G + 5
    qkv = randn((T, (H + 2 * KV) * d), tin, dev, 1) * 3
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([H * d, KV * d, KV * d], 1))
    gk, gv = randn((n_blocks, KV, G, d), tc, dev, 2), randn((n_blocks, KV, d, G), tc, dev, 3)
    gm = randn((n_blocks, KV, d), tc, dev, 4)
    rope = rope_table(rotary, max_pos, dev) if rotary else None
    qn, kn = (1 + 0.3 * randn(d, F32, dev, s) if norms else None for s in (5, 6))
    qb, kb, vb = (randn(h * d, F32, dev, s) if biases else None for h, s in ((H, 7), (KV, 8), (KV, 9)))
    rng = random.Random(T)
    # consecutive slots of blocks in any order (so that some complete), then padding and slots past the pool
    order = rng.sample(range(n_blocks), T // G + 1)
    slots = [order[i // G] * G + i % G for i in range(T)]
    pos = [rng.randrange(max_pos) for _ in range(T)]
    if T > 8:
        slots[3], slots[5] = -1, n_blocks * G
        pos[2], pos[4] = -1, max_pos
    slots, pos = ints(slots, dev), ints(pos, dev)
    live = (slots >= 0) & (slots < n_blocks * G)
    want_q = heads64(q, qb, qn, eps, rope, pos)
    want_k = heads64(k, kb, kn, eps, rope, pos)
    want_v = heads64(v, vb, None, eps, None, pos)
    out = randn((T, H, d), tq, dev, 10)
    out0, k0, v0, m0 = out.clone(), gk.clone(), gv.clone(), gm.clone()
    cache = P.PagedCache(gk, gv, gm)
    cache.append(q, k, v, pos, slots, out, rope, qn, kn, qb, kb, vb, eps=eps)
    near = (24 + d / 16) * 2.0 ** -24

    def close(got, want, dtype, largest):
        err = (got.double() - want).abs()
        assert bool((err <= half_step(dtype) * want.abs() * (1 + 2 * near) + near * largest + 1e-30 +
                     (2.0 ** -25 if dtype is HF else 0)).all()), float(err.max())

    # a rotated value's error is of the pair's size
    pair = lambda x: x.abs().amax(-1, keepdim=True) * 1.5  # noqa: E731
    close(out[live], want_q[live], tq, pair(want_q[live]))
    assert torch.equal(out[~live], out0[~live])
    s = slots[live].long()
    b, o = s // G, s % G
    close(gk[b, :, o], want_k[live], tc, pair(want_k[live]))
    close(gv[b, :, :, o], want_v[live], tc, pair(want_v[live]))
    keep = torch.ones((n_blocks, G), dtype=torch.bool, device=dev)
    keep[b, o] = False
    assert torch.equal(gk.transpose(1, 2)[keep], k0.transpose(1, 2)[keep])
    assert torch.equal(gv.permute(0, 3, 1, 2)[keep], v0.permute(0, 3, 1, 2)[keep])
    full = torch.unique(b[o == G - 1])
    want_m = gk[full].double().mean(2)
    err = (gm[full].double() - want_m).abs()
    assert bool((err <= half_step(tc) * want_m.abs() + G * 2.0 ** -24 * gk[full].double().abs().mean(2) +
                 (2.0 ** -25 if tc is HF else 0)).all())
    rest = torch.ones(n_blocks, dtype=torch.bool, device=dev)
    rest[full] = False
    assert torch.equal(gm[rest], m0[rest])
    if T >= 2 * G:
        assert full.numel() > 0
    # again, the queries in place
    if tin is tq:
        ik, iv = k0.clone(), v0.clone()
        P.PagedCache(ik, iv).append(q, k, v, pos, slots, q, rope, qn, kn, qb, kb, vb, eps=eps)
        assert torch.equal(ik, gk) and torch.equal(iv, gv) and torch.equal(q[live], out[live])


def test_append_of_no_rows_and_of_weights_anywhere(cuda):
    """A step without rows changes nothing; norm weights, biases and the rotation's table at any 4-byte address; rows of
    a wider projection."""
    d, H, KV, G, T = 128, 4, 2, 16, 5
    k, v = (torch.zeros(s, dtype=BF, device=cuda) for s in ((4, KV, G, d), (4, KV, d, G)))
    cache = P.PagedCache(k, v, torch.zeros((4, KV, d), dtype=BF, device=cuda))
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    x0 = torch.zeros((0, H + 2 * KV, d), dtype=F32, device=cuda)
    cache.append(x0[:, :H], x0[:, H:H + KV], x0[:, H + KV:], none, none, torch.zeros((0, H, d), device=cuda))
    assert torch.count_nonzero(k) == 0
    x = torch.randn((T, 64 + (H + 2 * KV) * d + 4), generator=gen(cuda, 1), device=cuda)[:, 64:-4].unflatten(1, (-1, d))
    pool = torch.randn(1 + d + d + H * d + 40 * d, generator=gen(cuda, 2), device=cuda)
    qn, kn, qb, rope = (t.clone() for t in (pool[1:1 + d], pool[1 + d:1 + 2 * d], pool[1 + 2 * d:1 + 2 * d + H * d],
                                            pool[-40 * d:].view(40, d)))
    odd = lambda t: torch.cat([pool[:1], t.reshape(-1)])[1:].view(t.shape)  # noqa: E731  4 bytes off 16
    pos, slots = ints([3, 0, 39, 7, 1], cuda), ints([17, 16, 63, 0, 5], cuda)
    outs = []
    for f in (lambda t: t, odd):
        out = torch.zeros((T, H, d), device=cuda)
        cache.append(x[:, :H], x[:, H:H + KV], x[:, H + KV:], pos, slots, out, f(rope), f(qn), f(kn), q_bias=f(qb))
        outs.append((out, k.clone(), v.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


# ---- attention ------------------------------------------------------------------------------------------------------

class Batch:
    """Sequences of the given lengths over a pool whose unwritten slots hold NaN and infinities."""

    def __init__(self, dev, lens, H, KV, d, G, cache, query, seed=0, spread=1.0):
        rng = random.Random(seed)
        self.H, self.KV, self.d, self.G, self.lens = H, KV, d, G, lens
        n = len(lens)
        need = [-(-t // G) for t in lens]
        n_blocks, width = sum(need) + 3, max(need + [1]) + 2
        perm = rng.sample(range(n_blocks), n_blocks)
        self.ids = rng.sample(range(n + 2), n)
        table, at = [[-1] * width for _ in range(n + 2)], 0
        length = [0] * (n + 2)
        self.k = randn((n_blocks, KV, G, d), cache, dev, seed + 1)
        self.v = randn((n_blocks, KV, d, G), cache, dev, seed + 2)
        used = torch.zeros((n_blocks, G), dtype=torch.bool, device=dev)
        for i, t, nb in zip(self.ids, lens, need):
            table[i][:nb] = perm[at:at + nb]
            length[i] = t
            for j in range(nb):
                used[perm[at + j], :min(G, t - j * G)] = True
            at += nb
        junk = torch.tensor([math.nan, math.inf, -math.inf, 60000.0], device=dev).to(cache)
        fill = junk[torch.randint(4, (n_blocks, G), generator=gen(dev, seed + 3), device=dev)]
        self.k = torch.where(used[:, None, :, None], self.k, fill[:, None, :, None]).contiguous()
        self.v = torch.where(used[:, None, None, :], self.v, fill[:, None, None, :]).contiguous()
        self.table = P.PagedTable(ints(table, dev), ints(length, dev), torch.zeros(n_blocks, dtype=torch.int32, device=dev),
                                  ints([0], dev), G)
        self.rows = table
        self.cache = P.PagedCache(self.k, self.v)
        self.q = (randn((n, H, d), F32, dev, seed + 4) * spread).to(query)
        self.tids = ints(self.ids, dev)

    def attend(self, lists=None, scale=None, width=0, stream=None):
        plan = P.PagedPlan(self.table, self.cache, len(self.lens), self.H, width)
        out = torch.full_like(self.q, 7.0)
        plan.update(ids=self.tids, stream=stream)
        self.cache.attend(self.q, out, plan, lists=lists, scale=scale, stream=stream)
        return out

    def check(self, out, scale=None, chosen=None, more=0.0):
        """Each output within its bound, and `more`; chosen(i, g): (blocks of the sequence, attended slots of each) or None for all."""
        scale = 1 / math.sqrt(self.d) if scale is None else scale
        group, worst = self.H // self.KV, 0.0
        for i, t in enumerate(self.lens):
            for g in range(self.KV):
                h = slice(g * group, (g + 1) * group)
                take = chosen(i, g) if chosen else [(b, min(self.G, t - b * self.G)) for b in range(-(-t // self.G))]
                ref, wt, size = attend64(self.q[i, h], self.k[:, g], self.v[:, g],
                                         [self.rows[self.ids[i]][b] for b, _ in take], [m for _, m in take], scale)
                bound = attend_bound(ref, wt, size, self.d, out.dtype, self.cache.dtype) + more
                err = (out[i, h].double() - ref).abs()
                assert bool((err <= bound).all()), (i, g, t, float(err.max()), float((err / bound.clamp(min=1e-30)).max()))
                if bound.numel() and float(bound.max()) > 0:
                    worst = max(worst, float((err / bound.clamp(min=1e-30)).max()))
        print(f"worst error / bound {worst:.2f}")


EDGE_LENS = [0, 1, 2, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000]
# (head size, heads, kv heads, block tokens, cache, query, spread of the queries)
ATTEND = [(128, 32, 4, 16, BF, BF, 2.0), (128, 32, 4, 32, BF, F32, 2.0), (64, 16, 16, 16, HF, HF, 1.0),
          (64, 8, 2, 64, HF, F32, 4.0), (256, 8, 1, 64, BF, BF, 1.0), (256, 4, 2, 16, HF, F32, 1.0),
          (128, 6, 2, 128, HF, HF, 2.0), (128, 40, 2, 16, BF, F32, 1.0), (64, 17, 1, 32, BF, BF, 1.0),
          (256, 16, 1, 128, BF, F32, 1.0)]


@pytest.mark.parametrize("d,H,KV,G,cache,query,spread", ATTEND)
def test_attend_lengths(cuda, d, H, KV, G, cache, query, spread):
    """Lengths at the edges of tiles, blocks, units and waves in one batch, none and one among them; groups of 1 to
    20 heads (17 and 20 take two tiles of columns). Empty sequences give zeros."""
    b = Batch(cuda, EDGE_LENS, H, KV, d, G, cache, query, seed=d + H, spread=spread)
    out = b.attend()
    b.check(out)
    assert torch.count_nonzero(out[EDGE_LENS.index(0)]) == 0
    assert torch.equal(out, b.attend())  # the same bits every time


@pytest.mark.parametrize("d,H,KV,G,cache,query,lens", [
    (128, 32, 4, 16, BF, BF, [70001]), (64, 16, 16, 16, HF, HF, [5000, 1, 12345, 300]),
    (128, 8, 8, 32, HF, F32, [20000, 0, 33333]), (256, 8, 1, 64, BF, F32, [40007, 128]),
    (128, 8, 2, 128, BF, BF, [9999] * 5 + [40000])])
def test_attend_long(cuda, d, H, KV, G, cache, query, lens):
    """Sequences split into many items and joined."""
    b = Batch(cuda, lens, H, KV, d, G, cache, query, seed=3, spread=2.0)
    b.check(b.attend())


@pytest.mark.parametrize("d,H,KV,query", [(128, 32, 4, BF), (64, 16, 16, BF), (256, 32, 2, F32)])
def test_repeated_calls_join_their_own_partials(cuda, d, H, KV, query):
    """Two batches of queries in turn over one plan whose items the last workgroup joins: every call gives the first
    call's bits, not what an earlier call left in the plan's memory."""
    b = Batch(cuda, [1500, 1000, 0, 129, 257] if d < 256 else [900, 129, 0, 128, 257], H, KV, d, 16, BF, query, seed=20)
    plan = P.PagedPlan(b.table, b.cache, 5, H)
    plan.update(ids=b.tids)
    qs = [b.q, (b.q * 0.5).contiguous()]
    first = [torch.empty_like(b.q) for _ in qs]
    for q, o in zip(qs, first):
        b.cache.attend(q, o, plan)
    b.check(first[0])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = [torch.empty((40, *b.q.shape), dtype=query, device=cuda) for _ in qs]
    for i in range(40):
        for q, o in zip(qs, outs):
            b.cache.attend(q, o[i], plan, stream=stream)
    torch.cuda.synchronize()
    for o, f in zip(outs, first):
        assert bool((o == f).all())


def test_attend_many_short(cuda):
    lens = [random.Random(1).randint(0, 40) for _ in range(700)]
    b = Batch(cuda, lens, 4, 2, 64, 16, BF, BF, seed=4)
    b.check(b.attend())


@pytest.mark.parametrize("query", [BF, F32])
def test_attend_other_ids_scale_and_strides(cuda, query):
    """Ids outside the table are empty sequences, one named twice is read twice; rows of q and out with gaps; a scale."""
    b = Batch(cuda, [50, 333, 0, 1025], 8, 2, 128, 16, BF, query, seed=5)
    out = b.attend(scale=0.5)
    b.check(out, scale=0.5)
    plan = P.PagedPlan(b.table, b.cache, 6, 8)
    ids = ints([b.ids[3], -1, b.ids[0], b.ids[3], b.table.max_seqs, 2 ** 31 - 1], cuda)
    wide_q = torch.full((6, 3, 8, 128), 9.0, dtype=query, device=cuda)
    wide_o = wide_q.clone()
    wide_q[:, 1] = b.q[[3, 0, 0, 3, 1, 2]]
    plan.update(ids=ids)
    b.cache.attend(wide_q[:, 1], wide_o[:, 1], plan, scale=0.5)
    got = wide_o[:, 1]
    # another batch may be split otherwise: the same within twice the bound (checked against fp64 itself)
    b2 = Batch.__new__(Batch)
    b2.__dict__ = dict(b.__dict__, lens=[1025, 0, 50, 1025, 0, 0], ids=[b.ids[3], 0, b.ids[0], b.ids[3], 0, 0],
                       q=wide_q[:, 1].contiguous())
    b2.check(got.contiguous(), scale=0.5)
    assert torch.equal(got[0], got[3])
    assert torch.count_nonzero(got[[1, 4, 5]]) == 0
    assert bool((wide_o[:, 0] == 9).all()) and bool((wide_o[:, 2] == 9).all())


@pytest.mark.parametrize("cache,query", [(BF, BF), (BF, F32), (HF, HF), (HF, F32)])
def test_scores_of_minus_infinity(cuda, cache, query):
    """Keys that make scores of -inf have no weight, also where they fill tiles or a whole item; where every score is
    -inf the output is a NaN, as the softmax is."""
    b = Batch(cuda, [100, 400, 64, 3000], 8, 2, 64, 16, cache, query, seed=6)
    b.q[:, :, 0] = b.q[:, :, 0].abs() + 0.5
    for i, masked in ((0, 40), (1, 300), (2, 64), (3, 2900)):
        for t in range(masked):
            b.k[b.rows[b.ids[i]][t // 16], :, t % 16, 0] = -math.inf
    out = b.attend()
    assert bool(torch.isnan(out[2]).all())
    for i, masked in ((0, 40), (1, 300), (3, 2900)):
        t = b.lens[i]
        for g in range(2):
            rows = [(b.rows[b.ids[i]][x // 16], x % 16) for x in range(masked, t)]
            kk = torch.stack([b.k[p, g, o] for p, o in rows]).double()
            vv = torch.stack([b.v[p, g, :, o] for p, o in rows]).double()
            q = b.q[i, 4 * g:4 * g + 4].double()
            p = torch.softmax(q @ kk.t().contiguous() / 8.0, 1)
            size = float((q.abs() @ kk.abs().t().contiguous()).max()) / 8
            bound = attend_bound(p @ vv, p @ vv.abs(), size, 64, query, cache)
            assert bool(((out[i, 4 * g:4 * g + 4].double() - p @ vv).abs() <= bound).all()), (i, g)


@pytest.mark.parametrize("cache,query", [(BF, BF), (BF, F32), (HF, HF), (HF, F32)])
def test_infinite_values_and_nans(cuda, cache, query):
    """An attended infinity makes its dimension infinite, an attended NaN its output; nothing else changes."""
    b = Batch(cuda, [200, 77], 4, 2, 64, 16, cache, query, seed=7, spread=0.1)
    clean = b.attend()
    b.v[b.rows[b.ids[0]][2], 0, 5, 3] = math.inf
    b.v[b.rows[b.ids[0]][2], 1, 6, 3] = -math.inf
    b.k[b.rows[b.ids[1]][1], 1, 4, 9] = math.nan
    out = b.attend()
    assert bool((out[0, :2, 5] == math.inf).all()) and bool((out[0, 2:, 6] == -math.inf).all())
    assert bool(torch.isnan(out[1, 2:]).all())
    same = torch.ones_like(out, dtype=torch.bool)
    same[0, :2, 5] = same[0, 2:, 6] = False
    same[1, 2:] = False
    assert torch.equal(out[same], clean[same])


@pytest.mark.parametrize("magnitude", [1e-30, 1e-6, 1e4, 1e20])
def test_fp32_queries_of_any_size_over_fp16(cuda, magnitude):
    """fp32 queries far outside fp16's range, with the scale that makes their scores ordinary."""
    b = Batch(cuda, [300, 65], 8, 2, 128, 16, HF, F32, seed=8)
    b.q *= magnitude
    scale = 1 / (magnitude * math.sqrt(128))
    b.check(b.attend(scale=scale), scale=scale)


def test_small_keys_and_values_of_fp16(cuda):
    """Keys and values far below fp16's least normal value (2^-14) are not flushed, and their outputs are as near as if
    they were 2^-14: a subnormal's exponent field is that of 2^-14, the matrix cores align the 32 products of a
    sum (weights of up to 2^14 times 2^-14) by these fields and cut off what lies 24 bits below, 2^-24 for each of three parts
    and as much for the sum they are added to, 8 2^-24 with the sums' own rounding; the sum of the weights is at least 2^14."""
    b = Batch(cuda, [300, 65, 1], 8, 2, 128, 16, HF, F32, seed=18)
    b.k *= 2.0 ** -16
    b.v *= 2.0 ** -18
    b.q *= 2.0 ** 16
    for t in (b.k, b.v):  # the junk of unwritten slots may have become finite: it stays unread
        t[torch.isnan(t)] = math.inf
    b.check(b.attend(), more=8 * 2.0 ** -38)


@pytest.mark.parametrize("query", [BF, F32])
def test_output_over_the_queries(cuda, query):
    """out may be q itself."""
    b = Batch(cuda, [3000, 0, 1, 700], 8, 2, 128, 16, BF, query, seed=19)
    want = b.attend()
    plan = P.PagedPlan(b.table, b.cache, 4, 8)
    plan.update(ids=b.tids)
    b.cache.attend(b.q, b.q, plan)
    assert torch.equal(b.q, want)


def test_bad_table_entries_are_skipped(cuda):
    """Entries outside the pool hold no tokens; with none left the output is zeros."""
    b = Batch(cuda, [100, 40, 16], 8, 2, 64, 16, BF, BF, seed=9)
    t = b.table.blocks
    t[b.ids[0], 1], t[b.ids[0], 3] = b.cache.n_blocks, -7
    t[b.ids[1], 0], t[b.ids[1], 2] = -2 ** 31, 2 ** 31 - 1
    t[b.ids[2], 0] = -1
    out = b.attend()

    def chosen(i, g):
        bad = {0: (1, 3), 1: (0, 2), 2: (0,)}[i]
        return [(x, min(16, b.lens[i] - 16 * x)) for x in range(-(-b.lens[i] // 16)) if x not in bad]

    b.check(out, chosen=chosen)
    assert torch.count_nonzero(out[2]) == 0


def test_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 elements, its blocks read and written at the far end."""
    G, KV, d, H = 16, 8, 128, 16
    n_blocks = 2 ** 32 // (G * KV * d) + 40
    k = torch.empty((n_blocks, KV, G, d), dtype=BF, device=cuda)
    v = torch.empty((n_blocks, KV, d, G), dtype=BF, device=cuda)
    m = torch.empty((n_blocks, KV, d), dtype=BF, device=cuda)
    t = P.PagedTable.create(2, 30, n_blocks, G, device=cuda)
    t.free_blocks.copy_(torch.arange(n_blocks, dtype=torch.int32, device=cuda))  # the far end on top
    cache = P.PagedCache(k, v, m)
    bufs = step_buffers(2, 400, cuda)
    t.extend(ints([200, 130], cuda), *bufs)
    assert bool((bufs[2][:330] >= (n_blocks - 30) * G).all())
    x = randn((400, H + 2 * KV, d), BF, cuda, 1)
    q_out = torch.empty((400, H, d), dtype=BF, device=cuda)
    cache.append(x[:, :H], x[:, H:H + KV], x[:, H + KV:], bufs[1], bufs[2], q_out)
    plan = P.PagedPlan(t, cache, 2, H)
    plan.update()
    out = torch.empty((2, H, d), dtype=BF, device=cuda)
    last = torch.tensor([199, 329], device=cuda)
    cache.attend(q_out[last], out, plan)
    for i, rows in ((0, slice(0, 200)), (1, slice(200, 330))):
        for g in range(KV):
            kk, vv = x[rows, H + g].double(), x[rows, H + KV + g].double()
            q = x[int(last[i]), 2 * g:2 * g + 2].double()
            p = torch.softmax(q @ kk.t().contiguous() / math.sqrt(d), 1)
            size = float((q.abs() @ kk.abs().t().contiguous()).max()) / math.sqrt(d)
            bound = attend_bound(p @ vv, p @ vv.abs(), size, d, BF, BF)
            assert bool(((out[i, 2 * g:2 * g + 2].double() - p @ vv).abs() <= bound).all()), (i, g)
    b = bufs[2][15].item() // G
    want = x[0:16, H:H + KV].double().mean(0)
    assert bool(((m[b].double() - want).abs() <= half_step(BF) * want.abs() + 2.0 ** -19).all())


# ---- lists ----------------------------------------------------------------------------------------------------------

def test_lists_of_blocks(cuda):
    """A caller's own lists: any blocks in any order, the sequence's last one among them, entries outside the sequence."""
    b = Batch(cuda, [300, 33, 1000, 0, 5], 8, 2, 64, 16, BF, F32, seed=10)
    lists = [[[18, 0, 5, 7], [3, 18, -1, 2]], [[0, 2, 1, -1], [2, 40, -9, 1]], [[62, 61, 0, 9], [1, 2, 3, 4]],
             [[0, 1, 2, 3], [-1, -1, -1, -1]], [[0, -1, -1, -1], [7, -1, -1, -1]]]
    out = b.attend(lists=ints(lists, cuda), width=4)

    def chosen(i, g):
        nb = -(-b.lens[i] // 16)
        take = lists[i][g][:min(nb, 4)]
        return [(x, max(min(16, b.lens[i] - 16 * x), 0)) for x in take if 0 <= x < nb]

    b.check(out, chosen=chosen)
    assert torch.count_nonzero(out[3]) == 0 and torch.count_nonzero(out[4, 4:]) == 0


def choose64(q, means, have, sinks, window, width):
    """One sequence and kv head: q [heads, d], its blocks' means."""
    if have <= width:
        return list(range(have)) + [-1] * (width - have)
    s = (q.double() @ means[sinks:have - window].double().t().contiguous())
    s = torch.where(torch.isnan(s), -math.inf, s).amax(0).float()
    best = torch.sort(s, descending=True, stable=True).indices[:width - sinks - window].tolist()
    return list(range(sinks)) + sorted(x + sinks for x in best) + list(range(have - window, have))


# (head size, heads, kv heads, block tokens, cache, query, sinks, window, budget, lengths)
SELECT = [(128, 32, 4, 16, BF, BF, 1, 4, 32, [30001, 700, 590, 593, 0, 1]), (64, 8, 2, 16, HF, F32, 0, 1, 5, [3000, 97, 96, 111]),
          (256, 8, 1, 64, BF, F32, 2, 2, 16, [20011, 1281, 1280]), (128, 20, 1, 32, HF, HF, 0, 3, 0, [5000, 64]),
          (64, 34, 2, 128, BF, BF, 3, 1, 9, [20000, 300]), (128, 4, 4, 16, BF, F32, 1, 2, 300, [70000, 5000]),
          (64, 2, 1, 16, BF, BF, 1, 1, 40, [150000, 8200 * 16])]


@pytest.mark.parametrize("d,H,KV,G,cache,query,sinks,window,budget,lens", SELECT)
def test_select(cuda, d, H, KV, G, cache, query, sinks, window, budget, lens):
    """The chosen blocks entry for entry, then the attention over them. Every fourth mean key equals its neighbour (equal scores:
    the lower block first); the means of blocks that are not full are NaN (never read)."""
    b = Batch(cuda, lens, H, KV, d, G, cache, query, seed=11)
    means = randn((b.cache.n_blocks, KV, d), cache, cuda, 12)
    for i, t in enumerate(lens):
        row = b.rows[b.ids[i]]
        for x in range(0, t // G - 1, 4):
            means[row[x + 1]] = means[row[x]]
        if t % G:
            means[row[t // G]] = math.nan
    cache_m = P.PagedCache(b.k, b.v, means)
    width = sinks + window + budget
    plan = P.PagedPlan(b.table, cache_m, len(lens), H, width)
    lists = torch.full((len(lens), KV, width), 99, dtype=torch.int32, device=cuda)
    plan.update(ids=b.tids)
    cache_m.select(b.q, plan, lists, sinks=sinks, window=window)
    group = H // KV
    for i, t in enumerate(lens):
        have = -(-t // G)
        pages = torch.tensor(b.rows[b.ids[i]][:have], dtype=torch.long, device=cuda)
        for g in range(KV):
            want = choose64(b.q[i, g * group:(g + 1) * group], means[pages, g], have, sinks, window, width)
            assert lists[i, g].tolist() == want, (i, g)
    out = torch.empty_like(b.q)
    cache_m.attend(b.q, out, plan, lists=lists)
    b.check(out, chosen=lambda i, g: [(x, min(G, b.lens[i] - x * G)) for x in lists[i, g].tolist() if x >= 0])


def test_select_with_nan_and_equal_scores(cuda):
    """Scores that are NaN count as -inf; where all are equal the lowest blocks are taken; -0 equals 0."""
    b = Batch(cuda, [16 * 40], 2, 1, 64, 16, BF, F32, seed=13)
    row = b.rows[b.ids[0]]
    means = torch.zeros((b.cache.n_blocks, 1, 64), dtype=BF, device=cuda)
    means[row[9]] = math.nan
    means[row[20]] = -0.0
    means[row[30], 0, 0] = 1.0
    c = P.PagedCache(b.k, b.v, means)
    plan = P.PagedPlan(b.table, c, 1, 2, 12)
    b.q[:] = 1.0
    lists = torch.zeros((1, 1, 12), dtype=torch.int32, device=cuda)
    plan.update(ids=b.tids)
    c.select(b.q, plan, lists, sinks=1, window=1)
    assert lists[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 8, 10, 30, 39]
    means[row[9]] = 0.0
    b.q[0, 0] = math.nan  # one head's scores: the other's stand
    c.select(b.q, plan, lists, sinks=1, window=1)
    assert lists[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 30, 39]
    b.q[:] = math.nan
    c.select(b.q, plan, lists, sinks=1, window=1)
    assert lists[0, 0].tolist() == list(range(11)) + [39]


@pytest.mark.parametrize("blocks,levels,big", [(300, 1, 1.0), (300, 3, 1.0), (1500, 2, 1e30), (5000, 7, 1.0), (300, 2, math.inf)])
def test_select_many_equal_scores(cuda, blocks, levels, big):
    """Scores of few different values, infinite ones among them: the lower blocks of the last value that fits."""
    b = Batch(cuda, [16 * blocks - 3], 2, 1, 64, 16, BF, F32, seed=blocks)
    pages = torch.tensor(b.rows[b.ids[0]][:blocks], device=cuda)
    means = torch.zeros((b.cache.n_blocks, 1, 64), dtype=BF, device=cuda)
    value = torch.randint(levels, (blocks,), generator=gen(cuda, 1), device=cuda).float() - 1
    means[pages, 0, 7] = torch.where(value == 0, 0.0, value * big).to(BF)
    b.q[:] = 0.0
    b.q[:, :, 7] = 3.0
    c = P.PagedCache(b.k, b.v, means)
    for budget in (1, blocks // 3, blocks - 5):
        plan = P.PagedPlan(b.table, c, 1, 2, budget + 3)
        lists = torch.zeros((1, 1, budget + 3), dtype=torch.int32, device=cuda)
        plan.update(ids=b.tids)
        c.select(b.q, plan, lists, sinks=1, window=2)
        scores = means[pages[1:-2], 0, 7].float() * 3
        want = torch.sort(torch.sort(scores, descending=True, stable=True).indices[:budget]).values + 1
        assert lists[0, 0].tolist() == [0] + want.tolist() + [blocks - 2, blocks - 1]


def test_lists_of_every_block_give_the_same_bits(cuda):
    """Selected lists that hold every block: the dense result bit for bit."""
    b = Batch(cuda, [500, 33, 0, 77], 8, 2, 128, 16, BF, BF, seed=14)
    dense = b.attend()
    c = P.PagedCache(b.k, b.v, torch.zeros((b.cache.n_blocks, 2, 128), dtype=BF, device=cuda))
    plan = P.PagedPlan(b.table, c, 4, 8, 40)
    lists = torch.zeros((4, 2, 40), dtype=torch.int32, device=cuda)
    plan.update(ids=b.tids)
    c.select(b.q, plan, lists, sinks=0, window=1)
    out = torch.empty_like(dense)
    c.attend(b.q, out, plan, lists=lists)
    assert torch.equal(out, dense)


# ---- together -------------------------------------------------------------------------------------------------------

class Server:
    """Prompts of three sequences, then steps of a token each, drafts taken back in between, one sequence ending and
    another starting in its place; the whole past of each sequence kept in fp64 beside it."""

    def __init__(self, dev, list_blocks=0):
        self.dev, self.H, self.KV, self.d, self.G = dev, 8, 2, 64, 16
        self.t = P.PagedTable.create(4, 24, 60, self.G, device=dev)
        self.cache = P.PagedCache.create(self.t, self.KV, self.d, BF, means=True)
        self.rope = rope_table(self.d, 512, dev)
        self.norm = 1 + 0.1 * randn(self.d, F32, dev, 99)
        self.max_rows = 256
        self.bufs = step_buffers(3, self.max_rows, dev)
        self.x = torch.zeros((self.max_rows, self.H + 2 * self.KV, self.d), dtype=BF, device=dev)
        self.q = torch.zeros((self.max_rows, self.H, self.d), dtype=F32, device=dev)
        self.plan = P.PagedPlan(self.t, self.cache, 3, self.H, list_blocks)
        self.lists = torch.zeros((3, self.KV, list_blocks), dtype=torch.int32, device=dev) if list_blocks else None
        self.last = torch.zeros((3, self.H, self.d), dtype=F32, device=dev)
        self.out = torch.zeros((3, self.H, self.d), dtype=F32, device=dev)
        self.ids, self.n_new = ints([0, 1, 2], dev), ints([1, 1, 1], dev)

    def step(self, stream=None):
        """The whole step from device memory: the same launches whatever the lengths."""
        self.t.extend(self.n_new, *self.bufs, ids=self.ids, stream=stream)
        x = self.x
        self.cache.append(x[:, :self.H], x[:, self.H:self.H + self.KV], x[:, self.H + self.KV:], self.bufs[1], self.bufs[2],
                          self.q, self.rope, q_norm=self.norm, k_norm=self.norm, stream=stream)
        with torch.cuda.stream(stream or torch.cuda.current_stream(self.dev)):
            # each sequence's last row (a sequence without new rows: some row)
            torch.index_select(self.q, 0, (self.bufs[0][1:] - 1).clamp(min=0).long(), out=self.last)
        self.plan.update(ids=self.ids, stream=stream)
        if self.lists is not None:
            self.cache.select(self.last, self.plan, self.lists, sinks=1, window=2, stream=stream)
        self.cache.attend(self.last, self.out, self.plan, lists=self.lists, stream=stream)


def serve(cuda, list_blocks, graph):
    s = Server(cuda, list_blocks)
    H, KV, d, G = s.H, s.KV, s.d, s.G
    past = {0: [], 1: [], 2: [], 3: []}  # raw rows of each table row's sequence
    plan = [([0, 1, 2], [50, 1, 120])] + [([0, 1, 2], [1, 1, 1])] * 20 + [([2, 0, 3], [3, 1, 70])] + \
        [([3, 2, 0], [1, 2, 1])] * 18
    g = None
    if graph:
        side = torch.cuda.Stream()
        s.n_new.zero_()
        side.wait_stream(torch.cuda.current_stream())
        s.step(stream=side)  # once uncaptured
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            s.step(stream=side)
        s.t.reset()
    for n, (ids, new) in enumerate(plan):
        if n == 21:  # sequence 1 ends, 2 takes its last five tokens back
            s.t.truncate(ints([0, 10 ** 6, len(past[2]) - 5], cuda), ids=ints([1, 0, 2], cuda))
            past[1], past[2] = [], past[2][:-5]
        T = sum(new)
        s.x.normal_(generator=gen(cuda, 1000 + n))
        at = 0
        for i, k in zip(ids, new):
            past[i] = past[i] + [s.x[at + j].clone() for j in range(k)]
            at += k
        s.ids.copy_(ints(ids, cuda))
        s.n_new.copy_(ints(new, cuda))
        if g:
            g.replay()
        else:
            s.step()
        torch.cuda.synchronize()
        assert s.bufs[3].tolist() == [0, 0, 0] and s.bufs[0].tolist()[-1] == T
        assert [s.t.len[i].item() for i in ids] == [len(past[i]) for i in ids]
        if n % 5 and n < 36:
            continue
        for b, i in enumerate(ids):
            rows = torch.stack(past[i])
            pos = torch.arange(len(past[i]), device=cuda)
            q64 = heads64(rows[-1:, :H], None, s.norm, 1e-6, s.rope, pos[-1:])[0]
            k64 = heads64(rows[:, H:H + KV], None, s.norm, 1e-6, s.rope, pos).to(BF).double()
            v64 = rows[:, H + KV:].double()
            for kv in range(KV):
                keep = torch.ones(len(past[i]), dtype=torch.bool, device=cuda)
                if list_blocks:
                    keep[:] = False
                    for x in s.lists[b, kv].tolist():
                        if x >= 0:
                            keep[x * G:(x + 1) * G] = True
                q, kk, vv = q64[4 * kv:4 * kv + 4], k64[keep, kv], v64[keep, kv]
                p = torch.softmax(q @ kk.t().contiguous() / 8, 1)
                size = float((q.abs() @ kk.abs().t().contiguous()).max()) / 8
                # a key next to the border of two bf16 values may be stored as the other one, one step (2^-7 of it at
                # most) off: where fp32's error of 2^-19 of the row's largest value reaches the border, few do; an
                # output then moves by the weight's change, at most 2^-7 of one term's share of the score
                bound = attend_bound(p @ vv, p @ vv.abs(), size, d, F32, BF) + (p @ vv.abs()) * 2.0 ** -7 * size / d * 8
                assert bool(((s.out[b, 4 * kv:4 * kv + 4].double() - p @ vv).abs() <= bound).all()), (n, b, kv)
    return s.out.clone()


@pytest.mark.parametrize("list_blocks", [0, 7])
def test_serving_steps(cuda, list_blocks):
    """Prompts, single tokens, tokens taken back, a sequence that ends and one that starts: eager calls and a captured
    graph of the whole step replayed for every one of them, checked on the way and equal at the end."""
    eager = serve(cuda, list_blocks, False)
    assert torch.equal(serve(cuda, list_blocks, True), eager)


def test_other_stream_and_two_plans(cuda):
    """Two plans on two streams at once give what one after the other gives."""
    b = Batch(cuda, [3000, 10, 777], 8, 2, 128, 16, BF, BF, seed=15)
    want = b.attend()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    plans = [P.PagedPlan(b.table, b.cache, 3, 8) for _ in range(2)]
    outs = [torch.zeros_like(b.q) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, p, o in zip((s1, s2), plans, outs):
            p.update(ids=b.tids, stream=s)
            b.cache.attend(b.q, o, p, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_a_plan_never_updated_writes_nothing(cuda):
    b = Batch(cuda, [30], 4, 2, 64, 16, BF, BF, seed=16)
    plan = P.PagedPlan(b.table, b.cache, 1, 4)
    out = torch.full_like(b.q, 7.0)
    b.cache.attend(b.q, out, plan)
    assert bool((out == 7).all())


def test_python_refusals(cuda):
    b = Batch(cuda, [30], 4, 2, 64, 16, BF, BF, seed=17)
    plan = P.PagedPlan(b.table, b.cache, 1, 4)
    plan.update(ids=b.tids)
    out = torch.empty_like(b.q)
    with pytest.raises(ValueError):
        b.cache.attend(b.q[:, :3], out, plan)
    with pytest.raises(ValueError):
        b.cache.attend(b.q.transpose(1, 2).contiguous().transpose(1, 2), out, plan)
    with pytest.raises(ValueError):
        b.cache.attend(b.q, out.float(), plan)
    with pytest.raises(ValueError):
        b.cache.attend(b.q.cpu(), out, plan)
    with pytest.raises(_lib.VireoError):
        b.cache.attend(b.q.half(), out.half(), plan)  # neither fp32 nor the cache's type
    with pytest.raises(_lib.VireoError):
        b.cache.attend(b.q, out, plan, scale=0.0)
    with pytest.raises(ValueError):
        b.cache.attend(b.q, out, plan, lists=torch.zeros((1, 2, 0), dtype=torch.int32, device=cuda))
    with pytest.raises(_lib.VireoError):
        b.cache.select(b.q, plan, torch.zeros((1, 2, 0), dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError):
        plan.update(ids=b.tids.long())
    with pytest.raises(ValueError):
        b.table.extend(None, *step_buffers(1, 4, cuda), ids=ints([0, 1], cuda))
    with pytest.raises(_lib.VireoError):
        b.table.extend(None, *step_buffers(9, 4, cuda))  # more sequences than the table has
    with pytest.raises(ValueError):
        P.PagedCache(b.k, b.v.transpose(2, 3).contiguous())
    with pytest.raises(_lib.VireoError):
        P.PagedPlan(b.table, b.cache, 1, 5)  # heads do not divide
    x = torch.zeros((2, 8 * 64 + 4), dtype=BF, device=cuda)[:, 4:].unflatten(1, (8, 64))  # rows 8 bytes off
    pos = ints([0, 0], cuda)
    with pytest.raises(_lib.VireoError):
        b.cache.append(x[:, :4], x[:, 4:6], x[:, 6:], pos, pos, torch.empty((2, 4, 64), dtype=BF, device=cuda))
