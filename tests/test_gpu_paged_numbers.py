"""The paged cache's attention at the corners of its arithmetic (include/vireo_paged.h), against fp64 with bounds
derived from the roundings that are left."""
import math

import pytest
import torch

from paged_ref import attend64, half_step
from test_gpu_paged import BF, F32, HF, Batch, ints, randn
from vireo_amd import paged as P

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of fp32


def working(weight64, size, d):
    """What fp32 arithmetic before the result's one rounding may be off by (paged_ref.attend_bound without its
    cut-off weights): 32 + 3 d / 32 half steps of a score into the weights and their sum, 16 for the rest."""
    return weight64 * (2 * U * ((32 + 3 * d // 32) * size + 16))


def check_rounded_once(b, out, scale=None, more=0.0):
    """Every output is the nearest value of its type to some value within working() of the fp64 result."""
    scale = 1 / math.sqrt(b.d) if scale is None else scale
    group = b.H // b.KV
    for i, t in enumerate(b.lens):
        for g in range(b.KV):
            h = slice(g * group, (g + 1) * group)
            pages = b.rows[b.ids[i]][:-(-t // b.G)]
            ref, wt, size = attend64(b.q[i, h], b.k[:, g], b.v[:, g], pages,
                                     [min(b.G, t - x * b.G) for x in range(len(pages))], scale)
            tol = working(wt, size, b.d) + more
            # rounding to nearest does not change an order
            lo, hi = (ref - tol).to(out.dtype), (ref + tol).to(out.dtype)
            bad = ~((out[i, h] >= lo) & (out[i, h] <= hi))
            assert not bool(bad.any()), (i, g, t, int(bad.sum()), float((out[i, h].double() - ref).abs().max()))


@pytest.mark.parametrize("d,H,KV,G,cache", [(128, 32, 4, 16, BF), (64, 16, 16, 32, BF), (256, 8, 2, 64, BF),
                                            (128, 32, 4, 16, HF), (256, 8, 2, 16, HF)])
def test_results_in_16_bits_are_rounded_once(cuda, d, H, KV, G, cache):
    """Weights in full: values of one sign, a level of its own for every dimension, so that a bias of the weights (of
    2^-17 of them, if 16 bits were kept) would take results past the borders of their type's values."""
    lens = [1000, 900, 1, 127, 640, 77, 512, 333]
    b = Batch(cuda, lens, H, KV, d, G, cache, cache, seed=31, spread=0.02)
    level = 1 + torch.arange(d, device=cuda) / d
    live = torch.isfinite(b.v) & (b.v.abs() < 100)  # the junk of unwritten slots stays
    b.v.copy_(torch.where(live, (level[:, None] + 0.2 * b.v.float()).to(cache), b.v))
    check_rounded_once(b, b.attend())


@pytest.mark.parametrize("scale,magnitude", [(1e-30, 1e-12), (1 / math.sqrt(128), 4e-41), (1 / math.sqrt(128), 1e-42),
                                             (1e-45, 1.0), (3e38, 1e-39), (3e38, 1e-44), (1e-38, 1e37), (1e-42, 1e37)])
def test_scales_and_fp32_queries_of_any_size_over_fp16(cuda, scale, magnitude):
    """Scale and queries each anywhere in fp32's range, their scores ordinary or as good as 0 (then every weight is the
    same); lengths that fill their last tile and lengths that do not."""
    b = Batch(cuda, [300, 65, 1000, 31, 128], 8, 2, 128, 16, HF, F32, seed=33)
    b.q *= magnitude
    scale = float(torch.tensor(scale, dtype=F32))
    b.check(b.attend(scale=scale), scale=scale)


@pytest.mark.parametrize("cache,query,big,step", [(BF, BF, 2.0 ** 40, 1.0), (BF, BF, 2.0 ** 100, 1.0), (BF, F32, 1.7e30, 1.0),
                                                  (HF, HF, 60000.0, 1024.0), (HF, F32, 1.7e10, 1.0), (HF, F32, 3e33, 16.0)])
def test_scores_of_any_size(cuda, cache, query, big, step):
    """Scores so large that only the largest has a weight: queries of one dimension and keys of few bits there, so that
    every sum is exact and the largest, at two tokens of each sequence, far above the next. The result is the mean of their
    values (weights of 1 and 0)."""
    b = Batch(cuda, [300, 65, 3000, 31, 128], 8, 2, 128, 16, cache, query, seed=34)
    b.q.zero_()
    b.q[:, :, 5] = big
    live = torch.isfinite(b.k) & (b.k.abs() < 100)
    b.k.copy_(torch.where(live, torch.round(b.k * 4) * step, b.k))
    tops = [(t // 3, t - 2) for t in b.lens]
    for i, ts in enumerate(tops):
        for t in ts:
            b.k[b.rows[b.ids[i]][t // 16], :, t % 16, 5] = 27 * step
    out = b.attend()
    for i, ts in enumerate(tops):
        at = [(b.rows[b.ids[i]][t // 16], t % 16) for t in ts]
        for g in range(2):
            vv = torch.stack([b.v[p, g, :, o] for p, o in at]).double()
            want, tol = vv.mean(0), working(vv.abs().mean(0), 0.0, 128)
            err = (out[i, 4 * g:4 * g + 4].double() - want).abs()
            assert bool((err <= half_step(query) * want.abs() + tol).all()), (i, g, float(err.max()))


@pytest.mark.parametrize("query", [HF, F32])
def test_tokens_without_weight_add_nothing(cuda, query):
    """One token's weight is e^44 times every other's, whose values are 60 000 times its own: 32 767 of them add
    10^-10 to a result of 1. 256 sequences that are the same, so that each is one workgroup's and the others follow the one
    in its wave."""
    G, n, t, d = 16, 256, 32768, 64
    k, v = torch.zeros((t // G, 1, G, d), dtype=HF, device=cuda), torch.full((t // G, 1, d, G), 60000.0, dtype=HF, device=cuda)
    k[0, 0, 0, 0], v[0, 0, :, 0] = 44.0, 1.0
    table = P.PagedTable(torch.arange(t // G, dtype=torch.int32, device=cuda)[None].contiguous(), ints([t], cuda),
                         torch.zeros(t // G, dtype=torch.int32, device=cuda), ints([0], cuda), G)
    cache = P.PagedCache(k, v)
    plan = P.PagedPlan(table, cache, n, 1)
    plan.update(ids=torch.zeros(n, dtype=torch.int32, device=cuda))
    q = torch.zeros((n, 1, d), dtype=query, device=cuda)
    q[:, :, 0] = 1.0
    out = torch.empty_like(q)
    cache.attend(q, out, plan, scale=1.0)
    want = 1 + 32767 * math.exp(-44) * 60000
    err = (out.double() - want).abs().max()
    assert float(err) <= half_step(query) + float(working(torch.tensor(1.0), 44.0, d)), float(err)


@pytest.mark.parametrize("query", [BF, F32])
def test_large_values_under_a_weight_of_zero(cuda, query):
    """Values of 3 10^38 where the key makes a score of -inf add nothing."""
    b = Batch(cuda, [40, 200], 4, 2, 64, 16, BF, query, seed=35)
    b.q[:, :, 0] = b.q[:, :, 0].abs() + 0.5
    clean = [b.k.clone(), b.v.clone()]
    for i, first in ((0, 3), (1, 150)):
        for x in range(first, b.lens[i]):
            p, o = b.rows[b.ids[i]][x // 16], x % 16
            b.k[p, :, o, 0], b.v[p, :, :, o] = -math.inf, 3e38
    out = b.attend()
    b.k, b.v, b.lens = *clean, [3, 150]
    b.check(out)


@pytest.mark.parametrize("cache,query", [(BF, BF), (BF, F32), (HF, HF), (HF, F32)])
@pytest.mark.parametrize("gap,d,G", [(0.0, 64, 16), (5.0, 128, 64), (20.0, 256, 16), (44.0, 64, 128), (44.0, 128, 16),
                                     (80.0, 64, 16), (80.0, 256, 64)])
def test_infinite_values_under_any_weight(cuda, cache, query, gap, d, G):
    """A token's infinite value makes its dimension infinite under every weight that fp32 holds, e^-80 of the largest
    too, in tiles before and after the largest; one of each sign, or a NaN, makes it a NaN; other dimensions keep their bits."""
    b = Batch(cuda, [200, 2000, 33], 4, 2, d, G, cache, query, seed=36)
    live = torch.isfinite(b.k) & (b.k.abs() < 100)
    b.k.copy_(torch.where(live, torch.zeros_like(b.k), b.k))
    b.q.fill_(1.0)
    spots = [[3, 150, 77], [40, 1990, 1033], [2, 32, 17]]
    for i, ts in enumerate(spots):
        for t in ts:
            b.k[b.rows[b.ids[i]][t // G], :, t % G, 1] = -gap
    clean = b.attend(scale=1.0)
    b.check(clean, scale=1.0)
    want = clean.clone()
    for i, ts in enumerate(spots):
        for t, dim, value in zip(ts + ts, (5, 6, 7, 8, 8, 9), (math.inf, -math.inf, math.nan, math.inf, -math.inf, -math.inf)):
            b.v[b.rows[b.ids[i]][t // G], 1, dim, t % G] = value
        want[i, 2:, 5], want[i, 2:, 6], want[i, 2:, 9] = math.inf, -math.inf, -math.inf
        want[i, 2:, 7] = want[i, 2:, 8] = math.nan
    out = b.attend(scale=1.0)
    assert bool(((out == want) | (torch.isnan(out) & torch.isnan(want))).all())


@pytest.mark.parametrize("cache", [BF, HF])
def test_zero_elements_of_fp32_queries(cuda, cache):
    """Where a query's element is 0 the key's does not count, however large: the scores are 0, the weights equal."""
    b = Batch(cuda, [300, 65, 1000], 8, 2, 128, 16, cache, F32, seed=37)
    live = torch.isfinite(b.k) & (b.k.abs() < 100)
    large = torch.where(b.k > 0, 6e4, -6e4) if cache is HF else torch.where(b.k > 0, 3e38, -3e38)
    large[..., 0] = 0.0
    b.k.copy_(torch.where(live, large.to(cache), b.k))
    b.q.zero_()
    b.q[:, :, 0] = 1e4
    b.check(b.attend())


@pytest.mark.parametrize("magnitude,scale", [(1e-30, 1e30), (1e-35, 1e35), (1e-37, 1e37), (1e-38, 1e38), (1e-41, 3e38), (1e30, 1e-30)])
def test_fp32_queries_of_any_size_over_bf16(cuda, magnitude, scale):
    """Parts of a small query are not lost below bf16's least normal value (2^-126)."""
    b = Batch(cuda, [300, 65, 1000], 8, 2, 128, 16, BF, F32, seed=38)
    b.q *= magnitude
    scale = float(torch.tensor(scale / math.sqrt(128), dtype=F32))
    b.check(b.attend(scale=scale), scale=scale)


@pytest.mark.parametrize("cache,small", [(BF, 1e-30), (BF, 1e-40), (HF, 1e-4), (HF, 1e-20), (HF, 1e-40)])
def test_infinite_keys_of_any_element(cuda, cache, small):
    """A key of -inf makes a score of -inf with a query's element however small, its largest being about 1."""
    b = Batch(cuda, [100, 400], 8, 2, 64, 16, cache, F32, seed=39)
    b.q[:, :, 9] = small
    clean = [b.k.clone(), b.v.clone()]
    for i, first in ((0, 60), (1, 300)):
        for x in range(first, b.lens[i]):
            b.k[b.rows[b.ids[i]][x // 16], :, x % 16, 9] = -math.inf
    out = b.attend()
    b.k, b.v, b.lens = *clean, [60, 300]
    b.check(out)


# ---- the largest sizes ----------------------------------------------------------------------------------------------

def test_plan_of_more_units_than_a_sum_holds(cuda):
    """4 096 times one sequence of 2^31 - 32 tokens: 2^36 units of 128, past the 31 bits of the plan's sums. No more
    items than the plan's memory holds (2 048 and one more per sequence), and each sequence has one."""
    G, n = 16, 4096
    width = 2 ** 27 - 2
    table = P.PagedTable(torch.zeros((1, width), dtype=torch.int32, device=cuda), ints([width * G], cuda),
                         torch.zeros(8, dtype=torch.int32, device=cuda), ints([0], cuda), G)
    cache = P.PagedCache(*(torch.zeros(s, dtype=BF, device=cuda) for s in ((8, 1, G, 64), (8, 1, 64, G))))
    plan = P.PagedPlan(table, cache, n, 1)
    plan.update(ids=torch.zeros(n, dtype=torch.int32, device=cuda))
    items = plan.mem[:8].view(torch.int32)[1].item()  # the split begins with its tag and its number of items
    assert n <= items <= 2048 + n


def test_a_step_with_room_for_every_row(cuda):
    """Row buffers of 2^31 - 1 rows: the last ones are written too."""
    rows = 2 ** 31 - 1
    t = P.PagedTable.create(2, 4, 8, 16, device=cuda)
    positions, slots = (torch.full((rows,), 77, dtype=torch.int32, device=cuda) for _ in range(2))
    start, status = ints([7, 7, 7], cuda), ints([7, 7], cuda)
    t.extend(ints([3, 20], cuda), start, positions, slots, status)
    assert start.tolist() == [0, 3, 23] and status.tolist() == [0, 0]
    assert positions[:24].tolist() == [0, 1, 2, *range(20), 0]
    assert slots[:23].tolist() == [0, 1, 2, *range(16, 36)]
    for at in range(23, rows, 2 ** 28):
        assert bool((positions[at:at + 2 ** 28] == 0).all()) and bool((slots[at:at + 2 ** 28] == -1).all())


def test_the_most_sequences_and_heads(cuda):
    """4 096 sequences of 4 096 heads, all empty but the last, which is split and joined by the second launch."""
    n, H, d, G, t = 4096, 4096, 64, 16, 5000
    nb = -(-t // G)
    blocks = torch.zeros((n, nb), dtype=torch.int32, device=cuda)
    blocks[n - 1] = torch.arange(nb, dtype=torch.int32, device=cuda)
    length = torch.zeros(n, dtype=torch.int32, device=cuda)
    length[n - 1] = t
    table = P.PagedTable(blocks, length, torch.zeros(nb, dtype=torch.int32, device=cuda), ints([0], cuda), G)
    k, v = randn((nb, 1, G, d), BF, cuda, 41), randn((nb, 1, d, G), BF, cuda, 42)
    cache = P.PagedCache(k, v)
    plan = P.PagedPlan(table, cache, n, H)
    plan.update()
    q = torch.zeros((n, H, d), dtype=BF, device=cuda)
    q[n - 1] = randn((H, d), BF, cuda, 43)
    out = torch.full_like(q, 7.0)
    cache.attend(q, out, plan)
    assert not bool(out[:n - 1].any())
    ref, weight, size = attend64(q[n - 1], k[:, 0], v[:, 0], list(range(nb)), [min(G, t - x * G) for x in range(nb)], 0.125)
    err = (out[n - 1].double() - ref).abs()
    assert bool((err <= half_step(BF) * ref.abs() + working(weight, size, d)).all())


@pytest.mark.parametrize("H,KV,cache,query", [(1, 1, BF, F32), (2, 2, HF, HF), (4, 1, BF, BF), (6, 2, HF, F32)])
def test_joins_of_more_items_than_one_go_of_wide_heads(cuda, H, KV, cache, query):
    """Up to 32 items of heads of 256, of which the last workgroup takes 16 at a time; alone and beside others."""
    for lens in ([4096], [4000, 0, 1, 3001]):
        b = Batch(cuda, lens, H, KV, 256, 64, cache, query, seed=44, spread=2.0)
        b.table = P.PagedTable(b.table.blocks[:, :64].contiguous(), b.table.len, b.table.free_blocks, b.table.n_free, 64)
        out = b.attend()
        b.check(out)
        assert torch.equal(out, b.attend())


@pytest.mark.parametrize("G", [16, 128])
@pytest.mark.parametrize("value", [3e38, 1e-39, -2.5e38])
def test_means_of_the_largest_and_smallest_keys(cuda, G, value):
    """A block's mean key where the sum of its keys is beyond fp32, and where keys are subnormal: equal keys' mean is the key."""
    k, v = (torch.zeros(s, dtype=BF, device=cuda) for s in ((2, 1, G, 64), (2, 1, 64, G)))
    means = torch.zeros((2, 1, 64), dtype=BF, device=cuda)
    x = torch.full((G, 3, 64), value, dtype=BF, device=cuda)
    rows = torch.arange(G, dtype=torch.int32, device=cuda)
    P.PagedCache(k, v, means).append(x[:, :1], x[:, 1:2], x[:, 2:], rows, rows + G, torch.zeros_like(x[:, :1]))
    assert bool((k[1] == x[0, 0, 0]).all()) and bool((means[1] == x[0, 0, 0]).all())
    assert not bool(means[0].any())


@pytest.mark.parametrize("query", [BF, F32])
@pytest.mark.parametrize("value", [3e38, -3.2e38])
def test_the_largest_values(cuda, query, value):
    """Values whose sum is beyond fp32: their mean is not."""
    b = Batch(cuda, [2, 33, 300, 3000], 8, 2, 128, 16, BF, query, seed=45)
    live = torch.isfinite(b.v) & (b.v.abs() < 100)
    b.v.copy_(torch.where(live, torch.tensor(value, dtype=BF, device=cuda), b.v))
    b.check(b.attend())
