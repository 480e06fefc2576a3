"""The paged cache's argument checks, which need no GPU: every call here is refused before any device work, and plans'
sizes follow from their shapes. And the plain bookkeeping of the GPU tests, on itself."""
import ctypes as C
import errno
import os
import random
import subprocess

import pytest

from paged_ref import E2BIG, EINVAL, ENOSPC, RefTable
from vireo_amd import _lib

BAD = -errno.EINVAL
PTR = 0x10000


def table(**kw):
    f = dict(max_seqs=4, max_blocks=8, n_blocks=16, block_tokens=16, blocks=PTR, len=PTR, free_blocks=PTR, n_free=PTR)
    f.update(kw)
    return _lib.PagedTableC(**f)


def cache(**kw):
    f = dict(type=30, n_blocks=16, block_tokens=16, n_kv_heads=2, head_size=128, k=PTR, v=PTR, means=PTR)
    f.update(kw)
    return _lib.PagedCacheC(**f)


def plan(t, **kw):
    f = dict(table=C.pointer(t), ids=None, n=3, n_heads=8, n_kv_heads=2, head_size=128, list_blocks=0, mem=PTR)
    f.update(kw)
    return _lib.PagedPlanC(**f)


BAD_TABLES = [dict(max_seqs=0), dict(max_seqs=4097), dict(max_blocks=0), dict(n_blocks=0), dict(block_tokens=0),
              dict(block_tokens=24), dict(block_tokens=8), dict(block_tokens=256), dict(n_blocks=2 ** 27),
              dict(max_blocks=2 ** 27), dict(blocks=None), dict(len=None), dict(free_blocks=None), dict(n_free=None)]


@pytest.mark.parametrize("bad", BAD_TABLES)
def test_tables_are_checked(lib, bad):
    t = table(**bad)
    assert lib.vireo_paged_reset(C.byref(t), None) == BAD
    assert lib.vireo_paged_extend(C.byref(t), None, None, 1, 1, PTR, PTR, PTR, PTR, None) == BAD
    assert lib.vireo_paged_truncate(C.byref(t), None, None, 1, None) == BAD
    p = plan(t)
    assert lib.vireo_paged_plan_bytes(C.byref(p)) == BAD
    assert lib.vireo_paged_plan_update(C.byref(p), None) == BAD


def test_extend_and_truncate_are_checked(lib):
    t = table()
    ok = [None, None, 2, 4, PTR, PTR, PTR, PTR]
    for i, v in ((2, -1), (2, 5), (3, -1), (4, None), (5, None), (6, None), (7, None)):
        args = list(ok)
        args[i] = v
        assert lib.vireo_paged_extend(C.byref(t), *args, None) == BAD, (i, v)
    assert lib.vireo_paged_extend(None, *ok, None) == BAD
    assert lib.vireo_paged_truncate(C.byref(t), None, None, -1, None) == BAD
    assert lib.vireo_paged_truncate(C.byref(t), None, None, 5, None) == BAD
    assert lib.vireo_paged_reset(None, None) == BAD


@pytest.mark.parametrize("bad", [dict(n=0), dict(n=4097), dict(n_heads=0), dict(n_heads=9), dict(n_heads=8192, n_kv_heads=1),
                                 dict(n_kv_heads=0), dict(head_size=96), dict(list_blocks=-1), dict(list_blocks=2 ** 27)])
def test_plans_are_checked(lib, bad):
    p = plan(table(), **bad)
    assert lib.vireo_paged_plan_bytes(C.byref(p)) == BAD
    assert lib.vireo_paged_plan_update(C.byref(p), None) == BAD
    assert lib.vireo_paged_attend(C.byref(cache()), C.byref(p), PTR, 30, 1024, 1.0, None, PTR, 1024, None) == BAD


def test_plan_bytes(lib):
    t = table()
    size = lambda **kw: lib.vireo_paged_plan_bytes(C.byref(plan(t, **kw)))  # noqa: E731
    assert 0 < size() < size(n_heads=16)
    assert size(list_blocks=4) >= size() + 3 * 2 * 8 * 4
    p = plan(t, mem=None)
    assert lib.vireo_paged_plan_update(C.byref(p), None) == BAD
    p = plan(t, mem=PTR + 16)  # 256-byte aligned
    assert lib.vireo_paged_plan_update(C.byref(p), None) == BAD
    p = plan(t, table=None)
    assert lib.vireo_paged_plan_bytes(C.byref(p)) == BAD


BAD_CACHES = [dict(type=0), dict(type=8), dict(n_blocks=0), dict(block_tokens=24), dict(n_kv_heads=0), dict(head_size=80),
              dict(k=None), dict(v=None), dict(k=PTR + 2), dict(v=PTR + 8), dict(means=PTR + 4), dict(n_blocks=2 ** 27)]


def rows(**kw):
    f = dict(rows=3, n_heads=8, type=0, q=PTR, k=PTR, v=PTR, q_stride=1024, k_stride=256, v_stride=256, eps=1e-6, rope=PTR,
             rotary=128, max_pos=10, positions=PTR, slots=PTR, q_out=PTR, q_out_type=0, q_out_stride=1024)
    f.update(kw)
    return _lib.PagedRowsC(**f)


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_caches_are_checked(lib, bad):
    c, r = cache(**bad), rows()
    assert lib.vireo_paged_append(C.byref(c), C.byref(r), None) == BAD
    p = plan(table())
    assert lib.vireo_paged_attend(C.byref(c), C.byref(p), PTR, 0, 1024, 1.0, None, PTR, 1024, None) == BAD


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(n_heads=0), dict(type=8), dict(q=None), dict(k=None), dict(v=None), dict(q=PTR + 4),
    dict(q_stride=1023), dict(q_stride=1022), dict(k_stride=252), dict(v_stride=255), dict(q_stride=-1024), dict(rotary=24),
    dict(rotary=144), dict(rotary=-16), dict(rope=None), dict(max_pos=0), dict(positions=None), dict(slots=None),
    dict(q_out=None), dict(q_out=PTR + 8), dict(q_out_type=1), dict(q_out_stride=512), dict(eps=-1.0),
    dict(eps=float("nan"))])
def test_rows_are_checked(lib, bad):
    assert lib.vireo_paged_append(C.byref(cache()), C.byref(rows(**bad)), None) == BAD


def test_attend_and_select_are_checked(lib):
    t = table()
    c, p, pl = cache(), plan(t), plan(t, list_blocks=5)
    ok = [PTR, 30, 1024, 1.0, None, PTR, 1024]
    for i, v in ((0, None), (0, PTR + 2), (1, 1), (1, 8), (2, 1020), (2, 512), (3, 0.0), (3, -1.0), (3, float("inf")),
                 (3, float("nan")), (4, PTR), (5, None), (5, PTR + 4), (6, 8)):
        args = list(ok)
        args[i] = v
        assert lib.vireo_paged_attend(C.byref(c), C.byref(p), *args, None) == BAD, (i, v)
    assert lib.vireo_paged_attend(C.byref(c), C.byref(pl), *ok, None) == BAD  # a plan with lists, none given
    # a cache of another shape than the plan's
    for kw in (dict(n_kv_heads=4), dict(head_size=64), dict(block_tokens=32), dict(n_blocks=17)):
        assert lib.vireo_paged_attend(C.byref(cache(**kw)), C.byref(p), *ok, None) == BAD
        assert lib.vireo_paged_select(C.byref(cache(**kw)), C.byref(pl), PTR, 30, 1024, 1, 1, PTR, None) == BAD
    ok = [PTR, 30, 1024, 1, 1, PTR]
    for i, v in ((0, None), (1, 1), (2, 1000), (3, -1), (3, 5), (4, 0), (4, 5), (5, None)):
        args = list(ok)
        args[i] = v
        assert lib.vireo_paged_select(C.byref(c), C.byref(pl), *args, None) == BAD, (i, v)
    assert lib.vireo_paged_select(C.byref(c), C.byref(p), *ok, None) == BAD  # a plan without lists
    assert lib.vireo_paged_select(C.byref(cache(means=None)), C.byref(pl), *ok, None) == BAD


def test_plain_bookkeeping_keeps_every_block():
    """No block is lost or owned twice, whatever the order of extensions and cuts."""
    rng, seen = random.Random(5), set()
    for _ in range(40):
        seqs, width, nb, G = rng.randint(1, 9), rng.randint(1, 9), rng.randint(1, 30), rng.choice([16, 32])
        t = RefTable(seqs, width, nb, G)
        for _ in range(12):
            ids = [rng.randrange(-1, seqs + 1) for _ in range(rng.randint(0, seqs))]
            start, pos, slots, st = t.extend(ids, [rng.randint(-1, 50) for _ in ids], 90)
            seen |= set(st)
            used = [s for s in slots if s >= 0]
            assert len(set(used)) == len(used)
            ids = [rng.randrange(-1, seqs + 1) for _ in range(rng.randint(0, seqs))]
            t.truncate(ids, [rng.randint(-1, 60) for _ in ids])
            own = [b for r, n in zip(t.blocks, t.len) for b in r[:-(-n // G)]]
            assert sorted(own + t.free[:t.n_free]) == list(range(nb))
    assert seen == {0, EINVAL, E2BIG, ENOSPC}


@pytest.mark.parametrize("language", [["-x", "c", "-std=c11"], ["-x", "c++", "-std=c++17"]], ids=["c11", "c++17"])
def test_header_stands_alone(language):
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    source = """#include <vireo_paged.h>
int64_t need(const vireo_paged_plan *p);
int64_t need(const vireo_paged_plan *p) { return vireo_paged_plan_bytes(p); }
"""
    r = subprocess.run(["gcc", *language, "-Wall", "-Wextra", "-Wpedantic", "-Werror", "-fsyntax-only", "-I", include, "-"],
                       input=source, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


@pytest.mark.parametrize("kw", [dict(q_out_stride=2048), dict(type=30, q_out_type=0), dict(type=0, q_out_type=30)])
def test_queries_in_place_keep_their_rows(lib, kw):
    """q_out at q's address with rows elsewhere or elements of another size would be written over rows still to be read."""
    assert lib.vireo_paged_append(C.byref(cache()), C.byref(rows(**kw)), None) == BAD


def test_attention_in_place_keeps_its_rows(lib):
    t = table()
    assert lib.vireo_paged_attend(C.byref(cache()), C.byref(plan(t)), PTR, 30, 1024, 1.0, None, PTR, 2048, None) == BAD


@pytest.mark.parametrize("hs,n_rows,n_heads", [(128, 2 ** 26, 8), (256, 2 ** 24, 30), (64, 2 ** 28, 8), (64, 2 ** 30, 1),
                                               (64, 2 ** 31 - 1, 65535)])
def test_more_rows_than_a_launch_takes(lib, hs, n_rows, n_heads):
    """Refused before any device work: 2^32 threads and more, 256 / (hs / 16) head rows to 256 of them."""
    c = cache(head_size=hs)
    r = rows(rows=n_rows, n_heads=n_heads, rotary=0, q_stride=n_heads * hs, k_stride=2 * hs, v_stride=2 * hs,
             q_out_stride=n_heads * hs)
    assert lib.vireo_paged_append(C.byref(c), C.byref(r), None) == -errno.E2BIG
