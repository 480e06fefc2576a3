"""Serving many sequences from one paged 16-bit key-value cache: the operators' calls as cases for timing and comparison.

A case is a dict of plain values; `kind` says which operator a pass calls:

  step    the bookkeeping of one serving step: sequences are cut back to the tokens that stand (drafts that were not
          accepted give their blocks back), then every sequence of the batch is extended by its new tokens: blocks from
          the free list, block tables, lengths, and each new token's position and slot.
  append  one layer's new rows on their way into the cache: biases, RMSNorm of every query and key head, rotation, and
          the keys and values written at the rows' slots (and the mean keys of the blocks that these rows complete).
  attend  one new token per sequence over the sequences' blocks, `layers` layers: the split of the batch's work is
          planned once, as a step does, and every layer attends by it.
  sparse  the same over few blocks of each sequence: the first, the last, and those whose mean key scores highest
          against the new token's queries; the chosen blocks and the attention over them.

Keys of a block lie token by token [kv head, token, dimension], values dimension by dimension [kv head, dimension,
token]. `own` says which side computes: the plain forms below, in torch, or the framework's operators.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
ROPE_BASE = 1000000.0
MAX_POS = 8192  # rows of the rotation table
SPARE_ROWS = 3  # sequences that the tables have room for beside the batch's
ENOSPC, E2BIG = -28, -7


def listed():
    return [
        # five conversations, a token each: the smallest step, whose latency every layer waits for
        {"name": "step-5", "kind": "step", "seqs": 5, "longest": 4000, "drafts": 1, "prompts": 0, "chunk": 0,
         "block": 16, "tight": False},
        # a busy server: sequences with drafts to check and a few chunks of prompts, in a pool that runs out
        {"name": "step-193-mixed-tight", "kind": "step", "seqs": 193, "longest": 30001, "drafts": 5, "prompts": 7,
         "chunk": 512, "block": 16, "tight": True},
        # one sequence's decode step at the benchmark's attention shape, 32-bit activations as the decode kernels make
        {"name": "append-1", "kind": "append", "rows": 1, "prompts": 0, "heads": 32, "kv_heads": 4, "head_size": 128,
         "rotary": 128, "block": 32, "input": "f32", "cache": "bf16", "query": "f32", "norms": True, "biases": False,
         "means": False},
        # a decode batch of a model with biases and no head norms, half of each head rotated
        {"name": "append-37-bias-f16", "kind": "append", "rows": 37, "prompts": 0, "heads": 16, "kv_heads": 16,
         "head_size": 64, "rotary": 32, "block": 16, "input": "f16", "cache": "f16", "query": "f16", "norms": False,
         "biases": True, "means": True},
        # prompts of a serving step, ragged against blocks and tiles
        {"name": "append-4093", "kind": "append", "rows": 4093, "prompts": 5, "heads": 32, "kv_heads": 4,
         "head_size": 128, "rotary": 128, "block": 16, "input": "bf16", "cache": "bf16", "query": "bf16",
         "norms": True, "biases": False, "means": True},
        # a short conversation, 32-bit queries
        {"name": "attend-1-ctx1000", "kind": "attend", "seqs": 1, "shortest": 1000, "longest": 1000, "heads": 32,
         "kv_heads": 4, "head_size": 128, "block": 32, "cache": "bf16", "query": "f32", "layers": 4},
        # a ragged batch of a model whose heads share nothing
        {"name": "attend-23-ragged-f16", "kind": "attend", "seqs": 23, "shortest": 1, "longest": 8191, "heads": 16,
         "kv_heads": 16, "head_size": 64, "block": 16, "cache": "f16", "query": "f16", "layers": 2},
        # one long document, alone
        {"name": "attend-1-ctx131071", "kind": "attend", "seqs": 1, "shortest": 131071, "longest": 131071, "heads": 32,
         "kv_heads": 4, "head_size": 128, "block": 32, "cache": "bf16", "query": "bf16", "layers": 2},
        # a full serving batch from short to long: the largest call
        {"name": "attend-64-ctx30001", "kind": "attend", "seqs": 64, "shortest": 500, "longest": 30001, "heads": 32,
         "kv_heads": 8, "head_size": 128, "block": 16, "cache": "bf16", "query": "bf16", "layers": 1},
        # a long conversation over a few of its blocks
        {"name": "sparse-1-ctx30001", "kind": "sparse", "seqs": 1, "shortest": 30001, "longest": 30001, "heads": 32,
         "kv_heads": 4, "head_size": 128, "block": 16, "cache": "bf16", "query": "bf16", "layers": 4, "sinks": 1,
         "window": 4, "budget": 32},
        # a batch of long documents, 32-bit queries
        {"name": "sparse-16-ctx65536", "kind": "sparse", "seqs": 16, "shortest": 9000, "longest": 65536, "heads": 32,
         "kv_heads": 8, "head_size": 128, "block": 16, "cache": "bf16", "query": "f32", "layers": 1, "sinks": 2,
         "window": 8, "budget": 128},
        # wide heads, one kv head, some sequences shorter than what would be chosen
        {"name": "sparse-7-wide-f16", "kind": "sparse", "seqs": 7, "shortest": 60, "longest": 20011, "heads": 8,
         "kv_heads": 1, "head_size": 256, "block": 64, "cache": "f16", "query": "f16", "layers": 2, "sinks": 1,
         "window": 2, "budget": 16},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(lo * (hi / lo) ** rng.random() + 0.5)))


def draw(rng):
    kind = rng.choice(["step", "append", "attend", "attend", "sparse", "sparse"])
    block = rng.choice([16, 32, 64])
    if kind == "step":
        seqs = _log_int(rng, 1, 190)
        return {"kind": "step", "seqs": seqs, "longest": _log_int(rng, 50, 30000), "drafts": rng.randint(1, 6),
                "prompts": rng.randint(0, min(7, seqs)), "chunk": _log_int(rng, 20, 500), "block": block,
                "tight": rng.random() < 0.3}
    heads, kv_heads = rng.choice([(32, 4), (16, 16), (32, 8), (8, 2), (8, 1), (6, 2)])
    d = rng.choice([64, 128, 256]) if heads <= 16 else rng.choice([64, 128])
    cache = rng.choice(["f16", "bf16"])
    query = rng.choice([cache, cache, "f32"])
    if kind == "append":
        rows = _log_int(rng, 1, 4000)
        return {"kind": "append", "rows": rows, "prompts": 0 if rows < 20 else rng.choice([0, rng.randint(1, 6)]),
                "heads": heads, "kv_heads": kv_heads, "head_size": d, "rotary": rng.choice([d, d, d // 2]),
                "block": block, "input": rng.choice(["f32", cache, "f16", "bf16"]), "cache": cache, "query": query,
                "norms": rng.random() < 0.6, "biases": rng.random() < 0.3, "means": rng.random() < 0.5}
    seqs = _log_int(rng, 1, 64)
    # the padded batch of the largest listed case holds 2 10^9 keys and values
    most = min(100000, 900000000 // (seqs * kv_heads * d))
    longest = _log_int(rng, 100, most)
    case = {"kind": kind, "seqs": seqs, "shortest": _log_int(rng, 1, longest), "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "head_size": d, "block": block, "cache": cache, "query": query,
            "layers": 2 if seqs * longest * kv_heads * d < 50000000 else 1}
    if kind == "sparse":
        case.update(sinks=rng.randint(0, 2), window=rng.randint(1, 8), budget=_log_int(rng, 4, 128))
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------

def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 1000003 + salt) % (1 << 62))
    return g


def _randn(shape, dtype, seed, salt):
    return torch.randn(shape, generator=_gen(seed, salt), device=DEV, dtype=dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cdiv(a, b):
    return -(-a // b)


def _lengths(case, rng):
    """Lengths spread from shortest to longest over their logarithm, in an order of the seed's."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    lens = [max(lo, min(hi, round(lo * (hi / lo) ** ((i + 1) / n)))) for i in range(n)]
    rng.shuffle(lens)
    return lens


def _tables(lens, block, rng, n_blocks, spare_blocks, max_blocks):
    """Block tables of sequences of these lengths whose blocks lie anywhere in a pool of n_blocks, of which
    spare_blocks more are free (others hold the rest)."""
    n = len(lens)
    rows = n + SPARE_ROWS
    ids = rng.sample(range(rows), n)
    perm = torch.randperm(n_blocks, generator=torch.Generator().manual_seed(rng.getrandbits(40))).tolist()
    table, length, at = [[-1] * max_blocks for _ in range(rows)], [0] * rows, 0
    for i, t in zip(ids, lens):
        nb = _cdiv(t, block)
        table[i][:nb] = perm[at:at + nb]
        length[i], at = t, at + nb
    free = perm[at:at + spare_blocks] + [0] * (n_blocks - spare_blocks)  # a stack, its top at the end
    return {"ids": _ints(ids), "blocks": _ints(table), "len": _ints(length), "free": _ints(free),
            "n_free": _ints([spare_blocks]), "block": block}


def _step_inputs(case, seed):
    rng = random.Random(seed * 7 + 1)
    n, block = case["seqs"], case["block"]
    base = [0 if i < case["prompts"] else rng.randint(1, case["longest"]) for i in range(n)]
    new = [case["chunk"] - rng.randrange(max(1, case["chunk"] // 3)) if i < case["prompts"]
           else rng.randint(1, case["drafts"]) for i in range(n)]
    both = list(zip(base, new))
    rng.shuffle(both)
    base, new = [b for b, _ in both], [t for _, t in both]
    need = sum(_cdiv(b + t, block) - _cdiv(b, block) for b, t in both)
    spare = need // 2 if case["tight"] else need + 10
    width = _cdiv(case["longest"] + case["drafts"] + case["chunk"], block)
    st = _tables(base, block, rng, n * (width + 1) + 10, spare, width)
    rows = n * case["drafts"] + case["prompts"] * case["chunk"] + 9  # rows of the step's buffers: some stay unused
    st.update(base=_ints(base), n_new=_ints(new), start=_ints([0] * (n + 1)), positions=_ints([0] * rows),
              slots=_ints([0] * rows), status=_ints([0] * n))
    return st


def _append_inputs(case, seed):
    rng = random.Random(seed * 7 + 2)
    T, H, KV, d, block = (case[k] for k in ("rows", "heads", "kv_heads", "head_size", "block"))
    kind, cache, R = TYPES[case["input"]], TYPES[case["cache"]], case["rotary"]
    # the rows' sequences: one token each, or `prompts` runs of consecutive tokens
    cuts = sorted(rng.sample(range(1, T), case["prompts"] - 1)) if case["prompts"] else list(range(1, T))
    runs = [b - a for a, b in zip([0] + cuts, cuts + [T])]
    first = [rng.randint(0, MAX_POS - r) for r in runs]
    n_blocks = (T // block + 2 * len(runs) if case["prompts"] else T) + 5
    perm = torch.randperm(n_blocks, generator=torch.Generator().manual_seed(rng.getrandbits(40))).tolist()
    pos, slots, at = [], [], 0
    for f, r in zip(first, runs):
        pos += range(f, f + r)
        slots += [perm[at + (f % block + j) // block] * block + (f + j) % block for j in range(r)]
        at += (f % block + r - 1) // block + 1
    freq = ROPE_BASE ** (-2.0 * torch.arange(R // 2, dtype=torch.float64, device=DEV) / R)
    ang = torch.arange(MAX_POS, dtype=torch.float64, device=DEV)[:, None] * freq
    st = {"qkv": _randn((T, (H + 2 * KV) * d), kind, seed, 1) * 1.5,  # as a joint projection leaves them
          "k": _randn((n_blocks, KV, block, d), cache, seed, 2), "v": _randn((n_blocks, KV, d, block), cache, seed, 3),
          "rope": torch.cat([torch.cos(ang), torch.sin(ang)], 1).float(), "positions": _ints(pos), "slots": _ints(slots),
          "q_out": torch.zeros((T, H, d), dtype=TYPES[case["query"]], device=DEV),
          "means": None, "q_norm": None, "k_norm": None, "q_bias": None, "k_bias": None, "v_bias": None}
    if case["means"]:
        st["means"] = st["k"].float().mean(2).to(cache)
    if case["norms"]:
        st.update(q_norm=1 + 0.2 * _randn(d, torch.float32, seed, 4), k_norm=1 + 0.2 * _randn(d, torch.float32, seed, 5))
    if case["biases"]:
        st.update(q_bias=_randn(H * d, torch.float32, seed, 6), k_bias=_randn(KV * d, torch.float32, seed, 7),
                  v_bias=_randn(KV * d, torch.float32, seed, 8))
    return st


def _attend_inputs(case, seed):
    rng = random.Random(seed * 7 + 3)
    L, n, H, KV, d, block = (case[k] for k in ("layers", "seqs", "heads", "kv_heads", "head_size", "block"))
    cache = TYPES[case["cache"]]
    lens = _lengths(case, rng)
    used = sum(_cdiv(t, block) for t in lens)
    st = _tables(lens, block, rng, used + 9, 9, _cdiv(case["longest"], block) + 4)
    n_blocks = st["free"].numel()
    # every layer's blocks in one pool; a sequence's unwritten slots hold what was there before
    st["k"] = _randn((L, n_blocks, KV, block, d), cache, seed, 11)
    st["v"] = _randn((L, n_blocks, KV, d, block), cache, seed, 12)
    st["q"] = (2 * _randn((L, n, H, d), torch.float32, seed, 13)).to(TYPES[case["query"]])
    st["out"] = torch.zeros((L, n, H, d), dtype=TYPES[case["query"]], device=DEV)
    st["lens"] = lens
    if case["kind"] == "sparse":
        # neighbouring tokens' keys have much in common
        st["k"] = st["k"] * 0.8 + 0.6 * _randn((L, n_blocks, KV, 1, d), cache, seed, 14)
        st["means"] = st["k"].float().mean(3).to(cache)
        st["lists"] = torch.zeros((L, n, KV, case["sinks"] + case["window"] + case["budget"]), dtype=torch.int32,
                                  device=DEV)
    return st


_INPUTS = {"step": _step_inputs, "append": _append_inputs, "attend": _attend_inputs, "sparse": _attend_inputs}


def prepare(case, seed):
    return dict(_INPUTS[case["kind"]](case, seed), case=case)


# ---- plain forms --------------------------------------------------------------------------------------------------

def _truncate(st):
    """Sequences cut back to `base` tokens; their blocks behind that go back on the free stack, so that the next
    extension takes them again in the same order."""
    ids, block = st["ids"].long(), st["block"]
    rows, old = st["blocks"][ids], st["len"][ids].long()
    new = torch.minimum(st["base"].long(), old)
    have, keep = (old + block - 1) // block, (new + block - 1) // block
    give = have - keep
    off = torch.cumsum(give, 0) - give
    j = torch.arange(rows.shape[1], device=DEV)
    gone = (j >= keep[:, None]) & (j < have[:, None])
    n_free, total = st["n_free"].long(), give.sum()
    at = torch.where(gone, n_free + total - 1 - (off[:, None] + j - keep[:, None]), st["free"].numel())
    free = torch.cat([st["free"], st["free"].new_zeros(1)])
    free.scatter_(0, at.reshape(-1), rows.reshape(-1))
    st["free"].copy_(free[:-1])
    st["n_free"].copy_(n_free + total)
    st["len"][ids] = new.int()


def _extend(st):
    """Room for every sequence's new tokens, in the batch's order while the free blocks last."""
    ids, block, n_new = st["ids"].long(), st["block"], st["n_new"].long()
    rows, old = st["blocks"][ids], st["len"][ids].long()
    T, width = st["slots"].numel(), rows.shape[1]
    start = torch.cumsum(torch.cat([n_new.new_zeros(1), n_new]), 0)
    have, want = (old + block - 1) // block, (old + n_new + block - 1) // block
    big = (want > width) | (start[1:] > T)
    need = torch.where(big, 0, want - have)
    upto = torch.cumsum(need, 0)
    n_free = st["n_free"].long()
    given = ~big & ((upto <= n_free) | (need == 0))
    j = torch.arange(width, device=DEV)
    fresh = given[:, None] & (j >= have[:, None]) & (j < want[:, None])
    at = n_free - 1 - ((upto - need)[:, None] + j - have[:, None])
    rows = torch.where(fresh, st["free"][at.clamp(0, st["free"].numel() - 1)], rows)
    st["blocks"][ids] = rows
    st["len"][ids] = torch.where(given, old + n_new, old).int()
    st["n_free"].copy_(n_free - torch.where(given & (need > 0), upto, 0).max())
    st["start"].copy_(start)
    st["status"].copy_(torch.where(big, E2BIG, torch.where(given, 0, ENOSPC)))
    r = torch.arange(T, device=DEV)
    seq = torch.searchsorted(start[1:], r, right=True)
    inside, seq = seq < ids.numel(), seq.clamp(max=ids.numel() - 1)
    pos = torch.where(inside, old[seq] + r - start[seq], 0)
    slot = rows[seq, (pos // block).clamp(max=width - 1)] * block + pos % block
    st["positions"].copy_(pos)
    st["slots"].copy_(torch.where(inside & given[seq], slot, -1))


def _heads(x, heads, bias, norm, st):
    """One kind of heads of the rows [T x heads x head size], in 32 bits: bias, RMSNorm, rotation (with a norm or not)."""
    x = x.float().reshape(x.shape[0], heads, -1)
    if bias is not None:
        x = x + bias.view(heads, -1)
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm
    R = st["rope"].shape[1]
    turn = st["rope"][st["positions"].long()][:, None]
    cos, sin = turn[..., :R // 2], turn[..., R // 2:]
    lo, hi = x[..., :R // 2], x[..., R // 2:R]
    return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos, x[..., R:]], -1)


def _append(st):
    case = st["case"]
    H, KV, d, block = case["heads"], case["kv_heads"], case["head_size"], case["block"]
    q, k, v = st["qkv"].split([H * d, KV * d, KV * d], 1)
    st["q_out"].copy_(_heads(q, H, st["q_bias"], st["q_norm"], st))
    k = _heads(k, KV, st["k_bias"], st["k_norm"], st)
    v = v.float() if st["v_bias"] is None else v.float() + st["v_bias"]
    at, off = st["slots"].long() // block, st["slots"].long() % block
    st["k"][at, :, off] = k.to(st["k"].dtype)
    st["v"][at, :, :, off] = v.reshape(-1, KV, d).to(st["v"].dtype)
    if st["means"] is not None:  # of the blocks whose last slot was written; the others' go into a row of their own
        whole = torch.cat([st["means"], st["means"][:1]])
        whole[torch.where(off == block - 1, at, len(whole) - 1)] = st["k"][at].float().mean(2).to(st["k"].dtype)
        st["means"].copy_(whole[:-1])


def _attention(st, blocks, count):
    """Softmax attention of every layer's and sequence's queries over the listed blocks [layers or 1, n, kv heads or 1,
    blocks], whose first count [n] tokens in order are attended."""
    case = st["case"]
    L, n, H, KV, d = (case[k] for k in ("layers", "seqs", "heads", "kv_heads", "head_size"))
    B = blocks.shape[3]
    l, g = torch.arange(L, device=DEV)[:, None, None, None], torch.arange(KV, device=DEV)[None, None, :, None]
    at = blocks.long().clamp(min=0)
    k = st["k"][l, at, g].float().reshape(L, n, KV, B * st["block"], d)
    v = st["v"][l, at, g].float().transpose(4, 5).reshape(L, n, KV, B * st["block"], d)
    q = st["q"].float().view(L, n, KV, H // KV, d)
    s = torch.matmul(q, k.transpose(3, 4)) * (1 / math.sqrt(d))
    live = torch.arange(B * st["block"], device=DEV) < count[:, None, None, None]
    s = torch.where(live, s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    st["out"].copy_((torch.matmul(p, v) / p.sum(-1, keepdim=True)).reshape(L, n, H, d))


def _attend(st):
    ids = st["ids"].long()
    blocks = st["blocks"][ids, :_cdiv(st["case"]["longest"], st["block"])]
    _attention(st, blocks[None, :, None], st["len"][ids])


def _sparse(st):
    case, block, ids = st["case"], st["block"], st["ids"].long()
    L, n, H, KV, d = (case[k] for k in ("layers", "seqs", "heads", "kv_heads", "head_size"))
    width, length = st["lists"].shape[3], st["len"][ids].long()
    B = max(width, _cdiv(case["longest"], block))
    rows = torch.nn.functional.pad(st["blocks"][ids], (0, width), value=-1)[:, :B]
    have = ((length + block - 1) // block)[:, None]
    # scores of the blocks' mean keys: sums of exact products in 64 bits, the largest of the group's heads, as 32 bits
    mean = st["means"][:, rows.long().clamp(min=0)].double().transpose(2, 3)  # [L, n, KV, B, d]
    s = torch.matmul(st["q"].double().view(L, n, KV, H // KV, d), mean.transpose(3, 4)).amax(3).float()
    j = torch.arange(B, device=DEV)
    always = (j < case["sinks"]) | (j >= have - case["window"]) | (have <= width)
    s = torch.where(always[None, :, None], math.inf, s)
    s = torch.where((j < have)[None, :, None], s, -math.inf)
    top = torch.sort(s, dim=-1, descending=True, stable=True).indices[..., :width]
    top = torch.sort(torch.where(top < have[:, None], top, B), dim=-1).values
    st["lists"].copy_(torch.where(top < B, top, -1))
    # every listed block but the last one of a sequence is full
    taken = torch.minimum(have[:, 0], torch.full_like(have[:, 0], width))
    count = taken * block - (have[:, 0] * block - length)
    pages = torch.gather(rows[None, :, None].expand(L, n, KV, B), 3, top.clamp(max=B - 1))
    _attention(st, pages, count)


# ---- the framework's operators --------------------------------------------------------------------------------------

_stream = None


def _serving_stream():
    """The stream that the program serves on (calls on the default stream are synchronous). It becomes the current one
    with the first pass: after the inputs that were made before, and before whatever is done with outputs later."""
    global _stream
    if _stream is None:
        _stream = torch.cuda.Stream()
        _stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(_stream)
    return _stream


def _handles(st):
    """The table, caches and work split over the program's own buffers, made on a state's first pass and kept."""
    if "table" not in st:
        from vireo_amd import paged
        case = st["case"]
        if "blocks" in st:
            st["table"] = paged.PagedTable(st["blocks"], st["len"], st["free"], st["n_free"], st["block"])
        if case["kind"] == "append":
            st["table"] = None
            st["cache"] = paged.PagedCache(st["k"], st["v"], st["means"])
        elif case["kind"] != "step":
            means = st.get("means")
            st["cache"] = [paged.PagedCache(st["k"][l], st["v"][l], None if means is None else means[l])
                           for l in range(case["layers"])]
            listed_blocks = st["lists"].shape[3] if "lists" in st else 0
            st["plan"] = paged.PagedPlan(st["table"], st["cache"][0], case["seqs"], case["heads"], listed_blocks)
    return st


def _run_own(st):
    case, s = _handles(st)["case"], _serving_stream()
    if case["kind"] == "step":
        st["table"].truncate(st["base"], ids=st["ids"], stream=s)
        st["table"].extend(st["n_new"], st["start"], st["positions"], st["slots"], st["status"], ids=st["ids"], stream=s)
    elif case["kind"] == "append":
        H, KV, d = case["heads"], case["kv_heads"], case["head_size"]
        q, k, v = st["qkv"].split([H * d, KV * d, KV * d], 1)
        st["cache"].append(q.unflatten(1, (H, d)), k.unflatten(1, (KV, d)), v.unflatten(1, (KV, d)), st["positions"],
                           st["slots"], st["q_out"], st["rope"], q_norm=st["q_norm"], k_norm=st["k_norm"],
                           q_bias=st["q_bias"], k_bias=st["k_bias"], v_bias=st["v_bias"], eps=EPS, stream=s)
    else:
        st["plan"].update(ids=st["ids"], stream=s)
        for l, cache in enumerate(st["cache"]):
            lists = None
            if case["kind"] == "sparse":
                lists = st["lists"][l]
                cache.select(st["q"][l], st["plan"], lists, sinks=case["sinks"], window=case["window"], stream=s)
            cache.attend(st["q"][l], st["out"][l], st["plan"], lists=lists, stream=s)


def run(state):
    kind = state["case"]["kind"]
    if own:
        _run_own(state)
    elif kind == "step":
        _truncate(state)
        _extend(state)
    elif kind == "append":
        _append(state)
    elif kind == "attend":
        _attend(state)
    else:
        _sparse(state)
    given = {"step": ("blocks", "len", "free", "n_free", "start", "positions", "slots", "status"),
             "append": ("q_out", "k", "v", "means"), "attend": ("out",), "sparse": ("out", "lists")}[kind]
    return {k: state[k] for k in given if state[k] is not None}


# ---- in 64 bits -----------------------------------------------------------------------------------------------------

def _exact_append(case, seed):
    st = _append_inputs(case, seed)
    T, H, KV, d, block = (case[k] for k in ("rows", "heads", "kv_heads", "head_size", "block"))
    x = st["qkv"].double().view(T, H + 2 * KV, d)
    if case["biases"]:
        x = x + torch.cat([st["q_bias"], st["k_bias"], st["v_bias"]]).double().view(1, -1, d)
    turned = x[:, :H + KV]
    if case["norms"]:
        w = torch.cat([st["q_norm"].expand(H, d), st["k_norm"].expand(KV, d)]).double()
        turned = turned / torch.sqrt(torch.linalg.vector_norm(turned, dim=-1, keepdim=True) ** 2 / d + EPS) * w
    half = case["rotary"] // 2
    table = st["rope"][st["positions"].long()].double()
    # the pair (j, j + half) as a complex number, turned by its angle
    pair = torch.complex(turned[..., :half], turned[..., half:2 * half])
    pair = pair * torch.complex(table[:, None, :half], table[:, None, half:])
    turned = torch.cat([pair.real, pair.imag, turned[..., 2 * half:]], -1)
    pages, offs = torch.div(st["slots"], block, rounding_mode="floor").tolist(), (st["slots"] % block).tolist()
    k, v = st["k"].double(), st["v"].double()
    where = torch.tensor(pages, device=DEV), torch.tensor(offs, device=DEV)
    k[where[0], :, where[1]] = turned[:, H:]
    v.transpose(2, 3)[where[0], :, where[1]] = x[:, H + KV:]
    out = {"q_out": turned[:, :H], "k": k, "v": v}
    if case["means"]:
        means = st["means"].double()
        full = sorted({p for p, o in zip(pages, offs) if o == block - 1})
        if full:
            stored = k[full].to(TYPES[case["cache"]]).double()
            means[full] = stored.sum(2) / block
        out["means"] = means
    return out


def _exact_attend(case, seed):
    st = _attend_inputs(case, seed)
    L, n, H, KV, d, block = (case[k] for k in ("layers", "seqs", "heads", "kv_heads", "head_size", "block"))
    group = H // KV
    out = torch.zeros((L, n, H, d), dtype=torch.float64, device=DEV)
    ids = st["ids"].tolist()
    for l in range(L):
        for i in range(n):
            t = st["lens"][i]
            nb = _cdiv(t, block)
            pages = st["blocks"][ids[i], :nb].long()
            for g in range(KV):
                q = st["q"][l, i, g * group:(g + 1) * group].double()
                chosen = torch.arange(nb, device=DEV)
                if case["kind"] == "sparse" and nb > st["lists"].shape[3]:
                    lo, hi = case["sinks"], nb - case["window"]
                    score = (st["means"][l, pages[lo:hi], g].double() @ q.t()).max(1).values.float()
                    best = torch.argsort(-score, stable=True)[:case["budget"]] + lo
                    chosen = torch.cat([chosen[:lo], torch.sort(best).values, chosen[hi:]])
                tokens = (chosen[:, None] * block + torch.arange(block, device=DEV)).reshape(-1) < t
                k = st["k"][l, pages[chosen], g].double().reshape(-1, d)[tokens]
                v = st["v"][l, pages[chosen], g].double().permute(0, 2, 1).reshape(-1, d)[tokens]
                w = torch.softmax(k @ q.t() / math.sqrt(d), 0)
                out[l, i, g * group:(g + 1) * group] = w.t() @ v
    return {"out": out, "lists": None} if case["kind"] == "sparse" else {"out": out}


def exact(case, seed):
    if case["kind"] == "step":  # whole numbers
        return None
    return _exact_append(case, seed) if case["kind"] == "append" else _exact_attend(case, seed)


# ---- work -----------------------------------------------------------------------------------------------------------

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["kind"] == "step":
        # lengths, new counts, statuses, the tables' new entries, positions and slots of the rows
        rows = case["seqs"] * (case["drafts"] + 1) / 2 + case["prompts"] * case["chunk"]
        return {"bytes": case["seqs"] * 32 + rows * 8 + rows / case["block"] * 16, "flops": 0}
    H, KV, d = case["heads"], case["kv_heads"], case["head_size"]
    if case["kind"] == "append":
        T = case["rows"]
        per = (H + 2 * KV) * d * size[case["input"]] + H * d * size[case["query"]] + 2 * KV * d * size[case["cache"]]
        turn = min(T, MAX_POS) * case["rotary"] * 4
        return {"bytes": T * (per + 8) + turn, "flops": T * (H + KV) * d * 8}
    L, block = case["layers"], case["block"]
    lens = _lengths(case, random.Random(0))
    if case["kind"] == "sparse":
        width = case["sinks"] + case["window"] + case["budget"]
        scored = sum(max(0, _cdiv(t, block) - case["sinks"] - case["window"]) for t in lens if _cdiv(t, block) > width)
        tokens = sum(min(t, width * block) for t in lens)
        more = {"bytes": scored * KV * d * size[case["cache"]] + len(lens) * KV * width * 4, "flops": 2 * scored * H * d}
    else:
        tokens, more = sum(lens), {"bytes": 0, "flops": 0}
    bytes_ = 2 * tokens * KV * d * size[case["cache"]] + 2 * len(lens) * H * d * size[case["query"]]
    return {"bytes": L * (bytes_ + more["bytes"]), "flops": L * (4 * tokens * H * d + more["flops"])}
