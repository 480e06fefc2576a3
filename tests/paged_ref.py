"""Plain forms of the paged cache's operators: the bookkeeping one sequence at a time in Python, the arithmetic in
fp64 torch."""
import errno
import math

import torch

OK, EINVAL, E2BIG, ENOSPC = 0, -errno.EINVAL, -errno.E2BIG, -errno.ENOSPC


class RefTable:
    """The table of include/vireo_paged.h as Python lists."""

    def __init__(self, max_seqs, max_blocks, n_blocks, G):
        self.max_blocks, self.G = max_blocks, G
        self.blocks = [[-1] * max_blocks for _ in range(max_seqs)]
        self.len = [0] * max_seqs
        self.free = list(range(n_blocks - 1, -1, -1))
        self.n_free = n_blocks

    def extend(self, ids, n_new, max_rows):
        """start, positions, slots, status."""
        G, seen = self.G, set()
        start, status, out = [0], [], []
        short = False
        for i, new in zip(ids, n_new):
            rows = max(new, 0)
            first = start[-1]
            start.append(first + rows)
            base = 0
            if not 0 <= i < len(self.len) or i in seen or new < 0:
                st = EINVAL
            else:
                base = self.len[i]
                have, want = -(-base // G), -(-(base + new) // G)
                if want > self.max_blocks or first + rows > max_rows:
                    st = E2BIG
                elif want > have and (short or want - have > self.n_free):
                    st, short = ENOSPC, True
                else:
                    st = OK
                    for b in range(have, want):
                        self.n_free -= 1
                        self.blocks[i][b] = self.free[self.n_free]
                    self.len[i] = base + new
            if 0 <= i < len(self.len):
                seen.add(i)
            status.append(st)
            for j in range(rows):
                p = base + j if st != EINVAL else 0
                out.append((p, self.blocks[i][p // G] * G + p % G if st == OK else -1))
        out = (out + [(0, -1)] * max_rows)[:max_rows]
        return start, [p for p, _ in out], [s for _, s in out], status

    def truncate(self, ids, new_len):
        seen, back = set(), []
        for i, to in zip(ids, new_len):
            if 0 <= i < len(self.len) and i not in seen and 0 <= to < self.len[i]:
                back += self.blocks[i][-(-to // self.G):-(-self.len[i] // self.G)]
                self.len[i] = to
            if 0 <= i < len(self.len):
                seen.add(i)
        for j, b in enumerate(reversed(back)):
            self.free[self.n_free + j] = b
        self.n_free += len(back)


def heads64(x, bias, norm, eps, rope, positions):
    """[T, heads, d] rows with bias, RMSNorm per head and rotation, in fp64. rope: [max_pos, rotary] or None."""
    x = x.double()
    if bias is not None:
        x = x + bias.double().view(1, x.shape[1], x.shape[2])
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double()
    if rope is not None:
        R, ok = rope.shape[1], ((positions >= 0) & (positions < rope.shape[0]))
        tab = rope[torch.where(ok, positions, torch.zeros_like(positions)).long()].double()[:, None]
        c, s = tab[..., :R // 2], tab[..., R // 2:]
        lo, hi = x[..., :R // 2], x[..., R // 2:R]
        x = torch.where(ok[:, None, None], torch.cat([lo * c - hi * s, lo * s + hi * c, x[..., R:]], -1), x)
    return x


def attend64(q, k, v, blocks, n_tokens, scale):
    """One sequence and kv head in fp64: q [heads, d], its blocks' numbers and how many of each one's slots are
    attended. Returns the output, sum p |v| and the largest sum |q k| scale (for error bounds); zeros with no token."""
    d = q.shape[1]
    ks = [k[b, :n].double() for b, n in zip(blocks, n_tokens) if n > 0]
    vs = [v[b, :, :n].double().t() for b, n in zip(blocks, n_tokens) if n > 0]
    if not ks:
        z = torch.zeros_like(q, dtype=torch.float64)
        return z, z, 0.0
    ks, vs, q = torch.cat(ks), torch.cat(vs), q.double()
    s = q @ ks.t().contiguous() * scale
    p = torch.exp(s - s.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    size = float((q.abs() @ ks.abs().t().contiguous()).max()) * scale if torch.isfinite(ks).all() else math.inf
    return p @ vs, p @ vs.abs(), size


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attend_bound(out64, weight64, size, d, dtype, cache):
    """How far an output may be from fp64: the result's rounding; its weights' truncation to 16 bits (bf16: what is cut
    off is less than 2^-15 of the leading bit) or 22 (fp16: less than 2^-21), none where the result is fp32 (three
    parts hold all 24 bits); and the scores' fp32 sums, each of at most 32 terms inside the matrix cores
    and d / 32 steps of at most 3 parts, whose relative error in units of 2^-24 goes into every weight twice (it and
    the sum), with 16 for the exponential, the scale and the sums over tokens."""
    u = 2.0 ** -24
    cut = 0.0 if dtype is torch.float32 else 2.0 ** -15 if cache is torch.bfloat16 else 2.0 ** -21
    return half_step(dtype) * out64.abs() + weight64 * (cut + 2 * u * ((32 + 3 * d // 32) * size + 16))
