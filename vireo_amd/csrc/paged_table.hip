// Block tables of the paged cache (API: include/vireo_paged.h): blocks taken
// and given back, positions and slots of a step's rows, and the split of a
// batch's attention, all from lengths that live on the device.
//
// The sequences of a batch are few (at most 4096) and depend on each other
// through prefix sums (whose blocks come first), so each call is one workgroup
// of 1024 threads with the batch in LDS: bound by its chain of dependent loads
// (ids -> lengths -> stack or table entries) and barriers, not by bytes. Only
// rows beyond kRowsHere go to a second launch over the whole chip.
#include <hip/hip_runtime.h>
#include <errno.h>
#include "paged.h"

namespace {

constexpr int kThreads = 1024, kFewThreads = 256;  // a batch of at most kFewThreads takes so many: barriers of 4 waves
// Rows that extend's one workgroup numbers itself, four per thread at a time; more
// take a second launch over the chip. 193 sequences, 4 558 rows: kernels of 4.5 and 3.7 us in
// two launches, 7.9 in one. 64 sequences, replayed in a graph: 4 096 rows 7.9 us in two and 7.5 in
// one, 8 192 rows 8.4 and 10.9, 16 384 rows 9.5 and 18.7; called one by one the second launch
// costs the host 3 us more.
constexpr int kRowsHere = 8192;
constexpr uint32_t kMaxRows = 0x7fffffff;

VH_DEV int lane_id() { return threadIdx.x & 63; }

// Sums that stop at 2^31 - 1 (adding in any order gives the same).
VH_DEV uint32_t add_sat(uint32_t a, uint32_t b) { return min(a + b, kMaxRows); }

// Exclusive prefix sum over the workgroup's NT threads; *total receives the sum.
// wsum: a word of LDS per wave (one barrier inside; wsum is read after it, so
// its next use needs another barrier in between).
template <int NT>
VH_DEV uint32_t block_scan(uint32_t v, uint32_t *wsum, uint32_t *total) {
    const int lane = lane_id(), wv = threadIdx.x >> 6;
    uint32_t s = v;
    s = add_sat(s, dpp_u<0x111>(s));
    s = add_sat(s, dpp_u<0x112>(s));
    s = add_sat(s, dpp_u<0x114>(s));
    s = add_sat(s, dpp_u<0x118>(s));
    s = add_sat(s, dpp_u<0x142, 0xA>(s));
    s = add_sat(s, dpp_u<0x143, 0xC>(s));
    if (lane == 63) wsum[wv] = s;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; w++) {
        const uint32_t u = wsum[w];
        before = w < wv ? add_sat(before, u) : before;
        all = add_sat(all, u);
    }
    *total = all;
    const uint32_t up = __shfl_up(s, 1);
    return add_sat(before, lane ? up : 0u);
}

// the last i < n with a[i] <= v (a ascending, a[0] <= v): the sequence that item v belongs to
VH_DEV int find(const uint32_t *a, int n, uint32_t v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (a[m] <= v) lo = m;
        else hi = m;
    }
    return lo;
}

VH_DEV int blocks_of(uint32_t tokens, int shift) { return int((tokens + (1u << shift) - 1) >> shift); }

struct TableArgs {
    int max_seqs, max_blocks, n_blocks, shift;  // block_tokens = 1 << shift
    int32_t *blocks, *len, *free_blocks, *n_free;
};

__global__ void __launch_bounds__(256) reset_kernel(TableArgs t) {
    const int64_t step = int64_t(gridDim.x) * 256, at = int64_t(blockIdx.x) * 256 + threadIdx.x;
    for (int64_t i = at; i < int64_t(t.max_seqs) * t.max_blocks; i += step) t.blocks[i] = -1;
    for (int64_t i = at; i < t.n_blocks; i += step) t.free_blocks[i] = t.n_blocks - 1 - int(i);
    for (int64_t i = at; i < t.max_seqs; i += step) t.len[i] = 0;
    if (at == 0) *t.n_free = t.n_blocks;
}

// The row of the table that batch entry i means, or -1 if it is out of range
// or an earlier entry means it too. owner: LDS, max_seqs words; one barrier
// before the answers.
template <int NT>
VH_DEV void claim(const int32_t *ids, int n, int max_seqs, int *owner) {
    for (int s = threadIdx.x; s < max_seqs; s += NT) owner[s] = n;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT) {
        const int id = ids ? ids[i] : i;
        if (id >= 0 && id < max_seqs) atomicMin(&owner[id], i);
    }
    __syncthreads();
}
VH_DEV int claimed(const int32_t *ids, int i, int max_seqs, const int *owner) {
    const int id = ids ? ids[i] : i;
    return id >= 0 && id < max_seqs && owner[id] == i ? id : -1;
}

// what extend knows of each sequence when it numbers rows and hands out blocks
struct Seq {
    int32_t row;       // of the table; -1: refused
    uint32_t base;     // tokens before
    int32_t have;      // blocks before; -1: not a sequence (its rows get position 0)
    uint32_t off;      // blocks taken by earlier sequences
};

// Positions and slots of rows r0, r0 + NT, ..., four at a time so that their loads
// are in flight together; blocks of before from the table, new ones from the stack
// below `top`.
template <int NT>
VH_DEV void number_rows(const TableArgs &t, const uint32_t *start, const Seq *seq, int n, int top, int max_rows,
                        int32_t *positions, int32_t *slots) {
    constexpr int U = 4;
    const int mask = (1 << t.shift) - 1;
    for (int r0 = threadIdx.x; r0 < max_rows; r0 += U * NT) {
        int pos[U];
        const int32_t *from[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t r = uint32_t(r0 + NT * u);
            pos[u] = 0;
            from[u] = nullptr;
            if (r < start[n] && r < uint32_t(max_rows)) {
                const int i = find(start, n, r);
                const Seq s = seq[i];
                if (s.have >= 0) pos[u] = int(s.base + (r - start[i]));
                const int b = pos[u] >> t.shift;
                if (s.row >= 0)
                    from[u] = b < s.have ? t.blocks + size_t(s.row) * t.max_blocks + b
                                         : t.free_blocks + (top - 1 - int(s.off + uint32_t(b - s.have)));
            }
        }
        int blk[U];
#pragma unroll
        for (int u = 0; u < U; u++) blk[u] = from[u] ? *from[u] : 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = r0 + NT * u;
            if (r >= max_rows) break;
            positions[r] = pos[u];
            slots[r] = from[u] ? (blk[u] << t.shift) + (pos[u] & mask) : -1;
        }
    }
}

// One workgroup. Every entry's status, the prefix sums of rows and of blocks,
// new table entries, lengths and the stack's height; then the rows' positions
// and slots, if they are few (rows_here). LDS: owner [max_seqs], start [n + 1],
// blocks' prefix sums [n + 1], Seq [n].
template <int NT>
__global__ void __launch_bounds__(NT) extend_kernel(TableArgs t, const int32_t *__restrict__ ids,
                                                          const int32_t *__restrict__ n_new, int n, int max_rows,
                                                          int32_t *__restrict__ start_out, int32_t *__restrict__ positions,
                                                          int32_t *__restrict__ slots, int32_t *__restrict__ status,
                                                          bool rows_here) {
    extern __shared__ uint32_t lds[];
    __shared__ uint32_t wsum[2][2][NT / 64];
    __shared__ uint32_t taken;
    int *owner = reinterpret_cast<int *>(lds);
    uint32_t *start = lds + t.max_seqs, *bsum = start + n + 1;
    Seq *seq = reinterpret_cast<Seq *>(bsum + n + 1);
    const int tid = threadIdx.x;
    const int n_free = min(max(*t.n_free, 0), t.n_blocks);
    if (tid == 0) taken = 0;
    claim<NT>(ids, n, t.max_seqs, owner);
    uint32_t rows = 0, blocks = 0;  // of the chunks before
    for (int c = 0; c < n; c += NT) {
        const int i = c + tid;
        int row = -1, st = -EINVAL, need = 0, have = 0;
        uint32_t grow = 0, base = 0;
        if (i < n) {
            row = claimed(ids, i, t.max_seqs, owner);
            const int want = n_new ? n_new[i] : 1;
            if (want >= 0) grow = uint32_t(want);
            if (row >= 0 && want >= 0) {
                base = uint32_t(max(t.len[row], 0));
                have = blocks_of(base, t.shift);
                st = 0;
            }
        }
        uint32_t all;
        const uint32_t r0 = add_sat(rows, block_scan<NT>(grow, wsum[0][(c / NT) & 1], &all));
        rows = add_sat(rows, all);
        if (st == 0) {
            const uint32_t to = add_sat(base, grow);
            if (blocks_of(to, t.shift) > t.max_blocks || add_sat(r0, grow) > uint32_t(max_rows)) st = -E2BIG;
            else need = blocks_of(to, t.shift) - have;
        }
        const uint32_t b0 = add_sat(blocks, block_scan<NT>(uint32_t(need), wsum[1][(c / NT) & 1], &all));
        blocks = add_sat(blocks, all);
        if (st == 0 && need > 0 && add_sat(b0, uint32_t(need)) > uint32_t(n_free)) st = -ENOSPC, need = 0;
        if (i < n) {
            start[i] = r0;
            start_out[i] = int32_t(r0);
            status[i] = st;
            seq[i] = Seq{st == 0 ? row : -1, base, st == -EINVAL ? -1 : have, b0};
            bsum[i] = b0;
            if (st == 0) {
                t.len[row] = int32_t(base + grow);
            }
        }
        // the wave's largest first: lanes' atomics on one word run one after another
        const uint32_t upto = wave_max_u(st == 0 && need > 0 ? b0 + uint32_t(need) : 0u);
        if (lane_id() == 0 && upto) atomicMax(&taken, upto);
    }
    if (tid == 0) {
        start[n] = rows;
        start_out[n] = int32_t(rows);
        bsum[n] = blocks;
    }
    __syncthreads();
    if (tid == 0 && taken) *t.n_free = n_free - int(taken);
    // new table entries: the sequences that took blocks hold the first `taken` of the prefix sums
    for (uint32_t b = tid; b < taken; b += NT) {
        const int i = find(bsum, n, b);
        const Seq s = seq[i];
        if (s.row >= 0)
            t.blocks[size_t(s.row) * t.max_blocks + s.have + int(b - s.off)] = t.free_blocks[n_free - 1 - int(b)];
    }
    if (rows_here) number_rows<NT>(t, start, seq, n, n_free, max_rows, positions, slots);
}

// Positions and slots of many rows, after extend_kernel has filled the table.
// Each workgroup has the batch's row numbers in LDS and takes kRowsPerGroup rows.
constexpr int kRowsPerGroup = 256;
__global__ void __launch_bounds__(kRowsPerGroup) rows_kernel(TableArgs t, const int32_t *__restrict__ ids, int n, int max_rows,
                                                   const int32_t *__restrict__ start_in,
                                                   const int32_t *__restrict__ status, int32_t *__restrict__ positions,
                                                   int32_t *__restrict__ slots) {
    extern __shared__ uint32_t start[];
    for (int i = threadIdx.x; i <= n; i += kRowsPerGroup) start[i] = uint32_t(start_in[i]);
    __syncthreads();
    if (blockIdx.x * kRowsPerGroup + threadIdx.x >= uint32_t(max_rows)) return;
    const int r = blockIdx.x * kRowsPerGroup + threadIdx.x;
    int pos = 0, slot = -1;
    if (uint32_t(r) < start[n]) {
        const int i = find(start, n, uint32_t(r)), st = status[i];
        if (st != -EINVAL) {  // a refused sequence's length is the one before
            const int id = ids ? ids[i] : i;
            pos = max(t.len[id], 0) - (st == 0 ? int(start[i + 1] - start[i]) : 0) + (r - int(start[i]));
            if (st == 0)
                slot = (t.blocks[size_t(id) * t.max_blocks + (pos >> t.shift)] << t.shift) +
                       (pos & ((1 << t.shift) - 1));
        }
    }
    positions[r] = pos;
    slots[r] = slot;
}

// One workgroup: the blocks that the batch's sequences give back, numbered in
// the batch's order and in the order of positions, go on the stack in reverse
// (the first on top). LDS: owner [max_seqs], prefix sums [n + 1], Seq [n].
template <int NT>
__global__ void __launch_bounds__(NT) truncate_kernel(TableArgs t, const int32_t *__restrict__ ids,
                                                            const int32_t *__restrict__ new_len, int n) {
    extern __shared__ uint32_t lds[];
    __shared__ uint32_t wsum[2][NT / 64];
    int *owner = reinterpret_cast<int *>(lds);
    uint32_t *bsum = lds + t.max_seqs;
    Seq *seq = reinterpret_cast<Seq *>(bsum + n + 1);
    const int tid = threadIdx.x;
    const int n_free = *t.n_free;
    claim<NT>(ids, n, t.max_seqs, owner);
    uint32_t blocks = 0;
    for (int c = 0; c < n; c += NT) {
        const int i = c + tid;
        int row = -1, keep = 0, have = 0;
        if (i < n) {
            row = claimed(ids, i, t.max_seqs, owner);
            const int to = new_len ? new_len[i] : 0;
            if (row >= 0 && to >= 0) {
                const int len = t.len[row];
                if (len > to) {
                    t.len[row] = to;
                    have = min(blocks_of(uint32_t(len), t.shift), t.max_blocks);
                    keep = min(blocks_of(uint32_t(to), t.shift), have);
                }
            }
        }
        uint32_t all;
        const uint32_t b0 = add_sat(blocks, block_scan<NT>(uint32_t(have - keep), wsum[(c / NT) & 1], &all));
        blocks = add_sat(blocks, all);
        if (i < n) {
            bsum[i] = b0;
            seq[i] = Seq{row, 0u, keep, b0};
        }
    }
    if (tid == 0) bsum[n] = blocks;
    __syncthreads();
    // a table that the caller filled may name blocks more often than there are any: the stack's end is its limit
    const int room = max(t.n_blocks - max(n_free, 0), 0), total = int(min(blocks, uint32_t(room)));
    for (int b = tid; b < total; b += NT) {
        const Seq s = seq[find(bsum, n, uint32_t(b))];
        t.free_blocks[max(n_free, 0) + total - 1 - b] =
            t.blocks[size_t(s.row) * t.max_blocks + s.have + (b - int(s.off))];
    }
    if (tid == 0 && total) *t.n_free = max(n_free, 0) + total;
}

// One workgroup: cut the batch into items. A sequence of u units (kPagedUnit
// tokens; an empty one has one, of no tokens) gets ceil(u / S) items and its units are dealt evenly over them. S is
// the batch's units / `whole`, or up to an eighth more, if the items then number
// at most `whole`: each CU has one, and they end together. Sequences that do not
// divide so (short ones beside long ones) are cut finer, S = units / `fine`, so that
// workgroups that end early take up others: 131 071 tokens alone 98 us (2 layers)
// whole and 125 fine; 64 sequences of 500 to 30 001 tokens 465 to 490 and 329, 23 of 1 to
// 8 191 67 and 54 (2 layers). With the first kernels 16 equal sequences took 79 and 84, and between
// the two 131 071 tokens 113 at 512, 121 at 1 024 and 162 at 4 096 workgroups (111 whole), the 64
// sequences 396, 364 and 354 (353 fine).
// LDS: items' prefix sums [n + 1], tokens [n], rows [n].
template <int NT>
__global__ void __launch_bounds__(NT) plan_kernel(TableArgs t, const int32_t *__restrict__ ids, int n, int whole,
                                                        int fine, int list_blocks, PlanHead *__restrict__ head,
                                                        PlanSeq *__restrict__ seqs,
                                                        int32_t *__restrict__ first, PlanItem *__restrict__ items,
                                                        uint32_t *__restrict__ arrivals, int n_arrivals, uint32_t tag) {
    extern __shared__ uint32_t lds[];
    __shared__ uint32_t wsum[2][2][NT / 64], many[3][NT / 64];
    uint32_t *fst = lds, *tok = fst + n + 1;
    int *rw = reinterpret_cast<int *>(tok + n);
    const int tid = threadIdx.x;
    const uint32_t most = uint32_t(t.max_blocks) << t.shift;
    uint32_t total = 0;
    for (int c = 0; c < n; c += NT) {
        const int i = c + tid;
        uint32_t tokens = 0;
        if (i < n) {
            const int id = ids ? ids[i] : i;
            const bool ok = id >= 0 && id < t.max_seqs;
            if (ok) tokens = min(uint32_t(max(t.len[id], 0)), most);
            const int blocks = blocks_of(tokens, t.shift);
            if (list_blocks) tokens = uint32_t(min(blocks, list_blocks)) << t.shift;
            tok[i] = tokens;
            rw[i] = ok ? id : 0;
            seqs[i] = PlanSeq{rw[i], blocks};
        }
        uint32_t all;
        block_scan<NT>((tokens + kPagedUnit - 1) / kPagedUnit, wsum[0][(c / NT) & 1], &all);
        total = add_sat(total, all);
    }
    // the least S of three that gives at most `whole` items
    uint32_t tries[3], mine[3] = {};
    tries[0] = max((total + whole - 1) / whole, 1u);
    tries[1] = tries[0] + (tries[0] + 15) / 16;
    tries[2] = tries[0] + (tries[0] + 7) / 8;
    for (int i = tid; i < n; i += NT) {
        const uint32_t u = (tok[i] + kPagedUnit - 1) / kPagedUnit;
#pragma unroll
        for (int k = 0; k < 3; k++) mine[k] += max((u + tries[k] - 1) / tries[k], 1u);
    }
    // (sums by wave: 64 lanes' atomics on one word run one after another, 5 us for a batch of 64)
#pragma unroll
    for (int k = 0; k < 3; k++) {
        mine[k] = wave_scan_u(mine[k]);
        if (lane_id() == 63) many[k][tid >> 6] = mine[k];
    }
    __syncthreads();
    // (a total that was cut off, of sequences that share most of their blocks, would give more items than there is room
    // for: each sequence gets one)
    uint32_t S = total < kMaxRows ? max((total + fine - 1) / fine, 1u) : 1u << 24;
#pragma unroll
    for (int k = 2; k >= 0; k--) {
        uint32_t m = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; w++) m += many[k][w];
        if (m <= uint32_t(whole)) S = tries[k];
    }
    uint32_t sum = 0;
    for (int c = 0; c < n; c += NT) {
        const int i = c + tid;
        uint32_t k = 0;
        if (i < n) {
            const uint32_t u = max((tok[i] + kPagedUnit - 1) / kPagedUnit, 1u), m = (u + S - 1) / S;
            k = (u + (u + m - 1) / m - 1) / ((u + m - 1) / m);  // items of ceil(u / m) units
        }
        uint32_t all;
        const uint32_t f = sum + block_scan<NT>(k, wsum[1][(c / NT) & 1], &all);
        sum += all;
        if (i < n) {
            fst[i] = f;
            first[i] = int32_t(f);
        }
    }
    if (tid == 0) {
        fst[n] = sum;
        first[n] = int32_t(sum);
        head->tag = tag;
        head->n_items = int32_t(sum);
    }
    __syncthreads();
    for (uint32_t x = tid; x < sum; x += NT) {
        const int i = find(fst, n, x);
        const uint32_t k = fst[i + 1] - fst[i], u = (tok[i] + kPagedUnit - 1) / kPagedUnit, per = (u + k - 1) / k;
        const uint32_t b = (x - fst[i]) * per * kPagedUnit, e = min(b + per * kPagedUnit, tok[i]);
        items[x] = PlanItem{rw[i], int32_t(b), int32_t(e), i, int32_t(fst[i]), int32_t(k), {0, 0}};
    }
    for (int x = tid; x < n_arrivals; x += NT) arrivals[x] = 0;
}

int log2i(int v) {
    int s = 0;
    while ((1 << s) < v) s++;
    return s;
}

TableArgs args_of(const vireo_paged_table *t) {
    return TableArgs{t->max_seqs, t->max_blocks, t->n_blocks, log2i(t->block_tokens),
                     t->blocks,   t->len,        t->free_blocks, t->n_free};
}

// LDS beyond 64 KB has to be asked for, per kernel and device
template <class F>
int allow_lds(F *f, size_t bytes) {
    if (bytes <= 65536) return 0;
    return vh_check(hipFuncSetAttribute(reinterpret_cast<const void *>(f), hipFuncAttributeMaxDynamicSharedMemorySize,
                                        int(bytes)));
}

// Items that a plan aims at per kv head (and tile of 16 query heads): whole, one
// workgroup per CU over all of them; fine, eight.
int plan_slots(const vireo_paged_plan *p, int groups) {
    const int s = groups / (p->n_kv_heads * vh_plan_head_tiles(p));
    return s > 1 ? s : 1;
}
constexpr int kWholeGroups = 256, kFineGroups = 2048;

}  // namespace

int vh_plan_head_tiles(const vireo_paged_plan *p) { return (p->n_heads / p->n_kv_heads + 15) / 16; }

bool vh_plan_ok(const vireo_paged_plan *p) {
    return p && vh_table_ok(p->table) && p->n >= 1 && p->n <= kPagedMaxSeqs && p->n_kv_heads >= 1 && p->n_heads >= 1 &&
           p->n_heads <= 4096 && p->n_heads % p->n_kv_heads == 0 &&
           (p->head_size == 64 || p->head_size == 128 || p->head_size == 256) && p->list_blocks >= 0 &&
           int64_t(p->list_blocks) * p->table->block_tokens < (int64_t(1) << 31);
}

PlanView vh_plan_view(const vireo_paged_plan *p) {
    PlanView v{};
    char *m = static_cast<char *>(p->mem);
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        char *q = m + at;
        at += (bytes + 255) & ~int64_t(255);
        return q;
    };
    // no more items than units that the table (or the lists) can hold
    const int64_t most = p->list_blocks && p->list_blocks < p->table->max_blocks ? p->list_blocks : p->table->max_blocks;
    const int64_t each = (most * p->table->block_tokens + kPagedUnit - 1) / kPagedUnit, units = each * p->n;
    v.cap = int(units < plan_slots(p, kFineGroups) + p->n ? units : plan_slots(p, kFineGroups) + p->n);
    v.head = reinterpret_cast<PlanHead *>(take(sizeof(PlanHead)));
    v.seqs = reinterpret_cast<PlanSeq *>(take(int64_t(p->n) * sizeof(PlanSeq)));
    v.first = reinterpret_cast<int32_t *>(take(int64_t(p->n + 1) * 4));
    v.items = reinterpret_cast<PlanItem *>(take(int64_t(v.cap) * sizeof(PlanItem)));
    v.keys = reinterpret_cast<uint32_t *>(
        take(p->list_blocks ? int64_t(p->n) * p->n_kv_heads * p->table->max_blocks * 4 : 0));
    v.ml = reinterpret_cast<float2 *>(take(int64_t(v.cap) * p->n_heads * 8));
    v.part = reinterpret_cast<float *>(take(int64_t(v.cap) * p->n_heads * p->head_size * 4));
    const int hpg = p->n_heads / p->n_kv_heads;
    v.join = each <= kJoinUnits && each * (hpg < 16 ? hpg : 16) <= kJoinHeads;
    if (v.join)
        v.arrivals = reinterpret_cast<uint32_t *>(take(int64_t(p->n) * p->n_kv_heads * vh_plan_head_tiles(p) * 4));
    v.bytes = at;
    // of the shapes that the memory's layout and its indexes follow from
    uint32_t h = 0x9e3779b9u;
    for (int x : {p->n, p->n_heads, p->n_kv_heads, p->head_size, p->list_blocks, p->table->max_seqs,
                  p->table->max_blocks, p->table->block_tokens})
        h = (h ^ uint32_t(x)) * 0x01000193u + 0x7f4a7c15u;
    v.tag = h;
    return v;
}

extern "C" int vireo_paged_reset(const vireo_paged_table *t, void *stream) {
    if (!vh_table_ok(t)) return -EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t most = int64_t(t->max_seqs) * t->max_blocks > t->n_blocks ? int64_t(t->max_seqs) * t->max_blocks
                                                                            : int64_t(t->n_blocks);
    const int64_t groups = (most + 1023) / 1024;
    hipLaunchKernelGGL(reset_kernel, dim3(unsigned(groups < 2048 ? groups : 2048)), dim3(256), 0, s, args_of(t));
    return vh_finish(s, vh_check(hipGetLastError()));
}

extern "C" int vireo_paged_extend(const vireo_paged_table *t, const int32_t *ids, const int32_t *n_new, int n,
                                  int max_rows, int32_t *start, int32_t *positions, int32_t *slots, int32_t *status,
                                  void *stream) {
    if (!vh_table_ok(t) || n < 0 || n > t->max_seqs || max_rows < 0 || !start || (n > 0 && !status) ||
        (max_rows > 0 && (!positions || !slots)))
        return -EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const TableArgs a = args_of(t);
    const bool here = max_rows <= kRowsHere;
    const size_t lds = 4 * size_t(t->max_seqs) + 8 * size_t(n + 1) + sizeof(Seq) * size_t(n);
    if (n <= kFewThreads && max_rows <= kFewThreads && t->max_seqs <= kThreads) {
        hipLaunchKernelGGL(extend_kernel<kFewThreads>, dim3(1), dim3(kFewThreads), lds, s, a, ids, n_new, n, max_rows,
                           start, positions, slots, status, here);
    } else {
        if (int rc = allow_lds(extend_kernel<kThreads>, lds)) return rc;
        hipLaunchKernelGGL(extend_kernel<kThreads>, dim3(1), dim3(kThreads), lds, s, a, ids, n_new, n, max_rows, start,
                           positions, slots, status, here);
    }
    if (!here)
        hipLaunchKernelGGL(rows_kernel, dim3((uint32_t(max_rows) + kRowsPerGroup - 1) / kRowsPerGroup), dim3(kRowsPerGroup),
                           4 * size_t(n + 1), s, a, ids, n, max_rows, start, status, positions, slots);
    return vh_finish(s, vh_check(hipGetLastError()));
}

extern "C" int vireo_paged_truncate(const vireo_paged_table *t, const int32_t *ids, const int32_t *new_len, int n,
                                    void *stream) {
    if (!vh_table_ok(t) || n < 0 || n > t->max_seqs) return -EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (n == 0) return vh_finish(s, 0);
    const size_t lds = 4 * size_t(t->max_seqs) + 4 * size_t(n + 1) + sizeof(Seq) * size_t(n);
    if (n <= kFewThreads && t->max_seqs <= kThreads) {
        hipLaunchKernelGGL(truncate_kernel<kFewThreads>, dim3(1), dim3(kFewThreads), lds, s, args_of(t), ids, new_len, n);
    } else {
        if (int rc = allow_lds(truncate_kernel<kThreads>, lds)) return rc;
        hipLaunchKernelGGL(truncate_kernel<kThreads>, dim3(1), dim3(kThreads), lds, s, args_of(t), ids, new_len, n);
    }
    return vh_finish(s, vh_check(hipGetLastError()));
}

extern "C" int64_t vireo_paged_plan_bytes(const vireo_paged_plan *p) {
    if (!vh_plan_ok(p)) return -EINVAL;
    return vh_plan_view(p).bytes;
}

extern "C" int vireo_paged_plan_update(const vireo_paged_plan *p, void *stream) {
    if (!vh_plan_ok(p) || !p->mem || (reinterpret_cast<uintptr_t>(p->mem) & 255u)) return -EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const PlanView v = vh_plan_view(p);
    const size_t lds = 4 * size_t(p->n + 1) + 8 * size_t(p->n);
    const int n_arrivals = v.join ? p->n * p->n_kv_heads * vh_plan_head_tiles(p) : 0;
    const int whole = plan_slots(p, kWholeGroups), fine = plan_slots(p, kFineGroups);
    if (p->n <= kFewThreads)
        hipLaunchKernelGGL(plan_kernel<kFewThreads>, dim3(1), dim3(kFewThreads), lds, s, args_of(p->table), p->ids, p->n,
                           whole, fine, p->list_blocks, v.head, v.seqs, v.first, v.items,
                           v.arrivals, n_arrivals, v.tag);
    else
        hipLaunchKernelGGL(plan_kernel<kThreads>, dim3(1), dim3(kThreads), lds, s, args_of(p->table), p->ids, p->n,
                           whole, fine, p->list_blocks, v.head, v.seqs, v.first, v.items,
                           v.arrivals, n_arrivals, v.tag);
    return vh_finish(s, vh_check(hipGetLastError()));
}
