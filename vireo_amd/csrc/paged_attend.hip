// Attention of one new token per sequence over the paged cache (API:
// include/vireo_paged.h), split over the sequences' lengths and joined.
//
//   out = sum_t e^(s_t - M) v_t / sum_t e^(s_t - M),  s_t = scale q . k_t,  M = max s_t
//
// A workgroup takes one item of the plan (a run of one sequence's tokens) and
// one kv head with up to 16 of its query heads; its four waves take a quarter
// of the run's 32-token tiles each. Per tile, all in registers:
//
//   S^T = K Q^T   v_mfma 16x16x32: rows are 16 tokens, columns the 16 heads, the
//                 32 a run of head dimensions. Two such products make the tile:
//                 row r of product u is token 8 (r / 4) + 4 u + r % 4, so the four
//                 results of a lane from each are its head's scores of tokens
//                 8 g .. 8 g + 7 (g = lane / 16).
//   weights       an online softmax: the running maximum over the head's four
//                 lanes, e^(scale (s - m)) in fp32, the sum per lane.
//   O^T += V^T P^T  rows are 16 dimensions, columns the heads, the 32 the tile's
//                 tokens: the lane's 8 weights are its operand as they stand, and 16
//                 consecutive bytes of the cache (8 tokens of a dimension) are V^T's.
//
// No weight, key or value passes through LDS or another lane; that is why
// values lie dimension by dimension in their block. Keys are requested again as
// soon as the scores are formed and values as soon as they are weighed, so a
// wave has a tile of 64 hs bytes in flight nearly all the time. They are read
// once, with the non-temporal hint: 64 sequences of 500 to 30 001 tokens (1.9 GB)
// 343 -> 318 us (324 with what came later, 6.0 TB/s) - but for the values of blocks of 64 slots and more, whose lines
// two tiles share (16 sequences, 275 MB: 78 us with the hint, 67 without; 60 in
// blocks of 16 and 32). Bound by that read; the matrix cores are busy for 8 % of the
// time for the 64 sequences (16-bit queries).
//
// Precision: products of 16-bit parts are exact in the matrix cores and their
// sums fp32 (fp16 values below 2^-14 are not flushed, but their products are added
// as if they were that large: absolute errors of 2^-38 of the largest weight). An fp32
// query is the sum of three truncated 16-bit parts (under a power of two per
// head: Queries), and so is a weight, whatever the result's type: a result is rounded
// once. (Two parts hold 16 bits of a weight in bf16; truncated, they took some results
// past a border between two bf16 values. The third part's products cost nothing beside
// the read: 64 sequences 329.4 us with two and 328.4 with three, 131 071 tokens alone
// 97.2 and 97.4.) The sum of weights is of the fp32 values. Over fp16 a query's value is
// cut off at 2^-38 of the head's largest, a weight at 2^-38 of the largest that its wave
// has seen. Infinite keys and values meet parts that are 0, whose products are NaN:
// where a wave finds a NaN in its sums it goes over its tiles again, with the least
// value of its sign in place of such parts of a query's value (in every call that would
// be seen beside large keys), and with weights that are all the same.
//
// Waves merge through LDS. A sequence of one item is then written; others' partial
// results are joined in the items' order, so that the bits are the same every time:
// by a second launch (merge_kernel), or, where a sequence can have but few units
// (short tables and lists of blocks: paged.h), by the last workgroup to arrive. Its
// inputs are stored and loaded past the dies' L2s (sc1), each store completed before
// its workgroup counts as arrived: a release fence instead would write back the L2.
#include <hip/hip_runtime.h>
#include <errno.h>
#include <math.h>
#include "paged.h"

namespace {

constexpr float kLowest = -3.4028234663852886e38f;

struct AttendArgs {
    const uint16_t *k, *v;
    int n_blocks, n_kv, shift;  // block_tokens = 1 << shift
    const int32_t *table, *len;
    int max_blocks;
    const int32_t *lists;  // or null
    int list_blocks;
    const void *q;
    int64_t q_stride;
    float mant;  // scale log2(e) = mant 2^expo: scores in powers of two
    int expo;
    int n_heads, hpg, tiles;  // query heads, of a kv head, tiles of 16 of those
    void *out;
    int64_t out_stride;
    uint32_t type;  // of q and out
    PlanHead *head;
    const PlanItem *items;
    const int32_t *first;
    uint32_t tag;
    float *part;
    float2 *ml;
    uint32_t *arrivals;  // or null: merge_kernel joins the items
};

// the wave's value of lane l's v (l the same on every lane)
VH_DEV int at_lane(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
// What an output is multiplied by at the end: nothing attended, zeros; every
// score -inf (no weight at all), a NaN, as the softmax of them is.
VH_DEV float inverse(float M, float L) {
    return M == -INFINITY ? 0.0f : L == 0.0f ? __builtin_nanf("") : 1.0f / L;
}

// four results
template <uint32_t T, bool QF>
VH_DEV void store4(void *out, int64_t at, f32x4 y) {
    if constexpr (QF)
        *reinterpret_cast<f32x4 *>(static_cast<float *>(out) + at) = y;
    else
        *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(out) + at) = u32x2{El<T>::pack(y[0], y[1]), El<T>::pack(y[2], y[3])};
}

// D: head size; T: the cache's type; QF: fp32 queries and results (else T's);
// ONCE: blocks of 16 or 32 slots, whose lines of values belong to one tile
template <int D, uint32_t T, bool QF, bool ONCE>
__global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) attend_kernel(AttendArgs a) {
    constexpr int KS = D / 32, DT = D / 16;              // steps of a score, 16-dimension tiles of an output
    constexpr int QP = Queries<D, T, QF>::P;             // parts of a query
    constexpr int WP = 3;                                // parts of a weight
    constexpr int RS = D + 4;                            // LDS row of a head: its 16 lanes on different banks
    __shared__ __align__(16) float red[4][16][RS];
    __shared__ float2 wml[4][16];
    // heads vary fastest: a block's kv heads are neighbours in memory, and the
    // plan's unused items come last
    const int item = blockIdx.y, hg = blockIdx.x;
    const uint32_t tag = a.head->tag;
    const int n_items = a.head->n_items;
    const PlanItem it = a.items[item];
    if (tag != a.tag || item >= n_items) return;  // not this plan's split, or not an item of it
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int g = hg / a.tiles, z = hg - g * a.tiles;
    const int seq = it.seq, h0 = g * a.hpg + z * 16, nh = min(16, a.hpg - z * 16);
    const int shift = a.shift, G = 1 << shift;

    // the queries: column col's head, dimensions 32 s + 8 grp .. + 7 of step s
    // (formed below, once the first keys and values are requested too)
    Queries<D, T, QF> query;
    const int64_t q0 = seq * a.q_stride + int64_t(h0 + min(col, nh - 1)) * D + 8 * grp;
    query.load(a.q, q0);

    // the wave's tiles, and the blocks behind them, 64 at a time: lane e holds
    // block e0 + e of the sequence (or of its list) and how many of its slots
    // are attended (0: not a block)
    const int T0 = (it.end - it.begin + 31) >> 5;
    const int i0 = T0 * wv / 4, i1 = T0 * (wv + 1) / 4;
    const int32_t *tab = a.table + size_t(it.row) * a.max_blocks;
    const int length = a.lists ? a.len[it.row] : 0;
    const int32_t *list = a.lists ? a.lists + (size_t(seq) * a.n_kv + g) * a.list_blocks : nullptr;
    int e0 = 0, blk = 0, cnt = 0;
    auto blocks_from = [&](int e) {
        e0 = e;
        const int mine = e + lane;
        int b = -1, n = 0;
        if (int64_t(mine) << shift < it.end) {
            b = mine;
            n = min(G, it.end - (mine << shift));
            if (list) {
                b = list[mine];
                n = b >= 0 && b < a.max_blocks ? min(max(length - (b << shift), 0), G) : 0;
            }
        }
        blk = n > 0 ? tab[b] : -1;
        cnt = blk >= 0 && blk < a.n_blocks ? n : 0;
        if (cnt == 0) blk = 0;
    };
    // tile i's two 16-token halves: the blocks they lie in, and where in them (a
    // tile has at most two blocks of 16 slots)
    const size_t head_tile = size_t(D) << shift;  // elements of a block of one kv head
    struct Where {
        size_t base[2];  // element of the half's block
        int off[2];      // its first slot
        int n[2];        // its slots that are attended, of 16
    };
    auto where = [&](int i) {
        Where w;
        const int t = it.begin + 32 * i;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int tu = t + 16 * u, e = (tu >> shift) - e0;
            w.off[u] = tu & (G - 1);
            w.base[u] = (size_t(at_lane(blk, e)) * a.n_kv + g) * head_tile;
            w.n[u] = min(max(at_lane(cnt, e) - w.off[u], 0), 16);
        }
        return w;
    };
    // the lane's rows of K: row r = col of product u is token 8 (r / 4) + 4 u + r % 4 of the tile
    const int kt = 8 * ((col >> 2) & 1) + (col & 3), khalf = col >> 3;
    u32x4 kk[2][KS], vv[DT];
    auto load_k = [&](const Where &w) {
        const size_t base = khalf ? w.base[1] : w.base[0];
        const int off = khalf ? w.off[1] : w.off[0];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const uint16_t *p = a.k + base + size_t(off + kt + 4 * u) * D + 8 * grp;
#pragma unroll
            for (int s = 0; s < KS; s++) kk[u][s] = ldu4_once(p + 32 * s);
        }
    };
    auto load_v = [&](const Where &w) {
        const size_t base = grp >> 1 ? w.base[1] : w.base[0];
        const int off = (grp >> 1 ? w.off[1] : w.off[0]) + 8 * (grp & 1);
        const uint16_t *p = a.v + base + (size_t(col) << shift) + off;
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const uint16_t *pd = p + (size_t(16 * d) << shift);
            vv[d] = ONCE ? ldu4_once(pd) : ldu4(pd);
        }
    };

    float m, l;
    bool seen = false;  // a token was attended
    f32x4 acc[DT];
    Where w;
    u32x4 qw[QP][KS];
    float two, c;
    // the lane's 8 scores of the tile in kk
    auto scores = [&](float (&x)[8]) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int p = QP - 1; p >= 0; p--)
#pragma unroll
                for (int k = 0; k < KS; k++) s = El<T>::mfma(kk[u][k], qw[p][k], s);
#pragma unroll
            for (int j = 0; j < 4; j++) x[4 * u + j] = s[j];
        }
    };
    // no score and no value for slots that are not attended: what lies there is not to meet a weight of 0, it may be
    // an infinity or a NaN
    auto mask = [&](const Where &w, float (&x)[8]) {
        if (w.n[0] == 16 && w.n[1] == 16) return;  // the same on every lane
        // slots of the lane's 8 that are attended
        const int nv = min(max((grp >> 1 ? w.n[1] : w.n[0]) - 8 * (grp & 1), 0), 8);
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = j < nv ? x[j] : -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t keep = nv >= 2 * j + 2 ? 0xffffffffu : nv == 2 * j + 1 ? 0xffffu : 0u;
#pragma unroll
            for (int d = 0; d < DT; d++) vv[d][j] &= keep;
        }
    };
    // a weight, the largest 2^up (the difference before the scale: a large score's rounding would be an exponent)
    auto weight = [&](float x, float up) { return __builtin_amdgcn_exp2f(fmaf(x - m, c, up)); };
    // fp16: so that the parts of small ones keep their bits; bf16: so that sums of the largest values stay in fp32
    constexpr float kUp = T == VIREO_PAGED_F16 ? 14.0f : -24.0f;
    for (bool again = false;; again = true) {
        m = kLowest, l = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) acc[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        blocks_from((it.begin + 32 * i0) >> shift);
        w = where(i0);  // i0 < T0 but where T0 = 0; a wave without tiles reads one that it does not use
        load_k(w);
        load_v(w);
        __builtin_amdgcn_sched_barrier(0);
        int e;
        if (QF && again) {
            query.load(a.q, q0);
            e = query.template parts<true>(qw);
        } else {
            e = query.template parts<false>(qw);
        }
        // Neither 0, which would make a NaN of a slot's -inf, nor infinite. Products with the queries are below 2^40 where
        // scale 2^-e lies under 2^-126: all weights are the same either way.
        two = ldexpf(1.0f, min(max(a.expo - e, -126), 126)), c = a.mant * two;
        for (int i = i0; i < i1; i++) {
            float x[8];
            scores(x);
            const bool more = i + 1 < i1;
            Where next = w;
            if (more) {
                if (((it.begin + 32 * i + 63) >> shift) - e0 >= 64) blocks_from((it.begin + 32 * (i + 1)) >> shift);
                next = where(i + 1);
                load_k(next);
            }
            seen |= w.n[0] + w.n[1] > 0;
            mask(w, x);
            float mx = x[0];
#pragma unroll
            for (int j = 1; j < 8; j++) mx = fmaxf(mx, x[j]);
            const float mn = fmaxf(m, head_max(mx));
            const float cr = __builtin_amdgcn_exp2f((m - mn) * c);
            m = mn;
            float ps = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[j] = weight(x[j], kUp);
                ps += x[j];
            }
            l = fmaf(l, cr, ps);
            u32x4 pw[WP];
            split8<T, WP, false>(x, pw);
#pragma unroll
            for (int d = 0; d < DT; d++) acc[d] *= cr;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int p = WP - 1; p >= 0; p--) acc[d] = El<T>::mfma(vv[d], pw[p], acc[d]);
            w = next;
            if (more) load_v(w);
        }
        // A NaN may be an infinite key's, with a part of a query's value that is 0: once more, without such parts.
        if (!QF || again || !__any(l != l)) break;
    }
    // A NaN may be an infinite value's, under a weight of which a part is 0: what such values (and NaN) come to under
    // weights that are all the same, or 0, takes its place. Rare, and looked for once: 8 to 32 comparisons a wave.
    bool odd = false;
#pragma unroll
    for (int d = 0; d < DT; d++)
        odd |= __builtin_isunordered(acc[d][0], acc[d][1]) || __builtin_isunordered(acc[d][2], acc[d][3]);
    if (__any(odd)) {
        // the results so far are put aside: they would take registers that the loop above could not have
        float *aside = &red[wv][col][4 * grp];
#pragma unroll
        for (int d = 0; d < DT; d++) {
            *reinterpret_cast<f32x4 *>(aside + 16 * d) = acc[d];
            acc[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        blocks_from((it.begin + 32 * i0) >> shift);
        for (int i = i0; i < i1; i++) {
            if (((it.begin + 32 * i + 31) >> shift) - e0 >= 64) blocks_from((it.begin + 32 * i) >> shift);
            w = where(i);
            load_k(w);
            float x[8];
            scores(x);
            __builtin_amdgcn_sched_barrier(0);  // values into the keys' registers: no more of them than in the loop above
            load_v(w);
            mask(w, x);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[j] = weight(x[j], 0.0f);
                x[j] = x[j] > 0.0f ? (T == VIREO_PAGED_F16 ? 1.0f : 0x1p-24f) : x[j];  // a NaN stays one
            }
            u32x4 pw;
#pragma unroll
            for (int j = 0; j < 4; j++) pw[j] = El<T>::pack(x[2 * j], x[2 * j + 1]);
#pragma unroll
            for (int d = 0; d < DT; d++) acc[d] = El<T>::mfma(vv[d], pw, acc[d]);
        }
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const f32x4 y = *reinterpret_cast<const f32x4 *>(aside + 16 * d);
#pragma unroll
            for (int j = 0; j < 4; j++) acc[d][j] = y[j] != y[j] && !(fabsf(acc[d][j]) < INFINITY) ? acc[d][j] : y[j];
        }
    }
    l = head_sum(l);
    if (T == VIREO_PAGED_F16) l = l * 0x1p-14f;
    // the waves' maxima, from here on in units of the scale's mantissa (exact, so that those of equal scores stay
    // equal); -inf marks a wave that attended nothing
    if (grp == 0) wml[wv][col] = make_float2(seen ? fmaxf(m * two, kLowest) : -INFINITY, l);
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) M = fmaxf(M, wml[w][col].x);
    float f = 0.0f;
    if (M > -INFINITY) {
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float2 o = wml[w][col];
            const float fw = __builtin_amdgcn_exp2f((o.x - M) * a.mant);
            L = fmaf(o.y, fw, L);
            f = w == wv ? fw : f;
        }
    }
    if (T == VIREO_PAGED_F16) f *= 0x1p-14f;
#pragma unroll
    for (int d = 0; d < DT; d++) acc[d] *= f;
    // the first wave adds the others' outputs in order
    if (wv > 0) {
#pragma unroll
        for (int d = 0; d < DT; d++) *reinterpret_cast<f32x4 *>(&red[wv - 1][col][16 * d + 4 * grp]) = acc[d];
    }
    __syncthreads();
    // partials of the sequence's items, for this tile's first head; at most kJoinUnits items where they are joined here
    const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc(
        a.part + (size_t(it.first) * a.n_heads + h0) * D, 0, int(uint32_t(it.count * a.n_heads - h0) * D * 4u), 0x00020000);
    const __amdgpu_buffer_rsrc_t rm = __builtin_amdgcn_make_buffer_rsrc(
        a.ml + size_t(it.first) * a.n_heads + h0, 0, (it.count * a.n_heads - h0) * 8, 0x00020000);
    const int64_t o0 = seq * a.out_stride + int64_t(h0) * D;
    if (wv == 0 && col < nh) {
#pragma unroll
        for (int w = 0; w < 3; w++)
#pragma unroll
            for (int d = 0; d < DT; d++) acc[d] += *reinterpret_cast<const f32x4 *>(&red[w][col][16 * d + 4 * grp]);
        if (it.count == 1) {
            const float inv = inverse(M, L);
#pragma unroll
            for (int d = 0; d < DT; d++) store4<T, QF>(a.out, o0 + col * D + 16 * d + 4 * grp, acc[d] * inv);
        } else if (a.arrivals) {  // past the L2 of this die, which others do not keep coherent (sc1)
            const int at = (item - it.first) * a.n_heads + col;
            if (grp == 0)
                __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(M), __float_as_uint(L)}, rm, at * 8, 0, 16);
#pragma unroll
            for (int d = 0; d < DT; d++)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[d]), rp,
                                                       (at * D + 16 * d + 4 * grp) * 4, 0, 16);
        } else {
            const size_t ph = size_t(item) * a.n_heads + h0 + col;
            if (grp == 0) a.ml[ph] = make_float2(M, L);
#pragma unroll
            for (int d = 0; d < DT; d++) *reinterpret_cast<f32x4 *>(a.part + ph * D + 16 * d + 4 * grp) = acc[d];
        }
    }
    if (it.count == 1 || !a.arrivals) return;
    // The last of the sequence's items to arrive joins them all, in their order.
    __shared__ int last;
    if (wv == 0) {
        __builtin_amdgcn_s_waitcnt(0);  // the stores above have completed
        asm volatile("" ::: "memory");
        if (lane == 0) {
            uint32_t *arrived = a.arrivals + size_t(seq) * gridDim.x + hg;
            last = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == uint32_t(it.count - 1);
            if (last) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
        }
    }
    __syncthreads();
    if (!last) return;
    // D / 4 threads a head, HT heads a thread, U items of each at a time: 8 heads of at most U items in one go
    constexpr int ND = D / 4, NG = 256 / ND, HT = D <= 128 ? 1 : 2, U = D <= 128 ? 8 : 16;
    const int dq = threadIdx.x % ND;
    for (int h = threadIdx.x / ND; h < nh; h += HT * NG) {
        float m1[HT], l1[HT];
        f32x4 y[HT];
#pragma unroll
        for (int x = 0; x < HT; x++) m1[x] = -INFINITY, l1[x] = 0.0f, y[x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int i0 = 0; i0 < it.count; i0 += U) {
            u32x2 ml[HT][U];
            u32x4 v[HT][U];
#pragma unroll
            for (int x = 0; x < HT; x++)
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int at = min(i0 + u, it.count - 1) * a.n_heads + min(h + NG * x, nh - 1);
                    ml[x][u] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rm, at * 8, 0, 16));
                    v[x][u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rp, (at * D + 4 * dq) * 4, 0, 16));
                }
#pragma unroll
            for (int x = 0; x < HT; x++) {
                float big = m1[x];
#pragma unroll
                for (int u = 0; u < U; u++) big = fmaxf(big, __uint_as_float(ml[x][u][0]));  // repeats of the last one too
                if (big == -INFINITY) continue;
                const float back = __builtin_amdgcn_exp2f((m1[x] - big) * a.mant);
                l1[x] *= back;
                y[x] *= back;
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (i0 + u < it.count) {
                        const float f1 = __builtin_amdgcn_exp2f((__uint_as_float(ml[x][u][0]) - big) * a.mant);
                        l1[x] = fmaf(__uint_as_float(ml[x][u][1]), f1, l1[x]);
                        y[x] += __builtin_bit_cast(f32x4, v[x][u]) * f1;
                    }
                m1[x] = big;
            }
        }
#pragma unroll
        for (int x = 0; x < HT; x++)
            if (h + NG * x < nh)
                store4<T, QF>(a.out, o0 + (h + NG * x) * D + 4 * dq, y[x] * inverse(m1[x], l1[x]));
    }
}

// A workgroup per (sequence, head) joins its items: thread i forms the weight of
// item i (256 at a time), groups of D / 4 threads take every NG-th item, four
// dimensions a thread, and are added in order. The first NG U items' outputs are
// requested with the weights' inputs, not after them. One thread per item's
// maximum in turn took 66 us for 256 items of 32 heads, this 6.7 (4.7 for 64).
template <int D, uint32_t T, bool QF>
__global__ void __launch_bounds__(256) merge_kernel(AttendArgs a) {
    constexpr int ND = D / 4, NG = 256 / ND, U = 8;
    __shared__ f32x4 red[NG][ND];
    __shared__ float fs[256], wm[4], wl[4];
    const int seq = blockIdx.y, h = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const uint32_t tag = a.head->tag;
    const int f0 = a.first[seq], n = a.first[seq + 1] - f0;
    if (tag != a.tag || n == 1) return;
    const int dq = tid % ND, grp = tid / ND;
    const f32x4 *part = reinterpret_cast<const f32x4 *>(a.part + (size_t(f0) * a.n_heads + h) * D) + dq;
    const size_t step = size_t(a.n_heads) * ND;
    const float2 *ml = a.ml + size_t(f0) * a.n_heads + h;
    f32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; u++) v[u] = n ? part[min(grp + NG * u, n - 1) * step] : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float M = -INFINITY;
    for (int i = tid; i < n; i += 256) M = fmaxf(M, ml[size_t(i) * a.n_heads].x);
    M = wave_max_f(M);
    if (lane == 0) wm[wv] = M;
    __syncthreads();
    M = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
    float L = 0.0f;
    for (int i0 = 0; i0 < n; i0 += 256) {
        const int m = min(256, n - i0);
        float f = 0.0f, l = 0.0f;
        if (tid < m) {
            const float2 o = ml[size_t(i0 + tid) * a.n_heads];
            if (o.x > -INFINITY) f = __builtin_amdgcn_exp2f((o.x - M) * a.mant), l = o.y * f;
        }
        fs[tid] = f;
        l = wave_sum_f(l);
        if (lane == 0) wl[wv] = l;
        __syncthreads();
        L += (wl[0] + wl[1]) + (wl[2] + wl[3]);
        for (int i = grp; i < m; i += NG * U) {
            if (i0 + i != grp)
#pragma unroll
                for (int u = 0; u < U; u++) v[u] = part[(i0 + min(i + NG * u, m - 1)) * step];
#pragma unroll
            for (int u = 0; u < U; u++)
                if (i + NG * u < m) y += v[u] * fs[i + NG * u];
        }
        __syncthreads();
    }
    red[grp][dq] = y;
    __syncthreads();
    if (grp) return;
#pragma unroll
    for (int u = 1; u < NG; u++) y += red[u][dq];
    store4<T, QF>(a.out, seq * a.out_stride + int64_t(h) * D + 4 * dq, y * inverse(M, L));
}

template <int D, uint32_t T, bool QF>
void launch_attend(const AttendArgs &a, int cap, int n, hipStream_t s) {
    const dim3 grid(a.n_kv * a.tiles, cap);
    if (a.shift < 6) hipLaunchKernelGGL((attend_kernel<D, T, QF, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attend_kernel<D, T, QF, false>), grid, dim3(256), 0, s, a);
    if (!a.arrivals) hipLaunchKernelGGL((merge_kernel<D, T, QF>), dim3(a.n_heads, n), dim3(256), 0, s, a);
}

template <int D>
void launch_types(uint32_t cache, const AttendArgs &a, int cap, int n, hipStream_t s) {
    const bool f = a.type == VIREO_PAGED_F32;
    if (cache == VIREO_PAGED_BF16)
        f ? launch_attend<D, VIREO_PAGED_BF16, true>(a, cap, n, s) : launch_attend<D, VIREO_PAGED_BF16, false>(a, cap, n, s);
    else
        f ? launch_attend<D, VIREO_PAGED_F16, true>(a, cap, n, s) : launch_attend<D, VIREO_PAGED_F16, false>(a, cap, n, s);
}

}  // namespace

extern "C" int vireo_paged_attend(const vireo_paged_cache *c, const vireo_paged_plan *p, const void *q, uint32_t type,
                                  int64_t q_stride, float scale, const int32_t *lists, void *out, int64_t out_stride,
                                  void *stream) {
    if (!vh_cache_ok(c) || !vh_plan_ok(p) || !p->mem || (reinterpret_cast<uintptr_t>(p->mem) & 255u) ||
        c->n_kv_heads != p->n_kv_heads || c->head_size != p->head_size || c->block_tokens != p->table->block_tokens ||
        c->n_blocks != p->table->n_blocks || (type != VIREO_PAGED_F32 && type != c->type) ||
        !vh_rows_ok(q, type, q_stride, p->n_heads, p->head_size, p->n) ||
        !vh_rows_ok(out, type, out_stride, p->n_heads, p->head_size, p->n) ||
        !vh_in_place_ok(q, type, q_stride, out, type, out_stride, p->n) || !(scale > 0.0f && scale < INFINITY) ||
        (lists != nullptr) != (p->list_blocks > 0))
        return -EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const PlanView v = vh_plan_view(p);
    int shift = 4;
    while ((1 << shift) < c->block_tokens) shift++;
    int expo;
    const double mant = 2.0 * frexp(double(scale) * 1.4426950408889634, &expo);
    const AttendArgs a{static_cast<const uint16_t *>(c->k), static_cast<const uint16_t *>(c->v), c->n_blocks,
                       c->n_kv_heads, shift, p->table->blocks, p->table->len, p->table->max_blocks, lists,
                       p->list_blocks, q, q_stride, float(mant), expo - 1, p->n_heads, p->n_heads / p->n_kv_heads,
                       vh_plan_head_tiles(p), out, out_stride, type, v.head, v.items, v.first, v.tag, v.part, v.ml, v.arrivals};
    if (c->head_size == 64) launch_types<64>(c->type, a, v.cap, p->n, s);
    else if (c->head_size == 128) launch_types<128>(c->type, a, v.cap, p->n, s);
    else launch_types<256>(c->type, a, v.cap, p->n, s);
    return vh_finish(s, vh_check(hipGetLastError()));
}
