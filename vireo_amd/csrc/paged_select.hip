// The blocks worth attending to (vireo_paged_select, include/vireo_paged.h):
// every sequence's first and last blocks and those between whose mean key
// scores highest against the new token's queries.
//
//   score_b = float32(max_h sum_j q_hj m_bj), the sum in fp64
//
// A sum of fp64 products of 16-bit and fp32 values is within 2^-50 of exact in
// any order, so the fp32 score, and with it which of two blocks is higher, does
// not depend on how the sum is split. (An fp32 sum would leave the order of
// near blocks to the split.)
//
// score_kernel: 16 lanes per mean key (16-bit, D / 16 consecutive values a
// lane), four keys per group of 16 lanes; per query head the lanes' four sums are
// transposed while they are reduced (5 exchanges instead of 16). 228 000 mean keys of
// 128 (58 MB, 16 sequences of 9 000 to 65 536 tokens) against 4 heads each take 19.6 us
// (24.2 with a block's kv heads far apart in the grid); against one head each 14.2,
// which is the read; the rest is fp64. The fp64 matrix cores took 46.8 (140 cycles a 16x16x4 product),
// and 16-bit matrix products that leave only the heads near the highest to fp64 33.9
// (their operand reads 64 bytes of a key at a time).
// choose_kernel: a workgroup per (sequence, kv head), its keys in registers,
// finds the budget's lowest key by 8-bit digits of its distance from the lowest one
// (two or three, where keys differ by their last bits four) and writes the blocks in
// order by one prefix sum. Bound by its chain of loads, barriers and LDS atomics.
#include <hip/hip_runtime.h>
#include <errno.h>
#include "paged.h"

namespace {

constexpr int kScoreRows = 64;  // mean keys per workgroup of score_kernel
constexpr int kHeads = 16;      // query heads in LDS at a time
constexpr int kThreads = 1024;  // of choose_kernel

struct SelectArgs {
    const uint16_t *means;
    uint32_t cache_type;
    int n_blocks, n_kv;
    const int32_t *table;
    int max_blocks;
    const PlanHead *head;
    const PlanSeq *seqs;
    uint32_t tag;
    const void *q;
    uint32_t q_type;
    int64_t q_stride;
    int hpg;
    int sinks, window, width;  // width: of a list
    uint32_t *keys;
    int32_t *lists;
};

// a float as an unsigned integer in the floats' order (-0 as 0)
VH_DEV uint32_t ordered(float f) {
    const uint32_t u = __float_as_uint(f + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// v of the lane 1 (xor) / 2 (xor) / 4 / 8 (rotated within 16) away
VH_DEV double swap1(double v) { return dpp_d<0xB1>(v); }
VH_DEV double swap2(double v) { return dpp_d<0x4E>(v); }
VH_DEV double ror4(double v) { return dpp_d<0x124>(v); }
VH_DEV double ror8(double v) { return dpp_d<0x128>(v); }

// keys[(i n_kv + g) max_blocks + b] = ordered score of block b, sinks <= b < have - window
template <int D, uint32_t T>
__global__ void __launch_bounds__(256) score_kernel(SelectArgs a) {
    constexpr int E = D / 16;
    __shared__ __align__(16) float qs[kHeads][D];
    const int i = blockIdx.z, g = blockIdx.x;  // a block's kv heads lie side by side
    const PlanSeq sq = a.seqs[i];
    const int row = sq.row, have = sq.blocks, b0 = a.sinks + blockIdx.y * kScoreRows, hi = have - a.window;
    if (a.head->tag != a.tag || have <= a.width || b0 >= hi) return;
    const int lane = threadIdx.x & 63, sub = lane & 15;
    // the group's four mean keys: blocks b .. b + 3 (past the end: the last one again)
    const int b = b0 + 4 * int(threadIdx.x >> 4);
    float m[4][E];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int blk = a.table[size_t(row) * a.max_blocks + min(b + r, hi - 1)];
        const bool ok = blk >= 0 && blk < a.n_blocks;
        const uint16_t *p = a.means + (size_t(ok ? blk : 0) * a.n_kv + g) * D + sub * E;
#pragma unroll
        for (int j = 0; j < E; j += 4) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(p + j);
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const float2 f = El<T>::unpack(w[x]);
                m[r][j + 2 * x] = f.x;
                m[r][j + 2 * x + 1] = f.y;
            }
        }
        if (!ok) m[r][0] = __builtin_nanf("");  // a block outside the pool: last
    }
    double best = -INFINITY;
    for (int h0 = 0; h0 < a.hpg; h0 += kHeads) {
        const int nh = min(kHeads, a.hpg - h0);
        if (h0) __syncthreads();
        for (int x = threadIdx.x * 8; x < nh * D; x += 256 * 8) {
            float v[8];
            ld8(a.q, a.q_type, i * a.q_stride + int64_t(g * a.hpg + h0) * D + x, v);
            float *dst = &qs[0][0] + x;
#pragma unroll
            for (int j = 0; j < 8; j++) dst[j] = v[j];
        }
        __syncthreads();
        for (int h = 0; h < nh; h++) {
            double s[4] = {};
#pragma unroll
            for (int j = 0; j < E; j++) {
                const double q = qs[h][sub * E + j];
#pragma unroll
                for (int r = 0; r < 4; r++) s[r] = fma(q, double(m[r][j]), s[r]);
            }
            // lane sub ends with row sub % 4's sum
            const bool odd = sub & 1, high = sub & 2;
            double u0 = odd ? s[1] : s[0], u1 = odd ? s[3] : s[2];
            u0 += swap1(odd ? s[0] : s[1]);
            u1 += swap1(odd ? s[2] : s[3]);
            double v = high ? u1 : u0;
            v += swap2(high ? u0 : u1);
            v += ror8(v);
            v += ror4(v);
            best = fmax(best, v);  // a NaN counts as -inf
        }
    }
    if (sub < 4 && b + sub < hi) a.keys[(size_t(i) * a.n_kv + g) * a.max_blocks + b + sub] = ordered(float(best));
}

// Keys that a thread of choose_kernel holds in registers; a sequence with more
// candidates reads them again in every pass.
constexpr int kHeld = 8;

__global__ void __launch_bounds__(kThreads) choose_kernel(SelectArgs a) {
    __shared__ uint32_t hist[2][256], wlo[kThreads / 64], whi[kThreads / 64];
    __shared__ uint64_t wsum[kThreads / 64];
    __shared__ uint32_t found, left, there;
    const int g = blockIdx.x, i = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int have = a.seqs[i].blocks;
    if (a.head->tag != a.tag) return;
    int32_t *list = a.lists + (size_t(i) * a.n_kv + g) * a.width;
    if (have <= a.width) {
        for (int x = tid; x < a.width; x += kThreads) list[x] = x < have ? x : -1;
        return;
    }
    const int budget = a.width - a.sinks - a.window, n = have - a.sinks - a.window;  // n > budget
    const uint32_t *keys = a.keys + (size_t(i) * a.n_kv + g) * a.max_blocks + a.sinks;
    // thread tid's candidates: x0 .. x0 + per - 1 (below n), in order
    const int per = (n + kThreads - 1) / kThreads, x0 = tid * per, cnt = max(min(per, n - x0), 0);
    const bool held = per <= kHeld;
    uint32_t k[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; j++) k[j] = held && j < cnt ? keys[x0 + j] : 0;
    for (int x = tid; x < a.sinks; x += kThreads) list[x] = x;
    for (int x = tid; x < a.window; x += kThreads) list[a.sinks + budget + x] = have - a.window + x;
    if (budget == 0) return;
    auto each = [&](auto f) {
        if (held) {
#pragma unroll
            for (int j = 0; j < kHeld; j++)
                if (j < cnt) f(x0 + j, k[j]);
        } else {
            for (int j = 0; j < cnt; j++) f(x0 + j, keys[x0 + j]);
        }
    };
    // the range of the keys: digits are of key - lowest, so that they spread
    uint32_t lo = 0xffffffffu, hi = 0;
    each([&](int, uint32_t key) { lo = min(lo, key), hi = max(hi, key); });
    hi = wave_max_u(hi);
    lo = ~wave_max_u(~lo);
    if (lane == 0) wlo[wv] = lo, whi[wv] = hi;
    if (tid < 512) hist[tid >> 8][tid & 255] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) lo = min(lo, wlo[w]), hi = max(hi, whi[w]);
    // `need` of the keys whose (key - lo) >> shift is `top` are taken, and all above
    int shift = 32 - __clz(hi - lo);  // __clz(0) is 32
    uint32_t top = 0, need = uint32_t(budget);
    for (int pass = 0; shift > 0; pass++) {
        const int bits = min(shift, 8);
        uint32_t *now = hist[pass & 1];
        shift -= bits;
        each([&](int, uint32_t key) {
            const uint32_t v = (key - lo) >> shift;
            if (uint64_t(v) >> bits == top) atomicAdd(&now[v & ((1u << bits) - 1)], 1u);
        });
        __syncthreads();
        if (wv == 0) {  // lane l: digits 255 - 4 l .. 252 - 4 l
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) sum += c[j] = now[255 - 4 * lane - j];
            uint32_t upto = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t u = __shfl_up(upto, o);
                if (lane >= o) upto += u;
            }
            uint32_t before = upto - sum;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (before < need && before + c[j] >= need)
                    found = uint32_t(255 - 4 * lane - j), left = need - before, there = c[j];
                before += c[j];
            }
        } else if (wv >= 4 && wv < 8) {
            hist[(pass & 1) ^ 1][tid & 255] = 0;  // read last in the pass before
        }
        __syncthreads();
        top = (top << bits) | found;
        need = left;
        if (there == need) break;  // all of them: the lower digits do not matter
    }
    // the keys above and the first `need` equal ones, in order: one prefix sum of both counts
    uint32_t above = 0, equal = 0;
    each([&](int, uint32_t key) {
        const uint32_t v = uint32_t(uint64_t(key - lo) >> shift);
        above += v > top, equal += v == top;
    });
    const uint64_t mine = (uint64_t(equal) << 32) | above;
    uint64_t s = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t u = __shfl_up(s, o);
        if (lane >= o) s += u;
    }
    if (lane == 63) wsum[wv] = s;
    __syncthreads();
    uint64_t before = s - mine;
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++)
        if (w < wv) before += wsum[w];
    uint32_t gt = uint32_t(before), eq = uint32_t(before >> 32);
    each([&](int x, uint32_t key) {
        const uint32_t v = uint32_t(uint64_t(key - lo) >> shift);
        const bool take = v > top || (v == top && eq < need);
        if (take) list[a.sinks + gt + min(eq, need)] = a.sinks + x;
        gt += v > top, eq += v == top;
    });
}

}  // namespace

extern "C" int vireo_paged_select(const vireo_paged_cache *c, const vireo_paged_plan *p, const void *q, uint32_t type,
                                  int64_t q_stride, int sinks, int window, int32_t *lists, void *stream) {
    if (!vh_cache_ok(c) || !c->means || !vh_plan_ok(p) || !p->mem || (reinterpret_cast<uintptr_t>(p->mem) & 255u) ||
        c->n_kv_heads != p->n_kv_heads || c->head_size != p->head_size || c->block_tokens != p->table->block_tokens ||
        c->n_blocks != p->table->n_blocks || (type != VIREO_PAGED_F32 && type != c->type) ||
        !vh_rows_ok(q, type, q_stride, p->n_heads, p->head_size, p->n) || sinks < 0 || window < 1 ||
        p->list_blocks == 0 || int64_t(sinks) + window > p->list_blocks || !lists)
        return -EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const PlanView v = vh_plan_view(p);
    const SelectArgs a{static_cast<const uint16_t *>(c->means), c->type, c->n_blocks, c->n_kv_heads, p->table->blocks,
                       p->table->max_blocks, v.head, v.seqs, v.tag, q, type, q_stride, p->n_heads / p->n_kv_heads, sinks,
                       window, p->list_blocks, v.keys, lists};
    const int cand = p->table->max_blocks - sinks - window;
    if (p->table->max_blocks > p->list_blocks && p->list_blocks > sinks + window) {
        const dim3 grid(c->n_kv_heads, (cand + kScoreRows - 1) / kScoreRows, p->n);
        const bool bf = c->type == VIREO_PAGED_BF16;
#define SCORE(D)                                                                                                   \
    if (c->head_size == D) {                                                                                       \
        if (bf) hipLaunchKernelGGL((score_kernel<D, VIREO_PAGED_BF16>), grid, dim3(256), 0, s, a);                  \
        else hipLaunchKernelGGL((score_kernel<D, VIREO_PAGED_F16>), grid, dim3(256), 0, s, a);                      \
    }
        SCORE(64)
        SCORE(128)
        SCORE(256)
#undef SCORE
    }
    hipLaunchKernelGGL(choose_kernel, dim3(c->n_kv_heads, p->n), dim3(kThreads), 0, s, a);
    return vh_finish(s, vh_check(hipGetLastError()));
}
