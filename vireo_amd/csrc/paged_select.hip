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
// transposed while they are reduced (5 exchanges instead of 16). Bound by the
// read of the mean keys where the batch is large and by fp64 operations where
// a kv head has many query heads.
// choose_kernel: a workgroup per (sequence, kv head) finds the budget's lowest
// key by four 8-bit digits from the top and writes the blocks in order. Bound
// by its passes over the keys (L2) and their barriers.
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
    int n_blocks, n_kv, shift;
    const int32_t *ids, *table, *len;
    int max_seqs, max_blocks;
    const void *q;
    uint32_t q_type;
    int64_t q_stride;
    int hpg;
    int sinks, window, width;  // width: of a list
    uint32_t *keys;
    int32_t *lists;
};

// the sequence's blocks
VH_DEV int blocks_have(const SelectArgs &a, int i, int *row) {
    const int id = a.ids ? a.ids[i] : i;
    if (id < 0 || id >= a.max_seqs) return 0;
    *row = id;
    const uint32_t len = uint32_t(max(a.len[id], 0));
    return min(int((len + (1u << a.shift) - 1) >> a.shift), a.max_blocks);
}

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
    const int i = blockIdx.z, g = blockIdx.y;
    int row = 0;
    const int have = blocks_have(a, i, &row);
    const int b0 = a.sinks + blockIdx.x * kScoreRows, hi = have - a.window;
    if (have <= a.width || b0 >= hi) return;
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

__global__ void __launch_bounds__(kThreads) choose_kernel(SelectArgs a) {
    __shared__ uint32_t hist[256], wsum[kThreads / 64];
    __shared__ uint32_t found, left;
    const int g = blockIdx.x, i = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    int row = 0;
    const int have = blocks_have(a, i, &row);
    int32_t *list = a.lists + (size_t(i) * a.n_kv + g) * a.width;
    if (have <= a.width) {
        for (int x = tid; x < a.width; x += kThreads) list[x] = x < have ? x : -1;
        return;
    }
    const int budget = a.width - a.sinks - a.window, n = have - a.sinks - a.window;  // n > budget
    const uint32_t *keys = a.keys + (size_t(i) * a.n_kv + g) * a.max_blocks + a.sinks;
    for (int x = tid; x < a.sinks; x += kThreads) list[x] = x;
    for (int x = tid; x < a.window; x += kThreads) list[a.sinks + budget + x] = have - a.window + x;
    if (budget == 0) return;
    // the budget-th highest key, digit by digit; `need` of the keys that share its digits so far are taken
    uint32_t key = 0, need = uint32_t(budget);
    for (int d = 24; d >= 0; d -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int x = tid; x < n; x += kThreads) {
            const uint32_t k = keys[x];
            if (d == 24 || (k >> (d + 8)) == (key >> (d + 8))) atomicAdd(&hist[(k >> d) & 255], 1u);
        }
        __syncthreads();
        if (wv == 0) {  // lane l: digits 255 - 4 l .. 252 - 4 l
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) sum += c[j] = hist[255 - 4 * lane - j];
            uint32_t upto = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t u = __shfl_up(upto, o);
                if (lane >= o) upto += u;
            }
            uint32_t before = upto - sum;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (before < need && before + c[j] >= need) found = uint32_t(255 - 4 * lane - j), left = need - before;
                before += c[j];
            }
        }
        __syncthreads();
        key |= found << d;
        need = left;
    }
    // the keys above it and the first `need` equal ones, in order
    uint32_t above = 0, equal = 0;
    for (int x0 = 0; x0 < n; x0 += kThreads) {
        const int x = x0 + tid;
        const uint32_t k = x < n ? keys[x] : 0;
        const bool gt = x < n && k > key, eq = x < n && k == key;
        // both counts in one word: at most 1024 each
        const uint32_t mine = (gt ? 1u : 0u) | (eq ? 65536u : 0u);
        uint32_t s = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t u = __shfl_up(s, o);
            if (lane >= o) s += u;
        }
        __syncthreads();  // wsum is free
        if (lane == 63) wsum[wv] = s;
        __syncthreads();
        uint32_t before = s - mine, all = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 64; w++) {
            if (w < wv) before += wsum[w];
            all += wsum[w];
        }
        const uint32_t eb = equal + (before >> 16), gb = above + (before & 65535u);
        if (gt || (eq && eb < need)) list[a.sinks + gb + min(eb, need)] = a.sinks + x;
        above += all & 65535u;
        equal += all >> 16;
    }
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
    int shift = 4;
    while ((1 << shift) < c->block_tokens) shift++;
    const SelectArgs a{static_cast<const uint16_t *>(c->means), c->type, c->n_blocks, c->n_kv_heads, shift, p->ids,
                       p->table->blocks, p->table->len, p->table->max_seqs, p->table->max_blocks, q, type, q_stride,
                       p->n_heads / p->n_kv_heads, sinks, window, p->list_blocks, vh_plan_view(p).keys, lists};
    const int cand = p->table->max_blocks - sinks - window;
    if (p->table->max_blocks > p->list_blocks && p->list_blocks > sinks + window) {
        const dim3 grid((cand + kScoreRows - 1) / kScoreRows, c->n_kv_heads, p->n);
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
