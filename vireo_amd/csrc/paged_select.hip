// The blocks worth attending to (vireo_paged_select, include/vireo_paged.h):
// every sequence's first and last blocks and those between whose mean key
// scores highest against the new token's queries.
//
//   score_b = float32(max_h sum_j q_hj m_bj), the sum in fp64
//
// A sum of fp64 products of 16-bit and fp32 values is within 2^-45 of their sizes'
// sum of exact in any order, so that the fp32 score, and with it which of two blocks is
// higher, hangs on how the sum is split only where it lies that near to a border between two
// fp32 values. (An fp32 sum would leave the order of near blocks to the split.)
//
// score_kernel: 16 lanes per mean key (16-bit, D / 16 consecutive values a
// lane), four keys per group of 16 lanes; per query head the lanes' four sums are
// transposed while they are reduced (5 exchanges instead of 16). 228 000 mean keys of
// 128 (58 MB, 16 sequences of 9 000 to 65 536 tokens) against 4 heads each take 18.7 to
// 19.2 us (19.6 beside 24.2 with a block's kv heads far apart in the grid); against one head each
// 14.2, which is the read; the rest is fp64. The fp64 matrix cores took 46.8, and
// 16-bit matrix products that leave only the heads near the highest to fp64 33.9.
// The grid is as wide as the table, whatever the lengths: workgroups behind a sequence's end return.
// choose_kernel: a workgroup per (sequence, kv head), its keys in registers
// (but for tables of more than 8 192 candidates, below), finds the budget's lowest score by a histogram of 256 bins of their range and the
// ranks of the scores in its bin, and writes the blocks in order by one prefix sum.
// Bound by its chain of loads, barriers and LDS atomics.
#include <hip/hip_runtime.h>
#include <errno.h>
#include "paged.h"

namespace {

constexpr int kScoreRows = 64;  // mean keys per workgroup of score_kernel
constexpr int kHeads = 16;      // query heads in LDS at a time

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

VH_DEV float score_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
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

// Keys of a bin that one wave ranks against each other; more are told apart by digits.
constexpr uint32_t kFew = 64;
// the most candidates of a sequence: 64 keys per thread of 1024
constexpr int kMaxCandidates = 65536;

// HELD: keys that a thread holds in registers (the host takes the fewest threads and
// keys that hold every candidate that the table has room for). Straight code over them: a loop's keys from memory
// or both forms of every pass took 7.4 us for 1 871 candidates, this 5.4. 64 keys of
// 1024 threads do not fit the 128 registers of each and spill (396 words): one sequence of 30 001
// tokens takes 9.9 us for scores and choice in tables of 65 536 tokens and 10.4 of 131 136, but 58.6 of
// 262 144 (blocks of 16, 4 kv heads), 150 000 tokens 62.5.
template <int NT, int HELD>
__global__ void __launch_bounds__(NT) choose_kernel(SelectArgs a) {
    __shared__ uint32_t hist[2][256], wlo[NT / 64], whi[NT / 64];
    __shared__ uint2 wsum[NT / 64];
    __shared__ uint32_t found, left, there, n_few, few[kFew];
    const int g = blockIdx.x, i = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int have = a.seqs[i].blocks;
    if (a.head->tag != a.tag) return;
    int32_t *list = a.lists + (size_t(i) * a.n_kv + g) * a.width;
    if (have <= a.width) {
        for (int x = tid; x < a.width; x += NT) list[x] = x < have ? x : -1;
        return;
    }
    const int budget = a.width - a.sinks - a.window, n = have - a.sinks - a.window;  // n > budget
    const uint32_t *keys = a.keys + (size_t(i) * a.n_kv + g) * a.max_blocks + a.sinks;
    // thread tid's candidates: x0 .. x0 + cnt - 1, in order
    const int per = (n + NT - 1) / NT, x0 = tid * per, cnt = max(min(per, n - x0), 0);
    uint32_t k[HELD];
#pragma unroll
    for (int j = 0; j < HELD; j++) k[j] = j < cnt ? keys[x0 + j] : 0;  // no score's key is 0
    for (int x = tid; x < a.sinks; x += NT) list[x] = x;
    for (int x = tid; x < a.window; x += NT) list[a.sinks + budget + x] = have - a.window + x;
    if (budget == 0) return;
    // A bin of the scores' range that holds the budget's lowest: of 256 equal ones
    // from the lowest score to the highest (digits of the keys would put scores of one
    // exponent together). The bin of a score does not fall as the score rises: each step of
    // its arithmetic is monotonous.
    uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
    for (int j = 0; j < HELD; j++) lo = min(lo, k[j] - 1), hi = max(hi, k[j]);  // 0 - 1: not the lowest
    hi = wave_max_u(hi);
    lo = ~wave_max_u(~lo);
    if (lane == 0) wlo[wv] = lo, whi[wv] = hi;
    for (int x = tid; x < 512; x += NT) hist[x >> 8][x & 255] = 0;
    if (tid == 0) n_few = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; w++) lo = min(lo, wlo[w]), hi = max(hi, whi[w]);
    const float flo = score_of(lo + 1), per_bin = 256.0f / (score_of(hi) - flo);
    const bool even = per_bin > 0.0f && per_bin < INFINITY && flo > -INFINITY;  // else all in bin 0
    auto bin_of = [&](uint32_t key) {
        return key == 0 ? -1 : even ? min(int((score_of(key) - flo) * per_bin), 255) : 0;
    };
    // wave 0: the digit of `now`'s 256 that the need-th from the top falls into, to found, left, there
    auto digit = [&](const uint32_t *now, uint32_t need) {
        uint32_t c[4], sum = 0;  // lane l: 255 - 4 l .. 252 - 4 l
#pragma unroll
        for (int j = 0; j < 4; j++) sum += c[j] = now[255 - 4 * lane - j];
        uint32_t before = wave_scan_u(sum) - sum;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (before < need && before + c[j] >= need)
                found = uint32_t(255 - 4 * lane - j), left = need - before, there = c[j];
            before += c[j];
        }
    };
    uint32_t need = uint32_t(budget);
#pragma unroll
    for (int j = 0; j < HELD; j++)
        if (k[j]) atomicAdd(&hist[0][bin_of(k[j])], 1u);
    __syncthreads();
    if (wv == 0) digit(hist[0], need);
    __syncthreads();
    // the candidates of the bins above, and those of the bin itself
    const int bin = int(found);
    uint64_t above = 0, same = 0;
#pragma unroll
    for (int j = 0; j < HELD; j++) {
        const int at = bin_of(k[j]);
        above |= uint64_t(at > bin) << j;
        same |= uint64_t(at == bin) << j;
    }
    // of the bin's keys, those above `least` are taken, and the first `need` of those equal to it
    uint32_t least = 0;
    need = left;
    if (there == need) {
        need = 0;  // all of them
    } else if (there <= kFew) {
#pragma unroll
        for (int j = 0; j < HELD; j++)
            if ((same >> j) & 1) few[atomicAdd(&n_few, 1u)] = k[j];
        __syncthreads();
        if (wv == 0) {
            const int m = int(there);
            const uint32_t mine = lane < m ? few[lane] : 0;
            uint32_t gt = 0, ge = 0;
            for (int j = 0; j < m; j++) {
                const uint32_t o = uint32_t(__builtin_amdgcn_readlane(int(mine), j));
                gt += o > mine, ge += o >= mine;
            }
            if (lane < m && gt < need && ge >= need) found = mine, left = need - gt;  // equal ones write the same
        }
        __syncthreads();
        least = found;
        need = left;
    } else {  // digit by digit from the top
        uint32_t top = 0;
        for (int d = 24, pass = 1; d >= 0; d -= 8, pass++) {
            uint32_t *now = hist[pass & 1];
#pragma unroll
            for (int j = 0; j < HELD; j++)
                if (((same >> j) & 1) && (d == 24 || k[j] >> (d + 8) == top)) atomicAdd(&now[(k[j] >> d) & 255], 1u);
            __syncthreads();
            if (wv == 0) digit(now, need);
            else
                for (int x = tid - 64; x < 256; x += NT - 64) hist[(pass & 1) ^ 1][x] = 0;  // read last in the pass before
            __syncthreads();
            top = (top << 8) | found;
            need = left;
        }
        least = top;
    }
    // those taken, in order: one prefix sum of the ones above and of the equal ones
    uint64_t equal = 0;
#pragma unroll
    for (int j = 0; j < HELD; j++) {
        above |= uint64_t(((same >> j) & 1) && k[j] > least) << j;
        equal |= uint64_t(((same >> j) & 1) && k[j] == least) << j;
    }
    const uint32_t na = __popcll(above), ne = __popcll(equal);
    uint32_t gt = wave_scan_u(na), eq = wave_scan_u(ne);
    if (lane == 63) wsum[wv] = make_uint2(gt, eq);
    __syncthreads();
    gt -= na, eq -= ne;
#pragma unroll
    for (int w = 0; w < NT / 64; w++)
        if (w < wv) gt += wsum[w].x, eq += wsum[w].y;
    for (uint64_t m = above | equal; m; m &= m - 1) {
        const int j = __builtin_ctzll(m);
        const bool is_eq = (equal >> j) & 1;
        if (!is_eq || eq < need) list[a.sinks + gt + min(eq, need)] = a.sinks + x0 + j;
        gt += !is_eq, eq += is_eq;
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
    const PlanView v = vh_plan_view(p);
    const SelectArgs a{static_cast<const uint16_t *>(c->means), c->type, c->n_blocks, c->n_kv_heads, p->table->blocks,
                       p->table->max_blocks, v.head, v.seqs, v.tag, q, type, q_stride, p->n_heads / p->n_kv_heads, sinks,
                       window, p->list_blocks, v.keys, lists};
    const int cand = p->table->max_blocks - sinks - window;
    if (cand > kMaxCandidates) return -E2BIG;
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
    const dim3 lists_of(c->n_kv_heads, p->n);
    if (cand <= 256 * 8) hipLaunchKernelGGL((choose_kernel<256, 8>), lists_of, dim3(256), 0, s, a);
    else if (cand <= 512 * 8) hipLaunchKernelGGL((choose_kernel<512, 8>), lists_of, dim3(512), 0, s, a);
    else if (cand <= 1024 * 8) hipLaunchKernelGGL((choose_kernel<1024, 8>), lists_of, dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((choose_kernel<1024, 64>), lists_of, dim3(1024), 0, s, a);
    return vh_finish(s, vh_check(hipGetLastError()));
}
