// A step's rows into the paged cache (API: include/vireo_paged.h): per head of
// q and k the bias, RMSNorm and NEOX rotation, rounded once into q_out or the
// cache; v into the cache; the mean key of each block that a row completes.
//
//   y = x + b;  z = y / sqrt(mean(y^2) + eps) * w;
//   (z_j, z_{j+R/2}) -> (z_j c_j - z_{j+R/2} s_j, z_j s_j + z_{j+R/2} c_j), j < R/2
//
// One pass: every head row is read once and written once. A row of hs values
// takes hs / 16 lanes; a lane holds two runs of 8 values that are each other's
// rotation partners (values 8 i .. and R/2 + 8 i ..), so loads and stores are
// 16 bytes wide, the norm's sum is a few DPP adds and the rotation needs no
// exchange. Values go through LDS, 16 rows of a kv head at a time, so that a
// store's lanes are neighbouring tokens of few dimensions. Queries are stored
// with the non-temporal hint (4 093 rows, 84 MB: 22.9 -> 19.2 us, 4.4 TB/s with the
// launch). Bound by bytes for prompts and by its loads' round trip for a decode batch.
#include <hip/hip_runtime.h>
#include <errno.h>
#include "paged.h"

namespace {

constexpr int kVRows = 16;  // rows of a workgroup that stores values

struct AppendArgs {
    vireo_paged_rows r;
    uint16_t *k, *v;
    uint32_t cache_type;
    int n_kv, shift;  // block_tokens = 1 << shift
    int slots;        // of the pool
    int qk_groups;    // workgroups of queries and keys; those behind store values
};

// A head of a row's queries or keys per group of lanes. (Four heads per group, the
// rotation and norm weights read once for them: 4 093 rows 27.4 us, two 24.7, one 22.9:
// the loads in flight count, not the ones that the L1 answers.)
template <int HS>
VH_DEV void append_qk(const AppendArgs &a) {
    constexpr int LPR = HS / 16;  // lanes per head row
    const vireo_paged_rows &r = a.r;
    const int per_row = r.n_heads + a.n_kv, ln = threadIdx.x % LPR;
    const uint32_t total = uint32_t(r.rows) * per_row, unit = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    const bool there = unit < total;  // every lane stays for the sums
    const uint32_t idx = there ? unit : total - 1;
    const int t = int(idx / per_row), hh = int(idx - uint32_t(t) * per_row);
    const bool key = hh >= r.n_heads;
    const int h = key ? hh - r.n_heads : hh;
    const int slot = r.slots[t], pos = r.positions[t];
    // the lane's two runs of 8 values
    const int R = r.rotary, turned = R / 16;
    const int i0 = ln < turned ? 8 * ln : R + 16 * (ln - turned), i1 = ln < turned ? R / 2 + 8 * ln : i0 + 8;
    float x[2][8], y[2][8];
    {
        const int64_t o = t * (key ? r.k_stride : r.q_stride) + int64_t(h) * HS;
        ld8(key ? r.k : r.q, r.type, o + i0, x[0]);
        ld8(key ? r.k : r.q, r.type, o + i1, x[1]);
    }
    if (const float *bias = key ? r.k_bias : r.q_bias) {
        ld8(bias, VIREO_PAGED_F32, int64_t(h) * HS + i0, y[0]);
        ld8(bias, VIREO_PAGED_F32, int64_t(h) * HS + i1, y[1]);
#pragma unroll
        for (int j = 0; j < 8; j++) x[0][j] += y[0][j], x[1][j] += y[1][j];
    }
    if (const float *norm = key ? r.k_norm : r.q_norm) {
        ld8(norm, VIREO_PAGED_F32, i0, y[0]);
        ld8(norm, VIREO_PAGED_F32, i1, y[1]);
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) ss = fmaf(x[0][j], x[0][j], fmaf(x[1][j], x[1][j], ss));
        const float s = 1.0f / sqrtf(group_sum<LPR>(ss) * (1.0f / HS) + r.eps);
#pragma unroll
        for (int j = 0; j < 8; j++) x[0][j] *= s * y[0][j], x[1][j] *= s * y[1][j];
    }
    if (ln < turned && pos >= 0 && pos < r.max_pos) {
        const float *tab = r.rope + size_t(pos) * R + 8 * ln;
        ld8(tab, VIREO_PAGED_F32, 0, y[0]);
        ld8(tab, VIREO_PAGED_F32, R / 2, y[1]);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float lo = x[0][j], hi = x[1][j];
            x[0][j] = lo * y[0][j] - hi * y[1][j];
            x[1][j] = lo * y[1][j] + hi * y[0][j];
        }
    }
    if (!there || slot < 0 || slot >= a.slots) return;
    if (key) {
        const int G = 1 << a.shift, off = slot & (G - 1);
        uint16_t *k = a.k + ((size_t(slot >> a.shift) * a.n_kv + h) * G + off) * HS;
        *reinterpret_cast<u32x4 *>(k + i0) = pack8(x[0], a.cache_type);
        *reinterpret_cast<u32x4 *>(k + i1) = pack8(x[1], a.cache_type);
    } else {
        const int64_t o = t * r.q_out_stride + int64_t(h) * HS;
        st8_once(r.q_out, r.q_out_type, o + i0, x[0]);
        st8_once(r.q_out, r.q_out_type, o + i1, x[1]);
    }
}

// kVRows rows of one kv head's values: read row by row, stored dimension by
// dimension, 16 lanes a dimension's tokens (rows of one block lie side by side)
template <int HS>
VH_DEV void append_v(const AppendArgs &a) {
    constexpr int RS = HS / 2 + 1;  // words of an LDS row: a column's 16 rows on different banks
    __shared__ uint32_t tile[kVRows * RS];
    const vireo_paged_rows &r = a.r;
    const int unit = blockIdx.x - a.qk_groups, h = unit % a.n_kv, t0 = unit / a.n_kv * kVRows;
    constexpr int CH = HS / 8;  // runs of 8 values of a row
    for (int i = threadIdx.x; i < kVRows * CH; i += 256) {
        const int t = t0 + i / CH, j0 = i % CH * 8;
        if (t >= r.rows) break;
        float x[8];
        ld8(r.v, r.type, t * r.v_stride + int64_t(h) * HS + j0, x);
        if (r.v_bias) {
            float b[8];
            ld8(r.v_bias, VIREO_PAGED_F32, int64_t(h) * HS + j0, b);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] += b[j];
        }
        const u32x4 w = pack8(x, a.cache_type);
#pragma unroll
        for (int j = 0; j < 4; j++) tile[(i / CH) * RS + j0 / 2 + j] = w[j];
    }
    const int tt = threadIdx.x & 15, t = t0 + tt;
    const int slot = t < r.rows ? r.slots[t] : -1;
    __syncthreads();
    if (slot < 0 || slot >= a.slots) return;
    const int G = 1 << a.shift;
    uint16_t *v = a.v + (size_t(slot >> a.shift) * a.n_kv + h) * size_t(HS) * G + (slot & (G - 1));
#pragma unroll 4
    for (int j = 2 * (threadIdx.x >> 4); j < HS; j += 32) {
        const uint32_t w = tile[tt * RS + j / 2];
        v[size_t(j) * G] = uint16_t(w);
        v[size_t(j + 1) * G] = uint16_t(w >> 16);
    }
}

template <int HS>
__global__ void __launch_bounds__(256) append_kernel(AppendArgs a) {
    if (int(blockIdx.x) < a.qk_groups) append_qk<HS>(a);
    else append_v<HS>(a);
}

// The mean key of each block whose last slot a row wrote, from its keys as
// stored (so a block has the same mean however its tokens came). A workgroup
// looks at kMeanRows rows for one kv head, a wave per row: 16 lanes a token's HS
// values, four tokens at a time, added in order and then across the four.
constexpr int kMeanRows = 16;
template <int HS>
__global__ void __launch_bounds__(256) means_kernel(const int32_t *__restrict__ slots, int rows, int n_slots, int shift,
                                                    int n_kv, uint32_t type, const uint16_t *__restrict__ k,
                                                    uint16_t *__restrict__ means) {
    constexpr int E = HS / 16;  // values of a lane: E / 4 runs of 4, 64 apart
    const int lane = threadIdx.x & 63, sub = lane & 15, tok = lane >> 4, h = blockIdx.y, G = 1 << shift;
    for (int t = blockIdx.x * kMeanRows + (threadIdx.x >> 6); t < min(rows, int(blockIdx.x + 1) * kMeanRows); t += 4) {
        const int slot = slots[t];
        if (slot < 0 || slot >= n_slots || (slot & (G - 1)) != G - 1) continue;
        const size_t head = size_t(slot >> shift) * n_kv + h;
        const uint16_t *src = k + (head * G + tok) * HS + 4 * sub;
        const float share = 1.0f / float(G);  // a power of two: exact, and the sum does not leave fp32
        float sum[E] = {};
#pragma unroll 4
        for (int g = 0; g < G; g += 4)
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                const u32x2 w = *reinterpret_cast<const u32x2 *>(src + size_t(g) * HS + 16 * e);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float2 f = type == VIREO_PAGED_BF16 ? El<VIREO_PAGED_BF16>::unpack(w[j])
                                                              : El<VIREO_PAGED_F16>::unpack(w[j]);
                    sum[e + 2 * j] = fmaf(f.x, share, sum[e + 2 * j]);
                    sum[e + 2 * j + 1] = fmaf(f.y, share, sum[e + 2 * j + 1]);
                }
            }
#pragma unroll
        for (int e = 0; e < E; e++) {
            sum[e] += __shfl_xor(sum[e], 16);
            sum[e] += __shfl_xor(sum[e], 32);
        }
        if (tok == 0)
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                u32x2 w;
#pragma unroll
                for (int j = 0; j < 2; j++)
                    w[j] = type == VIREO_PAGED_BF16 ? El<VIREO_PAGED_BF16>::pack(sum[e + 2 * j], sum[e + 2 * j + 1])
                                                    : El<VIREO_PAGED_F16>::pack(sum[e + 2 * j], sum[e + 2 * j + 1]);
                *reinterpret_cast<u32x2 *>(means + head * HS + 16 * e + 4 * sub) = w;
            }
    }
}

template <int HS>
int launch_append(AppendArgs a, uint16_t *means, hipStream_t s) {
    const vireo_paged_rows &r = a.r;
    constexpr int kGroups = 256 / (HS / 16);  // head rows of a workgroup
    const int64_t heads = int64_t(r.rows) * (r.n_heads + a.n_kv), qk = (heads + kGroups - 1) / kGroups;
    const int64_t values = (int64_t(r.rows) + kVRows - 1) / kVRows * a.n_kv;
    if ((qk + values) * 256 >= int64_t(1) << 32) return -E2BIG;  // threads of a launch
    a.qk_groups = int(qk);
    hipLaunchKernelGGL(append_kernel<HS>, dim3(unsigned(qk + values)), dim3(256), 0, s, a);
    if (means)
        hipLaunchKernelGGL(means_kernel<HS>, dim3((r.rows + kMeanRows - 1) / kMeanRows, a.n_kv), dim3(256), 0, s,
                           r.slots, r.rows, a.slots, a.shift, a.n_kv, a.cache_type, a.k, means);
    return vh_check(hipGetLastError());
}

}  // namespace

extern "C" int vireo_paged_append(const vireo_paged_cache *c, const vireo_paged_rows *r, void *stream) {
    if (!vh_cache_ok(c) || !r || r->rows < 0 || r->n_heads < 1 || r->n_heads > 65535) return -EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (r->rows == 0) return vh_finish(s, 0);
    const int hs = c->head_size;
    if (!vh_rows_ok(r->q, r->type, r->q_stride, r->n_heads, hs, r->rows) ||
        !vh_rows_ok(r->k, r->type, r->k_stride, c->n_kv_heads, hs, r->rows) ||
        !vh_rows_ok(r->v, r->type, r->v_stride, c->n_kv_heads, hs, r->rows) ||
        !vh_rows_ok(r->q_out, r->q_out_type, r->q_out_stride, r->n_heads, hs, r->rows) ||
        !vh_in_place_ok(r->q, r->type, r->q_stride, r->q_out, r->q_out_type, r->q_out_stride, r->rows) ||
        (r->q_out_type != VIREO_PAGED_F32 && r->q_out_type != c->type) || !r->positions || !r->slots ||
        r->rotary < 0 || r->rotary % 16 || r->rotary > hs || (r->rotary > 0 && (!r->rope || r->max_pos < 1)) ||
        !(r->eps >= 0.0f))
        return -EINVAL;
    int shift = 4;
    while ((1 << shift) < c->block_tokens) shift++;
    const AppendArgs a{*r, static_cast<uint16_t *>(c->k), static_cast<uint16_t *>(c->v), c->type, c->n_kv_heads, shift,
                 c->n_blocks * c->block_tokens, 0};
    uint16_t *means = static_cast<uint16_t *>(c->means);
    const int rc = hs == 64    ? launch_append<64>(a, means, s)
                   : hs == 128 ? launch_append<128>(a, means, s)
                               : launch_append<256>(a, means, s);
    return rc == -E2BIG ? rc : vh_finish(s, rc);
}
