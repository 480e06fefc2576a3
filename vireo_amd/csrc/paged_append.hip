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
// exchange. Bound by bytes for prompts and by its loads' round trip for a
// decode batch.
#include <hip/hip_runtime.h>
#include <errno.h>
#include "paged.h"

namespace {

struct AppendArgs {
    vireo_paged_rows r;
    uint16_t *k, *v;
    uint32_t cache_type;
    int n_kv, shift;  // block_tokens = 1 << shift
    int slots;        // of the pool
};

template <int HS>
__global__ void __launch_bounds__(256) append_kernel(AppendArgs a) {
    constexpr int LPR = HS / 16;  // lanes per head row
    const vireo_paged_rows &r = a.r;
    const int per_row = r.n_heads + 2 * a.n_kv, ln = threadIdx.x % LPR;
    const int64_t total = int64_t(r.rows) * per_row;
    int64_t idx = int64_t(blockIdx.x) * (256 / LPR) + threadIdx.x / LPR;
    const bool there = idx < total;
    if (!there) idx = total - 1;  // every lane stays for the sums
    const int t = int(idx / per_row), hh = int(idx - int64_t(t) * per_row);
    const int kind = hh < r.n_heads ? 0 : hh < r.n_heads + a.n_kv ? 1 : 2;
    const int h = kind == 0 ? hh : hh - r.n_heads - (kind == 2 ? a.n_kv : 0);
    const int slot = r.slots[t], pos = r.positions[t];
    // the lane's two runs of 8 values
    const int R = r.rotary, turned = R / 16;
    const int i0 = ln < turned ? 8 * ln : R + 16 * (ln - turned), i1 = ln < turned ? R / 2 + 8 * ln : i0 + 8;
    float x[2][8];
    const void *src = kind == 0 ? r.q : kind == 1 ? r.k : r.v;
    const int64_t at = t * (kind == 0 ? r.q_stride : kind == 1 ? r.k_stride : r.v_stride) + int64_t(h) * HS;
    ld8(src, r.type, at + i0, x[0]);
    ld8(src, r.type, at + i1, x[1]);
    const float *bias = kind == 0 ? r.q_bias : kind == 1 ? r.k_bias : r.v_bias;
    const float *norm = kind == 0 ? r.q_norm : kind == 1 ? r.k_norm : nullptr;
    if (bias) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[0][j] += bias[size_t(h) * HS + i0 + j], x[1][j] += bias[size_t(h) * HS + i1 + j];
    }
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) ss = fmaf(x[0][j], x[0][j], fmaf(x[1][j], x[1][j], ss));
    ss = group_sum<LPR>(ss);
    if (norm) {
        const float s = 1.0f / sqrtf(ss * (1.0f / HS) + r.eps);
#pragma unroll
        for (int j = 0; j < 8; j++) x[0][j] *= s * norm[i0 + j], x[1][j] *= s * norm[i1 + j];
    }
    if (kind < 2 && ln < turned && pos >= 0 && pos < r.max_pos) {
        const float *tab = r.rope + size_t(pos) * R + 8 * ln;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float c = tab[j], s = tab[R / 2 + j], lo = x[0][j], hi = x[1][j];
            x[0][j] = lo * c - hi * s;
            x[1][j] = lo * s + hi * c;
        }
    }
    if (!there || slot < 0 || slot >= a.slots) return;
    if (kind == 0) {
        const int64_t o = t * r.q_out_stride + int64_t(h) * HS;
        st8(r.q_out, r.q_out_type, o + i0, x[0]);
        st8(r.q_out, r.q_out_type, o + i1, x[1]);
        return;
    }
    const int G = 1 << a.shift, off = slot & (G - 1);
    const size_t tile = (size_t(slot >> a.shift) * a.n_kv + h) * size_t(HS) * G;
    const u32x4 w0 = pack8(x[0], a.cache_type), w1 = pack8(x[1], a.cache_type);
    if (kind == 1) {
        uint16_t *k = a.k + tile + size_t(off) * HS;
        *reinterpret_cast<u32x4 *>(k + i0) = w0;
        *reinterpret_cast<u32x4 *>(k + i1) = w1;
    } else {
        uint16_t *v = a.v + tile + off;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[size_t(i0 + j) * G] = uint16_t(w0[j / 2] >> (16 * (j & 1)));
            v[size_t(i1 + j) * G] = uint16_t(w1[j / 2] >> (16 * (j & 1)));
        }
    }
}

// The mean key of each block whose last slot a row wrote, from its keys as
// stored (so a block has the same mean however its tokens came): a thread per
// 8 dimensions of a kv head adds the block's tokens in order in fp32.
__global__ void __launch_bounds__(256) means_kernel(const int32_t *__restrict__ slots, int n_slots, int shift, int n_kv,
                                                    int hs, uint32_t type, const uint16_t *__restrict__ k,
                                                    uint16_t *__restrict__ means) {
    const int slot = slots[blockIdx.x], G = 1 << shift;
    if (slot < 0 || slot >= n_slots || (slot & (G - 1)) != G - 1) return;
    const int per = hs / 8;
    const size_t blk = size_t(slot >> shift);
    for (int i = threadIdx.x; i < n_kv * per; i += 256) {
        const uint16_t *src = k + (blk * n_kv + i / per) * size_t(hs) * G + (i % per) * 8;
        float sum[8] = {};
#pragma unroll 8
        for (int g = 0; g < G; g++) {
            float x[8];
            ld8(src, type, int64_t(g) * hs, x);
#pragma unroll
            for (int j = 0; j < 8; j++) sum[j] += x[j];
        }
#pragma unroll
        for (int j = 0; j < 8; j++) sum[j] *= 1.0f / float(G);  // a power of two: exact
        st8(means, type, int64_t(blk * n_kv * hs) + int64_t(i) * 8, sum);
    }
}

template <int HS>
void launch_append(const AppendArgs &a, hipStream_t s) {
    const int64_t rows = int64_t(a.r.rows) * (a.r.n_heads + 2 * a.n_kv), per = 256 / (HS / 16);
    hipLaunchKernelGGL(append_kernel<HS>, dim3(unsigned((rows + per - 1) / per)), dim3(256), 0, s, a);
}

}  // namespace

extern "C" int vireo_paged_append(const vireo_paged_cache *c, const vireo_paged_rows *r, void *stream) {
    if (!vh_cache_ok(c) || !r || r->rows < 0 || r->n_heads < 1 || r->n_heads > 65535) return -EINVAL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int hs = c->head_size;
    if (!vh_rows_ok(r->q, r->type, r->q_stride, r->n_heads, hs, r->rows) ||
        !vh_rows_ok(r->k, r->type, r->k_stride, c->n_kv_heads, hs, r->rows) ||
        !vh_rows_ok(r->v, r->type, r->v_stride, c->n_kv_heads, hs, r->rows) ||
        !vh_rows_ok(r->q_out, r->q_out_type, r->q_out_stride, r->n_heads, hs, r->rows) ||
        (r->q_out_type != VIREO_PAGED_F32 && r->q_out_type != c->type) || !r->positions || !r->slots ||
        r->rotary < 0 || r->rotary % 16 || r->rotary > hs || (r->rotary > 0 && (!r->rope || r->max_pos < 1)) ||
        !(r->eps >= 0.0f))
        return -EINVAL;
    const int64_t heads = int64_t(r->rows) * (r->n_heads + 2 * int64_t(c->n_kv_heads));
    if (heads > (int64_t(1) << 31)) return -E2BIG;
    if (r->rows == 0) return vh_finish(s, 0);
    int shift = 4;
    while ((1 << shift) < c->block_tokens) shift++;
    AppendArgs a{*r, static_cast<uint16_t *>(c->k), static_cast<uint16_t *>(c->v), c->type, c->n_kv_heads, shift,
                 c->n_blocks * c->block_tokens};
    if (hs == 64) launch_append<64>(a, s);
    else if (hs == 128) launch_append<128>(a, s);
    else launch_append<256>(a, s);
    if (c->means)
        hipLaunchKernelGGL(means_kernel, dim3(r->rows), dim3(256), 0, s, r->slots, a.slots, shift, c->n_kv_heads, hs,
                           c->type, a.k, static_cast<uint16_t *>(c->means));
    return vh_finish(s, vh_check(hipGetLastError()));
}
