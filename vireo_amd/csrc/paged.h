// Shared by the paged cache's kernels (API: include/vireo_paged.h): argument
// checks, the layout of a plan's memory, and 16-bit element types.
#pragma once
#include "common.h"
#include "vireo_paged.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 hf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kPagedMaxSeqs = 4096;
constexpr int kPagedUnit = 128;  // tokens of the unit that a plan splits sequences by

// a pointer that is given and aligned to 16 bytes
inline bool vh_al16(const void *p) { return p && !(reinterpret_cast<uintptr_t>(p) & 15u); }

inline bool vh_table_ok(const vireo_paged_table *t) {
    return t && t->max_seqs >= 1 && t->max_seqs <= kPagedMaxSeqs && t->max_blocks >= 1 && t->n_blocks >= 1 &&
           (t->block_tokens == 16 || t->block_tokens == 32 || t->block_tokens == 64 || t->block_tokens == 128) &&
           int64_t(t->n_blocks) * t->block_tokens < (int64_t(1) << 31) &&
           int64_t(t->max_blocks) * t->block_tokens < (int64_t(1) << 31) && t->blocks && t->len && t->free_blocks &&
           t->n_free;
}

inline bool vh_cache_ok(const vireo_paged_cache *c) {
    return c && (c->type == VIREO_PAGED_F16 || c->type == VIREO_PAGED_BF16) && c->n_blocks >= 1 && c->n_kv_heads >= 1 &&
           c->n_kv_heads <= 65535 &&
           (c->block_tokens == 16 || c->block_tokens == 32 || c->block_tokens == 64 || c->block_tokens == 128) &&
           int64_t(c->n_blocks) * c->block_tokens < (int64_t(1) << 31) &&
           (c->head_size == 64 || c->head_size == 128 || c->head_size == 256) && vh_al16(c->k) && vh_al16(c->v) &&
           (!c->means || vh_al16(c->means));
}

// rows of `heads` heads of hs elements of `type`, `stride` elements apart, each 16-byte aligned
inline bool vh_rows_ok(const void *p, uint32_t type, int64_t stride, int64_t heads, int hs, int64_t rows) {
    if (!vh_al16(p) || (type != VIREO_PAGED_F32 && type != VIREO_PAGED_F16 && type != VIREO_PAGED_BF16)) return false;
    const int64_t per16 = type == VIREO_PAGED_F32 ? 4 : 8;
    return stride % per16 == 0 && (rows <= 1 || stride >= heads * hs) && stride >= 0 && stride < (int64_t(1) << 40);
}

// rows written over the ones they are made from have to lie where those lie: others are still to be read
inline bool vh_in_place_ok(const void *from, uint32_t from_type, int64_t from_stride, const void *to, uint32_t to_type,
                           int64_t to_stride, int64_t rows) {
    return from != to || ((from_type == VIREO_PAGED_F32) == (to_type == VIREO_PAGED_F32) &&
                          (rows <= 1 || from_stride == to_stride));
}

// ---- a plan's memory ------------------------------------------------------------
// A batch is cut into items: (sequence, run of kPagedUnit-token units), at least
// one per sequence. Items of a sequence are consecutive; first[i] is sequence i's
// first. Every kv head (and tile of 16 query heads of it) attends each item in one
// workgroup. Where the table or the lists leave a sequence few units, at most
// kJoinUnits and kJoinHeads units and heads of a workgroup together, the last
// workgroup of a sequence and kv head to finish joins its items (arrivals counts
// them), else a second launch does. Per call, joined and in two launches: one sequence,
// 8 heads of 128 a kv head 8 units 8.0 and 10.6 us, 16 units 9.2 and 10.7; 4 heads 8 units 8.1 and 10.4, 16
// units 9.8 and 10.6, 24 units 11.7 and 10.6, 32 units 13.7 and 10.7; 4 of 256 32 units 16.3
// and 13.5. 8 sequences, whose split gives each fewer items: 4 heads of 128 16 units 15.4 and
// 16.8, 32 units 24.5 and 26.5. So the rule costs one sequence alone 1 to 3 us between 17 and 32
// units and gains a batch 2. (In a graph the second launch costs 1 us less.)
constexpr int kJoinUnits = 32, kJoinHeads = 128;
struct PlanHead {
    uint32_t tag;  // written by an update of a plan of the same shape (vh_plan_tag)
    int32_t n_items;
    int32_t pad[14];
};
struct PlanItem {
    int32_t row;         // of the table
    int32_t begin, end;  // tokens (of the listed blocks, where the plan has lists)
    int32_t seq;         // in the batch
    int32_t first, count;  // the sequence's items
    int32_t pad[2];
};
struct PlanSeq {
    int32_t row, blocks;  // of the table; 0 blocks: an empty sequence, or not one
};
struct PlanView {
    PlanHead *head;
    PlanSeq *seqs;    // [n]
    int32_t *first;   // [n + 1]
    PlanItem *items;  // [cap]
    uint32_t *keys;   // [n x n_kv_heads x max_blocks] ordered scores (plans with lists)
    float2 *ml;       // [cap x n_heads] largest score (times a power of two) and sum of weights of each item's partial
    float *part;      // [cap x n_heads x head_size]
    uint32_t *arrivals;  // [n x n_kv_heads x head tiles], zero between calls
    int cap;
    bool join;  // arrivals is there
    uint32_t tag;
    int64_t bytes;
};
bool vh_plan_ok(const vireo_paged_plan *p);    // its fields but mem
PlanView vh_plan_view(const vireo_paged_plan *p);
int vh_plan_head_tiles(const vireo_paged_plan *p);  // tiles of 16 query heads per kv head

// ---- device ---------------------------------------------------------------------
VH_DEV float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
VH_DEV float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// 16-bit element types by the type number: two packed values <-> floats (rounded to nearest even)
template <uint32_t T>
struct El;
template <>
struct El<VIREO_PAGED_BF16> {
    static VH_DEV float2 unpack(uint32_t w) { return make_float2(bf_lo(w), bf_hi(w)); }
    static VH_DEV uint32_t pack(float a, float b) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, (b2){__bf16(a), __bf16(b)});
    }
    static VH_DEV f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
};
template <>
struct El<VIREO_PAGED_F16> {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    static VH_DEV float2 unpack(uint32_t w) {
        const h2 v = __builtin_bit_cast(h2, w);
        return make_float2(float(v[0]), float(v[1]));
    }
    static VH_DEV uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, (h2){_Float16(a), _Float16(b)});
    }
    static VH_DEV f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hf16x8, a), __builtin_bit_cast(hf16x8, b), c, 0,
                                                      0, 0);
    }
};
VH_DEV u32x4 ldu4(const void *p) { return *reinterpret_cast<const u32x4 *>(p); }
// Inclusive prefix sums over the wave by DPP (row shifts, then the rows' totals carried on); every lane active.
VH_DEV uint32_t wave_scan_u(uint32_t v) {
    v += dpp_u<0x111>(v);
    v += dpp_u<0x112>(v);
    v += dpp_u<0x114>(v);
    v += dpp_u<0x118>(v);
    v += dpp_u<0x142, 0xA>(v);
    v += dpp_u<0x143, 0xC>(v);
    return v;
}
// with the non-temporal hint: what a launch reads once
VH_DEV u32x4 ldu4_once(const void *p) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p)); }
// 8 consecutive elements of a type known at run time (the same for the whole launch) as floats
VH_DEV void ld8(const void *p, uint32_t type, int64_t i, float (&x)[8]) {
    if (type == VIREO_PAGED_F32) {
        const f32x4 a = reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i)[0];
        const f32x4 b = reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i)[1];
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = a[j], x[4 + j] = b[j];
        return;
    }
    const u32x4 w = ldu4(static_cast<const uint16_t *>(p) + i);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 v = type == VIREO_PAGED_BF16 ? El<VIREO_PAGED_BF16>::unpack(w[j]) : El<VIREO_PAGED_F16>::unpack(w[j]);
        x[2 * j] = v.x;
        x[2 * j + 1] = v.y;
    }
}
VH_DEV u32x4 pack8(const float (&x)[8], uint32_t type) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; j++)
        w[j] = type == VIREO_PAGED_BF16 ? El<VIREO_PAGED_BF16>::pack(x[2 * j], x[2 * j + 1])
                                        : El<VIREO_PAGED_F16>::pack(x[2 * j], x[2 * j + 1]);
    return w;
}
// 8 elements stored with the non-temporal hint
VH_DEV void st8_once(void *p, uint32_t type, int64_t i, const float (&x)[8]) {
    if (type == VIREO_PAGED_F32) {
        f32x4 *d = reinterpret_cast<f32x4 *>(static_cast<float *>(p) + i);
        __builtin_nontemporal_store(f32x4{x[0], x[1], x[2], x[3]}, d);
        __builtin_nontemporal_store(f32x4{x[4], x[5], x[6], x[7]}, d + 1);
    } else {
        __builtin_nontemporal_store(pack8(x, type), reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(p) + i));
    }
}
// the largest / the sum over the four lanes of a column (lanes l, l + 16, l + 32, l + 48)
VH_DEV float head_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
VH_DEV float head_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// x split into NP truncated 16-bit parts, the operand words of each. LEAST: parts of an x
// that is not 0 which would be 0 become the least value of its sign.
template <uint32_t T, int NP, bool LEAST>
VH_DEV void split8(const float (&x)[8], u32x4 (&w)[NP]) {
    constexpr float kLeast = T == VIREO_PAGED_BF16 ? 1.17549435e-38f : 5.9604645e-8f;  // 2^-126, 2^-24
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        float a = x[j], b = x[j + 1], la = 0.0f, lb = 0.0f;
        if constexpr (LEAST) {
            la = fminf(fabsf(a) * 0x1p127f, kLeast);  // 0 for a zero
            lb = fminf(fabsf(b) * 0x1p127f, kLeast);
            a = fabsf(a) < la ? copysignf(la, a) : a;
            b = fabsf(b) < lb ? copysignf(lb, b) : b;
        }
#pragma unroll
        for (int p = 0; p < NP; p++) {
            if (LEAST && p) {
                a = copysignf(fmaxf(fabsf(a), la), x[j]);
                b = copysignf(fmaxf(fabsf(b), lb), x[j + 1]);
            }
            if constexpr (T == VIREO_PAGED_BF16) {
                const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
                w[p][j / 2] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);  // the high halves
                a -= __uint_as_float(ua & 0xffff0000u);
                b -= __uint_as_float(ub & 0xffff0000u);
            } else {
                const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
                w[p][j / 2] = __builtin_bit_cast(uint32_t, h);
                a -= float(h[0]);
                b -= float(h[1]);
            }
        }
    }
}

// A matrix operand of queries of type F32 (QF) or T as parts of T: lane (col,
// grp) loads values 32 s + 0 .. 7 from element `at` on (its head's, 8 grp in) for
// each step s; load() only requests them, parts() waits. fp32 queries are taken under a
// power of two whose exponent parts() returns: over fp16 one that brings the head's largest
// into [2^14, 2^15), so that a value is cut off at 2^-38 of it; over bf16 one that
// brings it to 2^-60 where it is smaller, for the parts' sake (larger ones could
// leave fp32 with the keys). LEAST: as split8's.
template <int D, uint32_t T, bool QF>
struct Queries {
    static constexpr int KS = D / 32, P = QF ? 3 : 1;
    u32x4 raw[KS][QF ? 2 : 1];
    VH_DEV void load(const void *q, int64_t at) {
#pragma unroll
        for (int s = 0; s < KS; s++) {
            if constexpr (QF) {
                const float *p = static_cast<const float *>(q) + at + 32 * s;
                raw[s][0] = ldu4(p);
                raw[s][1] = ldu4(p + 4);
            } else {
                raw[s][0] = ldu4(static_cast<const uint16_t *>(q) + at + 32 * s);
            }
        }
    }
    template <bool LEAST>
    VH_DEV int parts(u32x4 (&w)[P][KS]) const {
        int e = 0;
        if constexpr (!QF) {
#pragma unroll
            for (int s = 0; s < KS; s++) w[0][s] = raw[s][0];
        } else {
            float x[KS][8], big = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[s][j] = __uint_as_float(raw[s][j >> 2][j & 3]);
                    big = fmaxf(big, fabsf(x[s][j]));
                }
            if (T == VIREO_PAGED_F16 || __any(big < 0x1p-60f)) {
                big = head_max(big);
                if (T == VIREO_PAGED_F16 ? big > 0.0f && big < INFINITY : big > 0.0f && big < 0x1p-60f)
                    e = (T == VIREO_PAGED_F16 ? 14 : -60) - ilogbf(big);
#pragma unroll
                for (int s = 0; s < KS; s++)
#pragma unroll
                    for (int j = 0; j < 8; j++) x[s][j] = ldexpf(x[s][j], e);
            }
#pragma unroll
            for (int s = 0; s < KS; s++) {
                u32x4 p[3];
                split8<T, 3, LEAST>(x[s], p);
#pragma unroll
                for (int k = 0; k < 3; k++) w[k][s] = p[k];
            }
        }
        return e;
    }
};
