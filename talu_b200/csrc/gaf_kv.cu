// The quantised KV cache: rows written (quantised) into their pages and read back, and the attention over it for head
// sizes that the tensor-core kernel does not take.
//
// A group of G values x along head_dim is stored as codes q, a bf16 scale s and a bf16 bias b:
//   b = bf16(min x),  s = bf16((max x - min x) f32(1 / maxq)),  q = clamp(rint((x - b) / s), 0, maxq),  value = q s + b
// (a product with the rounded reciprocal, since that is what dividing a tensor by a number comes to in torch on the GPU, so that a
// cache filled there has the same scales; a true quotient gives a scale one bf16 step apart in some 1 in 10^5 groups of f32 rows)
// b is exact for bf16 inputs (the minimum is one of them).  s and b are rounded to nearest once, because 16 bits each is
// what the format stores; the codes are taken against the rounded pair, which makes the rounding of s part of the grid and
// not an error of every value: only the top value can be off by more than half a step, (max x - min x) 2^-9 + s / 2.
// Differences are formed of halves (0.5 x - 0.5 b), which is exact scaling, so that no finite input overflows.
#include "gaf_attend.cuh"
#include "gaf_internal.h"

#include <cuda_bf16.h>

#include <cfloat>

namespace tgaf {
namespace {

constexpr int kThreadsKv = 256;

__device__ __forceinline__ float bf16_f32(uint32_t raw) { return __uint_as_float(raw << 16); }
__device__ __forceinline__ uint32_t f32_bf16(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Sequence of packed row t, or -1 for a row behind the last sequence.
__device__ __forceinline__ int seq_of(const KvSeqs &s, uint32_t t) {
    if (!s.cu) return static_cast<int>(t / s.per);
    uint32_t lo = 0, hi = s.batch + 1u;   // cu[lo - 1] <= t < cu[hi], with cu[-1] = -inf
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (s.cu[mid] <= static_cast<int64_t>(t)) lo = mid + 1u;
        else hi = mid;
    }
    return lo >= 1u && lo <= s.batch ? static_cast<int>(lo) - 1 : -1;
}
// Row of the cache that holds packed row t (head 0, K), or -1 where there is none.
__device__ __forceinline__ int64_t row_of(const KvView &kv, const KvSeqs &s, uint32_t t, unsigned int *error_word) {
    const int b = seq_of(s, t);
    if (b < 0) return -1;
    const int64_t end = s.cu ? static_cast<int64_t>(s.cu[b + 1]) : static_cast<int64_t>(b + 1) * s.per;
    const int64_t pos = static_cast<int64_t>(s.lens[b]) - (end - static_cast<int64_t>(t));
    if (pos < 0) return -1;
    const int64_t pi = pos >> kv.page_shift;
    const int32_t page = pi < s.width ? s.table[static_cast<uint64_t>(b) * s.table_stride + static_cast<uint64_t>(pi)] : -1;
    if (page < 0 || static_cast<uint32_t>(page) >= kv.pages) {
        atomicOr(error_word, kKvBadTable);
        return -1;
    }
    return ((static_cast<int64_t>(page) * 2 * kv.kv_heads) << kv.page_shift) + (pos & (kv.page_tokens - 1));
}

template <bool F32, bool VEC>
__device__ __forceinline__ void load8(const void *p, uint64_t at, float (&x)[8]) {
    if (F32) {
        const float *f = static_cast<const float *>(p) + at;
        if (VEC) {
            const float4 a = *reinterpret_cast<const float4 *>(f), b = *reinterpret_cast<const float4 *>(f + 4);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = f[i];
        }
    } else {
        const uint16_t *f = static_cast<const uint16_t *>(p) + at;
        if (VEC) {
            const uint4 a = *reinterpret_cast<const uint4 *>(f);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = bf16_f32(f[i]);
        }
    }
}
template <bool F32, bool VEC>
__device__ __forceinline__ void store8(void *p, uint64_t at, const float (&x)[8]) {
    if (F32) {
        float *f = static_cast<float *>(p) + at;
        if (VEC) {
            *reinterpret_cast<float4 *>(f) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4 *>(f + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = x[i];
        }
    } else {
        uint16_t *f = static_cast<uint16_t *>(p) + at;
        if (VEC) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = attend::pack_bf16x2(x[2 * i], x[2 * i + 1]);
            *reinterpret_cast<uint4 *>(f) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = static_cast<uint16_t>(f32_bf16(x[i]));
        }
    }
}

struct KvRows {
    const void *k, *v;
    KvStrides ks, vs;
};

// Both kernels: a CTA takes `tokens` packed rows; it looks up where they lie once, and its threads then walk the rows'
// vectors of 8 values (K heads, then V heads).  What bounds them: HBM, with enough rows; the index arithmetic has to stay
// small beside 8 values' work, so it is carried from step to step and each thread has up to kUnroll loads in flight (fewer in calls
// whose CTAs have few rows of few heads).
constexpr int kMaxTokens = 32;    // of a CTA
constexpr int kUnroll = 4;

// Position of a thread in the vectors of the CTA's rows.  FIXED: the vectors of a row divide the CTA's threads, so that a thread
// stays with one of them and only the row changes.
struct Place {
    uint32_t which, head, vec;
    uint32_t token;      // of the CTA
    int64_t row;         // of the cache; -1: none
};
template <bool FIXED>
struct Walk {
    uint32_t token, v, h;
    uint32_t step_token, step_v, per_token, per_row, per_row_inv;   // the last: 2^32 over the vectors of a row, rounded up
    const int64_t *rows;
    uint32_t tokens;

    __device__ __forceinline__ Walk(const KvView &kv, uint32_t tokens_, const int64_t *rows_) : rows(rows_), tokens(tokens_) {
        per_row = kv.head_dim >> 3;              // at most 32, so that the product in split() is exact for v below 2^27
        per_row_inv = 0xFFFFFFFFu / per_row + 1u;
        per_token = 2u * kv.kv_heads * per_row;
        token = threadIdx.x / per_token;
        v = threadIdx.x - token * per_token;
        step_token = kThreadsKv / per_token;
        step_v = kThreadsKv - step_token * per_token;
        split();
    }
    __device__ __forceinline__ void split() { h = __umulhi(v, per_row_inv); }
    __device__ __forceinline__ Place at(const KvView &kv) const {
        Place p;
        p.vec = v - h * per_row;
        p.which = h >= kv.kv_heads ? 1u : 0u;
        p.head = h - p.which * kv.kv_heads;
        p.token = token;
        const int64_t row0 = token < tokens ? rows[token] : -1;
        p.row = row0 < 0 ? -1 : row0 + (static_cast<int64_t>(h) << kv.page_shift);
        return p;
    }
    __device__ __forceinline__ void next() {
        token += step_token;
        if (FIXED) return;
        v += step_v;
        if (v >= per_token) v -= per_token, ++token;
        split();
    }
};
__device__ __forceinline__ void check_rows(const KvSeqs &s, unsigned int *error_word) {
    if (blockIdx.x == 0 && threadIdx.x == 0 && s.cu && s.cu[s.batch] > static_cast<int64_t>(s.total)) atomicOr(error_word, kKvBadRows);
}
__device__ __forceinline__ void find_rows(const KvView &kv, const KvSeqs &seqs, uint32_t tokens, int64_t *s_row, unsigned int *error_word) {
    check_rows(seqs, error_word);
    for (uint32_t x = threadIdx.x; x < tokens; x += kThreadsKv) {
        const uint64_t t = static_cast<uint64_t>(blockIdx.x) * tokens + x;
        s_row[x] = t < seqs.total ? row_of(kv, seqs, static_cast<uint32_t>(t), error_word) : -1;
    }
    __syncthreads();
}
// The tensor that holds a place's values, and their element in it.  (Selected, not indexed: an indexed parameter is copied to
// local memory: 113 against 96 us for the read-back of 72k tokens of 8 heads.)
__device__ __forceinline__ const void *tensor_of(const KvRows &x, const Place &p) { return p.which ? x.v : x.k; }
__device__ __forceinline__ uint64_t element_of(const KvRows &x, const Place &p, uint64_t first_token) {
    const uint64_t token_stride = p.which ? x.vs.token : x.ks.token, head_stride = p.which ? x.vs.head : x.ks.head;
    return (first_token + p.token) * token_stride + p.head * head_stride + p.vec * 8u;
}

// Pairs of f32 in one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// a / b, rounded to nearest, for r = 1 / b rounded to nearest: the product a r and one correction by its exact remainder
// (Markstein's theorem).  The codes are those of a division, ties included, at two instructions more than a product.
__device__ __forceinline__ uint64_t rounded_quotient2(uint64_t a, uint64_t minus_b, uint64_t r) {
    const uint64_t q = mul2(a, r);
    return fma2(fma2(q, minus_b, a), r, q);
}

// The group's lanes (G / 8 neighbours) share minimum and maximum.
template <bool F32, bool VEC, bool FIXED>
__global__ void __launch_bounds__(kThreadsKv) gaf_kv_append_kernel(const KvView kv, const KvSeqs seqs, const KvRows in, uint32_t tokens,
                                                                   unsigned int *error_word) {
    __shared__ int64_t s_row[kMaxTokens];
    find_rows(kv, seqs, tokens, s_row, error_word);
    Walk<FIXED> walk(kv, tokens, s_row);
    const uint64_t first_token = static_cast<uint64_t>(blockIdx.x) * tokens;
    const uint32_t steps = (tokens * walk.per_token + kThreadsKv - 1u) / kThreadsKv;
    const float maxq = kv.bits == 4u ? 15.0f : 255.0f, inv_maxq = __frcp_rn(0.5f * maxq);
    for (uint32_t step = 0; step < steps; step += kUnroll) {
        Place pl[kUnroll];
        float x[kUnroll][8];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k, walk.next()) {
            pl[k] = walk.at(kv);
            if (pl[k].row >= 0) {
                load8<F32, VEC>(tensor_of(in, pl[k]), element_of(in, pl[k], first_token), x[k]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[k][i] = 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            if (step + k >= steps) break;
            float lo = x[k][0], hi = x[k][0];
#pragma unroll
            for (int i = 1; i < 8; ++i) {
                lo = min_nan(lo, x[k][i]);
                hi = max_nan(hi, x[k][i]);
            }
            for (uint32_t o = kv.group >> 4; o >= 1u; o >>= 1) {
                lo = min_nan(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
                hi = max_nan(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
            }
            const float range = 0.5f * hi - 0.5f * lo;             // of halves: finite for finite values
            uint32_t sraw = f32_bf16(range * inv_maxq), braw = f32_bf16(lo);
            if ((braw & 0x7FFFu) == 0x7F80u) braw -= 1u;           // f32 values beyond the largest bf16
            float s = bf16_f32(sraw);
            if (s < FLT_MIN) s = 0.0f, sraw = 0u;
            const bool finite = range <= FLT_MAX;
            if (!finite) sraw = braw = 0x7FC0u, s = 0.0f;          // an infinity or a NaN in the group
            const float half_b = 0.5f * bf16_f32(braw), half_s = 0.5f * s;
            const float r = s > 0.0f ? __frcp_rn(half_s) : 0.0f;
            // adding 1.5 * 2^23 rounds to an integer (ties to even) and leaves it in the low bits
            constexpr float kMagic = 12582912.0f;
            float y[8];
            const uint64_t half2 = pair(0.5f, 0.5f), minus_hb2 = pair(-half_b, -half_b), minus_hs2 = pair(-half_s, -half_s), r2 = pair(r, r);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const uint64_t c2 = rounded_quotient2(fma2(pair(x[k][i], x[k][i + 1]), half2, minus_hb2), minus_hs2, r2);
                float c, d;
                asm("mov.b64 {%0, %1}, %2;" : "=f"(c), "=f"(d) : "l"(c2));
                y[i] = fminf(fmaxf(c, 0.0f), maxq) + kMagic;
                y[i + 1] = fminf(fmaxf(d, 0.0f), maxq) + kMagic;
            }
            if (pl[k].row < 0) continue;
            uint8_t *dst = kv.packed + pl[k].row * kv.row_bytes + pl[k].vec * kv.bits;   // 8 codes are `bits` bytes
            auto bytes = [](float a, float b, float c, float d) {      // the low bytes of four numbers
                return attend::prmt(attend::prmt(__float_as_uint(a), __float_as_uint(b), 0x0040u), attend::prmt(__float_as_uint(c), __float_as_uint(d), 0x0040u), 0x5410u);
            };
            if (kv.bits == 8u) {
                *reinterpret_cast<uint2 *>(dst) = make_uint2(bytes(y[0], y[1], y[2], y[3]), bytes(y[4], y[5], y[6], y[7]));
            } else {
                float z[4];       // code + 16 code' + 1.5 * 2^23, exact
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = fmaf(y[2 * i + 1] - kMagic, 16.0f, y[2 * i]);
                *reinterpret_cast<uint32_t *>(dst) = bytes(z[0], z[1], z[2], z[3]);
            }
            if ((pl[k].vec & ((kv.group >> 3) - 1u)) == 0u) {
                const int64_t g = pl[k].row * kv.groups + (pl[k].vec * 8u >> kv.group_shift);
                kv.scales[g] = static_cast<uint16_t>(sraw);
                kv.biases[g] = static_cast<uint16_t>(braw);
            }
        }
    }
}

template <bool F32, bool VEC, bool FIXED>
__global__ void __launch_bounds__(kThreadsKv) gaf_kv_read_kernel(const KvView kv, const KvSeqs seqs, const KvRows out, uint32_t tokens,
                                                                 unsigned int *error_word) {
    __shared__ int64_t s_row[kMaxTokens];
    find_rows(kv, seqs, tokens, s_row, error_word);
    Walk<FIXED> walk(kv, tokens, s_row);
    const uint64_t first_token = static_cast<uint64_t>(blockIdx.x) * tokens;
    const uint32_t steps = (tokens * walk.per_token + kThreadsKv - 1u) / kThreadsKv;
    for (uint32_t step = 0; step < steps; step += kUnroll) {
        Place pl[kUnroll];
        uint2 code[kUnroll];
        float s[kUnroll], b[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k, walk.next()) {
            pl[k] = walk.at(kv);
            if (pl[k].row < 0) continue;
            const uint8_t *src = kv.packed + pl[k].row * kv.row_bytes + pl[k].vec * kv.bits;
            if (kv.bits == 8u) code[k] = *reinterpret_cast<const uint2 *>(src);
            else code[k].x = *reinterpret_cast<const uint32_t *>(src);
            const int64_t g = pl[k].row * kv.groups + (pl[k].vec * 8u >> kv.group_shift);
            s[k] = bf16_f32(kv.scales[g]);
            b[k] = bf16_f32(kv.biases[g]);
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            if (pl[k].row < 0) continue;
            float x[8];
            if (kv.bits == 8u) {
#pragma unroll
                for (int i = 0; i < 8; ++i)      // 2^23 + code, less 2^23
                    x[i] = fmaf(__uint_as_float(attend::prmt(i < 4 ? code[k].x : code[k].y, 0x4B000000u, 0x7650u | (i & 3))) - 8388608.0f, s[k], b[k]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = fmaf(__uint_as_float(((code[k].x >> (4 * i)) & 15u) | 0x4B000000u) - 8388608.0f, s[k], b[k]);
            }
            store8<F32, VEC>(const_cast<void *>(tensor_of(out, pl[k])), element_of(out, pl[k], first_token), x);
        }
    }
}

// Rows of a CTA: as many as leave eight CTAs for each SM, so that the look-up in front of them is paid seldom and hidden
uint32_t rows_of_cta(const KvSeqs &seqs, int sm_count) {
    const uint32_t n = seqs.total / (static_cast<uint32_t>(sm_count) * 8u);
    return n < 1u ? 1u : n < static_cast<uint32_t>(kMaxTokens) ? n : kMaxTokens;
}

bool vec_ok(const void *p, KvStrides st, bool f32) {
    const uint64_t n = f32 ? 4u : 8u;   // elements of 16 bytes
    return reinterpret_cast<uintptr_t>(p) % 16u == 0u && st.token % n == 0u && st.head % n == 0u;
}

// ---- attention for any head size ------------------------------------------------------------------------------------
// CTA = one query row (token, head); its warps take every fourth run of 32 keys.  In a run a lane owns a key for the scores
// and 1 / 32 of the head for the weighted sum; one running maximum and sum per warp, joined at the end.
constexpr int kWarpsGen = 4;
constexpr int kMaxDim = 256;

__device__ __forceinline__ uint32_t code_at(const KvView &kv, const uint8_t *row, uint32_t d) {
    return kv.bits == 8u ? row[d] : (row[d >> 1] >> (4u * (d & 1u))) & 15u;
}

template <bool F32>
__global__ void __launch_bounds__(kWarpsGen * 32) gaf_attention_generic_kernel(const AttnArgs a) {
    __shared__ float s_q[kMaxDim];
    __shared__ float s_o[kWarpsGen][kMaxDim];
    __shared__ float s_m[kWarpsGen], s_l[kWarpsGen];
    const KvView &kv = a.kv;
    const uint32_t t = blockIdx.x / a.q_heads, hq = blockIdx.x % a.q_heads, head = hq / (a.q_heads / kv.kv_heads);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t D = kv.head_dim;
    check_rows(a.seqs, a.error_word);
    const int b = seq_of(a.seqs, t);
    if (b < 0) return;
    const int64_t begin = a.seqs.cu ? static_cast<int64_t>(a.seqs.cu[b]) : static_cast<int64_t>(b) * a.seqs.per;
    const int64_t end = a.seqs.cu ? static_cast<int64_t>(a.seqs.cu[b + 1]) : begin + a.seqs.per;
    if (static_cast<int64_t>(t) - begin >= static_cast<int64_t>(a.max_new)) {
        if (threadIdx.x == 0) atomicOr(a.error_word, kKvBadCount);
        return;
    }
    bool bad = false;
    for (uint32_t d = threadIdx.x; d < D; d += kWarpsGen * 32) {
        const uint64_t at = t * a.qs.token + hq * a.qs.head + d;
        s_q[d] = F32 ? static_cast<const float *>(a.q)[at] : bf16_f32(static_cast<const uint16_t *>(a.q)[at]);
        bad |= !(fabsf(s_q[d]) <= FLT_MAX);
    }
    // a row that is not finite gives NaN wherever it sees a key (its scores may all be -inf)
    const float scale = __syncthreads_or(bad) ? __uint_as_float(0x7FC00000u) : a.scale;
    const int64_t limit = static_cast<int64_t>(a.seqs.lens[b]) - (end - 1 - static_cast<int64_t>(t));   // keys seen
    float m = -INFINITY, l = 0.0f, o[kMaxDim / 32];
#pragma unroll
    for (int i = 0; i < kMaxDim / 32; ++i) o[i] = 0.0f;
    for (int part = a.prefix_table ? 0 : 1; part < 2; ++part) {
        const int64_t keys = part == 0 ? static_cast<int64_t>(a.prefix_len) : limit;
        const int32_t *table = part == 0 ? a.prefix_table : a.seqs.table + static_cast<uint64_t>(b) * a.seqs.table_stride;
        for (int64_t j0 = warp * 32; j0 < keys; j0 += kWarpsGen * 32) {
            const int64_t j = j0 + lane, pi = j >> kv.page_shift;
            int64_t krow = -1;
            if (j < keys) {
                const int32_t page = part == 0 || pi < a.seqs.width ? table[pi] : -1;
                if (page < 0 || static_cast<uint32_t>(page) >= kv.pages) atomicOr(a.error_word, kKvBadTable);
                else krow = ((static_cast<int64_t>(page) * 2 * kv.kv_heads + head) << kv.page_shift) + (j & (kv.page_tokens - 1));
            }
            float score = -INFINITY;
            if (krow >= 0) {
                score = 0.0f;
                const uint8_t *row = kv.packed + krow * kv.row_bytes;
                for (uint32_t g = 0; g < kv.groups; ++g) {
                    const float s = bf16_f32(kv.scales[krow * kv.groups + g]), bias = bf16_f32(kv.biases[krow * kv.groups + g]);
                    for (uint32_t d = g * kv.group; d < (g + 1u) * kv.group; ++d)
                        score = fmaf(s_q[d], fmaf(static_cast<float>(code_at(kv, row, d)), s, bias), score);
                }
                score *= scale;
            }
            float top = score;
            for (int x = 16; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
            const float m1 = fmaxf(m, top);
            if (m1 == -INFINITY && !__any_sync(0xFFFFFFFFu, score != score)) continue;   // no key of the run can be seen
            const float keep = m == m1 ? 1.0f : expf(m - m1);
            const float p = krow >= 0 ? expf(score - m1) : 0.0f;
            m = m1;
            l *= keep;
            float sum = p;
            for (int x = 16; x >= 1; x >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
            l += sum;
#pragma unroll
            for (int i = 0; i < kMaxDim / 32; ++i) o[i] *= keep;
            for (int k = 0; k < 32; ++k) {
                const int64_t kr = __shfl_sync(0xFFFFFFFFu, krow, k);
                const float pk = __shfl_sync(0xFFFFFFFFu, p, k);
                if (kr < 0) continue;
                const int64_t vrow = kr + (static_cast<int64_t>(kv.kv_heads) << kv.page_shift);
                const uint8_t *row = kv.packed + vrow * kv.row_bytes;
#pragma unroll
                for (int i = 0; i < kMaxDim / 32; ++i) {
                    const uint32_t d = i * 32u + lane;
                    if (d >= D) continue;
                    const int64_t g = vrow * kv.groups + (d >> kv.group_shift);
                    o[i] = fmaf(pk, fmaf(static_cast<float>(code_at(kv, row, d)), bf16_f32(kv.scales[g]), bf16_f32(kv.biases[g])), o[i]);
                }
            }
        }
    }
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
    for (int i = 0; i < kMaxDim / 32; ++i)
        if (i * 32u + lane < D) s_o[warp][i * 32 + lane] = o[i];
    __syncthreads();
    float top = -INFINITY, total = 0.0f;
    for (int w = 0; w < kWarpsGen; ++w) top = fmaxf(top, s_m[w]);
    for (int w = 0; w < kWarpsGen; ++w) total += s_m[w] == -INFINITY ? s_l[w] : s_l[w] * expf(s_m[w] - top);
    for (uint32_t d = threadIdx.x; d < D; d += kWarpsGen * 32) {
        float v = 0.0f;
        for (int w = 0; w < kWarpsGen; ++w) v += s_m[w] == -INFINITY ? s_o[w][d] : s_o[w][d] * expf(s_m[w] - top);
        v = total == 0.0f ? 0.0f : v / total;
        const uint64_t at = t * a.os.token + hq * a.os.head + d;
        if (F32) static_cast<float *>(a.out)[at] = v;
        else static_cast<uint16_t *>(a.out)[at] = static_cast<uint16_t>(f32_bf16(v));
    }
}

}  // namespace

cudaError_t kv_append(const KvView &kv, const KvSeqs &seqs, bool f32, const void *k, KvStrides ks, const void *v, KvStrides vs,
                      unsigned int *error_word, int sm_count, cudaStream_t stream) {
    if (seqs.total == 0) return cudaSuccess;
    const KvRows in = {k, v, ks, vs};
    const bool vec = vec_ok(k, ks, f32) && vec_ok(v, vs, f32);
    const uint32_t n = rows_of_cta(seqs, sm_count), grid = (seqs.total - 1u) / n + 1u;
    const bool fixed = kThreadsKv % (2u * kv.kv_heads * (kv.head_dim / 8u)) == 0u;
    auto go = [&](auto kernel) { kernel<<<grid, kThreadsKv, 0, stream>>>(kv, seqs, in, n, error_word); };
    if (f32 && vec && fixed) go(gaf_kv_append_kernel<true, true, true>);
    else if (f32 && vec) go(gaf_kv_append_kernel<true, true, false>);
    else if (f32) go(gaf_kv_append_kernel<true, false, false>);
    else if (vec && fixed) go(gaf_kv_append_kernel<false, true, true>);
    else if (vec) go(gaf_kv_append_kernel<false, true, false>);
    else go(gaf_kv_append_kernel<false, false, false>);
    return cudaGetLastError();
}

cudaError_t kv_read(const KvView &kv, const KvSeqs &seqs, bool f32, void *k, KvStrides ks, void *v, KvStrides vs,
                    unsigned int *error_word, int sm_count, cudaStream_t stream) {
    if (seqs.total == 0) return cudaSuccess;
    const KvRows out = {k, v, ks, vs};
    const bool vec = vec_ok(k, ks, f32) && vec_ok(v, vs, f32);
    const uint32_t n = rows_of_cta(seqs, sm_count), grid = (seqs.total - 1u) / n + 1u;
    const bool fixed = kThreadsKv % (2u * kv.kv_heads * (kv.head_dim / 8u)) == 0u;
    auto go = [&](auto kernel) { kernel<<<grid, kThreadsKv, 0, stream>>>(kv, seqs, out, n, error_word); };
    if (f32 && vec && fixed) go(gaf_kv_read_kernel<true, true, true>);
    else if (f32 && vec) go(gaf_kv_read_kernel<true, true, false>);
    else if (f32) go(gaf_kv_read_kernel<true, false, false>);
    else if (vec && fixed) go(gaf_kv_read_kernel<false, true, true>);
    else if (vec) go(gaf_kv_read_kernel<false, true, false>);
    else go(gaf_kv_read_kernel<false, false, false>);
    return cudaGetLastError();
}

cudaError_t attention_generic(const AttnArgs &a, bool f32, cudaStream_t stream) {
    if (a.seqs.total == 0) return cudaSuccess;
    const unsigned int grid = a.seqs.total * a.q_heads;
    if (f32) gaf_attention_generic_kernel<true><<<grid, kWarpsGen * 32, 0, stream>>>(a);
    else gaf_attention_generic_kernel<false><<<grid, kWarpsGen * 32, 0, stream>>>(a);
    return cudaGetLastError();
}

// Up to how many rows of a cached head and sequence the register-path kernel takes bf16 calls; `items`: sequences x cached heads.
// Its time grows with the rows, the tcgen05 kernel's hardly does; with fewer items than SMs every item is cut across many CTAs,
// and the larger units of the tcgen05 kernel leave fewer parts to join.  Measured (8 cached heads, 8 bits; register path
// against tcgen05, us), 24 sequences of 3000 tokens, then 4 of 800:
//   heads of 128   12 rows 61 / 113, 30 / 27    16 rows 63 / 114, 33 / 27    24 rows 110 / 114, 47 / 28    (32 rows: 168 / 112, 65 / 27)
//   heads of 64    12 rows 37 / 90, 21 / 22     16 rows 37 / 90, 21 / 22     24 rows 44 / 90, 28 / 22      32 rows 55 / 91, 37 / 22
// (times of captured calls; the tcgen05 kernel's joining pass is a launch of its own, some 4 us more where launches follow one
// another from the host, which decides for 16 rows against a shared prefix: 38 against 40 us for one of 1111 tokens.  With 4 bits:
// heads of 128 16 rows 62 / 112, 24 rows 87 / 114; otherwise the same.)
uint64_t narrow_rows(uint32_t head_dim, uint64_t items, bool prefix, int sm_count) {
    const bool few = items < static_cast<uint64_t>(sm_count);
    return head_dim == 128u ? (!few ? 24u : prefix ? 16u : 8u) : (few ? 16u : 32u);
}

bool attention_fast(const KvView &kv) { return kv.head_dim == 64u || kv.head_dim == 128u; }
// the tickets of the narrow kernel, then the cuts of the wide one
size_t attention_ticket_count(int sm_count) {
    static_assert(sizeof(attend::Cut) % sizeof(unsigned int) == 0 && attend::kMaxCtas % 2 == 0, "the cuts are 8-byte aligned");
    return static_cast<size_t>(sm_count) * (attend::kMaxCtas + sizeof(attend::Cut) / sizeof(unsigned int));
}
size_t attention_partial_bytes(int sm_count) {
    return static_cast<size_t>(sm_count) * attend::kMaxPartRows * (attend::kMaxDim + 2) * sizeof(float);
}

cudaError_t make_kv_tmap(const KvView &kv, CUtensorMap *out) {
    const uint64_t rows = static_cast<uint64_t>(kv.pages) * 2u * kv.kv_heads * kv.page_tokens;
    const uint32_t box = kv.page_tokens < static_cast<uint32_t>(attend::kKeys) ? kv.page_tokens : attend::kKeys;
    return make_row_tmap(kv.packed, rows, kv.row_bytes, box, out);
}

cudaError_t attention(const AttnArgs &a, const CUtensorMap &tmap, const AttnWorkspace &ws, bool f32, int sm_count, cudaStream_t stream) {
    attend::Params p;
    p.a = a;
    p.per_kv = a.q_heads / a.kv.kv_heads;
    p.partials = ws.partials;
    p.tickets = ws.tickets;
    p.cuts = reinterpret_cast<attend::Cut *>(ws.tickets + static_cast<size_t>(sm_count) * attend::kMaxCtas);
    p.prefix_o = ws.prefix;
    p.prefix_lse = ws.prefix ? ws.prefix + static_cast<uint64_t>(a.seqs.total) * a.q_heads * a.kv.head_dim : nullptr;
    p.o_vec = reinterpret_cast<uintptr_t>(a.out) % (f32 ? 16u : 8u) == 0u && a.os.token % 4u == 0u && a.os.head % 4u == 0u;
    p.q_vec = vec_ok(a.q, a.qs, f32);
    auto run = [&](uint64_t rows) {
        const uint64_t items = static_cast<uint64_t>(p.prefix_pass ? 1u : a.seqs.batch) * a.kv.kv_heads;
        if (!f32 && rows > narrow_rows(a.kv.head_dim, items, p.prefix_pass != 0u, sm_count)) {
            p.row_tiles = static_cast<uint32_t>((rows + 255u) / 256u);
            p.elements = p.prefix_pass ? p.row_tiles : p.row_tiles * a.seqs.batch;
            return attend::launch_wide(p, tmap, sm_count, stream);
        }
        // 8 rows a tile cost least where they suffice; more rows read the cache less often
        const int nt = rows <= 8u ? 1 : rows <= 16u || f32 ? 2 : rows <= 24u ? 3 : 4;
        p.row_tiles = static_cast<uint32_t>((rows + 8u * nt - 1u) / (8u * nt));
        p.elements = p.prefix_pass ? p.row_tiles : p.row_tiles * a.seqs.batch;
        const int limbs = f32 ? 2 : 1;
        if (a.kv.head_dim == 64u)
            return a.kv.bits == 4u ? attend::launch_d64_b4(p, tmap, nt, limbs, sm_count, stream) : attend::launch_d64_b8(p, tmap, nt, limbs, sm_count, stream);
        return a.kv.bits == 4u ? attend::launch_d128_b4(p, tmap, nt, limbs, sm_count, stream) : attend::launch_d128_b8(p, tmap, nt, limbs, sm_count, stream);
    };
    p.merge_prefix = 0u;
    if (a.prefix_table) {
        p.prefix_pass = 1u;
        const cudaError_t e = run(static_cast<uint64_t>(a.seqs.total) * p.per_kv);
        if (e != cudaSuccess) return e;
        p.merge_prefix = 1u;
    }
    p.prefix_pass = 0u;
    return run(static_cast<uint64_t>(a.max_new) * p.per_kv);
}

}  // namespace tgaf
