// Attention over the quantised KV cache on the tensor cores' register path, for few query rows per cached head.
//
//   out[r] = sum_j softmax_j(scale q_r . K_j) V_j,   K_jd = c_jd s_jg + b_jg (codes c, scale s and bias b of group g of d)
//
// Mathematics.  The affine map is taken out of the sums, so that the matrix products run on the codes as they are (exact in
// f16) and neither keys nor values are rounded:
//   q_r . K_j  = sum_g s_jg (sum_{d in g} q_rd (c_jd - h)) + (b_jg + h s_jg) (sum_{d in g} q_rd),   h = 2^(bits - 1)
//   out_rd     = sum_j (p_rj s_jg) (c_jd - h) + sum_j p_rj (b_jg + h s_jg)
// q is scaled by a power of two per row (so that it fits f16, which holds bf16's 8 bits and the codes) and the products
// p s are rounded to f16 once (2^-11 of each); everything else is f32.  The codes are centred because roundings
// are relative to s |c - h|: with plain codes they are relative to the distance from the group's minimum, some four times
// the value itself.  f16 and not bf16 for the products, although s is the caller's and of any size: unpacking a
// code to f16 takes two instructions a pair, to bf16 (8 bits of code in 8 bits of mantissa) four.  The range is kept by powers
// of two: weights p are formed against a reference m, an integer within 2^8 of the row's largest score (base 2), and the products of
// each group have a factor of their own per row, which keeps the largest of them between 2^4 and 2^15.  So a group whose
// scales are far below its neighbours' has weights of as many bits, and a weight loses some only below 2^-18 of the group's
// largest one, where its step is 2^-28 of that.  (With one factor for all groups, from the largest scale of each key, a group
// 2^20 below it was 1.6e-3 off in f32.  A factor per group costs some 1 % per unit, 0.3 to 1 us where a segment begins: 16
// sequences of 2560 tokens, 32 heads on 8, 8 bits: 24.8 -> 25.4 us, f32 28.5 -> 29.5.)
// LIMBS = 2 (f32 q): q and p s are split into two f16 terms each (22 bits).
//
// Both products are formed transposed (keys as the 16 rows of the MMA's A operand, query rows as its 8 columns): with one
// new token and 4 or 8 query heads per cached head, 8 columns are what there is, and an A operand of query rows would leave
// half of every instruction empty.  The scores' accumulators turn into the second product's B operand by movmatrix.
//
// What bounds it: the cache is read once (HBM), and every code is unpacked once (2 to 3 instructions per pair).  A unit is 64
// keys of one (head, sequence, row tile): codes by TMA (swizzled, so that the fragment reads below hit every bank once),
// scales and biases by bulk copies into the same ring stage.  Each of the four consumer warps owns 16 keys of the unit for
// both products, with its own reference and sum: no barrier between warps but at the end of a segment.  (32 keys a warp and
// units in turns: 85 against 78 us for 64 sequences of 2048 to 4096 tokens, 32 heads on 8, 8 bits: the code grows, and what is
// executed once a segment comes from far.)  The units of
// all items are cut into equal contiguous ranges over a grid that fills the GPU once, whatever the lengths are; an item cut
// across CTAs is joined by the last CTA to finish, in CTA order (the result does not depend on timing).
#pragma once
#include "gaf_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

namespace tgaf {
namespace attend {

constexpr int kKeys = 64;                      // keys of a unit
constexpr int kConsumers = 4;                  // consumer warps
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr float kLazy = 8.0f;                  // the reference follows only when it is exceeded by 2^8
constexpr int kTarget = 4;                     // a group's factor brings the largest p s of a row to 2^4 to 2^5 when it is set
constexpr int kMostExp = 15;                   // ... and keeps it below 2^15 (f16)
constexpr float kNoMax = -3.0e38f;             // reference of a row that has seen no key: finite, so that -inf scores give 0

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ float bf16_f32(uint32_t raw) { return __uint_as_float(raw << 16); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(20000u)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded: gives up after four seconds, or once another role of the CTA has.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag, unsigned int *error_word) {
    if (mbar_test(bar, parity)) return true;
    unsigned long long t0 = 0ull;
    for (uint32_t it = 0; it < (1u << 22); ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 63u) == 63u) {
            if (*abort_flag) return false;
            unsigned long long now;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (t0 == 0ull) t0 = now;
            else if (now - t0 > 4000000000ull) break;
        }
    }
    atomicOr(error_word, 0x10000u);
    *abort_flag = 1u;
    return false;
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *tmap, uint32_t c0, uint32_t c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
__device__ __forceinline__ uint32_t add_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// 2^e; 0 below the normal numbers
__device__ __forceinline__ float pow2_or_0(int e) { return e < -126 ? 0.0f : __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 mul_pair(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\t"
        "mov.b64 x, {%2, %3};\n\t"
        "mov.b64 y, {%4, %5};\n\t"
        "mul.rn.f32x2 x, x, y;\n\t"
        "mov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// barriers of the consumer warps
__device__ __forceinline__ void bar_consumers() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool bar_consumers_or(bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, 1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(v ? 1u : 0u)
        : "memory");
    return r != 0u;
}

struct Params {
    AttnArgs a;
    uint32_t per_kv;        // query heads of a cached head
    uint32_t row_tiles;     // row tiles of the largest sequence
    uint32_t elements;      // sequences x row_tiles
    uint32_t prefix_pass;   // 1: all rows against the shared prefix, results to prefix_o / prefix_lse
    uint32_t merge_prefix;  // 1: rows start from prefix_o / prefix_lse
    float *prefix_o;        // [rows][D] f32, normalised; row = token * q_heads + head
    float *prefix_lse;      // [rows], base 2
    float *partials;        // [2 * gridDim.x][R * (D + 2)]
    unsigned int *tickets;  // [gridDim.x], zero between launches
    struct Cut *cuts;       // [gridDim.x] of the wide kernel
    uint32_t q_vec, o_vec;  // rows of q / out can be read / written by vectors
};

// An item is one (cached head, element); an element one row tile of one sequence.
struct Item {
    uint32_t tiles;      // units
    int32_t keys;        // keys that its last row sees (within the table)
    int32_t first_seen;  // keys that its first row sees
    uint32_t rows;       // rows of the sequence
    uint32_t row0;       // first row of the tile
    int32_t seen0;       // keys that the sequence's first new token sees
    int64_t token0;      // packed row of the sequence's first new token
    int32_t seq;
};

// An item that begins in a CTA of the wide kernel and goes on in the next `parts` - 1; parts = 0: none.
struct Cut {
    Item item;
    uint32_t head, parts;
};

template <int R, int KEYS>
__device__ __forceinline__ Item item_at(const Params &p, uint32_t n) {
    Item it;
    const KvSeqs &s = p.a.seqs;
    const uint32_t b = n / p.row_tiles;
    it.row0 = (n - b * p.row_tiles) * R;
    it.seq = static_cast<int32_t>(b);
    if (p.prefix_pass) {
        it.rows = s.total * p.per_kv;
        it.token0 = 0;
        it.keys = it.first_seen = it.seen0 = static_cast<int32_t>(p.a.prefix_len);
        it.tiles = (p.a.prefix_len + KEYS - 1) / KEYS;
        return it;
    }
    int64_t begin, count;
    if (s.cu) {
        begin = s.cu[b];
        count = static_cast<int64_t>(s.cu[b + 1]) - begin;
    } else {
        begin = static_cast<int64_t>(b) * s.per;
        count = s.per;
    }
    const int64_t len = s.lens[b];
    if (count > static_cast<int64_t>(p.a.max_new)) {
        atomicOr(p.a.error_word, kKvBadCount);
    }
    int64_t take = count > static_cast<int64_t>(p.a.max_new) ? static_cast<int64_t>(p.a.max_new) : count;
    if (count > 0 && begin + count > static_cast<int64_t>(s.total)) {
        atomicOr(p.a.error_word, kKvBadRows);
        take = begin + take > static_cast<int64_t>(s.total) ? static_cast<int64_t>(s.total) - begin : take;
    }
    it.rows = take > 0 && begin >= 0 ? static_cast<uint32_t>(take) * p.per_kv : 0u;
    it.token0 = begin;
    it.keys = it.first_seen = it.seen0 = 0;
    it.tiles = 0;
    if (it.row0 >= it.rows) return it;
    const int64_t top = static_cast<int64_t>(s.width) << p.a.kv.page_shift;
    const int64_t seen0 = len - count + 1;
    const uint32_t last_row = it.row0 + R <= it.rows ? it.row0 + R - 1u : it.rows - 1u;
    int64_t keys = seen0 + last_row / p.per_kv;
    if (keys > top) {
        atomicOr(p.a.error_word, kKvBadTable);
        keys = top;
    }
    const int64_t first = seen0 + it.row0 / p.per_kv;
    it.keys = static_cast<int32_t>(keys < 0 ? 0 : keys);
    it.first_seen = static_cast<int32_t>(first < 0 ? 0 : first > keys ? keys : first);
    it.seen0 = static_cast<int32_t>(seen0 < -0x40000000ll ? -0x40000000ll : seen0);
    it.tiles = it.keys > 0 ? (static_cast<uint32_t>(it.keys) + KEYS - 1u) / KEYS : 1u;   // an item without keys is one empty unit
    return it;
}

// The item at (head, elem), or the next one that has units; there is one.
template <int R, int KEYS>
__device__ __forceinline__ Item next_item(const Params &p, uint32_t &head, uint32_t &elem) {
    Item item = item_at<R, KEYS>(p, elem);
    while (item.tiles == 0u) {
        if (++elem == p.elements) elem = 0u, ++head;
        item = item_at<R, KEYS>(p, elem);
    }
    return item;
}

// 64-bit quotients of numbers that hardly ever need 64 bits (a division in them costs some 150 clocks).
__device__ __forceinline__ uint64_t quotient(uint64_t a, uint64_t b) {
    return ((a | b) >> 32) == 0u ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}
// The CTA's share of all units: equal contiguous ranges, in the order cached head, element, unit.  A sum over the elements
// that every CTA forms alike; false: nothing to do.
struct Range {
    uint64_t u0, u1, units, ctas;
};
template <int R, int KEYS, int THREADS>
__device__ __forceinline__ bool cta_range(const Params &p, uint32_t *s_scan, uint32_t *s_begin, Range &out) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t per_thread = (p.elements + THREADS - 1u) / THREADS;
    const uint32_t n_lo = threadIdx.x * per_thread, n_hi = n_lo + per_thread < p.elements ? n_lo + per_thread : p.elements;
    uint32_t mine = 0;
    for (uint32_t n = n_lo; n < n_hi; ++n) mine += item_at<R, KEYS>(p, n).tiles;
    uint32_t pre = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, pre, o);
        if (lane >= o) pre += v;
    }
    if (lane == 31) s_scan[warp] = pre;
    __syncthreads();
    uint32_t per_head = 0;
    pre -= mine;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) pre += s_scan[w];
        per_head += s_scan[w];
    }
    out.units = static_cast<uint64_t>(per_head) * p.a.kv.kv_heads;
    if (out.units == 0) return false;
    // The row tiles of a prefix pass are items of one size: where that leaves hardly a CTA idle they are cut into as many parts each,
    // so that a CTA has a part of one item and writes one partial result instead of two.  (A prefix of 16384 tokens for 96
    // sequences, 24 items on 148 CTAs: 85 us for its pass, 93 without.  Sequences are not cut so: it would take a single one of 8000
    // tokens from 24 to 18 us, but long 4-bit contexts from 109 to 112 and 16 of 2500 in f32 from 24.7 to 26.6.)
    out.ctas = gridDim.x;
    const uint64_t items = static_cast<uint64_t>(p.elements) * p.a.kv.kv_heads;
    if (p.prefix_pass && items < out.ctas && gridDim.x % static_cast<uint32_t>(items) * 16u <= gridDim.x) out.ctas -= gridDim.x % static_cast<uint32_t>(items);
    if (out.units < out.ctas) out.ctas = out.units;
    if (blockIdx.x >= out.ctas) return false;
    out.u0 = quotient(out.units * blockIdx.x, out.ctas);
    out.u1 = quotient(out.units * (blockIdx.x + 1u), out.ctas);
    const uint32_t first_head = static_cast<uint32_t>(quotient(out.u0, per_head));
    const uint32_t start = static_cast<uint32_t>(out.u0 - static_cast<uint64_t>(first_head) * per_head);
    if (start >= pre && start < pre + mine) {
        uint32_t n = n_lo, at = pre;
        for (;; ++n) {
            const uint32_t t = item_at<R, KEYS>(p, n).tiles;
            if (start < at + t) break;
            at += t;
        }
        s_begin[0] = first_head;
        s_begin[1] = n;
        s_begin[2] = start - at;
    }
    __syncthreads();
    return true;
}

// Four values of a finished row: the prefix's part added, divided by the sum, rounded once.  top: base 2.
template <int D, bool F32>
__device__ __forceinline__ void finish_row(const Params &p, const Item &item, uint32_t head, uint32_t r, uint32_t d, float top, float sum, float4 v) {
    const uint32_t row = item.row0 + r;
    const uint64_t token = static_cast<uint64_t>(item.token0 + row / p.per_kv);
    const uint32_t hq = head * p.per_kv + row % p.per_kv;
    const uint64_t prow = token * p.a.q_heads + hq;
    if (p.prefix_pass) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        *reinterpret_cast<float4 *>(p.prefix_o + prow * D + d) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        if (d == 0) p.prefix_lse[prow] = sum == 0.0f ? -INFINITY : top + log2f(sum);
        return;
    }
    if (p.merge_prefix) {
        const float lse = p.prefix_lse[prow];
        const float both = fmaxf(top, lse);
        const float wa = top == both ? 1.0f : exp2_approx(top - both), wb = lse == both ? 1.0f : exp2_approx(lse - both);
        if (lse != -INFINITY) {
            const float4 x = *reinterpret_cast<const float4 *>(p.prefix_o + prow * D + d);
            v = make_float4(fmaf(x.x, wb, v.x * wa), fmaf(x.y, wb, v.y * wa), fmaf(x.z, wb, v.z * wa), fmaf(x.w, wb, v.w * wa));
            sum = fmaf(sum, wa, wb);
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const float y[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
    const uint64_t at = token * p.a.os.token + hq * p.a.os.head + d;
    if (F32) {
        float *dst = static_cast<float *>(p.a.out) + at;
        if (p.o_vec) *reinterpret_cast<float4 *>(dst) = make_float4(y[0], y[1], y[2], y[3]);
        else dst[0] = y[0], dst[1] = y[1], dst[2] = y[2], dst[3] = y[3];
    } else {
        uint16_t *dst = static_cast<uint16_t *>(p.a.out) + at;
        const uint32_t lo = pack_bf16x2(y[0], y[1]), hi = pack_bf16x2(y[2], y[3]);
        if (p.o_vec) *reinterpret_cast<uint2 *>(dst) = make_uint2(lo, hi);
        else dst[0] = static_cast<uint16_t>(lo), dst[1] = static_cast<uint16_t>(lo >> 16), dst[2] = static_cast<uint16_t>(hi), dst[3] = static_cast<uint16_t>(hi >> 16);
    }
}

template <int D, int BITS, int GROUP, int NT, int LIMBS>
struct Shape {
    static constexpr int R = 8 * NT;                       // rows of a tile
    static constexpr int RB = D * BITS / 8;                // bytes of a cached row
    static constexpr int GS = D / GROUP;                   // stored groups of a row
    static constexpr int PG = GROUP < 64 ? GROUP : 64;     // values that share a step of the products
    static constexpr int NP = D / PG;
    static constexpr int KS = D / 16;                      // k steps of the score product, m tiles of the other
    static constexpr int CODES = kKeys * RB;               // bytes of a unit's K (or V) codes
    static constexpr int SB = kKeys * GS * 2;              // bytes of a unit's K (or V) scales (or biases)
    static constexpr int STAGE = 2 * CODES + ((4 * SB + 1023) / 1024) * 1024;
    static constexpr int QF = LIMBS * NT * KS * 32 * 8;    // q as B fragments
    static constexpr int HALVES = NT >= 2 && NP >= 2 ? 2 : 1;   // the warps' sums are joined D / HALVES values at a time
    static constexpr int OW = D / HALVES + 4;              // pitch of a joined row (floats)
    static constexpr int JOIN = kConsumers * R * OW * 4;
    static constexpr int FACTORS = kConsumers * R * (GS + 1) * 4;      // by warp: factors by group and row, limits by row
    static constexpr int CTAS = NT >= 2 ? 2 : 3;           // per SM
    static constexpr int FIXED = QF + JOIN + FACTORS + 1024;
    static constexpr int FIT = (226 * 1024 / CTAS - 2048 - FIXED) / STAGE;
    static constexpr int STAGES = FIT > 6 ? 6 : FIT;
    static constexpr int SMEM = STAGES * STAGE + FIXED;
    static_assert(STAGES >= 2, "a ring needs two stages");
};

// Row of a 16-key tile that stands at position m (0..7; +8 for the second half): the order in which the fragment reads of
// both products touch every bank of shared memory once per phase under the swizzle of the row length.
template <int RB>
__device__ __forceinline__ uint32_t key_row(uint32_t m) {
    if (RB == 128) return m ^ ((m & 1u) << 2);
    if (RB == 64) return ((m ^ (m >> 2)) & 1u) | ((m >> 2) << 1) | (((m >> 1) & 1u) << 2);
    return m;
}
// Offset of byte `off` of a row in a unit's codes.
template <int RB>
__device__ __forceinline__ uint32_t code_offset(uint32_t row, uint32_t off) {
    const uint32_t x = RB == 128 ? (row & 7u) : RB == 64 ? ((row >> 1) & 3u) : ((row >> 2) & 1u);
    return row * RB + (off ^ (x << 4));
}
template <int BYTES>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t *w) {
    if (BYTES == 16) asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
    else if (BYTES == 8) asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    else if (BYTES == 4) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
    else asm volatile("{\n\t.reg .u16 h;\n\tld.shared.u16 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}" : "=r"(w[0]) : "r"(addr));
}
// The GS bf16 values of a row of scales or biases.
template <int GS>
__device__ __forceinline__ void row_f32(uint32_t addr, float (&v)[GS]) {
    uint32_t w[2];
    lds<GS * 2>(addr, w);
#pragma unroll
    for (int i = 0; i < GS; ++i) v[i] = (i & 1) ? __uint_as_float(w[i >> 1] & 0xFFFF0000u) : bf16_f32(w[i >> 1]);
}
// Codes as f16, exact.  A byte under 0x64 reads 1024 + code.  Of a word of 4-bit codes the lower nibbles of its bytes read
// 1024 + code and the upper ones, left where they are, 1024 + 16 code; the multiply-add takes out both.
constexpr uint32_t kF16One16th = 0x2C002C00u;
__device__ __forceinline__ uint32_t f16_low(uint32_t x, uint32_t minus) { return add_f16x2((x & 0x000F000Fu) | 0x64006400u, minus); }
__device__ __forceinline__ uint32_t f16_high(uint32_t x, uint32_t minus) { return fma_f16x2((x & 0x00F000F0u) | 0x64006400u, kF16One16th, minus); }
// K codes (less 2^(bits - 1)) of one k step as two A registers.
template <int BITS>
__device__ __forceinline__ void k_codes(const uint32_t *w, int step, uint32_t &lo, uint32_t &hi) {
    if (BITS == 8) {
        lo = add_f16x2(prmt(w[step], 0x64646464u, 0x4140u), 0xE480E480u);      // -(1024 + 128)
        hi = add_f16x2(prmt(w[step], 0x64646464u, 0x4342u), 0xE480E480u);
    } else {
        const uint32_t x = (step & 1) ? w[step >> 1] >> 8 : w[step >> 1];
        lo = f16_low(x, 0xE408E408u);        // -(1024 + 8)
        hi = f16_high(x, 0xD480D480u);       // -(64 + 8)
    }
}
// Element of q in a k step of the score product: what k_codes pairs with it.
template <int BITS, int PG>
__device__ __forceinline__ void q_place(uint32_t d, uint32_t &step, uint32_t &t, uint32_t &slot) {
    const uint32_t j = d / PG, in = d % PG, own = in % (PG / 4);
    t = in / (PG / 4);
    if (BITS == 8) {
        step = j * (PG / 16) + own / 4u;
        slot = own % 4u;
    } else {
        const uint32_t c = own % 8u;      // code of the word; pairs are (0,4) (1,5) | (2,6) (3,7)
        step = j * (PG / 16) + (own / 8u) * 2u + ((c & 2u) >> 1);
        slot = (c & 1u) * 2u + (c >> 2);
    }
}
// V codes c and c + 1 (less 2^(bits - 1)) of two keys' words as an A register each.
__device__ __forceinline__ void v_codes8(uint32_t w0, uint32_t w1, int c, uint32_t &first, uint32_t &second) {
    const uint32_t x = prmt(w0, w1, c == 0 ? 0x5140u : 0x7362u);
    first = add_f16x2(prmt(x, 0x64646464u, 0x4140u), 0xE480E480u);
    second = add_f16x2(prmt(x, 0x64646464u, 0x4342u), 0xE480E480u);
}
// x: half words of two keys, codes n = 0..3
__device__ __forceinline__ uint32_t v_codes4(uint32_t x, int n) {
    const uint32_t y = n >= 2 ? x >> 8 : x;
    return (n & 1) ? f16_high(y, 0xD480D480u) : f16_low(y, 0xE408E408u);      // -(64 + 8), -(1024 + 8)
}

template <int D, int BITS, int GROUP, int NT, int LIMBS>
__global__ void __launch_bounds__(kThreads, (Shape<D, BITS, GROUP, NT, LIMBS>::CTAS))
gaf_attend_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap tmap) {
    using S = Shape<D, BITS, GROUP, NT, LIMBS>;
    constexpr int R = S::R, RB = S::RB, GS = S::GS, PG = S::PG, NP = S::NP;
    constexpr bool kQReg = NT * LIMBS <= 2;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t s_full[S::STAGES], s_empty[S::STAGES];
    __shared__ uint32_t s_bad[S::STAGES];          // bit w: keys 16w.. of the unit are in no page
    __shared__ volatile uint32_t s_abort;
    __shared__ uint32_t s_scan[kThreads / 32];
    __shared__ uint32_t s_begin[3];
    __shared__ float s_f[R], s_qsum[R][NP];
    __shared__ int32_t s_seen[R];
    __shared__ float s_ml[kConsumers][R][2];
    __shared__ uint32_t s_last;
    __shared__ Item s_item;

    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *const base_ptr = smem_raw + (base - smem_u32(smem_raw));
    uint8_t *const qf_ptr = base_ptr + S::STAGES * S::STAGE;
    float *const join = reinterpret_cast<float *>(qf_ptr + S::QF);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float *const factor = join + S::JOIN / 4 + (warp < kConsumers ? warp : 0) * (R * (GS + 1)), *const limit = factor + R * GS;
    const KvView &kv = p.a.kv;

    if (threadIdx.x == 0) {
        s_abort = 0u;
        for (int s = 0; s < S::STAGES; ++s) {
            mbar_init(smem_u32(&s_full[s]), 1);
            mbar_init(smem_u32(&s_empty[s]), kConsumers);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    Range range;
    if (!cta_range<R, kKeys, kThreads>(p, s_scan, s_begin, range)) return;
    const uint64_t u0 = range.u0, u1 = range.u1, units = range.units, ctas = range.ctas;
    uint32_t head = s_begin[0], elem = s_begin[1], tile0 = s_begin[2];

    if (warp == kConsumers) {
        // ---------------- producer ----------------
        const uint32_t rows_part = kv.page_tokens < static_cast<uint32_t>(kKeys) ? kv.page_tokens : kKeys;
        const uint32_t part_shift = kv.page_shift < 6u ? kv.page_shift : 6u;
        uint32_t it = 0;
        bool ok = true;
        if (lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap)) : "memory");
        for (uint64_t u = u0; u < u1 && ok;) {
            const Item item = next_item<R, kKeys>(p, head, elem);
            const uint32_t left = item.tiles - tile0;
            const uint32_t count = u1 - u < left ? static_cast<uint32_t>(u1 - u) : left;
            const int32_t *table = p.prefix_pass ? p.a.prefix_table : p.a.seqs.table + static_cast<uint64_t>(item.seq) * p.a.seqs.table_stride;
            const uint32_t last_page = item.keys > 0 ? static_cast<uint32_t>(item.keys - 1) >> kv.page_shift : 0u;
            uint32_t page_base = (tile0 * kKeys) >> kv.page_shift;
            int32_t page_id = page_base + lane <= last_page && item.keys > 0 ? table[page_base + lane] : -1;
            for (uint32_t tile = tile0; tile < tile0 + count; ++tile, ++it) {
                const uint32_t stage = it % S::STAGES, pass = it / S::STAGES;
                const uint32_t key0 = tile * kKeys;
                const uint32_t need = static_cast<uint32_t>(item.keys) > key0 ? static_cast<uint32_t>(item.keys) - key0 : 0u;
                const uint32_t parts = ((need < static_cast<uint32_t>(kKeys) ? need : kKeys) + rows_part - 1u) >> part_shift;
                if ((key0 >> kv.page_shift) + (kKeys / 16) > page_base + 32u) {   // the ids of the unit's pages must be at hand
                    page_base = key0 >> kv.page_shift;
                    page_id = page_base + lane <= last_page ? table[page_base + lane] : -1;
                }
                if (pass > 0 && !mbar_wait(smem_u32(&s_empty[stage]), (pass - 1u) & 1u, &s_abort, p.a.error_word)) {
                    ok = false;
                    break;
                }
                // lane x < parts loads part x
                const uint32_t key = key0 + lane * rows_part;
                const int32_t id = __shfl_sync(0xFFFFFFFFu, page_id, ((key >> kv.page_shift) - page_base) & 31u);
                const bool wanted = static_cast<uint32_t>(lane) < parts;
                const bool good = wanted && id >= 0 && static_cast<uint32_t>(id) < kv.pages;
                const uint32_t good_mask = __ballot_sync(0xFFFFFFFFu, good), bad_mask = __ballot_sync(0xFFFFFFFFu, wanted && !good);
                const uint32_t bar = smem_u32(&s_full[stage]);
                if (lane == 0) {
                    uint32_t bad = 0;   // in 16-key steps
                    for (uint32_t x = 0; x < parts; ++x)
                        if ((bad_mask >> x) & 1u) bad |= ((1u << (rows_part >> 4)) - 1u) << (x * (rows_part >> 4));
                    s_bad[stage] = bad;
                    if (bad) atomicOr(p.a.error_word, kKvBadTable);
                    mbar_arrive_expect_tx(bar, __popc(good_mask) * rows_part * 2u * (RB + 2u * GS * 2u));
                }
                __syncwarp();
                if (good) {
                    const uint64_t row = ((static_cast<uint64_t>(id) * 2u * kv.kv_heads + head) << kv.page_shift) + (key & (kv.page_tokens - 1u));
                    const uint64_t vrow = row + (static_cast<uint64_t>(kv.kv_heads) << kv.page_shift);
                    const uint32_t dst = base + stage * S::STAGE, at = lane * rows_part;
                    tma_load_2d(dst + at * RB, &tmap, 0u, static_cast<uint32_t>(row), bar);
                    tma_load_2d(dst + S::CODES + at * RB, &tmap, 0u, static_cast<uint32_t>(vrow), bar);
                    const uint32_t sdst = dst + 2 * S::CODES + at * GS * 2, bytes = rows_part * GS * 2;
                    bulk_load(sdst, kv.scales + row * GS, bytes, bar);
                    bulk_load(sdst + S::SB, kv.biases + row * GS, bytes, bar);
                    bulk_load(sdst + 2 * S::SB, kv.scales + vrow * GS, bytes, bar);
                    bulk_load(sdst + 3 * S::SB, kv.biases + vrow * GS, bytes, bar);
                }
                __syncwarp();
            }
            u += count;
            tile0 = 0;
            if (++elem == p.elements) elem = 0, ++head;
        }
        if (!ok) {
            // given up: the copies in flight must land before the CTA may end
            const uint32_t first = it > static_cast<uint32_t>(S::STAGES) ? it - S::STAGES : 0u;
            for (uint32_t x = first; x < it; ++x)
                for (uint32_t tries = 0; tries < (1u << 20) && !mbar_try_wait(smem_u32(&s_full[x % S::STAGES]), (x / S::STAGES) & 1u); ++tries) {
                }
        }
        return;
    }

    // ---------------- consumers ----------------
    const uint32_t g = lane >> 2, t = lane & 3;
    const uint32_t wrow = warp * 16u;                             // this warp's first key of a unit
    constexpr int kPiece = PG / 4 * BITS / 8, vPiece = PG / 8 * BITS / 8;   // bytes of a row that a lane reads per step
    const uint32_t ra = wrow + key_row<RB>(g);                    // this lane's rows in the score product: ra, ra + 8
    // offsets in a stage; a row 8 further on lies 8 row lengths further on under every swizzle
    uint32_t k_off[NP], v_off[NP][2];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        k_off[j] = code_offset<RB>(ra, j * (PG * BITS / 8) + t * kPiece);
        v_off[j][0] = S::CODES + code_offset<RB>(wrow + key_row<RB>(2 * t), j * (PG * BITS / 8) + g * vPiece);
        v_off[j][1] = S::CODES + code_offset<RB>(wrow + key_row<RB>(2 * t + 1), j * (PG * BITS / 8) + g * vPiece);
    }
    const uint32_t s_off = 2 * S::CODES + ra * GS * 2;
    const uint32_t q_at = smem_u32(qf_ptr) + lane * 8;
    const float s_hidden = __uint_as_float(0xFF800000u);      // score of a key that a row does not see
    uint32_t it = 0;
    bool failed = false;
    // A warp's rows of q as they lie in memory.  Those of the next segment are fetched before the present one's units are worked
    // on: finding the item and waiting for its rows took a segment's start 1 to 2 us.
    constexpr int PL = D / 32, kRows = R / kConsumers, kRaw = LIMBS == 2 ? PL : PL / 2;
    uint32_t raw[kRows][kRaw];
    auto fetch_q = [&](const Item &item) {
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            const uint32_t row = item.row0 + warp + j * kConsumers;
#pragma unroll
            for (int i = 0; i < kRaw; ++i) raw[j][i] = 0u;
            if (row >= item.rows) continue;
            const uint32_t token = row / p.per_kv;
            const uint64_t at = static_cast<uint64_t>(item.token0 + token) * p.a.qs.token +
                                static_cast<uint64_t>(head * p.per_kv + row - token * p.per_kv) * p.a.qs.head + lane * PL;
            if (LIMBS == 2) {
                const uint32_t *src = static_cast<const uint32_t *>(p.a.q) + at;
#pragma unroll
                for (int i = 0; i < kRaw; ++i) raw[j][i] = src[i];
            } else {
                const uint16_t *src = static_cast<const uint16_t *>(p.a.q) + at;
                if (p.q_vec && kRaw == 2) {
                    const uint2 y = *reinterpret_cast<const uint2 *>(src);
                    raw[j][0] = y.x, raw[j][kRaw - 1] = y.y;
                } else if (p.q_vec) {
                    raw[j][0] = *reinterpret_cast<const uint32_t *>(src);
                } else {
#pragma unroll
                    for (int i = 0; i < kRaw; ++i) raw[j][i] = src[2 * i] | (static_cast<uint32_t>(src[2 * i + 1]) << 16);
                }
            }
        }
    };
    {
        const Item first = next_item<R, kKeys>(p, head, elem);
        if (threadIdx.x == 0) s_item = first;
        fetch_q(first);
        bar_consumers();
    }
    for (uint64_t u = u0; u < u1;) {
        const Item item = s_item;
        const uint32_t left = item.tiles - tile0;
        const uint32_t count = u1 - u < left ? static_cast<uint32_t>(u1 - u) : left;

        // ---- q of the tile's rows: scaled by a power of two, f16, as B fragments; sums per step; scale of the scores ----
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
            const int r = warp + j * kConsumers;
            const uint32_t row = item.row0 + r;
            const bool have = row < item.rows;
            float x[PL];
#pragma unroll
            for (int i = 0; i < PL; ++i)
                x[i] = LIMBS == 2 ? __uint_as_float(raw[j][LIMBS == 2 ? i : 0])
                                  : (i & 1) ? __uint_as_float(raw[j][LIMBS == 2 ? 0 : i / 2] & 0xFFFF0000u) : bf16_f32(raw[j][LIMBS == 2 ? 0 : i / 2]);
            uint32_t top = 0u;                                   // bits of the largest magnitude; NaN is above infinity
#pragma unroll
            for (int i = 0; i < PL; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
            // which of the two is a matter of the code around them: 4 bits, 12 sequences of 32771 tokens, 64 heads on 8: 113 us by shuffles, 118
            // by the other; 8 bits, 64 sequences of 2048 to 4096: 88.7 and 87.4, 16 of 2500 in f32: 30.1 and 29.3
            if (BITS == 8) {
                top = __reduce_max_sync(0xFFFFFFFFu, top);
            } else {
#pragma unroll
                for (int o = 16; o >= 1; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            }
            int e = static_cast<int>(top >> 23) - 127;           // 2^e <= top < 2^(e + 1)
            e = e < -100 ? -100 : e > 127 ? 127 : e;
            const float mul = __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < PL; ++i) {
                const uint32_t d = lane * PL + i;
                uint32_t step, tt, slot;
                q_place<BITS, PG>(d, step, tt, slot);
                float rest = x[i] * mul;
#pragma unroll
                for (int l = 0; l < LIMBS; ++l) {
                    const __half h = __float2half_rn(rest);
                    const float back = __half2float(h);
                    rest -= back;
                    sum += back;
                    const uint32_t at = (((l * NT + r / 8) * S::KS + step) * 32 + (r % 8) * 4 + tt) * 4 + slot;
                    reinterpret_cast<__half *>(qf_ptr)[at] = h;
                }
            }
#pragma unroll
            for (int o = 1; o < 32 / NP; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            if (lane % (32 / NP) == 0) s_qsum[r][lane / (32 / NP)] = sum;
            if (lane == 0) {
                // a row that is not finite gives NaN wherever it sees a key (its scores may all be -inf)
                s_f[r] = top < 0x7F800000u ? __uint_as_float(static_cast<uint32_t>(127 - 13 + e) << 23) * (p.a.scale * 1.4426950408889634f) : __uint_as_float(0x7FC00000u);
                const int32_t seen = p.prefix_pass ? item.seen0 : item.seen0 + static_cast<int32_t>(row / p.per_kv);
                s_seen[r] = have ? (seen < item.keys ? seen : item.keys) : 0;
            }
        }
        bar_consumers();
        // where this segment lies is kept, and the next one's rows are sent for
        const uint32_t this_head = head;
        if (u + count < u1) {
            if (++elem == p.elements) elem = 0, ++head;
            const Item next = next_item<R, kKeys>(p, head, elem);
            if (threadIdx.x == 0) s_item = next;       // read again behind the barriers of the segment's end
            fetch_q(next);
        }
        uint32_t qreg[kQReg ? LIMBS : 1][kQReg ? NT : 1][kQReg ? S::KS : 1][2];
        if (kQReg) {
#pragma unroll
            for (int l = 0; l < LIMBS; ++l)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < S::KS; ++k)
                        lds<8>(smem_u32(qf_ptr) + (((l * NT + nt) * S::KS + k) * 32 + lane) * 8, qreg[kQReg ? l : 0][kQReg ? nt : 0][kQReg ? k : 0]);
        }
        float f[NT][2], qsum[NT][2][NP];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                f[nt][c] = s_f[nt * 8 + 2 * t + c];
#pragma unroll
                for (int j = 0; j < NP; ++j) qsum[nt][c][j] = s_qsum[nt * 8 + 2 * t + c][j];
            }
        for (int x = lane; x < R * GS; x += 32) factor[x] = 0.0f;     // until the first unit: the largest products
        __syncwarp();
        float most_scale[GS];    // a power of two above the warp's scales of the segment so far; 0: none
#pragma unroll
        for (int i = 0; i < GS; ++i) most_scale[i] = 0.0f;
        float m[NT][2], l[NT][2], bsum[NT][2][GS], o[S::KS][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m[nt][c] = kNoMax;
                l[nt][c] = 0.0f;
#pragma unroll
                for (int i = 0; i < GS; ++i) bsum[nt][c][i] = 0.0f;
            }
#pragma unroll
        for (int i = 0; i < S::KS; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[i][nt][c] = 0.0f;

        bool fresh = true;       // this warp has summed no unit of the segment
        // One unit.  kBorder: some row of the tile does not see all its keys, or some of its keys are in no page.
        auto unit = [&](auto border_tag, uint32_t kc, int32_t key0, uint32_t bad) {
            constexpr bool kBorder = decltype(border_tag)::value;
            // ---- scores, transposed: [16 keys][8 NT rows] ----
            float s[NT][4];
            {
                float sa[GS], sb[GS], ba[GS], bb[GS];
                const uint32_t at = kc + s_off;
                row_f32<GS>(at, sa);
                row_f32<GS>(at + 8 * GS * 2, sb);
                row_f32<GS>(at + S::SB, ba);
                row_f32<GS>(at + S::SB + 8 * GS * 2, bb);
#pragma unroll
                for (int i = 0; i < GS; ++i) {
                    ba[i] = fmaf(static_cast<float>(1 << (BITS - 1)), sa[i], ba[i]);
                    bb[i] = fmaf(static_cast<float>(1 << (BITS - 1)), sb[i], bb[i]);
                }
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    constexpr int kWords = kPiece >= 4 ? kPiece / 4 : 1;
                    uint32_t wa[kWords], wb[kWords];
                    lds<kPiece>(kc + k_off[j], wa);
                    lds<kPiece>(kc + k_off[j] + 8 * RB, wb);
                    float acc[NT][4];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.0f;
#pragma unroll
                    for (int k = 0; k < PG / 16; ++k) {
                        uint32_t a[4];
                        k_codes<BITS>(wa, k, a[0], a[2]);
                        k_codes<BITS>(wb, k, a[1], a[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int lb = 0; lb < LIMBS; ++lb) {
                                if (kQReg) {
                                    const uint32_t *q = qreg[kQReg ? lb : 0][kQReg ? nt : 0][kQReg ? j * (PG / 16) + k : 0];
                                    mma_f16(acc[nt], a, q[0], q[1]);
                                } else {
                                    uint32_t q[2];
                                    lds<8>(q_at + ((lb * NT + nt) * S::KS + j * (PG / 16) + k) * 256, q);
                                    mma_f16(acc[nt], a, q[0], q[1]);
                                }
                            }
                    }
                    constexpr int kPer = GROUP / PG;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            s[nt][c] = j == 0 ? sa[0] * acc[nt][c] : fmaf(sa[j / kPer], acc[nt][c], s[nt][c]);
                            s[nt][2 + c] = j == 0 ? sb[0] * acc[nt][2 + c] : fmaf(sb[j / kPer], acc[nt][2 + c], s[nt][2 + c]);
                            s[nt][c] = fmaf(ba[j / kPer], qsum[nt][c][j], s[nt][c]);
                            s[nt][2 + c] = fmaf(bb[j / kPer], qsum[nt][c][j], s[nt][2 + c]);
                        }
                }
                if (kBorder) {
                    const int32_t pa = key0 + static_cast<int32_t>(ra), pb = pa + 8;
                    const bool gone = (bad >> warp) & 1u;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int32_t seen = gone ? 0 : s_seen[nt * 8 + 2 * t + c];
                            if (pa >= seen) s[nt][c] = s_hidden;
                            if (pb >= seen) s[nt][2 + c] = s_hidden;
                        }
                }
            }
            // ---- weights: against the row's reference and the groups' factors; both follow lazily ----
            float va[GS], vb[GS];     // scales of the values
            row_f32<GS>(kc + s_off + 2 * S::SB, va);
            row_f32<GS>(kc + s_off + 2 * S::SB + 8 * GS * 2, vb);
            bool grow = false;
#pragma unroll
            for (int i = 0; i < GS; ++i) grow |= fmaxf(fabsf(va[i]), fabsf(vb[i])) >= most_scale[i];
            float z[NT][4];
            auto weigh = [&]() {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        z[nt][c] = kBorder && s[nt][c] == s_hidden ? -INFINITY : fmaf(s[nt][c], f[nt][c & 1], -m[nt][c & 1]);
            };
            weigh();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float2 most = *reinterpret_cast<const float2 *>(limit + nt * 8 + 2 * t);
#pragma unroll
                for (int c = 0; c < 4; ++c) grow |= z[nt][c] > ((c & 1) ? most.y : most.x);
            }
            if (fresh || __any_sync(0xFFFFFFFFu, grow)) {
                // the largest finite scales of the warp's keys so far, rounded up to a power of two
#pragma unroll
                for (int i = 0; i < GS; ++i) {
                    const uint32_t x = __float_as_uint(va[i]) & 0x7FFFFFFFu, y = __float_as_uint(vb[i]) & 0x7FFFFFFFu;
                    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, max(x < 0x7F800000u ? x : 0u, y < 0x7F800000u ? y : 0u));
                    most_scale[i] = fmaxf(most_scale[i], __uint_as_float((top & 0x7F800000u) + 0x00800000u));
                }
                // 2^(kTarget - floor(log2 most)), at most 2^126
                auto fitting = [](float most) { return min(((254u + kTarget) << 23) - (__float_as_uint(most) & 0x7F800000u), 253u << 23); };
                // scores above the reference by that, and no more, keep all products in range; reach: a group's factor times its largest scale
                auto room = [](float reach) { return fminf(kLazy, static_cast<float>(kMostExp + 127 - static_cast<int>(__float_as_uint(reach) >> 23))); };
                // kFirst: nothing is summed yet.  Code that runs once a segment comes from far, so there is no more of it than needed: the
                // groups' largest products by atomics in the array of the factors, instead of 6 instructions for each in every lane (a
                // shared prefix of 1111 tokens for five sequences: 37.5 us, 38.9 with those)
                auto settle = [&](auto first_tag) {
                    constexpr bool kFirst = decltype(first_tag)::value;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        // the rows' largest scores, not their distance from the present reference, which may be none
                        float y[4], top[2], most[2][GS], up[2];
#pragma unroll
                        for (int c = 0; c < 4; ++c) y[c] = kBorder && s[nt][c] == s_hidden ? -INFINITY : s[nt][c] * f[nt][c & 1];
#pragma unroll
                        for (int c = 0; c < 2; ++c) top[c] = fmaxf(y[c], y[2 + c]);
#pragma unroll
                        for (int x = 4; x <= 16; x <<= 1)
#pragma unroll
                            for (int c = 0; c < 2; ++c) top[c] = fmaxf(top[c], __shfl_xor_sync(0xFFFFFFFFu, top[c], x));
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float next = fmaxf(m[nt][c], ceilf(top[c]));
                            up[c] = fminf(next - m[nt][c], 1000.0f);
                            m[nt][c] = next;
                            // the groups' largest products; a scale that is not finite counts for nothing or for the most
                            const float pa = exp2_approx(y[c] - next), pb = exp2_approx(y[2 + c] - next);
#pragma unroll
                            for (int i = 0; i < GS; ++i) {
                                most[c][i] = fmaxf(fmaxf(pa * fabsf(va[i]), pb * fabsf(vb[i])), 0.0f);
                                if (kFirst) atomicMax(reinterpret_cast<unsigned int *>(factor + i * R + nt * 8 + 2 * t + c), __float_as_uint(most[c][i]));
                            }
                        }
                        if (kFirst) continue;
#pragma unroll
                        for (int x = 4; x <= 16; x <<= 1)
#pragma unroll
                            for (int c = 0; c < 2 * GS; ++c) most[c / GS][c % GS] = fmaxf(most[c / GS][c % GS], __shfl_xor_sync(0xFFFFFFFFu, most[c / GS][c % GS], x));
                        float reach[2] = {0.0f, 0.0f};       // product of a group's factor and largest scale
#pragma unroll
                        for (int i = 0; i < GS; ++i) {
                            float *const at = factor + i * R + nt * 8 + 2 * t;
                            float set[2];
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const uint32_t fit = fitting(most[c][i]);
                                // the sums' present unit is 2^-have; it is kept while the products stay below 2^(kTarget + 8)
                                const int have = static_cast<int>(__float_as_uint(at[c]) >> 23) - 127 + static_cast<int>(up[c]), aim = static_cast<int>(fit >> 23) - 127;
                                const int want = have >= aim + 8 ? aim : min(have, 126);
                                const float ratio = pow2_or_0(want - have);
                                set[c] = pow2_or_0(want);
#pragma unroll
                                for (int k = i * (GROUP / 16); k < (i + 1) * (GROUP / 16); ++k) o[k][nt][c] *= ratio, o[k][nt][2 + c] *= ratio;
                                reach[c] = fmaxf(reach[c], set[c] * most_scale[i]);
                            }
                            __syncwarp();       // the row's lanes have read it
                            if (g == 0) *reinterpret_cast<float2 *>(at) = make_float2(set[0], set[1]);
                        }
                        if (g == 0) *reinterpret_cast<float2 *>(limit + nt * 8 + 2 * t) = make_float2(room(reach[0]), room(reach[1]));
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float keep = pow2_or_0(-static_cast<int>(up[c]));
                            l[nt][c] *= keep;
#pragma unroll
                            for (int i = 0; i < GS; ++i) bsum[nt][c][i] *= keep;
                        }
                    }
                    if (kFirst) {
                        // the array held the largest products: a lane for each
                        __syncwarp();
                        for (int x = lane; x < R * GS; x += 32) factor[x] = __uint_as_float(fitting(factor[x]));
                        __syncwarp();
                        if (lane < R) {
                            float reach = 0.0f;
#pragma unroll
                            for (int i = 0; i < GS; ++i) reach = fmaxf(reach, factor[i * R + lane] * most_scale[i]);
                            limit[lane] = room(reach);
                        }
                    }
                };
                if (fresh) settle(std::true_type());
                else settle(std::false_type());
                __syncwarp();
                weigh();
            }
            fresh = false;
            {
                // ---- weights times scales as B fragments, weights times biases ----
                uint32_t pf[LIMBS][GS][NT][2];
                float ba[GS], bb[GS];
                const uint32_t at = kc + s_off + 3 * S::SB;
                row_f32<GS>(at, ba);
                row_f32<GS>(at + 8 * GS * 2, bb);
#pragma unroll
                for (int i = 0; i < GS; ++i) {
                    ba[i] = fmaf(static_cast<float>(1 << (BITS - 1)), va[i], ba[i]);
                    bb[i] = fmaf(static_cast<float>(1 << (BITS - 1)), vb[i], bb[i]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float pr[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) pr[c] = exp2_approx(z[nt][c]);
                    l[nt][0] += pr[0] + pr[2];
                    l[nt][1] += pr[1] + pr[3];
#pragma unroll
                    for (int i = 0; i < GS; ++i) {
                        const float2 gr = *reinterpret_cast<const float2 *>(factor + i * R + nt * 8 + 2 * t);
                        const float2 xa = mul_pair(mul_pair(make_float2(pr[0], pr[1]), make_float2(va[i], va[i])), gr);
                        const float2 xb = mul_pair(mul_pair(make_float2(pr[2], pr[3]), make_float2(vb[i], vb[i])), gr);
                        float x[4] = {xa.x, xa.y, xb.x, xb.y};
                        if (kBorder) {   // rows behind the end may hold anything, NaN too
                            float y[4] = {pr[0] * ba[i], pr[1] * ba[i], pr[2] * bb[i], pr[3] * bb[i]};
#pragma unroll
                            for (int c = 0; c < 4; ++c)
                                if (z[nt][c] == -INFINITY) x[c] = 0.0f, y[c] = 0.0f;
                            bsum[nt][0][i] += y[0] + y[2];
                            bsum[nt][1][i] += y[1] + y[3];
                        } else {
                            bsum[nt][0][i] = fmaf(pr[0], ba[i], fmaf(pr[2], bb[i], bsum[nt][0][i]));
                            bsum[nt][1][i] = fmaf(pr[1], ba[i], fmaf(pr[3], bb[i], bsum[nt][1][i]));
                        }
#pragma unroll
                        for (int lb = 0; lb < LIMBS; ++lb) {
                            const uint32_t w0 = pack_f16x2(x[0], x[1]), w1 = pack_f16x2(x[2], x[3]);
                            pf[lb][i][nt][0] = transpose8x8(w0);
                            pf[lb][i][nt][1] = transpose8x8(w1);
                            if (lb + 1 < LIMBS) {
                                const float2 y0 = __half22float2(*reinterpret_cast<const __half2 *>(&w0)), y1 = __half22float2(*reinterpret_cast<const __half2 *>(&w1));
                                x[0] -= y0.x, x[1] -= y0.y, x[2] -= y1.x, x[3] -= y1.y;
                            }
                        }
                    }
                }
                // ---- weighted sums, transposed: [D][8 NT rows] ----
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    constexpr int kWords = vPiece >= 4 ? vPiece / 4 : 1;
                    uint32_t w[4][kWords];
                    lds<vPiece>(kc + v_off[j][0], w[0]);
                    lds<vPiece>(kc + v_off[j][1], w[1]);
                    lds<vPiece>(kc + v_off[j][0] + 8 * RB, w[2]);
                    lds<vPiece>(kc + v_off[j][1] + 8 * RB, w[3]);
#pragma unroll
                    for (int i = 0; i < PG / 16; ++i) {
                        uint32_t a[4];
                        if (BITS == 8) {
                            v_codes8(w[0][i >> 1], w[1][i >> 1], 2 * (i & 1), a[0], a[1]);
                            v_codes8(w[2][i >> 1], w[3][i >> 1], 2 * (i & 1), a[2], a[3]);
                        } else {
                            const uint32_t x = prmt(w[0][0], w[1][0], i < 2 ? 0x5410u : 0x7632u);
                            const uint32_t y = prmt(w[2][0], w[3][0], i < 2 ? 0x5410u : 0x7632u);
                            a[0] = v_codes4(x, 2 * (i & 1));
                            a[1] = v_codes4(x, 2 * (i & 1) + 1);
                            a[2] = v_codes4(y, 2 * (i & 1));
                            a[3] = v_codes4(y, 2 * (i & 1) + 1);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int lb = 0; lb < LIMBS; ++lb)
                                mma_f16(o[j * (PG / 16) + i][nt], a, pf[lb][j * PG / GROUP][nt][0], pf[lb][j * PG / GROUP][nt][1]);
                    }
                }
            }
        };
        for (uint32_t tile = tile0; tile < tile0 + count; ++tile, ++it) {
            const uint32_t stage = it % S::STAGES;
            if (!mbar_wait(smem_u32(&s_full[stage]), (it / S::STAGES) & 1u, &s_abort, p.a.error_word)) failed = true;
            const int32_t key0 = static_cast<int32_t>(tile * kKeys);
            const uint32_t bad = s_bad[stage];
            if (key0 + kKeys <= item.first_seen && bad == 0u) unit(std::false_type(), base + stage * S::STAGE, key0, 0u);
            else if (key0 + static_cast<int32_t>(wrow) < item.keys) unit(std::true_type(), base + stage * S::STAGE, key0, bad);
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s_empty[stage]));
        }

        // ---- end of the segment: the four warps' sums joined ----
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int x = 4; x <= 16; x <<= 1) {
                    l[nt][c] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][c], x);
#pragma unroll
                    for (int i = 0; i < GS; ++i) bsum[nt][c][i] += __shfl_xor_sync(0xFFFFFFFFu, bsum[nt][c][i], x);
                }
                if (g == 0) s_ml[warp][nt * 8 + 2 * t + c][0] = m[nt][c], s_ml[warp][nt * 8 + 2 * t + c][1] = l[nt][c];
            }
        if (bar_consumers_or(failed)) return;   // a wait ran out: all four leave here
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int r = nt * 8 + 2 * t + c;
                float top = s_ml[0][r][0];
#pragma unroll
                for (int w = 1; w < kConsumers; ++w) top = fmaxf(top, s_ml[w][r][0]);
                const float keep = m[nt][c] == top ? 1.0f : exp2_approx(m[nt][c] - top);
                float unit_of[GS];       // 1 / factor
#pragma unroll
                for (int i = 0; i < GS; ++i) unit_of[i] = __uint_as_float((254u << 23) - __float_as_uint(factor[i * R + r]));
#pragma unroll
                for (int i = 0; i < S::KS; ++i) {
                    const int gi = i * 16 / GROUP;
                    o[i][nt][c] = fmaf(o[i][nt][c], unit_of[gi], bsum[nt][c][gi]) * keep;
                    o[i][nt][2 + c] = fmaf(o[i][nt][2 + c], unit_of[gi], bsum[nt][c][gi]) * keep;
                }
            }
        const bool whole = tile0 == 0u && count == item.tiles;
        const uint32_t slot = 2u * blockIdx.x + (tile0 == 0u ? 1u : 0u);
        float *const part = p.partials + static_cast<uint64_t>(slot) * (R * (D + 2));
        auto row_sum = [&](int r, float &top, float &sum) {   // maximum and sum of a row over the warps
            top = s_ml[0][r][0];
#pragma unroll
            for (int w = 1; w < kConsumers; ++w) top = fmaxf(top, s_ml[w][r][0]);
            sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) sum += s_ml[w][r][1] * (s_ml[w][r][0] == top ? 1.0f : exp2_approx(s_ml[w][r][0] - top));
        };
        constexpr int kWide = D / S::HALVES;
#pragma unroll
        for (int half = 0; half < S::HALVES; ++half) {
            if (half) bar_consumers();
#pragma unroll
            for (int i = 0; i < S::KS / S::HALVES; ++i) {
                const int ii = half * (S::KS / S::HALVES) + i;
                const int d = ii / (PG / 16) * PG + (PG / 8) * g + 2 * (ii % (PG / 16)) - half * kWide;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        *reinterpret_cast<float2 *>(join + (warp * R + nt * 8 + 2 * t + c) * S::OW + d) = make_float2(o[ii][nt][c], o[ii][nt][2 + c]);
            }
            bar_consumers();
            for (int x = threadIdx.x; x < R * (kWide / 4); x += kConsumers * 32) {
                const int r = x / (kWide / 4), d = (x % (kWide / 4)) * 4;
                if (item.row0 + r >= item.rows) continue;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kConsumers; ++w) {
                    const float4 y = *reinterpret_cast<const float4 *>(join + (w * R + r) * S::OW + d);
                    v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
                }
                float top, sum;
                row_sum(r, top, sum);
                if (whole) {
                    finish_row<D, LIMBS == 2>(p, item, this_head, r, half * kWide + d, top, sum, v);
                } else {
                    __stcg(reinterpret_cast<float4 *>(part + r * D + half * kWide + d), v);
                    if (half == 0 && d == 0) {
                        __stcg(part + R * D + 2 * r, top);
                        __stcg(part + R * D + 2 * r + 1, sum);
                    }
                }
            }
        }
        if (!whole) {
            // the item's CTAs: the first holds its unit 0
            const uint64_t first_unit = u - tile0;
            const uint32_t c0 = static_cast<uint32_t>(quotient((first_unit + 1) * ctas - 1, units));
            const uint32_t c1 = static_cast<uint32_t>(quotient((first_unit + item.tiles) * ctas - 1, units));
            bar_consumers();
            if (threadIdx.x == 0) {
                __threadfence();      // for the whole CTA, whose writes the barrier puts before it
                const uint32_t seen = atomicAdd(p.tickets + c0, 1u);
                s_last = seen == c1 - c0;
                if (s_last) p.tickets[c0] = 0u;
            }
            bar_consumers();
            if (s_last) {
                __threadfence();
                auto part_of = [&](uint32_t c) { return p.partials + static_cast<uint64_t>(2u * c + (c == c0 ? 1u : 0u)) * (R * (D + 2)); };
                for (int x = threadIdx.x; x < R * (D / 4); x += kConsumers * 32) {
                    const int r = x / (D / 4), d = (x % (D / 4)) * 4;
                    if (item.row0 + r >= item.rows) continue;
                    float top = -INFINITY, sum = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (uint32_t c = c0; c <= c1; ++c) {
                        const float *src = part_of(c);
                        const float mc = __ldcg(src + R * D + 2 * r), lc = __ldcg(src + R * D + 2 * r + 1);
                        const float4 y = __ldcg(reinterpret_cast<const float4 *>(src + r * D + d));
                        const float both = fmaxf(top, mc);
                        const float wa = top == both ? 1.0f : exp2_approx(top - both), wb = mc == both ? 1.0f : exp2_approx(mc - both);
                        top = both;
                        sum = fmaf(sum, wa, lc * wb);
                        v = make_float4(fmaf(v.x, wa, y.x * wb), fmaf(v.y, wa, y.y * wb), fmaf(v.z, wa, y.z * wb), fmaf(v.w, wa, y.w * wb));
                    }
                    finish_row<D, LIMBS == 2>(p, item, this_head, r, d, top, sum, v);
                }
            }
        }
        bar_consumers();   // s_ml, the joined rows and q are free again
        u += count;
        tile0 = 0;
    }
}

// Something that is done once for each device (a kernel's shared-memory opt-in), from any host thread.
struct DeviceOnce {
    std::atomic<uint64_t> done{0};
    template <class F>
    cudaError_t run(F &&f) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0u;
        if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
        e = f();
        if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
        return e;
    }
};

template <int D, int BITS, int GROUP, int NT, int LIMBS>
cudaError_t launch(const Params &p, const CUtensorMap &tmap, int sm_count, cudaStream_t stream) {
    using S = Shape<D, BITS, GROUP, NT, LIMBS>;
    auto kernel = gaf_attend_kernel<D, BITS, GROUP, NT, LIMBS>;
    static DeviceOnce once;    // of this instance
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM); });
    if (e != cudaSuccess) return e;
    kernel<<<sm_count * S::CTAS, kThreads, S::SMEM, stream>>>(p, tmap);
    return cudaGetLastError();
}

// `nt`: 1 to 4 row tiles of 8 (4 for heads of 64 only; limbs = 2: 1 or 2)
cudaError_t launch_d64_b4(const Params &p, const CUtensorMap &tmap, int nt, int limbs, int sm_count, cudaStream_t stream);
cudaError_t launch_d64_b8(const Params &p, const CUtensorMap &tmap, int nt, int limbs, int sm_count, cudaStream_t stream);
cudaError_t launch_d128_b4(const Params &p, const CUtensorMap &tmap, int nt, int limbs, int sm_count, cudaStream_t stream);
cudaError_t launch_d128_b8(const Params &p, const CUtensorMap &tmap, int nt, int limbs, int sm_count, cudaStream_t stream);

template <int D, int BITS, int GROUP>
cudaError_t launch_rows(const Params &p, const CUtensorMap &tmap, int nt, int limbs, int sm_count, cudaStream_t stream) {
    if (limbs == 2) return nt == 1 ? launch<D, BITS, GROUP, 1, 2>(p, tmap, sm_count, stream) : launch<D, BITS, GROUP, 2, 2>(p, tmap, sm_count, stream);
    if (nt == 1) return launch<D, BITS, GROUP, 1, 1>(p, tmap, sm_count, stream);
    if (nt == 2) return launch<D, BITS, GROUP, 2, 1>(p, tmap, sm_count, stream);
    if constexpr (D == 64)
        if (nt == 4) return launch<D, BITS, GROUP, 4, 1>(p, tmap, sm_count, stream);
    return launch<D, BITS, GROUP, 3, 1>(p, tmap, sm_count, stream);
}

// tcgen05, bf16 rows (gaf_attend_wide.cuh): 256 rows a tile
cudaError_t launch_wide(const Params &p, const CUtensorMap &tmap, int sm_count, cudaStream_t stream);

constexpr int kMaxCtas = 4;             // per SM, of any instance (even: what follows the tickets is 8-byte aligned)
constexpr int kMaxPartRows = 256 * 2;   // rows of the partial results of an SM's CTAs (3 CTAs x 2 slots x 32 rows; 1 x 2 x 256)
constexpr int kMaxDim = 128;

}  // namespace attend
}  // namespace tgaf
