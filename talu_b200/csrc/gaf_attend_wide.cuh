// Attention over the quantised KV cache on tcgen05, for many query rows per cached head (prompts, shared prefixes).
//
// Mathematics.  Keys and values are dequantised to f16, 32 keys at a time with one power of two that brings their largest
// magnitude to 2^14..2^15.  bf16 would hold any range as it is, but its 8 bits on keys and values alone put the result 3e-3
// off; f16 rounds the centre of a group and the element itself, 2^-11 of each (an element that is small beside its group's centre is
// off by 2^-11 of the centre), and loses what is below 2^-39 of the largest magnitude.
//   w 2^-e = (c - h) (s 2^-e) + (b + h s) 2^-e,   h = 2^(bits - 1): the centred code and s 2^-e are exact in f16
// q is f16 with a power of two per row (exact), the weights are f16 (2^-11 of each), all statistics and sums f32.  Scores thus carry
// 2^-11 of each key element, which those of the register path do not.  The keys'
// power goes into the scores' factor, the values' into the weights: they are formed as 2^(y + e - m) (y: scores in base
// 2), where m follows the largest y + e instead of the largest y, and leave it again in the row's sum.
//
// One CTA per SM, 256 query rows (two MMA tiles of 128) against units of 128 keys:
//   warps 0-3, 4-7   softmax of tile 0 and 1, one row per thread: scores from tensor memory, weights (f16) back into the
//                    scores' columns, where the second product takes them as its A operand
//   warps 8-11       dequantise, one cached row per thread; K (K-major) and V (N-major) tiles have the same image
//   warp 12          issues the MMAs: per unit S_t = Q_t K^T and O_t += P_t V for both tiles; while one tile's softmax
//                    runs, the tensor core works for the other
//   warp 13          TMA of codes, bulk copies of scales and biases
// K and V tiles share a ring of three 32 KB buffers, their codes one of three stages: K(i), V(i), K(i+1), ...
//
// The reference is an integer and follows lazily: a row's largest weight is brought to 2^6 to 2^7 and rescaled (O, and the weights of
// the unit that are formed already: exactly) when it exceeds 2^15, so that weights keep their 11 bits down to 2^-20 of the largest and
// have a step of 2^-30 of it below.  (With 2^0 in place of 2^7, 40000 keys of 2^-22 each behind one key whose values are zero were
// 15 % off; 2^10 costs 4 %, 2^12 11 % more time.)  A row's thread takes 32 scores at a time
// and puts their weights into columns whose scores it has read.  Measured on a chunk of two prompts (768 and
// 1024 new tokens over 3750 and 5000 cached ones, 32 heads on 8): 216 us; 262 with a pass of its own for the maximum,
// 256 with that and two threads a row, 334 with two buffers of 64 keys for the scores (twice the MMAs, of half the
// width: the issuing warp does not keep up), 387 with everything unrolled (instruction cache).
// What bounds it: 2 x 128 x 128 exponentials per unit (16 per clock and SM) and as many clocks of tensor work; what keeps it
// from there is the way of one tile's unit through scores, softmax, weights and second product, which the other tile
// covers only in part.
#pragma once
#include "gaf_attend.cuh"

namespace tgaf {
namespace attend {

constexpr int kWideKeys = 128;
constexpr int kWideRows = 256;
constexpr int kWideThreads = 14 * 32;    // 128 registers each
constexpr int kDequantWarp0 = 8, kDequantWarps = 4, kMmaWarp = 12, kLoadWarp = 13;
constexpr int kInfo = 4;             // units whose side information is kept
constexpr float kWideTarget = 7.0f;  // a row's largest weight is brought to 2^6 to 2^7
constexpr float kWideMost = 15.0f;   // ... when it exceeds 2^15 (f16)
constexpr float kMinFactor = 1.0e-37f;   // of raw scores: not 0, since hidden ones are -inf
constexpr int kMinExp = -90;         // values below 2^-76 lose bits instead of pushing the sums of weights, 2^(15 + 90) a key, out of f32

__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(lbo >> 4) << 16;
    d |= static_cast<uint64_t>(sbo >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t pred;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xFFFFFFFF;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(pred));
    return pred != 0u;
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }   // -126 <= e <= 127

// Place of value d of a row in the tiles: 4-bit codes leave their words in the order 0 4 1 5 2 6 3 7, and the tiles keep it (in
// K and q alike, and in the columns of O).
template <int BITS>
__device__ __forceinline__ constexpr int value_at(int place) {   // value that stands at a place of its eight
    return BITS == 8 ? place : ((place & 1) * 4 + (place >> 1));
}

template <int D, int BITS, int GROUP>
struct Wide {
    static constexpr int RB = D * BITS / 8;
    static constexpr int GS = D / GROUP;
    static constexpr int PANELS = D / 64;                       // of 64 values: 128 bytes of f16
    static constexpr int PANEL = kWideKeys * 128;
    static constexpr int TILE = PANELS * PANEL;                 // a dequantised tile, or 128 rows of q
    static constexpr int TILES = 3;
    static constexpr int CODES = kWideKeys * RB;
    static constexpr int SB = kWideKeys * GS * 2;
    static constexpr int STAGE = CODES + (2 * SB + 1023) / 1024 * 1024;
    static constexpr int STAGES = 3;
    static constexpr int SMEM = 2 * TILE + TILES * TILE + STAGES * STAGE + 1024;
    static constexpr int PART = kWideRows * (D + 2);            // floats of a partial result
};

template <int D, int BITS, int GROUP>
__global__ void __launch_bounds__(kWideThreads, 1)
gaf_attend_wide_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap tmap) {
    using W = Wide<D, BITS, GROUP>;
    constexpr int RB = W::RB, GS = W::GS;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t s_code_full[W::STAGES], s_code_empty[W::STAGES];
    __shared__ __align__(8) uint64_t s_tile_full[W::TILES], s_tile_empty[W::TILES];
    __shared__ __align__(8) uint64_t s_q_ready[2], s_score[2], s_weights[2], s_done[2], s_idle;
    __shared__ uint32_t s_bad[W::STAGES];           // bit x: keys 16x.. of the unit are in no page
    // by unit and 32 keys: factor of the keys' scores, exponent of the values, 2^-exponent, groups of values that are not finite
    __shared__ float s_kmul[kInfo][4], s_vexp[kInfo][4], s_vinv[kInfo][4];
    __shared__ uint32_t s_kbad[kInfo];
    __shared__ __align__(16) uint32_t s_lost[kInfo][4];
    __shared__ uint8_t s_poison[kInfo][kWideKeys];  // by key
    __shared__ uint32_t s_tmem;
    __shared__ volatile uint32_t s_abort;
    __shared__ uint32_t s_scan[kWideThreads / 32];
    __shared__ uint32_t s_begin[3];

    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_base = base, tile_base = q_base + 2 * W::TILE, code_base = tile_base + W::TILES * W::TILE;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const KvView &kv = p.a.kv;

    if (threadIdx.x == 0) {
        s_abort = 0u;
        for (int i = 0; i < W::STAGES; ++i) {
            mbar_init(smem_u32(&s_code_full[i]), 1);
            mbar_init(smem_u32(&s_code_empty[i]), kDequantWarps);
        }
        for (int i = 0; i < W::TILES; ++i) {
            mbar_init(smem_u32(&s_tile_full[i]), kDequantWarps);
            mbar_init(smem_u32(&s_tile_empty[i]), 1);
        }
        mbar_init(smem_u32(&s_idle), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s_q_ready[i]), 128);
            mbar_init(smem_u32(&s_score[i]), 1);
            mbar_init(smem_u32(&s_weights[i]), 128);
            mbar_init(smem_u32(&s_done[i]), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    Range range;
    if (!cta_range<kWideRows, kWideKeys, kWideThreads>(p, s_scan, s_begin, range)) {
        if (threadIdx.x == 0) p.cuts[blockIdx.x].parts = 0u;
        return;
    }
    if (threadIdx.x == 0) p.cuts[blockIdx.x].parts = 0u;     // until a segment says otherwise
    const uint64_t u0 = range.u0, u1 = range.u1;
    uint32_t head = s_begin[0], elem = s_begin[1], tile0 = s_begin[2];
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = s_tmem;
    // scores of tile t: columns 128 t ..; sums: 256 + 128 t ..

    // Every wait is bounded.  After one has run out all waits return at once: the roles run their loops to the end without
    // data, so that they still meet at their barriers and leave together.
    bool ok = true;
    auto wait = [&](uint64_t &bar, uint32_t parity) {
        if (ok) ok = mbar_wait(smem_u32(&bar), parity, &s_abort, p.a.error_word);
    };

    if (warp == kLoadWarp) {
        const uint32_t rows_part = kv.page_tokens < static_cast<uint32_t>(kKeys) ? kv.page_tokens : kKeys;
        const uint32_t part_shift = kv.page_shift < 6u ? kv.page_shift : 6u;
        if (lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap)) : "memory");
        uint32_t hx = 0, issued = 0;    // half units
        for (uint64_t u = u0; u < u1;) {
            const Item item = next_item<kWideRows, kWideKeys>(p, head, elem);
            const uint32_t left = item.tiles - tile0;
            const uint32_t count = u1 - u < left ? static_cast<uint32_t>(u1 - u) : left;
            const int32_t *table = p.prefix_pass ? p.a.prefix_table : p.a.seqs.table + static_cast<uint64_t>(item.seq) * p.a.seqs.table_stride;
            const uint32_t last_page = item.keys > 0 ? static_cast<uint32_t>(item.keys - 1) >> kv.page_shift : 0u;
            uint32_t page_base = (tile0 * kWideKeys) >> kv.page_shift;
            int32_t page_id = page_base + lane <= last_page && item.keys > 0 ? table[page_base + lane] : -1;
            for (uint32_t tile = tile0; tile < tile0 + count; ++tile) {
                const uint32_t key0 = tile * kWideKeys;
                const uint32_t need = static_cast<uint32_t>(item.keys) > key0 ? static_cast<uint32_t>(item.keys) - key0 : 0u;
                const uint32_t parts = ((need < static_cast<uint32_t>(kWideKeys) ? need : kWideKeys) + rows_part - 1u) >> part_shift;
                if ((key0 >> kv.page_shift) + kWideKeys / 16 > page_base + 32u) {
                    page_base = key0 >> kv.page_shift;
                    page_id = page_base + lane <= last_page ? table[page_base + lane] : -1;
                }
                const uint32_t key = key0 + lane * rows_part;
                const int32_t id = __shfl_sync(0xFFFFFFFFu, page_id, ((key >> kv.page_shift) - page_base) & 31u);
                const bool wanted = static_cast<uint32_t>(lane) < parts;
                const bool good = wanted && id >= 0 && static_cast<uint32_t>(id) < kv.pages;
                const uint32_t good_mask = __ballot_sync(0xFFFFFFFFu, good), bad_mask = __ballot_sync(0xFFFFFFFFu, wanted && !good);
                const uint64_t krow = ((static_cast<uint64_t>(id) * 2u * kv.kv_heads + head) << kv.page_shift) + (key & (kv.page_tokens - 1u));
                for (int which = 0; which < 2; ++which, ++hx) {
                    const uint32_t stage = hx % W::STAGES, pass = hx / W::STAGES;
                    if (pass > 0) wait(s_code_empty[stage], (pass - 1u) & 1u);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) continue;
                    issued = hx + 1u;
                    const uint32_t bar = smem_u32(&s_code_full[stage]);
                    if (lane == 0) {
                        uint32_t bad = 0;
                        for (uint32_t x = 0; x < parts; ++x)
                            if ((bad_mask >> x) & 1u) bad |= ((1u << (rows_part >> 4)) - 1u) << (x * (rows_part >> 4));
                        s_bad[stage] = bad;
                        if (bad) atomicOr(p.a.error_word, kKvBadTable);
                        mbar_arrive_expect_tx(bar, __popc(good_mask) * rows_part * (RB + 2u * GS * 2u));
                    }
                    __syncwarp();
                    if (good) {
                        const uint64_t row = krow + (which ? static_cast<uint64_t>(kv.kv_heads) << kv.page_shift : 0ull);
                        const uint32_t dst = code_base + stage * W::STAGE, at = lane * rows_part;
                        tma_load_2d(dst + at * RB, &tmap, 0u, static_cast<uint32_t>(row), bar);
                        const uint32_t sdst = dst + W::CODES + at * GS * 2, bytes = rows_part * GS * 2;
                        bulk_load(sdst, kv.scales + row * GS, bytes, bar);
                        bulk_load(sdst + W::SB, kv.biases + row * GS, bytes, bar);
                    }
                    __syncwarp();
                }
            }
            u += count;
            tile0 = 0;
            if (++elem == p.elements) elem = 0, ++head;
        }
        if (!ok) {
            // given up: the copies in flight must land before the CTA may end
            for (uint32_t x = issued > static_cast<uint32_t>(W::STAGES) ? issued - W::STAGES : 0u; x < issued; ++x)
                for (uint32_t tries = 0; tries < (1u << 20) && !mbar_try_wait(smem_u32(&s_code_full[x % W::STAGES]), (x / W::STAGES) & 1u); ++tries) {
                }
        }
    } else if (warp == kMmaWarp) {
        constexpr uint32_t kIdesc = (1u << 4) | ((128u >> 4) << 24);                       // f16 x f16 -> f32, M = 128
        constexpr uint32_t kIdescS = kIdesc | ((kWideKeys >> 3) << 17);                    // N = 128 keys, both K-major
        constexpr uint32_t kIdescO = kIdesc | (1u << 16) | ((static_cast<uint32_t>(D) >> 3) << 17);   // N = D, V is N-major
        const uint64_t q_desc = desc_sw128(q_base, 16u, 1024u), k_desc = desc_sw128(tile_base, 16u, 1024u), v_desc = desc_sw128(tile_base, W::PANEL, 1024u);
        uint32_t kx = 0, weights_seen[2] = {0u, 0u}, q_seen[2] = {0u, 0u};
        for (uint64_t u = u0; u < u1;) {
            const Item item = next_item<kWideRows, kWideKeys>(p, head, elem);
            const uint32_t left = item.tiles - tile0;
            const uint32_t count = u1 - u < left ? static_cast<uint32_t>(u1 - u) : left;
            const uint32_t tiles = item.rows - item.row0 > 128u ? 2u : 1u;
            // O_t += P_t V of unit i
            auto second = [&](uint32_t t, uint32_t i) {
                const uint32_t vx = kx + 2u * i + 1u, buf = vx % W::TILES;
                if (t == 0u) wait(s_tile_full[buf], (vx / W::TILES) & 1u);
                const uint64_t vd = v_desc + ((buf * W::TILE) >> 4);
                const uint32_t out = tmem + 256u + 128u * t, in = tmem + 128u * t;
                const uint32_t add = i > 0u ? 1u : 0u, free_bar = smem_u32(&s_tile_empty[buf]), done_bar = smem_u32(&s_done[t]);
                const bool last_tile = t + 1u == tiles, last_unit = i + 1u == count;
                wait(s_weights[t], weights_seen[t]++ & 1u);
                fence_after();
                if (elect_one()) {
                    umma_ts(out, in, vd, kIdescO, add);
#pragma unroll
                    for (int k = 1; k < kWideKeys / 16; ++k) umma_ts(out, in + k * 8u, vd + k * 128u, kIdescO, 1u);
                    if (last_tile) umma_commit(free_bar);
                    if (last_unit) umma_commit(done_bar);
                }
                __syncwarp();
            };
            for (uint32_t i = 0; i < count; ++i) {
                const uint32_t kxi = kx + 2u * i, buf = kxi % W::TILES;
                const uint64_t kd = k_desc + ((buf * W::TILE) >> 4);
                const uint32_t free_bar = smem_u32(&s_tile_empty[buf]);
                wait(s_tile_full[buf], (kxi / W::TILES) & 1u);     // ready long before the weights as a rule
                for (uint32_t t = 0; t < tiles; ++t) {
                    if (i > 0) second(t, i - 1u);
                    else wait(s_q_ready[t], q_seen[t]++ & 1u);
                    const uint64_t qd = q_desc + ((t * W::TILE) >> 4);
                    const uint32_t out = tmem + 128u * t, score_bar = smem_u32(&s_score[t]);
                    const bool last_tile = t + 1u == tiles;
                    fence_after();
                    if (elect_one()) {
                        umma_ss(out, qd, kd, kIdescS, 0u);
#pragma unroll
                        for (int k = 1; k < D / 16; ++k) {
                            constexpr uint32_t kStep = W::PANEL >> 4;
                            umma_ss(out, qd + (k / 4) * kStep + (k % 4) * 2u, kd + (k / 4) * kStep + (k % 4) * 2u, kIdescS, 1u);
                        }
                        if (last_tile) umma_commit(free_bar);
                        umma_commit(score_bar);
                    }
                    __syncwarp();
                }
            }
            for (uint32_t t = 0; t < tiles; ++t) second(t, count - 1u);
            kx += 2u * count;
            u += count;
            tile0 = 0;
            if (++elem == p.elements) elem = 0, ++head;
        }
        // tensor memory is given back when nothing writes to it any more, on the way out of a failure too
        if (elect_one()) umma_commit(smem_u32(&s_idle));
        __syncwarp();
        for (uint32_t tries = 0; tries < (1u << 20) && !mbar_try_wait(smem_u32(&s_idle), 0u); ++tries) {
        }
        __syncwarp();
    } else if (warp >= kDequantWarp0) {
        // ---------------- dequantise: thread = cached row ----------------
        const uint32_t part = warp - kDequantWarp0;
        const uint32_t row = part * 32u + lane;
        const uint32_t swz = RB == 128 ? (row & 7u) : RB == 64 ? ((row >> 1) & 3u) : ((row >> 2) & 1u);
        constexpr float kHalf = static_cast<float>(1 << (BITS - 1)), kMost = static_cast<float>((1 << BITS) - 1);
        constexpr uint32_t kCentre = BITS == 8 ? 0xE480E480u : 0xE408E408u;     // -(1024 + h)
        constexpr uint32_t kCentreHigh = 0xD480D480u;                           // -(64 + 8)
        uint32_t hx = 0;
        for (uint64_t u = u0; u < u1;) {
            const Item item = next_item<kWideRows, kWideKeys>(p, head, elem);
            const uint32_t left = item.tiles - tile0;
            const uint32_t count = u1 - u < left ? static_cast<uint32_t>(u1 - u) : left;
            for (uint32_t tile = tile0; tile < tile0 + count; ++tile) {
#pragma unroll 1
                for (uint32_t which = 0; which < 2u; ++which, ++hx) {
                    const uint32_t stage = hx % W::STAGES, buf = hx % W::TILES, info = (hx >> 1) % kInfo;
                    wait(s_code_full[stage], (hx / W::STAGES) & 1u);
                    __syncwarp();
                    const uint32_t src = code_base + stage * W::STAGE;
                    const uint32_t bad = s_bad[stage];
                    const bool valid = static_cast<int32_t>(tile * kWideKeys + row) < item.keys && !((bad >> (row >> 4)) & 1u);
                    float s[GS], b[GS];
                    row_f32<GS>(src + W::CODES + row * GS * 2, s);
                    row_f32<GS>(src + W::CODES + W::SB + row * GS * 2, b);
                    uint32_t top = 0u, poison = 0u;      // bits of the largest finite magnitude
#pragma unroll
                    for (int i = 0; i < GS; ++i) {
                        if (!valid) s[i] = b[i] = 0.0f;
                        const float hi = fmaxf(fabsf(b[i]), fabsf(fmaf(kMost, s[i], b[i])));
                        if (hi - hi == 0.0f && s[i] - s[i] == 0.0f) top = max(top, __float_as_uint(hi));
                        else poison |= 1u << i;
                    }
                    top = __reduce_max_sync(0xFFFFFFFFu, top);
                    int e = static_cast<int>(top >> 23) - 127 - 14;
                    if (which == 0u) {
                        e = e < -114 ? -114 : e;
                        if (lane == 0) {
                            s_kmul[info][part] = pow2(e);
                            if (part == 0u) s_kbad[info] = bad;
                        }
                    } else {
                        e = e < kMinExp ? kMinExp : e;
                        // a value that is not finite must not reach rows that do not see its key: it is stored as zero, and rows
                        // that see it learn of it here
                        const uint32_t lost = __ballot_sync(0xFFFFFFFFu, poison != 0u);
                        if (lost) s_poison[info][row] = static_cast<uint8_t>(poison);
                        if (lane == 0) {
                            s_vexp[info][part] = static_cast<float>(e);
                            s_vinv[info][part] = pow2(-e);
                            s_lost[info][part] = lost;
                        }
                    }
                    const float mul = pow2(-e);          // e between -114 and 114
                    if (hx >= static_cast<uint32_t>(W::TILES)) wait(s_tile_empty[buf], (hx / W::TILES - 1u) & 1u);
                    __syncwarp();
                    constexpr int kChunks = RB / 16;                 // 16-byte chunks of codes in a row
                    constexpr int kOut = BITS == 8 ? 2 : 4;          // 16-byte chunks of f16 that 16 bytes of codes make
                    const uint32_t dst = tile_base + buf * W::TILE + row * 128u, from = src + row * RB, scale_at = src + W::CODES + row * GS * 2;
                    // not unrolled: the roles share the instruction cache
#pragma unroll 1
                    for (uint32_t g = 0; g < static_cast<uint32_t>(GS); ++g) {
                        uint32_t si, bi;
                        lds<2>(scale_at + g * 2u, &si);
                        lds<2>(scale_at + W::SB + g * 2u, &bi);
                        const bool none = !valid || (which == 1u && ((poison >> g) & 1u));
                        const float sg = none ? 0.0f : bf16_f32(si), bg = none ? 0.0f : bf16_f32(bi);
                        const float sc = sg * mul, bc = fmaf(kHalf, sg, bg) * mul;
                        const uint32_t sh = pack_f16x2(sc, sc), bh = pack_f16x2(bc, bc);
#pragma unroll 1
                        for (uint32_t c = g * (kChunks / GS); c < (g + 1u) * (kChunks / GS); ++c) {
                            uint32_t w[4];
                            lds<16>(from + ((c ^ swz) << 4), w);
#pragma unroll
                            for (int x = 0; x < kOut; ++x) {
                                const uint32_t to = c * kOut + x;
                                uint32_t y[4];
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    uint32_t code;
                                    if (BITS == 8) {
                                        code = add_f16x2(prmt(w[2 * x + (i >> 1)], 0x64646464u, (i & 1) ? 0x4342u : 0x4140u), kCentre);
                                    } else {
                                        const uint32_t n = i >= 2 ? w[x] >> 8 : w[x];
                                        code = (i & 1) ? f16_high(n, kCentreHigh) : f16_low(n, kCentre);
                                    }
                                    y[i] = fma_f16x2(code, sh, bh);
                                }
                                const uint32_t at = dst + (to / 8u) * W::PANEL + (((to & 7u) ^ (row & 7u)) << 4);
                                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
                            }
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&s_code_empty[stage]));
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&s_tile_full[buf]));
                }
            }
            u += count;
            tile0 = 0;
            if (++elem == p.elements) elem = 0, ++head;
        }
    } else {
        // ---------------- softmax: thread = query row ----------------
        const uint32_t t = warp >> 2, r = threadIdx.x & 127u;       // row r of tile t
        const uint32_t tm = tmem + ((static_cast<uint32_t>(warp) & 3u) << 21);     // this warp's lanes
        const uint32_t tm_s = tm + 128u * t, tm_o = tm + 256u + 128u * t;
        uint32_t kx = 0, scores_seen = 0, done_seen = 0;
        for (uint64_t u = u0; u < u1;) {
            const Item item = next_item<kWideRows, kWideKeys>(p, head, elem);
            const uint32_t left = item.tiles - tile0;
            const uint32_t count = u1 - u < left ? static_cast<uint32_t>(u1 - u) : left;
            const bool active = t == 0u || item.rows - item.row0 > 128u;
            const uint32_t row = item.row0 + t * 128u + r;
            const bool have = row < item.rows;
            float m = kNoMax, l = 0.0f;
            uint32_t poison = 0u;
            const bool whole = tile0 == 0u && count == item.tiles;
            float *const part = p.partials + static_cast<uint64_t>(2u * blockIdx.x + (tile0 == 0u ? 1u : 0u)) * W::PART;
            if (active) {
                // ---- q: scaled by a power of two, f16 ----
                float f;
                bool finite;
                {
                    uint32_t x[D / 2];      // bf16 pairs
#pragma unroll
                    for (int i = 0; i < D / 2; ++i) x[i] = 0u;
                    if (have) {
                        const uint16_t *src = static_cast<const uint16_t *>(p.a.q) + static_cast<uint64_t>(item.token0 + row / p.per_kv) * p.a.qs.token +
                                              static_cast<uint64_t>(head * p.per_kv + row % p.per_kv) * p.a.qs.head;
                        if (p.q_vec) {
#pragma unroll
                            for (int i = 0; i < D / 8; ++i) {
                                const uint4 y = *reinterpret_cast<const uint4 *>(src + 8 * i);
                                x[4 * i] = y.x, x[4 * i + 1] = y.y, x[4 * i + 2] = y.z, x[4 * i + 3] = y.w;
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < D / 2; ++i) x[i] = src[2 * i] | (static_cast<uint32_t>(src[2 * i + 1]) << 16);
                        }
                    }
                    uint32_t top = 0u;
#pragma unroll
                    for (int i = 0; i < D / 2; ++i) top = max(top, max((x[i] << 16) & 0x7FFFFFFFu, x[i] & 0x7FFF0000u));
                    finite = top < 0x7F800000u;
                    int e = static_cast<int>(top >> 23) - 127;
                    e = e < -100 ? -100 : e > 127 ? 127 : e;
                    // the sign of the scale goes to q, so that the largest raw score is the largest score
                    const float mul = p.a.scale < 0.0f ? -pow2(13 - e) : pow2(13 - e);
                    f = pow2(e - 13) * (fabsf(p.a.scale) * 1.4426950408889634f);
                    const uint32_t dst = q_base + t * W::TILE + r * 128u;
#pragma unroll
                    for (int c = 0; c < D / 8; ++c) {
                        uint32_t y[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int d0 = value_at<BITS>(2 * i), d1 = value_at<BITS>(2 * i + 1);
                            const uint32_t w0 = x[4 * c + d0 / 2], w1 = x[4 * c + d1 / 2];
                            y[i] = pack_f16x2(((d0 & 1) ? __uint_as_float(w0 & 0xFFFF0000u) : bf16_f32(w0)) * mul,
                                              ((d1 & 1) ? __uint_as_float(w1 & 0xFFFF0000u) : bf16_f32(w1)) * mul);
                        }
                        const uint32_t at = dst + (c / 8) * W::PANEL + (((c & 7) ^ (r & 7u)) << 4);
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
                    }
                }
                fence_async_smem();
                fence_before();
                mbar_arrive(smem_u32(&s_q_ready[t]));
                int32_t seen = p.prefix_pass ? item.seen0 : item.seen0 + static_cast<int32_t>(row / p.per_kv);
                seen = seen < item.keys ? seen : item.keys;

                for (uint32_t i = 0; i < count; ++i) {
                    const int32_t key0 = static_cast<int32_t>((tile0 + i) * kWideKeys);
                    const uint32_t vx = kx + 2u * i + 1u, info = (vx >> 1) % kInfo;
                    // in this order: the scores are proof that the fill before the values' in their buffer is over, without which
                    // the parity could be that of an older one (a tile that rests in a segment runs ahead of the other)
                    wait(s_score[t], scores_seen++ & 1u);
                    __syncwarp();
                    fence_after();
                    const uint32_t bad = s_kbad[info];
                    const bool border = key0 + kWideKeys > item.first_seen || bad != 0u;
                    // 32 keys: scores to weights, which take half of the columns of scores that have been read
                    auto chunk = [&](int c, uint32_t (&x)[32]) {
                        const float fk = fmaxf(f * s_kmul[info][c], kMinFactor), ve = s_vexp[info][c];
                        float tops[4] = {__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]), __uint_as_float(x[3])};
#pragma unroll
                        for (int k = 4; k < 32; ++k) tops[k & 3] = fmaxf(tops[k & 3], __uint_as_float(x[k]));
                        const float top = fmaf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), fk, ve);
                        if (__any_sync(0xFFFFFFFFu, top > m + kWideMost)) {
                            const float m1 = fmaxf(m, ceilf(top) - kWideTarget);
                            const float keep = pow2_or_0(-static_cast<int>(fminf(m1 - m, 1000.0f)));
                            m = m1;
                            l *= keep;
                            tmem_wait_st();      // the weights of the chunk before may still be on their way to the columns read here
#pragma unroll 1
                            for (int y = i > 0 ? 0 : D / 16; y < D / 16 + c; ++y) {     // O, then this unit's weights so far
                                uint32_t z[16];
                                const uint32_t at = y < D / 16 ? tm_o + 16u * y : tm_s + 16u * (y - D / 16);
                                tmem_ld16(at, z);
                                tmem_wait_ld();
#pragma unroll
                                for (int k = 0; k < 16; ++k) {
                                    if (y < D / 16) {
                                        z[k] = __float_as_uint(__uint_as_float(z[k]) * keep);
                                    } else {
                                        const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&z[k]));
                                        z[k] = pack_f16x2(v.x * keep, v.y * keep);
                                    }
                                }
                                tmem_st16(at, z);
                            }
                            tmem_wait_st();
                        }
                        const float use = ve - m;
                        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        uint32_t w[16];
                        float e[32];
#pragma unroll
                        for (int k = 0; k < 32; ++k) e[k] = fmaf(__uint_as_float(x[k]), fk, use);
#pragma unroll
                        for (int k = 0; k < 32; ++k) e[k] = exp2_approx(e[k]);
#pragma unroll
                        for (int k = 0; k < 32; ++k) sum[k & 3] += e[k];
#pragma unroll
                        for (int k = 0; k < 16; ++k) w[k] = pack_f16x2(e[2 * k], e[2 * k + 1]);
                        l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), s_vinv[info][c], l);
                        tmem_st16(tm_s + 16u * c, w);
                    };
                    if (border) {            // what the row does not see is taken out
#pragma unroll 1
                        for (int c = 0; c < 8; ++c) {
                            const int32_t left = (bad >> c) & 1u ? 0 : seen - key0 - 16 * c;
                            if (__all_sync(0xFFFFFFFFu, left >= 16)) continue;
                            uint32_t x[16];
                            tmem_ld16(tm_s + 16u * c, x);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 16; ++k)
                                if (k >= left) x[k] = 0xFF800000u;
                            tmem_st16(tm_s + 16u * c, x);
                        }
                        tmem_wait_st();
                    }
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t x[32];
                        tmem_ld32(tm_s + 32u * c, x);
                        if (c == 0) {
                            wait(s_tile_full[vx % W::TILES], (vx / W::TILES) & 1u);
                            __syncwarp();
                        }
                        tmem_wait_ld();
                        chunk(c, x);
                    }
                    const uint4 lost = *reinterpret_cast<const uint4 *>(s_lost[info]);
                    if (lost.x | lost.y | lost.z | lost.w) {
                        for (int k = 0; k < kWideKeys; ++k)
                            if (key0 + k < seen && ((s_lost[info][k >> 5] >> (k & 31)) & 1u)) poison |= s_poison[info][k];
                        __syncwarp();
                    }
                    tmem_wait_st();
                    fence_before();
                    mbar_arrive(smem_u32(&s_weights[t]));
                }
                // ---- end of the segment ----
                wait(s_done[t], done_seen++ & 1u);
                __syncwarp();
                fence_after();
                if (!finite && seen > 0) l = __uint_as_float(0x7FC00000u);    // a row that is not finite, whose scores may all be -inf
                if (!whole && have) {
                    __stcg(part + kWideRows * D + t * 128u + r, m);
                    __stcg(part + kWideRows * (D + 1) + t * 128u + r, l);
                }
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t raw[32];
                    tmem_ld32(tm_o + 32u * c, raw);
                    tmem_wait_ld();
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        if (!have) break;
                        float v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            // value 4x + k of the 32 stands at the place that its eight keep it
                            const int in = (4 * x + k) % 8, place = BITS == 8 ? in : ((in & 3) * 2 + (in >> 2));
                            v[k] = __uint_as_float(raw[(4 * x + k) / 8 * 8 + place]);
                        }
                        if ((poison >> (c * 32 / GROUP)) & 1u) v[0] = v[1] = v[2] = v[3] = __uint_as_float(0x7FC00000u);
                        const uint32_t d = 32u * c + 4u * x;
                        if (whole) finish_row<D, false>(p, item, head, t * 128u + r, d, m, l, make_float4(v[0], v[1], v[2], v[3]));
                        else __stcg(reinterpret_cast<float4 *>(part + (static_cast<uint64_t>(d / 4u) * kWideRows + t * 128u + r) * 4u), make_float4(v[0], v[1], v[2], v[3]));
                    }
                    __syncwarp();
                }
                fence_before();
            }
            kx += 2u * count;
            if (tile0 == 0u && !whole && threadIdx.x == 0) {
                // the item goes on in the next CTAs: the pass that joins their results finds it here
                const uint32_t last = static_cast<uint32_t>(((u + item.tiles) * range.ctas - 1) / range.units);
                Cut &cut = p.cuts[blockIdx.x];
                cut.item = item;
                cut.head = head;
                cut.parts = last - blockIdx.x + 1u;
            }
            u += count;
            tile0 = 0;
            if (++elem == p.elements) elem = 0, ++head;
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// Joins the results of items that were cut across CTAs: grid (CTAs of the wide kernel) x (blocks of 32 rows), thread = a row and
// every eighth four of its values, so that a warp reads 32 rows' neighbours of the partial results.
template <int D>
__global__ void __launch_bounds__(256) gaf_attend_join_kernel(const __grid_constant__ Params p) {
    constexpr int kPart = kWideRows * (D + 2);
    const Cut &cut = p.cuts[blockIdx.x];
    const uint32_t parts = cut.parts;
    if (parts == 0u) return;
    const Item item = cut.item;
    const uint32_t r = blockIdx.y * 32u + (threadIdx.x & 31u);
    if (item.row0 + r >= item.rows) return;
    auto part_of = [&](uint32_t c) { return p.partials + static_cast<uint64_t>(2u * (blockIdx.x + c) + (c == 0u ? 1u : 0u)) * kPart; };
    float top = kNoMax, sum = 0.0f;
    for (uint32_t c = 0; c < parts; ++c) top = fmaxf(top, part_of(c)[kWideRows * D + r]);
    for (uint32_t c = 0; c < parts; ++c) {
        const float mc = part_of(c)[kWideRows * D + r];
        sum += part_of(c)[kWideRows * (D + 1) + r] * (mc == top ? 1.0f : exp2_approx(mc - top));
    }
    float4 v[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t c = 0; c < parts; ++c) {
        const float *src = part_of(c);
        const float mc = src[kWideRows * D + r];
        const float wc = mc == top ? 1.0f : exp2_approx(mc - top);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const float4 x = *reinterpret_cast<const float4 *>(src + (static_cast<uint64_t>((threadIdx.x >> 5) + 8u * i) * kWideRows + r) * 4u);
            v[i] = make_float4(fmaf(x.x, wc, v[i].x), fmaf(x.y, wc, v[i].y), fmaf(x.z, wc, v[i].z), fmaf(x.w, wc, v[i].w));
        }
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) finish_row<D, false>(p, item, cut.head, r, ((threadIdx.x >> 5) + 8u * i) * 4u, top, sum, v[i]);
}

template <int D, int BITS, int GROUP>
cudaError_t launch_wide(const Params &p, const CUtensorMap &tmap, int sm_count, cudaStream_t stream) {
    using W = Wide<D, BITS, GROUP>;
    auto kernel = gaf_attend_wide_kernel<D, BITS, GROUP>;
    static DeviceOnce once;    // of this instance
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, W::SMEM); });
    if (e != cudaSuccess) return e;
    kernel<<<sm_count, kWideThreads, W::SMEM, stream>>>(p, tmap);
    gaf_attend_join_kernel<D><<<dim3(sm_count, kWideRows / 32), 256, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace attend
}  // namespace tgaf
