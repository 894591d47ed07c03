// Attention over the quantised KV cache on tcgen05, for many query rows per cached head (prompts, shared prefixes).
//
// Mathematics.  Keys and values are dequantised to f16, 32 keys at a time with one power of two that brings their largest
// magnitude to 2^14..2^15: 11 bits of every element that is within 2^-29 of that.  bf16 would hold any range as it is, but its
// 8 bits on keys and values alone put the result 3e-3 off; f16 leaves them at 2^-12.
//   w 2^-e = (c - h) (s 2^-e) + (b + h s) 2^-e,   h = 2^(bits - 1): the centred code and s 2^-e are exact in f16
// q is f16 with a power of two per row (exact), the weights are f16 (2^-12 of each), all statistics and sums f32.  The keys'
// power goes into the scores' factor, the values' into the weights: they are formed as 2^(y + e - m) (y: scores in base
// 2), where m follows the largest y + e instead of the largest y, and leave it again in the row's sum.
//
// One CTA per SM, 256 query rows (two MMA tiles of 128) against units of 128 keys:
//   warps 0-7, 8-15  softmax of tile 0 and 1, two threads per row with 64 keys each: scores from tensor memory, weights (f16)
//                    back into the scores' columns, where the second product takes them as its A operand
//   warps 16-19      dequantise, one cached row per thread; K (K-major) and V (N-major) tiles have the same image
//   warp 20          issues the MMAs: per unit S_t = Q_t K^T and O_t += P_t V for both tiles; while one tile's softmax
//                    runs, the tensor core works for the other
//   warp 21          TMA of codes, bulk copies of scales and biases
// K and V tiles share a ring of three 32 KB buffers, their codes one of three stages: K(i), V(i), K(i+1), ...
//
// The reference follows lazily, as in the narrow kernel: only when a row of the warp exceeds it by 2^8 is O rescaled in tensor
// memory.  The scores are read twice (maximum, weights), 32 at a time in loops that are not unrolled.  A chunk of two
// prompts (768 and 1024 new tokens over 3750 and 5000 cached ones, 32 heads on 8): 387 us with one unrolled pass that was
// repeated when the reference had to follow (it ran out of the instruction cache), 262 with two passes and one thread a
// row, TTT with two threads a row.
// What bounds it: 2 x 128 x 128 exponentials per unit (16 per clock and SM) and as many clocks of tensor work; what keeps it
// from there is the way of one tile's unit through scores, softmax, weights and second product, which the other tile
// covers only in part.
#pragma once
#include "gaf_attend.cuh"

namespace tgaf {
namespace attend {

constexpr int kWideKeys = 128;
constexpr int kWideRows = 256;
constexpr int kWideThreads = 22 * 32;    // 80 registers each
constexpr int kDequantWarp0 = 16, kDequantWarps = 4, kMmaWarp = 20, kLoadWarp = 21;
constexpr int kInfo = 4;             // units whose side information is kept
constexpr float kMinFactor = 1.0e-37f;   // of raw scores: not 0, since hidden ones are -inf
constexpr int kMinExp = -50;         // values below 2^-36 lose bits instead of pushing the weights out of f32

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
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
          "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
          "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
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
    __shared__ uint32_t s_kbad[kInfo], s_lost[kInfo][4];
    __shared__ uint8_t s_poison[kInfo][kWideKeys];  // by key
    __shared__ float s_pair[2][2][128];             // what the two threads of a row tell each other
    __shared__ uint32_t s_tmem;
    __shared__ volatile uint32_t s_abort;
    __shared__ uint32_t s_scan[kWideThreads / 32];
    __shared__ uint32_t s_begin[3];
    __shared__ uint32_t s_last;

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
            mbar_init(smem_u32(&s_q_ready[i]), 256);
            mbar_init(smem_u32(&s_score[i]), 1);
            mbar_init(smem_u32(&s_weights[i]), 256);
            mbar_init(smem_u32(&s_done[i]), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    Range range;
    if (!cta_range<kWideRows, kWideKeys, kWideThreads>(p, s_scan, s_begin, range)) return;
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
                    uint32_t sh[GS], bh[GS];
#pragma unroll
                    for (int i = 0; i < GS; ++i) {
                        if (which == 1u && ((poison >> i) & 1u)) s[i] = b[i] = 0.0f;
                        const float sc = s[i] * mul, bc = fmaf(kHalf, s[i], b[i]) * mul;
                        sh[i] = pack_f16x2(sc, sc);
                        bh[i] = pack_f16x2(bc, bc);
                    }
                    constexpr int kChunks = RB / 16;                 // 16-byte chunks of codes in a row
                    constexpr int kOut = BITS == 8 ? 2 : 4;          // 16-byte chunks of f16 that 16 bytes of codes make
                    uint32_t w[kChunks][4];
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) lds<16>(src + row * RB + ((c ^ swz) << 4), w[c]);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&s_code_empty[stage]));
                    if (hx >= static_cast<uint32_t>(W::TILES)) wait(s_tile_empty[buf], (hx / W::TILES - 1u) & 1u);
                    __syncwarp();
                    const uint32_t dst = tile_base + buf * W::TILE + row * 128u;
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
                        for (int x = 0; x < kOut; ++x) {
                            const int chunk = c * kOut + x, gi = chunk * 8 / GROUP;
                            uint32_t y[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                uint32_t code;
                                if (BITS == 8) {
                                    code = add_f16x2(prmt(w[c][2 * x + (i >> 1)], 0x64646464u, (i & 1) ? 0x4342u : 0x4140u), kCentre);
                                } else {
                                    const uint32_t n = i >= 2 ? w[c][x] >> 8 : w[c][x];
                                    code = (i & 1) ? f16_high(n, kCentreHigh) : f16_low(n, kCentre);
                                }
                                y[i] = fma_f16x2(code, sh[gi], bh[gi]);
                            }
                            const uint32_t at = dst + (chunk / 8) * W::PANEL + (((chunk & 7) ^ (row & 7u)) << 4);
                            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
                        }
                    }
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
        // ---------------- softmax: two threads per query row ----------------
        const uint32_t t = warp >> 3, half = (warp >> 2) & 1u, r = (warp & 3u) * 32u + lane;       // row r of tile t, keys 64 half ..
        const uint32_t tm = tmem + ((static_cast<uint32_t>(warp) & 3u) << 21);     // this warp's lanes
        const uint32_t tm_s = tm + 128u * t + 64u * half, tm_w = tm + 128u * t + 32u * half, tm_o = tm + 256u + 128u * t + (D / 2) * half;
        const uint32_t pair_bar = 1u + t * 4u + (warp & 3u);
        auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory"); };
        // the other thread's value; the barrier in front of the write keeps the last exchange's values until they are read
        auto exchange = [&](float v) {
            pair_sync();
            s_pair[t][half][r] = v;
            pair_sync();
            return s_pair[t][half ^ 1u][r];
        };
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
                // ---- q: scaled by a power of two, f16; each thread half of the row ----
                float f;
                {
                    uint32_t x[D / 4];      // bf16 pairs
#pragma unroll
                    for (int i = 0; i < D / 4; ++i) x[i] = 0u;
                    if (have) {
                        const uint16_t *src = static_cast<const uint16_t *>(p.a.q) + static_cast<uint64_t>(item.token0 + row / p.per_kv) * p.a.qs.token +
                                              static_cast<uint64_t>(head * p.per_kv + row % p.per_kv) * p.a.qs.head + half * (D / 2);
                        if (p.q_vec) {
#pragma unroll
                            for (int i = 0; i < D / 16; ++i) {
                                const uint4 y = *reinterpret_cast<const uint4 *>(src + 8 * i);
                                x[4 * i] = y.x, x[4 * i + 1] = y.y, x[4 * i + 2] = y.z, x[4 * i + 3] = y.w;
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < D / 4; ++i) x[i] = src[2 * i] | (static_cast<uint32_t>(src[2 * i + 1]) << 16);
                        }
                    }
                    uint32_t top = 0u;
#pragma unroll
                    for (int i = 0; i < D / 4; ++i) top = max(top, max((x[i] << 16) & 0x7FFFFFFFu, x[i] & 0x7FFF0000u));
                    __syncwarp();
                    top = max(top, __float_as_uint(exchange(__uint_as_float(top))));
                    int e = static_cast<int>(top >> 23) - 127;
                    e = e < -100 ? -100 : e > 127 ? 127 : e;
                    // the sign of the scale goes to q, so that the largest raw score is the largest score
                    const float mul = p.a.scale < 0.0f ? -pow2(13 - e) : pow2(13 - e);
                    f = pow2(e - 13) * (fabsf(p.a.scale) * 1.4426950408889634f);
                    const uint32_t dst = q_base + t * W::TILE + r * 128u + (D == 128 ? half * W::PANEL : 0u);
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t y[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int d0 = value_at<BITS>(2 * i), d1 = value_at<BITS>(2 * i + 1);
                            const uint32_t w0 = x[4 * c + d0 / 2], w1 = x[4 * c + d1 / 2];
                            y[i] = pack_f16x2(((d0 & 1) ? __uint_as_float(w0 & 0xFFFF0000u) : bf16_f32(w0)) * mul,
                                              ((d1 & 1) ? __uint_as_float(w1 & 0xFFFF0000u) : bf16_f32(w1)) * mul);
                        }
                        const uint32_t chunk = D == 128 ? c : half * (D / 16) + c;
                        const uint32_t at = dst + ((chunk ^ (r & 7u)) << 4);
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
                    // values are ready before the scores as a rule: waiting for them first takes that wait out of the way
                    const uint32_t vx = kx + 2u * i + 1u, info = (vx >> 1) % kInfo;
                    wait(s_tile_full[vx % W::TILES], (vx / W::TILES) & 1u);
                    wait(s_score[t], scores_seen++ & 1u);
                    __syncwarp();
                    fence_after();
                    const uint32_t bad = s_kbad[info];
                    // 32 raw scores; kBorder: those that the row does not see taken out
                    auto scores = [&](auto border_tag, int c, uint32_t (&raw)[32]) {
                        tmem_ld32(tm_s + 32u * c, raw);
                        tmem_wait_ld();
                        if (decltype(border_tag)::value) {
                            const int32_t left = seen - key0 - 64 * static_cast<int32_t>(half) - 32 * c;
                            const uint32_t gone = bad >> (4u * half + 2u * c);
#pragma unroll
                            for (int k = 0; k < 32; ++k)
                                if (k >= left || ((gone >> (k / 16)) & 1u)) raw[k] = 0xFF800000u;
                        }
                    };
                    auto unit = [&](auto border_tag) {
                        float top = -INFINITY;
#pragma unroll 1
                        for (int c = 0; c < 2; ++c) {
                            uint32_t raw[32];
                            scores(border_tag, c, raw);
                            float t0 = __uint_as_float(raw[0]), t1 = __uint_as_float(raw[1]);
#pragma unroll
                            for (int k = 2; k < 32; k += 2) {
                                t0 = fmaxf(t0, __uint_as_float(raw[k]));
                                t1 = fmaxf(t1, __uint_as_float(raw[k + 1]));
                            }
                            top = fmaxf(top, fmaf(fmaxf(t0, t1), fmaxf(f * s_kmul[info][2 * half + c], kMinFactor), s_vexp[info][2 * half + c]));
                        }
                        top = fmaxf(top, exchange(top));
                        if (__any_sync(0xFFFFFFFFu, top > m + kLazy)) {
                            const float m1 = fmaxf(m, top);
                            const float keep = m1 == m ? 1.0f : exp2_approx(m - m1);
                            m = m1;
                            l *= keep;
                            if (i > 0) {
#pragma unroll 1
                                for (int c = 0; c < D / 64; ++c) {
                                    uint32_t raw[32];
                                    tmem_ld32(tm_o + 32u * c, raw);
                                    tmem_wait_ld();
#pragma unroll
                                    for (int k = 0; k < 32; ++k) raw[k] = __float_as_uint(__uint_as_float(raw[k]) * keep);
                                    tmem_st32(tm_o + 32u * c, raw);
                                }
                            }
                        }
                        // the weights of 32 keys take 16 of the row's first 64 columns.  The other thread may still be reading
                        // scores there: its weights wait until both are through (the loop writes after its last read)
                        uint32_t w[32];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            uint32_t raw[32];
                            scores(border_tag, c, raw);
                            const float fk = fmaxf(f * s_kmul[info][2 * half + c], kMinFactor), use = s_vexp[info][2 * half + c] - m;
                            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                float e[16];
#pragma unroll
                                for (int k = 0; k < 16; ++k) e[k] = fmaf(__uint_as_float(raw[16 * y + k]), fk, use);
#pragma unroll
                                for (int k = 0; k < 16; ++k) e[k] = exp2_approx(e[k]);
#pragma unroll
                                for (int k = 0; k < 16; ++k) sum[k & 3] += e[k];
#pragma unroll
                                for (int k = 0; k < 8; ++k) w[16 * c + 8 * y + k] = pack_f16x2(e[2 * k], e[2 * k + 1]);
                            }
                            l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), s_vinv[info][2 * half + c], l);
                        }
                        pair_sync();
                        tmem_st32(tm_w, w);
                    };
                    if (key0 + kWideKeys > item.first_seen || bad != 0u) unit(std::true_type());
                    else unit(std::false_type());
                    if (s_lost[info][2 * half] | s_lost[info][2 * half + 1]) {
                        for (uint32_t k = 64u * half; k < 64u * half + 64u; ++k)
                            if (key0 + static_cast<int32_t>(k) < seen && ((s_lost[info][k >> 5] >> (k & 31u)) & 1u)) poison |= s_poison[info][k];
                        __syncwarp();
                    }
                    tmem_wait_st();
                    fence_before();
                    mbar_arrive(smem_u32(&s_weights[t]));
                }
                // ---- end of the segment ----
                l += exchange(l);
                poison |= __float_as_uint(exchange(__uint_as_float(poison)));
                wait(s_done[t], done_seen++ & 1u);
                __syncwarp();
                fence_after();
                if (!whole && have && half == 0u) {
                    __stcg(part + kWideRows * D + t * 128u + r, m);
                    __stcg(part + kWideRows * (D + 1) + t * 128u + r, l);
                }
#pragma unroll 1
                for (int c = 0; c < D / 64; ++c) {
                    uint32_t raw[32];
                    tmem_ld32(tm_o + 32u * c, raw);
                    tmem_wait_ld();
                    const uint32_t d0 = half * (D / 2) + 32u * c;
                    const bool lost = (poison >> (d0 / GROUP)) & 1u;
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        if (!have) break;
                        float v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            // value 4x + k of the 32 stands at the place that its eight keep it
                            const int in = (4 * x + k) % 8, place = BITS == 8 ? in : ((in & 3) * 2 + (in >> 2));
                            v[k] = lost ? __uint_as_float(0x7FC00000u) : __uint_as_float(raw[(4 * x + k) / 8 * 8 + place]);
                        }
                        const uint32_t d = d0 + 4u * x;
                        if (whole) finish_row<D, false>(p, item, head, t * 128u + r, d, m, l, make_float4(v[0], v[1], v[2], v[3]));
                        else __stcg(reinterpret_cast<float4 *>(part + (static_cast<uint64_t>(d / 4u) * kWideRows + t * 128u + r) * 4u), make_float4(v[0], v[1], v[2], v[3]));
                    }
                    __syncwarp();
                }
                fence_before();
            }
            kx += 2u * count;
            if (!whole) {
                const uint64_t first_unit = u - tile0;
                const uint32_t c0 = static_cast<uint32_t>(((first_unit + 1) * range.ctas - 1) / range.units);
                const uint32_t c1 = static_cast<uint32_t>(((first_unit + item.tiles) * range.ctas - 1) / range.units);
                __threadfence();
                asm volatile("bar.sync 9, 512;" ::: "memory");
                if (threadIdx.x == 0) {
                    const uint32_t seen = atomicAdd(p.tickets + c0, 1u);
                    s_last = seen == c1 - c0;
                    if (s_last) p.tickets[c0] = 0u;
                }
                asm volatile("bar.sync 9, 512;" ::: "memory");
                if (s_last && have) {
                    __threadfence();
                    const uint32_t rr = t * 128u + r;
                    auto part_of = [&](uint32_t c) { return p.partials + static_cast<uint64_t>(2u * c + (c == c0 ? 1u : 0u)) * W::PART; };
                    float top = kNoMax, sum = 0.0f;
                    for (uint32_t c = c0; c <= c1; ++c) top = fmaxf(top, __ldcg(part_of(c) + kWideRows * D + rr));
                    for (uint32_t c = c0; c <= c1; ++c) {
                        const float mc = __ldcg(part_of(c) + kWideRows * D + rr);
                        sum += __ldcg(part_of(c) + kWideRows * (D + 1) + rr) * (mc == top ? 1.0f : exp2_approx(mc - top));
                    }
                    for (uint32_t d = half * (D / 2); d < (half + 1u) * (D / 2); d += 8u) {
                        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f), w = v;
                        for (uint32_t c = c0; c <= c1; ++c) {
                            const float *src = part_of(c);
                            const float4 x = __ldcg(reinterpret_cast<const float4 *>(src + (static_cast<uint64_t>(d / 4u) * kWideRows + rr) * 4u));
                            const float4 y = __ldcg(reinterpret_cast<const float4 *>(src + (static_cast<uint64_t>(d / 4u + 1u) * kWideRows + rr) * 4u));
                            const float mc = __ldcg(src + kWideRows * D + rr);
                            const float wc = mc == top ? 1.0f : exp2_approx(mc - top);
                            v = make_float4(fmaf(x.x, wc, v.x), fmaf(x.y, wc, v.y), fmaf(x.z, wc, v.z), fmaf(x.w, wc, v.w));
                            w = make_float4(fmaf(y.x, wc, w.x), fmaf(y.y, wc, w.y), fmaf(y.z, wc, w.z), fmaf(y.w, wc, w.w));
                        }
                        finish_row<D, false>(p, item, head, rr, d, top, sum, v);
                        finish_row<D, false>(p, item, head, rr, d + 4u, top, sum, w);
                    }
                }
                asm volatile("bar.sync 9, 512;" ::: "memory");   // s_last is free again
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

template <int D, int BITS, int GROUP>
cudaError_t launch_wide(const Params &p, const CUtensorMap &tmap, int sm_count, cudaStream_t stream) {
    using W = Wide<D, BITS, GROUP>;
    auto kernel = gaf_attend_wide_kernel<D, BITS, GROUP>;
    static DeviceOnce once;    // of this instance
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, W::SMEM); });
    if (e != cudaSuccess) return e;
    kernel<<<sm_count, kWideThreads, W::SMEM, stream>>>(p, tmap);
    return cudaGetLastError();
}

}  // namespace attend
}  // namespace tgaf
