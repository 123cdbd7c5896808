// Paged attention on the tensor cores proper (tcgen05), for row tiles that are full: prompts, and a prefix whose rows come
// from the whole batch.  What is computed and how the work is divided stands in paged_attention.cuh.
//
// attn_tc_kernel<D, BF16>, one CTA per SM, row tiles of 256 = two halves of 128 that share every key tile of 128:
//   S_h = Q_h K^T   (128 x 128, accumulator in tensor memory, operands in shared memory)
//   P_h = 2^(scale_log2 S_h - m)   by eight warps: two threads per row, one for each 64 keys
//   O_h += P_h V    (P from tensor memory, where it replaces S; V as it lies in the page, rows = keys, MN-major operand)
// While one half's warps take exponentials, the tensor core works for the other.  (With one thread per row a half's way from S to
// P took 1700 cycles however few other warps there were, a single warp's latency, and the two halves could not cover
// each other's way through the tensor core.)  Warps: 0-7 and 8-15 the halves' softmax and epilogue; 16 loads key and value tiles page
// by page and clears the rows of V behind the last key (their weights are zero, but what lies there may be NaN); 17 issues
// the MMAs; 18-19 bring the query rows of the next item.
// The reference m is the row's maximum over its first tile and is only raised when the weights of a tile add up to more than
// 2^10: weights above 1 change no digit of a floating-point result, no maximum is taken per tile, and O in tensor
// memory is rescaled a few times per item at most instead of once per tile.
// Weights are rounded to the cache's type for the product with V; their sum is taken before the rounding, in float32.
//
// What bounds it: 4 x 2048 causal, 32 heads of 128, takes 202 us, 680 TFLOP/s of visible pairs, 0.41 of the measured cuBLAS rate.  A key tile of
// 256 x 128 takes about 4200 cycles; its MMAs need 2048 (and 2048 of the shared memory's, with the tiles' arrival), its
// exponentials 2048.  With the MMAs left out it takes 175 us, with the softmax left out 182, without epilogue and first maximum 182: no
// part alone, but the hand-overs between them.  Two S buffers of 64 keys per half, so that no softmax waits for the way
// through the tensor core, took 220 us (MMAs of 64 columns read their A operand twice as often).
#include <atomic>

#include "paged_attention.cuh"

namespace mxfp4 {
namespace {

constexpr int kTcThreads = 640;
constexpr int kTcR = 256, kTcK = 128;
constexpr float kHigh = 1024.0f;

template <int D>
struct TcCfg {
    static constexpr int kHalves = D / 64;                   // blocks of 64 elements (128 bytes) per row
    static constexpr int kTileBytes = kTcK * D * 2;          // K or V tile, or one half of Q
    static constexpr int kQBytes = 2 * kTileBytes;
    static constexpr int kStages = D == 128 ? 4 : 8;         // K and V tiles take turns
    static constexpr int kOutBytes = 16 * 2048;              // 32 rows x 64 bytes per softmax warp: results on their way out
    static constexpr int kWalkBytes = 16 * 80;                // the softmax warps' walks: they need the registers
    static constexpr int kSmemBytes = kQBytes + kStages * kTileBytes + kOutBytes + 1024 + 384 + kWalkBytes;
};

// Instruction descriptor of kind::f16 with float32 accumulation (see gemm_w4a16.cu), type 1 = bf16, 0 = f16; bit 16: the B
// operand is MN-major
__device__ __forceinline__ uint32_t idesc_f16(int n, bool bf16, bool b_mn) {
    const uint32_t t = bf16 ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// The one thread of a converged warp that issues for it.  The instruction's operands live in uniform registers; under elect.sync
// the compiler knows that a single thread is active, under `lane == 0` it does not and takes several times as long per MMA.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Operand descriptors as two words: the high one is the same for every tile of an operand.
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)acc)
                 : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc, bool acc) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d), "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"((uint32_t)acc)
                 : "memory");
}
// Words of a shared-memory descriptor with 128-byte swizzle and 8-row groups 1024 bytes apart (SBO).  K-major operand: rows of 64
// elements.  MN-major operand (V as it lies): blocks of 64 elements x 8 keys, the next 64 elements `lbo` bytes on.
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return ((saddr & 0x3FFFFu) >> 4) | ((lbo >> 4) << 16); }
// Loads from tensor memory that have arrived when the statement is done: nothing reads the registers earlier.
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
          "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
          "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
          "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
          "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
        "%26,%27,%28,%29,%30,%31};" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
        "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]),
        "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Weights of 16 scores into 8 words, and their sums.  (Taking a part of the exponentials by a polynomial on the multiply-add
// units, and packed pairs of multiply-adds, were measured: 204 us without either on 4 x 2048 causal, 32 heads, 205-219 with.)
template <bool BF16>
__device__ __forceinline__ void weights(const uint32_t* s, uint32_t* out, float scale, float ref, float (&sum)[4]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = exp2_fast(fmaf(__uint_as_float(s[2 * i]), scale, ref)), b = exp2_fast(fmaf(__uint_as_float(s[2 * i + 1]), scale, ref));
        sum[(2 * i) & 3] += a;
        sum[(2 * i + 1) & 3] += b;
        out[i] = pack2(BF16, a, b);
    }
}

// One key tile of an item's part, as every role sees it: t the tile of the item
struct TileKeys {
    bool pre;
    int key0, n;                     // first key, keys in the tile (128 or more: full; 0 or less: none)
};
__device__ __forceinline__ TileKeys tile_keys(const AttnWalk<kTcR, kTcK>& w, int own, int t) {
    TileKeys k;
    k.pre = t < w.prefix_tiles;
    k.key0 = (k.pre ? t : t - w.prefix_tiles) * kTcK;
    k.n = (k.pre ? w.prefix : own) - k.key0;
    return k;
}
// key tiles of [t0, t1) that half h has to see: rows of the first half see fewer of the last keys
__device__ __forceinline__ int half_tiles(const AttnParams& p, const AttnWalk<kTcR, kTcK>& w, int h) {
    if (w.s.n * p.group - w.rt * kTcR <= h * 128) return 0;
    int own = 0;
    if (p.keys != kPrefix) {
        int last = (w.rt * kTcR + (h + 1) * 128 - 1) / p.group;
        if (last > w.s.n - 1) last = w.s.n - 1;
        own = w.s.len - w.s.n + last + 1;
        if (own < 0) own = 0;
    }
    int end = w.prefix_tiles + (own + kTcK - 1) / kTcK;
    if (end > w.t1) end = w.t1;
    return end > w.t0 ? end - w.t0 : 0;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kTcThreads, 1) attn_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                const __grid_constant__ CUtensorMap map_v, const AttnParams p) {
    using C = TcCfg<D>;
    using Walk = AttnWalk<kTcR, kTcK>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    const uint32_t q_s = base, kv_s = base + C::kQBytes, out_s = kv_s + C::kStages * C::kTileBytes, bars = out_s + C::kOutBytes;
    auto kv_full = [&](int s) { return bars + 8u * s; };
    auto kv_empty = [&](int s) { return bars + 8u * (C::kStages + s); };
    const uint32_t more = bars + 16u * C::kStages;
    const uint32_t q_full = more, q_empty = more + 8;
    // the rows behind the last key have been cleared; one per slot, because the ends of the prefix and of a sequence may be
    // in the ring at the same time
    auto v_fixed = [&](int s) { return more + 88 + 8u * s; };
    auto s_full = [&](int h) { return more + 24 + 8u * h; };        // S_h is in tensor memory
    auto p_full = [&](int h) { return more + 40 + 8u * h; };        // P_h is, and O_h may be added to
    auto o_full = [&](int h) { return more + 56 + 8u * h; };        // P_h V has been added
    auto o_empty = [&](int h) { return more + 72 + 8u * h; };       // O_h has been read
    __shared__ AttnStart at;
    __shared__ int64_t sums[kTcThreads / 32];
    __shared__ int abort_word;
    __shared__ uint32_t tmem_word;
    volatile int* abort_flag = &abort_word;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
    if (tid == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(kv_full(s), 1);
            mbar_init(kv_empty(s), 1);
            mbar_init(v_fixed(s), 1);
        }
        mbar_init(q_full, 2);
        mbar_init(q_empty, 1);
        for (int h = 0; h < 2; ++h) {
            mbar_init(s_full(h), 1);
            mbar_init(p_full(h), 8);
            mbar_init(o_full(h), 1);
            mbar_init(o_empty(h), 8);
        }
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 17) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_word)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    MXFP4_CHAIN_PROLOGUE();
    attn_find_start<kTcR, kTcK, kTcThreads>(p, &at, sums);
    tc_fence_after();
    const uint32_t tmem = tmem_word;
    if (p.keys == kAll && tid == 0) p.cut[cta].x = -1;

    Walk w;
    const bool any = attn_begin(p, at, w);
    if (!any) {
        for (int r = tid; r < kTcR; r += kTcThreads) p.slot_lse[(int64_t)(2 * cta) * kTcR + r] = kNegInf;
    } else if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 16) {
            // -------------------------------------------------------------- key and value tiles
            const int box_rows = (1 << p.page_shift) < kTcK ? (1 << p.page_shift) : kTcK, boxes = kTcK / box_rows;
            const int page_mask = (1 << p.page_shift) - 1;
            const int kv = lane >> 4, pg = (lane & 15) / C::kHalves, half = (lane & 15) % C::kHalves;      // 16 lanes each: at most 8 boxes x 2
            uint32_t it = 0;
            bool ok = true;
            do {
                const int own = attn_own_keys<kTcR>(p, w.s, w.rt);
                const int* table = p.table + (int64_t)w.b * p.table_stride;
                for (int t = w.t0; t < w.t1 && ok; ++t) {
                    const TileKeys k = tile_keys(w, own, t);
                    const int issue = k.n <= 0 ? 0 : (k.n >= kTcK ? boxes : (k.n + box_rows - 1) / box_rows);
                    const bool mine = pg < issue;
                    const int key = k.key0 + pg * box_rows;
                    int page = 0;
                    if (mine) {
                        page = (k.pre ? p.prefix_pages : table)[key >> p.page_shift];
                        if ((unsigned)page >= (unsigned)p.num_pages) {       // outside the cache: reported, and read as zeros
                            page = p.num_pages;
                            if (p.status) atomicExch(p.status, MXFP4_E_BADARG);
                        }
                    }
#pragma unroll
                    for (int v = 0; v < 2; ++v, ++it) {
                        const int s = it % C::kStages;
                        ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait(kv_empty(s), ((it / C::kStages) & 1) ^ 1u, abort_flag));
                        if (!ok) break;
                        if (lane == 0) mbar_expect_tx(kv_full(s), (uint32_t)(issue * box_rows * D * 2));
                        __syncwarp();
                        if (mine && kv == v)
                            tma_load_4d(kv_s + s * C::kTileBytes + half * (kTcK * 128) + pg * box_rows * 128, v ? &map_v : &map_k, kv_full(s), half * 64,
                                        key & page_mask, w.h, page);
                    }
                    if (ok && k.n > 0 && k.n < kTcK) {
                        // the rows of V behind the last key: this warp knows the phase its own copies complete, and the ring
                        // holds work for the MMAs meanwhile
                        const int s = (it - 1) % C::kStages;
                        ok = __all_sync(0xFFFFFFFFu, mbar_wait(kv_full(s), ((it - 1) / C::kStages) & 1, abort_flag));
                        if (!ok) break;
                        for (int i = lane; i < (kTcK - k.n) * (D / 8); i += 32) {
                            const int r = k.n + i / (D / 8), ch = i % (D / 8);
                            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(kv_s + s * C::kTileBytes + (ch >> 3) * (kTcK * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)),
                                         "r"(0)
                                         : "memory");
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(v_fixed(s));
                    }
                }
            } while (ok && w.next(p));
        } else if (warp == 17) {
            // -------------------------------------------------------------- MMAs
            // This warp's own instructions lie between one half's weights and its next scores: no division, no look at the
            // walk and no clock inside the loop over the tiles.
            const uint32_t id_s = idesc_f16(kTcK, BF16, false), id_o = idesc_f16(D, BF16, true);
            const uint32_t q_lo = desc_lo(q_s, 16), k_lo = desc_lo(kv_s, 16), v_lo = desc_lo(kv_s, kTcK * 128);
            uint32_t slot = 0, phase = 0, fixes = 0, seen0 = 0, seen1 = 0, live0 = 0, live1 = 0, items = 0;    // phases as parities; fixes: one per slot
            bool ok = true;
            auto wait = [&](uint32_t bar, uint32_t parity) {
                if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) return true;
                return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag)) != 0;
            };
            auto scores = [&](int h, uint32_t sl) {
                if (elect_one()) {
                    const uint32_t a = q_lo + h * (C::kTileBytes >> 4), b = k_lo + sl * (C::kTileBytes >> 4);
#pragma unroll
                    for (int kb = 0; kb < D / 16; ++kb) {
                        constexpr uint32_t kHalf = kTcK * 128;
                        const uint32_t off = ((kb >> 2) * kHalf + (kb & 3) * 32) >> 4;
                        tc_mma_ss(tmem + h * 128, a + off, b + off, kDescHi, id_s, kb > 0);
                    }
                    tc_commit(s_full(h));
                }
                __syncwarp();
            };
            // P_h V of a tile
            auto values = [&](int h, uint32_t sl, bool first, uint32_t& seen, uint32_t& live) {
                if (!wait(p_full(h), seen)) return false;
                seen ^= 1u;
                if (first) {
                    if (!wait(o_empty(h), live ^ 1u)) return false;
                    live ^= 1u;
                }
                tc_fence_after();
                const uint32_t b = v_lo + sl * (C::kTileBytes >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int kb = 0; kb < kTcK / 16; ++kb) tc_mma_ts(tmem + 256 + h * D, tmem + h * 128 + kb * 8, b + (kb * 2048 >> 4), kDescHi, id_o, !first || kb > 0);
                    tc_commit(o_full(h));
                }
                __syncwarp();
                return true;
            };
            auto release = [&](uint32_t bar) {
                if (elect_one()) tc_commit(bar);
                __syncwarp();
            };
            do {
                const int own = attn_own_keys<kTcR>(p, w.s, w.rt), T = w.t1 - w.t0;
                const int n0 = half_tiles(p, w, 0), n1 = half_tiles(p, w, 1), most = n0 > n1 ? n0 : n1;
                // the tiles that end inside: the prefix's last and the sequence's last (of this item)
                const int ends0 = (w.prefix & (kTcK - 1)) ? w.prefix_tiles - 1 - w.t0 : -1;
                const int ends1 = (own & (kTcK - 1)) ? w.prefix_tiles + own / kTcK - w.t0 : -1;
                ok = wait(q_full, items) && wait(kv_full(slot), phase);
                if (!ok) break;
                items ^= 1u;
                tc_fence_after();
                if (n0 > 0) scores(0, slot);
                if (n1 > 0) scores(1, slot);
                release(kv_empty(slot));
                if (most <= 1) release(q_empty);
                for (int j = 0; j < T; ++j) {
                    if (++slot == C::kStages) { slot = 0; phase ^= 1u; }
                    const uint32_t sv = slot;
                    ok = wait(kv_full(sv), phase);
                    if (ok && (j == ends0 || j == ends1)) {
                        ok = wait(v_fixed(sv), (fixes >> sv) & 1);
                        fixes ^= 1u << sv;
                    }
                    if (++slot == C::kStages) { slot = 0; phase ^= 1u; }
                    if (ok && j + 1 < T) ok = wait(kv_full(slot), phase);     // before the weights: not on their way to the next scores
                    if (ok && j < n0) ok = values(0, sv, j == 0, seen0, live0);
                    if (!ok) break;
                    if (j + 1 < n0) scores(0, slot);
                    if (j < n1) ok = values(1, sv, j == 0, seen1, live1);
                    if (!ok) break;
                    if (j + 1 < n1) scores(1, slot);
                    release(kv_empty(sv));
                    if (j + 1 < T) release(kv_empty(slot));
                    if (most > 1 && j + 2 == most) release(q_empty);
                }
            } while (ok && w.next(p));
        } else {
            // -------------------------------------------------------------- query rows
            const int t64 = tid - 576;                                       // 0..63
            constexpr int kChunks = D / 8;
            uint32_t items = 0;
            bool ok = true;
            do {
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(q_empty, (items & 1) ^ 1u, abort_flag));
                if (!ok) break;
                if (p.q_box) {
                    // a half is a whole number of tokens: one copy per half and 64 elements.  Rows behind the sequence hold other
                    // sequences' queries or, behind the last token, zeros; nothing of theirs is stored.
                    if (t64 == 0) {
                        mbar_expect_tx(q_full, C::kQBytes);
#pragma unroll
                        for (int i = 0; i < 2 * C::kHalves; ++i)
                            tma_load_4d(q_s + (i / C::kHalves) * C::kTileBytes + (i % C::kHalves) * (128 * 128), &map_q, q_full, (i % C::kHalves) * 64, 0, w.h,
                                        w.s.start + (w.rt * 2 + i / C::kHalves) * p.q_box);
                    }
                    if (t64 == 32) mbar_arrive(q_full);
                    __syncwarp();
                    ++items;
                    continue;
                }
                const int rows = w.s.n * p.group - w.rt * kTcR;
                const int c = t64 % kChunks;
                const uint32_t col = (c >> 3) * (128 * 128), cc = c & 7;
                for (int r = t64 / kChunks; r < kTcR; r += 64 / kChunks) {
                    const int lr = w.rt * kTcR + r, t = lr / p.group, g = lr - t * p.group;
                    const bool in = r < rows;
                    const uint16_t* src = (const uint16_t*)p.q + (in ? (int64_t)(w.s.start + t) * p.q_row + (int64_t)(w.h * p.group + g) * p.q_head + c * 8 : 0);
                    const int rr = r & 127;
                    const uint32_t dst = q_s + (r >> 7) * C::kTileBytes + col + rr * 128 + ((cc ^ (rr & 7)) << 4);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
                ++items;
            } while (ok && w.next(p));
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        // ------------------------------------------------------------------ softmax and results, two threads per row
        const int h = warp >> 3, part = (warp >> 2) & 1, r = h * 128 + (warp & 3) * 32 + lane;     // part: which 64 keys; r: row of the tile
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + h * 128 + part * 64 + lanes, tp = tmem + h * 128 + part * 32 + lanes, to = tmem + 256 + h * D + part * (D / 2) + lanes;
        const int pair_bar = 1 + h * 4 + (warp & 3);                         // the two warps of 32 rows
        auto pair_any = [&](bool x) {
            uint32_t any_of;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                         : "=r"(any_of) : "r"((uint32_t)x), "r"(pair_bar) : "memory");
            return any_of != 0;
        };
        auto pair_sync = [&]() { asm volatile("barrier.cta.sync %0, 64;" ::"r"(pair_bar) : "memory"); };
        // (A wait that ran out is told to the other warp in the same way: neither is left behind at a barrier.)
        // the other thread's value, by way of the space where results leave
        auto swap = [&](float x) {
            float y;
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(out_s + warp * 2048 + lane * 4), "f"(x) : "memory");
            pair_sync();
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(out_s + (warp ^ 4) * 2048 + lane * 4) : "memory");
            pair_sync();
            return y;
        };
        uint32_t c = 0;                                                      // tiles this half has seen
        bool ok = true, more = true;
        const Walk start = w;
        Walk& w = *reinterpret_cast<Walk*>(smem_raw + (bars - raw) + 384 + warp * 80);
        static_assert(sizeof(Walk) <= 80 && 3 * 8 * C::kStages + 88 <= 384, "room");
        if (lane == 0) w = start;
        __syncwarp();
        do {
            const int rows = w.s.n * p.group - w.rt * kTcR;
            const int n = half_tiles(p, w, h), lr = w.rt * kTcR + r, tok = lr / p.group, head = w.h * p.group + lr - tok * p.group;
            const int lim = w.s.len - w.s.n + tok + 1, t0 = w.t0, prefix = w.prefix, prefix_tiles = w.prefix_tiles;
            const bool in = r < rows;
            float m = kNegInf, l = 0.0f;                                     // m: reference of the weights, times scale_log2; l: of this thread's keys
            for (int j = 0; j < n; ++j, ++c) {
                const int t = t0 + j;
                const bool pre = t < prefix_tiles;
                const int key0 = (pre ? t : t - prefix_tiles) * kTcK + part * 64, end = (pre ? prefix : lim) - key0;
                ok = !pair_any(!mbar_wait(s_full(h), c & 1, abort_flag));
                if (!ok) break;
                tc_fence_after();
                uint32_t a[16], out[32];                                     // scores, weights packed
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const bool masked = __any_sync(0xFFFFFFFFu, end < 64);
                bool high = j == 0;
                if (j > 0) {
                    // In the hope that the tile raises no maximum by much, its weights are taken against the old one at once; where
                    // their sum says otherwise all is done again below.
                    const float ref = m == kNegInf ? 0.0f : -m;
                    if (!masked) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            tc_ld16(ts + q * 16, a);
                            weights<BF16>(a, out + q * 8, p.scale_log2, ref, sum);
                        }
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            tc_ld16(ts + q * 16, a);
#pragma unroll
                            for (int i = 0; i < 16; ++i) a[i] = q * 16 + i < end ? a[i] : __float_as_uint(kNegInf);
                            weights<BF16>(a, out + q * 8, p.scale_log2, ref, sum);
                        }
                    }
                    high = !((sum[0] + sum[1]) + (sum[2] + sum[3]) <= (m == kNegInf ? 0.0f : kHigh));
                }
                if (pair_any(high)) {
                    float top = kNegInf;
#pragma unroll 1
                    for (int q = 0; q < 64; q += 16) {
                        tc_ld16(ts + q, a);
#pragma unroll
                        for (int i = 0; i < 16; ++i) top = fmaxf(top, q + i < end ? __uint_as_float(a[i]) : kNegInf);
                    }
                    const float mt = fmaxf(top, swap(top)) * p.scale_log2;
                    const float nm = fmaxf(m, mt), f = nm == kNegInf ? 1.0f : exp2_fast(m - nm);
                    m = nm;
                    l *= f;
                    if (j > 0) {
                        ok = !pair_any(!mbar_wait(o_full(h), (c - 1) & 1, abort_flag));
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int i = 0; i < D / 2; i += 32) {
                            tc_ld32(to + i, out);
#pragma unroll
                            for (int e = 0; e < 32; ++e) out[e] = __float_as_uint(__uint_as_float(out[e]) * f);
                            tc_st32(to + i, out);
                        }
                    }
                    const float ref = m == kNegInf ? 0.0f : -m;              // nothing seen yet: every weight is 2^-inf = 0
                    sum[0] = sum[1] = sum[2] = sum[3] = 0.0f;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        tc_ld16(ts + q * 16, a);
#pragma unroll
                        for (int i = 0; i < 16; ++i) a[i] = q * 16 + i < end ? a[i] : __float_as_uint(kNegInf);
                        weights<BF16>(a, out + q * 8, p.scale_log2, ref, sum);
                    }
                    pair_sync();                                             // both have read their scores: weights may take their place
                }
                tc_st32(tp, out);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(h));
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            }
            if (!ok) break;
            l += swap(l);

            // ---------------------------------------------------------------- the item's (or the part's) result
            const bool first = w.t0 == 0, whole = first && w.t1 == w.tiles;
            const int64_t slot = first ? 2 * cta + 1 : 2 * cta, at_row = (int64_t)(w.s.start + tok) * p.heads + head;
            int c_end = cta;
            if (first && !whole) c_end = attn_cta_of(w.last_unit(at.w1), at.total);
            if (p.keys == kAll && first && !whole && tid == 0)
                p.cut[cta] = make_int4(c_end, w.s.start, w.rt * kTcR, (w.h << 9) | (rows < kTcR ? rows : kTcR));
            const float inv = l == 0.0f ? 0.0f : 1.0f / l, lse2 = l == 0.0f ? kNegInf : m + log2f(l);
            if (in && part == 0) {
                if (whole && p.keys == kAll) {
                    if (p.lse) p.lse[at_row] = lse2 * kLn2;
                } else if (whole) {
                    p.rows_lse[at_row] = lse2;
                } else {
                    p.slot_lse[slot * kTcR + r] = lse2;
                }
                if (p.keys != kAll && first) p.rows_seg[at_row] = whole ? make_int2(-1, -1) : make_int2(cta, c_end);
            }
            if (n > 0) {
                ok = !pair_any(!mbar_wait(o_full(h), (c - 1) & 1, abort_flag));
                if (!ok) break;
                tc_fence_after();
            }
            // Rows leave by way of shared memory: a thread has (half) a row, but a store of 32 rows' pieces costs 32 cycles where one
            // of eight 64-byte pieces costs eight.
            const bool final = whole && p.keys == kAll;
            const uint64_t mine = !in ? 0 : final ? (uint64_t)((uint16_t*)p.out + (int64_t)(w.s.start + tok) * p.out_row + (int64_t)head * p.out_head + part * (D / 2))
                                                  : (uint64_t)((whole ? p.rows_o + at_row * D : p.slot_o + (slot * kTcR + r) * D) + part * (D / 2));
            const uint32_t stage = out_s + warp * 2048;
            auto put = [&](const uint32_t* v, int byte) {                     // 64 bytes of this thread's row, `byte` into its part
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)), "r"(v[4 * i]), "r"(v[4 * i + 1]),
                                 "r"(v[4 * i + 2]), "r"(v[4 * i + 3])
                                 : "memory");
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = i * 8 + (lane >> 2), ch = lane & 3;
                    uint4 x;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(stage + row * 64 + ((ch ^ ((row >> 1) & 3)) << 4)) : "memory");
                    const uint64_t dst = __shfl_sync(0xFFFFFFFFu, mine, row);
                    if (dst) *reinterpret_cast<uint4*>(dst + byte + ch * 16) = x;
                }
                __syncwarp();
            };
#pragma unroll 1
            for (int i = 0; i < D / 2; i += 32) {
                uint32_t o[32];
                if (n > 0) tc_ld32(to + i, o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = n > 0 ? __float_as_uint(__uint_as_float(o[e]) * inv) : 0u;
                if (final) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = pack2(BF16, __uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
                    put(o, i * 2);
                } else {
                    put(o, i * 4);
                    put(o + 16, i * 4 + 64);
                }
            }
            if (n > 0) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(o_empty(h));
            }
            __syncwarp();
            if (lane == 0) more = w.next(p);
            more = __shfl_sync(0xFFFFFFFFu, more, 0);
            __syncwarp();
        } while (more);
    }

    // ---------------------------------------------------------------------- teardown
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        // a wait ran out: reported, and copies and MMAs in flight retire before tensor and shared memory are given back
        if (tid == 0) {
            if (p.status) atomicExch(p.status, MXFP4_E_TIMEOUT);
            for (int i = 0; i < 2000; ++i) __nanosleep(1000);
        }
        __syncthreads();
    }
    if (warp == 17) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int D, bool BF16>
int launch_tc(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const AttnParams& p, int grid, cudaStream_t st) {
    using C = TcCfg<D>;
    static_assert(C::kSmemBytes <= 227 * 1024, "shared memory");
    static std::atomic<bool> configured[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(attn_tc_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
        if (e != cudaSuccess) return cuda_fail(e, "mxfp4_paged_attention: cudaFuncSetAttribute");
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    const cudaError_t e = launch_smem(attn_tc_kernel<D, BF16>, (unsigned)grid, kTcThreads, (size_t)C::kSmemBytes, st, mq, mk, mv, p);
    if (e != cudaSuccess) return cuda_fail(e, "mxfp4_paged_attention");
    return MXFP4_OK;
}

}  // namespace

int launch_attn_tc(int head_dim, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const AttnParams& p, int grid, cudaStream_t st) {
    if (head_dim == 64) return p.bf16 ? launch_tc<64, true>(mq, mk, mv, p, grid, st) : launch_tc<64, false>(mq, mk, mv, p, grid, st);
    return p.bf16 ? launch_tc<128, true>(mq, mk, mv, p, grid, st) : launch_tc<128, false>(mq, mk, mv, p, grid, st);
}

}  // namespace mxfp4
