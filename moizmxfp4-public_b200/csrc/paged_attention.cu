// Attention over a paged key/value cache: the kernel for few rows (decode), the kernels that join partial results, and the
// C-ABI entry.  What is computed and how the work is divided stands in paged_attention.cuh.
//
// Row tiles of 256 rows go to paged_attention_tc.cu.
//
// attn_rows_kernel<D, RW>: HBM-bound, one query token per sequence reads every key and value once for a handful of rows.
// A producer warp brings tiles of 64 keys (K and V, page by page through 4-D tensor maps whose box is a page or a part of
// one) into a ring; four warps take them from there with mma.sync m16n8k16: the tensor work of such a tile is a tenth of
// the time its bytes take, so the accumulators stay in registers and nothing is gained by tensor memory here.  RW = 1: 16
// rows, every warp takes 16 of the tile's keys with statistics of its own, joined when the item ends; RW = 4: 64 rows,
// every warp takes 16 of them and all keys.  Scores, statistics and sums are float32; the weights are rounded to the
// cache's type for the product with V (they are at most 1 and their sum is taken before the rounding).
#include <atomic>
#include <initializer_list>

#include "paged_attention.cuh"

namespace mxfp4 {
namespace {

constexpr int kRowsThreads = 160;        // warps 0-3 compute, warp 4 loads
constexpr int kRowsKeys = 64;            // keys per tile

template <int D, int RW>
struct RowsCfg {
    static constexpr int kR = 16 * RW;
    static constexpr int kRowBytes = D * 2 > 128 ? 128 : D * 2;              // bytes of a key per block of the swizzled tile
    static constexpr int kHalves = D * 2 / kRowBytes;
    static constexpr int kTileBytes = kRowsKeys * D * 2;                     // K or V
    static constexpr int kStageBytes = 2 * kTileBytes;
    static constexpr int kStages = D == 128 ? 3 : (D == 64 ? 6 : 10);        // two CTAs per SM
    static constexpr int kJoinBytes = 4 * 16 * (D / 4) * 4 + 4 * 16 * 8;     // RW = 1: a quarter of every warp's result, its statistics
    static constexpr int kSmemBytes = kStages * kStageBytes + kJoinBytes + 1024 + 512;
};

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D, int RW, bool BF16>
__global__ void __launch_bounds__(kRowsThreads, 2) attn_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                    const AttnParams p) {
    using C = RowsCfg<D, RW>;
    constexpr int R = C::kR, K = kRowsKeys, KW = 4 / RW, KB = 4 / KW;       // KB: blocks of 16 keys per warp and tile
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - raw);
    float* join = reinterpret_cast<float*>(base_ptr + C::kStages * C::kStageBytes);
    float2* join_ml = reinterpret_cast<float2*>(join + 4 * 16 * (D / 4));
    const uint32_t bars = base + C::kStages * C::kStageBytes + C::kJoinBytes;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (C::kStages + s); };
    __shared__ AttnStart at;
    __shared__ int64_t sums[kRowsThreads / 32];
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 4);
        }
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    MXFP4_CHAIN_PROLOGUE();
    attn_find_start<R, K, kRowsThreads>(p, &at, sums);
    const int cta = blockIdx.x;
    if (p.keys == kAll && tid == 0) p.cut[cta].x = -1;

    AttnWalk<R, K> w;
    if (!attn_begin(p, at, w)) {
        // nothing to do: whoever joins an item that runs past this CTA finds an empty part
        if (tid < R) p.slot_lse[(int64_t)(2 * cta) * R + tid] = kNegInf;
        return;
    }

    if (warp == 4) {
        // ------------------------------------------------------------------ producer
        const int box_rows = (1 << p.page_shift) < K ? (1 << p.page_shift) : K, boxes = K / box_rows;
        const int per = boxes * C::kHalves;
        const int kv = lane / per, half = lane % C::kHalves, pg = (lane % per) / C::kHalves;
        const int page_mask = (1 << p.page_shift) - 1;
        uint32_t it = 0;
        bool ok = true;
        do {
            const int own = attn_own_keys<R>(p, w.s, w.rt);
            for (int t = w.t0; t < w.t1 && ok; ++t, ++it) {
                const bool pre = t < w.prefix_tiles;
                const int key0 = (pre ? t : t - w.prefix_tiles) * K, n = (pre ? w.prefix : own) - key0;
                const int* pages = pre ? p.prefix_pages : p.table + (int64_t)w.b * p.table_stride;
                const int issue = n <= 0 ? 0 : (n >= K ? boxes : (n + box_rows - 1) / box_rows);
                const bool mine = kv < 2 && pg < issue;
                const int key = key0 + pg * box_rows;
                int page = 0;
                if (mine) {
                    page = pages[key >> p.page_shift];
                    if ((unsigned)page >= (unsigned)p.num_pages) {           // outside the cache: reported, and read as zeros
                        page = p.num_pages;
                        if (p.status) atomicExch(p.status, MXFP4_E_BADARG);
                    }
                }
                const int s = it % C::kStages;
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(empty_bar(s), ((it / C::kStages) & 1) ^ 1u, abort_flag));
                if (!ok) break;
                if (lane == 0) mbar_expect_tx(full_bar(s), (uint32_t)(issue * box_rows * D * 2 * 2));
                __syncwarp();
                if (mine)
                    tma_load_4d(base + s * C::kStageBytes + kv * C::kTileBytes + half * (K * C::kRowBytes) + pg * box_rows * C::kRowBytes, kv ? &map_v : &map_k,
                                full_bar(s), half * 64, key & page_mask, w.h, page);
            }
        } while (ok && w.next(p));
    } else {
        // ------------------------------------------------------------------ consumers
        const int rw = RW == 1 ? 0 : warp, kw = RW == 1 ? warp : 0;
        const int r0 = rw * 16 + (lane >> 2), mat = lane >> 3;
        uint32_t it = 0;
        bool ok = true;
        // A warp whose wait ran out takes the same steps as the others, without computing, up to the next barrier of the four, where
        // all learn of it: none is left behind at one.
        auto all_ok = [&](bool mine) {
            uint32_t lost;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.eq.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(lost) : "r"((uint32_t)mine) : "memory");
            return lost == 0;
        };
        auto chunk_addr = [&](uint32_t tile, int row, int c) {
            if (D >= 64) return tile + (c >> 3) * (K * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
            return tile + row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
        };
        do {
            const int rows = w.s.n * p.group - w.rt * R;                     // of the item, may exceed R
            const int own = attn_own_keys<R>(p, w.s, w.rt);
            // this thread's two rows
            int lim[2];
            int64_t q_off[2];
            bool there[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = r0 + 8 * i, lr = w.rt * R + r;
                there[i] = r < rows;
                const int t = lr / p.group, g = lr - t * p.group;
                lim[i] = w.s.len - w.s.n + t + 1;
                q_off[i] = (int64_t)(w.s.start + t) * p.q_row + (int64_t)(w.h * p.group + g) * p.q_head;
            }
            uint32_t qf[D / 16][4];
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = kk * 16 + (i >> 1) * 8 + (lane & 3) * 2;
                    qf[kk][i] = there[i & 1] ? *reinterpret_cast<const uint32_t*>((const uint16_t*)p.q + q_off[i & 1] + d) : 0u;
                }
            float o[D / 8][4];
#pragma unroll
            for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
            float m[2] = {kNegInf, kNegInf}, l[2] = {0.0f, 0.0f};

            for (int t = w.t0; t < w.t1; ++t, ++it) {
                const bool pre = t < w.prefix_tiles;
                const int key0 = (pre ? t : t - w.prefix_tiles) * K, n = (pre ? w.prefix : own) - key0;
                const int s = it % C::kStages;
                ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait(full_bar(s), (it / C::kStages) & 1, abort_flag));
                const uint32_t tk = base + s * C::kStageBytes, tv = tk + C::kTileBytes;
                if (n < K) {
                    // values behind the last key weigh nothing, but what lies there may be anything: zeros instead
                    const int from = n < 0 ? 0 : n;
                    for (int i = tid; i < (K - from) * (D / 8); i += 128)
                        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(chunk_addr(tv, from + i / (D / 8), i % (D / 8))), "r"(0) : "memory");
                    ok = all_ok(ok);
                    if (!ok) break;
                }
                if (ok && n > kw * 16) {
                    float c[2 * KB][4];
#pragma unroll
                    for (int i = 0; i < 2 * KB; ++i) c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0.0f;
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                        for (int kb = 0; kb < KB; ++kb) {
                            uint32_t b[4];
                            ldsm_x4(chunk_addr(tk, (kw * KB + kb) * 16 + (mat >> 1) * 8 + (lane & 7), 2 * kk + (mat & 1)), b);
                            mma_16816<BF16>(c[2 * kb], qf[kk], b[0], b[1]);
                            mma_16816<BF16>(c[2 * kb + 1], qf[kk], b[2], b[3]);
                        }
                    float top[2] = {kNegInf, kNegInf};
#pragma unroll
                    for (int nt = 0; nt < 2 * KB; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = key0 + kw * KB * 16 + nt * 8 + (lane & 3) * 2 + (i & 1);
                            const float v = c[nt][i] * p.scale_log2;
                            c[nt][i] = key < (pre ? w.prefix : lim[i >> 1]) ? v : kNegInf;
                            top[i >> 1] = fmaxf(top[i >> 1], c[nt][i]);
                        }
                    float alpha[2], ref[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 1));
                        top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 2));
                        const float nm = fmaxf(m[i], top[i]);
                        ref[i] = nm == kNegInf ? 0.0f : nm;                  // nothing seen yet: every weight is 2^-inf = 0
                        alpha[i] = exp2_fast(m[i] - ref[i]);
                        m[i] = nm;
                        l[i] *= alpha[i];
                    }
#pragma unroll
                    for (int nt = 0; nt < 2 * KB; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            c[nt][i] = exp2_fast(c[nt][i] - ref[i >> 1]);
                            l[i >> 1] += c[nt][i];
                        }
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        o[i][0] *= alpha[0]; o[i][1] *= alpha[0]; o[i][2] *= alpha[1]; o[i][3] *= alpha[1];
                    }
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) {
                        const uint32_t a[4] = {pack2(BF16, c[2 * kb][0], c[2 * kb][1]), pack2(BF16, c[2 * kb][2], c[2 * kb][3]),
                                               pack2(BF16, c[2 * kb + 1][0], c[2 * kb + 1][1]), pack2(BF16, c[2 * kb + 1][2], c[2 * kb + 1][3])};
#pragma unroll
                        for (int dc = 0; dc < D / 8; dc += 2) {
                            uint32_t b[4];
                            ldsm_x4_t(chunk_addr(tv, (kw * KB + kb) * 16 + (mat & 1) * 8 + (lane & 7), dc + (mat >> 1)), b);
                            mma_16816<BF16>(o[dc], a, b[0], b[1]);
                            mma_16816<BF16>(o[dc + 1], a, b[2], b[3]);
                        }
                    }
                }
                if (n < K) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the zeros, before the next copy into this slot
                __syncwarp();
                if (lane == 0) mbar_arrive(empty_bar(s));
            }
            ok = all_ok(ok);
            if (!ok) break;

            // ---------------------------------------------------------------- the item's (or the part's) result
            const bool first = w.t0 == 0, last = w.t1 == w.tiles;
            const bool whole = first && last;
            const int64_t slot = first ? 2 * cta + 1 : 2 * cta;
            int c_end = cta;
            if (first && !last) c_end = attn_cta_of(w.last_unit(at.w1), at.total);
            if (p.keys == kAll && first && !last && tid == 0)
                p.cut[cta] = make_int4(c_end, w.s.start, w.rt * R, (w.h << 9) | (rows < R ? rows : R));
            // writes elements [d, d + N) of row r (of the tile): v normalised, lse2 the base-2 log of the row's sum
            auto put = [&](int r, int d, const float* v, int N) {
                const int lr = w.rt * R + r, t = lr / p.group, hd = w.h * p.group + lr - t * p.group;
                if (whole && p.keys == kAll) {
                    uint16_t* dst = (uint16_t*)p.out + (int64_t)(w.s.start + t) * p.out_row + (int64_t)hd * p.out_head + d;
                    if (N == 1) { *dst = (uint16_t)pack2(BF16, v[0], 0.0f); return; }
                    for (int i = 0; i < N; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack2(BF16, v[i], v[i + 1]);
                } else {
                    float* dst = whole ? p.rows_o + ((int64_t)(w.s.start + t) * p.heads + hd) * D + d : p.slot_o + (slot * R + r) * D + d;
                    for (int i = 0; i < N; ++i) dst[i] = v[i];
                }
            };
            auto put_lse = [&](int r, float lse2) {
                const int lr = w.rt * R + r, t = lr / p.group, hd = w.h * p.group + lr - t * p.group;
                const int64_t at_row = (int64_t)(w.s.start + t) * p.heads + hd;
                if (whole && p.keys == kAll) {
                    if (p.lse) p.lse[at_row] = lse2 * kLn2;
                } else if (whole) {
                    p.rows_lse[at_row] = lse2;
                } else {
                    p.slot_lse[slot * R + r] = lse2;
                }
                if (p.keys != kAll && first) p.rows_seg[at_row] = whole ? make_int2(-1, -1) : make_int2(cta, c_end);
            };
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 1);
                l[i] += __shfl_xor_sync(0xFFFFFFFFu, l[i], 2);
            }
            if (RW == 1) {
                if ((lane & 3) == 0) {
                    join_ml[warp * 16 + r0] = make_float2(m[0], l[0]);
                    join_ml[warp * 16 + r0 + 8] = make_float2(m[1], l[1]);
                }
                const int jr = tid >> 3, jc = (tid & 7) * (D / 32);          // this thread's row and columns of each quarter
                float wt[4], sum = 0.0f, top = kNegInf;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const int nt = q * (D / 32) + i;
                        float* dst = join + (warp * 16 + r0) * (D / 4) + i * 8 + (lane & 3) * 2;
                        *reinterpret_cast<float2*>(dst) = make_float2(o[nt][0], o[nt][1]);
                        *reinterpret_cast<float2*>(dst + 8 * (D / 4)) = make_float2(o[nt][2], o[nt][3]);
                    }
                    asm volatile("bar.sync 1, 128;" ::: "memory");
                    if (q == 0) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) top = fmaxf(top, join_ml[i * 16 + jr].x);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 ml = join_ml[i * 16 + jr];
                            wt[i] = ml.x == kNegInf ? 0.0f : exp2_fast(ml.x - top);
                            sum += wt[i] * ml.y;
                        }
                        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;   // a row that sees nothing: zeros
#pragma unroll
                        for (int i = 0; i < 4; ++i) wt[i] *= inv;
                    }
                    float v[D / 32];
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        v[i] = 0.0f;
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[i] += wt[k] * join[(k * 16 + jr) * (D / 4) + jc + i];
                    }
                    if (jr < rows) put(jr, q * (D / 4) + jc, v, D / 32);
                    asm volatile("bar.sync 1, 128;" ::: "memory");
                }
                if (jr < rows && (tid & 7) == 0) put_lse(jr, sum == 0.0f ? kNegInf : top + log2f(sum));
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = r0 + 8 * i;
                    if (r < rows) {
                        const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
#pragma unroll
                        for (int nt = 0; nt < D / 8; ++nt) {
                            const float v[2] = {o[nt][2 * i] * inv, o[nt][2 * i + 1] * inv};
                            put(r, nt * 8 + (lane & 3) * 2, v, 2);
                        }
                        if ((lane & 3) == 0) put_lse(r, l[i] == 0.0f ? kNegInf : m[i] + log2f(l[i]));
                    }
                }
            }
        } while (w.next(p));
    }
    if (*abort_flag) {
        // a wait ran out: reported, and copies in flight land before the block's shared memory is given back
        if (lane == 0 && p.status) atomicExch(p.status, MXFP4_E_TIMEOUT);
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    }
}

// ---------------------------------------------------------------------------------------------- joining the parts
// A warp adds one row's parts: o = sum w_i o_i / sum w_i with w_i = 2^(lse_i - max).  Lane i brings part i (up to 32 at a time), so
// that all loads of a row are under way at once; then lane holds D / 32 elements of the sum.
template <int D>
struct RowSum {
    float top, sum, v[D / 32];
    __device__ __forceinline__ void init() {
        top = kNegInf; sum = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) v[i] = 0.0f;
    }
    // n parts; lane i < n has part i's base-2 log-sum (-inf: empty, its elements mean nothing) and its elements
    __device__ __forceinline__ void add(int n, float lse2, const float* o, int lane) {
        float mx = lse2;
#pragma unroll
        for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, d));
        const float nt = fmaxf(top, mx);
        if (nt == kNegInf) return;
        const float a = top == kNegInf ? 0.0f : exp2_fast(top - nt), w = lse2 == kNegInf ? 0.0f : exp2_fast(lse2 - nt);
        float all = w;
#pragma unroll
        for (int d = 16; d; d >>= 1) all += __shfl_xor_sync(0xFFFFFFFFu, all, d);
        top = nt;
        sum = sum * a + all;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) v[i] *= a;
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
            const float wk = __shfl_sync(0xFFFFFFFFu, w, k);
            const float* ok = (const float*)__shfl_sync(0xFFFFFFFFu, (unsigned long long)o, k);
            float x[D / 32];
            if (D == 128) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(ok + lane * 4);
            else if (D == 64) *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(ok + lane * 2);
            else x[0] = ok[lane];
#pragma unroll
            for (int i = 0; i < D / 32; ++i) v[i] += wk > 0.0f ? wk * x[i] : 0.0f;
        }
    }
    __device__ __forceinline__ void put(const AttnParams& p, int64_t token, int head, int lane) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        uint16_t* dst = (uint16_t*)p.out + token * p.out_row + (int64_t)head * p.out_head + lane * (D / 32);
        if (D == 32) *dst = (uint16_t)pack2(p.bf16, v[0] * inv, 0.0f);
        else
#pragma unroll
            for (int i = 0; i + 1 < D / 32; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack2(p.bf16, v[i] * inv, v[i + 1] * inv);
        if (lane == 0 && p.lse) p.lse[token * p.heads + head] = sum == 0.0f ? kNegInf : (top + log2f(sum)) * kLn2;
    }
};

// zeros (and a log-sum of -inf) for the query rows that belong to no sequence, where the caller asked for it
template <int D>
__device__ __forceinline__ void fill_rest(const AttnParams& p, int warps_of_block) {
    const int first = p.starts[0], end = p.starts[p.batch];
    const int64_t step = (int64_t)gridDim.x * gridDim.y * warps_of_block;
    const int64_t before = first < 0 ? 0 : (first > p.tokens ? p.tokens : first), behind = end < 0 ? 0 : (end > p.tokens ? p.tokens : end);
    const int64_t n = (before + (p.tokens > behind ? p.tokens - behind : 0)) * p.heads;
    RowSum<D> z;
    z.init();
    for (int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * warps_of_block + (threadIdx.x >> 5); i < n; i += step) {
        const int64_t t = i / p.heads;
        z.put(p, t < before ? t : behind + (t - before), (int)(i % p.heads), threadIdx.x & 31);
    }
}

// kAll: blocks (c, y) join the item that began in CTA c of the main launch and went on behind it
template <int D>
__global__ void __launch_bounds__(256) attn_join_cut_kernel(const AttnParams p, int R, int rest) {
    MXFP4_CHAIN_PROLOGUE();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x;
    const int4 cut = p.cut[c];
    if (cut.x >= 0) {
        const int h = cut.w >> 9, rows = cut.w & 511;
        for (int r = blockIdx.y * 8 + warp; r < rows; r += 8 * gridDim.y) {
            RowSum<D> a;
            a.init();
            for (int first = c; first <= cut.x; first += 32) {
                const int n = cut.x - first + 1 < 32 ? cut.x - first + 1 : 32, i = first + lane;
                const int64_t at = (int64_t)(i == c ? 2 * i + 1 : 2 * i) * R + r;
                a.add(n, lane < n ? p.slot_lse[at] : kNegInf, p.slot_o + (lane < n ? at : (int64_t)r) * D, lane);
            }
            const int lr = cut.z + r, t = lr / p.group;
            a.put(p, cut.y + t, h * p.group + lr - t * p.group, lane);
        }
    }
    if (rest) fill_rest<D>(p, 8);
}

struct AttnPart {                    // what a kOwn or kPrefix launch left
    const float *slot_o, *slot_lse, *rows_o, *rows_lse;
    const int2* seg;
    int R, grid;
};
// Number of parts that a launch left of a row, and part i of them.
__device__ __forceinline__ int part_count(const AttnPart& s, int2 g) { return g.x == -1 ? 1 : (g.x < 0 || g.y < g.x || g.y >= s.grid ? 0 : g.y - g.x + 1); }
template <int D>
__device__ __forceinline__ float part_at(const AttnPart& s, int2 g, int i, int64_t row, int r, const float*& o) {
    const int64_t at = (int64_t)(i == 0 ? 2 * g.x + 1 : 2 * (g.x + i)) * s.R + r;
    o = g.x == -1 ? s.rows_o + row * D : s.slot_o + at * D;
    return g.x == -1 ? s.rows_lse[row] : s.slot_lse[at];
}

// kOwn and kPrefix results of every row: a warp per (token, head)
template <int D>
__global__ void __launch_bounds__(256) attn_join_rows_kernel(const AttnParams p, const AttnPart own, const AttnPart pre, int rest) {
    MXFP4_CHAIN_PROLOGUE();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row < (int64_t)p.tokens * p.heads) {
        const int token = (int)(row / p.heads), head = (int)(row - (int64_t)token * p.heads), g = head % p.group;
        // the row's sequence: its place within its row tile
        int first = token;
        bool there = true;
        if (p.starts) {
            int lo = 0, hi = p.batch;                                         // the last b with starts[b] <= token
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (p.starts[mid + 1] <= token) lo = mid + 1;
                else hi = mid;
            }
            there = lo < p.batch && p.starts[lo] <= token;
            first = there ? p.starts[lo] : 0;
            if (first < 0) first = 0;
        }
        if (there) {
            RowSum<D> a;
            a.init();
            const int r_own = (int)(((int64_t)(token - first) * p.group + g) % own.R), r_pre = (int)(((int64_t)token * p.group + g) % pre.R);
            const bool prefix = *p.prefix_len > 0 && p.prefix_table_pages > 0;
            const int2 s_own = own.seg[row], s_pre = prefix ? pre.seg[row] : make_int2(-2, -2);
            const int n_own = part_count(own, s_own), n = n_own + part_count(pre, s_pre);
            for (int i0 = 0; i0 < n; i0 += 32) {
                const int i = i0 + lane;
                const float* o = own.rows_o;
                float lse2 = kNegInf;
                if (i < n_own) lse2 = part_at<D>(own, s_own, i, row, r_own, o);
                else if (i < n) lse2 = part_at<D>(pre, s_pre, i - n_own, row, r_pre, o);
                a.add(n - i0 < 32 ? n - i0 : 32, lse2, o, lane);
            }
            a.put(p, token, head, lane);
        }
    }
    if (rest) fill_rest<D>(p, 8);
}

// ---------------------------------------------------------------------------------------------- host
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
    static std::atomic<EncodeTiledFn> fn{nullptr};
    if (!fn.load()) {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qres) == cudaSuccess && qres == cudaDriverEntryPointSuccess)
            fn.store((EncodeTiledFn)f);
    }
    return fn.load();
}

// cache [pages, kv_heads, page_size, D] with any strides: boxes of 64 elements (32 when D = 32) x `keys` tokens of one page
// and head, swizzled to the box's row width; a page outside the cache reads as zeros
int make_cache_map(CUtensorMap* map, const void* ptr, const mxfp4_paged_attention_args* a, const int64_t* stride, int keys) {
    EncodeTiledFn enc = encode_tiled();
    if (!enc) { set_error("cuTensorMapEncodeTiled is not available from this driver"); return MXFP4_E_CUDA; }
    const int box_rows = a->page_size < keys ? a->page_size : keys, width = a->head_dim < 64 ? a->head_dim : 64;
    cuuint64_t dims[4] = {(cuuint64_t)a->head_dim, (cuuint64_t)a->page_size, (cuuint64_t)a->kv_heads, (cuuint64_t)a->num_pages};
    cuuint64_t strides[3] = {(cuuint64_t)stride[2] * 2, (cuuint64_t)stride[1] * 2, (cuuint64_t)stride[0] * 2};
    cuuint32_t box[4] = {(cuuint32_t)width, (cuuint32_t)box_rows, 1, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = enc(map, a->dtype == MXFP4_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(ptr), dims, strides,
                    box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, width == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled (cache) failed with CUresult %d", (int)r); return MXFP4_E_CUDA; }
    return MXFP4_OK;
}

// queries [tokens, kv_heads, group, D]: boxes of 64 elements x the whole group x as many tokens as fill 128 rows
int make_query_map(CUtensorMap* map, const mxfp4_paged_attention_args* a, int tokens) {
    EncodeTiledFn enc = encode_tiled();
    if (!enc) { set_error("cuTensorMapEncodeTiled is not available from this driver"); return MXFP4_E_CUDA; }
    const int group = a->heads / a->kv_heads;
    cuuint64_t dims[4] = {(cuuint64_t)a->head_dim, (cuuint64_t)group, (cuuint64_t)a->kv_heads, (cuuint64_t)a->tokens};
    cuuint64_t strides[3] = {(cuuint64_t)a->q_stride[1] * 2, (cuuint64_t)a->q_stride[1] * group * 2, (cuuint64_t)a->q_stride[0] * 2};
    cuuint32_t box[4] = {64, (cuuint32_t)group, 1, (cuuint32_t)tokens};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = enc(map, a->dtype == MXFP4_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(a->q), dims, strides,
                    box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled (queries) failed with CUresult %d", (int)r); return MXFP4_E_CUDA; }
    return MXFP4_OK;
}

template <int D, int RW, bool BF16>
int launch_rows(const CUtensorMap& mk, const CUtensorMap& mv, const AttnParams& p, int grid, cudaStream_t st) {
    using C = RowsCfg<D, RW>;
    static std::atomic<bool> configured[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(attn_rows_kernel<D, RW, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
        if (e != cudaSuccess) return cuda_fail(e, "mxfp4_paged_attention: cudaFuncSetAttribute");
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    const cudaError_t e = launch_smem(attn_rows_kernel<D, RW, BF16>, (unsigned)grid, kRowsThreads, (size_t)C::kSmemBytes, st, mk, mv, p);
    if (e != cudaSuccess) return cuda_fail(e, "mxfp4_paged_attention");
    return MXFP4_OK;
}
template <int D>
int launch_rows_any(int R, const CUtensorMap& mk, const CUtensorMap& mv, const AttnParams& p, int grid, cudaStream_t st) {
    if (p.bf16) return R == 16 ? launch_rows<D, 1, true>(mk, mv, p, grid, st) : launch_rows<D, 4, true>(mk, mv, p, grid, st);
    return R == 16 ? launch_rows<D, 1, false>(mk, mv, p, grid, st) : launch_rows<D, 4, false>(mk, mv, p, grid, st);
}

// The launches of one call and where the workspace of each lies.
struct AttnPlan {
    bool stacked;                    // kOwn + kPrefix instead of kAll
    int R[2], grid[2];               // [0]: kAll or kOwn, [1]: kPrefix
    int64_t slot_o[2], slot_lse[2], rows_o[2], rows_lse[2], seg[2], cut, bytes;
};

int64_t take(int64_t& at, int64_t bytes) {
    const int64_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
}

AttnPlan plan_of(const mxfp4_paged_attention_args* a) {
    AttnPlan l = {};
    const int64_t group = a->heads / a->kv_heads, rows = a->tokens * group, each = a->batch ? rows / a->batch : 0;
    // The prefix is computed once for all rows where a sequence alone would leave most of a row tile empty; sequences
    // that fill their tiles read it with their own keys, which saves the joining of two results per row.
    l.stacked = a->prefix_pages && a->prefix_table_pages > 0 && a->batch > 1 && each < 64;
    const bool wide = a->head_dim >= 64;
    l.R[0] = each <= 16 ? 16 : (each <= 64 || !wide ? 64 : 256);
    l.R[1] = rows <= 16 ? 16 : (rows <= 64 || !wide ? 64 : 256);
    for (int i = 0; i < 2; ++i) l.grid[i] = l.R[i] == 256 ? num_sms() : 2 * num_sms();
    int64_t at = 0;
    for (int i = 0; i < (l.stacked ? 2 : 1); ++i) {
        l.slot_o[i] = take(at, (int64_t)2 * l.grid[i] * l.R[i] * a->head_dim * 4);
        l.slot_lse[i] = take(at, (int64_t)2 * l.grid[i] * l.R[i] * 4);
        if (l.stacked) {
            l.rows_o[i] = take(at, a->tokens * a->heads * a->head_dim * 4);
            l.rows_lse[i] = take(at, a->tokens * a->heads * 4);
            l.seg[i] = take(at, a->tokens * a->heads * 8);
        }
    }
    if (!l.stacked) l.cut = take(at, (int64_t)l.grid[0] * 16);
    l.bytes = at;
    return l;
}

int check_args(const mxfp4_paged_attention_args* a) {
    if (!a) { set_error("mxfp4_paged_attention: null arguments"); return MXFP4_E_BADARG; }
    if (a->dtype != MXFP4_DT_BF16 && a->dtype != MXFP4_DT_F16) { set_error("mxfp4_paged_attention: dtype %d (bfloat16 or float16)", a->dtype); return MXFP4_E_BADARG; }
    if (a->tokens < 0 || a->batch < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->num_pages < 0 || a->table_pages < 0 || a->prefix_table_pages < 0) {
        set_error("mxfp4_paged_attention: negative size");
        return MXFP4_E_SHAPE;
    }
    if (a->heads % a->kv_heads) { set_error("mxfp4_paged_attention: %d heads are not a multiple of %d key heads", a->heads, a->kv_heads); return MXFP4_E_SHAPE; }
    if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) { set_error("mxfp4_paged_attention: head_dim %d (32, 64 or 128)", a->head_dim); return MXFP4_E_UNSUPPORTED; }
    if (a->page_size < 16 || a->page_size > 1024 || (a->page_size & (a->page_size - 1))) {
        set_error("mxfp4_paged_attention: page_size %d (a power of two from 16 to 1024)", a->page_size);
        return MXFP4_E_UNSUPPORTED;
    }
    const int64_t group = a->heads / a->kv_heads;
    if (a->tokens * group > 0x3FFFFFFF || a->tokens * (int64_t)a->heads > 0x3FFFFFFF || a->batch > 0x3FFFFFFF || a->kv_heads > 65535 || a->num_pages > 0x3FFFFFFF ||
        a->table_pages * (int64_t)a->page_size > 0x3FFFFFFF || a->prefix_table_pages * (int64_t)a->page_size > 0x3FFFFFFF) {
        set_error("mxfp4_paged_attention: size too large");
        return MXFP4_E_SHAPE;
    }
    if (!(a->scale > 1e-30 && a->scale < 1e30)) { set_error("mxfp4_paged_attention: scale %g must be positive and finite", a->scale); return MXFP4_E_BADARG; }
    if (!a->q_starts && a->tokens != a->batch) {
        set_error("mxfp4_paged_attention: %lld query rows for %lld sequences need q_starts", (long long)a->tokens, (long long)a->batch);
        return MXFP4_E_SHAPE;
    }
    return MXFP4_OK;
}

template <int D>
int run_attention(const mxfp4_paged_attention_args* a, const AttnPlan& l, AttnParams p, cudaStream_t st) {
    int rc;
    uint8_t* ws = (uint8_t*)a->workspace;
    AttnPart part[2] = {};
    for (int i = 0; i < (l.stacked ? 2 : 1); ++i) {
        p.keys = l.stacked ? (i ? kPrefix : kOwn) : kAll;
        p.slot_o = (float*)(ws + l.slot_o[i]); p.slot_lse = (float*)(ws + l.slot_lse[i]);
        p.rows_o = (float*)(ws + l.rows_o[i]); p.rows_lse = (float*)(ws + l.rows_lse[i]); p.rows_seg = (int2*)(ws + l.seg[i]);
        p.cut = (int4*)(ws + l.cut);
        CUtensorMap mk, mv;
        const int keys = l.R[i] == 256 ? 128 : kRowsKeys;
        if ((rc = make_cache_map(&mk, a->k_cache, a, a->k_cache_stride, keys))) return rc;
        if ((rc = make_cache_map(&mv, a->v_cache, a, a->v_cache_stride, keys))) return rc;
        if (l.R[i] == 256) {
            CUtensorMap mq = {};
            p.q_box = p.group <= 128 && 128 % p.group == 0 && p.q_row > 0 && p.q_head > 0 ? 128 / p.group : 0;
            if (p.q_box && (rc = make_query_map(&mq, a, p.q_box))) return rc;
            rc = launch_attn_tc(D, mq, mk, mv, p, l.grid[i], st);
        } else {
            rc = launch_rows_any<D>(l.R[i], mk, mv, p, l.grid[i], st);
        }
        if (rc) return rc;
        part[i] = AttnPart{p.slot_o, p.slot_lse, p.rows_o, p.rows_lse, p.rows_seg, l.R[i], l.grid[i]};
    }
    const int rest = a->fill_rest && p.starts;
    cudaError_t e;
    if (l.stacked) e = launch_smem(attn_join_rows_kernel<D>, (unsigned)((a->tokens * a->heads + 7) / 8), 256, 0, st, p, part[0], part[1], rest);
    else e = launch_smem(attn_join_cut_kernel<D>, dim3((unsigned)l.grid[0], (unsigned)(l.R[0] + 31) / 32, 1), 256, 0, st, p, l.R[0], rest);
    if (e != cudaSuccess) return cuda_fail(e, "mxfp4_paged_attention: join");
    return MXFP4_OK;
}

}  // namespace
}  // namespace mxfp4

extern "C" int64_t mxfp4_paged_attention_workspace_bytes(const mxfp4_paged_attention_args* a) {
    using namespace mxfp4;
    if (check_args(a)) return -1;
    return plan_of(a).bytes;
}

extern "C" int mxfp4_paged_attention(const mxfp4_paged_attention_args* args, void* stream) {
    using namespace mxfp4;
    const int rc = check_args(args);
    if (rc) return rc;
    mxfp4_paged_attention_args own = *args;
    own.q_stride[0] = used_stride(own.q_stride[0], own.tokens); own.q_stride[1] = used_stride(own.q_stride[1], own.heads);
    own.out_stride[0] = used_stride(own.out_stride[0], own.tokens); own.out_stride[1] = used_stride(own.out_stride[1], own.heads);
    for (int64_t* st : {own.k_cache_stride, own.v_cache_stride}) {
        st[0] = used_stride(st[0], own.num_pages); st[1] = used_stride(st[1], own.kv_heads); st[2] = used_stride(st[2], own.page_size);
    }
    const mxfp4_paged_attention_args* a = &own;
    if (a->tokens == 0) return MXFP4_OK;
    if (a->num_pages == 0 || a->batch == 0) { set_error("mxfp4_paged_attention: query rows without a sequence or a cache"); return MXFP4_E_SHAPE; }
    if (!a->q || !a->out || !a->seq_lens || (a->table_pages && !a->block_tables) || !a->workspace || !a->k_cache || !a->v_cache ||
        (a->prefix_pages && !a->prefix_len)) {
        set_error("mxfp4_paged_attention: null pointer");
        return MXFP4_E_BADARG;
    }
    int64_t strides = a->q_stride[0] | a->q_stride[1] | a->out_stride[0] | a->out_stride[1];
    for (int i = 0; i < 3; ++i) strides |= a->k_cache_stride[i] | a->v_cache_stride[i];
    const uintptr_t ptrs = (uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)a->k_cache | (uintptr_t)a->v_cache;
    if (strides % 8 || ptrs % 16 || (uintptr_t)a->workspace % 256) {
        set_error("mxfp4_paged_attention: q, out and the caches must be 16-byte aligned with strides of multiples of 8 elements, the workspace 256-byte aligned");
        return MXFP4_E_ALIGN;
    }
    const AttnPlan l = plan_of(a);
    if (a->workspace_bytes < l.bytes) {
        set_error("mxfp4_paged_attention: workspace of %lld bytes, %lld needed", (long long)a->workspace_bytes, (long long)l.bytes);
        return MXFP4_E_WORKSPACE;
    }
    AttnParams p = {};
    p.q = a->q; p.q_row = a->q_stride[0]; p.q_head = a->q_stride[1];
    p.out = a->out; p.out_row = a->out_stride[0]; p.out_head = a->out_stride[1];
    p.lse = a->lse;
    p.lens = a->seq_lens; p.starts = a->q_starts; p.table = a->block_tables; p.table_stride = a->table_stride; p.table_pages = (int)a->table_pages;
    p.prefix_pages = a->prefix_table_pages > 0 ? a->prefix_pages : nullptr;
    p.prefix_len = a->prefix_len; p.prefix_table_pages = (int)a->prefix_table_pages;
    p.batch = (int)a->batch; p.tokens = (int)a->tokens; p.heads = a->heads; p.kv_heads = a->kv_heads; p.group = a->heads / a->kv_heads;
    p.page_shift = 31 - __builtin_clz((unsigned)a->page_size); p.num_pages = (int)a->num_pages;
    p.scale_log2 = (float)(a->scale * 1.4426950408889634074);
    p.bf16 = a->dtype == MXFP4_DT_BF16;
    p.status = a->status_dev;
    cudaStream_t st = (cudaStream_t)stream;
    switch (a->head_dim) {
        case 32: return run_attention<32>(a, l, p, st);
        case 64: return run_attention<64>(a, l, p, st);
        default: return run_attention<128>(a, l, p, st);
    }
}
