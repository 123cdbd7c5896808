// Shared pieces of the paged attention kernels: parameters, the division of the work over the CTAs, the page-wise tile
// loads and the form of partial results.
//
// out[t, head] = softmax_j(scale * q[t, head] . k[j]) v[j] over the keys j that token t sees: all `prefix_len` keys of the
// prefix, which the whole batch shares, and the first len - n + i + 1 of its sequence's own `len` keys, where t is the
// i-th of the sequence's n query tokens.  A token that sees nothing gets zeros and a log-sum of -inf.
//
// The heads that share a key head are stacked with the tokens into the rows of a tile (row = token * group + head in the
// group), so that a key is read once for all of them.  An item is one row tile of one key head against all the keys that
// the launch gives it; its cost in units is its number of key tiles and a constant for its beginning and end.  The grid
// is as large as the GPU holds, and CTA c takes the units [W c / P, W (c + 1) / P) of the W in all, in the order (sequence,
// row tile, key head, key): every CTA gets the same number of units whatever the lengths, and an item crosses from a CTA to
// the next at most once per CTA.  Lengths are read on the device, so that a captured launch follows them.
//
// Which keys a launch gives its items:
//   kAll     the prefix, then the sequence's own: the tile's result is final unless the item was cut
//   kOwn     the sequence's own only, kPrefix the prefix only with the rows of ALL sequences stacked into full tiles,
//            which reads the prefix once for the batch: joined per row afterwards
// A cut item leaves its parts in slots of the workspace, two per CTA: slot 2c for the part that began in an earlier CTA,
// slot 2c + 1 for the part that goes on in the next one.  A part is the normalised float32 result and the base-2 log of
// its sum of weights, -inf where it has none.
#pragma once
#include "gemm_mxf4_tc.cuh"

namespace mxfp4 {

enum AttnKeys { kAll = 0, kOwn = 1, kPrefix = 2 };

struct AttnParams {
    const void* q;
    int64_t q_row, q_head;
    void* out;                       // [tokens, heads, D]
    int64_t out_row, out_head;
    float* lse;                      // [tokens, heads] natural log, or null
    const int* lens;                 // [batch] own keys
    const int* starts;               // [batch + 1] first query row of every sequence, or null: one row each
    const int* table;                // [batch, table_pages] own pages
    int64_t table_stride;
    int table_pages;
    const int* prefix_pages;         // [prefix_table_pages], or null
    const int* prefix_len;           // one int
    int prefix_table_pages;
    int batch, tokens, heads, kv_heads, group;
    int page_shift, num_pages;
    float scale_log2;                // scale * log2(e)
    int keys;                        // AttnKeys
    int bf16;
    int q_box;                       // tokens per half row tile where the group divides it (their rows come by TMA), else 0
    float* slot_o;                   // [2 * grid][row tile][D]
    float* slot_lse;                 // [2 * grid][row tile]
    float* rows_o;                   // kOwn / kPrefix: [tokens * heads][D], results of items that were not cut
    float* rows_lse;                 // [tokens * heads]
    int2* rows_seg;                  // [tokens * heads] {CTA where the item began, CTA where it ended; -1: rows_o has it; -2: nothing}
    int4* cut;                       // kAll: [grid] {CTA where the item that goes on behind this CTA ends, or -1; first token; first row; key head << 9 | rows}
    int* status;
};

// paged_attention_tc.cu: head_dim 64 or 128, row tiles of 256, boxes of at most 128 keys; map_q when p.q_box is set
int launch_attn_tc(int head_dim, const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v, const AttnParams& p, int grid, cudaStream_t stream);

namespace {

constexpr float kNegInf = -__builtin_huge_valf();

// What one sequence brings to a launch.  In kPrefix launches there is one "sequence" of all tokens.
struct AttnSeq {
    int start, n, len;
};

__device__ __forceinline__ int prefix_keys(const AttnParams& p) {
    if (!p.prefix_pages || p.keys == kOwn) return 0;
    const int most = p.prefix_table_pages << p.page_shift, n = *p.prefix_len;
    return n < 0 ? 0 : (n > most ? most : n);
}
__device__ __forceinline__ AttnSeq attn_seq(const AttnParams& p, int b) {
    AttnSeq s;
    if (p.keys == kPrefix) {
        s.start = 0; s.n = p.tokens; s.len = 0;
        return s;
    }
    const int most = p.table_pages << p.page_shift, len = p.lens[b];
    s.len = len < 0 ? 0 : (len > most ? most : len);
    if (p.starts) {
        const int a = p.starts[b], e = p.starts[b + 1];
        s.start = a < 0 ? 0 : (a > p.tokens ? p.tokens : a);
        s.n = (e > p.tokens ? p.tokens : e) - s.start;
        if (s.n < 0) s.n = 0;
    } else {
        s.start = b; s.n = 1;
    }
    return s;
}

template <int R>
__device__ __forceinline__ int attn_row_tiles(const AttnParams& p, const AttnSeq& s) { return (s.n * p.group + R - 1) / R; }

// own keys that the last row of a row tile sees: no other row of it sees more
template <int R>
__device__ __forceinline__ int attn_own_keys(const AttnParams& p, const AttnSeq& s, int rt) {
    if (p.keys == kPrefix) return 0;
    int last = ((rt + 1) * R - 1) / p.group;                 // rows and keys are below 2^30
    if (last > s.n - 1) last = s.n - 1;
    const int k = s.len - s.n + last + 1;
    return k < 0 ? 0 : k;
}
// key tiles of one item; an item without keys still counts as one, because its rows have to be written
template <int R, int K>
__device__ __forceinline__ int attn_tiles(const AttnParams& p, const AttnSeq& s, int rt, int prefix_tiles) {
    const int t = prefix_tiles + (attn_own_keys<R>(p, s, rt) + K - 1) / K;
    return t < 1 ? 1 : t;
}
// What an item costs besides its key tiles, in key tiles: filling the pipeline, the result.  Measured: without it the CTA whose
// share was 31 prompt tiles of two key tiles each took twice the others' time (4 x 2048 causal 358 us against 223 with 3; 2 and
// 4: 230, 226); 64 sequences of 1 to 700 keys 39.5 us with 1, 34.3 with 3 to 5, 35.0 with 8.
template <int R>
__device__ __forceinline__ constexpr int attn_item_cost() { return R == 256 ? 3 : 4; }

template <int R, int K>
__device__ __forceinline__ int64_t attn_seq_units(const AttnParams& p, const AttnSeq& s, int prefix_tiles) {
    int64_t sum = 0;
    const int rts = attn_row_tiles<R>(p, s);
    for (int rt = 0; rt < rts; ++rt) sum += attn_tiles<R, K>(p, s, rt, prefix_tiles) + attn_item_cost<R>();
    return sum * p.kv_heads;
}

// The walk of a CTA over its units.  Every role of a CTA has its own copy and takes the same steps.
template <int R, int K>
struct AttnWalk {
    AttnSeq s;
    int b, rt, h;                    // the item: sequence, row tile, key head
    int tiles;                       // key tiles of the whole item
    int u0, u1;                      // this CTA's part of its units (the constant cost comes first) ...
    int t0, t1;                      // ... and of its key tiles
    int64_t left;                    // units of the CTA from u0 on
    int prefix, prefix_tiles;

    __device__ __forceinline__ bool cut() {
        constexpr int E = attn_item_cost<R>();
        u1 = (int64_t)(tiles + E - u0) > left ? u0 + (int)left : tiles + E;
        t0 = u0 > E ? u0 - E : 0;
        t1 = u1 > E ? u1 - E : 0;
        return t1 > t0;              // a CTA that ends within an item's constant cost leaves the whole item to the next
    }
    // the last unit of the item among all units
    __device__ __forceinline__ int64_t last_unit(int64_t w1) const { return w1 - left - u0 + tiles + attn_item_cost<R>() - 1; }
    // to the first item at or behind sequence b that has rows
    __device__ __forceinline__ void load(const AttnParams& p) {
        s = attn_seq(p, b);
        while (s.n <= 0 && b + 1 < p.batch) s = attn_seq(p, ++b);
    }
    __device__ __forceinline__ bool next(const AttnParams& p) {
        left -= u1 - u0;
        if (left <= 0) return false;
        u0 = 0;
        if (++h == p.kv_heads) {
            h = 0;
            if (++rt == attn_row_tiles<R>(p, s)) {
                rt = 0;
                ++b;
                load(p);
            }
            tiles = attn_tiles<R, K>(p, s, rt, prefix_tiles);
        }
        return cut();
    }
};

struct AttnStart {                   // in shared memory: where the CTA begins
    int64_t w0, w1, total, seq_first;
    int b;
};

// All threads of the block: the number W of units and the sequence of this CTA's first one.  A thread adds up a
// contiguous range of the sequences; the one whose range holds the first unit walks it again.  W = 0: nothing to do.
template <int R, int K, int kThreadsOfBlock>
__device__ __forceinline__ void attn_find_start(const AttnParams& p, AttnStart* at, int64_t* sums /* [kThreadsOfBlock / 32] */) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int seqs = p.keys == kPrefix ? 1 : p.batch;
    const int prefix_tiles = (prefix_keys(p) + K - 1) / K;
    const int b0 = (int)((int64_t)seqs * tid / kThreadsOfBlock), b1 = (int)((int64_t)seqs * (tid + 1) / kThreadsOfBlock);
    int64_t mine = 0;
    bool bad = false;
    if (!(p.keys == kPrefix && prefix_tiles == 0)) {
        for (int b = b0; b < b1; ++b) {
            mine += attn_seq_units<R, K>(p, attn_seq(p, b), prefix_tiles);
            if (p.keys != kPrefix) {
                bad |= p.lens[b] < 0 || p.lens[b] > (p.table_pages << p.page_shift);
                if (p.starts) bad |= p.starts[b] < 0 || p.starts[b] > p.starts[b + 1] || p.starts[b + 1] > p.tokens;
            }
        }
    }
    if (tid == 0 && p.prefix_pages) bad |= *p.prefix_len < 0 || *p.prefix_len > (p.prefix_table_pages << p.page_shift);
    if (bad && blockIdx.x == 0 && p.status) atomicExch(p.status, MXFP4_E_SHAPE);
    int64_t incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(0xFFFFFFFFu, incl, d);
        if (lane >= d) incl += o;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    int64_t before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kThreadsOfBlock / 32; ++w) {
        if (w < warp) before += sums[w];
        total += sums[w];
    }
    const int64_t excl = before + incl - mine;
    const int64_t w0 = total * blockIdx.x / gridDim.x, w1 = total * (blockIdx.x + 1) / gridDim.x;
    if (tid == 0) { at->w0 = w0; at->w1 = w1; at->total = total; }
    if (mine > 0 && excl <= w0 && w0 < excl + mine) {
        int64_t at_b = excl;
        for (int b = b0; b < b1; ++b) {
            const int64_t n = attn_seq_units<R, K>(p, attn_seq(p, b), prefix_tiles);
            if (w0 < at_b + n) { at->b = b; at->seq_first = at_b; break; }
            at_b += n;
        }
    }
    __syncthreads();
}

template <int R, int K>
__device__ __forceinline__ bool attn_begin(const AttnParams& p, const AttnStart& at, AttnWalk<R, K>& w) {
    if (at.w1 <= at.w0) return false;
    w.prefix = prefix_keys(p);
    w.prefix_tiles = (w.prefix + K - 1) / K;
    w.b = at.b;
    w.s = attn_seq(p, w.b);
    w.left = at.w1 - at.w0;
    int64_t off = at.w0 - at.seq_first;
    int units;
    for (w.rt = 0;; ++w.rt) {
        w.tiles = attn_tiles<R, K>(p, w.s, w.rt, w.prefix_tiles);
        units = w.tiles + attn_item_cost<R>();
        if (off < (int64_t)units * p.kv_heads) break;
        off -= (int64_t)units * p.kv_heads;
    }
    w.h = (int)(off / units);
    w.u0 = (int)(off - (int64_t)w.h * units);
    return w.cut();
}

// CTA that holds unit w of `total`: the last c with total * c / grid <= w
__device__ __forceinline__ int attn_cta_of(int64_t w, int64_t total) { return (int)(((w + 1) * gridDim.x - 1) / total); }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map),
                 "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
                 : "memory");
}

// Stores of a pair / four results in the output's type
__device__ __forceinline__ uint32_t pack2(int bf16, float a, float b) {
    if (bf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

constexpr float kLn2 = 0.69314718055994530942f;

template <typename... KArgs, typename... Args>
inline cudaError_t launch_smem(void (*kernel)(KArgs...), dim3 grid, unsigned block, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

}  // namespace
}  // namespace mxfp4
