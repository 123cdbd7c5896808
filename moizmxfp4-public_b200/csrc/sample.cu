// The next token of every row of logits from one given uniform number: temperature, top-k, top-p, min-p.
//
// Tokens are taken in descending order of their logits, equal ones by index, and every filter keeps a beginning of that
// order; so all that a filter has to yield is the weight of what it keeps, and the kept weight is the smallest of them.
// The sampled token, the k-th token and the last token of top-p are all "the first token whose cumulative count or weight
// reaches a target", which one routine finds without sorting: a histogram of counts and weights over the leading 11 bits of
// the (order-preserving) key, a scan, then histograms of the next bits inside the bin that holds the target (one more for
// 16-bit logits, two more for float32), and for equal keys the rank among them, found by counting in index order.
//
// Weights are fixed-point: rint(exp((l - max) / T) * 2^shift) with 2^shift * vocab < 2^63, the exponential in 64 bits.  Sums
// of integers do not depend on the order of the additions, so atomics on the histograms leave nothing to chance, and 45
// bits after the point at a vocabulary of 2^17 keep cumulative weights good to 1e-11, where float32 sums would move borders
// between tokens by 1e-7 and change what is sampled.
//
// A cluster of CTAs takes a row: each its contiguous piece, kept in shared memory where it fits, so that the logits are
// read once; histograms are added over distributed shared memory.  Bound by latency (a dozen cluster barriers) for few rows
// and by the 64-bit exponentials and shared-memory atomics for many.
#include <cooperative_groups.h>

#include "mxfp4_common.cuh"

namespace mxfp4 {
namespace {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;

struct SampleParams {
    const void* logits;
    int64_t ld;
    int vocab, shift, levels, piece;         // piece: logits per CTA, cached in shared memory when `cached`
    int cached;
    const float *uniforms, *temperature, *top_p, *min_p;
    const int* top_k;
    double temperature_value, top_p_value, min_p_value;
    int64_t top_k_value;
    int64_t* tokens;
    float* logprobs;
};

// Order-preserving key, inverted: ascending keys are descending logits.  NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float l) {
    if (l != l) l = -__builtin_huge_valf();
    const uint32_t u = __float_as_uint(l + 0.0f);
    return (u & 0x80000000u) ? u : ~(u | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key : (~key & 0x7FFFFFFFu)); }

struct Found {
    uint32_t bin;
    uint64_t before_count, before_weight;
};

struct SampleShared {
    uint32_t count[kBins], lo[kBins], hi[kBins];       // this CTA's histogram
    uint64_t sum_weight[2][kBins];                     // this CTA's slice of the cluster's histogram: [0] leading bits, [1] the level at hand
    uint32_t sum_count[2][kBins];
    uint64_t total_weight[2][kMaxCluster];             // of every CTA's slice
    uint32_t total_count[2][kMaxCluster];
    Found found[2];
    uint64_t warp_weight[kSampleThreads / 32];
    uint32_t warp_count[kSampleThreads / 32];
    uint32_t best[kMaxCluster];
    uint64_t kept[kMaxCluster];
    uint32_t ties[kMaxCluster];
};

template <typename T>
struct Sampler {
    const SampleParams& p;
    SampleShared& sh;
    cg::cluster_group cl;
    const T* data;                                     // this CTA's piece
    int n;                                             // logits in it
    int rank, size, slice;                             // slice: bins of the cluster's histogram per CTA
    int finds;
    double inv_t, unit;
    float top;

    __device__ __forceinline__ void sync() {
        if (size == 1) __syncthreads();
        else cl.sync();
    }
    template <typename V> __device__ __forceinline__ V* at(V* local, int r) { return size == 1 ? local : cl.map_shared_rank(local, r); }

    // weight relative to the maximum's; -inf has none at any temperature, an infinite one among them
    __device__ __forceinline__ double share(float l) const { return l == -__builtin_huge_valf() ? 0.0 : exp(((double)l - (double)top) * inv_t); }
    __device__ __forceinline__ uint64_t fixed(double e) const { return (uint64_t)(e * unit + 0.5); }

    __device__ __forceinline__ void clear() {
        for (int i = threadIdx.x; i < kBins; i += kSampleThreads) sh.count[i] = sh.lo[i] = sh.hi[i] = 0;
        __syncthreads();
    }
    __device__ __forceinline__ void add(uint32_t bin, uint64_t w) {
        atomicAdd(&sh.count[bin], 1u);
        const uint32_t lo = (uint32_t)w;
        const uint32_t carry = lo && atomicAdd(&sh.lo[bin], lo) + lo < lo ? 1u : 0u;
        if (uint32_t hi = (uint32_t)(w >> 32) + carry) atomicAdd(&sh.hi[bin], hi);
    }
    // The cluster's histogram of level `slot` from the CTAs' own, this CTA's slice of it, and the totals of all slices.
    // Leaves the CTA's own histogram cleared.
    __device__ __forceinline__ void gather(int slot) {
        sync();
        uint64_t weight = 0;
        uint32_t count = 0;
        for (int i = threadIdx.x; i < slice; i += kSampleThreads) {
            const int b = rank * slice + i;
            uint64_t w = 0;
            uint32_t c = 0;
            for (int r = 0; r < size; ++r) {
                w += ((uint64_t)at(sh.hi, r)[b] << 32) + at(sh.lo, r)[b];
                c += at(sh.count, r)[b];
            }
            sh.sum_weight[slot][i] = w;
            sh.sum_count[slot][i] = c;
            weight += w;
            count += c;
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            weight += __shfl_xor_sync(0xFFFFFFFFu, weight, d);
            count += __shfl_xor_sync(0xFFFFFFFFu, count, d);
        }
        if ((threadIdx.x & 31) == 0) { sh.warp_weight[threadIdx.x >> 5] = weight; sh.warp_count[threadIdx.x >> 5] = count; }
        __syncthreads();
        if (threadIdx.x < size) {
            weight = 0; count = 0;
            for (int i = 0; i < kSampleThreads / 32; ++i) { weight += sh.warp_weight[i]; count += sh.warp_count[i]; }
            at(&sh, threadIdx.x)->total_weight[slot][rank] = weight;
            at(&sh, threadIdx.x)->total_count[slot][rank] = count;
        }
        sync();
        clear();
    }
    // The first bin where the running weight (or count) reaches `target`, which the level's total does.
    __device__ __forceinline__ Found find(int slot, bool by_weight, uint64_t target) {
        Found& out = sh.found[finds & 1];
        uint64_t weight = 0, count = 0;
        int r = 0;
        for (; r < size - 1; ++r) {
            if ((by_weight ? weight + sh.total_weight[slot][r] : count + sh.total_count[slot][r]) >= target) break;
            weight += sh.total_weight[slot][r];
            count += sh.total_count[slot][r];
        }
        if (r == rank) {                                // this CTA's slice holds it
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = (slice + kSampleThreads - 1) / kSampleThreads, i0 = threadIdx.x * per;
            uint64_t w = 0, c = 0;
            for (int i = i0; i < i0 + per && i < slice; ++i) { w += sh.sum_weight[slot][i]; c += sh.sum_count[slot][i]; }
            uint64_t wi = w, ci = c;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint64_t a = __shfl_up_sync(0xFFFFFFFFu, wi, d), b = __shfl_up_sync(0xFFFFFFFFu, ci, d);
                if (lane >= d) { wi += a; ci += b; }
            }
            if (lane == 31) { sh.warp_weight[warp] = wi; sh.warp_count[warp] = (uint32_t)ci; }
            __syncthreads();
            for (int i = 0; i < warp; ++i) { weight += sh.warp_weight[i]; count += sh.warp_count[i]; }
            weight += wi - w;
            count += ci - c;
            if ((by_weight ? weight : count) < target && target <= (by_weight ? weight + w : count + c)) {
                for (int i = i0; i < i0 + per && i < slice; ++i) {
                    const uint64_t bw = sh.sum_weight[slot][i], bc = sh.sum_count[slot][i];
                    if ((by_weight ? weight + bw : count + bc) >= target) {
                        for (int q = 0; q < size; ++q) {
                            Found* f = at(&out, q);
                            f->bin = (uint32_t)(rank * slice + i);
                            f->before_count = count;
                            f->before_weight = weight;
                        }
                        break;
                    }
                    weight += bw;
                    count += bc;
                }
            }
        }
        sync();
        ++finds;
        return out;
    }
    struct Place {
        uint32_t key;                                  // of the token
        uint64_t rank;                                 // among the tokens with that key, in index order
        uint64_t weight;                               // of all tokens up to and with it
    };
    // The first token whose cumulative weight (or count) reaches `target`; the leading bits' histogram is in slot 0.
    __device__ __forceinline__ Place select(bool by_weight, uint64_t target) {
        Found f = find(0, by_weight, target);
        uint32_t prefix = f.bin;
        uint64_t before = f.before_weight;
        target -= by_weight ? f.before_weight : f.before_count;
        int used = 11;
        for (int level = 1; level < p.levels; ++level) {
            const int bits = 32 - used < 11 ? 32 - used : 11, down = 32 - used - bits;
            for (int i = threadIdx.x; i < n; i += kSampleThreads) {
                const float l = to_f32<T>(data[i]);
                const uint32_t k = key_of(l);
                if (k >> (32 - used) == prefix) add((k >> down) & ((1u << bits) - 1), fixed(share(logit_of(k))));
            }
            gather(1);
            f = find(1, by_weight, target);
            prefix = (prefix << bits) | f.bin;
            before += f.before_weight;
            target -= by_weight ? f.before_weight : f.before_count;
            used += bits;
        }
        Place out;
        out.key = prefix;
        if (used < 32) {
            // 16-bit logits: the bits below are those of a float32 whose mantissa ends in zeros
            const uint32_t low = (1u << (32 - used)) - 1;
            out.key = (prefix << (32 - used)) | ((prefix >> (used - 1)) & 1u ? 0u : low);
        }
        const uint64_t w = fixed(share(logit_of(out.key)));
        out.rank = by_weight ? (target - 1) / (w ? w : 1) : target - 1;
        out.weight = before + (out.rank + 1) * w;
        return out;
    }
};

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleParams p) {
    MXFP4_CHAIN_PROLOGUE();
    extern __shared__ __align__(16) uint8_t smem_raw[];
    SampleShared& sh = *reinterpret_cast<SampleShared*>(smem_raw);
    T* cache = reinterpret_cast<T*>(smem_raw + (sizeof(SampleShared) + 15) / 16 * 16);
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), size = (int)cl.num_blocks(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / size;
    const int from = rank * p.piece, n = p.vocab - from < p.piece ? (p.vocab - from < 0 ? 0 : p.vocab - from) : p.piece;
    const T* src = (const T*)p.logits + row * p.ld + from;
    Sampler<T> s{p, sh, cl, p.cached ? cache : src, n, rank, size, kBins / size, 0, 0.0, 0.0, 0.0f};

    // the row's maximum
    uint32_t best = 0xFFFFFFFFu;
    for (int i = tid; i < n; i += kSampleThreads) {
        const T v = src[i];
        if (p.cached) cache[i] = v;
        const uint32_t k = key_of(to_f32<T>(v));
        best = k < best ? k : best;
    }
    best = __reduce_min_sync(0xFFFFFFFFu, best);
    if (lane == 0) sh.warp_count[warp] = best;
    s.clear();
    if (tid < size) {
        for (int i = 0; i < kSampleThreads / 32; ++i) best = sh.warp_count[i] < best ? sh.warp_count[i] : best;
        s.at(&sh, tid)->best[rank] = best;
    }
    s.sync();
    best = sh.best[0];
    for (int r = 1; r < size; ++r) best = sh.best[r] < best ? sh.best[r] : best;
    s.top = logit_of(best);
    const double heat = p.temperature ? (double)p.temperature[row] : p.temperature_value;
    const bool finite = s.top - s.top == 0.0f;

    typename Sampler<T>::Place pick{best, 0, 0};
    double logprob = 0.0;
    if (heat > 0.0 && finite) {
        const int64_t top_k = p.top_k ? p.top_k[row] : p.top_k_value;
        const double top_p = p.top_p ? (double)p.top_p[row] : p.top_p_value;
        double min_p = p.min_p ? (double)p.min_p[row] : p.min_p_value;
        min_p = min_p > 1.0 ? 1.0 : min_p;
        s.inv_t = 1.0 / heat;
        s.unit = (double)(1ull << p.shift);
        uint64_t above = 0;
        for (int i = tid; i < n; i += kSampleThreads) {
            const uint32_t k = key_of(to_f32<T>(s.data[i]));
            const double e = s.share(logit_of(k));
            const uint64_t w = s.fixed(e);
            s.add(k >> 21, w);
            if (e >= min_p) above += w;
        }
        s.gather(0);
        uint64_t kept = 0;
        for (int r = 0; r < size; ++r) kept += sh.total_weight[0][r];
        if (min_p > 0.0) {
#pragma unroll
            for (int d = 16; d; d >>= 1) above += __shfl_xor_sync(0xFFFFFFFFu, above, d);
            if (lane == 0) sh.warp_weight[warp] = above;
            __syncthreads();
            if (tid < size) {
                above = 0;
                for (int i = 0; i < kSampleThreads / 32; ++i) above += sh.warp_weight[i];
                s.at(&sh, tid)->kept[rank] = above;
            }
            s.sync();
            above = 0;
            for (int r = 0; r < size; ++r) above += sh.kept[r];
        }
        if (top_k > 0 && top_k < p.vocab) {
            const uint64_t w = s.select(false, (uint64_t)top_k).weight;
            kept = w < kept ? w : kept;
        }
        if (top_p < 1.0) {
            const double goal = ceil(top_p * (double)kept);
            uint64_t target = goal >= 1.0 ? (uint64_t)goal : 1;
            target = target < kept ? target : kept;
            const uint64_t w = s.select(true, target).weight;
            kept = w < kept ? w : kept;
        }
        if (min_p > 0.0) kept = above < kept ? above : kept;
        const double u = (double)p.uniforms[row];
        uint64_t target = u > 0.0 ? (u < 1.0 ? (uint64_t)(u * (double)kept) : kept) : 0;
        target = target < kept ? target + 1 : kept;
        pick = s.select(true, target);
        logprob = ((double)logit_of(pick.key) - (double)s.top) * s.inv_t - log((double)kept / s.unit);
    }

    // the token: the pick.rank-th of its key in index order.  Warps take contiguous runs of the piece.
    const int run = (n + kSampleThreads / 32 - 1) / (kSampleThreads / 32), i0 = warp * run, i1 = i0 + run < n ? i0 + run : n;
    uint32_t mine = 0;
    for (int i = i0 + lane; i < i1; i += 32) mine += key_of(to_f32<T>(s.data[i])) == pick.key;
    mine = __reduce_add_sync(0xFFFFFFFFu, mine);
    __syncthreads();
    if (lane == 0) sh.warp_count[warp] = mine;
    __syncthreads();
    if (tid < size) {
        uint32_t all = 0;
        for (int i = 0; i < kSampleThreads / 32; ++i) all += sh.warp_count[i];
        s.at(&sh, tid)->ties[rank] = all;
    }
    s.sync();
    uint64_t before = 0;
    for (int r = 0; r < rank; ++r) before += sh.ties[r];
    for (int i = 0; i < warp; ++i) before += sh.warp_count[i];
    if (pick.rank >= before && pick.rank < before + mine) {
        uint32_t left = (uint32_t)(pick.rank - before);
        for (int b = i0; b < i1; b += 32) {
            const bool hit = b + lane < i1 && key_of(to_f32<T>(s.data[b + lane])) == pick.key;
            const uint32_t votes = __ballot_sync(0xFFFFFFFFu, hit), c = __popc(votes);
            if (left < c) {
                if (hit && __popc(votes & ((1u << lane) - 1)) == left) {
                    p.tokens[row] = from + b + lane;
                    if (p.logprobs) p.logprobs[row] = (float)logprob;
                }
                break;
            }
            left -= c;
        }
    }
}

template <typename T>
int launch_sample(SampleParams& p, int64_t rows, cudaStream_t st) {
    // As many CTAs per row as keep the GPU full (two per SM), and enough for the row to fit into their shared memory.
    int size = 1;
    while (size < kMaxCluster && rows * size * 2 <= 2 * (int64_t)num_sms() && p.vocab / size > 2048) size *= 2;
    constexpr int64_t kCache = 96 * 1024;
    while (size < kMaxCluster && (int64_t)p.vocab * (int64_t)sizeof(T) > kCache * size) size *= 2;
    p.piece = ((p.vocab + size - 1) / size + 7) / 8 * 8;
    p.cached = (int64_t)p.piece * (int64_t)sizeof(T) <= kCache;
    const size_t smem = (sizeof(SampleShared) + 15) / 16 * 16 + (p.cached ? (size_t)p.piece * sizeof(T) : 0);
    cudaError_t e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(SampleShared) + 16 + kCache));
    if (e != cudaSuccess) return cuda_fail(e, "mxfp4_sample: cudaFuncSetAttribute");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * size), 1, 1);
    cfg.blockDim = dim3(kSampleThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)size;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, p);
    if (e != cudaSuccess) return cuda_fail(e, "mxfp4_sample");
    return MXFP4_OK;
}

}  // namespace
}  // namespace mxfp4

extern "C" int mxfp4_sample(const mxfp4_sample_args* a, void* stream) {
    using namespace mxfp4;
    if (!a) { set_error("mxfp4_sample: null arguments"); return MXFP4_E_BADARG; }
    if (a->dtype != MXFP4_DT_BF16 && a->dtype != MXFP4_DT_F16 && a->dtype != MXFP4_DT_F32) { set_error("mxfp4_sample: unknown dtype %d", a->dtype); return MXFP4_E_BADARG; }
    if (a->rows < 0 || a->vocab < 0 || a->ld < a->vocab) { set_error("mxfp4_sample: negative size or ld < vocab"); return MXFP4_E_SHAPE; }
    if (a->rows == 0) return MXFP4_OK;
    if (a->vocab == 0 || a->vocab > (1 << 24) || a->rows > (1 << 26)) { set_error("mxfp4_sample: vocab %lld (1 to 2^24) or rows %lld (at most 2^26)", (long long)a->vocab, (long long)a->rows); return MXFP4_E_SHAPE; }
    if (!a->logits || !a->uniforms || !a->tokens) { set_error("mxfp4_sample: null pointer"); return MXFP4_E_BADARG; }
    SampleParams p;
    p.logits = a->logits; p.ld = a->ld; p.vocab = (int)a->vocab;
    int bits = 0;
    while ((int64_t(1) << bits) < a->vocab) ++bits;
    p.shift = 62 - bits;
    p.levels = a->dtype == MXFP4_DT_F32 ? 3 : 2;
    p.uniforms = a->uniforms; p.temperature = a->temperature; p.top_p = a->top_p; p.min_p = a->min_p; p.top_k = a->top_k;
    p.temperature_value = a->temperature_value; p.top_p_value = a->top_p_value; p.min_p_value = a->min_p_value; p.top_k_value = a->top_k_value;
    p.tokens = a->tokens; p.logprobs = a->logprobs;
    cudaStream_t st = (cudaStream_t)stream;
    switch (a->dtype) {
        case MXFP4_DT_BF16: return launch_sample<__nv_bfloat16>(p, a->rows, st);
        case MXFP4_DT_F16: return launch_sample<__half>(p, a->rows, st);
        default: return launch_sample<float>(p, a->rows, st);
    }
}
