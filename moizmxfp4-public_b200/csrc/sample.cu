// The next token of every row of logits from one given uniform number: temperature, top-k, top-p, min-p.
//
// Tokens are taken in descending order of their logits, equal ones by index, and every filter keeps a beginning of that
// order; so all that a filter has to yield is the weight of what it keeps, and the kept weight is the smallest of them.
// The k-th token, the last token of top-p and the sampled one are all "the first token whose cumulative count or weight
// reaches a target", which one routine finds without sorting the row: a histogram of counts and weights over 128 bins that
// are linear in the scaled logit finds the bin, a second one over 128 parts of that bin its part where the bin is full, and
// the few tokens of that are put in order in shared memory.  Where the bins up to the target hold few tokens altogether (top-k of
// 40, a narrow top-p), all of them are put in order once and the later targets are read off.  Bins and parts are intervals of
// logits, so that a look at the row for the tokens of one costs two comparisons each.  (Thousands of equal logits: radix
// histograms over their keys and a count in index order instead.)
//
// Weights are fixed-point: rint(exp((l - max) / T) * 2^shift) with 2^shift * vocab < 2^63, the exponential in 64 bits by a
// table of 2^(j/256) and a polynomial (Tang's method), within 2^-42 of its value.  Sums of integers do not depend on the order of the additions, so
// atomics on the histograms leave nothing to chance, and 45 bits after the point at a vocabulary of 2^17 keep cumulative
// weights good to 1e-11, where float32 sums would move borders between tokens by 1e-7 and change what is sampled.
//
// One CTA of 1024 threads per row; few long rows are divided among the CTAs of a cluster, which add up their histograms and
// exchange the lists of a bin's tokens, and many rows that L2 holds are taken by CTAs of 512 threads, two on an SM.  A histogram
// has a column for each lane, so that no two lanes of a warp meet at an address (with one column for all, 131072 logits spent
// most of their time in conflicts).  The row is read from memory once when it fits into shared memory, else again from L2.
// Measured: one row of 32000 bf16 with top-k 40 and top-p 14 us, one of 131072 with top-p 34 us, 128 rows of 32000 37 us
// (latency: barriers and selections one after the other), 257 rows of 131072 float32 189 us (instructions: the weights and the
// histogram's additions take 45% of the cycles, two looks for the tokens of a bin 13% each, the first read 9%).
#include <atomic>
#include <type_traits>

#include "mxfp4_common.cuh"

namespace mxfp4 {
namespace {

constexpr int kBins = 128;                       // linear bins of a level, 32 columns each
constexpr int kParts = 128;                      // parts of a bin; a part is one step of the exponential's table
constexpr int kRadix = 2048;
constexpr int kList = 4608;                      // tokens of a bin that are brought together
constexpr int kSort = 512;                       // tokens that are put in order at most
constexpr int kFew = 256;                        // up to so many without a look at the bin's parts
constexpr int kTable = 256;
constexpr int kMaxRanks = 8;                      // CTAs that share a row

struct SampleParams {
    const void* logits;
    int64_t ld;
    int vocab, shift, cached, ranks;
    const float *uniforms, *temperature, *top_p, *min_p;
    const int* top_k;
    double temperature_value, top_p_value, min_p_value;
    int64_t top_k_value;
    int64_t* tokens;
    float* logprobs;
};

// Order-preserving key, inverted: ascending keys are descending logits.  -0 is 0.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t u = __float_as_uint(l + 0.0f);
    return (u & 0x80000000u) ? u : ~(u | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key : (~key & 0x7FFFFFFFu)); }

struct SampleShared {
    union {
        struct { uint32_t count[kBins][32], lo[kBins][32], hi[kBins][32]; } bins;
        struct { uint32_t count[kRadix], lo[kRadix], hi[kRadix]; } radix;
        struct { uint64_t list[kList], part[kSort], order[kSort]; };   // key << 32 | index: of a bin, of a part of it, in order
    };
    uint64_t weight[2][kBins];                   // sums of the bins: [0] the row's, [1] the parts of one of them
    uint32_t count[2][kBins];
    double table[kTable];
    uint64_t warp64[32];
    uint32_t warp32[32];
    uint64_t found[4];
    uint32_t listed, part_count[kParts], part_lo[kParts], part_hi[kParts], ends[2];
    uint64_t own_weight[2][kBins];               // this CTA's part of a level's sums
    uint32_t own_count[2][kBins];
    uint32_t place[kSort];
    uint64_t told[2];                            // a number for the other CTAs of the row, two in turn
};

// The CTAs of a row, a cluster: what one has in shared memory is read by the others behind a barrier of all.
template <bool kMany>
struct Ranks {
    int rank_, count_;
    uint32_t turn;

    __device__ __forceinline__ int rank() const { return kMany ? rank_ : 0; }
    __device__ __forceinline__ int count() const { return kMany ? count_ : 1; }

    __device__ __forceinline__ void sync() const {
        if (kMany) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
        else __syncthreads();
    }
    // rank r's copy of a variable in shared memory
    template <typename U>
    __device__ __forceinline__ const volatile U* of(const U* own, int r) const {
        if (!kMany) return own;
        uint64_t a;
        asm("mapa.u64 %0, %1, %2;" : "=l"(a) : "l"((uint64_t)own), "r"(r));
        return (const volatile U*)a;
    }
    // In lane r of every warp what rank r said, and `none` in the lanes behind.  A slot is written again two calls later, behind
    // the barrier of the call between, at which all ranks have read it.
    __device__ __forceinline__ uint64_t say(SampleShared& sh, uint64_t v, uint64_t none) {
        const int lane = threadIdx.x & 31;
        uint64_t* slot = &sh.told[turn++ & 1];
        if (threadIdx.x == 0) *slot = v;
        sync();
        return lane < count() ? *of(slot, lane) : none;
    }
    __device__ __forceinline__ uint64_t sum(uint64_t x) const {                // of a warp's lanes
#pragma unroll
        for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
        return x;
    }
};

struct Place {
    uint32_t key;                                // of the token
    int64_t index;
    uint64_t weight;                             // of all tokens up to and with it
};

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
    using type = __nv_bfloat162;
    static __device__ __forceinline__ type both_down(float x) { return __bfloat162bfloat162(__float2bfloat16_rd(x)); }
    static __device__ __forceinline__ type both_up(float x) { return __bfloat162bfloat162(__float2bfloat16_ru(x)); }
};
template <> struct Pair<__half> {
    using type = __half2;
    static __device__ __forceinline__ type both_down(float x) { return __half2half2(__float2half_rd(x)); }
    static __device__ __forceinline__ type both_up(float x) { return __half2half2(__float2half_ru(x)); }
};

template <typename T, int kThreads, bool kMany>
struct Sampler {
    static constexpr int kWarps = kThreads / 32;
    static constexpr int kVec = 16 / sizeof(T);
    const SampleParams& p;
    SampleShared& sh;
    const T* src;                                // the row
    uint4* cache;
    int head, chunks;                            // whole 16-byte chunks begin behind `head` logits
    int begin_, end_;                            // this CTA's chunks of them
    Ranks<kMany> ranks;
    bool cached;
    double inv_t, top, least;                    // least: (l - max) / T below which a weight rounds to nothing
    uint32_t sorted = 0;                         // that many first tokens of the row are in order, one per thread:
    uint64_t token = 0, ahead = 0, mass = 0;     // key << 32 | index, the weight in front of it, its own

    __device__ __forceinline__ int begin() const { return kMany ? begin_ : 0; }
    __device__ __forceinline__ int end() const { return kMany ? end_ : chunks; }

    // f(index, logit) for every logit; a warp's lanes take neighbouring chunks
    template <typename F>
    __device__ __forceinline__ void each(F f, bool from_memory = false, bool keep = false) {
        const uint4* whole = reinterpret_cast<const uint4*>(src + head);
        for (int c = begin() + threadIdx.x; c < end(); c += kThreads) {
            union { uint4 v; T e[kVec]; } x;
            x.v = cached && !from_memory ? cache[c - begin()] : whole[c];
            if (keep) cache[c - begin()] = x.v;
            const int i0 = head + c * kVec;
#pragma unroll
            for (int k = 0; k < kVec; ++k) f(i0 + k, to_f32<T>(x.e[k]));
        }
        edges(f);
    }
    // f(index, logit) for what lies in front of the first whole chunk and behind the last
    template <typename F>
    __device__ __forceinline__ void edges(F f) {
        if (ranks.rank()) return;
        const int behind = head + chunks * kVec;
        if ((int)threadIdx.x < head) f((int)threadIdx.x, to_f32<T>(src[threadIdx.x]));
        if (behind + (int)threadIdx.x < p.vocab) f(behind + (int)threadIdx.x, to_f32<T>(src[behind + threadIdx.x]));
    }

    // g(logits) for every whole chunk and f(logit) for the rest
    template <typename G, typename F>
    __device__ __forceinline__ void each_chunk(G g, F f) {
        const uint4* whole = reinterpret_cast<const uint4*>(src + head);
        for (int c = begin() + threadIdx.x; c < end(); c += kThreads) {
            union { uint4 v; T e[kVec]; } x;
            x.v = cached ? cache[c - begin()] : whole[c];
            float l[kVec];
#pragma unroll
            for (int k = 0; k < kVec; ++k) l[k] = to_f32<T>(x.e[k]);
            g(l);
        }
        edges([&](int, float l) { f(l); });
    }

    static constexpr int kLast = kBins * kParts - 1;
    // Steps of ln 2 / 256 that a logit's scaled distance from the maximum is, and e^x 2^shift.  The steps are the histogram's places:
    // bin = steps / 128, part = steps % 128.  They never fall as the logit falls; NaN counts as -inf.
    // kWide: vocab > 2048, where weights are below 2^52 and no logit above `least` reaches the last steps.
    template <bool kWide = false>
    __device__ __forceinline__ int steps_of(float l, double& r) const {
        const double x = ((double)l - top) * inv_t;
        if (!(x > least)) return kLast;                                        // -inf at any temperature among them
        const double t = fma(x, 369.3299304675746 /* 256 / ln 2 */, 6755399441055744.0 /* 1.5 * 2^52: the nearest integer in the low bits */);
        const int n = -__double2loint(t);
        r = fma(t - 6755399441055744.0, -0.0027076061740622863 /* ln 2 / 256 */, x);
        return kWide || n < kLast ? n : kLast - 1;
    }
    __device__ __forceinline__ double scaled(int steps, double r) const {
        if (steps == kLast) return 0.0;
        double q = fma(r, 1.0 / 6.0, 0.5);                                     // e^r - 1 to r^3: |r| <= ln 2 / 512, r^4 / 24 < 2^-42
        q = fma(r * r, q, r);
        const double s = sh.table[-steps & (kTable - 1)], e = fma(s, q, s);
        return __hiloint2double(__double2hiint(e) + ((p.shift - ((steps + kTable - 1) / kTable)) << 20), __double2loint(e));
    }
    __device__ __forceinline__ uint64_t weight_of(float l) const {
        double r = 0.0;
        const int n = steps_of(l, r);
        return __double2ull_rn(scaled(n, r));
    }
    // The first key whose steps reach `goal`, found by a warp: 32 guesses at a time, from a narrow range around the logit at that
    // distance where the answer lies in there, else from all.
    __device__ __forceinline__ uint32_t first_key(int goal) const {
        const int lane = threadIdx.x & 31;
        uint32_t lo = key_of((float)top), hi = 0xFF800000u;                    // of the maximum, of -inf; hi itself reaches every goal
        auto short_of = [&](uint32_t key) {
            double r;
            return steps_of(logit_of(key), r) < goal;
        };
        const float guess = (float)(top - ((double)goal - 0.5) * (0.0027076061740622863 / inv_t));
        if (guess - guess == 0.0f) {
            const uint32_t g = key_of(guess), from = g > lo + 15 ? g - 15 : lo, to = from + 31 < hi ? from + 31 : hi;
            if (from >= lo && from < to) {
                const uint32_t at = from + lane;
                const uint32_t votes = __ballot_sync(0xFFFFFFFFu, at < to && short_of(at));
                const uint32_t n = __popc(votes);
                // guesses that fall short come first: the answer lies among these keys where the first falls short (or is the
                // maximum's own) and one does not
                if ((n > 0 || from == lo) && from + n < to) return from + n;
            }
        }
        while (lo < hi) {
            const uint32_t step = (hi - lo) / 32 + 1, at = lo + lane * step;
            const uint32_t n = __popc(__ballot_sync(0xFFFFFFFFu, at >= lo && at < hi && short_of(at)));
            const uint32_t old = lo;
            if (n > 0) lo = old + (n - 1) * step + 1;
            if (n < 32 && old + n * step >= old && old + n * step < hi) hi = old + n * step;
        }
        return lo;
    }
    struct Inside {                              // whether a logit's steps are in [from, to)
        float high, low;
        bool nan;
        __device__ __forceinline__ bool operator()(float l) const { return (l <= high && l >= low) || (nan && l != l); }
    };
    __device__ __forceinline__ Inside inside(int from, int to) {
        const int warp = threadIdx.x >> 5;
        if (warp == 0) {
            const uint32_t k = first_key(from);
            if (threadIdx.x == 0) sh.ends[0] = k;
        } else if (warp == 1) {
            const uint32_t k = to > kLast ? 0xFF800000u : first_key(to) - 1;
            if (threadIdx.x == 32) sh.ends[1] = k;
        }
        __syncthreads();
        const Inside in{logit_of(sh.ends[0]), logit_of(sh.ends[1]), to > kLast};
        __syncthreads();
        return in;
    }

    static __device__ __forceinline__ void add64(uint32_t* lo, uint32_t* hi, uint64_t w) {
        const uint32_t l = (uint32_t)w;
        uint32_t h = (uint32_t)(w >> 32);
        if (l && atomicAdd(lo, l) > 0xFFFFFFFFu - l) ++h;                      // a carry
        if (h) atomicAdd(hi, h);
    }
    __device__ __forceinline__ void clear_bins() {
        uint4* b = reinterpret_cast<uint4*>(&sh.bins);
        for (int i = threadIdx.x; i < (int)(sizeof(sh.bins) / 16); i += kThreads) b[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    __device__ __forceinline__ void add_bin(int bin, uint64_t w) {
        const int lane = threadIdx.x & 31;
        atomicAdd(&sh.bins.count[bin][lane], 1u);
        add64(&sh.bins.lo[bin][lane], &sh.bins.hi[bin][lane], w);
    }
    // sums of the columns over all CTAs of the row; the histogram is free again behind it
    __device__ __forceinline__ void sum_bins(int level) {
        __syncthreads();
        const int lane = threadIdx.x & 31;
        for (int b = threadIdx.x >> 5; b < kBins; b += kWarps) {
            // no sum of weights reaches 2^63, so 32 high words add up within 32 bits, and so do halves of the low ones
            const uint32_t lo = sh.bins.lo[b][lane], c = __reduce_add_sync(0xFFFFFFFFu, sh.bins.count[b][lane]);
            const uint64_t w = ((uint64_t)__reduce_add_sync(0xFFFFFFFFu, sh.bins.hi[b][lane]) << 32) +
                               ((uint64_t)__reduce_add_sync(0xFFFFFFFFu, lo >> 16) << 16) + __reduce_add_sync(0xFFFFFFFFu, lo & 0xFFFFu);
            if (lane == 0) (kMany ? sh.own_weight : sh.weight)[level][b] = w;
            if (lane == 0) (kMany ? sh.own_count : sh.count)[level][b] = c;
        }
        ranks.sync();
        if (kMany) share(level);
    }
    // the CTAs' own sums into one; they may be written again behind the next barrier of all
    __device__ __forceinline__ void share(int level) {
        static_assert(kMaxRanks == 8 && (!kMany || kBins * kMaxRanks == kThreads), "a thread for a bin of a CTA");
        const int b = threadIdx.x / kMaxRanks, r = threadIdx.x % kMaxRanks;
        uint64_t w = r < ranks.count() ? ranks.of(sh.own_weight[level], r)[b] : 0;
        uint32_t c = r < ranks.count() ? ranks.of(sh.own_count[level], r)[b] : 0;
#pragma unroll
        for (int d = kMaxRanks / 2; d; d >>= 1) {
            w += __shfl_xor_sync(0xFFFFFFFFu, w, d);
            c += __shfl_xor_sync(0xFFFFFFFFu, c, d);
        }
        if (r == 0) { sh.weight[level][b] = w; sh.count[level][b] = c; }
        __syncthreads();
    }
    // The first bin where the running weight (or count) reaches `target`, which the level's total does; target becomes what
    // is left of it in the bin, before grows by the weight in front.
    __device__ __forceinline__ int find_bin(int level, bool by_weight, uint64_t& target, uint64_t& before, uint64_t& tokens) {
        if (threadIdx.x < 32) {
            const int lane = threadIdx.x, per = kBins / 32;
            uint64_t w = 0, c = 0;
            for (int i = 0; i < per; ++i) { w += sh.weight[level][lane * per + i]; c += sh.count[level][lane * per + i]; }
            uint64_t wi = w, ci = c;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint64_t a = __shfl_up_sync(0xFFFFFFFFu, wi, d), b = __shfl_up_sync(0xFFFFFFFFu, ci, d);
                if (lane >= d) { wi += a; ci += b; }
            }
            uint64_t run_w = wi - w, run_c = ci - c;
            if ((by_weight ? run_w : run_c) < target && target <= (by_weight ? wi : ci)) {
                int b = lane * per;
                for (;; ++b) {
                    const uint64_t bw = sh.weight[level][b], bc = sh.count[level][b];
                    if ((by_weight ? run_w + bw : run_c + bc) >= target || b == lane * per + per - 1) break;
                    run_w += bw;
                    run_c += bc;
                }
                sh.found[0] = (uint64_t)b; sh.found[1] = run_w; sh.found[2] = run_c;
            }
        }
        __syncthreads();
        const int b = (int)sh.found[0];
        before += sh.found[1];
        tokens = sh.found[2];
        target -= by_weight ? sh.found[1] : tokens;
        __syncthreads();
        return b;
    }
    // exclusive sum over the block
    __device__ __forceinline__ uint64_t scan(uint64_t v) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        uint64_t incl = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint64_t a = __shfl_up_sync(0xFFFFFFFFu, incl, d);
            if (lane >= d) incl += a;
        }
        if (lane == 31) sh.warp64[warp] = incl;
        __syncthreads();
        if (warp == 0) {
            uint64_t s = lane < kWarps ? sh.warp64[lane] : 0, si = s;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint64_t a = __shfl_up_sync(0xFFFFFFFFu, si, d);
                if (lane >= d) si += a;
            }
            sh.warp64[lane] = si - s;
        }
        __syncthreads();
        const uint64_t r = sh.warp64[warp] + incl - v;
        __syncthreads();
        return r;
    }

    // The first token whose cumulative weight (or count) reaches `target`; the row's bins are summed in level 0.
    __device__ __forceinline__ Place select(bool by_weight, uint64_t target) {
        if (sorted) return of_sorted(by_weight, target, 0, sorted);            // a later target is never behind an earlier one
        const uint64_t goal = target;
        uint64_t before = 0, tokens = 0;
        const int bin = find_bin(0, by_weight, target, before, tokens);
        // The bin's logits are an interval: from the first key of its first step to the last one in front of the next bin's.
        int from = bin * kParts, to = bin == kBins - 1 ? kLast + 1 : from + kParts;
        uint32_t n = sh.count[0][bin];
        // all up to here, where they are few, since later targets lie among them
        if (tokens + n <= kFew) {
            sorted = (uint32_t)tokens + n;
            collect(inside(0, to));
            return from_list(by_weight, goal, 0, sorted, sh.list);
        }
        Inside in = inside(from, to);
        if (n > kFew) {
            // the bin's parts: from its tokens brought together, or from a second look at the row where they are too many
            if (n <= kList) {
                collect(in);
                for (int i = threadIdx.x; i < kParts; i += kThreads) sh.part_count[i] = sh.part_lo[i] = sh.part_hi[i] = 0;
                __syncthreads();
                for (int i = threadIdx.x; i < (int)n; i += kThreads) {
                    double r = 0.0;
                    const int m = steps_of(logit_of((uint32_t)(sh.list[i] >> 32)), r), q = m & (kParts - 1);
                    atomicAdd(&sh.part_count[q], 1u);
                    add64(&sh.part_lo[q], &sh.part_hi[q], __double2ull_rn(scaled(m, r)));
                }
                __syncthreads();
                if (threadIdx.x < kParts) {
                    sh.weight[1][threadIdx.x] = ((uint64_t)sh.part_hi[threadIdx.x] << 32) + sh.part_lo[threadIdx.x];
                    sh.count[1][threadIdx.x] = sh.part_count[threadIdx.x];
                }
                __syncthreads();
            } else {
                clear_bins();
                each([&](int, float l) {
                    if (!in(l)) return;
                    double r = 0.0;
                    const int m = steps_of(l, r);
                    add_bin(m & (kParts - 1), __double2ull_rn(scaled(m, r)));
                });
                sum_bins(1);
            }
            from += find_bin(1, by_weight, target, before, tokens);
            to = from == kLast ? kLast + 1 : from + 1;
            const uint32_t all = n;
            n = sh.count[1][from & (kParts - 1)];
            in = inside(from, to);
            if (n > kSort) return from_radix(by_weight, target, before, in);
            if (all <= kList) {
                if (threadIdx.x == 0) sh.listed = 0;
                __syncthreads();
                for (int i = threadIdx.x; i < (int)all; i += kThreads) {
                    const uint64_t x = sh.list[i];
                    if (in(logit_of((uint32_t)(x >> 32)))) sh.part[atomicAdd(&sh.listed, 1u)] = x;
                }
                __syncthreads();
                return from_list(by_weight, target, before, n, sh.part);
            }
        }
        collect(in);
        return from_list(by_weight, target, before, n, sh.list);
    }

    // Which logits of a chunk the interval has, a bit each: element k at 16 * (k % 2) + k / 2 for 16-bit types, else at k.
    template <bool kNan>
    static __device__ __forceinline__ uint32_t hits(const uint4& v, const Inside& in) {
        uint32_t m = 0;
        if constexpr (sizeof(T) == 4) {
            const float l[4] = {__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
#pragma unroll
            for (int k = 0; k < 4; ++k) m |= (kNan ? !(l[k] > in.high) && !(l[k] < in.low) : l[k] <= in.high && l[k] >= in.low) ? 1u << k : 0u;
        } else {
            // two comparisons at once; the ends of the interval rounded inwards to the type
            using T2 = typename Pair<T>::type;
            const T2 high = Pair<T>::both_down(in.high), low = Pair<T>::both_up(in.low);
            union { uint4 v; T2 e[4]; } x;
            x.v = v;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                m |= ((kNan ? __hleu2_mask(x.e[j], high) & __hgeu2_mask(x.e[j], low) : __hle2_mask(x.e[j], high) & __hge2_mask(x.e[j], low)) & 0x00010001u) << j;
        }
        return m;
    }
    template <bool kNan>
    __device__ __forceinline__ void list_inside(const Inside& in) {
        const uint4* whole = reinterpret_cast<const uint4*>(src + head);
        const int lane = threadIdx.x & 31;
        auto put = [&](uint32_t at, float l, int i) { sh.list[at] = (uint64_t)key_of(l != l ? -__builtin_huge_valf() : l) << 32 | (uint32_t)i; };
        constexpr int kAhead = 16 / kVec;                                      // 16 logits of each lane, for which a warp takes its room in the list at once
        for (int c = begin() + (threadIdx.x & ~31); c < end(); c += kAhead * kThreads) {
            uint4 x[kAhead];
            uint32_t mine = 0;
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int at = c + a * kThreads + lane;
                if (at < end()) x[a] = cached ? cache[at - begin()] : whole[at];
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
                if (c + a * kThreads + lane < end()) mine |= hits<kNan>(x[a], in) << (4 * a);
            if (!__any_sync(0xFFFFFFFFu, mine)) continue;
            const uint32_t n = __popc(mine);
            uint32_t at = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, at, d);
                if (lane >= d) at += other;
            }
            uint32_t room = 0;
            if (lane == 31) room = atomicAdd(&sh.listed, at);
            at += __shfl_sync(0xFFFFFFFFu, room, 31) - n;
            for (; mine; mine &= mine - 1) {
                const int b = __ffs(mine) - 1, chunk = c + (b & 15) / 4 * kThreads + lane, k = sizeof(T) == 4 ? b & 3 : 2 * (b & 3) + (b >> 4);
                const T l = cached ? reinterpret_cast<const T*>(cache + (chunk - begin()))[k] : src[head + chunk * kVec + k];
                put(at++, to_f32<T>(l), head + chunk * kVec + k);
            }
            __syncwarp();
        }
        edges([&](int i, float l) {
            if (in(l)) put(atomicAdd(&sh.listed, 1u), l, i);
        });
    }

    // the interval's tokens into the list, in any order, in every CTA of the row
    __device__ __forceinline__ void collect(const Inside& in) {
        if (threadIdx.x == 0) sh.listed = 0;
        __syncthreads();
        if (in.nan) list_inside<true>(in);
        else list_inside<false>(in);
        ranks.sync();
        if (!kMany) return;
        // the other CTAs' lists behind this one's own: lane r knows the length of rank r's
        const int lane = threadIdx.x & 31;
        const uint32_t own = sh.listed, theirs = lane < ranks.count() && lane != ranks.rank() ? *ranks.of(&sh.listed, lane) : 0;
        uint32_t upto = theirs;
#pragma unroll
        for (int d = 1; d < kMaxRanks; d <<= 1) {
            const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, upto, d);
            if (lane >= d) upto += other;
        }
        uint32_t ends[kMaxRanks];
#pragma unroll
        for (int r = 0; r < kMaxRanks; ++r) ends[r] = __shfl_sync(0xFFFFFFFFu, upto, r);
        for (uint32_t i = threadIdx.x; i < ends[kMaxRanks - 1]; i += kThreads) {
            int r = 0;
            uint32_t first = 0;
#pragma unroll
            for (int q = 0; q < kMaxRanks - 1; ++q)
                if (i >= ends[q]) { r = q + 1; first = ends[q]; }
            sh.list[own + i] = ranks.of(sh.list, r)[i - first];
        }
        ranks.sync();                                                          // their lists have been read
    }

    // n <= kSort tokens, among which the target is reached
    __device__ __forceinline__ Place from_list(bool by_weight, uint64_t target, uint64_t before, uint32_t n, uint64_t* list) {
        // A token's place is the number of those in front of it.  All threads count: `size` tokens side by side, each thread's share
        // of the others the same within a warp.  (128 rows of 32000 with their own settings: 50 us with a bitonic sort, 38 with this.)
        int size = 128;
        while (size < (int)n) size *= 2;
        if (threadIdx.x < n) sh.place[threadIdx.x] = 0;
        __syncthreads();
        const uint32_t teams = kThreads / size, each_of = (n + teams - 1) / teams, team = threadIdx.x / size, who = threadIdx.x % size;
        if (who < n) {
            const uint64_t mine = list[who];
            const uint32_t last = (team + 1) * each_of < n ? (team + 1) * each_of : n;
            uint32_t place = 0;
#pragma unroll 4
            for (uint32_t i = team * each_of; i < last; ++i) place += list[i] < mine;
            if (place) atomicAdd(&sh.place[who], place);
        }
        __syncthreads();
        if (threadIdx.x < n) sh.order[sh.place[threadIdx.x]] = list[threadIdx.x];
        __syncthreads();
        static_assert(kSort <= kThreads, "a token per thread");
        token = threadIdx.x < n ? sh.order[threadIdx.x] : 0;
        mass = threadIdx.x < n ? weight_of(logit_of((uint32_t)(token >> 32))) : 0;
        ahead = scan(mass);
        return of_sorted(by_weight, target, before, n);
    }
    // among the n tokens that the threads have in order, with `before` in front of them
    __device__ __forceinline__ Place of_sorted(bool by_weight, uint64_t target, uint64_t before, uint32_t n) {
        if (threadIdx.x < n && (by_weight ? ahead < target && target <= ahead + mass : (uint64_t)threadIdx.x + 1 == target)) {
            sh.found[0] = token;
            sh.found[1] = ahead + mass;
        }
        __syncthreads();
        Place r;
        r.key = (uint32_t)(sh.found[0] >> 32);
        r.index = (int64_t)(sh.found[0] & 0xFFFFFFFFu);
        r.weight = before + sh.found[1];
        __syncthreads();
        return r;
    }

    template <typename In>
    __device__ __forceinline__ Place from_radix(bool by_weight, uint64_t target, uint64_t before, const In& inside) {
        uint32_t prefix = 0;
        int used = 0;
        for (int level = 0; level < 3; ++level) {
            const int bits = level < 2 ? 11 : 10, down = 32 - used - bits;
            for (int i = threadIdx.x; i < kRadix; i += kThreads) sh.radix.count[i] = sh.radix.lo[i] = sh.radix.hi[i] = 0;
            __syncthreads();
            each([&](int, float l) {
                const uint32_t k = key_of(l != l ? -__builtin_huge_valf() : l);
                if (!inside(l) || (used && k >> (32 - used) != prefix)) return;
                const uint32_t b = (k >> down) & ((1u << bits) - 1);
                atomicAdd(&sh.radix.count[b], 1u);
                add64(&sh.radix.lo[b], &sh.radix.hi[b], weight_of(l));
            });
            ranks.sync();
            constexpr int kPer = kRadix / kThreads;                            // a thread's bins lie side by side
            uint64_t w[kPer], c[kPer], all_w = 0, all_c = 0;
            for (int i = 0; i < kPer; ++i) {
                const int b = kPer * threadIdx.x + i;
                w[i] = c[i] = 0;
                for (int r = 0; r < ranks.count(); ++r) {
                    w[i] += ((uint64_t)ranks.of(sh.radix.hi, r)[b] << 32) + ranks.of(sh.radix.lo, r)[b];
                    c[i] += ranks.of(sh.radix.count, r)[b];
                }
                all_w += w[i];
                all_c += c[i];
            }
            uint64_t run_w = scan(all_w), run_c = scan(all_c);
            for (int i = 0; i < kPer; ++i) {
                const uint64_t from = by_weight ? run_w : run_c, to = from + (by_weight ? w[i] : c[i]);
                if (from < target && target <= to) { sh.found[0] = kPer * threadIdx.x + i; sh.found[1] = run_w; sh.found[2] = run_c; }
                run_w += w[i];
                run_c += c[i];
            }
            __syncthreads();
            prefix = (prefix << bits) | (uint32_t)sh.found[0];
            before += sh.found[1];
            target -= by_weight ? sh.found[1] : sh.found[2];
            used += bits;
            ranks.sync();                                                      // the others have read this histogram
        }
        // equal logits from here on: the rank-th of them in index order.  CTAs and warps take contiguous runs of the row.
        const uint64_t w = weight_of(logit_of(prefix));
        const uint64_t rank = by_weight ? (target - 1) / (w ? w : 1) : target - 1;
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = (p.vocab + ranks.count() - 1) / ranks.count();
        const int last = (ranks.rank() + 1) * share < p.vocab ? (ranks.rank() + 1) * share : p.vocab, run = (share + kWarps - 1) / kWarps;
        const int i0 = ranks.rank() * share + warp * run, i1 = i0 + run < last ? i0 + run : last;
        auto hit = [&](int i) {
            if (i >= i1) return false;
            const float l = to_f32<T>(src[i]);
            return key_of(l != l ? -__builtin_huge_valf() : l) == prefix;
        };
        uint32_t mine = 0;
        for (int b = i0; b < i1; b += 32) mine += __popc(__ballot_sync(0xFFFFFFFFu, hit(b + lane)));
        const uint64_t first = scan(lane == 0 ? mine : 0);
        if (threadIdx.x == kThreads - 32) sh.found[0] = first + mine;
        if (threadIdx.x == 0) sh.found[3] = 0;
        __syncthreads();
        const uint64_t theirs = ranks.say(sh, sh.found[0], 0);
        const uint64_t ahead = __shfl_sync(0xFFFFFFFFu, first, 0) + ranks.sum(lane < ranks.rank() ? theirs : 0);
        if (rank >= ahead && rank < ahead + mine) {
            uint32_t left = (uint32_t)(rank - ahead);
            for (int b = i0; b < i1; b += 32) {
                const uint32_t votes = __ballot_sync(0xFFFFFFFFu, hit(b + lane));
                const uint32_t c = __popc(votes);
                if (left < c) {
                    if ((votes >> lane & 1) && __popc(votes & ((1u << lane) - 1)) == left) sh.found[3] = (uint64_t)(b + lane);             // of one CTA, 0 in the others
                    break;
                }
                left -= c;
            }
        }
        __syncthreads();
        Place r;
        r.key = prefix;
        r.index = (int64_t)ranks.sum(ranks.say(sh, sh.found[3], 0));
        r.weight = before + (rank + 1) * w;
        __syncthreads();
        return r;
    }
};

template <typename T, int kThreads, bool kMany>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) sample_kernel(const SampleParams p) {
    MXFP4_CHAIN_PROLOGUE();
    extern __shared__ __align__(16) uint8_t smem_raw[];
    SampleShared& sh = *reinterpret_cast<SampleShared*>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Ranks<kMany> ranks{0, p.ranks, 0};
    if (kMany) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(ranks.rank_));
    const int64_t row = kMany ? blockIdx.x / p.ranks : blockIdx.x;
    const T* src = (const T*)p.logits + row * p.ld;
    int head = (int)((16 - (uintptr_t)src % 16) % 16 / sizeof(T));
    if (head > p.vocab) head = p.vocab;
    using S = Sampler<T, kThreads, kMany>;
    const int chunks = (p.vocab - head) / S::kVec, share = (chunks + ranks.count() - 1) / ranks.count();
    const int begin = ranks.rank() * share < chunks ? ranks.rank() * share : chunks, end = begin + share < chunks ? begin + share : chunks;
    S s{p, sh, src, reinterpret_cast<uint4*>(smem_raw + (sizeof(SampleShared) + 15) / 16 * 16), head, chunks, begin, end, ranks, p.cached != 0,
        0.0, 0.0, 0.0};
    static_assert(kTable <= kThreads && kRadix % kThreads == 0, "");
    if (tid < kTable) sh.table[tid] = exp2((double)tid / kTable);

    float top = -__builtin_huge_valf();                                        // the row's maximum; NaN is passed over
    s.each([&](int, float l) { top = fmaxf(top, l); }, true, s.cached);
    auto block_min = [&](uint32_t x) {
        x = __reduce_min_sync(0xFFFFFFFFu, x);
        __syncthreads();
        if (lane == 0) sh.warp32[warp] = x;
        __syncthreads();
        x = __reduce_min_sync(0xFFFFFFFFu, sh.warp32[lane % S::kWarps]);
        return !kMany ? x : __reduce_min_sync(0xFFFFFFFFu, (uint32_t)s.ranks.say(sh, x, 0xFFFFFFFFu));
    };
    top = logit_of(block_min(key_of(top)));
    s.top = top;
    const double heat = p.temperature ? (double)p.temperature[row] : p.temperature_value;
    if (!(heat > 0.0) || top - top != 0.0f) {                                  // greedy, or a maximum that is infinite: its lowest index
        uint32_t first = 0xFFFFFFFFu;
        s.each([&](int i, float l) {
            if ((l == top || (l != l && top == -__builtin_huge_valf())) && (uint32_t)i < first) first = (uint32_t)i;
        });
        first = block_min(first);
        if (tid == 0 && s.ranks.rank() == 0) {
            p.tokens[row] = (int64_t)first;
            if (p.logprobs) p.logprobs[row] = 0.0f;
        }
        if (kMany) s.ranks.sync();                                 // no CTA ends while its numbers are read
        return;
    }
    s.clear_bins();
    const int64_t top_k = p.top_k ? p.top_k[row] : p.top_k_value;
    const double top_p = p.top_p ? (double)p.top_p[row] : p.top_p_value;
    double min_p = p.min_p ? (double)p.min_p[row] : p.min_p_value;
    min_p = min_p > 1.0 ? 1.0 : min_p;
    const double unit = (double)(1ull << p.shift), least_scaled = min_p * unit;
    s.inv_t = 1.0 / heat;
    s.least = -0.69314718055994531 * (p.shift + 2);

    uint64_t above = 0;
    auto weigh = [&](auto wide) {
        // rint(e): below 2^52 the sum with 2^52 has it in its low bits
        auto whole = [&](double e) {
            return wide.value ? (uint64_t)__double_as_longlong(e + 4503599627370496.0) & 0xFFFFFFFFFFFFFull : (uint64_t)__double2ull_rn(e);
        };
        const bool floor = min_p > 0.0;
        s.each_chunk([&](const float (&l)[S::kVec]) {
            // all weights of a chunk before the first histogram access: nothing is read behind an atomic
            int n[S::kVec];
            uint64_t w[S::kVec];
#pragma unroll
            for (int k = 0; k < S::kVec; ++k) {
                double r = 0.0;
                n[k] = s.template steps_of<wide.value>(l[k], r);
                const double e = s.scaled(n[k], r);
                w[k] = whole(e);
                if (floor && e >= least_scaled) above += w[k];
            }
#pragma unroll
            for (int k = 0; k < S::kVec; ++k) s.add_bin(n[k] / kParts, w[k]);
        }, [&](float l) {
            double r = 0.0;
            const int n = s.template steps_of<wide.value>(l, r);
            const double e = s.scaled(n, r);
            const uint64_t w = whole(e);
            s.add_bin(n / kParts, w);
            if (floor && e >= least_scaled) above += w;
        });
    };
    if (p.shift < 51) weigh(std::true_type{});
    else weigh(std::false_type{});
    s.sum_bins(0);
    uint64_t kept = 0;
#pragma unroll
    for (int b = lane; b < kBins; b += 32) kept += sh.weight[0][b];
#pragma unroll
    for (int d = 16; d; d >>= 1) kept += __shfl_xor_sync(0xFFFFFFFFu, kept, d);
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
    if (min_p > 0.0) {
        const uint64_t ahead = s.scan(above);
        if (tid == kThreads - 1) sh.found[3] = ahead + above;
        __syncthreads();
        const uint64_t all = s.ranks.sum(s.ranks.say(sh, sh.found[3], 0));
        kept = all < kept ? all : kept;
        __syncthreads();
    }
    const double u = (double)p.uniforms[row];
    uint64_t target = u > 0.0 ? (u < 1.0 ? (uint64_t)(u * (double)kept) : kept) : 0;
    target = target < kept ? target + 1 : kept;
    const Place pick = s.select(true, target);
    if (tid == 0 && s.ranks.rank() == 0) {
        p.tokens[row] = pick.index;
        if (p.logprobs) p.logprobs[row] = (float)(((double)logit_of(pick.key) - s.top) * s.inv_t - log((double)kept / unit));
    }
    if (kMany) s.ranks.sync();
}

template <typename T, int kThreads, bool kMany>
int launch_sample_with(SampleParams& p, int64_t rows, int64_t fixed, int64_t row, cudaStream_t st) {
    static std::atomic<bool> configured[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(sample_kernel<T, kThreads, kMany>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e != cudaSuccess) return cuda_fail(e, "mxfp4_sample: cudaFuncSetAttribute");
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * p.ranks), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = (size_t)(fixed + (p.cached ? row : 0));
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.ranks > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T, kThreads, kMany>, p);
    if (e != cudaSuccess) return cuda_fail(e, "mxfp4_sample");
    return MXFP4_OK;
}

template <typename T>
int launch_sample(SampleParams& p, int64_t rows, cudaStream_t st) {
    const int64_t fixed = (int64_t)(sizeof(SampleShared) + 15) / 16 * 16;
    // CTAs for a row, as many as run at once: a cluster of 8 needs 8 free SMs of one GPC, so that 16 of them take two turns (16 rows
    // of 32000: 29 us, with clusters of 4 15 us).  One row of 131072: 96 us with one CTA, 47 with 4, 40 with 8; one of 4096, where the
    // exchange costs more than it saves: 10 us with one CTA, 13 with 2.
    p.ranks = 1;
    if (p.vocab >= 8192) p.ranks = 16 * rows <= num_sms() ? 8 : 9 * rows <= 2 * num_sms() ? 4 : 2 * rows <= num_sms() ? 2 : 1;
    const int64_t row = ((p.vocab + p.ranks - 1) / p.ranks * (int64_t)sizeof(T) + 47) / 16 * 16;
    // Two CTAs on an SM hide each other's barriers (600 rows of 32000: 148 us with one, 132 with two; 290 of 10000: 55 and 38) where
    // there are rows enough for both (160 rows of 32000: 50 and 65) and L2 holds all that are under way (257 of 131072 float32: 201
    // and 244).
    const bool halves = 2 * rows >= 3 * num_sms() && 2 * num_sms() * row <= (64 << 20);
    p.cached = fixed + row <= (halves ? 113 : 227) * 1024;
    if (p.ranks > 1) return launch_sample_with<T, 1024, true>(p, rows, fixed, row, st);
    return halves ? launch_sample_with<T, 512, false>(p, rows, fixed, row, st) : launch_sample_with<T, 1024, false>(p, rows, fixed, row, st);
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
