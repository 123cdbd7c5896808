// Rotary positions on the way into a paged key/value cache: one launch between the q|k|v projection and attention.
//
// For token n at position p, pair i of a head (i < rotary/2) and angle a = p * inv_freq[i]:
//   (y0, y1) = scaling * (x0 cos a - x1 sin a,  x0 sin a + x1 cos a)
// on the elements (i, i + rotary/2) of the head (half layout) or (2i, 2i + 1) (interleaved layout); elements from `rotary`
// on are left alone, unscaled.  q goes to q_out, k to row slots[n] of the cache (page slots[n] / page_size), v there as it
// is.  The angle is formed and reduced to a fraction of a turn in 64 bits, because a float32 angle of position 10^6 is
// already 0.06 rad off; sine and cosine of the reduced angle, and the rotation, are float32, rounded once to the type.
//
// HBM-bound: (heads + 2 kv_heads) * head_dim elements of a token in and out.  A CTA takes two tokens (or a part of one's heads,
// when there are few), puts their sines and cosines in shared memory once for all heads, and moves 8 elements per load; a
// thread owns both members of its pairs, so q_out may be q itself.  Measured: 8191 tokens of 64 + 8 heads of 128, float16: 77 us =
// 4.4 TB/s, two thirds of the copy bandwidth.
#include "mxfp4_common.cuh"

namespace mxfp4 {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kMaxPairs = 512;           // sines and cosines of a CTA: of one token or of several
// Tokens per CTA where there are many: the second one's loads follow the first one's stores without the wait for slot and
// angles.  8191 tokens of 64 + 8 heads of 128: 83 us with one, 77 with two, 84 with four and eight.
constexpr int kPer = 2;

struct RopeParams {
    const void *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    void* q_out;
    int64_t qo_row, qo_head;
    void *kc, *vc;
    int64_t kc_page, kc_head, kc_token, vc_page, vc_head, vc_token;
    const int64_t *positions, *slots;
    const double* inv_freq;
    double scaling;
    int64_t num_slots, tokens;
    int per;                                 // tokens per CTA
    int heads, kv_heads, head_dim, rotary, interleaved, page_size;
    int* status;
};

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int W>
struct alignas(sizeof(T) * W < 16 ? sizeof(T) * W : 16) Chunk {
    T e[W];
};

// W = 8: chunks of eight elements, everything 16-byte aligned; W = 1: any stride, any even rotary width
template <typename T, int W, bool kInter>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const RopeParams p) {
    MXFP4_CHAIN_PROLOGUE();
    __shared__ float2 turns[kMaxPairs];
    __shared__ int64_t places[kPer][2];                               // page and row of the slot; page -1: not stored
    const int64_t n0 = (int64_t)blockIdx.x * p.per;
    const int pairs = p.rotary >> 1, count = p.tokens - n0 < p.per ? (int)(p.tokens - n0) : p.per;
    if (threadIdx.x < count) {
        const int64_t slot = p.slots[n0 + threadIdx.x];
        const bool keep = slot >= 0 && slot < p.num_slots;
        if (!keep && slot >= 0 && blockIdx.y == 0 && p.status) atomicExch(p.status, MXFP4_E_BADARG);
        places[threadIdx.x][0] = keep ? slot / p.page_size : -1;
        places[threadIdx.x][1] = keep ? slot % p.page_size : 0;
    }
    for (int i = threadIdx.x; i < count * pairs; i += kRopeThreads) {
        const int token = i / pairs;
        const double t = (double)p.positions[n0 + token] * p.inv_freq[i - token * pairs] * 0.15915494309189533577;      // turns
        float s, c;
        sincospif(2.0f * (float)(t - rint(t)), &s, &c);
        turns[i] = make_float2((float)(c * p.scaling), (float)(s * p.scaling));
    }
    __syncthreads();
    for (int token = 0; token < count; ++token) {
        const int64_t n = n0 + token;
        const float2* turn = turns + token * pairs;
        const int64_t* place = places[token];
        const bool keep = place[0] >= 0;

        // Units of a rotated head: in the half layout a chunk of the first half with its partner of the second, and the chunks
        // behind; else its chunks.  A thread steps from unit to unit without a division.
        const int turned = kInter ? 0 : pairs / W, units = turned + (kInter ? p.head_dim : p.head_dim - p.rotary) / W;
        const int first = blockIdx.y * kRopeThreads + threadIdx.x, step = kRopeThreads * gridDim.y;
        {
            const int dh = step / units, dw = step - dh * units, heads = keep ? p.heads + p.kv_heads : p.heads;
            const T *q = (const T*)p.q + n * p.q_row, *k = (const T*)p.k + n * p.k_row;
            T *qo = (T*)p.q_out + n * p.qo_row, *kc = (T*)p.kc + place[0] * p.kc_page + place[1] * p.kc_token;
            int h = first / units, w = first - h * units;
            while (h < heads) {
                const T* src[2];
                T* dst[2];
                Chunk<T, W> a[2], b[2];
                int at[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {                                   // two units' loads under way together
                    src[i] = nullptr;
                    if (h < heads) {
                        at[i] = w < turned || kInter ? w * W : p.rotary + (w - turned) * W;
                        const bool of_q = h < p.heads;
                        src[i] = (of_q ? q + h * p.q_head : k + (h - p.heads) * p.k_head) + at[i];
                        dst[i] = (of_q ? qo + h * p.qo_head : kc + (h - p.heads) * p.kc_head) + at[i];
                        if (W == 1 && kInter && at[i] < p.rotary) {
                            if (at[i] & 1) src[i] = nullptr;                    // the even member's thread turns the pair
                            else { a[i].e[0] = src[i][0]; b[i].e[0] = src[i][1]; }
                        } else {
                            a[i] = *reinterpret_cast<const Chunk<T, W>*>(src[i]);
                            if (!kInter && at[i] < pairs) b[i] = *reinterpret_cast<const Chunk<T, W>*>(src[i] + pairs);
                        }
                    }
                    h += dh;
                    w += dw;
                    if (w >= units) { w -= units; ++h; }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (!src[i]) continue;
                    if (!kInter && at[i] < pairs) {
#pragma unroll
                        for (int e = 0; e < W; ++e) {
                            const float2 cs = turn[at[i] + e];
                            const float x0 = to_f32<T>(a[i].e[e]), x1 = to_f32<T>(b[i].e[e]);
                            a[i].e[e] = from_f32<T>(x0 * cs.x - x1 * cs.y);
                            b[i].e[e] = from_f32<T>(x0 * cs.y + x1 * cs.x);
                        }
                        *reinterpret_cast<Chunk<T, W>*>(dst[i] + pairs) = b[i];
                    } else if (kInter && at[i] < p.rotary) {
#pragma unroll
                        for (int e = 0; e < W; e += 2) {
                            const float2 cs = turn[(at[i] + e) >> 1];
                            T& partner = W == 1 ? b[i].e[0] : a[i].e[W == 1 ? 0 : e + 1];
                            const float x0 = to_f32<T>(a[i].e[e]), x1 = to_f32<T>(partner);
                            a[i].e[e] = from_f32<T>(x0 * cs.x - x1 * cs.y);
                            partner = from_f32<T>(x0 * cs.y + x1 * cs.x);
                        }
                        if (W == 1) dst[i][1] = b[i].e[0];
                    }
                    *reinterpret_cast<Chunk<T, W>*>(dst[i]) = a[i];
                }
            }
        }
        if (keep) {
            const int per = p.head_dim / W, dh = step / per, dw = step - dh * per;
            const T* v = (const T*)p.v + n * p.v_row;
            T* vc = (T*)p.vc + place[0] * p.vc_page + place[1] * p.vc_token;
            for (int h = first / per, w = first - h * per; h < p.kv_heads;) {
                *reinterpret_cast<Chunk<T, W>*>(vc + h * p.vc_head + w * W) = *reinterpret_cast<const Chunk<T, W>*>(v + h * p.v_head + w * W);
                h += dh;
                w += dw;
                if (w >= per) { w -= per; ++h; }
            }
        }
    }
}

template <typename T>
int launch_rope(RopeParams p, int64_t tokens, bool wide, cudaStream_t st) {
    // few tokens: a token's heads are spread over CTAs, so that one token is not one SM's work; each has 128 units at least
    p.tokens = tokens;
    const int pairs = p.rotary > 2 ? p.rotary / 2 : 1;
    p.per = kPer;
    while (p.per > 1 && (p.per * pairs > kMaxPairs || tokens < (int64_t)p.per * 8 * num_sms())) p.per /= 2;
    const int64_t units = (int64_t)(p.heads + 2 * p.kv_heads) * (p.head_dim / (wide ? 8 : 1));
    int64_t split = 2 * (int64_t)num_sms() / tokens, most = (units + 127) / 128;
    split = split < 1 ? 1 : (split > most ? most : split);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((tokens + p.per - 1) / p.per), (unsigned)split, 1);
    cfg.blockDim = dim3(kRopeThreads, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    void (*const kernel)(RopeParams) = p.interleaved ? (wide ? rope_append_kernel<T, 8, true> : rope_append_kernel<T, 1, true>)
                                                     : (wide ? rope_append_kernel<T, 8, false> : rope_append_kernel<T, 1, false>);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess) return cuda_fail(e, "mxfp4_rope_append");
    return MXFP4_OK;
}

}  // namespace
}  // namespace mxfp4

extern "C" int mxfp4_rope_append(const mxfp4_rope_append_args* a, void* stream) {
    using namespace mxfp4;
    if (!a) { set_error("mxfp4_rope_append: null arguments"); return MXFP4_E_BADARG; }
    if (a->dtype != MXFP4_DT_BF16 && a->dtype != MXFP4_DT_F16 && a->dtype != MXFP4_DT_F32) { set_error("mxfp4_rope_append: unknown dtype %d", a->dtype); return MXFP4_E_BADARG; }
    if (a->tokens < 0 || a->heads < 0 || a->kv_heads < 0 || a->head_dim <= 0 || a->num_pages < 0 || a->page_size <= 0) { set_error("mxfp4_rope_append: negative size"); return MXFP4_E_SHAPE; }
    if (a->rotary < 0 || a->rotary % 2 || a->rotary > a->head_dim || a->rotary > 2 * kMaxPairs) {
        set_error("mxfp4_rope_append: rotary width %d must be even, at most the head's %d and at most %d", a->rotary, a->head_dim, 2 * kMaxPairs);
        return MXFP4_E_SHAPE;
    }
    if (a->tokens == 0 || a->heads + a->kv_heads == 0) return MXFP4_OK;
    if (a->tokens > 0x7FFFFFFF || (int64_t)(a->heads + 2 * (int64_t)a->kv_heads) * a->head_dim > 0x3FFFFFFF) { set_error("mxfp4_rope_append: size too large"); return MXFP4_E_SHAPE; }
    if (!a->positions || !a->slots || (a->rotary && !a->inv_freq) || (a->heads && (!a->q || !a->q_out)) ||
        (a->kv_heads && (!a->k || !a->v || !a->k_cache || !a->v_cache))) {
        set_error("mxfp4_rope_append: null pointer");
        return MXFP4_E_BADARG;
    }
    RopeParams p;
    p.q = a->q; p.k = a->k; p.v = a->v; p.q_out = a->q_out; p.kc = a->k_cache; p.vc = a->v_cache;
    const int64_t n = a->tokens, h = a->heads, kv = a->kv_heads;
    p.q_row = used_stride(a->q_stride[0], n); p.q_head = used_stride(a->q_stride[1], h); p.k_row = used_stride(a->k_stride[0], n);
    p.k_head = used_stride(a->k_stride[1], kv); p.v_row = used_stride(a->v_stride[0], n); p.v_head = used_stride(a->v_stride[1], kv);
    p.qo_row = used_stride(a->q_out_stride[0], n); p.qo_head = used_stride(a->q_out_stride[1], h);
    p.kc_page = used_stride(a->k_cache_stride[0], a->num_pages); p.kc_head = used_stride(a->k_cache_stride[1], kv);
    p.kc_token = used_stride(a->k_cache_stride[2], a->page_size);
    p.vc_page = used_stride(a->v_cache_stride[0], a->num_pages); p.vc_head = used_stride(a->v_cache_stride[1], kv);
    p.vc_token = used_stride(a->v_cache_stride[2], a->page_size);
    p.positions = a->positions; p.slots = a->slots; p.inv_freq = a->inv_freq; p.scaling = a->scaling;
    p.num_slots = a->num_pages * a->page_size; p.page_size = a->page_size;
    p.heads = a->heads; p.kv_heads = a->kv_heads; p.head_dim = a->head_dim; p.rotary = a->rotary; p.interleaved = a->interleaved ? 1 : 0;
    p.status = a->status_dev;
    // eight elements per access wherever every row starts on 16 bytes and no chunk crosses the end of the rotated part
    const int64_t strides = p.q_row | p.q_head | p.k_row | p.k_head | p.v_row | p.v_head | p.qo_row | p.qo_head | p.kc_page | p.kc_head | p.kc_token |
                            p.vc_page | p.vc_head | p.vc_token;
    const uintptr_t ptrs = (uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.q_out | (uintptr_t)p.kc | (uintptr_t)p.vc;
    const bool wide = strides % 8 == 0 && ptrs % 16 == 0 && p.head_dim % 8 == 0 && p.rotary % (p.interleaved ? 8 : 16) == 0;
    cudaStream_t st = (cudaStream_t)stream;
    switch (a->dtype) {
        case MXFP4_DT_BF16: return launch_rope<__nv_bfloat16>(p, a->tokens, wide, st);
        case MXFP4_DT_F16: return launch_rope<__half>(p, a->tokens, wide, st);
        default: return launch_rope<float>(p, a->tokens, wide, st);
    }
}
