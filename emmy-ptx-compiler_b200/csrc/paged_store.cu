// emb_paged_store: norm of each query and key head, position rotation, and the store of keys and values into the pages
// of a cache, in one pass over a step's rows.
//
//   y = x / sqrt(mean(x^2) + eps) * weight;  pairs (a, b) of the first `rot` dims -> (a c - b s, b c + a s)
//
// Bound by HBM on prompts: every element is read once and written once. A head row stays in registers from its load to its
// store: LANES = dim / 8 lanes hold two pieces of four elements each, chosen so that both elements of every pair to be
// rotated are in one lane (pieces j and rot/2 + j of the rotated dims, or eight neighbours), and the mean of squares is a
// butterfly over the lanes. With the norm's weight w, what a row's pair becomes is linear in it but for the norm:
//   a' = r (a [w_a c] - b [w_b s]),  b' = r (b [w_b c] + a [w_a s]),  r = 1 / sqrt(mean + eps)
// and the brackets are a token's and not a row's: a group of LANES lanes takes up to MOST_HEADS heads of one token, the
// next AHEAD of them loaded while AHEAD are at work, and has the brackets, the slot and the addresses ready for all of them. A group has heads of one
// kind only (q, k or v). Measured on 16384 tokens of 32 + 8 + 8 heads of 128, bf16, 407 MB: 79 us = 5.15 TB/s, 0.79 of the
// measured copy rate (with the elements in order, the partners fetched by shuffles and heads of all kinds in a group: 130 us;
// 16-byte pieces of half as many lanes: 101; packed f32x2 arithmetic: no change). Two thirds of the issue slots are taken, by
// addresses, conversions and shuffles as much as by arithmetic, and reads and 256-byte row writes are mixed in HBM; which of the
// two is the bound has not been told apart. Into an e4m3 cache: 72 us, 0.79. With few heads a group's start is a larger part (slot
// or position, then angles and weight, before the first store, and nothing of the next group's meanwhile): 10456 tokens of 8 + 8 +
// 8 heads of 128, f16, 133 MB: 36 us, 0.57. Small steps are bound by the launch: 4.5 us a call for 8 to 1001 tokens.

#include <algorithm>

#include "paged_common.cuh"

namespace {

using namespace emb::paged;

// 2, 8 and 8 CTAs an SM were the best of AHEAD 1, 2, 4, 8, MOST_HEADS 2 to 24 and 5 to 8 CTAs (79 us; the others 80 to 103)
constexpr int THREADS = 128, AHEAD = 2, MOST_HEADS = 8;

// how a launch's groups fall on a token: chunks of `heads` heads of q, of k and of v behind one another
struct Chunks {
    Divisor all;
    int heads, q, k;
};

__device__ __forceinline__ uint2 load_piece(const char* at) {  // not through the read-only path: q may be q_out
    uint2 r;
    asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(at) : "memory");
    return r;
}

enum Kind { Q, K, V };

// the rows of one group, C: the type they are stored in
template <class T, class C, int LANES, bool INTERLEAVED>
__device__ __forceinline__ void rows_of(const emb_paged_store_t& a, Kind kind, int count, const char* from, int64_t from_step, char* to, int64_t to_step, int i, uint32_t mask) {
    const int lane = threadIdx.x % LANES, half = a.rot / 2;
    const bool turns = kind != V && (INTERLEAVED ? lane * 8 : lane * 4) < (INTERLEAVED ? a.rot : half);
    // the dims of this lane's pieces
    const int d0 = INTERLEAVED ? lane * 8 : lane * 4 < half ? lane * 4 : a.rot + (lane * 4 - half) * 2;
    const int d1 = !INTERLEAVED && lane * 4 < half ? half + d0 : d0 + 4;
    const char* const from0 = from + d0 * 2;
    const char* const from1 = from + d1 * 2;
    char* const to0 = to + d0 * static_cast<int>(sizeof(C));
    char* const to1 = to + d1 * static_cast<int>(sizeof(C));

    uint2 next[AHEAD][2];
    const auto load = [&](int h0) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (h0 + u < count) next[u][0] = load_piece(from0 + (h0 + u) * from_step), next[u][1] = load_piece(from1 + (h0 + u) * from_step);
    };
    load(0);

    const T* const weight = static_cast<const T*>(kind == Q ? a.q_weight : kind == K ? a.k_weight : nullptr);
    // x'[e] = r (x[e] own[e] + x[partner of e] other[e])
    float own[8], other[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) own[e] = 1.f, other[e] = 0.f;
    if (weight) {
        Vec4<T>::widen(*reinterpret_cast<const uint2*>(weight + d0), own);
        Vec4<T>::widen(*reinterpret_cast<const uint2*>(weight + d1), own + 4);
    }
    if (turns) {
        const int position = a.positions[i];
        const bool known = position >= 0 && position < a.rope_rows;
        const float* const angles = a.rope + static_cast<long long>(known ? position : 0) * a.rot + lane * 4;
        const float4 c4 = *reinterpret_cast<const float4*>(angles), s4 = *reinterpret_cast<const float4*>(angles + half);
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int x = INTERLEAVED ? 2 * p : p, y = INTERLEAVED ? 2 * p + 1 : p + 4;
            const float cosine = known ? c[p] : __int_as_float(0x7fffffff), wx = own[x], wy = own[y];
            own[x] = wx * cosine, other[x] = -wy * s[p];
            own[y] = wy * cosine, other[y] = wx * s[p];
        }
    }
    const float unit = sizeof(C) == 1 ? 1.f / (kind == K ? a.cache.k_scale : a.cache.v_scale) : 1.f;

    for (int h0 = 0; h0 < count; h0 += AHEAD) {
        uint2 raw[AHEAD][2];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) raw[u][0] = next[u][0], raw[u][1] = next[u][1];
        load(h0 + AHEAD);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (h0 + u >= count) break;
            char* const out0 = to0 + (h0 + u) * to_step;
            char* const out1 = to1 + (h0 + u) * to_step;
            if (sizeof(C) == 2 && kind == V) {
                *reinterpret_cast<uint2*>(out0) = raw[u][0], *reinterpret_cast<uint2*>(out1) = raw[u][1];
                continue;
            }
            float x[8], r = unit;
            Vec4<T>::widen(raw[u][0], x);
            Vec4<T>::widen(raw[u][1], x + 4);
            if (weight) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
                for (int d = LANES / 2; d; d >>= 1) sum += __shfl_xor_sync(mask, sum, d);
                r *= rsqrtf(fmaf(sum, 1.f / (LANES * 8), a.eps));
            }
            float y[8];
            if (turns) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int partner = INTERLEAVED ? e ^ 1 : e ^ 4;
                    y[e] = r * fmaf(x[e], own[e], x[partner] * other[e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = r * (x[e] * own[e]);
            }
            *reinterpret_cast<typename Vec4<C>::raw*>(out0) = Vec4<C>::narrow(y);
            *reinterpret_cast<typename Vec4<C>::raw*>(out1) = Vec4<C>::narrow(y + 4);
        }
    }
}

template <class T, class C, int LANES, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS, 8) paged_store_kernel(const emb_paged_store_t a, const Chunks chunks) {
    const uint32_t mask = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << ((threadIdx.x & 31) / LANES * LANES);  // the group's lanes
    follow_on();
    const uint32_t work = blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES, i = chunks.all.over(work);
    if (i >= static_cast<uint32_t>(a.tokens)) return;
    const int chunk = work - i * chunks.all.d;
    if (chunk < chunks.q) {
        const int h = chunk * chunks.heads;
        rows_of<T, T, LANES, INTERLEAVED>(a, Q, min(chunks.heads, a.heads - h), static_cast<const char*>(a.q) + (i * a.q_stride[0] + h * a.q_stride[1]) * 2, a.q_stride[1] * 2,
                                          static_cast<char*>(a.q_out) + (i * a.out_stride[0] + h * a.out_stride[1]) * 2, a.out_stride[1] * 2, i, mask);
        return;
    }
    const int slot = a.slots[i];
    if (slot < 0 || slot >= a.cache.pages * a.cache.page_size) return;
    const int64_t page = slot / a.cache.page_size, in_page = slot % a.cache.page_size;
    const bool is_k = chunk < chunks.q + chunks.k;
    const int h = (chunk - chunks.q - (is_k ? 0 : chunks.k)) * chunks.heads;
    const int64_t* const stride = is_k ? a.cache.k_stride : a.cache.v_stride;
    const int64_t* const from_stride = is_k ? a.k_stride : a.v_stride;
    constexpr int SIZE = sizeof(C);
    rows_of<T, C, LANES, INTERLEAVED>(a, is_k ? K : V, min(chunks.heads, a.cache.kv_heads - h), static_cast<const char*>(is_k ? a.k : a.v) + (i * from_stride[0] + h * from_stride[1]) * 2, from_stride[1] * 2,
                                      static_cast<char*>(is_k ? a.cache.k : a.cache.v) + (page * stride[0] + in_page * stride[1] + h * stride[2]) * SIZE, stride[2] * SIZE, i, mask);
}

template <class T, class C, int LANES> int run(const emb_paged_store_t& a, cudaStream_t stream) {
    constexpr int GROUPS = THREADS / LANES;
    const int sms = sm_count();
    if (!sms) return refuse("paged_store: the current device cannot be asked for its SMs");
    // a head per group while there are fewer rows than places for groups, then more
    const int64_t rows = static_cast<int64_t>(a.tokens) * (a.heads + 2 * a.cache.kv_heads), places = static_cast<int64_t>(sms) * 8 * GROUPS;
    const int heads = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rows / places, MOST_HEADS)));
    const int q = (a.heads + heads - 1) / heads, k = (a.cache.kv_heads + heads - 1) / heads, all = q + 2 * k;
    const int64_t work = static_cast<int64_t>(a.tokens) * all;
    if (work >= (1ll << 31) - GROUPS) return refuse("paged_store: %d rows of %d heads in one call", a.tokens, a.heads);
    const auto kernel = a.interleaved ? paged_store_kernel<T, C, LANES, true> : paged_store_kernel<T, C, LANES, false>;
    return launched("launch of paged_store", launch(kernel, dim3(static_cast<unsigned>((work + GROUPS - 1) / GROUPS)), THREADS, 0, stream, a, Chunks{Divisor(all), heads, q, k}));
}

template <class T, class C> int run_dim(const emb_paged_store_t& a, cudaStream_t stream) {
    return a.cache.dim == 64 ? run<T, C, 8>(a, stream) : a.cache.dim == 128 ? run<T, C, 16>(a, stream) : run<T, C, 32>(a, stream);
}

}  // namespace

extern "C" int emb_paged_store(const emb_paged_store_t* args, void* stream) {
    if (!args) return refuse("paged_store: null arguments");
    const emb_paged_store_t& a = *args;
    if (int r = check_cache("paged_store", a.cache, a.dtype)) return r;
    if (a.tokens < 0 || a.heads < 1 || a.heads > 65535) return refuse("paged_store: %d rows of %d heads", a.tokens, a.heads);
    if (a.rot < 0 || a.rot > a.cache.dim || a.rot % 16) return refuse("paged_store: rotation of %d dims: a multiple of 16 up to the head dim %d", a.rot, a.cache.dim);
    if (a.rot && (!a.rope || !aligned16(a.rope) || a.rope_rows < 1)) return refuse("paged_store: a rotation without a table, or one that is not 16-byte aligned");
    if (!(a.eps >= 0.f)) return refuse("paged_store: eps is negative or NaN");
    for (const void* p : {a.q_weight, a.k_weight})
        if (!aligned16(p)) return refuse("paged_store: a norm weight is not 16-byte aligned");
    if (a.tokens == 0) return 0;
    if (!a.slots || (a.rot && !a.positions)) return refuse("paged_store: null slots or positions");
    for (const void* p : {a.q, a.k, a.v, static_cast<const void*>(a.q_out)})
        if (!p || !aligned16(p)) return refuse("paged_store: q, k, v or q_out is null or not 16-byte aligned");
    for (const int64_t* s : {a.q_stride, a.k_stride, a.v_stride, a.out_stride})
        if (!stride_fits(s[0], 2) || !stride_fits(s[1], 2)) return refuse("paged_store: a stride of q, k, v or q_out is not a multiple of 16 bytes below 2^32 elements");
    const int64_t rows[2] = {a.tokens, a.heads}, slots[3] = {a.cache.pages, a.cache.page_size, a.cache.kv_heads};
    if (!rows_apart(rows, a.out_stride, a.cache.dim)) return refuse("paged_store: rows of q_out overlap");
    if (!rows_apart(slots, a.cache.k_stride, a.cache.dim) || !rows_apart(slots, a.cache.v_stride, a.cache.dim)) return refuse("paged_store: slots of the cache overlap");
    const int64_t n = a.tokens;
    const int kv_heads = a.cache.kv_heads, dim = a.cache.dim;
    const Area written[3] = {rows_at("q_out", a.q_out, n, a.heads, dim, a.out_stride), pages_at("the keys' pages", a.cache, a.cache.k, a.cache.k_stride),
                             pages_at("the values' pages", a.cache, a.cache.v, a.cache.v_stride)};
    const Area read[8] = {rows_at("q", a.q, n, a.heads, dim, a.q_stride), rows_at("k", a.k, n, kv_heads, dim, a.k_stride), rows_at("v", a.v, n, kv_heads, dim, a.v_stride),
                          Area("slots", a.slots, n * 4), Area("positions", a.rot ? a.positions : nullptr, n * 4),
                          Area("rope", a.rot ? a.rope : nullptr, int64_t(a.rope_rows) * a.rot * 4), Area("q_weight", a.q_weight, dim * 2), Area("k_weight", a.k_weight, dim * 2)};
    const char* which[2];
    if (touches(written, read, &read[0], which)) return refuse("paged_store: %s and %s share memory", which[0], which[1]);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.dtype == EMB_F16) return a.cache.dtype == EMB_U8 ? run_dim<__half, E4m3>(a, s) : run_dim<__half, __half>(a, s);
    return a.cache.dtype == EMB_U8 ? run_dim<__nv_bfloat16, E4m3>(a, s) : run_dim<__nv_bfloat16, __nv_bfloat16>(a, s);
}
