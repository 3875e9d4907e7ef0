// emb_paged_store: norm of each query and key head, position rotation, and the store of keys and values into the pages
// of a cache, in one pass over a step's rows.
//
//   y = x / sqrt(mean(x^2) + eps) * weight;  pairs (a, b) of the first `rot` dims -> (a c - b s, b c + a s)
//
// Bound by HBM on prompts: every element is read once and written once, so a head row stays in registers from its load to
// its store: LANES = dim / 8 lanes hold eight elements each (one 16-byte access), the mean is a butterfly over them, and
// in the half-split rotation an element's partner is in the same register of the lane rot / 16 away.

#include "paged_common.cuh"

namespace {

using namespace emb::paged;

constexpr int THREADS = 128;

template <class T, class C, int LANES> __global__ void __launch_bounds__(THREADS) paged_store_kernel(const emb_paged_store_t a) {
    const int lane = threadIdx.x % LANES;
    follow_on();
    const int all_heads = a.heads + 2 * a.cache.kv_heads;
    const long long rows = static_cast<long long>(a.tokens) * all_heads;
    const long long row = static_cast<long long>(blockIdx.x) * (THREADS / LANES) + threadIdx.x / LANES;
    const bool real = row < rows;
    const int i = real ? static_cast<int>(row / all_heads) : 0;
    const int h = real ? static_cast<int>(row % all_heads) : 0;
    const bool is_q = h < a.heads, is_v = h >= a.heads + a.cache.kv_heads;
    const int kv = is_q ? 0 : is_v ? h - a.heads - a.cache.kv_heads : h - a.heads;
    const T* from = is_q   ? static_cast<const T*>(a.q) + i * a.q_stride[0] + h * a.q_stride[1]
                    : is_v ? static_cast<const T*>(a.v) + i * a.v_stride[0] + kv * a.v_stride[1]
                           : static_cast<const T*>(a.k) + i * a.k_stride[0] + kv * a.k_stride[1];
    float x[8];
    Vec8<T>::widen(*reinterpret_cast<const uint4*>(from + lane * 8), x);

    const void* weight = is_q ? a.q_weight : a.k_weight;
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += x[e] * x[e];
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (weight && !is_v) {
        const float inv = rsqrtf(sum / (LANES * 8) + a.eps);
        float w[8];
        Vec8<T>::widen(reinterpret_cast<const uint4*>(weight)[lane], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * w[e];
    }

    if (a.rot) {
        const int d0 = lane * 8, half = a.rot / 2;
        const bool turns = d0 < a.rot && !is_v;
        const int position = a.positions[i];
        const bool known = position >= 0 && position < a.rope_rows;
        const float* angles = a.rope + static_cast<long long>(known ? position : 0) * a.rot;
        const float nan = __int_as_float(0x7fffffff);
        if (a.interleaved) {
            if (turns) {
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const float c = known ? angles[d0 / 2 + p] : nan, s = known ? angles[half + d0 / 2 + p] : nan;
                    const float u = x[2 * p], w = x[2 * p + 1];
                    x[2 * p] = u * c - w * s, x[2 * p + 1] = w * c + u * s;
                }
            }
        } else {
            const bool low = d0 < half;
            const int group = (threadIdx.x & 31) / LANES * LANES;
            const int partner = group + (!turns ? lane : low ? lane + half / 8 : lane - half / 8);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float other = __shfl_sync(0xffffffffu, x[e], partner);
                if (turns) {
                    const int j = (low ? d0 : d0 - half) + e;
                    const float c = known ? angles[j] : nan, s = known ? angles[half + j] : nan;
                    x[e] = low ? x[e] * c - other * s : x[e] * c + other * s;
                }
            }
        }
    }
    if (!real) return;
    if (is_q) {
        T* to = static_cast<T*>(a.q_out) + i * a.out_stride[0] + h * a.out_stride[1];
        reinterpret_cast<uint4*>(to)[lane] = Vec8<T>::narrow(x);
        return;
    }
    const int slot = a.slots[i];
    if (slot < 0 || slot >= a.cache.pages * a.cache.page_size) return;
    const long long page = slot / a.cache.page_size, in_page = slot % a.cache.page_size;
    const int64_t* stride = is_v ? a.cache.v_stride : a.cache.k_stride;
    if (a.cache.dtype == EMB_U8) {
        const float scale = is_v ? a.cache.v_scale : a.cache.k_scale;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fdiv_rn(x[e], scale);
    }
    C* to = static_cast<C*>(is_v ? a.cache.v : a.cache.k) + page * stride[0] + in_page * stride[1] + kv * stride[2];
    reinterpret_cast<typename Vec8<C>::raw*>(to)[lane] = Vec8<C>::narrow(x);
}

template <class T, class C> int run_dim(const emb_paged_store_t& a, cudaStream_t stream) {
    const long long rows = static_cast<long long>(a.tokens) * (a.heads + 2 * a.cache.kv_heads);
    const int per_cta = THREADS / (a.cache.dim / 8);
    const long long grid = (rows + per_cta - 1) / per_cta;
    if (grid > 0x7fffffffll) return refuse("paged_store: %lld head rows in one call", rows);
    const auto kernel = a.cache.dim == 64 ? paged_store_kernel<T, C, 8> : a.cache.dim == 128 ? paged_store_kernel<T, C, 16> : paged_store_kernel<T, C, 32>;
    return launched("launch of paged_store", launch(kernel, static_cast<unsigned>(grid), THREADS, 0, stream, a));
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
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.dtype == EMB_F16) return a.cache.dtype == EMB_U8 ? run_dim<__half, E4m3>(a, s) : run_dim<__half, __half>(a, s);
    return a.cache.dtype == EMB_U8 ? run_dim<__nv_bfloat16, E4m3>(a, s) : run_dim<__nv_bfloat16, __nv_bfloat16>(a, s);
}
