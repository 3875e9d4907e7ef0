// emb_paged_attend: attention of one new token of each request over the pages of a cache.
//
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q . k_j,  m = max_j s_j
//
// One pass over the keys with the running maximum and sum of the softmax: when a key raises the maximum from m to m', what
// was summed is scaled by exp(m - m'). A group of DIM / 8 lanes holds eight dims each of one (request, query head).

#include "paged_common.cuh"

namespace {

using namespace emb::paged;

constexpr int THREADS = 128;

template <class T, class C, int LANES> __global__ void __launch_bounds__(THREADS) paged_attend_kernel(const emb_paged_attend_t a) {
    const int lane = threadIdx.x % LANES;
    const long long rows = static_cast<long long>(a.requests) * a.heads;
    const long long row = static_cast<long long>(blockIdx.x) * (THREADS / LANES) + threadIdx.x / LANES;
    const bool real = row < rows;
    const int b = real ? static_cast<int>(row / a.heads) : 0, h = real ? static_cast<int>(row % a.heads) : 0;
    const int kv = h / (a.heads / a.cache.kv_heads);
    const long long capacity = static_cast<long long>(a.table_width) * a.cache.page_size;
    const long long asked = real ? max(a.lengths[b], 0) : 0;
    const long long end = min(asked, capacity);
    const long long begin = a.window && asked > a.window ? asked - a.window : 0;
    const unsigned mask = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << ((threadIdx.x & 31) / LANES * LANES);
    const float nan = __int_as_float(0x7fffffff);

    float q[8], o[8] = {};
    Vec8<T>::widen(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.q_stride[0] + h * a.q_stride[1])[lane], q);
    const float scale = a.scale * a.cache.k_scale;
    float top = -INFINITY, total = asked > capacity ? nan : 0.f;
    for (long long j = begin; j < end; ++j) {
        const int page = a.table[b * a.table_stride + j / a.cache.page_size];
        if (page < 0 || page >= a.cache.pages) {
            total = nan;
            continue;
        }
        const long long in_page = j % a.cache.page_size;
        float k[8], v[8];
        Vec8<C>::widen(reinterpret_cast<const typename Vec8<C>::raw*>(static_cast<const C*>(a.cache.k) + page * a.cache.k_stride[0] + in_page * a.cache.k_stride[1] + kv * a.cache.k_stride[2])[lane], k);
        Vec8<C>::widen(reinterpret_cast<const typename Vec8<C>::raw*>(static_cast<const C*>(a.cache.v) + page * a.cache.v_stride[0] + in_page * a.cache.v_stride[1] + kv * a.cache.v_stride[2])[lane], v);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(q[e], k[e], s);
#pragma unroll
        for (int d = LANES / 2; d; d >>= 1) s += __shfl_xor_sync(mask, s, d);
        s *= scale;
        const float raised = fmaxf(top, s);
        const float keep = raised == -INFINITY ? 1.f : expf(top - raised), p = s == -INFINITY ? 0.f : expf(s - raised);
        total = total * keep + p;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = o[e] * keep + p * v[e];
        top = raised;
    }
    if (!real) return;
    const float inv = total == 0.f ? 0.f : a.cache.v_scale / total;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= inv;
    T* to = static_cast<T*>(a.out) + b * a.out_stride[0] + h * a.out_stride[1];
    reinterpret_cast<uint4*>(to)[lane] = Vec8<T>::narrow(o);
    if (a.lse && lane == 0) a.lse[row] = total == 0.f ? -INFINITY : top + logf(total);
}

template <class T, class C> int run_dim(const emb_paged_attend_t& a, cudaStream_t stream) {
    const long long rows = static_cast<long long>(a.requests) * a.heads;
    const int per_cta = THREADS / (a.cache.dim / 8);
    const long long grid = (rows + per_cta - 1) / per_cta;
    if (grid > 0x7fffffffll) return refuse("paged_attend: %lld rows in one call", rows);
    switch (a.cache.dim) {
        case 64: paged_attend_kernel<T, C, 8><<<static_cast<unsigned>(grid), THREADS, 0, stream>>>(a); break;
        case 128: paged_attend_kernel<T, C, 16><<<static_cast<unsigned>(grid), THREADS, 0, stream>>>(a); break;
        default: paged_attend_kernel<T, C, 32><<<static_cast<unsigned>(grid), THREADS, 0, stream>>>(a); break;
    }
    return launched("launch of paged_attend");
}

}  // namespace

extern "C" int emb_paged_attend(const emb_paged_attend_t* args, void* stream) {
    if (!args) return refuse("paged_attend: null arguments");
    const emb_paged_attend_t& a = *args;
    if (int r = check_cache("paged_attend", a.cache, a.dtype)) return r;
    if (a.requests < 0 || a.heads < 1 || a.heads > 65535 || a.heads % a.cache.kv_heads)
        return refuse("paged_attend: %d requests of %d heads over %d key heads: a multiple of the key heads", a.requests, a.heads, a.cache.kv_heads);
    if (a.table_width < 1 || static_cast<int64_t>(a.table_width) * a.cache.page_size >= (1ll << 31) || a.table_stride < 0)
        return refuse("paged_attend: a table row of %d pages of %d tokens", a.table_width, a.cache.page_size);
    if (a.window < 0) return refuse("paged_attend: a negative window");
    if (!(a.scale > -INFINITY && a.scale < INFINITY)) return refuse("paged_attend: the scale is not a finite number");
    if (a.requests == 0) return 0;
    if (!a.table || !a.lengths) return refuse("paged_attend: null table or lengths");
    if (!a.q || !a.out || !aligned16(a.q) || !aligned16(a.out)) return refuse("paged_attend: q or out is null or not 16-byte aligned");
    for (const int64_t* s : {a.q_stride, a.out_stride})
        if (!stride_fits(s[0], 2) || !stride_fits(s[1], 2)) return refuse("paged_attend: a stride of q or out is not a multiple of 16 bytes below 2^32 elements");
    const int64_t rows[2] = {a.requests, a.heads};
    if (!rows_apart(rows, a.out_stride, a.cache.dim)) return refuse("paged_attend: rows of out overlap");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.dtype == EMB_F16) return a.cache.dtype == EMB_U8 ? run_dim<__half, E4m3>(a, s) : run_dim<__half, __half>(a, s);
    return a.cache.dtype == EMB_U8 ? run_dim<__nv_bfloat16, E4m3>(a, s) : run_dim<__nv_bfloat16, __nv_bfloat16>(a, s);
}
