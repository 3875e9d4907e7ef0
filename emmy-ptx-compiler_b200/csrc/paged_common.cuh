// What the operators over a paged key-value cache share: error texts, argument checks of the cache, and the
// conversions between f32 and the types a row is held in.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cfloat>
#include <cstdarg>
#include <cstdio>

#include "emmy_b200.h"
#include "paged_overlap.h"

int emb_fail_text(int code, const char* text);  // shim.cpp

namespace emb {
namespace paged {

inline int refuse(const char* fmt, ...) {
    char text[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    return emb_fail_text(EMB_E_ARGUMENT, text);
}

inline int launched(const char* what, cudaError_t e) {
    if (e == cudaSuccess) return 0;
    char text[256];
    snprintf(text, sizeof text, "%s: %s", what, cudaGetErrorString(e));
    return emb_fail_text(static_cast<int>(e), text);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// a row's stride in elements of `size` bytes: a whole number of 16-byte pieces, and small enough that no product with a
// 31-bit count leaves 63 bits
inline bool stride_fits(int64_t stride, int size) { return stride >= 0 && stride < (1ll << 32) && stride * size % 16 == 0; }

// whether the rows of `dim` elements that two or three counted strides name are all apart (what is written has to be)
template <int N> inline bool rows_apart(const int64_t (&count)[N], const int64_t (&stride)[N], int64_t dim) {
    bool used[N] = {};
    int64_t extent = dim;
    for (int k = 0; k < N; ++k) {
        int best = -1;
        for (int i = 0; i < N; ++i)
            if (!used[i] && count[i] > 1 && (best < 0 || stride[i] < stride[best])) best = i;
        if (best < 0) break;
        if (stride[best] < extent) return false;
        extent = stride[best] * (count[best] - 1) + extent;
        used[best] = true;
    }
    return true;
}

inline int check_cache(const char* who, const emb_paged_cache_t& c, int q_dtype) {
    if (q_dtype != EMB_F16 && q_dtype != EMB_BF16) return refuse("%s: q is f16 or bf16", who);
    if (c.dtype != EMB_U8 && c.dtype != q_dtype) return refuse("%s: the cache holds q's type or e4m3 codes", who);
    if (c.dim != 64 && c.dim != 128 && c.dim != 256) return refuse("%s: head dim %d is not 64, 128 or 256", who, c.dim);
    if (c.pages < 1 || c.page_size < 1 || static_cast<int64_t>(c.pages) * c.page_size >= (1ll << 31))
        return refuse("%s: %d pages of %d tokens: at least one of each, and less than 2^31 slots", who, c.pages, c.page_size);
    if (c.kv_heads < 1 || c.kv_heads > 65535) return refuse("%s: %d key heads", who, c.kv_heads);
    if (!c.k || !c.v || !aligned16(c.k) || !aligned16(c.v)) return refuse("%s: pages are null or not 16-byte aligned", who);
    const int size = c.dtype == EMB_U8 ? 1 : 2;
    for (int i = 0; i < 3; ++i)
        if (!stride_fits(c.k_stride[i], size) || !stride_fits(c.v_stride[i], size))
            return refuse("%s: a stride of the pages is not a multiple of 16 bytes below 2^32 elements", who);
    for (const float scale : {c.k_scale, c.v_scale}) {
        // (of a subnormal number the reciprocal may be infinite)
        if (!(scale >= FLT_MIN && scale <= 3.0e38f)) return refuse("%s: a cache scale of %g is not a positive number between 1.2e-38 and 3e38", who, static_cast<double>(scale));
        if (c.dtype != EMB_U8 && scale != 1.f) return refuse("%s: scales belong to a cache of e4m3 codes", who);
    }
    return 0;
}

// rows [n, heads, dim] of 16 bits, and the pages of a cache
inline Area rows_at(const char* name, const void* p, int64_t n, int heads, int dim, const int64_t (&stride)[2]) {
    return Area(name, p, dim * 2).by(heads, stride[1] * 2).by(n, stride[0] * 2);
}
inline Area pages_at(const char* name, const emb_paged_cache_t& c, const void* p, const int64_t (&stride)[3]) {
    const int size = c.dtype == EMB_U8 ? 1 : 2;
    return Area(name, p, c.dim * size).by(c.kv_heads, stride[2] * size).by(c.page_size, stride[1] * size).by(c.pages, stride[0] * size);
}

constexpr int MAX_DEVICES = 64;

// SMs of the current device; 0 where that cannot be had
inline int sm_count() {
    static std::atomic<int> known[MAX_DEVICES];  // (threads that race here store the same number)
    int device = -1;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= MAX_DEVICES) return 0;
    int n = known[device].load(std::memory_order_relaxed);
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
        known[device].store(n, std::memory_order_relaxed);
    }
    return n;
}

// division by a number known to the host: floor(x / d) for x < 2^31
struct Divisor {
    uint32_t d, magic, shift;
    explicit Divisor(uint32_t d_) : d(d_) {
        shift = 0;
        while ((1ull << shift) < d) ++shift;
        magic = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t over(uint32_t x) const { return (__umulhi(x, magic) + x) >> shift; }
};

// Every kernel here is launched as a programmatic dependent of the work before it in the stream: it starts as that work's
// CTAs end, and before its first access to memory it waits until the work is complete and visible (follow_on). None of them
// lets its successor start earlier: CTAs that only wait then hold places that the running kernel's successors need (an
// early launch_dependents cost attend 2 to 43 % of a pass back to back, and assign half of one).
template <class... P, class... A> inline cudaError_t launch(void (*kernel)(P...), dim3 grid, unsigned block, unsigned smem, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid, config.blockDim = dim3(block), config.dynamicSmemBytes = smem, config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute, config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
}
__device__ __forceinline__ void follow_on() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

struct E4m3 {
    uint8_t code;
};

// four consecutive elements of a row <-> f32
template <class T> struct Vec4;

template <> struct Vec4<__half> {
    using raw = uint2;
    static __device__ __forceinline__ void widen(const raw& r, float* x) {
        const float2 lo = __half22float2(reinterpret_cast<const __half2&>(r.x)), hi = __half22float2(reinterpret_cast<const __half2&>(r.y));
        x[0] = lo.x, x[1] = lo.y, x[2] = hi.x, x[3] = hi.y;
    }
    static __device__ __forceinline__ raw narrow(const float* x) {
        const __half2 lo = __floats2half2_rn(x[0], x[1]), hi = __floats2half2_rn(x[2], x[3]);
        return make_uint2(reinterpret_cast<const uint32_t&>(lo), reinterpret_cast<const uint32_t&>(hi));
    }
};

template <> struct Vec4<__nv_bfloat16> {
    using raw = uint2;
    static __device__ __forceinline__ void widen(const raw& r, float* x) {
        x[0] = __uint_as_float(r.x << 16), x[1] = __uint_as_float(r.x & 0xffff0000u);
        x[2] = __uint_as_float(r.y << 16), x[3] = __uint_as_float(r.y & 0xffff0000u);
    }
    static __device__ __forceinline__ raw narrow(const float* x) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
        return make_uint2(reinterpret_cast<const uint32_t&>(lo), reinterpret_cast<const uint32_t&>(hi));
    }
};

template <> struct Vec4<E4m3> {
    using raw = uint32_t;
    // nearest even, saturating at +-448; NaN stays NaN
    static __device__ __forceinline__ raw narrow(const float* x) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
};

}  // namespace paged
}  // namespace emb
