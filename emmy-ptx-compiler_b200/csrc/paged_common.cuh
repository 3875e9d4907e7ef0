// What the operators over a paged key-value cache share: error texts, argument checks of the cache, and the
// conversions between f32 and the types a row is held in.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdarg>
#include <cstdio>

#include "emmy_b200.h"

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
    if (!(c.k_scale > 0.f) || !(c.v_scale > 0.f) || c.k_scale > 3.0e38f || c.v_scale > 3.0e38f) return refuse("%s: a cache scale is not a positive number", who);
    return 0;
}

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

// eight consecutive elements of a row <-> f32; a load is one 16-byte (8-byte for codes) access
template <class T> struct Vec8;

template <> struct Vec8<__half> {
    using raw = uint4;
    static __device__ __forceinline__ void widen(const raw& r, float (&x)[8]) {
        const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(h[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ raw narrow(const float (&x)[8]) {
        raw r;
        __half2* h = reinterpret_cast<__half2*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        return r;
    }
};

template <> struct Vec8<__nv_bfloat16> {
    using raw = uint4;
    static __device__ __forceinline__ void widen(const raw& r, float (&x)[8]) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __bfloat1622float2(h[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ raw narrow(const float (&x)[8]) {
        raw r;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        return r;
    }
};

template <> struct Vec8<E4m3> {
    using raw = uint2;
    static __device__ __forceinline__ void widen(const raw& r, float (&x)[8]) {
        const __nv_fp8x2_storage_t* c = reinterpret_cast<const __nv_fp8x2_storage_t*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h(__nv_cvt_fp8x2_to_halfraw2(c[i], __NV_E4M3));  // exact: e4m3 is a subset of f16
            const float2 f = __half22float2(h);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
    // nearest even, saturating at +-448; NaN stays NaN
    static __device__ __forceinline__ raw narrow(const float (&x)[8]) {
        raw r;
        __nv_fp8x2_storage_t* c = reinterpret_cast<__nv_fp8x2_storage_t*>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * i], x[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
        return r;
    }
};

}  // namespace paged
}  // namespace emb
