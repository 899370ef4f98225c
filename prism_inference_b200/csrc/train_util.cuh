// train_util.cuh - what the entry points of the trainable sub-block (row_ops.cu, gated_ffn.cu)
// share: value types, 16-byte vectors of them, and the host checks of row tensors.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "host_util.h"

namespace prism {

template <typename T>
PRISM_DEV float to_f32(T v);
template <>
PRISM_DEV float to_f32<float>(float v) { return v; }
template <>
PRISM_DEV float to_f32<__half>(__half v) { return __half2float(v); }
template <>
PRISM_DEV float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
PRISM_DEV T from_f32(float v);
template <>
PRISM_DEV float from_f32<float>(float v) { return v; }
template <>
PRISM_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
PRISM_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two fp32 -> packed 16-bit pair (lo = a), round to nearest even
template <typename T>
PRISM_DEV uint32_t pack2(float a, float b);
template <>
PRISM_DEV uint32_t pack2<__half>(float a, float b) { return pack_h2(a, b); }
template <>
PRISM_DEV uint32_t pack2<__nv_bfloat16>(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
    return r;
}
template <typename T>
PRISM_DEV void unpack2(uint32_t v, float& a, float& b);
template <>
PRISM_DEV void unpack2<__half>(uint32_t v, float& a, float& b) {
    a = lo_h2f(v);
    b = hi_h2f(v);
}
template <>
PRISM_DEV void unpack2<__nv_bfloat16>(uint32_t v, float& a, float& b) {
    a = __uint_as_float(v << 16);
    b = __uint_as_float(v & 0xffff0000u);
}

// cudaFuncSetAttribute(MaxDynamicSharedMemorySize) once a kernel and device (`done`: the kernel's own bit
// per device; setting it twice from two threads does no harm)
template <typename K>
inline cudaError_t allow_smem(K kernel, int bytes, int device, std::atomic<uint64_t>& done) {
    const uint64_t bit = 1ull << (device & 63);
    if (device < 64 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && device < 64) done.fetch_or(bit, std::memory_order_release);
    return e;
}

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
inline int cuda_rc(cudaError_t e, const char* what) {
    return e == cudaSuccess ? PRISM_OK : set_error(PRISM_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

inline int dtype_bytes(int dtype) { return dtype == PRISM_DTYPE_F32 ? 4 : 2; }
inline bool dtype_known(int dtype) {
    return dtype == PRISM_DTYPE_F16 || dtype == PRISM_DTYPE_BF16 || dtype == PRISM_DTYPE_F32;
}

// Offsets of a tensor's rows in elements: far from what 64 bits hold in bytes, also beside an address
inline bool extent_ok(int64_t rows, int64_t stride) { return rows <= 1 || stride <= ((int64_t)1 << 60) / rows; }

// Do two blocks of memory of na and nb bytes share one?
inline bool bytes_overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
    return a && b && pa < pb + nb && pb < pa + na;
}

// Do two tensors of `rows` rows of `dim` values share a byte?  Column slices of one wider buffer
// (same stride, disjoint column ranges) do not; two tensors whose byte ranges meet with unlike
// strides count as sharing.
inline bool rows_overlap(const void* a, int64_t sa, const void* b, int64_t sb, int64_t rows, int64_t dim, int64_t es) {
    if (!a || !b || rows <= 0) return false;
    const intptr_t pa = reinterpret_cast<intptr_t>(a), pb = reinterpret_cast<intptr_t>(b);
    const intptr_t ea = pa + ((rows - 1) * sa + dim) * es, eb = pb + ((rows - 1) * sb + dim) * es;
    if (ea <= pb || eb <= pa) return false;
    if (sa != sb) return true;
    const int64_t pitch = sa * es;
    int64_t d = (int64_t)(pb - pa) % pitch;
    if (d < 0) d += pitch;
    return d < dim * es || pitch - d < dim * es;
}

}  // namespace prism
