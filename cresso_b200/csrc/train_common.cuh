// Shared device helpers of the training operators (embedding, block norm, distillation).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/cresso_b200_train.h"
#include "cresso_common.cuh"
#include "cresso_status.h"

namespace cresso {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Element i of an array whose type is only known at run time (weights, gates,
// teacher logits: small next to the rows they go with, so the branch is uniform
// and its loads hit in cache).
__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
    if (dtype == CRESSO_DTYPE_F32) return static_cast<const float*>(p)[i];
    if (dtype == CRESSO_DTYPE_F16) return to_float(static_cast<const __half*>(p)[i]);
    return to_float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
    if (dtype == CRESSO_DTYPE_F32)
        static_cast<float*>(p)[i] = v;
    else if (dtype == CRESSO_DTYPE_F16)
        static_cast<__half*>(p)[i] = from_float<__half>(v);
    else
        static_cast<__nv_bfloat16*>(p)[i] = from_float<__nv_bfloat16>(v);
}

__device__ __forceinline__ int64_t load_id(const void* p, int bytes, int64_t i) {
    return bytes == 8 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Sum over the block, the same in every thread and in a fixed order; `sh` holds
// one float per warp.  Ends with a barrier, so that `sh` can be used again.
__device__ __forceinline__ float block_sum(float v, float* sh) {
    const int warps = blockDim.x >> 5;
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = (threadIdx.x & 31) < warps ? sh[threadIdx.x & 31] : 0.0f;
    s = warp_sum(s);
    __syncthreads();
    return s;
}
__device__ __forceinline__ float block_max(float v, float* sh) {
    const int warps = blockDim.x >> 5;
    v = warp_max(v);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = (threadIdx.x & 31) < warps ? sh[threadIdx.x & 31] : -INFINITY;
    s = warp_max(s);
    __syncthreads();
    return s;
}

// VEC elements of T between memory and float registers, as the widest accesses that
// VEC * sizeof(T) bytes allow; p is aligned to min(16, VEC * sizeof(T)).
template <int BYTES>
struct Word;
template <>
struct Word<2> { using type = unsigned short; };
template <>
struct Word<4> { using type = unsigned int; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<16> { using type = uint4; };

// VEC elements as they lie in memory.
template <typename T, int VEC>
struct Raw {
    static constexpr int kBytes = VEC * (int)sizeof(T) < 16 ? VEC * (int)sizeof(T) : 16;
    static constexpr int kWords = VEC * (int)sizeof(T) / kBytes;
    using W = typename Word<kBytes>::type;
    union {
        W w[kWords];
        T t[VEC];
    };
    __device__ __forceinline__ Raw() {}
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const W*>(p)[i];
    }
    __device__ __forceinline__ void load_once(const T* p) {  // read-only data
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = __ldg(reinterpret_cast<const W*>(p) + i);
    }
    __device__ __forceinline__ float get(int i) const { return to_float(t[i]); }
};

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[VEC]) {
    Raw<T, VEC> u;
    u.load(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = u.get(i);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[VEC]) {
    constexpr int B = VEC * (int)sizeof(T) < 16 ? VEC * (int)sizeof(T) : 16, N = VEC * (int)sizeof(T) / B;
    using W = typename Word<B>::type;
    union {
        W w[N];
        T t[VEC];
    } u;
#pragma unroll
    for (int i = 0; i < VEC; ++i) u.t[i] = from_float<T>(f[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<W*>(p)[i] = u.w[i];
}

// The same for global memory, with 32-byte accesses (sm_100) where VEC elements have 32
// bytes: a warp's access then covers whole sectors.  p is aligned to min(32, VEC *
// sizeof(T)).  load_global reads data that the kernel does not write.
struct alignas(32) Word32 {
    uint32_t w[8];
};
__device__ __forceinline__ Word32 load_word32(const void* p) {
    Word32 v;
    asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
        : "l"(p));
    return v;
}
__device__ __forceinline__ void store_word32(void* p, const Word32& v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v.w[0]), "r"(v.w[1]),
                 "r"(v.w[2]), "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7])
                 : "memory");
}
template <typename T, int VEC>
__device__ __forceinline__ void load_global(const T* p, float (&f)[VEC]) {
    if constexpr (VEC * sizeof(T) == 32) {
        const Word32 v = load_word32(p);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = __uint_as_float(v.w[i]);
    } else {
        Raw<T, VEC> u;
        u.load_once(p);
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = u.get(i);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_global(T* p, const float (&f)[VEC]) {
    if constexpr (VEC * sizeof(T) == 32) {
        Word32 v;
#pragma unroll
        for (int i = 0; i < VEC; ++i) v.w[i] = __float_as_uint(f[i]);
        store_word32(p, v);
    } else {
        store_vec<T, VEC>(p, f);
    }
}

// Asynchronous copy of VEC elements from global to shared memory in 16-, 8- or 4-byte
// pieces, counted by copy_commit / copy_wait; 2-byte pieces are copied at once.
template <typename T, int VEC>
__device__ __forceinline__ void copy_vec(T* dst, const T* src) {
    constexpr int B = VEC * (int)sizeof(T) < 16 ? VEC * (int)sizeof(T) : 16, N = VEC * (int)sizeof(T) / B;
    if constexpr (B == 2) {
        *reinterpret_cast<unsigned short*>(dst) = *reinterpret_cast<const unsigned short*>(src);
    } else {
        const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
        const char* s = reinterpret_cast<const char*>(src);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (B == 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + 16 * i), "l"(s + 16 * i) : "memory");
            else
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d + B * i), "l"(s + B * i), "n"(B)
                             : "memory");
        }
    }
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// Launch of a kernel that begins with previous_kernel_done() and may be set up while the
// stream's previous kernel still runs.
__device__ __forceinline__ void previous_kernel_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void next_kernel_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename K, typename... Args>
cudaError_t launch_overlapped(K kernel, dim3 grid, int threads, int smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

inline bool aligned_to(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

inline bool train_dtype_ok(int64_t d) { return d == CRESSO_DTYPE_F32 || d == CRESSO_DTYPE_F16 || d == CRESSO_DTYPE_BF16; }
inline int64_t dtype_bytes(int64_t d) { return d == CRESSO_DTYPE_F32 ? 4 : 2; }

// f(T()) with the element type of a dtype code.
template <typename F>
int with_dtype(int64_t d, F f) {
    if (d == CRESSO_DTYPE_F32) return f(float());
    if (d == CRESSO_DTYPE_F16) return f(__half());
    return f(__nv_bfloat16());
}

}  // namespace cresso
