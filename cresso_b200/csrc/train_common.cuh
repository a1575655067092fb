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

// Two packed 16-bit elements and their float values: one instruction an element to read,
// one for both to write.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// VEC elements as they lie in memory: 32-bit registers (one 16-bit element in a register of
// its own).  Global 32-byte accesses exist on sm_100; a warp's access then covers whole
// sectors.  Pointers are aligned to min(32, VEC * sizeof(T)), in shared memory to 16.
template <typename T, int VEC>
struct Raw {
    static constexpr int kBytes = VEC * (int)sizeof(T);
    static constexpr int kWords = kBytes < 4 ? 1 : kBytes / 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void load(const T* p) {  // any memory
        if constexpr (kBytes == 2)
            w[0] = *reinterpret_cast<const unsigned short*>(p);
        else if constexpr (kBytes == 4)
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        else if constexpr (kBytes == 8)
            set(0, *reinterpret_cast<const uint2*>(p));
        else
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) set(4 * i, reinterpret_cast<const uint4*>(p)[i]);
    }
    __device__ __forceinline__ void load_global(const T* p) {  // data that the kernel does not write
        if constexpr (kBytes == 32)
            asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                : "l"(p));
        else if constexpr (kBytes == 2)
            w[0] = __ldg(reinterpret_cast<const unsigned short*>(p));
        else if constexpr (kBytes == 4)
            w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
        else if constexpr (kBytes == 8)
            set(0, __ldg(reinterpret_cast<const uint2*>(p)));
        else
            set(0, __ldg(reinterpret_cast<const uint4*>(p)));
    }
    __device__ __forceinline__ void store(T* p) const {  // global memory
        if constexpr (kBytes == 32)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
                         "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
        else if constexpr (kBytes == 2)
            *reinterpret_cast<unsigned short*>(p) = (unsigned short)w[0];
        else if constexpr (kBytes == 4)
            *reinterpret_cast<uint32_t*>(p) = w[0];
        else if constexpr (kBytes == 8)
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ void to(float (&f)[VEC]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = __uint_as_float(w[i]);
        } else if constexpr (VEC == 1) {
            f[0] = unpack2<T>(w[0]).x;
        } else {
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                const float2 v = unpack2<T>(w[i]);
                f[2 * i] = v.x;
                f[2 * i + 1] = v.y;
            }
        }
    }
    __device__ __forceinline__ void from(const float (&f)[VEC]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) w[i] = __float_as_uint(f[i]);
        } else if constexpr (VEC == 1) {
            w[0] = pack2<T>(f[0], 0.0f);
        } else {
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
        }
    }

private:
    __device__ __forceinline__ void set(int i, uint2 v) {
        w[i] = v.x;
        w[i + 1] = v.y;
    }
    __device__ __forceinline__ void set(int i, uint4 v) {
        w[i] = v.x;
        w[i + 1] = v.y;
        w[i + 2] = v.z;
        w[i + 3] = v.w;
    }
};

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&f)[VEC]) {
    Raw<T, VEC> u;
    u.load(p);
    u.to(f);
}
template <typename T, int VEC>
__device__ __forceinline__ void load_global(const T* p, float (&f)[VEC]) {
    Raw<T, VEC> u;
    u.load_global(p);
    u.to(f);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_global(T* p, const float (&f)[VEC]) {
    Raw<T, VEC> u;
    u.from(f);
    u.store(p);
}

// f(p) with a pointer of the array's run-time type: one uniform branch for all its loads.
template <typename F>
__device__ __forceinline__ void with_any(const void* p, int dtype, F f) {
    if (dtype == CRESSO_DTYPE_F32)
        f(static_cast<const float*>(p));
    else if (dtype == CRESSO_DTYPE_F16)
        f(static_cast<const __half*>(p));
    else
        f(static_cast<const __nv_bfloat16*>(p));
}

// VEC elements of an array whose type is only known at run time; the branch is uniform.
template <int VEC>
__device__ __forceinline__ void store_any_vec(void* p, int dtype, int64_t i, const float (&f)[VEC]) {
    if (dtype == CRESSO_DTYPE_F32)
        store_global<float, VEC>(static_cast<float*>(p) + i, f);
    else if (dtype == CRESSO_DTYPE_F16)
        store_global<__half, VEC>(static_cast<__half*>(p) + i, f);
    else
        store_global<__nv_bfloat16, VEC>(static_cast<__nv_bfloat16*>(p) + i, f);
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
