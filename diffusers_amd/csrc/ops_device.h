// ops_device.h — element types and small device helpers shared by the operator kernels (op_*.hip).
#pragma once
#include "ops.h"

typedef __bf16 bf16_t;
typedef float floatx4 __attribute__((ext_vector_type(4)));
template <typename T, int N> struct VecOf { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T> struct VecOf<T, 1> { typedef T type; };
template <typename T> constexpr int kVec = 16 / (int)sizeof(T);         // elements of a 16-byte access

template <int N, typename T> __device__ __forceinline__ void vec_get(const typename VecOf<T, N>::type& v, float (&f)[N])
{
    if constexpr (N == 1) f[0] = (float)v;
    else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = (float)v[i];
    }
}
template <int N, typename T> __device__ __forceinline__ typename VecOf<T, N>::type vec_set(const float (&f)[N])
{
    typename VecOf<T, N>::type v;
    if constexpr (N == 1) v = (T)f[0];
    else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (T)f[i];
    }
    return v;
}
// a parameter that is stored either in fp32 or in the activations' type
template <typename T> __device__ __forceinline__ float param_at(const void* p, bool f32, long long i)
{
    return f32 ? ((const float*)p)[i] : (float)((const T*)p)[i];
}
template <typename T> __device__ __forceinline__ void param_put(void* p, bool f32, long long i, float v)
{
    if (f32) ((float*)p)[i] = v;
    else ((T*)p)[i] = (T)v;
}

typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
constexpr unsigned kOob = 0x80000000u;          // past the window of a buffer descriptor: such a lane of a load brings zeros
// ---- matrix instructions: 16 rows by 16 columns by 64 bytes of the contraction.  Operands: lane l holds 16 bytes of row (column) l & 15, chunk l >> 4;
// result: lane l holds rows 4 (l >> 4) .. + 3 of column l & 15.
template <typename T> struct Frag { typename VecOf<T, kVec<T>>::type v; };
__device__ __forceinline__ floatx4 mma(const Frag<half_t>& a, const Frag<half_t>& b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v, b.v, c, 0, 0, 0); }
__device__ __forceinline__ floatx4 mma(const Frag<bf16_t>& a, const Frag<bf16_t>& b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0); }
__device__ __forceinline__ floatx4 mma(const Frag<float>& a, const Frag<float>& b, floatx4 c)
{
    // lane group g holds elements 4g..4g+3 of the contraction in both operands: instruction j takes element j of every group
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
    return c;
}

// 16 bytes a lane, global memory to LDS, no registers between: lane l of the wave writes lds + 16 l.  Written out so that the waits are the
// kernels' own (a compiler-visible load into LDS makes every later LDS read wait for all of them).  It stays where it is written.
__device__ __forceinline__ void dma16(uintx4 rsrc, unsigned voff, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory", "m0");
}
// Waits for this wave's loads (and stores).  The builtin, not text: the compiler has to know that its own loads have arrived too, or it waits again, for the
// loads into LDS, wherever one of their registers is used next.
__device__ __forceinline__ void wait_loads()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);
    asm volatile("" ::: "memory");
}
// every wave of the workgroup is here, with its LDS reads done
__device__ __forceinline__ void meet()
{
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ uintx4 make_rsrc(const char* p, unsigned bytes = kOob)
{
    const unsigned long long a = (unsigned long long)p;
    return uintx4{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)a), (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32)), (unsigned)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

// calls f with a value of the element type that `dtype` names
template <typename F> static inline void op_dispatch(int dtype, F&& f)
{
    if (dtype == SDE_F16) f(half_t{});
    else if (dtype == SDE_BF16) f(bf16_t{});
    else f(float{});
}
