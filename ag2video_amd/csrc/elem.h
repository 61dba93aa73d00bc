// Element types of the operators that take fp32, bf16 and fp16 tensors (group_norm.hip, embed.hip): 16-byte vectors at the element's own
// alignment, widened to fp32 for every sum and product and rounded once (to nearest even) where a result is stored.
#pragma once
#include "common.h"

#define AG2V_F32 0
#define AG2V_BF16 1
#define AG2V_F16 2

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
// A row of an odd width starts at any multiple of the element's size: global memory takes 16-byte accesses at every one of them, so
// there is one load path and no variant by alignment.
typedef u32x4 u32x4_a2 __attribute__((aligned(2), may_alias));
typedef u32x4 u32x4_a4 __attribute__((aligned(4), may_alias));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

struct ElemF32 {
    typedef float T;
    typedef u32x4_a4 raw;
    static constexpr int V = 4;
    static __device__ __forceinline__ float widen(T v) { return v; }
    static __device__ __forceinline__ T narrow(float v) { return v; }
    static __device__ __forceinline__ void unpack(u32x4 r, float (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[4]) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(v[i]);
        return r;
    }
};
struct ElemBF16 {
    typedef unsigned short T;
    typedef u32x4_a2 raw;
    static constexpr int V = 8;
    static __device__ __forceinline__ float widen(T v) { return __uint_as_float((unsigned)v << 16); }
    static __device__ __forceinline__ T narrow(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
    static __device__ __forceinline__ void unpack(u32x4 r, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(r[i] << 16);
            v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[8]) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bf16x2 h;
            h[0] = (__bf16)v[2 * i];
            h[1] = (__bf16)v[2 * i + 1];
            r[i] = __builtin_bit_cast(unsigned, h);
        }
        return r;
    }
};
struct ElemF16 {
    typedef unsigned short T;
    typedef u32x4_a2 raw;
    static constexpr int V = 8;
    static __device__ __forceinline__ float widen(T v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ T narrow(float v) { return __builtin_bit_cast(unsigned short, (_Float16)v); }
    static __device__ __forceinline__ void unpack(u32x4 r, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned u = r[i];      // (a bit cast of the vector's element itself takes element 0)
            const f16x2 h = __builtin_bit_cast(f16x2, u);
            v[2 * i] = (float)h[0];
            v[2 * i + 1] = (float)h[1];
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[8]) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f16x2 h;
            h[0] = (_Float16)v[2 * i];
            h[1] = (_Float16)v[2 * i + 1];
            r[i] = __builtin_bit_cast(unsigned, h);
        }
        return r;
    }
};

// Accesses of tensors beyond these sizes go past the caches (template argument NT).  Results of more than the L2s hold together would leave
// them full of lines that the next kernel has to write back before it can read: the statistics behind a 134 MB result of group_norm_act
// took 41 us after ordinary stores and 31 us after these; smaller results stay where the next operator finds them.  Reads that are the last
// ones of a tensor of over a quarter of the Infinity Cache leave what is still needed there: lookups of 102 MB behind the gradient's sums of
// as much took 38 us after ordinary loads and 28 us after these; at 67 MB the two did not differ.
#define AG2V_NT_STORE_BYTES (32LL << 20)
#define AG2V_NT_LOAD_BYTES (64LL << 20)

// nv of the E::V elements at p (the last vector of a row whose width is no multiple of V); the rest reads as zero.
template <class E, bool NT = false>
__device__ __forceinline__ u32x4 load_vec(const typename E::T* p, int nv) {
    if (nv >= E::V) {
        if (NT) return __builtin_nontemporal_load(reinterpret_cast<const typename E::raw*>(p));
        return *reinterpret_cast<const typename E::raw*>(p);
    }
    float v[E::V];
#pragma unroll
    for (int i = 0; i < E::V; ++i) v[i] = i < nv ? E::widen(p[i]) : 0.f;
    return E::pack(v);
}
template <class E, bool NT = false>
__device__ __forceinline__ void store_vec(typename E::T* p, int nv, const float (&v)[E::V]) {
    if (nv >= E::V) {
        if (NT) __builtin_nontemporal_store(E::pack(v), reinterpret_cast<typename E::raw*>(p));
        else *reinterpret_cast<typename E::raw*>(p) = E::pack(v);
        return;
    }
#pragma unroll
    for (int i = 0; i < E::V; ++i)
        if (i < nv) p[i] = E::narrow(v[i]);
}

// The last vector of a row whose width is no multiple of V is loaded so that it ends with the row; its first `dup` elements are the vector
// before's, and only the others are stored (that vector's lane may round its own differently: the compiler is free to fuse a product into the
// conversion for one element of a vector and not for another).
template <class E, bool NT = false>
__device__ __forceinline__ void store_tail(typename E::T* p, int dup, int width, const float (&v)[E::V]) {
    if (dup == 0 || width < E::V) {
        store_vec<E, NT>(p, width, v);
        return;
    }
    typedef unsigned u32_a2 __attribute__((aligned(2), may_alias));
    typedef unsigned long long u64_a2 __attribute__((aligned(2), may_alias));
    const u32x4 r = E::pack(v);
    unsigned long long lo = r[0] | (unsigned long long)r[1] << 32, hi = r[2] | (unsigned long long)r[3] << 32;
    const int bits = dup * (int)sizeof(typename E::T) * 8, bytes = 16 - (bits >> 3);
    if (bits >= 64) {
        lo = hi >> (bits - 64);
    } else {
        lo = lo >> bits | hi << (64 - bits);
        hi >>= bits;
    }
    char* q = (char*)(p + dup);
    if (bytes & 8) {
        *reinterpret_cast<u64_a2*>(q) = lo;
        lo = hi;
        q += 8;
    }
    if (bytes & 4) {
        *reinterpret_cast<u32_a2*>(q) = (unsigned)lo;
        lo >>= 32;
        q += 4;
    }
    if (bytes & 2) *reinterpret_cast<unsigned short*>(q) = (unsigned short)lo;
}

// One value of a tensor whose type is a kernel argument (the same branch for every lane).
__device__ __forceinline__ float load_any(const void* p, int dtype, long long i) {
    if (dtype == AG2V_F32) return ((const float*)p)[i];
    const unsigned short v = ((const unsigned short*)p)[i];
    return dtype == AG2V_BF16 ? ElemBF16::widen(v) : ElemF16::widen(v);
}
__device__ __forceinline__ void store_any(void* p, int dtype, long long i, float v) {
    if (dtype == AG2V_F32) ((float*)p)[i] = v;
    else if (dtype == AG2V_BF16) ((unsigned short*)p)[i] = ElemBF16::narrow(v);
    else ((unsigned short*)p)[i] = ElemF16::narrow(v);
}
