// rt_elem.hpp — the element types of the network-block operators: loads, stores and conversions in 16-byte chunks.
#pragma once

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// The same with the alignment of one element only: global memory takes such accesses whole.
struct __attribute__((packed, aligned(2))) Chunk16 { u32x4 v; };
struct __attribute__((packed, aligned(2))) Chunk8 { unsigned long long v; };

template <int DT> struct Elem;
template <> struct Elem<RT_F32> { typedef float T; typedef f32x4 Quad; };
template <> struct Elem<RT_BF16> { typedef __bf16 T; typedef bf16x4 Quad; };
template <> struct Elem<RT_F16> { typedef _Float16 T; typedef f16x4 Quad; };
template <int DT> constexpr int ES = (int)sizeof(typename Elem<DT>::T);
template <int DT> constexpr int EPC = 16 / ES<DT>;          // elements in a 16-byte chunk

// v rounded to the type, from the float32 that it is.  float16: the compiler may fold a product before it into an instruction that
// rounds once instead (v_fma_mixlo_f16), here and not there; one value in 16000 would then depend on which store a call's
// alignment gives it, and differ from what n_lo is the rest of.
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T to_elem(float v) {
    if (DT == RT_F16) asm("" : "+v"(v));
    return (typename Elem<DT>::T)v;
}

// `valid` of the EPC elements at p, zeros behind them.  AL: p is 16-byte aligned and a chunk is all valid or not at all.
template <int DT, bool AL>
__device__ __forceinline__ u32x4 load_chunk(const void* p, int valid) {
    u32x4 r = {0, 0, 0, 0};
    if (AL) {
        if (valid > 0) r = *(const u32x4*)p;
    } else if (valid >= EPC<DT>) {
        r = ((const Chunk16*)p)->v;
    } else if (ES<DT> == 4) {
        const unsigned* q = (const unsigned*)p;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < valid) r[e] = q[e];
    } else {
        const unsigned short* q = (const unsigned short*)p;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < valid) r[e >> 1] |= (unsigned)q[e] << (16 * (e & 1));
    }
    return r;
}

template <int DT>
__device__ __forceinline__ void chunk_to_f32(u32x4 c, float (&v)[EPC<DT>]) {
    if (ES<DT> == 4) {
        const f32x4 f = __builtin_bit_cast(f32x4, c);
#pragma unroll
        for (int e = 0; e < EPC<DT>; ++e) v[e] = f[e & 3];
    } else if (DT == RT_BF16) {
#pragma unroll
        for (int e = 0; e < EPC<DT>; ++e) {
            const unsigned w = (e & 1) ? (c[e >> 1] & 0xffff0000u) : (c[e >> 1] << 16);
            v[e] = __builtin_bit_cast(float, w);
        }
    } else {
        const f16x8 h = __builtin_bit_cast(f16x8, c);
#pragma unroll
        for (int e = 0; e < EPC<DT>; ++e) v[e] = (float)h[e & 7];
    }
}

// Rounds to nearest even, once, and writes `valid` elements.
template <int DT, bool AL>
__device__ __forceinline__ void store_chunk(void* p, const float (&v)[EPC<DT>], int valid) {
    typedef typename Elem<DT>::T T;
    if (valid >= EPC<DT>) {
        union { T t[EPC<DT>]; u32x4 c; } u;
#pragma unroll
        for (int e = 0; e < EPC<DT>; ++e) u.t[e] = to_elem<DT>(v[e]);
        if (AL) *(u32x4*)p = u.c; else ((Chunk16*)p)->v = u.c;
    } else {
#pragma unroll
        for (int e = 0; e < EPC<DT>; ++e)
            if (e < valid) ((T*)p)[e] = to_elem<DT>(v[e]);
    }
}

// Four neighbouring elements, of which `valid` exist; the address has the alignment of one element.
template <int DT>
__device__ __forceinline__ void store4(void* p, f32x4 v, int valid) {
    typedef typename Elem<DT>::T T;
    if (valid >= 4) {
        union { T t[4]; u32x4 c; unsigned long long h; } u;
#pragma unroll
        for (int e = 0; e < 4; ++e) u.t[e] = to_elem<DT>(v[e]);
        if (ES<DT> == 4) ((Chunk16*)p)->v = u.c; else ((Chunk8*)p)->v = u.h;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < valid) ((T*)p)[e] = to_elem<DT>(v[e]);
    }
}

template <int DT>
__device__ __forceinline__ f32x4 load4(const void* p, int valid) {
    typedef typename Elem<DT>::T T;
    f32x4 r = {0, 0, 0, 0};
    if (valid >= 4) {
        union { T t[4]; u32x4 c; unsigned long long h; } u;
        if (ES<DT> == 4) u.c = ((const Chunk16*)p)->v; else u.h = ((const Chunk8*)p)->v;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (float)u.t[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < valid) r[e] = (float)((const T*)p)[e];
    }
    return r;
}
