// What the operators on the two ends of the vocabulary share (vocab_logprobs.hip, vocab_embedding.hip): element types,
// 16-byte accesses, maxima in single instructions.
#pragma once

#include "common.hip.h"

namespace pcfgnat {

typedef unsigned int vec16 __attribute__((ext_vector_type(4)));  // one 16-byte global access
typedef vec16 vec16_any __attribute__((aligned(2)));               // the same at the address of any element

typedef _Float16 f16;
typedef __bf16 bf16;

// Maxima of registers as one instruction each.  Written in assembly because fmaxf and its packed form on values from memory
// or another lane come out with one more instruction for every operand, which quiets NaNs that the maximum itself sets
// aside (it returns the other operand); the loops here are bound by the number of instructions.
__device__ __forceinline__ float max2_raw(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float max3_raw(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ unsigned pk_max_raw(unsigned a, unsigned b) {
    unsigned r;
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
// The maximum over a wave, in every lane: within the rows of 16 by partner lanes, across them by row broadcasts (rows 1 and 3
// take row 0's and 2's, rows 2 and 3 take the first half's), the last lane's to all.  The s_nops are the two wait states
// that a DPP read needs after the write of its register.
__device__ __forceinline__ float wave_max_raw(float v) {
    asm("s_nop 1\n\tv_max_f32_dpp %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_mirror row_mask:0xf bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_bcast:15 row_mask:0xa bank_mask:0xf\n\t"
        "s_nop 1\n\tv_max_f32_dpp %0, %0, %0 row_bcast:31 row_mask:0xc bank_mask:0xf\n\t"
        "s_nop 1"
        : "+v"(v));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Running maximum of 16-byte chunks, NaN left aside: packed for float16, two elements an instruction, widened otherwise.
template <typename T>
struct ChunkMax {
    float m = NEG_INF_F;
    __device__ __forceinline__ void take(const vec16 &v) {
        typedef T vecT __attribute__((ext_vector_type(16 / sizeof(T))));
        const vecT t = __builtin_bit_cast(vecT, v);
#pragma unroll
        for (int i = 0; i < (int)(16 / sizeof(T)); i += 2) m = max3_raw(m, (float)t[i], (float)t[i + 1]);
    }
    __device__ __forceinline__ void take(const ChunkMax &o) { m = max2_raw(m, o.m); }
    __device__ __forceinline__ float value() const { return m; }
};
template <>
struct ChunkMax<f16> {
    unsigned m = 0xFC00FC00u;
    __device__ __forceinline__ void take(const vec16 &v) { m = pk_max_raw(pk_max_raw(m, pk_max_raw(v.x, v.y)), pk_max_raw(v.z, v.w)); }
    __device__ __forceinline__ void take(const ChunkMax &o) { m = pk_max_raw(m, o.m); }
    __device__ __forceinline__ float value() const {
        typedef f16 f16x2 __attribute__((ext_vector_type(2)));
        const f16x2 h = __builtin_bit_cast(f16x2, m);
        return max2_raw((float)h.x, (float)h.y);
    }
};

// Element types.  N: elements of one 16-byte access; widening to float is exact, narrowing rounds to nearest even (by the
// conversion instructions of gfx950), once per value.
template <typename T>
struct VocabElem {
    static constexpr int N = 16 / (int)sizeof(T);
    static constexpr unsigned LOWEST_BIT = sizeof(T) == 4 ? 1u : (float)(T)1.00390625f == 1.f ? 1u << 16 : 1u << 13;  // of the widened value
    typedef ChunkMax<T> Max;
    typedef T vecT __attribute__((ext_vector_type(N)));
    typedef float vecF __attribute__((ext_vector_type(N)));
    __device__ static __forceinline__ void unpack(const vec16 &v, float (&o)[N]) {
        const vecT t = __builtin_bit_cast(vecT, v);
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = (float)t[i];
    }
    __device__ static __forceinline__ vec16 pack(const float (&o)[N]) {
        vecF f;
#pragma unroll
        for (int i = 0; i < N; i++) f[i] = o[i];
        return __builtin_bit_cast(vec16, __builtin_convertvector(f, vecT));
    }
};

// Splits n elements at any element address into [head scalars][16-byte chunks][tail scalars].
template <typename T>
struct Span {
    int head, nvec, tail;
    __device__ __forceinline__ Span(const T *x, int n) {
        constexpr int N = VocabElem<T>::N;
        const int h = (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T));
        head = h < n ? h : n;
        nvec = (n - head) / N;
        tail = n - head - nvec * N;
    }
    // the scalar of thread `tid` (one at most), or -1
    __device__ __forceinline__ int edge(int tid) const {
        if (tid < head) return tid;
        if (tid < head + tail) return head + nvec * VocabElem<T>::N + (tid - head);
        return -1;
    }
};

inline int vocab_elem_bytes(int dtype) { return dtype == PCFGNAT_F32 ? 4 : 2; }
inline bool vocab_dtype_ok(int dtype) { return dtype == PCFGNAT_F16 || dtype == PCFGNAT_BF16 || dtype == PCFGNAT_F32; }

}  // namespace pcfgnat
