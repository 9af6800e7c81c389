// What the operators on the two ends of the vocabulary share (vocab_logprobs.hip, vocab_embedding.hip): element types,
// 16-byte accesses, wave reductions of 64-bit keys.
#pragma once

#include "common.hip.h"

namespace pcfgnat {

typedef unsigned int vec16 __attribute__((ext_vector_type(4)));  // one 16-byte global access
typedef vec16 vec16_any __attribute__((aligned(2)));               // the same at the address of any element

typedef _Float16 f16;
typedef __bf16 bf16;

// Running maximum of 16-byte chunks, NaN left aside (as the hardware's maximum does): packed for float16, two elements an
// instruction, widened otherwise.
template <typename T>
struct ChunkMax {
    float m = NEG_INF_F;
    __device__ __forceinline__ void take(const vec16 &v) {
        typedef T vecT __attribute__((ext_vector_type(16 / sizeof(T))));
        const vecT t = __builtin_bit_cast(vecT, v);
#pragma unroll
        for (int i = 0; i < (int)(16 / sizeof(T)); i++) m = fmaxf(m, (float)t[i]);
    }
    __device__ __forceinline__ void take(const ChunkMax &o) { m = fmaxf(m, o.m); }
    __device__ __forceinline__ float value() const { return m; }
};
template <>
struct ChunkMax<f16> {
    typedef f16 f16x2 __attribute__((ext_vector_type(2)));
    f16x2 m = {(f16)NEG_INF_F, (f16)NEG_INF_F};
    __device__ __forceinline__ void take(const vec16 &v) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned pair = v[i];  // (a copy: the address of a vector's element is not its own)
            m = __builtin_elementwise_max(m, __builtin_bit_cast(f16x2, pair));
        }
    }
    __device__ __forceinline__ void take(const ChunkMax &o) { m = __builtin_elementwise_max(m, o.m); }
    __device__ __forceinline__ float value() const { return fmaxf((float)m.x, (float)m.y); }
};

// Element types.  N: elements of one 16-byte access; widening to float is exact, narrowing rounds to nearest even (by the
// conversion instructions of gfx950), once per value.
template <typename T>
struct VocabElem {
    static constexpr int N = 16 / (int)sizeof(T);
    typedef ChunkMax<T> Max;
    typedef T vecT __attribute__((ext_vector_type(N)));
    typedef float vecF __attribute__((ext_vector_type(N)));
    __device__ static __forceinline__ float widen(T x) { return (float)x; }
    __device__ static __forceinline__ T narrow(float x) { return (T)x; }
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

// Sixteen bytes of -inf.
template <typename T>
__device__ __forceinline__ vec16 minus_infinities() {
    float o[VocabElem<T>::N];
#pragma unroll
    for (int i = 0; i < VocabElem<T>::N; i++) o[i] = NEG_INF_F;
    return VocabElem<T>::pack(o);
}

inline int vocab_elem_bytes(int dtype) { return dtype == PCFGNAT_F32 ? 4 : 2; }
inline bool vocab_dtype_ok(int dtype) { return dtype == PCFGNAT_F16 || dtype == PCFGNAT_BF16 || dtype == PCFGNAT_F32; }

}  // namespace pcfgnat
