// What the operators on the two ends of the vocabulary share (vocab_logprobs.hip, vocab_embedding.hip): element types,
// 16-byte accesses, wave reductions of 64-bit keys.
#pragma once

#include "common.hip.h"

namespace pcfgnat {

typedef unsigned int vec16 __attribute__((ext_vector_type(4)));  // one 16-byte global access

// Element types.  N: elements of one 16-byte access; widening to float is exact, narrowing rounds to nearest even (by the
// conversion instructions of gfx950), once per value.
template <typename T>
struct VocabElem {
    static constexpr int N = 16 / (int)sizeof(T);
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
typedef _Float16 f16;
typedef __bf16 bf16;

inline int vocab_elem_bytes(int dtype) { return dtype == PCFGNAT_F32 ? 4 : 2; }
inline bool vocab_dtype_ok(int dtype) { return dtype == PCFGNAT_F16 || dtype == PCFGNAT_BF16 || dtype == PCFGNAT_F32; }

}  // namespace pcfgnat
