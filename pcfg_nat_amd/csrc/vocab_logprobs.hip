// Log-probabilities of given tokens over rows of vocabulary logits, with the entropy of the row and its top alternatives,
// and the gradient of all three.
//
//   lp_v = (x_v - m) - log Z,  m = max x,  Z = sum exp(x - m),   H = log Z - sum exp(x - m) (x - m) / Z
//   dx_v = sum_j g_j [v = id_j] - p_v (G + gH (lp_v + H)),  j over the token and the alternatives, G = sum_j g_j
//
// Conventions at the edges (tests/test_vocab_ops.py holds each of them): a masked entry (-inf) adds nothing to the entropy
// and has no gradient of its own; a row of nothing but -inf has log-probabilities of -inf, entropy 0 and gradient 0; a NaN
// or +inf makes every log-probability of its row NaN; in the order of the alternatives NaN counts as largest, the two
// zeros as equal, and equal values go to the lower index.  A negative token leaves its row out: it is not read.
#include "vocab.hip.h"

namespace pcfgnat {
namespace {

constexpr int MAX_TOP = 64;

struct LogprobArgs {
    const int64_t *tokens;
    float *logprobs, *entropy, *top_logprobs;
    int64_t *top_tokens;
    float *stats;  // m, log Z and H of every row, [3][rows]
    int64_t rows, inner, so, si;
    int V, top;
};

// Order of the alternatives as a whole number: value first (NaN largest, -0 = +0), then the lower index.  Never 0
// and never all ones, so both can stand for "no key".
__device__ __forceinline__ unsigned order_of(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const unsigned b = __float_as_uint(x + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ unsigned long long key_of(float x, int i) {
    return ((unsigned long long)order_of(x) << 32) | (0xFFFFFFFEu - (unsigned)i);
}
__device__ __forceinline__ float value_of(unsigned long long key) {
    const unsigned o = (unsigned)(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ int index_of(unsigned long long key) { return (int)(0xFFFFFFFEu - (unsigned)key); }

__device__ __forceinline__ unsigned long long wave_max_key(unsigned long long v) {
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long w = __shfl_xor(v, o);
        v = w > v ? w : v;
    }
    return v;
}

template <typename T>
__device__ __forceinline__ const T *row_at(const T *logits, const LogprobArgs &a, int64_t r) {
    const int64_t b = r / a.inner;
    return logits + b * a.so + (r - b * a.inner) * a.si;
}

template <typename T>
__global__ __launch_bounds__(256) void logprobs_kernel(const T *__restrict__ logits, LogprobArgs a) {
    __shared__ float s_f[8];
    __shared__ unsigned long long s_k[4];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t tok = a.tokens ? a.tokens[r] : 0;
    if (tok < 0) {
        if (tid == 0) {
            a.logprobs[r] = 0.f;
            if (a.entropy) a.entropy[r] = 0.f;
        }
        if (tid < a.top) {
            a.top_logprobs[r * a.top + tid] = NEG_INF_F;
            a.top_tokens[r * a.top + tid] = -1;
        }
        return;
    }
    const T *x = row_at(logits, a, r);
    float m = NEG_INF_F;
    for (int i = tid; i < a.V; i += 256) m = fmaxf(m, (float)x[i]);
    m = wave_max(m);
    if (lane == 0) s_f[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_f[0], s_f[1]), fmaxf(s_f[2], s_f[3]));
    const bool empty = m == NEG_INF_F;
    if (empty) m = 0.f;
    float z = 0.f, s = 0.f;
    for (int i = tid; i < a.V; i += 256) {
        const float d = (float)x[i] - m, e = __expf(d);
        z += e;
        s += e * fmaxf(d, -1e30f);
    }
    z = wave_sum(z);
    s = wave_sum(s);
    __syncthreads();
    if (lane == 0) {
        s_f[wave] = z;
        s_f[4 + wave] = s;
    }
    __syncthreads();
    z = (s_f[0] + s_f[1]) + (s_f[2] + s_f[3]);
    s = (s_f[4] + s_f[5]) + (s_f[6] + s_f[7]);
    const bool none = z == 0.f;  // nothing but -inf (a NaN makes z NaN)
    const float lz = logf(z), H = none ? 0.f : lz - s / z;
    if (tid == 0) {
        if (a.tokens) a.logprobs[r] = tok >= a.V ? __builtin_nanf("") : none ? NEG_INF_F : ((float)x[tok] - m) - lz;
        if (a.entropy) a.entropy[r] = H;
        if (a.stats) {
            a.stats[r] = m;
            a.stats[a.rows + r] = lz;
            a.stats[2 * a.rows + r] = H;
        }
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.top; k++) {
        unsigned long long best = 0;
        for (int i = tid; i < a.V; i += 256) {
            const unsigned long long key = key_of((float)x[i], i);
            if (key < last && key > best) best = key;
        }
        best = wave_max_key(best);
        __syncthreads();
        if (lane == 0) s_k[wave] = best;
        __syncthreads();
        for (int w = 0; w < 4; w++) best = s_k[w] > best ? s_k[w] : best;
        last = best;
        if (tid == 0) {
            const float v = (float)x[index_of(best)];
            a.top_logprobs[r * a.top + k] = none ? NEG_INF_F : (v - m) - lz;
            a.top_tokens[r * a.top + k] = index_of(best);
        }
    }
}

struct LogprobGradArgs {
    const int64_t *tokens, *top_tokens;
    const float *stats, *g_logprobs, *g_entropy, *g_top;
    int64_t rows, inner, so, si;
    int V, top;
};

template <typename T>
__global__ __launch_bounds__(256) void logprobs_grad_kernel(const T *__restrict__ logits, T *__restrict__ grad, LogprobGradArgs a) {
    __shared__ float s_g[MAX_TOP + 1];
    __shared__ int64_t s_i[MAX_TOP + 1];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x;
    T *dx = grad + r * a.V;
    const int64_t tok = a.tokens ? a.tokens[r] : 0;
    const float lz = tok < 0 ? NEG_INF_F : a.stats[a.rows + r];
    if (lz == NEG_INF_F) {
        for (int i = tid; i < a.V; i += 256) dx[i] = (T)0.f;
        return;
    }
    const int64_t b = r / a.inner;
    const T *x = logits + b * a.so + (r - b * a.inner) * a.si;
    const float m = a.stats[r], H = a.stats[2 * a.rows + r];
    const float gh = a.g_entropy ? a.g_entropy[r] : 0.f;
    if (tid <= a.top) {
        float g = 0.f;
        int64_t id = -1;
        if (tid == 0 && a.g_logprobs) {
            id = tok;
            g = tok >= a.V ? __builtin_nanf("") : a.g_logprobs[r];
        } else if (tid > 0 && a.g_top) {
            id = a.top_tokens[r * a.top + tid - 1];
            g = a.g_top[r * a.top + tid - 1];
        }
        s_g[tid] = g;
        s_i[tid] = id;
    }
    __syncthreads();
    float G = 0.f;
    for (int k = 0; k <= a.top; k++) G += s_g[k];
    for (int i = tid; i < a.V; i += 256) {
        const float lp = ((float)x[i] - m) - lz;
        float v = -__expf(lp) * (G + gh * (fmaxf(lp, -1e30f) + H));
        for (int k = 0; k <= a.top; k++)
            if (s_i[k] == i) v += s_g[k];
        dx[i] = (T)v;
    }
}

int check_sizes(const char *who, int dtype, int64_t outer, int64_t inner, int64_t so, int64_t si, int64_t V, int top) {
    PCFGNAT_REQUIRE(vocab_dtype_ok(dtype), "%s: logits must be float16, bfloat16 or float32", who);
    PCFGNAT_REQUIRE(outer >= 0 && inner >= 0 && (outer == 0 || inner <= 2147483647 / outer) && V >= 1 && V <= (1 << 30) && so >= 0 && si >= 0,
                    "%s: bad dimensions", who);
    PCFGNAT_REQUIRE(top >= 0 && top <= MAX_TOP && top <= V, "%s: between 0 and %d alternatives, at most the vocabulary (got %d of %lld)", who,
                    MAX_TOP, top, (long long)V);
    return PCFGNAT_OK;
}

}  // namespace
}  // namespace pcfgnat

using namespace pcfgnat;

extern "C" size_t pcfgnat_token_logprobs_workspace_bytes(int dtype, int64_t rows, int64_t V, int top) {
    (void)dtype;
    (void)rows;
    (void)V;
    (void)top;
    return 0;
}

extern "C" int pcfgnat_token_logprobs(const void *logits, int dtype, int64_t outer, int64_t inner, int64_t stride_outer,
                                      int64_t stride_inner, const int64_t *tokens, float *logprobs, float *entropy, int top,
                                      float *top_logprobs, int64_t *top_tokens, float *stats, void *workspace, int64_t V, void *stream) {
    const int rc = check_sizes("token_logprobs", dtype, outer, inner, stride_outer, stride_inner, V, top);
    if (rc != PCFGNAT_OK) return rc;
    if (outer * inner == 0) return PCFGNAT_OK;
    PCFGNAT_REQUIRE(logits && (tokens == nullptr) == (logprobs == nullptr) && (top == 0 || (top_logprobs && top_tokens)),
                    "token_logprobs: null pointer");
    const int64_t rows = outer * inner;
    const LogprobArgs a{tokens, logprobs, entropy, top_logprobs, top_tokens, stats, rows, inner, stride_outer, stride_inner, (int)V, top};
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)rows), block(256);
    if (dtype == PCFGNAT_F16) hipLaunchKernelGGL(logprobs_kernel<f16>, grid, block, 0, s, (const f16 *)logits, a);
    else if (dtype == PCFGNAT_BF16) hipLaunchKernelGGL(logprobs_kernel<bf16>, grid, block, 0, s, (const bf16 *)logits, a);
    else hipLaunchKernelGGL(logprobs_kernel<float>, grid, block, 0, s, (const float *)logits, a);
    PCFGNAT_HIP_CHECK(hipGetLastError());
    return PCFGNAT_OK;
}

extern "C" int pcfgnat_token_logprobs_backward(const void *logits, int dtype, int64_t outer, int64_t inner, int64_t stride_outer,
                                               int64_t stride_inner, const int64_t *tokens, const int64_t *top_tokens, int top,
                                               const float *stats, const float *grad_logprobs, const float *grad_entropy,
                                               const float *grad_top, void *grad_logits, int64_t V, void *stream) {
    const int rc = check_sizes("token_logprobs_backward", dtype, outer, inner, stride_outer, stride_inner, V, top);
    if (rc != PCFGNAT_OK) return rc;
    if (outer * inner == 0) return PCFGNAT_OK;
    PCFGNAT_REQUIRE(logits && stats && grad_logits && (tokens || !grad_logprobs) && (top_tokens || !grad_top || top == 0),
                    "token_logprobs_backward: null pointer");
    const int64_t rows = outer * inner;
    const LogprobGradArgs a{tokens, top_tokens, stats, grad_logprobs, grad_entropy, grad_top, rows, inner, stride_outer, stride_inner, (int)V, top};
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)rows), block(256);
    if (dtype == PCFGNAT_F16) hipLaunchKernelGGL(logprobs_grad_kernel<f16>, grid, block, 0, s, (const f16 *)logits, (f16 *)grad_logits, a);
    else if (dtype == PCFGNAT_BF16)
        hipLaunchKernelGGL(logprobs_grad_kernel<bf16>, grid, block, 0, s, (const bf16 *)logits, (bf16 *)grad_logits, a);
    else hipLaunchKernelGGL(logprobs_grad_kernel<float>, grid, block, 0, s, (const float *)logits, (float *)grad_logits, a);
    PCFGNAT_HIP_CHECK(hipGetLastError());
    return PCFGNAT_OK;
}
