// Scaled embedding lookup out[n] = scale * W[token_n] and its gradient dW[v] = scale * sum of g[n] over the n with
// token_n = v, summed in float32 in ascending n and rounded once.  A negative token is a zero row, one at or beyond V a
// row of NaN; neither has a gradient, nor has the padding index.
#include "vocab.hip.h"

namespace pcfgnat {
namespace {

// One 16-byte chunk of a row of D elements at column c: whole, or the D - c elements that are left (zeros behind them).
template <typename T>
__device__ __forceinline__ vec16 load_columns(const T *row, int64_t c, int64_t D) {
    constexpr int N = VocabElem<T>::N;
    if (c + N <= D) return *reinterpret_cast<const vec16_any *>(row + c);
    typename VocabElem<T>::vecT t;
#pragma unroll
    for (int i = 0; i < N; i++) t[i] = c + i < D ? row[c + i] : (T)0.f;
    return __builtin_bit_cast(vec16, t);
}
template <typename T>
__device__ __forceinline__ void store_columns(T *row, int64_t c, int64_t D, const vec16 &v) {
    constexpr int N = VocabElem<T>::N;
    if (c + N <= D) {
        *reinterpret_cast<vec16_any *>(row + c) = v;
        return;
    }
    const typename VocabElem<T>::vecT t = __builtin_bit_cast(typename VocabElem<T>::vecT, v);
#pragma unroll
    for (int i = 0; i < N; i++)
        if (c + i < D) row[c + i] = t[i];
}

// ---- lookup ----------------------------------------------------------------------------------------------------
// The output is one run of N * D elements, written in aligned chunks of 16 bytes: a thread takes LOOKUP_U of them, finds the
// row of each (one 64-bit division a workgroup, 32-bit ones from there), and has all its reads of the weight on their way
// before the first store.  A chunk that lies across the end of a row (D no multiple of a chunk) goes element by element.
constexpr int LOOKUP_U = 4;
template <typename T>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const T *__restrict__ weight, int64_t wstride, const int64_t *__restrict__ tokens,
                                                            float scale, T *__restrict__ out, int64_t N, int64_t V, unsigned D) {
    constexpr int E = VocabElem<T>::N;
    const int64_t first = (int64_t)blockIdx.x * (256 * LOOKUP_U * E), total = N * D;
    const int64_t row0 = first / D;
    const unsigned col0 = (unsigned)(first - row0 * D);
    vec16 w[LOOKUP_U];
    int64_t tok[LOOKUP_U];
#pragma unroll
    for (int u = 0; u < LOOKUP_U; u++) {
        const unsigned at = (threadIdx.x + 256 * u) * E, in = col0 + at, row = in / D;
        tok[u] = first + at < total ? tokens[row0 + row] : -1;
    }
#pragma unroll
    for (int u = 0; u < LOOKUP_U; u++) {
        const unsigned in = col0 + (threadIdx.x + 256 * u) * E, c = in - in / D * D;
        if (tok[u] >= 0 && tok[u] < V && c + E <= D) w[u] = *reinterpret_cast<const vec16_any *>(weight + tok[u] * wstride + c);
    }
#pragma unroll
    for (int u = 0; u < LOOKUP_U; u++) {
        const unsigned at = (threadIdx.x + 256 * u) * E, in = col0 + at, row = in / D, c = in - row * D;
        if (first + at >= total) continue;
        T *o = out + first + at;
        if (c + E <= D) {
            float f[E];
            if (tok[u] >= 0 && tok[u] < V) {
                VocabElem<T>::unpack(w[u], f);
#pragma unroll
                for (int k = 0; k < E; k++) f[k] *= scale;
            } else {
#pragma unroll
                for (int k = 0; k < E; k++) f[k] = tok[u] < 0 ? 0.f : __builtin_nanf("");
            }
            *reinterpret_cast<vec16_any *>(o) = VocabElem<T>::pack(f);
        } else {
            int64_t t = tok[u], r = row0 + row;
            unsigned cc = c;
            for (int k = 0; k < E && first + at + k < total; k++) {
                if (cc == D) {
                    cc = 0;
                    t = tokens[++r];
                }
                o[k] = (T)(t < 0 ? 0.f : t >= V ? __builtin_nanf("") : scale * (float)weight[t * wstride + cc]);
                cc++;
            }
        }
    }
}

// ---- gradient --------------------------------------------------------------------------------------------------
// Three launches, no atomics on results: the tokens in the order (token, position), sums over pieces of that order, joins of
// the sums of a token whose run was cut.  The order is a function of the tokens alone, so are the sums.
//
// What bounds it: writing all of dW (41 MB at 40000 x 512 float16, 6 us at the rate of a fill) and reading g once.  A decoder
// input of a glanced graph holds one token in most places, so runs are cut evenly by position, not by token.
struct Plan {
    int64_t N;       // positions
    int piece;       // positions of the order that one wave sums
    int64_t pieces;  // ceil(N / piece)
};
inline Plan plan_of(int64_t N, int64_t D) {
    // enough waves for the chip while pieces stay long enough that the cut runs' sums are few
    const int64_t waves = N * ((D + 511) / 512) / 2048;
    int piece = 8;
    while (piece < 64 && piece * 2 <= waves) piece *= 2;
    return Plan{N, piece, (N + piece - 1) / piece};
}
// workspace: number of positions in the order (16 bytes), positions [N], tokens [N] in the order, sums of cut runs
// [pieces][2][D] float32
inline size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }
inline size_t order_bytes(const Plan &p) { return align16((size_t)p.N * 4); }

constexpr int SORT_NT = 1024, SORT_NW = SORT_NT / 64;
constexpr int MAX_STRIP = 1024;

// Every workgroup owns a strip of the vocabulary and looks for its tokens among all of them, each wave in its sixteenth of
// the positions: first how often each occurs (and how many tokens lie below the strip, which is where the strip's part of
// the order begins: no workgroup waits for another), then each to its place, in ascending position.  Lanes with the same
// token take their places together.  The rows of the strip that no token selects are zeroed here.
template <typename T>
__global__ __launch_bounds__(SORT_NT) void embedding_order_kernel(const int64_t *__restrict__ tokens, int64_t padding_idx, int N, int64_t V,
                                                                  int strip, int64_t D, T *__restrict__ dweight, int *__restrict__ count,
                                                                  int *__restrict__ order_pos, int *__restrict__ order_tok) {
    __shared__ int s_at[SORT_NW][MAX_STRIP];
    __shared__ int s_total[MAX_STRIP];
    __shared__ int s_below[SORT_NW], s_wave[SORT_NW];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t lo = (int64_t)blockIdx.x * strip;
    const int ids = V - lo < strip ? (int)(V - lo) : strip;
    for (int i = lane; i < ids; i += 64) s_at[wave][i] = 0;
    const int groups = (N + 63) / 64, each = (groups + SORT_NW - 1) / SORT_NW;
    const int from = wave * each, to = from + each < groups ? from + each : groups;
    // the token of a lane relative to the strip, or -1; tokens below the strip are counted
    const auto local = [&](int g, int *below) {
        const int64_t t = g * 64 + lane < N ? tokens[(int64_t)g * 64 + lane] : -1;
        const bool real = t >= 0 && t < V && t != padding_idx;
        if (below) *below += __popcll(__ballot(real && t < lo));
        return real && t >= lo && t < lo + ids ? (int)(t - lo) : -1;
    };
    int below = 0;
    for (int g = from; g < to; g++) {
        const int t = local(g, &below);
        unsigned long long left = __ballot(t >= 0);
        while (left) {
            const int leader = __builtin_ctzll(left), id = __builtin_amdgcn_readlane(t, leader);
            const unsigned long long same = __ballot(t == id);
            if (lane == leader) s_at[wave][id] += __popcll(same);
            left &= ~same;
        }
    }
    if (lane == 0) s_below[wave] = below;
    __syncthreads();
    // exclusive sums over (token, wave)
    int mine = 0;
    if (tid < ids)
        for (int w = 0; w < SORT_NW; w++) mine += s_at[w][tid];
    int upto = mine;
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(upto, d);
        if (lane >= d) upto += v;
    }
    if (lane == 63) s_wave[wave] = upto;
    __syncthreads();
    int base = upto - mine;
    for (int w = 0; w < SORT_NW; w++) {
        base += s_below[w];
        if (w < wave) base += s_wave[w];
    }
    if (tid < ids) {
        int at = base;
        for (int w = 0; w < SORT_NW; w++) {
            const int c = s_at[w][tid];
            s_at[w][tid] = at;
            at += c;
        }
        s_total[tid] = mine;
        if (lo + tid == V - 1) *count = at;
    }
    __syncthreads();
    for (int g = from; g < to; g++) {
        const int t = local(g, nullptr);
        unsigned long long left = __ballot(t >= 0);
        while (left) {
            const int leader = __builtin_ctzll(left), id = __builtin_amdgcn_readlane(t, leader);
            const unsigned long long same = __ballot(t == id);
            int at = 0;
            if (lane == leader) at = atomicAdd(&s_at[wave][id], __popcll(same));
            at = __builtin_amdgcn_readlane(at, leader) + __popcll(same & ((1ull << lane) - 1));
            if (t == id) {
                order_pos[at] = g * 64 + lane;
                order_tok[at] = (int)(lo + id);
            }
            left &= ~same;
        }
    }
    const vec16 zero = {0u, 0u, 0u, 0u};
    for (int i = wave; i < ids; i += SORT_NW)
        if (s_total[i] == 0) {
            T *row = dweight + (lo + i) * D;
            for (int64_t c = (int64_t)lane * VocabElem<T>::N; c < D; c += 64 * VocabElem<T>::N) store_columns(row, c, D, zero);
        }
}

// A wave sums one piece of the order over a tile of 64 chunks of columns, 8 rows of g on their way at a time.  Runs that begin
// and end inside the piece are finished; the sums of the first and the last, where they go on outside, are left for the join.
constexpr int SUM_U = 8;
template <typename T>
__global__ __launch_bounds__(256) void embedding_sum_kernel(const T *__restrict__ g, int64_t gstride, float scale, T *__restrict__ dweight,
                                                            int64_t D, int tiles, int piece, int64_t pieces, const int *__restrict__ count,
                                                            const int *__restrict__ order_pos, const int *__restrict__ order_tok,
                                                            float *__restrict__ cut) {
    constexpr int E = VocabElem<T>::N;
    const int64_t task = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int64_t p = task / tiles;
    if (p >= pieces) return;
    const int total = *count;
    const int64_t c = ((task - p * tiles) * 64 + lane) * E;
    const int64_t from = p * piece;
    if (from >= total) return;
    const int n = total - from < piece ? (int)(total - from) : piece;
    const int my_pos = lane < n ? order_pos[from + lane] : 0, my_tok = lane < n ? order_tok[from + lane] : -1;
    const int before = from > 0 ? order_tok[from - 1] : -1, after = from + n < total ? order_tok[from + n] : -1;
    float acc[E];
#pragma unroll
    for (int k = 0; k < E; k++) acc[k] = 0.f;
    bool opened_before = before == __builtin_amdgcn_readlane(my_tok, 0);
    for (int j0 = 0; j0 < n; j0 += SUM_U) {
        vec16 buf[SUM_U];
#pragma unroll
        for (int u = 0; u < SUM_U; u++)
            if (j0 + u < n && c < D) buf[u] = load_columns(g + (int64_t)__builtin_amdgcn_readlane(my_pos, j0 + u) * gstride, c, D);
#pragma unroll
        for (int u = 0; u < SUM_U; u++) {
            const int j = j0 + u;
            if (j < n) {
                float o[E];
                VocabElem<T>::unpack(buf[u], o);
#pragma unroll
                for (int k = 0; k < E; k++) acc[k] += o[k];
                const int tok = __builtin_amdgcn_readlane(my_tok, j);
                const int next = j + 1 < n ? __builtin_amdgcn_readlane(my_tok, j + 1) : after;
                const bool last = j + 1 == n;
                if (next != tok || last) {
                    const bool goes_on = last && next == tok;
                    if (c < D) {
                        if (opened_before || goes_on) {  // slot 0: a run from before (whether or not it ends here), slot 1: one that begins here
                            float *to = cut + (p * 2 + (opened_before ? 0 : 1)) * D;
#pragma unroll
                            for (int k = 0; k < E; k++)
                                if (c + k < D) to[c + k] = acc[k];
                        } else {
                            float f[E];
#pragma unroll
                            for (int k = 0; k < E; k++) f[k] = acc[k] * scale;
                            store_columns(dweight + (int64_t)tok * D, c, D, VocabElem<T>::pack(f));
                        }
                    }
                    opened_before = false;
#pragma unroll
                    for (int k = 0; k < E; k++) acc[k] = 0.f;
                }
            }
        }
    }
}

// Joins the sums of a run that begins in piece p and goes on behind it, in the order of the pieces: each wave of the workgroup
// takes a stretch of them, the stretches are added in order.
constexpr int JOIN_NW = 8;
template <typename T>
__global__ __launch_bounds__(JOIN_NW * 64) void embedding_join_kernel(float scale, T *__restrict__ dweight, int64_t D, int piece, int64_t pieces,
                                                                      const int *__restrict__ count, const int *__restrict__ order_tok,
                                                                      const float *__restrict__ cut) {
    __shared__ float s_sum[JOIN_NW][64];
    const int64_t p = blockIdx.x, from = p * piece, end = from + piece;
    const int total = *count, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (end >= total) return;
    const int tok = order_tok[end];
    if (order_tok[end - 1] != tok) return;                                                    // nothing goes on
    if (order_tok[from] == tok && from > 0 && order_tok[from - 1] == tok) return;             // it began before
    // pieces behind p that the run reaches: those whose first position holds its token
    int64_t reach = 0;
    for (int64_t q = p + 1;; q += 64) {
        const bool in = q + lane < pieces && (q + lane) * piece < total && order_tok[(q + lane) * piece] == tok;
        const unsigned long long out = ~__ballot(in);
        reach += out ? __builtin_ctzll(out) : 64;
        if (out) break;
    }
    const int64_t each = (reach + JOIN_NW - 1) / JOIN_NW, a = p + 1 + wave * each, b = a + each < p + 1 + reach ? a + each : p + 1 + reach;
    for (int64_t c0 = (int64_t)blockIdx.y * 64; c0 < D; c0 += (int64_t)gridDim.y * 64) {
        const int64_t c = c0 + lane;
        float acc = 0.f;
        if (c < D) {
            if (wave == 0) acc = cut[(p * 2 + 1) * D + c];
#pragma unroll 8
            for (int64_t q = a; q < b; q++) acc += cut[q * 2 * D + c];
        }
        s_sum[wave][lane] = acc;
        __syncthreads();
        if (wave == 0 && c < D) {
#pragma unroll
            for (int w = 1; w < JOIN_NW; w++) acc += s_sum[w][lane];
            dweight[(int64_t)tok * D + c] = (T)(acc * scale);
        }
        __syncthreads();
    }
}

template <typename T>
int forward(const void *weight, int64_t wstride, const int64_t *tokens, float scale, void *out, int64_t N, int64_t V, int64_t D,
            hipStream_t s) {
    const int64_t each = 256 * LOOKUP_U * VocabElem<T>::N, blocks = (N * D + each - 1) / each;
    PCFGNAT_REQUIRE(blocks <= 2147483647, "token_embedding: the output is too large for one call");
    hipLaunchKernelGGL(embedding_fwd_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, (const T *)weight, wstride, tokens, scale, (T *)out, N,
                       V, (unsigned)D);
    PCFGNAT_HIP_CHECK(hipGetLastError());
    return PCFGNAT_OK;
}
template <typename T>
int backward(const void *g, int64_t gstride, const int64_t *tokens, float scale, int64_t padding_idx, void *dweight, void *workspace,
             int64_t N, int64_t V, int64_t D, hipStream_t s) {
    const Plan p = plan_of(N, D);
    const int tiles = (int)((D + 64 * VocabElem<T>::N - 1) / (64 * VocabElem<T>::N));
    const int64_t sum_blocks = (p.pieces * tiles + 3) / 4;
    PCFGNAT_REQUIRE(sum_blocks <= 2147483647, "token_embedding_backward: the gradient is too large for one call");
    char *w = (char *)workspace;
    int *count = (int *)w, *order_pos = (int *)(w + 16), *order_tok = (int *)(w + 16 + order_bytes(p));
    float *cut = (float *)(w + 16 + 2 * order_bytes(p));
    int64_t strip = (V + 255) / 256;
    strip = strip < 16 ? 16 : strip > MAX_STRIP ? MAX_STRIP : strip;
    hipLaunchKernelGGL(embedding_order_kernel<T>, dim3((unsigned)((V + strip - 1) / strip)), dim3(SORT_NT), 0, s, tokens, padding_idx, (int)N, V,
                       (int)strip, D, (T *)dweight, count, order_pos, order_tok);
    PCFGNAT_HIP_CHECK(hipGetLastError());
    if (N == 0) return PCFGNAT_OK;
    hipLaunchKernelGGL(embedding_sum_kernel<T>, dim3((unsigned)sum_blocks), dim3(256), 0, s, (const T *)g, gstride, scale, (T *)dweight, D,
                       tiles, p.piece, p.pieces, count, order_pos, order_tok, cut);
    PCFGNAT_HIP_CHECK(hipGetLastError());
    if (p.pieces > 1) {
        const unsigned split = (unsigned)((D + 63) / 64 < 64 ? (D + 63) / 64 : 64);
        hipLaunchKernelGGL(embedding_join_kernel<T>, dim3((unsigned)p.pieces, split), dim3(JOIN_NW * 64), 0, s, scale, (T *)dweight, D, p.piece,
                           p.pieces, count, order_tok, cut);
        PCFGNAT_HIP_CHECK(hipGetLastError());
    }
    return PCFGNAT_OK;
}

constexpr int64_t MAX_TOKENS = 2147483647 - 4096;  // positions are kept in 32 bits
constexpr int64_t MAX_VOCAB = 1 << 26;
constexpr int64_t MAX_DIM = 1 << 20;

}  // namespace
}  // namespace pcfgnat

using namespace pcfgnat;

extern "C" int pcfgnat_token_embedding(const void *weight, int dtype, int64_t weight_stride, const int64_t *tokens, float scale, void *out,
                                       int64_t N, int64_t V, int64_t D, void *stream) {
    PCFGNAT_REQUIRE(vocab_dtype_ok(dtype), "token_embedding: the weight must be float16, bfloat16 or float32");
    PCFGNAT_REQUIRE(N >= 0 && N <= MAX_TOKENS && V >= 1 && V <= MAX_VOCAB && D >= 1 && D <= MAX_DIM && weight_stride >= D,
                    "token_embedding: bad dimensions");
    if (N == 0) return PCFGNAT_OK;
    PCFGNAT_REQUIRE(weight && tokens && out, "token_embedding: null pointer");
    hipStream_t s = (hipStream_t)stream;
    if (dtype == PCFGNAT_F16) return forward<f16>(weight, weight_stride, tokens, scale, out, N, V, D, s);
    if (dtype == PCFGNAT_BF16) return forward<bf16>(weight, weight_stride, tokens, scale, out, N, V, D, s);
    return forward<float>(weight, weight_stride, tokens, scale, out, N, V, D, s);
}

extern "C" size_t pcfgnat_token_embedding_backward_workspace_bytes(int64_t N, int64_t V, int64_t D) {
    if (N < 0 || N > MAX_TOKENS || V < 1 || D < 1 || D > MAX_DIM) return 0;
    const Plan p = plan_of(N, D);
    return 16 + 2 * order_bytes(p) + align16((size_t)p.pieces * 2 * D * 4);
}

extern "C" int pcfgnat_token_embedding_backward(const void *grad_out, int dtype, int64_t grad_stride, const int64_t *tokens, float scale,
                                                int64_t padding_idx, void *grad_weight, void *workspace, int64_t N, int64_t V, int64_t D,
                                                void *stream) {
    PCFGNAT_REQUIRE(vocab_dtype_ok(dtype), "token_embedding_backward: the gradient must be float16, bfloat16 or float32");
    PCFGNAT_REQUIRE(N >= 0 && N <= MAX_TOKENS && V >= 1 && V <= MAX_VOCAB && D >= 1 && D <= MAX_DIM && grad_stride >= 0,
                    "token_embedding_backward: bad dimensions");
    PCFGNAT_REQUIRE(grad_weight && workspace && (N == 0 || (grad_out && tokens)), "token_embedding_backward: null pointer");
    hipStream_t s = (hipStream_t)stream;
    if (dtype == PCFGNAT_F16) return backward<f16>(grad_out, grad_stride, tokens, scale, padding_idx, grad_weight, workspace, N, V, D, s);
    if (dtype == PCFGNAT_BF16) return backward<bf16>(grad_out, grad_stride, tokens, scale, padding_idx, grad_weight, workspace, N, V, D, s);
    return backward<float>(grad_out, grad_stride, tokens, scale, padding_idx, grad_weight, workspace, N, V, D, s);
}
