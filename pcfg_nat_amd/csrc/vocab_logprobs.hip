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
constexpr int MAX_PARTS = 64;
constexpr int64_t MAX_LOGPROB_VOCAB = (int64_t)MAX_PARTS * 256 * 20 * 4;  // of what a part's workgroup holds, of float32

struct LogprobArgs {
    const int64_t *tokens;
    float *logprobs, *entropy, *top_logprobs;
    int64_t *top_tokens;
    float *stats;  // m, log Z and H of every row, [3][rows]
    int64_t rows, inner, so, si;
    int V, top;
};

// Makes the compiler forget what it knows about a chunk in registers, so that each pass widens it anew instead of keeping
// the wide values alive.
__device__ __forceinline__ void opaque(vec16 &v) { asm volatile("" : "+v"(v)); }

// Order of the alternatives as a whole number: value first (NaN largest, -0 = +0), then the lower index.  Never 0
// and never all ones, so both can stand for "no key".
__device__ __forceinline__ unsigned order_of(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const unsigned b = __float_as_uint(x + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
constexpr unsigned LOWEST_ORDER = 0x007FFFFFu;  // of -inf
__device__ __forceinline__ unsigned long long key_of(float x, int i) {
    return ((unsigned long long)order_of(x) << 32) | (0xFFFFFFFEu - (unsigned)i);
}
__device__ __forceinline__ float value_of_order(unsigned o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o); }
__device__ __forceinline__ float value_of(unsigned long long key) { return value_of_order((unsigned)(key >> 32)); }
__device__ __forceinline__ int index_of(unsigned long long key) { return (int)(0xFFFFFFFEu - (unsigned)key); }

// The rows of a launch: x and y of the grid (a dimension of a grid ends at 2^32 threads), parts of a row z.
constexpr int64_t GRID_X = 1 << 20;
inline dim3 row_grid(int64_t rows, int64_t parts = 1) {
    return dim3((unsigned)(rows < GRID_X ? rows : GRID_X), (unsigned)((rows + GRID_X - 1) / GRID_X), (unsigned)parts);
}
__device__ __forceinline__ unsigned row_of_grid() { return blockIdx.y * (unsigned)GRID_X + blockIdx.x; }

// Row r of the logits.  (rows < 2^31: a 32-bit division, and none at all where one stride covers the rows)
template <typename T>
__device__ __forceinline__ const T *row_at(const T *logits, unsigned r, int64_t inner, int64_t so, int64_t si, bool one_stride) {
    if (one_stride) return logits + (int64_t)r * si;
    const unsigned b = r / (unsigned)inner;
    return logits + (int64_t)b * so + (int64_t)(r - b * (unsigned)inner) * si;
}

template <int NT>
struct Shared {
    static constexpr int NW = NT / 64;
    static constexpr int MAX_KEYS = NT == 64 ? 256 : 1024;  // candidates that the workgroup puts in order
    float max[NW], tau[NW], z[NW], s[NW];
    int count[NW];
    int n;
    unsigned long long key[MAX_KEYS];
};

template <int NT>
__device__ __forceinline__ int block_count(int v, Shared<NT> &sh, int tid) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((tid & 63) == 0) sh.count[tid >> 6] = v;
    __syncthreads();
    int t = 0;
    for (int w = 0; w < Shared<NT>::NW; w++) t += sh.count[w];
    return t;
}

// Appends the keys of those of N values (indexes first, first + 1, ...) that `want` names to the list, as far as it goes; their
// number is counted on.
template <int NT, int N, typename Want>
__device__ __forceinline__ void append_keys(Shared<NT> &sh, const float (&o)[N], int first, Want want) {
    unsigned which = 0;
#pragma unroll
    for (int k = 0; k < N; k++) which |= want(o[k]) ? 1u << k : 0u;
    if (which == 0) return;
    int at = atomicAdd(&sh.n, __popc(which));
#pragma unroll
    for (int k = 0; k < N; k++)
        if (which & (1u << k)) {
            if (at < Shared<NT>::MAX_KEYS) sh.key[at] = key_of(o[k], first + k);
            at++;
        }
}

// The q-th largest of a wave's values, which hold no NaN, equal ones counted one by one (fewer than q above -inf: -inf): the
// largest taken away again and again, or, where that are many times, bit by bit as far down as the type has bits.
template <typename T, int G>
__device__ __forceinline__ float nth_largest_bitwise(const float (&v)[G], int q) {
    unsigned t = 0;
    for (unsigned bit = 0x80000000u; bit >= VocabElem<T>::LOWEST_BIT; bit >>= 1) {
        const float trial = (t | bit) > LOWEST_ORDER ? value_of_order(t | bit) : NEG_INF_F;
        int have = 0;
#pragma unroll
        for (int g = 0; g < G; g++) have += __popcll(__ballot(v[g] >= trial));
        if (have >= q) t |= bit;
    }
    if (!(t & 0x80000000u)) t |= VocabElem<T>::LOWEST_BIT - 1;  // (a negative value's order has ones below its last bit)
    return t > LOWEST_ORDER ? value_of_order(t) : NEG_INF_F;
}
template <typename T>
__device__ __forceinline__ float nth_largest(float v, float largest, int q) {
    if (q > 8) {
        const float one[1] = {v};
        return nth_largest_bitwise<T, 1>(one, q);
    }
    for (;;) {
        const int equal = __popcll(__ballot(v == largest));
        q -= equal > 0 ? equal : 1;
        if (q <= 0) return largest;
        v = v == largest ? NEG_INF_F : v;
        largest = wave_max_raw(v);
    }
}

// Calls f(the values of a chunk, or the one of the scalar besides; their first index) for the elements of a span, reading them
// from memory, two chunks a thread on their way at once.
template <typename T, int NT, typename F>
__device__ __forceinline__ void for_each(const T *x, const Span<T> &sp, int tid, F f) {
    constexpr int N = VocabElem<T>::N, U = 2;
    const int e = sp.edge(tid);
    if (e >= 0) {
        const float o[1] = {(float)x[e]};
        f(o, e);
    }
    const vec16 *xv = reinterpret_cast<const vec16 *>(x + sp.head);
    for (int c = tid; c < sp.nvec; c += U * NT) {
        vec16 v[U];
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = xv[c + u * NT < sp.nvec ? c + u * NT : c];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (c + u * NT < sp.nvec) {
                float o[N];
                VocabElem<T>::unpack(v[u], o);
                f(o, sp.head + (c + u * NT) * N);
            }
    }
}

__device__ unsigned long long g_selections;  // diagnostic: rows whose alternatives went through select_any

// The `want` largest of a span whatever it holds (NaN, a constant, a mask that leaves fewer than `want`), where at least `want`
// elements lie at or above `guess` in the order of `order_of`.  Everything above the guess is listed: where that is at least
// `want` and fits (a NaN among ordinary logits) nothing else is done; where it is fewer (most of the span is one value, a
// mask's) the lowest indexes of those equal to the guess follow.  Otherwise the want-th largest is found bit by bit first.
// Reads the span again for each step.  Returns how many keys it leaves in sh.key, `want` or more.
template <typename T, int NT>
__device__ __forceinline__ int select_any(const T *x, const Span<T> &sp, int want, unsigned guess, Shared<NT> &sh, int tid) {
    constexpr int N = VocabElem<T>::N;
    if (tid == 0) atomicAdd(&g_selections, 1ULL);
    const vec16 *xv = reinterpret_cast<const vec16 *>(x + sp.head);
    const auto list_above = [&](unsigned t) {
        __syncthreads();
        if (tid == 0) sh.n = 0;
        __syncthreads();
        for_each<T, NT>(x, sp, tid, [&](const auto &o, int first) { append_keys<NT>(sh, o, first, [&](float v) { return order_of(v) > t; }); });
        __syncthreads();
        return sh.n;
    };
    unsigned t = guess;
    int n = list_above(t);  // (the same for every thread)
    if (n > Shared<NT>::MAX_KEYS) {
        t = 0;
        for (unsigned bit = 0x80000000u; bit != 0; bit >>= 1) {
            int k = 0;
            for_each<T, NT>(x, sp, tid, [&](const auto &o, int) {
                for (const float v : o) k += order_of(v) >= (t | bit) ? 1 : 0;
            });
            if (block_count<NT>(k, sh, tid) >= want) t |= bit;
        }
        n = list_above(t);
    }
    const int above = n;
    // ties in ascending index: the head, rounds of one chunk a thread, the tail
    const int rounds = (sp.nvec + NT - 1) / NT;
    for (int round = -1; round <= rounds && n < want; round++) {
        float o[N];
        int first = 0, have = 0;
        if (round == -1 || round == rounds) {
            first = round == -1 ? tid : sp.head + sp.nvec * N + tid;
            have = tid < (round == -1 ? sp.head : sp.tail) ? 1 : 0;
            if (have) o[0] = (float)x[first];
        } else if (tid + round * NT < sp.nvec) {
            first = sp.head + (tid + round * NT) * N;
            have = N;
            VocabElem<T>::unpack(xv[tid + round * NT], o);
        }
        int mine = 0;
#pragma unroll
        for (int i = 0; i < N; i++) mine += i < have && order_of(o[i]) == t ? 1 : 0;
        int upto = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const int w = __shfl_up(upto, d);
            if ((tid & 63) >= d) upto += w;
        }
        __syncthreads();
        if ((tid & 63) == 63) sh.count[tid >> 6] = upto;
        __syncthreads();
        int before = upto - mine, all = 0;
        for (int w = 0; w < Shared<NT>::NW; w++) {
            if (w < (tid >> 6)) before += sh.count[w];
            all += sh.count[w];
        }
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < have && order_of(o[i]) == t) {
                if (n + before < want) sh.key[n + before] = key_of(o[i], first + i);
                before++;
            }
        n += all;
        __syncthreads();
    }
    return above < want ? want : above;
}

// What one workgroup finds in its part of a row, in base 2: z = sum of 2^t, s = sum of 2^t t, where t = (x - m) log2 e + shift.
// (shift: the rounding of m log2 e, which the sums share and the results undo.)  m = -inf, z = 0 where there is nothing.
struct Part {
    float m, z, s, shift;
};
// How far from zero the maximum may lie for that.  2^shift is the largest term of the sums, so the shift has to stay far within
// float32's exponents: below 2^24 it is at most 1, half a step of the product; at 5e9 it reaches 256, and 2^256 and 2^-256 are
// inf and 0.  (All of float16 lies below.)
constexpr float MAX_SHIFTED = 16777216.f;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// One workgroup of NT threads over n elements at x, with up to MAXC chunks of 16 bytes a thread in registers: memory is
// read once, all loads on their way together.
//
// Sums: one fused multiply-add (which also widens a float16), one exponential, one addition and one multiply-add an
// element.  Where an entry is -inf its t is too and s becomes NaN; a wave that finds one forms its s again from the
// registers, with t clamped.  Rows whose largest entry lies so far from zero that 2^shift could leave float32 take the careful
// form, which subtracts the maximum first, needs no shift, and reads them again (6400 rows of 40000 bfloat16 142 us instead of 87).
//
// Alternatives: from every wave the q-th largest of its lanes' maxima (q = top / waves, rounded up), equal ones counted one by
// one, the lowest of them over the waves: at least `top` elements lie at or above it, and of ordinary logits hardly more (some 30 for 20 of
// 40000).  The chunks that hold one are known from the first pass's maxima; they alone are read again and their candidates
// listed, to be put in order by counting.  What overflows the list (a constant, a mask) or holds a NaN goes to select_any.
// Leaves in sh.key[0..kept) the keys of the candidates, all of the `top` largest among them.
// With `lanes` the alternatives are left to another launch: each lane leaves the maximum of its elements there.
template <typename T, int NT, int MAXC>
__device__ __forceinline__ Part scan_part(const T *x, int n, int top, bool keep, Shared<NT> &sh, int tid, int &kept, float *lanes) {
    constexpr int N = VocabElem<T>::N;
    constexpr int NW = NT / 64, FEW = 2;
    const Span<T> sp(x, n);
    const int wave = tid >> 6, lane = tid & 63;
    const vec16 *xv = reinterpret_cast<const vec16 *>(x + sp.head);
    // (no branch around a load, whose result would be waited for at its end: threads behind the last chunk read that one again)
    vec16 buf[MAXC];
    const int ei = sp.edge(tid);
    const T edge_raw = x[ei >= 0 ? ei : 0];
    if (sp.nvec == 0) {
#pragma unroll
        for (int i = 0; i < MAXC; i++) buf[i] = vec16{0u, 0u, 0u, 0u};
    } else if (keep) {  // the backward reads the row again: leave it in the memory-side cache
#pragma unroll
        for (int i = 0; i < MAXC; i++) buf[i] = xv[tid + i * NT < sp.nvec ? tid + i * NT : sp.nvec - 1];
    } else {
#pragma unroll
        for (int i = 0; i < MAXC; i++) buf[i] = __builtin_nontemporal_load(xv + (tid + i * NT < sp.nvec ? tid + i * NT : sp.nvec - 1));
    }
    if (tid == 0) sh.n = 0;

    typename VocabElem<T>::Max cm[MAXC], mx;
#pragma unroll
    for (int i = 0; i < MAXC; i++) {
        cm[i].take(buf[i]);
        if (tid + i * NT >= sp.nvec) cm[i] = typename VocabElem<T>::Max();
        mx.take(cm[i]);
    }
    const float edge = ei >= 0 ? (float)edge_raw : NEG_INF_F;
    const float mine = max2_raw(mx.value(), edge);
    if (lanes != nullptr) lanes[tid] = mine;
    float m = wave_max_raw(mine), tau = m;
    if (NW == 1 && MAXC <= FEW && top > 24) {
        // one wave, a short row and a long list: the top-th largest element itself (maxima would leave a good part of the row)
        float o[MAXC * N + 1];
        o[MAXC * N] = edge;
#pragma unroll
        for (int i = 0; i < MAXC; i++) {
            float c[N];
            VocabElem<T>::unpack(buf[i], c);
#pragma unroll
            for (int k = 0; k < N; k++) o[i * N + k] = tid + i * NT < sp.nvec ? c[k] : NEG_INF_F;
        }
        tau = nth_largest_bitwise<T>(o, top);
    } else if (NW == 1 && top > 24) {
        // two maxima a lane: twice as many as the longest list, so that their top-th largest leaves little besides
        typename VocabElem<T>::Max half[2];
#pragma unroll
        for (int i = 0; i < MAXC; i++) half[i & 1].take(cm[i]);
        const float o[2] = {max2_raw(half[0].value(), edge), half[1].value()};
        tau = nth_largest_bitwise<T>(o, top);
    } else if (top > 0) {
        tau = nth_largest<T>(mine, m, (top + NW - 1) / NW);
    }
    if (lane == 0) {
        sh.max[wave] = m;
        sh.tau[wave] = tau;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) {
        m = max2_raw(m, sh.max[w]);
        tau = sh.tau[w] < tau ? sh.tau[w] : tau;
    }
    // chunks that hold a candidate: out of the registers where a thread has few, read again where it has many - the first
    // one's read is on its way during the sums
    unsigned hold = 0;
    vec16 held = {0u, 0u, 0u, 0u};
    if (top > 0) {
#pragma unroll
        for (int i = 0; i < MAXC; i++)
            if (cm[i].value() >= tau && tid + i * NT < sp.nvec) hold |= 1u << i;
        if (MAXC > FEW && hold) held = xv[tid + __builtin_ctz(hold) * NT];
    }
    const float mm = m == NEG_INF_F ? 0.f : m;
    float z = 0.f, s = 0.f, shift = 0.f;
    const bool careful = !(fabsf(mm) < MAX_SHIFTED);
    if (!careful) {
        const float nb = -(mm * LOG2E);
        shift = __builtin_fmaf(mm, LOG2E, nb);
        if (ei >= 0) {
            const float t = __builtin_fmaf(edge, LOG2E, nb);
            z = __builtin_amdgcn_exp2f(t);
            s = z * t;
        }
#pragma unroll
        for (int i = 0; i < MAXC; i++) {
            opaque(buf[i]);
            if (tid + i * NT < sp.nvec) {
                float o[N];
                VocabElem<T>::unpack(buf[i], o);
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const float t = __builtin_fmaf(o[k], LOG2E, nb), e = __builtin_amdgcn_exp2f(t);
                    z += e;
                    s = __builtin_fmaf(e, t, s);
                }
            }
        }
        if (__ballot(s != s) != 0) {
            s = 0.f;
            const auto add = [&](float v) {
                const float t = __builtin_fmaf(v, LOG2E, nb);
                s = __builtin_fmaf(__builtin_amdgcn_exp2f(t), fmaxf(t, -1e30f), s);
            };
            if (ei >= 0) add(edge);
#pragma unroll
            for (int i = 0; i < MAXC; i++) {
                opaque(buf[i]);
                if (tid + i * NT < sp.nvec) {
                    float o[N];
                    VocabElem<T>::unpack(buf[i], o);
#pragma unroll
                    for (int k = 0; k < N; k++) add(o[k]);
                }
            }
        }
    }
    if (top > 0) {
        const auto take = [&](float v, int i) {
            if (v >= tau) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < Shared<NT>::MAX_KEYS) sh.key[at] = key_of(v, i);
                else hold = 0;  // (too many: not worth the rest)
            }
        };
        if (ei >= 0) take(edge, ei);
        float o[N];
        if (MAXC <= FEW) {
#pragma unroll
            for (int i = 0; i < MAXC; i++)
                if (hold & (1u << i)) {
                    VocabElem<T>::unpack(buf[i], o);
#pragma unroll
                    for (int k = 0; k < N; k++) take(o[k], sp.head + (tid + i * NT) * N + k);
                }
        } else {
            while (hold) {
                const int c = tid + __builtin_ctz(hold) * NT;
                VocabElem<T>::unpack(held, o);
                hold &= hold - 1;
                if (hold) held = xv[tid + __builtin_ctz(hold) * NT];
#pragma unroll
                for (int k = 0; k < N; k++) take(o[k], sp.head + c * N + k);
            }
        }
    }
    if (careful)  // (the same for every thread)
        for_each<T, NT>(x, sp, tid, [&](const auto &o, int) {
            for (const float v : o) {
                const float d = v - mm, e = __builtin_amdgcn_exp2f(d * LOG2E);
                z += e;
                s = __builtin_fmaf(e, fmaxf(d, -1e30f) * LOG2E, s);
            }
        });
    z = wave_sum(z);
    s = wave_sum(s);
    if (lane == 0) {
        sh.z[wave] = z;
        sh.s[wave] = s;
    }
    __syncthreads();
    z = sh.z[0];
    s = sh.s[0];
#pragma unroll
    for (int w = 1; w < NW; w++) {
        z += sh.z[w];
        s += sh.s[w];
    }
    if (top > 0) {
        const int want = top < n ? top : n;
        kept = sh.n;
        if (kept > Shared<NT>::MAX_KEYS || kept < want || z != z) {  // (the same for every thread)
            kept = select_any<T, NT>(x, sp, want, order_of(tau), sh, tid);
        }
    }
    return Part{m, z, s, shift};
}

// The results of a row but its alternatives, by one thread.
__device__ __forceinline__ void write_row(const LogprobArgs &a, int64_t r, int64_t tok, float x_tok, float mm, float lz, float H, bool none) {
    if (a.tokens) a.logprobs[r] = tok >= a.V ? __builtin_nanf("") : none ? NEG_INF_F : (x_tok - mm) - lz;
    if (a.entropy) a.entropy[r] = H;
    if (a.stats) {
        a.stats[r] = mm;
        a.stats[a.rows + r] = lz;
        a.stats[2 * a.rows + r] = H;
    }
}
__device__ __forceinline__ void write_left_out(const LogprobArgs &a, int64_t r, int tid) {
    if (tid == 0) {
        a.logprobs[r] = 0.f;
        if (a.entropy) a.entropy[r] = 0.f;
    }
    for (int k = tid; k < a.top; k += 64) {
        a.top_logprobs[r * a.top + k] = NEG_INF_F;
        a.top_tokens[r * a.top + k] = -1;
    }
}
// Calls f(key, place) for the keys whose place among the n in LDS - how many are larger - is below `top`; eight lanes count
// for each key.
template <int NT, typename F>
__device__ __forceinline__ void in_order(const unsigned long long *keys, int n, int top, int tid, F f) {
    for (int i0 = 0; i0 < n; i0 += NT / 8) {
        const int i = i0 + (tid >> 3);
        const unsigned long long key = i < n ? keys[i] : ~0ull;
        int rank = 0;
#pragma unroll 4
        for (int j = tid & 7; j < n; j += 8) rank += keys[j] > key ? 1 : 0;
        rank += dpp_i<DPP_QUAD_XOR1>(rank);
        rank += dpp_i<DPP_QUAD_XOR2>(rank);
        rank += dpp_i<DPP_ROW_HALF_MIRROR>(rank);
        if ((tid & 7) == 0 && i < n && rank < top) f(key, rank);
    }
}

// A workgroup per row, the whole of it in registers, so that memory is read once.  What bounds it is that read where the rows are
// many: 6400 rows of 40000 float16 with 20 alternatives and entropy, 512 MB, take 89 us, 5.8 TB/s (a read alone reaches 6.4);
// 5120 rows, a third of them left out, without alternatives, 274 MB, take 51 us, 5.3 TB/s, where a backward is to come: then
// the reads leave the rows in the memory-side cache (past it 46 us, but the backward 139 us instead of 94).  One row of 40000 takes 6 us: the
// launch, then load, maxima, sums and alternatives one behind the other.  Short rows are bound by these steps of each
// workgroup: 16000 rows of 8000 float16 with 20 alternatives 53 us, 4.8 TB/s (without 45 us), of 1000 with 5 15 us (9 us).
template <typename T, int NT, int MAXC>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(MAXC >= 16 ? 4 : 1))) void logprobs_kernel(const T *__restrict__ logits, LogprobArgs a) {
    __shared__ Shared<NT> sh;
    const unsigned r = row_of_grid();
    if (r >= a.rows) return;
    const int tid = threadIdx.x;
    const int64_t tok = a.tokens ? a.tokens[r] : 0;
    if (tok < 0) {
        if (tid < 64) write_left_out(a, r, tid);
        return;
    }
    const T *x = row_at(logits, r, a.inner, a.so, a.si, a.inner == a.rows);
    const T x_tok = x[tok < a.V ? tok : 0];
    int kept = 0;
    const Part p = scan_part<T, NT, MAXC>(x, a.V, a.top, a.stats != nullptr, sh, tid, kept, nullptr);
    const bool none = p.z == 0.f;  // nothing but -inf (a NaN makes z NaN)
    const float mm = none ? 0.f : p.m, l2 = log2f(p.z), lz = (l2 - p.shift) * LN2, H = none ? 0.f : (l2 - p.s / p.z) * LN2;
    if (tid == 0) write_row(a, r, tok, (float)x_tok, mm, lz, H, none);
    in_order<NT>(sh.key, kept, a.top, tid, [&](unsigned long long key, int k) {
        a.top_tokens[(int64_t)r * a.top + k] = index_of(key);
        a.top_logprobs[(int64_t)r * a.top + k] = none ? NEG_INF_F : (value_of(key) - mm) - lz;
    });
}

// A row in several parts, where it is more than the registers of a workgroup hold.  Each part's workgroup leaves its sums and
// the maximum of every lane's elements in the workspace: two words, then PART_NT floats (64 rows of 250007 float32, 64 MB, in
// 13 parts each: 12.4 us, 5.2 TB/s, 832 workgroups being little more than three a CU) ...
constexpr int PART_NT = 256, PART_MAXC = 20;
constexpr int PART_WORDS = 2 + PART_NT / 2;
template <typename T>
__global__ __launch_bounds__(PART_NT) void logprobs_part_kernel(const T *__restrict__ logits, LogprobArgs a, int part_len,
                                                                unsigned long long *__restrict__ work) {
    __shared__ Shared<PART_NT> sh;
    const unsigned r = row_of_grid();
    if (r >= a.rows) return;
    const int part = blockIdx.z, parts = gridDim.z, tid = threadIdx.x;
    if (a.tokens && a.tokens[r] < 0) return;
    const int base = part * part_len;
    const T *x = row_at(logits, r, a.inner, a.so, a.si, a.inner == a.rows) + base;
    const int n = a.V - base < part_len ? a.V - base : part_len;
    unsigned long long *out = work + ((int64_t)r * parts + part) * PART_WORDS;
    int none = 0;
    const Part p = scan_part<T, PART_NT, PART_MAXC>(x, n, 0, true, sh, tid, none, a.top > 0 ? reinterpret_cast<float *>(out + 2) : nullptr);
    if (tid == 0) {
        out[0] = ((unsigned long long)__float_as_uint(p.z) << 32) | __float_as_uint(p.m);
        out[1] = ((unsigned long long)__float_as_uint(p.shift) << 32) | __float_as_uint(p.s);
    }
}

// ... and a workgroup per row joins the sums, rescaled to the row's maximum, and finds the alternatives: a threshold from the
// lanes' maxima as scan_part takes it from its own, the lanes at or above it (hardly more than `top` of some thousand),
// whose elements alone are read again, their candidates in order.  It is a chain of three reads, each waiting for the one
// before, 11.4 us of 1024 threads for 64 alternatives of 64 rows; where the rows are many, smaller workgroups that overlap
// each other are faster (both launches with 1024 and with 256 threads, 20 alternatives: 2000 rows of 131000 float16 162 and 116 us,
// 256 rows of 250007 float32 53 and 52 us, 128 rows 31 and 33 us, 64 rows 20.5 and 23.4 us).  (Ordered lists from every part
// instead: 38 instead of 25 us for 64 alternatives of those 64 rows.)
template <typename T, int JOIN_NT>
__global__ __launch_bounds__(JOIN_NT) void logprobs_join_kernel(const T *__restrict__ logits, LogprobArgs a, int part_len, int parts,
                                                                const unsigned long long *__restrict__ work) {
    constexpr int N = VocabElem<T>::N, NW = JOIN_NT / 64, MAX_LANES = 512;
    __shared__ Shared<JOIN_NT> sh;
    __shared__ int s_lane[MAX_LANES];
    __shared__ int s_lanes;
    const unsigned r = row_of_grid();
    if (r >= a.rows) return;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t tok = a.tokens ? a.tokens[r] : 0;
    if (tok < 0) {
        if (tid < 64) write_left_out(a, r, tid);
        return;
    }
    const T *x = row_at(logits, r, a.inner, a.so, a.si, a.inner == a.rows);
    const T x_tok = x[tok < a.V ? tok : 0];
    const unsigned long long *in = work + (int64_t)r * parts * PART_WORDS;
    // the lanes' maxima: U a thread on their way from here on, more than that are read again.  Every wave takes the same
    // number of lanes of every part, the threshold being taken from all waves: a wave without lanes (three parts have 768 for
    // 1024 threads) or with those of one part alone, which may be masked, would send the row to select_any (64 rows of 50257
    // float32, 20 alternatives: 196 us, as it is 12.8; 64 of 70001 with a quarter masked: 250 and 14).
    constexpr int U = 4, SHARE = PART_NT / NW, AT_ONCE = 64 / SHARE;
    const int all = a.top > 0 ? parts * PART_NT : 0;
    const auto lane_at = [&](int u) { return (lane / SHARE + u * AT_ONCE) * PART_NT + wave * SHARE + lane % SHARE; };
    const auto lane_max = [&](int l) { return reinterpret_cast<const float *>(in + (l / PART_NT) * PART_WORDS + 2)[l % PART_NT]; };
    float v[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int l = lane_at(u);
        v[u] = lane_max(l < all ? l : 0);  // (without alternatives nobody has written it and nobody looks at it)
        if (l >= all) v[u] = NEG_INF_F;
    }
    // every wave forms the row's sums, lane by lane over the parts
    float m_p = NEG_INF_F, z_p = 0.f, s_p = 0.f, shift_p = 0.f;
    if (lane < parts) {
        const unsigned long long zm = in[lane * PART_WORDS], hs = in[lane * PART_WORDS + 1];
        m_p = __uint_as_float((unsigned)zm);
        z_p = __uint_as_float((unsigned)(zm >> 32));
        s_p = __uint_as_float((unsigned)hs);
        shift_p = __uint_as_float((unsigned)(hs >> 32));
    }
    const float m = wave_max(m_p), mm = m == NEG_INF_F ? 0.f : m;
    float z = 0.f, s = 0.f;
    if (z_p != 0.f) {  // (a part that holds a NaN makes z NaN)
        // a part's t is larger than the row's by the rounding of its own maximum and by the distance of the two maxima
        const float d = __builtin_fmaf(fmaxf(m_p - mm, -1e30f), LOG2E, -shift_p), f = exp2f(d);
        z = z_p * f;
        s = f * (s_p + z_p * d);
    }
    z = wave_sum(z);
    s = wave_sum(s);
    const bool none = z == 0.f;
    const float l2 = log2f(z), lz = l2 * LN2, H = none ? 0.f : (l2 - s / z) * LN2;
    if (tid == 0) write_row(a, r, tok, (float)x_tok, mm, lz, H, none);
    if (a.top == 0) return;

    float mine = NEG_INF_F;
#pragma unroll
    for (int u = 0; u < U; u++) mine = max2_raw(mine, v[u]);
    for (int u = U; lane_at(u) < all; u++) mine = max2_raw(mine, lane_max(lane_at(u)));
    float tau = nth_largest<T>(mine, wave_max_raw(mine), (a.top + NW - 1) / NW);
    if (lane == 0) sh.tau[wave] = tau;
    if (tid == 0) sh.n = s_lanes = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) tau = sh.tau[w] < tau ? sh.tau[w] : tau;
    const auto list = [&](float max, int l) {
        if (max >= tau) {
            const int at = atomicAdd(&s_lanes, 1);
            if (at < MAX_LANES) s_lane[at] = l;
        }
    };
#pragma unroll
    for (int u = 0; u < U; u++)
        if (lane_at(u) < all) list(v[u], lane_at(u));
    for (int u = U; lane_at(u) < all; u++) list(lane_max(lane_at(u)), lane_at(u));
    __syncthreads();
    const int lanes = s_lanes;
    bool fits = lanes <= MAX_LANES && z == z;
    if (fits) {
        const auto take = [&](float v, int i) {
            if (v >= tau) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < Shared<JOIN_NT>::MAX_KEYS) sh.key[at] = key_of(v, i);
            }
        };
        // an item is one chunk of a lane, its last item the scalar that the lane may hold besides
        const int items = lanes * (PART_MAXC + 1);
        for (int i0 = tid; i0 < items; i0 += 4 * JOIN_NT) {
            vec16 v[4];
            int at[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                at[u] = -1;
                const int i = i0 + u * JOIN_NT;
                if (i >= items) continue;
                const int l = s_lane[i / (PART_MAXC + 1)], k = i % (PART_MAXC + 1), part = l / PART_NT, t = l % PART_NT;
                const int base = part * part_len, n = a.V - base < part_len ? a.V - base : part_len;
                const Span<T> sp(x + base, n);
                if (k == PART_MAXC) {
                    const int e = sp.edge(t);
                    if (e >= 0) take((float)x[base + e], base + e);
                } else if (t + k * PART_NT < sp.nvec) {
                    at[u] = base + sp.head + (t + k * PART_NT) * N;
                    v[u] = *reinterpret_cast<const vec16 *>(x + at[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (at[u] >= 0) {
                    float o[N];
                    VocabElem<T>::unpack(v[u], o);
#pragma unroll
                    for (int k = 0; k < N; k++) take(o[k], at[u] + k);
                }
        }
    }
    __syncthreads();
    int n = sh.n;
    if (!fits || n > Shared<JOIN_NT>::MAX_KEYS || n < a.top) {  // (the same for every thread)
        n = select_any<T, JOIN_NT>(x, Span<T>(x, a.V), a.top, order_of(tau), sh, tid);
    }
    in_order<JOIN_NT>(sh.key, n, a.top, tid, [&](unsigned long long key, int k) {
        a.top_tokens[(int64_t)r * a.top + k] = index_of(key);
        a.top_logprobs[(int64_t)r * a.top + k] = none ? NEG_INF_F : (value_of(key) - mm) - lz;
    });
}

// How a call is cut: parts of a row, each of at most MAX_CHUNKS chunks of 16 bytes.  A row that fits one workgroup's registers is
// one part however few the rows are: a second launch for the join costs more than the larger workgroup (one row of 40000
// float16: 6.4 us in one part, 8.6 us in nine; 100 rows: 7.8 and 11.2 us).
struct Cut {
    int parts, len;
};
constexpr int MAX_CHUNKS = 512 * 20, PART_CHUNKS = PART_NT * PART_MAXC;
inline Cut cut_of(int es, int64_t V) {
    const int64_t n = 16 / es, chunks = (V + n - 1) / n;
    if (chunks <= MAX_CHUNKS) return Cut{1, (int)V};
    const int64_t parts = (chunks + PART_CHUNKS - 1) / PART_CHUNKS, len = (chunks + parts - 1) / parts * n;
    return Cut{(int)((V + len - 1) / len), (int)len};
}

template <typename T, int NT, int MAXC>
void launch_rows(const T *x, const LogprobArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((logprobs_kernel<T, NT, MAXC>), row_grid(a.rows), dim3(NT), 0, s, x, a);
}
template <typename T>
int launch_forward(const void *logits, const LogprobArgs &a, void *work, hipStream_t s) {
    const T *x = (const T *)logits;
    const Cut c = cut_of((int)sizeof(T), a.V);
    const int chunks = (c.len + VocabElem<T>::N - 1) / VocabElem<T>::N;
    if (c.parts > 1) {
        unsigned long long *w = (unsigned long long *)work;
        hipLaunchKernelGGL(logprobs_part_kernel<T>, row_grid(a.rows, c.parts), dim3(PART_NT), 0, s, x, a, c.len, w);
        PCFGNAT_HIP_CHECK(hipGetLastError());
        if (a.rows < 192) hipLaunchKernelGGL((logprobs_join_kernel<T, 1024>), row_grid(a.rows), dim3(1024), 0, s, x, a, c.len, c.parts, w);
        else hipLaunchKernelGGL((logprobs_join_kernel<T, 256>), row_grid(a.rows), dim3(256), 0, s, x, a, c.len, c.parts, w);
        PCFGNAT_HIP_CHECK(hipGetLastError());
        return PCFGNAT_OK;
    }
    // The smallest workgroup whose registers hold the row without spilling: many small ones hide each other's latency, but where
    // they do not fill the chip a row's own latency counts.  Of float16 with 5, 8 or 20 alternatives:
    //    16000 rows of 8000, 20:  128 x 8 53 us, 256 x 4 67 us, 64 x 16 54 us         300 rows:  7.6, 6.5 and 9.0 us
    //    6400 rows of 40000, 20:  256 x 20 89 us, 512 x 10 94 us, 1024 x 5 196 us     100 rows, 8:  7.5, 7.0 and 7.0 us
    // (every wave of a workgroup has to have elements: the alternatives' threshold is taken from all of them)
    if (chunks <= 64 * 2) launch_rows<T, 64, 2>(x, a, s);
    else if (chunks <= 64 * 8) launch_rows<T, 64, 8>(x, a, s);
    else if (chunks <= 256 * 4 && a.rows < 1024) launch_rows<T, 256, 4>(x, a, s);
    else if (chunks <= 128 * 8) launch_rows<T, 128, 8>(x, a, s);
    else if (chunks <= 256 * 10) launch_rows<T, 256, 10>(x, a, s);
    else if (chunks <= 512 * 10 && a.rows < 512) launch_rows<T, 512, 10>(x, a, s);
    else if (chunks <= 256 * 20) launch_rows<T, 256, 20>(x, a, s);
    else launch_rows<T, 512, 20>(x, a, s);
    PCFGNAT_HIP_CHECK(hipGetLastError());
    return PCFGNAT_OK;
}

struct LogprobGradArgs {
    const int64_t *tokens, *top_tokens;
    const float *stats, *g_logprobs, *g_entropy, *g_top;
    int64_t rows, inner, so, si;
    int V, top;
};

// The gradient of one part of a row by one workgroup: NT threads, MAXC chunks of 16 bytes each, read once, written once.  What bounds
// it is memory: 5120 rows of 40000 float16, a third left out, 274 MB read and 410 MB written, take 90 us, 7.6 TB/s (part of the
// reads comes from the memory-side cache, where the forward left them); 1001 rows of 50021 bfloat16 with four alternatives,
// 190 MB in unaligned rows, 34 us, 5.6 TB/s.  Waves of 64 threads for rows of up to 128 chunks, otherwise 256.  The
// chunks follow the alignment of the gradient's row; the logits' row may lie otherwise and is read unaligned.  The entries
// at which something arrives besides (the token, the alternatives) are flagged by chunk in LDS, so that an ordinary chunk
// pays one byte of LDS for them, and are added before the one rounding, in the order of the list.
template <typename T, int NT, int MAXC>
__global__ __launch_bounds__(NT) void logprobs_grad_kernel(const T *__restrict__ logits, T *__restrict__ grad, LogprobGradArgs a) {
    constexpr int N = VocabElem<T>::N;
    __shared__ float s_g[MAX_TOP + 1];
    __shared__ int s_i[MAX_TOP + 1];
    __shared__ unsigned s_hit[NT * MAXC / 4];  // a byte for each chunk
    const unsigned r = row_of_grid();
    if (r >= a.rows) return;
    const int tid = threadIdx.x;
    const int base = blockIdx.z * (NT * MAXC * N), n = a.V - base < NT * MAXC * N ? a.V - base : NT * MAXC * N;
    T *dx = grad + (int64_t)r * a.V + base;
    const Span<T> sp(dx, n);
    vec16 *dv = reinterpret_cast<vec16 *>(dx + sp.head);
    const int64_t tok = a.tokens ? a.tokens[r] : 0;
    const float lz = tok < 0 ? NEG_INF_F : a.stats[a.rows + r];
    const int ei = sp.edge(tid);
    if (lz == NEG_INF_F) {  // left out, or nothing but -inf
        const vec16 zero = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < MAXC; i++)
            if (tid + i * NT < sp.nvec) __builtin_nontemporal_store(zero, dv + tid + i * NT);
        if (ei >= 0) dx[ei] = (T)0.f;
        return;
    }
    const T *x = row_at(logits, r, a.inner, a.so, a.si, a.inner == a.rows) + base;
    const vec16_any *xv = reinterpret_cast<const vec16_any *>(x + sp.head);
    vec16 buf[MAXC];
    const T edge = x[ei >= 0 ? ei : 0];
    if (sp.nvec > 0) {  // (threads behind the last chunk read that one again: no branch around a load)
#pragma unroll
        for (int i = 0; i < MAXC; i++) buf[i] = __builtin_nontemporal_load(xv + (tid + i * NT < sp.nvec ? tid + i * NT : sp.nvec - 1));
    } else {
#pragma unroll
        for (int i = 0; i < MAXC; i++) buf[i] = vec16{0u, 0u, 0u, 0u};
    }
    const float m = a.stats[r], H = a.stats[2 * a.rows + r];
    const float gh = a.g_entropy ? a.g_entropy[r] : 0.f;
    for (int i = tid; i < NT * MAXC / 4; i += NT) s_hit[i] = 0;
    for (int k = tid; k <= a.top; k += NT) {
        float g = 0.f;
        int id = -1;
        if (k == 0 && a.g_logprobs) {
            id = tok < a.V ? (int)tok : -1;
            g = tok < a.V ? a.g_logprobs[r] : __builtin_nanf("");
        } else if (k > 0 && a.g_top) {
            id = (int)a.top_tokens[(int64_t)r * a.top + k - 1];
            g = a.g_top[(int64_t)r * a.top + k - 1];
        }
        s_g[k] = g;
        s_i[k] = id < 0 ? -1 : id - base;  // (negative: before this part)
    }
    __syncthreads();
    for (int k = tid; k <= a.top; k += NT) {
        const int at = s_i[k] - sp.head;
        if (at >= 0 && at < sp.nvec * N) atomicOr(&s_hit[at / N / 4], 1u << (8 * (at / N % 4)));
    }
    __syncthreads();
    float K = 0.f;
    for (int k = 0; k <= a.top; k++) K += s_g[k];
    K = __builtin_fmaf(gh, H, K);
    // (below -200 the probability is 0 in float32; the bound keeps its product with gh, which may be large, from becoming 0 * inf)
    const auto of = [&](float v) {
        const float lp = (v - m) - lz;
        return -__builtin_amdgcn_exp2f(lp * LOG2E) * __builtin_fmaf(gh, fmaxf(lp, -200.f), K);
    };
    if (ei >= 0) {
        float g = of((float)edge);
        for (int k = 0; k <= a.top; k++) g += s_i[k] == ei ? s_g[k] : 0.f;
        dx[ei] = (T)g;
    }
    const unsigned char *hit = reinterpret_cast<const unsigned char *>(s_hit);
#pragma unroll
    for (int i = 0; i < MAXC; i++) {
        const int c = tid + i * NT;
        float o[N];
        VocabElem<T>::unpack(buf[i], o);
#pragma unroll
        for (int k = 0; k < N; k++) o[k] = of(o[k]);
        if (c < sp.nvec) {
            if (hit[c]) {
#pragma unroll 1
                for (int e = 0; e <= a.top; e++) {
                    const int at = s_i[e] - (sp.head + c * N);
#pragma unroll
                    for (int k = 0; k < N; k++) o[k] += at == k ? s_g[e] : 0.f;
                }
            }
            __builtin_nontemporal_store(VocabElem<T>::pack(o), dv + c);
        }
    }
}

template <typename T, int NT, int MAXC>
void launch_grad_parts(const T *x, T *dx, const LogprobGradArgs &a, hipStream_t s) {
    const int part = NT * MAXC * VocabElem<T>::N;
    hipLaunchKernelGGL((logprobs_grad_kernel<T, NT, MAXC>), row_grid(a.rows, (a.V + part - 1) / part), dim3(NT), 0, s, x, dx, a);
}
template <typename T>
int launch_backward(const void *logits, void *grad, const LogprobGradArgs &a, hipStream_t s) {
    if (a.V <= 64 * 2 * VocabElem<T>::N) launch_grad_parts<T, 64, 2>((const T *)logits, (T *)grad, a, s);
    else launch_grad_parts<T, 256, 4>((const T *)logits, (T *)grad, a, s);
    PCFGNAT_HIP_CHECK(hipGetLastError());
    return PCFGNAT_OK;
}

int check_sizes(const char *who, int dtype, int64_t outer, int64_t inner, int64_t so, int64_t si, int64_t V, int top) {
    PCFGNAT_REQUIRE(vocab_dtype_ok(dtype), "%s: logits must be float16, bfloat16 or float32", who);
    PCFGNAT_REQUIRE(outer >= 0 && inner >= 0 && (outer == 0 || inner <= 2147483647 / outer) && V >= 1 && so >= 0 && si >= 0, "%s: bad dimensions",
                    who);
    PCFGNAT_REQUIRE(V <= MAX_LOGPROB_VOCAB, "%s: a vocabulary of at most %lld entries (got %lld)", who, (long long)MAX_LOGPROB_VOCAB, (long long)V);
    PCFGNAT_REQUIRE(top >= 0 && top <= MAX_TOP && top <= V, "%s: between 0 and %d alternatives, at most the vocabulary (got %d of %lld)", who,
                    MAX_TOP, top, (long long)V);
    return PCFGNAT_OK;
}

}  // namespace
}  // namespace pcfgnat

using namespace pcfgnat;

extern "C" size_t pcfgnat_token_logprobs_workspace_bytes(int dtype, int64_t rows, int64_t V, int top) {
    if (!vocab_dtype_ok(dtype) || rows <= 0 || V < 1 || V > MAX_LOGPROB_VOCAB || top < 0) return 0;
    const Cut c = cut_of(vocab_elem_bytes(dtype), V);
    return c.parts == 1 ? 0 : (size_t)rows * c.parts * PART_WORDS * 8;
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
    PCFGNAT_REQUIRE(workspace || pcfgnat_token_logprobs_workspace_bytes(dtype, rows, V, top) == 0, "token_logprobs: null workspace");
    if (dtype == PCFGNAT_F16) return launch_forward<f16>(logits, a, workspace, s);
    if (dtype == PCFGNAT_BF16) return launch_forward<bf16>(logits, a, workspace, s);
    return launch_forward<float>(logits, a, workspace, s);
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
    if (dtype == PCFGNAT_F16) return launch_backward<f16>(logits, grad_logits, a, s);
    if (dtype == PCFGNAT_BF16) return launch_backward<bf16>(logits, grad_logits, a, s);
    return launch_backward<float>(logits, grad_logits, a, s);
}

extern "C" int pcfgnat_token_logprobs_selections(unsigned long long *rows, int reset) {
    unsigned long long h = 0;
    PCFGNAT_HIP_CHECK(hipMemcpyFromSymbol(&h, HIP_SYMBOL(g_selections), sizeof(h)));
    if (rows) *rows = h;
    if (reset) {
        const unsigned long long z = 0;
        PCFGNAT_HIP_CHECK(hipMemcpyToSymbol(HIP_SYMBOL(g_selections), &z, sizeof(z)));
    }
    return PCFGNAT_OK;
}
