// Scaled embedding lookup out[n] = scale * W[token_n] and its gradient dW[v] = scale * sum of g[n] over the n with
// token_n = v, summed in float32 in an order that the tokens alone decide, and rounded once.  A negative token is a zero row, one at or beyond V a
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
// What bounds it is memory: 131072 tokens of 128000 x 1024 bfloat16, 268 MB written and as much read, take 83 us, 6.4 TB/s (one
// read at a time 93 us); 5120 of 40000 x 512 4.2 us, one token 1.5 us, both less than the host's time for a launch.
// NARROW (here and below): rows shorter than a chunk.
constexpr int LOOKUP_U = 4;
template <typename T, bool NARROW>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const T *__restrict__ weight, int64_t wstride, const int64_t *__restrict__ tokens,
                                                            float scale, T *__restrict__ out, int64_t N, int64_t V, unsigned D) {
    constexpr int E = VocabElem<T>::N;
    const int64_t first = (int64_t)blockIdx.x * (256 * LOOKUP_U * E), total = N * D;
    const int64_t row0 = first / D;
    const unsigned col0 = (unsigned)(first - row0 * D);
    vec16 w[LOOKUP_U];
    int64_t tok[LOOKUP_U];
    // (no branch around a load, whose result would be waited for at its end: what lies behind the output's end, across a row's
    // end or outside the vocabulary reads some other place and is not used)
#pragma unroll
    for (int u = 0; u < LOOKUP_U; u++) {
        const unsigned at = (threadIdx.x + 256 * u) * E, row = (col0 + at) / D;
        tok[u] = tokens[first + at < total ? row0 + row : N - 1];
    }
#pragma unroll
    for (int u = 0; u < LOOKUP_U; u++) {
        const unsigned in = col0 + (threadIdx.x + 256 * u) * E, c = in - in / D * D;
        if (!NARROW) w[u] = *reinterpret_cast<const vec16_any *>(weight + (tok[u] >= 0 && tok[u] < V ? tok[u] : 0) * wstride + (c + E <= D ? c : D - E));
    }
#pragma unroll
    for (int u = 0; u < LOOKUP_U; u++) {
        const unsigned at = (threadIdx.x + 256 * u) * E, in = col0 + at, row = in / D, c = in - row * D;
        if (first + at >= total) continue;
        T *o = out + first + at;
        if (!NARROW && c + E <= D) {
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
#pragma unroll 1
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
// No atomics on results.  Three launches: the positions in an order that groups them by token (ascending within it), sums over
// pieces of that order, joins of the sums of a token whose run was cut.  Many positions take a fourth, for the order; few take
// one launch for all.  The order is a function of the tokens alone, so are the sums.
//
// What bounds it: writing all of dW (262 MB at 64000 x 2048 bfloat16, 38 us at the rate of a fill) and reading g once (32768
// positions, 134 MB, 21 us); the four launches of that case take 81 us, the three of 5120 positions of 40000 x 512 float16 20 to 24 us
// (41 and 5 MB, of which 8 us the order).  A decoder input of a glanced graph holds one token in most places, so runs are cut evenly by
// position, not by token.
struct Plan {
    int64_t N;       // positions
    int piece;       // positions of the order that one wave sums
    int64_t pieces;  // ceil(N / piece)
};
inline Plan plan_of(int64_t N, int64_t D) {
    // enough waves for the chip while pieces stay long enough that the cut runs' sums are few
    const int64_t waves = N * ((D + 511) / 512) / 2048;
    int piece = 16;
    while (piece < 64 && piece * 2 <= waves) piece *= 2;
    return Plan{N, piece, (N + piece - 1) / piece};
}
// workspace: number of positions in the order (16 bytes), positions [N], tokens [N] in the order, occurrences and begin of
// each token [V], [V], sums of cut runs [pieces][2][D] float32; for many positions also tokens, positions and bounds of the
// tiles spread over the owners
inline bool spread_pays(int64_t N, int64_t V);
inline size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }
inline size_t order_bytes(const Plan &p) { return align16((size_t)p.N * 4); }

constexpr int SORT_NT = 1024, SORT_NW = SORT_NT / 64;
constexpr int MAX_OWN = 1024;   // tokens of the vocabulary that one workgroup owns, at the most
constexpr int SORT_LIST = 256;  // tokens of its own that a wave remembers from the first look to the second
constexpr int SORT_U = 4;       // groups of 64 positions whose reads are on their way together

// Workgroup b of 2^block_bits owns the tokens b, b + 2^block_bits, ... of the vocabulary - spread, because vocabularies are
// sorted by frequency: in strips the first workgroup would place half of all tokens - and looks for them among all
// positions, each wave in its sixteenth: first how often each occurs (and how many belong to the workgroups before this
// one, which is where its part of the order begins: no workgroup waits for another), then each to its place, in ascending
// position.  What bounds it is the look at every position, a dozen instructions for 64 (8 us for 5120 positions of 40000
// tokens, 11 us for 16384 of 64000, 77 us for 131072 of 300000); the second look goes over the few
// that the first has listed, or, where a wave has met more than its list holds (a common token), over all again.
// The lanes that hold the same token are found by one ballot for each bit of the token; the last of them moves the token's
// cursor on for all, so 64 positions cost the same whether they hold one token or 64.
template <int NT, int LIST>
struct OrderShared {
    unsigned list[NT / 64][LIST];
    int below[NT / 64], wave[NT / 64];
};
// All positions, each wave its share: from * 64 up to to * 64.  The next round's reads are ahead of what f stores, so that a
// wait for them (the hardware counts both in order) is none for the stores.  Masks of lanes are scalar: a group of 64 is a
// handful of vector instructions where it holds none of the own tokens.
template <int NT>
struct LookAtAll {
    const uint64_t *words;
    int64_t padding_idx, V;
    int N, from, to, lane;
    __device__ __forceinline__ LookAtAll(const int64_t *tokens, int64_t padding, int n, int64_t v)
        : words(reinterpret_cast<const uint64_t *>(tokens)), padding_idx(padding), V(v), N(n), lane((int)threadIdx.x & 63) {
        const int groups = (int)(((int64_t)N + 63) / 64), each = (groups + NT / 64 - 1) / (NT / 64);
        from = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) * each;
        to = from + each < groups ? from + each : groups;
    }
    template <typename F>
    __device__ __forceinline__ void operator()(F f) const {
        if (from >= to) return;
        uint64_t w[SORT_U], next[SORT_U];
        const auto load = [&](uint64_t (&to_w)[SORT_U], int g) {
            if (((int64_t)g + SORT_U) * 64 <= N) {
                const uint64_t *at = words + (int64_t)g * 64;
#pragma unroll
                for (int u = 0; u < SORT_U; u++) to_w[u] = at[u * 64 + lane];
            } else {  // (the last position again behind the end)
#pragma unroll
                for (int u = 0; u < SORT_U; u++) {
                    const int64_t at = ((int64_t)g + u) * 64 + lane;
                    to_w[u] = words[at < N ? at : N - 1];
                }
            }
        };
        load(w, from);
        for (int g = from; g < to; g += SORT_U) {
            load(next, g + SORT_U);
            if (g + SORT_U <= to && ((int64_t)g + SORT_U) * 64 <= N) {
#pragma unroll
                for (int u = 0; u < SORT_U; u++)
                    f(w[u], __ballot(w[u] < (uint64_t)V) & __ballot(w[u] != (uint64_t)padding_idx), (g + u - from) * 64 + lane);
            } else {
#pragma unroll
                for (int u = 0; u < SORT_U; u++) {
                    const int64_t left = g + u < to ? N - ((int64_t)g + u) * 64 : 0;
                    const unsigned long long there = left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
                    f(w[u], there & __ballot(w[u] < (uint64_t)V) & __ballot(w[u] != (uint64_t)padding_idx), (g + u - from) * 64 + lane);
                }
            }
#pragma unroll
            for (int u = 0; u < SORT_U; u++) w[u] = next[u];
        }
    }
};

// The work of one such workgroup of NT threads: its tokens are `block`, block + 2^block_bits, ..., `ids` <= NT of them.  s_at:
// [NT / 64][ids] in LDS.  count(id, begin, n, before) is called by thread id, emit(place, position from the wave's first, id) for each of the own
// tokens; begin and place count from this workgroup's first, `before` are the tokens of the workgroups before it.
// `look(f)` calls f(token, the lanes that hold a real one, the lanes' positions counted from the wave's first) for all that
// the wave has to look at, in ascending position.
template <int NT, int LIST, typename Look, typename Count, typename Emit>
__device__ __forceinline__ void order_own(int block, int block_bits, int own_bits, int ids, int *s_at, OrderShared<NT, LIST> &sh, Look look, Count count,
                                          Emit emit) {
    constexpr int NW = NT / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int block_mask = (1 << block_bits) - 1;
    int *at_wave = s_at + wave * ids;
    for (int i = lane; i < ids; i += 64) at_wave[i] = 0;
    // appends the own tokens of a group to the wave's list (a ring)
    const auto append = [&](uint64_t w, unsigned long long own, int pos, int &listed) {
        if ((own >> lane) & 1)
            sh.list[wave][(listed + __popcll(own & ((1ull << lane) - 1))) & (LIST - 1)] =
                (unsigned)(w >> block_bits) << 22 | (unsigned)pos;
        listed += __popcll(own);
    };
    int below = 0, listed = 0;
    look([&](uint64_t w, unsigned long long is, int pos) {
        const int owner = (int)w & block_mask;
        below += __popcll(is & __ballot(owner < block));
        const unsigned long long own = is & __ballot(owner == block);
        if (own == 0) return;
        const int id = (int)(w >> block_bits), leader = __builtin_ctzll(own);
        if (own & __ballot(id != __builtin_amdgcn_readlane(id, leader))) {
            if ((own >> lane) & 1) atomicAdd(&at_wave[id], 1);
        } else if (lane == leader) {  // one token alone is common: a run's; LDS takes additions to one place one after the other
            atomicAdd(&at_wave[id], __popcll(own));
        }
        append(w, own, pos, listed);
    });
    if (lane == 0) sh.below[wave] = below;
    __syncthreads();
    // exclusive sums over (token, wave)
    int mine = 0;
    if (tid < ids) {
#pragma unroll
        for (int w = 0; w < NW; w++) mine += s_at[w * ids + tid];
    }
    int upto = mine;
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(upto, d);
        if (lane >= d) upto += v;
    }
    if (lane == 63) sh.wave[wave] = upto;
    __syncthreads();
    int base = upto - mine, all_before = 0, all_own = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
        all_before += sh.below[w];
        if (w < wave) base += sh.wave[w];
        all_own += sh.wave[w];
    }
    if (tid < ids) {
        int at = base;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const int n = s_at[w * ids + tid];
            s_at[w * ids + tid] = at;
            at += n;
        }
    }
    count(tid < ids ? tid : -1, base, mine, all_before, all_own);
    __syncthreads();
    // `n` listed tokens, from the first-th on, to their places
    const auto place = [&](int first, int n) {
        const bool own = lane < n;
        const unsigned e = sh.list[wave][(first + (own ? lane : 0)) & (LIST - 1)];
        const int id = (int)(e >> 22);
        unsigned long long same = __ballot(own);
        if (same & __ballot(id != __builtin_amdgcn_readfirstlane(id)))
            for (int bit = 0; bit < own_bits; bit++) {
                const bool one = (id >> bit) & 1;
                const unsigned long long set = __ballot(one);
                same &= one ? set : ~set;
            }
        if (own) {
            // (the cursor of this wave alone; read by all lanes of the token before the last of them writes it)
            const int at = __hip_atomic_load(&at_wave[id], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            const int rank = __popcll(same & ((1ull << lane) - 1)), all = __popcll(same);
            if (rank == all - 1) __hip_atomic_store(&at_wave[id], at + all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            emit(at + rank, (int)(e & 0x3FFFFF), id);
        }
        __builtin_amdgcn_wave_barrier();
    };
    int placed = 0;
    if (listed > LIST) {  // the list was overwritten: once more, placing 64 whenever there are
        listed = 0;
        look([&](uint64_t w, unsigned long long is, int pos) {
            const unsigned long long own = is & __ballot(((int)w & block_mask) == block);
            if (own == 0) return;
            append(w, own, pos, listed);
            if (listed - placed >= 64) {
                __builtin_amdgcn_wave_barrier();
                place(placed, 64);
                placed += 64;
            }
        });
    }
    __builtin_amdgcn_wave_barrier();
    for (; placed < listed; placed += 64) place(placed, listed - placed < 64 ? listed - placed : 64);
}

__global__ __launch_bounds__(SORT_NT) void embedding_order_kernel(const int64_t *__restrict__ tokens, int64_t padding_idx, int N, int64_t V,
                                                                  int block_bits, int own_bits, int *__restrict__ count,
                                                                  int *__restrict__ counts, int *__restrict__ starts,
                                                                  int *__restrict__ order_pos, int *__restrict__ order_tok) {
    extern __shared__ int s_at[];  // [SORT_NW][ids]: occurrences, then cursors
    __shared__ OrderShared<SORT_NT, SORT_LIST> sh;
    const int block = (int)blockIdx.x, block_mask = (1 << block_bits) - 1;
    const int ids = (int)((V - block + block_mask) >> block_bits);
    const LookAtAll<SORT_NT> look(tokens, padding_idx, N, V);
    int first = 0;
    order_own<SORT_NT, SORT_LIST>(
        block, block_bits, own_bits, ids, s_at, sh, look,
        [&](int id, int begin, int n, int before, int own) {
            first = before;
            if (id >= 0) {
                counts[((int64_t)id << block_bits) + block] = n;
                starts[((int64_t)id << block_bits) + block] = before + begin;
            }
            if (block == block_mask && threadIdx.x == 0) *count = before + own;
        },
        [&](int place, int pos, int id) {
            order_pos[first + place] = look.from * 64 + pos;
            order_tok[first + place] = (id << block_bits) + block;
        });
}

// Many positions: every workgroup looking at all of them is too much (131072 positions of 128000 x 1024, all launches: 187 us,
// spread 148 us; of 40000 x 64 94 and 56 us; 32768 of 64000 take as long either way, 14 and 6.2 + 8.8 us), so they are first
// spread over the owners.  A tile of SPREAD positions is brought into the order (owner, position) by a workgroup: places
// among the tokens of one owner by ballots within the wave, by counts over waves and owners in LDS.  Leaves the tile's tokens
// and positions in that order and where each owner's begin (one more for the end) ...
constexpr int SPREAD_NT = 512, SPREAD_Q = 4, SPREAD = SPREAD_NT * SPREAD_Q, OWNERS = 256;
// The owners are OWNERS at most, each of MAX_OWN tokens: larger vocabularies keep the look at all positions, by more workgroups
// still, which is a step in time from one row to the next (131072 positions of 262144 and of 262145 rows: 6.5 + 22 us and 77 us
// for the order, 65 and 114 us a training pass at 16 columns; a million positions 249 and 682 us a pass).
constexpr int SPREAD_FROM = 16384;  // positions
__global__ __launch_bounds__(SPREAD_NT) void embedding_spread_kernel(const int64_t *__restrict__ tokens, int64_t padding_idx, int N, int64_t V,
                                                                     int *__restrict__ spread_tok, int *__restrict__ spread_pos,
                                                                     int *__restrict__ bounds) {
    constexpr int NW = SPREAD_NT / 64;
    __shared__ int s_at[NW][OWNERS];
    __shared__ int s_wave[OWNERS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = lane; i < OWNERS; i += 64) s_at[wave][i] = 0;
    const int64_t tile = blockIdx.x, at0 = tile * SPREAD + wave * (64 * SPREAD_Q) + lane;
    uint64_t w[SPREAD_Q];
#pragma unroll
    for (int q = 0; q < SPREAD_Q; q++) w[q] = reinterpret_cast<const uint64_t *>(tokens)[at0 + q * 64 < N ? at0 + q * 64 : N - 1];
    int place[SPREAD_Q];
#pragma unroll
    for (int q = 0; q < SPREAD_Q; q++) {
        const bool real = at0 + q * 64 < N && w[q] < (uint64_t)V && w[q] != (uint64_t)padding_idx;
        const int owner = (int)w[q] & (OWNERS - 1);
        unsigned long long same = __ballot(real);
#pragma unroll
        for (int bit = 0; bit < 8; bit++) {
            const bool one = (owner >> bit) & 1;
            const unsigned long long set = __ballot(one);
            same &= one ? set : ~set;
        }
        place[q] = -1;
        if (real) {
            // (this wave's counts alone; read by all lanes of the owner before the last of them writes)
            const int at = __hip_atomic_load(&s_at[wave][owner], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            const int rank = __popcll(same & ((1ull << lane) - 1)), all = __popcll(same);
            if (rank == all - 1) __hip_atomic_store(&s_at[wave][owner], at + all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            place[q] = at + rank;
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    int mine = 0, upto = 0;
    if (tid < OWNERS) {
#pragma unroll
        for (int k = 0; k < NW; k++) {
            const int c = s_at[k][tid];
            s_at[k][tid] = mine;
            mine += c;
        }
        upto = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(upto, d);
            if (lane >= d) upto += v;
        }
        if (lane == 63) s_wave[wave] = upto;
    }
    __syncthreads();
    if (tid < OWNERS) {
        int base = upto - mine;
        for (int k = 0; k < wave; k++) base += s_wave[k];
#pragma unroll
        for (int k = 0; k < NW; k++) s_at[k][tid] += base;
        int *out = bounds + tile * (OWNERS + 1);
        out[tid] = base;
        if (tid == OWNERS - 1) out[OWNERS] = base + mine;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < SPREAD_Q; q++)
        if (place[q] >= 0) {
            const int64_t to = tile * SPREAD + s_at[wave][(int)w[q] & (OWNERS - 1)] + place[q];
            spread_tok[to] = (int)w[q];
            spread_pos[to] = (int)(at0 + q * 64);
        }
}

inline bool spread_pays(int64_t N, int64_t V) { return N > SPREAD_FROM && V >= OWNERS && V <= (int64_t)OWNERS * MAX_OWN; }
inline size_t spread_bytes(int64_t N, int64_t V) {
    if (!spread_pays(N, V)) return 0;
    const size_t tiles = (size_t)((N + SPREAD - 1) / SPREAD);
    return tiles * (2 * SPREAD + OWNERS + 1) * 4;
}

// ... and the owners order theirs, each wave a sixteenth of the tiles.  What bounds it is the owner of the commonest token, whose
// positions one CU brings in order, some 70 instructions for 64 of them: 8.8 us for 32768 positions, 20 us for 131072, of
// tokens whose frequency falls off with their rank, and 73 us where six tenths of those are one token.
__global__ __launch_bounds__(SORT_NT) void embedding_gather_kernel(const int *__restrict__ spread_tok, const int *__restrict__ spread_pos,
                                                                   const int *__restrict__ bounds, int tiles, int64_t V, int own_bits,
                                                                   int *__restrict__ count, int *__restrict__ counts, int *__restrict__ starts,
                                                                   int *__restrict__ order_pos, int *__restrict__ order_tok) {
    extern __shared__ int s_at[];  // [SORT_NW][ids]
    __shared__ OrderShared<SORT_NT, SORT_LIST> sh;
    __shared__ int s_before[SORT_NW];
    const int block = (int)blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ids = (int)((V - block + OWNERS - 1) / OWNERS);
    // tokens of the owners before this one: where its own begin, over all tiles
    int before = 0;
    for (int t = tid; t < tiles; t += SORT_NT) before += bounds[(int64_t)t * (OWNERS + 1) + block];
    for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o);
    if (lane == 0) s_before[wave] = before;
    const int each = (tiles + SORT_NW - 1) / SORT_NW, t0 = wave * each, t1 = t0 + each < tiles ? t0 + each : tiles;
    constexpr int U = 4;
    const auto look = [&](auto f) {
        for (int first = t0; first < t1; first += 64) {  // the bounds of 64 tiles at a time
            const int64_t at = (int64_t)(first + lane < t1 ? first + lane : t1 - 1) * (OWNERS + 1) + block;
            const int begins = bounds[at], ends = bounds[at + 1];
            for (int t = first; t < first + 64 && t < t1; t++) {
                const int begin = __builtin_amdgcn_readlane(begins, t - first), end = __builtin_amdgcn_readlane(ends, t - first);
                for (int j = begin; j < end; j += 64 * U) {  // (a common token's owner: as many reads on their way together)
                    int tok[U], pos[U];
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const int64_t e = (int64_t)t * SPREAD + (j + u * 64 + lane < end ? j + u * 64 + lane : end - 1);
                        tok[u] = spread_tok[e];
                        pos[u] = spread_pos[e];
                    }
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const int left = end - j - u * 64;
                        if (left > 0) f((uint64_t)(unsigned)tok[u], left >= 64 ? ~0ull : (1ull << left) - 1, pos[u] - t0 * SPREAD);
                    }
                }
            }
        }
    };
    int first = 0;
    order_own<SORT_NT, SORT_LIST>(
        block, 8, own_bits, ids, s_at, sh, look,
        [&](int id, int begin, int n, int, int own) {
            for (int w = 0; w < SORT_NW; w++) first += s_before[w];
            if (id >= 0) {
                counts[(int64_t)id * OWNERS + block] = n;
                starts[(int64_t)id * OWNERS + block] = first + begin;
            }
            if (block == OWNERS - 1 && tid == 0) *count = first + own;
        },
        [&](int place, int pos, int id) {
            order_pos[first + place] = t0 * SPREAD + pos;
            order_tok[first + place] = id * OWNERS + block;
        });
}

// Few positions: order and sums in one launch.  A workgroup owns up to 256 tokens of the vocabulary (as above) and 256 bytes
// of columns, orders the positions of its tokens in LDS and sums: sixteen lanes a token, its rows in ascending position; a
// token met more than HEAVY times by all the groups of sixteen, each every 32nd occurrence, and their sums in order.  Rows of
// tokens that do not occur are zeroed.
//
// What bounds it: every workgroup looks at all positions, so positions times tiles of columns; and that it writes the rows in
// strips, so their bytes.  In one launch and in three (replayed from a graph), of float16, a fifth of the tokens the same one:
//    100 of  40000 x  512   13.6   17.4 us        3000 of 40000 x  512   19.6   19.3 us       8192 of  1000 x   64   14.3   17.4 us
//   1000 of  40000 x 1024   22.7   24.4 us        4096 of 40000 x  512   22.0   20.1 us       8192 of 40000 x  512   30.6   22.5 us
// At the limit of the looks, 18432, one launch takes up to 3.3 us more of the GPU and 6 to 7 us less of the host, whose 40 us a
// small training step waits for (41 and 47 us a pass on either side of the limit):
//   4600 of  40000 x  512   23.9   20.6 us        2300 of 40000 x 1024   28.0   25.0 us       6100 of 10007 x  384   19.3   18.8 us
//   4700 of  40000 x  512   24.5   20.0 us        2400 of 40000 x 1024   28.4   25.4 us       6200 of 10007 x  384   20.7   18.9 us
// The limit of the bytes, 2^27: below it one launch gains in all of these, above it some lose and others still gain.
//    100 of 130000 x  512   23.7   33.0 us         100 of 132000 x 512   28.4   33.8 us        100 of 200000 x 512    37     49.4 us
//   3000 of 130000 x  512   32.0   36.1 us        3000 of 132000 x 512   39.2   36.7 us
//    100 of 100000 x  333 float32  28.1  36.6 us   100 of 101000 x 333 float32  28.5  37.2 us   100 of 200000 x 333 float32  102  69 us
// (Strips of 128 bytes by 256 threads: 23 and 42 us where this has 20 and 31; sixteen rows of a heavy token on their way
// instead of eight: 32 instead of 27 us for 100 of 65000 x 1024, for want of registers; two launches, the sums behind
// embedding_order_kernel: 40 us for 5120 of 40000 x 512.)
constexpr int DIRECT_NT = 512, DIRECT_LANES = 16, DIRECT_GROUPS = DIRECT_NT / DIRECT_LANES;
constexpr int DIRECT_TOKENS = 8192, HEAVY = 32, DIRECT_OWN = 256;
constexpr int DIRECT_LIST = DIRECT_TOKENS / (DIRECT_NT / 64);  // all that a wave looks at: no second look (common tokens: 34 -> 28 us)
constexpr int64_t DIRECT_LOOKS = 18432, DIRECT_TILES = 8, DIRECT_VOCAB = 1 << 18, DIRECT_BYTES = 1 << 27;
inline int64_t direct_tiles(int es, int64_t D) { return (D * es + 16 * DIRECT_LANES - 1) / (16 * DIRECT_LANES); }
inline bool direct_pays(int es, int64_t N, int64_t V, int64_t D) {
    return D * es >= 16 && N <= DIRECT_TOKENS && V <= DIRECT_VOCAB && V * D * es <= DIRECT_BYTES && direct_tiles(es, D) <= DIRECT_TILES &&
           N * direct_tiles(es, D) <= DIRECT_LOOKS;
}
template <typename T>
__global__ __launch_bounds__(DIRECT_NT) void embedding_direct_kernel(const T *__restrict__ g, int64_t gstride, const int64_t *__restrict__ tokens,
                                                                     float scale, int64_t padding_idx, T *__restrict__ dweight, int N, int64_t V,
                                                                     int64_t D, int block_bits, int own_bits) {
    constexpr int E = VocabElem<T>::N;
    struct Sort {
        OrderShared<DIRECT_NT, DIRECT_LIST> order;
        int at[DIRECT_NT / 64 * DIRECT_OWN];
    };
    __shared__ union {
        Sort sort;
        float sum[DIRECT_GROUPS][DIRECT_LANES * E];
    } sh;
    __shared__ int s_begin[DIRECT_OWN], s_count[DIRECT_OWN], s_heavy[DIRECT_TOKENS / HEAVY], s_heavies;
    extern __shared__ unsigned short s_pos[];  // [N]
    const int tid = threadIdx.x, lane = tid % DIRECT_LANES, group = tid / DIRECT_LANES;
    const int block = (int)blockIdx.x, block_mask = (1 << block_bits) - 1;
    const int ids = (int)((V - block + block_mask) >> block_bits);
    if (tid == 0) s_heavies = 0;
    __syncthreads();
    const LookAtAll<DIRECT_NT> look(tokens, padding_idx, N, V);
    order_own<DIRECT_NT, DIRECT_LIST>(
        block, block_bits, own_bits, ids, sh.sort.at, sh.sort.order, look,
        [&](int id, int begin, int n, int, int) {
            if (id < 0) return;
            s_begin[id] = begin;
            s_count[id] = n;
            if (n > HEAVY) s_heavy[atomicAdd(&s_heavies, 1)] = id;
        },
        [&](int place, int pos, int) { s_pos[place] = (unsigned short)(look.from * 64 + pos); });
    __syncthreads();
    // (the last columns of D no multiple of a chunk: the row's last whole chunk, whose first columns a neighbour writes too)
    const int64_t c0 = ((int64_t)blockIdx.y * DIRECT_LANES + lane) * E, c = c0 + E <= D ? c0 : D - E;
    const bool live = c0 < D;
    const auto row = [&](int j) { return *reinterpret_cast<const vec16_any *>(g + (int64_t)s_pos[j] * gstride + c); };
    const auto add = [&](float (&acc)[E], const vec16 &v) {
        float o[E];
        VocabElem<T>::unpack(v, o);
#pragma unroll
        for (int k = 0; k < E; k++) acc[k] += o[k];
    };
    for (int i = group; i < ids; i += DIRECT_GROUPS) {
        const int b = s_begin[i], n = s_count[i];
        if (n > HEAVY) continue;
        float acc[E];
#pragma unroll
        for (int k = 0; k < E; k++) acc[k] = 0.f;
        constexpr int U = 4;
        for (int j = 0; j < n; j += U) {
            vec16 buf[U];
#pragma unroll
            for (int u = 0; u < U; u++) buf[u] = row(b + (j + u < n ? j + u : n - 1));
#pragma unroll
            for (int u = 0; u < U; u++)
                if (j + u < n) add(acc, buf[u]);
        }
#pragma unroll
        for (int k = 0; k < E; k++) acc[k] *= scale;
        if (live) *reinterpret_cast<vec16_any *>(dweight + (((int64_t)i << block_bits) + block) * D + c) = VocabElem<T>::pack(acc);
    }
    const int heavies = s_heavies;
    for (int h = 0; h < heavies; h++) {
        const int i = s_heavy[h], b = s_begin[i], n = s_count[i];
        float acc[E];
#pragma unroll
        for (int k = 0; k < E; k++) acc[k] = 0.f;
        constexpr int U = 8;
        for (int j = group; j < n; j += U * DIRECT_GROUPS) {
            vec16 buf[U];
#pragma unroll
            for (int u = 0; u < U; u++) buf[u] = row(b + (j + u * DIRECT_GROUPS < n ? j + u * DIRECT_GROUPS : n - 1));
#pragma unroll
            for (int u = 0; u < U; u++)
                if (j + u * DIRECT_GROUPS < n) add(acc, buf[u]);
        }
        __syncthreads();  // (the last heavy token's sums, or the order's lists, are done with)
#pragma unroll
        for (int k = 0; k < E; k++) sh.sum[group][lane * E + k] = acc[k];
        __syncthreads();
        if (tid < DIRECT_LANES * E) {
            float all = 0.f;
#pragma unroll
            for (int w = 0; w < DIRECT_GROUPS; w++) all += sh.sum[w][tid];
            const int64_t from = ((int64_t)blockIdx.y * DIRECT_LANES + tid / E) * E;
            if (from < D) dweight[(((int64_t)i << block_bits) + block) * D + (from + E <= D ? from : D - E) + tid % E] = (T)(all * scale);
        }
    }
}

// A wave sums one piece of the order over a tile of 64 chunks of columns, 8 rows of g on their way at a time.  Runs that begin
// and end inside the piece are finished; the sums of the first and the last, where they go on outside, are left for the join.
// The waves behind the last piece zero the rows that no token selects, beside the others' reads, neighbouring rows as one run in
// aligned chunks (row by row: 100 positions of 200000 x 333 float32 81 us instead of 69, of 200000 x 64 float16 23 instead of 20).
// What bounds it is memory: 32768
// positions of 64000 x 2048 bfloat16, 134 MB read and 262 MB written, all launches 81 us, of which 14 the order and 7 the joins; with finished
// rows that stay in the caches, too, 94 us (rows of zeros that stay there: 107 us; g read past them: 101 us).
constexpr int SUM_U = 8;
inline int zero_rows_of(int64_t row_bytes) {  // rows that one of them looks at
    int rows = 8;
    while (rows < 64 && rows * row_bytes < 8192) rows *= 2;
    return rows;
}
template <typename T, bool NARROW>
__global__ __launch_bounds__(256) void embedding_sum_kernel(const T *__restrict__ g, int64_t gstride, float scale, T *__restrict__ dweight,
                                                            int64_t D, int tiles, int piece, int64_t pieces, int64_t V, int zero_rows, const int *__restrict__ count,
                                                            const int *__restrict__ counts, const int *__restrict__ order_pos,
                                                            const int *__restrict__ order_tok, float *__restrict__ cut) {
    constexpr int E = VocabElem<T>::N;
    const int64_t task = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int64_t p = task / tiles;
    if (p >= pieces) {
        const vec16 zero = {0u, 0u, 0u, 0u};
        const int64_t v0 = (task - pieces * tiles) * zero_rows;
        unsigned long long rows = __ballot(lane < zero_rows && v0 + lane < V && counts[v0 + lane < V ? v0 + lane : 0] == 0);
        while (rows) {  // runs of neighbouring rows
            const int at = __builtin_ctzll(rows), n = ~(rows >> at) ? __builtin_ctzll(~(rows >> at)) : 64;
            T *row = dweight + (v0 + at) * D;
            const Span<T> sp(row, (int)(n * D));
            const int e = sp.edge(lane);
            if (e >= 0) row[e] = (T)0.f;
            vec16 *to = reinterpret_cast<vec16 *>(row + sp.head);
            for (int c = lane; c < sp.nvec; c += 64) __builtin_nontemporal_store(zero, to + c);
            rows = n == 64 ? 0 : rows & ~(((1ull << n) - 1) << at);
        }
        return;
    }
    const int total = *count;
    const int64_t from = p * piece;
    if (from >= total) return;
    const int n = total - from < piece ? (int)(total - from) : piece;
    const int my_pos = order_pos[from + (lane < n ? lane : 0)], my_tok = order_tok[from + (lane < n ? lane : 0)];
    const int before = order_tok[from > 0 ? from - 1 : 0], after = order_tok[from + n < total ? from + n : from];
    // Columns of a lane: the last ones of a row of D no multiple of a chunk are taken as the row's last whole chunk, whose first
    // columns a neighbour sums and writes too, to the same values; narrower rows than a chunk go element by element.
    const int64_t c0 = ((task - p * tiles) * 64 + lane) * E;
    const bool live = c0 < D;
    const int64_t c = NARROW ? 0 : c0 + E <= D ? c0 : D - E;
    float acc[E];
#pragma unroll
    for (int k = 0; k < E; k++) acc[k] = 0.f;
    bool opened_before = from > 0 && before == __builtin_amdgcn_readlane(my_tok, 0);
    for (int j0 = 0; j0 < n; j0 += SUM_U) {
        vec16 buf[SUM_U];
#pragma unroll
        for (int u = 0; u < SUM_U; u++) {  // (no branch around a load: the last row again behind the end)
            const T *row = g + (int64_t)__builtin_amdgcn_readlane(my_pos, j0 + u < n ? j0 + u : n - 1) * gstride;
            if (!NARROW) buf[u] = *reinterpret_cast<const vec16_any *>(row + c);
            else buf[u] = load_columns(row, 0, D);
        }
#pragma unroll
        for (int u = 0; u < SUM_U; u++) {
            const int j = j0 + u;
            if (j < n) {
                float o[E];
                VocabElem<T>::unpack(buf[u], o);
#pragma unroll
                for (int k = 0; k < E; k++) acc[k] += o[k];
                const int tok = __builtin_amdgcn_readlane(my_tok, j);
                const bool last = j + 1 == n;
                const bool goes_on = last ? from + n < total && after == tok : __builtin_amdgcn_readlane(my_tok, j + 1) == tok;
                if (last || !goes_on) {
                    if (live) {
                        if (opened_before || goes_on) {  // slot 0: a run from before (whether or not it ends here), slot 1: one that begins here
                            float *to = cut + (p * 2 + (opened_before ? 0 : 1)) * D + c;
#pragma unroll
                            for (int k = 0; k < E; k++)
                                if (!NARROW || k < D) to[k] = acc[k];
                        } else {
                            float f[E];
#pragma unroll
                            for (int k = 0; k < E; k++) f[k] = acc[k] * scale;
                            if (NARROW) store_columns(dweight + (int64_t)tok * D, c, D, VocabElem<T>::pack(f));
                            else __builtin_nontemporal_store(VocabElem<T>::pack(f), reinterpret_cast<vec16_any *>(dweight + (int64_t)tok * D + c));
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
// takes a stretch of them, the stretches are added in order.  A workgroup covers 256 columns.  (5 to 8 us, of which most is the
// launch and one chain of reads: bounds, then the sums eight at a time.)
constexpr int JOIN_NW = 4;
typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));
template <typename T>
__global__ __launch_bounds__(JOIN_NW * 64) void embedding_join_kernel(float scale, T *__restrict__ dweight, int64_t D, int piece,
                                                                      const int *__restrict__ count, const int *__restrict__ counts,
                                                                      const int *__restrict__ starts, const int *__restrict__ order_tok,
                                                                      const float *__restrict__ cut) {
    __shared__ float4_any s_sum[JOIN_NW][64];
    const int64_t p = blockIdx.x, end = (p + 1) * piece;
    const int total = *count, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (end >= total) return;
    const int tok = order_tok[end], start = starts[tok], behind = start + counts[tok];
    if (start >= end || start < p * piece) return;  // it begins with the next piece, or began before this one
    const int64_t reach = (behind - 1) / piece - p;  // pieces behind p that hold a part of the run
    const int64_t each = (reach + JOIN_NW - 1) / JOIN_NW, a = p + 1 + wave * each, b = a + each < p + 1 + reach ? a + each : p + 1 + reach;
    for (int64_t c0 = (int64_t)blockIdx.y * 256; c0 < D; c0 += (int64_t)gridDim.y * 256) {
        // (the last columns of D no multiple of four: the row's last four, as in the sums)
        const bool live = c0 + lane * 4 < D;
        const int64_t c = D < 4 ? 0 : c0 + lane * 4 + 4 <= D ? c0 + lane * 4 : D - 4;
        float4_any acc = {0.f, 0.f, 0.f, 0.f};
        if (D >= 4) {
            if (wave == 0) acc = *reinterpret_cast<const float4_any *>(cut + (p * 2 + 1) * D + c);
#pragma unroll 8
            for (int64_t q = a; q < b; q++) acc += *reinterpret_cast<const float4_any *>(cut + q * 2 * D + c);
        } else {
            for (int k = 0; k < D; k++) {
                if (wave == 0) acc[k] = cut[(p * 2 + 1) * D + k];
                for (int64_t q = a; q < b; q++) acc[k] += cut[q * 2 * D + k];
            }
        }
        s_sum[wave][lane] = acc;
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int w = 1; w < JOIN_NW; w++) acc += s_sum[w][lane];
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (live && c + k < D) dweight[(int64_t)tok * D + c + k] = (T)(acc[k] * scale);
        }
        __syncthreads();
    }
}

constexpr int64_t MAX_BLOCKS = (1 << 24) - 1;  // of 256 threads: a dimension of a grid ends at 2^32 threads

template <typename T>
int forward(const void *weight, int64_t wstride, const int64_t *tokens, float scale, void *out, int64_t N, int64_t V, int64_t D,
            hipStream_t s) {
    const int64_t each = 256 * LOOKUP_U * VocabElem<T>::N, blocks = (N * D + each - 1) / each;
    PCFGNAT_REQUIRE(blocks <= MAX_BLOCKS, "token_embedding: the output is too large for one call");
    if (D < VocabElem<T>::N)
        hipLaunchKernelGGL((embedding_fwd_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, s, (const T *)weight, wstride, tokens, scale,
                           (T *)out, N, V, (unsigned)D);
    else
        hipLaunchKernelGGL((embedding_fwd_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, s, (const T *)weight, wstride, tokens, scale,
                           (T *)out, N, V, (unsigned)D);
    PCFGNAT_HIP_CHECK(hipGetLastError());
    return PCFGNAT_OK;
}
template <typename T>
int backward(const void *g, int64_t gstride, const int64_t *tokens, float scale, int64_t padding_idx, void *dweight, void *workspace,
             int64_t N, int64_t V, int64_t D, hipStream_t s) {
    const bool direct = direct_pays((int)sizeof(T), N, V, D);
    // 256 workgroups own the vocabulary, fewer a smaller one, more where they would own too much each
    int block_bits = 0, own_bits = 0;
    while (block_bits < 8 && ((int64_t)2 << block_bits) <= V) block_bits++;
    while (((V - 1) >> block_bits) + 1 > (direct ? DIRECT_OWN : MAX_OWN)) block_bits++;
    while (((int64_t)1 << own_bits) < ((V - 1) >> block_bits) + 1) own_bits++;
    if (direct) {
        hipLaunchKernelGGL(embedding_direct_kernel<T>, dim3(1u << block_bits, (unsigned)direct_tiles((int)sizeof(T), D)), dim3(DIRECT_NT),
                           (size_t)(N + 1) * 2, s, (const T *)g, gstride, tokens, scale, padding_idx, (T *)dweight, (int)N, V, D, block_bits,
                           own_bits);
        PCFGNAT_HIP_CHECK(hipGetLastError());
        return PCFGNAT_OK;
    }
    const Plan p = plan_of(N, D);
    const int tiles = (int)((D + 64 * VocabElem<T>::N - 1) / (64 * VocabElem<T>::N));
    const int zero_rows = zero_rows_of(D * (int64_t)sizeof(T));
    const int64_t sum_blocks = (p.pieces * tiles + (V + zero_rows - 1) / zero_rows + 3) / 4;
    PCFGNAT_REQUIRE(sum_blocks <= MAX_BLOCKS, "token_embedding_backward: the gradient is too large for one call");
    char *w = (char *)workspace;
    int *count = (int *)w, *order_pos = (int *)(w + 16), *order_tok = (int *)(w + 16 + order_bytes(p));
    int *counts = (int *)(w + 16 + 2 * order_bytes(p)), *starts = (int *)((char *)counts + align16((size_t)V * 4));
    float *cut = (float *)((char *)starts + align16((size_t)V * 4));
    const size_t lds = (size_t)SORT_NW * (((V - 1) >> block_bits) + 1) * 4;
    if (lds > 47 * 1024) {  // (with the static 16.6 KiB, what needs no leave)
        PCFGNAT_DYNAMIC_LDS(embedding_order_kernel, SORT_NW * MAX_OWN * 4);
        PCFGNAT_DYNAMIC_LDS(embedding_gather_kernel, SORT_NW * MAX_OWN * 4);
    }
    if (spread_pays(N, V)) {
        const int64_t tiles = (N + SPREAD - 1) / SPREAD;
        int *spread_tok = (int *)((char *)cut + align16((size_t)p.pieces * 2 * D * 4)), *spread_pos = spread_tok + tiles * SPREAD;
        int *bounds = spread_pos + tiles * SPREAD;
        hipLaunchKernelGGL(embedding_spread_kernel, dim3((unsigned)tiles), dim3(SPREAD_NT), 0, s, tokens, padding_idx, (int)N, V, spread_tok,
                           spread_pos, bounds);
        PCFGNAT_HIP_CHECK(hipGetLastError());
        hipLaunchKernelGGL(embedding_gather_kernel, dim3(OWNERS), dim3(SORT_NT), lds, s, spread_tok, spread_pos, bounds, (int)tiles, V, own_bits,
                           count, counts, starts, order_pos, order_tok);
    } else {
        hipLaunchKernelGGL(embedding_order_kernel, dim3(1u << block_bits), dim3(SORT_NT), lds, s, tokens, padding_idx, (int)N, V, block_bits,
                           own_bits, count, counts, starts, order_pos, order_tok);
    }
    PCFGNAT_HIP_CHECK(hipGetLastError());
    if (D < VocabElem<T>::N)
        hipLaunchKernelGGL((embedding_sum_kernel<T, true>), dim3((unsigned)sum_blocks), dim3(256), 0, s, (const T *)g, gstride, scale,
                           (T *)dweight, D, tiles, p.piece, p.pieces, V, zero_rows, count, counts, order_pos, order_tok, cut);
    else
        hipLaunchKernelGGL((embedding_sum_kernel<T, false>), dim3((unsigned)sum_blocks), dim3(256), 0, s, (const T *)g, gstride, scale,
                           (T *)dweight, D, tiles, p.piece, p.pieces, V, zero_rows, count, counts, order_pos, order_tok, cut);
    PCFGNAT_HIP_CHECK(hipGetLastError());
    if (p.pieces > 1) {
        const unsigned split = (unsigned)((D + 255) / 256 < 64 ? (D + 255) / 256 : 64);
        hipLaunchKernelGGL(embedding_join_kernel<T>, dim3((unsigned)p.pieces, split), dim3(JOIN_NW * 64), 0, s, scale, (T *)dweight, D, p.piece,
                           count, counts, starts, order_tok, cut);
        PCFGNAT_HIP_CHECK(hipGetLastError());
    }
    return PCFGNAT_OK;
}

constexpr int64_t MAX_TOKENS = (int64_t)SORT_NW << 22;  // (a list entry keeps 22 bits of a position in its wave's sixteenth)
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

extern "C" size_t pcfgnat_token_embedding_backward_workspace_bytes(int dtype, int64_t N, int64_t V, int64_t D) {
    if (!vocab_dtype_ok(dtype) || N < 0 || N > MAX_TOKENS || V < 1 || V > MAX_VOCAB || D < 1 || D > MAX_DIM) return 0;
    if (direct_pays(vocab_elem_bytes(dtype), N, V, D)) return 0;
    const Plan p = plan_of(N, D);
    return 16 + 2 * order_bytes(p) + 2 * align16((size_t)V * 4) + align16((size_t)p.pieces * 2 * D * 4) + align16(spread_bytes(N, V));
}

extern "C" int pcfgnat_token_embedding_backward(const void *grad_out, int dtype, int64_t grad_stride, const int64_t *tokens, float scale,
                                                int64_t padding_idx, void *grad_weight, void *workspace, int64_t N, int64_t V, int64_t D,
                                                void *stream) {
    PCFGNAT_REQUIRE(vocab_dtype_ok(dtype), "token_embedding_backward: the gradient must be float16, bfloat16 or float32");
    PCFGNAT_REQUIRE(N >= 0 && N <= MAX_TOKENS && V >= 1 && V <= MAX_VOCAB && D >= 1 && D <= MAX_DIM && grad_stride >= 0,
                    "token_embedding_backward: bad dimensions");
    PCFGNAT_REQUIRE(grad_weight && (N == 0 || (grad_out && tokens)) &&
                        (workspace || pcfgnat_token_embedding_backward_workspace_bytes(dtype, N, V, D) == 0),
                    "token_embedding_backward: null pointer");
    hipStream_t s = (hipStream_t)stream;
    if (dtype == PCFGNAT_F16) return backward<f16>(grad_out, grad_stride, tokens, scale, padding_idx, grad_weight, workspace, N, V, D, s);
    if (dtype == PCFGNAT_BF16) return backward<bf16>(grad_out, grad_stride, tokens, scale, padding_idx, grad_weight, workspace, N, V, D, s);
    return backward<float>(grad_out, grad_stride, tokens, scale, padding_idx, grad_weight, workspace, N, V, D, s);
}
