// The k best logits of every row, in order, with the probability mass outside them (elg_top_logits).
//
// Order: larger value first, equal values by the lower index; NaN above +inf.  One 64-bit composite (order_key(value), ~index) per element
// carries both, composites are unique, so "the k largest composites" has one answer whatever the order in which threads find them.
//
// Selection without sorting the row: T threads each know the largest key of their own elements; the k-th largest of these T <= maxima is a
// lower bound of the k-th largest element (k different elements reach it), and only a few more than k elements do.  These candidates are
// gathered into LDS (any order) and ranked by counting: rank = number of larger composites.  Rows that defeat the bound (thousands of equal
// values) fall back to a bisection over the keys of all elements, with equal values taken in index order.
#include "elg_logits.h"
#include <type_traits>

namespace elg {
namespace {

constexpr int WAVE_CAP = 256;             // candidates of a wave
constexpr int TOP_CAP = 1024;             // candidates kept in LDS; more of them: the bisection over the whole row

struct TopArgs {
    const char* z;
    long long stride_bytes;
    long long R;
    int V, k;
    float c2;                             // log2(e) / temperature
    char* values;
    int* idx;
    float* tail;
    unsigned k_inv;                       // ceil(2^32 / k); 0 for k = 1
};

__device__ __forceinline__ unsigned long long composite(unsigned key, int n) {
    return ((unsigned long long)key << 32) | (unsigned)~n;
}

template <int T>
struct Count {                            // block-wide counts; one barrier each, buffers alternate as in BlockRed
    int* buf;                             // 2 * T / 64 ints of LDS
    int flip = 0;
    __device__ explicit Count(int* b) : buf(b) {}
    __device__ __forceinline__ int sum_wave_uniform(int c) {
        int* s = buf + flip * (T / 64);
        flip ^= 1;
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = c;
        __syncthreads();
        int r = 0;
#pragma unroll
        for (int w = 0; w < T / 64; ++w) r += s[w];
        return r;
    }
    __device__ __forceinline__ int of(bool p) { return sum_wave_uniform(__popcll(__ballot(p))); }
    // total of a per-thread count, and the count of the threads in front of this one
    __device__ __forceinline__ int scan(int c, int& before) {
        int incl = c;
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d, 64);
            if (lane >= d) incl += o;
        }
        int* s = buf + flip * (T / 64);
        flip ^= 1;
        if (lane == 63) s[threadIdx.x >> 6] = incl;
        __syncthreads();
        int tot = 0, pre = 0;
#pragma unroll
        for (int w = 0; w < T / 64; ++w) {
            if (w < (int)(threadIdx.x >> 6)) pre += s[w];
            tot += s[w];
        }
        before = pre + incl - c;
        return tot;
    }
};

// A register of one f32 or two 16-bit elements <-> the order keys of the same width, in place: three operations for either.  These keys
// tell -0 from 0 and put NaN at both ends; the callers see to both.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
template <int DT> struct WordKey {                                    // two 16-bit keys
    static constexpr unsigned NEG_INF = DT == ELG_BF16 ? 0x007Fu : 0x03FFu, POS_INF = DT == ELG_BF16 ? 0xFF80u : 0xFC00u, ZERO = 0x8000u, TOP = 0xFFFFu;
    static __device__ __forceinline__ unsigned to(unsigned w) {
        const s16x2 sign = __builtin_bit_cast(s16x2, w) >> 15;
        return w ^ (__builtin_bit_cast(unsigned, sign) | 0x80008000u);
    }
    static __device__ __forceinline__ unsigned from(unsigned k) {
        const s16x2 sign = __builtin_bit_cast(s16x2, k) >> 15;
        return k ^ (~__builtin_bit_cast(unsigned, sign) | 0x80008000u);
    }
    static __device__ __forceinline__ unsigned hi(unsigned a, unsigned b) {
        return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
    }
    static __device__ __forceinline__ unsigned lo(unsigned a, unsigned b) {
        return __builtin_bit_cast(unsigned, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
    }
    static __device__ __forceinline__ unsigned highest(unsigned w) { return max(w >> 16, w & 0xFFFFu); }
    static __device__ __forceinline__ unsigned lowest(unsigned w) { return min(w >> 16, w & 0xFFFFu); }
    static __device__ __forceinline__ unsigned at(const u32x4& z, int e) { return (e & 1) ? z[e >> 1] >> 16 : z[e >> 1] & 0xFFFFu; }
};
template <> struct WordKey<ELG_F32> {
    static constexpr unsigned NEG_INF = KEY_NEG_INF, POS_INF = 0xFF800000u, ZERO = 0x80000000u, TOP = 0xFFFFFFFFu;
    static __device__ __forceinline__ unsigned to(unsigned w) { return w ^ ((unsigned)((int)w >> 31) | 0x80000000u); }
    static __device__ __forceinline__ unsigned from(unsigned k) { return k ^ (~(unsigned)((int)k >> 31) | 0x80000000u); }
    static __device__ __forceinline__ unsigned hi(unsigned a, unsigned b) { return max(a, b); }
    static __device__ __forceinline__ unsigned lo(unsigned a, unsigned b) { return min(a, b); }
    static __device__ __forceinline__ unsigned highest(unsigned w) { return w; }
    static __device__ __forceinline__ unsigned lowest(unsigned w) { return w; }
    static __device__ __forceinline__ unsigned at(const u32x4& z, int e) { return z[e]; }
};
// the key of one element given as a float
template <int DT>
__device__ __forceinline__ unsigned word_key(float f) {
    if constexpr (DT == ELG_F32) return WordKey<DT>::to((unsigned)f2i(f));
    else if constexpr (DT == ELG_BF16) return WordKey<DT>::to((unsigned)f2i(f) >> 16) & 0xFFFFu;
    else return WordKey<DT>::to((unsigned)__builtin_bit_cast(unsigned short, (_Float16)f)) & 0xFFFFu;
}

template <int T>
struct TopShared {
    unsigned long long found[T / 64][WAVE_CAP];       // as a wave finds them
    int n_found[T / 64];
    __attribute__((aligned(16))) unsigned long long cand[TOP_CAP + 8];       // all of them, in any order
    unsigned long long win[TOP_CAP];      // in order
    float fred[2 * 2 * (T / 64)];
    int cred[2 * (T / 64)];
    unsigned kred[2 * (T / 64)];
    int n_cand;
};

// `need` elements of order key `key`, lowest indices first, into win[at ...]: the row is read from its start as far as that takes
template <int DT, int T>
__device__ __forceinline__ void take_ties(const void* row, int V, unsigned key, int at, int need, unsigned long long* win, Count<T>& cnt) {
    const int tid = threadIdx.x, shift = shift_of<DT>(row), nch = (shift + V + VEC<DT> - 1) / VEC<DT>;
    for (int c0 = 0; need > 0 && c0 < nch; c0 += T) {
        const int c = c0 + tid;
        unsigned hit = 0;
        if (c < nch) {
            float v[VEC<DT>];
            unpack<DT>(load_chunk<DT>(row, shift, V, c, 0u), v);
#pragma unroll
            for (int e = 0; e < VEC<DT>; ++e) {
                const int n = c * VEC<DT> + e - shift;
                if (n >= 0 && n < V && order_key(v[e]) == key) hit |= 1u << e;
            }
        }
        int before;
        const int tot = cnt.scan(__popc(hit), before);
        for (; hit && before < need; ++before) {
            const int e = __ffs(hit) - 1;
            hit &= hit - 1;
            win[at + before] = composite(key, c * VEC<DT> + e - shift);
        }
        at += min(tot, need);
        need -= min(tot, need);
    }
}

// the candidates in order into win, the first k of it written out; what the others of them and the rest weigh
template <int DT, int T>
__device__ __forceinline__ void finish_row(const TopArgs& A, long long r, const void* row, int found, unsigned tie_key, int tie_need, float rest, bool rest_known,
                                           TopShared<T>& sh, Count<T>& cnt, BlockRed<T / 64>& red) {
    const int tid = threadIdx.x, k = A.k;
    // rank by counting; composites are unique, and none is 0
    if (tid < 8) sh.cand[found + tid] = 0ull;
    __syncthreads();
    for (int i = tid; i < found; i += T) {
        const unsigned long long me = sh.cand[i];
        int rank = 0;
        for (int j = 0; j < found; j += 8) {          // eight at a time: one LDS latency, not eight
            ulonglong2 o[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) o[u] = *reinterpret_cast<const ulonglong2*>(sh.cand + j + 2 * u);
#pragma unroll
            for (int u = 0; u < 4; ++u) rank += (o[u].x > me) + (o[u].y > me);
        }
        sh.win[rank] = me;
    }
    take_ties<DT, T>(row, A.V, tie_key, min(found, k), tie_need, sh.win, cnt);
    __syncthreads();
    for (int i = tid; i < k; i += T) {
        const unsigned long long w = sh.win[i];
        reinterpret_cast<elem_t<DT>*>(A.values)[r * k + i] = (elem_t<DT>)key_value((unsigned)(w >> 32));
        A.idx[r * k + i] = (int)~(unsigned)w;
    }
    if (A.tail) {
        // mass outside the winners: summed apart from the winners' own, so that a small tail keeps its digits
        const unsigned long long last = sh.win[k - 1];
        const float m = key_value((unsigned)(sh.win[0] >> 32));
        float top = 0.f;
        if (!(m > ELG_NEG_INF || m != m)) rest = 0.f;           // no open node: nothing to weigh
        else {
            for (int i = tid; i < k; i += T) top += ex2((key_value((unsigned)(sh.win[i] >> 32)) - m) * A.c2);
            if (rest_known) {
                for (int i = k + tid; i < found; i += T) rest += ex2((key_value((unsigned)(sh.win[i] >> 32)) - m) * A.c2);
            } else {
                const int shift = shift_of<DT>(row), nch = (shift + A.V + VEC<DT> - 1) / VEC<DT>;
                rest = 0.f;
                for (int c = tid; c < nch; c += T) {
                    float v[VEC<DT>];
                    unpack<DT>(load_chunk<DT>(row, shift, A.V, c, PAD_NEG_INF<DT>), v);
#pragma unroll
                    for (int e = 0; e < VEC<DT>; ++e)
                        if (composite(order_key(v[e]), c * VEC<DT> + e - shift) < last) rest += ex2((v[e] - m) * A.c2);
                }
            }
        }
        const float2 s = red.sum2(top, rest);
        if (tid == 0) A.tail[r] = s.x + s.y > 0.f || s.x != s.x || s.y != s.y ? s.y / (s.x + s.y) : 0.f;
    }
    __syncthreads();                      // win, cand and n_cand are written again by the next row
}

// A row by order keys of whole elements, read again by every pass: rows no workgroup can hold, rows with NaN, rows with so many equal values
// that the bound does not separate them.
template <int DT, int T>
__device__ __noinline__ void top_row_again(const TopArgs& A, long long r, TopShared<T>& sh) {
    __syncthreads();                      // the reductions' buffers start over
    BlockRed<T / 64> red(sh.fred);
    Count<T> cnt(sh.cred);
    const char* row = A.z + r * A.stride_bytes;
    const int tid = threadIdx.x, V = A.V, k = A.k, shift = shift_of<DT>(row), nch = (shift + V + VEC<DT> - 1) / VEC<DT>;
    // f(key, index) for every element of this thread; positions outside the row come as closed nodes
    auto each = [&](auto&& f) {
        for (int c = tid; c < nch; c += T) {
            float v[VEC<DT>];
            unpack<DT>(load_chunk<DT>(row, shift, V, c, PAD_NEG_INF<DT>), v);
#pragma unroll
            for (int e = 0; e < VEC<DT>; ++e) f(order_key(v[e]), c * VEC<DT> + e - shift);
        }
    };
    // ---- the threads' maxima over open nodes, and a bound from them
    unsigned kmax = 0;
    each([&](unsigned key, int) { if (key > KEY_NEG_INF) kmax = max(kmax, key); });
    if (tid == 0) sh.n_cand = 0;
    unsigned lo = KEY_NEG_INF + 1, hi = 0xFFFFFFFFu;
    if (cnt.of(kmax >= lo) >= k) {
        while (lo < hi) {
            const unsigned mid = lo + (hi - lo) / 2 + 1;
            const int c = cnt.of(kmax >= mid);
            if (c >= k) {
                lo = mid;
                if (c == k) break;
            } else hi = mid - 1;
        }
    }
    if (kmax >= lo)
        each([&](unsigned key, int n) {
            if (key >= lo) {
                const int p = atomicAdd(&sh.n_cand, 1);
                if (p < TOP_CAP) sh.cand[p] = composite(key, n);
            }
        });
    __syncthreads();
    int found = sh.n_cand, tie_need = 0;
    unsigned tie_key = 0;
    if (found > TOP_CAP) {
        // every wave has its count before n_cand starts over: where the bound is the NaN key already the search below takes no step, and none of
        // its barriers stands between
        __syncthreads();
        // the k-th largest key of all elements: count(>= lo) >= k holds throughout
        hi = 0xFFFFFFFFu;
        while (lo < hi) {
            const unsigned mid = lo + (hi - lo) / 2 + 1;
            int c = 0;
            each([&](unsigned key, int) { c += key >= mid; });
            int before;
            c = cnt.scan(c, before);
            if (c >= k) {
                lo = mid;
                if (c == k) break;
            } else hi = mid - 1;
        }
        if (tid == 0) sh.n_cand = 0;
        __syncthreads();
        each([&](unsigned key, int n) {
            if (key > lo) sh.cand[atomicAdd(&sh.n_cand, 1)] = composite(key, n);       // at most k of them
        });
        __syncthreads();
        found = sh.n_cand;
        tie_key = lo;
        tie_need = k - found;
    } else if (found < k) {
        tie_key = KEY_NEG_INF;                                                   // closed nodes fill the rest
        tie_need = k - found;
    }
    finish_row<DT, T>(A, r, row, found, tie_key, tie_need, 0.f, false, sh, cnt, red);
}

// One workgroup per row, the row in registers as order keys, C chunks a thread.  One pass for the threads' maxima, one that gathers the
// candidates and sums the exponentials of everything below the bound.
// 512 x 131072 bf16, the best 128: 83 us where its bytes take 28.  One workgroup takes all of a CU's registers, half of them for its row of 256 KB,
// so each CU works its two rows off one after the other, and between loading them stand the maxima (two 16-bit keys to an operation), the
// bound's bisection and the ranking, with nothing in flight behind them.  The candidates ranked eight at a time, 112 -> 90 us; keys formed in
// place of floats, 120 -> 112 us.
template <int DT, int T, int C>
__global__ __launch_bounds__(T, 4) void top_row_kernel(const TopArgs A) {
    using W = WordKey<DT>;
    __shared__ TopShared<T> sh;
    const int tid = threadIdx.x, k = A.k;
    BlockRed<T / 64> red(sh.fred);
    Count<T> cnt(sh.cred);
    for (long long r = blockIdx.x; r < A.R; r += gridDim.x) {
        const char* row = A.z + r * A.stride_bytes;
        const Span<DT> sp(row, A.V);
        auto place = [&]() { int t = tid; asm volatile("" : "+v"(t)); return t; };      // (see distill_row_kernel)
        u32x4 z[C];
        const int t0 = place();
#pragma unroll
        for (int c = 0; c < C; ++c) {
            constexpr unsigned pad = PAD_NEG_INF<DT>;
            z[c] = u32x4{pad, pad, pad, pad};
            if (t0 >= sp.c_lo - c * T && t0 < sp.c_hi - c * T) z[c] = sp.chunk(t0 + c * T);
        }
        const int edge = sp.edge(tid);
        const float ze = edge >= 0 ? elem<DT>(row, edge) : ELG_NEG_INF;
        // ---- keys, the threads' extremes
        unsigned mx = 0u, mn = 0xFFFFFFFFu;
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned w = W::to(z[c][i]);
                z[c][i] = w;
                mx = W::hi(mx, w);
                mn = W::lo(mn, w);
            }
            asm volatile("" : "+v"(z[c]), "+v"(mx), "+v"(mn));
        }
        unsigned kmax = W::highest(mx), kmin = W::lowest(mn);
        if (edge >= 0) {
            kmax = max(kmax, word_key<DT>(ze));
            kmin = min(kmin, word_key<DT>(ze));
        }
        unsigned best = kmax;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) best = max(best, (unsigned)__shfl_xor((int)best, d, 64));
        if ((tid & 63) == 0) sh.kred[tid >> 6] = best;
        const int strange = cnt.of(kmin < W::NEG_INF || kmax > W::POS_INF);          // NaN of either sign
#pragma unroll
        for (int w = 0; w < T / 64; ++w) best = max(best, sh.kred[w]);
        if (strange) {
            top_row_again<DT, T>(A, r, sh);
            continue;
        }
        // ---- the k-th largest of the threads' maxima, or a little less: a few candidates more cost less than the steps that would spare them
        unsigned lo = W::NEG_INF + 1, hi = best;
        if (cnt.of(kmax >= lo) >= k) {
            while (lo < hi) {
                const unsigned mid = lo + (hi - lo) / 2 + 1;
                const int c = cnt.of(kmax >= mid);
                if (c >= k) {
                    lo = mid;
                    if (c <= k + k / 8 + 4) break;
                } else hi = mid - 1;
            }
        }
        if (lo == W::ZERO) --lo;                                                     // -0 equals 0
        // ---- candidates, and the sum over everything below them
        float bits_best;
        {
            const unsigned w = W::from(best);
            if constexpr (DT == ELG_F32) bits_best = i2f((int)w);
            else if constexpr (DT == ELG_BF16) bits_best = i2f((int)(w << 16));
            else bits_best = (float)__builtin_bit_cast(_Float16, (unsigned short)w);
        }
        const float m = bits_best;
        float rest[2] = {0.f, 0.f};
        // (a wave keeps its own list: no atomics, no waiting)
        int n_mine = 0;
        auto push = [&](bool hit, float f, int n) {
            const unsigned long long mask = __ballot(hit);
            const int p = n_mine + lanes_below(mask);
            if (hit && p < WAVE_CAP) sh.found[tid >> 6][p] = composite(order_key(f), n);
            n_mine += __popcll(mask);
        };
        const int t1 = place();
#pragma unroll
        for (int c = 0; c < C; ++c) {
            asm volatile("" : "+v"(z[c]));
            const unsigned top = W::highest(W::hi(W::hi(z[c][0], z[c][1]), W::hi(z[c][2], z[c][3])));
            const bool some = __any(top >= lo);
            if (!A.tail && !some) continue;
            u32x4 raw;
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[i] = W::from(z[c][i]);
            float v[VEC<DT>];
            unpack<DT>(raw, v);
            if (some) {
                const int n0 = (t1 + c * T) * VEC<DT> - sp.shift;
#pragma unroll
                for (int e = 0; e < VEC<DT>; ++e) {
                    const bool hit = W::at(z[c], e) >= lo;
                    push(hit, v[e], n0 + e);
                    v[e] = hit ? ELG_NEG_INF : v[e];
                }
            }
            if (A.tail) {
#pragma unroll
                for (int e = 0; e < VEC<DT>; ++e) rest[e & 1] += ex2((v[e] - m) * A.c2);
            }
            asm volatile("" : "+v"(rest[0]), "+v"(rest[1]));
        }
        {
            const bool hit = edge >= 0 && word_key<DT>(ze) >= lo;
            push(hit, ze, edge);
            if (edge >= 0 && !hit) rest[0] += ex2((ze - m) * A.c2);
        }
        if ((tid & 63) == 0) sh.n_found[tid >> 6] = n_mine;
        __syncthreads();
        int found = 0, at = 0;
        bool over = false;
#pragma unroll
        for (int w = 0; w < T / 64; ++w) {
            const int n = sh.n_found[w];
            if (w < (tid >> 6)) at += n;
            found += n;
            over = over || n > WAVE_CAP;
        }
        if (found > TOP_CAP || over) {
            top_row_again<DT, T>(A, r, sh);
            continue;
        }
        for (int i = tid & 63; i < n_mine; i += 64) sh.cand[at + i] = sh.found[tid >> 6][i];
        finish_row<DT, T>(A, r, row, found, KEY_NEG_INF, found < k ? k - found : 0, rest[0] + rest[1], true, sh, cnt, red);
    }
}

// rows that no workgroup can hold: read twice or more, the keys formed anew each time
template <int DT, int T>
__global__ __launch_bounds__(T) void top_long_kernel(const TopArgs A) {
    __shared__ TopShared<T> sh;
    for (long long r = blockIdx.x; r < A.R; r += gridDim.x) top_row_again<DT, T>(A, r, sh);
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Short rows: a bitonic sort in registers, eight lanes to a row.  A lane holds NE positions of the order; merges across lanes go through
// DPP alone (pairs, quads and mirrored halves of eight lanes are what it can reach in one step), merges inside a lane are plain registers.
// The sort key is a whole composite in one comparable register: for 16-bit types a 32-bit integer (16 bits of value, 16 of index), for f32 a
// double in [1, 2) whose 52 mantissa bits hold 32 of value and 20 of index -- v_max_f64 / v_min_f64 then order both at once, in two
// instructions where a comparison with selects takes five.
template <int DT>
struct Key32 {
    unsigned u;
    static __device__ __forceinline__ Key32 make(float f, int n) {
        const unsigned b = DT == ELG_BF16 ? (unsigned)f2i(f) >> 16 : (unsigned)__builtin_bit_cast(unsigned short, (_Float16)f);
        unsigned key = (b & 0x8000u) ? ~b & 0xFFFFu : b | 0x8000u;
        key = b == 0x8000u ? 0x8000u : key;                                   // -0 = +0
        key = f != f ? 0xFFFFu : key;
        return {key << 16 | (0xFFFFu - (unsigned)n)};
    }
    __device__ __forceinline__ float value() const {
        const unsigned key = u >> 16, b = (key & 0x8000u) ? key & 0x7FFFu : ~key & 0xFFFFu;
        return DT == ELG_BF16 ? i2f((int)(b << 16)) : (float)__builtin_bit_cast(_Float16, (unsigned short)b);
    }
    __device__ __forceinline__ int index() const { return (int)(0xFFFFu - (u & 0xFFFFu)); }
    static __device__ __forceinline__ Key32 hi(Key32 a, Key32 b) { return {max(a.u, b.u)}; }
    static __device__ __forceinline__ Key32 lo(Key32 a, Key32 b) { return {min(a.u, b.u)}; }
    template <int CTRL> __device__ __forceinline__ Key32 moved() const { return {(unsigned)__builtin_amdgcn_mov_dpp((int)u, CTRL, 0xF, 0xF, true)}; }
    __device__ __forceinline__ void raise(Key32 o) { asm("v_max_u32 %0, %0, %1" : "+v"(u) : "v"(o.u)); }
    __device__ __forceinline__ void lower(Key32 o) { asm("v_min_u32 %0, %0, %1" : "+v"(u) : "v"(o.u)); }
};
struct Key64 {
    double d;
    static __device__ __forceinline__ Key64 of(unsigned long long mantissa) { return {__builtin_bit_cast(double, 0x3FF0000000000000ull | mantissa)}; }
    static __device__ __forceinline__ Key64 make(float f, int n) { return of(((unsigned long long)order_key(f) << 20) | (0xFFFFFu - (unsigned)n)); }
    __device__ __forceinline__ float value() const { return key_value((unsigned)(__builtin_bit_cast(unsigned long long, d) >> 20)); }
    __device__ __forceinline__ int index() const { return (int)(0xFFFFFu - ((unsigned)__builtin_bit_cast(unsigned long long, d) & 0xFFFFFu)); }
    // (asm: the library maximum first quiets operands that come out of integer registers -- these are never NaN)
    static __device__ __forceinline__ Key64 hi(Key64 a, Key64 b) { Key64 r; asm("v_max_f64 %0, %1, %2" : "=v"(r.d) : "v"(a.d), "v"(b.d)); return r; }
    static __device__ __forceinline__ Key64 lo(Key64 a, Key64 b) { Key64 r; asm("v_min_f64 %0, %1, %2" : "=v"(r.d) : "v"(a.d), "v"(b.d)); return r; }
    template <int CTRL> __device__ __forceinline__ Key64 moved() const {
        const unsigned long long u = __builtin_bit_cast(unsigned long long, d);
        const unsigned l = (unsigned)__builtin_amdgcn_mov_dpp((int)(unsigned)u, CTRL, 0xF, 0xF, true);
        const unsigned h = (unsigned)__builtin_amdgcn_mov_dpp((int)(unsigned)(u >> 32), CTRL, 0xF, 0xF, true);
        return {__builtin_bit_cast(double, (unsigned long long)h << 32 | l)};
    }
    static __device__ __forceinline__ Key64 pick(bool up, Key64 a, Key64 b) { return (a.d > b.d) == up ? a : b; }
    __device__ __forceinline__ void raise(Key64 o) { asm("v_max_f64 %0, %0, %1" : "+v"(d) : "v"(o.d)); }
    __device__ __forceinline__ void lower(Key64 o) { asm("v_min_f64 %0, %0, %1" : "+v"(d) : "v"(o.d)); }
};
template <int DT> struct KeyOf { using K = Key32<DT>; };
template <> struct KeyOf<ELG_F32> { using K = Key64; };

// an odd-even merge sort's compare-exchanges
template <int N> struct Network {
    int a[N * 8] = {}, b[N * 8] = {}, n = 0;
    constexpr Network() {
        for (int p = 1; p < N; p *= 2)
            for (int q = p; q >= 1; q /= 2)
                for (int j = q % p; j + q < N; j += 2 * q)
                    for (int i = 0; i < q && i + j + q < N; ++i)
                        if ((i + j) / (2 * p) == (i + j + q) / (2 * p)) { a[n] = i + j; b[n] = i + j + q; ++n; }
    }
};

template <class K, int NE>
__device__ __forceinline__ void exchange(K (&x)[NE], int i, int j) {
    const K a = x[i], b = x[j];
    x[i] = K::hi(a, b);
    x[j] = K::lo(a, b);
}
template <class K, int NE>
__device__ __forceinline__ void merge_lane(K (&x)[NE]) {
#pragma unroll
    for (int d = NE / 2; d >= 1; d /= 2)
#pragma unroll
        for (int s = 0; s < NE; ++s)
            if (!(s & d)) exchange(x, s, s + d);
}
// the lanes that keep the larger of their pairs, then the others: two moves and two ordered operations a value
template <class K, int NE>
__device__ __forceinline__ void keep(K (&x)[NE], const K (&y)[NE], bool up) {
    if (up) {
#pragma unroll
        for (int s = 0; s < NE; ++s) x[s].raise(y[s]);
    } else {
#pragma unroll
        for (int s = 0; s < NE; ++s) x[s].lower(y[s]);
    }
}
template <int CTRL, class K, int NE>
__device__ __forceinline__ void across_mirror(K (&x)[NE], bool up) {
    K y[NE];
#pragma unroll
    for (int s = 0; s < NE; ++s) y[s] = x[NE - 1 - s].template moved<CTRL>();
    keep(x, y, up);
}
template <int CTRL, class K, int NE>
__device__ __forceinline__ void across(K (&x)[NE], bool up) {
    K y[NE];
#pragma unroll
    for (int s = 0; s < NE; ++s) y[s] = x[s].template moved<CTRL>();
    keep(x, y, up);
}

constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_MIRROR4 = 0x1B, DPP_MIRROR8 = 0x141;

// 8 rows to a wave, 4 waves to a workgroup (2 where 4 would need over 64 KB of LDS); waves never wait for each other.  LDS turns the lanes'
// runs of the order into the rows' packed output.
// 896000 rows of 101 f32, the best 40 and the tail: 219 us where its bytes take 137 (3.0 TB/s; 280 us in the first dozen calls of a process); the
// sort's exchanges bound it, not memory.
template <int DT, int NE>
__global__ __launch_bounds__(256, NE == 32 ? 3 : 4) void top_sort_kernel(const TopArgs A) {
    using K = typename KeyOf<DT>::K;
    extern __shared__ __attribute__((aligned(16))) unsigned char top_lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, g = lane >> 3, l = lane & 7, V = A.V, k = A.k;
    const int lanes_out = (k + NE - 1) / NE;               // lanes of a row that hold winners; a lane's run is padded by one against bank conflicts
    K* out = reinterpret_cast<K*>(top_lds) + wave * 8 * lanes_out * (NE + 1);
    constexpr Network<NE> net{};
    for (long long r0 = ((long long)blockIdx.x * waves + wave) * 8; r0 < A.R; r0 += (long long)gridDim.x * waves * 8) {
        const long long r = r0 + g;
        const bool valid = r < A.R;
        const elem_t<DT>* row = reinterpret_cast<const elem_t<DT>*>(A.z + (valid ? r : r0) * A.stride_bytes) + l;
        int n0 = l;
        asm volatile("" : "+v"(n0));      // the slots' node numbers are formed here, not kept in registers across the rows
        K x[NE];
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            float f = ELG_NEG_INF;                            // behind every node of the row: a closed one of a higher index
            if (i * 8 + 8 <= V) f = (float)row[i * 8];
            else if (i * 8 < V && i * 8 + n0 < V) f = (float)row[i * 8];
            x[i] = K::make(f, i * 8 + n0);
        }
#pragma unroll
        for (int c = 0; c < net.n; ++c) exchange(x, net.a[c], net.b[c]);
        across_mirror<DPP_XOR1>(x, !(l & 1));
        merge_lane(x);
        across_mirror<DPP_MIRROR4>(x, !(l & 2));
        across<DPP_XOR1>(x, !(l & 1));
        merge_lane(x);
        across_mirror<DPP_MIRROR8>(x, !(l & 4));
        across<DPP_XOR2>(x, !(l & 2));
        across<DPP_XOR1>(x, !(l & 1));
        merge_lane(x);
        // position l NE + s of the order is slot s of lane l
        if (A.tail) {
            const float m = __shfl(x[0].value(), lane & 56, 64);
            float top = 0.f, rest = 0.f;
            const int k_here = k - n0 * NE;          // of this lane's positions, how many are among the k
#pragma unroll
            for (int s = 0; s < NE; ++s) {
                const float e = ex2((x[s].value() - m) * A.c2);
                top += s < k_here ? e : 0.f;
                rest += s < k_here ? 0.f : e;
            }
            top = oct_sum(top);
            rest = oct_sum(rest);
            // a row without an open node gives (-inf) - (-inf) = NaN here
            if (l == 0 && valid) A.tail[r] = m > ELG_NEG_INF || m != m ? rest / (top + rest) : 0.f;
        }
        wave_lds_fence();
        if (n0 * NE < k) {
#pragma unroll
            for (int s = 0; s < NE; ++s) out[(g * lanes_out + n0) * (NE + 1) + s] = x[s];
        }
        wave_lds_fence();
        const int n_out = (int)(A.R - r0 < 8 ? A.R - r0 : 8) * k;
        for (int f = lane; f < n_out; f += 64) {
            const int og = k > 1 ? (int)__umulhi((unsigned)f, A.k_inv) : f, pos = f - og * k;            // f / k: exact for f < 2^11
            const K w = out[(og * lanes_out + pos / NE) * (NE + 1) + pos % NE];
            reinterpret_cast<elem_t<DT>*>(A.values)[r0 * k + f] = (elem_t<DT>)w.value();
            A.idx[r0 * k + f] = w.index();
        }
        wave_lds_fence();
    }
}

template <int DT, int NE>
void launch_sort(const TopArgs& A, hipStream_t s) {
    const size_t per_wave = (size_t)8 * ((A.k + NE - 1) / NE) * (NE + 1) * sizeof(typename KeyOf<DT>::K);
    const int waves = 4 * per_wave > 65536 ? 2 : 4;
    const long long want = (A.R + waves * 8 - 1) / (waves * 8);
    hipLaunchKernelGGL((top_sort_kernel<DT, NE>), dim3((unsigned)(want < 4096 ? want : 4096)), dim3(64 * waves), waves * per_wave, s, A);
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Rows of 257 to 2048 logits: a wave to a row, lane l holding the nodes i 64 + l.  The same selection as a workgroup's, with counts by
// ballot: a bound from the maxima of groups of NE / 4 nodes, the few candidates above it compacted through LDS, then sorted with one, two or
// four to a lane.
// 8000 rows of 1001 f16, the best 63 and the tail: 27 us where its bytes take 4.  All 8000 waves are resident at once, and 1290 vector and 680
// scalar instructions a row keep the vector units busy 70 % of the cycles a CU has work.
template <int NE>
struct WaveRow {
    unsigned key[NE];
    // number of the row's keys >= t, the same in every lane
    __device__ __forceinline__ int count(unsigned t) const {
        int c = 0;
#pragma unroll
        for (int i = 0; i < NE; ++i) c += __popcll(__ballot(key[i] >= t));
        return c;
    }
};

// lane i <- lane i ^ D, D = 4 and 8 by two mirrors, 16 and 32 by the lane swaps
template <int D>
__device__ __forceinline__ Key64 lane_xor(const Key64 k) {
    if constexpr (D == 1) return k.moved<DPP_XOR1>();
    else if constexpr (D == 2) return k.moved<DPP_XOR2>();
    else if constexpr (D == 4) return k.moved<DPP_MIRROR8>().template moved<DPP_MIRROR4>();
    else if constexpr (D == 8) return k.moved<0x128>();                      // row_ror:8
    else {
        const unsigned long long u = __builtin_bit_cast(unsigned long long, k.d);
        const unsigned lo = (unsigned)u, hi = (unsigned)(u >> 32);
        if constexpr (D == 16) {
            const u32x2_t a = __builtin_amdgcn_permlane16_swap(lo, lo, false, false), b = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
            const bool odd = threadIdx.x & 16;
            const unsigned l2 = odd ? a[0] : a[1], h2 = odd ? b[0] : b[1];
            return {__builtin_bit_cast(double, (unsigned long long)h2 << 32 | l2)};
        } else {
            const u32x2_t a = __builtin_amdgcn_permlane32_swap(lo, lo, false, false), b = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
            const bool odd = threadIdx.x & 32;
            const unsigned l2 = odd ? a[0] : a[1], h2 = odd ? b[0] : b[1];
            return {__builtin_bit_cast(double, (unsigned long long)h2 << 32 | l2)};
        }
    }
}
// position lane * E + s of the descending order, E elements to a lane; bitonic, every merge in one direction per block of lanes
template <int E, int D>
__device__ __forceinline__ void merge_lanes(Key64 (&x)[E], int lane, bool down) {
#pragma unroll
    for (int s = 0; s < E; ++s) {
        const Key64 o = lane_xor<D>(x[s]);
        x[s] = Key64::pick(!(lane & D) != down, x[s], o);
    }
    if constexpr (D > 1) merge_lanes<E, D / 2>(x, lane, down);
}
template <int E>
__device__ __forceinline__ void merge_slots(Key64 (&x)[E], bool down) {
#pragma unroll
    for (int d = E / 2; d >= 1; d /= 2)
#pragma unroll
        for (int s = 0; s < E; ++s)
            if (!(s & d)) {
                const Key64 a = x[s], b = x[s + d], h = Key64::hi(a, b), l = Key64::lo(a, b);
                x[s] = down ? l : h;
                x[s + d] = down ? h : l;
            }
}
template <int E, int D>
__device__ __forceinline__ void sort_lanes(Key64 (&x)[E], int lane) {
    if constexpr (D > 1) sort_lanes<E, D / 2>(x, lane);
    // blocks of 2 D lanes alternate in direction (the last block is the whole wave: descending)
    const bool down = D < 32 && (lane & (2 * D));
    merge_lanes<E, D>(x, lane, down);
    merge_slots<E>(x, down);
}
template <int E>
__device__ __forceinline__ void sort_wave(Key64 (&x)[E], int lane) {
    if constexpr (E > 1) {
#pragma unroll
        for (int p = 2; p <= E; p *= 2)
#pragma unroll
            for (int d = p / 2; d >= 1; d /= 2)
#pragma unroll
                for (int s = 0; s < E; ++s)
                    if (!(s & d)) {
                        const Key64 a = x[s], b = x[s + d], h = Key64::hi(a, b), l = Key64::lo(a, b);
                        const bool rev = p < E ? (s & p) != 0 : (lane & 1);
                        x[s] = rev ? l : h;
                        x[s + d] = rev ? h : l;
                    }
    }
    sort_lanes<E, 32>(x, lane);
}

template <int DT, int NE>
__global__ __launch_bounds__(256) void top_wave_kernel(const TopArgs A) {
    constexpr int CAP = 256, GR = 4;                       // candidates a wave can sort; groups of nodes a lane keeps maxima of
    __shared__ double cand_all[4 * CAP];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, V = A.V, k = A.k;
    Key64* cand = reinterpret_cast<Key64*>(cand_all) + wave * CAP;
    for (long long r = (long long)blockIdx.x * 4 + wave; r < A.R; r += (long long)gridDim.x * 4) {
        const elem_t<DT>* row = reinterpret_cast<const elem_t<DT>*>(A.z + r * A.stride_bytes) + lane;
        int n0 = lane;
        asm volatile("" : "+v"(n0));              // node numbers and their comparisons are formed where they are used, not kept across the rows
        WaveRow<NE> z;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            float f = ELG_NEG_INF;
            if (n0 < V - i * 64) f = (float)row[i * 64];
            z.key[i] = order_key(f);
        }
        unsigned gm[GR], best = 0;
#pragma unroll
        for (int g = 0; g < GR; ++g) {
            gm[g] = z.key[g * (NE / GR)];
#pragma unroll
            for (int i = 1; i < NE / GR; ++i) gm[g] = max(gm[g], z.key[g * (NE / GR) + i]);
            best = max(best, gm[g]);
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) best = max(best, (unsigned)__shfl_xor((int)best, d, 64));
        auto groups = [&](unsigned t) {
            int c = 0;
#pragma unroll
            for (int g = 0; g < GR; ++g) c += __popcll(__ballot(gm[g] >= t));
            return c;
        };
        // ---- a lower bound of the k-th best: the k-th best group maximum (open nodes only)
        unsigned lo = KEY_NEG_INF + 1, hi = best;
        if (groups(lo) >= k)
            while (lo < hi) {
                const unsigned mid = lo + (hi - lo) / 2 + 1;
                const int c = groups(mid);
                if (c >= k) {
                    lo = mid;
                    if (c <= k + k / 8 + 4) break;
                } else hi = mid - 1;
            }
        int found = z.count(lo), ties = 0;
        unsigned tie_key = 0;
        if (found > CAP) {                                 // too many: the k-th best key itself, then equal ones by index
            hi = best;
            while (lo < hi) {
                const unsigned mid = lo + (hi - lo) / 2 + 1;
                const int c = z.count(mid);
                if (c >= k) {
                    lo = mid;
                    if (c == k) break;
                } else hi = mid - 1;
            }
            tie_key = lo;
            found = lo < 0xFFFFFFFFu ? z.count(lo + 1) : 0;
            ties = k - found;
            ++lo;                                          // (NaN as the tie: lo wraps to 0, and nothing is above it)
            if (tie_key == 0xFFFFFFFFu) lo = 0xFFFFFFFFu;
        } else if (found < k) {                            // closed nodes fill the rest, by index
            tie_key = KEY_NEG_INF;
            ties = k - found;
        }
        // ---- compaction: nodes above the bound in any order, then the ties in index order
        wave_lds_fence();
        int at = 0;
        if (found > 0)
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const bool hit = z.key[i] >= lo && !(ties > 0 && z.key[i] == tie_key);
                const unsigned long long m = __ballot(hit);
                if (hit) cand[at + lanes_below(m)] = Key64::of(((unsigned long long)z.key[i] << 20) | (0xFFFFFu - (unsigned)(i * 64 + n0)));
                at += __popcll(m);
            }
        int need = ties;
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (need > 0) {
                const bool hit = z.key[i] == tie_key && n0 < V - i * 64;
                const unsigned long long m = __ballot(hit);
                const int b = lanes_below(m);
                if (hit && b < need) cand[at + b] = Key64::of(((unsigned long long)z.key[i] << 20) | (0xFFFFFu - (unsigned)(i * 64 + n0)));
                const int n = min(need, (int)__popcll(m));
                at += n;
                need -= n;
            }
        wave_lds_fence();
        // ---- order
        Key64 last;                                        // the k-th best
        auto finish = [&](auto tag) {
            constexpr int E = decltype(tag)::value;
            Key64 x[E];
#pragma unroll
            for (int s = 0; s < E; ++s) x[s] = s * 64 + lane < at ? cand[s * 64 + lane] : Key64::of(0);
            sort_wave<E>(x, lane);
            wave_lds_fence();
#pragma unroll
            for (int s = 0; s < E; ++s)
                if (lane * E + s < k) cand[lane * E + s] = x[s];
            wave_lds_fence();
        };
        if (at <= 64) finish(std::integral_constant<int, 1>{});
        else if (at <= 128) finish(std::integral_constant<int, 2>{});
        else finish(std::integral_constant<int, 4>{});
        for (int i = lane; i < k; i += 64) {
            const Key64 w = cand[i];
            reinterpret_cast<elem_t<DT>*>(A.values)[r * k + i] = (elem_t<DT>)w.value();
            A.idx[r * k + i] = w.index();
        }
        last = cand[k - 1];
        if (A.tail) {
            const float m = key_value(best);
            const unsigned long long lu = __builtin_bit_cast(unsigned long long, last.d) & 0xFFFFFFFFFFFFFull;
            const unsigned lkey = (unsigned)(lu >> 20);
            const int lidx = last.index();
            float top = 0.f, rest = 0.f;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const float e = ex2((key_value(z.key[i]) - m) * A.c2);
                const bool in = z.key[i] > lkey || (z.key[i] == lkey && n0 <= lidx - i * 64);
                top += in ? e : 0.f;
                rest += in ? 0.f : e;
            }
            top = wave_sum(top);
            rest = wave_sum(rest);
            if (lane == 0) A.tail[r] = m > ELG_NEG_INF || m != m ? rest / (top + rest) : 0.f;
        }
        wave_lds_fence();
    }
}

template <int DT, int T, int C>
void launch_row(const TopArgs& A, hipStream_t s) {
    const long long cap = 2048 * 256 / T;                  // workgroups: what the chip holds at once
    hipLaunchKernelGGL((top_row_kernel<DT, T, C>), dim3((unsigned)(A.R < cap ? A.R : cap)), dim3(T), 0, s, A);
}
template <int DT, int NE>
void launch_wave(const TopArgs& A, hipStream_t s) {
    const long long want = (A.R + 3) / 4;
    hipLaunchKernelGGL((top_wave_kernel<DT, NE>), dim3((unsigned)(want < 2048 ? want : 2048)), dim3(256), 0, s, A);
}

// Up to 256 logits: sorted, eight lanes a row.  Up to 2048: selected, a wave a row.  Longer: a workgroup a row, its size and the chunks a
// thread holds by what keeps the row in registers (up to 256 KB of them); beyond that the row is read by every pass.
// Both sides of the borders, f32, the best 30 and the tail: 15625 rows of 256 sorted in 12.7 us, by waves in 23.1; 3906 rows of 2048 by waves in
// 18.2, by workgroups in 36.0 (bf16: 13.1 / 24.0, 19.6 / 36.4).
template <int DT>
void launch_top(const TopArgs& A, hipStream_t s) {
    const bool aligned = !((uintptr_t)A.z & 15) && !(A.stride_bytes & 15);
    const int nch = (A.V + (aligned ? 0 : VEC<DT> - 1) + VEC<DT> - 1) / VEC<DT>;
    if (A.V <= 32) launch_sort<DT, 4>(A, s);
    else if (A.V <= 64) launch_sort<DT, 8>(A, s);
    else if (A.V <= 128) launch_sort<DT, 16>(A, s);
    else if (A.V <= 256) launch_sort<DT, 32>(A, s);
    else if (A.V <= 512) launch_wave<DT, 8>(A, s);
    else if (A.V <= 1024) launch_wave<DT, 16>(A, s);
    else if (A.V <= 2048) launch_wave<DT, 32>(A, s);
    else if (nch <= 256 * 4) launch_row<DT, 256, 4>(A, s);
    else if (nch <= 256 * 8) launch_row<DT, 256, 8>(A, s);
    else if (nch <= 256 * 16) launch_row<DT, 256, 16>(A, s);
    else if (nch <= 512 * 16) launch_row<DT, 512, 16>(A, s);
    else if (nch <= 1024 * 16) launch_row<DT, 1024, 16>(A, s);
    else hipLaunchKernelGGL((top_long_kernel<DT, 1024>), dim3((unsigned)(A.R < 512 ? A.R : 512)), dim3(1024), 0, s, A);
}

}  // namespace
}  // namespace elg

using namespace elg;

extern "C" int elg_top_logits(const void* z, int64_t z_stride, int type, int64_t R, int64_t V, int k, float temperature, void* values,
                              int32_t* idx, float* tail, void* stream) {
    if (type != ELG_F32 && type != ELG_BF16 && type != ELG_F16) return fail(ELG_EINVAL, "top_logits: unknown element type");
    if (R < 0 || V <= 0 || V > ELG_ROW_MAX_V) return fail(ELG_EINVAL, "top_logits: rows of 1 .. 2^24 logits");
    if (k < 1 || k > ELG_TOP_MAX_K || k > V) return fail(ELG_EINVAL, "top_logits: 1 <= k <= min(V, 256)");
    if (!(temperature >= 1e-15f && temperature <= 1e15f)) return fail(ELG_EINVAL, "top_logits: the temperature must lie in 1e-15 .. 1e15");
    if (R == 0) return ELG_OK;
    if (!z || !values || !idx) return fail(ELG_EINVAL, "top_logits: null buffer");
    const int es = type == ELG_F32 ? 4 : 2;
    if (((uintptr_t)z | (uintptr_t)values) % es) return fail(ELG_EINVAL, "top_logits: misaligned buffer");
    TopArgs A;
    A.z = (const char*)z;
    A.stride_bytes = z_stride * es;
    A.R = R; A.V = (int)V; A.k = k;
    A.c2 = LOG2E / temperature;
    A.k_inv = k > 1 ? (unsigned)((0x100000000ull + k - 1) / k) : 0u;
    A.values = (char*)values; A.idx = idx; A.tail = tail;
    (void)hipGetLastError();
    hipStream_t st = (hipStream_t)stream;
    type == ELG_F32 ? launch_top<ELG_F32>(A, st) : type == ELG_BF16 ? launch_top<ELG_BF16>(A, st) : launch_top<ELG_F16>(A, st);
    return launch_status("top_logits");
}
