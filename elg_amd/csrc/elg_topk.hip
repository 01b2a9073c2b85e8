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

namespace elg {
namespace {

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

// One workgroup per row; the row is read again (from L2) by every pass.
template <int DT, int T>
__global__ __launch_bounds__(T) void top_row_kernel(const TopArgs A) {
    __shared__ unsigned long long cand[TOP_CAP];
    __shared__ unsigned long long win[ELG_TOP_MAX_K];
    __shared__ float fred[2 * 2 * (T / 64)];
    __shared__ int cred[2 * (T / 64)];
    __shared__ int n_cand;
    const int tid = threadIdx.x, V = A.V, k = A.k;
    BlockRed<T / 64> red(fred);
    Count<T> cnt(cred);
    for (long long r = blockIdx.x; r < A.R; r += gridDim.x) {
        const char* row = A.z + r * A.stride_bytes;
        const int shift = shift_of<DT>(row), nch = (shift + V + VEC<DT> - 1) / VEC<DT>;
        auto each = [&](auto&& f) {       // f(key, index) for every element of this thread, closed nodes included
            for (int c = tid; c < nch; c += T) {
                float v[VEC<DT>];
                unpack<DT>(load_chunk<DT>(row, shift, V, c, 0u), v);
#pragma unroll
                for (int e = 0; e < VEC<DT>; ++e) {
                    const int n = c * VEC<DT> + e - shift;
                    if (n >= 0 && n < V) f(order_key(v[e]), n);
                }
            }
        };
        // r elements equal to `key`, lowest indices first, into win[at ...]; the last one's index is the same for every thread
        auto ties = [&](unsigned key, int at, int need) {
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
        };
        // ---- the threads' maxima over open nodes, and the largest of all
        unsigned kmax = 0;
        each([&](unsigned key, int) { if (key > KEY_NEG_INF) kmax = max(kmax, key); });
        if (tid == 0) n_cand = 0;
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
        // ---- candidates
        if (kmax >= lo)
            each([&](unsigned key, int n) {
                if (key >= lo) {
                    const int p = atomicAdd(&n_cand, 1);
                    if (p < TOP_CAP) cand[p] = composite(key, n);
                }
            });
        __syncthreads();
        int found = n_cand;
        int tie_need = 0;
        unsigned tie_key = 0;
        if (found > TOP_CAP) {
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
            if (tid == 0) n_cand = 0;
            __syncthreads();
            each([&](unsigned key, int n) {
                if (key > lo) cand[atomicAdd(&n_cand, 1)] = composite(key, n);       // fewer than k of them
            });
            __syncthreads();
            found = n_cand;
            tie_key = lo;
            tie_need = k - found;
        } else if (found < k) {
            tie_key = KEY_NEG_INF;                                                   // closed nodes fill the rest
            tie_need = k - found;
        }
        // ---- rank by counting; composites are unique
        for (int i = tid; i < found; i += T) {
            const unsigned long long me = cand[i];
            int rank = 0;
            for (int j = 0; j < found; ++j) rank += cand[j] > me;
            if (rank < k) win[rank] = me;
        }
        ties(tie_key, min(found, k), tie_need);
        __syncthreads();
        for (int i = tid; i < k; i += T) {
            const unsigned long long w = win[i];
            reinterpret_cast<elem_t<DT>*>(A.values)[r * k + i] = (elem_t<DT>)key_value((unsigned)(w >> 32));
            A.idx[r * k + i] = (int)~(unsigned)w;
        }
        if (A.tail) {
            // mass outside the winners: summed apart from the winners' own, so that a small tail keeps its digits
            const unsigned long long last = win[k - 1];
            const float m = key_value((unsigned)(win[0] >> 32));
            float top = 0.f, rest = 0.f;
            if (m > ELG_NEG_INF || m != m) {
                for (int i = tid; i < k; i += T) top += ex2((key_value((unsigned)(win[i] >> 32)) - m) * A.c2);
                each([&](unsigned key, int n) {
                    if (composite(key, n) < last) rest += ex2((key_value(key) - m) * A.c2);
                });
            }
            const float2 s = red.sum2(top, rest);
            if (tid == 0) A.tail[r] = s.x + s.y > 0.f || s.x != s.x || s.y != s.y ? s.y / (s.x + s.y) : 0.f;
        }
        __syncthreads();                  // win, cand and n_cand are written again by the next row
    }
}

}  // namespace
}  // namespace elg

using namespace elg;

extern "C" int elg_top_logits(const void* z, int64_t z_stride, int type, int64_t R, int64_t V, int k, float temperature, void* values,
                              int32_t* idx, float* tail, void* stream) {
    if (type != ELG_F32 && type != ELG_BF16 && type != ELG_F16) return fail(ELG_EINVAL, "top_logits: unknown element type");
    if (R < 0 || V <= 0 || V > ELG_ROW_MAX_V) return fail(ELG_EINVAL, "top_logits: rows of 1 .. 2^24 logits");
    if (k < 1 || k > ELG_TOP_MAX_K || k > V) return fail(ELG_EINVAL, "top_logits: 1 <= k <= min(V, 256)");
    if (!(temperature > 0.f) || temperature > 3.4e38f) return fail(ELG_EINVAL, "top_logits: the temperature must be positive and finite");
    if (R == 0) return ELG_OK;
    if (!z || !values || !idx) return fail(ELG_EINVAL, "top_logits: null buffer");
    const int es = type == ELG_F32 ? 4 : 2;
    if (((uintptr_t)z | (uintptr_t)values) % es) return fail(ELG_EINVAL, "top_logits: misaligned buffer");
    TopArgs A;
    A.z = (const char*)z;
    A.stride_bytes = z_stride * es;
    A.R = R; A.V = (int)V; A.k = k;
    A.c2 = LOG2E / temperature;
    A.values = (char*)values; A.idx = idx; A.tail = tail;
    (void)hipGetLastError();
    const dim3 grid((unsigned)(R < 16384 ? R : 16384));
    if (type == ELG_F32) hipLaunchKernelGGL((top_row_kernel<ELG_F32, 256>), grid, dim3(256), 0, (hipStream_t)stream, A);
    else if (type == ELG_BF16) hipLaunchKernelGGL((top_row_kernel<ELG_BF16, 256>), grid, dim3(256), 0, (hipStream_t)stream, A);
    else hipLaunchKernelGGL((top_row_kernel<ELG_F16, 256>), grid, dim3(256), 0, (hipStream_t)stream, A);
    return launch_status("top_logits");
}
