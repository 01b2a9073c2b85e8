// Distillation of a policy from a teacher's best logits: the loss of every row and its gradient (elg_distill_loss_grad).
//
//   q_j = (1 - a) softmax_j(t_j / tau)      over the row's k teacher entries (node i_j, logit t_j); a = the teacher's mass outside them
//   p   = softmax(z / tau),  p_rest = sum of p over the nodes that are no entry's
//   L   = tau^2 w [ sum_j q_j (log q_j - log p_{i_j}) + a (log a - log p_rest) ]
//   dL/dz_n = tau w [ p_n - sum_{j: i_j = n} q_j ]   for an entry's node,     tau w p_n [ 1 - a / p_rest ]   for the others
//
// The row's softmax is formed in two parts with a maximum of its own each: the entries' nodes (k gathered logits) and the rest.  p_rest is
// then a sum of positive terms -- 1 - sum p_{i_j} would keep no digit where the entries hold nearly everything -- and stays exact in f32
// where the best node is 50 or 100 above the rest.  An entry's node listed twice counts once in the softmax and twice in q.
//
// The work is one read of the logits and one write of the gradient; everything else of a row (k entries, a few scalars) is small.
#include "elg_logits.h"

namespace elg {
namespace {

struct DistillArgs {
    const char* z;
    long long z_stride;                   // bytes
    long long R;
    int V, k;
    const void* tv;
    const void* ti;
    int tv_type, ti_wide;
    const float* tail;
    const float* weight;
    const float* cot;
    int cot_stride;
    float tau, c2;                        // c2 = log2(e) / tau
    float scale;
    float* loss_rows;
    double* part;                         // one partial loss per workgroup, or null
    float* total;                         // the loss itself, where one workgroup sees every row; or null
    float4* rec;                          // two a row: what a long row's loss is formed from; or null
    char* grad;                           // (R, V) packed, or null
    long long g_stride;                   // bytes
    // the rows from r on, for a kernel that leaves its losses in rec
    DistillArgs from(long long r) const {
        DistillArgs C = *this;
        C.z += r * z_stride;
        C.tv = (const char*)tv + r * k * (tv_type == ELG_F32 ? 4 : 2);
        C.ti = (const char*)ti + r * k * (ti_wide ? 8 : 4);
        if (tail) C.tail += r;
        if (weight) C.weight += r;
        if (cot) C.cot += r * cot_stride;
        if (rec) C.rec += 2 * r;
        if (grad) C.grad += r * g_stride;
        return C;
    }
};

// The sum of distances between teacher and student goes 2^-9 times as large (exact), so that 256 distances of the lowest value of f32, which some
// close their nodes with, add up to a finite number.
constexpr float SD_SCALE = 0x1p-9f;
// the logarithms are formed in base 2, like the exponentials, and brought to base e at their end
constexpr float LN2 = 0.6931471805599453f;
__device__ __forceinline__ float lg2(float x) { return __builtin_amdgcn_logf(x); }       // v_log_f32

// ---------------------------------------------------------------------------------------------------------------------------------
// Long rows: T >= ELG_TOP_MAX_K threads, thread j < k holding entry j, the row in 16-byte chunks.  A bitmap in LDS tells a chunk which of its
// nodes are entries': they stay out of the rest's sum, are written like the others and then written over.

// entry j = threadIdx.x of row r
struct Entry {
    int i = -1;                           // its node
    float t = ELG_NEG_INF, z = ELG_NEG_INF;
    __device__ __forceinline__ void load(const DistillArgs& A, long long r) {
        if ((int)threadIdx.x >= A.k) return;
        const long long at = r * A.k + threadIdx.x, n = index_any(A.ti, at, A.ti_wide);
        if (n >= 0 && n < A.V) {
            i = (int)n;
            t = elem_any(A.tv, at, A.tv_type);
        }
    }
    template <int DT> __device__ __forceinline__ void gather(const void* row) { if (i >= 0) z = elem<DT>(row, i); }
    // is this the first entry of its node (first), and is it the only one?  idx: the row's nodes in LDS, padded to fours with -2
    __device__ __forceinline__ void twins(const int* idx, int k, bool& first, bool& only) const {
        first = only = i >= 0;
        if (i < 0) return;
        const int me = threadIdx.x;
        for (int j = 0; j < k; j += 4) {
            const int4 o = *reinterpret_cast<const int4*>(idx + j);
            const unsigned m = (o.x == i) | (o.y == i) << 1 | (o.z == i) << 2 | (o.w == i) << 3;
            const unsigned own = (me >> 2) == (j >> 2) ? 1u << (me & 3) : 0u;
            only = only && (m & ~own) == 0u;
            first = first && (j > me || (m & (own ? own - 1u : 15u)) == 0u);
        }
    }
};

// What a row comes down to, given its maxima and sums; the same in every thread.
struct RowScalars {
    bool live;
    float q_scale, m, inv_S, c_rest, m_rest, G;
    float a, S, st, sr, sd;
    // mt, mz, mr: largest teacher logit, entry's logit, other logit (-inf: none); st, sz, sr: sums of exponentials relative to each;
    // sd: sum over entries of e^((t - mt) / tau) ((t - mt) - (z - m)), times SD_SCALE
    __device__ __forceinline__ RowScalars(const DistillArgs& A, long long r, float w, float mt, float mz, float mr, float st_, float sz, float sr_, float sd_)
        : st(st_), sr(sr_), sd(sd_) {
        a = A.tail ? A.tail[r] : 0.f;
        a = a > 1.f ? 1.f : a < 0.f ? 0.f : a;
        m = fmaxf(mz, mr);
        m_rest = mr > ELG_NEG_INF ? mr : 0.f;
        const float f_top = mz > ELG_NEG_INF ? ex2((mz - m) * A.c2) : 0.f, f_rest = mr > ELG_NEG_INF ? ex2((mr - m) * A.c2) : 0.f;
        S = sz * f_top + sr * f_rest;
        live = !(S <= 0.f) && !(st <= 0.f);
        inv_S = __builtin_amdgcn_rcpf(S);
        q_scale = st <= 0.f ? 0.f : (1.f - a) * __builtin_amdgcn_rcpf(st);
        const float cot = A.cot ? A.cot[r * A.cot_stride] : 1.f;
        G = live ? A.scale * cot * w * A.tau : 0.f;
        c_rest = live ? G * (f_rest * inv_S - (a > 0.f && sr > 0.f ? a * __builtin_amdgcn_rcpf(sr) : 0.f)) : 0.f;
        for (float* x : {&q_scale, &m, &inv_S, &c_rest, &m_rest, &G, &S}) *x = i2f(__builtin_amdgcn_readfirstlane(f2i(*x)));
    }
    // what a row's loss is formed from later (S = 0: it has none)
    __device__ __forceinline__ void record(const DistillArgs& A, long long r, float w) const {
        A.rec[2 * r] = make_float4(live ? S : 0.f, st, sr, sd);
        A.rec[2 * r + 1] = make_float4(a, m_rest - m, w, 0.f);
    }
};

// The losses of long rows from their records, in 64 bits: v_log_f32 is off by a half step of 1 near 1, the same way in every row, and a student
// near its teacher has both its logarithms there.  A thread a row, away from the kernels that hold a row in registers; one partial sum a workgroup.
__global__ __launch_bounds__(256) void distill_long_loss_kernel(const DistillArgs A) {
    __shared__ double red[4];
    double lacc = 0.0;
    for (long long r = (long long)blockIdx.x * 256 + threadIdx.x; r < A.R; r += (long long)gridDim.x * 256) {
        const float4 u = A.rec[2 * r], v = A.rec[2 * r + 1];
        double L = 0.0;
        if (u.x != 0.f) {
            const double t = 1.0 / (double)A.tau, d = (double)v.x, S = (double)u.x, st = (double)u.y;
            if (!(v.x >= 1.f)) L = (1.0 - d) * ((double)u.w / SD_SCALE / st * t + log((1.0 - d) / st * S));
            if (v.x > 0.f) L += d * (log(d * S / (double)u.z) - (double)v.y * t);
            L *= (double)A.tau * (double)A.tau * (double)v.z;
        }
        if (A.loss_rows) A.loss_rows[r] = (float)(L * (double)A.scale);
        lacc += L;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) lacc += __shfl_xor(lacc, d, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = lacc;
    __syncthreads();
    if (threadIdx.x == 0) {
        const double all = (red[0] + red[1]) + (red[2] + red[3]);
        if (A.total) A.total[0] = (float)(all * (double)A.scale);
        else if (A.part) A.part[blockIdx.x] = all;
    }
}

// N sums or maxima over the workgroup: one LDS exchange, one barrier; buffers alternate
template <int W, int N>
struct BlockN {
    float* buf;                           // 2 * W * N floats
    int flip = 0;
    __device__ explicit BlockN(float* b) : buf(b) {}
    template <bool MAX> __device__ __forceinline__ void run(float (&v)[N]) {
        float* s = buf + flip * W * N;
        flip ^= 1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = MAX ? wave_max(v[i]) : wave_sum(v[i]);
            if ((threadIdx.x & 63) == 0) s[(threadIdx.x >> 6) * N + i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = s[i];
        for (int w = 1; w < W; ++w)
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = MAX ? fmaxf(v[i], s[w * N + i]) : v[i] + s[w * N + i];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i2f(__builtin_amdgcn_readfirstlane(f2i(v[i])));      // the same in every lane: a scalar register
    }
};

// running maximum and sum of exponentials of the nodes that are no entry's, a few chunks at a time
struct Rest {
    float m = ELG_NEG_INF, s = 0.f;
    template <int N> __device__ __forceinline__ void add(const float (&v)[N], float c2) {
        float cm = v[0];
#pragma unroll
        for (int i = 1; i < N; ++i) cm = fmaxf(cm, v[i]);
        if (cm > m) {
            s = m > ELG_NEG_INF ? s * ex2((m - cm) * c2) : s;
            m = cm;
        }
        const float ref = m > ELG_NEG_INF ? m : 0.f;
        float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < N; ++i) t[i & 3] += ex2((v[i] - ref) * c2);
        s += (t[0] + t[1]) + (t[2] + t[3]);
        asm volatile("" : "+v"(s), "+v"(m));          // finished before the next values are unpacked
    }
    __device__ __forceinline__ float to(float all, float c2) const { return m > ELG_NEG_INF ? s * ex2((m - all) * c2) : s; }
};

template <int DT>
__device__ __forceinline__ void hide_entries(float (&v)[VEC<DT>], unsigned b) {
    if (__any(b & ((1u << VEC<DT>) - 1u)))            // most chunks hold none
#pragma unroll
        for (int e = 0; e < VEC<DT>; ++e) v[e] = (b >> e) & 1u ? ELG_NEG_INF : v[e];
}
// the gradient of a chunk, all its nodes taken as the rest's
template <int DT>
__device__ __forceinline__ void rest_grad(float (&v)[VEC<DT>], const RowScalars& s, float c2) {
#pragma unroll
    for (int e = 0; e < VEC<DT>; ++e) v[e] = s.live ? ex2((v[e] - s.m_rest) * c2) * s.c_rest : 0.f;
}
template <int DT>
__device__ __forceinline__ void entry_grad(void* grow, const Entry& en, const int* idx, const float* ee, int k, bool only, const RowScalars& s, float c2, float mine) {
    float q = mine;
    if (!only) {                                      // the node's masses in entry order
        q = 0.f;
        for (int j = 0; j < k; ++j) q += idx[j] == en.i ? ee[j] : 0.f;
    }
    reinterpret_cast<elem_t<DT>*>(grow)[en.i] = (elem_t<DT>)(s.G * (ex2((en.z - s.m) * c2) * s.inv_S - q * s.q_scale));
}

// zero or the rest's gradient into the chunks [c_lo, c_hi) that thread t owns, t + i step, i < C, and its edge element
template <int DT, int C>
__device__ __forceinline__ void store_rest(char* grow, const Span<DT>& sp, int t, int step, int c_hi, u32x4 (&zr)[C], int edge, float ze, const RowScalars& s, float c2) {
    const bool wide = shift_of<DT>(grow) == sp.shift;          // the gradient's rows lie like the logits': whole chunks
    elem_t<DT>* g0 = reinterpret_cast<elem_t<DT>*>(grow);
    char* gbase = grow - ((uintptr_t)grow & 15);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = t + c * step;
        if (at >= c_hi) break;
        float v[VEC<DT>];
        asm volatile("" : "+v"(zr[c]));       // unpacked again, not kept unpacked
        unpack<DT>(zr[c], v);
        rest_grad<DT>(v, s, c2);
        if (at >= sp.c_lo) {
            if (wide) *reinterpret_cast<u32x4*>(gbase + 16u * (unsigned)at) = pack<DT>(v);
            else {
#pragma unroll
                for (int e = 0; e < VEC<DT>; ++e) g0[at * VEC<DT> - sp.shift + e] = (elem_t<DT>)v[e];
            }
        }
    }
    if (edge >= 0) {
        float v[VEC<DT>] = {ze};
        rest_grad<DT>(v, s, c2);
        g0[edge] = (elem_t<DT>)v[0];
    }
}
template <int DT>
__device__ __forceinline__ void store_zero(char* grow, const Span<DT>& sp, int t, int step, int c_hi, int edge) {
    const bool wide = shift_of<DT>(grow) == sp.shift;
    elem_t<DT>* g0 = reinterpret_cast<elem_t<DT>*>(grow);
    char* gbase = grow - ((uintptr_t)grow & 15);
    for (int at = t; at < c_hi; at += step) {
        if (at < sp.c_lo) continue;
        if (wide) *reinterpret_cast<u32x4*>(gbase + 16u * (unsigned)at) = u32x4{0u, 0u, 0u, 0u};
        else {
#pragma unroll
            for (int e = 0; e < VEC<DT>; ++e) g0[at * VEC<DT> - sp.shift + e] = (elem_t<DT>)0.f;
        }
    }
    if (edge >= 0) g0[edge] = (elem_t<DT>)0.f;
}

// One workgroup per row, the row in registers, C chunks a thread (T C 16 bytes of it): one read, one write.  What bounds it is memory as long as
// two workgroups or more share a CU and their phases overlap (3125 x 32000 f32: 4.5 TB/s); the workgroup of a row of 256 KB takes the CU's
// registers alone (2048 x 131072 bf16: 282 us, 3.8 TB/s).
template <int DT, int T, int C>
__global__ __launch_bounds__(T, 4) void distill_row_kernel(const DistillArgs A) {
    static_assert(T >= ELG_TOP_MAX_K, "one entry per thread");
    constexpr int W = T / 64;
    __shared__ unsigned bits[T * C * VEC<DT> / 32];
    __shared__ __attribute__((aligned(16))) int eidx[ELG_TOP_MAX_K];
    __shared__ float ee[ELG_TOP_MAX_K];
    __shared__ float mred[2 * W * 3], sred[2 * W * 4];
    const int tid = threadIdx.x, V = A.V, k = A.k;
    BlockN<W, 3> bmax(mred);
    BlockN<W, 4> bsum(sred);
    for (int i = tid; i < T * C * VEC<DT> / 32; i += T) bits[i] = 0u;
    if (tid < ELG_TOP_MAX_K) eidx[tid] = -2;
    __syncthreads();
    for (long long r = blockIdx.x; r < A.R; r += gridDim.x) {
        const char* row = A.z + r * A.z_stride;
        char* grow = A.grad ? A.grad + r * A.g_stride : nullptr;
        const Span<DT> sp(row, V);
        const float w = A.weight ? A.weight[r] : 1.f;
        const int edge = sp.edge(tid);
        if (w == 0.f) {                   // the row is not looked at
            if (tid == 0 && A.rec) A.rec[2 * r] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (grow) store_zero<DT>(grow, sp, tid, T, sp.c_hi, edge);
            continue;
        }
        Entry en;
        en.load(A, r);
        // (what each pass needs of a chunk's place is formed there: kept from pass to pass it would not leave room for the row)
        auto place = [&]() { int t = tid; asm volatile("" : "+v"(t)); return t; };
        u32x4 zr[C];
        const int t0 = place();
#pragma unroll
        for (int c = 0; c < C; ++c) {
            constexpr unsigned pad = PAD_NEG_INF<DT>;
            zr[c] = u32x4{pad, pad, pad, pad};
            if (t0 >= sp.c_lo - c * T && t0 < sp.c_hi - c * T) zr[c] = sp.chunk(t0 + c * T);
        }
        float ze = edge >= 0 ? elem<DT>(row, edge) : ELG_NEG_INF;
        if (tid < k) eidx[tid] = en.i;
        if (en.i >= 0) atomicOr(bits + ((en.i + sp.shift) >> 5), 1u << ((en.i + sp.shift) & 31));
        __syncthreads();
        en.gather<DT>(row);
        bool first, only;
        en.twins(eidx, k, first, only);
        // ---- the rest's maximum and sum, as the chunks arrive
        Rest rest;
        const int t1 = place();
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int pos = (t1 + c * T) * VEC<DT>;
            float v[VEC<DT>];
            unpack<DT>(zr[c], v);
            hide_entries<DT>(v, bits[pos >> 5] >> (pos & 31));
            rest.add(v, A.c2);
        }
        if (edge >= 0) {
            const float v[1] = {bits[(edge + sp.shift) >> 5] >> ((edge + sp.shift) & 31) & 1u ? ELG_NEG_INF : ze};
            rest.add(v, A.c2);
        }
        float mx[3] = {en.t, en.z, rest.m};
        bmax.template run<true>(mx);
        const float tm = mx[0] > ELG_NEG_INF ? mx[0] : 0.f, zm = mx[1] > ELG_NEG_INF ? mx[1] : 0.f, m = fmaxf(mx[1], mx[2]);
        const float mine = en.i >= 0 ? ex2((en.t - tm) * A.c2) : 0.f;
        float sm[4] = {mine, first ? ex2((en.z - zm) * A.c2) : 0.f, rest.to(mx[2], A.c2),
                       mine > 0.f || mine != mine ? mine * (SD_SCALE * ((en.t - tm) - (en.z - m))) : 0.f};
        if (tid < k) ee[tid] = mine;
        if (en.i >= 0) bits[(en.i + sp.shift) >> 5] = 0u;              // clean for the next row
        bsum.template run<false>(sm);
        const RowScalars s(A, r, w, mx[0], mx[1], mx[2], sm[0], sm[1], sm[2], sm[3]);
        if (tid == 0 && A.rec) s.record(A, r, w);
        if (grow) {
            store_rest<DT, C>(grow, sp, place(), T, sp.c_hi, zr, edge, ze, s, A.c2);
            __syncthreads();
            if (first && s.live) entry_grad<DT>(grow, en, eidx, ee, k, only, s, A.c2, mine);
        }
        __syncthreads();                  // the entries' LDS is written again by the next row
    }
}

// Few long rows, or rows beyond what a workgroup can hold: a row is split into segments of SEG_T SEG_C chunks, a workgroup each.  The first
// kernel leaves every segment's maximum and sum, the second joins them and writes the segments' gradients.
// 6 rows of 100003 f32: 4 and 6.4 us, with nothing but launches and two passes over 2.4 MB in them.
constexpr int SEG_T = 256, SEG_C = 4;

template <int DT>
__device__ __forceinline__ void load_segment(u32x4 (&zr)[SEG_C], const Span<DT>& sp, int c0) {
#pragma unroll
    for (int c = 0; c < SEG_C; ++c) {
        constexpr unsigned pad = PAD_NEG_INF<DT>;
        const int at = c0 + c * SEG_T;
        zr[c] = u32x4{pad, pad, pad, pad};
        if (at >= sp.c_lo && at < sp.c_hi) zr[c] = sp.chunk(at);
    }
}

template <int DT>
__global__ __launch_bounds__(SEG_T) void distill_part_kernel(const DistillArgs A, float2* __restrict__ parts, int segs) {
    constexpr int W = SEG_T / 64, POS = SEG_T * SEG_C * VEC<DT>;
    __shared__ unsigned bits[POS / 32];
    __shared__ unsigned edge_bits;
    __shared__ float mred[2 * W], sred[2 * W];
    const int tid = threadIdx.x, V = A.V;
    const long long r = blockIdx.x / segs;
    const int seg = (int)(blockIdx.x - r * segs), c_lo = seg * SEG_T * SEG_C;
    const char* row = A.z + r * A.z_stride;
    const Span<DT> sp(row, V);
    if (A.weight && A.weight[r] == 0.f) return;
    Entry en;
    en.load(A, r);
    u32x4 zr[SEG_C];
    load_segment<DT>(zr, sp, c_lo + tid);
    const int edge = seg == segs - 1 ? sp.edge(tid) : -1;             // the last segment takes the elements outside whole chunks
    const float ze = edge >= 0 ? elem<DT>(row, edge) : ELG_NEG_INF;
    for (int i = tid; i < POS / 32; i += SEG_T) bits[i] = 0u;
    if (tid == 0) edge_bits = 0u;
    __syncthreads();
    const int p = en.i + sp.shift - c_lo * VEC<DT>;
    if (en.i >= 0 && p >= 0 && p < POS) atomicOr(bits + (p >> 5), 1u << (p & 31));
    if (en.i >= 0 && ((en.i + sp.shift) / VEC<DT> < sp.c_lo || (en.i + sp.shift) / VEC<DT> >= sp.c_hi)) atomicOr(&edge_bits, 1u << sp.edge_slot(en.i));
    __syncthreads();
    Rest rest;
#pragma unroll
    for (int c = 0; c < SEG_C; ++c) {
        const int pos = (tid + c * SEG_T) * VEC<DT>;
        float v[VEC<DT>];
        unpack<DT>(zr[c], v);
        hide_entries<DT>(v, bits[pos >> 5] >> (pos & 31));
        rest.add(v, A.c2);
    }
    if (edge >= 0) {
        const float v[1] = {edge_bits >> tid & 1u ? ELG_NEG_INF : ze};
        rest.add(v, A.c2);
    }
    BlockN<W, 1> bmax(mred), bsum(sred);
    float m[1] = {rest.m};
    bmax.template run<true>(m);
    float s[1] = {rest.to(m[0], A.c2)};
    bsum.template run<false>(s);
    if (tid == 0) parts[blockIdx.x] = make_float2(m[0], s[0]);
}

template <int DT>
__global__ __launch_bounds__(SEG_T) void distill_join_kernel(const DistillArgs A, const float2* __restrict__ parts, int segs, int grid_segs) {
    constexpr int W = SEG_T / 64;
    __shared__ __attribute__((aligned(16))) int eidx[ELG_TOP_MAX_K];
    __shared__ float ee[ELG_TOP_MAX_K];
    __shared__ float mred[2 * W * 3], sred[2 * W * 4];
    const int tid = threadIdx.x, V = A.V, k = A.k;
    const long long r = blockIdx.x / grid_segs;
    const int seg = (int)(blockIdx.x - r * grid_segs), c_lo = seg * SEG_T * SEG_C;
    const char* row = A.z + r * A.z_stride;
    char* grow = A.grad ? A.grad + r * A.g_stride : nullptr;
    const Span<DT> sp(row, V);
    const int c_end = min(sp.c_hi, c_lo + SEG_T * SEG_C), edge = seg == grid_segs - 1 ? sp.edge(tid) : -1;
    const float w = A.weight ? A.weight[r] : 1.f;
    if (w == 0.f) {
        if (tid == 0 && seg == 0 && A.rec) A.rec[2 * r] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (grow) store_zero<DT>(grow, sp, c_lo + tid, SEG_T, c_end, edge);
        return;
    }
    Entry en;
    en.load(A, r);
    Rest rest;                            // of the segments this thread joins
    for (int i = tid; i < segs; i += SEG_T) {
        const float2 p = parts[r * segs + i];
        const float all = fmaxf(rest.m, p.x);
        const float ref = all > ELG_NEG_INF ? all : 0.f;
        rest.s = (rest.m > ELG_NEG_INF ? rest.s * ex2((rest.m - ref) * A.c2) : rest.s) + (p.x > ELG_NEG_INF ? p.y * ex2((p.x - ref) * A.c2) : p.y);
        rest.m = all;
    }
    u32x4 zr[SEG_C];
    if (grow) load_segment<DT>(zr, sp, c_lo + tid);
    const float ze = grow && edge >= 0 ? elem<DT>(row, edge) : ELG_NEG_INF;
    if (tid < ELG_TOP_MAX_K) eidx[tid] = tid < k ? en.i : -2;
    en.gather<DT>(row);
    float mx[3] = {en.t, en.z, rest.m};
    BlockN<W, 3> bmax(mred);
    BlockN<W, 4> bsum(sred);
    bmax.template run<true>(mx);
    bool first, only;
    en.twins(eidx, k, first, only);
    const float tm = mx[0] > ELG_NEG_INF ? mx[0] : 0.f, zm = mx[1] > ELG_NEG_INF ? mx[1] : 0.f, m = fmaxf(mx[1], mx[2]);
    const float mine = en.i >= 0 ? ex2((en.t - tm) * A.c2) : 0.f;
    float sm[4] = {mine, first ? ex2((en.z - zm) * A.c2) : 0.f, rest.to(mx[2], A.c2),
                   mine > 0.f || mine != mine ? mine * (SD_SCALE * ((en.t - tm) - (en.z - m))) : 0.f};
    if (tid < k) ee[tid] = mine;
    bsum.template run<false>(sm);
    const RowScalars s(A, r, w, mx[0], mx[1], mx[2], sm[0], sm[1], sm[2], sm[3]);
    if (tid == 0 && seg == 0 && A.rec) s.record(A, r, w);
    if (!grow) return;
    store_rest<DT, SEG_C>(grow, sp, c_lo + tid, SEG_T, c_end, zr, edge, ze, s, A.c2);
    __syncthreads();
    // an entry's gradient is written by the workgroup that has written its node
    const int c_of = (en.i + sp.shift) / VEC<DT>;
    const bool whole = c_of >= sp.c_lo && c_of < sp.c_hi;
    if (first && s.live && (whole ? c_of >= c_lo && c_of < c_end : seg == grid_segs - 1)) entry_grad<DT>(grow, en, eidx, ee, k, only, s, A.c2, mine);
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Short rows, G lanes per row (16: four rows to a wave; 64: one).  Lane l holds the nodes n = i G + l, i < NE, and the entries
// j = e G + l, e < KE, in registers; a row is read and written in runs of G elements, whatever its alignment, and up to 16 nodes a lane the
// next row is on its way while this one is worked on (the stores of a row would otherwise stand between it and the next row's loads).
// A row of LDS, one float per node, carries what nodes and entries have to tell each other: first the nodes' logits, picked up by the entries,
// then the entries' teacher masses, picked up by the nodes (-0 marks a node of no entry, and -0 + q = q exactly).  Node n lies at
// (n % G) PN + n / G there: a lane's own nodes are side by side, so that it moves them 16 bytes at a time, and lanes lie PN apart, so that their
// banks do not meet.  Waves never wait for each other.
// The loss of a row takes v_log_f32 and v_rcp_f32, 1 ulp each.  Formed in 64 bits it is no nearer (3.2e-7 off over the rows below either way: the
// f32 sums and exponentials beneath the logarithms are what is off) and takes 289 us for 246.
// 896000 rows of 101 f32 with 40 entries: 246 us, 3.75 TB/s of needed bytes where a copy reaches 4.75; the vector units are busy 72 % of it.
// Instead of one float at a time, aligned 16-byte pieces of whole runs of rows turned through LDS took 358 us, with LDS busy 72 % of it.
template <int G> __device__ __forceinline__ float gsum(float v) { return G == 16 ? row16_sum(v) : wave_sum(v); }
template <int G> __device__ __forceinline__ float gmax(float v) { return G == 16 ? row16_max(v) : wave_max(v); }

template <int DT, int G, int NE, int KE>
struct ShortRow {
    float w, z[NE], t[KE];
    int i[KE];
    __device__ __forceinline__ void load(const DistillArgs& A, long long r, float weight, int l, bool plain_entries) {
        w = weight;
#pragma unroll
        for (int e = 0; e < KE; ++e) { i[e] = -1; t[e] = ELG_NEG_INF; }
#pragma unroll
        for (int n = 0; n < NE; ++n) z[n] = ELG_NEG_INF;
        if (w == 0.f) return;             // (a NaN weight is not 0)
        const int k = A.k, V = A.V;
        if (plain_entries) {
            const int* ti = reinterpret_cast<const int*>(A.ti) + r * k + l;
            const float* tv = reinterpret_cast<const float*>(A.tv) + r * k + l;
#pragma unroll
            for (int e = 0; e < KE; ++e)
                if (l < k - e * G) {
                    i[e] = ti[e * G];
                    t[e] = tv[e * G];
                }
        } else {
#pragma unroll
            for (int e = 0; e < KE; ++e)
                if (l < k - e * G) {
                    const long long n = index_any(A.ti, r * k + e * G + l, A.ti_wide);
                    i[e] = n >= 0 && n < V ? (int)n : -1;
                    t[e] = elem_any(A.tv, r * k + e * G + l, A.tv_type);
                }
        }
        const elem_t<DT>* row = reinterpret_cast<const elem_t<DT>*>(A.z + r * A.z_stride) + l;
#pragma unroll
        for (int n = 0; n < NE; ++n) {
            if (n * G + G <= V) z[n] = (float)row[n * G];
            else if (l < V - n * G) z[n] = (float)row[n * G];
        }
    }
};

template <int DT, int G, int NE, int KE>
__global__ __launch_bounds__(256) void distill_small_kernel(const DistillArgs A) {
    constexpr int RW = 64 / G, PN = NE == 4 ? 4 : NE + 4, P = G * PN + 4;
    constexpr bool AHEAD = NE <= 16;      // registers for the next row too
    __shared__ __attribute__((aligned(16))) float qs_all[4 * RW * P];
    __shared__ double dred[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane / G, l0 = lane % G, V = A.V;
    float* qs = qs_all + (wave * RW + g) * P;
    const bool plain_entries = A.tv_type == ELG_F32 && !A.ti_wide;
    const long long step = (long long)gridDim.x * 4 * RW;
    auto weight_of = [&](long long r) { return r < A.R ? A.weight ? A.weight[r] : 1.f : 0.f; };
    double lacc = 0.0;
    long long r0 = ((long long)blockIdx.x * 4 + wave) * RW;
    float w_next = weight_of(r0 + step + g);          // weights are two rows ahead: they decide whether the next row is loaded
    ShortRow<DT, G, NE, KE> next;
    next.load(A, r0 + g, weight_of(r0 + g), l0, plain_entries);
    for (; r0 < A.R; r0 += step) {
        const long long r = r0 + g;
        const bool valid = r < A.R;
        int l = l0;
        asm volatile("" : "+v"(l));       // the comparisons with node numbers are formed where they are used, not kept across the rows
        ShortRow<DT, G, NE, KE> x = next;
        // ---- the entries' logits
        float* mine = qs + l * PN;
        wave_lds_fence();
#pragma unroll
        for (int n = 0; n < NE; n += 4) *reinterpret_cast<float4*>(mine + n) = make_float4(x.z[n], x.z[n + 1], x.z[n + 2], x.z[n + 3]);
        wave_lds_fence();
        float zi[KE];
        int at[KE];                       // an entry's place in LDS, -1: absent
#pragma unroll
        for (int e = 0; e < KE; ++e) {
            const bool ok = (unsigned)x.i[e] < (unsigned)V;
            at[e] = ok ? (x.i[e] % G) * PN + x.i[e] / G : -1;
            x.t[e] = ok ? x.t[e] : ELG_NEG_INF;
            zi[e] = ok ? qs[at[e]] : ELG_NEG_INF;
        }
        float a = A.tail && valid ? A.tail[r] : 0.f;
        const float w_after = weight_of(r + 2 * step);
        if (AHEAD) next.load(A, r + step, w_next, l, plain_entries);
        a = a > 1.f ? 1.f : a < 0.f ? 0.f : a;
        // ---- the teacher's masses, still to be scaled
        float tm = x.t[0], mz = zi[0];
#pragma unroll
        for (int e = 1; e < KE; ++e) {
            tm = fmaxf(tm, x.t[e]);
            mz = fmaxf(mz, zi[e]);
        }
        tm = gmax<G>(tm);
        mz = gmax<G>(mz);
        tm = tm > ELG_NEG_INF ? tm : 0.f;
        const float z_ref = mz > ELG_NEG_INF ? mz : 0.f;
        float q[KE], st = 0.f, sz = 0.f;
#pragma unroll
        for (int e = 0; e < KE; ++e) {
            q[e] = at[e] >= 0 ? fabsf(ex2((x.t[e] - tm) * A.c2)) : 0.f;       // (a NaN can carry a sign: only the mark is to have one)
            st += q[e];
        }
        auto clear = [&]() {
            wave_lds_fence();
#pragma unroll
            for (int n = 0; n < NE; n += 4) *reinterpret_cast<float4*>(mine + n) = make_float4(-0.f, -0.f, -0.f, -0.f);
            wave_lds_fence();
        };
        constexpr int MARK = (int)0x80000000;
        clear();
        // Is some node listed twice?  Every entry leaves its number at its node and looks whether it is still there: two plain accesses for what
        // a returning LDS addition of floats would tell at several times the cycles.
        bool first[KE], twice = false;    // the first entry of its node counts it in the softmax
#pragma unroll
        for (int e = 0; e < KE; ++e) {
            first[e] = at[e] >= 0;
            if (at[e] >= 0) qs[at[e]] = i2f(e * G + l);
        }
        wave_lds_fence();
#pragma unroll
        for (int e = 0; e < KE; ++e)
            if (at[e] >= 0) twice = twice || f2i(qs[at[e]]) != e * G + l;
        wave_lds_fence();
#pragma unroll
        for (int e = 0; e < KE; ++e)
            if (at[e] >= 0) qs[at[e]] = q[e];
        if (__any(twice)) {               // then the masses are added up in entry order
            clear();
#pragma unroll
            for (int e = 0; e < KE; ++e)
#pragma unroll 1
                for (int j = 0; j < G; ++j) {
                    if (j == l && at[e] >= 0) {
                        const float old = qs[at[e]];
                        first[e] = f2i(old) == MARK;
                        qs[at[e]] = old + q[e];
                    }
                    wave_lds_fence();
                }
        }
        wave_lds_fence();
        float qv[NE];
#pragma unroll
        for (int n = 0; n < NE; n += 4) {
            const float4 f = *reinterpret_cast<const float4*>(mine + n);
            qv[n] = f.x; qv[n + 1] = f.y; qv[n + 2] = f.z; qv[n + 3] = f.w;
        }
#pragma unroll
        for (int e = 0; e < KE; ++e) sz += first[e] ? ex2((zi[e] - z_ref) * A.c2) : 0.f;
        // ---- the nodes: z becomes e^(z - the maximum of its part)
        float mr = ELG_NEG_INF;
#pragma unroll
        for (int n = 0; n < NE; ++n) mr = fmaxf(mr, f2i(qv[n]) < 0 ? x.z[n] : ELG_NEG_INF);
        mr = gmax<G>(mr);
        const float m_rest = mr > ELG_NEG_INF ? mr : 0.f, m = fmaxf(mz, mr);
        float sr = 0.f, sd = 0.f;
#pragma unroll
        for (int n = 0; n < NE; ++n) {
            const bool rest = f2i(qv[n]) < 0;
            x.z[n] = ex2((x.z[n] - (rest ? m_rest : z_ref)) * A.c2);
            sr += rest ? x.z[n] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < KE; ++e) sd += q[e] > 0.f || q[e] != q[e] ? q[e] * (SD_SCALE * ((x.t[e] - tm) - (zi[e] - m))) : 0.f;
        st = gsum<G>(st);
        sz = gsum<G>(sz);
        sr = gsum<G>(sr);
        // ---- the row's scalars
        const float f_top = mz > ELG_NEG_INF ? ex2((mz - m) * A.c2) : 0.f, f_rest = mr > ELG_NEG_INF ? ex2((mr - m) * A.c2) : 0.f;
        const float S = sz * f_top + sr * f_rest, inv_S = __builtin_amdgcn_rcpf(S), inv_sr = __builtin_amdgcn_rcpf(sr);
        const float q_scale = st <= 0.f ? 0.f : (1.f - a) * __builtin_amdgcn_rcpf(st);
        const bool live = x.w != 0.f && !(S <= 0.f) && !(st <= 0.f);
        if (A.loss_rows || A.part || A.total) {
            const float d = gsum<G>(sd);
            // The distances times tau^2 c2 ln 2 = tau, apart from the logarithms: a distance of the type's lowest value times c2 would be infinite.
            // All of it SD_SCALE times as large until it has met its weight.
            float L = 0.f, lg = 0.f;
            if (!(a >= 1.f)) {
                L = (d * q_scale) * A.tau;
                lg = (1.f - a) * lg2(q_scale * S);
            }
            if (a > 0.f) {
                // v_log_f32 takes a subnormal for 0, and a S / sr can be one long before a is: a small mass goes in 2^64 times as large
                const bool small = a < 1e-18f;
                lg += a * (lg2((small ? a * 0x1p64f : a) * S * inv_sr) - (small ? 64.f : 0.f));
                L -= (SD_SCALE * a * A.tau) * (m_rest - m);
                if (sr <= 0.f) lg = -ELG_NEG_INF * S;              // any mass on a rest that the student has closed (S: 1 or more, or NaN)
            }
            L = live ? (L + lg * (SD_SCALE * LN2 * A.tau * A.tau)) * x.w * (1.f / SD_SCALE) : 0.f;
            if (l == 0 && valid) {
                if (A.loss_rows) A.loss_rows[r] = L * A.scale;
                lacc += (double)L;
            }
        }
        // ---- gradient
        if (A.grad) {
            const float cot = A.cot && valid ? A.cot[r * A.cot_stride] : 1.f;
            const float Gr = live ? A.scale * cot * x.w * A.tau : 0.f;
            const float c_rest = live ? Gr * (f_rest * inv_S - (a > 0.f && sr > 0.f ? a * inv_sr : 0.f)) : 0.f;
            const float Gq = live ? Gr * q_scale : 0.f, c_top = live ? Gr * f_top * inv_S : 0.f;
            if (__any(!live))             // (whatever the nodes of a row without a gradient came to)
#pragma unroll
                for (int n = 0; n < NE; ++n) {
                    x.z[n] = live ? x.z[n] : 0.f;
                    qv[n] = live ? qv[n] : 0.f;
                }
            elem_t<DT>* grow = reinterpret_cast<elem_t<DT>*>(A.grad + r * A.g_stride) + l;
            auto put = [&](int n, float gn) {
                if (n * G + G <= V) grow[n * G] = (elem_t<DT>)gn;
                else if (l < V - n * G) grow[n * G] = (elem_t<DT>)gn;
            };
            // A NaN or infinity among the teacher's logits or in the cotangent: the masses stay with the entries' nodes, and the difference is
            // formed before it is scaled (infinity less infinity).  In other rows a node of no entry adds Gq (-0), which changes nothing.
            const bool odd = live && !(fabsf(Gq) < -ELG_NEG_INF);
            if (__any(odd)) {
                const float p_top = f_top * inv_S;
                if (valid)
#pragma unroll
                    for (int n = 0; n < NE; ++n) {
                        const bool rest = f2i(qv[n]) < 0;
                        const float usual = fmaf(x.z[n], rest ? c_rest : c_top, -Gq * qv[n]);
                        put(n, odd ? rest ? x.z[n] * c_rest : Gr * (x.z[n] * p_top - qv[n] * q_scale) : usual);
                    }
            } else if (valid) {
#pragma unroll
                for (int n = 0; n < NE; ++n) put(n, fmaf(x.z[n], f2i(qv[n]) < 0 ? c_rest : c_top, -Gq * qv[n]));
            }
        }
        if (!AHEAD) next.load(A, r + step, w_next, l, plain_entries);
        w_next = w_after;
    }
    if (A.part || A.total) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) lacc += __shfl_xor(lacc, d, 64);
        if (lane == 0) dred[wave] = lacc;
        __syncthreads();
        if (threadIdx.x == 0) {
            const double all = (dred[0] + dred[1]) + (dred[2] + dred[3]);
            if (A.total) A.total[0] = (float)(all * (double)A.scale);
            else A.part[blockIdx.x] = all;
        }
    }
}

// the workgroups' partial losses in workgroup order: the same bits in every run
__global__ __launch_bounds__(256) void distill_total_kernel(const double* __restrict__ part, int n, float scale, float* __restrict__ total) {
    __shared__ double s[256];
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) v += part[i];
    s[threadIdx.x] = v;
    __syncthreads();
    for (int d = 128; d > 0; d >>= 1) {
        if ((int)threadIdx.x < d) s[threadIdx.x] += s[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) total[0] = (float)(s[0] * (double)scale);
}

constexpr int MAX_GRID = 2048;

template <int DT, int G, int NE, int KE>
void launch_small(const DistillArgs& A, int grid, hipStream_t s) {
    hipLaunchKernelGGL((distill_small_kernel<DT, G, NE, KE>), dim3((unsigned)grid), dim3(256), 0, s, A);
}

// How a call is laid out, from its sizes alone (the scratch it needs follows from them too).
struct Plan {
    int lanes;                            // of a short row; 0: a workgroup or more
    bool split;
    int segs;
    long long grid;                       // workgroups of the kernel that sees the rows
    long long parts;                      // partial losses; 1: the loss itself is written, no scratch for them
    Plan(long long R, long long V, int type) {
        const int vec = type == ELG_F32 ? 4 : 8;
        // rows that no workgroup can hold, or so few long ones that most of the chip would idle.  Loss and gradient, split / by a workgroup each:
        // 65536 f32, 6 rows 11 / 18 us, 64 rows 18.6 / 21.2, 128 rows 25.7 / 23.7, 256 rows 42 / 32.5; 9001 f32, 6 rows 11.2 / 12.2, 64 rows
        // 11.6 / 12.2, 192 rows 13.7 / 13.1; 131072 bf16, 64 rows 21.7 / 29, 128 rows 29 / 31, 192 rows 40 / 34
        lanes = V <= 256 ? 16 : V <= 2048 ? 64 : 0;
        split = !lanes && (V > 1024 * 16 * vec || (R <= 64 && V > 1024 * vec));
        segs = split ? (int)((V + vec - 1 + SEG_T * SEG_C * vec - 1) / (SEG_T * SEG_C * vec)) : 0;     // a row may start inside its first 16 bytes
        const long long rows_wg = lanes == 16 ? 16 : lanes == 64 ? 4 : 1, want = (R + rows_wg - 1) / rows_wg;
        grid = want < MAX_GRID ? want : MAX_GRID;
        // so few short rows that one workgroup forms their total: a launch and the scratch saved.  Long rows: a thread a row
        parts = lanes ? (want <= 8 ? 1 : grid) : R <= 1024 ? 1 : (R + 255) / 256 < 256 ? (R + 255) / 256 : 256;
    }
    // partial losses | records of long rows | segments of split ones
    long long rec_at() const { return parts > 1 ? 8 * ((parts + 1) / 2 * 2) : 0; }
    long long segs_at(long long R) const { return rec_at() + (lanes ? 0 : 32 * R); }
    long long bytes(long long R) const { return segs_at(R) + 8 * R * segs; }
};

template <int DT, int T, int C>
void launch_row(const DistillArgs& A, int grid, hipStream_t s) {
    hipLaunchKernelGGL((distill_row_kernel<DT, T, C>), dim3((unsigned)grid), dim3(T), 0, s, A);
}

// Rows of up to 256 logits take a quarter of a wave, up to 2048 a wave (the registers of a lane sized by the next power of two), longer ones a
// workgroup or several.  Both sides of the borders, f32, loss and gradient with 30 entries: 15625 rows of 256 in 14.2 us by quarters, 19.5 by
// waves; 3906 rows of 2048 in 18.9 us by waves, 27.8 by workgroups.  Entry slots a lane, 200000 rows of 101: k = 16 with 1 / 3 / 16 slots 51 / 53 /
// 108 us, k = 48 with 3 / 16 slots 60 / 112, k = 63 with 16 slots 113; 20000 rows of 1001 by waves, k = 64 with 1 / 4 slots 39.5 / 40.5.
template <int DT>
void launch(const DistillArgs& A, const Plan& P, float2* parts, hipStream_t s) {
    const int V = A.V, k = A.k, grid = P.lanes && A.total ? 1 : (int)P.grid;
    // chunks a row can span: its own and, unless every row starts on 16 bytes, what the first line holds in front of it
    const bool aligned = !((uintptr_t)A.z & 15) && !(A.z_stride & 15);
    const int nch = (V + (aligned ? 0 : VEC<DT> - 1) + VEC<DT> - 1) / VEC<DT>;
    auto fits = [&](int g, int ne) { return V <= g * ne; };
    if (P.lanes == 16) {
        if (k > 48) fits(16, 8) ? launch_small<DT, 16, 8, 16>(A, grid, s) : launch_small<DT, 16, 16, 16>(A, grid, s);
        else if (k > 16) fits(16, 4) ? launch_small<DT, 16, 4, 3>(A, grid, s) : fits(16, 8) ? launch_small<DT, 16, 8, 3>(A, grid, s) : launch_small<DT, 16, 16, 3>(A, grid, s);
        else fits(16, 4) ? launch_small<DT, 16, 4, 1>(A, grid, s) : fits(16, 8) ? launch_small<DT, 16, 8, 1>(A, grid, s) : launch_small<DT, 16, 16, 1>(A, grid, s);
    } else if (P.lanes == 64) {
        if (k <= 64) fits(64, 8) ? launch_small<DT, 64, 8, 1>(A, grid, s) : fits(64, 16) ? launch_small<DT, 64, 16, 1>(A, grid, s) : launch_small<DT, 64, 32, 1>(A, grid, s);
        else fits(64, 8) ? launch_small<DT, 64, 8, 4>(A, grid, s) : fits(64, 16) ? launch_small<DT, 64, 16, 4>(A, grid, s) : launch_small<DT, 64, 32, 4>(A, grid, s);
    } else if (P.split) {
        const int grad_segs = A.grad ? P.segs : 1;
        const long long at_once = LAUNCH_WG / P.segs;          // rows of a launch
        for (long long r = 0; r < A.R; r += at_once) {
            const long long n = A.R - r < at_once ? A.R - r : at_once;
            const DistillArgs C = A.from(r);
            hipLaunchKernelGGL((distill_part_kernel<DT>), dim3((unsigned)(n * P.segs)), dim3(SEG_T), 0, s, C, parts, P.segs);
            hipLaunchKernelGGL((distill_join_kernel<DT>), dim3((unsigned)(n * grad_segs)), dim3(SEG_T), 0, s, C, parts, P.segs, grad_segs);
        }
    } else if (nch <= 256 * 4) launch_row<DT, 256, 4>(A, grid, s);
    else if (nch <= 256 * 8) launch_row<DT, 256, 8>(A, grid, s);
    else if (nch <= 256 * 16) launch_row<DT, 256, 16>(A, grid, s);
    else if (nch <= 512 * 16) launch_row<DT, 512, 16>(A, grid, s);
    else if (nch <= 1024 * 16) launch_row<DT, 1024, 16>(A, grid, s);
    else launch_row<DT, 1024, 17>(A, grid, s);
}

}  // namespace
}  // namespace elg

using namespace elg;

extern "C" int64_t elg_distill_ws_bytes(int64_t R, int64_t V, int type) {
    if (R <= 0 || V <= 0 || V > ELG_ROW_MAX_V) return 0;
    return Plan(R, V, type).bytes(R);
}

extern "C" int elg_distill_loss_grad(const void* z, int64_t z_stride, int type, int64_t R, int64_t V, const void* top_values, int top_type,
                                     const void* top_idx, int idx_wide, int k, const float* tail, float temperature, const float* weight,
                                     const float* cot, int cot_stride, float scale, float* loss_rows, float* loss_total, void* grad,
                                     void* ws, int64_t ws_bytes, void* stream) {
    if (type != ELG_F32 && type != ELG_BF16 && type != ELG_F16) return fail(ELG_EINVAL, "distill: unknown element type");
    if (top_type != ELG_F32 && top_type != ELG_BF16 && top_type != ELG_F16) return fail(ELG_EINVAL, "distill: unknown type of the teacher's logits");
    if (R < 0 || V <= 0 || V > ELG_ROW_MAX_V) return fail(ELG_EINVAL, "distill: rows of 1 .. 2^24 logits");
    if (k < 1 || k > ELG_TOP_MAX_K) return fail(ELG_EINVAL, "distill: 1 <= k <= 256 teacher entries a row");
    if (!(temperature >= 1e-15f && temperature <= 1e15f)) return fail(ELG_EINVAL, "distill: the temperature must lie in 1e-15 .. 1e15");
    if (cot_stride != 0 && cot_stride != 1) return fail(ELG_EINVAL, "distill: the cotangent is one number or one per row");
    if (!loss_rows && !loss_total && !grad) return fail(ELG_EINVAL, "distill: nothing to compute");
    if (R > 0 && (!z || !top_values || !top_idx)) return fail(ELG_EINVAL, "distill: null buffer");
    const Plan P(R, V, type);
    const bool want_loss = loss_rows || loss_total, scratch = P.split || (P.lanes ? loss_total && P.parts > 1 : want_loss);
    if (R > 0 && scratch && (!ws || ws_bytes < P.bytes(R))) return fail(ELG_EINVAL, "distill: needs elg_distill_ws_bytes() of scratch");
    if (R == 0 && !loss_total) return ELG_OK;
    const int es = type == ELG_F32 ? 4 : 2;
    if (((uintptr_t)z | (uintptr_t)grad) % es || (uintptr_t)top_values % (top_type == ELG_F32 ? 4 : 2) || (uintptr_t)top_idx % (idx_wide ? 8 : 4) || (uintptr_t)ws % 16)
        return fail(ELG_EINVAL, "distill: misaligned buffer");
    DistillArgs A;
    A.z = (const char*)z; A.z_stride = z_stride * es; A.R = R; A.V = (int)V; A.k = k;
    A.tv = top_values; A.ti = top_idx; A.tv_type = top_type; A.ti_wide = idx_wide != 0;
    A.tail = tail; A.weight = weight; A.cot = cot; A.cot_stride = cot_stride;
    A.tau = temperature; A.c2 = LOG2E / temperature; A.scale = scale;
    A.loss_rows = loss_rows;
    A.part = loss_total && P.parts > 1 ? (double*)ws : nullptr;
    A.total = loss_total && P.parts == 1 ? loss_total : nullptr;
    A.rec = want_loss && !P.lanes && R > 0 ? reinterpret_cast<float4*>((char*)ws + P.rec_at()) : nullptr;
    A.grad = (char*)grad; A.g_stride = V * es;
    (void)hipGetLastError();
    hipStream_t st = (hipStream_t)stream;
    if (R > 0) {
        float2* parts = reinterpret_cast<float2*>((char*)ws + P.segs_at(R));
        type == ELG_F32 ? launch<ELG_F32>(A, P, parts, st) : type == ELG_BF16 ? launch<ELG_BF16>(A, P, parts, st) : launch<ELG_F16>(A, P, parts, st);
        if (A.rec) hipLaunchKernelGGL(distill_long_loss_kernel, dim3((unsigned)(P.parts > 1 ? P.parts : R > 256 ? (A.total ? 1 : 4) : 1)), dim3(256), 0, st, A);
    }
    if (loss_total && (A.part || R == 0))
        hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(256), 0, st, (const double*)ws, R > 0 ? (int)P.parts : 0, scale, loss_total);
    return launch_status("distill");
}
