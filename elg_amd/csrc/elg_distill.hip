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
    char* grad;                           // (R, V) packed, or null
    long long g_stride;                   // bytes
};

constexpr float TINY_MASS = 1e-36f;       // a (log a - log p_rest) below this is nothing in f32
__device__ __forceinline__ float ln(float x) { return __builtin_amdgcn_logf(x) * 0.6931471805599453f; }

constexpr int SEG = 65536;                // window positions whose membership bits are held at a time

// One workgroup per row, T >= ELG_TOP_MAX_K threads: thread j < k holds entry j.  C > 0: the row stays in registers, C chunks a thread;
// C = 0: it is read once for the sums and once for the gradient.
template <int DT, int T, int C>
__global__ __launch_bounds__(T) void distill_row_kernel(const DistillArgs A) {
    static_assert(T >= ELG_TOP_MAX_K, "one entry per thread");
    constexpr int W = T / 64, BITS = C ? T * C * VEC<DT> : SEG;
    __shared__ unsigned bits[BITS / 32];
    __shared__ int eidx[ELG_TOP_MAX_K];
    __shared__ float eq[ELG_TOP_MAX_K];
    __shared__ float fred[2 * 2 * W];
    const int tid = threadIdx.x, V = A.V, k = A.k;
    BlockRed<W> red(fred);
    double lacc = 0.0;
    for (long long r = blockIdx.x; r < A.R; r += gridDim.x) {
        const char* row = A.z + r * A.z_stride;
        char* grow = A.grad ? A.grad + r * A.g_stride : nullptr;
        const int shift = shift_of<DT>(row), nch = (shift + V + VEC<DT> - 1) / VEC<DT>;
        const float w = A.weight ? A.weight[r] : 1.f;
        // ---- entries
        int ei = -1;
        float et = ELG_NEG_INF, zi = ELG_NEG_INF;
        if (w != 0.f && tid < k) {
            const long long i = index_any(A.ti, r * k + tid, A.ti_wide);
            if (i >= 0 && i < V) {
                ei = (int)i;
                et = elem_any(A.tv, r * k + tid, A.tv_type);
                zi = elem<DT>(row, i);
            }
        }
        u32x4 zr[C ? C : 1];
        if (C && w != 0.f) {
#pragma unroll
            for (int c = 0; c < C; ++c)
                zr[c] = tid + c * T < nch ? load_chunk<DT>(row, shift, V, tid + c * T, PAD_NEG_INF<DT>) : u32x4{PAD_NEG_INF<DT>, PAD_NEG_INF<DT>, PAD_NEG_INF<DT>, PAD_NEG_INF<DT>};
        }
        if (w == 0.f) {                   // the row is not looked at
            if (tid == 0 && A.loss_rows) A.loss_rows[r] = 0.f;
            if (grow) {
                const float zero[VEC<DT>] = {};
                for (int c = tid; c < nch; c += T) store_chunk<DT>(grow, shift, V, c, zero);
            }
            continue;
        }
        if (tid < k) eidx[tid] = ei;
        const float2 mx = red.max2(et, zi);
        const float tm = mx.x > ELG_NEG_INF ? mx.x : 0.f, m_top = mx.y > ELG_NEG_INF ? mx.y : 0.f;
        const float ee = ei >= 0 ? ex2((et - tm) * A.c2) : 0.f;
        // first entry of its node?  (k broadcast reads; equal nodes are counted once in the softmax)
        bool first = ei >= 0;
        if (tid < k)
            for (int j = 0; j < tid; ++j) first = first && eidx[j] != ei;
        const float2 sm = red.sum2(ee, first ? ex2((zi - m_top) * A.c2) : 0.f);
        const float st = sm.x, s_top = sm.y;
        float a = A.tail ? A.tail[r] : 0.f;
        a = a > 1.f ? 1.f : a < 0.f ? 0.f : a;
        const float q = ei >= 0 && ee > 0.f ? ee * ((1.f - a) / st) : 0.f * ee;
        if (tid < k) eq[tid] = q;
        // ---- the rest: maximum and sum over the nodes of no entry
        float rm = ELG_NEG_INF, rs = 0.f;
        if (C) {
            for (int i = tid; i < (nch * VEC<DT> + 31) / 32; i += T) bits[i] = 0u;
            __syncthreads();
            if (ei >= 0) atomicOr(bits + ((ei + shift) >> 5), 1u << ((ei + shift) & 31));
            __syncthreads();
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int pos = (tid + c * T) * VEC<DT>;
                const unsigned b = tid + c * T < nch ? bits[pos >> 5] >> (pos & 31) : 0u;
                float v[VEC<DT>];
                unpack<DT>(zr[c], v);
#pragma unroll
                for (int e = 0; e < VEC<DT>; ++e) rm = fmaxf(rm, (b >> e) & 1u ? ELG_NEG_INF : v[e]);
            }
            rm = red.max2(rm, rm).x;
            const float ref = rm > ELG_NEG_INF ? rm : 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int pos = (tid + c * T) * VEC<DT>;
                const unsigned b = tid + c * T < nch ? bits[pos >> 5] >> (pos & 31) : 0u;
                float v[VEC<DT>];
                unpack<DT>(zr[c], v);
#pragma unroll
                for (int e = 0; e < VEC<DT>; ++e) rs += (b >> e) & 1u ? 0.f : ex2((v[e] - ref) * A.c2);
            }
        } else {
            for (int s0 = 0; s0 < nch * VEC<DT>; s0 += SEG) {
                const int s1 = min(s0 + SEG, nch * VEC<DT>);
                __syncthreads();
                for (int i = tid; i < SEG / 32; i += T) bits[i] = 0u;
                __syncthreads();
                if (ei >= 0 && ei + shift >= s0 && ei + shift < s1) atomicOr(bits + ((ei + shift - s0) >> 5), 1u << ((ei + shift) & 31));
                __syncthreads();
                for (int c = s0 / VEC<DT> + tid; c < s1 / VEC<DT>; c += T) {
                    const int pos = c * VEC<DT> - s0;
                    const unsigned b = bits[pos >> 5] >> (pos & 31);
                    float v[VEC<DT>], cm = ELG_NEG_INF;
                    unpack<DT>(load_chunk<DT>(row, shift, V, c, PAD_NEG_INF<DT>), v);
#pragma unroll
                    for (int e = 0; e < VEC<DT>; ++e) {
                        v[e] = (b >> e) & 1u ? ELG_NEG_INF : v[e];
                        cm = fmaxf(cm, v[e]);
                    }
                    if (cm > rm) {
                        rs = rm > ELG_NEG_INF ? rs * ex2((rm - cm) * A.c2) : rs;
                        rm = cm;
                    }
                    const float ref = rm > ELG_NEG_INF ? rm : 0.f;
#pragma unroll
                    for (int e = 0; e < VEC<DT>; ++e) rs += ex2((v[e] - ref) * A.c2);
                }
            }
            const float all = red.max2(rm, rm).x;
            rs = rm > ELG_NEG_INF ? rs * ex2((rm - all) * A.c2) : rs;
            rm = all;
        }
        // ---- the row's scalars and its loss
        const float m_rest = rm > ELG_NEG_INF ? rm : 0.f;
        const float m = fmaxf(mx.y, rm);
        const float f_top = mx.y > ELG_NEG_INF ? ex2((m_top - m) * A.c2) : 0.f, f_rest = rm > ELG_NEG_INF ? ex2((m_rest - m) * A.c2) : 0.f;
        const float part_loss = q > 0.f || q != q ? q * (((et - tm) - (zi - m)) / A.tau) : 0.f;
        const float2 lr = red.sum2(rs, part_loss);
        const float s_rest = lr.x;
        const float S = s_top * f_top + s_rest * f_rest;
        const bool live = !(S <= 0.f) && !(st <= 0.f);
        const float logS = logf(S);
        if (tid == 0) {
            float L = 0.f;
            if (live) {
                L = lr.y;
                if (a < 1.f) L += (1.f - a) * (logf((1.f - a) / st) + logS);
                if (a > 0.f) L += a * (logf(a) - ((m_rest - m) / A.tau + logf(s_rest) - logS));
                L *= A.tau * A.tau * w;
            }
            if (A.loss_rows) A.loss_rows[r] = L * A.scale;
            lacc += (double)L;
        }
        // ---- gradient: every node as one of the rest first, then the entries' nodes on top of it
        if (grow) {
            const float cot = A.cot ? A.cot[r * A.cot_stride] : 1.f;
            const float G = live ? A.scale * cot * w * A.tau : 0.f;
            const float c_rest = live ? G * (f_rest / S - (a > 0.f && s_rest > 0.f ? a / s_rest : 0.f)) : 0.f;
            if (C) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    if (tid + c * T >= nch) break;
                    float v[VEC<DT>];
                    unpack<DT>(zr[c], v);
#pragma unroll
                    for (int e = 0; e < VEC<DT>; ++e) v[e] = live ? ex2((v[e] - m_rest) * A.c2) * c_rest : 0.f;
                    store_chunk<DT>(grow, shift, V, tid + c * T, v);
                }
            } else {
                for (int c = tid; c < nch; c += T) {
                    float v[VEC<DT>];
                    unpack<DT>(load_chunk<DT>(row, shift, V, c, PAD_NEG_INF<DT>), v);
#pragma unroll
                    for (int e = 0; e < VEC<DT>; ++e) v[e] = live ? ex2((v[e] - m_rest) * A.c2) * c_rest : 0.f;
                    store_chunk<DT>(grow, shift, V, c, v);
                }
            }
            __syncthreads();
            if (first && live) {
                float qn = 0.f;
                for (int j = 0; j < k; ++j) qn += eidx[j] == ei ? eq[j] : 0.f;
                reinterpret_cast<elem_t<DT>*>(grow)[ei] = (elem_t<DT>)(G * (ex2((zi - m) * A.c2) / S - qn));
            }
        }
        __syncthreads();                  // the entries' LDS is written again by the next row
    }
    if (A.part && tid == 0) A.part[blockIdx.x] = lacc;
}

// Short rows, G lanes per row (16: four rows to a wave; 64: one).  Lane l holds the nodes n = i G + l, i < NE, and the entries
// j = e G + l, e < KE, in registers; a row is read and written in runs of G elements, whatever its alignment.  The row's teacher masses are
// spread over a row of LDS, one float per node, where the lane that owns the node picks them up: -0 marks a node of no entry, and
// -0 + q = q exactly.  Waves never wait for each other.
template <int G> __device__ __forceinline__ float gsum(float v) { return G == 16 ? row16_sum(v) : wave_sum(v); }
template <int G> __device__ __forceinline__ float gmax(float v) { return G == 16 ? row16_max(v) : wave_max(v); }

template <int DT, int G, int NE, int KE, bool TAIL>
__global__ __launch_bounds__(256) void distill_small_kernel(const DistillArgs A) {
    // a row of LDS is padded so that the rows of a wave's four groups start 16 banks apart
    constexpr int RW = 64 / G, P = G * NE + (G == 16 ? 16 : 0);
    __shared__ float qs_all[4 * RW * P];
    __shared__ double dred[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane / G, l = lane % G, V = A.V, k = A.k;
    float* qs = qs_all + (wave * RW + g) * P;
    const bool plain_entries = A.tv_type == ELG_F32 && !A.ti_wide;
    const float inv_tau = 1.f / A.tau;
    double lacc = 0.0;
    for (long long r0 = ((long long)blockIdx.x * 4 + wave) * RW; r0 < A.R; r0 += (long long)gridDim.x * 4 * RW) {
        const long long r = r0 + g;
        const bool valid = r < A.R;
        const float w = !valid ? 0.f : A.weight ? A.weight[r] : 1.f;
        const bool on = w != 0.f;
        const elem_t<DT>* row = reinterpret_cast<const elem_t<DT>*>(A.z + (valid ? r : 0) * A.z_stride);
        // ---- entries and nodes
        const int kk = on ? k : 0, vv = on ? V : 0;
        int ei[KE];
        float et[KE], zi[KE];
        if (plain_entries) {
            const int* ti = reinterpret_cast<const int*>(A.ti) + r * k;
            const float* tv = reinterpret_cast<const float*>(A.tv) + r * k;
#pragma unroll
            for (int e = 0; e < KE; ++e) {
                const int j = e * G + l;
                ei[e] = j < kk ? ti[j] : -1;
                et[e] = j < kk ? tv[j] : ELG_NEG_INF;
            }
        } else {
#pragma unroll
            for (int e = 0; e < KE; ++e) {
                const int j = e * G + l;
                ei[e] = -1;
                et[e] = ELG_NEG_INF;
                if (j < kk) {
                    const long long i = index_any(A.ti, r * k + j, A.ti_wide);
                    ei[e] = i >= 0 && i < V ? (int)i : -1;
                    et[e] = elem_any(A.tv, r * k + j, A.tv_type);
                }
            }
        }
        float v[NE];
#pragma unroll
        for (int i = 0; i < NE; ++i) v[i] = i * G + l < vv ? (float)row[i * G + l] : ELG_NEG_INF;
#pragma unroll
        for (int e = 0; e < KE; ++e) {
            const bool ok = (unsigned)ei[e] < (unsigned)V;
            ei[e] = ok ? ei[e] : -1;
            et[e] = ok ? et[e] : ELG_NEG_INF;
            zi[e] = ok ? (float)row[ei[e]] : ELG_NEG_INF;
        }
        float a = TAIL && on ? A.tail[r] : 0.f;
        a = a > 1.f ? 1.f : a < 0.f ? 0.f : a;
        // ---- the teacher's masses
        float tm = et[0];
#pragma unroll
        for (int e = 1; e < KE; ++e) tm = fmaxf(tm, et[e]);
        tm = gmax<G>(tm);
        tm = tm > ELG_NEG_INF ? tm : 0.f;
        float q[KE], st = 0.f;
#pragma unroll
        for (int e = 0; e < KE; ++e) {
            q[e] = ei[e] >= 0 ? ex2((et[e] - tm) * A.c2) : 0.f;
            st += q[e];
        }
        st = gsum<G>(st);
        const float qscale = st <= 0.f ? 0.f : (1.f - a) * __builtin_amdgcn_rcpf(st);
#pragma unroll
        for (int e = 0; e < KE; ++e) q[e] *= qscale;
        auto clear = [&]() {
            wave_lds_fence();
#pragma unroll
            for (int i = 0; i < NE; ++i) qs[i * G + l] = -0.f;
            wave_lds_fence();
        };
        clear();
        bool twice = false;
#pragma unroll
        for (int e = 0; e < KE; ++e)
            if (ei[e] >= 0) {
                const float old = __hip_atomic_fetch_add(qs + ei[e], q[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                twice = twice || f2i(old) != (int)0x80000000;
            }
        if (__any(twice)) {               // some node is listed twice: add its masses again, in entry order, so that the bits are the same in every run
            clear();
#pragma unroll
            for (int e = 0; e < KE; ++e)
#pragma unroll 1
                for (int j = 0; j < G; ++j) {
                    if (j == l && ei[e] >= 0) qs[ei[e]] += q[e];
                    wave_lds_fence();
                }
        }
        wave_lds_fence();
        float qv[NE];
#pragma unroll
        for (int i = 0; i < NE; ++i) qv[i] = qs[i * G + l];
        // ---- the student's softmax; v becomes e^(z - its part's maximum)
        float m, S, f_top = 1.f, f_rest = 0.f, s_rest = 0.f, m_rest = 0.f;
        if (TAIL) {
            float mt = ELG_NEG_INF, mr = ELG_NEG_INF;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const bool top = f2i(qv[i]) >= 0;
                mt = fmaxf(mt, top ? v[i] : ELG_NEG_INF);
                mr = fmaxf(mr, top ? ELG_NEG_INF : v[i]);
            }
            mt = gmax<G>(mt);
            mr = gmax<G>(mr);
            m = fmaxf(mt, mr);
            const float m_top = mt > ELG_NEG_INF ? mt : 0.f;
            m_rest = mr > ELG_NEG_INF ? mr : 0.f;
            float s_top = 0.f;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const bool top = f2i(qv[i]) >= 0;
                v[i] = ex2((v[i] - (top ? m_top : m_rest)) * A.c2);
                s_top += top ? v[i] : 0.f;
                s_rest += top ? 0.f : v[i];
            }
            s_top = gsum<G>(s_top);
            s_rest = gsum<G>(s_rest);
            f_top = mt > ELG_NEG_INF ? ex2((m_top - m) * A.c2) : 0.f;
            f_rest = mr > ELG_NEG_INF ? ex2((m_rest - m) * A.c2) : 0.f;
            S = s_top * f_top + s_rest * f_rest;
        } else {
            m = v[0];
#pragma unroll
            for (int i = 1; i < NE; ++i) m = fmaxf(m, v[i]);
            m = gmax<G>(m);
            const float ref = m > ELG_NEG_INF ? m : 0.f;
            S = 0.f;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                v[i] = ex2((v[i] - ref) * A.c2);
                S += v[i];
            }
            S = gsum<G>(S);
        }
        const bool live = on && !(S <= 0.f) && !(st <= 0.f);
        const float inv_S = __builtin_amdgcn_rcpf(S);
        // ---- loss
        if (A.loss_rows || A.part) {
            float L = 0.f;
#pragma unroll
            for (int e = 0; e < KE; ++e) L += q[e] > 0.f || q[e] != q[e] ? q[e] * ((et[e] - tm) - (zi[e] - m)) : 0.f;
            L = gsum<G>(L) * inv_tau;
            if (a < 1.f) L += (1.f - a) * ln(qscale * S);
            if (TAIL && a > TINY_MASS) L += a * (ln(a * S * __builtin_amdgcn_rcpf(s_rest)) - (m_rest - m) * inv_tau);
            L = live ? L * (A.tau * A.tau * w) : 0.f;
            if (l == 0 && valid) {
                if (A.loss_rows) A.loss_rows[r] = L * A.scale;
                lacc += (double)L;
            }
        }
        // ---- gradient
        if (A.grad && valid) {
            const float cot = A.cot ? A.cot[r * A.cot_stride] : 1.f;
            const float Gr = live ? A.scale * cot * w * A.tau : 0.f, c_top = live ? Gr * f_top * inv_S : 0.f;
            float c_rest = c_top;
            if (TAIL) c_rest = live ? Gr * (f_rest * inv_S - (a > 0.f && s_rest > 0.f ? a * __builtin_amdgcn_rcpf(s_rest) : 0.f)) : 0.f;
            elem_t<DT>* grow = reinterpret_cast<elem_t<DT>*>(A.grad + r * A.g_stride);
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const float t = fmaf(live ? v[i] : 0.f, !TAIL || f2i(qv[i]) >= 0 ? c_top : c_rest, -Gr * qv[i]);
                if (i * G + l < V) grow[i * G + l] = (elem_t<DT>)t;
            }
        }
    }
    if (A.part) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) lacc += __shfl_xor(lacc, d, 64);
        if (lane == 0) dred[wave] = lacc;
        __syncthreads();
        if (threadIdx.x == 0) A.part[blockIdx.x] = (dred[0] + dred[1]) + (dred[2] + dred[3]);
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
    if (A.tail) hipLaunchKernelGGL((distill_small_kernel<DT, G, NE, KE, true>), dim3((unsigned)grid), dim3(256), 0, s, A);
    else hipLaunchKernelGGL((distill_small_kernel<DT, G, NE, KE, false>), dim3((unsigned)grid), dim3(256), 0, s, A);
}

// Rows of up to 256 logits take a quarter of a wave, up to 2048 a wave, longer ones a workgroup; the registers of a lane are sized by the
// next power of two.
template <int DT>
int launch(const DistillArgs& A, hipStream_t s) {
    const int V = A.V, k = A.k;
    const long long rows_wg = V <= 256 ? 16 : V <= 2048 ? 4 : 1, want = (A.R + rows_wg - 1) / rows_wg;
    const int grid = (int)(want < MAX_GRID ? want : MAX_GRID);
    if (V <= 256) {
        if (k > 48) V <= 128 ? launch_small<DT, 16, 8, 16>(A, grid, s) : launch_small<DT, 16, 16, 16>(A, grid, s);
        else if (k > 16) V <= 64 ? launch_small<DT, 16, 4, 3>(A, grid, s) : V <= 128 ? launch_small<DT, 16, 8, 3>(A, grid, s) : launch_small<DT, 16, 16, 3>(A, grid, s);
        else if (V <= 32) launch_small<DT, 16, 2, 1>(A, grid, s);
        else V <= 64 ? launch_small<DT, 16, 4, 1>(A, grid, s) : V <= 128 ? launch_small<DT, 16, 8, 1>(A, grid, s) : launch_small<DT, 16, 16, 1>(A, grid, s);
    } else if (V <= 2048) {
        if (k <= 64) V <= 512 ? launch_small<DT, 64, 8, 1>(A, grid, s) : V <= 1024 ? launch_small<DT, 64, 16, 1>(A, grid, s) : launch_small<DT, 64, 32, 1>(A, grid, s);
        else V <= 512 ? launch_small<DT, 64, 8, 4>(A, grid, s) : V <= 1024 ? launch_small<DT, 64, 16, 4>(A, grid, s) : launch_small<DT, 64, 32, 4>(A, grid, s);
    } else hipLaunchKernelGGL((distill_row_kernel<DT, 256, 0>), dim3((unsigned)grid), dim3(256), 0, s, A);
    return grid;
}

}  // namespace
}  // namespace elg

using namespace elg;

extern "C" int64_t elg_distill_ws_bytes(int64_t R, int64_t V, int type) {
    (void)V; (void)type;
    return 8 * (R < MAX_GRID ? (R > 0 ? R : 1) : MAX_GRID);
}

extern "C" int elg_distill_loss_grad(const void* z, int64_t z_stride, int type, int64_t R, int64_t V, const void* top_values, int top_type,
                                     const void* top_idx, int idx_wide, int k, const float* tail, float temperature, const float* weight,
                                     const float* cot, int cot_stride, float scale, float* loss_rows, float* loss_total, void* grad,
                                     void* ws, int64_t ws_bytes, void* stream) {
    if (type != ELG_F32 && type != ELG_BF16 && type != ELG_F16) return fail(ELG_EINVAL, "distill: unknown element type");
    if (top_type != ELG_F32 && top_type != ELG_BF16 && top_type != ELG_F16) return fail(ELG_EINVAL, "distill: unknown type of the teacher's logits");
    if (R < 0 || V <= 0 || V > ELG_ROW_MAX_V) return fail(ELG_EINVAL, "distill: rows of 1 .. 2^24 logits");
    if (k < 1 || k > ELG_TOP_MAX_K) return fail(ELG_EINVAL, "distill: 1 <= k <= 256 teacher entries a row");
    if (!(temperature > 0.f) || temperature > 3.4e38f) return fail(ELG_EINVAL, "distill: the temperature must be positive and finite");
    if (cot_stride != 0 && cot_stride != 1) return fail(ELG_EINVAL, "distill: the cotangent is one number or one per row");
    if (!loss_rows && !loss_total && !grad) return fail(ELG_EINVAL, "distill: nothing to compute");
    if (R > 0 && (!z || !top_values || !top_idx)) return fail(ELG_EINVAL, "distill: null buffer");
    if (loss_total && (!ws || ws_bytes < elg_distill_ws_bytes(R, V, type))) return fail(ELG_EINVAL, "distill: loss_total needs elg_distill_ws_bytes() of scratch");
    if (R == 0 && !loss_total) return ELG_OK;
    const int es = type == ELG_F32 ? 4 : 2;
    if (((uintptr_t)z | (uintptr_t)grad) % es || (uintptr_t)top_values % (top_type == ELG_F32 ? 4 : 2) || (uintptr_t)top_idx % (idx_wide ? 8 : 4) || (uintptr_t)ws % 8)
        return fail(ELG_EINVAL, "distill: misaligned buffer");
    DistillArgs A;
    A.z = (const char*)z; A.z_stride = z_stride * es; A.R = R; A.V = (int)V; A.k = k;
    A.tv = top_values; A.ti = top_idx; A.tv_type = top_type; A.ti_wide = idx_wide != 0;
    A.tail = tail; A.weight = weight; A.cot = cot; A.cot_stride = cot_stride;
    A.tau = temperature; A.c2 = LOG2E / temperature; A.scale = scale;
    A.loss_rows = loss_rows; A.part = loss_total ? (double*)ws : nullptr;
    A.grad = (char*)grad; A.g_stride = V * es;
    (void)hipGetLastError();
    int G = 0;
    if (R > 0) {
        hipStream_t st = (hipStream_t)stream;
        G = type == ELG_F32 ? launch<ELG_F32>(A, st) : type == ELG_BF16 ? launch<ELG_BF16>(A, st) : launch<ELG_F16>(A, st);
    }
    if (loss_total) hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, (const double*)ws, G, scale, loss_total);
    return launch_status("distill");
}
