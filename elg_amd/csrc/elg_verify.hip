// Verification of drafted choices against the target policy's probabilities, from given uniforms (elg_verify_draft).
//
// Draft i of a sequence is accepted while  u_i q_i(x_i) < p_i(x_i);  the first refusal replaces it by a draw from the positive part of
// p - q (so that accepted and replaced choices together are distributed as the target), an unrefused draft is followed by a draw from
// the target's next row.  A draw is  the first n with  cumsum(r)_n > u sum(r).
//
// Every product, sum and comparison is in 64 bits: products of two f32 are exact there, and a draw near a border depends on the order of
// the additions only in the last of 53 bits.
#include "elg_logits.h"

namespace elg {
namespace {

struct VerifyArgs {
    const char *p, *q;
    long long pb, ps, qb, qs;             // bytes: per sequence, per step
    const void* tok;
    int tok_wide;
    long long tok_stride;                 // elements
    const float* u;
    long long u_stride;
    const int* lengths;
    int G, V;
    int* out;
    int* accepted;
};

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}
__device__ __forceinline__ double wave_scan_d(double v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

// accepted drafts of sequence b, the same for every lane of the wave that calls it
template <int DT>
__device__ __forceinline__ int accept_prefix(const VerifyArgs& A, long long b, int lane, int n) {
    int a = 0;
    for (int i0 = 0; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        bool ok = false;
        if (i < n) {
            const long long x = index_any(A.tok, b * A.tok_stride + i, A.tok_wide);
            if (x >= 0 && x < A.V) {
                const double px = (double)elem<DT>(A.p + b * A.pb + i * A.ps, x);
                const double qx = A.q ? (double)elem<DT>(A.q + b * A.qb + i * A.qs, x) : 1.0;
                ok = (double)A.u[b * A.u_stride + i] * qx < px;
            }
        }
        const unsigned long long m = __ballot(ok);
        const int run = ~m ? __ffsll((long long)~m) - 1 : 64;
        a += run;
        if (run < 64) break;
    }
    return min(a, n);
}

// What is drawn from: the target's row, less the draft's row where there is one, or less the refused choice alone.
template <int DT>
struct Residual {
    const char *p, *q;
    int ban;                              // without a draft row: the choice that was refused
    int V, shift;
    __device__ __forceinline__ void chunk(int c, double (&r)[VEC<DT>]) const {
        float a[VEC<DT>];
        unpack<DT>(load_chunk<DT>(p, shift, V, c, 0u), a);
        if (q) {
            const elem_t<DT>* qq = reinterpret_cast<const elem_t<DT>*>(q);
            const int n0 = c * VEC<DT> - shift;
            float s[VEC<DT>] = {};
            if (n0 >= 0 && n0 + VEC<DT> <= V && !((uintptr_t)(qq + n0) & 15)) unpack<DT>(*reinterpret_cast<const u32x4*>(qq + n0), s);
            else {
#pragma unroll
                for (int e = 0; e < VEC<DT>; ++e)
                    if (n0 + e >= 0 && n0 + e < V) s[e] = (float)qq[n0 + e];
            }
#pragma unroll
            for (int e = 0; e < VEC<DT>; ++e) {
                const double d = (double)a[e] - (double)s[e];
                r[e] = d > 0.0 ? d : 0.0;
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC<DT>; ++e) r[e] = a[e] > 0.f && c * VEC<DT> + e - shift != ban ? (double)a[e] : 0.0;
        }
    }
};

// One workgroup per sequence.  A wave sums a contiguous part of the row; the wave in whose part the draw falls walks it again.
template <int DT, int T>
__global__ __launch_bounds__(T) void verify_kernel(const VerifyArgs A) {
    constexpr int W = T / 64;
    __shared__ double wsum[W];
    __shared__ int sh_a, sh_n;
    const long long b = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = A.lengths ? min(max(A.lengths[b], 0), A.G) : A.G;
    if (wave == 0) {
        const int a = accept_prefix<DT>(A, b, lane, n);
        if (lane == 0) { sh_a = a; sh_n = -1; }
    }
    __syncthreads();
    const int a = sh_a;
    Residual<DT> R;
    R.p = A.p + b * A.pb + a * A.ps;
    R.q = a < n && A.q ? A.q + b * A.qb + a * A.qs : nullptr;
    R.ban = a < n && !A.q ? (int)max(-1LL, min((long long)A.V, index_any(A.tok, b * A.tok_stride + a, A.tok_wide))) : -1;
    R.V = A.V;
    R.shift = shift_of<DT>(R.p);
    const int nch = (R.shift + A.V + VEC<DT> - 1) / VEC<DT>;
    const int per = (nch + W - 1) / W, c_lo = min(wave * per, nch), c_hi = min(c_lo + per, nch);
    double total = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        double s = 0.0;
        for (int c = c_lo + lane; c < c_hi; c += 64) {
            double r[VEC<DT>];
            R.chunk(c, r);
#pragma unroll
            for (int e = 0; e < VEC<DT>; ++e) s += r[e];
        }
        s = wave_sum_d(s);
        __syncthreads();
        if (lane == 0) wsum[wave] = s;
        __syncthreads();
        total = 0.0;
        for (int w = 0; w < W; ++w) total += wsum[w];
        if (total > 0.0 || (!R.q && R.ban < 0)) break;
        R.q = nullptr;                    // nothing of the target is left over the draft: its own row
        R.ban = -1;
    }
    if (total > 0.0) {
        const double t = (double)A.u[b * A.u_stride + A.G] * total;
        // the first wave whose part passes t; if rounding leaves none, the last one that holds anything
        int own = -1;
        double before = 0.0, acc = 0.0;
        for (int w = 0; w < W; ++w) {
            if (wsum[w] > 0.0) {
                own = w;
                before = acc;
                if (acc + wsum[w] > t) break;
            }
            acc += wsum[w];
        }
        if (wave == own) {
            int pick = -1;
            for (int c0 = c_lo; c0 < c_hi; c0 += 64) {
                const int c = c0 + lane;
                double r[VEC<DT>], s = 0.0;
                if (c < c_hi) {
                    R.chunk(c, r);
#pragma unroll
                    for (int e = 0; e < VEC<DT>; ++e) s += r[e];
                }
                const double incl = wave_scan_d(s, lane);
                const unsigned long long some = __ballot(s > 0.0), over = __ballot(s > 0.0 && before + incl > t);
                if (some) {               // the lane that passes t, else (for the case that no later one does) the last that holds anything
                    const int src = over ? __ffsll((long long)over) - 1 : 63 - __clzll((long long)some);
                    int n_mine = -1;
                    if (lane == src) {
                        double cum = before + (incl - s);
#pragma unroll
                        for (int e = 0; e < VEC<DT>; ++e) {
                            if (r[e] > 0.0 && !(n_mine >= 0 && cum > t)) n_mine = c * VEC<DT> + e - R.shift;
                            cum += r[e];
                        }
                    }
                    pick = __shfl(n_mine, src, 64);
                    if (over) break;
                }
                before += __shfl(incl, 63, 64);
            }
            if (lane == 0) sh_n = pick;
        }
    }
    __syncthreads();
    const int drawn = sh_n;
    for (int i = tid; i <= A.G; i += T)
        A.out[b * (A.G + 1) + i] = i < a ? (int)index_any(A.tok, b * A.tok_stride + i, A.tok_wide) : i == a ? drawn : -1;
    if (tid == 0) A.accepted[b] = a;
}

}  // namespace
}  // namespace elg

using namespace elg;

extern "C" int elg_verify_draft(const void* target, int64_t target_bstride, int64_t target_sstride, const void* draft, int64_t draft_bstride,
                                int64_t draft_sstride, int type, const void* tokens, int tokens_wide, int64_t tokens_stride,
                                const float* uniforms, int64_t uniforms_stride, const int32_t* lengths, int64_t B, int G, int64_t V,
                                int32_t* out_tokens, int32_t* accepted, void* stream) {
    if (type != ELG_F32 && type != ELG_BF16 && type != ELG_F16) return fail(ELG_EINVAL, "verify_draft: unknown element type");
    if (B < 0 || B > 0x7FFFFFFF || G < 0 || G > ELG_DRAFT_MAX || V <= 0 || V > ELG_ROW_MAX_V)
        return fail(ELG_EINVAL, "verify_draft: up to 1024 drafts a sequence over rows of 1 .. 2^24 probabilities");
    if (B == 0) return ELG_OK;
    if (!target || (G > 0 && !tokens) || !uniforms || !out_tokens || !accepted) return fail(ELG_EINVAL, "verify_draft: null buffer");
    const int es = type == ELG_F32 ? 4 : 2;
    if (((uintptr_t)target | (uintptr_t)draft) % es || (uintptr_t)tokens % (tokens_wide ? 8 : 4)) return fail(ELG_EINVAL, "verify_draft: misaligned buffer");
    VerifyArgs A;
    A.p = (const char*)target; A.q = (const char*)draft;
    A.pb = target_bstride * es; A.ps = target_sstride * es; A.qb = draft_bstride * es; A.qs = draft_sstride * es;
    A.tok = tokens; A.tok_wide = tokens_wide != 0; A.tok_stride = tokens_stride;
    A.u = uniforms; A.u_stride = uniforms_stride; A.lengths = lengths;
    A.G = G; A.V = (int)V; A.out = out_tokens; A.accepted = accepted;
    (void)hipGetLastError();
    const dim3 grid((unsigned)B);
    if (type == ELG_F32) hipLaunchKernelGGL((verify_kernel<ELG_F32, 256>), grid, dim3(256), 0, (hipStream_t)stream, A);
    else if (type == ELG_BF16) hipLaunchKernelGGL((verify_kernel<ELG_BF16, 256>), grid, dim3(256), 0, (hipStream_t)stream, A);
    else hipLaunchKernelGGL((verify_kernel<ELG_F16, 256>), grid, dim3(256), 0, (hipStream_t)stream, A);
    return launch_status("verify_draft");
}
