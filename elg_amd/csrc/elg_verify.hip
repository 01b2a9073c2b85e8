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

template <int DT>
__device__ __forceinline__ Residual<DT> residual_of(const VerifyArgs& A, long long b, int a, int n) {
    Residual<DT> R;
    R.p = A.p + b * A.pb + a * A.ps;
    R.q = a < n && A.q ? A.q + b * A.qb + a * A.qs : nullptr;
    R.ban = a < n && !A.q ? (int)max(-1LL, min((long long)A.V, index_any(A.tok, b * A.tok_stride + a, A.tok_wide))) : -1;
    R.V = A.V;
    R.shift = shift_of<DT>(R.p);
    return R;
}

__device__ __forceinline__ int drafts_of(const VerifyArgs& A, long long b) { return A.lengths ? min(max(A.lengths[b], 0), A.G) : A.G; }

__device__ __forceinline__ void answer(const VerifyArgs& A, long long b, int a, int drawn, int t, int step) {
    for (int i = t; i <= A.G; i += step)
        A.out[b * (A.G + 1) + i] = i < a ? (int)index_any(A.tok, b * A.tok_stride + i, A.tok_wide) : i == a ? drawn : -1;
    if (t == 0) A.accepted[b] = a;
}

// One wave: the element among the lanes' runs (lane order, N to a lane) where the running sum from `before` passes t; where rounding lets none
// pass, the last one that holds anything; -1 if none does.  The same in every lane.  N elements of lane l sit at node l_first + e.
template <int N>
__device__ __forceinline__ int pick_in_wave(const double (&r)[N], double before, double t, int first_node, int lane, bool& passed) {
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < N; ++e) s += r[e];
    const double incl = wave_scan_d(s, lane);
    const unsigned long long some = __ballot(s > 0.0), over = __ballot(s > 0.0 && before + incl > t);
    passed = over != 0ull;
    if (!some) return -1;
    const int src = over ? __ffsll((long long)over) - 1 : 63 - __clzll((long long)some);
    int mine = -1;
    double cum = before + (incl - s);
#pragma unroll
    for (int e = 0; e < N; ++e) {
        if (r[e] > 0.0 && !(mine >= 0 && cum > t)) mine = first_node + e;
        cum += r[e];
    }
    return __shfl(mine, src, 64);
}

// Rows of up to 64 NE probabilities: a wave to a sequence, lane l holding the nodes i 64 + l.  The sum of each run of 64 is formed once; only
// the run in which the draw falls is scanned.
// 6400 sequences of 8 drafts over 101 nodes: 7.4 us; one step of 100 sequences 4.4 us, a launch with a chain of four dependent reads in it.
template <int DT, int NE>
__global__ __launch_bounds__(256) void verify_wave_kernel(const VerifyArgs A, long long B) {
    const int lane = threadIdx.x & 63;
    const long long b = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b >= B) return;
    const int n = drafts_of(A, b), a = accept_prefix<DT>(A, b, lane, n);
    const Residual<DT> R = residual_of<DT>(A, b, a, n);
    double p[NE], r[NE], sum[NE], total = 0.0;
    float pv[NE], qv[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        pv[i] = i * 64 + lane < A.V ? elem<DT>(R.p, i * 64 + lane) : 0.f;
        qv[i] = R.q && i * 64 + lane < A.V ? elem<DT>(R.q, i * 64 + lane) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        p[i] = pv[i] > 0.f ? (double)pv[i] : 0.0;
        const double d = (double)pv[i] - (double)qv[i];
        r[i] = R.q ? (d > 0.0 ? d : 0.0) : i * 64 + lane == R.ban ? 0.0 : p[i];
        sum[i] = wave_sum_d(r[i]);
        total += sum[i];
    }
    if (!(total > 0.0)) {                 // nothing of the target is left over the draft: its own row
        total = 0.0;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            r[i] = p[i];
            sum[i] = wave_sum_d(p[i]);
            total += sum[i];
        }
    }
    int drawn = -1;
    if (total > 0.0) {
        const double t = (double)A.u[b * (A.u_stride) + A.G] * total;
        double before = 0.0;
        bool passed = false;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            if (!passed && sum[i] > 0.0) {
                const double one[1] = {r[i]};
                // (the last run that holds anything is scanned too if none passes)
                bool last = true;
#pragma unroll
                for (int j = i + 1; j < NE; ++j) last = last && !(sum[j] > 0.0);
                if (last || before + sum[i] > t) {
                    const int at = pick_in_wave<1>(one, before, t, i * 64 + lane, lane, passed);
                    if (at >= 0) drawn = at;
                }
            }
            before += sum[i];
        }
    }
    answer(A, b, a, drawn, lane, 64);
}

// Longer rows, in segments of RUNS runs of 64 chunks, four runs to a wave of a workgroup.
// 48 sequences over 131072 probabilities in bf16 (25 MB of two rows each): 12 us for the segments' sums, 10 us for the pick, where the bytes take
// 5.3.  The sums convert every probability to 64 bits; the pick waits for the acceptance, the segments, a segment and a run, one after the other.
constexpr int RUNS = 16;

// the sums of a segment's runs, of what is drawn from (x) and of the target's own row (y), into LDS
template <int DT>
__device__ __forceinline__ void run_sums(const Residual<DT>& R, int c0, int nch, double2* sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Residual<DT> own = R;
    own.q = nullptr;
    own.ban = -1;
#pragma unroll
    for (int i = 0; i < RUNS / 4; ++i) {
        const int run = wave * (RUNS / 4) + i, c = c0 + run * 64 + lane;
        double s = 0.0, so = 0.0;
        if (c < nch) {
            double r[VEC<DT>];
            R.chunk(c, r);
#pragma unroll
            for (int e = 0; e < VEC<DT>; ++e) s += r[e];
            own.chunk(c, r);
#pragma unroll
            for (int e = 0; e < VEC<DT>; ++e) so += r[e];
        }
        s = wave_sum_d(s);
        so = wave_sum_d(so);
        if (lane == 0) sums[run] = make_double2(s, so);
    }
}
// The draw within a segment, by the first wave: the run the sum passes t in (or the last that holds anything), then the chunk, then the node.
template <int DT>
__device__ __forceinline__ int pick_in_segment(Residual<DT> R, int c0, int nch, const double2* sums, bool own, double before, double t) {
    const int lane = threadIdx.x & 63;
    if (own) { R.q = nullptr; R.ban = -1; }
    int run = -1;
    double at = before, acc = before;
    for (int i = 0; i < RUNS; ++i) {
        const double s = own ? sums[i].y : sums[i].x;
        if (s > 0.0) {
            run = i;
            at = acc;
            if (acc + s > t) break;
        }
        acc += s;
    }
    if (run < 0) return -1;
    const int c = c0 + run * 64 + lane;
    double r[VEC<DT>] = {};
    if (c < nch) R.chunk(c, r);
    bool passed;
    return pick_in_wave<VEC<DT>>(r, at, t, c * VEC<DT> - R.shift, lane, passed);
}

// a row of one segment: one workgroup, one launch
template <int DT>
__global__ __launch_bounds__(256) void verify_row_kernel(const VerifyArgs A) {
    __shared__ double2 sums[RUNS];
    __shared__ int sh_a;
    const long long b = blockIdx.x;
    const int tid = threadIdx.x, n = drafts_of(A, b);
    if (tid < 64) {
        const int a = accept_prefix<DT>(A, b, tid, n);
        if (tid == 0) sh_a = a;
    }
    __syncthreads();
    const int a = sh_a;
    const Residual<DT> R = residual_of<DT>(A, b, a, n);
    const int nch = (R.shift + A.V + VEC<DT> - 1) / VEC<DT>;
    run_sums<DT>(R, 0, nch, sums);
    __syncthreads();
    if (tid >= 64) return;
    double total = 0.0, own = 0.0;
    for (int i = 0; i < RUNS; ++i) { total += sums[i].x; own += sums[i].y; }
    const bool fallback = !(total > 0.0);
    total = fallback ? own : total;
    int drawn = -1;
    if (total > 0.0) drawn = pick_in_segment<DT>(R, 0, nch, sums, fallback, 0.0, (double)A.u[b * A.u_stride + A.G] * total);
    answer(A, b, a, drawn, tid, 64);
}

// a row of several segments: their sums first, a workgroup each, then the draw
template <int DT>
__global__ __launch_bounds__(256) void verify_part_kernel(const VerifyArgs A, double2* __restrict__ parts, int segs) {
    __shared__ double2 sums[RUNS];
    __shared__ int sh_a;
    const long long b = blockIdx.x / segs;
    const int seg = (int)(blockIdx.x - b * segs), tid = threadIdx.x, n = drafts_of(A, b);
    if (tid < 64) {
        const int a = accept_prefix<DT>(A, b, tid, n);
        if (tid == 0) {
            sh_a = a;
            if (seg == 0) A.accepted[b] = a;
        }
    }
    __syncthreads();
    const Residual<DT> R = residual_of<DT>(A, b, sh_a, n);
    run_sums<DT>(R, seg * RUNS * 64, (R.shift + A.V + VEC<DT> - 1) / VEC<DT>, sums);
    __syncthreads();
    if (tid == 0) {
        double2 s = make_double2(0.0, 0.0);
        for (int i = 0; i < RUNS; ++i) { s.x += sums[i].x; s.y += sums[i].y; }
        parts[blockIdx.x] = s;
    }
}
template <int DT>
__global__ __launch_bounds__(256) void verify_pick_kernel(const VerifyArgs A, const double2* __restrict__ parts, int segs) {
    __shared__ double2 sums[RUNS];
    const long long b = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, n = drafts_of(A, b), a = A.accepted[b];
    const Residual<DT> R = residual_of<DT>(A, b, a, n);
    const double2* part = parts + b * segs;
    // every wave finds the segment: totals first, then the first one that the draw passes (or the last that holds anything)
    double total = 0.0, own = 0.0;
    for (int i = lane; i < segs; i += 64) { total += part[i].x; own += part[i].y; }
    total = wave_sum_d(total);
    own = wave_sum_d(own);
    const bool fallback = !(total > 0.0);
    total = fallback ? own : total;
    int seg = -1;
    double t = 0.0, before = 0.0, acc = 0.0;
    if (total > 0.0) {
        t = (double)A.u[b * A.u_stride + A.G] * total;
        bool passed = false;
        for (int i0 = 0; i0 < segs && !passed; i0 += 64) {
            const double s = i0 + lane < segs ? (fallback ? part[i0 + lane].y : part[i0 + lane].x) : 0.0;
            const double incl = wave_scan_d(s, lane);
            const unsigned long long some = __ballot(s > 0.0), over = __ballot(s > 0.0 && acc + incl > t);
            passed = over != 0ull;
            if (some) {
                const int src = over ? __ffsll((long long)over) - 1 : 63 - __clzll((long long)some);
                seg = i0 + src;
                before = __shfl(acc + (incl - s), src, 64);
            }
            acc += __shfl(incl, 63, 64);
        }
    }
    int drawn = -1;
    if (seg >= 0) {
        const int nch = (R.shift + A.V + VEC<DT> - 1) / VEC<DT>;
        run_sums<DT>(R, seg * RUNS * 64, nch, sums);
        __syncthreads();
        if (tid < 64) drawn = pick_in_segment<DT>(R, seg * RUNS * 64, nch, sums, fallback, before, t);
    }
    if (tid < 64) answer(A, b, a, drawn, tid, 64);
}

// segments of the longest row that V probabilities can make (a row may start inside its first 16 bytes)
int segments(int64_t V, int type) {
    const int vec = type == ELG_F32 ? 4 : 8;
    return (int)(((V + 2 * vec - 2) / vec + RUNS * 64 - 1) / (RUNS * 64));
}

template <int DT>
void launch_part(const VerifyArgs& A, long long B, int segs, double2* parts, hipStream_t s) {
    const dim3 waves((unsigned)((B + 3) / 4)), all((unsigned)B);
    if (A.V <= 128) hipLaunchKernelGGL((verify_wave_kernel<DT, 2>), waves, dim3(256), 0, s, A, B);
    else if (A.V <= 512) hipLaunchKernelGGL((verify_wave_kernel<DT, 8>), waves, dim3(256), 0, s, A, B);
    else if (A.V <= 1024) hipLaunchKernelGGL((verify_wave_kernel<DT, 16>), waves, dim3(256), 0, s, A, B);
    else if (segs == 1) hipLaunchKernelGGL((verify_row_kernel<DT>), all, dim3(256), 0, s, A);
    else {
        hipLaunchKernelGGL((verify_part_kernel<DT>), dim3((unsigned)(B * segs)), dim3(256), 0, s, A, parts, segs);
        hipLaunchKernelGGL((verify_pick_kernel<DT>), all, dim3(256), 0, s, A, (const double2*)parts, segs);
    }
}
// As many sequences at a time as a launch has workgroups for.  A wave a sequence up to 1024 probabilities, a workgroup beyond: 4000 sequences of 4
// drafts in f32 take 5.1 us by waves and 22.2 by workgroups over 101 probabilities, 11.7 / 22.5 over 400, 25.8 / 23.4 over 700, 29.9 / 24.1 over
// 1024 (100 sequences: 3.9 / 6.3, 6.4 / 5.7, 9.3 / 6.0, 10.1 / 6.4).
template <int DT>
void launch(const VerifyArgs& A, long long B, double2* parts, hipStream_t s) {
    const int segs = segments(A.V, DT);
    const long long at_once = A.V <= 1024 ? 4 * LAUNCH_WG : LAUNCH_WG / segs;
    for (long long b = 0; b < B; b += at_once) {
        VerifyArgs C = A;
        C.p += b * A.pb;
        if (A.q) C.q += b * A.qb;
        C.tok = (const char*)A.tok + b * A.tok_stride * (A.tok_wide ? 8 : 4);
        C.u += b * A.u_stride;
        if (A.lengths) C.lengths += b;
        C.out += b * (A.G + 1);
        C.accepted += b;
        launch_part<DT>(C, B - b < at_once ? B - b : at_once, segs, parts, s);         // (parts: read before the next ones are written)
    }
}

}  // namespace
}  // namespace elg

using namespace elg;

extern "C" int64_t elg_verify_ws_bytes(int64_t B, int64_t V, int type) {
    if (B <= 0 || V <= 1024 || V > ELG_ROW_MAX_V) return 0;
    const int segs = segments(V, type);
    return segs > 1 ? 16 * B * segs : 0;
}

extern "C" int elg_verify_draft(const void* target, int64_t target_bstride, int64_t target_sstride, const void* draft, int64_t draft_bstride,
                                int64_t draft_sstride, int type, const void* tokens, int tokens_wide, int64_t tokens_stride,
                                const float* uniforms, int64_t uniforms_stride, const int32_t* lengths, int64_t B, int G, int64_t V,
                                int32_t* out_tokens, int32_t* accepted, void* ws, int64_t ws_bytes, void* stream) {
    if (type != ELG_F32 && type != ELG_BF16 && type != ELG_F16) return fail(ELG_EINVAL, "verify_draft: unknown element type");
    if (B < 0 || B > 0x7FFFFFFF || G < 0 || G > ELG_DRAFT_MAX || V <= 0 || V > ELG_ROW_MAX_V)
        return fail(ELG_EINVAL, "verify_draft: up to 1024 drafts a sequence over rows of 1 .. 2^24 probabilities");
    if (B == 0) return ELG_OK;
    if (!target || (G > 0 && !tokens) || !uniforms || !out_tokens || !accepted) return fail(ELG_EINVAL, "verify_draft: null buffer");
    const int es = type == ELG_F32 ? 4 : 2;
    if (((uintptr_t)target | (uintptr_t)draft) % es || (uintptr_t)tokens % (tokens_wide ? 8 : 4)) return fail(ELG_EINVAL, "verify_draft: misaligned buffer");
    const int64_t need = elg_verify_ws_bytes(B, V, type);
    if (need > 0 && (!ws || ws_bytes < need || (uintptr_t)ws % 16)) return fail(ELG_EINVAL, "verify_draft: needs elg_verify_ws_bytes() of scratch");
    VerifyArgs A;
    A.p = (const char*)target; A.q = (const char*)draft;
    A.pb = target_bstride * es; A.ps = target_sstride * es; A.qb = draft_bstride * es; A.qs = draft_sstride * es;
    A.tok = tokens; A.tok_wide = tokens_wide != 0; A.tok_stride = tokens_stride;
    A.u = uniforms; A.u_stride = uniforms_stride; A.lengths = lengths;
    A.G = G; A.V = (int)V; A.out = out_tokens; A.accepted = accepted;
    (void)hipGetLastError();
    double2* parts = reinterpret_cast<double2*>(ws);
    hipStream_t st = (hipStream_t)stream;
    type == ELG_F32 ? launch<ELG_F32>(A, B, parts, st) : type == ELG_BF16 ? launch<ELG_BF16>(A, B, parts, st) : launch<ELG_F16>(A, B, parts, st);
    return launch_status("verify_draft");
}
