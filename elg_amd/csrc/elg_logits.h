// Shared device helpers of the row operators over node logits and probabilities (elg_topk.hip, elg_distill.hip, elg_verify.hip).
//
// A row of V elements is walked in 16-byte chunks of the ALIGNED address range around it: `shift` elements in front of the row share its
// first 16-byte line, element n sits at window position n + shift, chunk c holds positions c * VEC ... + VEC - 1.  Rows of odd length
// (101 nodes: the rows of a rollout) start at any element alignment, and every chunk but a row's first and last is still one wide load.
#pragma once
#include "elg_common.h"
#include "../../include/elg_hip.h"
#include <string>

namespace elg {
int fail(int code, const std::string& msg);
int launch_status(const char* what);

// Workgroups of 256 threads that one launch can have: its threads are counted in 32 bits, and beyond them the grid wraps without an error.
constexpr long long LAUNCH_WG = 0xFFFFFFFFLL / 256;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int DT> struct ElemOf;
template <> struct ElemOf<ELG_F32> { using T = float; };
template <> struct ElemOf<ELG_BF16> { using T = __bf16; };
template <> struct ElemOf<ELG_F16> { using T = _Float16; };
template <int DT> using elem_t = typename ElemOf<DT>::T;
template <int DT> constexpr int VEC = 16 / (int)sizeof(elem_t<DT>);       // elements of a chunk

template <int DT>
__device__ __forceinline__ float elem(const void* base, long long i) {
    return (float)reinterpret_cast<const elem_t<DT>*>(base)[i];
}
// the same with the type known at run time only (the few entries of a teacher's row)
__device__ __forceinline__ float elem_any(const void* base, long long i, int type) {
    return type == ELG_F32 ? elem<ELG_F32>(base, i) : type == ELG_BF16 ? elem<ELG_BF16>(base, i) : elem<ELG_F16>(base, i);
}
__device__ __forceinline__ long long index_any(const void* base, long long i, int wide) {
    return wide ? reinterpret_cast<const long long*>(base)[i] : (long long)reinterpret_cast<const int*>(base)[i];
}

template <int DT>
__device__ __forceinline__ void unpack(const u32x4 r, float (&v)[VEC<DT>]) {
    if constexpr (DT == ELG_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i2f((int)r[i]);
    } else if constexpr (DT == ELG_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = i2f((int)(r[i] << 16));
            v[2 * i + 1] = i2f((int)(r[i] & 0xFFFF0000u));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned u = r[i];      // a scalar of its own: the bit cast of a vector's element would read element 0
            const f16x2 h = __builtin_bit_cast(f16x2, u);
            v[2 * i] = (float)h[0];
            v[2 * i + 1] = (float)h[1];
        }
    }
}
// round to nearest even, once
template <int DT>
__device__ __forceinline__ u32x4 pack(const float (&v)[VEC<DT>]) {
    u32x4 r;
    if constexpr (DT == ELG_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = (unsigned)f2i(v[i]);
    } else if constexpr (DT == ELG_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(unsigned, bf16x2{(__bf16)v[2 * i], (__bf16)v[2 * i + 1]});
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(unsigned, f16x2{(_Float16)v[2 * i], (_Float16)v[2 * i + 1]});
    }
    return r;
}

template <int DT>
__device__ __forceinline__ int shift_of(const void* row) {
    return (int)((uintptr_t)row & 15) / (int)sizeof(elem_t<DT>);
}
// chunk c of a row, as stored; positions outside the row read as `pad` (the bits of one element, repeated)
template <int DT>
__device__ __forceinline__ u32x4 load_chunk(const void* row, int shift, int V, int c, unsigned pad) {
    const int n0 = c * VEC<DT> - shift;
    const elem_t<DT>* p = reinterpret_cast<const elem_t<DT>*>(row);
    if (n0 >= 0 && n0 + VEC<DT> <= V) return *reinterpret_cast<const u32x4*>(p + n0);
    u32x4 r = {pad, pad, pad, pad};
#pragma unroll
    for (int e = 0; e < VEC<DT>; ++e) {
        const int n = n0 + e;
        if (n >= 0 && n < V) {
            if constexpr (DT == ELG_F32) r[e] = reinterpret_cast<const unsigned*>(row)[n];
            else {
                const unsigned h = reinterpret_cast<const unsigned short*>(row)[n];
                r[e >> 1] = (e & 1) ? (r[e >> 1] & 0x0000FFFFu) | (h << 16) : (r[e >> 1] & 0xFFFF0000u) | h;
            }
        }
    }
    return r;
}
// the bits of -inf, as load_chunk's pad
template <int DT> constexpr unsigned PAD_NEG_INF = DT == ELG_F32 ? 0xFF800000u : DT == ELG_BF16 ? 0xFF80FF80u : 0xFC00FC00u;

// The same row as whole chunks [c_lo, c_hi) and the few elements in front of and behind them: loops over whole chunks need no per-chunk
// case distinction, and thread t < 2 VEC takes the single element edge(t) besides.  For rows of at least 2 VEC elements.
template <int DT>
struct Span {
    const char* base;                     // 16-byte aligned; chunk c is at base + 16 c
    int shift, c_lo, c_hi, V;
    __device__ __forceinline__ Span(const void* row, int V_) : V(V_) {
        shift = shift_of<DT>(row);
        base = reinterpret_cast<const char*>(row) - ((uintptr_t)row & 15);
        c_lo = shift ? 1 : 0;
        c_hi = (shift + V) / VEC<DT>;
    }
    __device__ __forceinline__ int edge(int t) const {
        const int head = shift ? VEC<DT> - shift : 0, tail = c_hi * VEC<DT> - shift;
        const int n = t < head ? t : tail + t - head;
        return n < V && t < 2 * VEC<DT> ? n : -1;
    }
    // the thread whose edge element is n (n outside the whole chunks)
    __device__ __forceinline__ int edge_slot(int n) const {
        const int head = shift ? VEC<DT> - shift : 0;
        return n < head ? n : head + n - (c_hi * VEC<DT> - shift);
    }
    __device__ __forceinline__ u32x4 chunk(int c) const { return *reinterpret_cast<const u32x4*>(base + 16u * (unsigned)c); }
};

// block-wide sums: one LDS exchange and one barrier; `slot` alternates between two buffers so that a wave may enter the next
// reduction while another still reads this one.  Every thread gets the result, added in wave order (the same bits in every run).
template <int W>
struct BlockRed {
    float* buf;              // 2 * 2 * W floats of LDS
    int flip = 0;
    __device__ explicit BlockRed(float* b) : buf(b) {}
    __device__ __forceinline__ float2 sum2(float a, float b) {
        a = wave_sum(a);
        b = wave_sum(b);
        float* s = buf + flip * 2 * W;
        flip ^= 1;
        if ((threadIdx.x & 63) == 0) { s[2 * (threadIdx.x >> 6)] = a; s[2 * (threadIdx.x >> 6) + 1] = b; }
        __syncthreads();
        float2 r = make_float2(s[0], s[1]);
#pragma unroll
        for (int w = 1; w < W; ++w) { r.x += s[2 * w]; r.y += s[2 * w + 1]; }
        return r;
    }
};

constexpr float LOG2E = 1.4426950408889634f;
// exp2 of a difference that is <= 0 where it matters; v_exp_f32 is 1 ulp
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// Order-preserving key of a float: larger value, larger key; -0 = +0; every NaN above +inf.
constexpr unsigned KEY_NEG_INF = 0x007FFFFFu;
__device__ __forceinline__ unsigned order_key(float f) {
    const int u = f2i(f + 0.0f);                                        // -0 + 0 = +0
    return f != f ? 0xFFFFFFFFu : (unsigned)(u ^ ((u >> 31) | (int)0x80000000));
}
__device__ __forceinline__ float key_value(unsigned k) {               // (the NaN key gives back a NaN)
    return i2f((int)k ^ ((~(int)k >> 31) | (int)0x80000000));
}
}  // namespace elg
