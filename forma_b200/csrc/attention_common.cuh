// Pieces that the tensor-core attention kernels share: softmax arithmetic on
// score rows, TMEM stores, the warp-level MMA with its cp.async rings, and the
// host side's tensor-map entry point and row layouts.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "async.cuh"
#include "device_common.cuh"
#include "kernels.h"
#include "tc.cuh"

namespace fb {
namespace {

constexpr int TQ = 128, TK = 128;  // query rows and keys of a tcgen05 tile

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^x for a pair of values on the FMA/ALU pipes, for a share of the softmax
// exponentials so that the transcendental unit (MUFU ex2) is not the only
// engine producing them.  Cody-Waite split x = n + f: n is the nearest
// integer, obtained by adding and subtracting 1.5 * 2^23, and |f| <= 1/2; 2^f
// comes from a degree-3 polynomial whose coefficients minimise the maximum
// relative error on [-1/2, 1/2] (a linear program over a dense grid; 7.5e-5,
// below the 2^-11 rounding of an F16 P and the 2^-9 of a BF16 one); n is
// added to the exponent field (the low 9 bits of t's pattern hold n mod 512).
// Inputs are clamped to -127 first; at n = -127 a polynomial value below 1
// carries its exponent field below zero, which the final max with 0 turns
// into exactly 0, so -inf (a masked score) gives 0 and a fully masked row
// keeps a zero sum.  A NaN passes the clamp and comes back with 0 x at the end
// (the integer steps lose it; a finite x adds nothing there).  The f32x2 forms
// process both values in one instruction.
__device__ __forceinline__ float max2_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float2 ex2_poly2(float2 x) {
    const float2 M = make_float2(12582912.0f, 12582912.0f);
    const float2 xc = make_float2(max2_nan(x.x, -127.0f), max2_nan(x.y, -127.0f));
    const float2 t = __fadd2_rn(xc, M);
    const float2 n = __fadd2_rn(t, make_float2(-12582912.0f, -12582912.0f));
    const float2 f = __ffma2_rn(n, make_float2(-1.0f, -1.0f), xc);  // exact: xc - n
    float2 q = __ffma2_rn(make_float2(0.0551716685295105f, 0.0551716685295105f), f,
                          make_float2(0.2426111251115799f, 0.2426111251115799f));
    q = __ffma2_rn(q, f, make_float2(0.6932609677314758f, 0.6932609677314758f));
    q = __ffma2_rn(q, f, make_float2(0.9999280571937561f, 0.9999280571937561f));
    const int bx = (int)(__float_as_uint(q.x) + (__float_as_uint(t.x) << 23));
    const int by = (int)(__float_as_uint(q.y) + (__float_as_uint(t.y) << 23));
    return __ffma2_rn(xc, make_float2(0.0f, 0.0f), make_float2(__int_as_float(max(bx, 0)), __int_as_float(max(by, 0))));
}

// Three-input extremes.  A NaN score is skipped by the row maximum but its
// exponential is NaN, which makes the row's sum and every output of the row
// NaN, as an elementwise max/exp/sum over the row would (measured: the
// NaN-propagating form costs ~1% of the kernel and changes no result).
__device__ __forceinline__ float max3n(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float min3n(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, uint32_t fmt) {
    uint32_t r;
    if (fmt)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

template <int FMT>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (FMT == 1)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int FMT>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (FMT == 1) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

constexpr int DEC_WARPS = 4;
constexpr int DEC_STAGES = 3;  // 16-key stages per warp: two in flight while one is consumed

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared-memory positions (16-byte chunks) of a stage's K and V rows: XOR
// swizzles under which every 8-lane phase of the fragment reads below touches
// eight distinct 16-byte bank groups.  K: lane (g, c) reads chunks
// c*D/32 .. of rows g and 8 + g; V: chunk(s) g*D/64 .. of rows 2c, 2c+1,
// 2c+8, 2c+9.
template <int D>
__device__ __forceinline__ uint32_t k_chunk(uint32_t row, uint32_t chunk) {
    if constexpr (D == 128) return chunk ^ (((chunk >> 3) & 1u) | ((row & 1u) << 1));
    else return chunk ^ (row & 1u);
}
__device__ __forceinline__ uint32_t v_chunk(uint32_t row, uint32_t chunk) { return chunk ^ (((row >> 1) & 3u) << 1); }

// ------------------------------------------------------------------ host

PFN_cuTensorMapEncodeTiled_v12000 encode_tiled_attn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// One operand's rows as a 4-D box source {depth, rows, heads, batch}: element
// strides of the row, head and (merged) batch axes; unit axes may have any
// stride and a stride-0 batch axis (broadcast) becomes a single batch index.
struct RowsLayout {
    uint64_t rows = 0, heads = 1, batch = 1;
    uint64_t s_row = 0, s_head = 0, s_batch = 0;
    bool batch_bcast = false;
};

// Merges the batch axes [0, nb) of the row nest into one (count, stride):
// the non-unit axes must nest row-major (stride[i] = stride[i+1] * dim[i+1])
// or all have stride 0 (broadcast).
bool merge_batch(const AttnArgs& a, const uint64_t* st, int nb, RowsLayout* o) {
    uint64_t count = 1, stride = 0;
    bool any = false, all_zero = true;
    int last = -1;
    for (int i = nb - 1; i >= 0; --i) {
        if (a.row_dims[i] == 1) continue;
        count *= a.row_dims[i];
        if (st[i] != 0) all_zero = false;
        if (!any) {
            stride = st[i];
            any = true;
        } else if (st[i] != st[last] * a.row_dims[last]) {
            if (!(st[i] == 0 && st[last] == 0)) return false;
        }
        last = i;
    }
    if (any && all_zero) {
        o->batch = 1;
        o->s_batch = 0;
        o->batch_bcast = true;
        return true;
    }
    if (any && stride == 0) return false;  // mixed broadcast and strided batch axes
    o->batch = count;
    o->s_batch = stride;
    return true;
}

}  // namespace
}  // namespace fb
