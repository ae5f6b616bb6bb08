// Log probabilities of given tokens with entropy and top alternatives, and
// their gradient for the logits.
//
// With m the row maximum, S0 = sum e^(x - m) and S1 = sum (x - m) e^(x - m):
//   lse = m + log S0,  logprob = x_t - lse,  entropy = log S0 - S1 / S0
//   d(gl * logprob + gh * entropy) / dx_v = gl ([v = t] - p_v) - gh p_v (log p_v + entropy)
// with p_v = e^(x_v - lse).
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "device_common.cuh"
#include "kernels.h"

namespace fb {
namespace {

constexpr int BLOCK = 256;

__device__ __forceinline__ uint64_t row_at(const RowOut& o, uint64_t row) { return o.offset + nest_offset(o.nest, row); }
__device__ __forceinline__ float row_value(const RowOut& o, uint64_t row) {
    return static_cast<const float*>(o.data)[row_at(o, row)];
}
__device__ __forceinline__ void row_store(const RowOut& o, uint64_t row, float v) {
    if (o.data) static_cast<float*>(o.data)[row_at(o, row)] = v;
}
__device__ __forceinline__ float row_nan() { return __int_as_float(0x7fffffff); }

// Total-order keys of the stored patterns: unsigned comparison orders them as
// IEEE's total order does the values.  They are made from integer loads: on a
// loaded float the compiler may turn the sign-bit arithmetic into fabs and
// fneg, which do not keep a NaN's sign.
template <typename T>
struct Bits {  // 16-bit patterns
    using U = uint16_t;
    static __device__ __forceinline__ uint32_t key(uint32_t b) { return (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u); }
    static __device__ __forceinline__ uint32_t pattern(uint32_t k) { return (k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu); }
    static __device__ __forceinline__ float value(uint32_t b) {
        if constexpr (std::is_same<T, __half>::value) return f16_bits_to_float((uint16_t)b);
        else return bf16_bits_to_float((uint16_t)b);
    }
};
template <>
struct Bits<float> {
    using U = uint32_t;
    static __device__ __forceinline__ uint32_t key(uint32_t b) { return (b & 0x80000000u) ? ~b : (b | 0x80000000u); }
    static __device__ __forceinline__ uint32_t pattern(uint32_t k) { return (k & 0x80000000u) ? (k & 0x7fffffffu) : ~k; }
    static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b); }
};

// log probability of target t given the row's lse
template <typename T>
__device__ __forceinline__ float target_logprob(const T* x, const Nest& inner, uint64_t cols, uint32_t t, float lse) {
    if (t == FB_NO_TOKEN) return 0.0f;
    if (t >= cols) return row_nan();
    return Elem<T>::load(x + nest_offset(inner, t)) - lse;
}

// Any layout: one block per row, the row read once for its maximum, once for
// the sums (f64) and once per alternative (the largest (value, lowest index)
// below the previous one).  Bound: L2 and latency, 2 + k passes; 256 x 50021
// f32 with a class stride of 256: 197 us, with 5 alternatives 537 us.
template <typename T>
__global__ void __launch_bounds__(BLOCK) token_rows_kernel(TokenArgs a) {
    __shared__ uint64_t keys[BLOCK / 32];
    __shared__ double sums[BLOCK / 32];
    const Rows& in = a.logits;
    for (uint64_t row = blockIdx.x; row < in.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(in.data) + in.offset + nest_offset(in.outer, row);
        // key of (value, index): larger value first, then the lower index
        auto largest_below = [&](uint64_t bound) {
            uint64_t best = 0;
            for (uint64_t c = threadIdx.x; c < in.cols; c += BLOCK) {
                const uint32_t b = __ldg(reinterpret_cast<const typename Bits<T>::U*>(x + nest_offset(in.inner, c)));
                const uint64_t k = ((uint64_t)Bits<T>::key(b) << 32) | (0xffffffffu - (uint32_t)c);
                if (k < bound && k > best) best = k;
            }
            return block_max_u64<BLOCK>(best, keys);
        };
        const uint64_t top = largest_below(~0ull);  // no index reaches 2^32 - 1, so no key is ~0
        const float m = Bits<T>::value(Bits<T>::pattern((uint32_t)(top >> 32)));
        double s0 = 0.0, s1 = 0.0;
        for (uint64_t c = threadIdx.x; c < in.cols; c += BLOCK) {
            const double z = (double)Elem<T>::load(x + nest_offset(in.inner, c)) - (double)m;
            const double e = exp(z);
            s0 += e;
            if (e > 0.0) s1 += z * e;
        }
        s0 = block_sum<BLOCK>(s0, sums);
        s1 = block_sum<BLOCK>(s1, sums);
        const double ls = log(s0);
        const float lse = (float)((double)m + ls);
        if (threadIdx.x == 0) {
            row_store(a.lse, row, lse);
            row_store(a.entropy, row, (float)(ls - s1 / s0));
            if (a.logprob.data)
                row_store(a.logprob, row,
                          target_logprob<T>(x, in.inner, in.cols, a.targets[a.target_offset + nest_offset(a.target_nest, row)], lse));
        }
        uint64_t bound = ~0ull;
        for (uint32_t k = 0; k < a.top; ++k) {
            bound = k == 0 ? top : largest_below(bound);
            if (threadIdx.x == 0) {
                a.top_index[row * a.top + k] = 0xffffffffu - (uint32_t)bound;
                a.top_logprob[row * a.top + k] = Bits<T>::value(Bits<T>::pattern((uint32_t)(bound >> 32))) - lse;
            }
        }
    }
}

// A logit that this kernel may overwrite: a plain load, not the read-only path.
template <typename T>
__device__ __forceinline__ float logit(const T* p) {
    return Bits<T>::value(*reinterpret_cast<const typename Bits<T>::U*>(p));
}

// Gradient of one logit.  A term whose coefficient is 0 is 0 whatever x is.
__device__ __forceinline__ float logit_grad(float x, float lse, float h, float gl, float gh, bool at_target) {
    const float z = x - lse, p = expf(z);
    float d = 0.0f;
    if (gl != 0.0f) d = gl * ((at_target ? 1.0f : 0.0f) - p);
    if (gh != 0.0f) d -= p > 0.0f || p != p ? gh * (p * (z + h)) : 0.0f;
    return d;
}

// Any layout: chunks of rows over the blocks.  Bound: the loads' latency; 256 x
// 50021 f32 with a class stride of 256: 131 us, 0.8 TB/s.
template <typename T, typename O>
__global__ void __launch_bounds__(BLOCK) token_grad_rows_kernel(TokenGradArgs a) {
    const Rows& in = a.logits;
    const uint64_t chunks = (in.cols + 4 * BLOCK - 1) / (4 * BLOCK);
    for (uint64_t u = blockIdx.x; u < in.rows * chunks; u += gridDim.x) {
        const uint64_t row = u / chunks, c0 = u % chunks * (4 * BLOCK);
        const T* x = static_cast<const T*>(in.data) + in.offset + nest_offset(in.outer, row);
        O* out = reinterpret_cast<O*>(a.out.data) + a.out.offset + nest_offset(a.out.outer, row);
        const uint32_t t = a.targets[a.target_offset + nest_offset(a.target_nest, row)];
        const float lse = row_value(a.lse, row);
        const float gl = t < in.cols ? row_value(a.g_logprob, row) : 0.0f;
        const float gh = a.g_entropy.data ? row_value(a.g_entropy, row) : 0.0f;
        const float h = gh != 0.0f ? row_value(a.entropy, row) : 0.0f;
        for (uint64_t c = c0 + threadIdx.x; c < min(c0 + 4 * BLOCK, in.cols); c += BLOCK) {
            const float d = logit_grad(logit<T>(x + nest_offset(in.inner, c)), lse, h, gl, gh, c == t);
            O* p = out + nest_offset(a.out.inner, c);
            if constexpr (sizeof(O) == 4) *p = d;
            else *p = a.out.dtype == FB_BF16 ? encode_bf16(d) : encode_f16(d);
        }
    }
}

// ------------------------------------------------- contiguous rows: one pass
//
// A row is read once, 16 bytes per lane and load, for everything but the
// alternatives.  Sums are kept against a reference m shared by a warp, its
// running maximum: with d_v = (x_v - m) log2 e,
//   S0 = sum 2^d_v,  S1 = sum d_v 2^d_v,
//   lse = m + ln S0,  entropy = ln S0 - ln 2 S1 / S0.
// x - m is subtracted before it is scaled (two packed operations instead of
// one FMA): the maximum's own term is then exactly 1, a row of one class has
// entropy and log probability exactly 0, and no m overflows.  Only a
// segment's maximum (packed 16-bit maxima, one redux) is compared with m, so
// rescales by 2^((m - m') log2 e) are rare.  d is clamped at -200 (2^-200
// flushes to 0) where that matters, which keeps a masked class's 0 * -inf out
// of S1; the NaN-propagating clamp keeps a NaN in it.
//
// Alternatives.  The k-th largest of the maxima of disjoint sets of lanes (to 16
// bits, by a binary search over ballots) is a lower bound t of the row's k-th
// largest value, and the maxima of the row's segments (kept in shared memory)
// say where values >= t lie: about k segments are read again (L2), the values
// >= t collected with their indices and put in order by counting.  More than
// CAND of them (a row of few distinct values), and rows with NaN or +inf, take a
// scan per alternative instead.  (Keeping a maximum per lane and segment, to
// read 64 bytes again instead of a segment, measured slower up to 5
// alternatives and no faster at 20 for rows under 50k classes.)
//
// Bound: HBM (the ex2 unit is 3/4 busy at the full rate with 16-bit logits),
// and the few microseconds per row in which its CTA puts the alternatives in
// order and loads nothing.  8200 x 131072 BF16: 375 us, 5.7 TB/s; with 5
// alternatives 415 us, 5.2 TB/s; 2048 rows 104 and 121 to 128 us; f32 1024 x 131072
// 86 and 96 us, 6.2 and 5.6 TB/s.  64 x 32000 with 8: 11 us, 1 x 50021 with 20:
// 12 us, latency.  (Measured and not kept: one persistent CTA per slot over
// several rows; a second launch that splits the rows of a partial last wave, 6%
// at 740 rows and nothing at 2048.)
// Few rows are split over the CTAs of a cluster, each with its own sums and
// alternatives, joined through distributed shared memory.
constexpr int SM_WARPS = 32;   // resident warps per SM (64 registers a thread)
constexpr int CAND = 1024;     // candidates that are put in order by counting
constexpr int MAX_SEGS = 512;  // segment maxima kept per CTA
constexpr float L2E = 1.4426950408889634f;

struct TokenPartial {  // one CTA's part of a row
    float m, s0, s1;
    uint64_t top[FB_MAX_TOP];  // (key << 32 | ~index), largest first; 0: none
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ uint32_t packed_max(uint32_t a, uint32_t b, __nv_bfloat16) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t packed_max(uint32_t a, uint32_t b, __half) {
    const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Per-row values with one stride (elements; 0 for a single value): the
// streaming kernels index them without the nests' divisions.
struct RowVec {
    void* p = nullptr;
    uint64_t stride = 0;
    template <typename V>
    __device__ __forceinline__ V& at(uint64_t row) const {
        return static_cast<V*>(p)[row * stride];
    }
};
bool row_vec(void* data, uint64_t offset, const Nest& n, RowVec* v) {
    if (n.rank > 1) return false;
    v->p = data ? static_cast<uint32_t*>(data) + offset : nullptr;
    v->stride = n.rank ? n.strides[0] : 0;
    return true;
}
bool row_vec(const RowOut& o, RowVec* v) { return row_vec(o.data, o.offset, o.nest, v); }

struct StreamArgs {
    const void* x;  // row 0
    uint64_t rows, cols, row_stride;
    RowVec targets, logprob, entropy, lse;
    float* top_logprob;
    uint32_t* top_index;
    uint32_t top;
    uint32_t parts, part_segs, mult;
};
struct GradArgs {
    const void* x;
    void* out;
    uint64_t cols, x_stride, out_stride;
    uint32_t chunks;
    RowVec targets, lse, g_logprob, entropy, g_entropy;
};

// A 16-byte vector as words; how a type's words are widened and compared.
template <typename T>
struct Words {
    static constexpr int E = 8;  // elements per vector
    static constexpr uint32_t LOWEST = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;  // -inf
    static __device__ __forceinline__ uint32_t maximum(uint32_t a, uint32_t b) { return packed_max(a, b, T()); }
    // pattern of the larger half
    static __device__ __forceinline__ uint32_t top(uint32_t w) { return maximum(w, __byte_perm(w, 0, 0x1032)) & 0xffffu; }
    static __device__ __forceinline__ float2 widen(uint32_t w) {
        if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<__half2*>(&w));
        else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
};
template <>
struct Words<float> {
    static constexpr int E = 4;
    static constexpr uint32_t LOWEST = 0xff800000u;
    static __device__ __forceinline__ uint32_t maximum(uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }
    static __device__ __forceinline__ uint32_t top(uint32_t w) { return w; }
};

// A contiguous row seen as aligned 16-byte vectors; vector 0 and the last one
// may hold elements of its neighbours, which read as -inf.
template <typename T>
struct RowVectors {
    using U = typename Bits<T>::U;
    static constexpr int E = Words<T>::E;
    const U* x;          // element 0
    uint32_t head;       // elements of vector 0 before element 0
    uint64_t end;        // head + columns
    __device__ __forceinline__ RowVectors(const T* row, uint64_t cols)
        : x(reinterpret_cast<const U*>(row)),
          head((uint32_t)(reinterpret_cast<uintptr_t>(row) & 15u) / (uint32_t)sizeof(U)),
          end(head + cols) {}
    __device__ __forceinline__ uint64_t vectors() const { return (end + E - 1) / E; }
    // NC: through the read-only path (not where the row is being overwritten)
    template <bool NC>
    __device__ __forceinline__ uint4 load(uint64_t j) const {
        const uint64_t v = j * E;
        if (v >= head && v + E <= end) {
            const uint4* p = reinterpret_cast<const uint4*>(x + (v - head));
            return NC ? __ldg(p) : *p;
        }
        uint4 r = make_uint4(Words<T>::LOWEST, Words<T>::LOWEST, Words<T>::LOWEST, Words<T>::LOWEST);
        if (v >= end) return r;
        uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (v + e >= head && v + e < end) {
                const uint32_t b = NC ? __ldg(x + (v + e - head)) : x[v + e - head];
                if constexpr (E == 4) w[e] = b;
                else w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | (b << 16) : (w[e / 2] & 0xffff0000u) | b;
            }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

__device__ __forceinline__ uint32_t mapa_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float ld_peer_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint64_t ld_peer_u64(uint32_t addr) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sync_cluster() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// Base-2 exponent of x against the reference m.
__device__ __forceinline__ float below(float x, float m) { return max_nan((x - m) * L2E, -200.0f); }

// {m, S0, S1} += another part's: both brought to the larger reference.
__device__ __forceinline__ void join_sums(float& m, float& s0, float& s1, float m2, float t0, float t1) {
    if (t0 == 0.0f) return;
    if (s0 == 0.0f) {
        m = m2, s0 = t0, s1 = t1;
        return;
    }
    const float top = fmaxf(m, m2), da = below(m, top), db = below(m2, top), a = ex2_approx(da), b = ex2_approx(db);
    s1 = fmaf(da, s0, s1) * a + fmaf(db, t0, t1) * b;
    s0 = s0 * a + t0 * b;
    m = top;
}

// `parts` CTAs (a cluster when > 1) per row, `part_segs` segments of 32 * VPL
// vectors each; `mult` segments share a kept maximum.
template <typename T, int VPL, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, SM_WARPS / WARPS) token_stream_kernel(StreamArgs a) {
    constexpr int THREADS = 32 * WARPS;
    using W = Words<T>;
    constexpr int NW = VPL * 4;
    __shared__ uint32_t tkey[THREADS], okey[32];  // maxima of the threads, and of WARPS lanes each
    __shared__ uint32_t seg_max[MAX_SEGS];
    __shared__ uint64_t cand[CAND];
    __shared__ uint64_t scan_keys[WARPS];
    __shared__ float wsum[3][WARPS];
    __shared__ uint32_t n_cand;
    __shared__ TokenPartial mine;
    const uint32_t parts = a.parts, mult = a.mult;
    const uint64_t row = blockIdx.x / parts;
    const uint32_t part = blockIdx.x % parts;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* x = static_cast<const T*>(a.x) + row * a.row_stride;
    const RowVectors<T> rv(x, a.cols);
    const uint32_t nseg = (uint32_t)((rv.vectors() + 32 * VPL - 1) / (32 * VPL));
    const uint32_t seg0 = min(part * a.part_segs, nseg), seg1 = min(seg0 + a.part_segs, nseg);
    const uint32_t groups = (seg1 - seg0 + mult - 1) / mult;
    if (threadIdx.x == 0) n_cand = 0u;
    // A warp takes groups of `mult` segments in turn with the others.
    auto seg_after = [&](uint32_t seg) {
        return mult == 1 ? seg + WARPS : (seg - seg0 + 1) % mult ? seg + 1 : seg + 1 + (WARPS - 1) * mult;
    };
    // segments [in0, in1) lie inside the row: no vector of theirs is partial
    const uint32_t per_seg = 32 * VPL * W::E;
    const uint32_t in0 = rv.head ? 1u : 0u, in1 = (uint32_t)(rv.end / per_seg);
    const uint4* xv = reinterpret_cast<const uint4*>(rv.x - rv.head) + lane;  // vector `lane` of segment 0
    auto load_seg = [&](uint32_t seg, uint32_t (&w)[NW]) {
        if (seg >= in0 && seg < in1) {
            const uint4* p = xv + (uint64_t)seg * (32 * VPL);
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const uint4 v = __ldg(p + i * 32);
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const uint4 v = rv.template load<true>((uint64_t)seg * (32 * VPL) + i * 32 + lane);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    };
    float m = 0.0f;  // the reference: 0 while nothing but -inf was seen
    float2 s0 = make_float2(0.f, 0.f), s1 = make_float2(0.f, 0.f);
    uint32_t run = 0u, own_max = W::LOWEST;
    uint32_t w[NW];
    uint32_t group_max = 0u;
    if (seg0 + warp * mult < seg1) load_seg(seg0 + warp * mult, w);
    for (uint32_t seg = seg0 + warp * mult, after; seg < seg1; seg = after) {
        uint32_t next[NW];  // the next segment's loads are in flight while this one is summed
        after = seg_after(seg);
        if (after < seg1) load_seg(after, next);
        uint32_t mx = w[0];
#pragma unroll
        for (int i = 1; i < NW; ++i) mx = W::maximum(mx, w[i]);
        own_max = W::maximum(own_max, mx);
        const uint32_t top = __reduce_max_sync(0xffffffffu, Bits<T>::key(W::top(mx)));
        if (a.top) {
            const uint32_t i = mult == 1 ? seg - seg0 : (seg - seg0) / mult;
            group_max = mult == 1 || (seg - seg0) % mult == 0 ? top : max(group_max, top);
            if (lane == 0) seg_max[i] = group_max;
        }
        if (top > run) {
            run = top;
            const float v = Bits<T>::value(Bits<T>::pattern(top));
            const float m2 = v == -__int_as_float(0x7f800000) ? 0.0f : v;
            const float dm = below(m, m2), f = ex2_approx(dm);
            const float t0 = s0.x + s0.y, t1 = s1.x + s1.y;
            s0 = make_float2(t0 == 0.0f ? 0.0f : t0 * f, 0.0f);
            s1 = make_float2(t0 == 0.0f ? 0.0f : fmaf(dm, t0, t1) * f, 0.0f);
            m = m2;
        }
        // Without the clamp a class at -inf (or further below than the floats
        // reach) makes the segment's S1 NaN: only then is it taken again with it.
        float2 a0, a1;
        auto sum = [&](auto clamp) {
            const float2 l2 = make_float2(L2E, L2E), nm = make_float2(-m, -m);
            constexpr int PAIRS = W::E == 8 ? NW : NW / 2;
            a0 = a1 = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                float2 v;
                if constexpr (W::E == 8) v = W::widen(w[i]);
                else v = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
                float2 d = __fmul2_rn(__fadd2_rn(v, nm), l2);
                if (clamp) d.x = max_nan(d.x, -200.0f), d.y = max_nan(d.y, -200.0f);
                const float2 e = make_float2(ex2_approx(d.x), ex2_approx(d.y));
                a0 = __fadd2_rn(a0, e);
                a1 = __ffma2_rn(e, d, a1);
            }
        };
        sum(std::false_type());
        const float t1 = a1.x + a1.y;
        if (__any_sync(0xffffffffu, t1 != t1)) sum(std::true_type());
        s0 = __fadd2_rn(s0, a0);
        s1 = __fadd2_rn(s1, a1);
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = next[i];
    }
    {
        const float t0 = warp_sum_f(s0.x + s0.y), t1 = warp_sum_f(s1.x + s1.y);
        if (lane == 0) wsum[0][warp] = m, wsum[1][warp] = t0, wsum[2][warp] = t1;
        if (a.top) {
            uint32_t key = Bits<T>::key(W::top(own_max));
            tkey[threadIdx.x] = key;
#pragma unroll
            for (int o = 1; o < WARPS; o <<= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
            if (lane % WARPS == 0) okey[threadIdx.x / WARPS] = key;
        }
    }
    __syncthreads();
    // The warps' sums, joined by each warp's first lanes.
    float M, S0, S1;
    {
        const int i = lane & (WARPS - 1);
        const float mi = wsum[0][i], t0 = wsum[1][i], t1 = wsum[2][i];
        M = t0 == 0.0f ? -__int_as_float(0x7f800000) : mi;
#pragma unroll
        for (int o = 1; o < WARPS; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float d = t0 == 0.0f ? 0.0f : below(mi, M), f = ex2_approx(d);
        S0 = t0 * f;
        S1 = t0 == 0.0f ? 0.0f : fmaf(d, t0, t1) * f;
#pragma unroll
        for (int o = 1; o < WARPS; o <<= 1) {
            S0 += __shfl_xor_sync(0xffffffffu, S0, o);
            S1 += __shfl_xor_sync(0xffffffffu, S1, o);
        }
    }

    const float ls = S0 == 0.0f ? row_nan() : logf(S0);  // log S0
    if (a.top) {
        const uint32_t k = a.top;
        if (parts > 1 && threadIdx.x < FB_MAX_TOP) mine.top[threadIdx.x] = 0ull;
        // t: the largest 16-bit prefix that k maxima reach, bit by bit, found
        // by each warp for itself: of the lane groups' 32 maxima for few
        // alternatives (k = 20 leaves about 30 values to put in order), where k
        // groups have any values, else of the threads' (fewer than k maxima bound
        // nothing: all values would be candidates, and a scan per alternative
        // took 29 us for 16 x 25000 with 20 in four parts, against 12).
        constexpr int SHIFT = W::E == 8 ? 0 : 16;
        uint32_t t = 0;
        constexpr uint32_t NONE = W::LOWEST >> SHIFT & 0xffffu;  // -inf
        const bool groups_do = __popc(__ballot_sync(0xffffffffu, okey[lane] >> SHIFT > (~NONE & 0xffffu))) >= (int)k;
        if (k <= 20 && groups_do) {
            const uint32_t v = okey[lane] >> SHIFT;
#pragma unroll
            for (uint32_t bit = 0x8000u; bit; bit >>= 1)
                if (__popc(__ballot_sync(0xffffffffu, v >= (t | bit))) >= k) t |= bit;
        } else {
            uint32_t v[WARPS];
#pragma unroll
            for (int i = 0; i < WARPS; ++i) v[i] = tkey[i * 32 + lane] >> SHIFT;
#pragma unroll 1
            for (uint32_t bit = 0x8000u; bit; bit >>= 1) {
                uint32_t n = 0;
#pragma unroll
                for (int i = 0; i < WARPS; ++i) n += v[i] >= (t | bit);
                if (__reduce_add_sync(0xffffffffu, n) >= k) t |= bit;
            }
        }
        t <<= SHIFT;
        const bool fine = S0 == S0;  // no NaN and no +inf among the values
        if (fine) {
            // The segments that reach t are read again; values at least t (as
            // numbers: a zero of the other sign comes along) are collected.
            float tv = Bits<T>::value(Bits<T>::pattern(t));
            if (tv != tv) tv = -__int_as_float(0x7f800000);  // a prefix of -inf names a NaN
            for (uint32_t g0 = 0; g0 < groups; g0 += 32 * WARPS) {
                const uint32_t lane_g = g0 + lane * WARPS + warp;
                uint32_t hits = __ballot_sync(0xffffffffu, lane_g < groups && seg_max[min(lane_g, MAX_SEGS - 1u)] >= t);
                for (; hits; hits &= hits - 1) {
                    const uint32_t g = g0 + (__ffs(hits) - 1) * WARPS + warp;
                    for (uint32_t seg = seg0 + g * mult; seg < min(seg0 + (g + 1) * mult, seg1); ++seg) {
                        uint32_t y[NW];
                        load_seg(seg, y);
                        const uint64_t v0 = ((uint64_t)seg * (32 * VPL) + lane) * W::E;
                        auto take = [&](uint32_t bits, int e) {
                            const uint64_t v = v0 + (uint64_t)(e / W::E) * 32 * W::E + e % W::E;
                            if (v < rv.head || v >= rv.end) return;
                            const uint32_t n = atomicAdd(&n_cand, 1u);
                            if (n < CAND) cand[n] = ((uint64_t)Bits<T>::key(bits) << 32) | (0xffffffffu - (uint32_t)(v - rv.head));
                        };
#pragma unroll
                        for (int i = 0; i < NW; ++i) {
                            if constexpr (W::E == 8) {
                                const float2 f = W::widen(y[i]);
                                if (fmaxf(f.x, f.y) >= tv) {
                                    if (f.x >= tv) take(y[i] & 0xffffu, 2 * i);
                                    if (f.y >= tv) take(y[i] >> 16, 2 * i + 1);
                                }
                            } else if (__uint_as_float(y[i]) >= tv) {
                                take(y[i], i);
                            }
                        }
                    }
                }
            }
        }
        __syncthreads();
        const uint32_t n = n_cand;
        if (fine && n <= CAND) {
            // Places by counting; a whole row's go out from here.
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                const uint64_t me = cand[i];
                uint32_t rank = 0;
#pragma unroll 4
                for (uint32_t j = 0; j < n; ++j) rank += cand[j] > me;
                if (rank >= k) continue;
                if (parts > 1) {
                    mine.top[rank] = me;
                } else {
                    a.top_index[row * k + rank] = 0xffffffffu - (uint32_t)me;
                    a.top_logprob[row * k + rank] = (Bits<T>::value(Bits<T>::pattern((uint32_t)(me >> 32))) - M) - ls;
                }
            }
        } else {
            const uint64_t v0 = max((uint64_t)seg0 * (32 * VPL) * W::E, (uint64_t)rv.head);
            const uint64_t v1 = min((uint64_t)seg1 * (32 * VPL) * W::E, rv.end);
            uint64_t bound = ~0ull;
            for (uint32_t r = 0; r < k && bound; ++r) {
                uint64_t best = 0;
                for (uint64_t v = v0 + threadIdx.x; v < v1; v += THREADS) {
                    const uint64_t q = ((uint64_t)Bits<T>::key(__ldg(rv.x + (v - rv.head))) << 32) |
                                       (0xffffffffu - (uint32_t)(v - rv.head));
                    if (q < bound && q > best) best = q;
                }
                bound = block_max_u64<THREADS>(best, scan_keys);
                if (threadIdx.x != 0) continue;
                if (parts > 1) {
                    mine.top[r] = bound;
                } else {
                    a.top_index[row * k + r] = 0xffffffffu - (uint32_t)bound;
                    a.top_logprob[row * k + r] = (Bits<T>::value(Bits<T>::pattern((uint32_t)(bound >> 32))) - M) - ls;
                }
            }
        }
    }
    auto store_row = [&](float ls) {
        if (a.lse.p) a.lse.at<float>(row) = M + ls;
        if (a.entropy.p) a.entropy.at<float>(row) = ls - S1 / S0 * 0.6931471805599453f;
        if (a.logprob.p) {
            const uint32_t t = a.targets.at<uint32_t>(row);
            float r = 0.0f;
            if (t != FB_NO_TOKEN) r = t < a.cols ? (Elem<T>::load(x + t) - M) - ls : row_nan();
            a.logprob.at<float>(row) = r;
        }
    };
    if (parts == 1) {
        if (threadIdx.x == THREADS - 1) store_row(ls);
        return;
    }
    if (threadIdx.x == 0) mine.m = M, mine.s0 = S0, mine.s1 = S1;
    sync_cluster();  // every part's sums and list are in its shared memory
    if (part == 0) {
        const uint32_t at = (uint32_t)__cvta_generic_to_shared(&mine);
        const uint32_t off = (uint32_t)(reinterpret_cast<const char*>(mine.top) - reinterpret_cast<const char*>(&mine));
        const uint32_t n = parts * a.top;
        for (uint32_t i = threadIdx.x; i < n; i += THREADS)
            cand[i] = ld_peer_u64(mapa_rank(at + off, i / a.top) + (i % a.top) * 8);
        for (uint32_t p = 1; p < parts; ++p) {
            const uint32_t peer = mapa_rank(at, p);
            join_sums(M, S0, S1, ld_peer_f32(peer), ld_peer_f32(peer + 4), ld_peer_f32(peer + 8));
        }
        const float lsr = S0 == 0.0f ? row_nan() : logf(S0);
        if (threadIdx.x == THREADS - 1) store_row(lsr);
        __syncthreads();
        // the parts' alternatives in one list: places by counting
        for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
            const uint64_t me = cand[i];
            if (me == 0) continue;
            uint32_t rank = 0;
#pragma unroll 4
            for (uint32_t j = 0; j < n; ++j) rank += cand[j] > me;
            if (rank >= a.top) continue;
            a.top_index[row * a.top + rank] = 0xffffffffu - (uint32_t)me;
            a.top_logprob[row * a.top + rank] = (Bits<T>::value(Bits<T>::pattern((uint32_t)(me >> 32))) - M) - lsr;
        }
    }
    sync_cluster();  // a part's sums and list stay until they are read
}

template <typename T, int VPL, int WARPS>
int launch_stream(const TokenArgs& a, cudaStream_t st) {
    const Rows& in = a.logits;
    const uint64_t E = Words<T>::E, seg = 32 * VPL;
    const uint64_t nseg = ((in.cols + 2 * E - 2) / E + seg - 1) / seg;  // at the worst alignment
    // Parts per row: powers of two up to a cluster of four, while the grid is
    // under eight CTAs per SM and a part keeps two segments per warp, or under
    // one per SM and it keeps half a segment per warp.
    uint64_t parts = 1;
    const uint64_t sms = (uint64_t)sm_count();
    while (parts < 4 && ((in.rows * parts * 2 <= sms * 8 && nseg >= parts * 2 * 2 * WARPS) ||
                         (in.rows * parts * 2 <= sms && nseg >= parts * WARPS)))
        parts *= 2;
    // The last part must hold more lanes with values than alternatives asked for
    // (else it has no bound, see above: 16 x 16500 with 50 took 43 us).
    while (parts > 1 && a.top > 0 && nseg < (parts - 1) * ((nseg + parts - 1) / parts) + 2 + (a.top + 31) / 32) parts /= 2;
    const uint64_t part_segs = (nseg + parts - 1) / parts;
    const uint64_t mult = (part_segs + MAX_SEGS - 1) / MAX_SEGS;
    if (in.rows * parts > 0x7fffffffull || nseg > 0xffffffffull) return FB_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(in.rows * parts));
    cfg.blockDim = dim3(32 * WARPS);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)parts;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    StreamArgs k{};
    k.x = static_cast<const T*>(in.data) + in.offset;
    k.rows = in.rows, k.cols = in.cols, k.row_stride = in.row_stride;
    if (!row_vec(const_cast<uint32_t*>(a.targets), a.target_offset, a.target_nest, &k.targets) || !row_vec(a.logprob, &k.logprob) ||
        !row_vec(a.entropy, &k.entropy) || !row_vec(a.lse, &k.lse))
        return FB_ERR_UNSUPPORTED;
    k.top_logprob = a.top_logprob, k.top_index = a.top_index, k.top = a.top;
    k.parts = (uint32_t)parts, k.part_segs = (uint32_t)part_segs, k.mult = (uint32_t)mult;
    (void)cudaLaunchKernelEx(&cfg, token_stream_kernel<T, VPL, WARPS>, k);
    count_launch("token_stream_kernel");
    return launch_status("kernel launch");
}

template <typename T>
int launch_t(const TokenArgs& a, cudaStream_t st) {
    if (a.logits.contiguous_rows) {
        // Short rows: one vector per lane and segment, so that every warp has
        // one from 8 * 32 vectors on.
        const bool brief = a.logits.cols <= (uint64_t)Words<T>::E * 32 * 4 * 8;
        // CTAs of four warps leave less of an SM idle while one of them puts
        // its alternatives in order; of eight, a last wave is shorter.  Four
        // where the rows fill the GPU and their waves (twice as long) cost at
        // most an eighth more.  Top 5, us, four | eight: 8200 x 32000 152 |
        // 171, 700 x 16000 17 | 19, 740 x 131072 60 | 64, 2048 x 131072 127 |
        // 127; where the rule keeps eight, 1776 x 131072 118 | 109.
        const uint64_t slots = (uint64_t)sm_count() * (SM_WARPS / 8), waves = (a.logits.rows + slots - 1) / slots;
        const bool four = a.logits.rows > slots && 16 * ((waves + 1) / 2) <= 9 * waves;
        const int r = brief ? four ? launch_stream<T, 1, 4>(a, st) : launch_stream<T, 1, 8>(a, st)
                            : four ? launch_stream<T, 4, 4>(a, st) : launch_stream<T, 4, 8>(a, st);
        if (r != FB_ERR_UNSUPPORTED) return r;
    }
    const unsigned blocks = (unsigned)std::min<uint64_t>(a.logits.rows, (uint64_t)sm_count() * 32);
    token_rows_kernel<T><<<blocks, BLOCK, 0, st>>>(a);
    count_launch("token_rows_kernel");
    return launch_status("kernel launch");
}

// Contiguous rows whose output vectors line up with the logits': 16 bytes per
// lane and load.  With d = (x - lse) log2 e, p = 2^d and
//   grad = gl [v = t] - p (gl + gh (log p + entropy)) = gl [v = t] + 2^d (A + B d),
//   A = -(gl + gh entropy), B = -gh ln 2:
// four packed operations, two clamps and two ex2 for a pair of elements; d is
// clamped at -200 (2^-200 flushes to 0) so that a masked class's -inf meets no
// 0 or infinity.
// Bound: HBM, one read and one write.  Loads are issued before the row's
// scalars arrive; each block does one chunk of 4 vectors per thread.
// 2048 x 131072 BF16: 170 to 183 us back to back (6.3 to 5.9 TB/s), 191 to 193 us (5.6
// TB/s) with other logits and another output every call; into f32 270 us, 6.0 TB/s.
template <typename T, typename U>  // U: patterns of the output, T's own or f32's
__global__ void __launch_bounds__(BLOCK) token_grad_stream_kernel(GradArgs a) {
    using W = Words<T>;
    constexpr int E = W::E, N = 4;
    constexpr bool LOW = sizeof(U) == 2;
    const uint64_t row = blockIdx.x / a.chunks;
    const uint64_t j0 = (uint64_t)(blockIdx.x % a.chunks) * (N * BLOCK) + threadIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    U* out = static_cast<U*>(a.out) + row * a.out_stride;
    const RowVectors<T> rv(x, a.cols);
    uint32_t w[N][4];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint4 v = rv.template load<false>(j0 + i * BLOCK);
        w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
    }
    const uint32_t t = a.targets.at<const uint32_t>(row);
    const float lse = a.lse.at<const float>(row);
    const float gl = t < a.cols ? a.g_logprob.at<const float>(row) : 0.0f;
    const float gh = a.g_entropy.p ? a.g_entropy.at<const float>(row) : 0.0f;
    const float h = gh != 0.0f ? a.entropy.at<const float>(row) : 0.0f;
    const bool zero = gl == 0.0f && gh == 0.0f;
    const float A = -fmaf(gh, h, gl), B = -gh * 0.6931471805599453f;
    const uint64_t at = (uint64_t)t + rv.head;  // the target's place among the vectors' elements
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint64_t v = (j0 + i * BLOCK) * E;
        if (v >= rv.end) break;
        float g[E];
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            float2 y;
            if constexpr (E == 8) y = W::widen(w[i][e / 2]);
            else y = make_float2(__uint_as_float(w[i][e]), __uint_as_float(w[i][e + 1]));
            float2 d = __fmul2_rn(__fadd2_rn(y, make_float2(-lse, -lse)), make_float2(L2E, L2E));
            d.x = max_nan(d.x, -200.0f), d.y = max_nan(d.y, -200.0f);
            const float2 k = __ffma2_rn(d, make_float2(B, B), make_float2(A, A));
            g[e] = zero ? 0.0f : ex2_approx(d.x) * k.x;
            g[e + 1] = zero ? 0.0f : ex2_approx(d.y) * k.y;
        }
        if (at - v < (uint64_t)E && gl != 0.0f) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (at == v + e) g[e] += gl;
        }
        constexpr int WORDS = E * sizeof(U) / 4;
        uint32_t o[WORDS];
#pragma unroll
        for (int e = 0; e < WORDS; ++e) {
            if constexpr (LOW) o[e] = encode_low_pair(g[2 * e], g[2 * e + 1], std::is_same<T, __half>::value ? FB_F16 : FB_BF16);
            else o[e] = __float_as_uint(g[e]);
        }
        if (v >= rv.head && v + E <= rv.end) {
#pragma unroll
            for (int e = 0; e < WORDS; e += 4)
                __stcs(reinterpret_cast<uint4*>(out + (v - rv.head)) + e / 4, make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]));
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (v + e >= rv.head && v + e < rv.end) {
                    if constexpr (LOW) out[v + e - rv.head] = (U)(e % 2 ? o[e / 2] >> 16 : o[e / 2] & 0xffffu);
                    else out[v + e - rv.head] = o[e];
                }
        }
    }
}

template <typename T>
int launch_grad_t(const TokenGradArgs& a, cudaStream_t st) {
    const Rows& in = a.logits;
    constexpr uint64_t esz = sizeof(typename Bits<T>::U);
    const uint64_t osz = a.out.dtype == FB_F32 ? 4 : esz, step = 16 / osz;  // step: output elements of 16 bytes
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(in.data) + in.offset * esz;
    const uintptr_t o0 = reinterpret_cast<uintptr_t>(a.out.data) + a.out.offset * osz;
    // Output elements sit in their 16 bytes as the logits do in theirs.
    if (in.contiguous_rows && a.out.contiguous_rows && (x0 / esz - o0 / osz) % step == 0 &&
        (in.row_stride - a.out.row_stride) % step == 0) {
        const uint64_t vectors = (in.cols + 2 * Words<T>::E - 2) / Words<T>::E, chunks = (vectors + 4 * BLOCK - 1) / (4 * BLOCK);
        GradArgs k{};
        const bool strided = row_vec(const_cast<uint32_t*>(a.targets), a.target_offset, a.target_nest, &k.targets) &&
                             row_vec(a.lse, &k.lse) && row_vec(a.g_logprob, &k.g_logprob) && row_vec(a.entropy, &k.entropy) &&
                             row_vec(a.g_entropy, &k.g_entropy);
        if (strided && in.rows * chunks <= 0x7fffffffull) {
            k.x = reinterpret_cast<const void*>(x0), k.out = reinterpret_cast<void*>(o0);
            k.cols = in.cols, k.x_stride = in.row_stride, k.out_stride = a.out.row_stride;
            k.chunks = (uint32_t)chunks;
            if (osz == esz) token_grad_stream_kernel<T, typename Bits<T>::U><<<(unsigned)(in.rows * chunks), BLOCK, 0, st>>>(k);
            else token_grad_stream_kernel<T, uint32_t><<<(unsigned)(in.rows * chunks), BLOCK, 0, st>>>(k);
            count_launch("token_grad_stream_kernel");
            return launch_status("kernel launch");
        }
    }
    const uint64_t chunks = (a.logits.cols + 4 * BLOCK - 1) / (4 * BLOCK);
    const unsigned blocks = (unsigned)std::min<uint64_t>(a.logits.rows * chunks, (uint64_t)sm_count() * 64);
    if (a.out.dtype == FB_F32) token_grad_rows_kernel<T, float><<<blocks, BLOCK, 0, st>>>(a);
    else token_grad_rows_kernel<T, uint16_t><<<blocks, BLOCK, 0, st>>>(a);
    count_launch("token_grad_rows_kernel");
    return launch_status("kernel launch");
}

}  // namespace

int launch_token_logprobs(const TokenArgs& a, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (a.logits.dtype) {
        case FB_F32: return launch_t<float>(a, st);
        case FB_BF16: return launch_t<__nv_bfloat16>(a, st);
        case FB_F16: return launch_t<__half>(a, st);
        default: return FB_ERR_DTYPE;
    }
}

int launch_token_logprobs_grad(const TokenGradArgs& a, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (a.logits.dtype) {
        case FB_F32: return launch_grad_t<float>(a, st);
        case FB_BF16: return launch_grad_t<__nv_bfloat16>(a, st);
        case FB_F16: return launch_grad_t<__half>(a, st);
        default: return FB_ERR_DTYPE;
    }
}

}  // namespace fb
