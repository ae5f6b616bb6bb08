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
// below the previous one).
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

// Gradient of one logit.  A term whose coefficient is 0 is 0 whatever x is.
__device__ __forceinline__ float logit_grad(float x, float lse, float h, float gl, float gh, bool at_target) {
    const float z = x - lse, p = expf(z);
    float d = 0.0f;
    if (gl != 0.0f) d = gl * ((at_target ? 1.0f : 0.0f) - p);
    if (gh != 0.0f) d -= p > 0.0f || p != p ? gh * (p * (z + h)) : 0.0f;
    return d;
}

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
            const float d = logit_grad(Elem<T>::load(x + nest_offset(in.inner, c)), lse, h, gl, gh, c == t);
            O* p = out + nest_offset(a.out.inner, c);
            if constexpr (sizeof(O) == 4) *p = d;
            else *p = a.out.dtype == FB_BF16 ? encode_bf16(d) : encode_f16(d);
        }
    }
}

template <typename T>
int launch_t(const TokenArgs& a, cudaStream_t st) {
    const unsigned blocks = (unsigned)std::min<uint64_t>(a.logits.rows, (uint64_t)sm_count() * 32);
    token_rows_kernel<T><<<blocks, BLOCK, 0, st>>>(a);
    count_launch("token_rows_kernel");
    return launch_status("kernel launch");
}

template <typename T>
int launch_grad_t(const TokenGradArgs& a, cudaStream_t st) {
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
