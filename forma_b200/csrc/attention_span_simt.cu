// Windowed and shared-prefix attention on CUDA cores: any strides, depths and
// types.
//
// One block of four warps owns a query row.  Its visible keys are up to three
// spans - the shared prefix, the first keys that stay visible (sinks) and the
// window before the query's position - and the warps take the spans' 32-key
// tiles in turn, one key per lane, each with its own online softmax in f64
// (as the general attention kernel keeps it, so f32 results stay within 1e-5);
// the four states are joined through shared memory.  Hidden keys are not
// read at all.
//
// Bound: the f64 states and one row's loads at a time, not memory: f32, 2
// sequences x 8 heads x 512 queries, window 1024, D = 64: 2.1 ms; single tokens
// of 16 sequences, 32/8 heads, window 4096, D = 128: 1.28 ms, 0.42 TB/s.
#include <cuda_runtime.h>

#include <algorithm>

#include "device_common.cuh"
#include "kernels.h"

namespace fb {
namespace {

constexpr int WARPS = 4;

struct SpanRow {
    uint64_t q, k, v, o;      // element offsets of the row, its head's first key and value, its output row
    uint64_t pk, pv;          // first prefix key and value of the head
    uint64_t batch, query;
};

__device__ __forceinline__ SpanRow span_row(const SpanArgs& s, uint64_t row) {
    const AttnArgs& a = s.base;
    SpanRow b{a.q_offset, a.k_offset, a.v_offset, a.o_offset, s.pk_offset, s.pv_offset, 0, 0};
    uint64_t rem = row, scale = 1;
    const int r = (int)a.row_rank;
#pragma unroll
    for (int d = FB_MAX_RANK - 1; d >= 0; --d) {
        if (d < r) {
            const uint64_t dim = a.row_dims[d], c = rem % dim;
            rem /= dim;
            const uint64_t kvc = d == r - 2 ? c / a.group_size : c;
            b.q += c * a.q_row_strides[d];
            b.k += kvc * a.k_row_strides[d];
            b.v += kvc * a.v_row_strides[d];
            b.o += c * a.o_row_strides[d];
            if (d == r - 1) b.query = c;
            if (d == r - 2) b.pk += kvc * s.pk_stride_head, b.pv += kvc * s.pv_stride_head;
            if (d < r - 2) {
                b.batch += c * scale;
                scale *= dim;
            }
        }
    }
    return b;
}

struct Span {  // keys [begin, end)
    uint64_t begin, end;
};

template <typename T, typename O>
__global__ void __launch_bounds__(32 * WARPS) span_simt_kernel(SpanArgs s) {
    const AttnArgs& a = s.base;
    extern __shared__ double smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t slot = a.value_depth + 34;  // O, 32 weights, {maximum, denominator}
    double* acc = smem + (uint64_t)warp * slot;
    double* wts = acc + a.value_depth;
    float* qrow = reinterpret_cast<float*>(smem + WARPS * slot);
    const double excluded = -__longlong_as_double(0x7ff0000000000000ll);
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const SpanRow b = span_row(s, row);
        const T* Q = static_cast<const T*>(a.q);
        for (uint64_t d = threadIdx.x; d < a.depth; d += blockDim.x) qrow[d] = Elem<T>::load(Q + b.q + d * a.q_stride_d);
        for (uint64_t d = lane; d < a.value_depth; d += 32) acc[d] = 0.0;
        __syncthreads();
        int64_t filled = (int64_t)a.keys;
        int64_t pos = s.offset + (int64_t)b.query;
        if (s.lengths) {
            filled = min(filled, (int64_t)s.lengths[b.batch * s.length_stride]);
            pos = filled - (int64_t)a.row_dims[a.row_rank - 1] + (int64_t)b.query;
        }
        const int64_t hi = max((int64_t)0, min(filled, pos + 1));
        int64_t lo = max((int64_t)0, pos - (int64_t)s.window + 1);  // window <= 2^62 (host)
        lo = min(lo, hi);
        const int64_t first = min((int64_t)min(s.sinks, (uint64_t)1 << 62), lo);
        const Span spans[3] = {{0, s.prefix_keys}, {0, (uint64_t)first}, {(uint64_t)lo, (uint64_t)hi}};
        double maximum = excluded, denominator = 0.0;
        uint64_t tile = 0;  // of all spans: warp w takes tiles w, w + WARPS, ...
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            const T* K = static_cast<const T*>(n == 0 ? s.pk : a.k) + (n == 0 ? b.pk : b.k);
            const T* V = static_cast<const T*>(n == 0 ? s.pv : a.v) + (n == 0 ? b.pv : b.v);
            const uint64_t k_key = n == 0 ? s.pk_stride_key : a.k_stride_key, k_d = n == 0 ? s.pk_stride_d : a.k_stride_d;
            const uint64_t v_key = n == 0 ? s.pv_stride_key : a.v_stride_key, v_d = n == 0 ? s.pv_stride_d : a.v_stride_d;
            for (uint64_t begin = spans[n].begin; begin < spans[n].end; begin += 32, ++tile) {
                if (tile % WARPS != (uint64_t)warp) continue;
                const uint64_t key = begin + lane;
                double score = excluded;
                if (key < spans[n].end) {
                    double dot = 0.0;
                    const T* kp = K + key * k_key;
                    for (uint64_t d = 0; d < a.depth; ++d) dot += (double)qrow[d] * (double)Elem<T>::load(kp + d * k_d);
                    score = dot * (double)a.scale;
                }
                // One maximum for the whole warp, so that all lanes go on or
                // none does: a NaN compares false either way and would leave its
                // own lane with another maximum than the rest.  It takes part
                // through its weight, which makes the row NaN.
                const bool nan = __any_sync(0xffffffffu, score != score);
                double tile_max = score == score ? score : excluded;
#pragma unroll
                for (int x = 16; x; x >>= 1) {
                    const double o = __shfl_xor_sync(0xffffffffu, tile_max, x);
                    tile_max = o > tile_max ? o : tile_max;
                }
                // Every visible score -inf (infinite operands): no weight, as
                // the general kernel has it.
                if (tile_max == excluded && !nan) continue;
                const double next = maximum > tile_max ? maximum : tile_max;
                const double alpha = denominator == 0.0 ? 0.0 : exp(maximum - next);
                maximum = next;
                const double w = score == excluded ? 0.0 : exp(score - maximum);
                denominator = denominator * alpha + warp_sum(w);
                wts[lane] = w;
                __syncwarp();
                for (uint64_t d = lane; d < a.value_depth; d += 32) {
                    double r = acc[d] * alpha;
                    for (int j = 0; j < 32; ++j) {
                        const double wj = wts[j];
                        if (wj != 0.0) r += wj * (double)Elem<T>::load(V + (begin + j) * v_key + d * v_d);
                    }
                    acc[d] = r;
                }
                __syncwarp();
            }
        }
        if (lane == 0) wts[32] = maximum, wts[33] = denominator;
        __syncthreads();
        double M = excluded, L = 0.0, wgt[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const double* st = smem + (uint64_t)w * slot + a.value_depth + 32;
            if (st[1] != 0.0) M = st[0] > M ? st[0] : M;
        }
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const double* st = smem + (uint64_t)w * slot + a.value_depth + 32;
            wgt[w] = st[1] != 0.0 ? exp(st[0] - M) : 0.0;
            L += st[1] * wgt[w];
        }
        O* out = reinterpret_cast<O*>(a.out) + b.o;
        for (uint64_t d = threadIdx.x; d < a.value_depth; d += blockDim.x) {
            double r = 0.0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w)
                if (wgt[w] != 0.0) r += wgt[w] * smem[(uint64_t)w * slot + d];
            const float f = L == 0.0 ? 0.0f : (float)(r / L);
            if constexpr (sizeof(O) == 4) out[d * a.o_stride_d] = f;
            else out[d * a.o_stride_d] = a.out_low == FB_BF16 ? encode_bf16(f) : encode_f16(f);
        }
        __syncthreads();  // the next row reuses shared memory
    }
}

template <typename T>
int launch_t(const SpanArgs& s, uint64_t smem, unsigned blocks, cudaStream_t st) {
    auto kernel = s.base.out_low ? span_simt_kernel<T, uint16_t> : span_simt_kernel<T, float>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return launch_status("shared-memory attribute");
    kernel<<<blocks, 32 * WARPS, smem, st>>>(s);
    count_launch("span_simt_kernel");
    return launch_status("kernel launch");
}

}  // namespace

int launch_span_simt(const SpanArgs& s, void* stream) {
    const AttnArgs& a = s.base;
    if (a.rows == 0) return FB_OK;
    const uint64_t smem = (WARPS * (a.value_depth + 34) + (a.depth + 1) / 2) * sizeof(double);
    if (smem > 200 * 1024) return FB_ERR_UNSUPPORTED;
    const unsigned blocks = (unsigned)std::min<uint64_t>(a.rows, (uint64_t)sm_count() * 64);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (a.dtype) {
        case FB_F32: return launch_t<float>(s, smem, blocks, st);
        case FB_BF16: return launch_t<__nv_bfloat16>(s, smem, blocks, st);
        case FB_F16: return launch_t<__half>(s, smem, blocks, st);
        default: return FB_ERR_DTYPE;
    }
}

}  // namespace fb
