// Windowed attention (last `window` keys and the first `sinks`) and attention
// over a prefix shared by the batch, for 16-bit operands at depth 64 and 128.
//
// Many query rows per key/value head: span_tile_kernel, a tcgen05 flash kernel
// over the key tiles that a block of rows can see.  At most 16 rows per
// key/value head (single tokens of a few sequences' heads): span_decode_kernel,
// warp-level MMAs under a stream of exactly the visible keys.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "attention_common.cuh"

namespace fb {
namespace {

__device__ uint32_t g_span_status;

// ------------------------------------------------------------- key spans

// A block of queries at positions pa .. pb (pa <= pb) over n filled keys sees
// no key outside [0, first) and [lo, hi], first <= lo: hi = min(pb, n - 1),
// lo = max(0, pa - window + 1).  hi < 0: nothing at all; lo > hi: only first.
//
// 32 bits hold all of it: L and Lk are at most 2^30, so positions and window
// starts clamped to +-2^30 by the host select the same keys.
struct SpanKeys {
    int32_t pos0, low0;     // without lengths: query 0's position, its window's first key (may be negative)
    int32_t window, sinks;  // at most 2^30
    int32_t after;          // with lengths: queries of the call behind this launch's last
    const uint32_t* lengths;
    uint64_t length_stride;
};
struct SpanBase {  // of one sequence
    int32_t filled, pos0, low0;
};
__device__ __forceinline__ SpanBase span_base(const SpanKeys& k, uint32_t b, uint32_t L, uint32_t Lk) {
    SpanBase s{(int32_t)Lk, k.pos0, k.low0};
    if (k.lengths) {
        s.filled = (int32_t)min(Lk, k.lengths[b * k.length_stride]);
        s.pos0 = s.filled - (int32_t)L - k.after;
        s.low0 = s.pos0 - k.window + 1;
    }
    return s;
}
struct Reach {
    int32_t first, lo, hi;
};
// of queries la .. lb
__device__ __forceinline__ Reach reach(const SpanBase& s, int32_t la, int32_t lb, int32_t sinks) {
    Reach r;
    r.hi = min(s.pos0 + lb, s.filled - 1);
    r.lo = max(0, s.low0 + la);
    r.first = max(0, min(min(sinks, r.lo), r.hi + 1));
    return r;
}

// What a key range leaves for a query row: O[D] = sum P V unnormalised, and a
// head {base, l}, l = sum P, base the log2 reference of P's exponentials
// (l = 0: no key seen).  Joined, with M the largest base of those with l > 0:
// O = sum O_r 2^(base_r - M) / sum l_r 2^(base_r - M).

// --------------------------------------------------------- tcgen05 tiles
//
// A tile is up to 128 query rows that share a key/value head: GB query heads
// x LB consecutive queries x NB sequences, gathered by one 4-D TMA box over
// {depth, heads, queries, batch}, so that grouped heads share the key tiles
// whatever Q's strides are.  A work item is two tiles and the key tiles that
// either sees; a tile of rows takes part only in the key tiles that it sees.
// CTAs are persistent, one per SM: the next item's loads start while this
// one's last products and epilogue run.  An item costs 5.8k cycles besides its
// key tiles (the epilogue 3k, the last product 0.9k, masks 1k per edge; 22k
// when each item was a CTA), a key tile 3.4k.
//   warp 0      TMA: both Q tiles, then K and V tiles of 128 keys through
//               rings of 2 (D = 128) or 4 (D = 64) slots
//   warp 2      the items' plans
//   warp 1      TMEM and MMA issue: S_t = Q_t K^T, O_t += P_t V, the two
//               tiles in turn so that one's products run during the other's
//               softmax; value rows that no query sees are zeroed in shared
//               memory first (a weight of 0 does not hide a NaN there)
//   warps 4-11  softmax, one query row per thread: lazy running maximum
//               (raised, and O rescaled, only past 2^8), P over S in TMEM; at
//               an item's end O / l, or a record, through shared memory and
//               TMA stores of 128 bytes per row
// P is handed over in two halves, so that the products of its first 64 keys run
// while the others' exponentials are taken (164 -> 149 us for 8192 queries,
// window 1024, 32/8 heads, D = 128).
// P is rounded to the operands' type, the only one the matrix unit takes beside
// V's.  With the output's own rounding it is the result's error: 0.0022 (BF16)
// and 2.9e-4 (F16) of the outputs' norm, 0.0016 and 2.1e-4 by the output alone.
// Bound: the chain of one tile's softmax (1850 cycles), the second half of its
// P V and its next S (800) and their hand-overs; the tensor pipe is busy 2100
// of a key tile's 3400 cycles.  8192 queries, 32/8 heads, D = 128, short runs of
// calls back to back: window 1024 149 us (860 TFLOP/s over the visible pairs),
// 4096 355 us (1170), no window 455 us (1210); in longer runs, under the power
// cap, window 1024 takes 166 to 170 us.
// Otherwise this is attn_fwd_kernel's pipeline; see there for the orderings and
// the bounded waits, and weight_shift for the scale of the weights.
struct SpanTileParams {
    uint32_t B, H, L, Lk;          // sequences, query heads, queries, keys per head
    uint32_t group;                // query heads per key/value head
    uint32_t GB, LB, NB, rows;     // the tile's box and its row count GB * LB * NB
    uint32_t l_tiles, tiles;       // tiles along the queries; tiles of one unit
    uint32_t units, groups, items; // units; pairs of tiles per unit; units x groups x splits
    uint32_t head_blocks;          // H / GB
    uint32_t shared_keys;          // 1: every row sees all Lk keys of batch 0 (the shared prefix)
    uint32_t k_batch_bcast, v_batch_bcast;
    SpanKeys keys;
    float scale_log2, shift;
    float hidden;                  // what a hidden key's raw score becomes: its logit is -inf whatever the scale's sign
    uint32_t splits;               // key ranges of a pair
    // Output: through tmO, a 5-D map {D, records, heads, queries, batch}; for
    // records (heads not null) the one at index first + split of each row, its
    // head at ((b * H + h) * L + l) * stride + first + split.
    float2* heads;
    uint32_t stride, first;
    uint32_t out_low;              // 16-bit output: FB_BF16 / FB_F16
};

template <int D>
struct TCfg {
    static constexpr int THREADS = 3 * 128;
    static constexpr int BOXES = D / 64;
    static constexpr int Q_BYTES = TQ * D * 2;
    static constexpr int K_BYTES = TK * D * 2;
    static constexpr int STAGE_BYTES = 2 * K_BYTES;
    static constexpr int STAGES = D == 64 ? 4 : 2;
    static constexpr int OUT_BYTES = TQ * 128;     // a tile's rows, 128 bytes of each on their way out
    static constexpr int SMEM = 1024 + 2 * Q_BYTES + STAGES * STAGE_BYTES + 2 * OUT_BYTES + 384;
    static __device__ __forceinline__ uint32_t s_col(int t) { return (uint32_t)(t * TK); }
    static __device__ __forceinline__ uint32_t o_col(int t) { return (uint32_t)(2 * TK + t * 128); }
};

// One work item: up to two tiles of a unit and one key range.  A warp of its
// own works it out and leaves it in shared memory, PLANS items ahead at most
// (its few hundred dependent integer instructions took the producer 10k cycles
// per item, most of what an item cost besides its key tiles).
//
// Its keys are numbered through: virtual key v is key v below `s16` (the first
// keys, rounded up to 16) and key v - s16 + lo from there on, lo the earliest
// window's start; where the two meet, s16 = lo = 0.  Virtual tiles hold 128
// virtual keys: the one that holds the border is gathered from 16-row boxes,
// the others are one box at any key, so the first keys cost no tile of their
// own and a window starts a tile.
constexpr int PLANS = 4;
struct TileItem {
    uint32_t split, head0, kv_head, unit_b;
    uint32_t b0[2], l0[2];          // first sequence and first query of each query tile
    bool real[2];
    uint32_t s16, lo;
    uint32_t j0, n_kv;              // this range of the virtual tiles
    // Query tile t sees n_t of them: those of index (from j0) below near[t],
    // then those from far[t] on.
    uint32_t n_t[2], near[2], far[2];
    SpanBase base;
    // Virtual keys that no query of the item sees although its tiles hold
    // them: [gap0, gap1), between the first keys and the window (under 16),
    // and those from stop on.  A weight of 0 does not make up for a NaN or an
    // infinity in their value rows.  Queries of other items may see some of
    // them; where the item's last tile holds only such (stop of 2^31 - 1), or
    // zeros past the tensor's end, they are left as they are.
    uint32_t gap0, gap1;
    int32_t stop;
    static __device__ __forceinline__ uint32_t after(uint32_t j, uint32_t near, uint32_t far) {
        return j + 1 < near ? j + 1 : max(j + 1, far);
    }
    // virtual key numbers of the keys from lo on: key + shift()
    __device__ __forceinline__ int32_t shift() const { return (int32_t)s16 - (int32_t)lo; }
    __device__ __forceinline__ void set(const SpanTileParams& p, uint32_t item) {
        // Last queries (the most keys under a long window) of every unit first.
        uint32_t rest = item;
        split = 0;
        if (p.splits > 1) rest = item / p.splits, split = item - rest * p.splits;
        const uint32_t rank = rest / p.units, unit = rest - rank * p.units, group = p.groups - 1 - rank;
        unit_b = unit / p.head_blocks;  // 0 with shared keys
        head0 = (unit - unit_b * p.head_blocks) * p.GB, kv_head = head0 / p.group;
        if (p.shared_keys) {  // every row of every tile sees all keys
            base = SpanBase{(int32_t)p.Lk, 0, 0};
            const uint32_t all = (p.Lk + TK - 1) / TK, per = p.splits > 1 ? (all + p.splits - 1) / p.splits : all;
            j0 = min(split * per, all);
            n_kv = min(per, all - j0);
            s16 = lo = 0;
            gap0 = gap1 = 0, stop = 0x7fffffff;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t tile = group * 2 + t;
                real[t] = tile < p.tiles;
                b0[t] = tile / p.l_tiles * p.NB, l0[t] = tile % p.l_tiles * p.LB;
                n_t[t] = real[t] ? n_kv : 0, near[t] = 0, far[t] = 0;
            }
            return;
        }
        base = span_base(p.keys, unit_b, p.L, p.Lk);
        Reach rc[2];
        int32_t first = 0, start = 0x7fffffff, last = -1;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t tile = group * 2 + t;
            real[t] = tile < p.tiles;
            b0[t] = unit_b, l0[t] = tile * p.LB;
            rc[t] = Reach{0, 0, -1};
            if (!real[t]) continue;
            rc[t] = reach(base, (int32_t)l0[t], (int32_t)min(l0[t] + p.LB, p.L) - 1, p.keys.sinks);
            if (rc[t].hi < 0) continue;
            first = max(first, rc[t].first);
            if (rc[t].lo <= rc[t].hi) start = min(start, rc[t].lo), last = max(last, rc[t].hi);
        }
        uint32_t s = (uint32_t)(first + 15) / 16 * 16, end;
        gap0 = gap1 = (uint32_t)first;
        if (last < 0) {  // the first keys alone
            s = 0, start = 0, end = (uint32_t)first;
        } else if ((uint32_t)start <= s) {  // one run
            gap1 = (uint32_t)max(first, start);
            s = 0, start = 0, end = (uint32_t)last + 1;
        } else {
            gap1 = s;
            end = s + (uint32_t)(last - start) + 1;
        }
        if (base.low0 <= first) gap1 = gap0;  // the call's earliest window reaches down to the first keys
        s16 = s, lo = (uint32_t)start;
        const int32_t seen = last < 0 ? first : min(base.filled, base.pos0 + (int32_t)p.L);
        stop = seen < (int32_t)p.Lk ? seen + shift() : 0x7fffffff;
        const uint32_t all = (end + TK - 1) / TK, per = p.splits > 1 ? (all + p.splits - 1) / p.splits : all;
        j0 = min(split * per, all);
        const uint32_t j1 = min(j0 + per, all);
        n_kv = j1 - j0;
        auto overlap = [&](uint32_t x0, uint32_t x1) {
            const uint32_t y0 = max(x0, j0), y1 = min(x1, j1);
            return y1 > y0 ? y1 - y0 : 0u;
        };
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            uint32_t ns = 0, a0 = 0, e = 0;
            if (rc[t].hi >= 0) {
                ns = (uint32_t)(rc[t].first + TK - 1) / TK;
                if (rc[t].lo <= rc[t].hi) {
                    a0 = max(((uint32_t)(rc[t].lo - start) + s) / TK, ns);
                    e = max(((uint32_t)(rc[t].hi - start) + s) / TK + 1, a0);
                }
            }
            n_t[t] = overlap(0, ns) + overlap(a0, e);
            near[t] = overlap(0, ns), far[t] = max(a0, j0) - j0;
        }
    }
};

// Whether `v` holds in all 128 threads of named barrier `id`.
__device__ __forceinline__ bool tile_all(int id, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred q, a;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.and.pred a, %2, 128, q;\n\tselp.u32 %0, 1, 0, a;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(id)
        : "memory");
    return r != 0;
}

// TMA tensor store shared -> global through a 5-D map; elements outside the
// map's extents are not written.
__device__ __forceinline__ void tma_store_5d(const CUtensorMap* map, int32_t x, int32_t y, int32_t z, int32_t w, int32_t v,
                                             const void* src) {
    asm volatile("cp.async.bulk.tensor.5d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4, %5}], [%6];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(smem_u32(src))
                 : "memory");
}

// acc + the two 16-bit weights of a packed word, each sum in f32.
template <int FMT>
__device__ __forceinline__ float2 add_weights(float2 acc, uint32_t w) {
    if constexpr (FMT == 1)
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.rn.f32.bf16 %0, l, %0;\n\tadd.rn.f32.bf16 %1, h, %1;\n\t}"
            : "+f"(acc.x), "+f"(acc.y)
            : "r"(w));
    else
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tadd.rn.f32.f16 %0, l, %0;\n\tadd.rn.f32.f16 %1, h, %1;\n\t}"
            : "+f"(acc.x), "+f"(acc.y)
            : "r"(w));
    return acc;
}

__device__ __forceinline__ void prefetch_tensormap(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

template <int D, int FMT>
__global__ void __launch_bounds__(TCfg<D>::THREADS, 1) span_tile_kernel(const __grid_constant__ CUtensorMap tmQ,
                                                                       const __grid_constant__ CUtensorMap tmK,
                                                                       const __grid_constant__ CUtensorMap tmV,
                                                                       const __grid_constant__ CUtensorMap tmK16,
                                                                       const __grid_constant__ CUtensorMap tmV16,
                                                                       const __grid_constant__ CUtensorMap tmO, SpanTileParams p) {
    using C = TCfg<D>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sQ = smem;
    unsigned char* sKV = sQ + 2 * C::Q_BYTES;
    unsigned char* sOut = sKV + C::STAGES * C::STAGE_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sOut + 2 * C::OUT_BYTES);
    uint64_t* k_full = bars;
    uint64_t* k_empty = k_full + C::STAGES;
    uint64_t* v_full = k_empty + C::STAGES;
    uint64_t* v_empty = v_full + C::STAGES;
    uint64_t* q_full = v_empty + C::STAGES;   // [2]
    uint64_t* q_empty = q_full + 2;
    uint64_t* s_full = q_empty + 2;
    uint64_t* p_full = s_full + 2;
    uint64_t* o_done = p_full + 2;
    uint64_t* o_free = o_done + 2;            // O read out of TMEM
    uint64_t* plan_full = o_free + 2;         // [PLANS]
    uint64_t* plan_empty = plan_full + PLANS;
    uint64_t* p_half = plan_empty + PLANS;    // [2]: P of the first 64 keys is written
    uint64_t* drain = p_half + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    __shared__ TileItem plans[PLANS];
    // Item i of this CTA: rounds over the grid run back and forth, so that no
    // CTA gets the longest item of every round.
    auto item_at = [&](uint32_t i) { return i * gridDim.x + (i & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x); };

    // The launch that follows may start while this one ends (where it was made
    // so); it waits for this grid's results itself.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&q_full[t], 1);
            mbar_init(&q_empty[t], 1);
            mbar_init(&s_full[t], 1);
            mbar_init(&p_half[t], 4);
            mbar_init(&p_full[t], 4);
            mbar_init(&o_done[t], 1);
            mbar_init(&o_free[t], 128);
        }
        for (int i = 0; i < PLANS; ++i) {
            mbar_init(&plan_full[i], 1);
            mbar_init(&plan_empty[i], 10);  // the loading, issuing and softmax warps
        }
        mbar_init(drain, 1);
        fence_barrier_init();
    }
    if (warp == 3 && lane == 0) {
        prefetch_tensormap(&tmQ);
        prefetch_tensormap(&tmK);
        prefetch_tensormap(&tmV);
        prefetch_tensormap(&tmO);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (warp == 2 && lane == 0 && item_at(0) < p.items) plans[0].set(p, item_at(0));
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Registers: the block has 3 x 128 x 168; the first four warps keep 104 each
    // thread and the softmax groups take 200 (104 + 2 x 200 = 3 x 168), which
    // holds a row of 128 scores without spills.
    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 0 && lane == 0) {
        // ------------------------------------------------ TMA producer
        // Loads of an item's tiles start as soon as the items before it have
        // left the buffers: Q_t once its last S_t is computed, K and V through
        // rings that run on across items (g: ring index of the next K / V).
        uint32_t g = 0, q_loads[2] = {0, 0};
        uint32_t issued_k = 0, issued_v = 0;
        bool failed = false;
        for (uint32_t i = 0; item_at(i) < p.items && !failed; ++i) {
            if (!mbar_wait(&plan_full[i % PLANS], (i / PLANS) & 1)) {
                failed = true;
                break;
            }
            const TileItem& it = plans[i % PLANS];
            const int32_t k_b = p.shared_keys || p.k_batch_bcast ? 0 : (int32_t)it.unit_b;
            const int32_t v_b = p.shared_keys || p.v_batch_bcast ? 0 : (int32_t)it.unit_b;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (it.n_t[t] == 0 || failed) continue;
                if (!mbar_wait(&q_empty[t], (q_loads[t] & 1) ^ 1)) {
                    failed = true;
                    break;
                }
                mbar_arrive_expect_tx(&q_full[t], p.rows * (uint32_t)(D * 2));
                for (int b = 0; b < C::BOXES; ++b)
                    tma_load_4d(sQ + t * C::Q_BYTES + b * (TQ * 128), &tmQ, b * 64, (int32_t)it.head0, (int32_t)it.l0[t],
                                (int32_t)it.b0[t], &q_full[t]);
                ++q_loads[t];
            }
            for (uint32_t j = 0; j < it.n_kv && !failed; ++j, ++g) {
                const uint32_t s = g % C::STAGES, ph = ((g / C::STAGES) & 1) ^ 1;
                const uint32_t v0 = (it.j0 + j) * TK;  // virtual tile's first key
                const bool border = v0 < it.s16 && v0 + TK > it.s16;
                const int32_t key = (int32_t)(v0 < it.s16 ? v0 : v0 - it.s16 + it.lo);
                auto load = [&](unsigned char* dst, const CUtensorMap* tm, const CUtensorMap* tm16, int32_t batch, uint64_t* bar) {
                    mbar_arrive_expect_tx(bar, C::K_BYTES);
                    for (int b = 0; b < C::BOXES; ++b) {
                        if (!border) {
                            tma_load_4d(dst + b * (TK * 128), tm, b * 64, key, (int32_t)it.kv_head, batch, bar);
                            continue;
                        }
                        for (uint32_t r = 0; r < TK; r += 16) {
                            const uint32_t v = v0 + r;
                            tma_load_4d(dst + b * (TK * 128) + r * 128, tm16, b * 64, (int32_t)(v < it.s16 ? v : v - it.s16 + it.lo),
                                        (int32_t)it.kv_head, batch, bar);
                        }
                    }
                };
                unsigned char* kd = sKV + s * C::STAGE_BYTES;
                if (!mbar_wait(&k_empty[s], ph)) {
                    failed = true;
                    break;
                }
                load(kd, &tmK, &tmK16, k_b, &k_full[s]);
                ++issued_k;
                if (!mbar_wait(&v_empty[s], ph)) {
                    failed = true;
                    break;
                }
                load(kd + C::K_BYTES, &tmV, &tmV16, v_b, &v_full[s]);
                ++issued_v;
            }
            mbar_arrive(&plan_empty[i % PLANS]);
        }
        // the copies still in flight land (bounded) before the block ends
        if (failed) atomicOr(&g_span_status, 1u << DEV_ATTN_TIMEOUT);
        for (uint32_t j = issued_k >= C::STAGES ? issued_k - C::STAGES : 0; failed && j < issued_k; ++j)
            (void)mbar_wait(&k_full[j % C::STAGES], (j / C::STAGES) & 1);
        for (uint32_t j = issued_v >= C::STAGES ? issued_v - C::STAGES : 0; failed && j < issued_v; ++j)
            (void)mbar_wait(&v_full[j % C::STAGES], (j / C::STAGES) & 1);
        for (int t = 0; t < 2 && failed; ++t)
            if (q_loads[t]) (void)mbar_wait(&q_full[t], (q_loads[t] - 1) & 1);
    } else if (warp == 2 && lane == 0) {
        // ------------------------------------------------ planner
        for (uint32_t i = 0, item; (item = item_at(i)) < p.items; ++i) {
            if (!mbar_wait(&plan_empty[i % PLANS], ((i / PLANS) & 1) ^ 1)) {
                atomicOr(&g_span_status, 1u << DEV_ATTN_TIMEOUT);
                break;
            }
            if (i > 0) plans[i % PLANS].set(p, item);  // (the first was made above)
            mbar_arrive(&plan_full[i % PLANS]);
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        const uint32_t idesc_s = f16_idesc(FMT, TQ, TK);
        const uint32_t idesc_o = f16_idesc(FMT, TQ, D) | (1u << 16);  // B (V) is MN-major
        auto wait = [](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); };
        // Descriptors are made where they are used: kept over the loop they
        // would take more registers than there are.
        auto opaque = [](uint32_t v) {
            asm volatile("" : "+r"(v));
            return v;
        };
        bool ok = true;
        // g: ring index of the item's first K / V; taken: S_t / PV_t pairs so
        // far; outs: items in which tile t had any
        uint32_t g = 0, taken[2] = {0, 0}, outs[2] = {0, 0};
        for (uint32_t n = 0; item_at(n) < p.items; ++n) {
            if (!(ok = ok && wait(&plan_full[n % PLANS], (n / PLANS) & 1))) break;
            const TileItem& it = plans[n % PLANS];
            const uint32_t n_kv = it.n_kv, n_t[2] = {it.n_t[0], it.n_t[1]}, near[2] = {it.near[0], it.near[1]},
                           far[2] = {it.far[0], it.far[1]};
            const bool gap = it.gap1 > it.gap0;
            // left: S_t still to come in this item
            auto issue_s = [&](int t, uint32_t j, uint32_t left) -> bool {
                const uint32_t s = (g + j) % C::STAGES;
                if (!wait(&k_full[s], ((g + j) / C::STAGES) & 1)) return false;
                tc_fence_after();
                const uint64_t qd = sw128_desc(opaque(smem_u32(sQ + t * C::Q_BYTES)));
                const uint64_t kd = sw128_desc(opaque(smem_u32(sKV + s * C::STAGE_BYTES)));
                const uint32_t d = tmem + C::s_col(t);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = (uint32_t)((k / 4) * (TQ * 128) + (k % 4) * 32);
                    umma_f16_ss_warp(d, desc_add(qd, off), desc_add(kd, off), idesc_s, k != 0);
                }
                umma_commit_warp(&s_full[t]);
                if (left == 0) umma_commit_warp(&q_empty[t]);
                return true;
            };
            auto issue_pv = [&](int t, uint32_t j, uint32_t i) -> bool {
                const uint32_t s = (g + j) % C::STAGES;
                if (!wait(&p_half[t], taken[t] & 1)) return false;
                // the first product of an item overwrites O_t: the item
                // before it must have been read out
                if (i == 0 && !wait(&o_free[t], (outs[t] & 1) ^ 1)) return false;
                tc_fence_after();
                const uint64_t vd = sw128_mn_desc(opaque(smem_u32(sKV + s * C::STAGE_BYTES + C::K_BYTES)), TK * 128);
                const uint32_t d = tmem + C::o_col(t), a = tmem + C::s_col(t);
                umma_f16_ts_warp(d, a, vd, idesc_o, i != 0);
#pragma unroll
                for (int k = 1; k < TK / 16; ++k) {
                    if (k == TK / 32) {  // the second 64 keys' weights
                        if (!wait(&p_full[t], taken[t] & 1)) return false;
                        tc_fence_after();
                    }
                    umma_f16_ts_warp(d, a + k * 8, desc_add(vd, k * 16 * 128), idesc_o, 1u);
                }
                if (i + 1 == n_t[t]) {
                    umma_commit_warp(&o_done[t]);
                    ++outs[t];
                }
                ++taken[t];
                return true;
            };
            uint32_t at[2], done[2] = {0, 0};
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                at[t] = n_t[t] ? (near[t] ? 0 : far[t]) : n_kv;
                if (!ok || at[t] >= n_kv) continue;
                ok = wait(&q_full[t], outs[t] & 1) && issue_s(t, at[t], n_t[t] - 1);
            }
            if (ok && n_kv > 0) umma_commit_warp(&k_empty[g % C::STAGES]);  // the first K consumed by every S of it
            for (uint32_t j = 0; ok && j < n_kv; ++j) {
                const uint32_t s = (g + j) % C::STAGES;
                ok = wait(&v_full[s], ((g + j) / C::STAGES) & 1);
                if (ok && ((gap && it.gap0 / TK == it.j0 + j) || (j + 1 == n_kv && it.stop < (int32_t)((it.j0 + n_kv) * TK)))) {
                    // value rows that no query of the item sees: zeros
                    const uint32_t v0 = (it.j0 + j) * TK;
                    unsigned char* v = sKV + s * C::STAGE_BYTES + C::K_BYTES;
                    auto clear = [&](uint32_t from, uint32_t to) {
                        for (int b = 0; b < C::BOXES; ++b)
                            for (uint32_t o = from * 128 + lane * 16; o < to * 128; o += 512)
                                *reinterpret_cast<uint4*>(v + b * (TK * 128) + o) = make_uint4(0u, 0u, 0u, 0u);
                    };
                    if (gap && it.gap0 / TK == it.j0 + j) clear(it.gap0 - v0, min(it.gap1 - v0, (uint32_t)TK));
                    if (it.stop < (int32_t)(v0 + TK)) clear((uint32_t)max(it.stop - (int32_t)v0, 0), TK);
                    fence_proxy_async_smem();
                    __syncwarp();
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (!ok || at[t] != j) continue;
                    ok = issue_pv(t, j, done[t]);
                    ++done[t];
                    at[t] = done[t] < n_t[t] ? TileItem::after(j, near[t], far[t]) : n_kv;
                    if (ok && at[t] < n_kv) ok = issue_s(t, at[t], n_t[t] - done[t] - 1);
                }
                // V(j) is free once every PV(j) has completed, K(j + 1) once
                // every S(j + 1) has (each was issued by now)
                if (ok) umma_commit_warp(&v_empty[s]);
                if (ok && j + 1 < n_kv) umma_commit_warp(&k_empty[(g + j + 1) % C::STAGES]);
            }
            g += n_kv;
            __syncwarp();
            if (lane == 0) mbar_arrive(&plan_empty[n % PLANS]);
        }
        if (!ok && lane == 0) atomicOr(&g_span_status, 1u << DEV_ATTN_TIMEOUT);
        umma_commit_warp(drain);
        (void)wait(drain, 0);
    }
    } else {
        // ------------------------------------------------ softmax / epilogue
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int t = (warp - 4) / 4, quarter = warp & 3;
        const uint32_t row = (uint32_t)(quarter * 32 + lane);
        const uint32_t tm_s = tmem + ((uint32_t)(quarter * 32) << 16) + C::s_col(t);
        const uint32_t tm_o = tmem + ((uint32_t)(quarter * 32) << 16) + C::o_col(t);
        const float NEG = -__int_as_float(0x7f800000);
        const float sl = p.scale_log2;
        // the row's place in the box: head, query and sequence, 8 bits each
        const uint32_t place = row % p.GB | row / p.GB % p.LB << 8 | row / (p.GB * p.LB) << 16;
        uint32_t steps = 0, outs = 0;  // S_t taken, items with any, over all items
        bool ok = true;
        for (uint32_t turn = 0; item_at(turn) < p.items; ++turn) {
            // (the tile's four warps go on or none does: they meet at barriers)
            if (!(ok = tile_all(1 + t, ok && mbar_wait(&plan_full[turn % PLANS], (turn / PLANS) & 1)))) {
                atomicOr(&g_span_status, 1u << DEV_ATTN_TIMEOUT);
                break;
            }
            const TileItem& it = plans[turn % PLANS];
            const uint32_t n = it.n_t[t];
            uint32_t j = it.near[t] ? 0 : it.far[t];  // this tile's key tiles, n in all
            // virtual keys of this row: below vsink, and [vlow, vhigh]
            int32_t vsink, vlow, vhigh;
            {
                const int32_t l = (int32_t)(it.l0[t] + (place >> 8 & 0xffu));
                const int32_t high = p.shared_keys ? (int32_t)p.Lk - 1 : max(-1, min(it.base.pos0 + l, it.base.filled - 1));
                vsink = p.shared_keys ? 0 : min(p.keys.sinks, high + 1);
                vlow = p.shared_keys ? 0 : max(0, min(0x3fffffff, it.base.low0 + l)) + it.shift();
                vhigh = high + it.shift();
            }
            float m_used = NEG;  // running max (log2 units)
            float lsum = 0.0f;
            for (uint32_t i = 0; i < n && ok; ++i, ++steps) {
                const int32_t v0 = (int32_t)((it.j0 + j) * TK);
                j = TileItem::after(j, it.near[t], it.far[t]);
                // Wait outcomes are made warp-uniform: tcgen05.ld/st are .sync.aligned.
                if (!__all_sync(0xffffffffu, mbar_wait(&s_full[t], steps & 1))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                float x[TK];
                {
                    uint32_t r[TK];
#pragma unroll
                    for (int c = 0; c < TK; c += 32) tmem_ld32(tm_s + c, *reinterpret_cast<uint32_t(*)[32]>(&r[c]));
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < TK; ++e) x[e] = __uint_as_float(r[e]);
                }
                // Hidden keys are masked in the raw scores, only in the tiles that
                // hold some: past the row's position or the filled keys, or between
                // the first keys and the window.  A word of bits per 32 keys says
                // which are seen; a warp's rows are neighbours, so most words are
                // whole in all of them.
                if (__any_sync(0xffffffffu, v0 + TK - 1 > vhigh || v0 < vlow)) {
                    auto below = [](int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
#pragma unroll
                    for (int c = 0; c < TK; c += 32) {
                        const uint32_t seen = below(vsink - v0 - c) | (below(vhigh + 1 - v0 - c) & ~below(vlow - v0 - c));
                        if (__any_sync(0xffffffffu, seen != 0xffffffffu)) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) x[c + e] = seen & (1u << e) ? x[c + e] : p.hidden;
                        }
                    }
                }
                if (sl == 0.0f) {  // logits 0, hidden keys stay -inf
#pragma unroll
                    for (int e = 0; e < TK; ++e) x[e] = x[e] == NEG ? NEG : 0.0f * x[e];
                }
                // Four chains of three-input extremes of the raw scores (the
                // logits' maximum is the minimum under a negative scale).
                float mx[4] = {x[0], x[1], x[2], x[3]};
                if (sl < 0.0f) {
#pragma unroll
                    for (int e = 4; e < TK - 4; e += 8)
#pragma unroll
                        for (int a = 0; a < 4; ++a) mx[a] = min3n(mx[a], x[e + 2 * a], x[e + 2 * a + 1]);
                    mx[0] = min3n(mx[0], x[TK - 4], x[TK - 3]);
                    mx[1] = min3n(mx[1], x[TK - 2], x[TK - 1]);
                } else {
#pragma unroll
                    for (int e = 4; e < TK - 4; e += 8)
#pragma unroll
                        for (int a = 0; a < 4; ++a) mx[a] = max3n(mx[a], x[e + 2 * a], x[e + 2 * a + 1]);
                    mx[0] = max3n(mx[0], x[TK - 4], x[TK - 3]);
                    mx[1] = max3n(mx[1], x[TK - 2], x[TK - 1]);
                }
                const float mul = sl == 0.0f ? 1.0f : sl;
                float mt = (sl < 0.0f ? min3n(min3n(mx[0], mx[1], mx[2]), mx[3], mx[3])
                                      : max3n(max3n(mx[0], mx[1], mx[2]), mx[3], mx[3])) * mul;
                float alpha = 1.0f;
                bool rescale = false;
                if (mt > m_used + 8.0f) {
                    alpha = m_used == NEG ? 0.0f : ex2(m_used - mt);
                    rescale = i > 0 && m_used != NEG;
                    m_used = mt;
                }
                if (__any_sync(0xffffffffu, rescale)) {
                    // O_t is quiescent: S_t of this step completed after PV_t
                    // of the last, and PV_t of this one waits for the arrivals.
                    const float f = rescale ? alpha : 1.0f;
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t r[32];
                        tmem_ld32(tm_o + c * 32, r);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * f);
                        tmem_st32(tm_o + c * 32, r);
                    }
                }
                const float ref = m_used == NEG ? 0.0f : m_used + p.shift;
                float2 lsa[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                // Packed pairs overwrite the scores they came from, so P needs no
                // registers of its own; one pair in eight takes the polynomial.
                // The row sum adds the weights as they were rounded, so that the
                // rounding of a dominant one cancels, after the hand-over and with
                // adds that widen their 16-bit operand (unpacking them first: 149
                // -> 165 us for 8192 queries, window 1024).
                uint32_t* xb = reinterpret_cast<uint32_t*>(x);
                const float2 sl2 = make_float2(mul, mul), nb2 = make_float2(-ref, -ref);
#pragma unroll
                for (int c = 0; c < TK / 32; ++c) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float2 z = __ffma2_rn(make_float2(x[c * 32 + 2 * e], x[c * 32 + 2 * e + 1]), sl2, nb2);
                        const float2 w = (e & 7) == 7 ? ex2_poly2(z) : make_float2(ex2(z.x), ex2(z.y));
                        xb[c * 32 + e] = pack2(w.x, w.y, FMT);
                    }
                    tmem_st16(tm_s + c * 16, *reinterpret_cast<const uint32_t(*)[16]>(&xb[c * 32]));
                    if (c == TK / 64 - 1) {  // half of P: its products may start
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_half[t]);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
#pragma unroll
                for (int e = 0; e < TK / 2; ++e) lsa[e & 3] = add_weights<FMT>(lsa[e & 3], xb[(e / 16) * 32 + e % 16]);
                const float2 l2 = __fadd2_rn(__fadd2_rn(lsa[0], lsa[1]), __fadd2_rn(lsa[2], lsa[3]));
                lsum = lsum * alpha + (l2.x + l2.y);
            }
            if (ok && n > 0 && !__all_sync(0xffffffffu, mbar_wait(&o_done[t], outs & 1))) ok = false;
            if (!ok) atomicOr(&g_span_status, 1u << DEV_ATTN_TIMEOUT);
            tc_fence_after();
            const bool load = ok && n > 0;
            const bool real = it.real[t];
            const uint32_t head0 = it.head0, l0 = it.l0[t], b0 = it.b0[t], record = p.first + it.split;
            float inv = load && (lsum > 0.0f || lsum != lsum) ? 1.0f / lsum : 0.0f;
            if (p.heads) {
                inv = 1.0f;
                const uint32_t head = head0 + (place & 0xffu), l = l0 + (place >> 8 & 0xffu), b = b0 + (place >> 16);
                if (real && row < p.rows && l < p.L && b < p.B)
                    p.heads[(((uint64_t)b * p.H + head) * p.L + l) * p.stride + record] =
                        make_float2(m_used == NEG ? 0.0f : m_used + p.shift, load ? lsum : 0.0f);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&plan_empty[turn % PLANS]);  // the plan is no longer needed
            // 128 bytes of every row at a time: staged in shared memory under
            // the map's swizzle, written by one TMA store per tile.  (Stores
            // from registers, one row per lane, hold the load/store unit for a
            // line per lane: 6k to 9k cycles per tile against 2k.)
            const uint32_t step = p.out_low ? 64 : 32;  // columns
            unsigned char* stage = sOut + t * C::OUT_BYTES;
            const uint32_t swz = row & 7u;
#pragma unroll 1
            for (uint32_t c = 0; c < (uint32_t)D; c += step) {
                // the staged bytes of the store before this one have been read
                if (threadIdx.x % 128 == 0) bulk_wait_read_all();
                asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (h * 32 >= (int)step) break;
                    uint32_t r[32];
                    if (load) {
                        tmem_ld32(tm_o + c + h * 32, r);
                        tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) r[e] = 0u;
                    }
                    if (p.out_low) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            uint32_t w[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                w[k] = pack2(__uint_as_float(r[8 * e + 2 * k]) * inv, __uint_as_float(r[8 * e + 2 * k + 1]) * inv, FMT);
                            *reinterpret_cast<uint4*>(stage + row * 128 + (((uint32_t)(h * 4 + e) ^ swz) * 16)) =
                                make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            *reinterpret_cast<float4*>(stage + row * 128 + (((uint32_t)e ^ swz) * 16)) =
                                make_float4(__uint_as_float(r[4 * e]) * inv, __uint_as_float(r[4 * e + 1]) * inv,
                                            __uint_as_float(r[4 * e + 2]) * inv, __uint_as_float(r[4 * e + 3]) * inv);
                    }
                }
                if (c + step == (uint32_t)D && load) {
                    tc_fence_before();
                    mbar_arrive(&o_free[t]);  // O_t is out of TMEM
                }
                fence_proxy_async_smem();  // the staged rows are visible to the TMA store
                asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory");
                if (threadIdx.x % 128 == 0 && real) {
                    tma_store_5d(&tmO, (int32_t)c, (int32_t)record, (int32_t)head0, (int32_t)l0, (int32_t)b0, stage);
                    bulk_commit_group();
                }
            }
            if (n > 0) ++outs;
        }
        if (threadIdx.x % 128 == 0) bulk_wait_read_all();  // shared memory stays valid until the stores have read it
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // in a chain: ends after the launch before it
}

// ------------------------------------------------------ joining records

template <int D>
struct RowPiece {  // the D / 32 columns lane * D / 32 .. of one row
    static constexpr int N = D / 32;
    float v[N];
};
template <int D>
__device__ __forceinline__ RowPiece<D> load_piece(const float* row, uint32_t lane) {
    RowPiece<D> r;
    if constexpr (D == 128) {
        const float4 f = __ldcg(reinterpret_cast<const float4*>(row) + lane);
        r.v[0] = f.x, r.v[1] = f.y, r.v[2] = f.z, r.v[3] = f.w;
    } else {
        const float2 f = __ldcg(reinterpret_cast<const float2*>(row) + lane);
        r.v[0] = f.x, r.v[1] = f.y;
    }
    return r;
}
template <int D>
__device__ __forceinline__ void store_piece(void* out, uint32_t out_low, uint64_t row_at, uint32_t lane, const float (&o)[D / 32],
                                            float inv) {
    const uint64_t at = row_at + lane * (D / 32);
    if (out_low) {
        uint16_t* d = static_cast<uint16_t*>(out) + at;
#pragma unroll
        for (int i = 0; i < D / 32; i += 2)
            *reinterpret_cast<uint32_t*>(d + i) = encode_low_pair(o[i] * inv, o[i + 1] * inv, out_low);
    } else {
        float* d = static_cast<float*>(out) + at;
#pragma unroll
        for (int i = 0; i < D / 32; i += 2) *reinterpret_cast<float2*>(d + i) = make_float2(o[i] * inv, o[i + 1] * inv);
    }
}

// A warp joins the records 0 .. n - 1 of one row, in order, to the state
// {M, L, o} it has (L = 0: nothing yet); head(i) and row(i) are where record i
// lies.  Eight records at a time, all their loads in flight together.
template <int D, typename Head, typename Row>
__device__ __forceinline__ void join_records(uint32_t n, Head head, Row row, float& M, float& L, float (&o)[D / 32]) {
    const uint32_t lane = threadIdx.x & 31;
    const float NEG = -__int_as_float(0x7f800000);
    for (uint32_t i0 = 0; i0 < n; i0 += 8) {
        const uint32_t m = min(n - i0, 8u);
        float2 h = make_float2(0.0f, 0.0f);
        if (lane < m) h = __ldcg(head(i0 + lane));
        RowPiece<D> r[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e)
            if (e < m) r[e] = load_piece<D>(row(i0 + e), lane);
        float top = h.y == 0.0f ? NEG : h.x;
#pragma unroll
        for (int x = 4; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        top = fmaxf(__shfl_sync(0xffffffffu, top, 0), L == 0.0f ? NEG : M);
        if (top == NEG) continue;
        const float keep = L == 0.0f ? 0.0f : exp2f(M - top);
        L *= keep;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] *= keep;
        M = top;
        const float w = h.y == 0.0f ? 0.0f : exp2f(h.x - M), lw = h.y * w;
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            if (e >= m) break;
            const float we = __shfl_sync(0xffffffffu, w, e);
            L += __shfl_sync(0xffffffffu, lw, e);
            if (we == 0.0f) continue;  // nothing seen, or underflow: O is not multiplied by 0
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] = fmaf(r[e].v[i], we, o[i]);
        }
    }
}
__device__ __forceinline__ float inverse(float l) { return l > 0.0f || l != l ? 1.0f / l : 0.0f; }

// One warp per row.
struct SpanMergeParams {
    const float2* heads;
    const float* part;
    uint64_t rows;
    uint32_t count, H, L;
    void* out;
    uint32_t out_low;
    uint64_t o_sb, o_sh, o_sl;
};

// A row of records per warp.  Bound: L2, each record read once; 16 x 33 queries
// of 32 heads, D = 128, three records each (26 MB): 10 us by itself, of which the
// launch before hides the start.
template <int D>
__global__ void __launch_bounds__(256) span_merge_kernel(SpanMergeParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the records are written
    const uint64_t w = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (w >= p.rows) return;
    float M = -__int_as_float(0x7f800000), L = 0.0f, o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = 0.0f;
    const float2* heads = p.heads + w * p.count;
    const float* part = p.part + w * p.count * D;
    join_records<D>(p.count, [&](uint32_t i) { return heads + i; }, [&](uint32_t i) { return part + i * D; }, M, L, o);
    const uint64_t q = w % p.L, h = w / p.L % p.H, b = w / p.L / p.H;
    store_piece<D>(p.out, p.out_low, b * p.o_sb + h * p.o_sh + q * p.o_sl, threadIdx.x & 31, o, inverse(L));
}

// ---------------------------------------------------------- few query rows
//
// At most 16 query rows share a key/value head (G x L): one 16-row block of
// warp-level MMAs (m16n8k16) per (sequence, key/value head), as in
// attn_decode16_kernel (see there for the depth permutation and the combine),
// over exactly the keys that the rows see: virtual key v of a sequence is key
// v < s ? v : v + lo - s, with s first keys and the window [lo, hi].  Weights are
// rounded and summed as span_tile_kernel's.
//
// Work split: the visible keys of all (sequence, key/value head) units, in
// 64-key tiles, are dealt out evenly: CTA c takes the tiles [c q, (c + 1) q)
// of their concatenation, whatever unit borders fall inside, so that ragged
// lengths and unit counts that do not divide the GPU leave no SM idle.  Each
// CTA finds its first unit from a block scan over the lengths.  Per unit that
// a CTA enters, its NW warps take a share of the keys each through
// three-stage cp.async rings and combine in shared memory.  A unit inside one
// CTA is finished there; otherwise its CTAs leave records and the last to
// arrive (a counter per unit, reset by it) joins them in CTA order, so results
// do not depend on who is last.  After a span_tile_kernel over a shared prefix
// the launch overlaps that kernel (programmatic dependent launch) on the SMs it
// leaves free; its records are joined at the same place where all CTAs fit
// there, else by a launch of their own (waiting CTAs would keep others out).
// Bound: HBM, the visible keys and values once: 16 sequences, 32/8 heads, D =
// 128, window 16384: 178 us, 6.0 TB/s; window 4096 55 us, 4.9 TB/s.  Single users
// are bound by latency, and by the 50 GB/s that one SM draws: 260 keys 9.4 us.
// (Clusters of CTAs per short unit, joined through distributed shared memory,
// took 504 keys from 12.4 to 10.0 us but 260 keys from 9.4 to 9.7 and long streams 1%
// up; three stages in flight instead of two made long streams 2% slower.)
constexpr int DTILE = 64;  // keys

struct SpanDecodeParams {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint64_t q_sb, q_sh, q_sl, k_sb, k_sh, k_sk, v_sb, v_sh, v_sk;
    uint32_t B, H, Hkv, G, L, Lk;
    SpanKeys keys;
    float scale_log2, shift;
    uint32_t whole_units; // 1: CTA i takes all of unit i
    float2* part_heads;   // two records x 16 rows per CTA
    float* part;
    uint32_t* arrived;    // per unit, 0 between launches
    // Records of the shared prefix, ((b * H + h) * L + l) * records + i, or null:
    // the first `records` are joined here (join), or this kernel's results
    // become the last of them and another launch joins all.
    float2* prefix_heads;
    float* prefix;
    uint32_t records, join;
    void* out;
    uint32_t out_low;
    uint64_t o_sb, o_sh, o_sl;
};

struct UnitKeys {
    SpanBase base;
    uint32_t s, lo, count;    // first keys, window start, visible keys
    uint32_t tiles;           // at least 1, so that every unit has a CTA
};
__device__ __forceinline__ UnitKeys unit_keys(const SpanDecodeParams& p, uint32_t b) {
    UnitKeys u;
    u.base = span_base(p.keys, b, p.L, p.Lk);
    const Reach r = reach(u.base, 0, (int32_t)p.L - 1, p.keys.sinks);
    u.s = (uint32_t)r.first;
    u.lo = min((uint32_t)r.lo, p.Lk);
    u.count = u.s + (r.hi >= r.lo ? (uint32_t)(r.hi - r.lo + 1) : 0u);
    u.tiles = max(1u, (u.count + DTILE - 1) / DTILE);
    return u;
}

template <int D, int NW>  // NW warps
struct DCfg {
    static constexpr int CPR = D / 8;            // 16-byte chunks per K / V row
    static constexpr int STAGE = 2 * 16 * CPR;   // chunks per stage: 16 K rows, 16 V rows
    static constexpr int RING = DEC_STAGES * STAGE;
    static constexpr int SMEM = NW * RING * 16;
    static_assert(RING * 16 >= 16 * (2 * D + 2) * 4, "a warp's rows and the CTA's fit a ring");
};

template <int D, int FMT, int NW>
__global__ void __launch_bounds__(32 * NW) span_decode_kernel(SpanDecodeParams p) {
    using C = DCfg<D, NW>;
    constexpr int QW = D / 8, KS = D / 16, NJ = D / 8, CPR = C::CPR, STAGE = C::STAGE;
    extern __shared__ uint4 dsm[];
    __shared__ uint32_t scan[NW], found[2], last;
    __shared__ float2 heads[16];     // the CTA's combined records: heads; rows in `cmb`, the upper part of warp 0's ring
    __shared__ float wts[16][NW];    // the warps' weights in them
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, c = lane & 3;
    uint4* ring = dsm + (size_t)warp * C::RING;
    const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);
    float* cmb = reinterpret_cast<float*>(dsm) + 16 * (D + 2);
    const uint32_t R = p.G * p.L;
    const float NEG = -__int_as_float(0x7f800000);

    // This CTA's tiles and its first unit.
    uint32_t T, t_begin, b, hkv, tin;
    if (p.whole_units) {
        b = blockIdx.x / p.Hkv, hkv = blockIdx.x % p.Hkv, tin = 0;
        t_begin = 0, T = unit_keys(p, b).tiles;
    } else if (!p.keys.lengths) {
        const uint32_t tpu = unit_keys(p, 0).tiles;
        T = p.B * p.Hkv * tpu;
        const uint32_t q = (T + gridDim.x - 1) / gridDim.x;
        t_begin = blockIdx.x * q;
        b = t_begin / (tpu * p.Hkv), hkv = t_begin / tpu % p.Hkv, tin = t_begin % tpu;
    } else {
        const uint32_t per = (p.B + 32 * NW - 1) / (32 * NW);
        const uint32_t b0 = min(threadIdx.x * per, p.B), b1 = min(b0 + per, p.B);
        uint32_t mine = 0;
        for (uint32_t i = b0; i < b1; ++i) mine += unit_keys(p, i).tiles * p.Hkv;
        uint32_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        if (lane == 31) scan[warp] = incl;
        __syncthreads();
        uint32_t before = incl - mine;
        T = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            if (w < warp) before += scan[w];
            T += scan[w];
        }
        const uint32_t q = (T + gridDim.x - 1) / gridDim.x;
        t_begin = blockIdx.x * q;
        if (t_begin >= before && t_begin < before + mine) {
            uint32_t at = before, i = b0;
            for (; i + 1 < b1; ++i) {
                const uint32_t n = unit_keys(p, i).tiles * p.Hkv;
                if (t_begin < at + n) break;
                at += n;
            }
            found[0] = i, found[1] = t_begin - at;
        }
        __syncthreads();
        b = found[0];
        const uint32_t tpu = t_begin < T ? unit_keys(p, b).tiles : 1u;
        hkv = found[1] / tpu, tin = found[1] % tpu;
    }
    const uint32_t per_cta = p.whole_units ? T : (T + gridDim.x - 1) / gridDim.x;
    if (t_begin >= T) {
        if (p.prefix && blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const uint32_t t_end = min(t_begin + per_cta, T);

    for (uint32_t t = t_begin; t < t_end;) {
        const UnitKeys u = unit_keys(p, b);
        const uint32_t seg = min(u.tiles - tin, t_end - t);
        const uint32_t v_begin = tin * DTILE, v_end = min((tin + seg) * DTILE, u.count);
        const uint32_t quarter = ((v_end > v_begin ? v_end - v_begin : 0u) + 16 * NW - 1) / (16 * NW) * 16;
        const uint32_t k_begin = min(v_begin + warp * quarter, v_end), k_end = min(k_begin + quarter, v_end);
        // Q fragments of rows g and g + 8 (zeros past R); row r is query head r / L, query r % L
        uint32_t qa[2][QW];
        int32_t high[2], low[2];  // keys (sinks or [low, high]) of the rows
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            const uint32_t r = (uint32_t)(g + 8 * rr);
            const int32_t lq = (int32_t)(r % p.L);
            high[rr] = r < R ? max(-1, min(u.base.pos0 + lq, (int32_t)p.Lk)) : -1;
            low[rr] = max(0, u.base.low0 + lq);
            if (r < R) {
                const uint32_t h = hkv * p.G + r / p.L, l = r % p.L;
                const uint4* src = reinterpret_cast<const uint4*>(p.q + b * p.q_sb + h * p.q_sh + l * p.q_sl + c * (D / 4));
#pragma unroll
                for (int i = 0; i < QW / 4; ++i) {
                    const uint4 w = src[i];
                    qa[rr][4 * i] = w.x, qa[rr][4 * i + 1] = w.y, qa[rr][4 * i + 2] = w.z, qa[rr][4 * i + 3] = w.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < QW; ++i) qa[rr][i] = 0u;
            }
        }
        const uint32_t skip = u.lo - u.s;
        // Virtual keys [open, shut) are seen by every row: from the last
        // query's window on, up to the first query's position.
        const uint32_t last_low = (uint32_t)max((int32_t)u.lo, u.base.low0 + (int32_t)p.L - 1);
        const uint32_t open = last_low - skip, shut = (uint32_t)max(0, min((int32_t)k_end, u.base.pos0 + 1 - (int32_t)skip));
        const int32_t sinks = p.keys.sinks;
        const uint16_t* kbase = p.k + (uint64_t)b * p.k_sb + (uint64_t)hkv * p.k_sh;
        const uint16_t* vbase = p.v + (uint64_t)b * p.v_sb + (uint64_t)hkv * p.v_sh;
        // One stage: virtual keys v0 .. v0 + 15 of K then V, 16 bytes per copy.
        // Copy n of a lane is chunk lane % CPR of row lane / CPR + n * RPC.
        // Stages inside the window and the range step a pointer; the others
        // number each key, those past the range zero-filled (source size 0,
        // address in bounds).
        constexpr int RPC = 32 / CPR, COPIES = 16 / RPC;
        const uint32_t crow = (uint32_t)lane / CPR, chunk = (uint32_t)lane % CPR;
        const uint64_t k_step = (uint64_t)RPC * p.k_sk, v_step = (uint64_t)RPC * p.v_sk;
        auto issue = [&](uint32_t v0, int slot) {
            const uint32_t dst0 = ring_s + (uint32_t)(slot * STAGE * 16);
            if (v0 >= u.s && v0 + 16 <= k_end) {
                const uint16_t* ks = kbase + (uint64_t)(v0 + skip + crow) * p.k_sk + chunk * 8;
                const uint16_t* vs = vbase + (uint64_t)(v0 + skip + crow) * p.v_sk + chunk * 8;
#pragma unroll
                for (int n = 0; n < COPIES; ++n, ks += k_step)
                    cp_async16(dst0 + ((crow + n * RPC) * CPR + k_chunk<D>(crow + n * RPC, chunk)) * 16, ks, 16u);
#pragma unroll
                for (int n = 0; n < COPIES; ++n, vs += v_step)
                    cp_async16(dst0 + (16 * CPR + (crow + n * RPC) * CPR + v_chunk(crow + n * RPC, chunk)) * 16, vs, 16u);
                return;
            }
#pragma unroll
            for (int n = 0; n < 2 * COPIES; ++n) {
                const uint32_t kv = n / COPIES, row = crow + (n % COPIES) * RPC;
                const bool in = v0 + row < k_end;
                const uint32_t vk = in ? v0 + row : k_begin, key = vk < u.s ? vk : vk + skip;
                const uint16_t* src = kv ? vbase + (uint64_t)key * p.v_sk + chunk * 8 : kbase + (uint64_t)key * p.k_sk + chunk * 8;
                const uint32_t pc = kv ? v_chunk(row, chunk) : k_chunk<D>(row, chunk);
                cp_async16(dst0 + (kv * 16 * CPR + row * CPR + pc) * 16, src, in ? 16u : 0u);
            }
        };
        float o[NJ][4];
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        float m[2] = {NEG, NEG}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < DEC_STAGES - 1; ++st) {
            if (k_begin + 16 * st < k_end) issue(k_begin + 16 * st, st);
            cp_async_commit();
        }
        int slot = 0;
        for (uint32_t v0 = k_begin; v0 < k_end; v0 += 16) {
            cp_async_wait<DEC_STAGES - 2>();  // this stage's copies (all but the newest group) have landed
            __syncwarp();
            const uint4* kst = ring + slot * STAGE;
            const uint4* vst = kst + 16 * CPR;
            float s[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                uint32_t kw[QW];
                const uint32_t row = (uint32_t)(8 * n + g);
#pragma unroll
                for (int i = 0; i < QW / 4; ++i) {
                    const uint4 w = kst[row * CPR + k_chunk<D>(row, (uint32_t)(c * (QW / 4) + i))];
                    kw[4 * i] = w.x, kw[4 * i + 1] = w.y, kw[4 * i + 2] = w.z, kw[4 * i + 3] = w.w;
                }
                // two chains of dependent products instead of one
                float s2[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ks += 2) {
                    mma16816<FMT>(s[n], qa[0][2 * ks], qa[1][2 * ks], qa[0][2 * ks + 1], qa[1][2 * ks + 1], kw[2 * ks], kw[2 * ks + 1]);
                    mma16816<FMT>(s2, qa[0][2 * ks + 2], qa[1][2 * ks + 2], qa[0][2 * ks + 3], qa[1][2 * ks + 3], kw[2 * ks + 2],
                                  kw[2 * ks + 3]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] += s2[e];
            }
            // V words of keys 2c, 2c+1, 2c+8, 2c+9 at columns g*D/8 ..
            uint32_t vw[4][NJ / 2];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const uint32_t row = (uint32_t)(2 * c + (n & 1) + 8 * (n >> 1));
                if constexpr (NJ / 8 == 2) {
                    const uint32_t odd = (uint32_t)(g & 1);
                    const uint4 w0 = vst[row * CPR + v_chunk(row, (uint32_t)(2 * g) + odd)];
                    const uint4 w1 = vst[row * CPR + v_chunk(row, (uint32_t)(2 * g) + (odd ^ 1u))];
                    const uint4 lo = odd ? w1 : w0, hi = odd ? w0 : w1;
                    vw[n][0] = lo.x, vw[n][1] = lo.y, vw[n][2] = lo.z, vw[n][3] = lo.w;
                    vw[n][4] = hi.x, vw[n][5] = hi.y, vw[n][6] = hi.z, vw[n][7] = hi.w;
                } else {
                    const uint4 w = vst[row * CPR + v_chunk(row, (uint32_t)g)];
                    vw[n][0] = w.x, vw[n][1] = w.y, vw[n][2] = w.z, vw[n][3] = w.w;
                }
            }
            __syncwarp();  // every lane has read this slot: it may be refilled
            if (v0 + 16 * (DEC_STAGES - 1) < k_end) issue(v0 + 16 * (DEC_STAGES - 1), (slot + DEC_STAGES - 1) % DEC_STAGES);
            cp_async_commit();
            slot = slot + 1 == DEC_STAGES ? 0 : slot + 1;
            // scores in log2 units, masked: s[n][e] is row g + 8 * (e >> 1), virtual key v0 + 8n + 2c + (e & 1)
            float mx[2] = {NEG, NEG};
            if (v0 >= open && v0 + 16 <= shut) {  // seen by every row
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] *= p.scale_log2;
            } else {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int rr = e >> 1;
                        const uint32_t vk = v0 + 8 * n + 2 * c + (e & 1);
                        const int32_t key = (int32_t)(vk < u.s ? vk : vk + skip);
                        const bool seen = vk < k_end && key <= high[rr] && (key >= low[rr] || key < sinks);
                        s[n][e] = seen ? s[n][e] * p.scale_log2 : NEG;
                    }
            }
#pragma unroll
            for (int rr = 0; rr < 2; ++rr)
                mx[rr] = fmaxf(fmaxf(s[0][2 * rr], s[0][2 * rr + 1]), fmaxf(s[1][2 * rr], s[1][2 * rr + 1]));
            float alpha[2], base[2];
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
                mx[rr] = fmaxf(mx[rr], __shfl_xor_sync(0xffffffffu, mx[rr], 1));
                mx[rr] = fmaxf(mx[rr], __shfl_xor_sync(0xffffffffu, mx[rr], 2));
                const float mn = fmaxf(m[rr], mx[rr]);
                alpha[rr] = m[rr] == NEG ? 0.0f : ex2(m[rr] - mn);
                m[rr] = mn;
                base[rr] = mn == NEG ? 0.0f : mn + p.shift;
            }
            // P as the A operand of PV: rows g / g + 8, keys 2c, 2c+1 (tile 0) and 8 + 2c, 9 + 2c (tile 1)
            uint32_t pa[4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int rr = 0; rr < 2; ++rr)
                    pa[2 * n + rr] = pack2(ex2(s[n][2 * rr] - base[rr]), ex2(s[n][2 * rr + 1] - base[rr]), FMT);
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
                const float2 w0 = unpack2<FMT>(pa[rr]), w1 = unpack2<FMT>(pa[2 + rr]);
                l[rr] = fmaf(l[rr], alpha[rr], (w0.x + w0.y) + (w1.x + w1.y));
            }
            if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    o[j][0] *= alpha[0], o[j][1] *= alpha[0];
                    o[j][2] *= alpha[1], o[j][3] *= alpha[1];
                }
            }
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const uint32_t half = (j & 1) ? 0x7632u : 0x5410u;  // high or low 16-bit halves of the word pair
                const uint32_t b0 = __byte_perm(vw[0][j / 2], vw[1][j / 2], half);
                const uint32_t b1 = __byte_perm(vw[2][j / 2], vw[3][j / 2], half);
                mma16816<FMT>(o[j], pa[0], pa[1], pa[2], pa[3], b0, b1);
            }
        }
        cp_async_wait<0>();
        // The warps combine: each leaves {m, l, O} per row in its own (drained)
        // ring, then the CTA writes one record per row to `cmb`.
        float* xs = reinterpret_cast<float*>(ring);  // [16 rows][D + 2]
        __syncwarp();
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 1);
            l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 2);
            float* x = xs + (g + 8 * rr) * (D + 2);
            if (c == 0) {
                x[0] = m[rr];
                x[1] = l[rr];
            }
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                x[2 + 2 * c * NJ + j] = o[j][2 * rr];
                x[2 + (2 * c + 1) * NJ + j] = o[j][2 * rr + 1];
            }
        }
        __syncthreads();
        const bool whole = tin == 0 && seg == u.tiles;
        const uint64_t slot0 = ((uint64_t)blockIdx.x * 2 + (t == t_begin ? 0 : 1)) * 16;  // this segment's records
        auto warp_row = [&](uint32_t w, uint32_t r) { return reinterpret_cast<const float*>(dsm + (size_t)w * C::RING) + r * (D + 2); };
        if (threadIdx.x < R) {
            const uint32_t r = threadIdx.x;
            float M = NEG, Lr = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w)
                if (warp_row(w, r)[1] != 0.0f) M = fmaxf(M, warp_row(w, r)[0]);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float lw = warp_row(w, r)[1], wt = lw != 0.0f ? exp2f(warp_row(w, r)[0] - M) : 0.0f;
                wts[r][w] = wt;
                Lr = fmaf(lw, wt, Lr);
            }
            const float2 h = make_float2(M == NEG ? 0.0f : M + p.shift, Lr);
            if (whole) heads[r] = h;
            else p.part_heads[slot0 + r] = h;
        }
        __syncthreads();
        {
            float* rows = whole ? cmb : p.part + slot0 * D;
            for (uint32_t i = threadIdx.x; i < R * D; i += 32 * NW) {
                const uint32_t r = i / D, d = i % D;
                float acc = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; ++w)
                    if (wts[r][w] != 0.0f) acc = fmaf(warp_row(w, r)[2 + d], wts[r][w], acc);
                rows[i] = acc;
            }
        }
        // Which CTAs share the unit: those of its first and last tiles.
        const uint32_t u_begin = t - tin, c0 = u_begin / per_cta, c1 = (u_begin + u.tiles - 1) / per_cta;
        bool finish = whole;
        if (!whole) {
            __threadfence();  // this thread's record values before the arrival
            __syncthreads();
            if (threadIdx.x == 0) {
                uint32_t* at = p.arrived + (uint64_t)b * p.Hkv + hkv;
                const uint32_t n = atomicAdd(at, 1u);
                last = n == c1 - c0;
                if (last) *at = 0u;  // re-armed for the next launch
                __threadfence();
            }
            __syncthreads();
            finish = last;
        } else {
            __syncthreads();  // cmb
        }
        if (finish) {
            if (p.join) asm volatile("griddepcontrol.wait;" ::: "memory");  // the prefix's records are written
            for (uint32_t r = warp; r < R; r += NW) {
                float M = NEG, Lr = 0.0f, acc[D / 32];
#pragma unroll
                for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
                if (whole) {
                    M = heads[r].x, Lr = heads[r].y;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) acc[i] = cmb[r * D + lane * (D / 32) + i];
                } else {
                    // CTA c0 entered the unit as its first segment only if the
                    // unit begins at the CTA's first tile
                    const uint32_t second = u_begin == c0 * per_cta ? 0u : 1u;
                    auto place = [&](uint32_t i) { return ((uint64_t)(c0 + i) * 2 + (i == 0 ? second : 0u)) * 16 + r; };
                    join_records<D>(c1 - c0 + 1, [&](uint32_t i) { return p.part_heads + place(i); },
                                    [&](uint32_t i) { return p.part + place(i) * D; }, M, Lr, acc);
                }
                const uint32_t h = hkv * p.G + r / p.L, q = r % p.L;
                if (p.prefix) {
                    const uint64_t at = (((uint64_t)b * p.H + h) * p.L + q) * p.records;
                    if (!p.join) {
                        const uint64_t mine = at + p.records - 1;
                        if (lane == 0) p.prefix_heads[mine] = make_float2(M == NEG ? 0.0f : M, Lr);
                        store_piece<D>(p.prefix, 0, mine * D, lane, acc, 1.0f);
                        continue;
                    }
                    join_records<D>(p.records, [&](uint32_t i) { return p.prefix_heads + at + i; },
                                    [&](uint32_t i) { return p.prefix + (at + i) * D; }, M, Lr, acc);
                }
                store_piece<D>(p.out, p.out_low, (uint64_t)b * p.o_sb + (uint64_t)h * p.o_sh + (uint64_t)q * p.o_sl, lane, acc,
                               inverse(Lr));
            }
        }
        __syncthreads();  // the rings and cmb are free again
        t += seg;
        tin = 0;
        if (++hkv == p.Hkv) hkv = 0, ++b;
    }
    // One CTA that ends after the prefix's launch is enough for the grid to.
    if (p.prefix && blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ------------------------------------------------------------------ host

// A map {D, n...} with element strides s of the outer axes (unit axes: any)
// and 128-byte boxes {128 / esz, box...}; false when the
// strides or the base do not suit TMA.
template <int N>
bool span_map(CUtensorMap* map, const void* ptr, uint32_t dtype, uint64_t D, const uint64_t (&n)[N], const uint64_t (&s)[N],
              const uint32_t (&box)[N], bool promote) {
    auto enc = encode_tiled_attn();
    if (!enc || reinterpret_cast<uintptr_t>(ptr) % 16) return false;
    const uint64_t esz = dtype == FB_F32 ? 4 : 2;
    cuuint64_t dims[N + 1] = {D}, strides[N];
    cuuint32_t boxes[N + 1] = {(cuuint32_t)(128 / esz)}, estr[N + 1] = {1};
    uint64_t filler = (D * esz + 15) / 16 * 16;
    for (int i = 0; i < N; ++i) {
        uint64_t sb = s[i] * esz;
        if (n[i] == 0 || n[i] > (1ull << 31)) return false;
        if (n[i] == 1 && (sb == 0 || sb % 16 || sb >= (1ull << 40))) sb = filler;
        if (sb == 0 || sb % 16 || sb >= (1ull << 40)) return false;
        strides[i] = sb;
        dims[i + 1] = n[i], boxes[i + 1] = box[i], estr[i + 1] = 1;
        filler = (sb * n[i] + 15) / 16 * 16;
        if (filler >= (1ull << 40)) filler = 16;
    }
    const CUtensorMapDataType type = dtype == FB_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : dtype == FB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                        : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return enc(map, type, N + 1, const_cast<void*>(ptr), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, promote ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_NONE,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Operands of a call the tensor cores take: layouts with merged batch axes.
struct SpanOperands {
    RowsLayout q, k, v, o;
    uint64_t B, H, Hkv, L, Lk, G, D;
    uint32_t fmt;
    const void *qp, *kp, *vp;
    void* op;
};

// Weights are 2^(logit - reference - shift).  BF16: see attn_fwd_kernel.  F16
// holds nothing below 2^-25, and many keys that far below one add up (131072
// keys 18 nats below it are 0.2% of the row): a shift of -7 puts the largest
// weight, 2^8 past the reference at most, at 2^15, and keeps all keys down to
// 2^-32 of the row's largest.
float weight_shift(uint32_t fmt, uint64_t keys) {
    return fmt ? 9.0f + std::ceil(std::log2((float)std::max<uint64_t>(keys, 1))) : -7.0f;
}

// Most keys that one accumulator takes.  The matrix units align products to
// the accumulator and cut them off at 2^-25 of it, so n keys can leave up to
// n 2^-25 of a row out of O (measured with 16384 keys of weight 2^-18 to 2^-27
// beside one of 1: 2^-25.1 a key at most; below 2^-25 nothing of them arrives).
// At u 2^25 keys, u the type's unit roundoff (2^-8, 2^-11), that is u, no more than
// a weight's own rounding; longer ranges are divided and joined in f32.  (32/8 heads,
// D = 128, F16: a prompt of 32768 without a window 8.4 -> 9.1 ms, single tokens
// of 16 sequences of 65536 keys 681 -> 689 us.)
uint64_t range_keys(uint32_t fmt) { return fmt ? 131072 : 16384; }

uint64_t largest_divisor(uint64_t n, uint64_t most) {
    uint64_t d = std::min(n, most);
    while (n % d) --d;
    return d;
}

// How span_tile_kernel covers a call's query rows, and its key ranges.
struct TileGrid {
    uint64_t GB, LB, NB;     // the tile's box
    uint64_t tiles, units;   // tiles per unit
    uint64_t splits;
};

// The box: all heads of a group (their largest divisor up to 128) and, over
// the shared prefix, whose mask does not depend on the row, the LB queries x
// NB sequences that make the fewest tiles (33 queries of 16 sequences, groups
// of 4: 2 x 16, 17 tiles; 32 x 1 would make 32, half of them nearly empty).
// Key ranges when the pairs of tiles alone do not fill the GPU: about one CTA
// per SM, at least two key tiles each.  (A key tile takes a CTA 1.8 us with two
// tiles of rows and hardly less with one, so rows are always paired.)
// Where span_decode_kernel streams the own keys meanwhile (`streamed` bytes of
// them) on the SMs that the tiles leave free, the number of ranges that ends
// both soonest: a key tile next to that stream takes 2.2 us (5 us more for a CTA's start and end),
// the stream 5.8 TB/s, which 70% of the SMs keep up, a record a write and a read
// (64 sequences x 8192 shared keys + 512 own: 8 ranges, 64 CTAs, not 16).
TileGrid tile_grid(const SpanArgs& s, const SpanOperands& a, bool shared, double streamed = 0.0) {
    TileGrid g{};
    g.GB = largest_divisor(a.G, TQ);
    const uint64_t room = TQ / g.GB;
    g.LB = std::min(a.L, room), g.NB = 1;
    auto count = [&](uint64_t lb, uint64_t nb) { return (a.L + lb - 1) / lb * ((a.B + nb - 1) / nb); };
    if (shared) {
        for (uint64_t lb = 1; lb <= std::min(a.L, room); ++lb) {
            const uint64_t nb = std::min(a.B, room / lb);
            if (lb == 1 || count(lb, nb) < count(g.LB, g.NB)) g.LB = lb, g.NB = nb;
        }
    }
    g.tiles = shared ? count(g.LB, g.NB) : (a.L + g.LB - 1) / g.LB;
    g.units = a.H / g.GB * (shared ? 1 : a.B);
    uint64_t keys = ((shared ? s.prefix_keys : a.Lk) + TK - 1) / TK;  // tiles that a CTA walks at most
    if (!shared)
        keys = std::min(keys, (std::min(s.sinks, a.Lk) + std::min(s.window, a.Lk) + 2 * g.LB + 16 + TK - 1) / TK);
    const uint64_t sms = (uint64_t)sm_count();
    const uint64_t ctas = g.units * ((g.tiles + 1) / 2);
    const uint64_t most = range_keys(a.fmt) / TK, least = std::max<uint64_t>(1, (keys + most - 1) / most);
    g.splits = least;
    if (ctas < sms && keys >= 4) {
        const double stream = streamed / 5.8e6, record = (double)(a.B * a.H * a.L) * a.D * 8 / 5.0e6;
        double lowest = INFINITY;
        for (uint64_t want = least; want <= std::max(least, std::min<uint64_t>(sms / ctas, keys / 2)); ++want) {
            const uint64_t per = (keys + want - 1) / want, n = (keys + per - 1) / per;
            const double tiles = (double)per * 2.2 + 5.0, done = (double)(sms - std::min(sms, ctas * n)) * tiles;
            const double left = std::max(0.0, (stream * 0.7 * (double)sms - done) / (double)sms);
            const double cost = std::max(stream, tiles + left) + record * (double)n;
            if (cost < lowest) lowest = cost, g.splits = n;
        }
    }
    return g;
}

SpanKeys span_keys(const SpanArgs& s) {
    const int64_t big = 1ll << 30, far = 1ll << 40;  // (the window is at most 2^33)
    const int64_t pos0 = std::clamp(s.offset, -far, far), low0 = pos0 - (int64_t)s.window + 1;
    SpanKeys k{};
    k.pos0 = (int32_t)std::clamp(pos0, -big, big), k.low0 = (int32_t)std::clamp(low0, -big, big);
    k.window = (int32_t)std::min<uint64_t>(s.window, 1u << 30), k.sinks = (int32_t)std::min<uint64_t>(s.sinks, 1u << 30);
    k.after = (int32_t)s.after;
    k.lengths = s.lengths, k.length_stride = s.length_stride;
    return k;
}

// A launch that may begin while the stream's previous kernel ends (overlap):
// the kernel waits for it with griddepcontrol.wait before it touches anything
// that depends on it, and every one of a chain does so before it ends.
template <typename... P, typename... A>
void launch_after(void (*kernel)(P...), unsigned grid, unsigned threads, size_t smem, bool overlap, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap ? 1 : 0;
    (void)cudaLaunchKernelEx(&cfg, kernel, args...);
}

constexpr uint64_t RECORD_BYTES = 1ull << 30;

// Records of every query row, `count` each: heads, then rows; heads null: none.
struct Records {
    float2* heads = nullptr;
    float* rows = nullptr;
    uint32_t count = 0;
};
template <int D>
bool get_records(cudaStream_t st, const SpanOperands& a, uint64_t count, int slot, uint64_t n, Records* r) {
    const uint64_t heads = (n * count * sizeof(float2) + 255) / 256 * 256;
    char* p = static_cast<char*>(scratch(st, heads + n * count * D * sizeof(float), slot));
    r->heads = reinterpret_cast<float2*>(p);
    r->rows = reinterpret_cast<float*>(p + heads);
    r->count = (uint32_t)count;
    return p != nullptr;
}

// The tcgen05 kernel over the shared prefix (shared = true) or over the
// sequences' own keys: records from index `first` on, or output rows.
template <int D>
int launch_tiles(const SpanArgs& s, const SpanOperands& a, bool shared, const Records& rec, uint32_t first, const TileGrid& g,
                 float shift, bool overlap, cudaStream_t st) {
    using C = TCfg<D>;
    SpanTileParams p{};
    p.B = (uint32_t)a.B, p.H = (uint32_t)a.H, p.L = (uint32_t)a.L;
    p.Lk = (uint32_t)(shared ? s.prefix_keys : a.Lk);
    p.group = (uint32_t)a.G;
    p.GB = (uint32_t)g.GB, p.LB = (uint32_t)g.LB, p.NB = (uint32_t)g.NB;
    p.rows = p.GB * p.LB * p.NB;
    p.l_tiles = (p.L + p.LB - 1) / p.LB;
    p.tiles = (uint32_t)g.tiles;
    p.groups = (p.tiles + 1) / 2;
    p.head_blocks = p.H / p.GB;
    p.shared_keys = shared ? 1 : 0;
    p.k_batch_bcast = a.k.batch_bcast ? 1 : 0, p.v_batch_bcast = a.v.batch_bcast ? 1 : 0;
    p.keys = span_keys(s);
    if (shared) p.keys.lengths = nullptr;
    p.scale_log2 = s.base.scale * 1.4426950408889634f;
    p.shift = shift;
    p.hidden = p.scale_log2 < 0.0f ? INFINITY : -INFINITY;
    p.splits = (uint32_t)g.splits;
    p.heads = rec.heads, p.stride = rec.count, p.first = first;
    p.out_low = rec.heads ? 0 : s.base.out_low;
    CUtensorMap tq, tk, tv, tk16{}, tv16{}, to;
    const uint32_t dt = a.fmt ? FB_BF16 : FB_F16;
    const uint32_t qbox[3] = {p.GB, p.LB, p.NB}, kbox[3] = {TK, 1, 1}, kbox16[3] = {16, 1, 1};
    if (!span_map<3>(&tq, a.qp, dt, D, {a.H, a.L, a.B}, {a.q.s_head, a.q.s_row, a.q.s_batch}, qbox, true)) return FB_ERR_UNSUPPORTED;
    if (shared) {
        const uint16_t* pk = static_cast<const uint16_t*>(s.pk) + s.pk_offset;
        const uint16_t* pv = static_cast<const uint16_t*>(s.pv) + s.pv_offset;
        if (!span_map<3>(&tk, pk, dt, D, {s.prefix_keys, a.Hkv, 1}, {s.pk_stride_key, s.pk_stride_head, 0}, kbox, true) ||
            !span_map<3>(&tv, pv, dt, D, {s.prefix_keys, a.Hkv, 1}, {s.pv_stride_key, s.pv_stride_head, 0}, kbox, true))
            return FB_ERR_UNSUPPORTED;
    } else {
        if (!span_map<3>(&tk, a.kp, dt, D, {a.Lk, a.Hkv, a.k.batch}, {a.k.s_row, a.k.s_head, a.k.s_batch}, kbox, true) ||
            !span_map<3>(&tv, a.vp, dt, D, {a.Lk, a.Hkv, a.v.batch}, {a.v.s_row, a.v.s_head, a.v.s_batch}, kbox, true) ||
            !span_map<3>(&tk16, a.kp, dt, D, {a.Lk, a.Hkv, a.k.batch}, {a.k.s_row, a.k.s_head, a.k.s_batch}, kbox16, true) ||
            !span_map<3>(&tv16, a.vp, dt, D, {a.Lk, a.Hkv, a.v.batch}, {a.v.s_row, a.v.s_head, a.v.s_batch}, kbox16, true))
            return FB_ERR_UNSUPPORTED;
    }
    const uint32_t obox[4] = {1, p.GB, p.LB, p.NB};
    const uint64_t row = (uint64_t)rec.count * D;
    if (rec.heads ? !span_map<4>(&to, rec.rows, FB_F32, D, {rec.count, a.H, a.L, a.B}, {(uint64_t)D, a.L * row, row, a.H * a.L * row}, obox, false)
                  : !span_map<4>(&to, a.op, s.base.out_low ? s.base.out_low : (uint32_t)FB_F32, D, {1, a.H, a.L, a.B},
                                 {0, a.o.s_head, a.o.s_row, a.o.s_batch}, obox, false))
        return FB_ERR_UNSUPPORTED;
    const uint64_t items = g.units * p.groups * p.splits;
    if (items > 0x7fffffffull) return FB_ERR_UNSUPPORTED;
    p.units = (uint32_t)g.units, p.items = (uint32_t)items;
    const uint64_t grid = std::min<uint64_t>(items, (uint64_t)sm_count());
    auto kernel = a.fmt ? span_tile_kernel<D, 1> : span_tile_kernel<D, 0>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
        return launch_status("shared-memory attribute");
    launch_after(kernel, (unsigned)grid, C::THREADS, C::SMEM, overlap, st, tq, tk, tv, tk16, tv16, to, p);
    count_launch(kernel_name("span_tile_kernel", {D, shared ? 1 : 0}).c_str());
    return launch_status("kernel launch");
}

template <int D>
int launch_merge(const SpanArgs& s, const SpanOperands& a, const Records& rec, cudaStream_t st) {
    SpanMergeParams m{};
    m.heads = rec.heads, m.part = rec.rows;
    m.rows = a.B * a.H * a.L;
    m.count = rec.count;
    m.H = (uint32_t)a.H, m.L = (uint32_t)a.L;
    m.out = a.op, m.out_low = s.base.out_low;
    m.o_sb = a.o.s_batch, m.o_sh = a.o.s_head, m.o_sl = a.o.s_row;
    if ((m.rows + 7) / 8 > 0x7fffffffull) return FB_ERR_UNSUPPORTED;
    launch_after(span_merge_kernel<D>, (unsigned)((m.rows + 7) / 8), 256, 0, true, st, m);
    count_launch(kernel_name("span_merge_kernel", {D}).c_str());
    return launch_status("kernel launch");
}

// span_decode_kernel's CTAs.  A unit of at most 512 keys is one CTA's (four
// warps stream it in the time that joining two CTAs' records takes), of two
// warps when there are more units than CTAs of four fit the GPU at once; longer
// ones are dealt out to two CTAs per SM, at least two tiles each once every SM
// has one, and to more where a warp would take more than range_keys.
struct DecodeGrid {
    uint64_t ctas = 0;
    bool whole = false;
    unsigned warps = 4;
};
bool decode_grid(const SpanArgs& s, const SpanOperands& a, DecodeGrid* g) {
    const uint64_t units = a.B * a.Hkv, sms = (uint64_t)sm_count();
    // the most 64-key tiles that a unit can have, over all lengths
    const uint64_t seen = std::min<uint64_t>(a.Lk, std::min(s.sinks, a.Lk) + std::min(s.window, a.Lk) + a.L);
    const uint64_t tiles = units * std::max<uint64_t>(1, (seen + DTILE - 1) / DTILE);
    if (tiles > 0x7fffffffull) return false;
    g->whole = seen <= 8 * DTILE;
    g->warps = g->whole && units > 2 * sms ? 2 : 4;
    g->ctas = g->whole ? units : tiles <= sms ? tiles : std::min<uint64_t>(2 * sms, std::max(sms, tiles / 2));
    const uint64_t most = 4 * range_keys(a.fmt) / DTILE;  // tiles of a CTA of four warps
    if (!g->whole) g->ctas = std::max(g->ctas, (tiles + most - 1) / most);
    return true;
}

template <int D>
int launch_decode(const SpanArgs& s, const SpanOperands& a, const DecodeGrid& g, const Records& prefix, bool join, float shift,
                  cudaStream_t st) {
    const bool whole = g.whole;
    const uint64_t grid = g.ctas, units = a.B * a.Hkv;
    SpanDecodeParams d{};
    d.whole_units = whole ? 1 : 0;
    if (!whole) {
        Records own;
        if (!get_records<D>(st, a, 1, SCRATCH_SPAN_PART, grid * 2 * 16, &own)) return FB_ERR_DRIVER;
        d.part_heads = own.heads, d.part = own.rows;
        d.arrived = static_cast<uint32_t*>(scratch(st, units * sizeof(uint32_t), SCRATCH_SPAN_COUNT));
        if (!d.arrived) return FB_ERR_DRIVER;
    }
    d.q = static_cast<const uint16_t*>(a.qp), d.k = static_cast<const uint16_t*>(a.kp), d.v = static_cast<const uint16_t*>(a.vp);
    d.q_sb = a.q.s_batch, d.q_sh = a.q.s_head, d.q_sl = a.q.s_row;
    d.k_sb = a.k.batch_bcast ? 0 : a.k.s_batch, d.k_sh = a.k.s_head, d.k_sk = a.k.s_row;
    d.v_sb = a.v.batch_bcast ? 0 : a.v.s_batch, d.v_sh = a.v.s_head, d.v_sk = a.v.s_row;
    d.B = (uint32_t)a.B, d.H = (uint32_t)a.H, d.Hkv = (uint32_t)a.Hkv, d.G = (uint32_t)a.G;
    d.L = (uint32_t)a.L, d.Lk = (uint32_t)a.Lk;
    d.keys = span_keys(s);
    d.scale_log2 = s.base.scale * 1.4426950408889634f;
    d.shift = shift;
    d.prefix_heads = prefix.heads, d.prefix = prefix.rows, d.records = prefix.count, d.join = join ? 1 : 0;
    d.out = a.op, d.out_low = s.base.out_low;
    d.o_sb = a.o.s_batch, d.o_sh = a.o.s_head, d.o_sl = a.o.s_row;
    const bool two = g.warps == 2;
    auto kernel = two ? a.fmt ? span_decode_kernel<D, 1, 2> : span_decode_kernel<D, 0, 2>
                      : a.fmt ? span_decode_kernel<D, 1, 4> : span_decode_kernel<D, 0, 4>;
    const int smem = two ? DCfg<D, 2>::SMEM : DCfg<D, 4>::SMEM;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return launch_status("shared-memory attribute");
    launch_after(kernel, (unsigned)grid, 32 * g.warps, smem, prefix.heads != nullptr, st, d);
    count_launch(kernel_name("span_decode_kernel", {D, (int)a.fmt, (int)g.warps}).c_str());
    return launch_status("kernel launch");
}

template <int D>
int launch_span(const SpanArgs& s, const SpanOperands& a, cudaStream_t st) {
    const bool prefix = s.prefix_keys > 0, own = a.Lk > 0, few = a.G * a.L <= 16;
    const float shift = weight_shift(a.fmt, a.Lk + s.prefix_keys);
    const double streamed = few ? (double)(a.B * a.Hkv * a.Lk) * a.D * 4 : 0.0;
    const TileGrid pg = prefix ? tile_grid(s, a, true, streamed) : TileGrid{};
    const TileGrid og = own && !few ? tile_grid(s, a, false) : TileGrid{};
    const uint64_t ps = pg.splits, rows = a.B * a.H * a.L;
    // Records per row: the prefix's ranges and the own keys', none where the
    // tiles write the output themselves.
    const uint64_t count = few ? prefix ? ps + 1 : 0 : ps + og.splits > 1 ? ps + og.splits : 0;
    Records rec;
    // For as many sequences at a time, or queries of one, as keep the records
    // within RECORD_BYTES: a launch fills the GPU long before that.
    const uint64_t row_bytes = count * (D * sizeof(float) + sizeof(float2));
    if (rows * row_bytes > RECORD_BYTES && (a.B > 1 || a.L > 1)) {
        const bool batch = a.B > 1;
        const uint64_t n = batch ? a.B : a.L, bytes = a.H * (batch ? a.L : 1) * row_bytes;
        uint64_t step = std::min(n - 1, std::max<uint64_t>(1, RECORD_BYTES / bytes));
        if (!batch && step > TQ) step = step / TQ * TQ;
        for (uint64_t at = 0; at < n; at += step) {
            SpanArgs sb = s;
            SpanOperands ab = a;
            const uint64_t m = std::min(step, n - at);
            const uint64_t out_bytes = s.base.out_low ? 2 : 4;
            if (batch) {
                ab.B = m;
                auto part = [&](RowsLayout& l) {
                    if (!l.batch_bcast) l.batch = m;
                    return l.batch_bcast ? 0 : at * l.s_batch;
                };
                ab.qp = static_cast<const uint16_t*>(a.qp) + part(ab.q);
                ab.kp = static_cast<const uint16_t*>(a.kp) + part(ab.k);
                ab.vp = static_cast<const uint16_t*>(a.vp) + part(ab.v);
                ab.op = static_cast<char*>(a.op) + part(ab.o) * out_bytes;
                if (s.lengths) sb.lengths = s.lengths + at * s.length_stride;
            } else {
                ab.L = ab.q.rows = ab.o.rows = m;
                ab.qp = static_cast<const uint16_t*>(a.qp) + at * a.q.s_row;
                ab.op = static_cast<char*>(a.op) + at * a.o.s_row * out_bytes;
                sb.offset += (int64_t)at;
                sb.after += n - at - m;
            }
            if (int r = launch_span<D>(sb, ab, st); r != FB_OK) return r;
        }
        return FB_OK;
    }
    if (few) {  // the own keys streamed, the prefix's records joined there
        DecodeGrid dg;
        if (!decode_grid(s, a, &dg)) return FB_ERR_UNSUPPORTED;
        if (!prefix) return launch_decode<D>(s, a, dg, rec, false, shift, st);
        const uint64_t sms = (uint64_t)sm_count(), busy = std::min(sms, pg.units * ((pg.tiles + 1) / 2) * ps);
        const bool join = dg.ctas <= 2 * (sms - busy) || !own;
        if (!get_records<D>(st, a, join ? ps : ps + 1, SCRATCH_SPAN, rows, &rec)) return FB_ERR_DRIVER;
        if (int r = launch_tiles<D>(s, a, true, rec, 0, pg, shift, false, st); r != FB_OK) return r;
        if (!own) return launch_merge<D>(s, a, rec, st);
        if (int r = launch_decode<D>(s, a, dg, rec, join, shift, st); r != FB_OK) return r;
        return join ? FB_OK : launch_merge<D>(s, a, rec, st);
    }
    if (!count) return launch_tiles<D>(s, a, prefix, rec, 0, prefix ? pg : og, shift, false, st);
    if (!get_records<D>(st, a, count, SCRATCH_SPAN, rows, &rec)) return FB_ERR_DRIVER;
    if (prefix)
        if (int r = launch_tiles<D>(s, a, true, rec, 0, pg, shift, false, st); r != FB_OK) return r;
    if (own)
        if (int r = launch_tiles<D>(s, a, false, rec, (uint32_t)ps, og, shift, prefix, st); r != FB_OK) return r;
    return launch_merge<D>(s, a, rec, st);
}

}  // namespace

uint32_t read_span_status() {
    uint32_t v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_span_status, sizeof(v)) != cudaSuccess) return 0xffffffffu;
    cudaMemcpyToSymbol(g_span_status, &zero, sizeof(zero));
    return v;
}

int launch_span_tc(const SpanArgs& s, void* stream) {
    const AttnArgs& a = s.base;
    if (a.dtype != FB_BF16 && a.dtype != FB_F16) return FB_ERR_UNSUPPORTED;
    if (a.depth != a.value_depth || (a.depth != 64 && a.depth != 128)) return FB_ERR_UNSUPPORTED;
    if (a.row_rank < 2 || a.rows == 0 || (a.keys == 0 && s.prefix_keys == 0)) return FB_ERR_UNSUPPORTED;
    if (a.q_stride_d != 1 || a.o_stride_d != 1) return FB_ERR_UNSUPPORTED;
    if (a.keys > 0 && (a.k_stride_d != 1 || a.v_stride_d != 1)) return FB_ERR_UNSUPPORTED;
    if (s.prefix_keys > 0 && (s.pk_stride_d != 1 || s.pv_stride_d != 1)) return FB_ERR_UNSUPPORTED;
    const int r = (int)a.row_rank;
    SpanOperands x;
    x.L = a.row_dims[r - 1], x.H = a.row_dims[r - 2], x.Lk = a.keys, x.G = a.group_size, x.D = a.depth;
    x.Hkv = x.H / x.G;
    x.fmt = a.dtype == FB_BF16 ? 1 : 0;
    if (x.L > (1u << 30) || x.Lk > (1u << 30) || s.prefix_keys > (1u << 30)) return FB_ERR_UNSUPPORTED;
    x.q.rows = x.L, x.q.heads = x.H, x.q.s_row = a.q_row_strides[r - 1], x.q.s_head = a.q_row_strides[r - 2];
    x.k.rows = x.Lk, x.k.heads = x.Hkv, x.k.s_row = a.k_stride_key, x.k.s_head = a.k_row_strides[r - 2];
    x.v.rows = x.Lk, x.v.heads = x.Hkv, x.v.s_row = a.v_stride_key, x.v.s_head = a.v_row_strides[r - 2];
    x.o.rows = x.L, x.o.heads = x.H, x.o.s_row = a.o_row_strides[r - 1], x.o.s_head = a.o_row_strides[r - 2];
    if (!merge_batch(a, a.q_row_strides, r - 2, &x.q) || !merge_batch(a, a.k_row_strides, r - 2, &x.k) ||
        !merge_batch(a, a.v_row_strides, r - 2, &x.v) || !merge_batch(a, a.o_row_strides, r - 2, &x.o))
        return FB_ERR_UNSUPPORTED;
    if (x.q.batch_bcast || x.o.batch_bcast) return FB_ERR_UNSUPPORTED;
    x.B = x.q.batch;
    if (x.B * x.H * x.L != a.rows || x.o.batch != x.B || a.rows > 0x7fffffffull) return FB_ERR_UNSUPPORTED;
    if ((!x.k.batch_bcast && x.k.batch != x.B) || (!x.v.batch_bcast && x.v.batch != x.B)) return FB_ERR_UNSUPPORTED;
    // rows of 16-byte vectors: bases, and strides of axes with more than one index
    auto aligned = [](const void* p, uint64_t esz, const RowsLayout& l) {
        const uint64_t v = 16 / esz;
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (l.rows <= 1 || l.s_row % v == 0) &&
               (l.heads <= 1 || l.s_head % v == 0) && (l.batch <= 1 || l.s_batch % v == 0);
    };
    x.qp = static_cast<const uint16_t*>(a.q) + a.q_offset;
    x.kp = static_cast<const uint16_t*>(a.k) + a.k_offset;
    x.vp = static_cast<const uint16_t*>(a.v) + a.v_offset;
    x.op = a.out_low ? static_cast<void*>(reinterpret_cast<uint16_t*>(a.out) + a.o_offset) : static_cast<void*>(a.out + a.o_offset);
    if (!aligned(x.qp, 2, x.q) || !aligned(x.op, a.out_low ? 2 : 4, x.o)) return FB_ERR_UNSUPPORTED;
    if (x.Lk > 0 && (!aligned(x.kp, 2, x.k) || !aligned(x.vp, 2, x.v))) return FB_ERR_UNSUPPORTED;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a.depth == 64 ? launch_span<64>(s, x, st) : launch_span<128>(s, x, st);
}

}  // namespace fb
