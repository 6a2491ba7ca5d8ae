// Attention of long chunks over a paged K/V cache on the tensor cores (tcgen05), head dim 128.
//
// The skeleton is that of the dense kernel (attn_fwd.cuh): persistent CTAs, work items of two 128-row tiles, the K/V ring in
// pairs [V(j-1) | K(j)], one issuing thread, one query row per softmax thread, a softmax without a maximum pass whose row sum
// guards the reference.  What differs:
//   * A work item is (sequence, rows, kv head).  A row tile holds 128 / g tokens of the g heads that share the kv head, so
//     shared heads cost no extra pass over the keys; lengths, rows and the page table are read on the device.
//   * Items are of very different lengths (ragged sequences, causal rows) and seldom a multiple of the SMs.  So the items are
//     laid end to end, each as long as its key tiles and kItemCost more, and every CTA takes an equal run of that line, which
//     may begin and end inside an item.  Parts of an item go to a workspace with their log-sum-exp and one small kernel joins
//     them, in order.  (Whole items dealt in snake order, cut in equal key ranges by a cost model, took 912 us for 4 680 rows x
//     12 heads over 28 080 keys -- 228 items on 148 SMs -- and 512 us for three ragged chunks of 600 items.)
//   * Key tiles are 128 keys at multiples of 128: those of the window, then those of the sinks (a reference taken from a few sinks would
//     not hold for long: 460 against 404 us for three ragged chunks over 4-bit pages).  Pages outside are not touched.
//   * bf16 pages: one lane of the loader warp per page (or half a page of 256 rows) issues that page's TMA boxes; boxes
//     of which the item sees nothing take a page coordinate past the pool, which reads as zeros.  In the few tiles that
//     the item's visible keys only cover in part, one warp ("fixer") then zeroes V's rows that no row of the item sees: a P of
//     zero times whatever memory holds there must be zero.
//   * 4-bit pages: the loader brings the packed codes by bulk copies, four more warps expand them to f16 into the swizzled
//     tiles that TMA would have written, and bring Q as f16.  Both products then run in f16: a value zero + step code is rounded
//     once, by 2^-11 at most (in bf16 the roundings of K and V, 2^-8 each, would be of the size of the output's own), P by 2^-11.
//     f16's range stays out of it: K and V of an item and every row of q are brought to the upper end of f16 by powers of two,
//     which go into the row's softmax scale and the output's.  Two warps survey the scales of an item's keys while the item before is
//     at work.  Values down to 2^-26 of the largest of their item keep their 11 bits.  (A factor a tile instead, worked out when its
//     scales come: 400 -> 436 us for three ragged chunks, most of it a wait and a load a tile in the softmax.)
//     P's reference is set 2^6 below the maximum that it is taken from: P up to 2^15 fits, and P is zero only 2^30 below it.
// Bound by the tensor pipe and by what feeds it (128 x 128 x 16 products from shared memory take all of its bandwidth): 4 680 rows x
// 12 heads over 28 080 bf16 keys 710 us under the profiler = 1 137 TFLOP/s, tensor pipe 62 % of the active cycles (690-830 us in a
// loop, at the power cap); three ragged chunks of up to 1 501 tokens, 40 heads on 8, windows of 4 100 keys (35 tiles an item, five of
// them cut by the mask) 326 us with bf16 pages, 56 %, and 402 us with 4-bit pages, 45 % (in a graph, with the join, 306-345 and 365-390).
// ptxas spills 56 bytes a thread over bf16 pages and 88 over 4-bit ones.
#pragma once
#include "attn_fwd.cuh"
#include "paged.cuh"

namespace fvpg {

constexpr int kChunkTile = 128;  // keys
constexpr int kChunkRows = 128;  // query rows of a row tile; an item has two

struct ChunkJob {
    Pool pool;
    Batch batch;
    Mask mask;
    const uint16_t* q;
    long long q_tok, q_head;
    uint16_t* out;
    float *part_o, *part_lse;  // [2 per run, 256 rows, 128] and [2 per run, 256]: a part that does not begin its item, one that does
    struct ChunkSplit* split;  // [run]: the item that begins in the run and ends in another
    int* wait_status;          // the first status word
    long long wait_cycles;
    int heads, group, tile_tokens, items, box_rows;  // items: (sequence, kv head, row block), row blocks fastest
    int phases;
    Div by_group, by_blocks, by_heads;  // row blocks of a plane; kv heads
    float sl2;
};
constexpr int kItemCost = 4;   // what an item costs beside its key tiles, in key tiles: the pipeline fills and drains, the output
constexpr int kLeastRun = 4;   // the shortest run worth a CTA (8: 23 against 16 us for 16 items of two tiles)
struct ChunkSplit {
    int valid, q0, nq, tok0, head, tiles, cost, runs;
    long long start, total;  // where the item begins on the line, and how long the line is
};
// The first key tile of an item that lies behind position y of its length: the fixed cost comes first, and no part is a
// sliver of one tile.
__host__ __device__ inline int tile_behind(int y, int tiles) {
    if (y >= tiles + kItemCost) return tiles;
    const int t = y - kItemCost;
    return t < 2 ? 0 : tiles - t < 2 ? tiles : t;
}

#if defined(__CUDA_ARCH_FEAT_SM100_ALL) || defined(__CUDA_ARCH_FEAT_SM103_ALL) || !defined(__CUDA_ARCH__)

using fvattn::as_f;
using fvattn::as_u;
using fvattn::Cols;
using fvattn::RowState;
using fvattn::Smem;
using fvattn::neg_inf;
using namespace fvp;

// Shared memory: the dense kernel's map.  After its barriers, bf16: a barrier for each pair slot, "V's invisible rows are
// zeroed".  4 bits: two stages of packed codes, [V(j-1) | K(j)] as they lie in the pages, take the place of the third Q slot;
// their barriers and scales come last.
constexpr uint32_t kVFixed = Smem::total;
constexpr uint32_t kCodeFull = kVFixed + 8 * fvattn::kKvPairs, kCodeFree = kCodeFull + 16;
// Of item i, in slot i & 1: K's and V's sizes are there; the rows' sizes are too; all of them have been read.
constexpr uint32_t kSurveyed = kCodeFree + 16, kItemReady = kSurveyed + 16, kItemFree = kItemReady + 16;
constexpr uint32_t kFirstDone = kItemFree + 16, kFirstTop = kFirstDone + 16;  // [K | V]: the softmax warps' share of a run's first survey
constexpr uint32_t kSizes = (kFirstTop + 8 + 15) & ~15u;         // [item & 1][K | V]: Size
constexpr uint32_t kScales = kSizes + 32;                        // [stage][V | K][128 keys] (step, zero)
constexpr uint32_t kRowSizes = kScales + 2 * 1024;               // [item & 1][row tile][128 rows] exponents, a byte each
constexpr uint32_t kScratch = kRowSizes;                         // find_run's, before there are any
constexpr uint32_t kRun = kRowSizes + 4 * kChunkRows;            // this CTA's run
constexpr uint32_t kChunkSmem = kRun + 64;
constexpr uint32_t kCodes = Smem::q + 2 * fvattn::kSlotBytes;   // [stage][V | K][128 keys][64 bytes]
static_assert(kVFixed % 8 == 0 && kChunkSmem <= 232448 && fvattn::kQSlots == 3 && fvattn::kSlotBytes == 32768, "shared memory");
static_assert(fvattn::kKvPairs == 2 && fvattn::kEarlyKeys == 128, "the ring in pairs, P handed over whole");

template <bool Q4>
struct Roles {
    static constexpr int kWarps = Q4 ? 16 : 12;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kLoader = 8, kIssuer = 9, kFixer = 10;  // (fixer: bf16)
    static constexpr int kSurveyor = 10;                         // 4 bits: warps 10 (K) and 11 (V)
    static constexpr int kExpander = 12, kExpanders = 4;         // 4 bits: warps 12-15, one on each of the SM's schedulers
    static constexpr uint32_t kQ = Q4 ? 2 : fvattn::kQSlots;     // Q slots
};

// What an item covers; every role works it out for itself, from the same numbers.
struct Work {
    Seq seq;
    Span span;
    int s, head, tok0;          // first token of the item inside the call's tokens of the sequence
    int sinks, first, tiles;    // its key tiles: those of the window, then those of the sinks
    int u0, n;                  // this CTA's part of them
    FV_DEV int pos0() const { return seq.len - seq.nq; }
    FV_DEV int key(int j) const {
        const int u = u0 + j;
        return (u < tiles - sinks ? first + u : u - (tiles - sinks)) * kChunkTile;
    }
    FV_DEV bool sees(int j) const { return (j >= span.lo && j < span.hi) || j < span.sink; }
    FV_DEV bool whole(int k0) const { return (k0 >= span.lo && k0 + kChunkTile <= span.hi) || k0 + kChunkTile <= span.sink; }
    FV_DEV bool begins() const { return u0 == 0; }
    FV_DEV bool ends() const { return u0 + n == tiles; }
};
// Item number i: its rows and tiles, and its cost; 0 when there are no such rows.
FV_DEV int item_at(const ChunkJob& jb, int i, Work& w) {
    const int plane = i / jb.by_blocks;
    w.s = plane / jb.by_heads;
    w.head = plane - w.s * jb.pool.kv_heads;
    w.seq = seq_of(jb.batch, w.s);
    w.tok0 = (i - plane * (int)jb.by_blocks.d) * 2 * jb.tile_tokens;
    w.tiles = 0;
    if (w.tok0 >= w.seq.nq) return 0;
    const int last = min(w.tok0 + 2 * jb.tile_tokens, w.seq.nq) - 1;
    w.span = span_of(jb.mask, w.pos0() + w.tok0, w.pos0() + last, w.seq.len);
    w.sinks = (w.span.sink + kChunkTile - 1) / kChunkTile;
    w.first = max(w.span.lo / kChunkTile, w.sinks);
    w.tiles = w.sinks + max(0, (w.span.hi + kChunkTile - 1) / kChunkTile - w.first);
    return w.tiles + kItemCost;
}
// This CTA's runs of the line: number blockIdx + p gridDim of `runs` equal ones, p = 0 .. phases - 1.
constexpr int kMaxPhases = 4;
struct Run {
    long long total;
    int runs;
    struct Start {
        int item, off, length;  // the item that the run begins in, where in it, and the run's length
    } start[kMaxPhases];
    FV_DEV long long edge(int v) const { return total * v / runs; }
};
static_assert(sizeof(Run) <= 64 && kRun % 8 == 0, "shared memory");
// Warp-inclusive sum.
FV_DEV long long scan_warp(long long x, int lane) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(kFullWarp, x, d);
        if (lane >= d) x += y;
    }
    return x;
}
// The whole CTA adds up the line (a run of items a thread) and finds its places on it.  `scratch`: 32 long longs.
FV_DEV void find_run(const ChunkJob& jb, Run* run, long long* scratch) {
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = (int)blockDim.x >> 5;
    const int per = (jb.items + (int)blockDim.x - 1) / (int)blockDim.x;
    const int i0 = min(tid * per, jb.items), i1 = min(i0 + per, jb.items);
    long long mine = 0;
    Work w;
    for (int i = i0; i < i1; i++) mine += item_at(jb, i, w);
    const long long incl = scan_warp(mine, lane);
    if (lane == 31) scratch[warp] = incl;
    __syncthreads();
    long long before = 0, total = 0;
    for (int i = 0; i < warps; i++) {
        if (i < warp) before += scratch[i];
        total += scratch[i];
    }
    const long long excl = before + incl - mine;
    const int runs = (int)max(1ll, min((long long)gridDim.x * jb.phases, total / kLeastRun));
    if (tid == 0) {
        run->total = total;
        run->runs = runs;
    }
    for (int p = 0; p < jb.phases; p++) {
        const int v = (int)blockIdx.x + p * (int)gridDim.x;
        const bool idle = v >= runs || total == 0;
        const long long from = idle ? 0 : total * v / runs, to = idle ? 0 : total * (v + 1) / runs;
        if (tid == 0) run->start[p].length = (int)(to - from);
        if (from < to && from >= excl && from < excl + mine) {
            long long at = excl;
            for (int i = i0; i < i1; i++) {
                const int cost = item_at(jb, i, w);
                if (from < at + cost) {
                    run->start[p].item = i;
                    run->start[p].off = (int)(from - at);
                    break;
                }
                at += cost;
            }
        }
    }
    __syncthreads();
}
// The items of the CTA's runs, in order.
struct Walk {
    const Run& run;
    int phase = -1, item = 0, off = 0, left = 0;
    FV_DEV explicit Walk(const Run& r) : run(r) {}
    FV_DEV int number() const { return (int)blockIdx.x + phase * (int)gridDim.x; }  // of the run
    // The next item with key tiles (`empty`: or with rows that see no key).  *ahead: what is left of the run from where this item
    // began on the line.
    FV_DEV bool next(const ChunkJob& jb, Work& w, bool empty, int* ahead = nullptr) {
        for (;;) {
            if (left <= 0 || item >= jb.items) {
                if (++phase >= jb.phases) return false;
                left = run.start[phase].length;
                item = run.start[phase].item;
                off = run.start[phase].off;
                continue;
            }
            const int cost = item_at(jb, item, w);
            const int end = min(cost, off + left);
            w.u0 = tile_behind(off, w.tiles);
            w.n = tile_behind(end, w.tiles) - w.u0;
            if (ahead) *ahead = left + off;
            left -= end - off;
            off = end;
            const bool done = end == cost;
            if (done) {
                off = 0;
                item++;
            }
            if (cost > 0 && (w.n > 0 || (empty && w.tiles == 0 && done))) return true;
        }
    }
};

struct ChunkWait {
    uint32_t sbase;
    int* status;
    long long cycles;
    int role;
    FV_DEV bool operator()(uint32_t bar, uint32_t parity) const {
        if (mbar_try(bar, parity)) return true;
        const long long t0 = clock64();
        uint32_t n = 0;
        while (!mbar_try(bar, parity)) {
            if (((++n) & 63u) == 0u) {
                uint32_t gone;
                asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(gone) : "r"(sbase + Smem::abort_flag) : "memory");
                if (gone) return false;
                if (clock64() - t0 > cycles) {
                    asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(sbase + Smem::abort_flag), "r"(1u) : "memory");
                    atomicCAS(status, FV_ST_OK, FV_ST_TIMEOUT_BASE + role);
                    return false;
                }
            }
        }
        return true;
    }
};

// ------------------------------------------------------------------------------------------------- products
// kind::f16 with both operands bf16 (as umma_idesc_bf16) or both f16 (type fields 0).
template <bool F16>
__host__ __device__ constexpr uint32_t chunk_idesc(uint32_t b_mn_major) {
    return F16 ? (1u << 4) | (b_mn_major << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24) : umma_idesc_bf16(128, 128, b_mn_major);
}
template <bool F16>
FV_DEV void chunk_scores(uint32_t tS, uint64_t qd, uint64_t kd) {
    constexpr uint32_t idesc = chunk_idesc<F16>(0);
    asm volatile(
        "{\n\t.reg .pred pt, pf;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 pf, %3, %3;\n\tsetp.eq.b32 pt, %3, %3;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, pf;\n\t"
        FV_QK_STEP(2) FV_QK_STEP(4) FV_QK_STEP(6) FV_QK_STEP(1024) FV_QK_STEP(1026) FV_QK_STEP(1028) FV_QK_STEP(1030)
        "}"
        ::"r"(tS), "l"(qd), "l"(kd), "r"(idesc)
        : "memory");
}
template <bool F16>
FV_DEV void chunk_output(uint32_t tO, uint32_t tP, uint64_t vd, bool fresh) {
    constexpr uint32_t idesc = chunk_idesc<F16>(1);
    asm volatile(
        "{\n\t.reg .pred pt, p0;\n\t.reg .b64 b;\n\t.reg .b32 t;\n\t"
        "setp.eq.b32 p0, %4, 0;\n\tsetp.eq.b32 pt, %3, %3;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p0;\n\t"
        FV_PV_STEP(8, 128) FV_PV_STEP(16, 256) FV_PV_STEP(24, 384) FV_PV_STEP(32, 512) FV_PV_STEP(40, 640)
        FV_PV_STEP(48, 768) FV_PV_STEP(56, 896)
        "}"
        ::"r"(tO), "r"(tP), "l"(vd), "r"(idesc), "r"(fresh ? 1u : 0u)
        : "memory");
}

// ---------------------------------------------------------------------------------------- sizes (4-bit pages)
// The power of two that numbers of which the largest has the biased exponent e are divided by for f16: what is left is below 2^13, values
// zero + step code (twice the larger of |zero| and 8 |step| at most) below 2^14.  Limited so that the factors stay normal numbers.
FV_DEV int size_of(int e) { return min(max(e, 24), 250) - 139; }
FV_DEV float power_of_two(int e) { return __int_as_float((127 + e) << 23); }
FV_DEV int exponent_of(float x) { return (int)(__float_as_uint(x) >> 23); }  // x >= 0
// The larger magnitudes of two pairs of bf16 (their signs mean nothing; a NaN gives way to a number).
FV_DEV uint32_t larger_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
FV_DEV uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
FV_DEV uint32_t twice_bf16(int e) { return 0x00010001u * ((uint32_t)(127 + e) << 7); }  // 2^e, two of it

// A survey: the largest |zero| or 8 |step| of the keys that an item sees, of K or V, as the bits of an f32.  Tiles first, first + stride, ..;
// all of a warp, and each lane gets the result.  Pages are looked up a box a lane, for up to 32 boxes at a time; of a tile's scales
// a lane holds four keys, four tiles are in flight (eight: more code in all, 404 -> 412 us for three ragged chunks).
FV_DEV uint32_t survey(const ChunkJob& jb, const Work& w, int which, int first, int stride, int lane) {
    constexpr int kAhead = 4;
    constexpr uint32_t kNone = 0xffffffffu;
    const uint32_t* scales = which ? jb.pool.v_scale : jb.pool.k_scale;
    const int log_box = min(jb.pool.log_rows, 7), log_boxes = 7 - log_box, per = 32 >> log_boxes;  // boxes of a tile, tiles of a look-up
    const int tiles = (w.n - first + stride - 1) / stride;                                        // (of this warp; may be less than one)
    uint32_t top_step = 0, top_zero = 0;
#pragma unroll 1
    for (int j0 = 0; j0 < tiles; j0 += per) {
        uint32_t row = kNone;
        if (j0 + (lane >> log_boxes) < tiles) {
            const int a = w.key(first + stride * (j0 + (lane >> log_boxes))) + ((lane << log_box) & (kChunkTile - 1)), b = a + (1 << log_box);
            if ((a < w.span.hi && b > w.span.lo) || a < w.span.sink) {
                const int page = page_of(jb.pool, jb.batch, w.s, a);
                if (page >= 0) row = (uint32_t)pool_row(jb.pool, page, w.head, a);
            }
        }
        const int end = min(per, tiles - j0);
#pragma unroll 1
        for (int t0 = 0; t0 < end; t0 += kAhead) {
            uint4 x[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                const uint32_t r = __shfl_sync(fvpg::kFullWarp, row, ((t0 + i) << log_boxes) + ((4 * lane) >> log_box));
                x[i] = make_uint4(0, 0, 0, 0);
                if (t0 + i < end && r != kNone) x[i] = __ldg(reinterpret_cast<const uint4*>(scales + r + ((4 * lane) & ((1 << log_box) - 1))));
            }
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                const int key = t0 + i < end ? w.key(first + stride * (j0 + t0 + i)) : 0;
                if (!w.whole(key)) {
                    if (!w.sees(key + 4 * lane)) x[i].x = 0;
                    if (!w.sees(key + 4 * lane + 1)) x[i].y = 0;
                    if (!w.sees(key + 4 * lane + 2)) x[i].z = 0;
                    if (!w.sees(key + 4 * lane + 3)) x[i].w = 0;
                }
                const uint32_t pair[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t step = pair[k] << 17, zero = pair[k] & 0x7fff0000u;  // (step: a bit further up)
                    if (step < 0xff000000u && zero < 0x7f800000u) {                     // (a row that is not finite has no say)
                        top_step = max(top_step, step);
                        top_zero = max(top_zero, zero);
                    }
                }
            }
        }
    }
    const float top = fmaxf(8.f * __uint_as_float(top_step >> 1), __uint_as_float(top_zero));
    return __reduce_max_sync(fvpg::kFullWarp, __float_as_uint(top));
}
// A run's first item has nothing to hide its survey behind: the softmax warps, which wait anyway, take four fifths of it.  (220 tiles
// of 28 080 keys would else take 23 us.)
constexpr int kFirstSurvey = 1 + fvattn::kSoftmaxWarps / 2;  // warps of each of K and V
struct Size {
    float by;     // 2^size
    uint32_t up;  // 2^-size as two bf16
};
static __device__ __noinline__ void first_survey(const ChunkJob& jb, const Run& run, uint32_t sbase, int warp, int lane) {
    const int which = warp & 1;
    Walk walk(run);
    Work w;
    if (!walk.next(jb, w, false)) return;
    const uint32_t top = survey(jb, w, which, 1 + (warp >> 1), kFirstSurvey, lane);
    if (lane == 0) {
        asm volatile("red.shared.max.u32 [%0], %1;" ::"r"(sbase + kFirstTop + 4u * which), "r"(top) : "memory");
        mbar_arrive(sbase + kFirstDone + 8u * which);
    }
}

// -------------------------------------------------------------------------------------------------- softmax
FV_DEV uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool F16>
FV_DEV uint32_t pack_p(float lo, float hi) {
    return F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}
// A row sum of P above this could leave P's type.
template <bool F16>
constexpr float kChunkGuard = F16 ? 32768.f : fvattn::kGuard;
// A reference is set 2^this below the maximum that it is taken from.
template <bool F16>
constexpr float kChunkBelow = F16 ? 6.f : 0.f;
// As fvattn::exp32: 2^(u sl2 + noff) of 32 columns to packed pairs, every fourth pair on the FMA pipe (POLY: bf16 pages; with 4-bit
// ones the expander wants the issue slots that this takes, three ragged chunks 388 with and 377 us without).
template <bool F16, bool POLY>
FV_DEV void chunk_exp32(const uint32_t (&u)[32], uint32_t* pw, uint64_t s2, uint64_t nf, uint64_t& acc0, uint64_t& acc1, float& top) {
#pragma unroll
    for (int w = 0; w < 16; w++) {
        float t0, t1, p0, p1;
        unpack_f32x2(fma_f32x2(pack_f32x2(as_f(u[2 * w]), as_f(u[2 * w + 1])), s2, nf), t0, t1);
        if (POLY && (w & 3) == 3) {
            top = max3(top, t0, t1);
            ex2_poly_x2(t0, t1, p0, p1);
        } else {
            p0 = ex2(t0);
            p1 = ex2(t1);
        }
        const uint64_t pp = pack_f32x2(p0, p1);
        if (w & 1) acc1 = add_f32x2(acc1, pp);
        else acc0 = add_f32x2(acc0, pp);
        pw[w] = pack_p<F16>(p0, p1);
    }
}

// Bit c: the row sees column c0 + c of the tile.  (Three comparisons a column instead took more than the exponentials.)
FV_DEV uint32_t seen_bits(const Cols& k, int c0) {
    auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; };
    return (below(k.hi - c0) & ~below(k.lo - c0)) | below(k.sink - c0);
}
FV_DEV void hide_columns(uint32_t (&u)[32], uint32_t seen) {
#pragma unroll
    for (int c = 0; c < 32; c++) u[c] = (seen & (1u << c)) ? u[c] : as_u(neg_inf());
}

template <bool F16>
FV_DEV void unpack_p(uint32_t w, float& lo, float& hi) {
    if (F16) {
        asm("{\n\t.reg .f16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(lo), "=f"(hi) : "r"(w));
    } else {
        lo = as_f(w << 16);
        hi = as_f(w & 0xffff0000u);
    }
}
// The reference of this lane's row moves for chunk c of the tile: to `below` the chunk's largest where there was none, else by a
// whole power of two, so that the P stored already (chunks 0 .. c - 1) stay exact.  O, the sum and that P are rescaled.
template <bool F16>
FV_DEV void move_reference(uint32_t tS, uint32_t tO, int c, float cand, bool have_o, float& m, float& l) {
    float a = 1.f;
    if (cand > m + 7.f) {  // (32 columns above a quarter of the guard have one above 2^8)
        const float want = cand - kChunkBelow<F16>;
        if (m == neg_inf()) {
            a = 0.f;
            m = want;
        } else {
            const float k = ceilf(want - m);
            a = ex2(-k);
            m += k;
        }
        l *= a;
    }
    if (!__any_sync(kFullWarp, a != 1.f)) return;
    auto rescale = [&](uint32_t at, bool packed) {
        uint32_t o[32];
        tmem_ld32_issue(at, o);
        tmem_ld_wait();
        tmem_pin(o);
#pragma unroll
        for (int i = 0; i < 32; i++) {
            float x = as_f(o[i]), y;
            if (packed) {
                unpack_p<F16>(o[i], x, y);
                o[i] = pack_p<F16>(x * a, y * a);
            } else {
                o[i] = as_u(x * a);
            }
        }
        tmem_st32(at, o);
    };
    if (have_o) {
#pragma unroll 1
        for (int q = 0; q < 4; q++) rescale(tO + 32u * q, false);
    }
    if (c > 0) {  // (16 columns a chunk; those behind them in the last 32 hold scores that are done with)
        tmem_st_wait();
#pragma unroll 1
        for (int q = 0; 2 * q < c; q++) rescale(tS + 32u * q, true);
    }
}

// A tile with invisible columns, or whose sum tripped the guard (out of line for the reasons that fvattn::careful_tile
// gives).  In one pass of four chunks of 32 columns, the invisible ones as -inf: P of a chunk (16 columns) takes the place of scores
// that have been read.  Where a row has no reference yet, or a chunk's sum is above a quarter of the guard (so that a tile that the hot path
// gave up always moves its reference), the reference moves there.  (With a pass
// for the maxima first: two sequences of 2 048 tokens, 32 heads on 8, 83 against 80 us, 4 bits 107 against 104.)
template <bool F16>
static __device__ __noinline__ void chunk_careful(uint32_t tS, uint32_t tO, uint32_t bt, Cols cols, float sl2, bool have_o, int lane,
                                                  RowState* rs) {
    float m = rs->m, l = rs->l;
    const uint64_t s2 = pack_f32x2(sl2, sl2);
#pragma unroll 1
    for (int c = 0; c < 4; c++) {
        uint32_t pw[16];
        const uint32_t seen = seen_bits(cols, 32 * c);
        if (__any_sync(kFullWarp, seen != 0u)) {
            for (bool moved = false;; moved = true) {
                uint32_t u[32];
                fvattn::load_chunk(tS, c, u);
                fvattn::land_chunk(u);
                hide_columns(u, seen);
                const float noff = m == neg_inf() ? 0.f : -m;
                const uint64_t nf = pack_f32x2(noff, noff);
                uint64_t acc0 = pack_f32x2(0.f, 0.f), acc1 = acc0;
                float top = 0.f;
                const bool none = __any_sync(kFullWarp, m == neg_inf() && seen != 0u);
                if (moved || !none) {
                    chunk_exp32<F16, false>(u, pw, s2, nf, acc0, acc1, top);
                    const float sum = fvattn::part_sum<false>(acc0, acc1, top);
                    if (moved || !__any_sync(kFullWarp, !(sum <= 0.25f * kChunkGuard<F16>))) {
                        l += sum;
                        break;
                    }
                }
                move_reference<F16>(tS, tO, c, fvattn::max32(u) * sl2, have_o, m, l);
            }
        } else {
#pragma unroll
            for (int w = 0; w < 16; w++) pw[w] = 0u;
        }
        tmem_st16(tS + 16u * (uint32_t)c, pw);
    }
    fvattn::publish(bt + Smem::p_ready, lane);
    rs->m = m;
    rs->l = l;
}

// Columns 32 q .. 32 q + 31 of the warp's 32 rows; `row` is this lane's output row or -1.  The 16-byte pieces are transposed
// between neighbouring lanes first, so that a store covers whole runs of a row (fvattn::store_cols32).
template <bool Q4, bool F32>
FV_DEV void chunk_store32(void* base, const uint32_t (&o)[32], float inv, int row, int q, int lane) {
    constexpr int G = F32 ? 8 : 4;
    uint4 p[G];
    float f[32];
#pragma unroll
    for (int c = 0; c < 32; c++) f[Q4 ? (c & 24) + ((c & 7) >> 1) + 4 * (c & 1) : c] = as_f(o[c]) * inv;  // (4 bits: see expand_unit)
#pragma unroll
    for (int c = 0; c < G; c++) {
        if (F32) p[c] = make_uint4(as_u(f[4 * c]), as_u(f[4 * c + 1]), as_u(f[4 * c + 2]), as_u(f[4 * c + 3]));
        else p[c] = make_uint4(pack_bf16x2(f[(8 * c) & 31], f[(8 * c + 1) & 31]), pack_bf16x2(f[(8 * c + 2) & 31], f[(8 * c + 3) & 31]),
                               pack_bf16x2(f[(8 * c + 4) & 31], f[(8 * c + 5) & 31]), pack_bf16x2(f[(8 * c + 6) & 31], f[(8 * c + 7) & 31]));
    }
    fvattn::transpose_pieces<G>(p, lane);
    const int l = lane & (G - 1);
#pragma unroll
    for (int k = 0; k < G; k++) {
        const int r = __shfl_sync(kFullWarp, row, (lane & ~(G - 1)) + k);
        if (r >= 0) {
            if (F32) *reinterpret_cast<uint4*>(static_cast<float*>(base) + (size_t)r * kD + 32 * q + 4 * l) = p[k];
            else *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + (size_t)r * kD + 32 * q + 8 * l) = p[k];
        }
    }
}
template <bool Q4, bool F32>
static __device__ __noinline__ void chunk_write(void* base, uint32_t tO, float inv, int row, bool have_o, int lane) {
#pragma unroll 1
    for (int q = 0; q < 4; q++) {
        uint32_t o[32];
        if (have_o) {
            tmem_ld32_issue(tO + 32u * q, o);
            tmem_ld_wait();
            tmem_pin(o);
        } else {
#pragma unroll
            for (int c = 0; c < 32; c++) o[c] = 0u;
        }
        chunk_store32<Q4, F32>(base, o, inv, row, q, lane);
    }
}

template <bool Q4>
FV_DEV void chunk_softmax(const ChunkJob& jb, const Run& run, uint32_t sbase, uint32_t tmem, int warp, int lane, const ChunkWait& wait) {
    const int tile = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t tS = lanes + fvattn::tmem_scores((uint32_t)tile), tO = lanes + fvattn::tmem_output((uint32_t)tile);
    const uint32_t bt = sbase + 8u * (uint32_t)tile;
    float sl2 = jb.sl2;
    const int row_tok = row / jb.by_group, row_head = row - row_tok * jb.group;
    uint32_t s_count = 0, o_count = 0, item = 0;  // (item: those with key tiles)
    if (Q4) first_survey(jb, run, sbase, warp, lane);
    Walk walk(run);
    Work w;
    int ahead = 0;
    bool more = walk.next(jb, w, true, &ahead);
    while (more) {
        const int tok = w.tok0 + tile * jb.tile_tokens + row_tok;
        const bool live = row_tok < jb.tile_tokens && tok < w.seq.nq;
        const int pos = w.pos0() + tok;
        const Span rsp = span_of(jb.mask, pos, pos, w.seq.len);
        RowState rs{neg_inf(), 0.f};
        if (Q4 && w.n > 0) {  // the row's softmax scale, with the sizes of its q and of the item's K
            if (!__all_sync(kFullWarp, wait(sbase + kItemReady + 8u * (item & 1u), (item >> 1) & 1u))) return;
            uint32_t e;
            float k;
            asm volatile("ld.shared.u8 %0, [%1];" : "=r"(e) : "r"(sbase + kRowSizes + 2 * kChunkRows * (item & 1u) + threadIdx.x) : "memory");
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(k) : "r"(sbase + kSizes + 16u * (item & 1u)) : "memory");
            // (a row of q with an infinity has scores that are not numbers)
            sl2 = e == 255u ? __int_as_float(0x7fffffff) : jb.sl2 * power_of_two(size_of((int)e)) * k;
        }
        for (int j = 0; j < w.n; j++) {
            if (!__all_sync(kFullWarp, wait(bt + Smem::s_ready, s_count & 1u))) return;
            s_count++;
            tc_fence_after();
            const int k0 = w.key(j);
            Cols cols{0, 0, 0, false};  // (a row that is none: nothing visible, and no say in the votes)
            if (live) {
                cols.lo = rsp.lo - k0;
                cols.hi = min(rsp.hi - k0, kChunkTile);
                cols.sink = min(rsp.sink - k0, kChunkTile);
                cols.whole = (cols.lo <= 0 && cols.hi >= kChunkTile) || cols.sink >= kChunkTile;
            }
            bool hot = __all_sync(kFullWarp, cols.whole || !live);
            if (hot) {
                uint32_t u0[32], u1[32], pw[64];
                fvattn::load_chunk(tS, 0, u0);
                fvattn::land_chunk(u0);
                if (rs.m == neg_inf()) rs.m = live ? fvattn::max32(u0) * sl2 - kChunkBelow<Q4> : 0.f;
                const uint64_t s2 = pack_f32x2(sl2, sl2), nf = pack_f32x2(-rs.m, -rs.m);
                uint64_t acc0 = pack_f32x2(0.f, 0.f), acc1 = acc0;
                float top = 0.f;
                fvattn::load_chunk(tS, 1, u1);
                chunk_exp32<Q4, !Q4>(u0, pw, s2, nf, acc0, acc1, top);
                fvattn::land_chunk(u1);
                fvattn::load_chunk(tS, 2, u0);
                chunk_exp32<Q4, !Q4>(u1, pw + 16, s2, nf, acc0, acc1, top);
                fvattn::land_chunk(u0);
                fvattn::load_chunk(tS, 3, u1);
                chunk_exp32<Q4, !Q4>(u0, pw + 32, s2, nf, acc0, acc1, top);
                fvattn::land_chunk(u1);
                chunk_exp32<Q4, !Q4>(u1, pw + 48, s2, nf, acc0, acc1, top);
                const float sum = fvattn::part_sum<!Q4>(acc0, acc1, top);
                if (__any_sync(kFullWarp, live && !(sum <= kChunkGuard<Q4>))) {
                    hot = false;  // nothing of this tile is stored
                } else {
                    fvattn::store_early(tS, pw);
                    fvattn::publish(bt + Smem::p_ready, lane);
                    rs.l += sum;
                }
            }
            if (!hot) chunk_careful<Q4>(tS, tO, bt, cols, sl2, j > 0, lane, &rs);
        }
        const int number = walk.number();
        const bool have_o = w.n > 0, begins = w.begins(), part = !(begins && w.ends());
        const int out_row = !live ? -1 : part ? tile * kChunkRows + row : (w.seq.q0 + tok) * jb.heads + w.head * jb.group + row_head;
        if (begins && part && threadIdx.x == 0)
            jb.split[number] = ChunkSplit{1, w.seq.q0, w.seq.nq, w.tok0, w.head, w.tiles, w.tiles + kItemCost, run.runs, run.edge(number + 1) - ahead, run.total};
        more = walk.next(jb, w, true, &ahead);  // (looked up while the last product runs)
        if (have_o) {
            if (!__all_sync(kFullWarp, wait(bt + Smem::o_ready, o_count & 1u))) return;
            o_count++;
            tc_fence_after();
        }
        float inv = rs.l > 0.f ? 1.f / rs.l : 0.f;
        if (Q4 && have_o) {
            float v;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(sbase + kSizes + 16u * (item & 1u) + 8u) : "memory");
            inv *= v;
            fvattn::warp_arrive(sbase + kItemFree + 8u * (item & 1u), lane);
            item++;
        }
        if (!part) {
            chunk_write<Q4, false>(jb.out, tO, inv, out_row, have_o, lane);
        } else {
            const size_t slot = 2 * (size_t)number + (begins ? 1 : 0);
            chunk_write<Q4, true>(jb.part_o + slot * 2 * kChunkRows * kD, tO, inv, out_row, have_o, lane);
            if (out_row >= 0)
                jb.part_lse[slot * 2 * kChunkRows + out_row] = rs.l > 0.f ? rs.m + log2f(rs.l) : rs.l == 0.f ? neg_inf() : -neg_inf();  // (+inf: not a number)
        }
    }
}

// --------------------------------------------------------------------------------- loader and fixer (bf16 pages)
FV_DEV void chunk_loader(const CUtensorMap* mq, const CUtensorMap* mk, const CUtensorMap* mv, const ChunkJob& jb, const Run& run,
                         uint32_t sbase, int lane, const ChunkWait& wait) {
    using namespace fvattn;
    uint32_t qn = 0, kvn = 0;
    if (lane == 0) {
        tma_prefetch_desc(mq);
        tma_prefetch_desc(mk);
        tma_prefetch_desc(mv);
    }
    const uint32_t q_bytes = (uint32_t)(jb.tile_tokens * jb.group) * 128u;  // of one 64-column panel
    auto ok_all = [&](uint32_t bar, uint32_t parity) { return __all_sync(fvpg::kFullWarp, wait(bar, parity)) != 0; };
    auto load_q = [&](const Work& w, int tile) -> bool {
        const uint32_t slot = qn % kQSlots, use = qn / kQSlots;
        if (use > 0 && !ok_all(sbase + Smem::q_free + 8u * slot, (use - 1u) & 1u)) return false;
        const uint32_t dst = sbase + Smem::q + slot * kSlotBytes, bar = sbase + Smem::q_full + 8u * slot;
        if (lane == 0) {
            const int tok = w.seq.q0 + w.tok0 + tile * jb.tile_tokens;  // rows of other sequences or past the end: never stored
            mbar_expect_tx(bar, 2 * q_bytes);
            tma_load4(dst, mq, bar, 0, w.head * jb.group, tok, 0);
            tma_load4(dst + kPanelBytes, mq, bar, 64, w.head * jb.group, tok, 0);
        }
        qn++;
        return true;
    };
    const int boxes = kChunkTile / jb.box_rows;
    // Page of this lane's box of the key tile at k0; past the pool (zeros) where the item sees nothing of it.
    auto box_page = [&](const Work& w, int k0) -> int {
        if (lane >= boxes) return jb.pool.pages;
        const int a = k0 + lane * jb.box_rows, b = a + jb.box_rows;
        if (!((a < w.span.hi && b > w.span.lo) || a < w.span.sink)) return jb.pool.pages;
        const int page = page_of(jb.pool, jb.batch, w.s, a);
        return page < 0 ? jb.pool.pages : page;
    };
    auto load_tile = [&](const CUtensorMap* map, uint32_t dst, uint32_t bar, int k0, int page, int head) {
        const int row = (k0 + lane * jb.box_rows) & ((1 << jb.pool.log_rows) - 1);
        const uint32_t at = dst + (uint32_t)(lane * jb.box_rows) * 128u;
        tma_load4(at, map, bar, 0, row, head, page);
        tma_load4(at + kPanelBytes, map, bar, 64, row, head, page);
    };
    Walk walk(run);
    Work w, nw;
    bool ok = true;
    bool have = walk.next(jb, w, false);
    if (have) ok = load_q(w, 0) && load_q(w, 1);
    while (ok && have) {
        const bool more = walk.next(jb, nw, false);
        if (more) ok = load_q(nw, 0);
        int page = box_page(w, w.key(0)), prev = 0;
        for (int j = 0; ok && j <= w.n; j++) {
            const int ahead = j + 1 < w.n ? box_page(w, w.key(j + 1)) : 0;  // (the look-up's latency runs under the wait)
            const uint32_t slot = kvn % kKvPairs, use = kvn / kKvPairs;
            if (use > 0 && !ok_all(sbase + Smem::kv_free + 8u * slot, (use - 1u) & 1u)) { ok = false; break; }
            const uint32_t dst = sbase + Smem::kv + slot * 2u * kSlotBytes, bar = sbase + Smem::kv_full + 8u * slot;
            if (lane == 0) mbar_expect_tx(bar, (j > 0 ? kSlotBytes : 0u) + (j < w.n ? kSlotBytes : 0u));
            __syncwarp();
            if (lane < boxes) {
                if (j > 0) load_tile(mv, dst, bar, w.key(j - 1), prev, w.head);
                if (j < w.n) load_tile(mk, dst + kSlotBytes, bar, w.key(j), page, w.head);
            }
            kvn++;
            prev = page;
            page = ahead;
        }
        if (ok && more) ok = load_q(nw, 1);
        w = nw;
        have = more;
    }
    __syncwarp();
    if (lane == 0) {  // copies in flight must land before the CTA's shared memory goes away
        for (uint32_t s = 0; s < (uint32_t)kQSlots && s < qn; s++) {
            const uint32_t last = ((qn - 1u - s) / kQSlots) * kQSlots + s;
            mbar_drain(sbase + Smem::q_full + 8u * s, (last / kQSlots) & 1u);
        }
        for (uint32_t s = 0; s < (uint32_t)kKvPairs && s < kvn; s++) {
            const uint32_t last = ((kvn - 1u - s) / kKvPairs) * kKvPairs + s;
            mbar_drain(sbase + Smem::kv_full + 8u * s, (last / kKvPairs) & 1u);
        }
    }
}

// Follows the pairs one by one (it has a share in kv_free, so it can neither run ahead of a phase nor miss one).
FV_DEV void chunk_fixer(const ChunkJob& jb, const Run& run, uint32_t sbase, int lane, const ChunkWait& wait) {
    using namespace fvattn;
    uint32_t pn = 0;
    Walk walk(run);
    Work w;
    while (walk.next(jb, w, false)) {
        for (int j = 0; j <= w.n; j++) {
            const uint32_t slot = pn % kKvPairs;
            if (!__all_sync(fvpg::kFullWarp, wait(sbase + Smem::kv_full + 8u * slot, (pn / kKvPairs) & 1u))) return;
            if (j > 0 && !w.whole(w.key(j - 1))) {
                const int k0 = w.key(j - 1);
                const uint32_t v = sbase + Smem::kv + slot * 2u * kSlotBytes;
                for (int r = lane; r < kChunkTile; r += 32) {
                    if (w.sees(k0 + r)) continue;
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v + 128u * r + 16u * c), "r"(0) : "memory");
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v + kPanelBytes + 128u * r + 16u * c), "r"(0) : "memory");
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the tensor cores read the rows
                warp_arrive(sbase + kVFixed + 8u * slot, lane);
            }
            warp_arrive(sbase + Smem::kv_free + 8u * slot, lane);
            pn++;
        }
    }
}

// ------------------------------------------------------------------------------------ expander (4-bit pages)
FV_DEV uint32_t add_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
FV_DEV uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
FV_DEV uint32_t pack_f16x2_inf(float lo, float hi) {  // (a row that is not finite stays one)
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
FV_DEV uint32_t and_or(uint32_t a, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));
    return r;
}
FV_DEV void store_piece(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// The unit of the expander's work: 8 neighbouring rows, a quarter (32 values, one 16-byte load) a lane.  Piece j (8 values) of
// quarter q of a row goes to piece_base(...) ^ (j << 4): the 128 x 128 tile has two 64-column panels, and the 128-byte
// swizzle puts piece c of row r into slot (c ^ r) & 7 of its panel's row.
FV_DEV uint32_t piece_base(uint32_t tile, int row, int q) {
    return tile + (uint32_t)(q >> 1) * fvattn::kPanelBytes + 128u * (uint32_t)row + 16u * (uint32_t)(((4 * (q & 1)) ^ row) & 7);
}
// Eight values of a word stand in a piece in the order 0 4 1 5 2 6 3 7: the pairs that one mask gives.  Q's pieces get the
// same order (the sum over d does not care), and the output's columns are put back when they are stored.
// f16 values (zero + step code) up, `up` a power of two as two bf16: a nibble is or-ed into 1024's mantissa (unit 1) where it lies, 1024 + n or 1024 + 16 n, an
// addition or multiply-add makes it n - 8 exactly, and one more multiply-add rounds once.
FV_DEV void expand_unit(uint4 c, uint32_t sz, uint32_t up, uint32_t base, int q) {
    sz = mul_bf16x2(sz, up);
    const uint32_t sz16 = pack_f16x2_inf(__uint_as_float(sz << 16), __uint_as_float(sz & 0xffff0000u));
    const uint32_t s2 = __byte_perm(sz16, 0, 0x1010), z2 = __byte_perm(sz16, 0, 0x3232);
    // (Quarters 0 and 2, 1 and 3 meet in the same banks, in different panels: the upper two take their words in the order 2 3 0 1.)
    const bool swap = q >= 2;
    const uint32_t word[4] = {swap ? c.z : c.x, swap ? c.w : c.y, swap ? c.x : c.z, swap ? c.y : c.w};
    base ^= swap ? 32u : 0u;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t w = word[j], v = w >> 8;
        const uint32_t h0 = add_f16x2(and_or(w, 0x000f000fu, 0x64006400u), 0xe408e408u);               // - 1032
        const uint32_t h1 = fma_f16x2(and_or(w, 0x00f000f0u, 0x64006400u), 0x2c002c00u, 0xd480d480u);  // / 16 - 72
        const uint32_t h2 = add_f16x2(and_or(v, 0x000f000fu, 0x64006400u), 0xe408e408u);
        const uint32_t h3 = fma_f16x2(and_or(v, 0x00f000f0u, 0x64006400u), 0x2c002c00u, 0xd480d480u);
        store_piece(base ^ (16u * j), fma_f16x2(h0, s2, z2), fma_f16x2(h1, s2, z2), fma_f16x2(h2, s2, z2), fma_f16x2(h3, s2, z2));
    }
}
// A pair's 32 units are dealt to the warps in turn.  Four warps, one per scheduler: their instructions come out of the softmax
// warps' issue slots, and six (two schedulers with two of them) were slower, 430 against 412 us for three ragged chunks
// when that was the kernel's time; without the arithmetic of the expansion it would have been 363.  (A first form with one key row a lane and page look-ups and loads of its
// own took 709: look-ups and loads are the loader's since.)
FV_DEV void chunk_expander(const ChunkJob& jb, const Run& run, uint32_t sbase, int wid, int lane, const ChunkWait& wait) {
    using namespace fvattn;
    using R = Roles<true>;
    constexpr int kW = R::kExpanders;
    uint32_t qn = 0, kvn = 0, item = 0;
    const int r8 = lane >> 2, q = lane & 3;  // this lane's row of a unit and its quarter
    auto ok_all = [&](uint32_t bar, uint32_t parity) { return __all_sync(fvpg::kFullWarp, wait(bar, parity)) != 0; };
    auto arrive = [&](uint32_t bar) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the tensor cores read what was stored
        warp_arrive(bar, lane);
    };
    auto load_q = [&](const Work& w, int tile) -> bool {
        const uint32_t slot = qn % R::kQ, use = qn / R::kQ;
        if (use > 0 && !ok_all(sbase + Smem::q_free + 8u * slot, (use - 1u) & 1u)) return false;
        const uint32_t dst = sbase + Smem::q + slot * kSlotBytes;
#pragma unroll 1
        for (int u = wid; u < 16; u += kW) {
            const int row = 8 * u + r8, row_tok = row / jb.by_group, tok = w.tok0 + tile * jb.tile_tokens + row_tok;
            const bool live = row_tok < jb.tile_tokens && tok < w.seq.nq;
            const uint16_t* p = jb.q + (long long)(w.seq.q0 + (live ? tok : 0)) * jb.q_tok +
                                (long long)(w.head * jb.group + (live ? row - row_tok * jb.group : 0)) * jb.q_head + 32 * q;
            const uint32_t base = piece_base(dst, row, q);
            uint4 x[4];
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[j] = live ? __ldg(reinterpret_cast<const uint4*>(p) + j) : make_uint4(0, 0, 0, 0);
                top = larger_bf16x2(larger_bf16x2(top, larger_bf16x2(x[j].x, x[j].y)), larger_bf16x2(x[j].z, x[j].w));
            }
            top = larger_bf16x2(top, __shfl_xor_sync(fvpg::kFullWarp, top, 1));
            top = larger_bf16x2(top, __shfl_xor_sync(fvpg::kFullWarp, top, 2)) & 0x7fff7fffu;
            const int e = (int)(max(top & 0xffffu, top >> 16) >> 7);
            if (q == 0)
                asm volatile("st.shared.u8 [%0], %1;" ::"r"(sbase + kRowSizes + kChunkRows * (2 * (item & 1u) + tile) + row), "r"(e) : "memory");
            const uint32_t up = twice_bf16(-size_of(e));
            auto low = [](uint32_t a, uint32_t b) { return pack_f16x2(__uint_as_float(a << 16), __uint_as_float(b << 16)); };
            auto high = [](uint32_t a, uint32_t b) { return pack_f16x2(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u)); };
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t a = mul_bf16x2(x[j].x, up), b = mul_bf16x2(x[j].y, up), c = mul_bf16x2(x[j].z, up), d = mul_bf16x2(x[j].w, up);
                store_piece(base ^ (16u * j), low(a, c), high(a, c), low(b, d), high(b, d));
            }
        }
        arrive(sbase + Smem::q_full + 8u * slot);
        qn++;
        return true;
    };
    Walk walk(run);
    Work w;
    while (walk.next(jb, w, false)) {
        if (!load_q(w, 0) || !load_q(w, 1)) return;
        if (!ok_all(sbase + kSurveyed + 8u * (item & 1u), (item >> 1) & 1u)) return;
        uint32_t up_k, up_v;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(up_k) : "r"(sbase + kSizes + 16u * (item & 1u) + 4u) : "memory");
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(up_v) : "r"(sbase + kSizes + 16u * (item & 1u) + 12u) : "memory");
        warp_arrive(sbase + kItemReady + 8u * (item & 1u), lane);
        item++;
        for (int j = 0; j <= w.n; j++) {
            const uint32_t slot = kvn % kKvPairs, use = kvn / kKvPairs;  // (as many code stages as pair slots)
            if (!ok_all(sbase + kCodeFull + 8u * slot, use & 1u)) return;
            if (use > 0 && !ok_all(sbase + Smem::kv_free + 8u * slot, (use - 1u) & 1u)) return;
            const uint32_t codes = sbase + kCodes + slot * 16384u, scales = sbase + kScales + slot * 1024u;
            const uint32_t dst = sbase + Smem::kv + slot * 2u * kSlotBytes;
            const int v0 = j > 0 ? w.key(j - 1) : 0, k0 = j < w.n ? w.key(j) : 0;
            const bool v_whole = j > 0 && w.whole(v0), k_whole = j < w.n && w.whole(k0);
#pragma unroll 2
            for (int u = wid; u < 32; u += kW) {  // units 0-15: V(j-1), 16-31: K(j)
                const bool is_k = u >= 16;
                if (is_k ? j == w.n : j == 0) continue;
                const int row = 8 * (u & 15) + r8;
                uint4 c;
                uint32_t sz;
                asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(c.x), "=r"(c.y), "=r"(c.z), "=r"(c.w) : "r"(codes + 512u * u + 16u * lane) : "memory");
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(sz) : "r"(scales + 32u * u + 4u * r8) : "memory");
                // A key that the item does not see counts as zeros whatever memory holds.
                if (!(is_k ? k_whole : v_whole) && !w.sees((is_k ? k0 : v0) + row)) sz = 0u;
                expand_unit(c, sz, is_k ? up_k : up_v, piece_base(dst + (is_k ? kSlotBytes : 0u), row, q), q);
            }
            arrive(sbase + Smem::kv_full + 8u * slot);
            if (lane == 0) mbar_arrive(sbase + kCodeFree + 8u * slot);  // (arrive() has met the warp: its reads are done)
            kvn++;
        }
    }
}

// The sizes of an item's K or V, an item ahead of the expander (which is what the tensor cores wait for).
FV_DEV void chunk_surveyor(const ChunkJob& jb, const Run& run, uint32_t sbase, int which, int lane, const ChunkWait& wait) {
    uint32_t item = 0;
    int before[2] = {0, 0};  // key tiles of the last two items
    Walk walk(run);
    Work w;
    while (walk.next(jb, w, false)) {
        uint32_t top = survey(jb, w, which, 0, item == 0 ? kFirstSurvey : 1, lane);
        const uint32_t slot = item & 1u;
        if (item == 0) {
            if (!__all_sync(fvpg::kFullWarp, wait(sbase + kFirstDone + 8u * which, 0))) return;
            uint32_t others;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(others) : "r"(sbase + kFirstTop + 4u * which) : "memory");
            top = max(top, others);
        } else if (item > 1) {  // (the only wait that lasts for a whole item: some 3 500 cycles a tile)
            ChunkWait patient = wait;
            patient.cycles += 16384ll * (before[0] + before[1]);
            if (!__all_sync(fvpg::kFullWarp, patient(sbase + kItemFree + 8u * slot, ((item >> 1) - 1u) & 1u))) return;
        }
        before[0] = before[1];
        before[1] = w.n;
        const int size = size_of((int)(top >> 23));
        if (lane == 0) {
            asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(sbase + kSizes + 16u * slot + 8u * which), "r"(__float_as_uint(power_of_two(size))), "r"(twice_bf16(-size)) : "memory");
            mbar_arrive(sbase + kSurveyed + 8u * slot);
        }
        item++;
    }
}

// The codes: one lane per page box brings its rows of K(j) and of V(j-1) and their scales by bulk copies (a page holds them as one
// run each).  Boxes of which the item sees nothing, and pages outside the pool, are left out: the expander zeroes what is not seen.
FV_DEV void chunk_code_loader(const ChunkJob& jb, const Run& run, uint32_t sbase, int lane, const ChunkWait& wait) {
    using namespace fvattn;
    uint32_t kvn = 0;
    auto ok_all = [&](uint32_t bar, uint32_t parity) { return __all_sync(fvpg::kFullWarp, wait(bar, parity)) != 0; };
    const int boxes = kChunkTile / jb.box_rows;
    auto box_row = [&](const Work& w, int k0) -> long long {  // pool row of this lane's box, -1: none
        if (lane >= boxes) return -1;
        const int a = k0 + lane * jb.box_rows, b = a + jb.box_rows;
        if (!((a < w.span.hi && b > w.span.lo) || a < w.span.sink)) return -1;
        const int page = page_of(jb.pool, jb.batch, w.s, a);
        return page < 0 ? -1 : (long long)pool_row(jb.pool, page, w.head, a);
    };
    Walk walk(run);
    Work w;
    bool ok = true;
    while (ok && walk.next(jb, w, false)) {
        long long row = box_row(w, w.key(0)), prev = -1;
        for (int j = 0; j <= w.n; j++) {
            const long long ahead = j + 1 < w.n ? box_row(w, w.key(j + 1)) : -1;  // (the look-up's latency runs under the wait)
            const uint32_t slot = kvn % kKvPairs, use = kvn / kKvPairs;
            if (use > 0 && !ok_all(sbase + kCodeFree + 8u * slot, (use - 1u) & 1u)) { ok = false; break; }
            const bool k = j < w.n && row >= 0, v = j > 0 && prev >= 0;
            const uint32_t tiles = __popc(__ballot_sync(fvpg::kFullWarp, k)) + __popc(__ballot_sync(fvpg::kFullWarp, v));
            const uint32_t bar = sbase + kCodeFull + 8u * slot, code_bytes = (uint32_t)jb.box_rows * kQ4Bytes, scale_bytes = (uint32_t)jb.box_rows * 4;
            if (lane == 0) mbar_expect_tx(bar, tiles * (code_bytes + scale_bytes));
            __syncwarp();
            const uint32_t codes = sbase + kCodes + slot * 16384u + lane * code_bytes, scales = sbase + kScales + slot * 1024u + lane * scale_bytes;
            if (v) {
                bulk_load(codes, jb.pool.v + prev * kQ4Bytes, code_bytes, bar);
                bulk_load(scales, jb.pool.v_scale + prev, scale_bytes, bar);
            }
            if (k) {
                bulk_load(codes + 8192u, jb.pool.k + row * kQ4Bytes, code_bytes, bar);
                bulk_load(scales + 512u, jb.pool.k_scale + row, scale_bytes, bar);
            }
            kvn++;
            prev = row;
            row = ahead;
        }
    }
    __syncwarp();
    if (lane == 0) {  // copies in flight must land before the CTA's shared memory goes away
        for (uint32_t s = 0; s < (uint32_t)kKvPairs && s < kvn; s++) {
            const uint32_t last = ((kvn - 1u - s) / kKvPairs) * kKvPairs + s;
            mbar_drain(sbase + kCodeFull + 8u * s, (last / kKvPairs) & 1u);
        }
    }
}

// --------------------------------------------------------------------------------------------------- issuer
// Step j of an item: O_t += P_t(j-1) . V(j-1) for j > 0, then S_t = Q_t . K(j)^T for j < n, t = A then B, strictly in order
// (fvattn::issuer_thread).
template <bool Q4>
FV_DEV void chunk_issuer(const ChunkJob& jb, const Run& run, uint32_t sbase, uint32_t tmem, const ChunkWait& wait) {
    using namespace fvattn;
    uint32_t qn = 0, pn = 0, pc = 0;
    uint32_t fixed[kKvPairs] = {};  // V tiles of each slot that the fixer had to touch so far
    Walk walk(run);
    Work w;
    bool ok = true;
    while (ok && walk.next(jb, w, false)) {
        const uint32_t qa = qn % Roles<Q4>::kQ, qb = (qn + 1u) % Roles<Q4>::kQ;
        const uint32_t qa_par = (qn / Roles<Q4>::kQ) & 1u, qb_par = ((qn + 1u) / Roles<Q4>::kQ) & 1u;
        qn += 2;
        const uint64_t qd_a = umma_desc_sw128(sbase + Smem::q + qa * kSlotBytes, 16, 1024);
        const uint64_t qd_b = umma_desc_sw128(sbase + Smem::q + qb * kSlotBytes, 16, 1024);
#pragma unroll 1
        for (int j = 0; j <= w.n; j++) {
            const uint32_t slot = pn % kKvPairs;
            const uint32_t pair = sbase + Smem::kv + slot * 2u * kSlotBytes;
            if (!wait(sbase + Smem::kv_full + 8u * slot, (pn / kKvPairs) & 1u)) { ok = false; break; }
            if (!Q4 && j > 0 && !w.whole(w.key(j - 1))) {
                uint32_t& count = slot ? fixed[1] : fixed[0];
                if (!wait(sbase + kVFixed + 8u * slot, count & 1u)) { ok = false; break; }
                count++;
            }
            tc_fence_after();
            const uint64_t vd = umma_desc_sw128(pair, kPanelBytes, 1024);
            const uint64_t kd = umma_desc_sw128(pair + kSlotBytes, 16, 1024);
#pragma unroll
            for (uint32_t t = 0; t < 2; t++) {
                if (j > 0) {
                    if (!wait(sbase + 8u * t + Smem::p_ready, pc & 1u)) { ok = false; break; }
                    tc_fence_after();
                    chunk_output<Q4>(tmem + tmem_output(t), tmem + tmem_scores(t), vd, j == 1);
                }
                if (j == w.n) {
                    umma_commit(sbase + Smem::o_ready + 8u * t);
                    continue;
                }
                if (j == 0) {
                    if (!wait(sbase + Smem::q_full + 8u * (t ? qb : qa), t ? qb_par : qa_par)) { ok = false; break; }
                    tc_fence_after();
                }
                chunk_scores<Q4>(tmem + tmem_scores(t), t ? qd_b : qd_a, kd);
                umma_commit(sbase + Smem::s_ready + 8u * t);
                if (j == w.n - 1) umma_commit(sbase + Smem::q_free + 8u * (t ? qb : qa));
            }
            if (!ok) break;
            umma_commit(sbase + Smem::kv_free + 8u * slot);
            pn++;
            if (j > 0) pc++;
        }
    }
    umma_commit(sbase + Smem::drain);
    mbar_drain(sbase + Smem::drain, 0);
}

template <bool Q4>
FV_DEV void chunk_persistent(const CUtensorMap* mq, const CUtensorMap* mk, const CUtensorMap* mv, const ChunkJob& jb, unsigned char* smem) {
    using namespace fvattn;
    using R = Roles<Q4>;
    const uint32_t sbase = smem_u32(smem);
    const int warp = (int)(threadIdx.x >> 5), lane = (int)(threadIdx.x & 31);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Smem::abort_flag);
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + Smem::tmem_slot);
    const Run& run = *reinterpret_cast<const Run*>(smem + kRun);
    if (threadIdx.x == 0) {
        for (int p = 0; p < jb.phases; p++) jb.split[blockIdx.x + p * gridDim.x].valid = 0;
        const uint32_t producers = Q4 ? R::kExpanders : 1;  // the expander's warps, or one transaction count
        for (int s = 0; s < kQSlots; s++) {
            mbar_init(sbase + Smem::q_full + 8u * s, producers);
            mbar_init(sbase + Smem::q_free + 8u * s, 1);
        }
        for (int s = 0; s < kKvPairs; s++) {
            mbar_init(sbase + Smem::kv_full + 8u * s, producers);
            mbar_init(sbase + Smem::kv_free + 8u * s, Q4 ? 1 : 2);  // the issuer's commit (and the fixer)
            mbar_init(sbase + kVFixed + 8u * s, 1);
            mbar_init(sbase + kCodeFull + 8u * s, 1);
            mbar_init(sbase + kCodeFree + 8u * s, R::kExpanders);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(sbase + kFirstDone + 8u * s, kFirstSurvey - 1);
            mbar_init(sbase + kSurveyed + 8u * s, 2);
            mbar_init(sbase + kItemReady + 8u * s, R::kExpanders);
            mbar_init(sbase + kItemFree + 8u * s, kSoftmaxWarps);
        }
        for (int t = 0; t < 2; t++) {
            mbar_init(sbase + Smem::s_ready + 8u * t, 1);
            mbar_init(sbase + Smem::p_ready + 8u * t, 4);
            mbar_init(sbase + Smem::o_ready + 8u * t, 1);
        }
        mbar_init(sbase + Smem::drain, 1);
        *reinterpret_cast<volatile uint32_t*>(smem + kFirstTop) = *reinterpret_cast<volatile uint32_t*>(smem + kFirstTop + 4) = 0u;
        int bad = (*(volatile int*)jb.wait_status != FV_ST_OK) ? 1 : 0;  // a CTA that starts after another one gave up does nothing
        if (sbase & 1023u) {
            atomicCAS(jb.wait_status, FV_ST_OK, FV_ST_BAD_SMEM);
            bad = 1;
        }
        *abort_flag = bad;
        mbar_init_fence();
    }
    __syncthreads();
    if (*abort_flag) return;  // CTA-uniform
    find_run(jb, reinterpret_cast<Run*>(smem + kRun), reinterpret_cast<long long*>(smem + kScratch));
    if (run.start[0].length == 0) return;  // nothing on this CTA's part of the line (a later run is never longer)
    if (warp == R::kIssuer) tmem_alloc(sbase + Smem::tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto waiter = [&](int role) { return ChunkWait{sbase, jb.wait_status, jb.wait_cycles, role}; };
    // Registers: 384 x 168 = 256 x 216 + 128 x 72; 512 x 128 = 256 x 184 + 256 x 72.
    if (warp < kSoftmaxWarps) {
        if (Q4) asm volatile("setmaxnreg.inc.sync.aligned.u32 184;" ::: "memory");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;" ::: "memory");
        chunk_softmax<Q4>(jb, run, sbase, tmem, warp, lane, waiter(3));
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;" ::: "memory");
        if (warp == R::kIssuer) {
            if (lane == 0) chunk_issuer<Q4>(jb, run, sbase, tmem, waiter(2));
        } else if (Q4) {
            if (warp >= R::kExpander) chunk_expander(jb, run, sbase, warp - R::kExpander, lane, waiter(6));
            else if (warp >= R::kSurveyor) chunk_surveyor(jb, run, sbase, warp - R::kSurveyor, lane, waiter(4));
            else if (warp == R::kLoader) chunk_code_loader(jb, run, sbase, lane, waiter(1));
        } else if (warp == R::kLoader) {
            chunk_loader(mq, mk, mv, jb, run, sbase, lane, waiter(1));
        } else if (warp == R::kFixer) {
            chunk_fixer(jb, run, sbase, lane, waiter(4));
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == R::kIssuer) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

#endif  // sm_100a / host pass

}  // namespace fvpg
