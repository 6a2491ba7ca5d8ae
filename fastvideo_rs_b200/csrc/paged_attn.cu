// Attention of a ragged batch's queries over a paged K/V cache: block-causal with a sliding window and sinks, shared
// K/V heads, pages of bf16 or of 4 bits.  This file: the kernel for few query rows per K/V head (decode steps, short
// chunks), the kernels that join parts, the choice between this kernel and the one for long chunks (paged_fwd.cuh), and the C
// entries.
//
// Row r of a (sequence, kv head) is token r / g, head r % g of the heads that share that K/V head (g = heads /
// kv_heads): one pass over the keys serves all of them.
#include "fv_runtime.h"
#include "paged.cuh"
#include "paged_fwd.cuh"
#include "paged_host.h"
#include <cooperative_groups.h>
#include <math.h>
#include <stdlib.h>
#include <string.h>
#include <mutex>

namespace fvpg {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;
constexpr int kAttnThreads = 32 * kWarps;
constexpr int kMaxCluster = 8;  // CTAs of a portable cluster
// Keys a warp takes at a time: 16 are in one page (page_rows is a multiple of 16), 32 in one or two.
template <bool Q4>
constexpr int kTile = Q4 ? 32 : 16;

struct AttnArgs {
    Pool pool;
    Batch batch;
    Mask mask;
    const uint16_t* q;
    long long q_tok, q_head;  // strides in values
    uint16_t* out;            // [tokens, heads, 128]
    float* part_o;            // [splits, tokens * heads, 128] normalised, when splits > 1
    float* part_lse;          // [splits, tokens * heads], base 2
    int heads, group, splits;
    Div by_group, by_splits, by_blocks, by_heads;  // blocks of rows of a (sequence, kv head); kv heads
    int cluster;              // the key ranges of a block of rows are one cluster, which joins them itself
    float sl2;
    long long wait_cycles;
};

using fvattn::neg_inf;

// The key tiles a block of rows visits: those of [0, sink), then those of [lo, hi), each tile once.
template <int TILE>
struct Tiles {
    int sinks, first, count;
    FV_DEV explicit Tiles(const Span& s) {
        sinks = (s.sink + TILE - 1) / TILE;
        first = max(s.lo / TILE, sinks);
        count = sinks + max(0, (s.hi + TILE - 1) / TILE - first);
    }
    FV_DEV int key(int u) const { return (u < sinks ? u : first + (u - sinks)) * TILE; }
};

FV_DEV uint4 ld_stream(const void* p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
FV_DEV uint2 ld_stream2(const void* p) {
    uint2 r;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
    return r;
}
FV_DEV uint32_t ld_stream1(const void* p) {
    uint32_t r;
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(r) : "l"(p));
    return r;
}
// D (16 x 8 f32) += A (16 x 16) . B (16 x 8), both bf16 or both f16.  Lane 4 g + t holds of A rows g (a0, a2) and g + 8
// (a1, a3), of B column g, of D rows g (c0, c1) and g + 8 (c2, c3), columns 2 t and 2 t + 1.
template <bool F16>
FV_DEV void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transpose of an 8 x 8 tile of 16-bit values held one row per quad of lanes.
FV_DEV uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
FV_DEV uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
// The eight codes of a word as four f16 pairs, pair i from nibbles i and i + 4: a nibble n at bits 0-3 of a half word is the
// f16 number n 2^-24 as it stands (below f16's normal numbers, which the matrix unit multiplies exactly), at bits 4-7
// 16 n 2^-24.  One shift and four masks a word and nothing else: expanding the codes is what bounds this kernel (with the
// codes or-ed into 1024's mantissa and the 1024 taken off again by an addition it took 160 instead of 129 us for 32 sequences of
// 20 011 keys; as bytes for the 8-bit matrix instruction, q in two parts, 137).  The factors, and the 8 between n and the code, are taken out of the products' results.
FV_DEV void codes_f16(uint32_t w, uint32_t (&h)[4]) {
    const uint32_t v = w >> 8;
    h[0] = w & 0x000f000fu;
    h[1] = w & 0x00f000f0u;
    h[2] = v & 0x000f000fu;
    h[3] = v & 0x00f000f0u;
}
constexpr float kCodeUnit = 16777216.f;  // 2^24
FV_DEV float lo_f(uint32_t x) { return __uint_as_float(x << 16); }
FV_DEV float hi_f(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

FV_DEV uint32_t word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

// One tile of 16 keys in registers, as lane 4 g + t holds it; `row` is the pool row of the tile's first key, or kNoRow.
//   bf16  k0 / k1: keys g and g + 8, 16-byte pieces 4 n + t of their rows; v: keys 2t, 2t+1, 2t+8, 2t+9, pieces g and
//         g + 8 of their rows.  Straight from memory.
//   4 bit k0 / k1: values 32 t .. 32 t + 31 of keys g' and g' + 8; v: values 16 g .. 16 g + 15 of four keys; s0 / s1:
//         (step, zero) of keys g' and g' + 8.  Out of the warp's ring in shared memory.
constexpr uint32_t kNoRow = 0xffffffffu;
// The key of a 4-bit tile that stands in row g of the product: every second pair is swapped, so that the lanes that read V's
// rows 2 t side by side meet both halves of the banks.
FV_DEV int key_of_row(int g) { return g ^ ((g >> 1) & 1); }
template <bool Q4>
struct Keys;
template <>
struct Keys<false> {
    uint4 k0[4], k1[4];
    FV_DEV void load(const uint8_t* lane_k, uint32_t row) {
        if (row == kNoRow) {
#pragma unroll
            for (int n = 0; n < 4; n++) k0[n] = k1[n] = make_uint4(0, 0, 0, 0);
            return;
        }
        const uint8_t* r = lane_k + (size_t)row * 256;
#pragma unroll
        for (int n = 0; n < 4; n++) {
            k0[n] = ld_stream(r + 64 * n);
            k1[n] = ld_stream(r + 8 * 256 + 64 * n);
        }
    }
    static FV_DEV size_t lane_offset(int g, int t) { return (size_t)g * 256 + 16 * t; }
};
template <>
struct Keys<true> {
    uint4 k0, k1;
    uint32_t s0, s1;
};
template <bool Q4>
struct Values;
template <>
struct Values<false> {
    uint4 a[4], b[4];  // pieces g and g + 8 of keys 2t, 2t+1, 2t+8, 2t+9
    FV_DEV void load(const uint8_t* lane_v, uint32_t row) {
        if (row == kNoRow) {
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = b[i] = make_uint4(0, 0, 0, 0);
            return;
        }
        const uint8_t* r = lane_v + (size_t)row * 256;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int o = ((i & 1) + 8 * (i >> 1)) * 256;
            a[i] = ld_stream(r + o);
            b[i] = ld_stream(r + o + 128);
        }
    }
    static FV_DEV size_t lane_offset(int g, int t) { return (size_t)(2 * t) * 256 + 16 * g; }
    FV_DEV float step(int) const { return 1.f; }
};
template <>
struct Values<true> {
    uint2 a[4];
    uint32_t s0, s1;
    FV_DEV float step(int h) const { return __uint_as_float((h ? s1 : s0) << 16); }
};

// The ring of a warp (4 bits): a stage is a tile of 32 keys, K codes | V codes | K scales | V scales, brought by bulk copies (in
// pages of 32 rows and more one run of each array, in pages of 16 two), one mbarrier a stage.  A warp fills and waits for
// its own stages only.
struct Ring {
    static constexpr uint32_t kHalfBytes = 2 * 1024 + 2 * 64, kStageBytes = 2 * kHalfBytes;
    static constexpr uint32_t kV = 2048, kKs = 4096, kVs = 4224;
    static constexpr int kStages = 3;
    static constexpr uint32_t kWarpBytes = kStages * kStageBytes;
};
template <bool Q4, int ROWS>
struct DecodeSmem {
    static constexpr uint32_t kJoin = kWarps * ROWS * (kD + 4) * 4 + 2 * kWarps * ROWS * 4;  // the warps' results side by side
    static constexpr uint32_t kRing = Q4 ? kWarps * Ring::kWarpBytes : 0;                        // (the join comes after the ring)
    static constexpr uint32_t kBars = kRing > kJoin ? kRing : kJoin;
    static constexpr uint32_t kTotal = kBars + (Q4 ? kWarps * Ring::kStages * 8 : 0);
};
// Bounded wait for a stage; false after a timeout, which is reported.
struct WaitStage {
    int* status;
    long long cycles;
    FV_DEV bool operator()(uint32_t bar, uint32_t parity) const {
        if (fvp::mbar_try(bar, parity)) return true;
        const long long t0 = clock64();
        while (!fvp::mbar_try(bar, parity)) {
            if (clock64() - t0 > cycles) {
                atomicCAS(status, FV_ST_OK, FV_ST_TIMEOUT_BASE + 5);
                return false;
            }
        }
        return true;
    }
};
FV_DEV bool elect_one() {  // one lane of the converged warp
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
FV_DEV uint4 lds128(uint32_t a) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
    return r;
}
FV_DEV uint2 lds64(uint32_t a) {
    uint2 r;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a) : "memory");
    return r;
}
FV_DEV uint32_t lds32(uint32_t a) {
    uint32_t r;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a) : "memory");
    return r;
}

// Up to ROWS query rows (4 bits: 4, 8 or 16, bf16: 8 or 16).  The transposed products S^T = K . Q^T and O^T = V^T . P^T keep
// keys and head dim on the 16-wide side of the matrix instruction and the (few) query rows on the 8-wide one; the sums of
// either product may run in any order of d or key, so every lane's operands are whole 16-byte pieces as they lie in memory.
//
// A warp takes a run of tiles of its own.  Their pool rows are looked up 32 at a time, one tile a lane, a batch ahead.
// bf16, bound by HBM: a tile's K registers are loaded anew as soon as its scores are done and V's as soon as its product is, so
// that memory is always being read while the warp computes, straight into registers: 32 ragged sequences of up to 9 001 keys, 32
// heads on 8, 137 us = 6.10 TB/s, 0.93 of the measured copy bandwidth; 6 windows of 8 190 keys, 40 heads on 8, 34.5 us = 5.8 TB/s.
// 4 bits, bound by latency (issue slots 50 %, logic pipe 52 %, DRAM 53 %: nothing is full with 12 warps an SM): 32 keys are 4.3 KB, so a
// ring in shared memory runs three stages ahead: 32 sequences of up to 20 011 keys 110 us = 4.5 TB/s (loads into registers: 173).  Three
// CTAs an SM: with a fourth the registers no longer suffice, 128 against 123 us.  At most four rows stand on every other column of the products, which leaves half of the softmax: 123 -> 116 us.
template <bool Q4, int ROWS>
__global__ void __launch_bounds__(kAttnThreads, ROWS <= 8 ? 3 : 2) fv_paged_decode_kernel(const AttnArgs a) {
    constexpr int kRows = ROWS, NT = (ROWS + 7) / 8;  // groups of 8 rows, the columns of a product
    constexpr int EH = ROWS == 4 ? 1 : 2;             // columns of a product in a lane that stand for rows
    constexpr int SUB = kTile<Q4> / 16;  // products of 16 keys in a tile
    using Sm = DecodeSmem<Q4, ROWS>;
    extern __shared__ __align__(128) unsigned char decode_smem[];
    float (*sh_o)[kRows][kD + 4] = reinterpret_cast<float (*)[kRows][kD + 4]>(decode_smem);
    float (*sh_m)[kRows] = reinterpret_cast<float (*)[kRows]>(decode_smem + kWarps * kRows * (kD + 4) * 4);
    float (*sh_l)[kRows] = sh_m + kWarps;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    int b = blockIdx.x;
    const int ranges = b / a.by_splits, split = b - ranges * a.splits;
    b = ranges / a.by_blocks;
    const int rb = ranges - b * (int)a.by_blocks.d, s = b / a.by_heads, head = b - s * a.pool.kv_heads;
    const Seq seq = seq_of(a.batch, s);
    const int row0 = rb * kRows, rows = min(kRows, seq.nq * a.group - row0);
    if (rows <= 0) return;  // (the same for all key ranges of these rows)
    const int pos0 = seq.len - seq.nq;  // position of the sequence's first token of this call
    const int first = pos0 + row0 / a.by_group, last = pos0 + (row0 + rows - 1) / a.by_group;
    const Span span = span_of(a.mask, first, last, seq.len);
    const Tiles<kTile<Q4>> tiles(span);
    const int u0 = (int)((long long)tiles.count * split / a.splits), u1 = (int)((long long)tiles.count * (split + 1) / a.splits);
    const int w0 = u0 + (u1 - u0) * warp / kWarps, n_tiles = u0 + (u1 - u0) * (warp + 1) / kWarps - w0;

    // Tiles of which every row sees every key: inside the first row's end and the last row's start, or inside the sinks.
    int whole_lo, whole_hi, whole_sink;
    {
        const Span lowest = span_of(a.mask, first, first, seq.len), highest = span_of(a.mask, last, last, seq.len);
        whole_lo = highest.lo;
        whole_hi = lowest.hi;
        whole_sink = min(lowest.lo == 0 ? lowest.hi : lowest.sink, highest.lo == 0 ? highest.hi : highest.sink);
    }
    struct Feed {
        uint32_t row[SUB], whole;  // pool rows of this lane's tile (of its halves); bit i: tile i of the batch is whole
    };
    auto lookup = [&](int base) {
        Feed f;
        bool whole = false;
#pragma unroll
        for (int i = 0; i < SUB; i++) f.row[i] = kNoRow;
        if (base + lane < n_tiles) {
            const int key = tiles.key(w0 + base + lane);
#pragma unroll
            for (int i = 0; i < SUB; i++) {
                const int k = key + 16 * i;
                if (i > 0 && a.pool.log_rows > 4) {  // (the same page)
                    if (f.row[0] != kNoRow) f.row[i] = f.row[0] + 16;
                } else if (SUB == 1 || a.pool.log_rows > 4 || (k < span.hi && k + 16 > span.lo) || k < span.sink) {
                    const int page = page_of(a.pool, a.batch, s, k);
                    if (page >= 0) f.row[i] = (uint32_t)pool_row(a.pool, page, head, k);
                }
            }
            whole = f.row[0] != kNoRow && f.row[SUB - 1] != kNoRow &&
                    ((key >= whole_lo && key + kTile<Q4> <= whole_hi) || key + kTile<Q4> <= whole_sink);
        }
        f.whole = __ballot_sync(kFullWarp, whole);
        return f;
    };
    // q's rows are asked for first: they come while the page is looked up (16 sequences of up to 4 000 4-bit keys, 32 heads on 8: 20.8 -> 19.6 us).
    uint4 u[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int rq = ROWS == 4 ? ((g & 1) ? ROWS : g >> 1) : 8 * n + g, r = row0 + rq;
        if (rq < rows) {
            const int tok = r / a.by_group;
            const uint16_t* p = a.q + (size_t)(seq.q0 + tok) * a.q_tok + (size_t)(head * a.group + r - tok * a.group) * a.q_head;
#pragma unroll
            for (int i = 0; i < 4; i++) u[n][i] = *reinterpret_cast<const uint4*>(p + (Q4 ? 32 * t + 8 * i : 32 * i + 8 * t));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) u[n][i] = make_uint4(0, 0, 0, 0);
        }
    }
    Feed cur = lookup(0), nxt = lookup(32);
    Keys<Q4> kt[SUB];
    Values<Q4> vt[SUB];
    const uint8_t *lane_k = a.pool.k, *lane_v = a.pool.v;
    const uint32_t ring = fvp::smem_u32(decode_smem) + warp * Ring::kWarpBytes;
    const uint32_t bars = fvp::smem_u32(decode_smem) + Sm::kBars + warp * Ring::kStages * 8;
    // 4 bits: tile j of the batch that `cur` (j >= 32: `nxt`) holds into stage st.
    auto fill_stage = [&](int j, int st) {
        const uint32_t r0 = __shfl_sync(kFullWarp, j < 32 ? cur.row[0] : nxt.row[0], j & 31);
        const uint32_t r1 = __shfl_sync(kFullWarp, j < 32 ? cur.row[SUB - 1] : nxt.row[SUB - 1], j & 31);
        if (!elect_one()) return;
        const uint32_t bar = bars + 8 * st, dst = ring + st * Ring::kStageBytes;
        if (r0 != kNoRow && r1 == r0 + 16) {
            fvp::mbar_expect_tx(bar, Ring::kStageBytes);
            fvp::bulk_load(dst, a.pool.k + (size_t)r0 * kQ4Bytes, 2048, bar);
            fvp::bulk_load(dst + Ring::kV, a.pool.v + (size_t)r0 * kQ4Bytes, 2048, bar);
            fvp::bulk_load(dst + Ring::kKs, a.pool.k_scale + r0, 128, bar);
            fvp::bulk_load(dst + Ring::kVs, a.pool.v_scale + r0, 128, bar);
        } else {  // two pages, or a half without one
            fvp::mbar_expect_tx(bar, ((r0 != kNoRow) + (r1 != kNoRow)) * Ring::kHalfBytes);
#pragma unroll 1
            for (uint32_t i = 0; i < 2; i++) {
                const uint32_t row = i ? r1 : r0;
                if (row == kNoRow) continue;
                fvp::bulk_load(dst + 1024 * i, a.pool.k + (size_t)row * kQ4Bytes, 1024, bar);
                fvp::bulk_load(dst + Ring::kV + 1024 * i, a.pool.v + (size_t)row * kQ4Bytes, 1024, bar);
                fvp::bulk_load(dst + Ring::kKs + 64 * i, a.pool.k_scale + row, 64, bar);
                fvp::bulk_load(dst + Ring::kVs + 64 * i, a.pool.v_scale + row, 64, bar);
            }
        }
    };
    if constexpr (Q4) {
        if (lane == 0) {
            for (int st = 0; st < Ring::kStages; st++) fvp::mbar_init(bars + 8 * st, 1);
            fvp::mbar_init_fence();
        }
        __syncwarp();
        for (int st = 0; st < Ring::kStages && st < n_tiles; st++) fill_stage(st, st);
    } else {
        lane_k += Keys<false>::lane_offset(g, t);
        lane_v += Values<false>::lane_offset(g, t);
        const uint32_t row = __shfl_sync(kFullWarp, cur.row[0], 0);
        kt[0].load(lane_k, row);
        vt[0].load(lane_v, row);
    }

    // The row of group n that column 2 t + e stands for.  With at most four rows (4 bits) they take the even columns: the odd ones of a
    // lane then have no softmax.
    auto row_of = [&](int n, int e) { return ROWS == 4 ? t : 8 * n + 2 * t + e; };
    // Q^T: column g of each group of 8 rows, in the order of d that the keys' lanes hold.  4 bits: as f16, scaled by a power
    // of two that brings the row's largest value to 2^8 .. 2^9 (what falls below f16's range is 2^-32 of that), which goes into
    // the row's softmax scale; qsum: the row's sum in the same units.
    uint32_t qf[NT][16];
    float qsum[NT][2], sl2[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        if constexpr (Q4) {
            float top = 0.f, sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float x = lo_f(word(u[n][i], j)), y = hi_f(word(u[n][i], j));
                    top = fmaxf(top, fmaxf(fabsf(x), fabsf(y)));
                    sum += x + y;
                }
            }
            top = fmaxf(top, __shfl_xor_sync(kFullWarp, top, 1));
            top = fmaxf(top, __shfl_xor_sync(kFullWarp, top, 2));
            sum += __shfl_xor_sync(kFullWarp, sum, 1);
            sum += __shfl_xor_sync(kFullWarp, sum, 2);
            // 2^(8 - floor(log2 top)) and its inverse, from the exponent field (kept inside the normal numbers)
            const int e = min(max((int)(__float_as_uint(top) >> 23), 16), 246);
            const float up = __uint_as_float((uint32_t)(262 - e) << 23), down = __uint_as_float((uint32_t)(e - 8) << 23);
#pragma unroll
            for (int i = 0; i < 4; i++) {  // pairs (d, d + 4) of eight values: the nibbles that one mask gives
                const float up16 = up * 0.0625f;  // (the second and fourth pair meet codes that stand for 16 n)
                qf[n][4 * i + 0] = pack_f16x2(lo_f(u[n][i].x) * up, lo_f(u[n][i].z) * up);
                qf[n][4 * i + 1] = pack_f16x2(hi_f(u[n][i].x) * up16, hi_f(u[n][i].z) * up16);
                qf[n][4 * i + 2] = pack_f16x2(lo_f(u[n][i].y) * up, lo_f(u[n][i].w) * up);
                qf[n][4 * i + 3] = pack_f16x2(hi_f(u[n][i].y) * up16, hi_f(u[n][i].w) * up16);
            }
            // (an infinity in q: the scores are not numbers, where f16's largest value and zero * sum(q) would give something finite)
            const float scaled = sum * up * (1.f / kCodeUnit), back = top < -neg_inf() ? a.sl2 * down * kCodeUnit : __int_as_float(0x7fffffff);
            qsum[n][0] = __shfl_sync(kFullWarp, scaled, 8 * t);      // of row 2 t, which the lanes 4 (2 t) .. hold
            qsum[n][1] = __shfl_sync(kFullWarp, scaled, 8 * t + 4);  // of row 2 t + 1
            sl2[n][0] = __shfl_sync(kFullWarp, back, 8 * t);
            sl2[n][1] = __shfl_sync(kFullWarp, back, 8 * t + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int j = 0; j < 4; j++) qf[n][4 * i + j] = word(u[n][i], j);
            }
            qsum[n][0] = qsum[n][1] = 0.f;
            sl2[n][0] = sl2[n][1] = a.sl2;
        }
    }

    float o[NT][8][4];  // O^T: d by lane g and tile, rows row_of(n, 0) and row_of(n, 1)
    float m[NT][2], l[NT][2], z[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int i = 0; i < 8; i++) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
        m[n][0] = m[n][1] = neg_inf();
        l[n][0] = l[n][1] = z[n][0] = z[n][1] = 0.f;
    }

    int st = 0;  // 4 bits: the stage of this step and the phase of its barrier
    uint32_t phase = 0;
    const WaitStage wait_stage{a.batch.status - 1, a.wait_cycles};
    for (int v = 0; v < n_tiles; v++) {
        const int i0 = v & 31;
        if (v > 0 && i0 == 0) {
            cur = nxt;
            nxt = lookup(v + 32);
        }
        const bool more = v + 1 < n_tiles;
        uint32_t next_row = kNoRow, stage = 0;
        if constexpr (Q4) {
            stage = ring + st * Ring::kStageBytes;
            if (!__all_sync(kFullWarp, wait_stage(bars + 8 * st, phase))) {  // (given up and reported: what was asked for must land)
                for (int k = 0; k < Ring::kStages && v + k < n_tiles; k++) {
                    fvp::mbar_drain(bars + 8 * st, phase);
                    st = st + 1 == Ring::kStages ? 0 : st + 1;
                    phase ^= st == 0;
                }
                break;
            }
#pragma unroll
            for (int i = 0; i < SUB; i++) {
                kt[i].k0 = lds128(stage + 1024 * i + 64 * key_of_row(g) + 16 * t);
                kt[i].k1 = lds128(stage + 1024 * i + 64 * key_of_row(g) + 512 + 16 * t);
                kt[i].s0 = lds32(stage + Ring::kKs + 64 * i + 4 * key_of_row(g));
                kt[i].s1 = lds32(stage + Ring::kKs + 64 * i + 4 * key_of_row(g) + 32);
            }
        } else {
            next_row = __shfl_sync(kFullWarp, i0 + 1 < 32 ? cur.row[0] : nxt.row[0], (i0 + 1) & 31);
        }

        // c0, c1: key g, rows row_of(n, 0) and (n, 1); c2, c3: key g + 8.
        float c[SUB][NT][4];
#pragma unroll
        for (int i = 0; i < SUB; i++) {
#pragma unroll
            for (int n = 0; n < NT; n++) c[i][n][0] = c[i][n][1] = c[i][n][2] = c[i][n][3] = 0.f;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                uint32_t x0[4], x1[4];
                if constexpr (Q4) {
                    codes_f16(word(kt[i].k0, w), x0);
                    codes_f16(word(kt[i].k1, w), x1);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        x0[j] = word(kt[i].k0[w], j);
                        x1[j] = word(kt[i].k1[w], j);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
#pragma unroll
                    for (int n = 0; n < NT; n++) mma<Q4>(c[i][n], x0[j], x1[j], x0[j + 1], x1[j + 1], qf[n][4 * w + j], qf[n][4 * w + j + 1]);
                }
            }
            if constexpr (Q4) {  // q . (zero + step code) = step (q . n) + (zero - 8 step) sum(q), all by 2^-24
                const float s0 = lo_f(kt[i].s0), s1 = lo_f(kt[i].s1);
                const float z0 = fmaf(-8.f, s0, hi_f(kt[i].s0)), z1 = fmaf(-8.f, s1, hi_f(kt[i].s1));
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int e = 0; e < EH; e++) {
                        c[i][n][e] = fmaf(c[i][n][e], s0, z0 * qsum[n][e]);
                        c[i][n][2 + e] = fmaf(c[i][n][2 + e], s1, z1 * qsum[n][e]);
                    }
                }
            }
            if constexpr (!Q4) {
                if (more) kt[i].load(lane_k, next_row);
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) vt[i].a[k] = lds64(stage + Ring::kV + 1024 * i + 64 * (key_of_row(2 * t + (k & 1)) + 8 * (k >> 1)) + 8 * g);
                vt[i].s0 = lds32(stage + Ring::kVs + 64 * i + 4 * key_of_row(g));
                vt[i].s1 = lds32(stage + Ring::kVs + 64 * i + 4 * key_of_row(g) + 32);
            }
        }

        if (!((cur.whole >> i0) & 1u)) {
#pragma unroll
            for (int i = 0; i < SUB; i++) {
                const bool none = __shfl_sync(kFullWarp, cur.row[i], i0) == kNoRow;
                const int key0 = tiles.key(w0 + v) + 16 * i;
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int e = 0; e < EH; e++) {
                        const int r = row0 + row_of(n, e), p = pos0 + r / a.by_group;
                        const Span sp = span_of(a.mask, p, p, seq.len);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int j = key0 + (Q4 ? key_of_row(g) : g) + 8 * h;
                            if (none || !((j >= sp.lo && j < sp.hi) || j < sp.sink)) c[i][n][2 * h + e] = neg_inf();
                        }
                    }
                }
                // Values that no row of this block may see count as zero whatever they hold (0 times NaN is NaN).
                auto seen = [&](int j) { return !none && ((j >= span.lo && j < span.hi) || j < span.sink); };
                if constexpr (Q4) {
                    if (!seen(key0 + key_of_row(g))) vt[i].s0 = 0u;
                    if (!seen(key0 + key_of_row(g) + 8)) vt[i].s1 = 0u;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (!seen(key0 + 2 * t + (k & 1) + 8 * (k >> 1))) vt[i].a[k] = vt[i].b[k] = make_uint4(0, 0, 0, 0);
                }
            }
        }
        // Streaming softmax: P against the reference the row has; exact maxima are taken only where there is none yet, or
        // where a sum comes out above its guard (the reference cancels in O / l).  bf16: P itself must fit bf16 and the f32
        // sums, 2^40.  4 bits: V's step goes into P (the zeros are summed apart), so that both operands of the product are
        // exact but for P step, which is rounded to f16 and must fit it: 2^14; a reference bounds P step by 2^8, so that only
        // what is 2^32 below the largest is lost at f16's lower end.
        constexpr float kGuard = Q4 ? 16384.f : 1099511627776.f, kGuardP = 1.2676506e30f;  // 2^100
        float p[SUB][NT][4] = {}, ps[SUB][NT][4], sum = 0.f, sum_s = 0.f;
        auto weigh = [&vt, &p, &ps](int i, int n) {
            ps[i][n][1] = ps[i][n][3] = 0.f;
#pragma unroll
            for (int e = 0; e < EH; e++) {
                ps[i][n][e] = Q4 ? p[i][n][e] * vt[i].step(0) : p[i][n][e];
                ps[i][n][2 + e] = Q4 ? p[i][n][2 + e] * vt[i].step(1) : p[i][n][2 + e];
            }
        };
#pragma unroll
        for (int i = 0; i < SUB; i++) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int e = 0; e < EH; e++) {
                    p[i][n][e] = fvp::ex2(fmaf(c[i][n][e], sl2[n][e], -m[n][e]));
                    p[i][n][2 + e] = fvp::ex2(fmaf(c[i][n][2 + e], sl2[n][e], -m[n][e]));
                }
                weigh(i, n);
                if (Q4) sum += (p[i][n][0] + p[i][n][1]) + (p[i][n][2] + p[i][n][3]);
                sum_s += (ps[i][n][0] + ps[i][n][1]) + (ps[i][n][2] + ps[i][n][3]);
            }
        }
        if (__any_sync(kFullWarp, !(sum_s <= kGuard) || (Q4 && !(sum <= kGuardP)))) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int e = 0; e < EH; e++) {
                    float mx = neg_inf();
#pragma unroll
                    for (int i = 0; i < SUB; i++) {
                        const float t0 = c[i][n][e] * sl2[n][e], t1 = c[i][n][2 + e] * sl2[n][e];
                        if constexpr (Q4) {  // (a key whose values are all equal has step 0)
                            mx = fmaxf(mx, fmaxf(t0 + fmaxf(log2f(lo_f(vt[i].s0)), -60.f), t1 + fmaxf(log2f(lo_f(vt[i].s1)), -60.f)));
                        } else {
                            mx = fmaxf(mx, fmaxf(t0, t1));
                        }
                    }
                    mx = fmaxf(mx, __shfl_xor_sync(kFullWarp, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(kFullWarp, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(kFullWarp, mx, 16));
                    if (Q4) mx -= 8.f;
                    if (mx > m[n][e]) {
                        const float f = fvp::ex2(m[n][e] - mx);  // 0 when there was no reference
                        m[n][e] = mx;
                        l[n][e] *= f;
                        z[n][e] *= f;
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            o[n][i][e] *= f;
                            o[n][i][2 + e] *= f;
                        }
                    }
                    const float ref = m[n][e] == neg_inf() ? 0.f : m[n][e];  // (a row that has seen nothing yet: P = 0)
#pragma unroll
                    for (int i = 0; i < SUB; i++) {
                        p[i][n][e] = fvp::ex2(fmaf(c[i][n][e], sl2[n][e], -ref));
                        p[i][n][2 + e] = fvp::ex2(fmaf(c[i][n][2 + e], sl2[n][e], -ref));
                    }
                }
#pragma unroll
                for (int i = 0; i < SUB; i++) weigh(i, n);
            }
        }
#pragma unroll
        for (int i = 0; i < SUB; i++) {
            uint32_t pb[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int e = 0; e < EH; e++) l[n][e] += p[i][n][e] + p[i][n][2 + e];
                const uint32_t pk0 = pack_p<Q4>(ps[i][n][0], ps[i][n][1]), pk1 = pack_p<Q4>(ps[i][n][2], ps[i][n][3]);
                if constexpr (Q4) {
                    // P zero - 8 (P step), the latter as the product takes it: its rounding then meets the code, not the 8 as well
                    // (which could be a hundred times the value).
                    float r[4];
                    unpack_p<true>(pk0, r[0], r[1]);
                    unpack_p<true>(pk1, r[2], r[3]);
#pragma unroll
                    for (int e = 0; e < EH; e++)
                        z[n][e] = fmaf(-8.f, r[e] + r[2 + e], fmaf(p[i][n][e], hi_f(vt[i].s0), fmaf(p[i][n][2 + e], hi_f(vt[i].s1), z[n][e])));
                }
                pb[n][0] = transpose8(pk0);
                pb[n][1] = transpose8(pk1);
            }
            // O^T += V^T . P^T: the pair of one d and two neighbouring keys comes out of two keys' words.
            if constexpr (Q4) {
                // Words of both keys' nibbles 0-3 (h = 0) and 4-7, key by key in the halves: codes_f16 would pair nibble k
                // with k + 4 of one key's word; here the two halves are the two keys.
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t sel = h ? 0x7632 : 0x5410;
                    uint32_t x0[4], x1[4], x2[4], x3[4];
                    codes_f16(prmt(vt[i].a[0].x, vt[i].a[1].x, sel), x0);
                    codes_f16(prmt(vt[i].a[0].y, vt[i].a[1].y, sel), x1);
                    codes_f16(prmt(vt[i].a[2].x, vt[i].a[3].x, sel), x2);
                    codes_f16(prmt(vt[i].a[2].y, vt[i].a[3].y, sel), x3);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
#pragma unroll
                        for (int n = 0; n < NT; n++) mma<true>(o[n][4 * h + k], x0[k], x1[k], x2[k], x3[k], pb[n][0], pb[n][1]);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const uint32_t sel = (k & 1) ? 0x7632 : 0x5410;
                    const uint32_t a0 = prmt(word(vt[i].a[0], k / 2), word(vt[i].a[1], k / 2), sel);
                    const uint32_t a1 = prmt(word(vt[i].b[0], k / 2), word(vt[i].b[1], k / 2), sel);
                    const uint32_t a2 = prmt(word(vt[i].a[2], k / 2), word(vt[i].a[3], k / 2), sel);
                    const uint32_t a3 = prmt(word(vt[i].b[2], k / 2), word(vt[i].b[3], k / 2), sel);
#pragma unroll
                    for (int n = 0; n < NT; n++) mma<false>(o[n][k], a0, a1, a2, a3, pb[n][0], pb[n][1]);
                }
            }
            if constexpr (!Q4) {
                if (more) vt[i].load(lane_v, next_row);
            }
        }
        if constexpr (Q4) {
            __syncwarp();  // every lane has its operands out of the stage: fill it again
            if (v + Ring::kStages < n_tiles) fill_stage(i0 + Ring::kStages, st);
            st = st + 1 == Ring::kStages ? 0 : st + 1;
            phase ^= st == 0;
            // O holds sum P step n and z the sum of P (zero - 8 step): both grow with every key, their sum does not.  Every 256
            // keys z goes into O, so that f32 (whose sums the matrix unit truncates) never carries more than those keys' offset.
            if ((v & 7) == 7) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int e = 0; e < EH; e++) {
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) z[n][e] += __shfl_xor_sync(kFullWarp, z[n][e], d);
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            o[n][k][e] = fmaf(z[n][e], ((k & 1) ? 16.f : 1.f) / kCodeUnit, o[n][k][e]);
                            o[n][k][2 + e] = fmaf(z[n][e], ((k & 1) ? 16.f : 1.f) / kCodeUnit, o[n][k][2 + e]);
                        }
                        z[n][e] = 0.f;
                    }
                }
            }
        }
    }

    if (Q4) __syncthreads();  // (the join's memory is the ring's)
    // The four warps' results side by side, then joined.
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int e = 0; e < EH; e++) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                l[n][e] += __shfl_xor_sync(kFullWarp, l[n][e], d);
                z[n][e] += __shfl_xor_sync(kFullWarp, z[n][e], d);
            }
            if (!(l[n][e] >= 0.f)) m[n][e] = -neg_inf();  // a score that is not a number: the row comes out as one that is not
            const int r = row_of(n, e);
            if (g == 0) {
                sh_m[warp][r] = m[n][e];
                sh_l[warp][r] = l[n][e];
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float unit = Q4 ? ((i & 1) ? kCodeUnit / 16.f : kCodeUnit) : 1.f;
                sh_o[warp][r][Q4 ? 16 * g + i : 8 * g + i] = fmaf(o[n][i][e], unit, z[n][e]);
                sh_o[warp][r][Q4 ? 16 * g + 8 + i : 64 + 8 * g + i] = fmaf(o[n][i][2 + e], unit, z[n][e]);
            }
        }
    }
    __syncthreads();
    // A warp takes whole rows, warp + 4 i, four values a lane, all of them at a time (a value a thread, row after row, took 5 us of 16 rows).
    auto out_row = [&](int r) {
        const int tok = (row0 + r) / a.by_group;
        return (size_t)(seq.q0 + tok) * a.heads + head * a.group + (row0 + r - tok * a.group);
    };
    auto add = [](float4& acc, float f, const float4& x) {  // (what has no weight may hold anything)
        if (f == 0.f) return;
        acc.x = fmaf(f, x.x, acc.x);
        acc.y = fmaf(f, x.y, acc.y);
        acc.z = fmaf(f, x.z, acc.z);
        acc.w = fmaf(f, x.w, acc.w);
    };
    auto pack = [](const float4& x, float by) {
        return make_uint2(fvp::pack_bf16x2(x.x * by, x.y * by), fvp::pack_bf16x2(x.z * by, x.w * by));
    };
    constexpr int kMine = kRows / kWarps;
    float top[kMine], sum[kMine];  // the reference of a row, and the sum of P against it
    float4 acc[kMine];
#pragma unroll
    for (int i = 0; i < kMine; i++) {
        const int r = warp + kWarps * i;
        top[i] = sh_m[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; w++) top[i] = fmaxf(top[i], sh_m[w][r]);
        sum[i] = 0.f;
        acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float f = sh_m[w][r] == neg_inf() ? 0.f : fvp::ex2(sh_m[w][r] - top[i]);
            sum[i] = fmaf(f, sh_l[w][r], sum[i]);
            add(acc[i], f, *reinterpret_cast<const float4*>(&sh_o[w][r][4 * lane]));
        }
    }
    if (a.cluster) {
        // The key ranges of these rows are the CTAs of one cluster: each has joined its own warps, then the rows are dealt to
        // the CTAs, which read each other's parts over distributed shared memory, in the order of the ranges.
        cg::cluster_group cluster = cg::this_cluster();
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kMine; i++) {  // (rows of this warp's own)
            const int r = warp + kWarps * i;
            *reinterpret_cast<float4*>(&sh_o[0][r][4 * lane]) = acc[i];
            if (lane == 0) {
                sh_m[0][r] = top[i];
                sh_l[0][r] = sum[i];
            }
        }
        cluster.sync();
        for (int r = split + a.splits * warp; r < rows; r += a.splits * kWarps) {
            // (every load of the row on its way before the first is used: one after the other they took 2 us)
            float mi[kMaxCluster], li[kMaxCluster];
            float4 oi[kMaxCluster];
#pragma unroll
            for (int i = 0; i < kMaxCluster; i++) {
                mi[i] = neg_inf();
                li[i] = 0.f;
                oi[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < a.splits) {
                    mi[i] = *cluster.map_shared_rank(&sh_m[0][r], i);
                    li[i] = *cluster.map_shared_rank(&sh_l[0][r], i);
                    oi[i] = *cluster.map_shared_rank(reinterpret_cast<float4*>(&sh_o[0][r][4 * lane]), i);
                }
            }
            float m_all = mi[0], l_all = 0.f;
            float4 o_all = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 1; i < kMaxCluster; i++) m_all = fmaxf(m_all, mi[i]);
#pragma unroll
            for (int i = 0; i < kMaxCluster; i++) {
                const float f = mi[i] == neg_inf() ? 0.f : fvp::ex2(mi[i] - m_all);
                l_all = fmaf(f, li[i], l_all);
                add(o_all, f, oi[i]);
            }
            *reinterpret_cast<uint2*>(a.out + out_row(r) * kD + 4 * lane) = pack(o_all, m_all == neg_inf() ? 0.f : 1.f / l_all);
        }
        cluster.sync();  // (no CTA leaves while another one still reads its part)
        return;
    }
#pragma unroll
    for (int i = 0; i < kMine; i++) {
        const int r = warp + kWarps * i;
        if (r >= rows) break;
        const float by = top[i] == neg_inf() ? 0.f : 1.f / sum[i];
        const size_t oi = out_row(r);
        if (a.splits == 1) {
            *reinterpret_cast<uint2*>(a.out + oi * kD + 4 * lane) = pack(acc[i], by);
        } else {
            const size_t pi = (size_t)split * a.batch.tokens * a.heads + oi;
            *reinterpret_cast<float4*>(a.part_o + pi * kD + 4 * lane) = make_float4(acc[i].x * by, acc[i].y * by, acc[i].z * by, acc[i].w * by);
            if (lane == 0) a.part_lse[pi] = sum[i] > 0.f ? top[i] + log2f(sum[i]) : top[i];  // (no key: -inf; not a number: +inf)
        }
    }
}

// out = sum_s w_s O_s, w_s = 2^(lse_s - max) / sum: one warp per row, parts in their order.  Rows behind the last
// sequence stay as they were.
__global__ void __launch_bounds__(kAttnThreads) fv_paged_merge_kernel(const AttnArgs a) {
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5), rows = (long long)a.batch.tokens * a.heads;
    if (row >= rows) return;
    const int tok = (int)(row / a.heads);
    const int s = seq_of_token(a.batch.cu_q, a.batch.seqs, tok, lane);
    if (s >= a.batch.seqs) return;
    const Seq seq = seq_of(a.batch, s);
    if (tok < seq.q0 || tok >= seq.q0 + seq.nq) return;
    // (a lane a weight, and the loads of eight parts on their way before the first is used: one sequence of 20 011 keys, 8 heads on 1, 64
    // parts, 17 us for both kernels; one part after the other 27)
    float top = neg_inf();
    for (int i = lane; i < a.splits; i += 32) top = fmaxf(top, a.part_lse[(size_t)i * rows + row]);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullWarp, top, d));
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    for (int i0 = 0; i0 < a.splits && top != neg_inf(); i0 += 32) {
        const float w = i0 + lane < a.splits ? fvp::ex2(a.part_lse[(size_t)(i0 + lane) * rows + row] - top) : 0.f;
        const int here = min(32, a.splits - i0);
        constexpr int kAhead = 8;
        for (int i = 0; i < here; i += kAhead) {
            float4 x[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; j++)
                x[j] = __ldcg(reinterpret_cast<const float4*>(a.part_o + ((size_t)(i0 + min(i + j, here - 1)) * rows + row) * kD + 4 * lane));
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                const float wj = __shfl_sync(kFullWarp, w, (i + j) & 31);
                if (i + j >= here || wj == 0.f) continue;
                sum += wj;
                acc.x = fmaf(wj, x[j].x, acc.x);
                acc.y = fmaf(wj, x[j].y, acc.y);
                acc.z = fmaf(wj, x[j].z, acc.z);
                acc.w = fmaf(wj, x[j].w, acc.w);
            }
        }
    }
    if (top != neg_inf()) {
        const float inv = 1.f / sum;
        acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
    }
    *reinterpret_cast<uint2*>(a.out + (size_t)row * kD + 4 * lane) =
        make_uint2(fvp::pack_bf16x2(acc.x, acc.y), fvp::pack_bf16x2(acc.z, acc.w));
}

template <bool Q4>
__global__ void __launch_bounds__(Roles<Q4>::kThreads, 1)
fv_paged_chunk_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                      const __grid_constant__ ChunkJob jb) {
#if defined(__CUDA_ARCH_FEAT_SM100_ALL) || defined(__CUDA_ARCH_FEAT_SM103_ALL)
    extern __shared__ __align__(1024) unsigned char fv_smem[];
    chunk_persistent<Q4>(&mq, &mk, &mv, jb, fv_smem);
#endif
}

// The items that the chunk kernel's runs cut: the part that begins the item lies with the run that `split` belongs to, the
// others with the runs after it.  A warp a row; which parts there are is worked out once per block, a lane a run, and the
// weights of a row a lane a part (one lane doing both for every row took 34 us for the 147 cuts of a launch, this 8).
constexpr int kJoinBlocks = 16;  // of a split item's 256 rows
constexpr int kMaxRuns = 1024;   // of a launch
__global__ void __launch_bounds__(kAttnThreads) fv_paged_join_kernel(const ChunkJob jb) {
    __shared__ int slots[kMaxRuns];
    __shared__ int count;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x / kJoinBlocks, block = blockIdx.x - c * kJoinBlocks;
    const ChunkSplit sp = jb.split[c];
    if (!sp.valid) return;
    if (warp == 0) {
        int n = 1;
        if (lane == 0) slots[0] = 2 * c + 1;
        for (int k0 = c + 1; k0 < sp.runs; k0 += 32) {
            const int k = k0 + lane;
            bool mine = false, past = true;
            if (k < sp.runs) {
                const long long y = sp.total * k / sp.runs - sp.start, y1 = sp.total * (k + 1) / sp.runs - sp.start;
                past = y >= sp.cost;
                mine = !past && tile_behind((int)min(y1, (long long)sp.cost), sp.tiles) > tile_behind((int)y, sp.tiles);
            }
            const uint32_t have = __ballot_sync(kFullWarp, mine);
            const int at = n + __popc(have & ((1u << lane) - 1u));
            if (mine && at < kMaxRuns) slots[at] = 2 * k;
            n = min(n + __popc(have), kMaxRuns);
            if (__any_sync(kFullWarp, past)) break;
        }
        if (lane == 0) count = n;
    }
    __syncthreads();
    const int n = count;
    // The warp's rows go together, so that the loads of all of them are in flight at a time (one after the other: 34 against 15 us
    // under the profiler for 88 runs over 6 items of 40 rows, 12 against 7.4 for 148 over 40 of 256).
    constexpr int kRowsHere = 2 * kChunkRows / kJoinBlocks / kWarps;
    const int r0 = block * kRowsHere * kWarps + warp;  // its rows: r0 + kWarps i
    long long out[kRowsHere];  // -1: none
    bool any = false;
#pragma unroll
    for (int i = 0; i < kRowsHere; i++) {
        const int r = r0 + kWarps * i, tile = r / kChunkRows, row = r - tile * kChunkRows;
        const int row_tok = row / jb.by_group, tok = sp.tok0 + tile * jb.tile_tokens + row_tok;
        const bool live = row_tok < jb.tile_tokens && tok < sp.nq;
        out[i] = live ? (long long)(sp.q0 + tok) * jb.heads + sp.head * jb.group + (row - row_tok * jb.group) : -1;
        any |= live;
    }
    if (!any) return;
    float top[kRowsHere], sum[kRowsHere];
    float4 acc[kRowsHere];
#pragma unroll
    for (int i = 0; i < kRowsHere; i++) {
        top[i] = neg_inf();
        sum[i] = 0.f;
        acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    auto lse = [&](int k, int i) { return jb.part_lse[(size_t)slots[k] * 2 * kChunkRows + r0 + kWarps * i]; };
    for (int k = lane; k < n; k += 32) {
#pragma unroll
        for (int i = 0; i < kRowsHere; i++)
            if (out[i] >= 0) top[i] = fmaxf(top[i], lse(k, i));
    }
#pragma unroll
    for (int i = 0; i < kRowsHere; i++) {
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(kFullWarp, top[i], d));
    }
    for (int k0 = 0; k0 < n; k0 += 32) {
        float w[kRowsHere];
#pragma unroll
        for (int i = 0; i < kRowsHere; i++) w[i] = k0 + lane < n && top[i] != neg_inf() ? fvp::ex2(lse(k0 + lane, i) - top[i]) : 0.f;
        const int here = min(32, n - k0);
        constexpr int kAhead = 4;  // parts whose loads are on their way before the first is used
        for (int k = 0; k < here; k += kAhead) {
            float4 x[kAhead][kRowsHere];
#pragma unroll
            for (int j = 0; j < kAhead; j++) {  // (also of rows that are none: their sums are not stored)
                const float* part = jb.part_o + ((size_t)slots[k0 + min(k + j, here - 1)] * 2 * kChunkRows + r0) * kD + 4 * lane;
#pragma unroll
                for (int i = 0; i < kRowsHere; i++) x[j][i] = __ldcg(reinterpret_cast<const float4*>(part + (size_t)kWarps * i * kD));
            }
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                if (k + j >= here) break;
#pragma unroll
                for (int i = 0; i < kRowsHere; i++) {
                    const float wk = __shfl_sync(kFullWarp, w[i], k + j);
                    sum[i] += wk;
                    acc[i].x = fmaf(wk, x[j][i].x, acc[i].x);
                    acc[i].y = fmaf(wk, x[j][i].y, acc[i].y);
                    acc[i].z = fmaf(wk, x[j][i].z, acc[i].z);
                    acc[i].w = fmaf(wk, x[j][i].w, acc[i].w);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kRowsHere; i++) {
        if (out[i] < 0) continue;
        const float inv = sum[i] > 0.f ? 1.f / sum[i] : 0.f;
        *reinterpret_cast<uint2*>(jb.out + (size_t)out[i] * kD + 4 * lane) =
            make_uint2(fvp::pack_bf16x2(acc[i].x * inv, acc[i].y * inv), fvp::pack_bf16x2(acc[i].z * inv, acc[i].w * inv));
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------

struct Shape {
    bool chunk;  // the tensor-core kernel for long chunks
    int splits, row_blocks, block_rows, tile_tokens;
    bool cluster;
    int ctas, phases;  // of the chunk kernel
};
constexpr long long kL2Bytes = 126ll << 20;
// Key ranges: as many as fill the SMs once; where the rows alone nearly do, three times over, so that ragged ends even
// out.  Up to kMaxCluster ranges are one cluster, which joins its parts itself.  More need the merge kernel, which costs about 4 us: they
// are taken where they shorten a warp's run of tiles (0.72 us for 16 keys of bf16, 0.34 us of 4 bits) by more than that, with at least
// four of them left to it; of 4 bits, bound by the SMs' own pipes, two CTAs an SM are enough.  (One sequence of 20 011 keys, 32 heads on 8:
// 25 us in 55 ranges of bf16, 48 in 8; 16 us in 32 ranges of 4 bits, 20 in 8.  Of 4 001 keys: 14 and 12; 12 and 9.)
// `ctas` blocks of rows, of which `resident` run at a time.
static int key_ranges(long long ctas, int resident, long long keys, bool q4, int sms) {
    const long long tiles = (keys + 15) / 16, most = (tiles + 2 * kWarps - 1) / (2 * kWarps);  // at least 32 keys per warp
    long long n = resident / ctas;
    if (n < 2) n = (3ll * resident + ctas - 1) / ctas;
    if (n > kMaxCluster) {
        const long long full = q4 ? 2ll * sms / ctas : n, whole = tiles / (4 * kWarps);
        n = full < whole ? full : whole;
        if (n <= kMaxCluster || (q4 ? 0.34 : 0.72) * (double)(tiles / kWarps) * (1.0 / kMaxCluster - 1.0 / (double)n) < 4.0) n = kMaxCluster;
    }
    n = n < most ? n : most;
    return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
// How a call is cut.  Few rows per kv head: blocks of up to 16 rows, and the keys in ranges.  Many: items of 2 x 128 rows, one CTA
// per SM.  Which of the two: an estimate of both in us, fitted to 326 calls of 20 to 800 rows, 1 to 16 sequences of 200 to 20 011 keys, 1 and 8
// kv heads, both page formats, over which the choice costs 0.7 % more than the better kernel would, at worst half as much again (96 rows over
// 20 011 4-bit keys of 8 kv heads).  E.g. 8 kv heads, bf16: one sequence of
// 20 011 keys 20 rows 31 us in blocks of rows and 43 in items, 96 rows 116 and 43; sixteen of 200 keys 48 rows 17 and 19, 400 rows 51 and 27.
// FV_PAGED_KERNEL=rows or items (kept for A/B) takes the choice away.
static bool take_items(long long planes, long long rows, long long keys, bool q4, int sms) {
    const char* e = getenv("FV_PAGED_KERNEL");
    if (e && strcmp(e, "items") == 0) return true;
    if ((e && strcmp(e, "rows") == 0) || rows <= 16) return false;
    const long long ctas = planes * ((rows + 15) / 16);
    const int resident = 2 * sms, n = key_ranges(ctas, resident, keys, q4, sms);
    const double load = (double)ctas * n / resident, waves = load <= 1.0 ? 1.0 : 0.5 * (load + ceil(load));  // (their CTAs end at different times)
    const double in_rows = 5.0 + waves * ((q4 ? 3.8 : 2.2) + (q4 ? 0.49 : 0.85) * (double)keys / (16.0 * kWarps * n)) + (n > kMaxCluster ? 4.0 : 0.0);
    const double items = (double)planes * (double)((rows + 255) / 256), line = items * (double)((keys + kChunkTile - 1) / kChunkTile + kItemCost);
    const double runs = line < (double)kLeastRun * sms ? line / kLeastRun : (double)sms, parts = runs / items;
    const double in_items = (q4 ? 4.9 + 1.83 * line / runs : 4.3 + 1.66 * line / runs) + (parts > 1.0 ? 8.8 + 0.64 * (parts - 1.0) : 0.0);
    return in_items < in_rows;
}
static Shape shape_of(const fv_paged_kv* kv, const fv_paged_batch* b, int tokens, int heads, const Mask& m, int sms) {
    Shape s;
    const int group = heads / kv->kv_heads, max_q = b->max_q < tokens ? b->max_q : tokens;
    const long long rows = (long long)max_q * group;
    long long keys = b->max_kv;
    if (m.block > 0 && m.window > 0) {  // rows of one block see window blocks and the sinks, max_q rows a little more
        const long long most = ((long long)m.window + m.sink + 1) * m.block + max_q;
        keys = most < keys ? most : keys;
    }
    const bool q4 = kv->format == FV_PAGE_Q4;
    s.chunk = group <= kChunkRows && take_items((long long)b->seqs * kv->kv_heads, rows, keys, q4, sms);
    s.tile_tokens = s.chunk ? kChunkRows / group : 0;
    s.cluster = false;
    if (s.chunk) {
        s.block_rows = 0;
        s.splits = 1;
        s.row_blocks = (max_q + 2 * s.tile_tokens - 1) / (2 * s.tile_tokens);
        // (an upper bound of the line's length: with little work no more CTAs are launched than may find a run)
        const long long longest = (long long)b->seqs * kv->kv_heads * s.row_blocks * ((b->max_kv + kChunkTile - 1) / kChunkTile + kItemCost);
        const long long most = longest / kLeastRun;
        s.ctas = (int)(most < 1 ? 1 : most < sms ? most : sms);
        // Every CTA streams the keys of its items.  Where the keys of all items are more than L2 holds, the line is gone through in
        // four phases, all CTAs on a quarter of it at a time (4 680 rows x 40 heads over 28 080 bf16 keys: 3 297 -> 2 901 us, 12 heads:
        // 924 -> 827 us); where they fit that only makes more parts (1 501-token chunks over 69 MB of keys: 358 -> 422 us).
        const long long bytes = keys * b->seqs * kv->kv_heads * (q4 ? 2 * kQ4Bytes + 8 : 4 * kD);
        s.phases = bytes > kL2Bytes && longest / ((long long)s.ctas * kMaxPhases) >= 32 && s.ctas * kMaxPhases <= kMaxRuns ? kMaxPhases : 1;
        return s;
    }
    s.block_rows = rows > 8 ? 16 : rows <= 4 && q4 ? 4 : 8;
    s.row_blocks = (int)((rows + s.block_rows - 1) / s.block_rows);
    const long long ctas = (long long)b->seqs * kv->kv_heads * s.row_blocks;
    s.splits = key_ranges(ctas, sms * (s.block_rows <= 8 ? 3 : 2), keys, q4, sms);
    s.cluster = s.splits > 1 && s.splits <= kMaxCluster;
    return s;
}

// Scratch of a call: the parts of split rows (f32 and a log-sum-exp), for the chunk kernel two slots of 256 rows a CTA.
static size_t workspace_of(const Shape& s, size_t rows) {
    if (s.chunk) return (size_t)s.ctas * s.phases * (2 * 2 * kChunkRows * (kD + 1) * sizeof(float) + sizeof(ChunkSplit));
    return s.splits > 1 && !s.cluster ? s.splits * rows * (kD + 1) * sizeof(float) : 0;
}

static int launch_chunk(cudaStream_t st, const fv_paged_kv* kv, const AttnArgs& a, const Shape& s, int dev) {
    const bool q4 = kv->format == FV_PAGE_Q4;
    ChunkJob jb{};
    jb.pool = a.pool;
    jb.batch = a.batch;
    jb.mask = a.mask;
    jb.q = a.q;
    jb.q_tok = a.q_tok;
    jb.q_head = a.q_head;
    jb.out = a.out;
    const size_t slots = 2 * (size_t)s.ctas * s.phases * 2 * kChunkRows;  // rows of parts
    jb.part_o = a.part_o;
    jb.part_lse = jb.part_o + slots * kD;
    jb.split = reinterpret_cast<ChunkSplit*>(jb.part_lse + slots);
    jb.wait_status = a.batch.status - 1;
    jb.wait_cycles = FV_WAIT_CYCLES;
    jb.heads = a.heads;
    jb.group = a.group;
    jb.tile_tokens = s.tile_tokens;
    jb.by_group = a.by_group;
    jb.by_blocks = a.by_blocks;
    jb.by_heads = a.by_heads;
    const long long items = (long long)a.batch.seqs * a.pool.kv_heads * s.row_blocks;
    if (items > 0x3fffffffll) return FV_DECLINED;
    jb.items = (int)items;
    jb.phases = s.phases;
    jb.box_rows = kv->page_rows < kChunkTile ? kv->page_rows : kChunkTile;
    jb.sl2 = a.sl2;
    CUtensorMap mq{}, mk{}, mv{};
    if (!q4) {
        const uint64_t dq[4] = {128, (uint64_t)a.heads, (uint64_t)a.batch.tokens, 1};
        const uint64_t sq[3] = {(uint64_t)a.q_head * 2, (uint64_t)a.q_tok * 2, (uint64_t)a.q_tok * 2};
        const uint32_t bq[4] = {64, (uint32_t)a.group, (uint32_t)s.tile_tokens, 1};
        int rc = fvrt::encode_map4_box(&mq, a.q, dq, sq, bq);
        if (rc != FV_RAN) return rc;
        const uint64_t row = 256, head = row * kv->page_rows, page = head * kv->kv_heads;
        const uint64_t dk[4] = {128, (uint64_t)kv->page_rows, (uint64_t)kv->kv_heads, (uint64_t)kv->pages};
        const uint64_t sk[3] = {row, head, page};
        rc = fvrt::encode_map4_cached(&mk, kv->k, dk, sk, (uint32_t)jb.box_rows);
        if (rc != FV_RAN) return rc;
        rc = fvrt::encode_map4_cached(&mv, kv->v, dk, sk, (uint32_t)jb.box_rows);
        if (rc != FV_RAN) return rc;
    }
    {
        static bool attr_set[64][2] = {};
        static std::mutex attr_mu;
        std::lock_guard<std::mutex> lock(attr_mu);
        if (!attr_set[dev][q4]) {
            if (q4) FV_CUDA(cudaFuncSetAttribute(fv_paged_chunk_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kChunkSmem));
            else FV_CUDA(cudaFuncSetAttribute(fv_paged_chunk_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kChunkSmem));
            attr_set[dev][q4] = true;
        }
    }
    const unsigned grid = (unsigned)s.ctas;
    if (q4) fv_paged_chunk_kernel<true><<<grid, Roles<true>::kThreads, kChunkSmem, st>>>(mq, mk, mv, jb);
    else fv_paged_chunk_kernel<false><<<grid, Roles<false>::kThreads, kChunkSmem, st>>>(mq, mk, mv, jb);
    FV_CUDA(cudaGetLastError());
    if (grid > 1) {
        fv_paged_join_kernel<<<grid * s.phases * kJoinBlocks, kAttnThreads, 0, st>>>(jb);
        FV_CUDA(cudaGetLastError());
    }
    fvrt::ran_later(fvrt::kLogPagedChunk, "paged attention: fv_paged_chunk_kernel<%s> (sm_100a tcgen05, persistent, %d CTAs) %d sequences x %d heads / %d",
              q4 ? "4 bits" : "bf16", (int)grid, a.batch.seqs, a.heads, a.pool.kv_heads);
    return FV_RAN;
}

static int check_mask(const fv_paged_query& x, Mask* m) {
    if (x.mask_mode == FV_MASK_NONE) {
        *m = Mask{};
        return FV_RAN;
    }
    if (x.mask_mode != FV_MASK_BLOCK_CAUSAL) return fvrt::fail(FV_ERR_INVALID, "paged attention: unknown mask mode %d", x.mask_mode);
    if (x.block_tokens < 1 || x.window < 0 || x.sink < 0)
        return fvrt::fail(FV_ERR_INVALID, "paged attention: block-causal needs block_tokens >= 1, window, sink >= 0");
    *m = Mask{x.block_tokens, x.window, x.sink, Div::of(x.block_tokens)};
    return FV_RAN;
}

}  // namespace fvpg

extern "C" size_t fv_paged_attn_workspace_bytes(const fv_paged_kv* kv, const fv_paged_batch* b, const fv_paged_query* x) {
    using namespace fvpg;
    fvrt::clear_error();
    Mask m;
    int dev, sms;
    if (!kv || !b || !x || kv->kv_heads < 1 || x->heads < 1 || x->heads % kv->kv_heads || b->seqs < 1 || x->tokens < 1 || b->max_q < 1 ||
        check_mask(*x, &m) != FV_RAN || fvrt::require_sm100(&dev) != FV_RAN ||
        fvrt::sm_count(dev, &sms) != FV_RAN)
        return 0;
    return workspace_of(shape_of(kv, b, x->tokens, x->heads, m, sms), (size_t)x->tokens * x->heads);
}

extern "C" int fv_paged_attn_bf16(void* stream, const fv_paged_kv* kv, const fv_paged_batch* b, const fv_paged_query* x) {
    using namespace fvpg;
    fvrt::clear_error();
    if (!x) return fvrt::fail(FV_ERR_INVALID, "paged attention: null operand");
    const int tokens = x->tokens, heads = x->heads;
    const void* q = x->q;
    void *out = x->out, *workspace = x->workspace;
    const float scale = x->scale;
    AttnArgs a{};
    int rc = check_mask(*x, &a.mask);
    if (rc != FV_RAN) return rc;
    if (heads < 1 || (kv && kv->kv_heads > 0 && heads % kv->kv_heads))
        return fvrt::fail(FV_ERR_INVALID, "paged attention: %d heads over %d K/V heads", heads, kv ? kv->kv_heads : 0);
    if (!(scale > 0.f) || !isfinite(scale)) return fvrt::fail(FV_ERR_INVALID, "paged attention: scale must be positive and finite");
    int dev, sms;
    rc = check_paged("paged attention", kv, b, tokens, &a.pool, &a.batch, &dev);
    if (rc != FV_RAN) return rc;
    if (b->max_q == 0) return FV_DECLINED;
    if (!q || !out) return fvrt::fail(FV_ERR_INVALID, "paged attention: null operand");
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15)
        return fvrt::fail(FV_ERR_INVALID, "paged attention: operands must be 16-byte aligned");
    const long long q_tok = tokens == 1 ? kD : x->q_tok, q_head = heads == 1 ? kD : x->q_head;  // (that of an extent of one means nothing)
    if (((q_tok | q_head) & 7) || q_tok <= 0 || q_head <= 0)
        return fvrt::fail(FV_ERR_INVALID, "paged attention: strides must be positive multiples of 8 values");
    rc = fvrt::sm_count(dev, &sms);
    if (rc != FV_RAN) return rc;
    const size_t rows = (size_t)tokens * heads;
    if (rows > 0x7fffffffull) return FV_DECLINED;
    const Shape s = shape_of(kv, b, tokens, heads, a.mask, sms);
    const size_t need = workspace_of(s, rows);
    if (need > 0 && (!workspace || x->workspace_bytes < need))
        return fvrt::fail(FV_ERR_INVALID, "paged attention: workspace of %zu bytes, %zu needed", x->workspace_bytes, need);
    a.q = (const uint16_t*)q;
    a.q_tok = q_tok;
    a.q_head = q_head;
    a.out = (uint16_t*)out;
    a.part_o = (float*)workspace;
    a.part_lse = (float*)workspace + (size_t)s.splits * rows * kD;
    a.heads = heads;
    a.group = heads / kv->kv_heads;
    a.splits = s.splits;
    a.by_group = Div::of(a.group);
    a.by_splits = Div::of(s.splits);
    a.by_blocks = Div::of(s.row_blocks);
    a.by_heads = Div::of(kv->kv_heads);
    a.cluster = s.cluster;
    a.sl2 = scale * 1.4426950408889634f;
    a.wait_cycles = FV_WAIT_CYCLES;
    const long long grid = (long long)b->seqs * kv->kv_heads * s.row_blocks * s.splits;
    if (grid > 0x7fffffffll) return FV_DECLINED;
    cudaStream_t st = (cudaStream_t)stream;
    if (s.chunk) {
        return launch_chunk(st, kv, a, s, dev);
    }
    const bool q4 = kv->format == FV_PAGE_Q4;
    void (*fn)(AttnArgs);
    uint32_t smem;
    auto pick = [&](auto f, uint32_t bytes) {
        fn = f;
        smem = bytes;
    };
    if (q4 && s.block_rows == 4) pick(fv_paged_decode_kernel<true, 4>, DecodeSmem<true, 4>::kTotal);
    else if (q4 && s.block_rows == 8) pick(fv_paged_decode_kernel<true, 8>, DecodeSmem<true, 8>::kTotal);
    else if (q4) pick(fv_paged_decode_kernel<true, 16>, DecodeSmem<true, 16>::kTotal);
    else if (s.block_rows == 8) pick(fv_paged_decode_kernel<false, 8>, DecodeSmem<false, 8>::kTotal);
    else pick(fv_paged_decode_kernel<false, 16>, DecodeSmem<false, 16>::kTotal);
    if (q4) {  // (more shared memory than a launch gets unasked)
        static bool attr_set[64][17] = {};
        static std::mutex attr_mu;
        std::lock_guard<std::mutex> lock(attr_mu);
        if (!attr_set[dev][s.block_rows]) {
            FV_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            attr_set[dev][s.block_rows] = true;
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kAttnThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)s.splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = s.cluster ? 1 : 0;
    FV_CUDA(cudaLaunchKernelEx(&cfg, fn, a));
    if (s.splits > 1 && !s.cluster) {
        fv_paged_merge_kernel<<<(unsigned)((rows + kWarps - 1) / kWarps), kAttnThreads, 0, st>>>(a);
        FV_CUDA(cudaGetLastError());
    }
    fvrt::ran_later(fvrt::kLogPagedAttn, "paged attention: fv_paged_decode_kernel<%s, %d rows> %d sequences x %d heads / %d, %d key ranges",
              q4 ? "4 bits" : "bf16", s.block_rows, b->seqs, heads, kv->kv_heads, s.splits);
    return FV_RAN;
}
