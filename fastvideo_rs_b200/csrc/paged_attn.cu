// Attention of a ragged batch's queries over a paged K/V cache: block-causal with a sliding window and sinks, shared
// K/V heads, pages of bf16 or of 4 bits.  This file: the kernel for few query rows per K/V head (decode steps, short
// chunks), the merge of key ranges, and the C entry.
//
// Row r of a (sequence, kv head) is token r / g, head r % g of the heads that share that K/V head (g = heads /
// kv_heads): one pass over the keys serves all of them.
#include "fv_runtime.h"
#include "paged.cuh"
#include "paged_fwd.cuh"
#include "paged_host.h"
#include <math.h>
#include <mutex>

namespace fvpg {

constexpr int kWarps = 4;
constexpr int kAttnThreads = 32 * kWarps;
constexpr int kTile = 16;  // keys a warp takes at a time (one page holds them: page_rows is a multiple of 16)

struct AttnArgs {
    Pool pool;
    Batch batch;
    Mask mask;
    const uint16_t* q;
    long long q_tok, q_head;  // strides in values
    uint16_t* out;            // [tokens, heads, 128]
    float* part_o;            // [splits, tokens * heads, 128] normalised, when splits > 1
    float* part_lse;          // [splits, tokens * heads], base 2
    int heads, group, splits, row_blocks;
    float sl2;
};


using fvattn::neg_inf;

// The key tiles a block of rows visits: those of [0, sink), then those of [lo, hi), each tile once.
struct Tiles {
    int sinks, first, count;
    FV_DEV explicit Tiles(const Span& s) {
        sinks = (s.sink + kTile - 1) / kTile;
        first = max(s.lo / kTile, sinks);
        count = sinks + max(0, (s.hi + kTile - 1) / kTile - first);
    }
    FV_DEV int key(int u) const { return (u < sinks ? u : first + (u - sinks)) * kTile; }
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
// D (16 x 8 f32) += A (16 x 16 bf16) . B (16 x 8 bf16).  Lane 4 g + t holds of A rows g (a0, a2) and g + 8 (a1, a3), of B
// column g, of D rows g (c0, c1) and g + 8 (c2, c3), columns 2 t and 2 t + 1.
FV_DEV void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transpose of an 8 x 8 tile of bf16 held one row per quad of lanes.
FV_DEV uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
FV_DEV uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
// Codes n of nibbles i and i + 4 of x as the bf16 pair (128 + n): 128 has a unit in its last place of one, so or-ing the
// code into the mantissa is exact.
FV_DEV uint32_t codes128(uint32_t x, int i) { return ((x >> (4 * i)) & 0x000f000fu) | 0x43004300u; }
FV_DEV uint32_t sub136(uint32_t x) {  // (128 + n) - 136 = n - 8, exact
    uint32_t r;
    asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0xc308c308u));
    return r;
}
FV_DEV float lo_f(uint32_t x) { return __uint_as_float(x << 16); }
FV_DEV float hi_f(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// One tile of 16 keys in registers, as lane 4 g + t holds it.
//   bf16  k0 / k1: keys g and g + 8, 16-byte pieces 4 n + t of their rows; v: keys 2t, 2t+1, 2t+8, 2t+9, pieces g and
//         g + 8 of their rows.
//   4 bit k0[0] / k1[0]: values 32 t .. 32 t + 31 of keys g and g + 8; v4: values 16 g .. 16 g + 15 of the four keys;
//         ks / vs: (step, zero) of keys g and g + 8.
template <bool Q4>
struct Keys;
template <>
struct Keys<false> {
    uint4 k0[4], k1[4];
    FV_DEV void load(const Pool& p, int page, int head, int key, int g, int t) {
        if (page < 0) {
#pragma unroll
            for (int n = 0; n < 4; n++) k0[n] = k1[n] = make_uint4(0, 0, 0, 0);
            return;
        }
        const uint8_t* r = p.k + pool_row(p, page, head, key) * 256 + (size_t)g * 256 + 16 * t;
#pragma unroll
        for (int n = 0; n < 4; n++) {
            k0[n] = ld_stream(r + 64 * n);
            k1[n] = ld_stream(r + 8 * 256 + 64 * n);
        }
    }
};
template <>
struct Keys<true> {
    uint4 k0[1], k1[1];
    uint32_t s0, s1;
    FV_DEV void load(const Pool& p, int page, int head, int key, int g, int t) {
        if (page < 0) {
            k0[0] = k1[0] = make_uint4(0, 0, 0, 0);
            s0 = s1 = 0;
            return;
        }
        const size_t row = pool_row(p, page, head, key) + g;
        k0[0] = ld_stream(p.k + row * kQ4Bytes + 16 * t);
        k1[0] = ld_stream(p.k + (row + 8) * kQ4Bytes + 16 * t);
        s0 = ld_stream1(p.k_scale + row);
        s1 = ld_stream1(p.k_scale + row + 8);
    }
};
template <bool Q4>
struct Values;
template <>
struct Values<false> {
    uint4 a[4], b[4];  // pieces g and g + 8 of keys 2t, 2t+1, 2t+8, 2t+9
    FV_DEV void load(const Pool& p, int page, int head, int key, int g, int t) {
        if (page < 0) {
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = b[i] = make_uint4(0, 0, 0, 0);
            return;
        }
        const uint8_t* r = p.v + pool_row(p, page, head, key) * 256 + (size_t)(2 * t) * 256 + 16 * g;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int o = ((i & 1) + 8 * (i >> 1)) * 256;
            a[i] = ld_stream(r + o);
            b[i] = ld_stream(r + o + 128);
        }
    }
    FV_DEV void clear(int i) { a[i] = b[i] = make_uint4(0, 0, 0, 0); }
};
template <>
struct Values<true> {
    uint2 a[4];
    uint32_t s0, s1;
    FV_DEV void load(const Pool& p, int page, int head, int key, int g, int t) {
        if (page < 0) {
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = make_uint2(0, 0);
            s0 = s1 = 0;
            return;
        }
        const size_t row = pool_row(p, page, head, key);
#pragma unroll
        for (int i = 0; i < 4; i++) a[i] = ld_stream2(p.v + (row + 2 * t + (i & 1) + 8 * (i >> 1)) * kQ4Bytes + 8 * g);
        s0 = ld_stream1(p.v_scale + row + g);
        s1 = ld_stream1(p.v_scale + row + g + 8);
    }
};

FV_DEV uint32_t word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

// NT groups of 8 query rows.  The transposed products S^T = K . Q^T and O^T = V^T . P^T keep keys and head dim on the
// 16-wide side of the matrix instruction and the (few) query rows on the 8-wide one; the sums of either product may run
// in any order of d or key, so every lane's operands are whole 16-byte pieces as they lie in memory and no shared
// memory is needed on the way.
template <bool Q4, int NT>
__global__ void __launch_bounds__(kAttnThreads) fv_paged_decode_kernel(const AttnArgs a) {
    constexpr int kRows = 8 * NT;
    __shared__ float sh_o[kWarps][kRows][kD + 4];
    __shared__ float sh_m[kWarps][kRows], sh_l[kWarps][kRows];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    int b = blockIdx.x;
    const int split = b % a.splits;
    b /= a.splits;
    const int rb = b % a.row_blocks;
    b /= a.row_blocks;
    const int head = b % a.pool.kv_heads, s = b / a.pool.kv_heads;
    const Seq seq = seq_of(a.batch, s);
    const int row0 = rb * kRows, rows = min(kRows, seq.nq * a.group - row0);
    if (rows <= 0) return;
    const int pos0 = seq.len - seq.nq;  // position of the sequence's first token of this call
    const int first = pos0 + row0 / a.group, last = pos0 + (row0 + rows - 1) / a.group;
    const Span span = span_of(a.mask, first, last, seq.len);
    const Span lowest = span_of(a.mask, first, first, seq.len), highest = span_of(a.mask, last, last, seq.len);
    const Tiles tiles(span);
    // (every row sees the whole tile: inside the first row's end and the last row's start, or inside the sinks)
    const int whole_lo = highest.lo, whole_hi = lowest.hi;
    const int whole_sink = min(lowest.lo == 0 ? lowest.hi : lowest.sink, highest.lo == 0 ? highest.hi : highest.sink);
    const int u0 = (int)((long long)tiles.count * split / a.splits), u1 = (int)((long long)tiles.count * (split + 1) / a.splits);

    // Q^T: column g of each group of 8 rows, in the order of d that the keys' lanes hold.
    uint32_t qf[NT][16];
    float qsum[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = row0 + 8 * n + g;
        uint4 u[4];
        if (8 * n + g < rows) {
            const uint16_t* p = a.q + (size_t)(seq.q0 + r / a.group) * a.q_tok + (size_t)(head * a.group + r % a.group) * a.q_head;
#pragma unroll
            for (int i = 0; i < 4; i++) u[i] = *reinterpret_cast<const uint4*>(p + (Q4 ? 32 * t + 8 * i : 32 * i + 8 * t));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) u[i] = make_uint4(0, 0, 0, 0);
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (Q4) {  // pairs (d, d + 4) of eight values: the nibbles that one shift and mask give
                qf[n][4 * i + 0] = prmt(u[i].x, u[i].z, 0x5410);
                qf[n][4 * i + 1] = prmt(u[i].x, u[i].z, 0x7632);
                qf[n][4 * i + 2] = prmt(u[i].y, u[i].w, 0x5410);
                qf[n][4 * i + 3] = prmt(u[i].y, u[i].w, 0x7632);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) qf[n][4 * i + j] = word(u[i], j);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) sum += lo_f(word(u[i], j)) + hi_f(word(u[i], j));
        }
        if (Q4) {
            sum += __shfl_xor_sync(kFullWarp, sum, 1);
            sum += __shfl_xor_sync(kFullWarp, sum, 2);
            qsum[n][0] = __shfl_sync(kFullWarp, sum, 8 * t);      // of row 2 t, which the lanes 4 (2 t) .. hold
            qsum[n][1] = __shfl_sync(kFullWarp, sum, 8 * t + 4);  // of row 2 t + 1
        }
    }

    float o[NT][8][4];  // O^T: d by lane g and tile, rows 2 t and 2 t + 1
    float m[NT][2], l[NT][2], z[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int i = 0; i < 8; i++) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
        m[n][0] = m[n][1] = neg_inf();
        l[n][0] = l[n][1] = z[n][0] = z[n][1] = 0.f;
    }

    auto lookup = [&](int u) { return u < u1 ? page_of(a.pool, a.batch, s, tiles.key(u)) : -1; };
    Keys<Q4> kt;
    Values<Q4> vt;
    int u = u0 + warp;
    int page = lookup(u), page_next = lookup(u + kWarps);
    if (u < u1) {
        kt.load(a.pool, page, head, tiles.key(u), g, t);
        vt.load(a.pool, page, head, tiles.key(u), g, t);
    }
    while (u < u1) {
        const int key0 = tiles.key(u), un = u + kWarps;
        const int page_after = lookup(un + kWarps);
        float c[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    if (Q4) {
                        const uint32_t w0 = word(kt.k0[0], i), w1 = word(kt.k1[0], i);
                        mma(c[n], codes128(w0, 2 * j), codes128(w1, 2 * j), codes128(w0, 2 * j + 1), codes128(w1, 2 * j + 1),
                            qf[n][4 * i + 2 * j], qf[n][4 * i + 2 * j + 1]);
                    } else {
                        mma(c[n], word(kt.k0[Q4 ? 0 : i], 2 * j), word(kt.k1[Q4 ? 0 : i], 2 * j), word(kt.k0[Q4 ? 0 : i], 2 * j + 1),
                            word(kt.k1[Q4 ? 0 : i], 2 * j + 1), qf[n][4 * i + 2 * j], qf[n][4 * i + 2 * j + 1]);
                    }
                }
            }
        }
        if constexpr (Q4) {
            // q . (zero + step code) = step (q . (128 + n)) + (zero - 136 step) sum(q)
            const float s0 = lo_f(kt.s0), s1 = lo_f(kt.s1);
            const float z0 = fmaf(-136.f, s0, hi_f(kt.s0)), z1 = fmaf(-136.f, s1, hi_f(kt.s1));
#pragma unroll
            for (int n = 0; n < NT; n++) {
                c[n][0] = fmaf(c[n][0], s0, z0 * qsum[n][0]);
                c[n][1] = fmaf(c[n][1], s0, z0 * qsum[n][1]);
                c[n][2] = fmaf(c[n][2], s1, z1 * qsum[n][0]);
                c[n][3] = fmaf(c[n][3], s1, z1 * qsum[n][1]);
            }
        }
        if (un < u1) kt.load(a.pool, page_next, head, tiles.key(un), g, t);

        // c0, c1: key g, rows 2 t and 2 t + 1; c2, c3: key g + 8.
        const bool whole = page >= 0 && ((key0 >= whole_lo && key0 + kTile <= whole_hi) || key0 + kTile <= whole_sink);
        if (!whole) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int r = row0 + 8 * n + 2 * t + e, p = pos0 + r / a.group;
                    const Span sp = span_of(a.mask, p, p, seq.len);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int j = key0 + g + 8 * h;
                        if (page < 0 || !((j >= sp.lo && j < sp.hi) || j < sp.sink)) c[n][2 * h + e] = neg_inf();
                    }
                }
            }
            // Values that no row of this block may see count as zero whatever they hold (0 times NaN is NaN).
            auto seen = [&](int j) { return (j >= span.lo && j < span.hi) || j < span.sink; };
            if constexpr (Q4) {
                if (!seen(key0 + g)) vt.s0 = 0u;
                if (!seen(key0 + g + 8)) vt.s1 = 0u;
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (!seen(key0 + 2 * t + (i & 1) + 8 * (i >> 1))) vt.clear(i);
            }
        }
        // Streaming softmax: P against the reference the row has; the exact maximum is taken only where there is none
        // yet, or where a P comes out above 2^40 (bf16 and the f32 sums hold that; the reference cancels in O / l).
        float p[NT][4];
        bool trip = false;
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                p[n][e] = fvp::ex2(fmaf(c[n][e], a.sl2, -m[n][e & 1]));
                trip |= !(p[n][e] <= 1099511627776.f);
            }
        }
        if (__any_sync(kFullWarp, trip)) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float mx = fmaxf(c[n][e], c[n][2 + e]) * a.sl2;
                    mx = fmaxf(mx, __shfl_xor_sync(kFullWarp, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(kFullWarp, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(kFullWarp, mx, 16));
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
                    p[n][e] = fvp::ex2(fmaf(c[n][e], a.sl2, -ref));
                    p[n][2 + e] = fvp::ex2(fmaf(c[n][2 + e], a.sl2, -ref));
                }
            }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            l[n][0] += p[n][0] + p[n][2];
            l[n][1] += p[n][1] + p[n][3];
            if constexpr (Q4) {  // sum P (zero + step (n - 8)): the step goes into P, the zeros are summed apart
                const float s0 = lo_f(vt.s0), s1 = lo_f(vt.s1), z0 = hi_f(vt.s0), z1 = hi_f(vt.s1);
                z[n][0] += p[n][0] * z0 + p[n][2] * z1;
                z[n][1] += p[n][1] * z0 + p[n][3] * z1;
                pb[n][0] = transpose8(fvp::pack_bf16x2(p[n][0] * s0, p[n][1] * s0));
                pb[n][1] = transpose8(fvp::pack_bf16x2(p[n][2] * s1, p[n][3] * s1));
            } else {
                pb[n][0] = transpose8(fvp::pack_bf16x2(p[n][0], p[n][1]));
                pb[n][1] = transpose8(fvp::pack_bf16x2(p[n][2], p[n][3]));
            }
        }
        // O^T += V^T . P^T: the pair of one d and two neighbouring keys comes out of two keys' words.
        if constexpr (Q4) {
#pragma unroll
            for (int h = 0; h < 2; h++) {  // the low and the high half of each word: its nibbles 4 h .. 4 h + 3
                const uint32_t sel = h ? 0x7632 : 0x5410;
                const uint32_t x0 = prmt(vt.a[0].x, vt.a[1].x, sel), x1 = prmt(vt.a[0].y, vt.a[1].y, sel);
                const uint32_t x2 = prmt(vt.a[2].x, vt.a[3].x, sel), x3 = prmt(vt.a[2].y, vt.a[3].y, sel);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t a0 = sub136(codes128(x0, i)), a1 = sub136(codes128(x1, i));
                    const uint32_t a2 = sub136(codes128(x2, i)), a3 = sub136(codes128(x3, i));
#pragma unroll
                    for (int n = 0; n < NT; n++) mma(o[n][4 * h + i], a0, a1, a2, a3, pb[n][0], pb[n][1]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t sel = (i & 1) ? 0x7632 : 0x5410;
                const uint32_t a0 = prmt(word(vt.a[0], i / 2), word(vt.a[1], i / 2), sel);
                const uint32_t a1 = prmt(word(vt.b[0], i / 2), word(vt.b[1], i / 2), sel);
                const uint32_t a2 = prmt(word(vt.a[2], i / 2), word(vt.a[3], i / 2), sel);
                const uint32_t a3 = prmt(word(vt.b[2], i / 2), word(vt.b[3], i / 2), sel);
#pragma unroll
                for (int n = 0; n < NT; n++) mma(o[n][i], a0, a1, a2, a3, pb[n][0], pb[n][1]);
            }
        }
        if (un < u1) vt.load(a.pool, page_next, head, tiles.key(un), g, t);
        u = un;
        page = page_next;
        page_next = page_after;
    }

    // The four warps' results side by side, then joined.
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
                l[n][e] += __shfl_xor_sync(kFullWarp, l[n][e], d);
                z[n][e] += __shfl_xor_sync(kFullWarp, z[n][e], d);
            }
            const int r = 8 * n + 2 * t + e;
            if (g == 0) {
                sh_m[warp][r] = m[n][e];
                sh_l[warp][r] = l[n][e];
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                sh_o[warp][r][Q4 ? 16 * g + i : 8 * g + i] = o[n][i][e] + z[n][e];
                sh_o[warp][r][Q4 ? 16 * g + 8 + i : 64 + 8 * g + i] = o[n][i][2 + e] + z[n][e];
            }
        }
    }
    __syncthreads();
    const int d = threadIdx.x;  // kAttnThreads == kD
#pragma unroll
    for (int r = 0; r < kRows; r++) {
        if (r >= rows) break;
        float top = sh_m[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; w++) top = fmaxf(top, sh_m[w][r]);
        float sum = 0.f, acc = 0.f;
        if (top != neg_inf()) {
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float f = fvp::ex2(sh_m[w][r] - top);
                sum += f * sh_l[w][r];
                if (f != 0.f) acc += f * sh_o[w][r][d];
            }
            acc /= sum;
        }
        const int rr = row0 + r;
        const size_t oi = (size_t)(seq.q0 + rr / a.group) * a.heads + head * a.group + rr % a.group;
        if (a.splits == 1) {
            a.out[oi * kD + d] = (uint16_t)(fvp::pack_bf16x2(acc, 0.f));
        } else {
            const size_t pi = (size_t)split * a.batch.tokens * a.heads + oi;
            a.part_o[pi * kD + d] = acc;
            if (d == 0) a.part_lse[pi] = top == neg_inf() ? neg_inf() : top + log2f(sum);
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
    float top = neg_inf();
    for (int i = 0; i < a.splits; i++) top = fmaxf(top, a.part_lse[(size_t)i * rows + row]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    if (top != neg_inf()) {
        for (int i = 0; i < a.splits; i++) {
            const float w = fvp::ex2(a.part_lse[(size_t)i * rows + row] - top);
            if (w == 0.f) continue;
            const float4 x = *reinterpret_cast<const float4*>(a.part_o + ((size_t)i * rows + row) * kD + 4 * lane);
            sum += w;
            acc.x = fmaf(w, x.x, acc.x);
            acc.y = fmaf(w, x.y, acc.y);
            acc.z = fmaf(w, x.z, acc.z);
            acc.w = fmaf(w, x.w, acc.w);
        }
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

// ---- host --------------------------------------------------------------------------------------------------------------

struct Shape {
    bool chunk;  // the tensor-core kernel for long chunks
    int splits, row_blocks, nt, tile_tokens;
};
// How a call is cut.  Few rows per kv head: blocks of 8 or 16 rows, and the keys in `splits` ranges so that all SMs have
// work.  From kChunkFrom rows on: items of 2 x 128 rows, the keys cut where that evens out the waves.
constexpr int kChunkFrom = 33;
static Shape shape_of(const fv_paged_kv* kv, const fv_paged_batch* b, int heads, const Mask& m, int sms) {
    Shape s;
    const int group = heads / kv->kv_heads;
    const long long rows = (long long)b->max_q * group;
    s.chunk = rows >= kChunkFrom && group <= kChunkRows;
    s.tile_tokens = s.chunk ? kChunkRows / group : 0;
    if (s.chunk) {
        long long seen = b->max_kv;
        if (m.block > 0 && m.window > 0) {
            const long long some = ((long long)m.window + m.sink + 1) * m.block + 2 * s.tile_tokens;
            seen = some < seen ? some : seen;
        }
        const int tiles = (int)((seen + kChunkTile - 1) / kChunkTile);
        s.nt = 0;
        s.row_blocks = (b->max_q + 2 * s.tile_tokens - 1) / (2 * s.tile_tokens);
        const long long items = (long long)b->seqs * kv->kv_heads * s.row_blocks;
        // Time of a cut, in key tiles of a CTA: whole waves of equal items, each with a fixed cost of about four tiles,
        // and the merge's traffic (a part is 516 bytes a row; a key tile takes about 1.5 us, 7.5 MB at 5 TB/s).
        double best = 0;
        s.splits = 1;
        for (int n = 1; n <= 16 && (n == 1 || tiles >= 4 * n); n++) {
            const long long waves = (items * n + sms - 1) / sms;
            const double cost = (double)waves * ((tiles + n - 1) / n + 4) + (n > 1 ? 2.0 + (double)b->max_q * b->seqs * heads * n * 1032.0 / 7.5e6 : 0.0);
            if (n == 1 || cost < 0.95 * best) {
                best = cost;
                s.splits = n;
            }
        }
        return s;
    }
    s.nt = rows > 8 ? 2 : 1;
    s.row_blocks = (int)((rows + 8 * s.nt - 1) / (8 * s.nt));
    long long keys = b->max_kv;
    if (m.block > 0 && m.window > 0) {  // rows of one block see window blocks and the sinks, max_q rows a little more
        const long long most = ((long long)m.window + m.sink + 1) * m.block + b->max_q;
        keys = most < keys ? most : keys;
    }
    const long long ctas = (long long)b->seqs * kv->kv_heads * s.row_blocks;
    const long long want = (6ll * sms + ctas - 1) / ctas;      // CTAs of about two waves of three per SM
    const long long most = (keys + 4 * kTile * kWarps - 1) / (4 * kTile * kWarps);  // at least four tiles per warp
    long long n = want < most ? want : most;
    s.splits = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
    return s;
}

static int launch_chunk(cudaStream_t st, const fv_paged_kv* kv, const AttnArgs& a, const Shape& s, int dev, int sms) {
    const bool q4 = kv->format == FV_PAGE_Q4;
    ChunkJob jb{};
    jb.pool = a.pool;
    jb.batch = a.batch;
    jb.mask = a.mask;
    jb.q = a.q;
    jb.q_tok = a.q_tok;
    jb.q_head = a.q_head;
    jb.out = a.out;
    jb.part_o = a.part_o;
    jb.part_lse = a.part_lse;
    jb.wait_status = a.batch.status - 1;
    jb.wait_cycles = FV_WAIT_CYCLES;
    jb.heads = a.heads;
    jb.group = a.group;
    jb.tile_tokens = s.tile_tokens;
    jb.splits = s.splits;
    jb.planes = a.batch.seqs * a.pool.kv_heads;
    jb.q_blocks = s.row_blocks;
    const long long items = (long long)jb.planes * s.row_blocks * s.splits;
    if (items > 0x3fffffffll) return FV_DECLINED;
    jb.items = (int)items;
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
    const unsigned grid = (unsigned)(items < sms ? items : sms);
    if (q4) fv_paged_chunk_kernel<true><<<grid, Roles<true>::kThreads, kChunkSmem, st>>>(mq, mk, mv, jb);
    else fv_paged_chunk_kernel<false><<<grid, Roles<false>::kThreads, kChunkSmem, st>>>(mq, mk, mv, jb);
    FV_CUDA(cudaGetLastError());
    fvrt::ran(fvrt::kLogPagedChunk, "paged attention: fv_paged_chunk_kernel<%s> (sm_100a tcgen05, persistent, %u CTAs) %d sequences x %d heads / %d, %d key ranges",
              q4 ? "4 bits" : "bf16", grid, a.batch.seqs, a.heads, a.pool.kv_heads, s.splits);
    return FV_RAN;
}

static int check_mask(int mask_mode, int block_tokens, int window, int sink, Mask* m) {
    if (mask_mode == FV_MASK_NONE) {
        *m = Mask{0, 0, 0};
        return FV_RAN;
    }
    if (mask_mode != FV_MASK_BLOCK_CAUSAL) return fvrt::fail(FV_ERR_INVALID, "paged attention: unknown mask mode %d", mask_mode);
    if (block_tokens < 1 || window < 0 || sink < 0)
        return fvrt::fail(FV_ERR_INVALID, "paged attention: block-causal needs block_tokens >= 1, window, sink >= 0");
    *m = Mask{block_tokens, window, sink};
    return FV_RAN;
}

}  // namespace fvpg

extern "C" size_t fv_paged_attn_workspace_bytes(const fv_paged_kv* kv, const fv_paged_batch* b, int tokens, int heads, int mask_mode,
                                                int block_tokens, int window, int sink) {
    using namespace fvpg;
    fvrt::clear_error();
    Mask m;
    int dev, sms;
    if (!kv || !b || kv->kv_heads < 1 || heads < 1 || heads % kv->kv_heads || b->seqs < 1 || tokens < 1 || b->max_q < 1 ||
        check_mask(mask_mode, block_tokens, window, sink, &m) != FV_RAN || fvrt::require_sm100(&dev) != FV_RAN ||
        fvrt::sm_count(dev, &sms) != FV_RAN)
        return 0;
    const Shape s = shape_of(kv, b, heads, m, sms);
    return s.splits > 1 ? (size_t)s.splits * tokens * heads * (kD + 1) * sizeof(float) : 0;
}

extern "C" int fv_paged_attn_bf16(void* stream, const fv_paged_kv* kv, const fv_paged_batch* b, int tokens, const void* q, long long q_tok,
                                  long long q_head, int heads, int mask_mode, int block_tokens, int window, int sink, float scale,
                                  void* out, void* workspace, size_t workspace_bytes) {
    using namespace fvpg;
    fvrt::clear_error();
    AttnArgs a{};
    int rc = check_mask(mask_mode, block_tokens, window, sink, &a.mask);
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
    if ((q_tok | q_head) & 7) return fvrt::fail(FV_ERR_INVALID, "paged attention: strides must be multiples of 8 values");
    rc = fvrt::sm_count(dev, &sms);
    if (rc != FV_RAN) return rc;
    const Shape s = shape_of(kv, b, heads, a.mask, sms);
    const size_t rows = (size_t)tokens * heads;
    if (s.splits > 1 && (!workspace || workspace_bytes < s.splits * rows * (kD + 1) * sizeof(float)))
        return fvrt::fail(FV_ERR_INVALID, "paged attention: workspace of %zu bytes, %zu needed", workspace_bytes,
                          s.splits * rows * (kD + 1) * sizeof(float));
    a.q = (const uint16_t*)q;
    a.q_tok = q_tok;
    a.q_head = q_head;
    a.out = (uint16_t*)out;
    a.part_o = (float*)workspace;
    a.part_lse = (float*)workspace + (size_t)s.splits * rows * kD;
    a.heads = heads;
    a.group = heads / kv->kv_heads;
    a.splits = s.splits;
    a.row_blocks = s.row_blocks;
    a.sl2 = scale * 1.4426950408889634f;
    const long long grid = (long long)b->seqs * kv->kv_heads * s.row_blocks * s.splits;
    if (grid > 0x7fffffffll || (long long)rows > 0x7fffffffll) return FV_DECLINED;
    cudaStream_t st = (cudaStream_t)stream;
    if (s.chunk) {
        rc = launch_chunk(st, kv, a, s, dev, sms);
        if (rc != FV_RAN) return rc;
        if (s.splits > 1) {
            fv_paged_merge_kernel<<<(unsigned)((rows + kWarps - 1) / kWarps), kAttnThreads, 0, st>>>(a);
            FV_CUDA(cudaGetLastError());
        }
        return FV_RAN;
    }
    const bool q4 = kv->format == FV_PAGE_Q4;
    if (q4 && s.nt == 1) fv_paged_decode_kernel<true, 1><<<(unsigned)grid, kAttnThreads, 0, st>>>(a);
    else if (q4) fv_paged_decode_kernel<true, 2><<<(unsigned)grid, kAttnThreads, 0, st>>>(a);
    else if (s.nt == 1) fv_paged_decode_kernel<false, 1><<<(unsigned)grid, kAttnThreads, 0, st>>>(a);
    else fv_paged_decode_kernel<false, 2><<<(unsigned)grid, kAttnThreads, 0, st>>>(a);
    FV_CUDA(cudaGetLastError());
    if (s.splits > 1) {
        fv_paged_merge_kernel<<<(unsigned)((rows + kWarps - 1) / kWarps), kAttnThreads, 0, st>>>(a);
        FV_CUDA(cudaGetLastError());
    }
    fvrt::ran(fvrt::kLogPagedAttn, "paged attention: fv_paged_decode_kernel<%s, %d rows> %d sequences x %d heads / %d, %d key ranges",
              q4 ? "4 bits" : "bf16", 8 * s.nt, b->seqs, heads, kv->kv_heads, s.splits);
    return FV_RAN;
}
