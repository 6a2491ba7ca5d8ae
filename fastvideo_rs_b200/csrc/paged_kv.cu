// Writing to and reading from a paged K/V cache (no counterpart in the reference: its causal cache is one contiguous
// buffer per sequence that is copied down past the sink for every block, crates/fastvideo-cudarc/src/wan/causal.rs:
// 541-628; over pages the rows in between are given back instead).
//
// Append: every token's K (and q) is rotated with its position's table row, V is taken as it is, and both land in the
// token's row of its sequence's page, in bf16 or in 4 bits; q goes to a packed tensor.  Rotation arithmetic is that of the
// BHSD rope kernel: f32, products and sums rounded separately, one rounding to bf16.  4 bits, per row of 128 values x:
//     step = bf16((max x - min x) / 15), zero = bf16(min x + 8 step), code = clamp(rint((x - zero) / step), -8, 7),
// stored as code + 8 (even value in the low half of a byte): a row stands for zero + step * code.  Where zero's rounding moved it by
// more than a quarter of a step (an offset of some 64 steps and more), step is the smallest bf16 whose codes still span the row:
//     step = max((max x - zero) / 7, (zero - min x) / 8), rounded up.
// So no value is more than half a step off: at the ends the codes fall short by a quarter of a step and 15 times step's rounding,
// 0.31 of it, or by nothing.  K is quantised from the f32 rotation, not from its bf16 rounding.  One scale for the whole row because its factor then leaves the
// attention's products (q . k = step (q . code) + zero sum(q)), so that these run on exact codes.
//
// HBM-bound: 8 lanes hold one row of one head (16 values a lane), a warp the same head of 4 neighbouring tokens, a CTA
// of 16: their rows lie side by side in a page, each lane keeps its token's cosines and sines in registers over all heads,
// and q's, K's and V's heads are loops of their own without a branch inside, four rows in flight per lane.  4 680 tokens x 3 x 40
// heads to bf16 pages: 50-52 us = 5.6-5.8 TB/s, 0.86 of the measured copy bandwidth (a token a CTA: 87).  To 4 bits: 5 016
// tokens x (40 + 2 x 8) heads 31 us, of which the bytes are 16: some 250 instructions a lane and row in 1.41 waves of CTAs (six run at a time
// on an SM), which leaves the issue slots 44 % busy.
#include "fv_runtime.h"
#include "paged.cuh"
#include "paged_host.h"

namespace fvpg {

constexpr int kThreads = 128;
constexpr int kTokens = kThreads / 8;  // of a CTA

struct AppendArgs {
    Pool pool;
    Batch batch;
    const uint16_t *q, *k, *v;
    uint16_t* q_out;
    long long q_tok, q_head, k_tok, k_head, v_tok, v_head;  // strides in values
    const float *cosv, *sinv;
    const int* positions;
    int table_rows, q_heads, parts;
};

FV_DEV void widen8(const uint4 u, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
FV_DEV uint4 narrow8(const float* x) {
    using fvp::pack_bf16x2;
    return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}
FV_DEV float bf16_of(float x) {
    return __uint_as_float(fvp::pack_bf16x2(0.f, x) & 0xffff0000u);
}
FV_DEV float min_nan(float a, float b, float c) {
    float r;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
FV_DEV float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
FV_DEV float fma_sat(float a, float b, float c) {  // clamped to 0 .. 1
    float r;
    asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// seq_of_token for the warp's four tokens (one per 8 lanes) at once.
FV_DEV int seq_of_slot(const int* cu, int seqs, int t, int lane) {
    int s = 0;
    for (int base = 0; base < seqs; base += 32) {
        const int end = base + lane < seqs ? __ldg(cu + base + lane + 1) : 0x7fffffff;
        bool more = false;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int n = __popc(__ballot_sync(kFullWarp, end <= __shfl_sync(kFullWarp, t, 8 * k)));
            if ((lane >> 3) == k) s += n;
            more |= n == 32;
        }
        if (!more) break;
    }
    return s;
}

// x[0 .. 7] are values 8 c .. 8 c + 7 of a row, x[8 .. 15] are 64 values further on; cs / sn the factors of its 8 pairs.
template <bool HALF>
FV_DEV void rotate16(float (&x)[16], const float (&cs)[8], const float (&sn)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int a = HALF ? i : 2 * i, b = HALF ? i + 8 : 2 * i + 1;
        const float xa = x[a], xb = x[b];
        x[a] = __fsub_rn(__fmul_rn(xa, cs[i]), __fmul_rn(xb, sn[i]));
        x[b] = __fadd_rn(__fmul_rn(xa, sn[i]), __fmul_rn(xb, cs[i]));
    }
}
// Four codes exactly as the rounded quotient gives them, where some lie near the middle h between two codes.  Without dividing:
// d = y - step h is exact, and the quotient rounds to h itself (whose nearest integer is the even one) while |d| is at most
// step times half a unit in h's last place, a quarter unit below a power of two.  Out of line.
static __device__ __noinline__ uint32_t settle4(float a, float b, float c4, float d4, float zero, float step, float inv) {
    const float x[4] = {a, b, c4, d4};
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float y = __fsub_rn(x[i], zero);
        float c;
        if (inv <= 3e38f) {
            c = fminf(fmaxf(__fmul_rn(y, inv), -8.f), 7.f);
            float r = rintf(c);
            const float e = __fsub_rn(c, r);
            if (fabsf(e) > 0.4999f) {
                const float h = r + copysignf(0.5f, e), mag = fabsf(h);
                const float d = copysignf(1.f, h) * __fmaf_rn(-step, h, y);  // > 0: farther from zero than h
                const float unit = __uint_as_float(__float_as_uint(mag) & 0x7f800000u) * 0x1p-24f * step;
                if (d > unit || d < (mag == 0.5f ? -0.5f * unit : -unit)) r = h + copysignf(0.5f, d * h);
                else r = rintf(h);
            }
            c = r;
        } else {  // (a step so small that its reciprocal overflows)
            c = rintf(__fdiv_rn(y, step));
        }
        c = fminf(fmaxf(c, -8.f), 7.f);
        w |= ((uint32_t)((int)c + 8) & 15u) << (4 * i);
    }
    return w;
}
// The same row in 4 bits: codes of this lane's 16 values as two words (8 values each), (step, zero) as one.  Collective
// over the warp.  (A row of one bf16 value has step 0 and codes 0.  A row with a value that is not finite has a step that is
// not: its codes say nothing, the row stands for NaN.)
FV_DEV void quantize16(const float (&x)[16], uint32_t& lo, uint32_t& hi, uint32_t& scale) {
    float mn = min_nan(x[0], x[1], x[2]), mx = max_nan(x[0], x[1], x[2]);
#pragma unroll
    for (int i = 3; i < 15; i += 2) {
        mn = min_nan(mn, x[i], x[i + 1]);
        mx = max_nan(mx, x[i], x[i + 1]);
    }
    mn = min_nan(mn, x[15], x[15]);
    mx = max_nan(mx, x[15], x[15]);
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
        const float a = __shfl_xor_sync(kFullWarp, mn, d), b = __shfl_xor_sync(kFullWarp, mx, d);
        mn = min_nan(mn, a, a);
        mx = max_nan(mx, b, b);
    }
    float step = bf16_of(__fdiv_rn(__fsub_rn(mx, mn), 15.f));
    const float mid = __fadd_rn(mn, __fmul_rn(8.f, step)), zero = bf16_of(mid);
    if (fabsf(zero - mid) > 0.25f * step) {
        const float wide = fmaxf(__fdiv_rn(__fsub_rn(mx, zero), 7.f), 0.125f * __fsub_rn(zero, mn));
        step = __uint_as_float((__float_as_uint(wide) + 0xffffu) & 0xffff0000u);  // up to the next bf16
    }
    scale = fvp::pack_bf16x2(step, zero);
    lo = hi = 0x88888888u;
    if (!(step > 0.f)) return;
    // code + 8 = 15 u, u = ((x - zero) / step + 8) / 15 clamped to 0 .. 1.  By the reciprocal 15 u is off by some 2^-20, which moves a
    // code only where it lies at the middle between two: a lane that meets such a value settles it apart.  (True divisions there cost: values
    // that came in as bf16 lie exactly in the middle often, in some row of every third warp.)  Adding 1.5 2^23 rounds to the nearest even
    // integer; four codes are put together as one number in f32, which 16 bits fit exactly.
    constexpr float kRound = 12582912.f;
    const float inv = __frcp_rn(step), inv15 = inv * (1.f / 15.f);
    uint32_t part[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        float r[4], middle = inv <= 3e38f ? 0.f : 1.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float u = fma_sat(__fsub_rn(x[4 * k + i], zero), inv15, 8.f / 15.f);
            r[i] = __fsub_rn(__fmaf_rn(u, 15.f, kRound), kRound);
            middle = fmaxf(middle, fabsf(__fmaf_rn(u, 15.f, -r[i])));
        }
        const float four = __fmaf_rn(__fmaf_rn(__fmaf_rn(r[3], 16.f, r[2]), 16.f, r[1]), 16.f, r[0]);
        part[k] = __float_as_uint(__fadd_rn(four, 8388608.f));  // its lowest 16 bits
        if (middle > 0.49998f) part[k] = settle4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3], zero, step, inv);
    }
    lo = __byte_perm(part[0], part[1], 0x5410);
    hi = __byte_perm(part[2], part[3], 0x5410);
}

// Rows of heads first, first + step, .. below `last`, UNROLL at a time: raw bits in, `use(head, u0, u1)` gets 16 values.
template <int UNROLL, class Use>
FV_DEV void for_heads(const uint16_t* src, long long stride, int first, int last, int step, const Use& use) {
    int h = first;
    for (; h + (UNROLL - 1) * step < last; h += UNROLL * step) {
        uint4 u[UNROLL][2];
#pragma unroll
        for (int i = 0; i < UNROLL; i++) {
            const uint4* p = reinterpret_cast<const uint4*>(src + (long long)(h + i * step) * stride);
            u[i][0] = __ldg(p);
            u[i][1] = __ldg(p + 8);
        }
#pragma unroll
        for (int i = 0; i < UNROLL; i++) use(h + i * step, u[i][0], u[i][1]);
    }
    for (; h < last; h += step) {
        const uint4* p = reinterpret_cast<const uint4*>(src + (long long)h * stride);
        use(h, __ldg(p), __ldg(p + 8));
    }
}

template <bool Q4, bool HALF>
__global__ void __launch_bounds__(kThreads) fv_paged_append_kernel(const AppendArgs a) {
    const int lane = threadIdx.x & 31, part = threadIdx.x & 7;
    const int block = blockIdx.x / a.parts, share = blockIdx.x - block * a.parts;
    const int t = min(block * kTokens + (int)(threadIdx.x >> 3), a.batch.tokens - 1);  // (a lane past the end repeats the last
    bool mine = block * kTokens + (int)(threadIdx.x >> 3) < a.batch.tokens;            // token's loads and stores nothing)
    const int s = seq_of_slot(a.batch.cu_q, a.batch.seqs, t, lane);
    int key = -1, page = -1;
    if (mine && s < a.batch.seqs) {
        const Seq seq = seq_of(a.batch, s);
        const int at = t - seq.q0;
        mine = at >= 0 && at < seq.nq;
        key = mine ? seq.len - seq.nq + at : -1;  // the token's index in its sequence
        if (key >= 0) page = page_of(a.pool, a.batch, s, key);
    } else {
        mine = false;  // behind the last sequence
    }
    const bool turn = a.cosv != nullptr;
    bool placed = key >= 0;
    float cs[8], sn[8];
    if (turn) {
        const int pos = a.positions ? __ldg(a.positions + t) : key;
        if (placed && (unsigned)pos >= (unsigned)a.table_rows) {
            report(a.batch.status, FV_ST_BAD_POSITION);
            placed = false;
        }
        const size_t row = (size_t)(placed ? pos : 0) * kD;
        if (HALF) {  // pairs (i, i + 64): this lane's are 8 part .. 8 part + 7
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float4 c = __ldg(reinterpret_cast<const float4*>(a.cosv + row + 8 * part) + i);
                const float4 n = __ldg(reinterpret_cast<const float4*>(a.sinv + row + 8 * part) + i);
                cs[4 * i] = c.x; cs[4 * i + 1] = c.y; cs[4 * i + 2] = c.z; cs[4 * i + 3] = c.w;
                sn[4 * i] = n.x; sn[4 * i + 1] = n.y; sn[4 * i + 2] = n.z; sn[4 * i + 3] = n.w;
            }
        } else {  // pairs (2 i, 2 i + 1): four in each of the lane's two pieces; the tables hold every value twice
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const size_t o = row + 8 * part + 64 * (i >> 1) + 4 * (i & 1);
                const float4 c = __ldg(reinterpret_cast<const float4*>(a.cosv + o));
                const float4 n = __ldg(reinterpret_cast<const float4*>(a.sinv + o));
                cs[2 * i] = c.x; cs[2 * i + 1] = c.z;
                sn[2 * i] = n.x; sn[2 * i + 1] = n.z;
            }
        }
    }
    // This CTA's share of the token's rows -- q's heads, then K's, then V's -- is every parts-th of them, so that each share has its
    // part of the rows that are quantised (with runs of rows the last share had them all: 46 against 31 us for 4 142 tokens of
    // 40 + 2 x 8 heads).
    const int hk = a.pool.kv_heads, parts = a.parts;
    auto first_of = [&](int before) { return (share + parts - before % parts) % parts; };  // `before` rows come before head 0
    for_heads<4>(a.q + t * a.q_tok + 8 * part, a.q_head, share, a.q_heads, parts, [&](int h, uint4 u0, uint4 u1) {
        if (!mine) return;
        if (!placed) {
            u0 = u1 = make_uint4(0, 0, 0, 0);
        } else if (turn) {
            float x[16];
            widen8(u0, x);
            widen8(u1, x + 8);
            rotate16<HALF>(x, cs, sn);
            u0 = narrow8(x);
            u1 = narrow8(x + 8);
        }
        uint4* o = reinterpret_cast<uint4*>(a.q_out + ((size_t)t * a.q_heads + h) * kD + 8 * part);
        o[0] = u0;
        o[8] = u1;
    });
    const bool store = placed && page >= 0;
    const size_t first = store ? pool_row(a.pool, page, 0, key) : 0;  // head h: h << log_rows rows further on
    auto put = [&](const uint8_t* pool, const uint32_t* scales, bool rotated) {
        return [=, &cs, &sn](int h, uint4 u0, uint4 u1) {
            const size_t row = first + ((size_t)h << a.pool.log_rows);
            if (Q4 || rotated) {
                float x[16];
                widen8(u0, x);
                widen8(u1, x + 8);
                if (rotated) rotate16<HALF>(x, cs, sn);
                if (Q4) {
                    uint32_t lo, hi, scale;
                    quantize16(x, lo, hi, scale);
                    if (!store) return;
                    uint32_t* o = reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(pool) + row * kQ4Bytes);
                    o[part] = lo;
                    o[8 + part] = hi;
                    if (part == 0) const_cast<uint32_t*>(scales)[row] = scale;
                    return;
                }
                u0 = narrow8(x);
                u1 = narrow8(x + 8);
            }
            if (!store) return;
            uint4* o = reinterpret_cast<uint4*>(const_cast<uint8_t*>(pool) + row * (2 * kD)) + part;
            o[0] = u0;
            o[8] = u1;
        };
    };
    constexpr int kUnroll = Q4 ? 2 : 4;
    const int k0 = first_of(a.q_heads), v0 = first_of(a.q_heads + hk);
    if (turn) for_heads<kUnroll>(a.k + t * a.k_tok + 8 * part, a.k_head, k0, hk, parts, put(a.pool.k, a.pool.k_scale, true));
    else for_heads<kUnroll>(a.k + t * a.k_tok + 8 * part, a.k_head, k0, hk, parts, put(a.pool.k, a.pool.k_scale, false));
    for_heads<kUnroll>(a.v + t * a.v_tok + 8 * part, a.v_head, v0, hk, parts, put(a.pool.v, a.pool.v_scale, false));
}

// Read: row r of the packed result is key first[s] + (r - cu_rows[s]) of sequence s, K and V, as bf16 (4-bit rows as the
// values they stand for, rounded once).  Keys that the sequence does not hold and rows behind the last one give zeros.
// The append's split: 8 lanes a row, a CTA 16 neighbouring rows of its share of the heads.  (Lane i holds values 8 i .. 8 i + 7 and
// 64 + 8 i ..: with 16 values side by side its two stores would each fill half of a 32-byte sector, 60 against 53 us for
// 32 760 rows x 12 heads of 4 bits.)
struct ReadArgs {
    Pool pool;
    Batch batch;
    const int *cu_rows, *first;
    uint16_t *k_out, *v_out;
    int rows, parts;
};

// 8 codes as bf16 values zero + step code: 128 + n by or-ing the code into 128's mantissa, 136 off is code exactly, and
// one fused multiply-add rounds once.
FV_DEV uint4 expand8(uint32_t w, uint32_t step2, uint32_t zero2) {
    const uint32_t odd = w >> 4;
    uint32_t h[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t pair = __byte_perm(w, odd, (uint32_t)(k | (k << 4) | ((4 + k) << 8) | ((4 + k) << 12)));
        uint32_t c = (pair & 0x000f000fu) | 0x43004300u;
        asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(c) : "r"(0xc308c308u));
        asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(h[k]) : "r"(c), "r"(step2), "r"(zero2));
    }
    return make_uint4(h[0], h[1], h[2], h[3]);
}

template <bool Q4>
__global__ void __launch_bounds__(kThreads) fv_paged_read_kernel(const ReadArgs a) {
    constexpr int UNROLL = 8;  // rows in flight
    const int lane = threadIdx.x & 31, part = threadIdx.x & 7;
    const int block = blockIdx.x / a.parts, share = blockIdx.x - block * a.parts;
    const int t = block * kTokens + (int)(threadIdx.x >> 3);
    const int s = seq_of_slot(a.cu_rows, a.batch.seqs, min(t, a.rows - 1), lane);
    if (t >= a.rows) return;
    long long key = -1;
    int page = -1;
    if (s < a.batch.seqs) {
        const int r0 = __ldg(a.cu_rows + s), r1 = __ldg(a.cu_rows + s + 1), len = __ldg(a.batch.kv_len + s);
        if (r0 < 0 || t < r0 || r1 <= t || len < 0 || len > a.batch.max_kv) {
            report(a.batch.status, FV_ST_BAD_BATCH);
        } else {
            key = (a.first ? (long long)__ldg(a.first + s) : (long long)len - (r1 - r0)) + (t - r0);
            if (key >= 0 && key < len) page = page_of(a.pool, a.batch, s, (int)key);
        }
    }
    const int hk = a.pool.kv_heads;
    const size_t first = page >= 0 ? pool_row(a.pool, page, 0, (int)key) : 0;
    const int r0 = (int)((long long)2 * hk * share / a.parts), r1 = (int)((long long)2 * hk * (share + 1) / a.parts);
    for (int r = r0; r < r1; r += UNROLL) {
        uint4 u[UNROLL][2];
        uint32_t sc[UNROLL];
#pragma unroll
        for (int i = 0; i < UNROLL; i++) {
            u[i][0] = u[i][1] = make_uint4(0, 0, 0, 0);
            sc[i] = 0;
            if (r + i >= r1 || page < 0) continue;
            const bool is_k = r + i < hk;
            const size_t row = first + ((size_t)(is_k ? r + i : r + i - hk) << a.pool.log_rows);
            const uint8_t* base = is_k ? a.pool.k : a.pool.v;
            if (Q4) {
                const uint32_t* p = reinterpret_cast<const uint32_t*>(base + row * kQ4Bytes) + part;
                u[i][0].x = __ldg(p);
                u[i][0].y = __ldg(p + 8);
                sc[i] = __ldg((is_k ? a.pool.k_scale : a.pool.v_scale) + row);
            } else {
                const uint4* p = reinterpret_cast<const uint4*>(base + row * (2 * kD)) + part;
                u[i][0] = __ldg(p);
                u[i][1] = __ldg(p + 8);
            }
        }
#pragma unroll
        for (int i = 0; i < UNROLL; i++) {
            if (r + i >= r1) continue;
            if (Q4 && page >= 0) {
                const uint32_t step2 = __byte_perm(sc[i], 0, 0x1010), zero2 = __byte_perm(sc[i], 0, 0x3232);
                u[i][1] = expand8(u[i][0].y, step2, zero2);
                u[i][0] = expand8(u[i][0].x, step2, zero2);
            }
            const bool is_k = r + i < hk;
            uint4* o = reinterpret_cast<uint4*>((is_k ? a.k_out : a.v_out) + ((size_t)t * hk + (is_k ? r + i : r + i - hk)) * kD) + part;
            __stcs(o, u[i][0]);  // (not read again here: 49 against 53 us for 32 760 rows x 12 heads of 4 bits)
            __stcs(o + 8, u[i][1]);
        }
    }
}

// ---- the host side shared by the paged entries ---------------------------------------------------------------------

int check_paged(const char* what, const fv_paged_kv* kv, const fv_paged_batch* b, int rows, Pool* pool, Batch* batch, int* dev) {
    if (!kv || !b) return fvrt::fail(FV_ERR_INVALID, "%s: null cache or batch", what);
    if (kv->format != FV_PAGE_BF16 && kv->format != FV_PAGE_Q4) return fvrt::fail(FV_ERR_INVALID, "%s: unknown page format %d", what, kv->format);
    if (kv->pages < 1 || kv->kv_heads < 1 || kv->kv_heads > 4096)
        return fvrt::fail(FV_ERR_INVALID, "%s: a pool of %d pages and %d heads", what, kv->pages, kv->kv_heads);
    if (kv->page_rows < 16 || kv->page_rows > 256 || (kv->page_rows & (kv->page_rows - 1)))
        return fvrt::fail(FV_ERR_INVALID, "%s: pages of %d rows (16, 32, 64, 128 or 256)", what, kv->page_rows);
    if (rows < 0 || b->seqs < 0 || b->max_q < 0 || b->max_kv < 0 || b->table_width < 0)
        return fvrt::fail(FV_ERR_INVALID, "%s: negative size in the batch", what);
    if ((long long)b->table_width * kv->page_rows < b->max_kv)
        return fvrt::fail(FV_ERR_INVALID, "%s: a table of %d pages of %d rows does not hold %d keys", what, b->table_width, kv->page_rows, b->max_kv);
    if (b->max_kv > 0x3fffffff || b->max_q > 0x3fffffff || rows > 0x3fffffff)
        return fvrt::fail(FV_ERR_INVALID, "%s: sequences of %d keys, %d of them new, %d rows", what, b->max_kv, b->max_q, rows);
    if ((long long)kv->pages * kv->kv_heads * kv->page_rows > 0xfffffff0ll)  // (the kernels number the pool's rows in 32 bits)
        return fvrt::fail(FV_ERR_INVALID, "%s: a pool of %d pages x %d heads x %d rows", what, kv->pages, kv->kv_heads, kv->page_rows);
    if (b->seqs == 0 || rows == 0) return FV_DECLINED;
    const int rc = fvrt::require_sm100(dev);
    if (rc != FV_RAN) return rc;
    if (!kv->k || !kv->v || !b->kv_len || !b->cu_q || (!b->page_table && b->table_width > 0))
        return fvrt::fail(FV_ERR_INVALID, "%s: null operand", what);
    uintptr_t bits = (uintptr_t)kv->k | (uintptr_t)kv->v;
    if (kv->format == FV_PAGE_Q4) {
        if (!kv->k_scale || !kv->v_scale) return fvrt::fail(FV_ERR_INVALID, "%s: 4-bit pages without scales", what);
        bits |= (uintptr_t)kv->k_scale | (uintptr_t)kv->v_scale;
    }
    if ((bits & 15) || (((uintptr_t)b->page_table | (uintptr_t)b->kv_len | (uintptr_t)b->cu_q) & 3))
        return fvrt::fail(FV_ERR_INVALID, "%s: pools must be 16-byte aligned, tables 4-byte aligned", what);
    int* status;
    const int rc2 = fvrt::status_word(*dev, &status);
    if (rc2 != FV_RAN) return rc2;
    int log_rows = 4;
    while ((1 << log_rows) < kv->page_rows) log_rows++;
    *pool = Pool{(const uint8_t*)kv->k, (const uint8_t*)kv->v, (const uint32_t*)kv->k_scale, (const uint32_t*)kv->v_scale,
                 kv->pages, log_rows, kv->kv_heads};
    *batch = Batch{b->page_table, b->kv_len, b->cu_q, b->seqs, b->table_width, rows, b->max_q, b->max_kv, status + 1};
    return FV_RAN;
}

// CTAs that share the heads of the same 16 tokens: about eight per SM with few tokens, as few as possible (one reads the tables'
// rows once for all heads) with many.
static int parts_for(int tokens, int rows, int sms) {
    const long long blocks = (tokens + kTokens - 1) / kTokens;
    const long long want = (8ll * sms + blocks / 2) / blocks;
    return (int)(want < 1 ? 1 : want > rows ? rows : want);
}

}  // namespace fvpg

extern "C" int fv_paged_append_bf16(void* stream, const fv_paged_kv* kv, const fv_paged_batch* b, const fv_paged_rows* x) {
    using namespace fvpg;
    fvrt::clear_error();
    if (!x) return fvrt::fail(FV_ERR_INVALID, "paged append: null operand");
    const void *k = x->k, *v = x->v, *q = x->q;
    void* q_out = x->q_out;
    const float *cosv = x->cosv, *sinv = x->sinv;
    const int tokens = x->tokens, q_heads = x->q_heads, table_rows = x->table_rows, pairing = x->pairing;
    AppendArgs a{};
    int dev;
    const int rc = check_paged("paged append", kv, b, tokens, &a.pool, &a.batch, &dev);
    if (rc != FV_RAN) return rc;
    if (!k || !v) return fvrt::fail(FV_ERR_INVALID, "paged append: null operand");
    if ((q != nullptr) != (q_out != nullptr) || (q && q_heads < 1) || q_heads > 4096)
        return fvrt::fail(FV_ERR_INVALID, "paged append: q, q_out and q_heads go together");
    if ((cosv != nullptr) != (sinv != nullptr) || (cosv && table_rows < 1) || (x->positions && !cosv))
        return fvrt::fail(FV_ERR_INVALID, "paged append: cos, sin, their rows and positions go together");
    if (pairing != FV_ROPE_INTERLEAVED && pairing != FV_ROPE_HALF)
        return fvrt::fail(FV_ERR_INVALID, "paged append: unknown pairing %d", pairing);
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)cosv | (uintptr_t)sinv) & 15)
        return fvrt::fail(FV_ERR_INVALID, "paged append: operands must be 16-byte aligned");
    if ((uintptr_t)x->positions & 3) return fvrt::fail(FV_ERR_INVALID, "paged append: positions must be 4-byte aligned");
    if ((x->k_tok | x->k_head | x->v_tok | x->v_head | (q ? x->q_tok | x->q_head : 0)) & 7)
        return fvrt::fail(FV_ERR_INVALID, "paged append: strides must be multiples of 8 values");
    a.q = (const uint16_t*)q;
    a.k = (const uint16_t*)k;
    a.v = (const uint16_t*)v;
    a.q_out = (uint16_t*)q_out;
    a.q_tok = x->q_tok; a.q_head = x->q_head; a.k_tok = x->k_tok; a.k_head = x->k_head; a.v_tok = x->v_tok; a.v_head = x->v_head;
    a.cosv = cosv;
    a.sinv = sinv;
    a.positions = x->positions;
    a.table_rows = table_rows;
    a.q_heads = q ? q_heads : 0;
    int sms;
    const int rc2 = fvrt::sm_count(dev, &sms);
    if (rc2 != FV_RAN) return rc2;
    a.parts = parts_for(tokens, a.q_heads + 2 * kv->kv_heads, sms);
    const long long grid = (((long long)tokens + kTokens - 1) / kTokens) * a.parts;
    if (grid > 0x7fffffffll) return FV_DECLINED;
    const bool q4 = kv->format == FV_PAGE_Q4, half = pairing == FV_ROPE_HALF;
    const auto fn = q4 ? (half ? fv_paged_append_kernel<true, true> : fv_paged_append_kernel<true, false>)
                       : (half ? fv_paged_append_kernel<false, true> : fv_paged_append_kernel<false, false>);
    fn<<<(unsigned)grid, kThreads, 0, (cudaStream_t)stream>>>(a);
    FV_CUDA(cudaGetLastError());
    fvrt::ran_later(fvrt::kLogPaged, "paged append: fv_paged_append_kernel<%s> %d tokens x (%d + 2 x %d) heads", q4 ? "4 bits" : "bf16",
              tokens, a.q_heads, kv->kv_heads);
    return FV_RAN;
}

extern "C" int fv_paged_read_bf16(void* stream, const fv_paged_kv* kv, const fv_paged_batch* b, const int* cu_rows, const int* first,
                                  int rows, void* k_out, void* v_out) {
    using namespace fvpg;
    fvrt::clear_error();
    ReadArgs a{};
    int dev;
    const int rc = check_paged("paged read", kv, b, rows, &a.pool, &a.batch, &dev);
    if (rc != FV_RAN) return rc;
    if (!cu_rows || !k_out || !v_out) return fvrt::fail(FV_ERR_INVALID, "paged read: null operand");
    if (((uintptr_t)k_out | (uintptr_t)v_out) & 15 || ((uintptr_t)cu_rows | (uintptr_t)first) & 3)
        return fvrt::fail(FV_ERR_INVALID, "paged read: results must be 16-byte aligned, tables 4-byte aligned");
    a.cu_rows = cu_rows;
    a.first = first;
    a.k_out = (uint16_t*)k_out;
    a.v_out = (uint16_t*)v_out;
    a.rows = rows;
    int sms;
    const int rc2 = fvrt::sm_count(dev, &sms);
    if (rc2 != FV_RAN) return rc2;
    a.parts = parts_for(rows, 2 * kv->kv_heads, sms);
    const long long grid = (((long long)rows + kTokens - 1) / kTokens) * a.parts;
    if (grid > 0x7fffffffll) return FV_DECLINED;
    if (kv->format == FV_PAGE_Q4) fv_paged_read_kernel<true><<<(unsigned)grid, kThreads, 0, (cudaStream_t)stream>>>(a);
    else fv_paged_read_kernel<false><<<(unsigned)grid, kThreads, 0, (cudaStream_t)stream>>>(a);
    FV_CUDA(cudaGetLastError());
    fvrt::ran_later(fvrt::kLogPaged, "paged read: fv_paged_read_kernel<%s> %d rows x 2 x %d heads", kv->format == FV_PAGE_Q4 ? "4 bits" : "bf16", rows,
              kv->kv_heads);
    return FV_RAN;
}
