// Writing to and reading from a paged K/V cache (no counterpart in the reference: its causal cache is one contiguous
// buffer per sequence that is copied down past the sink for every block, crates/fastvideo-cudarc/src/wan/causal.rs:
// 541-628; over pages the rows in between are given back instead).
//
// Append: every token's K (and q) is rotated with its position's table row, V is taken as it is, and both land in the
// token's row of its sequence's page, in bf16 or in 4 bits; q goes to a packed tensor.  Rotation arithmetic is that of the
// BHSD rope kernel: f32, products and sums rounded separately, one rounding to bf16.  4 bits, per row of 128 values x:
//     step = bf16((max x - min x) / 15), zero = bf16(min x + 8 step), code = clamp(rint((x - zero) / step), -8, 7),
// stored as code + 8 (even value in the low half of a byte): a row stands for zero + step * code.  K is quantised from
// the f32 rotation, not from its bf16 rounding.  One scale for the whole row because its factor then leaves the
// attention's products (q . k = step (q . code) + zero sum(q)), so that these run on exact codes.
//
// HBM-bound: 8 lanes hold one row of one head (16 values a lane: 8 from each half, so both kinds of pairs are inside a
// lane), a CTA works on one token and keeps its cosines and sines in registers over the heads it takes.
#include "fv_runtime.h"
#include "paged.cuh"
#include "paged_host.h"

namespace fvpg {

constexpr int kThreads = 128;
constexpr int kRowsAtOnce = kThreads / 8;  // rows (of one head each) that a CTA has in hand at a time

struct AppendArgs {
    Pool pool;
    Batch batch;
    const uint16_t *q, *k, *v;
    uint16_t* q_out;
    long long q_tok, q_head, k_tok, k_head, v_tok, v_head;  // strides in values
    const float *cosv, *sinv;
    const int* positions;
    int table_rows, q_heads, parts, half;
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
FV_DEV float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
FV_DEV float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// x[0 .. 7] are values 8 c .. 8 c + 7 of a row, x[8 .. 15] are 64 values further on; cs / sn the factors of its 8 pairs.
FV_DEV void rotate16(float (&x)[16], const float (&cs)[8], const float (&sn)[8], bool half) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int a = half ? i : 2 * i, b = half ? i + 8 : 2 * i + 1;
        const float xa = x[a], xb = x[b];
        x[a] = __fsub_rn(__fmul_rn(xa, cs[i]), __fmul_rn(xb, sn[i]));
        x[b] = __fadd_rn(__fmul_rn(xa, sn[i]), __fmul_rn(xb, cs[i]));
    }
}
// The same row in 4 bits: codes of this lane's 16 values as two words (8 values each), (step, zero) as one.  Collective
// over the row's 8 lanes (the callers' lanes of a row are live or not together).
FV_DEV void quantize16(const float (&x)[16], uint32_t& lo, uint32_t& hi, uint32_t& scale, uint32_t lanes) {
    float mn = x[0], mx = x[0];
#pragma unroll
    for (int i = 1; i < 16; i++) {
        mn = min_nan(mn, x[i]);
        mx = max_nan(mx, x[i]);
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
        mn = min_nan(mn, __shfl_xor_sync(lanes, mn, d));
        mx = max_nan(mx, __shfl_xor_sync(lanes, mx, d));
    }
    const float step = bf16_of(__fdiv_rn(__fsub_rn(mx, mn), 15.f));
    const float zero = bf16_of(__fadd_rn(mn, __fmul_rn(8.f, step)));
    scale = fvp::pack_bf16x2(step, zero);
    lo = hi = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        // (a row of one value has step 0: code 0.  A row with a value that is not finite has a step that is not: its
        // codes say nothing, the row stands for NaN.)
        float c = step > 0.f ? rintf(__fdiv_rn(__fsub_rn(x[i], zero), step)) : 0.f;
        c = fminf(fmaxf(c, -8.f), 7.f);
        const uint32_t n = (uint32_t)((int)c + 8) & 15u;
        if (i < 8) lo |= n << (4 * i);
        else hi |= n << (4 * (i - 8));
    }
}

template <bool Q4>
__global__ void __launch_bounds__(kThreads) fv_paged_append_kernel(const AppendArgs a) {
    const int lane = threadIdx.x & 31, part = threadIdx.x & 7, slot = threadIdx.x >> 3;
    const uint32_t lanes = 0xffu << (lane & 24);
    const int t = blockIdx.x / a.parts, block = blockIdx.x - t * a.parts;
    const int s = seq_of_token(a.batch.cu_q, a.batch.seqs, t, lane);
    if (s >= a.batch.seqs) return;  // behind the last sequence
    const Seq seq = seq_of(a.batch, s);
    const int at = t - seq.q0;
    if (at < 0 || at >= seq.nq) return;
    const int key = seq.len - seq.nq + at;  // the token's index in its sequence
    int page = -1;
    if (key >= 0) page = page_of(a.pool, a.batch, s, key);
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
        if (a.half) {  // pairs (i, i + 64): this lane's are 8 part .. 8 part + 7
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
    // Rows of this token: q's heads, then K's, then V's; dealt to the parts in runs of kRowsAtOnce.
    const int hk = a.pool.kv_heads, rows = a.q_heads + 2 * hk;
    for (int r = block * kRowsAtOnce + slot; r < rows; r += a.parts * kRowsAtOnce) {
        const bool is_q = r < a.q_heads, is_k = !is_q && r < a.q_heads + hk;
        const int head = is_q ? r : is_k ? r - a.q_heads : r - a.q_heads - hk;
        if (!is_q && page < 0) continue;
        const uint16_t* src = is_q ? a.q + t * a.q_tok + head * a.q_head : is_k ? a.k + t * a.k_tok + head * a.k_head
                                                                                : a.v + t * a.v_tok + head * a.v_head;
        const uint4 u0 = *reinterpret_cast<const uint4*>(src + 8 * part), u1 = *reinterpret_cast<const uint4*>(src + 64 + 8 * part);
        float x[16];
        widen8(u0, x);
        widen8(u1, x + 8);
        if (turn && (is_q || is_k)) rotate16(x, cs, sn, a.half);
        if (is_q) {
            uint16_t* o = a.q_out + ((size_t)t * a.q_heads + head) * kD + 8 * part;
            if (!placed) {
#pragma unroll
                for (int i = 0; i < 16; i++) x[i] = 0.f;
            }
            *reinterpret_cast<uint4*>(o) = narrow8(x);
            *reinterpret_cast<uint4*>(o + 64) = narrow8(x + 8);
            continue;
        }
        if (!placed) continue;
        const size_t row = pool_row(a.pool, page, head, key);
        uint8_t* base = const_cast<uint8_t*>(is_k ? a.pool.k : a.pool.v);
        if (Q4) {
            uint32_t lo, hi, scale;
            quantize16(x, lo, hi, scale, lanes);
            *reinterpret_cast<uint32_t*>(base + row * kQ4Bytes + 4 * part) = lo;
            *reinterpret_cast<uint32_t*>(base + row * kQ4Bytes + 32 + 4 * part) = hi;
            if (part == 0) const_cast<uint32_t*>(is_k ? a.pool.k_scale : a.pool.v_scale)[row] = scale;
        } else {
            uint16_t* o = reinterpret_cast<uint16_t*>(base) + row * kD + 8 * part;
            *reinterpret_cast<uint4*>(o) = narrow8(x);
            *reinterpret_cast<uint4*>(o + 64) = narrow8(x + 8);
        }
    }
}

// Read: row r of the packed result is key first[s] + (r - cu_rows[s]) of sequence s, K and V, as bf16 (4-bit rows as the
// values they stand for, rounded once).  Keys that the sequence does not hold and rows behind the last one give zeros.
struct ReadArgs {
    Pool pool;
    Batch batch;
    const int *cu_rows, *first;
    uint16_t *k_out, *v_out;
    int rows, parts;
};

template <bool Q4>
__global__ void __launch_bounds__(kThreads) fv_paged_read_kernel(const ReadArgs a) {
    const int lane = threadIdx.x & 31, part = threadIdx.x & 7, slot = threadIdx.x >> 3;
    const int t = blockIdx.x / a.parts, block = blockIdx.x - t * a.parts;
    const int s = seq_of_token(a.cu_rows, a.batch.seqs, t, lane);
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
    for (int r = block * kRowsAtOnce + slot; r < 2 * hk; r += a.parts * kRowsAtOnce) {
        const bool is_k = r < hk;
        const int head = is_k ? r : r - hk;
        uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0;
        if (page >= 0) {
            const size_t row = pool_row(a.pool, page, head, (int)key);
            const uint8_t* base = is_k ? a.pool.k : a.pool.v;
            if (Q4) {
                const uint32_t sc = __ldg((is_k ? a.pool.k_scale : a.pool.v_scale) + row);
                const uint32_t lo = __ldg(reinterpret_cast<const uint32_t*>(base + row * kQ4Bytes + 4 * part));
                const uint32_t hi = __ldg(reinterpret_cast<const uint32_t*>(base + row * kQ4Bytes + 32 + 4 * part));
                const float step = __uint_as_float(sc << 16), zero = __uint_as_float(sc & 0xffff0000u);
                float x[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {  // (step * code is exact in f32: 8 bits by 4)
                    const uint32_t n = ((i < 8 ? lo >> (4 * i) : hi >> (4 * (i - 8))) & 15u);
                    x[i] = fmaf(step, (float)((int)n - 8), zero);
                }
                u0 = narrow8(x);
                u1 = narrow8(x + 8);
            } else {
                const uint4* p = reinterpret_cast<const uint4*>(base + row * 2 * kD);
                u0 = __ldg(p + part);
                u1 = __ldg(p + 8 + part);
            }
        }
        uint16_t* o = (is_k ? a.k_out : a.v_out) + ((size_t)t * hk + head) * kD + 8 * part;
        *reinterpret_cast<uint4*>(o) = u0;
        *reinterpret_cast<uint4*>(o + 64) = u1;
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
    if (b->max_kv > 0x3fffffff) return fvrt::fail(FV_ERR_INVALID, "%s: sequences of %d keys", what, b->max_kv);
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

// CTAs per token: as many as keep the GPU busy when there are few tokens, as few as possible (one reads the tables'
// row once for all heads) when there are many.
static int parts_for(int tokens, int rows, int sms) {
    const int most = (rows + kRowsAtOnce - 1) / kRowsAtOnce;
    const long long want = (16ll * sms + tokens - 1) / tokens;
    return (int)(want < 1 ? 1 : want > most ? most : want);
}

}  // namespace fvpg

extern "C" int fv_paged_append_bf16(void* stream, const fv_paged_kv* kv, const fv_paged_batch* b, int tokens, const void* k, long long k_tok,
                                    long long k_head, const void* v, long long v_tok, long long v_head, const void* q,
                                    long long q_tok, long long q_head, int q_heads, void* q_out, const float* cosv,
                                    const float* sinv, int table_rows, const int* positions, int pairing) {
    using namespace fvpg;
    fvrt::clear_error();
    AppendArgs a{};
    int dev;
    const int rc = check_paged("paged append", kv, b, tokens, &a.pool, &a.batch, &dev);
    if (rc != FV_RAN) return rc;
    if (!k || !v) return fvrt::fail(FV_ERR_INVALID, "paged append: null operand");
    if ((q != nullptr) != (q_out != nullptr) || (q && q_heads < 1) || q_heads > 4096)
        return fvrt::fail(FV_ERR_INVALID, "paged append: q, q_out and q_heads go together");
    if ((cosv != nullptr) != (sinv != nullptr) || (cosv && table_rows < 1) || (positions && !cosv))
        return fvrt::fail(FV_ERR_INVALID, "paged append: cos, sin, their rows and positions go together");
    if (pairing != FV_ROPE_INTERLEAVED && pairing != FV_ROPE_HALF)
        return fvrt::fail(FV_ERR_INVALID, "paged append: unknown pairing %d", pairing);
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)cosv | (uintptr_t)sinv) & 15)
        return fvrt::fail(FV_ERR_INVALID, "paged append: operands must be 16-byte aligned");
    if ((k_tok | k_head | v_tok | v_head | (q ? q_tok | q_head : 0)) & 7)
        return fvrt::fail(FV_ERR_INVALID, "paged append: strides must be multiples of 8 values");
    a.q = (const uint16_t*)q;
    a.k = (const uint16_t*)k;
    a.v = (const uint16_t*)v;
    a.q_out = (uint16_t*)q_out;
    a.q_tok = q_tok; a.q_head = q_head; a.k_tok = k_tok; a.k_head = k_head; a.v_tok = v_tok; a.v_head = v_head;
    a.cosv = cosv;
    a.sinv = sinv;
    a.positions = positions;
    a.table_rows = table_rows;
    a.q_heads = q ? q_heads : 0;
    a.half = pairing == FV_ROPE_HALF;
    int sms;
    const int rc2 = fvrt::sm_count(dev, &sms);
    if (rc2 != FV_RAN) return rc2;
    a.parts = parts_for(tokens, a.q_heads + 2 * kv->kv_heads, sms);
    const long long grid = (long long)tokens * a.parts;
    if (grid > 0x7fffffffll) return FV_DECLINED;
    if (kv->format == FV_PAGE_Q4) fv_paged_append_kernel<true><<<(unsigned)grid, kThreads, 0, (cudaStream_t)stream>>>(a);
    else fv_paged_append_kernel<false><<<(unsigned)grid, kThreads, 0, (cudaStream_t)stream>>>(a);
    FV_CUDA(cudaGetLastError());
    fvrt::ran(fvrt::kLogPaged, "paged append: fv_paged_append_kernel<%s> %d tokens x (%d + 2 x %d) heads", kv->format == FV_PAGE_Q4 ? "4 bits" : "bf16",
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
    const long long grid = (long long)rows * a.parts;
    if (grid > 0x7fffffffll) return FV_DECLINED;
    if (kv->format == FV_PAGE_Q4) fv_paged_read_kernel<true><<<(unsigned)grid, kThreads, 0, (cudaStream_t)stream>>>(a);
    else fv_paged_read_kernel<false><<<(unsigned)grid, kThreads, 0, (cudaStream_t)stream>>>(a);
    FV_CUDA(cudaGetLastError());
    fvrt::ran(fvrt::kLogPaged, "paged read: fv_paged_read_kernel<%s> %d rows x 2 x %d heads", kv->format == FV_PAGE_Q4 ? "4 bits" : "bf16", rows,
              kv->kv_heads);
    return FV_RAN;
}
