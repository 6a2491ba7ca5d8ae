// What the kernels over a paged K/V cache share: the pool, the ragged batch, the page lookup and the visible keys of a
// query position.  Everything a kernel takes from device memory to address with (page ids, lengths, row offsets,
// positions) is checked against the sizes the host gave before it is used; what fails is left out and reported in the
// second status word (fv_device_status), so a broken table costs a wrong row, never an access out of range.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "fv_ptx.cuh"

// Codes of the second status word (the first one carries the bounded waits, which stop later launches; these do not).
#define FV_ST_BAD_PAGE 200      // a page that the call needs lies outside the pool, or past the table's width
#define FV_ST_BAD_BATCH 201     // cu_q is not ascending inside the batch's tokens, or a length is outside its bound
#define FV_ST_BAD_POSITION 202  // a position outside the rotation tables

namespace fvpg {

constexpr int kD = 128;
constexpr int kQ4Bytes = 64;  // a row of 128 4-bit codes
constexpr uint32_t kFullWarp = 0xffffffffu;

// The pool: K and V of one layer, [pages, kv_heads, page_rows, 128] bf16, or codes [pages, kv_heads, page_rows, 64] with
// (step, zero) pairs [pages, kv_heads, page_rows, 2] bf16.  page_rows = 1 << log_rows, at least 16.
struct Pool {
    const uint8_t *k, *v;
    const uint32_t *k_scale, *v_scale;
    int pages, log_rows, kv_heads;
};
struct Batch {
    const int* table;   // [seqs, table_width]
    const int* kv_len;  // [seqs]
    const int* cu_q;    // [seqs + 1]
    int seqs, table_width, tokens, max_q, max_kv;
    int* status;        // the data status word
};

FV_DEV void report(int* status, int code) { atomicCAS(status, 0, code); }

struct Seq {
    int q0, nq, len;
};
// Rows and length of sequence s; a sequence whose numbers break the batch's bounds counts as empty.
FV_DEV Seq seq_of(const Batch& b, int s) {
    Seq x;
    x.q0 = __ldg(b.cu_q + s);
    const int q1 = __ldg(b.cu_q + s + 1);
    x.len = __ldg(b.kv_len + s);
    x.nq = q1 - x.q0;
    if (x.q0 < 0 || q1 < x.q0 || q1 > b.tokens || x.nq > b.max_q || x.len < 0 || x.len > b.max_kv) {
        report(b.status, FV_ST_BAD_BATCH);
        x = Seq{0, 0, 0};
    }
    return x;
}
// The sequence that token t belongs to (the number of sequences that end at or before it): warp-collective, one round
// trip for up to 32 sequences.  seqs: behind the last one.
FV_DEV int seq_of_token(const int* cu, int seqs, int t, int lane) {
    int s = 0;
    for (int base = 0; base < seqs; base += 32) {
        const bool before = base + lane < seqs && __ldg(cu + base + lane + 1) <= t;
        const int n = __popc(__ballot_sync(kFullWarp, before));
        s += n;
        if (n < 32) break;
    }
    return s;
}
// Page id of key `key` of sequence s, or -1 (reported) when there is none inside the pool.
FV_DEV int page_of(const Pool& p, const Batch& b, int s, int key) {
    const int i = key >> p.log_rows;
    int page = -1;
    if (i < b.table_width) page = __ldg(b.table + (size_t)s * b.table_width + i);
    if ((unsigned)page >= (unsigned)p.pages) {
        report(b.status, FV_ST_BAD_PAGE);
        page = -1;
    }
    return page;
}
// Row number of (page, kv head, row in page) inside the pool.
FV_DEV size_t pool_row(const Pool& p, int page, int head, int key) {
    return ((((size_t)page * p.kv_heads + head) << p.log_rows) + (size_t)(key & ((1 << p.log_rows) - 1)));
}

// A divisor known on the host: quotients of 0 .. 2^31 - 1 by a multiplication (Granlund and Montgomery, Division by Invariant
// Integers using Multiplication, 1994).  The kernels' indices and masks divide a dozen times before anything is read; each division that is not
// one of these is a chain of some twenty instructions.
struct Div {
    uint32_t d, mul;
    int shift;
    static Div of(int d) {
        Div v{(uint32_t)d, 0, 0};
        while ((1ull << v.shift) < v.d) v.shift++;
        v.mul = (uint32_t)((((1ull << v.shift) - v.d) << 32) / v.d + 1);
        return v;
    }
};
FV_DEV int operator/(int n, const Div& v) { return (int)((__umulhi((uint32_t)n, v.mul) + (uint32_t)n) >> v.shift); }

// The mask: key j is visible to position p iff t_j <= t_p and (window == 0 or t_p - t_j < window or t_j < sink), with
// t = index / block; block == 0: every key below the sequence's length.
struct Mask {
    int block, window, sink;
    Div by_block;
};
// Keys that positions first .. last see between them: [0, sink) U [lo, hi), sink <= lo.
struct Span {
    int sink, lo, hi;
};
FV_DEV int mul_sat(int a, int b) {
    const long long v = (long long)a * (long long)b;
    return v > 0x7fffffffll ? 0x7fffffff : (int)v;
}
FV_DEV Span span_of(const Mask& m, int first, int last, int len) {
    if (m.block == 0) return Span{0, 0, len};
    if (last < 0) return Span{0, 0, 0};
    Span s;
    s.hi = min(len, mul_sat(last / m.by_block + 1, m.block));
    s.lo = 0;
    s.sink = 0;
    if (m.window > 0) {
        s.lo = mul_sat(max(0, max(first, 0) / m.by_block - m.window + 1), m.block);
        s.sink = min(mul_sat(m.sink, m.block), s.hi);
        if (s.sink >= s.lo) s.lo = s.sink = 0;
    }
    return s;
}

}  // namespace fvpg
