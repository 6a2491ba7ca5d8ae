"""The paged K/V cache on the GPU: appending, reading back and attention against plain 64-bit implementations
(tests/_paged.py, where the tolerances are derived), at the sizes and masks where it can go wrong."""
import math

import pytest
import torch

from _paged import D, BF16_HALF, Case, attend64, pack, quantize, rotate32, rotate64, seen_matrix, stands_for, unpack

pytestmark = pytest.mark.gpu

FMTS = ["bf16", "q4"]


@pytest.fixture(params=["rows", "items"])
def kernel(request, monkeypatch):
    """Either of the two attention kernels, whichever the sizes would choose."""
    monkeypatch.setenv("FV_PAGED_KERNEL", request.param)
    return request.param


def check(got, want, bound, what):
    assert torch.isfinite(got).all(), what
    err = (got.double().cpu() - want).abs()
    worst = float((err / bound).max()) if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound, max-abs {float(err.max()):.3e}"


def mask_of(mask):
    from fastvideo_rs_b200.sdpa import BlockCausal
    return None if mask is None else BlockCausal(*mask)


# (kv_len, nq, heads, kv_heads, page_rows, mask)
ATTEND = [
    ([1], [1], 1, 1, 16, (1, 0, 0)),                              # one token, one key
    ([17], [1], 3, 1, 16, (1, 0, 0)),                             # a tile and one key
    ([777], [1], 12, 12, 16, (1, 0, 0)),
    ([130, 0, 16, 5], [1, 0, 1, 1], 8, 2, 32, (1, 0, 0)),         # an empty sequence among others
    ([63, 1025], [1, 1], 10, 2, 64, (1, 0, 0)),                   # five heads to a key head
    ([300], [1], 16, 1, 128, (1, 0, 0)),                          # sixteen: two groups of eight rows
    ([300, 40], [1, 1], 21, 3, 256, (1, 0, 0)),
    ([515], [1], 4, 4, 16, (1, 100, 0)),                          # a window that starts inside a tile
    ([515, 90], [1, 1], 8, 2, 16, (1, 100, 5)),                   # and sinks
    ([515], [1], 8, 2, 32, (1, 1, 0)),                            # a window of the token itself
    ([40], [1], 8, 2, 32, (1, 50, 3)),                            # a window longer than the sequence
    ([77], [5], 2, 2, 16, (1, 0, 0)),                             # short chunks
    ([77, 200, 9], [9, 3, 9], 4, 2, 16, (1, 20, 2)),
    ([150], [150], 2, 1, 16, (1, 0, 0)),                          # a whole prompt
    ([150], [150], 2, 1, 16, (1, 33, 4)),
    ([700], [130], 4, 1, 64, (1, 0, 0)),                          # rows in several blocks
    ([900, 333], [300, 129], 8, 2, 32, (1, 257, 7)),
    ([513], [257], 3, 3, 64, (1, 0, 0)),
    ([640], [160], 2, 2, 64, (160, 0, 0)),                        # blocks of frames
    ([645], [170], 2, 2, 64, (80, 3, 1)),
    ([1000], [129], 2, 2, 16, (100, 2, 2)),                       # blocks that no tile divides
    ([333], [40], 6, 2, 32, None),                                # no mask
    ([2000], [1], 4, 1, 16, None),
    ([4100], [1], 8, 1, 64, (1, 0, 0)),                           # many key ranges
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("i", range(len(ATTEND)))
def test_attend_matches_the_formula(fvlib, kernel, fmt, i):
    from fastvideo_rs_b200 import paged, sdpa
    kv_len, nq, heads, hk, rows, mask = ATTEND[i]
    case = Case(fmt, kv_len, nq, heads, hk, rows, seed=100 + i)
    kv, batch, q = case.device()
    out = paged.attend(kv, batch, q, mask_of(mask))
    assert sdpa.device_status() == 0
    want, bound = case.expect(mask)
    check(out[: len(want)], want, bound, f"{fmt} {ATTEND[i]}")
    assert torch.equal(out, paged.attend(kv, batch, q, mask_of(mask)))  # the same bits again


# Work for the long-chunk kernel: ragged, cut across CTAs, parts joined.
LARGE = [
    ([3000, 1111], [600, 300], 4, 2, 64, (1, 0, 0)),
    ([4000], [700], 5, 1, 16, (1, 1500, 6)),
    ([2600, 90, 2000], [500, 90, 1], 6, 2, 128, (40, 9, 1)),
    ([6000], [1300], 2, 2, 32, None),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("i", range(len(LARGE)))
def test_long_chunks_cut_and_joined(fvlib, fmt, i, monkeypatch):
    from fastvideo_rs_b200 import _lib, paged, sdpa
    monkeypatch.setenv("FV_PAGED_KERNEL", "items")
    kv_len, nq, heads, hk, rows, mask = LARGE[i]
    case = Case(fmt, kv_len, nq, heads, hk, rows, seed=200 + i)
    kv, batch, q = case.device()
    out = paged.attend(kv, batch, q, mask_of(mask))
    assert "fv_paged_chunk_kernel" in _lib.last_kernel()
    assert sdpa.device_status() == 0
    want, bound = case.expect(mask)
    check(out, want, bound, f"{fmt} {LARGE[i]}")
    assert torch.equal(out, paged.attend(kv, batch, q, mask_of(mask)))


def test_which_kernel_runs(fvlib):
    from fastvideo_rs_b200 import _lib, paged
    for fmt in FMTS:
        for kv_len, nq, name in (([300], [1], "decode"), ([300], [60], "decode"), ([6000], [1300], "chunk")):
            kv, batch, q = Case(fmt, kv_len, nq, 4, 2, 64).device()
            paged.attend(kv, batch, q, mask_of((1, 0, 0)))
            assert f"fv_paged_{name}_kernel<{'4 bits' if fmt == 'q4' else 'bf16'}" in _lib.last_kernel()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("i", [2, 3, 7, 8, 12, 16, 19])
def test_memory_that_no_row_sees_has_no_influence(fvlib, kernel, fmt, i):
    """Rows behind the sequences, unused pages and pages outside of the window hold NaN or are given back."""
    from fastvideo_rs_b200 import paged, sdpa
    kv_len, nq, heads, hk, rows, mask = ATTEND[i]
    case = Case(fmt, kv_len, nq, heads, hk, rows, seed=100 + i, poison=True, drop=mask)
    for s, (n, m) in enumerate(zip(kv_len, nq)):  # keys that no row sees, in pages that others need
        hidden = (~seen_matrix(m, n, mask).any(0)).nonzero().flatten()
        page = case.table[s].long()[hidden // rows]
        live = page >= 0
        for name in ("k", "v"):
            (case.pool if fmt == "bf16" else case.scales)[name][page[live], :, (hidden % rows)[live]] = math.nan
    kv, batch, q = case.device()
    out = paged.attend(kv, batch, q, mask_of(mask))
    assert sdpa.device_status() == 0
    case2 = Case(fmt, kv_len, nq, heads, hk, rows, seed=100 + i, poison=True)
    want, bound = case2.expect(mask)
    check(out[: len(want)], want, bound, f"{fmt} {ATTEND[i]}")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("nq,heads", [(1, 8), (200, 4)])
def test_large_scores_move_the_reference(fvlib, kernel, fmt, nq, heads):
    """Scores that grow along the keys by far more than the softmax's guard: every tile outgrows the reference."""
    from fastvideo_rs_b200 import paged
    case = Case(fmt, [400], [nq], heads, 2, 16, seed=7)
    case.q = (case.q.float() * 30).to(torch.bfloat16)
    kv, batch, q = case.device()
    want, bound = case.expect((1, 0, 0))
    # (scores of several hundred: 128 products in f32 are off by about 2^-24 of the sum of their sizes, 2^-13 in the exponent)
    check(paged.attend(kv, batch, q, mask_of((1, 0, 0))), want, bound + 2.0 ** -9 * bound / BF16_HALF, fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_small_values_of_few_keys(fvlib, kernel, fmt):
    """Two and three keys: here single values near zero meet weights of one half, and nothing averages an error out."""
    from fastvideo_rs_b200 import paged
    for seed in range(40):
        case = Case(fmt, [15, 2, 3, 3], [15, 2, 3, 3], 8, 1, 64, seed=1000 + seed)
        kv, batch, q = case.device()
        want, bound = case.expect(None)
        check(paged.attend(kv, batch, q), want, bound, f"{fmt} {seed}")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("nq", [3, 150])
def test_rows_before_the_sequence_are_zero(fvlib, kernel, fmt, nq):
    """More new tokens than the sequence holds: the first rows have no position and see nothing."""
    from fastvideo_rs_b200 import paged, sdpa
    case = Case(fmt, [2], [nq], 4, 2, 16, seed=3)
    kv, batch, q = case.device()
    out = paged.attend(kv, batch, q, mask_of((1, 0, 0)))
    assert sdpa.device_status() == 0
    assert not out[: nq - 2].any() and out[nq - 2:].any()
    none = Case(fmt, [0, 5], [1, 1], 4, 2, 16, seed=3)
    kv, batch, q = none.device()
    out = paged.attend(kv, batch, q, mask_of((1, 0, 0)))
    assert not out[0].any() and out[1].any()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("nq", [1, 170])
def test_padded_batch_strides_stream_and_out(fvlib, kernel, fmt, nq):
    from fastvideo_rs_b200 import paged, sdpa
    case = Case(fmt, [500, 300], [nq, 1], 4, 2, 16, seed=5, pad=7)
    kv, batch, q = case.device()
    want, bound = case.expect((1, 64, 2))
    fused = torch.randn(case.tokens, 8 * D, device="cuda").to(torch.bfloat16)
    fused[:, 2 * D:6 * D] = q.flatten(1)
    view = fused[:, 2 * D:6 * D].view(case.tokens, 4, D)
    out = torch.full((case.tokens, 4, D), 3.0, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged.attend(kv, batch, view, mask_of((1, 64, 2)), out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert got is out and sdpa.device_status() == 0
    check(out[: nq + 1], want, bound, fmt)
    assert bool((out[nq + 1:] == 3.0).all())  # rows behind the last sequence stay as they were
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)  # another order of tokens and heads
    assert torch.equal(paged.attend(kv, batch, heads_first, mask_of((1, 64, 2)))[: nq + 1], out[: nq + 1])


@pytest.mark.parametrize("fmt", FMTS)
def test_scale_argument(fvlib, kernel, fmt):
    from fastvideo_rs_b200 import paged
    case = Case(fmt, [333], [20], 4, 2, 16, seed=6)
    kv, batch, q = case.device()
    want, bound = case.expect((1, 0, 0), scale=0.02)
    check(paged.attend(kv, batch, q, mask_of((1, 0, 0)), scale=0.02), want, bound, fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("nq", [1, 140])
def test_captured_call_follows_the_tables(fvlib, kernel, fmt, nq):
    """A captured call reads lengths, rows and tables anew at every replay, within the bounds it was captured with."""
    from fastvideo_rs_b200 import paged, sdpa
    a = Case(fmt, [900, 450], [nq, 1], 4, 2, 16, seed=8)
    kv, batch, q = a.device()
    paged.attend(kv, batch, q, mask_of((1, 0, 0)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.attend(kv, batch, q, mask_of((1, 0, 0)))
    for lens in ([900, 450], [nq + 1, 3], [640, 0]):
        batch.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert sdpa.device_status() == 0
        rows = {n: [x[:m] for x, m in zip(a.rows[n], lens)] for n in ("k", "v")}
        for s, m in enumerate(lens):
            o, mag = attend64(a.q[a.cu[s]:a.cu[s + 1]].double(), rows["k"][s], rows["v"][s], (1, 0, 0))
            room = BF16_HALF * o.abs() + (BF16_HALF + 2.0 ** -10) * (mag + (1.5 if fmt == "q4" else 0.0)) + 1e-30
            check(out[a.cu[s]:a.cu[s + 1]], o, room, f"{fmt} {lens}")


def tables(rows, pairing, seed=0):
    turn = 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * turn
    angle = angle.repeat_interleave(2, 1) if pairing == "interleaved" else angle.repeat(1, 2)
    return angle.cos().float(), angle.sin().float()


# (kv_len, nq, q_heads, kv_heads, page_rows, pad)
APPEND = [([1], [1], 1, 1, 16, 0), ([5], [5], 4, 4, 16, 2), ([777], [33], 12, 12, 64, 0), ([40, 17, 300, 0], [1, 17, 130, 0], 40, 8, 32, 5),
          ([4000], [4000], 3, 1, 256, 0), (list(range(1, 41)), [1] * 40, 8, 2, 16, 3), ([3], [6], 2, 2, 16, 0)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("pairing", ["interleaved", "half"])
@pytest.mark.parametrize("i", range(len(APPEND)))
def test_append_and_read_are_the_formula_bit_for_bit(fvlib, fmt, pairing, i):
    from fastvideo_rs_b200 import paged, sdpa
    kv_len, nq, heads, hk, rows, pad = APPEND[i]
    case = Case(fmt, kv_len, nq, heads, hk, rows, seed=50 + i, pad=pad)
    kv, batch, _ = case.device()
    before = {n: t.clone() for n, t in (("k", kv.k), ("v", kv.v))}
    g = torch.Generator().manual_seed(i)
    proj = torch.randn(case.tokens, (heads + 2 * hk) * D, generator=g).to(torch.bfloat16)
    cos, sin = tables(max(case.max_kv, 1), pairing)
    dev = proj.cuda()
    q, k, v = (x.view(case.tokens, -1, D) for x in dev.split([heads * D, hk * D, hk * D], 1))
    q_out = torch.full((case.tokens, heads, D), 5.0, dtype=torch.bfloat16, device="cuda")
    assert paged.append(kv, batch, k, v, q=q, cos=cos.cuda(), sin=sin.cuda(), pairing=pairing, q_out=q_out) is q_out
    k_read, v_read = paged.read(kv, batch, rows=case.tokens)
    assert sdpa.device_status() == 0
    live = sum(nq)
    assert bool((q_out[live:] == 5.0).all()) and not k_read[live:].any() and not v_read[live:].any()
    hq, hkk, hv = (x.cpu() for x in (q, k, v))
    touched = {n: torch.zeros(case.pages, rows, dtype=torch.bool) for n in ("k", "v")}
    for s, (n, m) in enumerate(zip(kv_len, nq)):
        for x in range(m):
            t, p = int(case.cu[s]) + x, n - m + x
            if p < 0:
                assert not q_out[t].any() and not k_read[t].any()
                continue
            page, row = int(case.table[s, p // rows]), p % rows
            touched["k"][page, row] = touched["v"][page, row] = True
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(kv_len, nq)])
    ok = pos >= 0
    c, sn = cos[pos.clamp(min=0)][:, None], sin[pos.clamp(min=0)][:, None]
    want_q = rotate32(hq[:live], c, sn, pairing)
    assert torch.equal(q_out[:live].cpu()[ok], want_q.to(torch.bfloat16)[ok])
    # the definition in 64 bits: at most one rounding to bf16 of values off by 2^-22 of |x|
    far = (want_q.double() - rotate64(hq[:live].double(), c.double(), sn.double(), pairing)).abs()
    assert float(far.max()) <= 2.0 ** -22 * float(hq.double().abs().max())
    want_k = rotate32(hkk[:live], c, sn, pairing)
    for name, x, got in (("k", want_k, k_read), ("v", hv[:live].float(), v_read)):
        if fmt == "bf16":
            want = x.to(torch.bfloat16)
        else:
            codes, sc = quantize(x)
            want = stands_for(pack(codes), sc).to(torch.bfloat16)
        assert torch.equal(got[:live].cpu()[ok], want[ok]), name
    for name, now in (("k", kv.k), ("v", kv.v)):  # nothing else in the pool has moved
        same = (now == before[name]).flatten(3).all(-1).all(1).cpu() if fmt == "q4" else \
            (now.view(torch.int16) == before[name].view(torch.int16)).all(-1).all(1).cpu()
        assert bool(same[~touched[name]].all()), name


def test_append_without_rotation_and_by_positions(fvlib):
    from fastvideo_rs_b200 import paged, sdpa
    case = Case("bf16", [50], [20], 4, 2, 16, seed=1)
    kv, batch, q = case.device()
    k, v = (torch.randn(20, 2, D, device="cuda").to(torch.bfloat16) for _ in range(2))
    assert paged.append(kv, batch, k, v) is None
    a, b = paged.read(kv, batch, rows=20)
    assert torch.equal(a, k) and torch.equal(b, v)
    same = paged.append(kv, batch, k, v, q=q)
    assert torch.equal(same, q)
    cos, sin = tables(400, "interleaved")
    where = torch.randperm(400, generator=torch.Generator().manual_seed(2))[:20].to(torch.int32)
    got = paged.append(kv, batch, k, v, q=q, cos=cos.cuda(), sin=sin.cuda(), positions=where.cuda())
    c, s = cos[where.long()][:, None], sin[where.long()][:, None]
    assert torch.equal(got.cpu(), rotate32(q.cpu(), c, s, "interleaved").to(torch.bfloat16))
    assert torch.equal(paged.read(kv, batch, rows=20)[0].cpu(), rotate32(k.cpu(), c, s, "interleaved").to(torch.bfloat16))
    assert sdpa.device_status() == 0


def test_four_bit_rows_of_odd_values(fvlib):
    """Rows of one value, of tiny, huge and lopsided values: the format's own formula, and at most half a step off."""
    from fastvideo_rs_b200 import paged
    rows = torch.stack([torch.zeros(D), torch.full((D,), 3.5), torch.full((D,), -1e-30), torch.linspace(0, 1e-38, D),
                        torch.linspace(-3e38, 0, D), torch.linspace(1000, 1001, D), torch.cat([torch.full((1,), 900.0), torch.zeros(D - 1)])])
    rows = rows.to(torch.bfloat16)
    n = len(rows)
    case = Case("q4", [n], [n], 1, 1, 16, seed=1)
    kv, batch, _ = case.device()
    x = rows.cuda()[:, None]
    paged.append(kv, batch, x, x)
    k, v = paged.read(kv, batch, rows=n)
    codes, sc = quantize(rows.float())
    assert torch.equal(k[:, 0].cpu(), stands_for(pack(codes), sc).to(torch.bfloat16)) and torch.equal(k, v)
    ordinary = quantize(torch.randn(500, D, generator=torch.Generator().manual_seed(0)))
    x = torch.randn(500, D, generator=torch.Generator().manual_seed(0))
    step = ordinary[1][:, :1].double()
    # half a step, and at the ends what the roundings of step (2^-8 of 15 steps) and zero (2^-8 of about 8 steps) add
    assert bool(((stands_for(pack(ordinary[0]), ordinary[1]) - x.double()).abs() <= step * (0.5 + 15 * BF16_HALF + 0.1)).all())


@pytest.mark.parametrize("fmt", FMTS)
def test_reading_whole_sequences_and_ranges(fvlib, fmt):
    from fastvideo_rs_b200 import paged, sdpa
    case = Case(fmt, [70, 0, 33], [1, 0, 1], 4, 2, 16, seed=4)
    kv, batch, _ = case.device()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    k, v = paged.read(kv, batch, rows=105, cu_rows=i32([0, 70, 70, 103]), first=i32([0, 0, 0]))
    for name, got in (("k", k), ("v", v)):
        want = torch.cat([case.rows[name][0], case.rows[name][2], torch.zeros(2, 2, D, dtype=torch.float64)])
        assert torch.equal(got.cpu(), want.to(torch.bfloat16)), name
    k, _ = paged.read(kv, batch, rows=9, cu_rows=i32([0, 4, 6, 9]), first=i32([-2, 0, 32]))  # rows that are not there: zero
    assert not k[:2].any() and torch.equal(k[2:4].cpu(), case.rows["k"][0][:2].to(torch.bfloat16)) and not k[4:6].any()
    assert torch.equal(k[6].cpu(), case.rows["k"][2][32].to(torch.bfloat16)) and not k[7:].any()
    assert sdpa.device_status() == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_streaming_run_equals_one_chunk(fvlib, kernel, fmt):
    """A prompt and then single tokens, appended and attended to step by step under a sliding window with sinks whose pages
    are given back as it slides, against the formula over everything that was appended."""
    from fastvideo_rs_b200 import paged, sdpa
    from fastvideo_rs_b200.sdpa import BlockCausal
    heads, hk, rows, total, prompt = 8, 2, 16, 150, 70
    mask = (1, 40, 5)
    g = torch.Generator().manual_seed(9)
    proj = torch.randn(total, (heads + 2 * hk) * D, generator=g).to(torch.bfloat16).cuda()
    q, k, v = (x.view(total, -1, D) for x in proj.split([heads * D, hk * D, hk * D], 1))
    cos, sin = (t.cuda() for t in tables(total, "half"))
    kv = paged.PagedKv.empty(8, rows, hk, fmt)
    free = list(range(7, -1, -1))
    table = torch.full((1, (total + rows - 1) // rows), -1, dtype=torch.int32)
    outs, at = [], 0
    kept = {}
    for n in [prompt] + [1] * (total - prompt):
        end = at + n
        for i in range(at // rows, (end + rows - 1) // rows):
            if table[0, i] < 0:
                table[0, i] = free.pop()
        batch = paged.PagedBatch(table.cuda(), torch.tensor([end], dtype=torch.int32).cuda(),
                                 torch.tensor([0, n], dtype=torch.int32).cuda(), max_q=n, max_kv=end)
        qr = paged.append(kv, batch, k[at:end], v[at:end], q=q[at:end], cos=cos, sin=sin, pairing="half")
        kr, vr = paged.read(kv, batch, rows=n)
        for p in range(at, end):
            kept[p] = (kr[p - at].cpu(), vr[p - at].cpu(), qr[p - at].cpu())
        outs.append(paged.attend(kv, batch, qr, BlockCausal(*mask)))
        at = end
        for i in range(table.shape[1]):  # pages that no later token sees
            if table[0, i] >= 0 and i * rows >= mask[2] and (i + 1) * rows <= at - mask[1] + 1:
                free.append(int(table[0, i]))
                table[0, i] = -1
    assert sdpa.device_status() == 0
    got = torch.cat(outs)
    ks, vs, qs = (torch.stack([kept[p][i] for p in range(total)]).double() for i in range(3))
    want, mag = attend64(qs, ks, vs, mask)
    # (4 bits: kept holds the values rounded to bf16 once more, 2^-8 of K in the scores: about 2^-8 |q| |k| / 11.3 < 0.04)
    room = (BF16_HALF * want.abs() + (BF16_HALF + 2.0 ** -10) * (mag + 1.5)) * (1 if fmt == "bf16" else 4) + (0 if fmt == "bf16" else 0.05 * mag)
    check(got, want, room, fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_wan_layer_streams_over_pages(fvlib, fmt):
    """WanSelfAttention.forward_paged block by block of frames, two rollouts of different lengths packed, under a window of
    blocks with a sink block, against norm, rotation and attention in 64 bits on what the cache was given."""
    from fastvideo_rs_b200 import paged, sdpa, wan
    from fastvideo_rs_b200.sdpa import BlockCausal
    heads, frame, frames = 3, 20, 7
    mask = (frame, 3, 1)
    g = torch.Generator().manual_seed(12)
    w = [1 + 0.1 * torch.randn(heads * D, generator=g) for _ in range(2)]
    layer = wan.WanSelfAttention((frames, 4, 5), heads, w[0].cuda(), w[1].cuda(), causal=BlockCausal(*mask))
    cos, sin = layer.cos.cpu().double(), layer.sin.cpu().double()
    qkv = torch.randn(2, frames * frame, 3 * heads * D, generator=g).to(torch.bfloat16)
    kv = paged.PagedKv.empty(24, 16, heads, fmt)
    table = torch.randperm(24, generator=g).to(torch.int32)[:18].view(2, 9).contiguous()
    have, seen = [0, 0], [[], []]
    for step in range(frames):
        new = [frame, frame if step % 2 == 0 else 0]  # the second rollout advances every other step
        rows = [qkv[s, have[s]:have[s] + new[s]] for s in range(2)]
        have = [a + b for a, b in zip(have, new)]
        cu = torch.tensor([0, new[0], new[0] + new[1]], dtype=torch.int32)
        batch = paged.PagedBatch(table.cuda(), torch.tensor(have, dtype=torch.int32).cuda(), cu.cuda(), max_q=frame, max_kv=max(have))
        out = layer.forward_paged(torch.cat(rows)[None].cuda(), kv, batch)
        assert out.shape == (sum(new), heads, D)
        kr, vr = (t.double().cpu() for t in paged.read(kv, batch, rows=sum(new)))
        for s in range(2):
            if not new[s]:
                continue
            part = slice(int(cu[s]), int(cu[s + 1]))
            x = rows[s].double().view(new[s], 3, heads * D)
            norm = [(y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6) * w[i].double()).view(-1, heads, D) for i, y in ((0, x[:, 0]), (1, x[:, 1]))]
            at = slice(have[s] - new[s], have[s])
            c, sn = cos[at][:, None], sin[at][:, None]
            q64, k64 = (rotate64(y, c, sn, "interleaved") for y in norm)
            if fmt == "bf16":  # two roundings to bf16, of values no larger than sqrt(2) of a pair's larger one
                assert float((kr[part] - k64).abs().max()) <= 2.0 * math.sqrt(2.0) * BF16_HALF * float(norm[1].abs().max())
                assert torch.equal(vr[part], x[:, 2].view(-1, heads, D))
            seen[s].append((kr[part], vr[part]))
            ks, vs = (torch.cat([t[i] for t in seen[s]]) for i in range(2))
            want, mag = attend64(q64, ks, vs, mask)
            # q is off by two roundings as well: each score by at most 2 sqrt(2) 2^-8 |q| |k| / sqrt(128), P by as much relatively;
            # 4 bits: read() rounds K and V to bf16 once more, and P's products' zeros come on top (|zero| <= 1.5)
            off = 2.0 * math.sqrt(2.0) * BF16_HALF * float(q64.norm(dim=-1).max() * ks.norm(dim=-1).max()) / math.sqrt(D)
            off = off * (1.0 if fmt == "bf16" else 2.0)
            check(out[part], want, BF16_HALF * want.abs() + (2 * BF16_HALF + off) * (mag + (1.5 if fmt == "q4" else 0.0)), f"{fmt} step {step} rollout {s}")
    assert sdpa.device_status() == 0


def test_rows_past_four_gigabytes(fvlib, kernel):
    """Pages whose byte offsets pass 32 bits."""
    from fastvideo_rs_b200 import paged, sdpa
    pages, rows = 70000, 256
    kv = paged.PagedKv.empty(pages, rows, 1)
    table = torch.tensor([[69999, 33000, 2]], dtype=torch.int32).cuda()
    n = 600
    batch = paged.PagedBatch(table, torch.tensor([n], dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(), max_q=n, max_kv=n)
    x = torch.randn(3, n, 1, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    q, k, v = x.cuda()
    paged.append(kv, batch, k, v)
    out = paged.attend(kv, batch, q, mask_of((1, 0, 0)))
    assert sdpa.device_status() == 0
    want, mag = attend64(x[0].double(), x[1].double(), x[2].double(), (1, 0, 0))
    check(out, want, BF16_HALF * want.abs() + (BF16_HALF + 2.0 ** -10) * mag, "far pages")


@pytest.mark.parametrize("nq", [1, 150])
def test_broken_tables_are_reported_and_not_followed(fvlib, kernel, nq):
    from fastvideo_rs_b200 import FvError, paged, sdpa
    mask = mask_of((1, 0, 0))
    case = Case("bf16", [400, 200], [nq, 1], 4, 2, 16, seed=11)
    kv, batch, q = case.device()
    good = paged.attend(kv, batch, q, mask)

    def reported(code):
        with pytest.raises(FvError, match=f"status {code}"):
            sdpa.device_status()
        assert sdpa.device_status() == 0

    for bad in (-1, case.pages, 1 << 30):
        batch.page_table[0, 3] = bad
        out = paged.attend(kv, batch, q, mask)
        reported(200)
        assert torch.equal(out[nq], good[nq])  # the other sequence is untouched
    batch.page_table[0, 3] = int(case.table[0, 3])
    k = torch.randn(case.tokens, 2, D, device="cuda").to(torch.bfloat16)
    batch.page_table[1, 199 // 16] = -5
    paged.append(kv, batch, k, k)
    reported(200)
    batch.page_table.copy_(case.table)
    paged.append(kv, batch, k, k, cos=torch.ones(100, D, device="cuda"), sin=torch.zeros(100, D, device="cuda"))
    reported(202)
    for t, i, x in ((batch.kv_len, 0, 401), (batch.kv_len, 0, -3), (batch.cu_q, 1, -1), (batch.cu_q, 2, 10 ** 6)):
        old = int(t[i])
        t[i] = x
        paged.attend(kv, batch, q, mask)
        reported(201)
        t[i] = old
    assert torch.equal(paged.attend(kv, batch, q, mask)[nq], good[nq])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("nq", [1, 150])
@pytest.mark.parametrize("kv_len", [400, 9000])
def test_a_query_that_is_not_a_number_stays_one(fvlib, kernel, fmt, nq, kv_len):
    """A NaN in q reaches its own row and no other, however many parts the row's keys are cut into."""
    from fastvideo_rs_b200 import paged
    case = Case(fmt, [kv_len], [nq], 4, 2, 64, seed=12)
    kv, batch, q = case.device()
    want, bound = case.expect((1, 0, 0))
    q[nq // 2, 1] = math.nan
    q[nq - 1, 2, 5] = math.nan
    out = paged.attend(kv, batch, q, mask_of((1, 0, 0)))
    bad = torch.zeros(nq, 4, dtype=torch.bool, device="cuda")
    bad[nq // 2, 1] = bad[nq - 1, 2] = True
    assert bool(out[bad].isnan().all())
    good = ~bad.cpu()
    check(out[~bad], want[good], bound[good], fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("nq", [1, 150])
@pytest.mark.parametrize("kv_len", [700, 9000])
def test_out_may_be_q(fvlib, kernel, fmt, nq, kv_len):
    from fastvideo_rs_b200 import paged
    case = Case(fmt, [kv_len, 300], [nq, 3], 8, 2, 32, seed=13)
    kv, batch, q = case.device()
    cos, sin = (t.cuda() for t in tables(kv_len, "half"))
    k = torch.randn(case.tokens, 2, D, device="cuda").to(torch.bfloat16)
    want_q = paged.append(kv, batch, k, k, q=q, cos=cos, sin=sin, pairing="half")
    want = paged.attend(kv, batch, want_q, mask_of((1, 0, 0)))
    assert paged.append(kv, batch, k, k, q=q, cos=cos, sin=sin, pairing="half", q_out=q) is q
    assert torch.equal(q, want_q)
    assert paged.attend(kv, batch, q, mask_of((1, 0, 0)), out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("nq", [1, 150])
def test_one_batch_serves_pools_of_both_formats(fvlib, kernel, nq):
    """Layers of both formats in turn, whose calls need scratch of different sizes, and bounds far above what the call holds."""
    from fastvideo_rs_b200 import paged
    b, c = (Case(fmt, [20011], [nq], 4, 1, 64, seed=14) for fmt in FMTS)
    kv, batch, q = b.device()
    kv4, batch4, q4 = c.device()
    wants = paged.attend(kv, batch, q, mask_of((1, 0, 0))), paged.attend(kv4, batch4, q4, mask_of((1, 0, 0)))
    batch4.page_table.copy_(batch.page_table)  # (both pools are laid out alike)
    assert torch.equal(b.table, c.table)
    wide = paged.PagedBatch(batch.page_table, batch.kv_len, batch.cu_q, max_q=(1 << 30) - 1, max_kv=20011)
    for shared in (batch, wide):
        for _ in range(2):
            assert torch.equal(paged.attend(kv, shared, q, mask_of((1, 0, 0))), wants[0])
            assert torch.equal(paged.attend(kv4, shared, q4, mask_of((1, 0, 0))), wants[1])


@pytest.mark.parametrize("fmt", FMTS)
def test_two_streams_at_once(fvlib, kernel, fmt):
    """Calls in flight side by side share no scratch."""
    from fastvideo_rs_b200 import paged, sdpa
    cases = [Case(fmt, [9000, 400], [nq, 2], 8, 2, 64, seed=15 + nq) for nq in (1, 200)]
    on = [c.device() for c in cases]
    wants = [paged.attend(kv, batch, q, mask_of((1, 0, 0))) for kv, batch, q in on]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in on]
    outs = [[], []]
    for _ in range(10):
        for i, (kv, batch, q) in enumerate(on):
            with torch.cuda.stream(streams[i]):
                outs[i].append(paged.attend(kv, batch, q, mask_of((1, 0, 0))))
    torch.cuda.synchronize()
    assert sdpa.device_status() == 0
    for want, got in zip(wants, outs):
        assert all(torch.equal(want, x) for x in got)


@pytest.mark.parametrize("fmt", FMTS)
def test_captured_steps_of_append_and_attend(fvlib, kernel, fmt):
    """A step of two layers -- append, attend, twice -- captured once and replayed for token after token, beside a second graph of the
    same step, equals the calls made one by one."""
    from fastvideo_rs_b200 import paged, sdpa
    heads, hk, rows, total, mask = 8, 2, 16, 40, mask_of((1, 20, 3))
    g = torch.Generator().manual_seed(16)
    proj = torch.randn(2, total, heads + 2 * hk, D, generator=g).to(torch.bfloat16).cuda()
    cos, sin = (t.cuda() for t in tables(total, "interleaved"))
    table = torch.arange((total + rows - 1) // rows, dtype=torch.int32, device="cuda")[None]
    mk = lambda: [paged.PagedKv.empty(table.shape[1], rows, hk, fmt) for _ in range(2)]
    batch = paged.PagedBatch(table, torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                             max_q=1, max_kv=total)
    token = torch.empty(2, 1, heads + 2 * hk, D, dtype=torch.bfloat16, device="cuda")

    def step(pools):
        outs = []
        for kv, x in zip(pools, token):
            q, k, v = x.split([heads, hk, hk], 1)
            outs.append(paged.attend(kv, batch, paged.append(kv, batch, k, v, q=q, cos=cos, sin=sin), mask))
        return torch.stack(outs)

    plain = mk()
    want = []
    for t in range(total):
        batch.kv_len.fill_(t + 1)
        token.copy_(proj[:, t:t + 1])
        want.append(step(plain))
    graphs = []
    for _ in range(2):
        pools, graph = mk(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(pools)
        graphs.append((pools, graph, out))
    for t in range(total):
        batch.kv_len.fill_(t + 1)
        token.copy_(proj[:, t:t + 1])
        for pools, graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for pools, graph, out in graphs:
            assert torch.equal(out, want[t])
    assert sdpa.device_status() == 0


def test_refusals(fvlib):
    from fastvideo_rs_b200 import FvError, paged
    from fastvideo_rs_b200.sdpa import BlockCausal
    case = Case("bf16", [40], [4], 4, 2, 16)
    kv, batch, q = case.device()
    k = torch.zeros(4, 2, D, dtype=torch.bfloat16, device="cuda")
    cos = torch.zeros(50, D, device="cuda")
    with pytest.raises(ValueError, match="heads over"):
        paged.attend(kv, batch, q[:, :3])
    with pytest.raises(ValueError, match="bfloat16"):
        paged.attend(kv, batch, q.float())
    with pytest.raises(ValueError, match="CUDA"):
        paged.attend(kv, batch, q.cpu())
    with pytest.raises(FvError, match="scale"):
        paged.attend(kv, batch, q, scale=-1.0)
    with pytest.raises(FvError, match="block_tokens"):
        paged.attend(kv, batch, q, BlockCausal(0, 1, 1))
    with pytest.raises(ValueError, match="range"):
        paged.attend(kv, batch, q, BlockCausal(1, -1, 1))
    with pytest.raises(ValueError, match="range"):
        paged.attend(kv, batch, q, BlockCausal(1, 1 << 31, 1))
    with pytest.raises(FvError, match="positive"):
        paged.attend(kv, batch, q[:1].expand(4, 4, D))
    with pytest.raises(FvError, match="aligned|multiples"):
        paged.attend(kv, batch, torch.zeros(4 * 4 * 132 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(4, 4, 132)[..., :128])
    with pytest.raises(ValueError, match="out must be"):
        paged.attend(kv, batch, q, out=torch.zeros(4, 8, D, dtype=torch.bfloat16, device="cuda")[:, :4])
    with pytest.raises(ValueError, match="go together"):
        paged.append(kv, batch, k, k, cos=cos)
    with pytest.raises(ValueError, match="float32"):
        paged.append(kv, batch, k, k, cos=cos, sin=cos.half())
    with pytest.raises(ValueError, match="pairing"):
        paged.append(kv, batch, k, k, pairing="both")
    with pytest.raises(ValueError, match="wanted"):
        paged.append(kv, batch, k, k[:3])
    with pytest.raises(ValueError, match="wanted"):
        paged.append(kv, batch, k[:, :1], k)
    with pytest.raises(ValueError, match="int32"):
        paged.append(kv, batch, k, k, cos=cos, sin=cos, positions=torch.zeros(4, dtype=torch.int64, device="cuda"))
    with pytest.raises(FvError, match="does not hold"):
        short = paged.PagedBatch(batch.page_table, batch.kv_len, batch.cu_q, max_q=4, max_kv=49)
        paged.attend(kv, short, q)
    # empty calls do nothing
    assert paged.attend(kv, batch, q[:0]).shape == (0, 4, D)
    paged.append(kv, batch, k[:0], k[:0])
    assert paged.read(kv, batch, rows=0)[0].shape == (0, 2, D)
    nobody = paged.PagedBatch(torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"),
                              torch.zeros(1, dtype=torch.int32, device="cuda"), max_q=1, max_kv=1)
    out = torch.full_like(q, 2.0)
    assert bool((paged.attend(kv, nobody, q, out=out) == 2.0).all())
    assert not paged.read(kv, nobody, rows=3)[0].any()
