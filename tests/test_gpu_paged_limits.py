"""The paged K/V cache at the ends of its ranges: values and rows far from one, tables and bounds at their ends, masks counted
key by key.  Tolerances count roundings (tests/_paged.py, and beside each test where they differ)."""
import ctypes
import math

import pytest
import torch

from _paged import D, BF16_HALF, Case, attend64, pack, rotate64, unpack

pytestmark = pytest.mark.gpu

FMTS = ["bf16", "q4"]
F16_HALF = torch.finfo(torch.float16).eps / 2


@pytest.fixture(params=["rows", "items"])
def kernel(request, monkeypatch):
    monkeypatch.setenv("FV_PAGED_KERNEL", request.param)
    return request.param


def mask_of(mask):
    from fastvideo_rs_b200.sdpa import BlockCausal
    return None if mask is None else BlockCausal(*mask)


def check(got, want, bound, what):
    assert torch.isfinite(got).all(), what
    err = (got.double().cpu() - want).abs()
    worst = float((err / bound).max()) if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound, max-abs {float(err.max()):.3e}"


# ---- the Wan layer over pages -----------------------------------------------------------------------------------------

def _stream(layer, qkv, frame, fmt, heads, loose=0):
    """The frames of qkv one after the other through layer.forward_paged; [tokens, heads, 128]."""
    from fastvideo_rs_b200 import paged
    total = qkv.shape[1]
    kv = paged.PagedKv.empty((total + 15) // 16, 16, heads, fmt)
    table = torch.arange((total + 15) // 16, dtype=torch.int32, device="cuda")[None]
    outs = []
    for end in range(frame, total + 1, frame):
        i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
        batch = paged.PagedBatch(table, i32(end), i32(0, frame), max_q=frame, max_kv=max(end, loose))
        outs.append(layer.forward_paged(qkv[:, end - frame:end].contiguous(), kv, batch))
    return torch.cat(outs)


@pytest.mark.parametrize("fmt", FMTS)
def test_wan_layer_streams_past_its_grid(fvlib, fmt):
    """Rollouts longer than the layer's grid: the same bits as from a layer whose grid holds them."""
    from fastvideo_rs_b200 import sdpa, wan
    from fastvideo_rs_b200.sdpa import BlockCausal
    heads, frame, frames = 2, 20, 7
    g = torch.Generator().manual_seed(21)
    w = [(1 + 0.1 * torch.randn(heads * D, generator=g)).cuda() for _ in range(2)]
    qkv = torch.randn(1, frames * frame, 3 * heads * D, generator=g).to(torch.bfloat16).cuda()
    mk = lambda n: wan.WanSelfAttention((n, 4, 5), heads, *w, causal=BlockCausal(frame, 3, 1))
    want = _stream(mk(frames), qkv, frame, fmt, heads)
    got = _stream(mk(2), qkv, frame, fmt, heads)
    assert sdpa.device_status() == 0
    assert torch.equal(got, want)
    # a bound above the grid with lengths inside it
    short = qkv[:, :2 * frame].contiguous()
    assert torch.equal(_stream(mk(2), short, frame, fmt, heads, loose=48), _stream(mk(frames), short, frame, fmt, heads, loose=48))


def test_longer_tables_are_not_made_while_a_graph_is_captured(fvlib):
    from fastvideo_rs_b200 import paged, wan
    w = torch.ones(2 * D, device="cuda")
    layer = wan.WanSelfAttention((1, 4, 5), 2, w, w)
    kv = paged.PagedKv.empty(4, 16, 2)
    kv.k.zero_(), kv.v.zero_()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    batch = paged.PagedBatch(i32(0, 1, 2)[None].contiguous(), i32(30), i32(0, 10), max_q=10, max_kv=30)
    qkv = torch.randn(1, 10, 6 * D, device="cuda").to(torch.bfloat16)
    layer_ready = wan.WanSelfAttention((1, 4, 5), 2, w, w)
    want = layer_ready.forward_paged(qkv, kv, batch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="captur"):
            layer.forward_paged(qkv, kv, batch)
        got = layer_ready.forward_paged(qkv, kv, batch)
    graph.replay()
    assert torch.equal(got, want)


# ---- the 4-bit format -------------------------------------------------------------------------------------------------

def quantize_rows(x):
    """(codes 0..15 uint8, (step, zero) bf16) of f32 rows, with the step widened where the rounding of zero asks for it."""
    lo, hi = x.amin(-1), x.amax(-1)
    step = ((hi - lo) / torch.full_like(hi, 15.0)).to(torch.bfloat16).float()
    mid = lo + 8.0 * step
    zero = mid.to(torch.bfloat16).float()
    wide = torch.maximum((hi - zero) / torch.full_like(hi, 7.0), (zero - lo) * 0.125)
    wide = ((wide.view(torch.int32) + 0xffff) & -65536).view(torch.float32)  # up to the next bf16
    step = torch.where((zero - mid).abs() > 0.25 * step, wide, step)
    c = torch.round((x - zero[..., None]) / step[..., None]).clamp(-8, 7)
    c = torch.where(step[..., None] > 0, c, torch.zeros_like(c))
    return (c + 8).to(torch.uint8), torch.stack([step, zero], -1).to(torch.bfloat16)


def _offset_rows():
    g = torch.Generator().manual_seed(30)
    rows = [torch.tensor([1000.0, 1004.0] * 64), torch.tensor([1000.0, 1004.0, 1008.0, 1000.0] * 32),
            torch.tensor([-1000.0] * 127 + [-996.0]), torch.full((D,), 1000.0), torch.zeros(D), torch.tensor([256.0, 258.0] * 64)]
    for _ in range(500):  # an offset of up to 2^14 ranges, either sign
        span, off = 2.0 ** float(torch.rand((), generator=g) * 20 - 10), 2.0 ** float(torch.rand((), generator=g) * 14)
        rows.append(span * (torch.randn(D, generator=g) + (off if len(rows) % 2 else -off)))
    for _ in range(100):
        rows.append(torch.randn(D, generator=g))
    return torch.stack(rows).to(torch.bfloat16)


def test_four_bit_rows_with_an_offset_read_back_within_half_a_step(fvlib):
    """The codes span the row whatever its offset is: no value is more than half a step off, and the step is no larger than the
    range and the roundings of zero and step make it."""
    from fastvideo_rs_b200 import paged
    x = _offset_rows()
    n = len(x)
    kv = paged.PagedKv.empty((n + 15) // 16, 16, 1, "q4")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    batch = paged.PagedBatch(torch.arange((n + 15) // 16, dtype=torch.int32, device="cuda")[None], i32(n), i32(0, n), max_q=n, max_kv=n)
    # K through a rotation whose f32 results are no bf16 values, V as it is
    turn = torch.linspace(0, 3, n)[:, None] * torch.ones(D)
    cos, sin = turn.cos(), turn.sin()
    paged.append(kv, batch, x.cuda()[:, None], x.cuda()[:, None], cos=cos.cuda(), sin=sin.cuda())
    turned = torch.empty(n, D)
    xf = x.float()
    turned[:, 0::2] = xf[:, 0::2] * cos[:, 0::2] - xf[:, 1::2] * sin[:, 0::2]
    turned[:, 1::2] = xf[:, 0::2] * sin[:, 0::2] + xf[:, 1::2] * cos[:, 0::2]
    for name, rows in (("v", xf), ("k", turned)):
        codes = unpack(getattr(kv, name).cpu()[:, 0].flatten(0, 1)[:n])
        scale = getattr(kv, name + "_scale").cpu()[:, 0].flatten(0, 1)[:n]
        want_codes, want_scale = quantize_rows(rows)
        assert torch.equal(scale, want_scale) and torch.equal(codes, want_codes), name
        step, zero = scale[:, :1].double(), scale[:, 1:].double()
        r = rows.double()
        off = (zero + step * (codes.double() - 8.0) - r).abs()
        # half a step; f32: the subtraction of zero 2^-24 of the difference, the quotient 2^-24 of up to 8 steps
        assert bool((off <= step * (0.5 + 2.0 ** -19)).all()), (name, float((off / step.clamp(min=1e-30)).max()))
        span, most = r.amax(-1) - r.amin(-1), r.abs().amax(-1)
        # (zero is 2^-8 of at most max |x| + a step off; step is rounded once, or up: 2^-7; three f32 roundings)
        assert bool((step[:, 0] <= (1 + 2.0 ** -6) * (span / 15 + BF16_HALF * (most + span / 15) / 7) + 1e-30).all()), name
    k, v = paged.read(kv, batch, rows=n)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()


# ---- 4-bit values far from one ----------------------------------------------------------------------------------------

def _scaled(case, name, power):
    """Every row of `name` times 2^power[s][j] (power: a number, or per sequence and key), exactly."""
    for s, n in enumerate(case.kv_len):
        p = power if not torch.is_tensor(power) else power[:n]
        f = 2.0 ** (p * torch.ones(n, dtype=torch.float64))
        case.rows[name][s] = case.rows[name][s] * f[:, None, None]
        j = torch.arange(n)
        page, row = case.table[s].long()[j // case.page_rows], j % case.page_rows
        case.scales[name][page, :, row] = (case.scales[name][page, :, row].double() * f[:, None, None]).to(torch.bfloat16)


@pytest.mark.parametrize("powers", [(0, 0, -24), (0, 0, 18), (0, 0, -60), (0, 0, 100), (20, -20, 0), (-18, 18, 0), (-40, 40, 30), (60, -60, -40), (-20, 0, -20)])
@pytest.mark.parametrize("nq,kv_len,mask", [(1, 700, (1, 0, 0)), (150, 700, (1, 0, 0)), (150, 1500, (1, 300, 5)), (40, 333, None)])
def test_four_bit_values_of_any_size(fvlib, kernel, powers, nq, kv_len, mask):
    """q, K and V times powers of two: what the f16 products of long chunks hold is a matter of the kernel, not of the caller."""
    from fastvideo_rs_b200 import paged, sdpa
    case = Case("q4", [kv_len, 90], [nq, 5], 4, 2, 16, seed=40)
    pq, pk, pv = powers
    case.q = (case.q.double() * 2.0 ** pq).to(torch.bfloat16)
    _scaled(case, "k", pk)
    _scaled(case, "v", pv)
    kv, batch, q = case.device()
    out = paged.attend(kv, batch, q, mask_of(mask))
    assert sdpa.device_status() == 0
    want, bound = case.expect(mask)
    check(out, want, bound, f"{powers} {nq} {kv_len}")


def test_four_bit_values_of_every_size_in_one_call(fvlib, kernel):
    """Keys whose V is of another size every 128 keys, from 2^-40 to 2^40."""
    from fastvideo_rs_b200 import paged, sdpa
    for seed, runs in enumerate(([0, -40, 40], [40, 0, -40, 0], [-12, 12, -7, 7, 17, -20], [3, -3])):
        n = 1400
        case = Case("q4", [n, 600], [200, 3], 4, 2, 32, seed=50 + seed)
        p = torch.tensor(runs, dtype=torch.float64).repeat_interleave(128).repeat(n)[:n]
        _scaled(case, "v", p)
        kv, batch, q = case.device()
        want, bound = case.expect((1, 0, 0))
        # (Case's bound adds the largest |zero| of all keys to the terms: here of the keys that carry the row's weights)
        per = []
        for s, (m, nq) in enumerate(zip(case.kv_len, case.nq)):
            qs = case.q[case.cu[s]:case.cu[s + 1]].double()
            j = torch.arange(m)
            page, row = case.table[s].long()[j // 32], j % 32
            sc = case.scales["v"][page, :, row].double()
            top = (sc[..., 1].abs() + 8 * sc[..., 0].abs())[..., None].expand(m, 2, D)
            per.append(attend64(qs, case.rows["k"][s], top, (1, 0, 0))[0])
        bound = BF16_HALF * want.abs() + (BF16_HALF + 2.0 ** -10) * torch.cat(per) + 1e-30
        out = paged.attend(kv, batch, q, mask_of((1, 0, 0)))
        assert sdpa.device_status() == 0
        check(out, want, bound, f"{runs}")


def test_rows_of_q_of_every_size(fvlib, kernel):
    from fastvideo_rs_b200 import paged
    case = Case("q4", [500], [140], 4, 2, 16, seed=60)
    p = torch.tensor([0, -30, 3, -9, 40, 0, -60, 1], dtype=torch.float64).repeat(70)
    case.q = case.q.double() * 2.0 ** torch.minimum(p, torch.tensor(1.0, dtype=torch.float64)).view(140, 4, 1)
    case.q = case.q.to(torch.bfloat16)
    kv, batch, q = case.device()
    want, bound = case.expect((1, 0, 0))
    check(paged.attend(kv, batch, q, mask_of((1, 0, 0))), want, bound, "rows")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("nq", [1, 150])
def test_an_infinite_query_is_not_a_number(fvlib, kernel, fmt, nq):
    """An infinity in q: the row is not a number (its scores are infinities of both signs), and no other row changes."""
    from fastvideo_rs_b200 import paged
    case = Case(fmt, [700], [nq], 4, 2, 64, seed=61)
    kv, batch, q = case.device()
    want, bound = case.expect((1, 0, 0))
    q[nq // 2, 1, 7] = math.inf
    q[nq - 1, 2, 5] = -math.inf
    out = paged.attend(kv, batch, q, mask_of((1, 0, 0)))
    bad = torch.zeros(nq, 4, dtype=torch.bool, device="cuda")
    bad[nq // 2, 1] = bad[nq - 1, 2] = True
    assert bool(out[bad].isnan().all())
    good = ~bad.cpu()
    check(out[~bad], want[good], bound[good], fmt)


def test_a_four_bit_row_that_is_not_finite_stands_for_nan(fvlib, kernel):
    """A row with an infinity was appended: whoever sees it gets what is not a number, other sequences nothing of it."""
    from fastvideo_rs_b200 import paged
    for which in ("k", "v"):
        for bad in (math.inf, -math.inf, math.nan):
            case = Case("q4", [300, 200], [140, 3], 4, 2, 16, seed=62)
            kv, batch, q = case.device()
            clean = paged.attend(kv, batch, q, mask_of((1, 0, 0)))
            x = torch.randn(case.tokens, 2, D, device="cuda").to(torch.bfloat16)
            y = x.clone()
            y[0, 1, 3] = bad  # the first token of the first sequence: key 160, which all 140 rows see
            paged.append(kv, batch, y if which == "k" else x, y if which == "v" else x)
            out = paged.attend(kv, batch, q, mask_of((1, 0, 0)))
            assert bool(out[:140, 2:].isnan().all()), (which, bad)
            assert not bool(out[140:].isnan().any()) and not bool(clean.isnan().any())


# ---- probabilities and masks, counted ---------------------------------------------------------------------------------

@pytest.mark.parametrize("heads", [2, 16])
def test_four_bit_probabilities_are_rounded_at_eleven_bits(fvlib, kernel, heads):
    """Scores and values that every product holds exactly, and outputs that nearly cancel: what is left is P's rounding, 2^-11."""
    from fastvideo_rs_b200 import paged
    g = torch.Generator().manual_seed(70)
    for n, nq in ((5, 5), (37, 20), (200, 70)):
        case = Case("q4", [n], [nq], heads, 1, 16, seed=70)
        codes = {"k": torch.full((n, 1, D), 8), "v": torch.randint(0, 16, (n, 1, D), generator=g)}
        codes["k"][:, 0, 0] = torch.randint(0, 16, (n,), generator=g)
        codes["v"][1::2] = (16 - codes["v"][0::2][: n // 2]).clamp(max=15)  # nearly the negative of the key before
        q = torch.zeros(nq, heads, D)
        q[..., 0] = torch.randint(1, 256, (nq, heads), generator=g) / 64.0
        case.q = q.to(torch.bfloat16)
        j = torch.arange(n)
        page, row = case.table[0].long()[j // 16], j % 16
        for name in ("k", "v"):
            case.pool[name][page, :, row] = pack(codes[name]).to(torch.uint8)
            case.scales[name][page, :, row] = torch.tensor([0.25, 0.0]).to(torch.bfloat16)
            case.rows[name] = [0.25 * (codes[name].double() - 8.0)]
        kv, batch, qd = case.device()
        out = paged.attend(kv, batch, qd, mask_of((1, 0, 0)))
        want, mag = attend64(case.q.double(), case.rows["k"][0], case.rows["v"][0], (1, 0, 0))
        # P: half a step of f16, 2^-11; the exponential and the f32 sums (scores up to 16: 2^-24 of them in the exponent, ex2 2^-22): 2^-15
        bound = BF16_HALF * want.abs() + (F16_HALF + 2.0 ** -15) * mag + 1e-30
        check(out, want, bound, f"{n}")


COUNTED = [([400], [1], (1, 0, 0)), ([400], [1], (1, 257, 0)), ([1031], [1], (1, 300, 5)), ([1031], [260], (1, 300, 5)), ([900], [333], (1, 129, 0)),
           ([777], [777], (1, 0, 0)), ([640], [160], (160, 2, 1)), ([1000], [129], (100, 2, 2)), ([515, 64], [3, 64], (7, 20, 3)), ([4100], [40], (1, 1000, 130))]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("i", range(len(COUNTED)))
def test_every_visible_key_counts_once(fvlib, kernel, fmt, i):
    """q of zeros: every visible key has the same weight.  V marks key j in column j % 128, so an output is a count of a few keys
    over the number of visible ones: a key too many or too few, anywhere, is far outside the roundings."""
    from fastvideo_rs_b200 import paged, sdpa
    kv_len, nq, mask = COUNTED[i]
    case = Case(fmt, kv_len, nq, 2, 1, 32, seed=80 + i)
    case.q = torch.zeros_like(case.q)
    for s, n in enumerate(kv_len):
        j = torch.arange(n)
        page, row = case.table[s].long()[j // 32], j % 32
        mark = torch.zeros(n, 1, D)
        mark[j, 0, j % D] = 1.0
        case.rows["v"][s] = mark.double()
        if fmt == "bf16":
            case.pool["v"][page, :, row] = mark.to(torch.bfloat16)
        else:
            case.pool["v"][page, :, row] = pack((8 + mark).to(torch.uint8))
            case.scales["v"][page, :, row] = torch.tensor([1.0, 0.0]).to(torch.bfloat16)
    kv, batch, q = case.device()
    out = paged.attend(kv, batch, q, mask_of(mask))
    assert sdpa.device_status() == 0
    want = torch.cat([attend64(case.q[case.cu[s]:case.cu[s + 1]].double(), case.rows["k"][s], case.rows["v"][s], mask)[0] for s in range(len(kv_len))])
    # P is a power of two or one, sums of up to 4 100 of them are exact in f32; the quotient and the parts' joins 2^-20; bf16
    check(out, want, (BF16_HALF + 2.0 ** -18) * want + 1e-30, f"{fmt} {COUNTED[i]}")


# ---- the Wan layer against its contiguous form ------------------------------------------------------------------------

def test_paged_layer_agrees_with_the_contiguous_one(fvlib):
    """One chunk-causal pass over a whole clip: forward_paged over bf16 pages against forward_self on the same projection."""
    from fastvideo_rs_b200 import paged, wan
    from fastvideo_rs_b200.sdpa import BlockCausal
    heads, frame, frames = 3, 20, 6
    g = torch.Generator().manual_seed(90)
    w = [(1 + 0.1 * torch.randn(heads * D, generator=g)).cuda() for _ in range(2)]
    qkv = torch.randn(1, frames * frame, 3 * heads * D, generator=g).to(torch.bfloat16).cuda()
    layer = wan.WanSelfAttention((frames, 4, 5), heads, *w, causal=BlockCausal(frame, 0, 0))
    want = layer.forward_self(qkv)[0].transpose(0, 1).double().cpu()
    got = _stream(layer, qkv, frame, "bf16", heads)
    q, k, v = (t[0].transpose(0, 1).double().cpu() for t in wan.qk_prep(qkv, *w, layer.cos, layer.sin, heads))
    o, mag = attend64(q, k, v, (frame, 0, 0))
    # q and k are off by one more rounding to bf16 (2^-8 of a pair's values, sqrt(2) of it after the rotation): each score by at
    # most 2 sqrt(2) 2^-8 |q| |k| / sqrt(128) -- by Cauchy -- and P by twice that; both sides round P and the result
    off = 2 * 2.0 * math.sqrt(2.0) * BF16_HALF * float(q.norm(dim=-1).max() * k.norm(dim=-1).max()) / math.sqrt(D)
    check(got, want, 2 * BF16_HALF * o.abs() + (2 * BF16_HALF + 2.0 ** -9 + off) * mag, "layer")
    # and no further from the 64-bit result than that
    check(got, o, BF16_HALF * o.abs() + (BF16_HALF + 2.0 ** -10 + off) * mag, "64 bits")


def test_sinks_move_on_by_appending_them_again(fvlib):
    """The rows of the sinks get the rotation of later positions by appending their raw keys once more with `positions`."""
    from fastvideo_rs_b200 import paged, sdpa, wan
    cos, sin = wan.wan_rope_tables((6, 4, 5))
    n, sink = 100, 20
    g = torch.Generator().manual_seed(91)
    k, v = (torch.randn(n, 2, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    kv = paged.PagedKv.empty(8, 16, 2)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table = torch.arange(7, dtype=torch.int32, device="cuda")[None]
    whole = paged.PagedBatch(table, i32(n), i32(0, n), max_q=n, max_kv=n)
    paged.append(kv, whole, k, v, cos=cos, sin=sin)
    before = paged.read(kv, whole, rows=n)
    head = paged.PagedBatch(table, i32(sink), i32(0, sink), max_q=sink, max_kv=sink)
    where = torch.arange(40, 40 + sink, dtype=torch.int32, device="cuda")
    paged.append(kv, head, k[:sink], v[:sink], cos=cos, sin=sin, positions=where)
    after = paged.read(kv, whole, rows=n)
    assert sdpa.device_status() == 0
    assert torch.equal(after[0][sink:], before[0][sink:]) and torch.equal(after[1], before[1])
    want = rotate64(k[:sink].double().cpu(), cos[where.long()].double().cpu()[:, None], sin[where.long()].double().cpu()[:, None], "interleaved")
    assert bool(((after[0][:sink].double().cpu() - want).abs() <= BF16_HALF * want.abs() + 2.0 ** -21 * k.abs().max().item()).all())


# ---- what is refused, reported and kept -------------------------------------------------------------------------------

def test_a_wait_that_ran_out_and_a_bad_page_are_both_told(fvlib):
    """One status read tells of the wait, the next one of the page."""
    from fastvideo_rs_b200 import FvError, paged, sdpa
    case = Case("bf16", [40], [1], 4, 2, 16, seed=1)
    kv, batch, q = case.device()
    batch.page_table[0, 1] = -1
    paged.attend(kv, batch, q, mask_of((1, 0, 0)))
    fvlib.fv_selftest_wait_timeout.argtypes = [ctypes.c_void_p, ctypes.c_longlong]
    assert fvlib.fv_selftest_wait_timeout(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), 100000) == 0
    with pytest.raises(FvError, match="wait"):
        sdpa.device_status()
    with pytest.raises(FvError, match="status 200"):
        sdpa.device_status()
    assert sdpa.device_status() == 0


def test_results_that_overlap_operands_are_refused(fvlib):
    """out may be q itself; anything in between would be read after it was written."""
    from fastvideo_rs_b200 import paged
    n, heads, hk = 20, 4, 2
    case = Case("bf16", [60], [n], heads, hk, 16, seed=2)
    kv, batch, _ = case.device()
    room = torch.randn(2 * n * 8 * D, device="cuda").to(torch.bfloat16)
    q = room[:n * heads * D].view(n, heads, D)
    late = room[8 * D:8 * D + n * heads * D].view(n, heads, D)
    fused = room[:n * 8 * D].view(n, 8, D)
    k = room[n * heads * D:][:n * hk * D].view(n, hk, D)
    with pytest.raises(ValueError, match="overlap"):
        paged.attend(kv, batch, q, out=late)
    with pytest.raises(ValueError, match="overlap"):
        paged.attend(kv, batch, fused[:, :heads], out=q)
    with pytest.raises(ValueError, match="overlap"):
        paged.append(kv, batch, k, k, q=q, q_out=late)
    with pytest.raises(ValueError, match="overlap"):
        paged.append(kv, batch, k, k, q=q.clone(), q_out=room[n * heads * D:2 * n * heads * D].view(n, heads, D))
    # side by side, and in place
    want = paged.attend(kv, batch, q, mask_of((1, 0, 0)))
    beside = room[n * heads * D:2 * n * heads * D].view(n, heads, D)
    assert torch.equal(paged.attend(kv, batch, q, mask_of((1, 0, 0)), out=beside), want)
    assert torch.equal(paged.attend(kv, batch, q, mask_of((1, 0, 0)), out=q), want)


def test_the_kernel_switch_may_change_under_a_batch(fvlib, monkeypatch):
    """FV_PAGED_KERNEL changes what scratch a call needs, also of a batch that has been asked before."""
    from fastvideo_rs_b200 import paged
    case = Case("q4", [9000], [30], 4, 1, 64, seed=3)
    kv, batch, q = case.device()
    want, bound = case.expect((1, 0, 0))
    for name in ("rows", "items", "rows", "items"):
        monkeypatch.setenv("FV_PAGED_KERNEL", name)
        check(paged.attend(kv, batch, q, mask_of((1, 0, 0))), want, bound, name)


def test_what_a_batch_keeps_does_not_grow(fvlib):
    """One batch with another number of packed rows at every call."""
    from fastvideo_rs_b200 import paged
    case = Case("bf16", [40], [1], 4, 2, 16, seed=4, pad=400)
    kv, batch, q = case.device()
    want = paged.attend(kv, batch, q)[:1]
    for n in range(1, 400):
        assert torch.equal(paged.attend(kv, batch, q[:n])[:1], want)
    assert len(batch._need) <= 64


def test_positions_must_be_aligned(fvlib):
    from fastvideo_rs_b200 import paged
    append = paged._entries()[0]
    case = Case("bf16", [40], [2], 1, 1, 16, seed=5)
    kv, batch, q = case.device()
    x = torch.zeros(2, 1, D, dtype=torch.bfloat16, device="cuda")
    table = torch.ones(40, D, device="cuda")
    where = torch.zeros(8, dtype=torch.int32, device="cuda")
    rows = paged._rows_struct.pack(x.data_ptr(), x.data_ptr(), 0, 0, table.data_ptr(), table.data_ptr(), where.data_ptr() + 2, D, D, D, D, 0, 0, 2, 0, 40, 0)
    assert append(None, kv._ref, batch._ref, rows) == -1 and b"aligned" in fvlib.fv_last_error()


# ---- many items a CTA -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt,heads,nq,n", [("q4", 40, 1030, 28100), ("bf16", 12, 2060, 24000)])
def test_keys_beyond_l2_in_phases(fvlib, fmt, heads, nq, n):
    """More keys than L2 holds: the long-chunk kernel goes through its line of items in four phases, several runs a CTA.  Against 64
    bits on a few rows of every head, at the ends of the row blocks and inside them."""
    from fastvideo_rs_b200 import _lib, paged, sdpa
    rows, mask = 128, (1, n - 600, 9)
    pages = (n + rows - 1) // rows
    g = torch.Generator(device="cuda").manual_seed(100)
    if fmt == "q4":
        pools = [torch.randint(0, 256, (pages, heads, rows, 64), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
        scales = [torch.stack([0.2 + 0.2 * torch.rand(pages, heads, rows, generator=g, device="cuda"),
                               0.3 * torch.randn(pages, heads, rows, generator=g, device="cuda")], -1).to(torch.bfloat16) for _ in range(2)]
        kv = paged.PagedKv(*pools, *scales)
    else:
        pools = [torch.randn(pages, heads, rows, D, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
        kv = paged.PagedKv(*pools)
    table = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)[None].contiguous()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    batch = paged.PagedBatch(table, i32(n), i32(0, nq), max_q=nq, max_kv=n)
    q = torch.randn(nq, heads, D, generator=g, device="cuda", dtype=torch.bfloat16)
    out = paged.attend(kv, batch, q, mask_of(mask))
    assert "fv_paged_chunk_kernel" in _lib.last_kernel() and sdpa.device_status() == 0
    assert torch.equal(out, paged.attend(kv, batch, q, mask_of(mask)))
    k, v = (t.double() for t in paged.read(kv, batch, rows=n, cu_rows=i32(0, n), first=i32(0)))
    if fmt == "q4":
        at = lambda t: t[table[0].long()].transpose(1, 2).flatten(0, 1)[:n]
        k, v = (at(s)[..., 1:].double() + at(s)[..., :1].double() * (torch.stack([at(p) & 15, at(p) >> 4], -1).flatten(-2).double() - 8.0)
                for p, s in zip(pools, scales))
    pick = torch.tensor([0, 1, 127, 128, 255, 256, 511, 700, 1023, 1024, nq - 1], device="cuda")
    p, j = pick[:, None] + n - nq, torch.arange(n, device="cuda")
    seen = (j <= p) & ((p - j < mask[1]) | (j < mask[2]))
    for h in range(heads):
        s = (q[pick, h].double() @ k[:, h].T / math.sqrt(D)).masked_fill(~seen, -math.inf)
        w = torch.softmax(s, -1)
        want, mag = w @ v[:, h], w @ v[:, h].abs()
        if fmt == "q4":
            mag = mag + 1.5
        err = (out[pick, h].double() - want).abs()
        assert bool((err <= BF16_HALF * want.abs() + (BF16_HALF + 2.0 ** -10) * mag).all()), (h, float(err.max()))
