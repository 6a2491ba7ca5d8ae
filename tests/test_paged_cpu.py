"""The paged K/V cache without a device: what its Python and C faces refuse, and the plain forms that the GPU tests lean on."""
import ctypes
import math

import pytest
import torch

from _paged import D, allows, attend64, pack, quantize, seen_matrix, stands_for, unpack


def test_handles_refuse_what_is_not_a_cache(fvlib):
    from fastvideo_rs_b200 import paged
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)
    with pytest.raises(ValueError, match="CUDA"):
        paged.PagedKv(z(2, 1, 16, 128), z(2, 1, 16, 128))
    for bad in (z(2, 1, 16, 64), z(2, 16, 128), z(2, 1, 16, 128, dtype=torch.float32)):
        with pytest.raises(ValueError, match="must be"):
            paged.PagedKv(bad, bad)
    for rows in (0, 8, 24, 512):
        with pytest.raises(ValueError, match="rows"):
            paged.PagedKv(z(2, 1, rows, 128), z(2, 1, rows, 128))
    with pytest.raises(ValueError, match="scales"):
        paged.PagedKv(z(2, 1, 16, 64, dtype=torch.uint8), z(2, 1, 16, 64, dtype=torch.uint8))
    with pytest.raises(ValueError, match="scales"):
        paged.PagedKv(z(2, 1, 16, 128), z(2, 1, 16, 128), z(2, 1, 16, 2), z(2, 1, 16, 2))
    with pytest.raises(ValueError, match="format"):
        paged.PagedKv.empty(1, 16, 1, "q5")
    with pytest.raises(ValueError, match="int32"):
        paged.PagedBatch(torch.zeros(1, 4, dtype=torch.int64), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), max_q=1, max_kv=1)
    with pytest.raises(ValueError, match="page_table"):
        paged.PagedBatch(torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), max_q=1, max_kv=1)


def test_batch_bounds(fvlib):
    from fastvideo_rs_b200 import paged
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)
    for kw in (dict(max_q=-1, max_kv=1), dict(max_q=1, max_kv=1 << 30), dict(max_q=1 << 32, max_kv=1)):
        with pytest.raises(ValueError, match="2\\^30|int32"):
            paged.PagedBatch(z(1, 4), z(1), z(2), **kw)


def _c(**kw):
    from fastvideo_rs_b200 import paged
    kv = dict(k=16, v=16, k_scale=None, v_scale=None, format=0, pages=4, page_rows=16, kv_heads=2)
    b = dict(page_table=16, kv_len=16, cu_q=16, seqs=1, table_width=4, max_q=1, max_kv=64)
    for n, x in kw.items():
        (kv if n in kv else b)[n] = x
    return paged._KvC(*kv.values()), paged._BatchC(*b.values())


def _rows(**kw):
    from fastvideo_rs_b200 import paged
    x = dict(k=16, v=16, q=0, q_out=0, cos=0, sin=0, positions=0, k_tok=256, k_head=128, v_tok=256, v_head=128, q_tok=0, q_head=0,
             tokens=1, q_heads=0, table_rows=0, pairing=0)
    x.update(kw)
    return paged._rows_struct.pack(*x.values())


def _query(**kw):
    from fastvideo_rs_b200 import paged
    x = dict(q=16, out=16, workspace=0, workspace_bytes=0, q_tok=512, q_head=128, tokens=1, heads=4, mode=1, block=1, window=0, sink=0, scale=0.1)
    x.update(kw)
    return paged._query_struct.pack(*x.values())


@pytest.mark.parametrize("kw,text", [(dict(format=2), b"format"), (dict(pages=0), b"pool"), (dict(kv_heads=0), b"pool"),
                                     (dict(page_rows=8), b"rows"), (dict(page_rows=48), b"rows"), (dict(page_rows=512), b"rows"),
                                     (dict(max_kv=65), b"does not hold"), (dict(seqs=-1), b"negative"), (dict(max_q=-1), b"negative")])
def test_c_entries_refuse_bad_sizes_before_any_device(fvlib, kw, text):
    from fastvideo_rs_b200 import paged
    append, read, need, attn = paged._entries()
    kv, b = _c(**kw)
    kr, br = ctypes.addressof(kv), ctypes.addressof(b)
    assert append(None, kr, br, _rows()) == -1
    assert text in fvlib.fv_last_error()
    assert read(None, kr, br, 16, None, 1, 16, 16) == -1 and text in fvlib.fv_last_error()
    assert attn(None, kr, br, _query()) == -1


def test_c_entries_refuse_and_decline(fvlib):
    from fastvideo_rs_b200 import paged
    append, read, need, attn = paged._entries()
    kv, b = _c()
    kr, br = ctypes.addressof(kv), ctypes.addressof(b)
    assert append(None, None, br, _rows()) == -1 and append(None, kr, br, None) == -1 and attn(None, kr, br, None) == -1
    for bad in (dict(heads=3), dict(scale=0.0), dict(scale=math.inf), dict(mode=7), dict(block=0), dict(window=-1), dict(sink=-1)):
        assert attn(None, kr, br, _query(**bad)) == -1, bad
    assert append(None, kr, br, _rows(tokens=1 << 30)) == -1 and read(None, kr, br, 16, None, 1 << 30, 16, 16) == -1
    # empty calls are declined before a device is asked for
    assert attn(None, kr, br, _query(tokens=0)) == 1
    assert append(None, kr, br, _rows(tokens=0)) == 1
    assert read(None, kr, br, 16, None, 0, 16, 16) == 1
    if not torch.cuda.is_available():  # no CPU path
        assert attn(None, kr, br, _query()) == -3 and append(None, kr, br, _rows()) == -3
        assert need(kr, br, _query()) == 0


@pytest.mark.parametrize("mask", [(1, 0, 0), (1, 5, 0), (1, 5, 3), (4, 2, 1), (7, 0, 0), (3, 1, 2)])
def test_plain_mask_is_the_predicate(mask):
    seen = seen_matrix(6, 23, mask)
    for i in range(6):
        for j in range(23):
            assert bool(seen[i, j]) == allows(17 + i, j, *mask)


def test_plain_mask_agrees_with_block_causal_from_the_sinks_on():
    """The cache's mask is BlockCausal's on every row from the last sink block on; before it the sinks stay causal."""
    from fastvideo_rs_b200.sdpa import BlockCausal
    for mask in ((1, 5, 3), (4, 2, 1), (3, 1, 2), (5, 0, 0)):
        m = BlockCausal(*mask)
        for p in range(30):
            for j in range(30):
                same = allows(p, j, *mask) == m.allows(p, j)
                assert same or (p // mask[0] < mask[2] and j // mask[0] > p // mask[0])


def test_plain_four_bit_format():
    x = torch.randn(300, D, generator=torch.Generator().manual_seed(1)) * torch.logspace(-3, 3, 300)[:, None]
    codes, sc = quantize(x)
    assert torch.equal(unpack(pack(codes)), codes)
    off = (stands_for(pack(codes), sc) - x.double()).abs() / sc[:, :1].double()
    # half a step; at the ends the rounding of the step (2^-8 of 15 steps) and of zero (2^-8 of at most ~8 steps) on top
    assert float(off.max()) <= 0.5 + 23 * 2.0 ** -8


def test_plain_attention_of_equal_keys_is_the_mean():
    q, v = torch.zeros(2, 4, D, dtype=torch.float64), torch.randn(9, 2, D, dtype=torch.float64)
    o, _ = attend64(q, torch.zeros_like(v), v, (1, 0, 0))
    assert torch.allclose(o[1, 3], v[:, 1].mean(0)) and torch.allclose(o[0, 0], v[:8, 0].mean(0))
