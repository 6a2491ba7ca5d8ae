"""The paged K/V cache at the ends of its ranges: values and rows far from one, tables and bounds at their ends, masks counted
key by key.  Tolerances count roundings (tests/_paged.py, and beside each test where they differ)."""
import ctypes
import math

import pytest
import torch

from _paged import D, BF16_HALF, Case, attend64, pack, rotate64, seen_matrix, unpack

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
