"""WanSelfAttention.forward_paged without a device: its rotation tables and what it refuses."""
import pytest
import torch


def _layer(grid):
    from fastvideo_rs_b200 import wan
    w = torch.ones(2 * 128)
    return wan.WanSelfAttention(grid, 2, w, w, device="cpu")


def test_tables_go_on_behind_the_grid(fvlib):
    layer, whole = _layer((2, 4, 5)), _layer((30, 4, 5))
    assert layer._tables(40)[0] is layer.cos and layer._tables(0)[1] is layer.sin
    kept = []
    for rows in (41, 60, 81, 333, 50, 40):
        cos, sin = layer._tables(rows)
        assert cos.shape[0] >= rows and cos.shape == sin.shape
        n = min(cos.shape[0], 600)
        assert torch.equal(cos[:n], whole.cos[:n]) and torch.equal(sin[:n], whole.sin[:n])
        kept.append(cos)
    assert kept[0] is kept[1] and kept[3] is kept[4] and kept[5] is layer.cos  # (once made they stay)
    assert len(layer._longer) == 3 and len(layer.cos) == 40


def test_a_layer_with_a_vsa_context_is_refused(fvlib):
    """forward_self takes the VSA route there; dense attention in its place would be another result without a word."""
    from fastvideo_rs_b200 import wan
    w = torch.ones(2 * 128)
    layer = wan.WanSelfAttention((2, 4, 5), 2, w, w, device="cpu", vsa=object())
    with pytest.raises(ValueError, match="VSA"):
        layer.forward_paged(torch.zeros(1, 4, 768, dtype=torch.bfloat16), None, None)
