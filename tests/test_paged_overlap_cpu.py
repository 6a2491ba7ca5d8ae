"""Which results of the paged calls share memory with an operand, decided without a device."""
import pytest
import torch

D = 128


def test_results_may_lie_beside_an_operand_and_in_its_gaps():
    from fastvideo_rs_b200.paged import _keep_apart
    room = torch.zeros(64 * D, dtype=torch.bfloat16)
    rows = lambda at, n, h: room[at * D:(at + n * h) * D].view(n, h, D)

    def told(out, t, in_place=False):
        n, h = t.shape[:2]
        try:
            _keep_apart("out", out, "q", t, n, h, t.stride(0) if n > 1 else D, t.stride(1) if h > 1 else D, in_place)
        except ValueError as e:
            assert "overlap" in str(e)
            return True
        return False

    q = rows(0, 4, 2)
    assert told(q, q) and not told(q, q, in_place=True)
    for at, bad in ((8, False), (7, True), (1, True), (40, False)):
        assert told(rows(at, 4, 2), q, in_place=True) == bad
        assert told(q, rows(at, 4, 2)) == bad
    wide = room.view(4, 16, D)[:, :2]  # two heads of sixteen: gaps of fourteen rows
    assert not told(rows(2, 7, 2), wide) and told(rows(2, 15, 1), wide) and told(rows(1, 1, 1), wide)
    assert told(rows(0, 4, 2), wide, in_place=True)  # begins where q does, but is not q
    assert not told(room[:0].view(0, 2, D), room[:0].view(0, 2, D))
    for seed in range(200):  # against the sets of values
        g = torch.Generator().manual_seed(seed)
        r = lambda lo, hi: int(torch.randint(lo, hi + 1, (), generator=g))
        n, h, sh = r(1, 3), r(1, 3), r(1, 4)
        st = r(1, 12)
        t = torch.as_strided(room, (n, h, D), (st * D, sh * D, 1), r(0, 8) * D)
        out = rows(r(0, 40), r(1, 3), r(1, 3))
        index = torch.arange(room.numel())
        mine = torch.as_strided(index, t.shape, t.stride(), t.storage_offset()).flatten()
        both = torch.isin(index[out.storage_offset():out.storage_offset() + out.numel()], mine).any()
        assert told(out, t) == bool(both), seed


def test_another_base_address_is_not_an_overlap():
    from fastvideo_rs_b200.paged import _keep_apart
    a, b = (torch.zeros(4, 2, D, dtype=torch.bfloat16) for _ in range(2))
    _keep_apart("out", a, "q", b, 4, 2, 2 * D, D)
    with pytest.raises(ValueError, match="overlaps q"):
        _keep_apart("out", a, "q", a[1:], 3, 2, 2 * D, D, in_place=True)
