"""page_slots on the CPU: every token without a page gets a slot that append reports, never the padding marker."""
import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_slots_of_tokens_without_a_page_are_reported(page):
    import moe_b200 as M

    table = torch.tensor([[3, -1], [-1, 0]], dtype=torch.int32)
    for seq, first, want in ((0, 0, 3 * page), (1, page, 0), (0, page, None), (1, 0, None)):
        pos = torch.arange(first, first + page, dtype=torch.int32)
        slots = M.page_slots(table, torch.full_like(pos, seq), pos, page)
        assert slots.dtype == torch.int64
        if want is None:
            assert (slots < -1).all(), slots  # at the page's last offset -page + offset would be -1
        else:
            assert slots.tolist() == list(range(want, want + page))


def test_positions_and_sequences_outside_the_table():
    import moe_b200 as M

    table = torch.tensor([[3, 1], [2, 0]], dtype=torch.int32)
    pos = torch.tensor([31, 32, -1, 5, 5, 1 << 30])
    seq = torch.tensor([0, 0, 0, 2, -1, 1])
    assert M.page_slots(table, seq, pos, 16).tolist() == [31, -2, -2, -2, -2, -2]
    empty = torch.zeros((2, 0), dtype=torch.int32)
    assert M.page_slots(empty, seq[:2], pos[:2], 16).tolist() == [-2, -2]
