"""What paged_attention refuses of a given result, on the CPU."""
import pytest
import torch


@pytest.mark.parametrize("shape", [(1, 4, 64), (6, 1, 64)])
def test_rows_on_top_of_each_other_are_refused(shape):
    """An expanded result has one place for several rows."""
    from flashvsr_sm89_ops import kv_pages, paged_attention
    i32, bf = torch.int32, torch.bfloat16
    with pytest.raises(ValueError, match="rows of their own"):
        paged_attention(torch.zeros(6, 4, 64, dtype=bf), kv_pages(4, 2, 64, device="cpu"),
                        torch.zeros(2, 3, dtype=i32), torch.zeros(2, dtype=i32),
                        out=torch.zeros(shape, dtype=bf).expand(6, 4, 64))
