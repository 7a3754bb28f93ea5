"""Results laid over memory that other blocks still read are refused; results beside it are fine."""
import pytest
import torch

from winnow_b200.packed_backend import keep_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("over", ["counts", "seq_lens", "keep", "page_table"])
def test_kept_lengths_over_what_other_layers_read(over):
    """Refused whether the native or the Python host looks at the call; a result beside them is fine."""
    pool = [torch.zeros(2, 4, 1, 16, 8, dtype=torch.uint8, device=DEV), torch.zeros(2, 4, 1, 16, dtype=torch.half, device=DEV)] * 2
    words = torch.zeros(4, 6, dtype=torch.int32, device=DEV)
    a = {"page_table": words[0].view(2, 3), "seq_lens": words[1, 1:3], "keep": words[2, :4].view(2, 2), "counts": words[3, 1:3]}
    a["seq_lens"].fill_(8)
    a["counts"].fill_(1)
    a["page_table"].copy_(i32([[0, -1, -1], [1, -1, -1]]))
    t = a[over].reshape(-1)
    for out in (t[:2], words.view(-1)[t.storage_offset() + 1:t.storage_offset() + 3]):
        with pytest.raises(ValueError, match="share memory"):
            keep_tokens(*pool, *a.values(), 4, out=out)
    assert keep_tokens(*pool, *a.values(), 4, out=words[1, 4:6]).tolist() == [5, 5]
