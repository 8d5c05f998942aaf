"""GPU: packed attention on the calls between the usual ones: empty batches of grouped heads, one token of each sequence, blocks that walk
several query heads, masks longer than a block keeps, padded batches that are causal and grouped, numbers that are tensors, transforms."""
import ctypes

import pytest

from tests._attention_ref import reference, worst
from tests.test_attention_gpu import _check, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("form", ["no sequence", "empty sequences", "empty batch", "sequences of no rows"])
def test_empty_calls_with_grouped_heads(form, biased):
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    lead = {"empty batch": (0, 7), "sequences of no rows": (3, 0)}.get(form, (0,))
    q, k = torch.empty(*lead, 8, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(*lead, 2, 64, dtype=torch.bfloat16, device="cuda")
    off = torch.zeros(1 if form == "no sequence" else 4, dtype=torch.int32, device="cuda") if len(lead) == 1 else None
    tab = torch.ones(32, 8, device="cuda") if biased else None
    out, lse = packed_attention(q, k, k, off, bias_table=tab, return_lse=True)
    dq, dk, dv, dtable = packed_attention_backward(q, q, k, k, out, lse, off, bias_table=tab)
    torch.cuda.synchronize()
    assert out.shape == dq.shape == q.shape and dk.shape == dv.shape == k.shape and lse.shape == (8, 0)
    assert dtable is None if tab is None else torch.equal(dtable, torch.zeros_like(tab))
