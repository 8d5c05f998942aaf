"""CPU: calls of the packed attention that its layers on the host decide: views, numbers that are tensors, transforms that cannot see the
kernels."""
import pytest


@pytest.mark.parametrize("index", [slice(0, 1), slice(4, 5), slice(-1, None)])
def test_a_batch_of_single_rows_may_be_a_view(index):
    """One token of each sequence of a [batch][length] tensor: rows a whole sequence apart."""
    import torch
    from rag_amd.attention import _rows
    x = torch.zeros(3, 10, 4, 64, dtype=torch.bfloat16)
    v = x[:, index]
    r = _rows("q", v, v.shape, x.dtype, x.device)
    assert (r.ptr, r.token_stride, r.head_stride) == (v.data_ptr(), 10 * 4 * 64, 64)


def test_views_whose_rows_are_not_evenly_spaced():
    import torch
    from rag_amd.attention import _rows
    x = torch.zeros(3, 10, 4, 64, dtype=torch.bfloat16)
    for v in (x[:, :2], x[:, ::3], x[:1].expand(3, -1, -1, -1), x.transpose(0, 1)):
        with pytest.raises(ValueError, match="evenly spaced"):
            _rows("q", v, v.shape, x.dtype, x.device)
    for v, stride in ((x[:, ::2], 2 * 256), (x[1:2, 3:7], 256), (x[1:2, :1], 256), (x[:, :, 1:3], 256)):
        assert _rows("q", v, v.shape, x.dtype, x.device).token_stride == stride
