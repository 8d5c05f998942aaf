"""CPU: calls of the packed attention that its layers on the host decide: views, numbers that are tensors, transforms that cannot see the
kernels."""
import pytest


def _stub(shape):
    """What the argument checks read of a tensor on a GPU."""
    import types
    import torch
    return types.SimpleNamespace(shape=torch.Size(shape), device=torch.device("cuda", 0), is_cuda=True, dtype=torch.bfloat16)


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


def test_a_scale_that_is_a_tensor_counts_as_it_stands_at_the_call():
    import numpy as np
    import torch
    from rag_amd.attention import _setup
    q = _stub((2, 5, 4, 64))
    t = torch.tensor(0.5)
    setup = lambda scale, **kw: _setup(q, q, q, None, kw.get("causal", False), scale, None, None, kw.get("max_distance", 128), kw.get("bidirectional"))[0]   # noqa: E731
    assert setup(t).scale == 0.5
    t *= 2
    assert setup(t).scale == 1.0
    a = np.array(0.25)
    assert setup(a).scale == 0.25
    a[...] = 0.75
    assert setup(a).scale == 0.75
    causal, dist, two = torch.tensor(False), torch.tensor(100), torch.tensor(True)
    c = setup(0.5, causal=causal, max_distance=dist, bidirectional=two)
    assert (c.causal, c.max_distance, c.bidirectional) == (0, 100, 1)
    causal.fill_(True), dist.fill_(200), two.fill_(False)
    c = setup(0.5, causal=causal, max_distance=dist, bidirectional=two)
    assert (c.causal, c.max_distance, c.bidirectional) == (1, 200, 0)
    assert setup(None).scale == 0.125


def test_a_scale_that_wants_a_gradient_is_refused():
    import torch
    from rag_amd.attention import packed_attention
    q = torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="gradient"):
        packed_attention(q, q, q, scale=torch.tensor(0.5, requires_grad=True))
    with torch.no_grad(), pytest.raises(ValueError, match="on the GPU"):       # nothing is lost here: refused for being on the CPU
        packed_attention(q, q, q, scale=torch.tensor(0.5, requires_grad=True))


@pytest.mark.parametrize("which", ["q", "k", "v", "bias_table", "scale"])
def test_forward_mode_derivatives_are_refused(which):
    """A dual tensor does not require a gradient: the kernels would run on its value and drop its tangent."""
    import torch
    import torch.autograd.forward_ad as fwad
    from rag_amd.attention import packed_attention
    q = torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16)
    x = dict(q=q, k=q, v=q, bias_table=torch.zeros(32, 4), scale=torch.tensor(0.5))
    with fwad.dual_level():
        x[which] = fwad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            packed_attention(**x)
        with pytest.raises(ValueError, match="on the GPU"):                    # a level alone refuses nothing
            packed_attention(q, q, q)


@pytest.mark.parametrize("which", ["dout", "q", "out", "lse", "bias_table"])
def test_forward_mode_derivatives_of_the_backward_pass_are_refused(which):
    import torch
    import torch.autograd.forward_ad as fwad
    from rag_amd.attention import packed_attention_backward
    q = torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16)
    x = dict(dout=q, q=q, k=q, v=q, out=q, lse=torch.zeros(4, 10), bias_table=torch.zeros(32, 4))
    with fwad.dual_level():
        x[which] = fwad.make_dual(x[which].clone(), torch.ones_like(x[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            packed_attention_backward(**x)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("how", ["make_fx", "make_fx pre_dispatch", "jit.trace"])
def test_tracing_is_refused(how, backward):
    """A trace would hold the allocation of the result and not the kernel that fills it."""
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx
    from rag_amd.attention import packed_attention, packed_attention_backward
    q, lse = torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16), torch.zeros(4, 10)

    def f(x):
        return packed_attention_backward(x, x, x, x, x, lse)[0] if backward else packed_attention(x, x, x)

    with pytest.raises(RuntimeError, match="trac"):
        if how == "jit.trace":
            torch.jit.trace(f, q, check_trace=False)
        else:
            make_fx(f, pre_dispatch=how.endswith("dispatch"))(q)
    with pytest.raises(ValueError, match="on the GPU"):                        # and afterwards as before
        f(q)


def test_workspace_of_calls_that_are_out_of_range():
    import ctypes
    from rag_amd import _capi
    lib, need = _capi.load(), ctypes.c_size_t(7)
    ok = dict(heads=4, kv_heads=2, head_dim=64, dtype=_capi.DTYPE_BF16, causal=0, zero_tail=0, scale=0.125, num_buckets=0, max_distance=0, bidirectional=0)
    for change, tokens, nseq in (({}, 1 << 31, 1), ({}, 100, 1 << 24), ({}, 100, (1 << 32) + 2), (dict(heads=65536, kv_heads=1), 100, 1), (dict(head_dim=136), 100, 1),
                                 (dict(head_dim=60), 100, 1), ({}, (1 << 62), 1), (dict(heads=65535, kv_heads=1), (1 << 31) - 5000, 1)):
        cfg = _capi.AttentionConfig(*{**ok, **change}.values())
        assert lib.mi_attention_backward_workspace(cfg, tokens, nseq, 1, ctypes.byref(need)) == -1 and need.value == 7, (change, tokens, nseq)
