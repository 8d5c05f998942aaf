"""GPU: packed attention, forward and backward, through rag_amd.attention against the plain 64-bit form, elementwise within the bounds
that tests/_attention_ref.py derives from the roundings the kernels make."""
import ctypes

import pytest

from tests._attention_ref import reference, worst

pytestmark = pytest.mark.gpu


def _make(lens, H, Hk, D, dtype="bf16", table=0, seed=0, extra=0, scale_q=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lens) + extra
    dt = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")          # noqa: E731
    x = dict(q=(r(T, H, D) * scale_q).to(dt), k=r(T, Hk, D).to(dt), v=r(T, Hk, D).to(dt), dout=r(T, H, D).to(dt))
    off = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    tab = r(table, H) if table else None
    return x, off, tab


def _check(x, off, lens, tab=None, mask=None, backward=True, **kw):
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    D = x["q"].shape[-1]
    scale = kw.pop("scale", None)
    causal = kw.get("causal", False)
    kw.setdefault("max_distance", 128)
    two = kw.pop("bidirectional", not causal)
    out, lse = packed_attention(x["q"], x["k"], x["v"], off, bias_table=tab, key_mask=mask, scale=scale, bidirectional=two, return_lse=True, **kw)
    ref = reference(x["q"], x["k"], x["v"], lens, causal, scale if scale else D ** -0.5, mask, tab, kw["max_distance"], two,
                    x["dout"] if backward else None)
    got = {"out": out, "lse": lse}
    if backward:
        grads = packed_attention_backward(x["dout"], x["q"], x["k"], x["v"], out, lse, off, bias_table=tab, key_mask=mask, scale=scale, bidirectional=two, **kw)
        got.update(zip(("dq", "dk", "dv"), grads))
        if tab is not None:
            got["dtable"] = grads[3]
        else:
            assert grads[3] is None
    torch.cuda.synchronize()
    off_by = {n: worst(y, ref, n) for n, y in got.items()}
    assert all(v <= 1.0 for v in off_by.values()), off_by
    return got, ref


LENS = [[1], [17], [31, 32, 33], [63, 64, 65], [127, 128, 129, 1], [5, 0, 200, 0, 1], [257, 3]]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("lens", LENS, ids=[str(i) for i in range(len(LENS))])
def test_lengths_and_head_sizes(lens, D, causal, dtype):
    x, off, _ = _make(lens, 4, 2, D, dtype, seed=len(lens) + D)
    _check(x, off, lens, causal=causal)


@pytest.mark.parametrize("D", [8, 24, 40, 72, 96, 120])
def test_head_sizes_between(D):
    lens = [70, 1, 130]
    x, off, tab = _make(lens, 3, 3, D, table=8, seed=D)
    _check(x, off, lens, tab=tab, causal=True, max_distance=20)


@pytest.mark.parametrize("H,Hk", [(1, 1), (2, 1), (3, 1), (6, 2), (8, 8), (12, 12), (16, 2), (20, 5)])
def test_grouped_heads(H, Hk):
    lens = [90, 33]
    x, off, tab = _make(lens, H, Hk, 64, table=16, seed=H)
    _check(x, off, lens, causal=True)
    _check(x, off, lens, tab=tab, max_distance=40)


@pytest.mark.parametrize("buckets,M,two,causal", [(32, 128, True, False), (32, 128, False, True), (32, 128, True, True), (32, 128, False, False), (4, 2, True, False),
                                                   (4, 9, True, True), (2, 5, False, True), (3, 7, False, True), (48, 300, True, False), (64, 1024, True, False),
                                                   (64, 40, False, True), (34, 90, True, False), (33, 17, False, True)])
@pytest.mark.parametrize("D,dtype", [(32, "bf16"), (128, "fp16")])
def test_bias_schemes(buckets, M, two, causal, D, dtype):
    lens = [3, 301, 64]
    x, off, tab = _make(lens, 2, 2, D, dtype, table=buckets, seed=buckets + M)
    _check(x, off, lens, tab=tab, causal=causal, max_distance=M, bidirectional=two)


def test_bias_over_a_long_sequence_with_far_buckets():
    lens = [1500]
    x, off, tab = _make(lens, 2, 1, 64, table=32, seed=5)
    _check(x, off, lens, tab=tab)
    _check(x, off, lens, tab=tab, causal=True)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_key_mask_with_holes_and_rows_without_keys(D, causal):
    import torch
    lens = [70, 40, 129]
    x, off, tab = _make(lens, 4, 2, D, table=32, seed=3)
    mask = (torch.rand(sum(lens), generator=torch.Generator().manual_seed(2)) < 0.6).to(torch.int32)
    mask[:5] = 0                                            # causal: rows 0 .. 4 attend nothing
    mask[70:110] = 0                                        # a sequence without any key
    mask = mask.cuda()
    got, _ = _check(x, off, lens, tab=tab, mask=mask, causal=causal)
    assert torch.all(got["out"][70:110] == 0) and torch.all(got["lse"][:, 70:110] == -float("inf")) and torch.all(got["dk"][mask == 0] == 0)
    # what masked keys hold does not matter
    y = {n: t.clone() for n, t in x.items()}
    y["k"][mask == 0] = float("nan")
    y["v"][mask == 0] = float("inf")
    again, _ = _check(y, off, lens, tab=tab, mask=mask, causal=causal)
    for n in got:
        assert torch.equal(got[n], again[n]), n


@pytest.mark.parametrize("mask", [False, True])
def test_padded_batch(mask):
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    B, L, H, Hk, D = 5, 77, 4, 4, 64
    lens = [L] * B
    x, _, tab = _make(lens, H, Hk, D, table=32, seed=9)
    km = None
    if mask:
        km = (torch.arange(L)[None, :] < torch.tensor([77, 3, 50, 0, 64])[:, None]).to(torch.int32).cuda()
    y = {n: t.view(B, L, *t.shape[1:]) for n, t in x.items()}
    out, lse = packed_attention(y["q"], y["k"], y["v"], key_mask=km, bias_table=tab, return_lse=True)
    grads = packed_attention_backward(y["dout"], y["q"], y["k"], y["v"], out, lse, key_mask=km, bias_table=tab)
    ref = reference(x["q"], x["k"], x["v"], lens, False, D ** -0.5, None if km is None else km.view(-1), tab, 128, True, x["dout"])
    for n, g in zip(("out", "lse", "dq", "dk", "dv", "dtable"), (out.view(-1, H, D), lse, *(t.view(-1, t.shape[-2], D) for t in grads[:3]), grads[3])):
        assert worst(g, ref, n) <= 1.0, n


def test_views_of_one_qkv_tensor_and_strided_outputs():
    """q, k, v as slices of one projection's rows (token stride 3 H D), dout transposed to [heads][tokens]."""
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    lens, H, D = [45, 100], 6, 32
    x, off, _ = _make(lens, H, H, D, seed=4)
    T = sum(lens)
    qkv = torch.stack((x["q"], x["k"], x["v"]), 1).contiguous()                  # [T][3][H][D]
    q, k, v = qkv[:, 0], qkv[:, 1], qkv[:, 2]
    do = x["dout"].transpose(0, 1).contiguous().transpose(0, 1)                  # [T][H][D] with strides (D, T D, 1)
    assert not q.is_contiguous() and not do.is_contiguous()
    want = packed_attention(x["q"], x["k"], x["v"], off, causal=True, return_lse=True)
    got = packed_attention(q, k, v, off, causal=True, return_lse=True)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    a = packed_attention_backward(x["dout"], x["q"], x["k"], x["v"], *want, off, causal=True)
    b = packed_attention_backward(do, q, k, v, *got, off, causal=True)
    assert all(torch.equal(s, t) for s, t in zip(a[:3], b[:3])) and T == q.shape[0]


def test_rows_beyond_two_to_the_31_elements():
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    T, pitch, H, D = 300, 8 * 1024 * 1024, 1, 64                                 # the last rows start behind element 2.4e9
    lens = [200, 100]
    x, off, _ = _make(lens, H, H, D, seed=6)
    big = torch.empty(T * pitch, dtype=torch.bfloat16, device="cuda")
    views = [torch.as_strided(big, (T, H, D), (pitch, D, 1), o) for o in (0, 64, 128)]
    for view, n in zip(views, "qkv"):
        view.copy_(x[n])
    want = packed_attention(x["q"], x["k"], x["v"], off, causal=True, return_lse=True)
    got = packed_attention(*views, off, causal=True, return_lse=True)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    a = packed_attention_backward(x["dout"], x["q"], x["k"], x["v"], *want, off, causal=True)
    b = packed_attention_backward(x["dout"], *views, *got, off, causal=True)
    assert all(torch.equal(s, t) for s, t in zip(a[:3], b[:3]))


def test_many_sequences():
    import torch
    lens = [i % 4 for i in range(5000)]                                          # more than 64 x 64: three rounds of the search
    x, off, tab = _make(lens, 2, 1, 32, table=32, seed=8)
    _check(x, off, lens, tab=tab, backward=False)
    lens = [0, 0, 3, 0, 1, 0] * 30
    x, off, tab = _make(lens, 2, 1, 32, table=32, seed=8)
    _check(x, off, lens, tab=tab, causal=True)
    assert torch.cuda.current_device() == 0


def test_sequences_do_not_reach_each_other():
    """NaN and infinities in one sequence, and behind the last, leave the others' results and gradients alone."""
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    lens = [40, 64, 33]
    for causal in (False, True):
        x, off, tab = _make(lens, 4, 2, 64, table=32, seed=12, extra=10)
        kw = dict(causal=causal, bias_table=tab)
        out, lse = packed_attention(x["q"], x["k"], x["v"], off, return_lse=True, **kw)
        grads = packed_attention_backward(x["dout"], x["q"], x["k"], x["v"], out, lse, off, **kw)
        y = {n: t.clone() for n, t in x.items()}
        for n in y:
            y[n][40:104:3] = float("nan")
            y[n][41:104:3] = float("inf")
            y[n][137:] = float("nan")
        out2, lse2 = packed_attention(y["q"], y["k"], y["v"], off, return_lse=True, **kw)
        grads2 = packed_attention_backward(y["dout"], y["q"], y["k"], y["v"], out2, lse2, off, **kw)
        for s, t in zip((out, *grads[:3]), (out2, *grads2[:3])):
            assert torch.equal(s[:40], t[:40]) and torch.equal(s[104:], t[104:])
            assert torch.isnan(t[40:104].float()).any()
        assert torch.equal(lse[:, :40], lse2[:, :40]) and torch.equal(lse[:, 104:], lse2[:, 104:])


def test_rows_behind_the_last_sequence():
    import torch
    from rag_amd import _capi
    from rag_amd.attention import packed_attention, packed_attention_backward
    lens = [30, 50]
    x, off, tab = _make(lens, 4, 2, 64, table=32, seed=1, extra=200)
    out, lse = packed_attention(x["q"], x["k"], x["v"], off, bias_table=tab, return_lse=True)
    grads = packed_attention_backward(x["dout"], x["q"], x["k"], x["v"], out, lse, off, bias_table=tab)
    for t in (out, *grads[:3]):
        assert torch.all(t[80:] == 0) and not torch.all(t[:80] == 0)
    assert torch.all(lse[:, 80:] == -float("inf"))
    # the C entry leaves them as they were unless asked
    y = torch.full_like(out, 7.0)
    z = torch.full_like(lse, 7.0)
    rows = lambda t: _capi.AttentionRows(t.data_ptr(), t.stride(0), t.stride(1))   # noqa: E731
    cfg = _capi.AttentionConfig(4, 2, 64, _capi.DTYPE_BF16, 0, 0, 64 ** -0.5, 32, 128, 1)
    lib, ctx = _capi.load(), _capi.get_ctx(0)
    _capi.check(lib.mi_attention_dev(ctx, cfg, x["q"].shape[0], 2, off.data_ptr(), None, rows(x["q"]), rows(x["k"]), rows(x["v"]), tab.data_ptr(), rows(y),
                                     z.data_ptr(), _capi.stream_arg(y.device)))
    assert torch.equal(y[:80], out[:80]) and torch.all(y[80:] == 7) and torch.equal(z[:, :80], lse[:, :80]) and torch.all(z[:, 80:] == 7)
    g = [torch.full_like(t, 7.0) for t in grads[:3]]
    need = ctypes.c_size_t()
    _capi.check(lib.mi_attention_backward_workspace(cfg, x["q"].shape[0], 2, 1, ctypes.byref(need)))
    work, dt = torch.empty(need.value, dtype=torch.uint8, device="cuda"), torch.empty_like(tab)
    _capi.check(lib.mi_attention_backward_dev(ctx, cfg, x["q"].shape[0], 2, off.data_ptr(), None, rows(x["q"]), rows(x["k"]), rows(x["v"]), tab.data_ptr(), rows(y),
                                              z.data_ptr(), rows(x["dout"]), *(rows(t) for t in g), dt.data_ptr(), work.data_ptr(), work.numel(), _capi.stream_arg(y.device)))
    for s, t in zip(grads[:3], g):
        assert torch.equal(s[:80], t[:80]) and torch.all(t[80:] == 7)
    assert torch.equal(dt, grads[3])


def test_no_rows_and_no_sequences():
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    e = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    tab = torch.ones(32, 4, device="cuda")
    for off in (torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")):
        out, lse = packed_attention(e, e, e, off, bias_table=tab, return_lse=True)
        assert out.shape == e.shape and lse.shape == (4, 0)
        g = packed_attention_backward(e, e, e, e, out, lse, off, bias_table=tab)
        assert g[0].shape == e.shape and torch.all(g[3] == 0)
    b = torch.empty(0, 7, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert packed_attention(b, b, b).shape == b.shape
    b = torch.empty(3, 0, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert packed_attention(b, b, b).shape == b.shape
    x, off, _ = _make([9], 4, 4, 64)                                             # rows, but no sequence
    assert torch.all(packed_attention(x["q"], x["k"], x["v"], off[:1]) == 0)


def test_extreme_scores_and_biases():
    import torch
    from rag_amd.attention import packed_attention
    lens = [100, 37]
    x, off, tab = _make(lens, 2, 2, 64, table=32, seed=2, scale_q=30.0)          # scores of several hundred: nearly one key per row
    _check(x, off, lens, tab=tab)
    _check(x, off, lens, causal=True)
    low = torch.finfo(torch.float32).min
    tab2 = tab.clone()
    tab2[16:] = -float("inf")                                                    # later keys are out: the same as a causal mask
    x, off, _ = _make(lens, 2, 2, 64, seed=2)
    got, _ = _check(x, off, lens, tab=tab2)
    tab3 = tab.clone()
    tab3[16:] = low                                                              # the type's lowest value: out as well, where another key is in
    assert torch.equal(packed_attention(x["q"], x["k"], x["v"], off, bias_table=tab3), got["out"])
    tab4 = torch.full_like(tab, -float("inf"))                                   # nothing attended anywhere
    got, _ = _check(x, off, lens, tab=tab4)
    assert torch.all(got["out"] == 0)
    tab5 = torch.full_like(tab, low)                                             # one bias for all keys cancels, whatever its size
    _check(x, off, lens, tab=tab5)
    for far in (low, -1e9, -1e4, -float("inf")):                                 # far keys out, before and behind: a window of 16 either way
        tab6 = tab.clone()
        tab6[10:16] = far
        tab6[26:] = far
        x, off, _ = _make([300, 37], 2, 2, 64, seed=2)
        _check(x, off, [300, 37], tab=tab6)
        _check(x, off, [300, 37], tab=tab6, causal=True, bidirectional=True)


def test_repeated_calls_give_the_same_bits():
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    x, off, tab = _make([700, 129, 64], 8, 2, 64, table=32, seed=21)
    first = None
    for _ in range(4):
        out, lse = packed_attention(x["q"], x["k"], x["v"], off, bias_table=tab, return_lse=True)
        now = (out, lse, *packed_attention_backward(x["dout"], x["q"], x["k"], x["v"], out, lse, off, bias_table=tab))
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_another_stream_than_the_default():
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    x, off, tab = _make([300, 64], 4, 4, 64, table=32, seed=22)
    want = packed_attention(x["q"], x["k"], x["v"], off, bias_table=tab, return_lse=True)
    wg = packed_attention_backward(x["dout"], x["q"], x["k"], x["v"], *want, off, bias_table=tab)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = {n: (t.float() * 1.0).to(t.dtype) for n, t in x.items()}             # produced on the side stream
        got = packed_attention(y["q"], y["k"], y["v"], off, bias_table=tab, return_lse=True)
        gg = packed_attention_backward(y["dout"], y["q"], y["k"], y["v"], *got, off, bias_table=tab)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*want, *wg), (*got, *gg)))


def test_two_graphs_with_eager_work_between_their_replays():
    """Forward and backward captured twice; new inputs written into the captured buffers; each replay equals the eager call."""
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward

    def step(x, off, tab, causal):
        out, lse = packed_attention(x["q"], x["k"], x["v"], off, bias_table=tab, causal=causal, return_lse=True)
        return (out, lse, *packed_attention_backward(x["dout"], x["q"], x["k"], x["v"], out, lse, off, bias_table=tab, causal=causal))

    held = []
    for i, (lens, causal) in enumerate([([200, 65], False), ([130, 1, 90], True)]):
        x, off, tab = _make(lens, 4, 2, 64, table=40 if i else 32, seed=30 + i)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, off, tab, causal)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(x, off, tab, causal)
        held.append((graph, x, off, tab, causal, res, lens))
    for turn in range(3):
        for i, (graph, x, off, tab, causal, res, lens) in enumerate(held):
            new, _, ntab = _make(lens, 4, 2, 64, table=tab.shape[0], seed=100 * turn + i)
            for n in x:
                x[n].copy_(new[n])
            tab.copy_(ntab)
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in res]
            want = step(new, off, ntab, causal)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, got)), (turn, i)


def test_refusals_of_the_python_layer():
    import torch
    from rag_amd import MI355Error
    from rag_amd.attention import packed_attention, packed_attention_backward
    x, off, tab = _make([20, 12], 4, 2, 64, table=32)
    q, k, v = x["q"], x["k"], x["v"]
    bad = [
        dict(q=q.float(), k=k.float(), v=v.float()),
        dict(k=k.half()),
        dict(k=k[:-1]),
        dict(v=v[:, :1]),
        dict(k=k[:, :, :32], v=v[:, :, :32]),
        dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)),
        dict(offsets=None),
        dict(offsets=off.long()),
        dict(offsets=off.cpu()),
        dict(offsets=off[:0]),
        dict(key_mask=torch.ones(32, dtype=torch.bool, device="cuda")),
        dict(key_mask=torch.ones(31, dtype=torch.int32, device="cuda")),
        dict(bias_table=tab.bfloat16()),
        dict(bias_table=tab[:, :2]),
        dict(bias_table=tab[:0]),
        dict(bias_table=tab.t().contiguous().t()),
        dict(q=q[:, :3], k=k, v=v),
        dict(q=torch.empty(32, 4, 60, dtype=torch.bfloat16, device="cuda"), k=torch.empty(32, 2, 60, dtype=torch.bfloat16, device="cuda"),
             v=torch.empty(32, 2, 60, dtype=torch.bfloat16, device="cuda")),
        dict(scale=-1.0),
        dict(bias_table=tab, max_distance=4),
        dict(bias_table=tab[:31].contiguous()),
        dict(q=q.view(2, 16, 4, 64), k=k.view(2, 16, 2, 64), v=v.view(2, 16, 2, 64)),       # offsets with a padded batch
    ]
    for i, b in enumerate(bad):
        kw = dict(q=q, k=k, v=v, offsets=off)
        kw.update(b)
        with pytest.raises((ValueError, MI355Error)):
            packed_attention(**kw)
            raise AssertionError(i)
    out, lse = packed_attention(q, k, v, off, return_lse=True)
    for b in (dict(lse=lse[:, :-1]), dict(lse=lse.double()), dict(out=out[:-1]), dict(dout=q.half()), dict(lse=lse.t().contiguous().t())):
        kw = dict(dout=x["dout"], q=q, k=k, v=v, out=out, lse=lse, offsets=off)
        kw.update(b)
        with pytest.raises(ValueError):
            packed_attention_backward(**kw)
