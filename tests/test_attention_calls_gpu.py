"""GPU: packed attention on the calls between the usual ones: empty batches of grouped heads, one token of each sequence, blocks that walk
several query heads, masks longer than a block keeps, padded batches that are causal and grouped, numbers that are tensors, transforms."""
import ctypes

import pytest

from tests._attention_ref import reference, worst
from tests.test_attention_gpu import _check, _make

pytestmark = pytest.mark.gpu


def _splits(H, Hk, D, tokens, nseq):
    """Into how many shares the backward pass divides a group's query heads, read off the workspace it asks for."""
    from rag_amd import _capi
    need = ctypes.c_size_t()
    cfg = _capi.AttentionConfig(H, Hk, D, _capi.DTYPE_BF16, 0, 1, 1.0, 0, 0, 0)
    _capi.check(_capi.load().mi_attention_backward_workspace(cfg, tokens, nseq, 1, ctypes.byref(need)))
    return max(1, (need.value - H * tokens * 8) // (2 * tokens * Hk * D * 4))


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


@pytest.mark.parametrize("at", [0, 4, -1])
def test_one_token_of_each_sequence_as_a_view(at):
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    x, _, _ = _make([40], 4, 2, 64, seed=3)
    y = {n: t.view(4, 10, *t.shape[1:])[:, at:at + 1 if at != -1 else None] for n, t in x.items()}
    z = {n: t.contiguous() for n, t in y.items()}
    assert not y["q"].is_contiguous() and y["q"].shape == (4, 1, 4, 64)
    a = packed_attention(y["q"], y["k"], y["v"], return_lse=True)
    b = packed_attention(z["q"], z["k"], z["v"], return_lse=True)
    g = packed_attention_backward(y["dout"], y["q"], y["k"], y["v"], *a)
    h = packed_attention_backward(z["dout"], z["q"], z["k"], z["v"], *b)
    assert all(torch.equal(s, t) for s, t in zip((*a, *g[:3]), (*b, *h[:3])))
    assert torch.equal(a[0], z["v"].repeat_interleave(2, 2))


@pytest.mark.parametrize("H,Hk,repeats,splits", [(8, 4, 44, 1), (8, 4, 17, 1), (16, 4, 12, 2), (16, 4, 9, 2), (32, 16, 12, 1)])
@pytest.mark.parametrize("table", [0, 32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,dtype", [(32, "bf16"), (64, "fp16"), (128, "bf16"), (128, "fp16")])
def test_blocks_that_walk_several_query_heads(D, dtype, causal, table, H, Hk, repeats, splits):
    """Large batches of grouped heads: a dK / dV block takes group / splits > 1 query heads one after another, up to head size 64 with its
    rows split over two waves (17 and 9 repeats: fewer than 1,024 blocks) or not.  The batch repeats a
    pattern of sequences, so that the 64-bit form is worked out for one: a repeat's results are the first's, bit for bit, and the
    table's gradient is the sum of the repeats'."""
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    lens = [200, 1, 0, 64, 130, 33, 7, 129]
    T = sum(lens)
    assert _splits(H, Hk, D, T * repeats, len(lens) * repeats) == splits < H // Hk
    x, _, tab = _make(lens, H, Hk, D, dtype, table=table, seed=D + H + causal)
    many = {n: t.repeat(repeats, 1, 1) for n, t in x.items()}
    off = torch.tensor([0] + lens * repeats, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    kw = dict(causal=causal, bias_table=tab, max_distance=64)
    out, lse = packed_attention(many["q"], many["k"], many["v"], off, return_lse=True, **kw)
    dq, dk, dv, dtable = packed_attention_backward(many["dout"], many["q"], many["k"], many["v"], out, lse, off, **kw)
    torch.cuda.synchronize()
    ref = reference(x["q"], x["k"], x["v"], lens, causal, D ** -0.5, None, tab, 64, not causal, x["dout"])
    for n, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        t = t.view(repeats, T, *t.shape[1:])
        assert torch.equal(t, t[:1].expand_as(t)), n
        assert worst(t[0], ref, n) <= 1.0, n
    assert worst(lse[:, :T], ref, "lse") <= 1.0
    if table:
        assert worst(dtable / repeats, ref, "dtable") <= 1.0


def _long_mask(L, seed):
    """Whole tiles of 64 keys in front (past the 64th), a stretch without keys, holes on both sides of tile 256, none in the last tiles."""
    import torch
    m = (torch.rand(L, generator=torch.Generator().manual_seed(seed)) < 0.6).int()
    m[:64 * 66 + 5] = 1
    m[64 * 66 + 5:64 * 68] = 0
    if L > 64 * 257:
        m[64 * 255 - 3:64 * 257 + 9] = 0
        m[64 * 255 + 20] = m[64 * 256 + 3] = 1
    m[L - 100:] = 0
    return m.cuda()


@pytest.mark.parametrize("causal,table", [(False, 0), (True, 32)])
@pytest.mark.parametrize("L", [4096 + 300, 16384 + 333])
def test_a_key_mask_over_many_tiles(L, causal, table):
    """Past 64 tiles a block scans its words in rounds, past 256 it reads the mask as it goes."""
    import torch
    x, off, tab = _make([L], 2, 1, 32, table=table, seed=L)
    mask = _long_mask(L, 7)
    assert int(mask.sum()) > L // 2
    for n in ("k", "v"):
        x[n][mask == 0] = float("nan")
    got, _ = _check(x, off, [L], tab=tab, mask=mask, causal=causal)
    assert torch.all(got["dk"][mask == 0] == 0) and torch.all(got["dv"][mask == 0] == 0)


@pytest.mark.parametrize("H,Hk", [(4, 4), (8, 2)])
@pytest.mark.parametrize("D,dtype", [(32, "fp16"), (64, "bf16"), (128, "bf16")])
@pytest.mark.parametrize("biased", [False, True])
def test_padded_batch_causal_and_grouped(biased, D, dtype, H, Hk):
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    B, L = 5, 150
    x, _, tab = _make([L] * B, H, Hk, D, dtype, table=32 if biased else 0, seed=D)
    at = torch.arange(L)[None, :]
    km = ((at < torch.tensor([150, 3, 70, 0, 64])[:, None]) & (at >= torch.tensor([0, 0, 5, 0, 1])[:, None])).int().cuda()   # also padded in front
    for n in ("k", "v"):
        x[n][km.view(-1) == 0] = float("nan")
    y = {n: t.view(B, L, *t.shape[1:]) for n, t in x.items()}
    kw = dict(causal=True, key_mask=km, bias_table=tab)
    out, lse = packed_attention(y["q"], y["k"], y["v"], return_lse=True, **kw)
    grads = packed_attention_backward(y["dout"], y["q"], y["k"], y["v"], out, lse, **kw)
    ref = reference(x["q"], x["k"], x["v"], [L] * B, True, D ** -0.5, km.view(-1), tab, 128, False, x["dout"])
    got = {"out": out.view(-1, H, D), "lse": lse, **{n: t.view(-1, t.shape[-2], D) for n, t in zip(("dq", "dk", "dv"), grads)}}
    if biased:
        got["dtable"] = grads[3]
    off_by = {n: worst(t, ref, n) for n, t in got.items()}
    assert all(v <= 1.0 for v in off_by.values()), off_by
    assert torch.all(out[2, :5] == 0) and torch.all(grads[0][2, :5] == 0)


def test_a_scale_that_is_a_tensor_counts_as_it_stands_at_the_call():
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    x, off, _ = _make([33, 80], 4, 4, 32, seed=5)
    q, k, v = x["q"], x["k"], x["v"]
    for device in ("cpu", "cuda"):
        t = torch.tensor(0.25, device=device)
        for value in (0.25, 0.5):
            t.fill_(value)
            assert torch.equal(packed_attention(q, k, v, off, scale=t), packed_attention(q, k, v, off, scale=value))
    # one that changes between an autograd step's two passes: both take the first
    out, lse = packed_attention(q, k, v, off, scale=0.5, return_lse=True)
    want = packed_attention_backward(x["dout"], q, k, v, out, lse, off, scale=0.5)
    leaf, t = q.clone().requires_grad_(), torch.tensor(0.5)
    got = packed_attention(leaf, k, v, off, scale=t)
    t.fill_(2.0)
    got.backward(x["dout"])
    assert torch.equal(got, out) and torch.equal(leaf.grad, want[0])


@pytest.mark.parametrize("which", ["q", "v", "bias_table"])
def test_forward_mode_derivatives_are_refused(which):
    import torch
    import torch.autograd.forward_ad as fwad
    from rag_amd.attention import packed_attention
    x, off, tab = _make([33], 4, 4, 32, table=32, seed=5)
    kw = dict(q=x["q"], k=x["k"], v=x["v"], bias_table=tab)
    want = packed_attention(offsets=off, **kw)
    with fwad.dual_level():
        assert torch.equal(packed_attention(offsets=off, **kw), want)
        kw[which] = fwad.make_dual(kw[which], torch.ones_like(kw[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            packed_attention(offsets=off, **kw)


def test_tracing_is_refused():
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx
    from rag_amd.attention import packed_attention
    x, off, _ = _make([33], 4, 4, 32, seed=5)
    f = lambda q: packed_attention(q, x["k"], x["v"], off)                       # noqa: E731
    with pytest.raises(RuntimeError, match="trac"):
        make_fx(f)(x["q"])
    with pytest.raises(RuntimeError, match="trac"):
        torch.jit.trace(f, x["q"], check_trace=False)
    assert torch.equal(f(x["q"]), f(x["q"]))


def test_a_finite_bias_counts_as_at_most_4096():
    """The stated bound: -5,000 and -6,000 are both -4,096, whichever other keys a row has, and the gradient is the table's as it counts."""
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    lens = [40, 7]
    for D in (32, 64, 128):
        x, off, tab = _make(lens, 4, 2, D, table=8, seed=D)
        tab[0, :2], tab[1:4, :2], tab[5:, :2] = -5000.0, -6000.0, -1e30
        tab[0, 2], tab[2, 2] = 5000.0, 1e30
        kept = tab.clamp(-4096, 4096)
        assert not torch.equal(kept, tab)
        res = []
        for t in (tab, kept):
            out, lse = packed_attention(x["q"], x["k"], x["v"], off, bias_table=t, max_distance=20, return_lse=True)
            res.append((out, lse, *packed_attention_backward(x["dout"], x["q"], x["k"], x["v"], out, lse, off, bias_table=t, max_distance=20)))
        assert all(torch.equal(a, b) for a, b in zip(*res))
        _check(x, off, lens, tab=tab, max_distance=20)
