"""GPU: packed attention in training: through autograd, two layers that share a table, and batches large enough for one wave per row."""
import pytest

from tests.test_attention_gpu import _check, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("table", [0, 32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D,dtype", [(32, "bf16"), (64, "fp16"), (64, "bf16"), (128, "bf16"), (128, "fp16")])
def test_many_rows(D, dtype, causal, table):
    """More than 1,024 blocks of 128 rows: a row's keys are no longer split over two waves."""
    lens = [150, 1, 0, 64, 33] * 27
    x, off, tab = _make(lens, 8, 4, D, dtype, table=table, seed=D + causal)
    _check(x, off, lens, tab=tab, causal=causal, max_distance=64)


@pytest.mark.parametrize("D", [32, 64])
def test_many_rows_under_a_key_mask(D):
    import torch
    lens = [150, 1, 0, 64, 33] * 27
    x, off, tab = _make(lens, 8, 8, D, table=32, seed=D)
    mask = (torch.rand(sum(lens), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.5).int()
    mask[:150] = 0                                           # a sequence without keys
    for n in ("k", "v"):
        x[n][mask == 0] = float("nan")
    x["dout"][:150] = 0
    _check(x, off, lens, tab=tab, mask=mask)


@pytest.mark.parametrize("D", [32, 128])
def test_more_than_65535_tiles_of_a_head(D):
    """70,000 sequences of one token (out = v, dv = dout, nothing else) around one of 70"""
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    from tests._attention_ref import reference, worst
    N, n = 70000, 70
    x, _, tab = _make([N + n], 8, 8, D, table=8, seed=D)
    off = torch.cat([torch.arange(N - 9), torch.arange(N - 9, N + 1) + n]).int().cuda()
    assert off.shape[0] == N + 1 and int(off[-1]) == N + n
    out, lse = packed_attention(x["q"], x["k"], x["v"], off, bias_table=tab, max_distance=20, return_lse=True)
    dq, dk, dv, dtable = packed_attention_backward(x["dout"], x["q"], x["k"], x["v"], out, lse, off, bias_table=tab, max_distance=20)
    torch.cuda.synchronize()
    long = slice(N - 10, N - 9 + n)
    part = {k: v[long] for k, v in x.items()}
    ref = reference(part["q"], part["k"], part["v"], [n + 1], False, D ** -0.5, None, tab, 20, True, part["dout"])
    got = {"out": out[long], "lse": lse[:, long], "dq": dq[long], "dk": dk[long], "dv": dv[long]}
    assert all(worst(y, ref, name) <= 1.0 for name, y in got.items())
    ones = torch.ones(N + n, dtype=torch.bool, device="cuda")
    ones[long] = False
    # p of the only key is 1 (backward: to fp32's last bits, which rounding it takes away); ds is the difference of two fp32 sums
    # of D products, in either order
    assert torch.equal(out[ones], x["v"][ones]) and torch.equal(dv[ones], x["dout"][ones])
    dp = (x["dout"].float().abs() * x["v"].float().abs()).sum(-1)
    for got, other in ((dq, x["k"]), (dk, x["q"])):
        assert bool((got.float().abs()[ones] <= 2.0 ** -22 * (D + 2) * dp[ones][..., None] * other.float().abs()[ones] + 1e-30).all())
    far = torch.arange(8, device="cuda") != 0                # one-token sequences know bucket 0 alone
    assert worst(dtable[far], {"dtable": ref["dtable"][far], "dtable_tol": ref["dtable_tol"][far]}, "dtable") <= 1.0


def _leaves(x, tab, which):
    import torch
    t = {n: x[n].clone().requires_grad_(n in which) for n in ("q", "k", "v")}
    t["table"] = tab.clone().requires_grad_("table" in which) if tab is not None else None
    return t


@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("which", ["q k v table", "q", "k", "v", "table", "k v"])
def test_autograd_gives_the_gradients_of_the_backward_call(which, padded):
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    which = which.split()
    x, off, tab = _make([60, 60], 4, 2, 64, table=32, seed=3)
    if padded:
        x = {n: t.view(2, 60, *t.shape[1:]) for n, t in x.items()}
        off = None
    out, lse = packed_attention(x["q"], x["k"], x["v"], off, bias_table=tab, causal=True, return_lse=True)
    want = dict(zip(("q", "k", "v", "table"), packed_attention_backward(x["dout"], x["q"], x["k"], x["v"], out, lse, off, bias_table=tab, causal=True)))
    t = _leaves(x, tab, which)
    got = packed_attention(t["q"], t["k"], t["v"], off, bias_table=t["table"], causal=True)
    assert torch.equal(got, out) and got.requires_grad
    got.backward(x["dout"])
    for n in want:
        if n in which:
            assert torch.equal(t[n].grad, want[n]), n
        else:
            assert t[n].grad is None
    o2, l2 = packed_attention(t["q"], t["k"], t["v"], off, bias_table=t["table"], causal=True, return_lse=True)
    assert torch.equal(l2, lse) and not l2.requires_grad and o2.requires_grad
    with torch.no_grad():
        assert not packed_attention(t["q"], t["k"], t["v"], off, bias_table=t["table"], causal=True).requires_grad


def test_a_loss_that_is_a_sum():
    """autograd hands the backward pass one expanded scalar"""
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    x, off, _ = _make([33, 80], 4, 4, 32, seed=5)
    t = _leaves(x, None, "qkv")
    packed_attention(t["q"], t["k"], t["v"], off).sum().backward()
    out, lse = packed_attention(x["q"], x["k"], x["v"], off, return_lse=True)
    want = packed_attention_backward(torch.ones_like(out), x["q"], x["k"], x["v"], out, lse, off)
    assert all(torch.equal(t[n].grad, w) for n, w in zip("qkv", want))


def test_two_layers_of_one_table_and_a_fused_projection():
    """Views of one QKV product, a table used twice, one query token after training: against the float32 plain form under autograd.  The
    plain form starts from the same 16-bit projections, so what differs is each layer's own rounding: a hidden state's error of 3 u per
    layer (p, out and the projection: u = 2^-8 each), relative to its largest size, twice, and again in the backward pass: 12 u."""
    import torch
    from rag_amd.attention import packed_attention, relative_position_buckets
    H, D, lens = 4, 32, [70, 1, 45]
    g = torch.Generator(device="cuda").manual_seed(8)
    T, E = sum(lens), H * D
    w0 = [torch.randn(3 * E, E, generator=g, device="cuda") * E ** -0.5 for _ in range(2)]
    h0 = torch.randn(T, E, generator=g, device="cuda").bfloat16()
    tab0 = torch.randn(32, H, generator=g, device="cuda")
    off = torch.tensor([0, 70, 71, 116], dtype=torch.int32, device="cuda")
    at = torch.arange(T)
    seq = torch.repeat_interleave(torch.arange(3), torch.tensor(lens))
    num = torch.from_numpy(relative_position_buckets((at[None, :] - at[:, None]).numpy(), 32, 128, True)).cuda().long()
    ok = (seq[:, None] == seq[None, :]).cuda()

    def run(plain):
        ws = [w.bfloat16().requires_grad_() for w in w0]
        tab = tab0.clone().requires_grad_()
        h = h0
        for w in ws:
            qkv = (h @ w.t()).view(T, 3, H, D)
            q, k, v = qkv[:, 0], qkv[:, 1], qkv[:, 2]
            if plain:
                q, k, v = (t.float().transpose(0, 1).contiguous() for t in (q, k, v))
                s = (q[:, :, None, :] * k[:, None, :, :]).sum(-1) * D ** -0.5 + tab[num].permute(2, 0, 1)
                p = s.masked_fill(~ok, -float("inf")).softmax(-1)
                a = (p[:, :, :, None] * v[:, None, :, :]).sum(2).transpose(0, 1).bfloat16()
            else:
                a = packed_attention(q, k, v, off, bias_table=tab)
            h = a.reshape(T, E)
        (h.float() ** 2).sum().backward()
        return [h.detach().float(), tab.grad] + [w.grad.float() for w in ws]

    for got, want in zip(run(False), run(True)):
        assert float((got - want).norm() / want.norm()) < 12 * 2.0 ** -8


def test_autograd_under_capture_is_refused():
    import torch
    from rag_amd.attention import packed_attention
    x, off, _ = _make([33, 80], 4, 4, 32, seed=5)
    t = _leaves(x, None, "q")
    packed_attention(t["q"], t["k"], t["v"], off)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = x["q"].clone()
        with pytest.raises(RuntimeError, match="graph capture"):
            packed_attention(t["q"], t["k"], t["v"], off)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, x["q"])


def test_second_derivatives_are_refused():
    import torch
    from rag_amd.attention import packed_attention
    x, off, _ = _make([33], 4, 4, 32, seed=5)
    t = _leaves(x, None, "q")
    (dq,) = torch.autograd.grad(packed_attention(t["q"], t["k"], t["v"], off).float().pow(2).sum(), t["q"], create_graph=True)
    with pytest.raises(RuntimeError):
        dq.sum().backward()
