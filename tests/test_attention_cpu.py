"""CPU: the packed attention's bucket scheme in whole numbers, and every refusal of its C entry points and Python layer that needs no
GPU (arguments are checked before anything touches the device)."""
import ctypes

import numpy as np
import pytest

from tests._attention_ref import bucket_of


def _lib():
    from rag_amd import _capi
    return _capi, _capi.load()


@pytest.mark.parametrize("bidirectional", [True, False])
def test_buckets_match_the_whole_number_definition(bidirectional):
    from rag_amd.attention import relative_position_buckets
    for buckets in list(range(4 if bidirectional else 2, 65, 2)) + ([] if bidirectional else [3, 5, 7, 33, 63]):
        n = buckets // 2 if bidirectional else buckets
        for M in {n // 2 + 1, n, 2 * n, 20, 33, 100, 127, 128, 256, 1000, 1024}:
            if not n // 2 < M <= 1024:
                continue
            rel = np.arange(-1030, 1031, 7 if M not in (128, 1024) else 1)
            got = relative_position_buckets(rel, buckets, M, bidirectional)
            want = [bucket_of(int(r), buckets, M, bidirectional) for r in rel]
            assert got.tolist() == want, (buckets, M)


def test_buckets_match_the_logarithm_in_its_usual_floating_point_form():
    """32 buckets up to distance 128, the usual setting, against m + log(d / m) / log(M / m) (n - m) in fp32 torch."""
    import torch
    from rag_amd.attention import relative_position_buckets
    r = torch.arange(-600, 601)
    n, d = 16, r.abs()
    far = 8 + (torch.log(d.float().clamp(min=1) / 8) / np.log(128 / 8) * 8).to(torch.long)
    want = torch.where(d < 8, d, far.clamp(max=n - 1)) + (r > 0) * n
    assert relative_position_buckets(r.numpy(), 32, 128, True).tolist() == want.tolist()
    assert relative_position_buckets(np.array([-(1 << 40), 1 << 40]), 32, 128, True).tolist() == [15, 31]


def test_bucket_schemes_that_are_refused():
    from rag_amd import MI355Error
    from rag_amd.attention import relative_position_buckets
    for args in [(1, 128, False), (2, 128, True), (7, 128, True), (66, 128, True), (65, 128, False), (32, 8, True), (32, 1025, True), (0, 128, True), (-4, 128, False)]:
        with pytest.raises(MI355Error):
            relative_position_buckets(np.arange(3), *args)


def _call(change=None, rows=None, tokens=64, nseq=2, offsets=4096, table=None, backward=False, **extra):
    """One call with a made-up context and addresses that nothing may look behind: it has to be refused by its arguments."""
    capi, lib = _lib()
    cfg = dict(heads=4, kv_heads=2, head_dim=64, dtype=capi.DTYPE_BF16, causal=0, zero_tail=0, scale=0.125, num_buckets=0, max_distance=0, bidirectional=0)
    cfg.update(change or {})
    c = capi.AttentionConfig(*cfg.values())
    hq, hk, D = cfg["heads"], cfg["kv_heads"], cfg["head_dim"]
    base = {n: [1 << 20, max(hq, 1) * D, D] for n in ("q", "out", "dout", "dq")}
    base.update({n: [1 << 20, max(hk, 1) * D, D] for n in ("k", "v", "dk", "dv")})
    for n, (i, x) in (rows or {}).items():
        base[n][i] = x
    R = {n: capi.AttentionRows(*x) for n, x in base.items()}
    ctx = extra.get("ctx", 4096)
    if not backward:
        rc = lib.mi_attention_dev(ctx, c, tokens, nseq, offsets, None, R["q"], R["k"], R["v"], table, R["out"], None, None)
    else:
        rc = lib.mi_attention_backward_dev(ctx, c, tokens, nseq, offsets, None, R["q"], R["k"], R["v"], table, R["out"], extra.get("lse", 4096), R["dout"],
                                           R["dq"], R["dk"], R["dv"], extra.get("dtable"), extra.get("work", 1 << 20), extra.get("bytes", 1 << 30), None)
    return rc, lib.mi_last_error().decode()


BAD = [
    (dict(ctx=None), "NULL"),
    (dict(change=dict(dtype=0)), "dtype"),
    (dict(change=dict(dtype=7)), "dtype"),
    (dict(change=dict(heads=0)), "heads"),
    (dict(change=dict(kv_heads=0)), "heads"),
    (dict(change=dict(kv_heads=3)), "multiple"),
    (dict(change=dict(heads=-4, kv_heads=-2)), "heads"),
    (dict(change=dict(head_dim=0)), "head_dim"),
    (dict(change=dict(head_dim=60)), "head_dim"),
    (dict(change=dict(head_dim=136)), "head_dim"),
    (dict(change=dict(scale=0.0)), "scale"),
    (dict(change=dict(scale=-1.0)), "scale"),
    (dict(change=dict(scale=1e-30)), "scale"),
    (dict(change=dict(scale=float("nan"))), "scale"),
    (dict(change=dict(scale=float("inf"))), "scale"),
    (dict(tokens=-1), "tokens"),
    (dict(tokens=1 << 31), "tokens"),
    (dict(nseq=-1), "sequences"),
    (dict(nseq=1 << 24), "sequences"),
    (dict(offsets=None, nseq=3), "one length"),
    (dict(offsets=None, nseq=0), "one length"),
    (dict(rows=dict(q=(0, None))), "q is NULL"),
    (dict(rows=dict(k=(0, (1 << 20) + 8))), "k is not 16-byte aligned"),
    (dict(rows=dict(v=(1, 132))), "strides of v"),
    (dict(rows=dict(out=(2, 68))), "strides of out"),
    (dict(rows=dict(v=(1, 1 << 24))), "2^24"),
    (dict(rows=dict(q=(1, 56))), "overlap"),
    (dict(rows=dict(k=(2, 0))), "overlap"),
    (dict(rows=dict(q=(1, -256))), "overlap"),
    (dict(change=dict(num_buckets=32, max_distance=128, bidirectional=1)), "bias_table is NULL"),
    (dict(table=4096), "without buckets"),
    (dict(change=dict(num_buckets=31, max_distance=128, bidirectional=1), table=4096), "num_buckets"),
    (dict(change=dict(num_buckets=32, max_distance=4, bidirectional=1), table=4096), "max_distance"),
    (dict(change=dict(heads=65535, kv_heads=1), tokens=(1 << 31) - 5000), "too many"),
]


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("kw,says", BAD, ids=[str(i) for i in range(len(BAD))])
def test_refused_by_its_arguments(kw, says, backward):
    rc, msg = _call(**kw, backward=backward)
    assert rc == -1 and says in msg, (rc, msg)


@pytest.mark.parametrize("kw,says", [(dict(lse=None), "lse"), (dict(dtable=4096), "dbias_table"), (dict(work=None), "workspace"), (dict(work=(1 << 20) + 128), "workspace"),
                                     (dict(bytes=100), "workspace of 100 bytes"), (dict(rows=dict(dq=(0, None))), "dq is NULL"),
                                     (dict(rows=dict(dk=(1, 100))), "strides of dk"), (dict(rows=dict(dv=(0, 8))), "dv is not 16-byte"),
                                     (dict(rows=dict(dout=(2, 8))), "dout")])
def test_backward_refused_by_its_own_arguments(kw, says):
    rc, msg = _call(**kw, backward=True)
    assert rc == -1 and says in msg, (rc, msg)


def test_too_many_sequences():
    for backward in (False, True):
        rc, msg = _call(change=dict(head_dim=128), nseq=1 << 21, backward=backward)
        assert rc == -1 and "too many" in msg, (rc, msg)


def test_workspace_sizes():
    capi, lib = _lib()
    need = ctypes.c_size_t()
    cfg = capi.AttentionConfig(4, 2, 64, capi.DTYPE_BF16, 0, 0, 0.125, 0, 0, 0)
    assert lib.mi_attention_backward_workspace(cfg, 1000, 3, 1, ctypes.byref(need)) == 0 and need.value >= 4 * 1000 * 4
    cfg.num_buckets, cfg.max_distance, cfg.bidirectional = 32, 128, 1
    plain = need.value
    assert lib.mi_attention_backward_workspace(cfg, 1000, 3, 1, ctypes.byref(need)) == 0 and need.value > plain
    assert lib.mi_attention_backward_workspace(cfg, 0, 0, 0, ctypes.byref(need)) == 0 and need.value == 0
    assert lib.mi_attention_backward_workspace(cfg, 1000, 3, 0, ctypes.byref(need)) == -1
    assert lib.mi_attention_backward_workspace(None, 1000, 3, 1, ctypes.byref(need)) == -1


def test_python_layer_refuses_cpu_tensors_and_wrong_ranks():
    import torch
    from rag_amd.attention import packed_attention, packed_attention_backward
    q = torch.zeros(4, 2, 32, dtype=torch.bfloat16)
    off = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError):
        packed_attention(q, q, q, off)
    with pytest.raises(ValueError):
        packed_attention(q[0], q[0], q[0], off)
    with pytest.raises(ValueError):
        packed_attention_backward(q, q, q, q, q, torch.zeros(2, 4), off)


@pytest.mark.parametrize("causal", [False, True])
def test_reference_gradients_against_differences(causal):
    """The formulas the kernels are held to, against central differences of the forward formula, all in 64 bits."""
    import torch
    from tests._attention_ref import reference
    torch.manual_seed(1)
    lens, H, Hk, D = [5, 0, 1, 9], 4, 2, 8
    T = sum(lens) + 2
    x = {n: torch.randn(T, h, D).bfloat16() for n, h in (("q", H), ("k", Hk), ("v", Hk), ("dout", H))}
    mask = torch.ones(T, dtype=torch.int32)
    mask[[2, 8, 9]] = 0
    table = torch.randn(8, H)
    kw = dict(lens=lens, causal=causal, scale=0.4, key_mask=mask, max_distance=6, bidirectional=not causal)
    ref = reference(x["q"], x["k"], x["v"], table=table, dout=x["dout"], **kw)

    def loss(change, t=table):
        y = dict(x)
        for n, d in change.items():
            y[n] = y[n].double() + d
        real = {n: v if v.dtype == torch.float64 else v.double() for n, v in y.items()}
        out = _forward(real["q"], real["k"], real["v"], t.double(), kw)
        return float((out * x["dout"].double()).sum())

    eps = 1e-5
    for n in ("q", "k", "v"):
        for _ in range(3):
            d = torch.randn(x[n].shape, dtype=torch.float64)
            diff = (loss({n: eps * d}) - loss({n: -eps * d})) / (2 * eps)
            assert abs(diff - float((ref["d" + n] * d).sum())) < 1e-6 * max(1.0, abs(diff))
    d = torch.randn(table.shape, dtype=torch.float64)
    diff = (loss({}, table.double() + eps * d) - loss({}, table.double() - eps * d)) / (2 * eps)
    assert abs(diff - float((ref["dtable"] * d).sum())) < 1e-6 * max(1.0, abs(diff))


def _forward(q, k, v, table, kw):
    import torch
    out, start = torch.zeros_like(q), 0
    for n in kw["lens"]:
        for i in range(n):
            js = [j for j in range(n) if kw["key_mask"][start + j] and (not kw["causal"] or j <= i)]
            for h in range(q.shape[1]):
                g = h // (q.shape[1] // k.shape[1])
                if js:
                    s = torch.stack([kw["scale"] * q[start + i, h] @ k[start + j, g] + table[bucket_of(j - i, table.shape[0], kw["max_distance"], kw["bidirectional"]), h] for j in js])
                    out[start + i, h] = torch.softmax(s, 0) @ torch.stack([v[start + j, g] for j in js])
        start += n
    return out


def test_position_bias_of_a_model():
    from rag_amd.encoder_weights import position_bias_from_state_dict
    import torch
    t = np.arange(12, dtype=np.float32).reshape(6, 2)
    cfg = {"num_attention_heads": 2, "relative_attention_num_buckets": 6}
    name = "encoder.relative_attention_bias.weight"
    assert position_bias_from_state_dict({}, {"num_attention_heads": 2}) is None
    for prefix in ("", "bert.", "0.auto_model."):
        got = position_bias_from_state_dict({prefix + name: t}, cfg)
        assert np.array_equal(got["bias_table"], t) and got["max_distance"] == 128 and got["bidirectional"]
    assert position_bias_from_state_dict({name: torch.from_numpy(t)}, {**cfg, "relative_attention_max_distance": 40})["max_distance"] == 40
    with pytest.raises(ValueError, match="hold no"):
        position_bias_from_state_dict({}, cfg)
    with pytest.raises(ValueError, match="shape"):
        position_bias_from_state_dict({name: t[:5]}, cfg)
