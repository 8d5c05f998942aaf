"""GPU: encoders with causal attention and / or a relative position bias (mi_encoder_set_attention) against a plain 64-bit encoder:
the projections, packed attention and the head run together, padded and packed, at latency and bulk sizes.

Tolerances: embeddings within 1e-3 in cosine, the bar of every encoder test here (hidden states are bf16 between kernels, 2^-8 relative
per rounding, averaged over the tokens); logits as in test_rerank_gpu.py.  A model with the wrong attention is 1e-2 and more away, which
each test checks as well."""
import json
import os

import numpy as np
import pytest

from tests._attention_ref import bucket_of

pytestmark = pytest.mark.gpu
TOL = 1e-3
FORMS = {"causal": (True, 0, 128), "bias": (False, 32, 128), "causal_bias": (True, 8, 20)}


def _table(buckets, heads, seed=4):
    return (np.random.default_rng(seed).standard_normal((buckets, heads)) * 3).astype(np.float32) if buckets else None


def _form(name, heads):
    causal, buckets, dist = FORMS[name]
    return {"causal": causal, "bias_table": _table(buckets, heads), "max_distance": dist}


def _bert64(cfg, blob, ids, types=None, causal=False, bias_table=None, max_distance=128):
    """Hidden states [n][H] of one sequence, float64."""
    from scipy.special import erf
    from rag_amd.encoder_weights import unpack_blob
    w = {k: v.astype(np.float64) for k, v in unpack_blob(cfg, blob).items()}
    n, nh = len(ids), cfg.num_attention_heads
    dh = cfg.hidden_size // nh

    def ln(x, p):
        x = x - x.mean(-1, keepdims=True)
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + cfg.layer_norm_eps) * w[p + ".weight"] + w[p + ".bias"]

    def lin(x, p):
        return x @ w[p + ".weight"].T + w[p + ".bias"]

    types = np.zeros(n, dtype=np.int64) if types is None else types
    h = ln(w["embeddings.word_embeddings.weight"][ids] + w["embeddings.position_embeddings.weight"][:n] +
           w["embeddings.token_type_embeddings.weight"][types], "embeddings.LayerNorm")
    rel = np.arange(n)[None, :] - np.arange(n)[:, None]
    add = np.zeros((nh, n, n))
    if bias_table is not None:
        num = np.array([bucket_of(int(r), bias_table.shape[0], max_distance, not causal) for r in range(-n + 1, n)])
        add = bias_table.astype(np.float64)[num[rel + n - 1]].transpose(2, 0, 1)
    if causal:
        add = np.where(rel > 0, -np.inf, add)
    for l in range(cfg.num_hidden_layers):
        p = f"encoder.layer.{l}."
        q, k, v = (lin(h, p + "attention.self." + x).reshape(n, nh, dh).transpose(1, 0, 2) for x in ("query", "key", "value"))
        s = q @ k.transpose(0, 2, 1) * dh ** -0.5 + add
        s = np.exp(s - s.max(-1, keepdims=True))
        a = (s / s.sum(-1, keepdims=True)) @ v
        h = ln(h + lin(a.transpose(1, 0, 2).reshape(n, -1), p + "attention.output.dense"), p + "attention.output.LayerNorm")
        m = lin(h, p + "intermediate.dense")
        h = ln(h + lin(0.5 * m * (1 + erf(m / np.sqrt(2))), p + "output.dense"), p + "output.LayerNorm")
    return h


def _embed64(cfg, blob, ids, **form):
    e = _bert64(cfg, blob, ids, **form).mean(0)
    return e / np.linalg.norm(e)


def _cos_err(a, b):
    a, b = a.astype(np.float64), np.asarray(b, dtype=np.float64)
    return 1 - (a * b).sum(-1) / np.linalg.norm(a, axis=-1) / np.linalg.norm(b, axis=-1)


def _encoder(heads=4, layers=2, seed=11, normalize=1):
    from rag_amd._capi import BertConfig
    from rag_amd.embeddings import Encoder
    from rag_amd.encoder_weights import random_blob
    cfg = BertConfig(700, 32 * heads, layers, heads, 4 * 32 * heads, 300, 2, 1e-12, normalize)
    blob = random_blob(cfg, seed=seed, init_range=0.15)
    return cfg, blob, Encoder(cfg, blob)


def _batch(lens, L, seed=1):
    rng = np.random.default_rng(seed)
    ids, mask = np.zeros((len(lens), L), dtype=np.int32), np.zeros((len(lens), L), dtype=np.int32)
    for i, n in enumerate(lens):
        ids[i, :n] = rng.integers(1, 700, size=n)
        mask[i, :n] = 1
    return ids, mask


@pytest.mark.parametrize("heads", [4, 12])
@pytest.mark.parametrize("form", list(FORMS))
def test_padded_packed_and_allocation_free_passes(form, heads):
    import torch
    cfg, blob, enc = _encoder(heads)
    lens = [1, 2, 31, 32, 33, 64, 100, 129, 203]
    ids, mask = _batch(lens, 203)
    plain = enc.encode_ids(ids, mask)
    f = _form(form, heads)
    enc.set_attention(**f)
    want = np.stack([_embed64(cfg, blob, ids[i, :n], **f) for i, n in enumerate(lens)])
    got = enc.encode_ids(ids, mask)
    assert np.all(_cos_err(got, want) < TOL), _cos_err(got, want)
    assert np.any(_cos_err(plain[2:], want[2:]) > 10 * TOL)
    flat = np.concatenate([ids[i, :n] for i, n in enumerate(lens)])
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
    assert np.all(_cos_err(enc.encode_ragged(flat, off), want) < TOL)
    dev = [torch.from_numpy(x[:6, :64].copy()).cuda() for x in (ids, mask)]
    small = enc.encode_ids_torch_noalloc(*dev).cpu().numpy()
    assert np.all(_cos_err(small, want[:6]) < TOL)
    enc.set_attention()
    assert np.array_equal(enc.encode_ids(ids, mask), plain)


def test_bulk_pass_of_many_sequences():
    cfg, blob, enc = _encoder(12, layers=1)
    f = _form("causal_bias", 12)
    enc.set_attention(**f)
    rng = np.random.default_rng(3)
    lens = rng.integers(1, 257, size=700)
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
    flat = rng.integers(0, 700, size=int(off[-1])).astype(np.int32)
    got = enc.encode_ragged(flat, off)                 # 90,000 tokens: several passes, on both lanes
    for i in range(0, 700, 35):
        assert _cos_err(got[i], _embed64(cfg, blob, flat[off[i]:off[i + 1]], **f)) < TOL, i
    ids, mask = _batch([256] * 100, 256)
    assert _cos_err(enc.encode_ids(ids, mask)[17], _embed64(cfg, blob, ids[17], **f)) < TOL


def test_classification_with_a_bias():
    from rag_amd.encoder_weights import random_head
    from tests.test_rerank_gpu import _logit_tol
    cfg, blob, enc = _encoder(4, normalize=0)
    head = random_head(cfg, num_labels=2, seed=7, init_range=0.1)
    enc.set_head(*head)
    f = _form("bias", 4)
    enc.set_attention(**f)
    lens = [3, 40, 77, 150]
    ids, mask = _batch(lens, 150)
    types = (np.arange(150)[None, :] >= 12).astype(np.int32) * mask
    got = enc.classify(ids, types, mask)
    want = np.stack([np.tanh(_bert64(cfg, blob, ids[i, :n], types[i, :n], **f)[0] @ head[0].T.astype(np.float64) + head[1]) @ head[2].T + head[3]
                     for i, n in enumerate(lens)])
    assert np.abs(got - want).max() < _logit_tol(head[0], head[2])


def test_a_captured_pass_replays_and_reads_the_current_table():
    import torch
    cfg, blob, enc = _encoder(4)
    f = _form("bias", 4)
    enc.set_attention(**f)
    ids, mask = _batch([9, 30, 48], 48)
    dev = [torch.from_numpy(x).cuda() for x in (ids, mask)]
    out = enc.encode_ids_torch_noalloc(*dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        enc.encode_ids_torch_noalloc(*dev, out)
    for seed in (4, 5, 6):
        f["bias_table"] = _table(32, 4, seed)
        torch.cuda.synchronize()
        enc.set_attention(**f)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, enc.encode_ids_torch(*dev))
        assert _cos_err(got.cpu().numpy()[2], _embed64(cfg, blob, ids[2], **f)) < TOL


def test_refusals_leave_the_encoder_as_it_was():
    from rag_amd import MI355Error
    cfg, blob, enc = _encoder(4)
    ids, mask = _batch([9, 30], 30)
    before = enc.encode_ids(ids, mask)
    for t in (np.zeros((8, 5)), np.zeros(8), np.zeros((0, 4))):
        with pytest.raises(ValueError):
            enc.set_attention(bias_table=t)
    for kw in ({"bias_table": np.zeros((66, 4))}, {"bias_table": np.zeros((7, 4))}, {"bias_table": np.zeros((32, 4)), "max_distance": 8},
               {"bias_table": np.zeros((32, 4)), "max_distance": 1025}):
        with pytest.raises(MI355Error):
            enc.set_attention(**kw)
    assert np.array_equal(enc.encode_ids(ids, mask), before)


def test_a_model_directory_with_a_bias(tmp_path):
    from safetensors.numpy import load_file, save_file
    from rag_amd import HuggingFaceEmbeddings
    from rag_amd.encoder_weights import load_local_dir
    from tests.test_retrievers import _write_model_dir
    path = str(tmp_path / "m")
    cfgd, _ = _write_model_dir(path)
    table = _table(16, 4)
    sd = load_file(os.path.join(path, "model.safetensors"))
    sd["bert.encoder.relative_attention_bias.weight"] = table
    save_file(sd, os.path.join(path, "model.safetensors"))
    with open(os.path.join(path, "config.json"), "w") as f:
        json.dump({**cfgd, "relative_attention_num_buckets": 16, "relative_attention_max_distance": 40}, f)
    cfg, blob = load_local_dir(path)
    text = "the cat sat on mat dogs chase red was flat index row the cat sat"
    for causal in (False, True):
        emb = HuggingFaceEmbeddings(model_name=path, model_kwargs={"device": 0, "causal": causal})
        ids = np.array(emb._tokenize([text])[0])
        # the loader's table has buckets for both directions, whether the model is causal or not
        h = _embed_both(cfg, blob, ids, table, 40, causal)
        assert _cos_err(np.array(emb.embed_query(text)), h) < TOL
        assert _cos_err(np.array(emb.embed_documents([text])[0]), h) < TOL


def _embed_both(cfg, blob, ids, table, dist, causal):
    if not causal:
        return _embed64(cfg, blob, ids, bias_table=table, max_distance=dist)
    # one-sided table of the same numbers: with d < side, bucket(d behind) of the two-sided scheme is its first half
    half = table[:table.shape[0] // 2]
    return _embed64(cfg, blob, ids, causal=True, bias_table=half, max_distance=dist)
