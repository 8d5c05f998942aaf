"""GPU: gradients in fp16 whose upstream values are small, as a loss's mean makes them, or of very different sizes.

ds = p (dp - D) is rounded to fp16 for the products, whose normal range ends at 2^-14.  The kernels carry it times a power of two that
keeps a lane's largest ds between 2^10 and 2^15, so its rounding is relative whatever the size of dout.  A gradient is linear in dout, so
dout 2^-12 is held to the bounds of dout, 2^-12 times as large.  (Not to the same bits: where dout 2^-12 is subnormal the matrix unit's
sum of its products can differ in fp32's last bit, which the bounds count.)"""
import pytest

from tests._attention_ref import reference, worst
from tests.test_attention_gpu import _check, _make

pytestmark = pytest.mark.gpu
DOWN = 2.0 ** -12


def _inputs(lens, H, Hk, D, table, seed, up_k):
    """dout in steps of 2^-6, so that dout 2^-12 is exact in fp16.  q and k with one of them up_k times as large, the other as much smaller:
    the scores stay, dq (or dk) keeps out of fp16's subnormals."""
    x, off, tab = _make(lens, H, Hk, D, "fp16", table=table, seed=seed)
    x["dout"] = (x["dout"].float() * 64).round().div(64).half()
    x["k"], x["q"] = x["k"] * up_k, x["q"] / up_k
    small = (x["dout"].float() * DOWN).half()
    assert bool((small.float() / DOWN == x["dout"].float()).all())
    return x, off, tab, small


def _gradients(x, dout, off, **kw):
    from rag_amd.attention import packed_attention, packed_attention_backward
    out, lse = packed_attention(x["q"], x["k"], x["v"], off, return_lse=True, **kw)
    return dict(zip(("dq", "dk", "dv", "dtable"), packed_attention_backward(dout, x["q"], x["k"], x["v"], out, lse, off, **kw)))


@pytest.mark.parametrize("lens,H,Hk", [([4096], 2, 1), ([300, 17, 70, 1], 4, 2), ([150, 1, 0, 64, 33] * 27, 8, 4)], ids=["long", "few", "many"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("table", [0, 32])
def test_small_gradients_against_64_bits(lens, H, Hk, D, causal, table):
    """Within the bounds of the larger dout, 2^-12 times as large, and half a step of fp16's subnormals for the result itself."""
    for up_k in (128.0, 1 / 128.0):
        x, off, tab, small = _inputs(lens, H, Hk, D, table, D, up_k)
        got = _gradients(x, small, off, causal=causal, bias_table=tab)
        ref = reference(x["q"], x["k"], x["v"], lens, causal, D ** -0.5, None, tab, 128, not causal, x["dout"])
        for n in ("dq" if up_k > 1 else "dk",) + (("dtable",) if table else ()):
            r = {n: ref[n], n + "_tol": ref[n + "_tol"] + (2.0 ** -25 / DOWN if n != "dtable" else 0.0)}
            assert worst(got[n].float() / DOWN, r, n) <= 1.0, (n, up_k)


@pytest.mark.parametrize("lens,H,Hk", [([700, 90], 4, 2), ([150, 1, 0, 64, 250] * 20, 8, 4)], ids=["few", "many"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("causal,table", [(False, 0), (True, 0), (True, 32), (False, 32)])
@pytest.mark.parametrize("rising", [True, False])
def test_rows_of_very_different_sizes(lens, H, Hk, D, causal, table, rising):
    """dout and v grow (or fall) by 2^18 along a sequence: the power of two has to move in the middle of a walk."""
    import torch
    x, off, tab = _make(lens, H, Hk, D, "fp16", table=table, seed=D + rising)
    at = torch.cat([torch.arange(n) / max(n - 1, 1) for n in lens]).cuda()
    size = torch.exp2((at if rising else 1 - at) * 18 - 12)[:, None, None]
    x["dout"], x["v"] = (x["dout"].float() * size).half(), (x["v"].float() * size).half()
    _check(x, off, lens, tab=tab, causal=causal)


def test_the_largest_gradients_stay_finite():
    """ds itself is beyond fp16's range, the gradients are not: the power of two goes below 1."""
    import torch
    lens = [130, 40]
    for D in (32, 64, 128):
        x, off, _ = _make(lens, 4, 2, D, "fp16", seed=D)
        x["v"], x["dout"] = x["v"] * 1024, x["dout"] * 1024
        x["q"], x["k"] = x["q"] / 128, x["k"] / 256
        got, ref = _check(x, off, lens, scale=0.5)
        assert float(ref["dk"].abs().max()) > 1000 and torch.isfinite(got["dk"]).all()
