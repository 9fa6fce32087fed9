"""The operators on device memory at the edges of their ranges: numbers that are not finite, very large
and very small scales, sizes of one, errors of several calls at once. The bounds are derived as in
test_gpu_train_ops.py, whose helpers are used here."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import test_gpu_train_ops as ops  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def m(esm):
    model = esm.Model(0)
    yield model
    model.check_device()
    model.close()


# ---- attention: scores that are not finite ----------------------------------------------------------

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_bad_rows_of_short_sequences_are_written(m, kind, bad):
    """A sequence of one key tile (32 rows) has no second step to wait for, whatever its scores are."""
    for H, dh in ((2, 64), (3, 24)):
        lens = [70, 1, 20, 31, 32, 33, 64, 65, 40]
        spoiled = range(1, 8)
        cu, qkv, _ = ops.attention_inputs(lens, H, dh, kind, seed=200 + dh)
        c, d = cu.tolist(), H * dh
        out, lse = ops.run_forward(m, cu, qkv, H, 70)
        qkv2 = qkv.clone()
        qkv2[c[1]:c[8]] = bad
        out2, lse2 = ops.run_forward(m, cu, qkv2, H, 70)
        m.check_device()
        for b in range(len(lens)):
            at = slice(c[b], c[b + 1])
            if b in spoiled:
                assert not torch.isfinite(out2[at]).any() and not torch.isfinite(lse2[:, at]).any()
            else:
                assert torch.equal(out2[at], out[at]) and torch.equal(lse2[:, at], lse[:, at])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_a_bad_key_shows_in_every_row(m, kind, bad):
    """One key of one head is not finite, at every place of the first and of a later key tile: every query of that
    sequence and head has a score that is NaN or +inf, so no distribution; other heads and sequences do not see it."""
    H, dh = 3, 32
    places = list(range(64)) + [0, 5, 19, 31]
    lens = [96] * 64 + [32] * 4
    cu, qkv, _ = ops.attention_inputs(lens, H, dh, kind, seed=210)
    c, d = cu.tolist(), H * dh
    qkv[:, dh:dh + 8] = qkv[:, dh:dh + 8].abs() + 0.5   # head 1's queries: an infinite key scores +inf
    out, lse = ops.run_forward(m, cu, qkv, H, 96)
    ops.check_forward(cu, qkv, H, out, lse)
    qkv2 = qkv.clone()
    for b, at in enumerate(places):
        qkv2[c[b] + at, d + dh + b % 8] = bad
    out2, lse2 = ops.run_forward(m, cu, qkv2, H, 96)
    m.check_device()
    head = slice(dh, 2 * dh)
    rows = torch.isnan(out2[:, head]).all(1) & torch.isnan(lse2[1])
    assert rows.all(), f"finite in {(~rows).sum().item()} rows, the first of sequence {int(rows.logical_not().nonzero()[0]) // 96}"
    out2[:, head], lse2[1] = out[:, head], lse[1]
    assert torch.equal(out2, out) and torch.equal(lse2, lse)


@pytest.mark.parametrize("dim, heads", [(640, 10), (320, 20)])
def test_encoder_forward_of_a_short_sequence_with_nan(esm, dim, heads):
    """The encoder's own attention: heads of 64 and of 16 columns, 1 to 33 tokens, one of them NaN."""
    cfg = esm.EsmConfig(dim, 4 * dim, 1, heads, 33, 64, 0)
    tensors = esm.synth_fp32_tensors(cfg, seed=3)
    tensors["tok_emb"].reshape(33, dim)[10] = math.nan
    model = esm.Model(0)
    model.load_tensors(cfg, esm.DTYPE_FP32, tensors)
    model.reserve(64, 1, 64)
    for n in (1, 20, 32, 33):
        seq = np.full(n, 5, dtype=np.int32)
        assert np.isfinite(model.forward([seq])["logits"]).all()
        seq[-1] = 10
        logits = model.forward([seq])["logits"]   # a wait that gave up would raise here
        assert not np.isfinite(logits[0, n - 1]).any()
    model.check_device()
    model.close()
