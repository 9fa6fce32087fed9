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
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_backward_of_bad_short_sequences_stays_alone(m, kind, bad):
    """Gradients of a spoiled sequence are not finite, and those of its neighbours what they were."""
    for H, dh in ((2, 64), (3, 24)):
        lens = [70, 1, 20, 31, 32, 33, 64, 65, 40]
        cu, qkv, dout = ops.attention_inputs(lens, H, dh, kind, seed=260 + dh)
        c, d = cu.tolist(), H * dh
        out, lse = ops.run_forward(m, cu, qkv, H, 70)
        dqkv = ops.run_backward(m, cu, qkv, H, 70, out, lse, dout)
        qkv2 = qkv.clone()
        qkv2[c[1]:c[8], d:] = bad                     # keys and values
        out2, lse2 = ops.run_forward(m, cu, qkv2, H, 70)
        dqkv2 = ops.run_backward(m, cu, qkv2, H, 70, out2, lse2, dout)
        m.check_device()
        assert torch.equal(dqkv2[:c[1]], dqkv[:c[1]]) and torch.equal(dqkv2[c[8]:], dqkv[c[8]:])
        assert not torch.isfinite(dqkv2[c[1]:c[8]]).any()


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


def check_exact_scores(cu, qkv, H, out, lse, scale):
    """Where every score is a multiple of its last bit in fp32, the products are exact, and exponentials take the
    difference to the maximum, which is exact too: the probabilities are as good as those of small scores."""
    U, d = ops.half_step(qkv.dtype), qkv.shape[1] // 3
    for a, b in ops.sequences(cu):
        q, k, v = (ops.split_heads(x, H) for x in qkv[a:b].split(d, 1))
        s = scale * q @ k.transpose(-1, -2)
        assert torch.equal((s / scale).float().double() * scale, s)
        want_lse = torch.logsumexp(s, -1)
        p = torch.softmax(s, -1)
        # Exponentials and their arguments (down to e^-40; below, they are less than U of nothing), sums of b - a terms.
        rel = 2.0 ** -20 + 40 * 4 * ops.E + (b - a) * ops.E
        want = p @ v
        ops.within(ops.split_heads(out[a:b], H), want, (U + rel) * (p @ v.abs()) + U * want.abs() + 2.0 ** -25, "out")
        ops.within(lse[:, a:b], want_lse, 8 * ops.E * want_lse.abs() + rel, "lse")


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("terms, step", [(1, 2.0 ** -7), (2, 2.0 ** 6), (8, 2.0 ** 8), (32, 2.0 ** 10)])
def test_attention_large_scores(m, kind, sign, terms, step):
    """Scores whose maximum is 2^19 to 2^31, where its product with log2 e rounds by up to 128, and whose
    differences are a few bits of that, beside rows with ordinary scores."""
    dh, lens = 64, [1, 20, 33, 150]
    T = sum(lens)
    cu, qkv, _ = ops.attention_inputs(lens, 1, dh, kind, seed=220)
    q, k = qkv[:, :dh], qkv[:, dh:2 * dh]
    q.zero_(), k.zero_()
    big = 2.0 ** 7 if terms == 1 else 2.0 ** 14
    q[:, :terms] = sign * big
    k[:, :terms] = big
    at = torch.arange(T, device="cuda")
    q[:, 40] = step                                  # S = sign * terms * big^2 + step * (0 .. 7)
    k[:, 40] = ((at * 5) % 8).to(k.dtype)
    q[3::7, :terms] = 0.0                            # ordinary rows in the same warps
    for scale in (0.25 / step, 1.0 / step, 16.0 / step, 256.0 / step):
        out, lse = ops.run_forward(m, cu, qkv, 1, 150, scale=scale)
        m.check_device()
        check_exact_scores(cu, qkv, 1, out, lse, scale)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_maximum_grows_through_large_scores(m, kind):
    """Key tiles whose scores rise from -2^24 through ordinary ones to 2^24 (log2), and fall again."""
    dh, L = 32, 300
    cu, qkv, _ = ops.attention_inputs([L], 1, dh, kind, seed=221)
    q, k = qkv[:, :dh], qkv[:, dh:2 * dh]
    q.zero_(), k.zero_()
    steps = [-2.0 ** 12, -2.0 ** 9, -8.0, -1.0, 0.0, 1.0, 2.0 ** 9, 2.0 ** 12, 2.0 ** 12, 2.0 ** 9]
    k[:, 0] = torch.tensor(steps, device="cuda").repeat_interleave(32)[:L].to(k.dtype)
    q[0::3, 0], q[1::3, 0], q[2::3, 0] = 2.0 ** 12, -2.0 ** 12, 1.0
    out, lse = ops.run_forward(m, cu, qkv, 1, L, scale=1.0)
    check_exact_scores(cu, qkv, 1, out, lse, 1.0)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("ruled_out", [1, 31, 32, 33, 64, 99])
def test_attention_scores_of_minus_infinity(m, kind, ruled_out):
    """Keys whose scores are -inf have no part in the result, also when they fill the first key tiles; a row that has
    nothing else has no distribution."""
    H, dh, L = 2, 24, 100
    cu, qkv, _ = ops.attention_inputs([L, 40, L], H, dh, kind, seed=222)
    d = H * dh
    qkv[:, :d] = qkv[:, :d].abs() + 0.25
    rest = qkv.clone()
    qkv[:ruled_out, d + 3] = -math.inf               # head 0 of the first sequence
    qkv[L + 40:, d + dh:2 * d] = -math.inf           # head 1 of the last one, every key
    out, lse = ops.run_forward(m, cu, qkv, H, L)
    m.check_device()
    other, other_lse = ops.run_forward(m, cu, rest, H, L)
    assert torch.isnan(out[L + 40:, dh:]).all() and (lse[1, L + 40:] == -math.inf).all()
    q, k, v = (x[:, 0] for x in rest[:L].double().unflatten(1, (3, H, dh)).unbind(1))
    s = dh ** -0.5 * q @ k[ruled_out:].t()
    p = torch.softmax(s, 1)
    es = ops.score_error(q, k, dh ** -0.5).amax()
    want = p @ v[ruled_out:]
    rel = ops.half_step(qkv.dtype) + 2 * es + 2.0 ** -19
    ops.within(out[:L, :dh], want, rel * (p @ v[ruled_out:].abs()) + ops.half_step(qkv.dtype) * want.abs() + 2.0 ** -25, "out")
    ops.within(lse[0, :L], torch.logsumexp(s, 1), es + 2.0 ** -19 + 8 * ops.E * s.abs().amax(1), "lse")
    out[:L, :dh], lse[0, :L] = other[:L, :dh], other_lse[0, :L]
    out[L + 40:, dh:], lse[1, L + 40:] = other[L + 40:, dh:], other_lse[1, L + 40:]
    assert torch.equal(out, other) and torch.equal(lse, other_lse)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n", range(20, 30))
def test_attention_backward_of_large_scores(m, kind, n):
    """lse / scale of every query spread over [2^n, 2^(n+1)) up to 1e9: it reaches the key items in parts of 16 bits."""
    dh, lens, scale = 64, [200, 33], 2.0 ** -19
    T = sum(lens)
    cu, qkv, dout = ops.attention_inputs(lens, 1, dh, kind, seed=230 + n)
    q, k = qkv[:, :dh], qkv[:, dh:2 * dh]
    q.zero_(), k.zero_()
    top = 2.0 ** 16 if n < 29 else 1.8 * 2.0 ** 15
    at = torch.arange(T, device="cuda")
    q[:, 0] = (2.0 ** 15 + (top - 2.0 ** 15) * ((at * 0.6180339887) % 1.0)).clamp(max=65000).to(q.dtype)
    q[:, 1] = (at * 37 % 256 * 8).to(q.dtype)
    q[:, 2] = 16.0
    k[:, 0], k[:, 1] = 2.0 ** (n - 15), 2.0 ** (n - 21)
    k[:, 2] = (12000 * ops.randn(231, T)).to(k.dtype)       # scores that differ by about 0.4
    out, lse = ops.run_forward(m, cu, qkv, 1, 200, scale=scale)
    ops.check_forward(cu, qkv, 1, out, lse, scale)
    dqkv = ops.run_backward(m, cu, qkv, 1, 200, out, lse, dout, scale=scale)
    ops.check_backward(cu, qkv, 1, out, lse, dout, dqkv, scale)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("grad", [1e-5, 1e-3, 0.05])
def test_attention_backward_of_small_sums(m, kind, grad):
    """Sums of dout out far below 1 beside large queries and keys: dS is a difference of them, and 0 for a single key."""
    for H, dh in ((3, 64), (200, 16), (500, 8)):
        lens = [1] * 20 + [2, 3, 40]
        cu, qkv, dout = ops.attention_inputs(lens, H, dh, kind, seed=245, grad=grad)
        qkv[:, :2 * H * dh] *= 30.0
        scale = 0.01 / dh
        out, lse = ops.run_forward(m, cu, qkv, H, 40, scale=scale)
        dqkv = ops.run_backward(m, cu, qkv, H, 40, out, lse, dout, scale=scale)
        ops.check_backward(cu, qkv, H, out, lse, dout, dqkv, scale)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("terms", [1, 2, 3])
def test_attention_backward_of_large_sums(m, kind, terms):
    """Sums of dout out up to 1e9, beside which the rest of dS is small."""
    dh, lens = 64, [150, 40]
    T = sum(lens)
    cu, qkv, dout = ops.attention_inputs(lens, 1, dh, kind, seed=240)
    v = qkv[:, 2 * dh:]
    v[:, :terms] = 2.0 ** 15
    dout[:, :terms] = (2.0 ** 13 * (0.51 + 0.48 * torch.rand(T, 1, device="cuda", generator=torch.Generator(device="cuda").manual_seed(241)))).to(dout.dtype)
    dout[:, 10:] *= 2.0 ** 12
    out, lse = ops.run_forward(m, cu, qkv, 1, 150)
    dqkv = ops.run_backward(m, cu, qkv, 1, 150, out, lse, dout)
    ops.check_backward(cu, qkv, 1, out, lse, dout, dqkv)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("lens", [[1, 5, 31, 32, 33], [257, 64], [700]], ids=str)
def test_attention_exponentials_are_exact_to_32_bits(m, monkeypatch, kind, lens):
    """The bounds of the helpers with what the operator's exponentials have: 2^-21, the exp2 instruction's 2^-22 or
    the polynomial's 2.2e-7 with their rounding, and sums of 32 of a row's columns at a time, then over the steps."""
    monkeypatch.setattr(ops, "X", 2.0 ** -21 + (32 + 3 * max(lens) / 32) * ops.E)
    for H, dh in ((3, 64), (2, 24)):
        cu, qkv, dout = ops.attention_inputs(lens, H, dh, kind, seed=250 + dh)
        out, lse = ops.run_forward(m, cu, qkv, H, max(lens))
        ops.check_forward(cu, qkv, H, out, lse)
        ops.check_backward(cu, qkv, H, out, lse, dout, ops.run_backward(m, cu, qkv, H, max(lens), out, lse, dout))


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


# ---- distillation: temperatures and large logits --------------------------------------------------------

def check_soft(x, ids, top, dloss, tau, loss, lse, dx):
    """check_distill with bounds that do not grow with |x| / tau: exponents are differences to the row's maximum,
    each with a relative error of 4 E, and 2^-21 in the exponential; lse and the loss are rounded once more."""
    V = x.shape[1]
    U = ops.half_step(x.dtype)
    want, want_lse, q, p, any_, _, _ = ops.distill_64(x, ids, top, tau)
    sums = (V / 32 + 64) * ops.E + 2.0 ** -20
    far = ((x.double() - x.double().amax(1, keepdim=True)) / tau).abs()
    eq = q * (sums + torch.where(q > 0, 8 * ops.E * far.clamp(max=200), 0.0) + 2.0 ** -17) + 1e-38
    there = (ids >= 0) & (ids < V)
    t = torch.where(there, top.double(), -math.inf) / tau
    far_t = torch.where(p.sum(1, keepdim=True) > 0, (t.amax(1, keepdim=True) - t).clamp(max=200), 0.0).amax(1, keepdim=True)
    ep = p * (2.0 ** -20 + 64 * ops.E + 8 * ops.E * far_t)
    g = (dloss.double() * tau * any_)[:, None]
    wx = g * (q - p)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 1e-38
    ops.within(dx, wx, U * wx.abs() + g.abs() * (eq + ep + 2 * ops.E * (q + p)) + tiny, "dlogits")
    ops.within(lse, want_lse, sums + 4 * ops.E * (x.double().amax(1) / tau).abs() + 4 * ops.E * want_lse.abs(), "lse")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V, k", [(33, 16), (33, 33), (64, 20), (65, 5), (1500, 32), (40000, 64)])
@pytest.mark.parametrize("tau", [1e-6, 1e-3, 0.05, 1.0])
def test_distill_gradient_at_low_temperatures_and_large_logits(m, kind, V, k, tau):
    """Rows around 20, 1000 and 0, with the row's spread a few tau where the type has such differences, and tied maxima."""
    T = 21
    step = {"f32": 2.0 ** -19, "f16": 2.0 ** -6, "bf16": 2.0 ** -3}[kind]  # the last bit of numbers around 20
    spread = max(step, tau)
    x = 20.0 + (3 * ops.randn(300 + V, T, V) * spread / step).round() * step
    x[::3] -= 20.0
    x[1::3] += 980.0
    x[5] = 20.0                     # all tied
    x[6, 1:4] = x[6].max() + 8 * spread   # three tied maxima far above the rest
    x = x.to(ops.KINDS[kind])
    top, ids = (x.float() + 1.5 * spread * ops.randn(301, T, V)).topk(k, 1)
    ids = ids.to(torch.int32)
    if k > 2:
        ids[1::4, k // 2:] = -1
    dloss = ops.randn(302, T)
    dloss[::5] = 0
    got = ops.run_distill(m, x, ids, top.contiguous(), dloss / tau, tau)
    check_soft(x, ids, top, dloss / tau, tau, *got)


def test_distill_tied_maxima_share_their_probability(m):
    for V in (33, 2000):
        x = torch.full((3, V), -5.0, device="cuda")
        x[:, 7] = x[:, 11] = 20.0
        ids, top = torch.tensor([[3]] * 3, dtype=torch.int32, device="cuda"), torch.zeros(3, 1, device="cuda")
        dloss = torch.full((3,), 1e6, device="cuda")
        _, _, dx = ops.run_distill(m, x, ids, top, dloss, 1e-6)
        want = torch.zeros(V, device="cuda")
        want[7] = want[11] = 0.5
        want[3] = -1.0
        assert torch.allclose(dx, want.expand(3, V), rtol=1e-5, atol=0)


@pytest.mark.parametrize("V", [33, 60, 500])
@pytest.mark.parametrize("tau", [10.0, 100.0])
def test_distill_loss_at_high_temperatures(m, V, tau):
    """The loss tends to half the variance of the logits' differences: a sum of order tau^-2 of terms of order 1, whose
    rounding is at most 2^-18: sums of V terms as in check_logprobs, two logarithms of at most log V, and their difference."""
    k = min(V, 60)
    x = 3 * ops.randn(310, 50, V)
    x[:, k:] -= 1000.0 * tau          # only the alternatives count
    ids = torch.arange(k, dtype=torch.int32, device="cuda").expand(50, k).contiguous()
    top = (x[:, :k] + ops.randn(311, 50, k)).contiguous()
    dloss = torch.ones(50, device="cuda")
    loss, lse, dx = ops.run_distill(m, x, ids, top, dloss, tau)
    want = ops.distill_64(x, ids, top, tau)[0]
    ops.within(loss, want, tau * tau * 2.0 ** -18 + 8 * ops.E * want.abs(), "loss")
    check_soft(x, ids, top, dloss, tau, loss, lse, dx)


def test_distill_refuses_temperatures_that_fp32_does_not_support(esm, m):
    x, ids, top, dloss = ops.distill_inputs(4, 33, 3, "f32", seed=99)
    for tau in (1e-7, 9.9e-7, 100.1, 1e3, 1e6):
        s, l = torch.full((4,), 7.0, device="cuda"), torch.full((4,), 7.0, device="cuda")
        with pytest.raises(esm.EsmError, match="temperature must be in") as e:
            m.distill_loss(x, ids, top, s, l, temperature=tau)
        assert e.value.code == esm.ESM_EINVAL
        with pytest.raises(esm.EsmError, match="temperature must be in"):
            m.distill_backward(x, ids, top, l, dloss, torch.empty_like(x), temperature=tau)
        assert (s == 7).all() and (l == 7).all()


@pytest.mark.parametrize("V", [33, 50, 300, 5000])
@pytest.mark.parametrize("k", [1, 3, 20, 33])
def test_distill_a_teacher_of_nan_alone_shows(m, V, k):
    """Rows whose present alternatives are all NaN, or NaN and -inf, are not rows without alternatives."""
    x = ops.logits_of(6, V, "f32", seed=320)
    ids = torch.arange(k, dtype=torch.int32, device="cuda").expand(6, k).contiguous()
    top = torch.full((6, k), math.nan, device="cuda")
    top[1, 1:] = -math.inf
    ids[2, : k - 1] = -1
    top[3] = 0.5
    top[4] = -math.inf
    ids[5] = V
    loss, lse, dx = ops.run_distill(m, x, ids, top, torch.ones(6, device="cuda"), 2.0)
    assert torch.isnan(loss[:3]).all() and torch.isfinite(loss[3]) and (loss[4:] == 0).all()
    for row in range(3):
        assert torch.isnan(dx[row, ids[row][ids[row] >= 0].long()]).any()
    assert torch.isfinite(dx[3]).all() and (dx[4:] == 0).all() and torch.isfinite(lse).all()


# ---- layouts ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("T", [1, 2, 77])
def test_attention_on_column_blocks_of_one_matrix(m, T):
    """qkv, out, dout and dqkv side by side in one matrix: their address ranges interlock, their elements do not."""
    H, dh = 2, 24
    d = H * dh
    cu, qkv, dout = ops.attention_inputs([T], H, dh, "f16", seed=400)
    out, lse = ops.run_forward(m, cu, qkv, H, T)
    dqkv = ops.run_backward(m, cu, qkv, H, T, out, lse, dout)
    store = torch.full((T, 8 * d + 8), 7.0, dtype=torch.float16, device="cuda")
    out2, qkv2, dqkv2, dout2 = store[:, :d], store[:, d:4 * d], store[:, 4 * d:7 * d], store[:, 7 * d:8 * d]
    qkv2.copy_(qkv), dout2.copy_(dout)
    lse2 = torch.empty_like(lse)
    ws = torch.empty(m.attention_backward_workspace(1, T, H), dtype=torch.uint8, device="cuda")
    m.attention(qkv2, cu, T, H, out2, lse2)
    m.attention_backward(qkv2, cu, T, H, out2, lse2, dout2, dqkv2, ws)
    assert torch.equal(out2, out) and torch.equal(lse2, lse) and torch.equal(dqkv2, dqkv)
    assert torch.equal(qkv2, qkv) and torch.equal(dout2, dout) and (store[:, 8 * d:] == 7.0).all()


def test_attention_of_one_row_takes_any_stride(m, esm):
    """No second row starts anywhere: the stride need not be a multiple of 16 bytes."""
    H, dh = 2, 8
    d = H * dh
    cu, qkv, dout = ops.attention_inputs([1], H, dh, "f16", seed=403)
    out, lse = ops.run_forward(m, cu, qkv, H, 1)
    dqkv = ops.run_backward(m, cu, qkv, H, 1, out, lse, dout)
    L, scale = esm.lib(), dh ** -0.5
    out2, lse2, dqkv2 = torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(dqkv)
    size = m.attention_backward_workspace(1, 1, H)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    for odd in (1, 3, 2 ** 33 + 1):
        rc = L.esm_attention(m._ctx, esm.TYPE_F16, qkv.data_ptr(), 3 * d + odd, cu.data_ptr(), 1, 1, 1, H, dh, scale,
                             out2.data_ptr(), d + odd, lse2.data_ptr(), None)
        assert rc == esm.ESM_OK, L.esm_last_error(m._ctx).decode()
        rc = L.esm_attention_backward(m._ctx, esm.TYPE_F16, qkv.data_ptr(), 3 * d + odd, cu.data_ptr(), 1, 1, 1, H, dh, scale,
                                      out2.data_ptr(), d + odd, lse2.data_ptr(), dout.data_ptr(), d + odd, dqkv2.data_ptr(),
                                      3 * d + odd, ws.data_ptr(), size, None)
        assert rc == esm.ESM_OK, L.esm_last_error(m._ctx).decode()
        assert torch.equal(out2, out) and torch.equal(lse2, lse) and torch.equal(dqkv2, dqkv)


def test_attention_of_the_most_heads(m):
    for kind, dh in (("f16", 8), ("bf16", 16)):
        H, lens = 65535, [2, 1]
        cu, qkv, dout = ops.attention_inputs(lens, H, dh, kind, seed=404)
        out, lse = ops.run_forward(m, cu, qkv, H, 2)
        dqkv = ops.run_backward(m, cu, qkv, H, 2, out, lse, dout)
        m.check_device()
        ops.check_forward(cu, qkv, H, out, lse)
        ops.check_backward(cu, qkv, H, out, lse, dout, dqkv)


def test_optional_statistics(m):
    """lse, mean and rstd may be left out; the results are the same."""
    cu, qkv, _ = ops.attention_inputs([40, 300], 3, 40, "bf16", seed=405)
    out, _ = ops.run_forward(m, cu, qkv, 3, 300)
    out2 = torch.empty_like(out)
    m.attention(qkv, cu, 300, 3, out2, stream=torch.cuda.current_stream())
    assert torch.equal(out, out2)
    for d in (64, 9001):
        x, w, b = ops.ln_inputs(50, d, "f32", seed=406)
        y, mean, rstd = ops.run_ln(m, x, w, b, "f16")
        y2 = torch.empty_like(y)
        m.layernorm(x, w, b, y2)
        assert torch.equal(y, y2)


@pytest.mark.parametrize("handle", [None, 0, 1, 2])
def test_streams_by_their_special_handles(m, handle):
    """The legacy default stream (null, cudaStreamLegacy) and the per-thread one."""
    cu, qkv, dout = ops.attention_inputs([40, 300], 3, 32, "f16", seed=407)
    out, lse = ops.run_forward(m, cu, qkv, 3, 300)
    dqkv = ops.run_backward(m, cu, qkv, 3, 300, out, lse, dout)
    out2, lse2, dqkv2 = torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(dqkv)
    ws = torch.empty(m.attention_backward_workspace(2, 340, 3), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    m.attention(qkv, cu, 300, 3, out2, lse2, stream=handle)
    m.attention_backward(qkv, cu, 300, 3, out2, lse2, dout, dqkv2, ws, stream=handle)
    torch.cuda.synchronize()
    assert torch.equal(out2, out) and torch.equal(lse2, lse) and torch.equal(dqkv2, dqkv)


def test_distill_gradient_beside_the_logits(m):
    x, ids, top, dloss = ops.distill_inputs(40, 33, 5, "f32", seed=401)
    want = ops.run_distill(m, x, ids, top, dloss, 1.0)
    store = torch.full((40, 70), 7.0, device="cuda")
    grad, logits = store[:, 1:34], store[:, 34:67]
    logits.copy_(x)
    loss, lse = torch.empty(40, device="cuda"), torch.empty(40, device="cuda")
    m.distill_loss(logits, ids, top, loss, lse)
    m.distill_backward(logits, ids, top, lse, dloss, grad)
    assert torch.equal(grad, want[2]) and torch.equal(logits, x) and (store[:, 0] == 7).all() and (store[:, 67:] == 7).all()


def test_column_blocks_that_share_elements_are_refused(m, esm):
    T, V = 9, 33
    x, ids, top, dloss = ops.distill_inputs(T, V, 5, "f32", seed=402)
    lse = torch.zeros(T, device="cuda")
    store = torch.zeros(T + 2, 70, device="cuda")

    def refused(logits, grad):
        for a, b in ((logits, grad), (grad, logits)):
            with pytest.raises(esm.EsmError, match="overlap") as e:
                m.distill_backward(a, ids, top, lse, dloss, b)
            assert e.value.code == esm.ESM_EINVAL

    rows = store[:T]
    refused(rows[:, :33], rows[:, 32:65])                 # one column in common
    refused(rows[:, :33], store[1:T + 1, 20:53])          # the same, a row further
    refused(rows[:, :33], store.view(-1)[70 + 52:].as_strided((T, 33), (70, 1)))   # its row's end meets the next row's start
    refused(rows[:, :33], store.view(-1)[37:].as_strided((T, 33), (69, 1)))          # other strides: not told apart


# ---- errors that are found on the device --------------------------------------------------------------

@pytest.fixture
def encoder(esm):
    cfg = esm.EsmConfig(320, 1280, 1, 20, 33, 64, 0)
    model = esm.Model(0)
    model.load_tensors(cfg, esm.DTYPE_FP32, esm.synth_fp32_tensors(cfg, seed=3))
    model.reserve(100, 4, 64)
    yield model
    model.close()


def bad_offsets(model):
    _, qkv, _ = ops.attention_inputs([64], 2, 16, "f16", seed=14)
    ops.run_forward(model, torch.tensor([0, 40, 30, 64], dtype=torch.int32, device="cuda"), qkv, 2, 45)


def test_an_operators_error_is_not_the_encoders(esm, encoder):
    """Bad offsets of an operator do not fail the context's encoder calls, which leave them to check_device."""
    seqs = [np.arange(n, dtype=np.int32) % 20 + 4 for n in (30, 12)]
    logits, scores = encoder.forward(seqs)["logits"], encoder.score(seqs)["logp"]
    bad_offsets(encoder)
    torch.cuda.synchronize()
    assert np.array_equal(encoder.forward(seqs)["logits"], logits)
    assert np.array_equal(encoder.score(seqs)["logp"], scores)
    with pytest.raises(esm.EsmError, match="token id"):
        encoder.forward([np.full(5, 77, dtype=np.int32)])
    with pytest.raises(esm.EsmError, match="cu_seqlens") as e:
        encoder.check_device()
    assert e.value.code == esm.ESM_EINVAL
    encoder.check_device()


def test_errors_on_another_stream_are_reported(esm, encoder):
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bad_offsets(encoder)
    s.synchronize()
    with pytest.raises(esm.EsmError, match="cu_seqlens"):
        encoder.check_device()
    encoder.check_device()


def test_errors_of_several_calls_are_all_named(esm, encoder):
    """Error bits are gathered until they are read: two bad arguments are not a wait that gave up."""
    cu = np.array([0, 5], dtype=np.int32)
    bad, logits = torch.full((5,), 77, dtype=torch.int32, device="cuda"), torch.empty(5, 33, device="cuda")
    for _ in range(2):
        encoder.forward_device(bad, cu, logits)
        bad_offsets(encoder)
        with pytest.raises(esm.EsmError, match="token id.*cu_seqlens") as e:
            encoder.check_device()
        assert e.value.code == esm.ESM_EINVAL
    encoder.check_device()
    encoder.forward_device(bad, cu, logits)
    assert encoder.probe_wait_timeout(20) == esm.ESM_ETIMEOUT
    message = esm.lib().esm_last_error(encoder._ctx).decode()
    assert "wait gave up" in message and "token id" in message
    encoder.check_device()


def test_a_bound_of_no_rows_is_checked_like_any_other(esm, m):
    """max_len = 0 with sequences that are not empty: they are longer than max_len, and esm_check_device says so."""
    cu, qkv, dout = ops.attention_inputs([3, 0, 61], 2, 16, "f16", seed=420)
    out, lse = ops.run_forward(m, cu, qkv, 2, 64)
    m.check_device()
    out0, lse0 = ops.run_forward(m, cu, qkv, 2, 0)
    assert (out0 == 7).all() and (lse0 == 7).all()
    with pytest.raises(esm.EsmError, match="cu_seqlens"):
        m.check_device()
    assert (ops.run_backward(m, cu, qkv, 2, 0, out, lse, dout) == 7).all()
    with pytest.raises(esm.EsmError, match="cu_seqlens"):
        m.check_device()
    cu.fill_(64)
    ops.run_backward(m, cu, qkv, 2, 0, *ops.run_forward(m, cu, qkv, 2, 0), dout)
    m.check_device()
