"""The operators on device memory (attention, LayerNorm, token log probabilities, distillation, and
their backward passes) against their formulas in 64 bits.

Tolerances are bounds, elementwise: a value of a 16-bit type is rounded by at most half a step, U =
eps / 2 relative (fp16 2^-11, bf16 2^-8); fp32 sums of n terms in blocks of 32 lanes lose at most
(n / 32 + 32) E of the sum of magnitudes, E = 2^-24; exponentials are taken with a relative error
of at most X = 2^-13 (twice the 7.5e-5 of the polynomial that the attention kernels use for a share of
them) plus the absolute error of their argument.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
X = 2.0 ** -13
KINDS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(kind):
    return torch.finfo(kind).eps / 2


@pytest.fixture(scope="module")
def m(esm):
    model = esm.Model(0)
    yield model
    model.check_device()
    model.close()


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def within(got, want, bound, what):
    got, want = got.double(), want.double()
    if got.numel() == 0:
        return
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    worst = int(over.argmax())
    assert float(over.max()) <= 0, (f"{what}: {float(got.flatten()[worst]):.6g} for {float(want.flatten()[worst]):.6g}, "
                                    f"allowed {float(bound.expand_as(want).flatten()[worst]):.3g}")


# ---- attention ------------------------------------------------------------------------------------

def attention_inputs(lens, H, dh, kind, seed=0, rows_behind=0, pad_cols=0, sharp=1.5, grad=0.05):
    T, d = sum(lens) + rows_behind, H * dh
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")
    qkv = torch.zeros(T, 3 * d + pad_cols, dtype=KINDS[kind], device="cuda")
    x = randn(seed, T, 3 * d)
    x[:, :d] *= sharp
    qkv[:, :3 * d] = x.to(KINDS[kind])
    dout = torch.zeros(T, d + pad_cols, dtype=KINDS[kind], device="cuda")
    dout[:, :d] = (grad * randn(seed + 1, T, d)).to(KINDS[kind])
    return cu, qkv[:, :3 * d], dout[:, :d]


def run_forward(m, cu, qkv, H, max_len, stream=None, scale=None):
    T, d = qkv.shape[0], qkv.shape[1] // 3
    out = torch.full((T, d), 7.0, dtype=qkv.dtype, device="cuda")
    lse = torch.full((H, T), 7.0, device="cuda")
    m.attention(qkv, cu, max_len, H, out, lse, scale=scale, stream=stream or torch.cuda.current_stream())
    return out, lse


def run_backward(m, cu, qkv, H, max_len, out, lse, dout, stream=None, scale=None):
    dqkv = torch.full((qkv.shape[0], qkv.shape[1]), 7.0, dtype=qkv.dtype, device="cuda")
    ws = torch.full((m.attention_backward_workspace(cu.numel() - 1, qkv.shape[0], H),), 255, dtype=torch.uint8, device="cuda")
    m.attention_backward(qkv, cu, max_len, H, out, lse, dout, dqkv, ws, scale=scale, stream=stream or torch.cuda.current_stream())
    return dqkv


def sequences(cu):
    c = cu.tolist()
    return [(a, b) for a, b in zip(c[:-1], c[1:]) if b > a]


def split_heads(x, H):
    return x.double().unflatten(-1, (H, -1)).transpose(0, 1)  # [H, L, dh]


def score_error(q, k, scale):
    """Bound of |S - exact|: fp32 accumulation of exact products, and fp32 arithmetic on the score."""
    dh = q.shape[-1]
    return (dh + 2) * E * abs(scale) * (q.abs() @ k.abs().transpose(-1, -2)) + 4 * E * abs(scale) * (q @ k.transpose(-1, -2)).abs()


def check_forward(cu, qkv, H, out, lse, scale=None):
    U = half_step(qkv.dtype)
    d = qkv.shape[1] // 3
    scale = (d // H) ** -0.5 if scale is None else scale
    for a, b in sequences(cu):
        q, k, v = (split_heads(x, H) for x in qkv[a:b].split(d, 1))
        s = scale * q @ k.transpose(-1, -2)
        es = score_error(q, k, scale).amax(-1, keepdim=True)
        want_lse = torch.logsumexp(s, -1)
        p = torch.exp(s - want_lse[..., None])
        want = p @ v
        mass = p @ v.abs()
        within(split_heads(out[a:b], H), want, (U + 2 * X + 2 * es) * mass + U * want.abs() + 2.0 ** -25, "out")
        within(lse[:, a:b], want_lse, es[..., 0] + X + 8 * E * want_lse.abs(), "lse")


def check_backward(cu, qkv, H, out, lse, dout, dqkv, scale=None):
    U = half_step(qkv.dtype)
    d = qkv.shape[1] // 3
    dh = d // H
    scale = dh ** -0.5 if scale is None else scale
    tiny = 2.0 ** -25 if qkv.dtype == torch.float16 else 1e-38
    for a, b in sequences(cu):
        q, k, v = (split_heads(x, H) for x in qkv[a:b].split(d, 1))
        o, g = split_heads(out[a:b], H), split_heads(dout[a:b], H)
        s = scale * q @ k.transpose(-1, -2)
        lse_ = lse[:, a:b].double()[..., None]
        p = torch.exp(s - lse_)
        ep = X + 2 * score_error(q, k, scale) + 8 * E * lse_.abs()  # relative error of p
        delta = (o * g).sum(-1, keepdim=True)
        dp = g @ v.transpose(-1, -2)
        ds = p * (dp - delta)
        # fp32 accumulation of dout V^T and of D, times p; and dS rounded, on the scale that its type is given
        e_ds = p * ((dh + 8) * E * (g.abs() @ v.abs().transpose(-1, -2) + (o * g).abs().sum(-1, keepdim=True) + delta.abs() + dp.abs()))
        floor = 2.0 ** -37 * dh * float(g.abs().max()) * float(v.abs().max()) + 1e-30
        e_ds = e_ds + (U + ep) * ds.abs() + floor
        e_pv = (U + ep) * p + 2.0 ** -38
        got = [split_heads(x, H) for x in dqkv[a:b].split(d, 1)]
        n = (b - a) * E  # fp32 accumulation over the rows
        want = scale * ds @ k
        within(got[0], want, U * want.abs() + abs(scale) * (e_ds + n * ds.abs()) @ k.abs() + tiny, "dq")
        want = scale * ds.transpose(-1, -2) @ q
        within(got[1], want, U * want.abs() + abs(scale) * (e_ds + n * ds.abs()).transpose(-1, -2) @ q.abs() + tiny, "dk")
        want = p.transpose(-1, -2) @ g
        within(got[2], want, U * want.abs() + (e_pv + n * p).transpose(-1, -2) @ g.abs() + tiny, "dv")


LENGTHS = [[1], [2, 1, 1], [0, 5, 0, 0, 9], [31, 32, 33], [63, 64, 65, 1], [127, 128, 129], [255, 257, 3, 256], [700]]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
def test_attention_lengths(m, kind, lens):
    for H, dh in ((3, 64), (2, 24)):
        cu, qkv, dout = attention_inputs(lens, H, dh, kind, seed=sum(lens) + dh)
        out, lse = run_forward(m, cu, qkv, H, max(lens))
        check_forward(cu, qkv, H, out, lse)
        check_backward(cu, qkv, H, out, lse, dout, run_backward(m, cu, qkv, H, max(lens), out, lse, dout))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dh", [8, 16, 24, 32, 40, 48, 56, 64])
def test_attention_head_dims(m, kind, dh):
    lens = [130, 0, 77]
    cu, qkv, dout = attention_inputs(lens, 5, dh, kind, seed=dh)
    out, lse = run_forward(m, cu, qkv, 5, 200)
    check_forward(cu, qkv, 5, out, lse)
    check_backward(cu, qkv, 5, out, lse, dout, run_backward(m, cu, qkv, 5, 200, out, lse, dout))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_row_strides_and_rows_behind(m, kind):
    H, dh, lens = 4, 32, [70, 129]
    cu, qkv, dout = attention_inputs(lens, H, dh, kind, seed=3, rows_behind=21, pad_cols=24)
    assert qkv.stride(0) == 3 * H * dh + 24
    qkv[sum(lens):] = math.nan      # rows behind the last sequence hold anything
    dout[sum(lens):] = math.inf
    out, lse = run_forward(m, cu, qkv, H, 129)
    check_forward(cu, qkv, H, out, lse)
    out[sum(lens):] = math.nan
    lse[:, sum(lens):] = math.nan
    dqkv = run_backward(m, cu, qkv, H, 129, out, lse, dout)
    check_backward(cu, qkv, H, out, lse, dout, dqkv)
    out, lse = run_forward(m, cu, qkv, H, 129)
    for x in (out, dqkv):
        assert (x[sum(lens):] == 7.0).all()
    assert (lse[:, sum(lens):] == 7.0).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_sequences_do_not_see_each_other(m, kind, bad):
    H, dh, lens = 2, 64, [100, 45, 190]
    cu, qkv, dout = attention_inputs(lens, H, dh, kind, seed=5)
    out, lse = run_forward(m, cu, qkv, H, 190)
    dqkv = run_backward(m, cu, qkv, H, 190, out, lse, dout)
    qkv2, dout2 = qkv.clone(), dout.clone()
    qkv2[100:145] = bad
    dout2[100:145] = bad
    out2, lse2 = run_forward(m, cu, qkv2, H, 190)
    dqkv2 = run_backward(m, cu, qkv2, H, 190, out2, lse2, dout2)
    for x, y in ((out, out2), (dqkv, dqkv2), (lse.t(), lse2.t())):
        assert torch.equal(x[:100], y[:100]) and torch.equal(x[145:], y[145:])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_sharp_and_flat_scores(m, kind):
    H, dh, lens = 2, 64, [300]
    for sharp, scale in ((40.0, None), (0.01, None), (1.0, 1e-3), (1.0, 0.3), (1.0, 1e-6), (0.001, 100.0)):
        cu, qkv, dout = attention_inputs(lens, H, dh, kind, seed=7, sharp=sharp)
        out, lse = run_forward(m, cu, qkv, H, 300, scale=scale)
        check_forward(cu, qkv, H, out, lse, scale)
        check_backward(cu, qkv, H, out, lse, dout, run_backward(m, cu, qkv, H, 300, out, lse, dout, scale=scale), scale)


def test_attention_late_maximum(m):
    """A row whose largest scores come last: the running maximum is far below them until then."""
    H, dh, L = 1, 64, 400
    for kind in ("f16", "bf16"):
        cu, qkv, dout = attention_inputs([L], H, dh, kind, seed=8, sharp=0.2)
        qkv[:, :dh] = 1.0
        qkv[:, dh:2 * dh] = torch.linspace(-40, 40, L, device="cuda")[:, None].to(qkv.dtype) / 8
        out, lse = run_forward(m, cu, qkv, H, L)
        check_forward(cu, qkv, H, out, lse)
        check_backward(cu, qkv, H, out, lse, dout, run_backward(m, cu, qkv, H, L, out, lse, dout))


@pytest.mark.parametrize("grad", [1e-6, 1.0, 300.0])
def test_attention_backward_small_and_large_gradients(m, grad):
    """fp16: dS of a gradient this small is far below the type's normal range, unless it is scaled."""
    H, dh, lens = 2, 32, [513, 20]
    cu, qkv, dout = attention_inputs(lens, H, dh, "f16", seed=9, grad=grad)
    out, lse = run_forward(m, cu, qkv, H, 513)
    check_backward(cu, qkv, H, out, lse, dout, run_backward(m, cu, qkv, H, 513, out, lse, dout))


def test_attention_backward_of_zeros(m):
    H, dh = 2, 64
    for kind in ("f16", "bf16"):
        cu, qkv, dout = attention_inputs([150], H, dh, kind, seed=10)
        dout.zero_()
        out, lse = run_forward(m, cu, qkv, H, 150)
        assert (run_backward(m, cu, qkv, H, 150, out, lse, dout) == 0).all()


def test_attention_gradient_against_differences(m):
    """<dqkv, t> against the central difference of <out(qkv), dout> along t, in 64 bits."""
    H, dh, L = 2, 16, 37
    d = H * dh
    cu, qkv, dout = attention_inputs([L], H, dh, "f16", seed=11)
    out, lse = run_forward(m, cu, qkv, H, L)
    dqkv = run_backward(m, cu, qkv, H, L, out, lse, dout).double()

    def loss(x):
        q, k, v = (x[:, i * d:(i + 1) * d].unflatten(1, (H, dh)).transpose(0, 1) for i in range(3))
        p = torch.softmax(q @ k.transpose(-1, -2) * dh ** -0.5, -1)
        return (p @ v * dout.double().unflatten(1, (H, dh)).transpose(0, 1)).sum()

    for part in range(3):
        t = torch.zeros_like(dqkv)
        t[:, part * d:(part + 1) * d] = dqkv[:, part * d:(part + 1) * d] / dqkv[:, part * d:(part + 1) * d].norm()
        h = 1e-4
        slope = float((loss(qkv.double() + h * t) - loss(qkv.double() - h * t)) / (2 * h))
        # Roundings of P or dS, of out inside D and of the gradient itself: three half steps of the
        # norms they act on, which are at most 4 times the gradient's norm here; h^2 is negligible.
        assert abs(float((dqkv * t).sum()) - slope) <= 3 * 4 * 2.0 ** -11 * float(dqkv.norm())


def test_attention_is_reproducible_and_capturable(m):
    H, dh, lens = 3, 64, [200, 1, 310]
    cu, qkv, dout = attention_inputs(lens, H, dh, "bf16", seed=12)
    T, d = qkv.shape[0], H * dh
    out, lse = run_forward(m, cu, qkv, H, 310)
    dqkv = run_backward(m, cu, qkv, H, 310, out, lse, dout)
    stream = torch.cuda.Stream()
    q2, g2, o2, l2 = torch.zeros_like(qkv), torch.zeros_like(dout), torch.zeros_like(out), torch.zeros_like(lse)
    dq2 = torch.zeros_like(dqkv)
    cu2 = torch.zeros_like(cu)
    ws = torch.empty(m.attention_backward_workspace(3, T, H), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        s = torch.cuda.current_stream()
        m.attention(q2, cu2, 310, H, o2, l2, stream=s)
        m.attention_backward(q2, cu2, 310, H, o2, l2, g2, dq2, ws, stream=s)
    q2.copy_(qkv), g2.copy_(dout), cu2.copy_(cu)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o2, out) and torch.equal(l2, lse) and torch.equal(dq2, dqkv)
    # Other lengths in the same graph.
    cu, qkv, dout = attention_inputs([310, 0, 201], H, dh, "bf16", seed=13)
    q2.copy_(qkv), g2.copy_(dout), cu2.copy_(cu)
    graph.replay()
    torch.cuda.synchronize()
    check_forward(cu, qkv, H, o2, l2)
    check_backward(cu, qkv, H, o2, l2, dout, dq2)


def test_attention_reports_offsets_that_do_not_fit(m, esm):
    H, dh = 2, 16
    _, qkv, dout = attention_inputs([64], H, dh, "f16", seed=14)
    for bad in ([0, 40, 30, 64], [0, 10, 20, 65], [0, 50, 60, 64], [-3, 10, 20, 30]):
        cu = torch.tensor(bad, dtype=torch.int32, device="cuda")
        out, lse = run_forward(m, cu, qkv, H, 45)
        with pytest.raises(esm.EsmError, match="cu_seqlens") as e:
            m.check_device()
        assert e.value.code == esm.ESM_EINVAL
        run_backward(m, cu, qkv, H, 45, out, lse, dout)
        with pytest.raises(esm.EsmError, match="cu_seqlens"):
            m.check_device()
    m.check_device()


def test_attention_refusals(m, esm):
    H, dh = 2, 16
    cu, qkv, dout = attention_inputs([64], H, dh, "f16", seed=15)
    out, lse = run_forward(m, cu, qkv, H, 64)
    dqkv, ws = torch.empty_like(qkv), torch.empty(m.attention_backward_workspace(1, 64, H), dtype=torch.uint8, device="cuda")

    def refused(match, code=esm.ESM_EINVAL, **kw):
        a = {"qkv": qkv, "cu": cu, "max_len": 64, "H": H, "out": out, "lse": lse, "dout": dout, "dqkv": dqkv, "ws": ws,
             "scale": None, **kw}
        with pytest.raises(esm.EsmError, match=match) as e:
            m.attention_backward(a["qkv"], a["cu"], a["max_len"], a["H"], a["out"], a["lse"], a["dout"], a["dqkv"], a["ws"], scale=a["scale"])
        assert e.value.code == code

    refused("max_len", max_len=65)
    refused("max_len", max_len=-1)
    refused("head_dim", H=8, lse=torch.zeros(8, 64, device="cuda"))   # 4 columns
    refused("head_dim", H=32, lse=torch.zeros(32, 64, device="cuda"))  # 1 column
    for scale in (math.inf, math.nan, 0.0, -0.3, 1e-7, 1e7):
        refused("scale", scale=scale)
    refused("workspace", code=esm.ESM_ECAPACITY, ws=ws[:16])
    refused("overlap", dqkv=qkv)
    refused("overlap", out=dout, dqkv=torch.cat([dout] * 4, 1)[:, :96].contiguous(), ws=dout.view(torch.uint8))
    refused("not device memory|not memory of", dout=dout.cpu())
    refused("16-byte", qkv=torch.empty(64, 100, dtype=torch.float16, device="cuda")[:, 1:97])
    refused("16-byte", qkv=torch.empty(64, 97, dtype=torch.float16, device="cuda")[:, :96])
    refused("ESM_F16 or ESM_BF16", **{n: x.float() for n, x in (("qkv", qkv), ("out", out), ("dout", dout), ("dqkv", dqkv))})


def test_attention_of_nothing(m):
    empty = torch.empty(0, 96, dtype=torch.float16, device="cuda")
    out = torch.empty(0, 32, dtype=torch.float16, device="cuda")
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    m.attention(empty, cu, 0, 2, out, torch.empty(2, 0, device="cuda"))
    cu, qkv, dout = attention_inputs([0, 0], 2, 16, "f16", rows_behind=5)
    out, lse = run_forward(m, cu, qkv, 2, 0)
    assert (out == 7).all() and (lse == 7).all()
    out, lse = run_forward(m, cu, qkv, 2, 5)
    dqkv = run_backward(m, cu, qkv, 2, 5, out, lse, dout)
    assert (out == 7).all() and (dqkv == 7).all()


# ---- LayerNorm ------------------------------------------------------------------------------------

def ln_inputs(T, d, x_kind, seed, outliers=True):
    x = randn(seed, T, d) + 0.5 * randn(seed + 1, T, 1)
    if outliers and d > 8:
        x[:, 3] *= 60
    return x.to(KINDS[x_kind]), 1 + 0.2 * randn(seed + 2, d), 0.1 * randn(seed + 3, d)


def run_ln(m, x, w, b, y_kind, eps=1e-5):
    T, d = x.shape
    y = torch.empty(T, d, dtype=KINDS[y_kind], device="cuda")
    mean, rstd = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    m.layernorm(x, w, b, y, mean, rstd, eps=eps, stream=torch.cuda.current_stream())
    return y, mean, rstd


def check_ln(x, w, b, y, mean, rstd, eps=1e-5):
    d = x.shape[1]
    G = (d / 32 + 32) * E
    x64, U = x.double(), half_step(y.dtype)
    mu = x64.mean(1, keepdim=True)
    c = x64 - mu
    var = (c * c).mean(1, keepdim=True)
    r = (var + eps) ** -0.5
    want = c * r * w.double() + b.double()
    e_mu = G * x64.abs().mean(1, keepdim=True)
    # The variance: its own sum, and the centre's error (second order) and each term's rounding.
    rel = G + 4 * E + (2 * E * x64.abs().mean(1, keepdim=True) + e_mu ** 2 * r) * r
    within(mean[:, None], mu, e_mu, "mean")
    within(rstd[:, None], r, rel * r, "rstd")
    xw = (c * r * w.double()).abs()
    bound = U * want.abs() + (e_mu + 2 * E * x64.abs()) * r * w.double().abs() + (rel + 4 * E) * xw + 4 * E * (xw + b.abs())
    within(y, want, bound + (2.0 ** -25 if y.dtype == torch.float16 else 0), "y")


def run_ln_backward(m, dy, x, w, mean, rstd, dres=None):
    T, d = x.shape
    dx = torch.empty_like(x)
    dw, db = torch.full((d,), 7.0, device="cuda"), torch.full((d,), 7.0, device="cuda")
    ws = torch.full((m.layernorm_backward_workspace(T, d),), 255, dtype=torch.uint8, device="cuda")
    m.layernorm_backward(dy, x, w, mean, rstd, dx, dw, db, ws, dres=dres, stream=torch.cuda.current_stream())
    return dx, dw, db


def check_ln_backward(dy, x, w, mean, rstd, dres, dx, dw, db):
    T, d = x.shape
    G = (d / 32 + 32) * E
    r = rstd.double()[:, None]
    xh = (x.double() - mean.double()[:, None]) * r
    e_xh = 2 * E * (x.double().abs() + mean.double().abs()[:, None]) * r + 2 * E * xh.abs()
    dy64 = dy.double()
    g = dy64 * w.double()
    mg, mgx = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    want = r * (g - mg - xh * mgx)
    e_mgx = G * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * e_xh).mean(1, keepdim=True)
    bound = r * (4 * E * g.abs() + G * g.abs().mean(1, keepdim=True) + 4 * E * mg.abs() + xh.abs() * e_mgx + (e_xh + 4 * E * xh.abs()) * mgx.abs())
    if dres is not None:
        want = want + dres.double()
        bound = bound + 2 * E * (dres.double().abs() + want.abs())
    tiny = 2.0 ** -25 if dx.dtype == torch.float16 else 0.0
    within(dx, want, bound + half_step(dx.dtype) * (want.abs() + bound) + tiny, "dx")
    # At most 1024 additions in a row on the way of a term into its sum.
    N = 1024 * E
    within(dw, (dy64 * xh).sum(0), N * (dy64 * xh).abs().sum(0) + (dy64.abs() * e_xh).sum(0) + 1e-30, "dw")
    within(db, dy64.sum(0), N * dy64.abs().sum(0) + 1e-30, "db")


@pytest.mark.parametrize("d", [1, 7, 16, 33, 320, 480, 640, 1000, 1280, 2560, 5121, 8192])
@pytest.mark.parametrize("T", [1, 3, 65])
def test_layernorm_sizes(m, T, d):
    for x_kind, y_kind in (("f32", "f16"), ("f32", "f32"), ("bf16", "bf16")):
        x, w, b = ln_inputs(T, d, x_kind, seed=T * 31 + d)
        y, mean, rstd = run_ln(m, x, w, b, y_kind)
        check_ln(x, w, b, y, mean, rstd)
        dy = (0.05 * randn(d, T, d)).to(KINDS[y_kind])
        for dres in (None, (0.05 * randn(d + 1, T, d)).to(KINDS[x_kind])):
            check_ln_backward(dy, x, w, mean, rstd, dres, *run_ln_backward(m, dy, x, w, mean, rstd, dres))


@pytest.mark.parametrize("x_kind", KINDS)
@pytest.mark.parametrize("y_kind", KINDS)
def test_layernorm_types_and_many_rows(m, x_kind, y_kind):
    T, d = 5003, 640
    x, w, b = ln_inputs(T, d, x_kind, seed=17)
    y, mean, rstd = run_ln(m, x, w, b, y_kind)
    check_ln(x, w, b, y, mean, rstd)
    dy = (0.05 * randn(18, T, d)).to(KINDS[y_kind])
    dres = randn(19, T, d).to(KINDS[x_kind])
    check_ln_backward(dy, x, w, mean, rstd, dres, *run_ln_backward(m, dy, x, w, mean, rstd, dres))


def test_layernorm_unaligned_buffers(m):
    """Views that start on an odd element: no 16-byte loads."""
    for d in (320, 1280):
        T = 9
        store = torch.zeros(T * d + 1, device="cuda")
        x, w, b = ln_inputs(T, d, "f32", seed=20)
        store[1:] = x.flatten()
        xo = store[1:].view(T, d)
        y = torch.empty(T * d + 1, dtype=torch.float16, device="cuda")[1:].view(T, d)
        mean, rstd = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
        wo = torch.cat([w, w])[1:d + 1]
        m.layernorm(xo, wo, b, y, mean, rstd)
        check_ln(xo, wo, b, y, mean, rstd)
        dy = torch.zeros(T * d + 1, dtype=torch.float16, device="cuda")[1:].view(T, d)
        dy.copy_(0.05 * randn(21, T, d))
        check_ln_backward(dy, xo, wo, mean, rstd, None, *run_ln_backward(m, dy, xo, wo, mean, rstd))


def test_layernorm_constant_rows_and_eps(m):
    for eps in (1e-5, 1e-12, 0.3):
        x, w, b = ln_inputs(6, 320, "f32", seed=22)
        x[1] = 0.0
        x[2] = 3.25
        y, mean, rstd = run_ln(m, x, w, b, "f32", eps)
        check_ln(x, w, b, y, mean, rstd, eps)
        assert torch.equal(y[1], b) and torch.equal(y[2], b)


def test_layernorm_a_bad_row_stays_alone(m):
    x, w, b = ln_inputs(70, 640, "f32", seed=23)
    y, mean, rstd = run_ln(m, x, w, b, "f16")
    dy = (0.05 * randn(24, 70, 640)).half()
    dx, _, _ = run_ln_backward(m, dy, x, w, mean, rstd)
    x2 = x.clone()
    x2[33, 5] = math.nan
    y2, mean2, rstd2 = run_ln(m, x2, w, b, "f16")
    dx2, _, _ = run_ln_backward(m, dy, x2, w, mean2, rstd2)
    keep = torch.arange(70, device="cuda") != 33
    assert torch.equal(y[keep], y2[keep]) and torch.equal(dx[keep], dx2[keep])
    assert torch.isnan(y2[33]).all()


def test_layernorm_gradient_against_differences(m):
    T, d = 5, 64
    x, w, b = ln_inputs(T, d, "f32", seed=25, outliers=False)
    _, mean, rstd = run_ln(m, x, w, b, "f32")
    dy = randn(26, T, d)
    grads = run_ln_backward(m, dy, x, w, mean, rstd)

    def loss(x, w, b):
        c = x - x.mean(1, keepdim=True)
        return ((c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * w + b) * dy.double()).sum()

    at = [x.double(), w.double(), b.double()]
    for i, g in enumerate(grads):
        t = g.double() / g.double().norm()
        h = 1e-4
        up, down = [list(at) for _ in range(2)]
        up[i], down[i] = at[i] + h * t, at[i] - h * t
        slope = float((loss(*up) - loss(*down)) / (2 * h))
        # fp32 statistics and sums: 100 roundings' worth; the difference's own error is of order h^2.
        assert abs(float((g.double() * t).sum()) - slope) <= (100 * E + 1e-6) * float(g.double().norm())


def test_layernorm_no_rows_reproducible_refusals(m, esm):
    d = 48
    w = torch.ones(d, device="cuda")
    none = torch.empty(0, d, device="cuda")
    dx, dw, db = run_ln_backward(m, none, none, w, torch.empty(0, device="cuda"), torch.empty(0, device="cuda"))
    assert (dw == 0).all() and (db == 0).all()
    m.layernorm(none, w, w, none)
    x, w, b = ln_inputs(3001, 320, "f32", seed=27)
    _, mean, rstd = run_ln(m, x, w, b, "f16")
    dy = randn(28, 3001, 320).half()
    first = run_ln_backward(m, dy, x, w, mean, rstd)
    for a, c in zip(first, run_ln_backward(m, dy, x, w, mean, rstd)):
        assert torch.equal(a, c)
    with pytest.raises(esm.EsmError, match="overlap"):
        m.layernorm(x, w, b, x)
    with pytest.raises(esm.EsmError, match="eps"):
        m.layernorm(x, w, b, torch.empty_like(x), eps=-1.0)
    with pytest.raises(esm.EsmError, match="workspace") as e:
        m.layernorm_backward(dy, x, w, mean, rstd, torch.empty_like(x), torch.empty_like(w), torch.empty_like(w), torch.empty(16, device="cuda"))
    assert e.value.code == esm.ESM_ECAPACITY
    with pytest.raises(esm.EsmError, match="not memory of|not device"):
        m.layernorm(x.cpu(), w, b, torch.empty_like(x))


# ---- log probabilities ------------------------------------------------------------------------------

def logits_of(T, V, kind, seed, spread=3.0):
    return (spread * randn(seed, T, V) + 2 * randn(seed + 1, T, 1)).to(KINDS[kind])


def run_logprobs(m, x, targets, k):
    T = x.shape[0]
    logp, ent = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    ids = torch.full((T, k), -7, dtype=torch.int32, device="cuda")
    top = torch.empty(T, k, device="cuda")
    m.token_logprobs(x, targets, logp, ent, ids if k else None, top if k else None, stream=torch.cuda.current_stream())
    return logp, ent, ids, top


def check_logprobs(x, targets, logp, ent, ids, top):
    V, k = x.shape[1], ids.shape[1]
    x64 = x.double()
    big = torch.where(x64.isfinite(), x64.abs(), 0.0).amax(1)
    lse = torch.logsumexp(x64, 1)
    e_lse = (V / 32 + 64) * E + 2.0 ** -20 + 8 * E * big
    lp = x64 - lse[:, None]
    ok = (targets >= 0) & (targets < V)
    want = torch.where(ok, lp.gather(1, targets.long().clamp(0, V - 1)[:, None])[:, 0], 0.0)
    assert torch.equal(logp == -math.inf, want == -math.inf)
    fin = want.isfinite()
    within(logp[fin], want[fin], (e_lse + 4 * E * want.abs())[fin], "logp")
    assert (logp[~ok] == 0).all()
    p = lp.exp()
    want = -torch.where(p > 0, p * lp, 0.0).sum(1)
    spread = torch.where(p > 0, p * (x64 - x64.amax(1, keepdim=True)).abs(), 0.0).sum(1)
    within(ent, want, e_lse + (1 + spread) * ((V / 32 + 64) * E + 2.0 ** -19), "entropy")
    order = torch.sort(x64, dim=1, descending=True, stable=True)
    assert torch.equal(ids.long(), order.indices[:, :k])
    want = order.values[:, :k] - lse[:, None]
    assert torch.equal(top == -math.inf, want == -math.inf)
    fin = want.isfinite()
    within(top[fin], want[fin], (e_lse[:, None] + 4 * E * want.abs())[fin], "top_logp")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T, V, k", [(1, 1, 1), (1, 33, 33), (3, 2, 2), (33, 20, 5), (129, 33, 1), (1000, 33, 6), (31, 64, 64), (40, 65, 7),
                                     (17, 127, 64), (9, 128, 3), (5, 1000, 64), (3, 4099, 17), (2, 50257, 64), (1, 131075, 5), (70, 33, 0)])
def test_logprobs_sizes(m, kind, T, V, k):
    x = logits_of(T, V, kind, seed=T + V)
    targets = torch.randint(-1, V + 1, (T,), device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(V))
    check_logprobs(x, targets, *run_logprobs(m, x, targets, k))


@pytest.mark.parametrize("V", [33, 257, 9001])
def test_logprobs_ties_masks_and_rows_without_a_distribution(m, V):
    T, k = 12, 16
    x = logits_of(T, V, "f32", seed=V)
    x[0] = 1.0                      # all equal
    x[1] = -math.inf                # one token can occur
    x[1, V // 2] = 4.0
    x[2, ::2] = -math.inf
    x[3] = torch.where(torch.arange(V, device="cuda") % 3 == 0, 0.0, -0.0)
    x[4] = torch.finfo(torch.float32).min
    x[5] = torch.finfo(torch.float32).min
    x[5, 3] = 100.0
    x[6] = x[6].round()             # many ties
    targets = torch.arange(T, dtype=torch.int32, device="cuda")
    bad = {7: math.nan, 8: math.inf}
    for r, v in bad.items():
        x[r, V - 1] = v
    x[9] = -math.inf
    logp, ent, ids, top = run_logprobs(m, x, targets, k)
    lost = [7, 8, 9]
    keep = [i for i in range(T) if i not in lost]
    check_logprobs(x[keep], targets[keep], logp[keep], ent[keep], ids[keep], top[keep])
    assert torch.isnan(logp[lost]).all() and torch.isnan(ent[lost]).all() and torch.isnan(top[lost]).all() and (ids[lost] == -1).all()


def test_logprobs_adversarial_order(m):
    """The largest logits at a fixed stride, so that they all fall to the same threads; and sorted rows."""
    V, k = 32768, 64
    x = randn(31, 8, V)
    at = torch.arange(V, device="cuda")
    x[4] += 40.0 * ((at // 4) % 512 < 32)     # one warp's worth of vectors, all far above the rest
    x[5] = ((at // 4) % 512 < 64).float()     # the same as ties
    x[6] = (at % 2).float()
    x[7] += 40.0 * ((at // 4) % 128 < 96)
    x[0, 5::256][:k] += 50
    x[1, ::1024] += 50
    x[2] = torch.linspace(-20, 20, V, device="cuda")
    x[3] = torch.linspace(20, -20, V, device="cuda")
    targets = torch.zeros(8, dtype=torch.int32, device="cuda")
    check_logprobs(x, targets, *run_logprobs(m, x, targets, k))
    for n in (1000, 4000):                    # the smaller blocks
        y = x[:, :n].contiguous()
        y[4] = 40.0 * ((at[:n] // 4) % 128 < 32) + randn(32, n)
        check_logprobs(y, targets, *run_logprobs(m, y, targets, 16))
        check_logprobs(y, targets, *run_logprobs(m, y, targets, k))


def test_logprobs_are_reproducible(m):
    for V, k in ((33, 8), (700, 9), (4000, 33), (32003, 64)):
        x = logits_of(64, V, "bf16", seed=V)
        targets = torch.full((64,), 5, dtype=torch.int32, device="cuda")
        first = run_logprobs(m, x, targets, k)
        for _ in range(3):
            for a, b in zip(first, run_logprobs(m, x, targets, k)):
                assert torch.equal(a, b)


def test_logprobs_row_strides_and_optional_outputs(m, esm):
    T, V = 50, 33
    store = logits_of(T, V + 7, "f16", seed=32)
    x = store[:, 2:2 + V]
    store[:, V + 2:] = math.nan
    store[:, :2] = math.nan
    targets = torch.full((T,), 4, dtype=torch.int32, device="cuda")
    full = run_logprobs(m, x, targets, 3)
    check_logprobs(x, targets, *full)
    logp, ent = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    m.token_logprobs(x, targets, logp)
    m.token_logprobs(x, entropy=ent)
    assert torch.equal(logp, full[0]) and torch.equal(ent, full[1])
    with pytest.raises(esm.EsmError, match="go together"):
        m.token_logprobs(x, targets)
    with pytest.raises(esm.EsmError, match="alternatives"):
        m.token_logprobs(x, top_ids=torch.empty(T, 34, dtype=torch.int32, device="cuda"), top_logp=torch.empty(T, 34, device="cuda"))
    big = logits_of(2, 100, "f32", seed=1)
    with pytest.raises(esm.EsmError, match="alternatives"):
        m.token_logprobs(big, top_ids=torch.empty(2, 65, dtype=torch.int32, device="cuda"), top_logp=torch.empty(2, 65, device="cuda"))
    m.token_logprobs(torch.empty(0, 33, device="cuda"), entropy=torch.empty(0, device="cuda"))


def test_score_is_the_forward_and_its_log_probabilities(esm):
    cfg = esm.EsmConfig(320, 1280, 1, 20, 33, 64, 0)
    model = esm.Model(0)
    model.load_tensors(cfg, esm.DTYPE_FP32, esm.synth_fp32_tensors(cfg, seed=3))
    model.reserve(200, 4, 64)
    seqs = [np.arange(n, dtype=np.int32) % 20 + 4 for n in (50, 1, 64, 17)]
    logits = model.forward(seqs)["logits"]
    targets = [(x * 7 + 3) % 35 - 1 for x in seqs]           # some outside the vocabulary
    for want, k in ((None, 0), (targets, 5)):
        got = model.score(seqs, want, k)
        for i, x in enumerate(seqs):
            n = len(x)
            row = torch.from_numpy(logits[i, :n]).cuda()
            t = torch.from_numpy((x if want is None else want[i]).astype(np.int32)).cuda()
            ids = torch.from_numpy(got["top_ids"][i, :n]).cuda() if k else torch.empty(n, 0, dtype=torch.int32, device="cuda")
            top = torch.from_numpy(got["top_logp"][i, :n]).cuda() if k else torch.empty(n, 0, device="cuda")
            check_logprobs(row, t, torch.from_numpy(got["logp"][i, :n]).cuda(), torch.from_numpy(got["entropy"][i, :n]).cuda(), ids, top)
            assert (got["logp"][i, n:] == 0).all() and (got["entropy"][i, n:] == 0).all()
            assert not k or ((got["top_ids"][i, n:] == -1).all() and (got["top_logp"][i, n:] == 0).all())
    for bad in ({"k": 34}, {"k": -1}, {"targets": targets[:3]}):
        with pytest.raises(esm.EsmError) as e:
            model.score(seqs, **bad)
        assert e.value.code == esm.ESM_EINVAL
    model.close()
    empty = esm.Model(0)
    with pytest.raises(esm.EsmError, match="no weights"):
        empty.score(seqs)
    empty.close()


# ---- distillation -----------------------------------------------------------------------------------

def distill_inputs(T, V, k, kind, seed):
    x = logits_of(T, V, kind, seed)
    top, ids = (x.float() + 1.5 * randn(seed + 5, T, V)).topk(k, 1)
    ids = ids.to(torch.int32)
    if k > 2:
        ids[1::3, k // 2:] = -1
        ids[2::3, 0] = V + 3            # outside the vocabulary: absent
        ids[0::3, 1] = ids[0::3, 0]     # the same alternative twice
    top = torch.where((ids < 0) | (ids >= V), math.nan, top)  # what absent entries hold does not matter
    dloss = randn(seed + 6, T)
    dloss[::4] = 0
    return x, ids, top.contiguous(), dloss


def run_distill(m, x, ids, top, dloss, tau):
    T, V = x.shape
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    dx = torch.full((T, V), 7.0, dtype=x.dtype, device="cuda")
    s = torch.cuda.current_stream()
    m.distill_loss(x, ids, top, loss, lse, temperature=tau, stream=s)
    m.distill_backward(x, ids, top, lse, dloss, dx, temperature=tau, stream=s)
    return loss, lse, dx


def distill_64(x, ids, top, tau):
    """(loss, q, p scattered over the vocabulary, bound of the relative errors of q) in 64 bits."""
    V = x.shape[1]
    y = x.double() / tau
    lse = torch.logsumexp(y, 1, keepdim=True)
    logq = y - lse
    there = (ids >= 0) & (ids < V)
    t = torch.where(there, top.double(), -math.inf) / tau
    any_ = (t > -math.inf).any(1, keepdim=True)
    logp = torch.where(any_, t - torch.logsumexp(t, 1, keepdim=True), -math.inf)
    p = logp.exp()
    at = torch.where(there, ids, 0).long()
    terms = torch.where(p > 0, p * (logp - logq.gather(1, at)), 0.0)
    loss = tau * tau * terms.sum(1)
    spread = tau * tau * torch.where(p > 0, p * (logp.abs() + logq.gather(1, at).abs()), 0.0).sum(1)
    full = torch.zeros_like(y).scatter_add(1, at, p)
    big = torch.where(y.isfinite(), y.abs(), 0.0).amax(1)
    big_t = torch.where(t.isfinite(), t.abs(), 0.0).amax(1)
    e = (V / 32 + 64) * E + 2.0 ** -20 + 8 * E * (big + big_t + lse[:, 0].abs())
    return loss, lse[:, 0], logq.exp(), full, any_[:, 0], spread, e


def check_distill(x, ids, top, dloss, tau, loss, lse, dx):
    U = half_step(x.dtype)
    want, want_lse, q, p, any_, spread, e = distill_64(x, ids, top, tau)
    within(lse, want_lse, e + 4 * E * want_lse.abs(), "lse")
    within(loss, want, 4 * e * (tau * tau + spread), "loss")
    g = (dloss.double() * tau * any_)[:, None]
    wx = g * (q - p)
    within(dx, wx, U * wx.abs() + 4 * g.abs() * e[:, None] * (q + p) + (2.0 ** -25 if x.dtype == torch.float16 else 1e-38), "dlogits")
    assert (dx[dloss == 0] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T, V, k, tau", [(1, 1, 1, 1.0), (5, 2, 2, 3.0), (100, 33, 16, 2.0), (65, 33, 33, 0.5), (31, 64, 64, 1.0), (20, 65, 9, 1.0),
                                          (9, 128, 64, 4.0), (7, 1000, 33, 1.0), (3, 32003, 64, 2.0), (2, 70001, 1, 1.0)])
def test_distill_sizes(m, kind, T, V, k, tau):
    x, ids, top, dloss = distill_inputs(T, V, k, kind, seed=V + k)
    check_distill(x, ids, top, dloss, tau, *run_distill(m, x, ids, top, dloss, tau))


@pytest.mark.parametrize("V", [33, 3001])
def test_distill_rows_without_alternatives_and_padding(m, V):
    x, ids, top, dloss = distill_inputs(9, V, 8, "f32", seed=41)
    dloss[:] = 1.0
    ids[0] = -1
    top[1] = -math.inf               # every alternative impossible
    top[1, 0] = math.nan
    ids[1] = torch.arange(8, device="cuda")
    ids[1, 0] = -5
    ids[2] = torch.arange(8, device="cuda") + 2
    top[2] = -math.inf               # one alternative has all
    top[2, 3] = 0.5
    ids[3] = 11                      # one id, eight times
    top[3] = torch.arange(8.0, device="cuda")
    loss, lse, dx = run_distill(m, x, ids, top, dloss, 2.0)
    check_distill(x, ids, top, dloss, 2.0, loss, lse, dx)
    assert loss[0] == 0 and loss[1] == 0 and (dx[:2] == 0).all()
    # A padded row's logits do not matter.
    x[5] = math.nan
    x[6] = math.inf
    dloss[5:7] = 0
    _, _, dx2 = run_distill(m, x, ids, top, dloss, 2.0)
    assert (dx2[5:7] == 0).all() and torch.equal(dx2[7:], dx[7:])
    # A token that the student rules out.
    x[7] = 0.0
    x[7, 4] = -math.inf
    ids[7] = torch.tensor([4, 5, 6, -1, -1, -1, -1, -1], device="cuda")
    top[7] = 0.0
    loss, _, dx = run_distill(m, x, ids, top, dloss, 1.0)
    assert loss[7] == math.inf
    want = torch.full((V,), 1.0 / (V - 1), dtype=torch.float64, device="cuda")
    want[4] = 0
    want[4:7] -= 1 / 3
    within(dx[7], want, torch.full_like(want, 1e-6), "dlogits of a token ruled out")


@pytest.mark.parametrize("V", [33, 300])
def test_distill_bad_numbers_show(m, V):
    """A NaN teacher logit of a present alternative, or student logit, is not hidden."""
    x, ids, top, dloss = distill_inputs(3, V, 2, "f32", seed=46)
    dloss[:] = 1.0
    top[0, 1] = math.nan
    x[1, 7] = math.nan
    loss, _, dx = run_distill(m, x, ids, top, dloss, 1.0)
    assert torch.isnan(loss[:2]).all() and torch.isfinite(loss[2])
    assert torch.isnan(dx[0, ids[0, 1].long()]) and torch.isnan(dx[1]).all() and torch.isfinite(dx[2]).all()


def test_distill_row_strides(m):
    T, V = 40, 33
    x, ids, top, dloss = distill_inputs(T, V, 5, "bf16", seed=43)
    store = torch.full((T, V + 9), math.nan, dtype=torch.bfloat16, device="cuda")
    store[:, 3:3 + V] = x
    xs = store[:, 3:3 + V]
    grad = torch.full((T, V + 5), 7.0, dtype=torch.bfloat16, device="cuda")
    loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
    m.distill_loss(xs, ids, top, loss, lse, temperature=1.0)
    m.distill_backward(xs, ids, top, lse, dloss, grad[:, 1:1 + V], temperature=1.0)
    check_distill(x, ids, top, dloss, 1.0, loss, lse, grad[:, 1:1 + V])
    assert (grad[:, 0] == 7).all() and (grad[:, 1 + V:] == 7).all()


def test_distill_gradient_against_differences(m):
    x, ids, top, dloss = distill_inputs(6, 33, 7, "f32", seed=44)
    _, _, dx = run_distill(m, x, ids, top, dloss, 1.5)
    g = dx.double()
    t = g / g.norm()

    def total(y):
        return float((distill_64(y, ids, top, 1.5)[0] * dloss.double()).sum())

    h = 1e-4
    slope = (total(x.double() + h * t) - total(x.double() - h * t)) / (2 * h)
    assert abs(float((g * t).sum()) - slope) <= (200 * E + 1e-6) * float(g.norm())


def test_distill_refusals(m, esm):
    x, ids, top, dloss = distill_inputs(4, 33, 5, "f32", seed=45)
    s, l = torch.empty(4, device="cuda"), torch.empty(4, device="cuda")
    for tau in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(esm.EsmError, match="temperature"):
            m.distill_loss(x, ids, top, s, l, temperature=tau)
        with pytest.raises(esm.EsmError, match="temperature"):
            m.distill_backward(x, ids, top, l, dloss, torch.empty_like(x), temperature=tau)
    with pytest.raises(esm.EsmError, match="overlap"):
        m.distill_loss(x, ids, top, s, s)
    with pytest.raises(esm.EsmError, match="overlap"):
        m.distill_backward(x, ids, top, l, dloss, x)
    with pytest.raises(esm.EsmError, match="alternatives"):
        m.distill_loss(x, ids[:, :0].contiguous(), top[:, :0].contiguous(), s, l)


# ---- a distillation step --------------------------------------------------------------------------

def test_a_distillation_step(m):
    """Teacher logits -> its top alternatives -> loss of a one-block student -> gradients of its
    input and LayerNorm weights, with torch's GEMMs in between, against autograd in 64 bits."""
    H, dh, V, k, tau = 4, 16, 33, 12, 2.0
    d, lens = H * dh, [50, 1, 90]
    T = sum(lens)
    cu = torch.tensor([0, 50, 51, 141], dtype=torch.int32, device="cuda")
    x = randn(51, T, d)
    lw, lb = 1 + 0.1 * randn(52, d), 0.1 * randn(53, d)
    wqkv, wo, wv = (randn(54 + i, *s) * d ** -0.5 for i, s in enumerate(((d, 3 * d), (d, d), (d, V))))
    teacher = 2 * randn(60, T, V)
    weight = torch.full((T,), 1.0 / T, device="cuda")

    ids, top = torch.empty(T, k, dtype=torch.int32, device="cuda"), torch.empty(T, k, device="cuda")
    m.token_logprobs(teacher, top_ids=ids, top_logp=top)
    # forward
    y, mean, rstd = run_ln(m, x, lw, lb, "f32")
    qkv = (y @ wqkv).half()
    a, lse_a = run_forward(m, cu, qkv, H, 90)
    x1 = x + a.float() @ wo
    logits = x1 @ wv
    loss, lse, dlogits = run_distill(m, logits, ids, top, weight, tau)
    # backward; the 16-bit gradients are scaled as in mixed-precision training
    up = 4096.0
    dx1 = dlogits @ wv.t()
    da = (up * dx1 @ wo.t()).half()
    dqkv = run_backward(m, cu, qkv, H, 90, a, lse_a, da)
    dy = dqkv.float() @ wqkv.t() / up
    dx, dw, db = run_ln_backward(m, dy, x, lw, mean, rstd, dx1)

    X_, lw_, lb_ = (t.double().requires_grad_() for t in (x, lw, lb))
    c = X_ - X_.mean(1, keepdim=True)
    yy = c * torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-5) * lw_ + lb_
    q = yy @ wqkv.double()
    outs = []
    for s0, s1 in ((0, 50), (50, 51), (51, 141)):
        qh, kh, vh = (t.unflatten(1, (H, dh)).transpose(0, 1) for t in q[s0:s1].split(d, 1))
        outs.append((torch.softmax(qh @ kh.transpose(-1, -2) * dh ** -0.5, -1) @ vh).transpose(0, 1).flatten(1))
    xx = X_ + torch.cat(outs) @ wo.double()
    total = distill_64(xx @ wv.double(), ids, top, tau)[0]
    want = torch.autograd.grad((total * weight.double()).sum(), (X_, lw_, lb_))
    # Six 16-bit roundings lie on the way (qkv, P, out, dout, dS, dqkv), each at most 2^-11 of the
    # norm of what it rounds; the products between them change a norm by a factor of at most 4 here.
    rel = 6 * 4 * 2.0 ** -11
    for got, ref in zip((dx, dw, db), want):
        assert float((got.double() - ref).norm()) <= rel * float(ref.norm())
    assert float((loss.double() - total.detach()).norm()) <= 3 * 4 * 2.0 ** -11 * float(total.detach().norm())


# ---- many sequences, long buffers, graphs and streams -------------------------------------------------

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("length", [1, 64, 128, 40])
def test_attention_of_many_short_sequences(m, kind, length):
    """Items of one or two steps, whole and partial tiles, several per block, and empty sequences between."""
    H, dh, B = 5, 32, 220
    lens = [length if b % 7 else 0 for b in range(B)]
    cu, qkv, dout = attention_inputs(lens, H, dh, kind, seed=70 + length)
    max_len = min(2 * length + 100, qkv.shape[0])   # a loose bound
    out, lse = run_forward(m, cu, qkv, H, max_len)
    check_forward(cu, qkv, H, out, lse)
    check_backward(cu, qkv, H, out, lse, dout, run_backward(m, cu, qkv, H, max_len, out, lse, dout))


def test_attention_of_the_most_sequences(m):
    lens = [0] * 65535
    for at in (0, 1, 30000, 65533, 65534):
        lens[at] = 20
    cu, qkv, dout = attention_inputs(lens, 2, 16, "f16", seed=80)
    out, lse = run_forward(m, cu, qkv, 2, 100)
    check_forward(cu, qkv, 2, out, lse)
    check_backward(cu, qkv, 2, out, lse, dout, run_backward(m, cu, qkv, 2, 100, out, lse, dout))


def test_attention_offsets_beyond_32_bits(m):
    """Rows 800,000 elements apart: the last ones lie more than 2^31 elements into the buffer."""
    H, dh, T, ld = 2, 64, 2800, 800000
    d = H * dh
    assert T * ld > 2 ** 31
    qkv = torch.empty(T, ld, dtype=torch.float16, device="cuda")[:, :3 * d]
    dqkv = torch.empty(T, ld, dtype=torch.float16, device="cuda")[:, :3 * d]
    cu = torch.tensor([0, 2500, 2731, 2800], dtype=torch.int32, device="cuda")
    qkv.copy_(randn(81, T, 3 * d))
    dout = (0.05 * randn(82, T, d)).half()
    out, lse = run_forward(m, cu, qkv, H, 2500)
    check_forward(cu, qkv.contiguous(), H, out, lse)
    ws = torch.empty(m.attention_backward_workspace(3, T, H), dtype=torch.uint8, device="cuda")
    m.attention_backward(qkv, cu, 2500, H, out, lse, dout, dqkv, ws, stream=torch.cuda.current_stream())
    check_backward(cu, qkv.contiguous(), H, out, lse, dout, dqkv.contiguous())


def test_layernorm_offsets_beyond_32_bits(m):
    T, d = 1_700_001, 1280
    assert T * d > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(83)
    x = torch.empty(T, d, dtype=torch.float16, device="cuda").normal_(generator=gen)
    w, b = 1 + 0.2 * randn(84, d), 0.1 * randn(85, d)
    y, mean, rstd = run_ln(m, x, w, b, "f16")
    ends = [slice(0, 100), slice(T - 100, T)]
    for at in ends:
        check_ln(x[at], w, b, y[at], mean[at], rstd[at])
    dy = y
    dx, dw, db = run_ln_backward(m, dy, x, w, mean, rstd)
    for at in ends:   # the rows' own gradient; that of the weights is over all of them
        small = run_ln_backward(m, dy[at], x[at], w, mean[at], rstd[at])
        check_ln_backward(dy[at], x[at], w, mean[at], rstd[at], None, dx[at], *small[1:])
    want_w, want_b, size_w, size_b = (torch.zeros(d, dtype=torch.float64, device="cuda") for _ in range(4))
    for at in range(0, T, 100_000):
        at = slice(at, at + 100_000)
        g, xh = dy[at].double(), (x[at].double() - mean[at].double()[:, None]) * rstd[at].double()[:, None]
        want_b += g.sum(0)
        size_b += g.abs().sum(0)
        want_w += (g * xh).sum(0)
        size_w += (g * xh).abs().sum(0)
    # At least 148 blocks share the rows, each adding its own up one after another. A term of dw also carries
    # the rounding of xh, a few E of |x| rstd (rstd and |x| are near 1 here).
    N = (T / 148 + 64) * E
    within(dw, want_w, N * size_w + 8 * E * size_b, "dw")
    within(db, want_b, N * size_b, "db")


def test_logits_offsets_beyond_32_bits(m):
    T, V, ld = 70_000, 33, 32768
    assert T * ld > 2 ** 31
    for V in (33, 300):
        x = torch.empty(T, ld, dtype=torch.float16, device="cuda")[:, :V]
        dx = torch.empty(T, ld, dtype=torch.float16, device="cuda")[:, :V]
        small, ids, top, dloss = distill_inputs(T, V, 4, "f16", seed=86)
        x.copy_(small)
        targets = ids[:, 0].contiguous()
        check_logprobs(small, targets, *run_logprobs(m, x, targets, 4))
        loss, lse = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
        m.distill_loss(x, ids, top, loss, lse, stream=torch.cuda.current_stream())
        m.distill_backward(x, ids, top, lse, dloss, dx, stream=torch.cuda.current_stream())
        check_distill(small, ids, top, dloss, 1.0, loss, lse, dx)


@pytest.mark.parametrize("T, d", [(384, 96), (385, 96), (384, 5121), (385, 5121), (2, 9000), (400, 9000), (3000, 8), (3000, 1)])
def test_layernorm_few_and_many_rows_and_wide_ones(m, T, d):
    x, w, b = ln_inputs(T, d, "f32", seed=87)
    y, mean, rstd = run_ln(m, x, w, b, "bf16")
    check_ln(x, w, b, y, mean, rstd)
    dy = (0.05 * randn(88, T, d)).bfloat16()
    dres = randn(89, T, d)
    check_ln_backward(dy, x, w, mean, rstd, dres, *run_ln_backward(m, dy, x, w, mean, rstd, dres))


def test_rows_operators_in_a_graph(m):
    """Captured calls answer for what their buffers hold when they are replayed."""
    for T, d, V in ((40, 64, 33), (900, 320, 3001)):
        k = 5
        x, w, b = ln_inputs(T, d, "f32", seed=90)
        dy = 0.05 * randn(91, T, d)
        logits, ids, top, dloss = distill_inputs(T, V, k, "f32", seed=92)
        targets = ids[:, 1].contiguous()
        buffers = [torch.zeros_like(t) for t in (x, dy, logits, dloss)]
        got = {}
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        run_ln(m, x, w, b, "f32")
        torch.cuda.synchronize()

        def step(x, dy, logits, dloss):
            y, mean, rstd = run_ln(m, x, w, b, "f32")
            return (y, mean, rstd, *run_ln_backward(m, dy, x, w, mean, rstd), *run_logprobs(m, logits, targets, k),
                    *run_distill(m, logits, ids, top, dloss, 2.0))

        with torch.cuda.graph(graph, stream=stream):
            got = step(*buffers)
        for buf, t in zip(buffers, (x, dy, logits, dloss)):
            buf.copy_(t)
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(got, step(x, dy, logits, dloss)):
            assert torch.equal(a, c)


def test_two_streams_at_once(m):
    """Calls that run side by side, with a workspace each, do not disturb one another."""
    H, dh = 4, 32
    inputs = [attention_inputs([300, 17, 250 + i], H, dh, "f16", seed=93 + i) for i in range(2)]
    norms = [(*ln_inputs(2000, 320, "f32", seed=95 + i), randn(97 + i, 2000, 320).half()) for i in range(2)]

    def step(i):
        cu, qkv, dout = inputs[i]
        out, lse = run_forward(m, cu, qkv, H, 300)
        x, w, b, dy = norms[i]
        y, mean, rstd = run_ln(m, x, w, b, "f16")
        return (out, lse, run_backward(m, cu, qkv, H, 300, out, lse, dout), y, *run_ln_backward(m, dy, x, w, mean, rstd))

    alone = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    together = []
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                together.append((i, step(i)))
    torch.cuda.synchronize()
    for i, got in together:
        for a, c in zip(got, alone[i]):
            assert torch.equal(a, c)


def test_limits_of_sizes_and_temperatures(m, esm):
    L, big = esm.lib(), 2 ** 30 + 1
    assert L.esm_token_logprobs(m._ctx, 0, None, big, 5, big, None, 0, None, None, None, None, None) == esm.ESM_EINVAL
    assert "vocabulary" in L.esm_last_error(m._ctx).decode()
    assert L.esm_layernorm(m._ctx, 0, 0, None, None, None, 1e-5, 1, big // 2 + 1, None, None, None, None) == esm.ESM_EINVAL
    assert "columns" in L.esm_last_error(m._ctx).decode()
    assert L.esm_attention(m._ctx, 1, None, 24, None, 1, big, 5, 1, 8, 1.0, None, 8, None, None) == esm.ESM_EINVAL
    assert "bad B, T" in L.esm_last_error(m._ctx).decode()
    x, ids, top, dloss = distill_inputs(4, 33, 3, "f32", seed=99)
    for tau in (1e-7, 1e7):
        with pytest.raises(esm.EsmError, match="temperature"):
            run_distill(m, x, ids, top, dloss, tau)


def test_score_refuses_more_than_was_reserved(esm):
    cfg = esm.EsmConfig(320, 1280, 1, 20, 33, 64, 0)
    model = esm.Model(0)
    model.load_tensors(cfg, esm.DTYPE_FP32, esm.synth_fp32_tensors(cfg, seed=3))
    seq = np.arange(10, dtype=np.int32) + 4
    with pytest.raises(esm.EsmError, match="esm_reserve"):
        model.score([seq])
    model.reserve(25, 3, 12)
    for seqs in ([seq[:2]] * 4, [seq] * 3, [np.tile(seq, 2)]):   # sequences, tokens, one sequence's length
        with pytest.raises(esm.EsmError) as e:
            model.score(seqs)
        assert e.value.code == esm.ESM_ECAPACITY
    with pytest.raises(esm.EsmError, match="length outside"):
        model.score([seq, seq[:0]])
    assert model.score([seq, seq])["logp"].shape == (2, 10)
    model.close()


@pytest.mark.parametrize("dh", [24, 64])
def test_attention_backward_of_ragged_batches_is_reproducible(m, dh):
    """Which block works on which item depends on timing here; the results do not."""
    lens = [int(n) for n in np.random.default_rng(dh).integers(1, 500, 40)]
    cu, qkv, dout = attention_inputs(lens, 12, dh, "f16", seed=100 + dh)
    out, lse = run_forward(m, cu, qkv, 12, 500)
    dqkv = run_backward(m, cu, qkv, 12, 500, out, lse, dout)
    check_backward(cu, qkv, 12, out, lse, dout, dqkv)
    for _ in range(3):
        assert torch.equal(run_backward(m, cu, qkv, 12, 500, out, lse, dout), dqkv)


@pytest.mark.parametrize("dh", [16, 64])
def test_attention_lse_is_exact_to_32_bits(m, dh):
    """Exponentials within 2^-21 of exact (2.2e-7, or the exp2 instruction's 2^-22 with its rounding), summed in 32
    bits: 32 of a row's columns at a time, then over the steps, and rescaled at most once a step."""
    H, lens = 3, [1, 2, 3, 5, 33, 64, 200, 700]
    cu, qkv, _ = attention_inputs(lens, H, dh, "bf16", seed=110 + dh, sharp=0.5)
    out, lse = run_forward(m, cu, qkv, H, 700)
    scale = dh ** -0.5
    for a, b in sequences(cu):
        q, k, _ = (split_heads(x, H) for x in qkv[a:b].split(H * dh, 1))
        want = torch.logsumexp(scale * q @ k.transpose(-1, -2), -1)
        es = score_error(q, k, scale).amax(-1)
        within(lse[:, a:b], want, es + 2.0 ** -21 + (32 + 3 * (b - a) / 32) * E + 8 * E * (1 + want.abs()), "lse")
