"""Block-scaled e4m3 (the quantiser, the dense and the grouped product) and the routing by scores, against their formulas in 64 bits.

Tolerances.  The narrowing is exact: every rounding point of its definition is reproduced.  A product of e4m3 values is exact in f32;
an MMA adds 32 of them to its accumulator with at least 23 bits kept, so a block's sum is off by at most 4 * 33 * 2^-23 of the sum of
magnitudes, and the f32 sums over the blocks add 2^-24 per block and three roundings of the scales: ``_sum_error``.  A result is then
off by half a step of its type: bf16 2^-8, e4m3 2^-4 (2^-10 of the scale among the subnormals), and SiLU by the error of its functions.
"""

import numpy as np
import pytest

from oracle import codec
from tests import util
from tests.util import bf16_randn, e4m3_randn, f32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qb():
    import quark_b200 as q

    q._lib.require_device(0)
    yield q
    q.runtime.synchronize()
    assert q._lib.device_status() == 0


def T(qb, arr, dtype=None):
    return qb.QuarkTensor.from_numpy(np.ascontiguousarray(arr), dtype=dtype)


def blocks(n):
    return -(-n // 128)


# ------------------------------------------------------------------------------------------------------------ narrowing


def narrow(x, tile=1, pow2=False):
    """The definition: f32 quotient, reciprocal and product, e4m3 by the codec.  x f32 [rows, cols] -> bytes, scales [row blocks, blocks]."""
    rows, cols = x.shape
    rb, kb = -(-rows // tile), blocks(cols)
    q, scale = np.zeros((rows, cols), np.uint8), np.ones((rb, kb), np.float32)
    for i in range(rb):
        for b in range(kb):
            at = np.s_[i * tile : (i + 1) * tile, b * 128 : (b + 1) * 128]
            part = x[at]
            top = np.float32(np.nanmax(np.abs(part))) if np.any(~np.isnan(part)) else np.float32(0)
            s = np.float32(1)
            if top != 0:
                s = max(np.float32(top / np.float32(448)), np.float32(2.0**-126))
                if pow2 and np.isfinite(top):
                    s = np.float32(2.0**-126)
                    while 448.0 * float(s) < float(top):
                        s = np.float32(s * 2)
            scale[i, b] = s
            with np.errstate(invalid="ignore"):
                q[at] = codec.f32_to_e4m3((part * (np.float32(1) / s)).astype(np.float32))
    return q, scale


@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 2048), (3, 112), (129, 272), (300, 640), (2500, 1040)])
@pytest.mark.parametrize("src", ["bf16", "f32"])
@pytest.mark.parametrize("tile", [1, 128])
@pytest.mark.parametrize("pow2", [False, True])
def test_narrowing_is_the_definition(qb, rows, cols, src, tile, pow2):
    r = util.rng([1, rows, cols])
    x = (r.standard_normal((rows, cols)) * np.exp2(r.integers(-20, 12, (rows, 1)))).astype(np.float32)
    x[rows // 2, : min(cols, 128)] = 0  # a block of zeros (tile 1)
    if src == "bf16":
        carrier = codec.f32_to_bf16(x)
        x = f32(carrier, "bf16")
    else:
        carrier = x
    q, s = qb.qf.quantize_e4m3_blocks(T(qb, carrier, src), tile_rows=tile, pow2=pow2)
    wq, ws = narrow(x, tile, pow2)
    assert q.dtype == "e4m3" and tuple(q.shape) == (rows, cols)
    np.testing.assert_array_equal(s.to_numpy(), ws.T if tile == 1 else ws)
    np.testing.assert_array_equal(q.to_numpy(), wq)


@pytest.mark.parametrize("pow2", [False, True])
def test_narrowing_of_extreme_values(qb, pow2):
    x = np.zeros((8, 256), np.float32)
    x[0, :3] = [1e-45, -1e-45, 0]  # the scale's lowest value keeps its reciprocal finite
    x[1, 0] = np.float32(3.3e38)
    x[2, :2] = [np.nan, 2.5]
    x[3, :] = np.nan
    x[4, :2] = [448.0 * 2.0**-5, 1]  # the top code exactly: no scale above it
    x[5, 0] = np.nextafter(np.float32(448.0), np.float32(1e9))
    x[6, 130] = -7.0
    x[7, :4] = [2.0**-126, 2.0**-130, -(2.0**-120), 0]
    q, s = qb.qf.quantize_e4m3_blocks(T(qb, x), pow2=pow2)
    wq, ws = narrow(x, 1, pow2)
    np.testing.assert_array_equal(s.to_numpy(), ws.T)
    got = q.to_numpy()
    nan = np.isnan(x)
    assert np.all((got[nan] & 0x7F) == 0x7F)
    np.testing.assert_array_equal(got[~nan], wq[~nan])
    x[:] = 1.0
    x[1, 5] = np.inf
    v = codec.e4m3_to_f32(qb.qf.quantize_e4m3_blocks(T(qb, x), pow2=pow2)[0].to_numpy())
    assert np.isnan(v[1, 5]) and np.all(v[1, :5] == 0) and np.all(v[0] == v[0, 0]) and np.all(v[1, 128:] == v[0, 0])


def test_narrowing_of_gathered_rows_and_of_a_batch(qb):
    r = util.rng(2)
    x = bf16_randn(r, (70, 400))
    X = T(qb, x, "bf16")
    q, s = (t.to_numpy() for t in qb.qf.quantize_e4m3_blocks(X))
    idx = np.array([5, -1, 69, 5, 70, 0, 1 << 30, -(1 << 31), 33], np.int32)
    out, sc = T(qb, np.full((9, 400), 0x55, np.uint8), "e4m3"), T(qb, np.full((4, 9), -3.0, np.float32))
    qb.qf.quantize_e4m3_blocks(X, row_index=T(qb, idx), out=out, scale_out=sc)
    o, c = out.to_numpy(), sc.to_numpy()
    for i, j in enumerate(idx):
        if 0 <= j < 70:
            np.testing.assert_array_equal(o[i], q[j])
            np.testing.assert_array_equal(c[:, i], s[:, j])
        else:  # left as they were
            assert np.all(o[i] == 0x55) and np.all(c[:, i] == -3.0)
    w = bf16_randn(r, (3, 200, 272))
    q, s = qb.qf.quantize_e4m3_blocks(T(qb, w, "bf16"), tile_rows=128)
    assert tuple(s.shape) == (3, 2, 3)
    for e in range(3):
        wq, ws = narrow(f32(w[e], "bf16"), 128)
        np.testing.assert_array_equal(q.to_numpy()[e], wq)
        np.testing.assert_array_equal(s.to_numpy()[e], ws)


# ------------------------------------------------------------------------------------------------------------- products


class Operands:
    def __init__(self, r, M, N, K, experts=1):
        kb = blocks(K)
        self.A, self.B = e4m3_randn(r, (M, K), 8.0), e4m3_randn(r, (experts * N, K), 8.0)
        self.sa = np.exp2(r.uniform(-6, 2, (kb, M))).astype(np.float32)
        self.sb = np.exp2(r.uniform(-9, -3, (experts, blocks(N), kb))).astype(np.float32)
        self.M, self.N, self.K, self.experts = M, N, K, experts

    def tensors(self, qb):
        return T(qb, self.A, "e4m3"), T(qb, self.B, "e4m3"), T(qb, self.sa), T(qb, self.sb.reshape(-1, self.sb.shape[2]) if self.experts == 1 else self.sb)

    def product(self, rows=slice(None), expert=0):
        """The sum in 64 bits and the sum of the magnitudes."""
        N = self.N
        a = codec.e4m3_to_f32(self.A[rows]).astype(np.float64) * np.repeat(self.sa[:, rows].T.astype(np.float64), 128, 1)[:, : self.K]
        sb = np.repeat(np.repeat(self.sb[expert].astype(np.float64), 128, 0)[:N], 128, 1)[:, : self.K]
        b = codec.e4m3_to_f32(self.B[expert * N : (expert + 1) * N]).astype(np.float64) * sb
        return a @ b.T, np.abs(a) @ np.abs(b).T

    def sum_error(self, mags):
        return mags * (4 * 33 * 2.0**-23 + (blocks(self.K) + 3) * 2.0**-24)


def silu(x):
    return x / (1 + np.exp(-x))


def epilogue(y, err, *, bias=None, act=None, gate=None, residual=None, groups=1, out="bf16"):
    """The epilogue in 64 bits and how far an f32 one may be off before the cast."""
    if bias is not None:
        y = y + f32(bias, "bf16").astype(np.float64)
        err = err + np.abs(y) * 2.0**-23
    if act:
        # |silu'| <= 1.1; bf16 goes through tanh.approx (2^-11 relative), else exp (2 + 1.16 |x| ulp) and a division of 2 ulp
        err = 1.1 * err + (np.abs(y) * 2.0**-12 if out == "bf16" else np.abs(silu(y)) * (6 + 1.2 * np.abs(y)) * 2.0**-23 + 1e-37)
        y = silu(y)
    if gate is not None:
        g = np.repeat(f32(gate, "bf16").astype(np.float64), y.shape[0] // groups, 0)
        y, err = f32(residual, "bf16").astype(np.float64) + g * y, err * np.abs(g)
        err = err + (np.abs(y) + np.abs(f32(residual, "bf16"))) * 2.0**-22
    return y, err


def check(got, scale, y, err, out, what=""):
    """``got`` as f32 values (e4m3: without their scales)."""
    if out == "e4m3":
        N = y.shape[1]
        tops = np.stack([np.abs(y[:, b * 128 : (b + 1) * 128]).max(1) for b in range(blocks(N))])
        err_top = np.stack([err[:, b * 128 : (b + 1) * 128].max(1) for b in range(blocks(N))])
        assert np.all(np.abs(scale * 448.0 - tops) <= err_top + tops * 2.0**-22), what
        s = np.repeat(scale.T.astype(np.float64), 128, 1)[:, :N]
        assert np.all(np.abs(got * s - y) <= np.abs(y) * 2.0**-4 + s * 2.0**-10 + err * (1 + 2.0**-3)), what
    else:
        half = 2.0**-8 if out == "bf16" else 2.0**-24
        bad = np.abs(got - y) > (np.abs(y) + err) * half + err
        assert not bad.any(), f"{what}: {bad.mean():.2e} of the values, worst at {np.argwhere(bad)[0]}"


def values(t):
    a = t.to_numpy()
    return a if t.dtype == "f32" else f32(a, "bf16") if t.dtype == "bf16" else codec.e4m3_to_f32(a)


@pytest.mark.parametrize("M,N,K", [
    (1, 8, 16), (1, 2048, 2048), (7, 72, 144), (128, 128, 128), (128, 512, 1152), (130, 264, 640), (257, 1000, 400), (300, 136, 5008), (5, 64, 8192),
])  # fmt: skip
@pytest.mark.parametrize("out", ["bf16", "f32", "e4m3"])
def test_product_of_block_scaled_operands(qb, M, N, K, out):
    r = util.rng([3, M, N, K])
    op = Operands(r, M, N, K)
    got = qb.qf.gemm_blocks(*op.tensors(qb), out_dtype=out)
    got, scale = got if out == "e4m3" else (got, None)
    y, mags = op.product()
    check(values(got), scale.to_numpy() if scale else None, y, op.sum_error(mags), out, f"{M}x{N}x{K} {out}")


@pytest.mark.parametrize("M,N,K,groups", [(1, 64, 128, 1), (6, 136, 272, 3), (256, 200, 384, 2), (384, 512, 2064, 1), (140, 264, 1024, 70)])
@pytest.mark.parametrize("kind", ["bias", "silu", "bias_silu", "gate", "bias_silu_gate"])
@pytest.mark.parametrize("out", ["bf16", "f32", "e4m3"])
def test_epilogues(qb, M, N, K, groups, kind, out):
    r = util.rng([4, M, N])
    op = Operands(r, M, N, K)
    kw, ref = {}, dict(out=out)
    if "bias" in kind:
        ref["bias"] = bf16_randn(r, (N,))
        kw["bias"] = T(qb, ref["bias"], "bf16")
    if "silu" in kind:
        ref["act"] = kw["activation"] = "silu"
    if "gate" in kind:
        ref.update(gate=bf16_randn(r, (groups, N)), residual=bf16_randn(r, (M, N)), groups=groups)
        kw.update(gate=T(qb, ref["gate"], "bf16"), residual=T(qb, ref["residual"], "bf16"), gate_groups=groups)
    got = qb.qf.gemm_blocks(*op.tensors(qb), out_dtype=out, **kw)
    got, scale = got if out == "e4m3" else (got, None)
    y, mags = op.product()
    y, err = epilogue(y, op.sum_error(mags), **ref)
    check(values(got), scale.to_numpy() if scale else None, y, err, out, f"{M}x{N}x{K} {kind} {out}")


@pytest.mark.parametrize("tile_n,split_k", [(64, 1), (128, 1), (256, 1), (64, 2), (64, 4), (64, 8)])
@pytest.mark.parametrize("M,N,K", [(3, 72, 2064), (200, 328, 1040)])
def test_forced_tiles_and_slices(qb, M, N, K, tile_n, split_k):
    r = util.rng([5, M])
    op = Operands(r, M, N, K)
    t = op.tensors(qb)
    y, mags = op.product()
    gate, res = bf16_randn(r, (1, N)), bf16_randn(r, (M, N))
    if split_k == 1 and tile_n > 64:
        q, s = qb.qf.gemm_blocks(*t, out_dtype="e4m3", tile_n=tile_n)
        check(values(q), s.to_numpy(), y, op.sum_error(mags), "e4m3", f"{tile_n}")
    for out, kw in (("f32", {}), ("bf16", dict(gate=T(qb, gate, "bf16"), residual=T(qb, res, "bf16"), activation="silu"))):
        got = qb.qf.gemm_blocks(*t, out_dtype=out, tile_n=tile_n, split_k=split_k, b_constant=True, **kw)
        w, err = epilogue(y, op.sum_error(mags), out=out, **(dict(act="silu", gate=gate, residual=res) if kw else {}))
        check(values(got), None, w, err, out, f"{tile_n} {split_k} {out}")


@pytest.mark.parametrize("tile_n", [128, 256])
def test_power_of_two_result_scales(qb, tile_n):
    r = util.rng(6)
    op = Operands(r, 140, 264, 512)
    q, s = qb.qf.gemm_blocks(*op.tensors(qb), out_dtype="e4m3", pow2=True, tile_n=tile_n)
    y, mags = op.product()
    err, sc = op.sum_error(mags), s.to_numpy()
    assert np.all(np.frexp(sc)[0] == 0.5)
    for b in range(3):
        top = np.abs(y[:, b * 128 : (b + 1) * 128]).max(1)
        assert np.all(448.0 * sc[b] >= top * (1 - 1e-5)) and np.all(224.0 * sc[b] <= top * (1 + 1e-5))
    wide = np.repeat(sc.T.astype(np.float64), 128, 1)[:, :264]
    assert np.all(np.abs(values(q) * wide - y) <= np.abs(y) * 2.0**-4 + wide * 2.0**-10 + err * (1 + 2.0**-3))


def test_dead_values_stay_in_their_row_and_column(qb):
    """NaN operands reach their own row and column only, and rows of a partial tile do not see what lies behind them."""
    r = util.rng(7)
    op = Operands(r, 133, 200, 256)
    op.A[40, 130], op.B[77, 3] = 0x7F, 0xFF
    got = values(qb.qf.gemm_blocks(*op.tensors(qb), out_dtype="f32"))
    bad = np.zeros((133, 200), bool)
    bad[40], bad[:, 77] = True, True
    np.testing.assert_array_equal(np.isnan(got), bad)


def test_quantised_linear_end_to_end(qb):
    """A linear through the quantisers: close to the unquantised product, and channels of very different size keep their relative precision."""
    r = util.rng(8)
    x = (r.standard_normal((96, 1024)) * np.exp2(r.integers(-10, 10, (1, 8))).repeat(128, 1)).astype(np.float32)
    w = (r.standard_normal((256, 1024)) * 0.03 / np.exp2(r.integers(-10, 10, (1, 8))).repeat(128, 1)).astype(np.float32)
    qf = qb.qf
    a, sa = qf.quantize_e4m3_blocks(T(qb, x))
    b, sb = qf.quantize_e4m3_blocks(T(qb, w), tile_rows=128)
    got = values(qf.gemm_blocks(a, b, sa, sb, out_dtype="f32"))
    want = x.astype(np.float64) @ w.astype(np.float64).T
    # every operand is off by at most 2^-4 of itself (uniformly about 0.29 of that): rounding noise of independent terms
    assert np.linalg.norm(got - want) <= 2 * 2.0**-4 * np.linalg.norm(want)


# --------------------------------------------------------------------------------------------------------------- experts


@pytest.mark.parametrize("live,N,K", [
    ([[128]], 64, 128),
    ([[128, 3], [1], [], [128, 128, 32]], 328, 192),
    ([[33], [5], [128, 64]], 136, 2064),
])  # fmt: skip
@pytest.mark.parametrize("out", ["bf16", "f32", "e4m3"])
@pytest.mark.parametrize("act,tile_n", [(None, 0), ("silu", 0), (None, 256), ("silu", 128), (None, 64)])
def test_grouped_product_by_expert_runs(qb, live, N, K, out, act, tile_n):
    if out == "e4m3" and tile_n == 64:
        with pytest.raises(qb._lib.QbError):  # a group of 128 results is one tile's
            qb.qf.gemm_grouped_blocks(*Operands(util.rng(9), 128, N, K, experts=1).tensors(qb), T(qb, np.zeros(1, np.int32)), T(qb, np.ones(1, np.int32)), n_experts=1,
                                      out_dtype=out, tile_n=tile_n)  # fmt: skip
        return
    r = util.rng([9, N, K])
    table = [(e, n) for e, runs in enumerate(live) for n in runs] + [(-1, 0), (len(live), 128)]  # the last one has no such expert
    te, tr = (np.array(c, np.int32) for c in zip(*table))
    M, E = 128 * len(table), len(live)
    op = Operands(r, M, N, K, experts=E)
    A, B, sa, sb = op.tensors(qb)
    carrier = {"bf16": np.uint16, "f32": np.float32, "e4m3": np.uint8}[out]
    o = T(qb, np.full((M, N), 85, carrier), out)
    so = T(qb, np.full((blocks(N), M), -5.0, np.float32)) if out == "e4m3" else None
    before = values(o)[0, 0]
    qb.qf.gemm_grouped_blocks(A, B, sa, sb, T(qb, te), T(qb, tr), n_experts=E, activation=act, out=o, scale_out=so, tile_n=tile_n)
    got = values(o)
    for i, (e, n) in enumerate(table):
        rows = slice(128 * i, 128 * i + (n if 0 <= e < E else 0))
        if rows.stop > rows.start:
            y, mags = op.product(rows, e)
            y, err = epilogue(y, op.sum_error(mags), act=act, out=out)
            check(got[rows], so.to_numpy()[:, rows] if so else None, y, err, out, f"tile {i}")
        assert np.all(got[rows.stop : 128 * (i + 1)] == before)  # left as they were
        if so:
            assert np.all(so.to_numpy()[:, rows.stop : 128 * (i + 1)] == -5.0)


# --------------------------------------------------------------------------------------------------------------- routing


def route_scores(logits, scoring):
    x = logits.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        if scoring == "softmax":
            m = x.max(1, keepdims=True)
            s = np.exp(x - np.where(np.isinf(m), 0, m))
            t = s.sum(1, keepdims=True)
            return np.where(t == 0, 0, s / t)
        return 1 / (1 + np.exp(-x))


def route(logits, bias, k, scoring, groups=1, kept=1, top=1, renorm=True, factor=1.0):
    M, E = logits.shape
    s = route_scores(logits, scoring)
    c = s + (bias.astype(np.float64) if bias is not None else 0)
    if groups > 1 and kept < groups:
        per = -np.sort(-c.reshape(M, groups, -1), 2)[:, :, :top].sum(2)
        keep = np.zeros((M, groups), bool)
        np.put_along_axis(keep, np.argsort(-per, 1, kind="stable")[:, :kept], True, 1)
        c = np.where(np.repeat(keep, E // groups, 1), c, -np.inf)
        c = np.where(np.repeat(keep, E // groups, 1) & np.isinf(c), -1e300, c)  # a masked expert of a kept group comes before the others
    e = np.argsort(-c, 1, kind="stable")[:, :k]
    w = np.take_along_axis(s, e, 1)
    if renorm:
        t = w.sum(1, keepdims=True)
        w = np.where(t == 0, 0, w / np.where(t == 0, 1, t))
    return e, w * factor


def slot_tables(e, E):
    M, k = e.shape
    n = min(E, M * k) + (M * k - min(E, M * k)) // 128
    st, ts, te, tr, at = np.full(n * 128, -1), np.zeros((M, k), int), np.full(n, -1), np.zeros(n, int), 0
    for x in range(E):
        m, j = np.nonzero(e == x)
        here = at * 128 + np.arange(m.size)
        st[here], ts[m, j] = m, here
        c = blocks(m.size)
        te[at : at + c], tr[at : at + c] = x, np.minimum(m.size - 128 * np.arange(c), 128)
        at += c
    return st, ts, te, tr


def check_routing(got, e, w, E):
    np.testing.assert_array_equal(got.experts.to_numpy(), e)
    # an exponential of 2 ulp, a sum of at most 32 (or a softmax over 512), a division, a product
    np.testing.assert_allclose(got.weights.to_numpy(), w, rtol=40 * 2.0**-24, atol=1e-37)
    st, ts, te, tr = slot_tables(e, E)
    np.testing.assert_array_equal(got.slot_token.to_numpy(), st)
    np.testing.assert_array_equal(got.token_slot.to_numpy(), ts)
    np.testing.assert_array_equal(got.tile_expert.to_numpy(), te)
    np.testing.assert_array_equal(got.tile_rows.to_numpy(), tr)
    sw = np.zeros(st.size, np.float32)
    sw[ts] = got.weights.to_numpy()
    np.testing.assert_array_equal(got.slot_weight.to_numpy(), sw)


@pytest.mark.parametrize("M,E,k,groups,kept,top", [
    (1, 8, 2, 1, 1, 1), (1, 256, 8, 8, 4, 2), (3, 1, 1, 1, 1, 1), (64, 64, 6, 8, 3, 1), (65, 160, 6, 8, 3, 2), (200, 96, 4, 4, 2, 2), (130, 40, 5, 8, 2, 1),
    (1000, 512, 32, 16, 8, 2), (2049, 256, 8, 8, 4, 2), (700, 16, 16, 1, 1, 1), (90, 300, 7, 30, 5, 2), (77, 512, 8, 32, 4, 1), (129, 264, 8, 4, 1, 2),
    (4, 64, 6, 8, 4, 2), (5, 64, 6, 8, 4, 2), (513, 128, 3, 4, 2, 1), (8200, 64, 8, 8, 4, 2),  # tokens of a block: 4, 4, 16, 64
])  # fmt: skip
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_routing(qb, M, E, k, groups, kept, top, scoring, biased):
    r = util.rng([10, M, E])
    dtype = "bf16" if (M + biased) % 2 else "f32"
    x = (1.5 * r.standard_normal((M, E))).astype(np.float32)
    if dtype == "bf16":
        carrier = codec.f32_to_bf16(x)  # many equal logits
        x = f32(carrier, "bf16")
    else:
        carrier = x
    bias = (0.1 * r.standard_normal(E)).astype(np.float32) if biased else None
    renorm, factor = M % 3 != 0, 2.5 if M % 2 else 1.0
    got = qb.qf.moe_route_scored(T(qb, carrier, dtype), T(qb, bias) if biased else None, top_k=k, scoring=scoring, n_groups=groups, topk_groups=kept, group_top=top,
                                 renormalize=renorm, factor=factor)  # fmt: skip
    check_routing(got, *route(x, bias, k, scoring, groups, kept, top, renorm, factor), E)
    plain = qb.qf.moe_route_scored(T(qb, carrier, dtype), T(qb, bias) if biased else None, top_k=k, scoring=scoring, n_groups=groups, topk_groups=kept, group_top=top,
                                   renormalize=renorm, factor=factor, tables=False)  # fmt: skip
    np.testing.assert_array_equal(plain.experts.to_numpy(), got.experts.to_numpy())
    np.testing.assert_array_equal(plain.weights.to_numpy(), got.weights.to_numpy())
    assert plain.slot_token is None


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept,top", [(1, 1, 1), (4, 2, 2), (4, 2, 1)])
@pytest.mark.parametrize("biased", [False, True])
def test_routing_of_equal_and_masked_logits(qb, scoring, groups, kept, top, biased):
    """Equal scores go to the lower index; -inf and the type's lowest value are never chosen while another expert is left; a row
    without any finite logit has weights 0."""
    r = util.rng([11, groups])
    M, E, k = 150, 32, 6
    x = r.integers(-2, 3, (M, E)).astype(np.float32) * 0.5
    x[3:40] = np.where(r.random((37, E)) < 0.7, -np.inf, x[3:40])
    x[40:70] = np.where(r.random((30, E)) < 0.7, np.float32(-3.3e38), x[40:70])
    x[5], x[6] = -np.inf, 0.0
    x[7, 9], x[8, 3] = 0.0, -0.0
    bias = (r.integers(-1, 2, E) * 0.125).astype(np.float32) if biased else None
    got = qb.qf.moe_route_scored(T(qb, x), T(qb, bias) if biased else None, top_k=k, scoring=scoring, n_groups=groups, topk_groups=kept, group_top=top)
    e, w = route(x, bias, k, scoring, groups, kept, top)
    if not biased and groups == 1:
        # the choice is on the logits: -inf after the lowest value, though both score 0
        e = np.argsort(-x.astype(np.float64), 1, kind="stable")[:, :k]
    if biased or groups == 1:
        check_routing(got, e, w, E)
    else:
        check_routing(got, got.experts.to_numpy(), w, E)  # (which of several experts of score 0 is left open)
    assert np.all(got.weights.to_numpy()[5] == 0)


@pytest.mark.parametrize("E,k,groups,kept,top", [(64, 6, 1, 1, 1), (64, 6, 8, 3, 2), (256, 32, 1, 1, 1), (16, 15, 1, 1, 1), (16, 16, 1, 1, 1), (40, 3, 8, 2, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dense", [False, True])
def test_routing_of_close_scores(qb, E, k, groups, kept, top, scoring, dense):
    """Scores that differ by less than a rounding to 32 bits are told apart, be it two of them or all."""
    r = util.rng([15, E, k])
    M = 200
    x = (1.5 * r.standard_normal((M, E))).astype(np.float32)
    bias = (0.1 * r.standard_normal(E)).astype(np.float32)
    if dense:
        x = (np.float32(0.5) + r.integers(-4, 5, (M, E)).astype(np.float32) * np.float32(2.0**-24)).astype(np.float32)
        bias[:] = r.integers(0, 2, E) * np.float32(0.25)
    else:  # expert 1 scores as expert 0 to the last bit or so, and expert 2 as 3 in other tokens
        for m in range(M):
            p, q = (0, 1) if m % 2 else (3, 2)
            s = 1 / (1 + np.exp(-x[m].astype(np.float64)))
            want = s[p] + float(bias[p]) - float(bias[q])
            if 1e-3 < want < 1 - 1e-3:
                x[m, q] = np.float32(np.log(want / (1 - want)))
                x[m, [p, q]] += np.float32(2.0) if m % 3 == 0 else 0
    got = qb.qf.moe_route_scored(T(qb, x), T(qb, bias), top_k=k, scoring=scoring, n_groups=groups, topk_groups=kept, group_top=top)
    e, w = route(x, bias, k, scoring, groups, kept, top)
    if dense and groups > 1:
        # Two experts one step up and down sum to two in the middle but for (2^-24)^2 of a score: below 2^-50, so 64 bits do not say which
        # group is first.  Any of the groups that close to the last one kept will do; the choice inside them is the formula's.
        c = route_scores(x, scoring) + bias.astype(np.float64)
        per = -np.sort(-c.reshape(M, groups, -1), 2)[:, :, :top].sum(2)
        last = -np.sort(-per, 1)[:, kept - 1]
        ge = got.experts.to_numpy()
        for m in range(M):
            used = set(ge[m] // (E // groups))
            assert all(per[m, g] >= last[m] - 2.0**-50 for g in used)
            kept_now = used | {g for g in range(groups) if per[m, g] > last[m] + 2.0**-50}
            assert len(kept_now) <= kept
            inside = np.where(np.isin(np.arange(E) // (E // groups), list(kept_now)), c[m], -np.inf)
            np.testing.assert_array_equal(ge[m], np.argsort(-inside, kind="stable")[:k])
        s = np.take_along_axis(route_scores(x, scoring), ge, 1)
        e, w = ge, s / s.sum(1, keepdims=True)
    check_routing(got, e, w, E)


@pytest.mark.parametrize("E,groups,kept,k", [(16, 4, 2, 3), (64, 8, 3, 6), (256, 8, 4, 8), (512, 16, 5, 8), (40, 5, 2, 4)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_routing_of_groups_whose_best_two_cancel(qb, E, groups, kept, k, scoring):
    """A group's best two values of large size and opposite sign: their sum is small, and what 32 bits lose of it goes by the size of the two."""
    r = util.rng([19, E])
    x = (1.5 * r.standard_normal((400, E))).astype(np.float32)
    bias = np.full((groups, E // groups), -1e6, np.float32)
    size = np.exp2(r.integers(4, 12, groups)).astype(np.float32)
    bias[:, 1], bias[:, -1] = size, -size  # (exact in 64 bits beside a score)
    bias = bias.reshape(-1)
    got = qb.qf.moe_route_scored(T(qb, x), T(qb, bias), top_k=k, scoring=scoring, n_groups=groups, topk_groups=kept, group_top=2)
    check_routing(got, *route(x, bias, k, scoring, groups, kept, 2), E)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("low", [-40.0, -95.0, -150.0, -400.0])
def test_weights_of_choices_with_tiny_scores(qb, scoring, low):
    """The bias picks experts whose scores are far below the row's: what the weights are made of underflows in 32 bits, their ratios do not."""
    r = util.rng([20, int(-low)])
    x = r.standard_normal((70, 64)).astype(np.float32)
    x[:, ::7] += np.float32(low)
    bias = np.zeros(64, np.float32)
    bias[::7] = 2.0 + np.arange(10)  # (apart, whatever the scores)
    for k, renorm in ((1, True), (4, True), (10, True), (4, False)):
        got = qb.qf.moe_route_scored(T(qb, x), T(qb, bias), top_k=k, scoring=scoring, renormalize=renorm)
        e, w = route(x, bias, k, scoring, renorm=renorm)
        assert np.all(e % 7 == 0)
        check_routing(got, e, w, 64)


def test_routing_of_nan(qb):
    """NaN is chosen last, stays in its row, and never leads an index out of range."""
    r = util.rng(12)
    x = r.standard_normal((70, 64)).astype(np.float32)
    clean = x.copy()
    x[10, 5], x[20], x[30, ::2] = np.nan, np.nan, np.nan
    for bias in (None, np.zeros(64, np.float32)):
        for groups in (1, 8):
            got = qb.qf.moe_route_scored(T(qb, x), None if bias is None else T(qb, bias), top_k=4, scoring="sigmoid", n_groups=groups, topk_groups=groups // 2 or 1, group_top=1)
            e = got.experts.to_numpy()
            assert e.min() >= 0 and e.max() < 64 and all(len(set(row)) == 4 for row in e)
            we, ww = route(clean, bias, 4, "sigmoid", groups, groups // 2 or 1, 1)
            rest = np.setdiff1d(np.arange(70), [10, 20, 30])
            np.testing.assert_array_equal(e[rest], we[rest])
            np.testing.assert_allclose(got.weights.to_numpy()[rest], ww[rest], rtol=40 * 2.0**-24)
            assert 5 not in e[10] and not np.any(e[30] % 2 == 0) and np.all(np.isnan(got.weights.to_numpy()[20]))


# -------------------------------------------------------------------------------------------------------------- together


def test_experts_from_logits_to_sum(qb):
    """Routing, gather with narrowing, both products, weighted sum, each fed what the one before made; eager, then as a replayed graph
    beside another one of the same stream."""
    r = util.rng(13)
    qf = qb.qf
    M, E, k, D, H = 150, 16, 3, 256, 384
    x, logits = bf16_randn(r, (M, D)), (1.5 * r.standard_normal((M, E))).astype(np.float32)
    win, wout = bf16_randn(r, (E, H, D), D**-0.5), bf16_randn(r, (E, D, H), H**-0.5)
    X, L = T(qb, x, "bf16"), T(qb, logits)
    w1, s1 = qf.quantize_e4m3_blocks(T(qb, win, "bf16"), tile_rows=128)
    w2, s2 = qf.quantize_e4m3_blocks(T(qb, wout, "bf16"), tile_rows=128)
    n = qf.moe_scored_slots(M, E, k)
    e = lambda *s, dt="f32": qb.QuarkTensor.zeros(*s, dtype=dt)  # noqa: E731

    def buffers():
        return dict(tables=[e(M, k, dt="s32"), e(M, k), e(n, dt="s32"), e(n), e(n // 128, dt="s32"), e(n // 128, dt="s32"), e(M, k, dt="s32")], xq=e(n, D, dt="e4m3"),
                    xs=e(2, n), hq=e(n, H, dt="e4m3"), hs=e(3, n), y=e(n, D), out=e(M, D, dt="bf16"))  # fmt: skip

    def run(b):
        t = qf.moe_route_scored(L, top_k=k, scoring="sigmoid", n_groups=4, topk_groups=2, group_top=2, factor=1.5, out=b["tables"])
        qf.quantize_e4m3_blocks(X, row_index=t.slot_token, out=b["xq"], scale_out=b["xs"])
        qf.gemm_grouped_blocks(b["xq"], w1, b["xs"], s1, t.tile_expert, t.tile_rows, n_experts=E, activation="silu", out=b["hq"], scale_out=b["hs"], b_constant=True)
        qf.gemm_grouped_blocks(b["hq"], w2, b["hs"], s2, t.tile_expert, t.tile_rows, n_experts=E, out=b["y"], b_constant=True)
        return qf.moe_reduce(b["y"], t.slot_weight, t.token_slot, out=b["out"])

    b = buffers()
    got = run(b).to_numpy()
    we, ww = route(logits, None, k, "sigmoid", 4, 2, 2, True, 1.5)
    check_routing(qf.Routing(*b["tables"]), we, ww, E)
    want = np.zeros((M, D))
    f64 = lambda t: f32(t, "bf16").astype(np.float64)  # noqa: E731
    for j in range(k):
        h = silu(np.einsum("md,mhd->mh", f64(x), f64(win)[we[:, j]]))
        want += ww[:, j : j + 1] * np.einsum("mh,mdh->md", h, f64(wout)[we[:, j]])
    # three narrowed operands in turn, each 2^-4 off at most
    assert np.linalg.norm(f32(got, "bf16") - want) <= 3 * 2.0**-4 * np.linalg.norm(want)
    # the same bits replayed, two graphs in turn and the eager call between them
    from quark_b200.runtime import stream

    made = []
    for _ in range(2):
        c = buffers()
        run(c)
        with stream.capture_graph() as cap:
            run(c)
        made.append((c, cap.graph))
    for c, _ in made:
        c["out"].zero_()
        c["y"].zero_()
    for c, g in made:
        g.launch()
        run(b)
    for c, _ in made:
        np.testing.assert_array_equal(c["out"].to_numpy(), got)


def test_calls_on_several_streams_and_replayed_at_once(qb):
    """Routings of many blocks (they meet in a workspace) with products in slices, eager on two streams and replayed from a graph on a third:
    every result is that of the call alone."""
    import ctypes as C

    lib, stream, qf, r = qb._lib.load(), qb.runtime.stream, qb.qf, util.rng(15)
    calls = []
    for M, E in ((4100, 256), (900, 64), (8192, 128)):
        logits, bias = T(qb, r.standard_normal((M, E)).astype(np.float32)), T(qb, (0.1 * r.standard_normal(E)).astype(np.float32))
        n = qf.moe_scored_slots(M, E, 6)
        shapes = [((M, 6), "s32"), ((M, 6), "f32"), ((n,), "s32"), ((n,), "f32"), ((n // 128,), "s32"), ((n // 128,), "s32"), ((M, 6), "s32")]
        outs = [qb.QuarkTensor.zeros(*shape, dtype=d) for shape, d in shapes]
        op, y = Operands(r, 40, 256, 2048).tensors(qb), qb.QuarkTensor.zeros(40, 256, dtype="f32")

        def call(a=(logits, bias), o=outs, op=op, y=y):
            qf.moe_route_scored(*a, top_k=6, scoring="sigmoid", n_groups=8, topk_groups=4, group_top=2, out=o)
            qf.gemm_blocks(*op, out=y, tile_n=64, split_k=4)

        calls.append((call, [*outs, y]))
    want = []
    for call, outs in calls:
        call()
        want.append([t.to_numpy() for t in outs])
        for t in outs:
            t.zero_()
    cap = qb.runtime.capture_graph()
    with cap:
        calls[2][0]()
    qb.runtime.synchronize()
    first, handles = qb.runtime.active_stream(), []
    for _ in range(2):
        p = C.c_void_p()
        qb._lib.check(lib.qb_stream_create(C.byref(p)))
        handles.append(int(p.value))
    try:
        for _ in range(20):
            for handle, run in zip([first, *handles], (calls[0][0], calls[1][0], cap.graph.launch)):
                stream.set_stream(handle)
                run()
    finally:
        stream.set_stream(first)
        qb._lib.check(lib.qb_device_sync())
    for (_, outs), w in zip(calls, want):
        for t, x in zip(outs, w):
            np.testing.assert_array_equal(t.to_numpy(), x)
    for handle in handles:
        qf._OF_STREAM.pop(handle, None)
        qb._lib.check(lib.qb_stream_destroy(C.c_void_p(handle)))


# ---------------------------------------------------------------------------------------------------- offsets past 32 bits


def test_rows_past_32_bits_of_elements(qb):
    """Narrowing and product of 4.3e9 elements each: the first and the last rows are those of a call with them alone."""
    qf, r = qb.qf, util.rng(16)
    M, N, K, part = 4_194_700, 1040, 1024, 300
    x, ends = bf16_randn(r, (2 * part, K)), (slice(0, part), slice(M - part, M))
    X = qb.QuarkTensor.zeros(M, K, dtype="bf16")
    for i, rows in enumerate(ends):
        X.rows(rows.start, rows.stop).copy_from_numpy(x[i * part : (i + 1) * part])
    w, sw = qf.quantize_e4m3_blocks(T(qb, bf16_randn(r, (N, K)), "bf16"), tile_rows=128)
    q, s = qf.quantize_e4m3_blocks(X)
    y = qf.gemm_blocks(q, w, s, sw, out_dtype="bf16", tile_n=128)
    assert np.all(y.rows(M // 2, M // 2 + 8).to_numpy() == 0)
    for i, rows in enumerate(ends):
        qe, se = qf.quantize_e4m3_blocks(T(qb, x[i * part : (i + 1) * part], "bf16"))
        np.testing.assert_array_equal(q.rows(rows.start, rows.stop).to_numpy(), qe.to_numpy())
        for b in range(K // 128):  # [block, row]
            np.testing.assert_array_equal(s.reshape(-1, 1).rows(b * M + rows.start, b * M + rows.stop).to_numpy()[:, 0], se.to_numpy()[b])
        np.testing.assert_array_equal(y.rows(rows.start, rows.stop).to_numpy(), qf.gemm_blocks(qe, w, se, sw, out_dtype="bf16", tile_n=128).to_numpy())


def test_experts_past_32_bits_of_elements(qb):
    """The last of 33 experts, whose weights lie behind 4.3e9 elements, gives what the dense product with its weights gives."""
    qf, r = qb.qf, util.rng(17)
    E, N, K = 33, 8192, 16384
    B = qb.QuarkTensor.empty(E * N, K, dtype="e4m3").zero_()
    B.rows((E - 1) * N, E * N).copy_from_numpy(np.resize(e4m3_randn(r, 1_000_003, 8.0), (N, K)))
    A, sa = T(qb, e4m3_randn(r, (128, K), 8.0), "e4m3"), T(qb, np.exp2(r.uniform(-6, 2, (K // 128, 128))).astype(np.float32))
    sb = np.exp2(r.uniform(-9, -3, (E, N // 128, K // 128))).astype(np.float32)
    got = qf.gemm_grouped_blocks(A, B, sa, T(qb, sb), T(qb, np.array([E - 1], np.int32)), T(qb, np.array([128], np.int32)), n_experts=E, out_dtype="f32", tile_n=128)
    want = qf.gemm_blocks(A, B.rows((E - 1) * N, E * N), sa, T(qb, sb[E - 1]), out_dtype="f32", tile_n=128)
    assert np.any(want.to_numpy() != 0)
    np.testing.assert_array_equal(got.to_numpy(), want.to_numpy())


def test_logits_past_31_bits_of_elements(qb):
    qf, r = qb.qf, util.rng(18)
    M, E, part = 4_194_400, 512, 100
    x, bias = r.standard_normal((part, E)).astype(np.float32), T(qb, (0.1 * r.standard_normal(E)).astype(np.float32))
    X = qb.QuarkTensor.zeros(M, E, dtype="f32")
    X.rows(M - part, M).copy_from_numpy(x)
    kw = dict(top_k=4, scoring="sigmoid", n_groups=16, topk_groups=4, group_top=2, tables=False)
    got, want = qf.moe_route_scored(X, bias, **kw), qf.moe_route_scored(T(qb, x), bias, **kw)
    np.testing.assert_array_equal(got.experts.rows(M - part, M).to_numpy(), want.experts.to_numpy())
    np.testing.assert_array_equal(got.weights.rows(M - part, M).to_numpy(), want.weights.to_numpy())


def test_calls_made_in_c_equal_the_python_path(qb, monkeypatch):
    """Same bytes with and without the extension, and the Python path's errors for what it does not take."""
    qf, r = qb.qf, util.rng(14)
    e = lambda *s, dt="bf16": qb.QuarkTensor.zeros(*s, dtype=dt)  # noqa: E731
    x, idx = T(qb, bf16_randn(r, (24, 256)), "bf16"), T(qb, np.arange(9, dtype=np.int32)[::-1])
    op, gp = Operands(r, 24, 136, 272), Operands(r, 256, 136, 272, experts=2)
    t, gt = op.tensors(qb), gp.tensors(qb)
    te, tr = T(qb, np.array([1, 0], np.int32)), T(qb, np.array([128, 7], np.int32))
    bias, gate, res = (T(qb, bf16_randn(r, s), "bf16") for s in ((136,), (2, 136), (24, 136)))
    lg, lb = T(qb, r.standard_normal((70, 16)).astype(np.float32)), T(qb, r.standard_normal(16).astype(np.float32))
    n = qf.moe_scored_slots(70, 16, 2)
    tabs = lambda: [e(70, 2, dt="s32"), e(70, 2, dt="f32"), e(n, dt="s32"), e(n, dt="f32"), e(n // 128, dt="s32"), e(n // 128, dt="s32"), e(70, 2, dt="s32")]  # noqa: E731
    calls = [
        lambda: qf.quantize_e4m3_blocks(x, out=e(24, 256, dt="e4m3"), scale_out=e(2, 24, dt="f32")),
        lambda: qf.quantize_e4m3_blocks(x, row_index=idx, pow2=True, out=e(9, 256, dt="e4m3"), scale_out=e(2, 9, dt="f32")),
        lambda: qf.quantize_e4m3_blocks(x.reshape(2, 12, 256), tile_rows=128, out=e(2, 12, 256, dt="e4m3"), scale_out=e(2, 1, 2, dt="f32")),
        lambda: [qf.gemm_blocks(*t, out=e(24, 136), bias=bias, activation="silu")],
        lambda: [qf.gemm_blocks(*t, out=e(24, 136, dt="f32"), gate=gate, residual=res, gate_groups=2, tile_n=64)],
        lambda: qf.gemm_blocks(*t, out=e(24, 136, dt="e4m3"), scale_out=e(2, 24, dt="f32"), pow2=True),
        lambda: qf.gemm_grouped_blocks(*gt, te, tr, n_experts=2, out=e(256, 136, dt="e4m3"), scale_out=e(2, 256, dt="f32"), activation="silu"),
        lambda: qf.moe_route_scored(lg, lb, top_k=2, scoring="sigmoid", n_groups=4, topk_groups=2, group_top=2, factor=2.0, out=tabs()),
        lambda: qf.moe_route_scored(lg, top_k=2, tables=False, out=tabs()[:2])[:2],
    ]
    wrong = [
        (TypeError, lambda: qf.quantize_e4m3_blocks(idx.reshape(1, 9), out=e(1, 9, dt="e4m3"), scale_out=e(1, dt="f32"))),
        (TypeError, lambda: qf.quantize_e4m3_blocks(x, out=e(24, 256), scale_out=e(2, 24, dt="f32"))),
        (ValueError, lambda: qf.quantize_e4m3_blocks(x, out=e(24, 240, dt="e4m3"), scale_out=e(2, 24, dt="f32"))),
        (ValueError, lambda: qf.quantize_e4m3_blocks(x, out=e(24, 256, dt="e4m3"), scale_out=e(24, dt="f32"))),
        (ValueError, lambda: qf.quantize_e4m3_blocks(x, tile_rows=64, out=e(24, 256, dt="e4m3"), scale_out=e(2, 24, dt="f32"))),
        (ValueError, lambda: qf.gemm_blocks(t[0], t[1], t[2], T(qb, np.ones((1, 3), np.float32)), out=e(24, 136))),
        (TypeError, lambda: qf.gemm_blocks(e(24, 272), t[1], t[2], t[3], out=e(24, 136))),
        (ValueError, lambda: qf.gemm_blocks(x, t[1], t[2], t[3], out=e(24, 136))),
        (ValueError, lambda: qf.gemm_blocks(*t, out=e(24, 136), gate=gate, residual=res, gate_groups=5)),
        (ValueError, lambda: qf.gemm_blocks(*t, out=e(24, 136), scale_out=e(2, 24, dt="f32"))),
        (ValueError, lambda: qf.gemm_grouped_blocks(*gt, te, tr, n_experts=3, out=e(256, 136))),
        (TypeError, lambda: qf.gemm_grouped_blocks(*gt, te, T(qb, np.ones(2, np.float32)), n_experts=2, out=e(256, 136))),
        (ValueError, lambda: qf.moe_route_scored(lg, top_k=2, scoring="max", out=tabs())),
        (ValueError, lambda: qf.moe_route_scored(lg, top_k=2, n_groups=3, out=tabs())),
        (ValueError, lambda: qf.moe_route_scored(lg, top_k=2, out=tabs()[:2])),
        (TypeError, lambda: qf.moe_route_scored(lg, x, top_k=2, out=tabs())),
    ]
    first = [[u.to_numpy() for u in c()] for c in calls]
    for kind, c in wrong:
        with pytest.raises(kind):
            c()
    monkeypatch.setattr(qf, "_fast", qb._lib._NoFastcall())
    for a, c in zip(first, calls):
        for u, v in zip(a, c()):
            np.testing.assert_array_equal(u, v.to_numpy())
    for kind, c in wrong:
        with pytest.raises(kind):
            c()
