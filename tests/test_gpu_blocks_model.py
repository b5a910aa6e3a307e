"""Block-scaled e4m3 and routing by scores through ``nn`` and the engine: the layers are the chain of their ``qf`` calls, bit for bit, and
close to the unquantised formula; sessions replay their graphs with the bits of the eager passes."""

import numpy as np
import pytest

from oracle import codec
from tests import util
from tests.test_gpu_blocks import blocks, check, epilogue, route
from tests.test_gpu_model import small_cfg
from tests.util import bf16_randn, f32

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


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("M", [1, 77])
def test_linear_with_block_scales(qb, M, bias):
    from quark_b200 import nn

    r = util.rng([20, M])
    K, N = 272, 200
    lin = nn.Linear(K, N, bias=bias)
    w, b, x = bf16_randn(r, (N, K), 0.05), bf16_randn(r, (N,)), bf16_randn(r, (M, K))
    lin.weight.data = T(qb, w, "bf16")
    if bias:
        lin.bias.data = T(qb, b, "bf16")
    lin.prepare(fp8=True, fp8_blocks=True)
    lin.prepare(fp8=True, fp8_blocks=True)  # once only
    X = T(qb, x, "bf16")
    y = lin(X, activation="silu")
    q, s = qb.qf.quantize_e4m3_blocks(X)
    pair = lin((q, s), activation="silu", out=qb.QuarkTensor.zeros(M, N))
    np.testing.assert_array_equal(y.to_numpy(), pair.to_numpy())
    wq, ws = qb.qf.quantize_e4m3_blocks(T(qb, w, "bf16"), tile_rows=128)
    np.testing.assert_array_equal(lin.weight.data.to_numpy(), wq.to_numpy())
    np.testing.assert_array_equal(lin.w_blocks.to_numpy(), ws.to_numpy())
    a = codec.e4m3_to_f32(q.to_numpy()).astype(np.float64) * np.repeat(s.to_numpy().T.astype(np.float64), 128, 1)[:, :K]
    wide = np.repeat(np.repeat(ws.to_numpy().astype(np.float64), 128, 0)[:N], 128, 1)[:, :K]
    v = codec.e4m3_to_f32(wq.to_numpy()).astype(np.float64) * wide
    want, err = epilogue(a @ v.T, np.abs(a) @ np.abs(v).T * (4 * 33 * 2.0**-23 + 6 * 2.0**-24), bias=b if bias else None, act="silu")
    check(f32(y.to_numpy(), "bf16"), None, want, err, "bf16", "linear")
    with pytest.raises(TypeError):
        lin(q)  # e4m3 without its scales
    with pytest.raises(ValueError):
        lin(X, gate=T(qb, bf16_randn(r, (1, N)), "bf16"))


@pytest.mark.parametrize("fuse", [False, True])
def test_mlp_hands_its_hidden_activations_over_with_their_scales(qb, fuse):
    from quark_b200 import nn

    r, qf = util.rng(21), qb.qf
    M, D, H = 130, 256, 640
    mlp = nn.MLP(D, H, D, fuse_silu=fuse)
    w1, w2, x = bf16_randn(r, (H, D), 0.06), bf16_randn(r, (D, H), 0.04), bf16_randn(r, (M, D))
    mlp.fc1.weight.data, mlp.fc2.weight.data = T(qb, w1, "bf16"), T(qb, w2, "bf16")
    for lin in (mlp.fc1, mlp.fc2):
        lin.prepare(fp8=True, fp8_blocks=True)
    gate, X = T(qb, bf16_randn(r, (1, D)), "bf16"), T(qb, x, "bf16")
    got = mlp(X, gate=gate, residual=X, out=qb.QuarkTensor.zeros(M, D)).to_numpy()
    q, s = qf.quantize_e4m3_blocks(X)
    (b1, s1), (b2, s2) = (qf.quantize_e4m3_blocks(T(qb, w, "bf16"), tile_rows=128) for w in (w1, w2))
    if fuse:
        h = qf.gemm_blocks(q, b1, s, s1, activation="silu", out_dtype="e4m3")
    else:
        h = qf.quantize_e4m3_blocks(qf.silu(qf.gemm_blocks(q, b1, s, s1)))
    np.testing.assert_array_equal(got, qf.gemm_blocks(h[0], b2, h[1], s2, gate=gate, residual=X).to_numpy())
    f = lambda t: f32(t, "bf16").astype(np.float64)  # noqa: E731
    hid = f(x) @ f(w1).T
    y = (hid / (1 + np.exp(-hid))) @ f(w2).T
    delta = (f32(got, "bf16") - f(x)) / f(gate.to_numpy())
    # four operands, each off by at most 2^-4 of itself; and bf16's 2^-8 of the sum over the gate
    big = np.abs(f(gate.to_numpy()))[0] > 0.1
    assert np.linalg.norm((delta - y)[:, big]) <= 4 * 2.0**-4 * np.linalg.norm(y[:, big]) + 10 * 2.0**-8 * np.linalg.norm(f(x)[:, big])


@pytest.mark.parametrize("scoring,fp8,fp8_blocks", [(None, True, True), ("softmax", True, True), ("sigmoid", True, True), ("sigmoid", False, False), ("sigmoid", True, False)])
@pytest.mark.parametrize("M", [1, 200])
def test_mixture_of_experts_routed_by_scores(qb, M, scoring, fp8, fp8_blocks):
    from quark_b200 import nn

    r, qf = util.rng([22, M]), qb.qf
    D, H, E, K = 256, 384, 16, 3
    kw = {} if scoring is None else dict(scoring=scoring, n_groups=4, topk_groups=2, group_top=2, renormalize=scoring == "sigmoid", route_scale=1.5, score_bias=True)
    moe = nn.MoE(M, D, H, E, K, **kw)
    x, wr = bf16_randn(r, (M, D)), bf16_randn(r, (E, D), 0.1)
    win, wout = bf16_randn(r, (E, H, D), D**-0.5), bf16_randn(r, (E, D, H), H**-0.5)
    bias = (0.1 * r.standard_normal(E)).astype(np.float32) if scoring else None
    moe.router.weight.data = T(qb, wr, "bf16")
    moe.expert_in.data, moe.expert_out.data = T(qb, win.reshape(E * H, D), "bf16"), T(qb, wout.reshape(E * D, H), "bf16")
    if scoring:
        assert "score_bias" in moe.state_dict()
        moe.score_bias.data = T(qb, bias)
    moe.prepare(fp8=fp8, fp8_blocks=fp8_blocks)
    X = T(qb, x, "bf16")
    got = f32(moe(X).to_numpy(), "bf16")
    logits = moe.router(X)
    logits = logits.to_numpy() if scoring else f32(logits.to_numpy(), "bf16")
    e, w = route(logits, bias, K, scoring or "softmax", *((4, 2, 2, scoring == "sigmoid", 1.5) if scoring else ()))
    np.testing.assert_array_equal(moe._bufs[("experts", (M, K), "s32")].to_numpy(), e)
    f = lambda t: f32(t, "bf16").astype(np.float64)  # noqa: E731
    want = np.zeros((M, D))
    for j in range(K):
        h = np.einsum("md,mhd->mh", f(x), f(win)[e[:, j]])
        want += w[:, j : j + 1] * np.einsum("mh,mdh->md", h / (1 + np.exp(-h)), f(wout)[e[:, j]])
    # four operands, each off by at most 2^-4 of itself (e4m3; without scales small values lose more, to 2^-10 absolute) or 2^-8 (bf16)
    step = (2.0**-4 if fp8_blocks else 2.0**-3) if fp8 else 2.0**-8
    assert np.linalg.norm(got - want) <= 4 * step * np.linalg.norm(want)


def test_refusals():
    from quark_b200 import nn  # noqa: F401
    from quark_b200.models import QuantConfig, Waypoint15Config

    for kw in (dict(scoring="max"), dict(scoring="sigmoid", schedule="dense"), dict(n_groups=2), dict(score_bias=True), dict(scoring="softmax", n_groups=3),
               dict(scoring="softmax", n_groups=8, topk_groups=4, group_top=2)):  # fmt: skip
        with pytest.raises(ValueError):
            nn.MoE(16, 128, 128, 8, 2, **kw)
    with pytest.raises(ValueError):
        nn.MoE(16, 128, 192, 8, 2).prepare(fp8=True, fp8_blocks=True)  # widths that are no whole tiles
    with pytest.raises(NotImplementedError):
        Waypoint15Config(fp8_blocks=True, tp_world=2)
    with pytest.raises(ValueError):
        Waypoint15Config(moe=True, moe_n_experts=64)  # more than 32 need scoring
    with pytest.raises(ValueError):
        Waypoint15Config(d_model=320, n_heads=5, n_kv_heads=5, moe=True, fp8_blocks=True, quant=QuantConfig.all_fp8())


@pytest.mark.parametrize("kw", [
    dict(),
    dict(fuse_silu=False, fuse_gate_residual=False),
    dict(fuse_qkv_post=False, quilt_factor=2),
    dict(moe=True, moe_n_experts=16, moe_top_k=2, moe_scoring="sigmoid", moe_n_groups=4, moe_topk_groups=2, moe_group_top=2, moe_score_bias=True, moe_route_scale=1.5),
    dict(fp8_scales=True),
])  # fmt: skip
def test_sessions(qb, kw):
    from quark_b200.models import QuantConfig, Waypoint15Config, make_params

    quant = QuantConfig(linear="fp8", kv_cache="bf16", attn_compute="bf16", moe="fp8")
    cfg = Waypoint15Config(**{**small_cfg(qb, "bf16").__dict__, "quant": quant, "fp8_blocks": True, **kw})
    params = make_params(cfg, seed=23, weight_std=0.04)
    r = util.rng(24)
    lats = [codec.f32_to_bf16(r.standard_normal((1, cfg.latent_numel)).astype(np.float32)) for _ in range(2)]
    noise = r.standard_normal((1, cfg.latent_numel)).astype(np.float32)
    outs = []
    for graph, c in ((False, cfg), (True, cfg), (False, Waypoint15Config(**{**cfg.__dict__, "quant": QuantConfig.all_bf16(), "fp8_blocks": False, "fp8_scales": False}))):
        eng = qb.Engine(cfg=c, quant=c.quant, params=params, use_graph=graph)
        if c is cfg:
            assert eng.model.blocks[0].qkv_proj.w_blocks is not None
        for lat in lats:
            eng.append_frame(lat)
        outs.append([eng.gen_frame(noise=noise).reshape(-1) for _ in range(2)])
    for a, b in zip(outs[0], outs[1]):
        np.testing.assert_array_equal(a, b)
    # Every linear's operands are off by 2 - 3 % (rms): with two branches of two or three linears in each of four blocks 15 - 20 % at
    # most if a branch were the whole of the stream, so a cosine of 0.98.
    assert util.cosine(f32(outs[0][0], "bf16"), f32(outs[2][0], "bf16")) >= 0.97
    assert np.any(outs[0][0] != outs[2][0])
