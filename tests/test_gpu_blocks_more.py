"""Block-scaled e4m3 and routing by scores: calls that follow one another closely, products whose CTAs walk several tiles, choices among
equal scores, weights of scores far apart.  Formulas and tolerances are those of ``test_gpu_blocks``."""

import numpy as np
import pytest

from oracle import codec
from tests import util
from tests.test_gpu_blocks import Operands, T, blocks, check, check_routing, epilogue, route, route_scores, values
from tests.util import bf16_randn, f32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qb():
    import quark_b200 as q

    q._lib.require_device(0)
    yield q
    q.runtime.synchronize()
    assert q._lib.device_status() == 0


# --------------------------------------------------------------------------------------------------------------- layers


def test_a_product_right_after_its_weight_was_narrowed(qb):
    """Rows that were narrowed before: nothing but the product follows the kernel that writes the weight.  The bits are those of the same call later."""
    from quark_b200 import nn

    r = util.rng(30)
    K, N = 8192, 8192
    x, s = qb.qf.quantize_e4m3_blocks(T(qb, bf16_randn(r, (3, K)), "bf16"))
    for seed in range(4):
        lin = nn.Linear(K, N)
        wide = T(qb, np.resize(bf16_randn(util.rng([31, seed]), (1_000_003,), 0.05), (N, K)), "bf16")
        lin.weight.data = wide  # (kept: giving its memory back would wait for the kernel that reads it)
        out = [qb.QuarkTensor.zeros(3, N) for _ in range(2)]
        qb.runtime.synchronize()
        lin.prepare(fp8=True, fp8_blocks=True)
        lin((x, s), out=out[0])
        qb.runtime.synchronize()
        lin((x, s), out=out[1])
        np.testing.assert_array_equal(out[0].to_numpy(), out[1].to_numpy())
        assert np.any(out[1].to_numpy() != 0)


@pytest.mark.parametrize("kw", [dict(), dict(moe=True, moe_n_experts=8, moe_top_k=2)])
def test_parameters_loaded_into_a_model_that_was_prepared(qb, kw):
    """A second set of parameters, and then the first again: every frame is that of a session made with them."""
    from quark_b200.models import QuantConfig, Waypoint15Config, make_params
    from tests.test_gpu_model import small_cfg

    quant = QuantConfig(linear="fp8", kv_cache="bf16", attn_compute="bf16", moe="fp8")
    cfg = Waypoint15Config(**{**small_cfg(qb, "bf16").__dict__, "quant": quant, "fp8_blocks": True, **kw})
    params = [make_params(cfg, seed=s, weight_std=0.04) for s in (32, 33)]
    noise = util.rng(34).standard_normal((1, cfg.latent_numel)).astype(np.float32)
    want, got = [], []
    for p in params:
        want.append(qb.Engine(cfg=cfg, quant=quant, params=p, use_graph=False).gen_frame(noise=noise).reshape(-1))
    eng = qb.Engine(cfg=cfg, quant=quant, params=params[0], use_graph=False)
    start = eng.snapshot()
    for p in (params[1], params[0]):
        eng.model.load_params(p)
        eng.model.prepare()
        eng.restore(start)
        got.append(eng.gen_frame(noise=noise).reshape(-1))
    np.testing.assert_array_equal(got[0], want[1])
    np.testing.assert_array_equal(got[1], want[0])
    assert np.any(want[0] != want[1])


@pytest.mark.parametrize("kw", [dict(fp8_blocks=True), dict(fp8_blocks=False), dict(fp8_blocks=True, moe=True, moe_n_experts=8, moe_top_k=2)])
def test_parameters_loaded_into_a_session_that_replays_its_frames(qb, kw):
    """Frames are captured before the other parameters come, and again behind them: a frame is the one of a session that calls one by one."""
    from quark_b200.models import QuantConfig, Waypoint15Config, make_params
    from tests.test_gpu_model import small_cfg

    quant = QuantConfig(linear="fp8", kv_cache="bf16", attn_compute="bf16", moe="fp8")
    cfg = Waypoint15Config(**{**small_cfg(qb, "bf16").__dict__, "quant": quant, **kw})
    params = [make_params(cfg, seed=s, weight_std=0.04) for s in (42, 43)]
    r = util.rng(44)
    noise = [r.standard_normal((1, cfg.latent_numel)).astype(np.float32) for _ in range(5)]
    frames = []
    for graph in (True, False):
        eng = qb.Engine(cfg=cfg, quant=quant, params=params[0], use_graph=graph)
        out = [eng.gen_frame(noise=n) for n in noise[:2]]
        eng.model.load_params(params[1])
        eng.model.prepare()
        out += [eng.gen_frame(noise=n) for n in noise[2:4]]
        assert (eng.gen._graph is not None) == graph
        eng.model.load_state_dict({k: v.to_numpy().copy() for k, v in eng.model.state_dict().items()})  # the same values in other memory
        frames.append(out + [eng.gen_frame(noise=noise[4])])
    for a, b in zip(*frames):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("kw", [
    dict(), dict(fp8_scales=True), dict(ctrl_conditioning=True), dict(value_residual=False), dict(quilt_factor=2),
    dict(moe=True, moe_n_experts=32, moe_top_k=4, moe_scoring="softmax", moe_n_groups=8, moe_topk_groups=3, moe_renormalize=False),
])  # fmt: skip
def test_sessions_with_everything_in_e4m3(qb, kw):
    """Block-scaled linears beside e4m3 caches and attention (the default of ``Engine``): the wirings that a block can have give the same
    bits, replayed or not, and stay close to the session without block scales and to the one in bf16."""
    from quark_b200.models import QuantConfig, Waypoint15Config, make_params
    from tests.test_gpu_model import small_cfg

    quant = QuantConfig.all_fp8()
    cfg = Waypoint15Config(**{**small_cfg(qb, "bf16").__dict__, "quant": quant, "fp8_blocks": True, **kw})
    params = make_params(cfg, seed=45, weight_std=0.04)
    r = util.rng(46)
    lats = [codec.f32_to_bf16(r.standard_normal((1, cfg.latent_numel)).astype(np.float32)) for _ in range(3)]
    noise = r.standard_normal((1, cfg.latent_numel)).astype(np.float32)
    ctrl = qb.CtrlInput(button={1, 5}, mouse=(0.3, -0.2)) if cfg.ctrl_conditioning else None
    outs = []
    wide = dict(quant=QuantConfig.all_bf16(), fp8_blocks=False, fp8_scales=False)
    for graph, other in ((True, {}), (False, {}), (False, dict(fuse_qkv_post=False)), (False, dict(fp8_blocks=False)), (False, wide)):
        c = Waypoint15Config(**{**cfg.__dict__, **other})
        eng = qb.Engine(cfg=c, quant=c.quant, params=params, use_graph=graph)
        for lat in lats:
            eng.append_frame(lat, ctrl) if ctrl else eng.append_frame(lat)
        outs.append([(eng.gen_frame(ctrl, noise=noise) if ctrl else eng.gen_frame(noise=noise)).reshape(-1) for _ in range(2)])
    for o in outs[1:3]:
        for a, b in zip(outs[0], o):
            np.testing.assert_array_equal(a, b)
    # as in test_sessions of the layers' file: linears off by 2 - 3 % (rms) each; caches and probabilities in e4m3 add as much again
    assert util.cosine(f32(outs[0][0], "bf16"), f32(outs[4][0], "bf16")) >= 0.95
    assert np.any(outs[0][0] != outs[3][0])


@pytest.mark.parametrize("first", ["bf16", "e4m3", "blocks"])
@pytest.mark.parametrize("second", ["bf16", "e4m3", "blocks"])
@pytest.mark.parametrize("fuse", [False, True])
def test_an_mlp_of_linears_narrowed_each_as_it_likes(qb, first, second, fuse):
    from quark_b200 import nn

    forms = {"bf16": {}, "e4m3": dict(fp8=True), "blocks": dict(fp8=True, fp8_blocks=True)}
    r = util.rng(40)
    M, D, H = 33, 256, 640
    w1, w2, x = bf16_randn(r, (H, D), 0.06), bf16_randn(r, (D, H), 0.04), bf16_randn(r, (M, D))
    mlp = nn.MLP(D, H, D, fuse_silu=fuse)
    mlp.fc1.load_weight(T(qb, w1, "bf16"))
    mlp.fc2.load_weight(T(qb, w2, "bf16"))
    mlp.fc1.prepare(**forms[first])
    mlp.fc2.prepare(**forms[second])
    got = f32(mlp(T(qb, x, "bf16")).to_numpy(), "bf16")
    f = lambda t: f32(t, "bf16").astype(np.float64)  # noqa: E731
    h = f(x) @ f(w1).T
    want = (h / (1 + np.exp(-h))) @ f(w2).T
    # four operands, each off by at most 2^-4 of itself (without scales 2^-10 absolute as well: of weights of 0.04 another 2^-5), or 2^-8
    step = {"bf16": 2.0**-8, "blocks": 2.0**-4, "e4m3": 2.0**-4 + 2.0**-5}
    assert np.linalg.norm(got - want) <= 2 * (step[first] + step[second] + 2.0**-8) * np.linalg.norm(want)


def test_a_state_with_its_scales_goes_from_layer_to_layer(qb):
    """As tensors and as host arrays: the layer that takes it gives what the other gave."""
    from quark_b200 import nn

    r = util.rng(41)
    x = T(qb, bf16_randn(r, (9, 384)), "bf16")
    lins = [nn.Linear(384, 200) for _ in range(3)]
    for lin in lins:
        lin.load_weight(T(qb, bf16_randn(r, (200, 384), 0.05), "bf16"))
        lin.prepare(fp8=True, fp8_blocks=True)
    want = lins[0](x).to_numpy()
    assert np.any(lins[1](x).to_numpy() != want)
    lins[1].load_state_dict(lins[0].state_dict())
    lins[2].load_state_dict({k: v.to_numpy() for k, v in lins[0].state_dict().items()})
    for lin in lins[1:]:
        np.testing.assert_array_equal(lin(x).to_numpy(), want)


# -------------------------------------------------------------------------------------------------------------- routing


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("low", [-70.0, -90.0, -95.0, -105.0, -120.0])
def test_weights_of_choices_on_both_sides_of_what_32_bits_hold(qb, scoring, low):
    """The bias picks experts of which some score far above the others: the small ones' weights are as close as the large ones', also where their
    scores are subnormal or 0 in 32 bits and the sum is not small."""
    r = util.rng([35, int(-low)])
    x = r.standard_normal((70, 64)).astype(np.float32)
    x[:, ::7] += np.float32(low)
    x[:, 7] += np.float32(0.5 * -low)  # one of the ten is about halfway
    bias = np.zeros(64, np.float32)
    bias[::7] = 2.0 + np.arange(10)
    for k in (2, 4, 10):
        got = qb.qf.moe_route_scored(T(qb, x), T(qb, bias), top_k=k, scoring=scoring, factor=2.5)
        e, w = route(x, bias, k, scoring, factor=2.5)
        check_routing(got, e, w, 64)
    masked = x.copy()
    masked[:, 14] = -np.inf  # chosen by its bias all the same, with weight 0
    got = qb.qf.moe_route_scored(T(qb, masked), T(qb, bias), top_k=10, scoring=scoring)
    e, w = route(masked, bias, 10, scoring)
    assert np.all((e == 14).sum(1) == 1) and np.all(w[e == 14] == 0)
    check_routing(got, e, w, 64)


def choice(values, groups, kept, top, k):
    """The kept groups by the sum of their best ``top`` values, then the best ``k`` inside them; equal ones: the lower index."""
    M, E = values.shape
    per = -np.sort(-values.reshape(M, groups, -1), 2)[:, :, :top].sum(2)
    keep = np.zeros((M, groups), bool)
    np.put_along_axis(keep, np.argsort(-per, 1, kind="stable")[:, :kept], True, 1)
    out = np.zeros((M, k), int)
    for m in range(M):
        inside = np.flatnonzero(np.repeat(keep[m], E // groups))
        out[m] = inside[np.argsort(-values[m, inside], kind="stable")[:k]]
    return out


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,kept,k", [(32, 4, 2, 6), (32, 8, 3, 12), (256, 8, 4, 8), (24, 4, 3, 5), (160, 8, 3, 6), (512, 16, 5, 32)])
@pytest.mark.parametrize("top", [1, 2])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_equal_groups_and_experts_without_a_bias(qb, scoring, E, groups, kept, k, top, dtype):
    """Every expert of every token, equal or masked, is the one the formula names: by the logits where groups go by their best one (-inf comes
    behind the lowest value), by the scores in 64 bits where they go by their best two."""
    r = util.rng([36, E, groups])
    M, low = 150, codec.bf16_to_f32(np.uint16(0xFF7F)) if dtype == "bf16" else np.float32(-3.4028235e38)
    # (no two levels are opposite: the sigmoids of such sum to 1 but for a rounding, and 64 bits would not say which group comes first)
    x = r.integers(-2, 3, (M, E)).astype(np.float32) * np.float32(0.5) + np.float32(0.3125)
    x[3:40] = np.where(r.random((37, E)) < 0.7, -np.inf, x[3:40])
    x[40:70] = np.where(r.random((30, E)) < 0.7, low, x[40:70])
    x[5], x[6], x[7] = -np.inf, 0.0, low
    x[8, :] = np.where(np.arange(E) % 3 == 0, -np.inf, low)
    x[9] = np.where(np.arange(E) < E // groups, 1.0, x[9])
    x[70:80, ::2] = -0.0
    x[70:80, 1::2] = 0.0
    X = T(qb, codec.f32_to_bf16(x), "bf16") if dtype == "bf16" else T(qb, x)
    got = qb.qf.moe_route_scored(X, top_k=k, scoring=scoring, n_groups=groups, topk_groups=kept, group_top=top)
    s = route_scores(x, scoring)
    e = choice(x.astype(np.float64) if top == 1 else s, groups, kept, top, k)
    w = np.take_along_axis(s, e, 1)
    t = w.sum(1, keepdims=True)
    check_routing(got, e, np.where(t == 0, 0, w / np.where(t == 0, 1, t)), E)


# ------------------------------------------------------------------------------------------------- several tiles to a CTA


@pytest.mark.parametrize("tile_n,M,N,K", [
    (64, 1700, 1400, 640), (64, 2000, 1096, 1152), (64, 2100, 1048, 144),
    (128, 2500, 2056, 640), (128, 2700, 1880, 1152), (128, 2500, 2000, 272), (128, 2500, 2000, 1024),
    (256, 2500, 4104, 640), (256, 2600, 3848, 384), (256, 2500, 4000, 128), (256, 2500, 4000, 1168),
])  # fmt: skip
@pytest.mark.parametrize("kind", ["plain", "bias_silu", "gate", "bias_silu_gate_groups"])
def test_several_tiles_of_a_cta(qb, tile_n, M, N, K, kind):
    """More tiles than SMs: a CTA's next tile meets the ring, the accumulators' buffers and the vectors per column as the last one left them.
    Blocks of K that go evenly into the buffers and ones that do not, with every epilogue and type that the width has."""
    tiles = -(-M // 128) * -(-N // tile_n)
    assert tiles > 2 * 148 or tile_n == 64 and tiles > 148
    r = util.rng([37, M, N, K])
    op = Operands(r, M, N, K)
    t = op.tensors(qb)
    y, mags = op.product()
    kw, ref = {}, {}
    if "bias" in kind:
        ref["bias"] = bf16_randn(r, (N,))
        kw["bias"] = T(qb, ref["bias"], "bf16")
    if "silu" in kind:
        ref["act"] = kw["activation"] = "silu"
    if "gate" in kind:
        groups = M // 50 if "groups" in kind else 1  # (50 rows: most tiles have several)
        ref.update(gate=bf16_randn(r, (groups, N)), residual=bf16_randn(r, (M, N)), groups=groups)
        kw.update(gate=T(qb, ref["gate"], "bf16"), residual=T(qb, ref["residual"], "bf16"), gate_groups=groups)
    for out in ("bf16", "f32", "e4m3"):
        if out == "e4m3" and tile_n == 64:
            continue
        want, err = epilogue(y, op.sum_error(mags), **ref, out=out)
        got = qb.qf.gemm_blocks(*t, out_dtype=out, tile_n=tile_n, split_k=1, b_constant=out == "bf16", **kw)
        got, scale = got if out == "e4m3" else (got, None)
        check(values(got), scale.to_numpy() if scale else None, want, err, out, f"{M}x{N}x{K} {tile_n} {kind} {out}")


@pytest.mark.parametrize("tile_n,N,K", [(64, 1048, 640), (64, 520, 1152), (128, 2056, 640), (128, 1048, 384), (256, 4104, 384), (256, 2056, 1152)])
@pytest.mark.parametrize("act", [None, "silu"])
def test_several_tiles_of_a_cta_by_experts(qb, tile_n, N, K, act):
    """The same over runs of experts: full tiles, tiles of few rows (whose copies are small ones), and tiles without tokens among them."""
    r = util.rng([38, N, K])
    E = 5
    rows = [128, 3, 0, 128, 31, 32, 33, 128, -7, 100, 1, 128, 64, 300, 17, 128, 0, 96, 128, 2, 128, 128, 40, 128, 5, 128, 128, 8, 77, 128, 128, 0, 128, 24, 128, 128, 128, 1, 128, 50]
    experts = [int(e) for e in r.integers(0, E, len(rows))]
    experts[4], experts[9], experts[20] = -1, E, 1 << 30  # no such experts
    M = 128 * len(rows)
    op = Operands(r, M, N, K, experts=E)
    A, B, sa, sb = op.tensors(qb)
    tables = T(qb, np.array(experts, np.int32)), T(qb, np.array(rows, np.int32))
    live = [slice(128 * i, 128 * i + (max(min(n, 128), 0) if 0 <= e < E else 0)) for i, (e, n) in enumerate(zip(experts, rows))]
    products = [op.product(at, e) if at.stop > at.start else None for at, e in zip(live, experts)]
    for out in ("bf16", "f32", "e4m3"):
        if out == "e4m3" and tile_n == 64:
            continue
        carrier = {"bf16": np.uint16, "f32": np.float32, "e4m3": np.uint8}[out]
        o = T(qb, np.full((M, N), 85, carrier), out)
        so = T(qb, np.full((blocks(N), M), -5.0, np.float32)) if out == "e4m3" else None
        before = values(o)[0, 0]
        qb.qf.gemm_grouped_blocks(A, B, sa, sb, *tables, n_experts=E, activation=act, out=o, scale_out=so, tile_n=tile_n)
        got, scales = values(o), so.to_numpy() if so else None
        for i, at in enumerate(live):
            if products[i] is not None:
                y, mags = products[i]
                y, err = epilogue(y, op.sum_error(mags), act=act, out=out)
                check(got[at], scales[:, at] if so else None, y, err, out, f"tile {i} {tile_n} {out}")
            assert np.all(got[at.stop : 128 * (i + 1)] == before)  # left as they were
            if so:
                assert np.all(scales[:, at.stop : 128 * (i + 1)] == -5.0)


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("E,groups,kept,top", [(64, 1, 1, 1), (64, 8, 4, 2), (64, 8, 4, 1), (160, 8, 3, 2)])
def test_a_softmax_over_nan_or_infinity(qb, biased, renorm, E, groups, kept, top):
    """All of such a row's scores are NaN by the formula, so all of its weights are, whichever experts it goes to; other rows do not see it."""
    r = util.rng([39, E])
    x = r.standard_normal((70, E)).astype(np.float32)
    clean = x.copy()
    x[10, 5], x[20], x[30, ::2], x[40, E - 1], x[50, 3], x[51, 7] = np.nan, np.nan, np.nan, np.inf, np.inf, -np.inf
    x[50, 4] = np.nan
    clean[51, 7] = -np.inf
    bias = (0.1 * r.standard_normal(E)).astype(np.float32) if biased else None
    got = qb.qf.moe_route_scored(T(qb, x), T(qb, bias) if biased else None, top_k=4, n_groups=groups, topk_groups=kept, group_top=top, renormalize=renorm)
    e, w = got.experts.to_numpy(), got.weights.to_numpy()
    assert e.min() >= 0 and e.max() < E and all(len(set(row)) == 4 for row in e)
    bad = [10, 20, 30, 40, 50]
    rest = np.setdiff1d(np.arange(70), bad)
    assert np.all(np.isnan(w[bad]))
    we, ww = route(clean, bias, 4, "softmax", groups, kept, top, renorm)
    np.testing.assert_array_equal(e[rest], we[rest])
    np.testing.assert_allclose(w[rest], ww[rest], rtol=40 * 2.0**-24)
