"""Block-scaled e4m3 and routing by scores: calls that follow one another closely, products whose CTAs walk several tiles, choices among
equal scores, weights of scores far apart.  Formulas and tolerances are those of ``test_gpu_blocks``."""

import numpy as np
import pytest

from tests import util
from tests.test_gpu_blocks import T, check_routing, route
from tests.util import bf16_randn

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
