"""Layers with block-scaled weights on the host: what they launch, wait for and keep, with the device calls replaced by a record of them."""

import pytest

from quark_b200 import nn
from quark_b200.runtime.tensor import QuarkTensor


def t(*shape, dtype="bf16"):
    """A tensor of made-up memory: nothing below reads it."""
    return QuarkTensor.borrow(1 << 20, shape, dtype)


class Record:
    """In the place of ``qf`` and of the stream: every call by its name, results of the right kind."""

    BLOCK = 128

    def __init__(self):
        self.calls = []

    def synchronize(self):
        self.calls.append("synchronize")

    def quantize_e4m3(self, X, out=None):
        self.calls.append("quantize_e4m3")
        return t(*X.shape, dtype="e4m3")

    def quantize_e4m3_rows(self, X):
        self.calls.append("quantize_e4m3_rows")
        return t(*X.shape, dtype="e4m3"), t(X.shape[0], dtype="f32")

    def quantize_e4m3_blocks(self, X, tile_rows=1, out=None, scale_out=None):
        self.calls.append(f"quantize_e4m3_blocks {tile_rows}")
        rows = -(-X.shape[0] // tile_rows)
        return t(*X.shape, dtype="e4m3"), t(*((rows, -(-X.shape[1] // 128)) if tile_rows > 1 else (-(-X.shape[1] // 128), rows)), dtype="f32")

    def gemm(self, A, B, out_dtype=None, activation=None, out=None, **kw):
        assert A.dtype in ("bf16", "e4m3") and (A.dtype == "bf16" or B.dtype == "e4m3")
        self.calls.append(f"gemm {A.dtype} {B.dtype} -> {out_dtype}")
        return t(A.shape[0], B.shape[0], dtype=out_dtype)

    def gemm_blocks(self, A, B, a_scale, b_scale, out_dtype=None, out=None, scale_out=None, **kw):
        assert A.dtype == B.dtype == "e4m3" and a_scale.dtype == b_scale.dtype == "f32"
        self.calls.append(f"gemm_blocks -> {out_dtype}")
        y = t(A.shape[0], B.shape[0], dtype=out_dtype)
        return y if out_dtype != "e4m3" else (y, t(-(-B.shape[0] // 128), A.shape[0], dtype="f32"))

    def silu(self, X, out=None, out_q=None):
        self.calls.append("silu" if out_q is None else "silu e4m3")


@pytest.fixture
def record(monkeypatch):
    r = Record()
    monkeypatch.setattr(QuarkTensor, "zeros", staticmethod(t))
    monkeypatch.setattr(QuarkTensor, "empty", staticmethod(t))
    monkeypatch.setattr(nn, "qf", r)
    monkeypatch.setattr(nn, "_stream", r, raising=False)
    return r


def test_a_narrowed_weight_is_in_place_before_the_first_product(record):
    """Products fetch weights ahead of the kernels before them (``b_constant``): the kernel that writes the weight may not be one of those."""
    lin = nn.Linear(256, 384)
    lin.prepare(fp8=True, fp8_blocks=True)
    assert record.calls == ["quantize_e4m3_blocks 128", "synchronize"]
    lin.prepare(fp8=True, fp8_blocks=True)  # once only
    assert len(record.calls) == 2


FORMS = {"bf16": {}, "e4m3": dict(fp8=True), "rows": dict(fp8=True, fp8_scaled=True), "blocks": dict(fp8=True, fp8_blocks=True)}


@pytest.mark.parametrize("first", list(FORMS))
@pytest.mark.parametrize("second", list(FORMS))
@pytest.mark.parametrize("fuse", [False, True])
def test_the_two_linears_of_an_mlp_are_narrowed_each_as_it_likes(record, first, second, fuse):
    """The hidden activations are handed over in a form that both know: e4m3 with its scales between two block-scaled linears, plain e4m3
    where neither is, else bf16."""
    mlp = nn.MLP(256, 512, 256, fuse_silu=fuse)
    mlp.fc1.prepare(**FORMS[first])
    mlp.fc2.prepare(**FORMS[second])
    del record.calls[:]
    y = mlp(t(5, 256))
    assert y.dtype == "bf16" and y.shape == (5, 256)
    h = "e4m3" if second != "bf16" and (first == "blocks") == (second == "blocks") else "bf16"
    if fuse:
        one = [f"gemm_blocks -> {h}"] if first == "blocks" else [f"gemm bf16 {'bf16' if first == 'bf16' else 'e4m3'} -> {h}"]
    else:
        emit = second in ("e4m3", "rows")
        h = "e4m3" if emit else "bf16"
        one = ["gemm_blocks -> bf16" if first == "blocks" else f"gemm bf16 {'bf16' if first == 'bf16' else 'e4m3'} -> bf16", "silu e4m3" if emit else "silu"]
    narrow = ["quantize_e4m3_blocks 1"]
    handed = fuse and h == "e4m3"
    two = (([] if handed else narrow) + ["gemm_blocks -> bf16"]) if second == "blocks" else [f"gemm {h} {'bf16' if second == 'bf16' else 'e4m3'} -> bf16"]
    assert record.calls == (narrow if first == "blocks" else []) + one + two


def test_a_pair_goes_with_block_scaled_weights_only(record):
    lin = nn.Linear(256, 128)
    pair = (t(4, 256, dtype="e4m3"), t(2, 4, dtype="f32"))
    for form in ("bf16", "e4m3"):
        lin.prepare(**FORMS[form])
        with pytest.raises(TypeError, match="pair"):
            lin(pair)


def test_scales_are_part_of_the_state(record):
    """The e4m3 bytes mean nothing without their scales: both are in ``state_dict``, and a state goes only into layers narrowed the same way."""
    a, b, plain = nn.Linear(256, 200), nn.Linear(256, 200), nn.Linear(256, 200)
    for lin in (a, b):
        lin.prepare(fp8=True, fp8_blocks=True)
    state = a.state_dict()
    assert list(state) == ["weight", "weight_blocks"] and state["weight_blocks"] is a.w_blocks and a.w_blocks.shape == (2, 2)
    b.load_state_dict(state)
    assert b.weight.data is a.weight.data and b.w_blocks is a.w_blocks
    with pytest.raises(KeyError, match="weight_blocks"):
        plain.load_state_dict(state)
    with pytest.raises(KeyError, match="weight_blocks"):
        b.load_state_dict(plain.state_dict())
    moe, other = nn.MoE(4, 128, 256, 8, 2), nn.MoE(4, 128, 256, 8, 2)
    moe.prepare(fp8=True, fp8_blocks=True)
    state = moe.state_dict()
    assert state["expert_in_blocks"].shape == (8 * 2, 1) and state["expert_out_blocks"].shape == (8 * 1, 2)
    with pytest.raises(KeyError, match="expert_in_blocks"):
        other.load_state_dict(state)


@pytest.mark.parametrize("form", ["e4m3", "rows", "blocks"])
def test_a_new_weight_is_narrowed_again(record, form):
    lin = nn.Linear(256, 200)
    lin.prepare(**FORMS[form])
    lin.load_weight(t(200, 256))
    assert lin.weight.data.dtype == "bf16" and lin.w_blocks is None and lin.w_scale is None and list(lin.state_dict()) == ["weight"]
    lin(t(4, 256))
    assert record.calls[-1] == "gemm bf16 bf16 -> bf16"
    del record.calls[:]
    lin.prepare(**FORMS[form])
    assert lin.weight.data.dtype == "e4m3" and (lin.w_blocks is not None) == (form == "blocks") and (lin.w_scale is not None) == (form == "rows")


def test_parameters_loaded_into_a_prepared_model(record, monkeypatch):
    """``load_params`` takes a model back to bf16 weights, and ``prepare`` narrows them again."""
    from quark_b200.models import QuantConfig, Waypoint15, Waypoint15Config, make_params
    from quark_b200.models import waypoint_15 as w

    monkeypatch.setattr(QuarkTensor, "from_numpy", staticmethod(lambda a, dtype=None: t(*a.shape, dtype=dtype or "f32")))
    monkeypatch.setattr(w, "_stream", record)
    for kw in (dict(), dict(moe=True, moe_n_experts=8, moe_top_k=2)):
        cfg = Waypoint15Config(d_model=128, n_layers=2, n_heads=2, n_kv_heads=1, height=8, width=8, channels=4, local_window=2, global_window=4, global_pinned_dilation=2,
                               fourier_dim=32, quant=QuantConfig.all_fp8(), fp8_blocks=True, **kw)  # fmt: skip
        model, params = Waypoint15(cfg), make_params(cfg)

        def forms(blk):
            lins = [blk.qkv_proj, blk.out_proj, *(() if cfg.moe else (blk.mlp.fc1, blk.mlp.fc2))]
            got = {(lin.weight.data.dtype, lin.w_blocks is not None) for lin in lins}
            if cfg.moe:
                got |= {(p.data.dtype, "expert_in_blocks" in blk.mlp.state_dict()) for p in (blk.mlp.expert_in, blk.mlp.expert_out)}
            return got

        for _ in range(2):
            model.load_params(params)
            assert all(forms(blk) == {("bf16", False)} for blk in model.blocks)
            model.prepare()
            assert all(forms(blk) == {("e4m3", True)} for blk in model.blocks)


def test_a_captured_frame_is_not_replayed_with_other_parameters():
    """The graph of a frame reads the memory of the parameters it was captured with: once one of them has been replaced it is not launched again."""
    from quark_b200.models.waypoint_15 import GenerateFrame

    class Model(nn.Module):
        def __init__(self):
            self.weight = nn.Parameter(t(8, 8))

    class Graph:
        launched = 0

        def launch(self):
            self.launched += 1

    class Latent:
        def copy_from(self, other):
            pass

    gen = GenerateFrame.__new__(GenerateFrame)
    gen.model, gen._ctrl_in, gen._in, gen._out = Model(), None, Latent(), "replayed"
    gen.forward = lambda latent, ctrl_input=None: "call by call"
    gen._graph = None
    assert gen("x") == "call by call" and not gen.captured()
    first = Graph()
    gen.hold(first)
    assert gen.captured() and gen("x") == "replayed" and first.launched == 1
    gen.model.load_state_dict({"weight": t(8, 8)})
    assert not gen.captured() and gen("x") == "call by call" and first.launched == 1 and gen._graph is None
    gen.hold(Graph())
    assert gen("x") == "replayed"
