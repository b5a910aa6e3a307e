"""Host side of the block-scaled products and of the routing by scores: what is refused, and sizes, without a GPU."""

import ctypes as C

import pytest

from quark_b200 import _lib
from quark_b200 import functional as qf
from quark_b200.runtime.tensor import QuarkTensor


def t(*shape, dtype="bf16", ptr=1 << 20):
    """A tensor of made-up memory: every call below is refused before anything could read it."""
    return QuarkTensor.borrow(ptr, shape, dtype)


ONE = C.c_void_p(1 << 20)


def last():
    return _lib.load().qb_last_error_string().decode()


def test_entry_points_refuse_on_the_host():
    lib = _lib.load()

    def quant(X=ONE, idx=None, out=ONE, sc=ONE, **kw):
        p = _lib.QuantBlocksParams(**{**dict(batch=1, rows=4, cols=32, src_rows=4, src_dtype=0, tile_rows=1, pow2=0), **kw})
        return lib.qb_quantize_e4m3_blocks(X, idx, out, sc, C.byref(p), None)

    assert quant(X=None) == -1 and quant(sc=None) == -1 and quant(rows=0) == -1 and quant(batch=0) == -1
    assert quant(cols=24) == -3 and "multiple of 16" in last()
    assert quant(X=C.c_void_p(8)) == -3 and quant(out=C.c_void_p(8)) == -3
    assert quant(src_dtype=1) == -1 and quant(tile_rows=64) == -1 and quant(src_rows=5) == -1
    assert quant(tile_rows=128, idx=ONE) == -2 and quant(batch=2) == -2
    assert lib.qb_quantize_e4m3_blocks(ONE, None, ONE, ONE, None, None) == -1

    def gemm(A=ONE, B=ONE, sa=ONE, sb=ONE, c=ONE, sc=None, bias=None, gate=None, res=None, **kw):
        p = _lib.GemmBlocksParams(**{**dict(M=16, N=16, K=32, c_dtype=0, activation=0, gate_groups=1, pow2=0, b_constant=0, tile_n=0, split_k=0), **kw})
        return lib.qb_gemm_blocks(A, B, sa, sb, c, sc, bias, gate, res, C.byref(p), None)

    assert gemm(M=0) == -1 and gemm(K=24) == -3 and gemm(N=12) == -3 and gemm(c_dtype=3) == -1 and gemm(activation=2) == -1
    assert gemm(tile_n=96) == -1 and gemm(split_k=9) == -1 and gemm(A=None) == -1 and gemm(sa=None) == -1 and gemm(sb=None) == -1
    assert gemm(gate=ONE) == -1 and gemm(sc=ONE) == -1 and gemm(c_dtype=1) == -1 and "scales" in last()
    assert gemm(B=C.c_void_p(8)) == -3 and gemm(sb=C.c_void_p(2)) == -3
    # a tile and slices that do not go together are no silent choice of others
    assert gemm(split_k=3) == -1 and gemm(split_k=2, tile_n=128) == -2 and gemm(split_k=2, c_dtype=1, sc=ONE) == -2 and "64 columns" in last()
    assert gemm(tile_n=64, c_dtype=1, sc=ONE) == -2

    def grouped(te=ONE, tr=ONE, experts=2, **kw):
        p = _lib.GemmBlocksParams(**{**dict(M=128, N=16, K=32, c_dtype=0, activation=0, gate_groups=1), **kw})
        return lib.qb_gemm_grouped_blocks(ONE, ONE, ONE, ONE, ONE, None, te, tr, experts, C.byref(p), None)

    assert grouped(te=None) == -1 and grouped(tr=None) == -1 and grouped(experts=0) == -1 and grouped(M=100) == -2 and grouped(M=0) == -2
    assert grouped(experts=1 << 30) == -1 and grouped(split_k=2) == -2

    def route(logits=ONE, bias=None, experts=ONE, weights=ONE, tabs=(ONE,) * 5, ws=None, ws_bytes=0, **kw):
        p = _lib.RouteParams(**{**dict(M=4, E=16, top_k=2, logits_dtype=2, scoring=0, n_groups=1, topk_groups=1, group_top=1, renormalize=1, factor=1.0), **kw})
        return lib.qb_moe_route_scored(logits, bias, experts, weights, *tabs, C.byref(p), ws, ws_bytes, None)

    assert route(logits=None) == -1 and route(experts=None) == -1 and route(tabs=(ONE, None, ONE, ONE, ONE)) == -1
    assert route(M=0) == -1 and route(E=0) == -1 and route(E=513) == -1 and route(top_k=17) == -1 and route(top_k=33, E=64) == -1
    assert route(logits_dtype=1) == -1 and route(scoring=2) == -1 and route(n_groups=3) == -1 and route(n_groups=4, topk_groups=5) == -1
    assert route(n_groups=8, topk_groups=1, top_k=3) == -1 and route(n_groups=16, topk_groups=4, group_top=2) == -1 and route(group_top=0) == -1
    assert route(logits=C.c_void_p(4)) == -3
    assert route(M=65) == -6 and "workspace" in last()  # more than one block of tokens


def test_sizes_of_the_slot_tables():
    lib = _lib.load()
    assert lib.qb_moe_scored_slots(1, 256, 8) == 8 * 128  # a tile per expert that can be chosen
    assert lib.qb_moe_scored_slots(64, 8, 1) == 8 * 128
    assert lib.qb_moe_scored_slots(512, 8, 2) == (8 + (1024 - 8) // 128) * 128
    assert lib.qb_moe_scored_slots(0, 8, 2) == 0 and lib.qb_moe_scored_slots(4, 8, 9) == 0
    for M, E, k in ((1, 8, 2), (300, 16, 3), (1000, 256, 8)):  # no routing needs more: the worst has full tiles and one token over, everywhere
        n = M * k
        worst = max(sum(-(-c // 128) for c in ([1] * (u - 1) + [n - (u - 1)])) for u in range(1, min(E, n) + 1))
        assert lib.qb_moe_scored_slots(M, E, k) // 128 >= worst
    p = _lib.RouteParams(M=4, E=256, top_k=8, logits_dtype=2, scoring=1, n_groups=8, topk_groups=4, group_top=2, renormalize=1, factor=1.0)
    assert lib.qb_moe_route_scored_workspace_bytes(C.byref(p)) == 0
    for M, counts in ((5, 2), (129, 33), (512, 64), (2048, 128), (8192, 128), (8193, 129)):  # behind the area that belongs to the GEMM's tile counters
        p.M = M
        assert lib.qb_moe_route_scored_workspace_bytes(C.byref(p)) == (64 << 10) + counts * 256


@pytest.mark.parametrize("kind,call", [
    (TypeError, lambda: qf.quantize_e4m3_blocks(t(4, 32, dtype="e4m3"))),
    (TypeError, lambda: qf.quantize_e4m3_blocks(t(4, 32), row_index=t(4, dtype="f32"))),
    (ValueError, lambda: qf.quantize_e4m3_blocks(t(4, 40))),
    (ValueError, lambda: qf.quantize_e4m3_blocks(t(32))),
    (ValueError, lambda: qf.quantize_e4m3_blocks(t(0, 32))),
    (ValueError, lambda: qf.quantize_e4m3_blocks(t(4, 32), tile_rows=2)),
    (ValueError, lambda: qf.quantize_e4m3_blocks(t(4, 32), tile_rows=128, row_index=t(4, dtype="s32"))),
    (ValueError, lambda: qf.quantize_e4m3_blocks(t(4, 32), row_index=t(0, dtype="s32"))),
    (TypeError, lambda: qf.gemm_blocks(t(4, 32), t(16, 32, dtype="e4m3"), t(1, 4, dtype="f32"), t(1, 1, dtype="f32"))),
    (TypeError, lambda: qf.gemm_blocks(t(4, 32, dtype="e4m3"), t(16, 32, dtype="e4m3"), t(1, 4), t(1, 1, dtype="f32"))),
    (ValueError, lambda: qf.gemm_blocks(t(4, 32, dtype="e4m3"), t(16, 48, dtype="e4m3"), t(1, 4, dtype="f32"), t(1, 1, dtype="f32"))),
    (ValueError, lambda: qf.gemm_blocks(t(0, 32, dtype="e4m3"), t(16, 32, dtype="e4m3"), t(1, 0, dtype="f32"), t(1, 1, dtype="f32"))),
    (ValueError, lambda: qf.gemm_blocks(t(4, 256, dtype="e4m3"), t(16, 256, dtype="e4m3"), t(1, 4, dtype="f32"), t(1, 2, dtype="f32"))),
    (ValueError, lambda: qf.gemm_blocks(t(4, 32, dtype="e4m3"), t(16, 32, dtype="e4m3"), t(1, 4, dtype="f32"), t(1, 1, dtype="f32"), activation="gelu")),
    (ValueError, lambda: qf.gemm_blocks(t(4, 32, dtype="e4m3"), t(16, 32, dtype="e4m3"), t(1, 4, dtype="f32"), t(1, 1, dtype="f32"), gate=t(1, 16))),
    (TypeError, lambda: qf.gemm_blocks(t(4, 32, dtype="e4m3"), t(16, 32, dtype="e4m3"), t(1, 4, dtype="f32"), t(1, 1, dtype="f32"), bias=t(16, dtype="f32"))),
    (TypeError, lambda: qf.gemm_blocks(t(4, 32, dtype="e4m3"), t(16, 32, dtype="e4m3"), t(1, 4, dtype="f32"), t(1, 1, dtype="f32"), out_dtype="s32")),
    (ValueError, lambda: qf.gemm_grouped_blocks(t(100, 32, dtype="e4m3"), t(16, 32, dtype="e4m3"), t(1, 100, dtype="f32"), t(1, 1, 1, dtype="f32"), t(1, dtype="s32"),
                                                t(1, dtype="s32"), n_experts=1)),
    (ValueError, lambda: qf.gemm_grouped_blocks(t(128, 32, dtype="e4m3"), t(16, 32, dtype="e4m3"), t(1, 128, dtype="f32"), t(1, 1, 1, dtype="f32"), t(2, dtype="s32"),
                                                t(1, dtype="s32"), n_experts=1)),
    (ValueError, lambda: qf.gemm_grouped_blocks(t(128, 32, dtype="e4m3"), t(15, 32, dtype="e4m3"), t(1, 128, dtype="f32"), t(1, 1, 1, dtype="f32"), t(1, dtype="s32"),
                                                t(1, dtype="s32"), n_experts=2)),
    (TypeError, lambda: qf.moe_route_scored(t(4, 16, dtype="e4m3"), top_k=2)),
    (TypeError, lambda: qf.moe_route_scored(t(16), top_k=2)),
    (ValueError, lambda: qf.moe_route_scored(t(0, 16), top_k=2)),
    (ValueError, lambda: qf.moe_route_scored(t(4, 16), top_k=0)),
    (ValueError, lambda: qf.moe_route_scored(t(4, 16), top_k=17)),
    (ValueError, lambda: qf.moe_route_scored(t(4, 1024), top_k=2)),
    (ValueError, lambda: qf.moe_route_scored(t(4, 16), top_k=2, n_groups=5)),
    (ValueError, lambda: qf.moe_route_scored(t(4, 16), top_k=2, n_groups=0)),
    (ValueError, lambda: qf.moe_route_scored(t(4, 16), top_k=5, n_groups=4, topk_groups=1)),
    (ValueError, lambda: qf.moe_route_scored(t(4, 16), top_k=2, n_groups=16, topk_groups=4, group_top=2)),
    (TypeError, lambda: qf.moe_route_scored(t(4, 16), t(16), top_k=2)),
    (ValueError, lambda: qf.moe_route_scored(t(4, 16), t(8, dtype="f32"), top_k=2)),
])  # fmt: skip
def test_python_checks(kind, call):
    with pytest.raises(kind):
        call()


def test_tables_of_more_tokens_than_a_call_can_number(monkeypatch):
    """Every block of the tables reads the counts of all: what 2^24 tokens leave is seconds of work, and past 2^28 the slots were numbered in too few bits."""
    lib = _lib.load()

    def route(tabs, **kw):
        p = _lib.RouteParams(**{**dict(M=(1 << 24) + 1, E=8, top_k=1, logits_dtype=0, scoring=0, n_groups=1, topk_groups=1, group_top=1, renormalize=1, factor=1.0), **kw})
        return lib.qb_moe_route_scored(ONE, None, ONE, ONE, *tabs, C.byref(p), ONE, 1 << 40, None)

    assert route((ONE,) * 5) == -2 and "16777216 tokens" in last()
    assert route((ONE,) * 5, M=1 << 28) == -2
    assert route((None,) * 5, M=1 << 30) == -1  # (without tables only the size of the result counts)
    big = t((1 << 24) + 1, 8)
    with pytest.raises(ValueError, match="16777216 tokens"):
        qf.moe_route_scored(big, top_k=1)
    n = qf.moe_scored_slots((1 << 24) + 1, 8, 1)
    out = [t(*s, dtype=d) for s, d in ((((1 << 24) + 1, 1), "s32"), (((1 << 24) + 1, 1), "f32"), ((n,), "s32"), ((n,), "f32"), ((n // 128,), "s32"), ((n // 128,), "s32"),
                                       (((1 << 24) + 1, 1), "s32"))]  # fmt: skip
    monkeypatch.setattr(qf, "_s", lambda: 1 << 20)
    with pytest.raises(ValueError, match="16777216 tokens"):
        qf.moe_route_scored(big, top_k=1, out=out)


def test_sizes_next_to_the_largest_number_are_refused():
    """The number of blocks and tiles of such a size left 32 bits: a contraction of 2^31 - 16 had a negative number of blocks in the kernel."""
    lib, top = _lib.load(), (1 << 31) - 16

    def gemm(**kw):
        p = _lib.GemmBlocksParams(**{**dict(M=16, N=16, K=32, c_dtype=0, activation=0, gate_groups=1), **kw})
        return lib.qb_gemm_blocks(ONE, ONE, ONE, ONE, ONE, None, None, None, None, C.byref(p), None)

    def quant(**kw):
        p = _lib.QuantBlocksParams(**{**dict(batch=1, rows=1, cols=32, src_rows=1, src_dtype=0, tile_rows=1, pow2=0), **kw})
        return lib.qb_quantize_e4m3_blocks(ONE, None, ONE, ONE, C.byref(p), None)

    for kw in (dict(M=top), dict(N=top), dict(K=top)):
        assert gemm(**kw) == -1 and "too large" in last(), kw
    for kw in (dict(cols=top), dict(rows=top, src_rows=top, tile_rows=128), dict(cols=top, tile_rows=128)):
        assert quant(**kw) == -1 and "too large" in last(), kw
