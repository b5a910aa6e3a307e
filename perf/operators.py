"""Block-scaled e4m3 and the routing of many experts, as cases that can be timed and compared.

A case is a dict of plain values.  Its ``"op"`` is one of

* ``quantize``  a matrix narrowed to e4m3 with one scale per 1 x 128 group of a row, or per 128 x 128 tile
* ``gemm``      a matrix product of such operands, with the epilogues of a linear
* ``route``     the choice of each token's experts, their weights, and the slot tables of the experts' products
* ``experts``   the products of slot-sorted rows with the weights of their experts

``run`` computes a case in plain torch operations, or, where ``own`` is set, by the calls that a user of the framework makes.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

TORCH = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "f32": torch.float32}
BYTES = {"bf16": 2, "e4m3": 1, "f32": 4}
BLOCK = 128  # values of the contraction under one scale; columns of a weight under one scale
TILE = 128  # slots of an expert's run are whole tiles of rows


def _blocks(n):
    return -(-n // BLOCK)


def _tiles(M, E, k):
    """Row tiles that any routing of ``M`` tokens to ``k`` of ``E`` experts each fits."""
    used = min(E, M * k)
    return used + (M * k - used) // TILE


# --------------------------------------------------------------------------------------------------------------- the cases


def _quantize(name, rows, cols, src="bf16", tile=1, pow2=False):
    c = dict(op="quantize", rows=rows, cols=cols, src=src, tile=tile, pow2=pow2)
    return dict(c, name=name) if name else c


def _gemm(name, M, N, K, out="bf16", epilogue="none", groups=1, pow2=False):
    c = dict(op="gemm", M=M, N=N, K=K, out=out, epilogue=epilogue, groups=groups, pow2=pow2)
    return dict(c, name=name) if name else c


def _route(name, M, E, k, scoring, *, groups=1, kept=1, top=1, bias=False, renorm=True, dtype="f32", factor=1.0):
    c = dict(op="route", M=M, E=E, k=k, scoring=scoring, groups=groups, kept=kept, top=top, bias=bias, renorm=renorm, dtype=dtype, factor=factor)
    return dict(c, name=name) if name else c


def _experts(name, M, E, k, N, K, out="bf16", silu=False):
    c = dict(op="experts", M=M, E=E, k=k, N=N, K=K, out=out, silu=silu)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one row of activations before a linear of a model of width 2048: the smallest call
        _quantize("quantize-row", 1, 2048),
        # the hidden activations of a 720p frame (512 tokens) before the second linear of the MLP, where no kernel before it narrows
        _quantize("quantize-720p-hidden", 512, 8192),
        # a large weight as it is loaded: tiles of 128 x 128, scales rounded up to powers of two
        _quantize("quantize-weight-8192", 8192, 8192, tile=128, pow2=True),
        # one token through the first linear of the MLP: 17 MB of weights for one row
        _gemm("gemm-row", 1, 8192, 2048),
        # the first linear of the MLP at 720p, whose output is the next product's operand
        _gemm("gemm-720p-fc1", 512, 8192, 2048, "e4m3", "silu"),
        # the second one, a long contraction with the gate and the residual
        _gemm("gemm-720p-fc2", 512, 2048, 8192, "bf16", "gate"),
        # a product whose sizes fit no tile and no block
        _gemm("gemm-ragged", 777, 1096, 1296, "f32", "bias_silu"),
        # the square product by which rates are quoted
        _gemm("gemm-8192", 8192, 8192, 8192),
        # one token choosing 8 of 256 experts: 8 groups of experts, 4 of them kept, sigmoid scores with a bias for balance
        _route("route-token", 1, 256, 8, "sigmoid", groups=8, kept=4, top=2, bias=True, factor=2.5),
        # the same for many tokens at once
        _route("route-8192", 8192, 256, 8, "sigmoid", groups=8, kept=4, top=2, bias=True, factor=2.5),
        # one 720p frame through the in-projections of 8 experts, 2 per token
        _experts("experts-720p-in", 512, 8, 2, 4096, 2048, "e4m3", True),
        # few tokens over many experts, the out-projections: every run is a small part of a tile
        _experts("experts-many-out", 100, 64, 6, 2048, 1408, "f32"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of ``step`` in ``[lo, hi]``, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step * step, max(-(-lo // step) * step, int(v / step + 0.5) * step))


def draw(rng):
    op = rng.choice(["quantize", "gemm", "gemm", "gemm", "route", "route", "experts", "experts"])
    if op == "quantize":
        return _quantize(None, _log(rng, 1, 8192), _log(rng, 64, 8192, 16), rng.choice(["bf16", "bf16", "f32"]), rng.choice([1, 1, 128]), rng.random() < 0.4)
    if op == "gemm":
        M, epilogue = _log(rng, 1, 8192), rng.choice(["none", "silu", "bias_silu", "gate"])
        groups = 2 if epilogue == "gate" and M % 2 == 0 and rng.random() < 0.3 else 1
        return _gemm(None, M, _log(rng, 64, 8192, 8), _log(rng, 64, 8192, 16), rng.choice(["bf16", "bf16", "f32", "e4m3"]), epilogue, groups, rng.random() < 0.3)
    if op == "route":
        M, E, scoring = _log(rng, 1, 8192), rng.choice([8, 16, 64, 96, 128, 256]), rng.choice(["softmax", "sigmoid"])
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if E // g >= 2])
        kept = rng.randint(1, groups)
        k = rng.randint(1, min(8, kept * (E // groups)))
        return _route(None, M, E, k, scoring, groups=groups, kept=kept, top=rng.choice([1, 2]), bias=rng.random() < 0.5, renorm=rng.random() < 0.7,
                      dtype=rng.choice(["bf16", "f32"]), factor=rng.choice([1.0, 2.5]))  # fmt: skip
    E = rng.choice([8, 8, 16, 32, 64])
    return _experts(None, _log(rng, 1, 512), E, rng.randint(1, min(6, E)), _log(rng, 256, 2048, 128), _log(rng, 256, 2048, 64), rng.choice(["bf16", "e4m3", "f32"]),
                    rng.random() < 0.5)  # fmt: skip


# ------------------------------------------------------------------------------------------------------------------ inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _activations(g, rows, cols):
    """Rows of different size, and some channels much larger than the others."""
    x = torch.randn((rows, cols), device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn((rows, 1), device="cuda", generator=g))
    return x * torch.exp(0.8 * torch.randn((1, cols), device="cuda", generator=g))


def _weight(g, rows, cols):
    return torch.randn((rows, cols), device="cuda", generator=g) * torch.exp(0.3 * torch.randn((rows, 1), device="cuda", generator=g)) * cols**-0.5


def _operands(g, M, N, K, pow2=False, experts=1):
    A, a_scale = _narrow(_activations(g, M, K), 1, pow2)
    B, b_scale = _narrow(_weight(g, experts * N, K), BLOCK, pow2)
    return dict(A=A, a_scale=a_scale, B=B, b_scale=b_scale)


def _outputs(rows, N, out):
    """Output buffers; slots that hold no token are left as they are."""
    d = dict(out=torch.zeros((rows, N), device="cuda", dtype=TORCH[out]))
    if out == "e4m3":
        d["scale_out"] = torch.zeros((_blocks(N), rows), device="cuda")
    return d


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["op"] == "quantize":
        x = _activations(g, c["rows"], c["cols"]) if c["tile"] == 1 else _weight(g, c["rows"], c["cols"])
        s = dict(x=x.to(TORCH[c["src"]]), out=torch.zeros_like(x, dtype=TORCH["e4m3"]))
        kb = _blocks(c["cols"])
        s["scale_out"] = torch.zeros((kb, c["rows"]) if c["tile"] == 1 else (_blocks(c["rows"]), kb), device="cuda")
    elif c["op"] == "gemm":
        M, N = c["M"], c["N"]
        s = {**_operands(g, M, N, c["K"], c["pow2"]), **_outputs(M, N, c["out"])}
        if "bias" in c["epilogue"]:
            s["bias"] = torch.randn((N,), device="cuda", generator=g).to(torch.bfloat16)
        if c["epilogue"] == "gate":
            s["gate"] = (0.2 * torch.randn((c["groups"], N), device="cuda", generator=g)).to(torch.bfloat16)
            s["residual"] = torch.randn((M, N), device="cuda", generator=g).to(torch.bfloat16)
    elif c["op"] == "route":
        M, E, k = c["M"], c["E"], c["k"]
        liked = torch.randn((1, E), device="cuda", generator=g)  # some experts are liked by all tokens, and the bias works against it
        s = dict(logits=(1.5 * torch.randn((M, E), device="cuda", generator=g) + 0.7 * liked).to(TORCH[c["dtype"]]))
        if c["bias"]:
            s["bias"] = (-0.1 * liked + 0.02 * torch.randn((1, E), device="cuda", generator=g)).reshape(E)
        tiles = _tiles(M, E, k)
        i32 = dict(device="cuda", dtype=torch.int32)
        s.update(experts=torch.zeros((M, k), **i32), weights=torch.zeros((M, k), device="cuda"), slot_token=torch.zeros(tiles * TILE, **i32),
                 slot_weight=torch.zeros(tiles * TILE, device="cuda"), tile_expert=torch.zeros(tiles, **i32), tile_rows=torch.zeros(tiles, **i32),
                 token_slot=torch.zeros((M, k), **i32))  # fmt: skip
    else:
        M, E, k = c["M"], c["E"], c["k"]
        logits = torch.randn((M, E), device="cuda", generator=g) + 0.5 * torch.randn((1, E), device="cuda", generator=g)
        experts = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :k]
        tables = _slots(experts, torch.ones_like(experts, dtype=torch.float32), E)
        n = tables["slot_token"].numel()
        s = {**_operands(g, n, c["N"], c["K"], experts=E), **_outputs(n, c["N"], c["out"])}
        s.update(tile_expert=tables["tile_expert"], tile_rows=tables["tile_rows"])
    s["c"] = dict(c)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------------------------------------------------- plain forms


def _padded(x, rows, cols):
    return torch.nn.functional.pad(x, (0, cols - x.shape[-1], 0, rows - x.shape[-2]))


def _narrow(x, tile, pow2):
    """e4m3 values and scales.  The rounding points are the operator's: the scale, its reciprocal and the product in f32."""
    x = x.float()
    rows, cols = x.shape
    kb, rb = _blocks(cols), -(-rows // tile)
    p = _padded(x, rb * tile, kb * BLOCK).view(rb, tile, kb, BLOCK)
    top = p.abs().amax(dim=(1, 3))
    if pow2:
        m, e = torch.frexp(top)  # the smallest 2^j with top <= 448 * 2^j = 0.875 * 2^(j + 9)
        scale = torch.ldexp(torch.ones_like(top), (e - 9 + (m > 0.875)).clamp(min=-126))
    else:
        scale = (top / torch.full_like(top, 448.0)).clamp(min=2.0**-126)  # (a division by a number may be a product with its reciprocal)
    scale = torch.where(top == 0, torch.ones_like(scale), scale)
    q = (p * (1.0 / scale)[:, None, :, None]).reshape(rb * tile, kb * BLOCK)[:rows, :cols].to(TORCH["e4m3"]).contiguous()
    return q, (scale.t() if tile == 1 else scale).contiguous()


def _widen_rows(q, scale):
    """[M, K] e4m3 with scales [blocks, M]."""
    return q.float() * scale.t().repeat_interleave(BLOCK, 1)[:, : q.shape[1]]


def _widen_tiles(q, scale):
    """[N, K] e4m3 with scales [blocks of N, blocks of K]."""
    return q.float() * scale.repeat_interleave(BLOCK, 0)[: q.shape[0]].repeat_interleave(BLOCK, 1)[:, : q.shape[1]]


def _epilogue(y, s, c):
    if "bias" in s:
        y = y + s["bias"].float()
    if c.get("silu") or "silu" in c.get("epilogue", ""):
        y = y / (1.0 + torch.exp(-y))
    if "gate" in s:
        y = s["residual"].float() + s["gate"].float().repeat_interleave(c["M"] // c["groups"], 0) * y
    return y


def _slots(experts, weights, E):
    """Slot tables: the choices sorted by expert (by token inside one), every expert's run starting at a whole tile."""
    M, k = experts.shape
    flat = experts.reshape(-1).long()
    tiles = _tiles(M, E, k)
    counts = torch.zeros(E, dtype=torch.long, device=flat.device).scatter_add_(0, flat, torch.ones_like(flat))
    per = (counts + TILE - 1) // TILE
    first = torch.cumsum(per, 0) - per  # first tile of each expert
    order = torch.sort(flat, stable=True)[1]
    before = torch.cumsum(counts, 0) - counts
    e = flat[order]
    slot = first[e] * TILE + torch.arange(M * k, device=flat.device) - before[e]
    i32 = dict(device=flat.device, dtype=torch.int32)
    slot_token = torch.full((tiles * TILE,), -1, **i32).scatter_(0, slot, (order // k).to(torch.int32))
    slot_weight = torch.zeros(tiles * TILE, device=flat.device).scatter_(0, slot, weights.reshape(-1)[order])
    token_slot = torch.zeros(M * k, **i32).scatter_(0, order, slot.to(torch.int32)).view(M, k)
    t = torch.arange(tiles, device=flat.device)
    last = torch.cumsum(per, 0)
    of = (t[:, None] >= last[None, :]).sum(1)  # expert of a tile; E past the last used tile
    live = of < E
    of0 = of.clamp(max=E - 1)
    rows = (counts[of0] - (t - first[of0]) * TILE).clamp(max=TILE)
    return dict(slot_token=slot_token, slot_weight=slot_weight, tile_expert=torch.where(live, of, -1).to(torch.int32),
                tile_rows=torch.where(live, rows, 0).to(torch.int32), token_slot=token_slot)  # fmt: skip


def _plain_route(s, c):
    M, E, k, G = c["M"], c["E"], c["k"], c["groups"]
    x = s["logits"].double()  # scores next to the border of a choice
    if c["scoring"] == "softmax":
        score = torch.exp(x - x.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    choice = score + s["bias"].double() if "bias" in s else score
    if G > 1:
        grouped = choice.view(M, G, E // G)
        best = torch.sort(grouped, dim=2, descending=True)[0][:, :, : c["top"]].sum(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True)[1][:, : c["kept"]]
        keep = torch.zeros((M, G), dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        choice = torch.where(keep[:, :, None], grouped, -math.inf).reshape(M, E)
    experts = torch.sort(choice, dim=1, descending=True, stable=True)[1][:, :k]
    w = score.gather(1, experts)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    w = (w * c["factor"]).float()
    t = _slots(experts, w, E)
    return [experts.to(torch.int32), w, t["slot_token"], t["slot_weight"], t["tile_expert"], t["tile_rows"], t["token_slot"]]


def _plain_experts(s, c):
    N, K, T = c["N"], c["K"], s["tile_expert"].numel()
    a = _widen_rows(s["A"], s["a_scale"]).view(T, TILE, K)
    e = s["tile_expert"].long().clamp(min=0)
    kb = _blocks(K)
    b = s["B"].view(c["E"], N, K)[e].float()
    b = b * s["b_scale"].view(c["E"], _blocks(N), kb)[e].repeat_interleave(BLOCK, 1)[:, :N].repeat_interleave(BLOCK, 2)[:, :, :K]
    y = _epilogue(torch.bmm(a, b.transpose(1, 2)), s, c)
    live = (torch.arange(TILE, device=y.device) < s["tile_rows"][:, None]).view(T, TILE, 1)
    return torch.where(live, y, 0.0).view(T * TILE, N), live.view(-1)


def _plain(s, c):
    if c["op"] == "quantize":
        return list(_narrow(s["x"], c["tile"], c["pow2"]))
    if c["op"] == "route":
        return _plain_route(s, c)
    if c["op"] == "gemm":
        y = _epilogue(_widen_rows(s["A"], s["a_scale"]) @ _widen_tiles(s["B"], s["b_scale"]).t(), s, c)
        live = None
    else:
        y, live = _plain_experts(s, c)
    if c["out"] != "e4m3":
        return [y.to(TORCH[c["out"]])]
    q, scale = _narrow(y, 1, False)
    return [q, scale if live is None else torch.where(live, scale, 0.0)]


# ------------------------------------------------------------------------------------------------- the framework's own calls


def _handles(s):
    """The framework's tensors over the buffers of ``prepare``: a user's program has its data in this form to begin with."""
    import quark_b200 as qb

    names = {torch.bfloat16: "bf16", torch.float8_e4m3fn: "e4m3", torch.float32: "f32", torch.int32: "s32"}
    return {k: qb.QuarkTensor.borrow(t.data_ptr(), tuple(t.shape), names[t.dtype], keepalive=t) for k, t in s.items() if isinstance(t, torch.Tensor)}


def _own(s, c):
    from quark_b200 import qf

    h = s.get("handles")
    if h is None:
        h = s["handles"] = _handles(s)
    if c["op"] == "quantize":
        qf.quantize_e4m3_blocks(h["x"], tile_rows=c["tile"], pow2=c["pow2"], out=h["out"], scale_out=h["scale_out"])
        return [s["out"], s["scale_out"]]
    if c["op"] == "route":
        tables = ("experts", "weights", "slot_token", "slot_weight", "tile_expert", "tile_rows", "token_slot")
        qf.moe_route_scored(h["logits"], h.get("bias"), top_k=c["k"], scoring=c["scoring"], n_groups=c["groups"], topk_groups=c["kept"], group_top=c["top"],
                            renormalize=c["renorm"], factor=c["factor"], out=[h[t] for t in tables])  # fmt: skip
        return [s[t] for t in tables]
    if c["op"] == "gemm":
        qf.gemm_blocks(h["A"], h["B"], h["a_scale"], h["b_scale"], activation="silu" if "silu" in c["epilogue"] else None, bias=h.get("bias"), gate=h.get("gate"),
                       residual=h.get("residual"), gate_groups=c["groups"], out=h["out"], scale_out=h.get("scale_out"), b_constant=True)  # fmt: skip
    else:
        qf.gemm_grouped_blocks(h["A"], h["B"], h["a_scale"], h["b_scale"], h["tile_expert"], h["tile_rows"], n_experts=c["E"], activation="silu" if c["silu"] else None,
                               out=h["out"], scale_out=h.get("scale_out"), b_constant=True)  # fmt: skip
    return [s["out"], s["scale_out"]] if c["out"] == "e4m3" else [s["out"]]


def run(state):
    return _own(state, state["c"]) if own else _plain(state, state["c"])


# ------------------------------------------------------------------------------------------------ the definition in 64 bits


def _np(t):
    return t.float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _to_e4m3(x):
    """The nearest value of 3 mantissa bits and exponents -6 to 8 (subnormals of 2^-9 below), ties to even, as f64."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-6))) - 3)
    return torch.clamp(torch.round(x / step) * step, -448.0, 448.0)


def _exact_narrow(y, tile, pow2, in_f32):
    """``in_f32``: the scale, its reciprocal and the product are rounded to f32, as the operator's definition has it for values given
    in f32 or bf16; for values that are themselves results, everything stays in 64 bits."""
    rows, cols = y.shape
    q, scales = torch.empty_like(y), torch.empty((-(-rows // tile), _blocks(cols)), dtype=torch.float64, device=y.device)
    r = (lambda t: t.float().double()) if in_f32 else (lambda t: t)
    for b in range(_blocks(cols)):
        part = y[:, b * BLOCK : (b + 1) * BLOCK]
        top = part.abs().amax(1)
        if tile > 1:
            top = torch.stack([t.max() for t in top.split(tile)])
        s = r(top / 448.0).clamp(min=2.0**-126)
        if pow2:
            s = torch.exp2(torch.ceil(torch.log2(s)))
            s = torch.where(s / 2 * 448.0 >= top, s / 2, s)  # (a logarithm a hair above a whole number, or a rounded quotient)
            s = torch.where(s * 448.0 < top, s * 2, s).clamp(min=2.0**-126)
        s = torch.where(top == 0, 1.0, s)
        scales[:, b] = s
        per_row = s.repeat_interleave(tile)[:rows, None]
        q[:, b * BLOCK : (b + 1) * BLOCK] = _to_e4m3(r(part * r(1.0 / per_row)))
    return q, (scales.t() if tile == 1 else scales).contiguous()


def _exact_product(a, a_scale, b, b_scale):
    """Block by block of the contraction, in f64."""
    N = b.shape[0]
    y = torch.zeros((a.shape[0], N), dtype=torch.float64, device=a.device)
    for i in range(_blocks(a.shape[1])):
        at = slice(i * BLOCK, (i + 1) * BLOCK)
        y += (a[:, at].double() @ b[:, at].double().t()) * a_scale[i].double()[:, None] * b_scale[:, i].double().repeat_interleave(BLOCK)[:N]
    return y


def _exact_epilogue(y, s, c):
    if "bias" in s:
        y = y + s["bias"].double()
    if c.get("silu") or "silu" in c.get("epilogue", ""):
        y = y * torch.sigmoid(y)
    if "gate" in s:
        per = c["M"] // c["groups"]
        y = torch.cat([s["residual"][g * per : (g + 1) * per].double() + s["gate"][g].double() * y[g * per : (g + 1) * per] for g in range(c["groups"])])
    return y


def _exact_route(s, c):
    x = _np(s["logits"]).astype(np.float64)
    M, E, k, G = c["M"], c["E"], c["k"], c["groups"]
    if c["scoring"] == "softmax":
        score = np.exp(x - x.max(1, keepdims=True))
        score /= score.sum(1, keepdims=True)
    else:
        score = 0.5 + 0.5 * np.tanh(0.5 * x)
        score = np.where(x < -1, np.exp(x) / (1 + np.exp(x)), score)
    choice = score + (_np(s["bias"]).astype(np.float64) if "bias" in s else 0.0)
    if G > 1:
        size = E // G
        per = np.stack([np.sort(choice[:, g * size : (g + 1) * size], 1)[:, ::-1][:, : c["top"]].sum(1) for g in range(G)], 1)
        kept = np.argsort(-per, 1, kind="stable")[:, : c["kept"]]
        for g in range(G):
            choice[(kept != g).all(1), g * size : (g + 1) * size] = -np.inf
    experts = np.argsort(-choice, 1, kind="stable")[:, :k]
    w = np.take_along_axis(score, experts, 1)
    if c["renorm"]:
        w = w / w.sum(1, keepdims=True)
    w = w * c["factor"]
    tiles = _tiles(M, E, k)
    slot_token, slot_weight, token_slot = np.full(tiles * TILE, -1), np.zeros(tiles * TILE), np.zeros((M, k), np.int64)
    tile_expert, tile_rows, at = np.full(tiles, -1), np.zeros(tiles, np.int64), 0
    for e in range(E):
        m, j = np.nonzero(experts == e)
        here = at * TILE + np.arange(m.size)
        slot_token[here], slot_weight[here], token_slot[m, j] = m, w[m, j], here
        n = -(-m.size // TILE)
        tile_expert[at : at + n] = e
        tile_rows[at : at + n] = np.minimum(m.size - TILE * np.arange(n), TILE)
        at += n
    return [experts.astype(np.int32), w, slot_token.astype(np.int32), slot_weight, tile_expert.astype(np.int32), tile_rows.astype(np.int32), token_slot.astype(np.int32)]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "quantize":
        return list(_exact_narrow(s["x"].double(), c["tile"], c["pow2"], True))
    if c["op"] == "route":
        return _exact_route(s, c)
    if c["op"] == "gemm":
        y = _exact_epilogue(_exact_product(s["A"], s["a_scale"], s["B"], s["b_scale"]), s, c)
        rows = torch.ones(y.shape[0], dtype=torch.bool, device=y.device)
    else:
        N, nb = c["N"], _blocks(c["N"])
        y = torch.zeros((s["A"].shape[0], N), dtype=torch.float64, device="cuda")
        rows = torch.zeros(y.shape[0], dtype=torch.bool, device="cuda")
        for t, (e, n) in enumerate(zip(s["tile_expert"].tolist(), s["tile_rows"].tolist())):
            if e >= 0:
                at = slice(t * TILE, t * TILE + n)
                y[at] = _exact_product(s["A"][at], s["a_scale"][:, at], s["B"][e * N : (e + 1) * N], s["b_scale"][e * nb : (e + 1) * nb])
                rows[at] = True
        y = torch.where(rows[:, None], _exact_epilogue(y, s, c), 0.0)
    if c["out"] != "e4m3":
        return [y]
    q, scale = _exact_narrow(y, 1, False, False)
    return [q, torch.where(rows, scale, 0.0)]


# ------------------------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    c = case
    if c["op"] == "quantize":
        n = c["rows"] * c["cols"]
        return dict(bytes=n * (BYTES[c["src"]] + 1) + 4 * _blocks(c["cols"]) * (c["rows"] if c["tile"] == 1 else _blocks(c["rows"])), flops=3 * n)
    if c["op"] == "route":
        n = c["M"] * c["k"]
        slots = _tiles(c["M"], c["E"], c["k"]) * TILE
        return dict(bytes=c["M"] * c["E"] * BYTES[c["dtype"]] + (4 * c["E"] if c["bias"] else 0) + 12 * n + 8 * slots + 8 * (slots // TILE), flops=8 * c["M"] * c["E"])
    N, K, kb = c["N"], c["K"], _blocks(c["K"])
    rows = c["M"] if c["op"] == "gemm" else c["M"] * c["k"]
    used = 1 if c["op"] == "gemm" else min(c["E"], rows)
    total = rows * (K + 4 * kb) + used * (N * K + 4 * kb * _blocks(N)) + rows * N * BYTES[c["out"]]
    if c["out"] == "e4m3":
        total += 4 * rows * _blocks(N)
    if c.get("epilogue") == "gate":
        total += 2 * rows * N + 2 * c["groups"] * N
    if "bias" in c.get("epilogue", ""):
        total += 2 * N
    return dict(bytes=total, flops=2 * rows * N * K)
