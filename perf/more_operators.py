"""The feed-forward half of a layer as cases that can be timed and compared: norms, codes for 8-bit products, experts.

Four kinds: the residual's addition and the norm behind it, with an output in 8 bits and scales for each token ("norm"); the
same ahead of a projection that multiplies those codes by 8-bit weights ("product"); routing of tokens to experts ("route");
and the experts' gated feed-forward networks, weighted and added to the residual ("experts").

Weights are those of the FullyConnected layout: blocks of 4 inputs x 4 outputs, [inputs / 4][outputs / 4][4 inputs][4 outputs], a
byte holds q + 128 or two nibbles q + 8, the even output in the low one; scales in fp16, [groups of inputs][outputs].
An expert's first matrix has the rows gate 0, up 0, gate 1, up 1, ...

Widths of 2048, 4096, 8192 and 14336, blocks of 32 and prompts of 2048 tokens are this repository's own sizes; numbers of
experts and the others are generic.
"""
import functools
import importlib
import math
import random

import torch

own = False

EPS = 1e-6


def _mld():
    return importlib.import_module("ml-drift_b200")


# ------------------------------------------------------------------------------------------------------------ cases
def _norm(tokens, width, type_, residual, offset, out, codes):
    """codes: "none", "symmetric" or "asymmetric"."""
    return {"kind": "norm", "tokens": tokens, "width": width, "type": type_, "residual": residual, "offset": offset, "out": out,
            "codes": codes}


def _product(tokens, width, outputs, codes):
    return {"kind": "product", "tokens": tokens, "width": width, "outputs": outputs, "type": "f16", "residual": True, "offset": 0.0,
            "out": False, "codes": codes}


def _route(tokens, experts, chosen, score, bias, groups, top_groups, best, renormalise, factor, type_):
    return {"kind": "route", "tokens": tokens, "experts": experts, "chosen": chosen, "score": score, "bias": bias, "groups": groups,
            "top_groups": top_groups, "best": best, "renormalise": renormalise, "factor": factor, "type": type_}


def _experts(tokens, padding, experts, chosen, width, inner, bits, block, act, residual):
    """The last `padding` tokens are rows of a batch that nobody has filled: they go to no expert."""
    return {"kind": "experts", "tokens": tokens, "padding": padding, "experts": experts, "chosen": chosen, "width": width,
            "inner": inner, "bits": bits, "block": block, "act": act, "residual": residual}


def listed():
    return [
        # One generated token between attention and the feed-forward network: the smallest call, nothing but latency.
        {"name": "norm_token", **_norm(1, 4096, "f16", True, 0.0, True, "none")},
        # fp32 tensors of an odd width with weights about zero; codes with zero points.
        {"name": "norm_f32_1155", **_norm(333, 1155, "f32", True, 1.0, True, "asymmetric")},
        # A long prompt: the sum, the norm in fp16 for one reader and in codes for another.
        {"name": "norm_prompt8191", **_norm(8191, 8192, "f16", True, 0.0, True, "symmetric")},
        # A ragged chunk of a prompt: norm and one projection on its codes.
        {"name": "product_77", **_product(77, 2048, 4096, "symmetric")},
        # A prompt through a wide projection, codes with zero points.
        {"name": "product_2048", **_product(2048, 4096, 14336, "asymmetric")},
        # One generated token finds its experts.
        {"name": "route_token", **_route(1, 128, 8, "softmax", False, 1, 1, 1, True, 1.0, "f16")},
        # A long prompt, a bias for balance, four of eight groups first.
        {"name": "route_prompt8192", **_route(8192, 256, 8, "sigmoid", True, 8, 4, 2, True, 2.5, "f32")},
        # One generated token through eight of 64 small experts.
        {"name": "experts_token", **_experts(1, 0, 64, 8, 2048, 768, 4, 32, "silu", True)},
        # A server's batch, one token each, two places empty; most experts have a token or a few.
        {"name": "experts_batch33", **_experts(33, 2, 64, 6, 2048, 1408, 4, 32, "silu", True)},
        # A few drafted tokens, two of eight large experts in 8 bits.
        {"name": "experts_int8_5", **_experts(5, 0, 8, 2, 4096, 14336, 8, 0, "gelu", False)},
        # A prompt over many small experts, ragged numbers of tokens to each.
        {"name": "experts_prompt2048", **_experts(2048, 0, 64, 8, 2048, 1024, 4, 32, "silu", True)},
        # A ragged prompt over few large experts.
        {"name": "experts_prompt1531", **_experts(1531, 30, 8, 2, 4096, 14336, 4, 32, "silu", True)},
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))


def draw(rng):
    kind = rng.choice(("norm", "product", "route", "experts", "experts", "experts"))
    if kind == "norm":
        width = rng.choice((_log(rng, 64, 8192), 64 * _log(rng, 1, 128)))
        codes = rng.choice(("none", "symmetric", "asymmetric"))
        tokens = min(_log(rng, 1, 16384), 8191 * 8192 // width)
        return _norm(tokens, width, rng.choice(("f16", "f16", "f32")), rng.random() < 0.8, rng.choice((0.0, 0.0, 1.0)),
                     codes == "none" or rng.random() < 0.5, codes)
    if kind == "product":
        return _product(_log(rng, 17, 2048), 16 * _log(rng, 16, 256), 8 * _log(rng, 32, 1792), rng.choice(("symmetric", "asymmetric")))
    if kind == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * max(2, _log(rng, 8, 512) // groups)
        top_groups = rng.randint(1, groups)
        chosen = min(rng.choice((1, 2, 4, 6, 8, 10, 16)), top_groups * (experts // groups))
        return _route(min(_log(rng, 1, 16384), 8192 * 256 // experts), experts, chosen, rng.choice(("softmax", "sigmoid")),
                      rng.random() < 0.5, groups, top_groups, rng.choice((1, 2)), rng.random() < 0.7, rng.choice((1.0, 2.5)),
                      rng.choice(("f16", "f32")))
    bits = rng.choice((4, 4, 8))
    experts = _log(rng, 4, 128)
    width, inner = 128 * _log(rng, 4, 32), 128 * _log(rng, 2, 112)
    while experts * width * inner > 8 * 4096 * 14336 * 4 // bits:
        if experts > 8:
            experts //= 2
        else:
            inner = max(128, inner // 256 * 128)
    chosen = min(rng.choice((1, 2, 4, 6, 8)), experts)
    tokens = rng.choice((1, _log(rng, 2, 16), _log(rng, 17, 128), _log(rng, 129, 2048)))
    while tokens > 1 and tokens * chosen * width * inner > 1501 * 2 * 4096 * 14336:
        tokens = (tokens + 1) // 2
    return _experts(tokens, rng.choice((0, 0, tokens // 16)), experts, chosen, width, inner, bits, rng.choice((32, 32, 64, 128)) if bits == 4 else 0,
                    rng.choice(("silu", "silu", "gelu")), rng.random() < 0.7)


@functools.lru_cache(None)
def _routing(tokens, padding, experts, chosen):
    """Experts of every token, some of them more popular than others: the same for every seed, since work() has to know them."""
    gen = torch.Generator().manual_seed(1000 * tokens + experts)
    logits = torch.randn(tokens, experts, generator=gen) + 0.5 * torch.randn(experts, generator=gen)
    ids = torch.topk(logits, chosen, dim=1).indices.int()
    ids[tokens - padding:] = -1
    return ids


def work(case):
    n = case["tokens"]
    if case["kind"] in ("norm", "product"):
        w, size = case["width"], 2 if case["type"] == "f16" else 4
        data = n * w * size * (3 if case["residual"] else 1) + w * size  # in, residual in and sum out
        if case["kind"] == "product":
            o = case["outputs"]
            return {"bytes": data + o * w + 2 * o + 2 * n * o, "flops": 2 * n * w * o}
        data += n * w * size if case["out"] else 0
        data += n * w + 8 * n if case["codes"] != "none" else 0
        return {"bytes": data, "flops": 6 * n * w}
    if case["kind"] == "route":
        e = case["experts"]
        return {"bytes": n * e * (2 if case["type"] == "f16" else 4) + 8 * n * case["chosen"] + (4 * e if case["bias"] else 0),
                "flops": 4 * n * e}
    ids = _routing(n, case["padding"], case["experts"], case["chosen"])
    used, pairs = int(torch.unique(ids[ids >= 0]).numel()), int((ids >= 0).sum())
    d, f = case["width"], case["inner"]
    scales = (2 * f * (d // case["block"]) + d * (f // case["block"])) * 2 if case["block"] else (2 * f + d) * 2
    return {"bytes": used * (3 * d * f * case["bits"] // 8 + scales) + 2 * n * d * (3 if case["residual"] else 2) + 8 * ids.numel(),
            "flops": 6 * pairs * d * f}


# ------------------------------------------------------------------------------------- what a program has in hand
def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _packed(codes, bits):
    """Codes [outputs][inputs] (int8) in blocks of 4 inputs x 4 outputs."""
    o, i = codes.shape
    blocks = codes.view(o // 4, 4, i // 4, 4).permute(2, 0, 3, 1).contiguous()  # [i / 4][o / 4][4 i][4 o]
    if bits == 8:
        return (blocks.view(-1).int() + 128).to(torch.uint8)
    nibbles = (blocks.view(-1, 2) + 8).to(torch.uint8)
    return nibbles[:, 0] | nibbles[:, 1] << 4


def _matrix(gen, o, i, bits, block):
    """A quantised matrix of o outputs and i inputs: packed codes, scales [groups][o]; products with inputs of size 1 have about size 1."""
    step = 2.6 if bits == 4 else 40.0
    codes = torch.empty(o, i, dtype=torch.int8, device="cuda")
    for at in range(0, o, 2048):
        rows = codes[at:at + 2048]
        rows.copy_(torch.round(_randn(gen, *rows.shape) * step).clamp_(-7 if bits == 4 else -127, 7 if bits == 4 else 127))
    groups = i // block if block else 1
    scales = torch.exp(0.2 * _randn(gen, groups, o)) / (step * math.sqrt(i))
    return codes, scales.half()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"norm": _prepare_norm, "product": _prepare_product, "route": _prepare_route, "experts": _prepare_experts}[case["kind"]](case, gen)


def _prepare_norm(case, gen):
    n, w = case["tokens"], case["width"]
    dtype = torch.float16 if case["type"] == "f16" else torch.float32
    channels = torch.exp(0.8 * _randn(gen, w))  # some channels of the residual stream are larger than the others
    empty = functools.partial(torch.empty, device="cuda")
    s = {"case": case, "x": _randn(gen, n, w).to(dtype), "residual": (_randn(gen, n, w) * channels).to(dtype) if case["residual"] else None,
         "weight": (1 - case["offset"] + 0.2 * _randn(gen, w)).to(dtype)}
    if case["residual"]:
        s["sum"] = empty(n, w, dtype=dtype)
    s["y"] = empty(n, w, dtype=dtype) if case["out"] else None
    if case["codes"] != "none":
        s["codes"], s["params"] = empty(n, -(-w // 16) * 16, dtype=torch.int8), empty(n, 3, dtype=torch.float32)
    return s


def _prepare_product(case, gen):
    s = _prepare_norm(case, gen)
    o, i = case["outputs"], case["width"]
    codes, scales = _matrix(gen, o, i, 8, 0)
    s["packed"], s["scales"] = _packed(codes, 8), scales
    s["totals"] = codes.sum(1, dtype=torch.int32)
    s["bias"] = (0.1 * _randn(gen, o)).half()
    s["out"] = torch.empty(case["tokens"], o, dtype=torch.float16, device="cuda")
    if own:
        m = _mld()
        s["plan"] = m.FullyConnectedPlan(o, i, 8, has_bias=True, max_tokens=case["tokens"], src_layout=m.LAYOUT_ROW_MAJOR,
                                         dst_layout=m.LAYOUT_ROW_MAJOR, prefill_act_quant=1 if case["codes"] == "symmetric" else 2)
        s["plan"].set_weights_sum(s["totals"])
    return s


def _prepare_route(case, gen):
    n, e = case["tokens"], case["experts"]
    logits = _randn(gen, n, e) * 1.5 + 0.5 * _randn(gen, e)
    s = {"case": case, "logits": logits.half() if case["type"] == "f16" else logits,
         "bias": 0.1 * _randn(gen, e) if case["bias"] else None,
         "ids": torch.empty(n, case["chosen"], dtype=torch.int32, device="cuda"),
         "weights": torch.empty(n, case["chosen"], dtype=torch.float32, device="cuda")}
    if own:
        m = _mld()
        s["router"] = m.MoeRouter(e, case["chosen"], score=m.MOE_SOFTMAX if case["score"] == "softmax" else m.MOE_SIGMOID,
                                  groups=case["groups"], top_groups=case["top_groups"], group_best=case["best"],
                                  renormalise=case["renormalise"], factor=case["factor"], f16=case["type"] == "f16")
    return s


def _prepare_experts(case, gen):
    n, e, k, d, f, bits, block = (case[x] for x in ("tokens", "experts", "chosen", "width", "inner", "bits", "block"))
    s = {"case": case, "x": _randn(gen, n, d).half(), "ids": _routing(n, case["padding"], e, k).cuda(),
         "weights": torch.softmax(_randn(gen, n, k), -1), "out": torch.empty(n, d, dtype=torch.float16, device="cuda"),
         "residual": (3 * _randn(gen, n, d)).half() if case["residual"] else None}
    for name, o, i in (("first", 2 * f, d), ("second", d, f)):
        s[name] = torch.empty(e, o * i * bits // 8, dtype=torch.uint8, device="cuda")
        s[name + "_scales"] = torch.empty(e, i // block if block else 1, o, dtype=torch.float16, device="cuda")
        for j in range(e):
            codes, s[name + "_scales"][j] = _matrix(gen, o, i, bits, block)
            s[name][j] = _packed(codes, bits)
    if own:
        m = _mld()
        s["plan"] = m.MoeExperts(e, k, d, f, weight_bits=bits, block=block, activation=m.MOE_SILU if case["act"] == "silu" else m.MOE_GELU_TANH,
                                 max_tokens=n)
    return s


# ------------------------------------------------------------------------------------------------------- one pass
def run(s):
    return {"norm": _run_norm, "product": _run_product, "route": _run_route, "experts": _run_experts}[s["case"]["kind"]](s)


def _values(codes, params, width):
    return codes[:, :width].float() * params[:, :1] + params[:, 1:2]


def _run_norm(s):
    case = s["case"]
    got = {}
    if own:
        coded = case["codes"] != "none"
        _mld().add_rms_norm(s["x"], weight=s["weight"], residual=s["residual"], sum_out=s.get("sum"), out=s["y"],
                            codes=s["codes"] if coded else None, params=s["params"] if coded else None,
                            symmetric=case["codes"] == "symmetric", eps=EPS, weight_offset=case["offset"])
        if case["residual"]:
            got["sum"] = s["sum"]
        if case["out"]:
            got["out"] = s["y"]
        if coded:
            got["codes"], got["params"] = s["codes"], s["params"]
    else:
        total, y, codes, params = _plain_norm(s)
        if case["residual"]:
            got["sum"] = total
        if case["out"]:
            got["out"] = y.to(total.dtype)
        if codes is not None:
            got["codes"], got["params"] = codes, params
    if "codes" in got:  # as the values that the codes stand for, with the scales and zero points
        codes, params = got.pop("codes"), got.pop("params")
        got["values"], got["steps"] = _values(codes, params, case["width"]), params[:, :2]
    return got


def _plain_norm(s):
    """(h in the tensors' type, y, codes or None, {scale, zero point} or None).  A row's codes do not hang on its norm, so they
    are taken of v = h w, and in 64 bits: v next to a border between two codes, or on one, as values of 16 bits often are."""
    case = s["case"]
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    wide = torch.float64 if case["codes"] != "none" else torch.float32
    v = h.to(wide)
    norm = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
    v = v * (case["offset"] + s["weight"].to(wide))
    if case["codes"] == "none":
        return h, v * norm, None, None
    if case["codes"] == "symmetric":
        top = v.abs().amax(-1, keepdim=True)
        step, zero = top * norm / 127, torch.zeros_like(top)
        codes = torch.floor(v * 127 / torch.where(top > 0, top, 1.0) + 0.5).clamp(-128, 127)
    else:
        low, high = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
        span = high - low
        step, zero = span * norm / 255, (low + span * (128 / 255)) * norm
        codes = torch.floor((v - low) * 255 / torch.where(span > 0, span, 1.0) + 0.5).clamp(0, 255) - 128
    return h, v * norm, codes.to(torch.int8), torch.cat((step, zero), -1).float()


def _run_product(s):
    case = s["case"]
    if own:
        _mld().add_rms_norm(s["x"], weight=s["weight"], residual=s["residual"], sum_out=s["sum"], codes=s["codes"], params=s["params"],
                            symmetric=case["codes"] == "symmetric", eps=EPS)
        s["plan"].run_codes(s["codes"], s["params"], s["packed"], s["scales"], s["out"], case["tokens"], bias=s["bias"])
        return {"sum": s["sum"], "out": s["out"]}
    h, _, codes, params = _plain_norm(s)
    w = _dequantised(s["packed"], s["scales"], case["outputs"], case["width"], 8)
    y = (codes.float() * params[:, :1] + params[:, 1:]) @ w.T + s["bias"].float()
    return {"sum": h, "out": y.half()}


def _dequantised(packed, scales, o, i, bits):
    """A matrix in fp32, [outputs][inputs]."""
    if bits == 4:
        blocks = torch.stack((packed & 15, packed >> 4), -1).view(i // 4, o // 4, 4, 4)
        zero = 8.0
    else:
        blocks = packed.view(i // 4, o // 4, 4, 4)
        zero = 128.0
    w = (blocks.float() - zero).permute(0, 2, 1, 3).reshape(scales.numel() // o, -1, o)  # [groups][inputs of a group][outputs]
    return (w * scales.view(-1, 1, o).float()).view(i, o).T


def _run_route(s):
    case = s["case"]
    if own:
        s["router"].run(s["logits"], s["ids"], s["weights"], bias=s["bias"])
        return {"ids": s["ids"], "weights": s["weights"]}
    x = s["logits"].double()  # 64 bits: two experts' values may be close
    n, e = x.shape
    if case["score"] == "softmax":
        score = torch.exp(x - x.amax(-1, keepdim=True))
        score = score / score.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    value = score if s["bias"] is None else score + s["bias"].double()
    if case["groups"] > 1:
        by_group = value.view(n, case["groups"], -1)
        best = by_group.sort(dim=-1, descending=True).values[..., :case["best"]].sum(-1)
        place = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros_like(best).scatter_(1, place, 1.0) > 0
        value = torch.where(kept[..., None], by_group, -math.inf).view(n, e)
    ids = torch.sort(value, dim=-1, descending=True, stable=True).indices[:, :case["chosen"]]
    weights = score.gather(1, ids)
    if case["renormalise"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return {"ids": ids.int(), "weights": (weights * case["factor"]).float()}


def _run_experts(s):
    case = s["case"]
    if own:
        s["plan"].run(s["x"], s["ids"], s["weights"], s["first"], s["first_scales"], s["second"], s["second_scales"], s["out"],
                      residual=s["residual"])
        return s["out"]
    d, f, bits = case["width"], case["inner"], case["bits"]
    x = s["x"].float()
    total = torch.zeros_like(x) if s["residual"] is None else s["residual"].float()
    for e in torch.unique(s["ids"]).tolist():
        if e < 0:
            continue
        token, place = torch.nonzero(s["ids"] == e, as_tuple=True)
        both = x[token] @ _dequantised(s["first"][e], s["first_scales"][e], 2 * f, d, bits).T
        gate, up = both[:, 0::2], both[:, 1::2]
        if case["act"] == "silu":
            gate = gate / (1 + torch.exp(-gate))
        else:
            gate = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate * gate * gate)))
        y = (gate * up) @ _dequantised(s["second"][e], s["second_scales"][e], d, f, bits).T
        total.index_add_(0, token, y * s["weights"][token, place][:, None])
    return total.half()


# ----------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "product": _exact_product, "route": _exact_route, "experts": _exact_experts}[case["kind"]](case, s)


def _exact_codes(case, s):
    """h, y, and for codes: (codes, scales, zero points), all in 64 bits."""
    h = s["x"].double()
    if case["residual"]:
        h = (h + s["residual"].double()).to(s["x"].dtype).double()
    w = s["weight"].double() + case["offset"]
    y = h * w * (h.square().sum(1, keepdim=True) / case["width"] + EPS).rsqrt()
    if case["codes"] == "none":
        return h, y, None
    v = h * w
    hi, lo, rms = v.max(1, keepdim=True).values, v.min(1, keepdim=True).values, (h.square().sum(1, keepdim=True) / case["width"] + EPS).sqrt()
    if case["codes"] == "symmetric":
        top = torch.maximum(hi, -lo)
        return h, y, (torch.floor(0.5 * (v * 254 / top + 1)), top / 127 / rms, torch.zeros_like(hi))
    scale = (hi - lo) / 255 / rms
    return h, y, (torch.floor(0.5 * ((v - lo) * 510 / (hi - lo) + 1)) - 128, scale, lo / rms + 128 * scale)


def _exact_norm(case, s):
    h, y, coded = _exact_codes(case, s)
    got = {}
    if case["residual"]:
        got["sum"] = h
    if case["out"]:
        got["out"] = y
    if coded is not None:
        codes, scale, zero = coded
        got["values"], got["steps"] = codes * scale + zero, torch.cat((scale, zero), 1)
    return got


def _exact_matrix(packed, scales, o, i, bits):
    """[outputs][inputs] in 64 bits, each value fetched from its place."""
    out, row = torch.arange(o, device="cuda"), torch.arange(i, device="cuda")
    got = torch.empty(o, i, dtype=torch.float64, device="cuda")
    per = i // scales.shape[0]
    for at in range(0, i, 256):
        k = row[at:at + 256][:, None]
        place = (k // 4 * (o // 4) + out // 4) * 16 + k % 4 * 4 + out % 4
        if bits == 8:
            code = packed[place].double() - 128
        else:
            code = (packed[place // 2] >> (place % 2 * 4).to(torch.uint8) & 15).double() - 8
        got[:, at:at + 256] = (code * scales.double()[k[:, 0] // per]).T
    return got


def _exact_product(case, s):
    h, _, (codes, scale, zero) = _exact_codes(case, s)
    w = _exact_matrix(s["packed"], s["scales"], case["outputs"], case["width"], 8)
    return {"sum": h, "out": (codes * scale + zero) @ w.T + s["bias"].double()}


def _exact_route(case, s):
    x = s["logits"].double()
    score = torch.softmax(x, -1) if case["score"] == "softmax" else torch.sigmoid(x)
    value = score.clone()
    if case["bias"]:
        value += s["bias"].double()
    per = case["experts"] // case["groups"]
    if case["groups"] > 1:
        of_group = [value[:, g * per:(g + 1) * per].topk(min(case["best"], per)).values.sum(1) for g in range(case["groups"])]
        of_group = torch.stack(of_group, 1)
        for _ in range(case["groups"] - case["top_groups"]):  # the worst group goes, of equal ones the last
            worst = case["groups"] - 1 - of_group.flip(1).argmin(1)
            of_group.scatter_(1, worst[:, None], math.inf)
            of_worst = torch.arange(case["experts"], device="cuda") // per == worst[:, None]
            value.masked_fill_(of_worst, -math.inf)
    ids = torch.empty(case["tokens"], case["chosen"], dtype=torch.int64, device="cuda")
    for j in range(case["chosen"]):
        top = value.max(1, keepdim=True).values
        ids[:, j] = (value == top).int().argmax(1)
        value.scatter_(1, ids[:, j:j + 1], -math.inf)
    weights = torch.gather(score, 1, ids)
    if case["renormalise"]:
        weights /= weights.sum(1, keepdim=True)
    return {"ids": ids.int(), "weights": weights * case["factor"]}


def _exact_experts(case, s):
    d, f = case["width"], case["inner"]
    out = torch.zeros(case["tokens"], d, dtype=torch.float64, device="cuda")
    if case["residual"]:
        out += s["residual"].double()
    for e in range(case["experts"]):
        weight = ((s["ids"] == e).double() * s["weights"].double()).sum(1)
        tokens = (s["ids"] == e).any(1).nonzero()[:, 0]
        if tokens.numel() == 0:
            continue
        w = _exact_matrix(s["first"][e], s["first_scales"][e], 2 * f, d, case["bits"])
        x = s["x"][tokens].double()
        gate, up = x @ w[0::2].T, x @ w[1::2].T
        if case["act"] == "silu":
            hidden = gate * torch.sigmoid(gate) * up
        else:
            hidden = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3))) * up
        del w
        w = _exact_matrix(s["second"][e], s["second_scales"][e], d, f, case["bits"])
        out[tokens] += weight[tokens, None] * (hidden @ w.T)
    return out
