"""Cases for the operators around quantised expert layers, each in a plain form and as a call of this package.

Operators (the case's "op"):
  route     router logits -> expert ids and weights of every token
  dispatch  tokens -> rows sorted by expert, quantised for the grouped matmuls, with group list and row lists
  linear    activations quantised to 4-bit codes with a scale per 16, times weights held that way
  experts   the grouped product of such rows with every expert's weights
  combine   the experts' output rows -> weighted sum per token

The plain forms are written in elementary tensor operations, in 32 bits (expert selection in 64), rounded once.
"""
import torch

own = False

FLOATS = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one token of a serving step through a router with 256 experts in 8 groups: latency alone
        {"name": "route_one", "op": "route", "tokens": 1, "experts": 256, "top_k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "kept": 4, "renormalize": True, "logits": "f32"},
        # a prompt batch through the same router
        {"name": "route_prompt", "op": "route", "tokens": 16384, "experts": 256, "top_k": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "kept": 4, "renormalize": True, "logits": "bf16"},
        # an odd batch through a small ungrouped softmax router
        {"name": "route_softmax", "op": "route", "tokens": 4099, "experts": 60, "top_k": 4, "score": "softmax",
         "bias": False, "groups": 1, "kept": 1, "renormalize": False, "logits": "f16"},
        # a serving step: 16 tokens to 8 of 64 experts as int8 rows
        {"name": "dispatch_step", "op": "dispatch", "tokens": 16, "experts": 64, "top_k": 8, "k": 4096,
         "format": "int8", "x": "bf16"},
        # a prompt batch as block-scaled 8-bit rows
        {"name": "dispatch_prompt", "op": "dispatch", "tokens": 8192, "experts": 64, "top_k": 8, "k": 7168,
         "format": "e4m3", "x": "bf16"},
        # a serving step through one 4-bit layer: the weights are read once
        {"name": "linear_step", "op": "linear", "m": 16, "n": 14336, "k": 4096, "x": "bf16"},
        # an odd prompt through a narrow projection: quantising is half of the work, ragged edges on both sides
        {"name": "linear_narrow", "op": "linear", "m": 4111, "n": 515, "k": 7168, "x": "bf16"},
        # a large prompt through a square layer
        {"name": "linear_prompt", "op": "linear", "m": 8192, "n": 8192, "k": 8192, "x": "bf16"},
        # a serving step of 32 tokens to 8 of 64 experts: every expert's weights are read for a few rows
        {"name": "experts_step", "op": "experts", "rows": 256, "experts": 64, "n": 4096, "k": 7168, "skew": 0.5},
        # a prompt of 4096 tokens to 8 of 64 experts
        {"name": "experts_prompt", "op": "experts", "rows": 32768, "experts": 64, "n": 4096, "k": 7168, "skew": 0.5},
        # a serving step's rows back to its tokens, with the shared expert's output
        {"name": "combine_step", "op": "combine", "tokens": 16, "top_k": 8, "n": 7168, "d": "bf16", "shared": True},
        # a prompt batch's rows back to its tokens
        {"name": "combine_prompt", "op": "combine", "tokens": 8192, "top_k": 8, "n": 7168, "d": "bf16", "shared": False},
    ]


def _spread(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["route", "dispatch", "linear", "experts", "combine"])
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = max(8 * groups, _spread(rng, 8, 256) // groups * groups)
        kept = rng.randint(max(1, groups // 2), groups)
        return {"op": op, "tokens": _spread(rng, 1, 16384), "experts": experts, "top_k": rng.randint(1, 8),
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups, "kept": kept,
                "renormalize": rng.random() < 0.6, "logits": rng.choice(["f32", "bf16", "f16"])}
    if op == "dispatch":
        experts = _spread(rng, 4, 256)
        return {"op": op, "tokens": _spread(rng, 1, 8192), "experts": experts, "top_k": rng.randint(1, min(8, experts)),
                "k": 32 * rng.randint(2, 224), "format": rng.choice(["int8", "e4m3"]),
                "x": rng.choice(["bf16", "f32"])}
    if op == "linear":
        return {"op": op, "m": _spread(rng, 1, 8192), "n": _spread(rng, 64, 8192), "k": 32 * _spread(rng, 2, 256),
                "x": rng.choice(["bf16", "f32"])}
    if op == "experts":
        return {"op": op, "rows": _spread(rng, 1, 16384), "experts": _spread(rng, 2, 64), "n": _spread(rng, 64, 4096),
                "k": 32 * _spread(rng, 4, 224), "skew": round(rng.uniform(0.1, 1.0), 3)}
    return {"op": op, "tokens": _spread(rng, 1, 8192), "top_k": rng.randint(1, 8), "n": _spread(rng, 16, 7168),
            "d": rng.choice(["bf16", "f32"]), "shared": rng.random() < 0.5}


def work(case):
    op = case["op"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        return {"bytes": t * e * size[case["logits"]] + t * k * 8 + (4 * e if case["bias"] else 0), "flops": 4 * t * e}
    if op == "dispatch":
        t, e, j, k = case["tokens"], case["experts"], case["top_k"], case["k"]
        scale = 4 if case["format"] == "int8" else (k // 32 + 1) // 2 * 2
        rows = t * j
        return {"bytes": t * k * size[case["x"]] + rows * 8 + rows * (k + scale) + rows * 12 + 8 * e,
                "flops": 3 * t * k}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * size[case["x"]] + n * (k // 2 + k // 16) + m * n * 2, "flops": 2 * m * n * k}
    if op == "experts":
        r, e, n, k = case["rows"], case["experts"], case["n"], case["k"]
        used = min(e, r)
        return {"bytes": r * (k // 2 + k // 16) + used * n * (k // 2 + k // 16) + r * n * 2 + 12 * e,
                "flops": 2 * r * n * k}
    t, j, n = case["tokens"], case["top_k"], case["n"]
    return {"bytes": t * j * n * size[case["d"]] + t * n * size[case["d"]] * (2 if case["shared"] else 1) + t * j * 8,
            "flops": 2 * t * j * n}


# ------------------------------------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(g, rows, k, dtype):
    # a few channels and a few tokens stand out, as in the residual stream
    x = torch.randn((rows, k), generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn((1, k), generator=g, device="cuda"))
    x *= torch.exp(0.3 * torch.randn((rows, 1), generator=g, device="cuda"))
    return x.to(dtype)


def _weights(g, count, n, k):
    """Weights quantised from a normal distribution: codes [count, n, k/2], scales tiled, and their tensor scale."""
    sample = 0.02 * torch.randn((65536, 16), generator=g, device="cuda")
    tensor_scale = sample.abs().max() / 2688.0
    codes, scale, _ = _quantize_fp4(sample, tensor_scale)
    packed = _pack(codes).view(torch.int64).reshape(-1)
    pick = torch.randint(0, 65536, (count * n * (k // 16),), generator=g, device="cuda", dtype=torch.int32)
    q = packed[pick].view(torch.uint8).reshape(count, n, k // 2)
    s = scale.reshape(-1).view(torch.uint8)[pick].reshape(count, n, k // 16)
    return q, _tile_scales(s), tensor_scale


def _group_sizes(g, rows, experts, skew):
    """Row counts of unevenly loaded experts, the largest at a few times the mean, as a tensor."""
    load = torch.softmax(skew * torch.randn((experts,), generator=g, device="cuda"), 0)
    draws = torch.multinomial(load, rows, replacement=True, generator=g)
    return torch.bincount(draws, minlength=experts)


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    state = {"case": case}
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        state["logits"] = (1.5 * torch.randn((t, e), generator=g, device="cuda")).to(FLOATS[case["logits"]])
        state["bias"] = 0.1 * torch.randn((e,), generator=g, device="cuda") if case["bias"] else None
        state["weights"] = torch.empty((t, k), dtype=torch.float32, device="cuda")
        state["ids"] = torch.empty((t, k), dtype=torch.int32, device="cuda")
    elif op == "dispatch":
        t, e, j, k = case["tokens"], case["experts"], case["top_k"], case["k"]
        logits = torch.randn((t, e), generator=g, device="cuda") + torch.randn((1, e), generator=g, device="cuda")
        top = torch.topk(torch.softmax(logits, 1), j, 1)
        state["ids"] = top.indices.to(torch.int32).contiguous()
        state["weights"] = top.values.contiguous()
        state["x"] = _activations(g, t, k, FLOATS[case["x"]])
        rows = t * j
        state["group_list"] = torch.zeros((e,), dtype=torch.int64, device="cuda")
        state["position"] = torch.zeros((t, j), dtype=torch.int32, device="cuda")
        state["row_index"] = torch.zeros((rows,), dtype=torch.int32, device="cuda")
        state["row_weight"] = torch.zeros((rows,), dtype=torch.float32, device="cuda")
        if case["format"] == "int8":
            state["q"] = torch.zeros((rows, k), dtype=torch.int8, device="cuda")
            state["scale"] = torch.zeros((rows,), dtype=torch.float32, device="cuda")
        else:
            state["q"] = torch.zeros((rows, k), dtype=torch.uint8, device="cuda")
            state["scale"] = torch.zeros((rows, (k // 32 + 1) // 2 * 2), dtype=torch.uint8, device="cuda")
    elif op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        state["x"] = _activations(g, m, k, FLOATS[case["x"]])
        q, s, w_scale = _weights(g, 1, n, k)
        state["w"], state["w_scale"] = q[0], s[0]
        # the activations' tensor scale as calibrated beforehand: some values of a batch may lie above it
        state["x_scale"] = (state["x"].float().square().mean().sqrt() * 14.3 / 2688.0).reshape(1)
        state["alpha"] = (state["x_scale"] * w_scale).reshape(1)
        state["d"] = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    elif op == "experts":
        r, e, n, k = case["rows"], case["experts"], case["n"], case["k"]
        x = _activations(g, r, k, torch.bfloat16)
        x_scale = x.abs().max().float() / 2688.0
        codes, scale, _ = _quantize_fp4(x.float(), x_scale)
        state["a"], state["a_scale"] = _pack(codes), scale.view(torch.uint8)
        state["w"], state["w_scale"], w_scale = _weights(g, e, n, k)
        # every expert's weights have a tensor scale of their own
        state["alpha"] = x_scale * w_scale * torch.exp(0.2 * torch.randn((e,), generator=g, device="cuda"))
        sizes = _group_sizes(g, r, e, case["skew"])
        state["group_list"] = torch.cumsum(sizes, 0)
        state["ends"] = [int(v) for v in state["group_list"].tolist()]
        state["d"] = torch.empty((r, n), dtype=torch.bfloat16, device="cuda")
    else:
        t, j, n = case["tokens"], case["top_k"], case["n"]
        state["rows"] = torch.randn((t * j, n), generator=g, device="cuda").to(FLOATS[case["d"]])
        state["position"] = torch.randperm(t * j, generator=g, device="cuda").to(torch.int32).reshape(t, j)
        w = torch.rand((t, j), generator=g, device="cuda")
        state["weights"] = 2.5 * w / w.sum(1, keepdim=True)
        state["shared"] = torch.randn((t, n), generator=g, device="cuda").to(FLOATS[case["d"]]) if case["shared"] else None
        state["out"] = torch.empty((t, n), dtype=FLOATS[case["d"]], device="cuda")
    return state


# ------------------------------------------------------------------------------------------------ plain forms

def _e2m1_values(device):
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return torch.tensor(grid + [-v for v in grid], dtype=torch.float32, device=device)


def _quantize_fp4(x, tensor_scale):
    """x fp32 [rows, k] -> codes uint8 [rows, k], scales float8_e4m3fn [rows, k/16], and what they stand for
    without the tensor scale, fp32 [rows, k].  A scale is amax / 6 of its 16 values, in units of tensor_scale; a code
    is the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, a tie going to the even code."""
    rows, k = x.shape
    blocks = x.reshape(rows, k // 16, 16)
    amax = blocks.abs().amax(2)
    scale = torch.div(amax, 6.0 * tensor_scale).clamp(max=448.0).to(torch.float8_e4m3fn)
    step = scale.float() * tensor_scale
    inverse = torch.where(step > 0, torch.reciprocal(step), torch.zeros_like(step))
    y = blocks * inverse[:, :, None]
    m = y.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
    code = (code + 8 * (y < 0)).to(torch.uint8)
    stands_for = _e2m1_values(x.device)[code.int()] * scale.float()[:, :, None]
    return code.reshape(rows, k), scale, stands_for.reshape(rows, k)


def _pack(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous()


def _unpack(q):
    """Packed codes [..., k/2] -> their values, fp32 [..., k]."""
    values = _e2m1_values(q.device)
    byte = torch.arange(256, device=q.device)
    pairs = torch.stack([values[byte & 15], values[byte >> 4]], 1)
    return pairs[q.int()].flatten(-2)


def _tile_scales(s):
    """Scale bytes [count, rows, blocks] -> [count, row blocks of 128, words of 4 blocks, 32, 4, 4]: the byte of row r and
    block b is [r // 128][b // 4][r % 32][r % 128 // 32][b % 4]."""
    count, rows, blocks = s.shape
    s = torch.nn.functional.pad(s, (0, -blocks % 4, 0, -rows % 128))
    s = s.reshape(count, s.shape[1] // 128, 4, 32, s.shape[2] // 4, 4)
    return s.permute(0, 1, 4, 3, 2, 5).contiguous()


def _untile_scales(t, rows, blocks):
    """The reverse of _tile_scales, as fp32 values [count, rows, blocks]."""
    count, rb, words = t.shape[:3]
    s = t.permute(0, 1, 4, 3, 2, 5).reshape(count, rb * 128, words * 4)[:, :rows, :blocks]
    return s.contiguous().view(torch.float8_e4m3fn).float()


def _dequantized(w, w_scale, n, k):
    """Weights [count, n, k] without their tensor scale, fp32."""
    count = w.shape[0]
    values = _unpack(w).reshape(count, n, k // 16, 16)
    values *= _untile_scales(w_scale, n, k // 16)[..., None]
    return values.reshape(count, n, k)


def _plain_route(s):
    c = s["case"]
    x = s["logits"].double()
    open_ = x > -float("inf")  # (a NaN is not open either)
    x = torch.where(open_, x, torch.full_like(x, -float("inf")))
    if c["score"] == "softmax":
        e = torch.exp(x - x.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = torch.sigmoid(x)
    # without a bias the order of the scores is the order of the logits
    key = score + s["bias"].double() if s["bias"] is not None else x
    if c["groups"] > 1:
        t, e = key.shape
        per = e // c["groups"]
        by_group = (key if s["bias"] is not None else score).reshape(t, c["groups"], per)
        group_key = torch.topk(by_group, min(2, per), 2).values.sum(2)
        rank = torch.sort(group_key, dim=1, descending=True, stable=True).indices[:, :c["kept"]]
        keep = torch.zeros_like(group_key, dtype=torch.bool).scatter(1, rank, True)
        key = torch.where(keep.repeat_interleave(per, 1), key, torch.full_like(key, -float("inf")))
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :c["top_k"]]
    weights = score.gather(1, ids)
    if c["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    return {"weights": weights.float(), "ids": ids.to(torch.int32)}


def _row_order(ids, experts):
    """Rows sorted by expert, a token's pairs in the order of the tokens: (pair of each row, row of each pair, ends)."""
    flat = ids.reshape(-1).long()
    pair = torch.sort(flat, stable=True).indices
    position = torch.empty_like(pair)
    position[pair] = torch.arange(pair.numel(), device=pair.device)
    return pair, position, torch.cumsum(torch.bincount(flat, minlength=experts), 0)


def _plain_dispatch(s):
    c = s["case"]
    pair, position, ends = _row_order(s["ids"], c["experts"])
    x = s["x"].float()
    if c["format"] == "int8":
        amax = x.abs().amax(1)
        inverse = torch.where(amax > 0, torch.div(torch.full_like(amax, 127.0), amax), torch.zeros_like(amax))
        q = torch.clamp(torch.round(x * inverse[:, None]), -127, 127).to(torch.int8)
        scale = torch.div(amax, torch.full_like(amax, 127.0))
    else:
        # one power of two per 32 values: the largest's exponent less 8; nearest code, a tie to the smaller magnitude
        t, k = x.shape
        blocks = x.reshape(t, k // 32, 32)
        amax = blocks.abs().amax(2)
        exponent = torch.where(amax < 1e-12, torch.zeros_like(amax), torch.frexp(amax).exponent - 9.0)
        y = (blocks * torch.exp2(-exponent)[..., None]).clamp(-448.0, 448.0)
        m = y.abs()
        grid = torch.exp2(torch.clamp(torch.frexp(m).exponent - 1.0, min=-6.0) - 3.0)
        low = torch.floor(m / grid)
        m = (low + (m / grid - low > 0.5)) * grid
        q = torch.where(y < 0, -m, m).reshape(t, k).to(torch.float8_e4m3fn).view(torch.uint8)
        scale = (exponent + 127.0).to(torch.uint8)
        scale = torch.nn.functional.pad(scale, (0, scale.shape[1] % 2), value=127)
    token = pair // c["top_k"]
    s["q"].copy_(q[token])
    s["scale"].copy_(scale[token])
    return _dispatch_outputs(s, s["q"], s["scale"], ends, token.to(torch.int32), s["weights"].reshape(-1)[pair],
                             position.to(torch.int32).reshape(c["tokens"], c["top_k"]))


def _dispatch_outputs(s, q, scale, group_list, row_index, row_weight, position):
    if s["case"]["format"] == "e4m3":
        q, scale = q.view(torch.float8_e4m3fn), scale.view(torch.float8_e8m0fnu)
    return {"q": q, "scale": scale, "group_list": group_list, "row_index": row_index, "row_weight": row_weight,
            "position": position}


def _plain_linear(s):
    c = s["case"]
    x = _quantize_fp4(s["x"].float(), s["x_scale"])[2]
    w = _dequantized(s["w"][None], s["w_scale"][None], c["n"], c["k"])[0]
    return ((x @ w.t()) * s["alpha"]).to(torch.bfloat16)


def _plain_experts(s):
    c = s["case"]
    k = c["k"]
    a = _unpack(s["a"]).reshape(c["rows"], k // 16, 16) * s["a_scale"].view(torch.float8_e4m3fn).float()[..., None]
    a = a.reshape(c["rows"], k)
    d = torch.empty((c["rows"], c["n"]), dtype=torch.bfloat16, device=a.device)
    begin = 0
    for e, end in enumerate(s["ends"]):  # (experts without rows are left out)
        if end > begin:
            w = _dequantized(s["w"][e:e + 1], s["w_scale"][e:e + 1], c["n"], k)[0]
            d[begin:end] = ((a[begin:end] @ w.t()) * s["alpha"][e]).to(torch.bfloat16)
        begin = end
    return d


def _plain_combine(s):
    rows = s["rows"][s["position"].long()].float()
    out = (rows * s["weights"][..., None]).sum(1)
    if s["shared"] is not None:
        out = out + s["shared"].float()
    return out.to(s["rows"].dtype)


# ------------------------------------------------------------------------------------------------ this package's calls

def _workspace(s, size):
    """The workspace that a program keeps beside its buffers."""
    if "workspace" not in s:
        s["workspace"] = torch.empty((max(size(), 256),), dtype=torch.uint8, device="cuda")
    return s["workspace"]


def _own(s):
    from catlass_b200 import capi
    c = s["case"]
    types = {"f32": capi.DTYPE_F32, "bf16": capi.DTYPE_BF16, "f16": capi.DTYPE_F16}
    if c["op"] == "route":
        capi.moe_route(s["logits"], s["weights"], s["ids"], c["tokens"], c["experts"], c["top_k"],
                       score=capi.ROUTE_SOFTMAX if c["score"] == "softmax" else capi.ROUTE_SIGMOID, bias=s["bias"],
                       groups=c["groups"], groups_kept=c["kept"], group_score=capi.ROUTE_GROUP_TOP2_SUM,
                       renormalize=c["renormalize"], logits_type=types[c["logits"]])
        return {"weights": s["weights"], "ids": s["ids"]}
    if c["op"] == "dispatch":
        ws = _workspace(s, lambda: capi.moe_dispatch_workspace_size(c["tokens"], c["experts"], c["top_k"]))
        capi.moe_dispatch(s["x"], s["ids"], s["weights"], s["group_list"], s["position"], c["tokens"], c["experts"],
                          c["top_k"], c["k"], capi.DISPATCH_INT8 if c["format"] == "int8" else capi.DISPATCH_MX_E4M3,
                          q=s["q"], scale=s["scale"], row_index=s["row_index"], row_weight=s["row_weight"],
                          x_type=types[c["x"]], workspace=ws)
        return _dispatch_outputs(s, s["q"], s["scale"], s["group_list"], s["row_index"], s["row_weight"], s["position"])
    if c["op"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        if "codes" not in s:  # the layer's buffers for its quantised activations
            s["codes"] = torch.empty((m, k // 2), dtype=torch.uint8, device="cuda")
            s["code_scales"] = torch.empty((capi.nvfp4_tiled_scale_bytes(m, k),), dtype=torch.uint8, device="cuda")
        ws = _workspace(s, lambda: capi.nvfp4_matmul_workspace_size(m, n, k, capi.NVFP4_SCALES_TILED,
                                                                    capi.NVFP4_SCALES_TILED))
        capi.nvfp4_quantize(s["x"], s["codes"], s["code_scales"], m, k, s["x_scale"], x_type=types[c["x"]],
                            scale_layout=capi.NVFP4_SCALES_TILED)
        capi.nvfp4_matmul(s["codes"], s["w"], s["code_scales"], s["w_scale"], s["d"], m, n, k, ws, alpha=s["alpha"],
                          scale_a_layout=capi.NVFP4_SCALES_TILED, scale_b_layout=capi.NVFP4_SCALES_TILED)
        return s["d"]
    if c["op"] == "experts":
        r, e, n, k = c["rows"], c["experts"], c["n"], c["k"]
        ws = _workspace(s, lambda: capi.nvfp4_grouped_matmul_workspace_size(r, n, k, e, capi.NVFP4_SCALES_TILED))
        capi.nvfp4_grouped_matmul(s["a"], s["w"], s["group_list"], s["a_scale"], s["w_scale"], s["d"], r, n, k, e, ws,
                                  alpha=s["alpha"], scale_b_layout=capi.NVFP4_SCALES_TILED,
                                  group_list_kind=capi.GROUP_LIST_PREFIX_SUMS)
        return s["d"]
    capi.moe_combine(s["rows"], s["position"], s["weights"], s["out"], c["tokens"], c["n"], c["top_k"],
                     d_type=types[c["d"]], out_type=types[c["d"]], shared=s["shared"])
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"route": _plain_route, "dispatch": _plain_dispatch, "linear": _plain_linear, "experts": _plain_experts,
            "combine": _plain_combine}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ 64-bit values

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")

    def codes_to_64(q):
        nibble = torch.stack([q & 15, q >> 4], -1).flatten(-2).long()
        return torch.where(nibble >= 8, -1.0, 1.0) * grid[nibble & 7]

    def scales_to_64(t, rows, blocks):  # tiled bytes of one matrix
        r = torch.arange(rows, device="cuda")[:, None]
        b = torch.arange(blocks, device="cuda")[None, :]
        byte = t[r // 128, b // 4, r % 32, r % 128 // 32, b % 4].long()
        e, f = byte >> 3 & 15, (byte & 7).double()
        return torch.where(e > 0, (1 + f / 8) * torch.exp2(e.double() - 7), f / 8 * 2.0 ** -6)

    if op == "route":
        p = s["logits"].double()
        p = torch.softmax(p, 1) if case["score"] == "softmax" else 1 / (1 + torch.exp(-p))
        key = p if s["bias"] is None else p + s["bias"].double()
        if case["groups"] > 1:
            g = key.reshape(key.shape[0], case["groups"], -1)
            best = g.sort(2, descending=True).values[:, :, :2].sum(2)
            floor = best.sort(1, descending=True).values[:, case["kept"] - 1, None]
            key = torch.where((best >= floor)[:, :, None], g, -float("inf")).reshape(key.shape)
        w = p.gather(1, key.topk(case["top_k"], 1).indices)
        return {"weights": w / w.sum(1, keepdim=True) if case["renormalize"] else w, "ids": None}
    if op == "dispatch":
        token = torch.argsort(s["ids"].reshape(-1).long(), stable=True) // case["top_k"]
        weight = s["weights"].double().reshape(-1)[torch.argsort(s["ids"].reshape(-1).long(), stable=True)]
        x = s["x"].double()
        if case["format"] == "int8":
            return {"scale": (x.abs().amax(1) / 127)[token], "row_weight": weight}
        b = x.reshape(x.shape[0], -1, 32)
        e = (b.abs().amax(2).clamp(min=1e-12).view(torch.int64) >> 52).double() - 1023 - 8  # the exponent field
        scale = torch.nn.functional.pad(torch.exp2(e), (0, e.shape[1] % 2), value=1.0)
        y = (b / torch.exp2(e)[..., None]).reshape(x.shape)
        # the values of the 8-bit codes in ascending order; the nearest one, the smaller where two are as near
        code = torch.arange(127, device="cuda")
        value = torch.where(code < 8, code / 512.0, (1 + (code & 7) / 8.0) * torch.exp2((code >> 3) - 7.0)).double()
        out = torch.bucketize(y.abs(), (value[1:] + value[:-1]) / 2, right=False)
        return {"q": (torch.sign(y) * value[out])[token], "scale": scale[token], "row_weight": weight}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        unit = s["x_scale"].double()
        x = s["x"].double().reshape(m, k // 16, 16)
        ratio = (x.abs().amax(2) / (6 * unit)).clamp(max=448.0)
        scale = ratio.float().to(torch.float8_e4m3fn).double()
        y = torch.where(scale[..., None] > 0, x / (scale * unit)[..., None], 0.0)
        # half-way points belong to the neighbour with the even code: below .25, 1.25, 2.5 and 5, above .75, 1.75 and 3.5
        middle = (grid[1:] + grid[:-1]) / 2
        up = torch.nextafter(middle, torch.zeros_like(middle))
        edge = torch.where(torch.arange(7, device="cuda") % 2 == 0, middle, up)
        y = torch.sign(y) * grid[torch.bucketize(y.abs(), edge, right=False)]
        x = (y * scale[..., None]).reshape(m, k)
        w = codes_to_64(s["w"]) * scales_to_64(s["w_scale"], n, k // 16).repeat_interleave(16, 1)
        return x @ w.t() * s["alpha"].double()
    if op == "experts":
        k, n = case["k"], case["n"]
        a = codes_to_64(s["a"]) * s["a_scale"].view(torch.float8_e4m3fn).double().repeat_interleave(16, 1)
        d, begin = torch.empty((case["rows"], n), dtype=torch.float64, device="cuda"), 0
        for e, end in enumerate(s["ends"]):
            if end > begin:
                w = codes_to_64(s["w"][e]) * scales_to_64(s["w_scale"][e], n, k // 16).repeat_interleave(16, 1)
                d[begin:end] = s["alpha"][e].double() * (a[begin:end] @ w.t())
            begin = end
        return d
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for j in range(case["top_k"]):
        out += s["weights"][:, j, None].double() * s["rows"][s["position"][:, j].long()].double()
    return out if s["shared"] is None else out + s["shared"].double()
