"""Expert layers end to end, as a serving step runs them: route, dispatch with quantisation, grouped matmuls, combine.  Every
step's output is held against the plain definition applied to the buffers that step read."""
import numpy as np
import pytest

import moe_reference as R
import oracle_lib as O

pytestmark = pytest.mark.gpu


def u8(torch, cuda, *shape):
    return torch.empty(shape, dtype=torch.uint8, device=cuda)


class Nvfp4Layer:
    """One NVFP4 expert layer with its buffers: hidden -> 2 * inner (act next to gate) -> hidden."""

    def __init__(self, torch, capi, cuda, tokens, hidden, inner, experts, top_k, seed):
        self.torch, self.capi = torch, capi
        self.shape = tokens, hidden, inner, experts, top_k
        rng = np.random.default_rng(seed)
        self.w, self.tensor_scale = [], []
        for n, k in ((2 * inner, hidden), (hidden, inner)):
            w = (rng.standard_normal((experts, n, k)) / np.sqrt(k)).astype(np.float32)
            g = np.float32(np.abs(w).max() / 2688)
            parts = [R.nvfp4_quantize(w[e], g) for e in range(experts)]
            tiled = np.stack([R.tile_scales(s) for _, s in parts])
            self.w.append((torch.from_numpy(np.stack([R.pack(c) for c, _ in parts])).to(cuda), torch.from_numpy(tiled).to(cuda),
                           np.stack([R.nvfp4_values(c, s) for c, s in parts])))
            self.tensor_scale.append(g)
        rows = tokens * top_k
        self.x_scale = torch.tensor([5.0 / 2688], device=cuda)
        self.h_scale = torch.tensor([3.0 / 2688], device=cuda)
        self.alpha = [torch.full((experts,), float(np.float32(s) * w), device=cuda)
                      for s, w in ((self.x_scale.item(), self.tensor_scale[0]), (self.h_scale.item(), self.tensor_scale[1]))]
        self.ids = torch.empty((tokens, top_k), dtype=torch.int32, device=cuda)
        self.weights = torch.empty((tokens, top_k), device=cuda)
        self.position = torch.empty_like(self.ids)
        self.group_list = torch.empty((experts,), dtype=torch.int64, device=cuda)
        self.a, self.a_scale = u8(torch, cuda, rows, hidden // 2), u8(torch, cuda, rows, hidden // 16)
        self.c = torch.empty((rows, 2 * inner), dtype=torch.bfloat16, device=cuda)
        self.h, self.h_scales = u8(torch, cuda, rows, inner // 2), u8(torch, cuda, rows, inner // 16)
        self.d = torch.empty((rows, hidden), dtype=torch.bfloat16, device=cuda)
        self.out = torch.empty((tokens, hidden), dtype=torch.bfloat16, device=cuda)
        need = [capi.nvfp4_grouped_matmul_workspace_size(rows, n, k, experts, 1)
                for n, k in ((2 * inner, hidden), (hidden, inner))] + [capi.moe_dispatch_workspace_size(tokens, experts, top_k)]
        self.ws = u8(torch, cuda, max(need + [256]))

    def run(self, x, logits, bias, shared):
        capi = self.capi
        t, hidden, inner, experts, top_k = self.shape
        rows = t * top_k
        capi.moe_route(logits, self.weights, self.ids, t, experts, top_k, score=capi.ROUTE_SIGMOID, bias=bias, scaling=2.5)
        capi.moe_dispatch(x, self.ids, self.weights, self.group_list, self.position, t, experts, top_k, hidden,
                          capi.DISPATCH_NVFP4, q=self.a, scale=self.a_scale, tensor_scale=self.x_scale, workspace=self.ws)
        kw = dict(scale_b_layout=capi.NVFP4_SCALES_TILED, group_list_kind=capi.GROUP_LIST_PREFIX_SUMS)
        capi.nvfp4_grouped_matmul(self.a, self.w[0][0], self.group_list, self.a_scale, self.w[0][1], self.c, rows, 2 * inner,
                                  hidden, experts, self.ws, alpha=self.alpha[0], **kw)
        capi.nvfp4_quantize(self.c, self.h, self.h_scales, rows, inner, self.h_scale, swiglu=True,
                            row_count=self.group_list[-1:])
        capi.nvfp4_grouped_matmul(self.h, self.w[1][0], self.group_list, self.h_scales, self.w[1][1], self.d, rows, hidden,
                                  inner, experts, self.ws, alpha=self.alpha[1], **kw)
        capi.moe_combine(self.d, self.position, self.weights, self.out, t, hidden, top_k, shared=shared)

    def check(self, x, logits, bias, shared):
        t, hidden, inner, experts, top_k = self.shape
        host = lambda v: v.double().cpu().numpy()  # noqa: E731
        want_ids, want_w = R.route(host(logits), top_k, True, host(bias), renormalize=True, scaling=2.5)
        ids, weights = self.ids.cpu().numpy(), host(self.weights)
        assert np.array_equal(ids, want_ids) and np.allclose(weights, want_w, rtol=2.0 ** -16, atol=0)
        sizes, position, pair = R.dispatch(ids, experts)
        assert np.array_equal(self.position.cpu().numpy(), position)
        assert np.array_equal(self.group_list.cpu().numpy(), np.cumsum(sizes))
        rows = pair.size
        codes, scale = R.nvfp4_quantize(x.float().cpu().numpy(), np.float32(self.x_scale.item()))
        assert np.array_equal(self.a.cpu().numpy()[:rows], R.pack(codes)[pair // top_k])
        assert np.array_equal(self.a_scale.cpu().numpy()[:rows], scale[pair // top_k])

        def product(q, s, w, alpha, d):
            v = R.nvfp4_values(R.unpack(q.cpu().numpy()), s.cpu().numpy())
            got, begin = host(d), 0
            for e, n in enumerate(sizes):
                f = float(alpha[e])
                want, size = f * (v[begin:begin + n] @ w[e].T), f * (np.abs(v[begin:begin + n]) @ np.abs(w[e]).T)
                bound = (w.shape[2] // 16 + 4) * 2.0 ** -22 * size + 1.01 * 2.0 ** -8 * np.abs(want)
                assert (np.abs(got[begin:begin + n] - want) <= bound).all()
                begin += n

        product(self.a, self.a_scale, self.w[0][2], self.alpha[0], self.c)
        # the quantised SwiGLU: a value differs from the exact one by at most half of its code's interval (1 in units of
        # scale * tensor scale, at the top of the grid) and by what a scale rounded down cuts off (6 / 16); what lies above
        # the tensor scale's range becomes its end, the scale 448 times the code 6 (the definition's two minima)
        c = host(self.c)[:rows]
        s = c[:, :inner] / (1 + np.exp(-c[:, :inner])) * c[:, inner:]
        unit = self.h_scale.item()
        h_scale = self.h_scales.cpu().numpy()[:rows]
        got = R.nvfp4_values(R.unpack(self.h.cpu().numpy()[:rows]), h_scale) * unit
        step = np.repeat(np.maximum(R.scale_values(h_scale), 2.0 ** -9), 16, 1) * unit
        s = np.clip(s, -2688 * unit, 2688 * unit)
        assert (np.abs(got - s) <= 1.4 * step).all()
        product(self.h, self.h_scales, self.w[1][2], self.alpha[1], self.d)
        d = host(self.d)
        want = host(shared)
        size = np.abs(want)
        for j in range(top_k):
            term = weights[:, j, None] * d[position[:, j]]
            want, size = want + term, size + np.abs(term)
        bound = (top_k + 1) * 2.0 ** -24 * size * 1.01 + 1.01 * 2.0 ** -8 * np.abs(want)
        assert (np.abs(host(self.out) - want) <= bound).all()


@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(1, 256, 128, 8, 2), (16, 512, 256, 16, 4), (300, 320, 192, 12, 3),
                                                               (700, 256, 256, 4, 2)])
def test_nvfp4_expert_layer(cuda, tokens, hidden, inner, experts, top_k):
    import torch
    from catlass_b200 import capi
    layer = Nvfp4Layer(torch, capi, cuda, tokens, hidden, inner, experts, top_k, tokens)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    new = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    x, shared = new(tokens, hidden).to(torch.bfloat16), new(tokens, hidden).to(torch.bfloat16)
    logits, bias = new(tokens, experts), 0.1 * new(experts)
    layer.run(x, logits, bias, shared)
    torch.cuda.synchronize()
    layer.check(x, logits, bias, shared)
    # captured, and replayed with other tokens
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.run(x, logits, bias, shared)
    for _ in range(2):
        x.copy_(new(tokens, hidden))
        logits.copy_(new(tokens, experts) + 2 * new(1, experts))
        graph.replay()
        torch.cuda.synchronize()
        layer.check(x, logits, bias, shared)
    assert capi.device_status()[0] == 0


def test_int8_expert_layer(cuda):
    """route, dispatch to int8 rows, the grouped W8A8 matmul, combine: bit for bit up to the combine."""
    import torch
    from catlass_b200 import capi
    tokens, k, n, experts, top_k = 200, 256, 384, 10, 3
    rng = np.random.default_rng(9)
    x = torch.from_numpy(rng.standard_normal((tokens, k)).astype(np.float32)).to(cuda).to(torch.bfloat16)
    logits = torch.from_numpy(rng.standard_normal((tokens, experts)).astype(np.float32)).to(cuda)
    b = rng.integers(-127, 128, (experts, k, n), dtype=np.int8)
    scale = rng.uniform(1e-3, 1e-2, (experts, n)).astype(np.float32)
    rows = tokens * top_k
    weights = torch.empty((tokens, top_k), device=cuda)
    ids = torch.empty((tokens, top_k), dtype=torch.int32, device=cuda)
    position, group_list = torch.empty_like(ids), torch.empty((experts,), dtype=torch.int64, device=cuda)
    q, s = torch.empty((rows, k), dtype=torch.int8, device=cuda), torch.empty((rows,), device=cuda)
    d = torch.empty((rows, n), dtype=torch.bfloat16, device=cuda)
    out = torch.empty((tokens, n), dtype=torch.bfloat16, device=cuda)
    capi.moe_route(logits, weights, ids, tokens, experts, top_k)
    capi.moe_dispatch(x, ids, weights, group_list, position, tokens, experts, top_k, k, capi.DISPATCH_INT8, q=q, scale=s,
                      workspace=u8(torch, cuda, max(256, capi.moe_dispatch_workspace_size(tokens, experts, top_k))))
    capi.grouped_quant_matmul(q, torch.from_numpy(b).to(cuda), group_list, torch.from_numpy(scale).to(cuda), s, d, rows, n, k,
                              experts, layout_b=capi.ROW_MAJOR)
    capi.moe_combine(d, position, weights, out, tokens, n, top_k)
    torch.cuda.synchronize()
    want_ids, want_w = R.route(logits.double().cpu().numpy(), top_k, False, renormalize=True)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    sizes, want_position, pair = R.dispatch(want_ids, experts)
    want_q, want_s = O.quantize_per_token_int8(x.float().cpu().numpy())
    want_d = O.bf16_bits(O.grouped_quant_matmul(want_q[pair // top_k], b, np.cumsum(sizes), scale, want_s[pair // top_k], rows, n,
                                                k, O.ROW_MAJOR))
    assert np.array_equal(d.view(torch.int16).cpu().numpy().view(np.uint16), want_d)
    values, w = d.double().cpu().numpy(), weights.double().cpu().numpy()
    terms = [w[:, j, None] * values[want_position[:, j]] for j in range(top_k)]
    want = sum(terms)
    bound = 1.01 * (top_k * 2.0 ** -24 * sum(np.abs(t) for t in terms) + 2.0 ** -8 * np.abs(want))
    assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()


def test_mx_expert_layer_and_both_ways_back(cuda):
    """dispatch to MX rows feeds the fused matmul + SwiGLU + quantisation; its result goes back to the tokens through the
    fused finalize routing and through a plain grouped matmul and combine: the same sums, up to their fp32 roundings."""
    import torch
    from catlass_b200 import capi
    tokens, k, inner, experts, top_k = 150, 256, 128, 6, 2
    rng = np.random.default_rng(12)
    dev = lambda v: torch.from_numpy(np.ascontiguousarray(v)).to(cuda)  # noqa: E731
    x = dev(rng.standard_normal((tokens, k)).astype(np.float32)).to(torch.bfloat16)
    w1 = [O.mx_quantize(rng.standard_normal((2 * inner, k)).astype(np.float32), O.MX_E4M3) for _ in range(experts)]
    w2 = [O.mx_quantize(rng.standard_normal((k, inner)).astype(np.float32), O.MX_E4M3) for _ in range(experts)]
    logits = dev(rng.standard_normal((tokens, experts)).astype(np.float32))
    rows = tokens * top_k
    weights, ids = torch.empty((tokens, top_k), device=cuda), torch.empty((tokens, top_k), dtype=torch.int32, device=cuda)
    position, group_list = torch.empty_like(ids), torch.empty((experts,), dtype=torch.int32, device=cuda)
    row_index, row_weight = torch.empty((rows,), dtype=torch.int64, device=cuda), torch.empty((rows,), device=cuda)
    q, s = u8(torch, cuda, rows, k), u8(torch, cuda, rows, k // 32)
    capi.moe_route(logits, weights, ids, tokens, experts, top_k)
    capi.moe_dispatch(x, ids, weights, group_list, position, tokens, experts, top_k, k, capi.DISPATCH_MX_E4M3, q=q, scale=s,
                      row_index=row_index, row_weight=row_weight, group_list_type=capi.GROUP_LIST_INT32,
                      group_list_kind=capi.GROUP_LIST_SIZES, row_index_type=capi.GROUP_LIST_INT64)
    h, hs = u8(torch, cuda, rows, inner), u8(torch, cuda, rows, inner // 32)
    stack = lambda ws: (dev(np.stack([v for v, _ in ws])), dev(np.stack([v for _, v in ws])))  # noqa: E731
    (b1, sb1), (b2, sb2) = stack(w1), stack(w2)
    lists = dict(group_list_type=capi.GROUP_LIST_INT32, group_list_kind=capi.GROUP_LIST_SIZES)
    capi.mx_grouped_swiglu_quant(q, b1, group_list, s, sb1, h, hs, rows, 2 * inner, k, experts,
                                 u8(torch, cuda, capi.mx_grouped_swiglu_quant_workspace_size(rows, 2 * inner, k, experts)),
                                 **lists)
    fused = torch.empty((tokens, k), device=cuda)
    capi.mx_grouped_finalize_routing(
        h, b2, group_list, hs, sb2, row_weight, row_index, fused, rows, k, inner, experts, tokens,
        u8(torch, cuda, capi.mx_grouped_finalize_routing_workspace_size(rows, k, inner, experts, tokens, deterministic=True)),
        row_index_type=capi.GROUP_LIST_INT64, deterministic=True, **lists)
    d, out = torch.empty((rows, k), device=cuda), torch.empty((tokens, k), device=cuda)
    capi.mx_grouped_matmul(h, b2, group_list, hs, sb2, d, rows, k, inner, experts, capi.MX_E4M3,
                           u8(torch, cuda, capi.mx_grouped_matmul_workspace_size(rows, k, inner, experts, capi.MX_E4M3)),
                           out_f32=True, **lists)
    capi.moe_combine(d, position, weights, out, tokens, k, top_k, d_type=capi.DTYPE_F32, out_type=capi.DTYPE_F32)
    torch.cuda.synchronize()
    assert capi.device_status()[0] == 0
    sizes, want_position, pair = R.dispatch(ids.cpu().numpy(), experts)
    assert np.array_equal(group_list.cpu().numpy(), sizes)
    assert np.array_equal(row_index.cpu().numpy(), pair // top_k)
    want_q, want_s = O.mx_quantize(x.float().cpu().numpy(), O.MX_E4M3)
    assert np.array_equal(q.cpu().numpy(), want_q[pair // top_k]) and np.array_equal(s.cpu().numpy(), want_s[pair // top_k])
    size = sum(np.abs(weights.double().cpu().numpy()[:, j, None] * d.double().cpu().numpy()[want_position[:, j]])
               for j in range(top_k))
    # two products and their sum on either side, each rounded by 2^-24
    assert (np.abs(fused.double().cpu().numpy() - out.double().cpu().numpy()) <= 4 * top_k * 2.0 ** -24 * size + 1e-30).all()
