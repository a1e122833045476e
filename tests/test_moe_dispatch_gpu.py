"""cb200_moe_dispatch and cb200_moe_combine against their plain definitions: lists and codes bit for bit."""
import numpy as np
import pytest

import moe_reference as R
import oracle_lib as O

pytestmark = pytest.mark.gpu


def routed(rng, tokens, experts, top_k, dropped=0.0):
    """Distinct experts per token, unevenly loaded, some pairs without an expert."""
    load = rng.standard_normal(experts) * 1.5
    ids = np.argsort(-(load + rng.gumbel(size=(tokens, experts))), axis=1)[:, :top_k].astype(np.int32)
    ids[rng.random(ids.shape) < dropped] = -1
    return ids, rng.random((tokens, top_k)).astype(np.float32)


class Outputs:
    def __init__(self, torch, capi, rows, experts, k, fmt, x_dtype, cuda, i32_list, i32_index):
        e = lambda shape, dt: torch.full(shape, 85, dtype=dt, device=cuda)  # noqa: E731
        self.group_list = e((experts,), torch.int32 if i32_list else torch.int64)
        self.row_index = e((rows,), torch.int32 if i32_index else torch.int64)
        self.row_weight = e((rows,), torch.float32)
        self.q = self.scale = None
        if fmt == capi.DISPATCH_COPY:
            self.q = e((rows, k), x_dtype)
        elif fmt == capi.DISPATCH_INT8:
            self.q, self.scale = e((rows, k), torch.int8), e((rows,), torch.float32)
        elif fmt == capi.DISPATCH_MX_E4M3:
            self.q, self.scale = e((rows, k), torch.uint8), e((rows, (k // 32 + 1) // 2 * 2), torch.uint8)
        elif fmt == capi.DISPATCH_NVFP4:
            self.q, self.scale = e((rows, k // 2), torch.uint8), e((rows, k // 16), torch.uint8)


def quantized(capi, x, fmt, tensor_scale):
    """Rows of codes and scales by the formats' definitions (x fp32 [tokens, k])."""
    if fmt == capi.DISPATCH_INT8:
        return O.quantize_per_token_int8(x)
    if fmt == capi.DISPATCH_MX_E4M3:
        q, scale = O.mx_quantize(x, O.MX_E4M3)
        return q, np.pad(scale, ((0, 0), (0, scale.shape[1] % 2)), constant_values=127)  # an even number of columns, 2^0
    codes, scale = R.nvfp4_quantize(x, tensor_scale)
    return R.pack(codes), scale


@pytest.mark.parametrize("tokens,experts,top_k,k,dropped", [
    (1, 1, 1, 32, 0), (1, 8, 8, 64, 0), (16, 64, 8, 4096, 0), (3, 5, 2, 32, 0.5), (128, 256, 8, 96, 0.1),   # one launch
    (129, 256, 8, 160, 0), (300, 64, 6, 1056, 0.2), (513, 1024, 4, 64, 0), (2500, 60, 4, 32, 0.05),        # sorted
    (70, 40, 32, 8224, 0), (40, 33, 32, 64, 1.0),
])
@pytest.mark.parametrize("fmt", ["INDEX", "COPY", "INT8", "MX_E4M3", "NVFP4"])
def test_dispatch_matches_the_definition(cuda, tokens, experts, top_k, k, dropped, fmt):
    import torch
    from catlass_b200 import capi
    fmt = getattr(capi, "DISPATCH_" + fmt)
    rng = np.random.default_rng(tokens * 7 + experts + fmt)
    ids, weights = routed(rng, tokens, experts, top_k, dropped)
    case = tokens + fmt                                   # types and kinds of lists vary from case to case
    dtype = (torch.bfloat16, torch.float32, torch.float16)[case % 3]
    prefix, i32_list, i32_index = case % 2 == 0, case % 4 < 2, case % 3 == 0
    pitch = k + (32 if case % 2 else 0)
    x = rng.standard_normal((tokens, pitch)).astype(np.float32) * rng.uniform(0.01, 20, (tokens, 1)).astype(np.float32)
    x[0, :16] = 0
    xd = torch.from_numpy(x).to(cuda).to(dtype)
    x = xd.float().cpu().numpy()[:, :k]
    g = np.float32(np.abs(x).max() / 2000)
    rows = tokens * top_k
    out = Outputs(torch, capi, rows, experts, k, fmt, dtype, cuda, i32_list, i32_index)
    position = torch.full((tokens, top_k), 85, dtype=torch.int32, device=cuda)
    ws = torch.empty((max(256, capi.moe_dispatch_workspace_size(tokens, experts, top_k)),), dtype=torch.uint8, device=cuda)
    capi.moe_dispatch(
        xd, torch.from_numpy(ids).to(cuda), torch.from_numpy(weights).to(cuda), out.group_list, position, tokens, experts, top_k,
        k, fmt, q=out.q, scale=out.scale, row_index=out.row_index, row_weight=out.row_weight,
        x_type={torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype], x_pitch=pitch if pitch != k else 0,
        tensor_scale=torch.tensor([g], device=cuda), workspace=ws,
        group_list_type=capi.GROUP_LIST_INT32 if i32_list else capi.GROUP_LIST_INT64,
        group_list_kind=capi.GROUP_LIST_PREFIX_SUMS if prefix else capi.GROUP_LIST_SIZES,
        row_index_type=capi.GROUP_LIST_INT32 if i32_index else capi.GROUP_LIST_INT64)
    torch.cuda.synchronize()
    sizes, want_position, pair = R.dispatch(ids, experts)
    n = pair.size
    assert np.array_equal(out.group_list.cpu().numpy(), np.cumsum(sizes) if prefix else sizes)
    assert np.array_equal(position.cpu().numpy(), want_position)
    assert np.array_equal(out.row_index.cpu().numpy()[:n], pair // top_k)
    assert np.array_equal(out.row_weight.cpu().numpy()[:n], weights.reshape(-1)[pair])
    assert (out.row_index[n:] == 85).all() and (out.row_weight[n:] == 85).all()
    if fmt == capi.DISPATCH_COPY:
        assert torch.equal(out.q[:n], xd[:, :k][torch.from_numpy(pair // top_k).to(cuda)])
    elif fmt != capi.DISPATCH_INDEX:
        q, scale = quantized(capi, x, fmt, g)
        assert np.array_equal(out.q.cpu().numpy()[:n], q[pair // top_k])
        assert np.array_equal(out.scale.cpu().numpy()[:n], scale[pair // top_k])
        assert (out.scale[n:] == 85).all()
    if out.q is not None:
        assert (out.q[n:] == 85).all()


def test_dispatch_of_a_shard_and_of_nothing(cuda):
    """expert_begin: only the pairs of experts 16 .. 23; a batch without tokens still writes its group list."""
    import torch
    from catlass_b200 import capi
    rng = np.random.default_rng(2)
    for tokens in (50, 700):
        ids, weights = routed(rng, tokens, 64, 6)
        ids[0, 0] = np.iinfo(np.int32).max
        ids[0, 1] = np.iinfo(np.int32).min
        out = Outputs(torch, capi, tokens * 6, 8, 32, capi.DISPATCH_INDEX, None, cuda, False, True)
        position = torch.empty((tokens, 6), dtype=torch.int32, device=cuda)
        ws = torch.empty((max(256, capi.moe_dispatch_workspace_size(tokens, 8, 6)),), dtype=torch.uint8, device=cuda)
        capi.moe_dispatch(None, torch.from_numpy(ids).to(cuda), torch.from_numpy(weights).to(cuda), out.group_list, position,
                          tokens, 8, 6, 0, capi.DISPATCH_INDEX, row_index=out.row_index, workspace=ws, expert_begin=16)
        sizes, want, pair = R.dispatch(ids, 8, 16)
        assert np.array_equal(out.group_list.cpu().numpy(), np.cumsum(sizes))
        assert np.array_equal(position.cpu().numpy(), want)
        assert np.array_equal(out.row_index.cpu().numpy()[:pair.size], pair // 6)
    empty = torch.empty((0, 6), dtype=torch.int32, device=cuda)
    capi.moe_dispatch(None, empty, None, out.group_list, empty, 0, 8, 6, 0, capi.DISPATCH_INDEX)
    assert (out.group_list == 0).all()


def test_dispatch_in_a_graph_and_back_to_back(cuda):
    """Replays with other routings, and two calls in a row on one stream that share a workspace."""
    import torch
    from catlass_b200 import capi
    rng = np.random.default_rng(4)
    tokens, experts, top_k, k = 600, 32, 4, 64
    x = torch.randn((tokens, k), device=cuda).to(torch.bfloat16)
    ids = torch.zeros((tokens, top_k), dtype=torch.int32, device=cuda)
    weights = torch.rand((tokens, top_k), device=cuda)
    out = [Outputs(torch, capi, tokens * top_k, experts, k, capi.DISPATCH_INT8, None, cuda, False, True) for _ in range(2)]
    position = [torch.empty((tokens, top_k), dtype=torch.int32, device=cuda) for _ in range(2)]
    ws = torch.empty((capi.moe_dispatch_workspace_size(tokens, experts, top_k),), dtype=torch.uint8, device=cuda)
    other = torch.zeros_like(ids)

    def both():
        for i, which in enumerate((ids, other)):
            capi.moe_dispatch(x, which, weights, out[i].group_list, position[i], tokens, experts, top_k, k,
                              capi.DISPATCH_INT8, q=out[i].q, scale=out[i].scale, row_index=out[i].row_index,
                              row_weight=out[i].row_weight, workspace=ws)

    both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    want_q, want_scale = O.quantize_per_token_int8(x.float().cpu().numpy())
    for _ in range(3):
        host = [routed(rng, tokens, experts, top_k)[0] for _ in range(2)]
        ids.copy_(torch.from_numpy(host[0]))
        other.copy_(torch.from_numpy(host[1]))
        graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            sizes, want, pair = R.dispatch(host[i], experts)
            assert np.array_equal(position[i].cpu().numpy(), want)
            assert np.array_equal(out[i].group_list.cpu().numpy(), np.cumsum(sizes))
            assert np.array_equal(out[i].q.cpu().numpy(), want_q[pair // top_k])
            assert np.array_equal(out[i].scale.cpu().numpy(), want_scale[pair // top_k])


def test_dispatch_refusals(cuda):
    import torch
    from catlass_b200 import capi
    ids = torch.zeros((600, 4), dtype=torch.int32, device=cuda)
    position, gl = torch.empty_like(ids), torch.empty((8,), dtype=torch.int64, device=cuda)
    before = capi.launch_count()
    with pytest.raises(capi.CallError):     # no workspace
        capi.moe_dispatch(None, ids, None, gl, position, 600, 8, 4, 0, capi.DISPATCH_INDEX)
    with pytest.raises(ValueError):         # a group list that is too short
        capi.moe_dispatch(None, ids, None, gl[:7], position, 600, 8, 4, 0, capi.DISPATCH_INDEX)
    with pytest.raises(ValueError):
        capi.moe_dispatch(None, ids, None, gl, position, 601, 8, 4, 0, capi.DISPATCH_INDEX)
    assert capi.launch_count() == before


# ---------------------------------------------------------------------------------------------------- combine

@pytest.mark.parametrize("tokens,top_k,n", [(1, 1, 1), (1, 8, 7168), (5, 3, 17), (16, 8, 2056), (33, 32, 130), (70, 9, 4096),
                                            (70000, 1, 8)])
@pytest.mark.parametrize("d_type,out_type", [("bfloat16", "bfloat16"), ("float32", "float32"), ("float16", "float32"),
                                             ("float32", "bfloat16"), ("bfloat16", "float16")])
def test_combine_matches_the_definition(cuda, tokens, top_k, n, d_type, out_type):
    import torch
    from catlass_b200 import capi
    code = {"float32": 0, "bfloat16": 1, "float16": 2}
    rng = np.random.default_rng(tokens + n)
    rows = tokens * top_k
    d = torch.from_numpy(rng.standard_normal((rows, n)).astype(np.float32)).to(cuda).to(getattr(torch, d_type))
    position = rng.permutation(rows).astype(np.int32).reshape(tokens, top_k)
    position[rng.random(position.shape) < 0.2] = -1
    if top_k > 1:
        position[0] = -1                                   # a token without any row
    d[0] = float("nan") if 0 not in position else d[0]     # rows that nobody reads may hold anything
    weights = rng.uniform(-1, 1, (tokens, top_k)).astype(np.float32)
    weights[position < 0] = np.nan                         # ... and weights of skipped slots
    shared = torch.from_numpy(rng.standard_normal((tokens, n)).astype(np.float32)).to(cuda).to(getattr(torch, out_type))
    x = d.double().cpu().numpy()
    for use_shared in (False, True):
        out = torch.full((tokens, n), 9.0, dtype=getattr(torch, out_type), device=cuda)
        capi.moe_combine(d, torch.from_numpy(position).to(cuda), torch.from_numpy(weights).to(cuda), out, tokens, n, top_k,
                         d_type=code[d_type], out_type=code[out_type], shared=shared if use_shared else None,
                         shared_weight=0.75)
        want = 0.75 * shared.double().cpu().numpy() if use_shared else np.zeros((tokens, n))
        size = np.abs(want)                                # sum of magnitudes, for the rounding of the fp32 sums
        for j in range(top_k):
            at = np.flatnonzero(position[:, j] >= 0)
            term = weights[at, j, None].astype(np.float64) * x[position[at, j]]
            want[at] += term
            size[at] += np.abs(term)
        # every fused multiply-add rounds once, by 2^-24 of a partial sum; then the output's half step
        step = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[out_type]
        bound = (top_k + 1) * 2.0 ** -24 * size * 1.01 + step * np.abs(want) * 1.01 + (2.0 ** -25 if out_type == "float16" else 0)
        got = out.double().cpu().numpy()
        assert (np.abs(got - want) <= bound).all()


def test_combine_refuses_and_skips(cuda):
    """Positions past the rows of d are skipped, not read."""
    import torch
    from catlass_b200 import capi
    d = torch.ones((4, 16), device=cuda)
    position = torch.tensor([[0, 4], [2147483647, 3]], dtype=torch.int32, device=cuda)
    w = torch.full((2, 2), 2.0, device=cuda)
    out = torch.empty((2, 16), device=cuda)
    capi.moe_combine(d, position, w, out, 2, 16, 2, rows=4, d_type=0, out_type=0)
    assert (out == 2).all()
    with pytest.raises(ValueError):
        capi.moe_combine(d, position, w, out, 2, 16, 2, rows=5, d_type=0, out_type=0)
    with pytest.raises(ValueError):
        capi.moe_combine(d, position, w, out, 3, 16, 2, rows=4, d_type=0, out_type=0)


def test_int64_ids_are_refused(cuda):
    import torch
    from catlass_b200 import capi
    ids = torch.zeros((16, 2), dtype=torch.int64, device=cuda)
    position, gl = torch.empty((16, 2), dtype=torch.int32, device=cuda), torch.empty((8,), dtype=torch.int64, device=cuda)
    with pytest.raises(ValueError, match="elements of 4 bytes"):
        capi.moe_dispatch(None, ids, None, gl, position, 16, 8, 2, 0, capi.DISPATCH_INDEX)
    x = torch.zeros((16, 64), device=cuda)
    q = torch.empty((32, 64), dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="x must have"):    # fp32 rows under the default type code, bf16
        capi.moe_dispatch(x, ids.to(torch.int32), None, gl, position, 16, 8, 2, 64, capi.DISPATCH_COPY, q=q)


@pytest.mark.parametrize("n", [7, 514, 4096])
def test_combine_onto_the_shared_rows(cuda, n):
    """out may be shared itself: every element is read by the thread that writes it.  Small integers: exact sums."""
    import torch
    from catlass_b200 import capi
    g = torch.Generator(device="cpu").manual_seed(n)
    d = torch.randint(-4, 5, (40, n), generator=g).to(torch.bfloat16).to(cuda)
    shared = torch.randint(-4, 5, (20, n), generator=g).to(torch.bfloat16).to(cuda)
    position = torch.randperm(40, generator=g).view(20, 2).to(torch.int32).to(cuda)
    w = torch.randint(1, 3, (20, 2), generator=g).float().to(cuda)
    want = shared.float() + (w[:, :, None] * d.float()[position.long()]).sum(1)
    capi.moe_combine(d, position, w, shared, 20, n, 2, shared=shared)
    assert torch.equal(shared.float(), want)
