"""cb200_nvfp4_matmul and its grouped form against the product in 64 bits.

Bound: the products of codes and scales are exact in fp32; what rounds is their sum.  The tensor core adds K in
blocks into an fp32 accumulator; each addition may lose two bits more than one fp32 rounding (2^-22 of the sum of
magnitudes S so far), and there are at most K/16 of them per output; alpha rounds once and the output by half a step of
its type."""
import numpy as np
import pytest

import moe_reference as R

pytestmark = pytest.mark.gpu

STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
CODE = {"float32": 0, "bfloat16": 1, "float16": 2}


def operand(rng, rows, k):
    """Codes, scale bytes and values; scales over the whole range of a trained tensor, some zero."""
    codes = rng.integers(0, 16, (rows, k)).astype(np.uint8)
    scale = np.clip(rng.normal(0x38, 9, (rows, k // 16)), 0, 0x7E).astype(np.uint8)
    scale[rng.random(scale.shape) < 0.03] = 0
    return codes, scale, R.nvfp4_values(codes, scale)


def close(got, want, size, k, dtype):
    bound = (k // 16 + 4) * 2.0 ** -22 * size + 1.01 * STEP[dtype] * np.abs(want) + (2.0 ** -24 if dtype == "float16" else 1e-37)
    top = 65504.0 if dtype == "float16" else np.inf
    over = np.abs(want) > top * 0.999
    bad = (np.abs(got - want) > bound) & ~over
    return not bad.any() and (np.abs(got[over]) >= top * 0.999).all()


def to(cuda, x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(cuda)


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 32), (1, 16, 64), (7, 130, 96), (16, 1024, 4096), (16, 40, 8192), (33, 300, 544), (100, 520, 1056), (128, 256, 512),
    (129, 257, 288), (300, 1000, 1056), (257, 520, 2080), (512, 512, 256), (1000, 776, 7168), (130, 64, 32), (1025, 2312, 416),
])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32", "float16"])
def test_matmul_matches_the_product(cuda, m, n, k, dtype):
    import torch
    from catlass_b200 import capi
    rng = np.random.default_rng(m * 31 + n * 7 + k)
    ca, sa, va = operand(rng, m, k)
    cb, sb, vb = operand(rng, n, k)
    alpha = np.float32(0.37)
    want = np.float64(alpha) * (va @ vb.T)
    size = np.float64(alpha) * (np.abs(va) @ np.abs(vb).T)
    a, b = to(cuda, R.pack(ca)), to(cuda, R.pack(cb))
    al = torch.tensor([alpha], device=cuda)
    for la in (0, 1):
        for lb in (0, 1):
            if k > 4096 and la != lb:
                continue
            d = torch.full((m, n), 7.0, dtype=getattr(torch, dtype), device=cuda)
            ws_bytes = capi.nvfp4_matmul_workspace_size(m, n, k, la, lb)
            assert (ws_bytes == 0) == (la == 1 and lb == 1)
            ws = torch.empty((max(ws_bytes, 1),), dtype=torch.uint8, device=cuda)
            capi.nvfp4_matmul(a, b, to(cuda, R.tile_scales(sa) if la else sa), to(cuda, R.tile_scales(sb) if lb else sb), d, m, n,
                              k, ws, alpha=al, scale_a_layout=la, scale_b_layout=lb, d_type=CODE[dtype])
            st, code = capi.device_status()
            assert st == 0, hex(code)
            assert close(d.double().cpu().numpy(), want, size, k, dtype), (la, lb)


@pytest.mark.parametrize("m,n,k,block_num", [(16, 512, 2048, 4), (200, 512, 512, 1), (600, 600, 320, 5), (64, 4096, 1024, 0),
                                             (700, 200, 352, 8), (768, 256, 1056, 8)])  # (four tiles of 192 rows)
def test_matmul_without_alpha_on_few_ctas(cuda, m, n, k, block_num):
    import torch
    from catlass_b200 import capi
    rng = np.random.default_rng(k)
    ca, sa, va = operand(rng, m, k)
    cb, sb, vb = operand(rng, n, k)
    outs = []
    for _ in range(2):
        d = torch.empty((m, n), device=cuda)
        capi.nvfp4_matmul(to(cuda, R.pack(ca)), to(cuda, R.pack(cb)), to(cuda, R.tile_scales(sa)), to(cuda, R.tile_scales(sb)), d,
                          m, n, k, scale_a_layout=1, scale_b_layout=1, d_type=0, block_num=block_num)
        outs.append(d)
    assert capi.device_status()[0] == 0
    assert torch.equal(outs[0], outs[1])
    assert close(outs[0].double().cpu().numpy(), va @ vb.T, np.abs(va) @ np.abs(vb).T, k, "float32")


@pytest.mark.parametrize("m", [20, 300])
def test_matmul_spreads_nan_to_its_row_and_column_only(cuda, m):
    import torch
    from catlass_b200 import capi
    rng = np.random.default_rng(m)
    n, k = 200, 96
    ca, sa, va = operand(rng, m, k)
    cb, sb, vb = operand(rng, n, k)
    sa[5, 2] = 0x7F
    sb[130, 5] = 0x7F
    d = torch.empty((m, n), device=cuda)
    ws = torch.empty((capi.nvfp4_matmul_workspace_size(m, n, k, 0, 0),), dtype=torch.uint8, device=cuda)
    capi.nvfp4_matmul(to(cuda, R.pack(ca)), to(cuda, R.pack(cb)), to(cuda, sa), to(cuda, sb), d, m, n, k, ws, d_type=0)
    got = d.double().cpu().numpy()
    bad = np.zeros((m, n), bool)
    bad[5] = bad[:, 130] = True
    assert np.isnan(got[bad]).all()
    assert close(np.where(bad, 0, got), np.where(bad, 0, va @ vb.T), np.abs(va) @ np.abs(vb).T, k, "float32")


def grouped(cuda, sizes, m, n, k, dtype="bfloat16", tiled=False, i32=False, prefix=False, glist=None, seed=0, alpha=True):
    import torch
    from catlass_b200 import capi
    rng = np.random.default_rng(seed + m + n)
    g = len(sizes)
    ca, sa, va = operand(rng, m, k)
    parts = [operand(rng, n, k) for _ in range(g)]
    al = rng.uniform(0.2, 2, g).astype(np.float32) if alpha else np.ones(g, np.float32)
    b = np.stack([R.pack(p[0]) for p in parts])
    sb = np.stack([R.tile_scales(p[1]) if tiled else p[1] for p in parts])
    if glist is None:
        glist = np.cumsum(sizes) if prefix else np.array(sizes)
    d = torch.full((m, n), 7.0, dtype=getattr(torch, dtype), device=cuda)
    ws = torch.empty((capi.nvfp4_grouped_matmul_workspace_size(m, n, k, g, int(tiled)),), dtype=torch.uint8, device=cuda)
    gl = to(cuda, np.asarray(glist).astype(np.int32 if i32 else np.int64))
    capi.nvfp4_grouped_matmul(to(cuda, R.pack(ca)), to(cuda, b), gl, to(cuda, sa), to(cuda, sb), d, m, n, k, g, ws,
                              alpha=to(cuda, al) if alpha else None, scale_b_layout=int(tiled), d_type=CODE[dtype],
                              group_list_type=int(i32), group_list_kind=int(prefix))
    st, code = capi.device_status()
    assert st == 0, hex(code)
    got = d.double().cpu().numpy()
    begin = 0
    for i, rows in enumerate(sizes):
        end = begin + rows
        v, w = va[begin:end], parts[i][2]
        f = np.float64(al[i])
        assert close(got[begin:end], f * (v @ w.T), f * (np.abs(v) @ np.abs(w).T), k, dtype), (i, rows)
        begin = end
    assert (got[begin:] == 7.0).all()


@pytest.mark.parametrize("sizes,m,n,k", [
    ([1], 1, 16, 32), ([3, 0, 5, 1], 9, 136, 96), ([0, 0, 0], 4, 64, 64), ([16, 1, 0, 17, 130], 170, 300, 352),
    ([2] * 40 + [0] * 30 + [7], 90, 256, 512), ([300, 0, 1, 129], 430, 264, 416), ([256, 257, 700], 1300, 520, 288),
    ([1000, 24], 1024, 1000, 256), ([0, 128, 0], 128, 129, 160), ([1] * 1024, 1024, 24, 64),
])
def test_grouped_matmul_matches_the_products(cuda, sizes, m, n, k):
    case = len(sizes) + m
    for j, dtype in enumerate(("bfloat16", "float32")):
        grouped(cuda, sizes, m, n, k, dtype, tiled=(case + j) % 2 == 0, i32=case % 3 == 0, prefix=j == 1, alpha=case % 2 == 0)


def test_grouped_matmul_lists_out_of_range(cuda):
    """Entries past m are clamped, negative sizes are empty, a prefix sum that falls leaves an empty group."""
    grouped(cuda, [10, 30, 0], 40, 64, 64, glist=[10, 1 << 40, 5])
    grouped(cuda, [0, 12, 28], 40, 64, 64, glist=[-4, 12, 99])
    grouped(cuda, [20, 0, 5], 40, 64, 64, prefix=True, glist=[20, 7, 25])
    grouped(cuda, [0, 40, 0], 40, 64, 64, prefix=True, glist=[-1, 1 << 40, -3])
    grouped(cuda, [0, 600, 0], 600, 64, 64, prefix=True, i32=True, glist=[-1, 2147483647, 3])


def test_matmuls_in_a_graph_on_another_stream(cuda):
    """Replays with other operands and other group lists; the eager result of the same call is the same bits."""
    import torch
    from catlass_b200 import capi
    rng = np.random.default_rng(6)
    m, n, k, g = 160, 264, 320, 5
    codes = [R.pack(operand(rng, m, k)[0]) for _ in range(3)]
    sa, sb = to(cuda, operand(rng, m, k)[1]), to(cuda, np.stack([operand(rng, n, k)[1] for _ in range(g)]))
    b = to(cuda, np.stack([R.pack(operand(rng, n, k)[0]) for _ in range(g)]))
    a = to(cuda, codes[0])
    lists = [[32, 32, 32, 32, 32], [0, 160, 0, 0, 0], [1, 2, 3, 4, 100]]
    gl = torch.tensor(lists[0], device=cuda)
    d, dense = torch.zeros((m, n), device=cuda), torch.zeros((m, n), device=cuda)
    ws = torch.empty((capi.nvfp4_grouped_matmul_workspace_size(m, n, k, g, 0),), dtype=torch.uint8, device=cuda)
    ws2 = torch.empty((capi.nvfp4_matmul_workspace_size(m, n, k, 0, 0),), dtype=torch.uint8, device=cuda)

    def both(to_grouped, to_dense):
        capi.nvfp4_grouped_matmul(a, b, gl, sa, sb, to_grouped, m, n, k, g, ws, d_type=0)
        capi.nvfp4_matmul(a, b, sa, sb, to_dense, m, n, k, ws2, d_type=0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        both(d, dense)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            both(d, dense)
        for i in range(3):
            a.copy_(to(cuda, codes[i]))
            gl.copy_(torch.tensor(lists[i], device=cuda))
            d.fill_(7.0)
            want, want_dense = torch.full_like(d, 7.0), torch.zeros_like(dense)
            graph.replay()
            both(want, want_dense)
            torch.cuda.synchronize()
            assert torch.equal(d, want) and torch.equal(dense, want_dense)
    assert capi.device_status()[0] == 0


def test_matmul_refusals(cuda):
    import torch
    from catlass_b200 import capi
    z = lambda n: torch.zeros((n,), dtype=torch.uint8, device=cuda)  # noqa: E731
    d = torch.zeros((8, 64), dtype=torch.bfloat16, device=cuda)
    before = capi.launch_count()
    with pytest.raises(capi.CallError):  # scales by rows need a workspace
        capi.nvfp4_matmul(z(8 * 32), z(64 * 32), z(512), z(512), d, 8, 64, 64)
    with pytest.raises(ValueError):      # tiled scales are larger
        capi.nvfp4_matmul(z(8 * 32), z(64 * 32), z(32), z(512), d, 8, 64, 64, scale_a_layout=1, scale_b_layout=1)
    with pytest.raises(ValueError):
        capi.nvfp4_matmul(z(8 * 32), z(64 * 32), z(512), z(512), d, 9, 64, 64, scale_a_layout=1, scale_b_layout=1)
    with pytest.raises(capi.CallError):  # k % 32
        capi.nvfp4_matmul(z(8 * 32), z(64 * 32), z(512), z(512), d, 8, 64, 48, scale_a_layout=1, scale_b_layout=1)
    with pytest.raises(capi.CallError):  # operands off 16-byte boundaries
        capi.nvfp4_matmul(z(8 * 32 + 8)[8:], z(64 * 32), z(512), z(512), d, 8, 64, 64, scale_a_layout=1, scale_b_layout=1)
    assert capi.launch_count() == before
