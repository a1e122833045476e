"""cb200_nvfp4_quantize against the plain definition: codes and scales bit for bit, both scale layouts."""
import numpy as np
import pytest

import moe_reference as R

pytestmark = pytest.mark.gpu


def quantize(torch, capi, x, g, rows, k, tiled=False, **kw):
    dev = x.device
    q = torch.full((rows, k // 2), 0x55, dtype=torch.uint8, device=dev)
    n = capi.nvfp4_tiled_scale_bytes(rows, k) if tiled else rows * (k // 16)
    scale = torch.full((n,), 0x55, dtype=torch.uint8, device=dev)
    code = {torch.float32: capi.DTYPE_F32, torch.bfloat16: capi.DTYPE_BF16, torch.float16: capi.DTYPE_F16}[x.dtype]
    capi.nvfp4_quantize(x, q, scale, rows, k, torch.tensor([g], dtype=torch.float32, device=dev), x_type=code,
                        scale_layout=capi.NVFP4_SCALES_TILED if tiled else capi.NVFP4_SCALES_ROWS, **kw)
    torch.cuda.synchronize()
    return q.cpu().numpy(), scale.cpu().numpy()


def read_scales(scale, rows, k, tiled):
    if not tiled:
        return scale.reshape(rows, k // 16)
    s, padding = R.untile_scales(scale, rows, k // 16)
    assert not padding.any()
    return s


@pytest.mark.parametrize("rows,k,pitch", [(1, 16, 0), (3, 48, 0), (7, 64, 80), (128, 1024, 0), (129, 80, 0), (300, 7168, 0),
                                          (33, 4112, 4128), (2, 65536, 0), (1500, 16, 0)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("tiled", [False, True])
def test_quantize_matches_the_definition(cuda, rows, k, pitch, dtype, tiled):
    import torch
    from catlass_b200 import capi
    rng = np.random.default_rng(rows + k)
    x = (rng.standard_normal((rows, pitch or k)) * np.exp(rng.standard_normal((rows, 1)))).astype(np.float32)
    x[0, :16] = 0.0
    x[-1, -1] = 40.0
    xd = torch.from_numpy(x).to(cuda).to(getattr(torch, dtype))
    x = xd.float().cpu().numpy()[:, :k]
    for g in (np.abs(x).max() / 2688, 0.37):
        q, scale = quantize(torch, capi, xd, g, rows, k, tiled, x_pitch=pitch)
        codes, want = R.nvfp4_quantize(x, np.float32(g))
        assert np.array_equal(read_scales(scale, rows, k, tiled), want)
        assert np.array_equal(R.unpack(q), codes)


def test_quantize_every_border(cuda):
    """Every half-way point of the codes, and the values next to it, with scales that are powers of two."""
    import torch
    from catlass_b200 import capi
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    vals = np.concatenate([borders, np.nextafter(borders, 0, dtype=np.float32), np.nextafter(borders, 9, dtype=np.float32),
                           R.E2M1.astype(np.float32)])
    vals = np.concatenate([vals, -vals])
    x = np.zeros((vals.size, 16), np.float32)
    x[:, 0] = 6.0
    x[:, 5] = vals
    for shift in (0, 3, -5):
        q, scale = quantize(torch, capi, torch.from_numpy(x * 2.0 ** shift).to(cuda), 2.0 ** -4, vals.size, 16)
        codes, want = R.nvfp4_quantize(x * np.float32(2.0 ** shift), np.float32(2.0 ** -4))
        assert np.array_equal(scale.reshape(want.shape), want) and np.array_equal(R.unpack(q), codes)
        ties = R.code_values(R.unpack(q))[:7, 5]
        assert list(ties) == [0, 1, 1, 2, 2, 4, 4]


def test_quantize_extremes(cuda):
    """Blocks that saturate or vanish, denormals, Inf and NaN."""
    import torch
    from catlass_b200 import capi
    inf, nan = np.inf, np.nan
    x = np.ones((10, 32), np.float32)
    x[0, 3], x[1, 4], x[2, 5] = nan, inf, -inf
    x[3] = 1e30
    x[4] = 1e-30
    x[5] = 1e-42
    x[6, ::2] = -0.0
    x[6, 1::2] = 0.0
    x[7, :16] = np.linspace(-9000, 9000, 16)
    x[8] = np.finfo(np.float32).max
    x[9] = 2.0 ** -10 * 6 * 0.5           # a scale half-way to the smallest one
    for g in (0.5, 1e-20, 1e20, np.float32(2.0 ** -126)):
        q, scale = quantize(torch, capi, torch.from_numpy(x).to(cuda), g, 10, 32)
        codes, want = R.nvfp4_quantize(x, np.float32(g))
        assert np.array_equal(scale.reshape(10, 2), want), g
        assert np.array_equal(R.unpack(q), codes), g
    assert (want[:3, 0] == 0x7F).all()


def test_quantize_every_scale(cuda):
    """Blocks whose scale runs through all E4M3 values and the half-way points between them."""
    import torch
    from catlass_b200 import capi
    v = R.e4m3_values()
    t = np.concatenate([v, (v[1:] + v[:-1]) / 2]).astype(np.float32)
    t = np.concatenate([t, np.nextafter(t, np.float32(0)), np.nextafter(t, np.float32(1000))])
    x = np.zeros((t.size, 16), np.float32)
    x[:, 7] = t * 6
    q, scale = quantize(torch, capi, torch.from_numpy(x).to(cuda), 1.0, t.size, 16)
    codes, want = R.nvfp4_quantize(x, np.float32(1.0))
    assert np.array_equal(scale.reshape(-1, 1), want) and np.array_equal(R.unpack(q), codes)


@pytest.mark.parametrize("rows,k,dtype,tiled", [(5, 16, "float32", False), (130, 2048, "bfloat16", True),
                                                (64, 80, "float16", False)])
def test_quantize_swiglu(cuda, rows, k, dtype, tiled):
    """act / (1 + exp(-act)) * gate in fp32.  expf, the sum, the quotient and the product are each off by at most a few
    units in the last place, 2^-20 in all; a scale or a code may therefore be the neighbour where the exact value lies
    within that distance (with a margin: 2^-18) of a half-way point, and nowhere else."""
    import torch
    from catlass_b200 import capi
    rng = np.random.default_rng(k)
    x = (3 * rng.standard_normal((rows, 2 * k))).astype(np.float32)
    xd = torch.from_numpy(x).to(cuda).to(getattr(torch, dtype))
    x = xd.double().cpu().numpy()
    s = x[:, :k] / (1 + np.exp(-x[:, :k])) * x[:, k:]
    g = np.float32(np.abs(s).max() / 2688)
    q, scale = quantize(torch, capi, xd, g, rows, k, tiled, swiglu=True)
    scale = read_scales(scale, rows, k, tiled)
    ratio = np.abs(s).reshape(rows, k // 16, 16).max(2) / (6 * np.float64(g))
    low, high = (R.nearest_even(np.minimum(ratio * (1 + d), 448), R.e4m3_values()) for d in (-2.0 ** -18, 2.0 ** -18))
    assert ((scale == low) | (scale == high)).all()
    step = np.repeat(R.scale_values(scale) * np.float64(g), 16, 1)
    y = np.divide(np.abs(s), step, out=np.zeros_like(s), where=step > 0)
    codes = R.unpack(q)
    low, high = (R.nearest_even(y * (1 + d), R.E2M1) for d in (-2.0 ** -18, 2.0 ** -18))
    assert (((codes & 7) == low) | ((codes & 7) == high)).all()
    assert ((codes >> 3 == np.signbit(s)) | ((codes & 7) == 0)).all()


def test_quantize_row_count(cuda):
    """Rows at or beyond the device-side count stay as they were."""
    import torch
    from catlass_b200 import capi
    x = torch.randn((40, 64), device=cuda)
    codes, _ = R.nvfp4_quantize(x.cpu().numpy(), np.float32(0.01))
    for dtype, code in ((torch.int64, capi.GROUP_LIST_INT64), (torch.int32, capi.GROUP_LIST_INT32)):
        for n, filled in ((-5, 0), (0, 0), (17, 17), (40, 40), (1 << 30, 40)):
            count = torch.tensor([1, n], dtype=dtype, device=cuda)
            q, _ = quantize(torch, capi, x, 0.01, 40, 64, row_count=count[1:], row_count_type=code)
            assert np.array_equal(q[:filled], R.pack(codes)[:filled]) and (q[filled:] == 0x55).all()


def test_quantize_short_buffers(cuda):
    import torch
    from catlass_b200 import capi
    x, g = torch.zeros((4, 64), device=cuda), torch.ones((1,), device=cuda)
    q, s = (torch.zeros((n,), dtype=torch.uint8, device=cuda) for n in (4 * 32, 16))
    for kw in (dict(rows=5, k=64), dict(rows=4, k=80), dict(rows=4, k=64, swiglu=True), dict(rows=4, k=64, x_pitch=80),
               dict(rows=4, k=64, scale_layout=capi.NVFP4_SCALES_TILED)):
        with pytest.raises(ValueError):
            capi.nvfp4_quantize(x, q, s, tensor_scale=g, x_type=capi.DTYPE_F32, **kw)
