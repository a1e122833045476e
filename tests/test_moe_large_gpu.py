"""Offsets that pass 32 bits: rows, codes and outputs behind the first 2^32 elements."""
import numpy as np
import pytest

import moe_reference as R

pytestmark = pytest.mark.gpu


def room(torch, gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip("needs more free device memory")


def test_combine_reads_rows_behind_4g_elements(cuda):
    import torch
    from catlass_b200 import capi
    room(torch, 12)
    rows, n = 66000, 65600                                  # 4.33e9 bf16 elements
    d = torch.empty((rows, n), dtype=torch.bfloat16, device=cuda)
    for r in (0, 1, rows - 1):
        d[r] = r % 97 + 1
    position = torch.tensor([[rows - 1, 0], [1, rows - 1], [rows, -1]], dtype=torch.int32, device=cuda)
    w = torch.tensor([[1.0, 2.0], [0.5, 0.25], [1.0, 1.0]], device=cuda)
    out = torch.empty((3, n), device=cuda)
    capi.moe_combine(d, position, w, out, 3, n, 2, rows=rows, out_type=capi.DTYPE_F32)
    last = (rows - 1) % 97 + 1
    for t, want in enumerate((last + 2.0, 1.0 + last / 4, 0.0)):
        assert (out[t] == want).all()


@pytest.mark.parametrize("tiled", [False, True])
def test_quantize_behind_4g_elements(cuda, tiled):
    import torch
    from catlass_b200 import capi
    room(torch, 16)
    rows, k = 66000, 65536 + 64
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device=cuda)
    tail = torch.randn((3, k), device=cuda).to(torch.bfloat16)
    x[-3:] = tail
    q = torch.empty((rows, k // 2), dtype=torch.uint8, device=cuda)
    scale = torch.empty((capi.nvfp4_tiled_scale_bytes(rows, k) if tiled else rows * (k // 16),), dtype=torch.uint8, device=cuda)
    capi.nvfp4_quantize(x, q, scale, rows, k, torch.tensor([0.002], device=cuda), scale_layout=int(tiled))
    codes, want = R.nvfp4_quantize(tail.float().cpu().numpy(), np.float32(0.002))
    assert np.array_equal(q[-3:].cpu().numpy(), R.pack(codes))
    if tiled:
        got = R.untile_scales(scale[-(k // 64) * 512:].cpu().numpy(), 128, k // 16)[0]
        last = rows % 128 or 128
        assert np.array_equal(got[last - 3:last], want)
    else:
        assert np.array_equal(scale.view(rows, k // 16)[-3:].cpu().numpy(), want)
    assert not q[:5].any()


def test_matmul_writes_behind_4g_elements(cuda):
    import torch
    from catlass_b200 import capi
    room(torch, 14)
    m, n, k = 66000, 65600, 32
    rng = np.random.default_rng(0)
    ca, cb = (rng.integers(0, 16, (r, k)).astype(np.uint8) for r in (m, n))
    one = lambda r: torch.full((r, k // 16), 0x38, dtype=torch.uint8, device=cuda)  # noqa: E731  (a scale of 1)
    a, b = (torch.from_numpy(R.pack(c)).to(cuda) for c in (ca, cb))
    d = torch.empty((m, n), dtype=torch.bfloat16, device=cuda)
    ws = torch.empty((capi.nvfp4_matmul_workspace_size(m, n, k),), dtype=torch.uint8, device=cuda)
    capi.nvfp4_matmul(a, b, one(m), one(n), d, m, n, k, ws)
    assert capi.device_status()[0] == 0
    for r in (0, 65535, m - 1):
        want = torch.from_numpy(R.code_values(ca[r]) @ R.code_values(cb).T).to(torch.bfloat16)  # (exact: sums of quarters)
        assert torch.equal(d[r].cpu(), want)
