"""Routing, dispatch, combine and the NVFP4 entry points on the host: the argument structs equal the header's, and what
cannot be run is refused before anything is launched."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest

import moe_reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def capi():
    from catlass_b200 import build, capi
    build.build()
    capi.load()
    return capi


def accepted(capi, name, args):
    return capi._function(name + "_can_implement", type(args))(ctypes.byref(args))


def refused(capi, name, args, **changes):
    """Status of the arguments with some fields changed."""
    other = type(args).from_buffer_copy(args)
    for field, value in changes.items():
        setattr(other, field, value)
    return accepted(capi, name, other) == capi.INVALID


def test_struct_layouts(capi):
    pairs = [("cb200_moe_route_args", capi.MoeRouteArgs), ("cb200_moe_dispatch_args", capi.MoeDispatchArgs),
             ("cb200_moe_combine_args", capi.MoeCombineArgs), ("cb200_nvfp4_quantize_args", capi.Nvfp4QuantizeArgs),
             ("cb200_nvfp4_matmul_args", capi.Nvfp4MatmulArgs),
             ("cb200_nvfp4_grouped_matmul_args", capi.Nvfp4GroupedMatmulArgs)]
    lines = []
    for cname, ctype in pairs:
        offsets = ", ".join(f"offsetof({cname}, {f[0]})" for f in ctype._fields_)
        lines.append('  printf("%s\\n", sizeof(%s), %s);' % (" ".join(["%zu"] * (len(ctype._fields_) + 1)), cname, offsets))
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"catlass_b200.h\"\nint main(void) {\n%s\n  return 0; }\n" % \
        "\n".join(lines)
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "t.c"), os.path.join(td, "t")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.strip().splitlines()
    for (cname, ctype), line in zip(pairs, out):
        want = [ctypes.sizeof(ctype)] + [getattr(ctype, f[0]).offset for f in ctype._fields_]
        assert [int(v) for v in line.split()] == want, cname


def test_route_refusals(capi):
    name = "cb200_moe_route"
    ok = capi.MoeRouteArgs(tokens=4, experts=64, top_k=8, score=0, groups=8, groups_kept=2, group_score=1, flags=1,
                           logits_type=0, scaling=1.0, logits=256, weights=256, ids=256)
    assert accepted(capi, name, ok) == capi.SUCCESS
    for change in (dict(experts=0), dict(experts=1025, groups=1, groups_kept=1), dict(top_k=0), dict(top_k=17), dict(top_k=33),
                   dict(groups=7), dict(groups=0), dict(groups=64, groups_kept=64), dict(groups_kept=0), dict(groups_kept=9),
                   dict(score=2), dict(group_score=2), dict(flags=2), dict(logits_type=3), dict(logits_pitch=63),
                   dict(logits=None), dict(logits=257), dict(weights=None), dict(ids=258), dict(bias=2), dict(token_count=1)):
        assert refused(capi, name, ok, **change), change
    assert not refused(capi, name, ok, tokens=0, logits=None, weights=None, ids=None)
    assert capi._function(name, type(ok))(None, None) == capi.INVALID


def test_dispatch_refusals(capi):
    name = "cb200_moe_dispatch"
    ok = capi.MoeDispatchArgs(tokens=4, experts=64, top_k=8, k=64, format=capi.DISPATCH_NVFP4, x_type=1, x=256, ids=256,
                              weights=256, tensor_scale=256, q=256, scale=256, group_list=256, position=256, row_index=256,
                              row_weight=256)
    assert accepted(capi, name, ok) == capi.SUCCESS
    for change in (dict(experts=0), dict(experts=1025), dict(top_k=0), dict(top_k=33), dict(format=5), dict(x_type=3), dict(k=24),
                   dict(x=None), dict(x=264), dict(q=None), dict(q=264), dict(scale=None), dict(tensor_scale=None),
                   dict(ids=None), dict(position=None), dict(weights=None), dict(group_list=None), dict(group_list=260),
                   dict(group_list_type=2), dict(group_list_kind=2), dict(row_index_type=2), dict(row_index=260),
                   dict(x_pitch=48), dict(x_pitch=68), dict(tokens=1 << 21), dict(format=capi.DISPATCH_MX_E4M3, k=48),
                   dict(format=capi.DISPATCH_INT8, k=8), dict(format=capi.DISPATCH_INT8, scale=258),
                   dict(format=capi.DISPATCH_COPY, k=12, x_pitch=16)):
        assert refused(capi, name, ok, **change), change
    assert not refused(capi, name, ok, weights=None, row_weight=None, row_index=None)
    assert not refused(capi, name, ok, format=capi.DISPATCH_INDEX, x=None, q=None, scale=None, tensor_scale=None)
    assert not refused(capi, name, ok, tokens=0, ids=None, position=None)
    # few pairs need no workspace, many need the counts of 128 chunks at most
    assert capi.moe_dispatch_workspace_size(16, 64, 8) == 0
    assert 0 < capi.moe_dispatch_workspace_size(1 << 20, 256, 8) <= 128 * 256 * 4
    assert capi._function(name, type(ok))(None, None) == capi.INVALID


def test_combine_refusals(capi):
    name = "cb200_moe_combine"
    ok = capi.MoeCombineArgs(tokens=4, top_k=8, n=64, rows=32, d_type=1, out_type=1, d=256, position=256, weights=256, out=256)
    assert accepted(capi, name, ok) == capi.SUCCESS
    for change in (dict(top_k=0), dict(top_k=33), dict(d_type=3), dict(out_type=3), dict(reserved=1), dict(d=None), dict(d=257),
                   dict(position=None), dict(position=258), dict(weights=None), dict(weights=258), dict(out=None),
                   dict(out=257), dict(shared=257), dict(out_type=0, out=258)):
        assert refused(capi, name, ok, **change), change
    assert not refused(capi, name, ok, rows=0, d=None)
    assert not refused(capi, name, ok, tokens=0, position=None, weights=None, out=None)


def test_nvfp4_quantize_refusals(capi):
    name = "cb200_nvfp4_quantize"
    ok = capi.Nvfp4QuantizeArgs(rows=4, k=64, x_type=1, x=256, tensor_scale=256, q=256, scale=256)
    assert accepted(capi, name, ok) == capi.SUCCESS
    for change in (dict(k=24), dict(x_type=3), dict(scale_layout=2), dict(flags=2), dict(row_count_type=2), dict(x=None),
                   dict(x=264), dict(tensor_scale=None), dict(q=None), dict(q=260), dict(scale=None), dict(x_pitch=48),
                   dict(x_pitch=68), dict(flags=1, x_pitch=64), dict(row_count=260), dict(tensor_scale=258)):
        assert refused(capi, name, ok, **change), change
    assert not refused(capi, name, ok, rows=0, x=None, q=None)
    assert capi.nvfp4_tiled_scale_bytes(129, 80) == 2 * 2 * 512
    lib_bytes = capi._function("cb200_nvfp4_tiled_scale_bytes", capi.MoeRouteArgs, ctypes.c_uint64)
    lib_bytes.argtypes = [ctypes.c_uint32, ctypes.c_uint32]
    for rows, k in ((0, 64), (1, 16), (128, 64), (129, 80), (1 << 20, 7168)):
        assert lib_bytes(rows, k) == capi.nvfp4_tiled_scale_bytes(rows, k)


def test_nvfp4_matmul_refusals(capi):
    dense = capi.Nvfp4MatmulArgs(m=16, n=64, k=64, d_type=1, a=256, b=256, scale_a=256, scale_b=256, d=256)
    groups = capi.Nvfp4GroupedMatmulArgs(m=16, n=64, k=64, group_count=4, d_type=1, a=256, b=256, group_list=256, scale_a=256,
                                         scale_b=256, d=256)
    for name, ok in (("cb200_nvfp4_matmul", dense), ("cb200_nvfp4_grouped_matmul_slice_m", groups)):
        assert accepted(capi, name, ok) == capi.SUCCESS
        for change in (dict(k=0), dict(k=48), dict(d_type=3), dict(scale_b_layout=2), dict(flags=1), dict(a=None), dict(a=264),
                       dict(b=None), dict(b=264), dict(scale_a=None), dict(scale_a=264), dict(scale_b=None), dict(d=None),
                       dict(d=264), dict(d=257, n=65), dict(alpha=258), dict(m=1 << 31)):
            assert refused(capi, name, ok, **change), (name, change)
        assert not refused(capi, name, ok, m=0, a=None, d=None)
        assert not refused(capi, name, ok, n=65, d=258)
        assert capi._function(name, type(ok))(None, None) == capi.INVALID
    assert refused(capi, "cb200_nvfp4_matmul", dense, scale_a_layout=2)
    for change in (dict(group_count=0), dict(group_count=1025), dict(group_list=None), dict(group_list=260),
                   dict(group_list_type=2), dict(group_list_kind=2)):
        assert refused(capi, "cb200_nvfp4_grouped_matmul_slice_m", groups, **change), change
    # only scales by rows, and row tables, need a workspace
    assert capi.nvfp4_matmul_workspace_size(4096, 4096, 4096, 1, 1) == 0
    assert capi.nvfp4_matmul_workspace_size(128, 256, 4096, 0, 1) == capi.nvfp4_tiled_scale_bytes(128, 4096)
    assert capi.nvfp4_matmul_workspace_size(16, 256, 4096, 1, 0) == capi.nvfp4_tiled_scale_bytes(256, 4096)
    assert capi.nvfp4_grouped_matmul_workspace_size(256, 4096, 7168, 64, 1) > 0


CPP = r"""
#include <cstdio>
#include "catlass_b200/device_gemm.hpp"
using namespace Catlass;
int main() {
    using Dense = Gemm::Device::DeviceGemm<Gemm::Kernel::Nvfp4Matmul>;
    using Grouped = Gemm::Device::DeviceGemm<Gemm::Kernel::GroupedNvfp4MatmulSliceM<int32_t>>;
    auto p = reinterpret_cast<uint8_t*>(256);
    Gemm::Kernel::Nvfp4Matmul::Arguments a;
    a.problemShape = GemmCoord{128, 256, 4096};
    a.ptrA = a.ptrB = a.ptrScaleA = a.ptrScaleB = a.ptrD = p;
    a.scaleLayoutB = CB200_NVFP4_SCALES_TILED;
    Gemm::Kernel::GroupedNvfp4MatmulSliceM<int32_t>::Arguments g;
    g.problemShape = GemmCoord{128, 256, 4096};
    g.problemCount = 4;
    g.ptrGroupList = g.ptrA = g.ptrB = g.ptrScaleA = g.ptrScaleB = g.ptrD = p;
    bool ok = Dense::CanImplement(a) == Status::kSuccess && Grouped::CanImplement(g) == Status::kSuccess;
    g.ptrGroupList = reinterpret_cast<uint8_t*>(260);   // aligned for int32, not for int64
    ok = ok && Grouped::CanImplement(g) == Status::kSuccess;
    size_t dense = Dense::GetWorkspaceSize(a);
    a.problemShape = GemmCoord{128, 256, 40};
    ok = ok && Dense::CanImplement(a) == Status::kInvalid;
    std::printf("%d %zu\n", ok ? 1 : 0, dense);
    return 0;
}
"""


def test_cpp_descriptors(capi):
    """The C++ descriptors of the NVFP4 matmuls compile, link and hand their members on."""
    lib = capi.library_path()
    with tempfile.TemporaryDirectory() as td:
        src, exe = os.path.join(td, "t.cpp"), os.path.join(td, "t")
        open(src, "w").write(CPP)
        subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "include"), src, "-o", exe, lib,
                        "-Wl,-rpath," + os.path.dirname(lib)], check=True)
        out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()
    assert out == ["1", str(capi.nvfp4_tiled_scale_bytes(128, 4096))]


def test_python_calls_check_their_tensors(capi):
    """Sizes and places of tensors are checked before an address is handed on."""
    torch = pytest.importorskip("torch")
    t = torch.zeros((4, 64))
    with pytest.raises(ValueError):
        capi.moe_route(t, t, t, 4, 64, 2)
    with pytest.raises(ValueError):
        capi.moe_route(t, t, t, 4, 64, 2, logits_type=9)
    with pytest.raises(ValueError):
        capi.moe_combine(t, t, t, t, 4, 64, 1)
    with pytest.raises(ValueError):
        capi.nvfp4_quantize(t, t, t, 4, 64, t)


def test_python_calls_refuse_sizes_and_element_types(capi):
    """Sizes that a 32-bit field would wrap, and tensors whose elements are not of the size the kernel reads."""
    torch = pytest.importorskip("torch")
    for bad in ((-1, 4), (4, 1 << 31), ((1 << 32) + 4, 4)):
        with pytest.raises(ValueError):
            capi._sizes(bad[0] | bad[1], *bad)
    capi._sizes(0 | ((1 << 31) - 1), 0, (1 << 31) - 1)
    ids = torch.zeros((8,), dtype=torch.int64)
    here = ids.get_device()
    with pytest.raises(ValueError):
        capi._buffer(ids, 32, "ids", here, 4)
    assert capi._buffer(ids.to(torch.int32), 32, "ids", here, 4) != 0
    assert capi._buffer(ids.view(torch.uint8), 32, "ids", here, 4) == ids.data_ptr()    # raw bytes
    with pytest.raises(ValueError):
        capi._rows(torch.zeros((4, 16)), 4, 16, 16, 2, "x", here)


def test_reference_rounding():
    """The plain definitions themselves: ties of both small formats, and a scale that lands on the largest value."""
    assert list(R.E2M1[R.nearest_even(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 99.0]), R.E2M1)]) == \
        [0, 1, 1, 2, 2, 4, 4, 6]
    x = np.zeros((1, 16), np.float32)
    x[0, 3] = -6 * 448.0
    codes, scale = R.nvfp4_quantize(x, 1.0)
    assert scale[0, 0] == 0x7E and codes[0, 3] == 15 and codes[0, 0] == 0
    s = np.arange(130 * 5, dtype=np.uint8).reshape(130, 5) % 120
    back, padding = R.untile_scales(R.tile_scales(s), 130, 5)
    assert np.array_equal(back, s) and not padding.any()
