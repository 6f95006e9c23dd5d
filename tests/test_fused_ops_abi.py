"""The fused ops between the residual stream and the projections without a GPU: record layouts and typed refusals, each
before any launch."""
import ctypes as C

import pytest

from roost_amd import abi

BF16, F32, F8, I32 = abi.DTYPE_BF16, abi.DTYPE_F32, abi.DTYPE_F8E4M3, abi.DTYPE_I32


def _span(address, n, dtype):
    s = abi.DeviceSpan()
    s.address, s.length, s.dtype = address, n, dtype
    return s


@pytest.fixture()
def ctx(kernels):
    c = kernels.create_context(0)
    yield c
    kernels.destroy_context(c)


def test_layouts():
    sizes = {"RoostAmdAddRmsNormParams": 160, "RoostAmdAddRmsNormQuantParams": 184, "RoostAmdSiluMulQuantParams": 128,
             "RoostAmdGemmLoraParams": 336}
    for name, size in sizes.items():
        assert C.sizeof(abi.EXTENSION_STRUCTS[name]) == size, name
    assert (abi.AddRmsNormParams.rows.offset, abi.AddRmsNormParams.eps.offset) == (128, 152)
    assert (abi.AddRmsNormQuantParams.rows.offset, abi.AddRmsNormQuantParams.group_size.offset) == (152, 180)
    assert (abi.SiluMulQuantParams.rows.offset, abi.SiluMulQuantParams.group_size.offset) == (104, 124)
    assert (abi.GemmLoraParams.output.offset, abi.GemmLoraParams.tokens.offset) == (272, 296)


def _norm(struct):
    p = abi.new(struct)
    quant = struct is abi.AddRmsNormQuantParams
    p.rows, p.dim, p.eps = 4, 256, 1e-6
    p.input, p.residual = _span(0x100000, 1024, BF16), _span(0x200000, 1024, F32)
    p.weight, p.residual_out = _span(0x300000, 256, BF16), _span(0x400000, 1024, F32)
    p.output = _span(0x500000, 1024, F8 if quant else BF16)
    if quant:
        p.scales = _span(0x600000, 8, F32)
        p.group_size = 128
    return p


def _refuse(kernels, run, make, change, want):
    p = make()
    change(p)
    assert run(p) == want, kernels.last_error()
    assert kernels.last_error()


def _set(path, value):
    def change(p):
        *outer, name = path.split(".")
        for o in outer:
            p = getattr(p, o)
        setattr(p, name, value)
    return change


NORM_REFUSALS = [
    ("struct_size", 64, abi.ABI_MISMATCH), ("abi_minor", 9, abi.ABI_MISMATCH), ("dim", 0, abi.UNSUPPORTED),
    ("dim", 32769, abi.UNSUPPORTED), ("input.dtype", abi.DTYPE_F16, abi.UNSUPPORTED),
    ("residual.dtype", abi.DTYPE_F16, abi.UNSUPPORTED), ("weight.dtype", F8, abi.UNSUPPORTED),
    ("weight.address", None, abi.INVALID_ARGUMENT), ("weight.length", 255, abi.INVALID_ARGUMENT),
    ("residual_out.dtype", BF16, abi.INVALID_ARGUMENT), ("input.length", 1023, abi.INVALID_ARGUMENT),
    ("input_stride", 255, abi.INVALID_ARGUMENT), ("input_stride", 257, abi.INVALID_ARGUMENT),  # four rows no longer fit
    ("output.length", 1000, abi.INVALID_ARGUMENT), ("output.dtype", F32, abi.INVALID_ARGUMENT),
    ("output.reserved0", 1, abi.INVALID_ARGUMENT), ("input.address", 0x100001, abi.INVALID_ARGUMENT),
    ("residual.address", 0x200002, abi.INVALID_ARGUMENT),
    ("output.address", 0x100200, abi.INVALID_ARGUMENT),      # over the input, not exactly it
    ("output.address", 0x200000, abi.INVALID_ARGUMENT),      # the residual's address, another type
    ("output.address", 0x400000, abi.INVALID_ARGUMENT),      # both outputs on one span
    ("residual_out.address", 0x300000, abi.INVALID_ARGUMENT),  # over the weight
]


@pytest.mark.parametrize("field,value,want", NORM_REFUSALS + [("reserved0", 3, abi.INVALID_ARGUMENT)])
def test_add_rms_norm_refusals(kernels, ctx, field, value, want):
    run = lambda p: kernels.dll.roost_amd_add_rms_norm_run(ctx, C.addressof(p), None)  # noqa: E731
    _refuse(kernels, run, lambda: _norm(abi.AddRmsNormParams), _set(field, value), want)


@pytest.mark.parametrize("field,value,want", NORM_REFUSALS + [
    ("group_size", 8, abi.UNSUPPORTED), ("group_size", 100, abi.UNSUPPORTED), ("group_size", 1024, abi.UNSUPPORTED),
    ("scales.length", 7, abi.INVALID_ARGUMENT), ("scales.dtype", BF16, abi.INVALID_ARGUMENT),
    ("scales.address", 0x100000, abi.INVALID_ARGUMENT), ("scales.address", 0x500010, abi.INVALID_ARGUMENT),
    ("scales.address", None, abi.INVALID_ARGUMENT)])
def test_add_rms_norm_quant_refusals(kernels, ctx, field, value, want):
    run = lambda p: kernels.dll.roost_amd_add_rms_norm_quant_run(ctx, C.addressof(p), None)  # noqa: E731
    _refuse(kernels, run, lambda: _norm(abi.AddRmsNormQuantParams), _set(field, value), want)


@pytest.mark.parametrize("apart,message", [(1200, "scales"), (400, "overlaps"), (2000, "overlaps")])
def test_column_views_of_one_tensor(kernels, ctx, apart, message):
    """Input (1,000 bytes) and output (250) in rows of 2,400 bytes: side by side they pass the overlap rule (the call is
    refused later, for its missing scales); sharing columns they do not, in the same row or past its end."""
    p = _norm(abi.AddRmsNormQuantParams)
    p.dim, p.input_stride, p.output_stride = 250, 600, 2400
    p.input, p.output = _span(0x100000, 3 * 600 + 250, F32), _span(0x100000 + apart, 3 * 2400 + 250, F8)
    if apart == 2000:
        p.input, p.output = _span(0x100000 + 2200, 3 * 600 + 250, F32), _span(0x100000 + 2400, 3 * 2400 + 250, F8)
    p.residual = p.residual_out = abi.DeviceSpan()
    p.weight.length = 250
    p.scales = abi.DeviceSpan()
    assert kernels.dll.roost_amd_add_rms_norm_quant_run(ctx, C.addressof(p), None) == abi.INVALID_ARGUMENT
    assert message in kernels.last_error(), kernels.last_error()


def _silu():
    p = abi.new(abi.SiluMulQuantParams)
    p.rows, p.dim, p.gate_stride, p.up_stride = 4, 256, 512, 512
    p.gate, p.up = _span(0x100000, 3 * 512 + 256, BF16), _span(0x100200, 3 * 512 + 256, BF16)
    p.output, p.scales = _span(0x500000, 1024, F8), _span(0x600000, 4, F32)
    return p


@pytest.mark.parametrize("field,value,want", [
    ("struct_size", 64, abi.ABI_MISMATCH), ("dim", 0, abi.UNSUPPORTED), ("dim", 32769, abi.UNSUPPORTED),
    ("gate.dtype", F8, abi.UNSUPPORTED), ("up.dtype", F32, abi.INVALID_ARGUMENT), ("up_stride", 100, abi.INVALID_ARGUMENT),
    ("output.address", 0x100300, abi.INVALID_ARGUMENT), ("scales.address", 0x500004, abi.INVALID_ARGUMENT),
    ("scales.length", 3, abi.INVALID_ARGUMENT), ("group_size", 48, abi.UNSUPPORTED), ("output.address", None, abi.INVALID_ARGUMENT)])
def test_silu_mul_quant_refusals(kernels, ctx, field, value, want):
    run = lambda p: kernels.dll.roost_amd_silu_mul_quant_run(ctx, C.addressof(p), None)  # noqa: E731
    _refuse(kernels, run, _silu, _set(field, value), want)


def _lora(dtype=BF16):
    low = F32 if dtype == F32 else BF16
    p = abi.new(abi.GemmLoraParams)
    p.tokens, p.batch, p.in_dim, p.out_dim, p.adapters, p.max_rank = 10, 3, 64, 48, 5, 16
    p.x, p.weight = _span(0x100000, 640, dtype), _span(0x200000, 48 * 64, dtype)
    p.lora_a, p.lora_b = _span(0x300000, 5 * 16 * 64, low), _span(0x400000, 5 * 48 * 16, low)
    p.lora_scale, p.ranks = _span(0x500000, 5, F32), _span(0x510000, 5, I32)
    p.lora_slots, p.cu_seqlens = _span(0x520000, 3, I32), _span(0x530000, 4, I32)
    p.addend, p.output = _span(0x600000, 480, BF16), _span(0x700000, 480, F32 if dtype == F32 else BF16)
    if dtype == F8:
        p.x_scale, p.w_scale = _span(0x540000, 10, F32), _span(0x550000, 48, F32)
    return p


def _run_lora(kernels, ctx, p):
    ws = abi.new(abi.Workspace)
    ws.device, ws.device_bytes = 0x900000, 1 << 20
    return kernels.dll.roost_amd_gemm_lora_run(ctx, C.addressof(p), C.addressof(ws), None)


@pytest.mark.parametrize("field,value,want", [
    ("struct_size", 64, abi.ABI_MISMATCH), ("reserved0", 1, abi.INVALID_ARGUMENT), ("x.dtype", abi.DTYPE_F16, abi.UNSUPPORTED),
    ("in_dim", 0, abi.UNSUPPORTED), ("in_dim", 60, abi.UNSUPPORTED), ("x_stride", 68, abi.UNSUPPORTED),
    ("x_stride", 56, abi.INVALID_ARGUMENT), ("x_stride", 72, abi.INVALID_ARGUMENT), ("out_dim", 0, abi.UNSUPPORTED),
    ("out_dim", 49, abi.INVALID_ARGUMENT), ("output_stride", 40, abi.INVALID_ARGUMENT), ("tokens", 11, abi.INVALID_ARGUMENT),
    ("tokens", 1 << 20, abi.UNSUPPORTED), ("batch", 4, abi.INVALID_ARGUMENT), ("batch", 1 << 30, abi.UNSUPPORTED),
    ("max_rank", 12, abi.UNSUPPORTED), ("max_rank", 136, abi.UNSUPPORTED), ("max_rank", 0, abi.UNSUPPORTED),
    ("max_rank", 24, abi.INVALID_ARGUMENT), ("adapters", 0, abi.UNSUPPORTED), ("adapters", 6, abi.INVALID_ARGUMENT),
    ("lora_a.dtype", F32, abi.INVALID_ARGUMENT), ("lora_b.address", None, abi.INVALID_ARGUMENT),
    ("lora_a.address", 0x300008, abi.INVALID_ARGUMENT), ("lora_b.address", 0x400002, abi.INVALID_ARGUMENT),
    ("lora_slots.address", None, abi.INVALID_ARGUMENT), ("cu_seqlens.address", None, abi.INVALID_ARGUMENT),
    ("cu_seqlens.length", 3, abi.INVALID_ARGUMENT), ("ranks.length", 4, abi.INVALID_ARGUMENT),
    ("x.address", 0x100008, abi.INVALID_ARGUMENT), ("weight.address", 0x200008, abi.INVALID_ARGUMENT),
    ("weight.dtype", F8, abi.INVALID_ARGUMENT), ("output.dtype", F8, abi.UNSUPPORTED),
    ("output.address", 0x600010, abi.INVALID_ARGUMENT), ("output.address", 0x100000, abi.INVALID_ARGUMENT),
    ("output.address", 0x200000, abi.INVALID_ARGUMENT), ("output.address", 0x52FFF0, abi.INVALID_ARGUMENT),
    ("addend.dtype", F8, abi.UNSUPPORTED), ("addend.length", 479, abi.INVALID_ARGUMENT),
    ("x_scale.address", 0x540000, abi.INVALID_ARGUMENT), ("lora_a.address", None, abi.INVALID_ARGUMENT)])
def test_gemm_lora_refusals(kernels, ctx, field, value, want):
    _refuse(kernels, lambda p: _run_lora(kernels, ctx, p), _lora, _set(field, value), want)


@pytest.mark.parametrize("field,value,want", [
    ("x_scale.address", None, abi.INVALID_ARGUMENT), ("w_scale.address", None, abi.INVALID_ARGUMENT),
    ("x_scale.length", 9, abi.INVALID_ARGUMENT), ("in_dim", 56, abi.UNSUPPORTED), ("lora_a.dtype", F8, abi.INVALID_ARGUMENT)])
def test_gemm_lora_8_bit_refusals(kernels, ctx, field, value, want):
    _refuse(kernels, lambda p: _run_lora(kernels, ctx, p), lambda: _lora(F8), _set(field, value), want)


def test_gemm_lora_neither_weight_nor_adapters(kernels, ctx):
    p = _lora()
    p.weight = p.lora_a = abi.DeviceSpan()
    p.adapters = p.max_rank = 0
    assert _run_lora(kernels, ctx, p) == abi.INVALID_ARGUMENT
    p = _lora(F32)
    p.output = _span(0x700000, 480, BF16)
    assert _run_lora(kernels, ctx, p) == abi.UNSUPPORTED


def test_gemm_lora_workspace(kernels, ctx):
    p, sizes = _lora(), abi.new(abi.WorkspaceSizes)
    query = kernels.dll.roost_amd_gemm_lora_workspace
    assert query(ctx, C.addressof(p), C.addressof(sizes)) == abi.OK
    assert sizes.device_bytes > 0 and sizes.device_alignment == 256 and sizes.pinned_host_bytes == sizes.plan_bytes == 0
    assert kernels.dll.roost_amd_gemm_lora_run(ctx, C.addressof(p), None, None) == abi.WORKSPACE_TOO_SMALL
    ws = abi.new(abi.Workspace)
    ws.device, ws.device_bytes = 0x900000, sizes.device_bytes - 1
    assert kernels.dll.roost_amd_gemm_lora_run(ctx, C.addressof(p), C.addressof(ws), None) == abi.WORKSPACE_TOO_SMALL
    ws.device, ws.device_bytes = 0x900010, sizes.device_bytes
    assert kernels.dll.roost_amd_gemm_lora_run(ctx, C.addressof(p), C.addressof(ws), None) == abi.WORKSPACE_TOO_SMALL
    p.max_rank = 12
    assert query(ctx, C.addressof(p), C.addressof(sizes)) == abi.UNSUPPORTED
    assert query(ctx, None, C.addressof(sizes)) == abi.INVALID_ARGUMENT
    assert query(None, C.addressof(p), C.addressof(sizes)) == abi.INVALID_ARGUMENT


def test_nothing_to_do(kernels, ctx):
    """No rows, or no sequences: OK without a launch, whatever the addresses."""
    for struct, fn in ((abi.AddRmsNormParams, "add_rms_norm"), (abi.AddRmsNormQuantParams, "add_rms_norm_quant")):
        p = _norm(struct)
        p.rows = 0
        assert getattr(kernels.dll, f"roost_amd_{fn}_run")(ctx, C.addressof(p), None) == abi.OK
    p = _silu()
    p.rows = 0
    assert kernels.dll.roost_amd_silu_mul_quant_run(ctx, C.addressof(p), None) == abi.OK
    for name in ("tokens", "batch"):
        p = _lora()
        setattr(p, name, 0)
        assert _run_lora(kernels, ctx, p) == abi.OK


def test_gemm_lora_row_limits(kernels, ctx):
    """Strides past what a tile's 32-bit offsets reach are refused; neighbouring columns of one tensor are not."""
    p = _lora()
    p.x_stride, p.x = (1 << 20) + 8, _span(0x100000, 10 << 21, BF16)
    assert _run_lora(kernels, ctx, p) == abi.UNSUPPORTED and "x_stride" in kernels.last_error()


def test_python_checks():
    """The mirrors refuse what the C records cannot carry before a record is made."""
    import torch

    import roost_amd

    t = torch.zeros(4, 16)
    assert roost_amd._rows(t[:, 2:10], "x", 4, 8)[1] == 16 and roost_amd._rows(t[:1, 2:10], "x", 1, 8)[1] == 8
    assert roost_amd._rows(t[:0], "x", 0, 16)[0].length == 0 and roost_amd._rows(None, "x", 4, 16)[1] == 0
    for bad, shape in ((t, (4, 8)), (t[0], (16, 1)), (t.T, (16, 4)), (t[:1].expand(4, 16), (4, 16)), (t[:, ::2], (4, 8))):
        with pytest.raises(ValueError, match="x: "):
            roost_amd._rows(bad, "x", *shape)
    with pytest.raises(ValueError, match="not one of"):
        roost_amd._rows(t, "up", 4, 16, (torch.bfloat16,))
    assert roost_amd._flat(t, "w", (4, 16)).length == 64 and not roost_amd._flat(None, "w", (4, 16)).address
    for bad, shape, dtype in ((t, (16, 4), None), (t[:, :8], (4, 8), None), (t, (4, 16), torch.int32)):
        with pytest.raises(ValueError, match="w: "):
            roost_amd._flat(bad, "w", shape, dtype)
    cu, slots = torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="tensors of one call are on"):
        roost_amd.gemm_lora_params(t, t, None, None, None, slots, cu, torch.zeros(4, 4))
    with pytest.raises(ValueError, match="tensors of one call are on"):
        roost_amd.add_rms_norm_params(t, None, t[0], None, t, eps=1e-6)
    with pytest.raises(ValueError, match="tensors of one call are on"):
        roost_amd.silu_mul_quant_params(t, t, t, t[:, :1])


@pytest.mark.parametrize("rows,dim", [(1 << 26, 64), (1 << 26, 512), (1 << 22, 8192), (1 << 22, 32768)])
def test_rows_of_a_launch(kernels, ctx, rows, dim):
    """Every row has a workgroup; a launch of 2^32 threads is refused by its size, one row fewer by its spans' lengths."""
    for struct, fn in ((abi.AddRmsNormParams, "add_rms_norm"), (abi.AddRmsNormQuantParams, "add_rms_norm_quant"),
                       (abi.SiluMulQuantParams, "silu_mul_quant")):
        for fewer, want in ((0, abi.UNSUPPORTED), (1, abi.INVALID_ARGUMENT)):
            p = _silu() if fn == "silu_mul_quant" else _norm(struct)
            p.rows, p.dim = rows - fewer, dim
            assert getattr(kernels.dll, f"roost_amd_{fn}_run")(ctx, C.addressof(p), None) == want, kernels.last_error()
