"""What of the expert layer's operators needs no GPU: record geometry, weight quantization, argument checks of the C ABI, and the
checks' order ahead of any device work."""

import ctypes

import pytest
import torch

import cabi
import nanoep_amd as ep
import operator_oracle as oracle
from nanoep_amd.examples import fp8_moe


def library():
    lib = cabi.lib()
    p, i, i64, f, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t
    lib.nanoep_fp8_record_bytes.restype = i64
    lib.nanoep_fp8_record_bytes.argtypes = [i64]
    lib.nanoep_rms_norm_fp8.argtypes = [p, p, p, i64, i, f, p, p, p, p]
    lib.nanoep_experts_linear.argtypes = [p, i64, p, i64, p, p, p, p, i64, i64, i, i, p, p]
    lib.nanoep_experts_gated_workspace_bytes.restype = sz
    lib.nanoep_experts_gated_workspace_bytes.argtypes = [i64, i64, i, i, i64, i64]
    lib.nanoep_experts_gated.argtypes = [p, i64, p, i64, p, p, p, p, i64, i64, i, i, p, p, sz, p]
    lib.nanoep_combine_weighted.argtypes = [p, i64, p, p, p, i64, i, i, p, p]
    lib.nanoep_combine_weighted_backward.argtypes = [p, p, i64, p, p, p, p, i64, i64, i, i, p, p, p]
    return lib


@pytest.mark.parametrize("columns", [16, 112, 128, 144, 256, 1024, 2816, 7168, 65536])
def test_records_hold_values_and_scales_and_can_be_dispatched(columns):
    size = library().nanoep_fp8_record_bytes(columns)
    used = columns + 4 * oracle.groups(columns)
    assert size % 512 == 0 and used <= size < used + 512
    assert ep.fp8_payload_width(columns) == size // 2
    payload = torch.arange(3 * size, dtype=torch.int64).to(torch.uint8).view(3, size).view(torch.bfloat16)
    rows = ep.Fp8Rows.of_payload(payload, columns)
    raw = payload.view(torch.uint8)
    assert torch.equal(rows.values.view(torch.uint8), raw[:, :columns])
    assert torch.equal(rows.scales.contiguous().view(torch.uint8).reshape(3, -1), raw[:, columns:used])
    assert rows.values.data_ptr() == payload.data_ptr()
    assert library().nanoep_fp8_record_bytes(0) == 0


@pytest.mark.parametrize("shape", [(1, 8, 16), (2, 128, 128), (3, 136, 272), (1, 300, 1024)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_weight(shape, dtype):
    weight = torch.randn(*shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    weight[0, :5] = 0
    got = ep.quantize_weight(weight)
    experts, columns, inner = shape
    assert got.values.shape == shape and got.scales.shape == (experts, oracle.groups(columns), oracle.groups(inner))
    scale = oracle.spread(got.scales.double().repeat_interleave(128, 1)[:, :columns], inner)
    error = (got.values.double() * scale - weight.double()).abs()
    assert (error <= torch.maximum(weight.double().abs() * oracle.FP8, scale * oracle.FP8_SMALL) * (1 + 8 * oracle.FP32)).all()
    for e in range(experts):
        for b in range(got.scales.shape[1]):
            for g in range(got.scales.shape[2]):
                block = weight[e, b * 128 : (b + 1) * 128, g * 128 : (g + 1) * 128].double().abs().max()
                want = block.clamp(min=oracle.SMALLEST_AMAX) / oracle.LARGEST
                assert abs(got.scales[e, b, g].double() - want) <= want * 2 * oracle.FP32
    assert not got.values[0, :5].float().any()


def test_the_c_abi_refuses_before_any_device_work():
    lib, null = library(), None
    bad = 1
    norm, linear, gated = lib.nanoep_rms_norm_fp8, lib.nanoep_experts_linear, lib.nanoep_experts_gated
    # no rows are nothing to do, whatever the pointers
    assert norm(null, null, null, 0, 256, 1e-6, null, null, null, null) == 0
    assert linear(null, 0, null, 0, null, null, null, null, 0, 1, 128, 128, null, null) == 0
    assert gated(null, 0, null, 0, null, null, null, null, 0, 1, 128, 128, null, null, 0, null) == 0
    assert lib.nanoep_combine_weighted(null, 0, null, null, null, 0, 256, 2, null, null) == 0
    assert lib.nanoep_combine_weighted_backward(null, null, 0, null, null, null, null, 0, 0, 256, 2, null, null, null) == 0
    # sizes
    for tokens, hidden, eps in ((-1, 256, 0.0), (1, 0, 0.0), (1, 24, 0.0), (1, 65552, 0.0), (1, 256, -1.0), (1, 256, float("nan"))):
        assert norm(64, null, 64, tokens, hidden, eps, 64, null, null, null) == bad
    # a residual without a place for the sum; no input; a pointer off its alignment
    assert norm(64, 64, 64, 1, 256, 0.0, 64, null, null, null) == bad
    assert norm(null, null, 64, 1, 256, 0.0, 64, null, null, null) == bad
    assert norm(72, null, 64, 1, 256, 0.0, 64, null, null, null) == bad
    for rows, experts, inner, columns in ((-1, 1, 128, 128), (1 << 31, 1, 128, 128), (1, 0, 128, 128), (1, 1, 8, 128), (1, 1, 0, 128), (1, 1, 128, 12), (1, 1, 128, 0)):
        assert linear(64, 128, 64, 1, 64, 64, null, null, rows, experts, inner, columns, 64, null) == bad
    assert gated(64, 128, 64, 1, 64, 64, null, null, 1, 1, 128, 48, 64, null, 0, null) == bad
    # strides shorter than the rows or off 16 bytes; one of the layout's arrays; more experts than one without a layout
    assert linear(64, 112, 64, 1, 64, 64, null, null, 2, 1, 128, 128, 64, null) == bad
    assert linear(64, 136, 64, 1, 64, 64, null, null, 2, 1, 128, 128, 64, null) == bad
    assert linear(64, 256, 64, 1, 64, 64, null, null, 2, 1, 256, 128, 64, null) == bad
    assert linear(64, 128, 64, 1, 64, 64, 64, null, 2, 2, 128, 128, 64, null) == bad
    assert linear(64, 128, 64, 1, 64, 64, null, null, 2, 2, 128, 128, 64, null) == bad
    assert linear(64, 128, 64, 1, 64, 64, null, null, 2, 1, 128, 128, 72, null) == bad
    # a gated product of few rows needs its workspace
    needed = lib.nanoep_experts_gated_workspace_bytes(2, 1, 128, 128, 128, 1)
    assert needed == 2 * 64 * 4
    assert gated(64, 128, 64, 1, 64, 64, null, null, 2, 1, 128, 128, 64, 64, needed - 1, null) == 3
    assert gated(64, 128, 64, 1, 64, 64, null, null, 2, 1, 128, 128, 64, null, needed, null) == bad
    assert lib.nanoep_experts_gated_workspace_bytes(1 << 16, 8, 1024, 4096, 1024, 8) == 0
    assert lib.nanoep_experts_gated_workspace_bytes(0, 1, 128, 128, 128, 1) == 0
    for rows, tokens, hidden, topk in ((-1, 1, 256, 1), (1, -1, 256, 1), (1, 1, 252, 1), (1, 1, 256, 0), (1, 1, 256, 33)):
        assert lib.nanoep_combine_weighted(64, rows, 64, 64, null, tokens, hidden, topk, 64, null) == bad
        assert lib.nanoep_combine_weighted_backward(64, 64, rows, 64, 64, null, null, 0, tokens, hidden, topk, 64, 64, null) == bad
    assert lib.nanoep_combine_weighted_backward(64, 64, 1, 64, 64, 64, null, 1, 1, 256, 1, 64, 64, null) == bad
    assert lib.nanoep_combine_weighted_backward(64, 64, 1, 64, 64, 64, 64, 0, 1, 256, 1, 64, 64, null) == bad


def test_cpu_tensors_are_refused():
    x, gamma = torch.zeros(2, 256, dtype=torch.bfloat16), torch.ones(256, dtype=torch.bfloat16)
    weight = ep.quantize_weight(torch.zeros(1, 32, 256))
    rows = ep.Fp8Rows(torch.zeros(2, 256).to(torch.float8_e4m3fn), torch.ones(2, 2))
    slots, weights = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1)
    for call in (lambda: ep.rms_norm_fp8(x, gamma), lambda: ep.experts_linear(rows, weight), lambda: ep.experts_gated(rows, weight),
                 lambda: ep.combine_weighted(x, slots, weights), lambda: ep.combine_weighted_backward(x, x, slots, weights)):
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            call()


def test_the_examples_arguments_are_checked():
    for arguments in (["--hidden", "200"], ["--intermediate", "8"], ["--topk", "9"], ["--tokens", "0"]):
        with pytest.raises(SystemExit):
            fp8_moe.parse_args(arguments)
