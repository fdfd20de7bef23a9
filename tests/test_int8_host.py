"""The int8 projections' refusals and shapes, without a GPU: argument checks of the C ABI before any
launch, the Python helpers on CPU tensors, the operators' Meta kernels."""

import ctypes

import pytest
import torch

from triton_mla import _lib, layer_ops


def _rows(**kw):
    p = _lib.TmlaInt8RowsParams()
    p.x = p.q = p.scale = 256
    p.x_stride = p.q_stride = 64
    p.m, p.k, p.dtype, p.eps = 2, 64, _lib.DTYPE_BF16, 1e-6
    for name, v in kw.items():
        setattr(p, name, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(m=0), _lib.OK),
    (dict(m=0, x=None, q=None, scale=None), _lib.OK),
    (dict(m=-1), _lib.ERR_INVALID_ARG),
    (dict(k=0), _lib.ERR_INVALID_ARG),
    (dict(dtype=3), _lib.ERR_INVALID_ARG),
    (dict(x=None), _lib.ERR_INVALID_ARG),
    (dict(q=None), _lib.ERR_INVALID_ARG),
    (dict(scale=None), _lib.ERR_INVALID_ARG),
    (dict(x_stride=63), _lib.ERR_INVALID_ARG),
    (dict(q_stride=63), _lib.ERR_INVALID_ARG),
    (dict(weight=256), _lib.ERR_INVALID_ARG),       # quantisation has no weight
    (dict(residual=256), _lib.ERR_INVALID_ARG),
    (dict(m=1 << 31), _lib.ERR_UNSUPPORTED),
    (dict(k=(1 << 30) + 1, x_stride=1 << 31, q_stride=1 << 31), _lib.ERR_UNSUPPORTED),
])
def test_quantize_int8_checks_its_arguments_before_any_launch(kw, code):
    assert _lib.load().tmla_quantize_int8(ctypes.byref(_rows(**kw)), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(m=0), _lib.OK),
    (dict(weight=None), _lib.ERR_INVALID_ARG),
    (dict(residual=256, residual_stride=64), _lib.ERR_INVALID_ARG),                       # no h
    (dict(residual=256, residual_stride=60, h=256, h_stride=64), _lib.ERR_INVALID_ARG),
    (dict(residual=256, residual_stride=64, h=256, h_stride=60), _lib.ERR_INVALID_ARG),
])
def test_rms_norm_int8_checks_its_arguments_before_any_launch(kw, code):
    p = _rows(**{"weight": 256, **kw})
    assert _lib.load().tmla_rms_norm_int8(ctypes.byref(p), None) == code


def _linear(**kw):
    p = _lib.TmlaLinearInt8Params()
    p.x = p.x_scale = p.w = p.w_scale = p.y = 256
    p.x_stride = p.w_stride = 64
    p.y_stride, p.m, p.n, p.k, p.dtype = 8, 2, 8, 64, _lib.DTYPE_BF16
    for name, v in kw.items():
        setattr(p, name, v)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(m=0), _lib.OK),
    (dict(n=0), _lib.OK),
    (dict(m=-1), _lib.ERR_INVALID_ARG),
    (dict(n=-1), _lib.ERR_INVALID_ARG),
    (dict(k=0), _lib.ERR_INVALID_ARG),
    (dict(dtype=3), _lib.ERR_INVALID_ARG),
    (dict(x=None), _lib.ERR_INVALID_ARG),
    (dict(x_scale=None), _lib.ERR_INVALID_ARG),
    (dict(w=None), _lib.ERR_INVALID_ARG),
    (dict(w_scale=None), _lib.ERR_INVALID_ARG),
    (dict(y=None), _lib.ERR_INVALID_ARG),
    (dict(x_stride=63), _lib.ERR_INVALID_ARG),
    (dict(w_stride=63), _lib.ERR_INVALID_ARG),
    (dict(y_stride=7), _lib.ERR_INVALID_ARG),
    (dict(m=(1 << 30) + 1), _lib.ERR_UNSUPPORTED),
    (dict(n=(1 << 30) + 1, y_stride=1 << 31), _lib.ERR_UNSUPPORTED),
    (dict(k=_lib.LINEAR_INT8_MAX_K + 1, x_stride=1 << 20, w_stride=1 << 20), _lib.ERR_UNSUPPORTED),
])
def test_linear_int8_checks_its_arguments_before_any_launch(kw, code):
    assert _lib.load().tmla_linear_int8(ctypes.byref(_linear(**kw)), None) == code


def test_null_parameter_structs_are_refused():
    lib = _lib.load()
    for fn in (lib.tmla_quantize_int8, lib.tmla_rms_norm_int8, lib.tmla_linear_int8):
        assert fn(None, None) == _lib.ERR_INVALID_ARG


def test_the_status_word_needs_somewhere_to_go():
    assert _lib.load().tmla_status_word(None) == _lib.ERR_INVALID_ARG


def test_int8_helpers_refuse_cpu_tensors():
    x, w = torch.zeros(4, 64), torch.ones(64)
    q, s = torch.zeros(4, 64, dtype=torch.int8), torch.ones(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        layer_ops.quantize_int8(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        layer_ops.rms_norm_int8(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        layer_ops.linear_int8(q, s, q, s)


def test_int8_operators_have_meta_kernels():
    """What torch.compile's tracing runs: shapes, dtypes and the 16-byte row strides of q."""
    ops = torch.ops.triton_mla
    x = torch.empty(5, 1001, dtype=torch.bfloat16, device="meta")
    q, scale = ops.quantize_int8(x, False)
    assert q.shape == (5, 1001) and q.dtype == torch.int8 and q.stride() == (1008, 1)
    assert scale.shape == (5,) and scale.dtype == torch.float32
    w = torch.empty(1001, dtype=torch.bfloat16, device="meta")
    q, scale, h = ops.rms_norm_int8(x, w, 1e-6, x, None, False)
    assert q.stride() == (1008, 1) and h.shape == x.shape and h.dtype == x.dtype
    assert ops.rms_norm_int8(x, w, 1e-6, None, None, False)[2].numel() == 0
    wq = torch.empty(70, 1001, dtype=torch.int8, device="meta")
    y = ops.linear_int8(q, scale, wq, torch.empty(70, device="meta"), torch.float16, False, None)
    assert y.shape == (5, 70) and y.dtype == torch.float16 and y.stride() == (72, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n", [(1, 1), (32, 249), (5, 1001), (3, 64), (0, 7), (4, 0)])
def test_padded_rows_lie_in_their_own_storage(dtype, m, n):
    """Rows of y, h and q are padded to 16 bytes, the last one too: what a TMA store may write there is the tensor's."""
    ops = torch.ops.triton_mla
    wq = torch.empty(n, 64, dtype=torch.int8, device="meta")
    xq, xs = torch.empty(m, 64, dtype=torch.int8, device="meta"), torch.empty(m, device="meta")
    tensors = [ops.linear_int8(xq, xs, wq, torch.empty(n, device="meta"), dtype, False, None)]
    if n:
        x, w = torch.empty(m, n, dtype=dtype, device="meta"), torch.empty(n, dtype=dtype, device="meta")
        q, _, h = ops.rms_norm_int8(x, w, 1e-6, x, None, False)
        tensors += [q, h, ops.quantize_int8(x, False)[0]]
    for t in tensors:
        row = -(-n * t.element_size() // 16) * 16
        assert t.shape == (m, n) and t.stride(1) == 1
        assert m < 2 or t.stride(0) * t.element_size() == max(row, t.element_size())
        assert t.untyped_storage().nbytes() >= m * row and t.storage_offset() == 0 and not t._is_view()


def _variant(m, n, k, dtype):
    """(CTAs of a tile, tokens of a tile, parts of k, tiles in a row: 1, 2 or more) on 148 SMs."""
    plan = (ctypes.c_int32 * 4)()
    assert _lib.load().tmla_linear_int8_plan(m, n, k, dtype, 148, plan) == _lib.OK
    return (*plan[:3], min(plan[3], 3))


@pytest.mark.parametrize("dtype", [_lib.DTYPE_BF16, _lib.DTYPE_FP32])
def test_the_gpu_tests_reach_every_variant_of_the_product(dtype):
    """Whatever constants choose the variant: the shapes that the GPU tests run in every type reach all variants that
    20,000 sizes (1 to 8192 tokens, spread over the logarithm) reach."""
    import math
    import random

    import test_int8_gpu as gpu

    rng = random.Random(11)

    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    run = {_variant(m, n, k, dtype) for m, n, k in gpu.LINEAR_SHAPES + gpu.VARIANT_SHAPES + gpu.MORE_VARIANT_SHAPES}
    for _ in range(20000):
        k = log(64, 16384)
        size = (log(1, 8192), log(64, min(24576, 7168 * 16384 // k)), k)
        assert _variant(*size, dtype) in run, (size, _variant(*size, dtype))


@pytest.mark.parametrize("kw,code", [
    (dict(m=0), _lib.ERR_INVALID_ARG),
    (dict(n=0), _lib.ERR_INVALID_ARG),
    (dict(k=0), _lib.ERR_INVALID_ARG),
    (dict(dtype=3), _lib.ERR_INVALID_ARG),
    (dict(num_sms=0), _lib.ERR_INVALID_ARG),
    (dict(plan=None), _lib.ERR_INVALID_ARG),
    (dict(m=(1 << 30) + 1), _lib.ERR_UNSUPPORTED),
    (dict(k=_lib.LINEAR_INT8_MAX_K + 1), _lib.ERR_UNSUPPORTED),
])
def test_the_plan_checks_its_arguments(kw, code):
    args = dict(m=1, n=1, k=1, dtype=_lib.DTYPE_BF16, num_sms=148, plan=(ctypes.c_int32 * 4)())
    args.update(kw)
    assert _lib.load().tmla_linear_int8_plan(*args.values()) == code
