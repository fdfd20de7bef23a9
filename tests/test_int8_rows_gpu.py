"""int8 rows (``layer_ops.quantize_int8``, ``rms_norm_int8``) at the borders of their definition: the integers bit for
bit, rows of every kernel variant, products that pass fp32, tensors that autograd watches.

Tolerances of a norm, in units u = 2^-24 as in ``test_int8_gpu``, for every variant: a thread adds up to 64 squares
in a row (8 vectors of 8 values, or k / 1024 + 8 for looped rows) and 10 more across threads.  rstd is off by half of
that and 6 u more, the scale by another 4 u, a value of y over the scale by 8 u more.
"""

import pytest
import torch

from test_int8_gpu import DTYPES, TINY, U, _check_quantize, _check_rows, _gen
from triton_mla import layer_ops

pytestmark = pytest.mark.gpu


def _rows(m, k, stride, offset, dtype, g, device, scale=1.0):
    """[m, k] with the given row stride, starting `offset` values into its memory."""
    flat = (torch.randn(m * stride + offset, generator=g, device=device) * scale).to(dtype)
    return flat.as_strided((m, k), (stride, 1), offset)


def _check_norm(x, w, eps=1e-6, residual=None):
    want_h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    q, scale, h = layer_ops.rms_norm_int8(x, w, eps, residual=residual)
    assert h is None if residual is None else torch.equal(h, want_h)
    f = want_h.double()
    y = f * w.double() * (f.square().mean(-1, keepdim=True) + eps).rsqrt()
    tol = ((max(64, x.shape[1] / 1024 + 8) + 10) / 2 + 6 + 4) * U * 1.01
    _check_rows(q, scale, y, tol, tol + 8 * U)


def _by_127(t):
    """True fp32 division (a Python number as the divisor would be multiplied by its reciprocal)."""
    return t / torch.full((1,), 127.0, device=t.device)


# (k, row stride, offset) of every variant: whole vectors of one warp and of several, with 1, 2, 4 and 8 of them a
# thread, each with and without a rest of the row; rows off 16-byte boundaries in registers and looped over;
# aligned rows beyond the registers, with and without a rest.
LAYOUTS = [
    (64, 64, 0), (513, 520, 0), (1001, 1008, 0), (1536, 2112, 0), (7168, 7168, 0), (7171, 7184, 0), (16387, 16400, 0),
    (32768, 32768, 0), (20005, 20016, 8), (100, 103, 1), (1001, 1003, 3), (8192, 8193, 1), (8193, 8195, 0),
    (10001, 10007, 5), (40001, 40003, 1), (40000, 40000, 0), (40001, 40016, 0),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,stride,offset", LAYOUTS)
def test_rows_of_every_variant(device, dtype, k, stride, offset):
    """Several rows a block, every alignment, with and without a residual, into a new h and in place."""
    g = _gen(device, k + stride)
    for m in (1, 5, 67):
        x = _rows(m, k, stride, offset, dtype, g, device, 3.0)
        r = _rows(m, k, stride, offset, dtype, g, device, 4.0)
        w = (1 + 0.2 * torch.randn(k + 1, generator=g, device=device)).to(dtype)
        for weight in (w[:k], w[1:]):
            _check_norm(x, weight)
            _check_norm(x, weight, residual=r)
        _check_quantize(x)
        target = r.clone() if m == 5 else _rows(m, k, stride, offset, dtype, g, device)   # packed rows, or r's layout
        target.copy_(r)
        q, s, h = layer_ops.rms_norm_int8(x, w[:k], residual=target)
        q2, s2, h2 = layer_ops.rms_norm_int8(x, w[:k], residual=target, residual_out=target)
        assert h2 is target and torch.equal(q2, q) and torch.equal(s2, s) and torch.equal(h2, h)


def _integers(y, scale):
    """The definition, bit for bit: y times the rounded 1 / scale, rounded to fp32 and to the nearest integer."""
    inv = torch.ones_like(scale) / scale
    return (y * inv[:, None]).round().to(torch.int8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,stride,offset", LAYOUTS)
def test_quantize_int8_gives_the_definition_bit_for_bit(device, dtype, k, stride, offset):
    """scale = max / 127 and q = rint(x (1 / scale)), each operation rounded to fp32.  Sixteenths between -9.375 and
    9.375 put many quotients next to half an integer (4.6875 / (9.375 / 127) = 63.5), where the product may fall on
    either side of x / scale; no integer is off by more than half a step and 2^-16."""
    g = _gen(device, k)
    for i in range(3):
        x = _rows(33, k, stride, offset, dtype, g, device, 2.5)
        if i:
            x.copy_((x.float() * 16).round().clamp(-150, 150) / 16)
        if i == 2:
            x[:, k // 2] = 9.375
        q, scale = layer_ops.quantize_int8(x)
        assert torch.equal(scale, _by_127(x.float().abs().amax(-1)))
        assert torch.equal(q, _integers(x.float(), scale))
        assert float((q.double() - x.double() / scale.double()[:, None]).abs().max()) <= 0.5 + 2.0 ** -16


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,stride,offset", LAYOUTS)
def test_rms_norm_int8_gives_the_definition_bit_for_bit(device, dtype, k, stride, offset):
    """h of +-1 and eps = 0: the mean square is exactly 1, so y = h w without a rounding."""
    g = _gen(device, k)
    x = _rows(33, k, stride, offset, dtype, g, device)
    x.copy_(torch.where(x < 0, -1.0, 1.0))
    w = ((torch.randn(k, generator=g, device=device) * 40).round().clamp(-150, 150) / 16).to(dtype)
    w[k // 2] = 9.375
    for residual in (None, torch.zeros_like(x)):
        q, scale, _ = layer_ops.rms_norm_int8(x, w, 0.0, residual=residual)
        assert torch.equal(scale, _by_127(torch.full_like(scale, 9.375)))
        assert torch.equal(q, _integers(x.float() * w.float(), scale))


def test_integers_at_the_ends_of_fp32(device):
    """Rows near the largest and the smallest fp32 values, subnormal ones among them."""
    g = _gen(device, 5)
    x = torch.randn(4, 4096, generator=g, device=device)
    x = x / x.abs().amax(-1, keepdim=True)
    x = x * torch.tensor([3.4e38, 2e-36, 1.4e-38, 1e-42], device=device)[:, None]
    for rows in (x, torch.nn.functional.pad(x, (0, 1))[:, :4096]):
        q, scale = layer_ops.quantize_int8(rows)
        assert torch.equal(scale, _by_127(x.abs().amax(-1)).clamp_min(TINY))
        assert torch.equal(q, _integers(x, scale))
        assert int(q[0].abs().max()) == 127 and not bool(q[3].any())


# ----------------------------------------------------------------------------- products and squares past fp32
FAR_LAYOUTS = [(100, 104, 0), (7168, 7168, 0), (32768, 32768, 0), (1001, 1003, 1), (10001, 10003, 1), (40000, 40000, 0)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("k,stride,offset", FAR_LAYOUTS)
def test_products_beyond_fp32(device, dtype, k, stride, offset):
    """|h w| above 3.4e38 with finite h and w is not a row without a scale: where the squares sum past fp32 too the
    norm is 0, where they do not y is what its formula says.  An infinity itself still leaves no scale."""
    g = _gen(device, k)
    x = _rows(7, k, stride, offset, dtype, g, device)
    ordinary = x.clone()
    w = (1 + 0.2 * torch.randn(k, generator=g, device=device)).to(dtype)
    w[1], w[2] = 4.0, 1e30
    x[1, 1] = 2e38                                        # h w = 8e38 and h^2 past fp32: zeros
    x[2, 2] = 1e12                                        # h w = 1e42, h^2 = 1e24: an ordinary norm
    x[3] = 1e15
    x[4, 1] = float("inf")
    x[5, 0] = float("nan")
    x[5, 2] = 1e12
    x[6, 1], x[6, 2] = 2e38, float("inf")
    for residual in (None, torch.zeros_like(x)):
        q, s, _ = layer_ops.rms_norm_int8(x, w, residual=residual)
        assert float(s[1]) == TINY and not bool(q[1].any())
        for bad in (4, 5, 6):
            assert bool(torch.isnan(s[bad])) and not bool(q[bad].any())
        for row in (0, 2, 3):
            _check_norm(x[row:row + 1], w, residual=None if residual is None else residual[row:row + 1])
            f = x[row].double()
            y = f * w.double() / (f.square().mean() + 1e-6).sqrt()
            assert abs(float(s[row]) - float(y.abs().max() / 127)) <= 1e-5 * float(s[row])
    w[2] = float("inf")
    q, s, _ = layer_ops.rms_norm_int8(ordinary, w)
    assert bool(torch.isnan(s).all()) and not bool(q.any()), "a weight without a value leaves no row a scale"


def test_eps_of_zero(device):
    """An all-zero row has no norm then (0 / 0): no scale, as a fp32 norm's NaN; the other rows are ordinary."""
    g = _gen(device, 9)
    x = torch.randn(3, 1536, generator=g, device=device)
    x[1] = 0
    w = torch.ones(1536, device=device)
    q, s, _ = layer_ops.rms_norm_int8(x, w, 0.0)
    assert bool(torch.isnan(s[1])) and not bool(q[1].any())
    _check_norm(x[::2].contiguous(), w, 0.0)


# ----------------------------------------------------------------------------- refusals
def test_a_watched_tensor_is_not_written_in_place(device):
    """Autograd cannot follow the operator, so a tensor that requires a gradient is not updated under it."""
    x = torch.randn(4, 64, device=device)
    w = torch.ones(64, device=device)
    leaf = torch.randn(4, 64, device=device, requires_grad=True)
    for watched in (leaf, leaf * 2):
        before = watched.detach().clone()
        with pytest.raises(RuntimeError, match="gradient"):
            layer_ops.rms_norm_int8(x, w, residual=watched, residual_out=watched)
        torch.cuda.synchronize()
        assert torch.equal(watched.detach(), before)
        with torch.no_grad():
            want = (x + before)
            _, _, h = layer_ops.rms_norm_int8(x, w, residual=watched, residual_out=watched)
            assert h is watched and torch.equal(watched.detach(), want)


def test_overlapping_rows_are_refused_by_name(device):
    x = torch.randn(1, 64, device=device)
    w = torch.ones(64, device=device)
    wide = torch.randn(4, 64, device=device)
    flat = torch.randn(400, device=device).as_strided((4, 64), (63, 1))
    assert layer_ops.quantize_int8(x)[0].shape == (1, 64)
    for rows in (x.expand(4, 64), flat):
        with pytest.raises(AssertionError, match="row stride"):
            layer_ops.quantize_int8(rows)
        with pytest.raises(AssertionError, match="row stride"):
            layer_ops.rms_norm_int8(rows, w)
        with pytest.raises(AssertionError, match="row stride"):
            layer_ops.rms_norm_int8(wide, w, residual=rows)
        with pytest.raises(AssertionError, match="row stride"):
            layer_ops.rms_norm_int8(wide, w, residual=wide, residual_out=rows)
    q, s = layer_ops.quantize_int8(wide)
    rows = q[:1].expand(4, 64)
    with pytest.raises(AssertionError, match="row stride"):
        layer_ops.linear_int8(rows, s, q, s)
    with pytest.raises(AssertionError, match="row stride"):
        layer_ops.linear_int8(q, s, rows, s)
