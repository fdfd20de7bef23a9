"""The int8 projections (``layer_ops.quantize_int8``, ``rms_norm_int8``, ``linear_int8``) against
their definitions in 64 bits.

Tolerances.  u = 2^-24 is the unit roundoff of fp32.
* quantize_int8: scale = fl(a / 127) is off by at most u relative; x / scale as x * fl(1 / scale) by
  3 u relative, 127 * 3 u absolute at most, before it is rounded to an integer.
* rms_norm_int8: the sum of squares adds c terms in a row in one thread (c = 8 per vector, 4 vectors, or
  k / 1024 + 8 for long rows) and 10 more across threads, so it is off by (c + 10) u, rstd by half of
  that plus the mean's, eps's and rsqrt's 1 + 1 + 4 u, and the scale by 4 u more (h w, times rstd,
  / 127).  rstd cancels from q: h w rstd / scale is off by 8 u relative.
* linear_int8: the int32 sum is exact; its conversion and the two scales cost 3 u, the output's
  rounding eps / 2 (an absolute 2^-25 below fp16's normal range).
"""

import pytest
import torch

from triton_mla import layer_ops, mla_decode, read_status

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = torch.finfo(torch.float32).tiny
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def _check_rows(q, scale, y, scale_tol, q_tol):
    """q and scale against the exact rows y (float64) they stand for."""
    ref = (y.abs().amax(-1) / 127).clamp_min(TINY)
    assert scale.dtype == torch.float32 and q.dtype == torch.int8 and scale.shape == y.shape[:1]
    assert bool(((scale.double() - ref).abs() <= scale_tol * ref).all())
    off = (q.double() - y / ref[:, None]).abs().max() if y.numel() else torch.tensor(0.0)
    assert float(off) <= 0.5 + q_tol * 127, float(off)
    assert int(q.int().abs().max()) <= 127 if y.numel() else True


def _check_quantize(x):
    q, scale = layer_ops.quantize_int8(x)
    assert q.shape == x.shape and q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0
    _check_rows(q, scale, x.double(), U * 1.01, 3 * U * 1.01)


def _check_norm(x, w, eps=1e-6, residual=None, **kw):
    want_h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    q, scale, h = layer_ops.rms_norm_int8(x, w, eps, residual=residual, **kw)
    if residual is None:
        assert h is None
    else:
        assert h.dtype == x.dtype and torch.equal(h, want_h)
    f = want_h.double()
    y = f * w.double() * (f.square().mean(-1, keepdim=True) + eps).rsqrt()
    chain = 32 if x.shape[1] <= 4096 * (16 // x.element_size()) else x.shape[1] / 1024 + 8
    tol = ((chain + 10) / 2 + 6 + 4) * U * 1.01
    _check_rows(q, scale, y, tol, tol + 8 * U)
    return q, scale, h


# One value, vector tails, one warp, several warps, vectors of several per thread, long rows.
WIDTHS = [1, 7, 8, 64, 129, 576, 1001, 1536, 7168, 16384, 40000]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", WIDTHS)
def test_quantize_int8_matches_the_definition(device, dtype, k):
    g = _gen(device, k)
    for m in (1, 5, 67):
        _check_quantize((torch.randn(m, k, generator=g, device=device) * 3).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", WIDTHS)
def test_rms_norm_int8_matches_the_definition(device, dtype, k):
    g = _gen(device, k + 1)
    for m in (1, 5, 67):
        x = torch.randn(m, k, generator=g, device=device).to(dtype)
        r = (torch.randn(m, k, generator=g, device=device) * 4).to(dtype)
        w = (1 + 0.2 * torch.randn(k, generator=g, device=device)).to(dtype)
        _check_norm(x, w)
        _check_norm(x, w, residual=r)


@pytest.mark.parametrize("k", [1536, 40000])
def test_many_rows(device, k):
    g = _gen(device, 3)
    m = 3001
    x = torch.randn(m, k, generator=g, device=device).to(torch.bfloat16)
    w = (1 + 0.2 * torch.randn(k, generator=g, device=device)).to(torch.bfloat16)
    _check_quantize(x)
    _check_norm(x, w, residual=x.flip(0).contiguous())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,offset,stride", [(1536, 0, 2112), (1536, 576, 2112), (100, 1, 103), (513, 3, 520)])
def test_rows_of_a_wider_matrix(device, dtype, k, offset, stride):
    """Strided rows, aligned for 16-byte accesses or not; every tensor with its own strides."""
    g = _gen(device, k + offset)
    wide = [torch.randn(9, stride, generator=g, device=device).to(dtype) for _ in range(3)]
    x, r, out = (t[:, offset:offset + k] for t in wide)
    w = torch.rand(k + 1, generator=g, device=device).to(dtype)[1:]
    before = wide[2].clone()
    _check_quantize(x)
    _check_norm(x, w)
    q, scale, h = _check_norm(x, w, residual=r, residual_out=out)
    assert h is out
    mask = torch.ones_like(before, dtype=torch.bool)
    mask[:, offset:offset + k] = False
    assert torch.equal(wide[2][mask], before[mask]), "only the rows themselves are written"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [1001, 7168, 40000])
def test_residual_updated_in_place(device, dtype, k):
    g = _gen(device, 21)
    x = torch.randn(6, k, generator=g, device=device).to(dtype)
    r = torch.randn(6, k, generator=g, device=device).to(dtype)
    w = torch.rand(k, generator=g, device=device).to(dtype)
    fresh = layer_ops.rms_norm_int8(x, w, residual=r)
    for target in ("residual", "x"):
        a, b = x.clone(), r.clone()
        q, scale, h = layer_ops.rms_norm_int8(a, w, residual=b, residual_out=b if target == "residual" else a)
        assert h is (b if target == "residual" else a)
        assert torch.equal(q, fresh[0]) and torch.equal(scale, fresh[1]) and torch.equal(h, fresh[2])
        assert torch.equal(a if target == "residual" else b, x if target == "residual" else r)


def test_padding_of_odd_rows_is_not_written(device):
    """The library writes k values per row, whatever the row stride."""
    import ctypes

    from triton_mla import _lib
    x = torch.randn(3, 37, device=device)
    q = torch.full((3, 48), 99, dtype=torch.int8, device=device)
    scale = torch.empty(4, device=device).fill_(7.0)
    p = _lib.TmlaInt8RowsParams(x=x.data_ptr(), x_stride=37, q=q.data_ptr(), q_stride=48, scale=scale.data_ptr(), m=3,
                                k=37, dtype=_lib.DTYPE_FP32)
    assert _lib.load().tmla_quantize_int8(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == 0
    assert bool((q[:, 37:] == 99).all()) and float(scale[3]) == 7.0
    assert torch.equal(q[:, :37], layer_ops.quantize_int8(x)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [50, 7168, 40000])
def test_special_rows(device, dtype, k):
    g = _gen(device, 4)
    x = torch.randn(7, k, generator=g, device=device).to(dtype)
    x[0] = 0
    x[1, k // 2] = float("nan")
    x[2, 3] = float("inf")
    x[3, k - 1] = -float("inf")
    x[4] *= 0
    x[4, 5] = torch.finfo(dtype).smallest_normal / 4   # subnormal, and the row's largest
    x[5, 7] = torch.finfo(dtype).max
    w = torch.ones(k, device=device, dtype=dtype)
    q, scale = layer_ops.quantize_int8(x)
    qn, sn, _ = layer_ops.rms_norm_int8(x, w)
    for a, s in ((q, scale), (qn, sn)):
        assert float(s[0]) == TINY and not a[0].any()
        for bad in (1, 2, 3):
            assert bool(torch.isnan(s[bad])) and not a[bad].any(), "no scale for a row with a NaN or an infinity"
        assert bool(torch.isfinite(s[[0, 4, 5, 6]]).all())
    assert int(q[5].abs().max()) == 127 and int(q[6].abs().max()) == 127
    _check_quantize(x[[0, 4, 5, 6]])
    y = layer_ops.linear_int8(q, scale, q[6:7], scale[6:7], torch.float32)
    assert torch.equal(torch.isnan(y[:, 0]).cpu(), torch.tensor([False, True, True, True, False, False, False]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("k", [100, 1001, 7168])
def test_squares_beyond_fp32_make_the_norm_zero(device, dtype, k):
    """The sum of squares is infinite, so 1 / rms is 0; the other rows are as they were."""
    g = _gen(device, k)
    x = torch.randn(3, k, generator=g, device=device).to(dtype)
    x[1] = 1e20
    q, scale, _ = layer_ops.rms_norm_int8(x, torch.ones(k, dtype=dtype, device=device))
    assert not bool(q[1].any()) and float(scale[1]) == 2.0 ** -126
    want_q, want_scale, _ = layer_ops.rms_norm_int8(x[::2].contiguous(), torch.ones(k, dtype=dtype, device=device))
    assert torch.equal(q[::2], want_q) and torch.equal(scale[::2], want_scale)


def test_empty_batches(device):
    x = torch.zeros(0, 64, device=device, dtype=torch.bfloat16)
    q, s = layer_ops.quantize_int8(x)
    assert q.shape == (0, 64) and s.shape == (0,)
    q, s, h = layer_ops.rms_norm_int8(x, torch.ones(64, device=device, dtype=torch.bfloat16), residual=x)
    assert q.shape == (0, 64) and h.shape == (0, 64)
    wq = torch.ones(5, 64, device=device, dtype=torch.int8)
    ws = torch.ones(5, device=device)
    assert layer_ops.linear_int8(q, s, wq, ws).shape == (0, 5)
    assert layer_ops.linear_int8(wq, ws, q, s).shape == (5, 0)


# ----------------------------------------------------------------------------- linear_int8
def _int8(rows, k, g, device, pad=None):
    stride = -(-k // 16) * 16 if pad is None else k + pad
    q = torch.randint(-128, 128, (rows, stride), generator=g, device=device, dtype=torch.int32).to(torch.int8)
    return q[:, :k]


def _check_linear(xq, xs, wq, ws, dtype, **kw):
    y = layer_ops.linear_int8(xq, xs, wq, ws, dtype, **kw)
    assert y.shape == (xq.shape[0], wq.shape[0]) and y.dtype == dtype
    _compare_linear(y, xq, xs, wq, ws)
    return y


def _compare_linear(y, xq, xs, wq, ws):
    dtype = y.dtype
    ref = (xq.double() @ wq.double().T) * xs.double()[:, None] * ws.double()
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    bound = ref.abs() * (half + 3 * U) * 1.01 + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    err = (y.double() - ref).abs()
    # The exact value's own rounding is right in any case (an overflow to infinity among it).
    bad = ~(err <= bound) & (y != ref.to(dtype))
    assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, "
                                 f"worst excess {float((err - bound).max()):.3e}")


# One token, decode batches, odd sizes in each direction, tile borders, batches of several tiles.
LINEAR_SHAPES = [
    (1, 1, 1), (1, 1, 16), (3, 5, 7), (1, 2112, 7168), (16, 7168, 16384), (16, 24576, 1536), (17, 129, 127),
    (33, 257, 129), (64, 1000, 512), (65, 4001, 2001), (100, 640, 16), (128, 128, 128), (129, 300, 1000),
    (255, 256, 300), (257, 513, 640), (500, 2112, 7168), (700, 100, 33), (1000, 999, 1001), (2048, 2112, 1536),
]


@pytest.mark.parametrize("m,n,k", LINEAR_SHAPES)
def test_linear_int8_matches_the_exact_product(device, m, n, k):
    g = _gen(device, m * 7 + n * 3 + k)
    xq, wq = _int8(m, k, g, device), _int8(n, k, g, device)
    xs = torch.rand(m, generator=g, device=device) * 0.02 + 1e-3
    ws = torch.rand(n, generator=g, device=device) * 1e-3 + 1e-5
    for dtype in DTYPES:
        _check_linear(xq, xs, wq, ws, dtype)
    assert read_status(device) == 0


# A small case of every variant (tile of tokens, CTA pairs, parts of k) that the library chooses, then of
# several tiles in a row for each that is not split.
VARIANT_SHAPES = [
    (1, 70, 66), (1, 9097, 2089), (1, 5754, 3398), (1, 3951, 8787), (1, 65, 8320), (17, 64, 80),
    (18, 8471, 3052), (24, 5684, 8484), (17, 71, 15101), (38, 65, 69), (39, 8631, 2514), (33, 5659, 3758),
    (34, 4091, 9255), (34, 70, 11457), (51, 75, 74), (3958, 65, 2550), (2372, 77, 2556), (1689, 81, 4931),
    (1173, 75, 8145), (72, 9497, 65), (6569, 87, 4202), (3391, 72, 7144), (3031, 68, 4511), (1783, 65, 15182),
    (114, 10078, 73), (7297, 65, 6314), (4782, 70, 4879), (3854, 87, 11186), (2162, 66, 12903), (134, 9547, 72),
    (3625, 365, 5775), (7118, 78, 10075), (4737, 70, 8667), (3215, 72, 12171), (483, 5081, 66),
    (4176, 307, 11977), (7899, 70, 9850), (6301, 72, 10216), (5919, 582, 64), (5333, 350, 13902),
    (7339, 75, 12801), (235, 14703, 74), (17, 22440, 6245), (17, 64, 916), (1, 66, 1411), (1, 71, 1927),
    (55, 20334, 3559), (1426, 75, 1424), (44, 64, 1827), (33, 70, 2955), (5343, 144, 4076), (2890, 69, 2424),
    (72, 4972, 2275), (1417, 64, 10880), (7684, 136, 2953), (3332, 149, 3462), (2149, 144, 5372),
    (746, 260, 9712), (131, 10624, 2419), (4780, 147, 3674), (3256, 129, 5229), (132, 2933, 7316),
    (163, 10646, 2141), (5776, 143, 4765), (2077, 412, 4822), (185, 3178, 10614), (211, 11068, 1768),
    (3147, 259, 6803), (4369, 136, 10008), (644, 1090, 10071), (235, 20162, 1012), (1422, 1072, 7063),
    (2680, 276, 9137), (233, 3468, 14580), (170, 20273, 92), (223, 23140, 77), (319, 19197, 74),
    (340, 24364, 67), (441, 20197, 74), (678, 16360, 74), (269, 23382, 770), (357, 20186, 654),
    (7849, 1322, 658), (3877, 3111, 719),
    (7, 8465, 7363), (1, 5743, 11131), (22, 8773, 8607), (18, 66, 16005), (47, 8535, 10130), (45, 5640, 12628),
    (1446, 69, 5406), (972, 66, 8517), (2082, 274, 5875), (2862, 73, 16210), (4345, 75, 11772),
    (3708, 70, 16189), (474, 2943, 10323), (5853, 65, 16150), (4674, 119, 16191), (514, 3015, 14526),
    (5480, 124, 16720), (421, 4734, 16695), (22, 20313, 11209), (524, 808, 4976), (707, 340, 9612),
    (1092, 857, 5245), (797, 823, 4691), (709, 546, 10453), (531, 1649, 5748), (908, 516, 11792),
    (1310, 1259, 7589), (1117, 780, 9094), (1464, 1172, 9467), (1021, 1069, 9215),
]


@pytest.mark.parametrize("m,n,k", VARIANT_SHAPES)
def test_linear_int8_variants(device, m, n, k):
    g = _gen(device, m + n + k)
    xq, wq = _int8(m, k, g, device), _int8(n, k, g, device)
    xs = torch.rand(m, generator=g, device=device) * 0.01 + 1e-3
    ws = torch.rand(n, generator=g, device=device) * 1e-3 + 1e-5
    for dtype in DTYPES:
        _check_linear(xq, xs, wq, ws, dtype)
    assert read_status(device) == 0


# The variants that the shapes above leave out, of fp32 output most of all: larger tiles of CTA pairs, split or not, and two
# and three tiles in a row of each (``test_int8_host`` checks that the lists reach every variant of either output size).
MORE_VARIANT_SHAPES = [
    (38, 19579, 66), (54, 19048, 5624), (66, 20867, 68), (73, 20347, 3639), (105, 20043, 66),
    (105, 20832, 2767), (135, 19542, 68), (193, 9671, 1834), (196, 3393, 10864), (224, 19019, 904),
    (233, 19641, 813), (271, 4648, 13396), (282, 19390, 1374), (291, 10444, 1167), (332, 18948, 820),
    (337, 15087, 65), (385, 2856, 8943), (400, 14673, 64), (417, 20003, 781), (524, 8343, 778), (673, 9756, 67),
    (1597, 278, 5487), (2052, 280, 5766), (2458, 1896, 774), (3458, 3063, 777),
]


@pytest.mark.parametrize("m,n,k", MORE_VARIANT_SHAPES)
def test_linear_int8_more_variants(device, m, n, k):
    test_linear_int8_variants(device, m, n, k)


@pytest.mark.parametrize("m,n,k,pad", [(5, 40, 100, 1), (70, 130, 257, 0), (16, 300, 1001, 2), (300, 65, 80, 3)])
def test_linear_int8_rows_of_any_alignment(device, m, n, k, pad):
    """Rows that do not start on 16-byte boundaries (x, w or both) give the same values."""
    g = _gen(device, 17)
    xs, ws = torch.rand(m, generator=g, device=device) * 0.01, torch.rand(n, generator=g, device=device) * 0.01
    aligned = _int8(m, k, g, device), _int8(n, k, g, device)
    y = _check_linear(aligned[0], xs, aligned[1], ws, torch.float32)
    x_odd, w_odd = _int8(m, k, g, device, pad), _int8(n, k, g, device, pad)
    x_odd.copy_(aligned[0])
    w_odd.copy_(aligned[1])
    for xq, wq in ((x_odd, aligned[1]), (aligned[0], w_odd), (x_odd, w_odd)):
        assert torch.equal(layer_ops.linear_int8(xq, xs, wq, ws, torch.float32), y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(5, 33, 64), (70, 1001, 300), (300, 515, 257), (600, 1027, 128), (64, 130, 7168)])
def test_linear_int8_into_rows_of_any_stride(device, dtype, m, n, k):
    """The library's y may have any row stride and start (here an odd one, and a column inside wider
    rows); nothing beside its rows is written."""
    import ctypes

    from triton_mla import _lib
    g = _gen(device, n)
    xq, wq = _int8(m, k, g, device), _int8(n, k, g, device)
    xs, ws = torch.rand(m, generator=g, device=device), torch.rand(n, generator=g, device=device)
    codes = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}
    for first, stride in ((0, n), (1, n + 6), (3, n + 9), (8, -(-n // 8) * 8 + 16)):
        buf = torch.full((m * stride + 64,), 7.0, device=device, dtype=dtype)
        y = torch.as_strided(buf, (m, n), (stride, 1), first)
        p = _lib.TmlaLinearInt8Params(xq.data_ptr(), xq.stride(0), xs.data_ptr(), wq.data_ptr(), wq.stride(0),
                                      ws.data_ptr(), y.data_ptr(), stride, m, n, k, codes[dtype], 0, None, 0)
        stream = torch.cuda.current_stream(device).cuda_stream
        assert _lib.load().tmla_linear_int8(ctypes.byref(p), ctypes.c_void_p(stream)) == 0
        _compare_linear(y, xq, xs, wq, ws)
        mask = torch.ones_like(buf, dtype=torch.bool)
        torch.as_strided(mask, (m, n), (stride, 1), first).fill_(False)
        assert bool((buf[mask] == 7.0).all()), "only y's rows are written"


@pytest.mark.parametrize("m", [4, 300])
def test_linear_int8_sums_that_fill_int32_are_exact(device, m):
    """All operands -128: the sum is k 2^14, at the longest k one step below 2^31."""
    k = 131071
    xq = torch.full((m, k + 1), -128, dtype=torch.int8, device=device)[:, :k]
    wq = torch.full((130, k + 1), -128, dtype=torch.int8, device=device)[:, :k]
    y = layer_ops.linear_int8(xq, torch.ones(m, device=device), wq, torch.ones(130, device=device), torch.float32)
    want = torch.full((m, 130), k * 16384, dtype=torch.float64, device=device).float()
    assert torch.equal(y, want)
    with pytest.raises(AssertionError):
        big = torch.zeros(1, 131072, dtype=torch.int8, device=device)
        layer_ops.linear_int8(big, torch.ones(1, device=device), big, torch.ones(1, device=device))


def test_linear_int8_refuses_bad_operands(device):
    q = torch.zeros(4, 64, dtype=torch.int8, device=device)
    s = torch.ones(4, device=device)
    for bad in ((q.float(), s, q, s), (q, s[:3], q, s), (q, s, q[:, :32], s), (q, s.double(), q, s), (q[0], s, q, s)):
        with pytest.raises(AssertionError):
            layer_ops.linear_int8(*bad)
    with pytest.raises(TypeError):
        layer_ops.linear_int8(q, s, q, s, torch.float64)
    with pytest.raises(AssertionError):
        layer_ops.linear_int8(q.T[:4, :4], s, q[:, :4], s)   # columns, not rows
    with pytest.raises(AssertionError):
        layer_ops.linear_int8(q, torch.ones(8, device=device)[::2], q, s)
    with pytest.raises(RuntimeError):
        layer_ops.linear_int8(q, s, q.cpu(), s)
    with pytest.raises(TypeError):
        layer_ops.quantize_int8(q.double())
    with pytest.raises(AssertionError):
        layer_ops.quantize_int8(torch.zeros(4, 4, device=device).T[:2])
    with pytest.raises(AssertionError):
        layer_ops.rms_norm_int8(torch.zeros(4, 8, device=device), torch.ones(9, device=device))
    with pytest.raises(AssertionError):
        layer_ops.rms_norm_int8(torch.zeros(4, 8, device=device), torch.ones(8, device=device),
                                residual_out=torch.zeros(4, 8, device=device))


def test_offsets_beyond_32_bits(device):
    """Rows and outputs past 2^31 elements: the last rows equal those of a call on them alone."""
    g = _gen(device, 40)
    m, k = 140001, 16384                                   # 2.3e9 values
    x = torch.randn(64, k, generator=g, device=device).to(torch.bfloat16).repeat(m // 64 + 1, 1)[:m]
    x[-5:] = torch.randn(5, k, generator=g, device=device).to(torch.bfloat16)
    w = torch.ones(k, device=device, dtype=torch.bfloat16)
    for call in (lambda t: layer_ops.quantize_int8(t), lambda t: layer_ops.rms_norm_int8(t, w, residual=t)):
        got, want = call(x), call(x[-5:].contiguous())
        for a, b in zip(got, want):
            assert torch.equal(a[-5:], b)
        del got
    q, s = layer_ops.quantize_int8(x[-5:, :128].contiguous())
    xq = q.repeat(14001, 1)                                # 70005 tokens x 33000 channels: 2.3e9 products
    wq, ws = _int8(33000, 128, g, device), torch.rand(33000, generator=g, device=device)
    y = layer_ops.linear_int8(xq, s.repeat(14001), wq, ws)
    _compare_linear(y[-5:], q, s, wq, ws)
    _compare_linear(y[:5], q, s, wq, ws)
    wide = torch.zeros(20, (1 << 27) + 16, dtype=torch.int8, device=device)   # rows 2^27 apart: 2.7e9 bytes
    wide[:, :128] = wq[:20]
    _compare_linear(layer_ops.linear_int8(q, s, wide[:, :128], ws[:20]), q, s, wq[:20], ws[:20])
    _compare_linear(layer_ops.linear_int8(wide[:, :128], ws[:20], q, s), wq[:20], ws[:20], q, s)
    odd = wide.view(-1)[: 19 * ((1 << 27) + 15) + 128].as_strided((20, 128), ((1 << 27) + 15, 1))
    odd.copy_(wq[:20])
    _compare_linear(layer_ops.linear_int8(q, s, odd, ws[:20]), q, s, wq[:20], ws[:20])


# ----------------------------------------------------------------------------- used together
class _Layer:
    """An MLA layer's decode step with int8 projections: the operators as a serving loop uses them."""

    def __init__(self, device, batch, heads, hidden, seed, dtype=torch.bfloat16):
        self.heads, self.dn, self.dr, self.dv, self.rank, self.q_rank = heads, 128, 64, 128, 512, 384
        self.page, pages = 64, 4
        g = _gen(device, seed)

        def weight(n, k):
            return (torch.randn(n, k, generator=g, device=device) * k ** -0.5).to(dtype)

        def norm(k):
            return (1 + 0.1 * torch.randn(k, generator=g, device=device)).to(dtype)

        self.w_a = layer_ops.quantize_int8(weight(self.q_rank + self.rank + self.dr, hidden))
        self.wq_b = layer_ops.quantize_int8(weight(heads * (self.dn + self.dr), self.q_rank))
        self.wo = layer_ops.quantize_int8(weight(hidden, heads * self.dv))
        self.wkv_b = weight(heads * (self.dn + self.dv), self.rank)
        self.norm_in, self.q_norm, self.kv_norm = norm(hidden), norm(self.q_rank), norm(self.rank)
        self.x = torch.randn(batch, hidden, generator=g, device=device).to(dtype)
        self.residual = torch.randn(batch, hidden, generator=g, device=device).to(dtype)
        self.bt = torch.randperm(batch * pages, generator=g, device=device).view(batch, pages).int()
        self.cache = torch.randn(batch * pages, self.page, self.rank + self.dr, generator=g, device=device).to(dtype)
        self.lens = torch.randint(0, pages * self.page - 1, (batch,), generator=g, device=device, dtype=torch.int32)

    def step(self, overlap):
        q, s, h = layer_ops.rms_norm_int8(self.x, self.norm_in, residual=self.residual)
        both = layer_ops.linear_int8(q, s, *self.w_a, overlap=overlap)
        qa, kva = both.split([self.q_rank, self.rank + self.dr], dim=-1)
        seqlens = torch.empty_like(self.lens)
        layer_ops.kv_norm_rope_append(kva, self.kv_norm, self.lens, self.cache, self.bt, 1e-6, 10000.0,
                                      seqlens_out=seqlens, overlap=overlap)
        qn, sn, _ = layer_ops.rms_norm_int8(qa, self.q_norm, overlap=overlap)
        qb = layer_ops.linear_int8(qn, sn, *self.wq_b, overlap=overlap)
        full = layer_ops.q_absorb_rope(qb.view(-1, self.heads, self.dn + self.dr), self.wkv_b, self.lens, self.dn,
                                       self.dv, 10000.0, overlap=overlap)
        o = mla_decode(full, self.cache, seqlens, self.bt, softmax_scale=192 ** -0.5, num_splits=1)
        o = layer_ops.o_unabsorb(o, self.wkv_b, self.dn, self.dv, overlap=overlap)
        oq, os = layer_ops.quantize_int8(o, overlap=overlap)
        y = layer_ops.linear_int8(oq, os, *self.wo, overlap=overlap)
        return dict(q=q, s=s, h=h, both=both, qn=qn, sn=sn, qb=qb, o=o, oq=oq, os=os, y=y)


@pytest.mark.parametrize("batch", [1, 13, 80])
def test_a_layer_step_with_int8_projections(device, batch):
    layer = _Layer(device, batch, 16, 1024, seed=batch)
    out = layer.step(overlap=False)
    torch.cuda.synchronize()
    assert read_status(device) == 0
    _compare_linear(out["both"], out["q"], out["s"], *layer.w_a)
    _compare_linear(out["qb"], out["qn"], out["sn"], *layer.wq_b)
    _compare_linear(out["y"], out["oq"], out["os"], *layer.wo)
    _check_norm(out["both"][:, :layer.q_rank], layer.q_norm)
    _check_rows(out["oq"], out["os"], out["o"].double(), U * 1.01, 3 * U * 1.01)
    # As programmatic launches, and in a captured graph, the same bits.
    for got in (layer.step(overlap=True), _captured(layer)):
        for name in out:
            assert torch.equal(got[name], out[name]), name


def _captured(layer):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step(overlap=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.step(overlap=True)
    for t in got.values():
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    return {name: t.clone() for name, t in got.items()}


def test_two_graphs_and_two_streams_at_once(device):
    """Calls keep nothing between them: two captured graphs replayed on two streams at the same
    time, over and over, and an eager call beside them, each give their own result."""
    g = _gen(device, 31)
    jobs = []
    for m, n, k in ((16, 2112, 7168), (40, 1536, 4096)):
        xq, wq = _int8(m, k, g, device), _int8(n, k, g, device)
        xs, ws = torch.rand(m, generator=g, device=device), torch.rand(n, generator=g, device=device)
        want = layer_ops.linear_int8(xq, xs, wq, ws, torch.float32)
        _compare_linear(want, xq, xs, wq, ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer_ops.linear_int8(xq, xs, wq, ws, torch.float32)
        jobs.append((graph, y, want, (xq, xs, wq, ws), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, y, want, args, stream in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
        eager = layer_ops.linear_int8(*jobs[0][3], torch.float32)
        torch.cuda.synchronize()
        assert torch.equal(eager, jobs[0][2])
        for graph, y, want, _, _ in jobs:
            assert torch.equal(y, want)
            y.zero_()
        torch.cuda.synchronize()


def test_first_calls_inside_a_capture(device):
    """A process whose first calls are captured: nothing has to be set up before."""
    import subprocess
    import sys

    from conftest import ROOT
    code = """
import torch
from triton_mla import layer_ops, read_status
x = torch.randn(40, 512, device="cuda", dtype=torch.bfloat16)
w = torch.ones(512, device="cuda", dtype=torch.bfloat16)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    q, s, h = layer_ops.rms_norm_int8(x, w, residual=x)
    y = layer_ops.linear_int8(q, s, q, s, torch.float32)
graph.replay()
torch.cuda.synchronize()
q2, s2, _ = layer_ops.rms_norm_int8(x, w, residual=x)
assert torch.equal(q, q2) and torch.equal(y, layer_ops.linear_int8(q2, s2, q2, s2, torch.float32))
assert read_status() == 0
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT / "triton-mla_b200", capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


def test_calls_on_another_stream(device):
    """The operators run on the current stream, and wait there for what came before on it."""
    g = _gen(device, 33)
    x = torch.randn(300, 7168, generator=g, device=device).to(torch.bfloat16)
    w = torch.ones(7168, device=device, dtype=torch.bfloat16)
    wq, ws = layer_ops.quantize_int8(torch.randn(512, 7168, generator=g, device=device))
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    late = torch.zeros_like(x)
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)          # about 10 ms before x is there
        late.copy_(x)
        q, s, h = layer_ops.rms_norm_int8(late, w, residual=late, overlap=True)
        y = layer_ops.linear_int8(q, s, wq, ws, overlap=True)
    stream.synchronize()
    want = layer_ops.rms_norm_int8(x, w, residual=x)
    assert torch.equal(q, want[0]) and torch.equal(s, want[1]) and torch.equal(h, want[2])
    assert torch.equal(y, layer_ops.linear_int8(want[0], want[1], wq, ws))


def test_a_weight_written_just_before(device):
    """Without ``overlap`` the kernel before may write the weight (it is quantised in the same stream)."""
    g = _gen(device, 34)
    x, s = _int8(16, 4096, g, device), torch.rand(16, generator=g, device=device)
    for i in range(10):
        w = torch.randn(2048, 4096, generator=g, device=device).to(torch.bfloat16)
        torch.cuda.synchronize()
        wq, ws = layer_ops.quantize_int8(w)
        y = layer_ops.linear_int8(x, s, wq, ws)
        torch.cuda.synchronize()
        assert torch.equal(y, layer_ops.linear_int8(x, s, wq, ws))
        _compare_linear(y, x, s, wq, ws)


@pytest.mark.parametrize("m,n,k", [(16, 2112, 7168), (256, 2048, 4096), (600, 4096, 1024)])
def test_a_weight_written_two_kernels_before(device, m, n, k):
    """With ``overlap`` only the kernel just before may not write the weight: one product (with another weight) lies
    between the quantisation of the weight and its product, which loads it ahead of its wait."""
    g = _gen(device, 35)
    x1, s1 = _int8(m, k, g, device), torch.rand(m, generator=g, device=device)
    w1, v1 = _int8(n, k, g, device), torch.rand(n, generator=g, device=device)
    x2, s2 = _int8(16, 1536, g, device), torch.rand(16, generator=g, device=device)
    for i in range(20):
        w = torch.randn(24576, 1536, generator=g, device=device).to(torch.bfloat16)
        torch.cuda.synchronize()
        w2, v2 = layer_ops.quantize_int8(w)
        y1 = layer_ops.linear_int8(x1, s1, w1, v1)
        y2 = layer_ops.linear_int8(x2, s2, w2, v2, overlap=True)
        torch.cuda.synchronize()
        assert torch.equal(y2, layer_ops.linear_int8(x2, s2, w2, v2))
        if i == 0:
            _compare_linear(y1, x1, s1, w1, v1)
            _compare_linear(y2, x2, s2, w2, v2)


def test_no_gradient_passes(device):
    x = torch.randn(4, 64, device=device, requires_grad=True)
    w = torch.ones(64, device=device, requires_grad=True)
    q, s, h = layer_ops.rms_norm_int8(x, w, residual=x)
    assert not s.requires_grad and not h.requires_grad
    assert not layer_ops.quantize_int8(x)[1].requires_grad
    y = torch.randn(4, 64, device=device)
    version = y._version
    layer_ops.rms_norm_int8(y, w.detach(), residual=y, residual_out=y)
    assert y._version > version, "a write in place is seen by autograd"


def test_int8_operators_compile_without_a_graph_break(device):
    def f(x, r, w, wq, ws):
        q, s, h = layer_ops.rms_norm_int8(x, w, residual=r)
        return layer_ops.linear_int8(q, s, wq, ws), h

    g = _gen(device, 8)
    x, r = (torch.randn(5, 200, generator=g, device=device).to(torch.bfloat16) for _ in range(2))
    w = torch.ones(200, device=device, dtype=torch.bfloat16)
    wq, ws = layer_ops.quantize_int8(torch.randn(70, 200, generator=g, device=device))
    for got, want in zip(torch.compile(f, fullgraph=True, backend="aot_eager")(x, r, w, wq, ws), f(x, r, w, wq, ws)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("m,n,k", [(16, 2112, 7168), (300, 700, 1024), (40, 130, 100)])
def test_a_timed_out_wait_returns_cleanly(device, m, n, k):
    """A bounded wait that runs out (the test-only stall: the first CTA never loads its first
    stage) sets TMLA_STATUS_TIMEOUT and the kernel returns; the tiles of the other CTAs are right,
    the stalled one's are left unwritten, and the next call is exact."""
    import ctypes

    from triton_mla import _lib
    from triton_mla.kernel import _status_word

    g = _gen(device, 11)
    xq, wq = _int8(m, k, g, device), _int8(n, k, g, device)
    xs, ws = torch.rand(m, generator=g, device=device), torch.rand(n, generator=g, device=device)
    y = torch.full((m, n), float("nan"), device=device)
    p = _lib.TmlaLinearInt8Params(xq.data_ptr(), xq.stride(0), xs.data_ptr(), wq.data_ptr(), wq.stride(0), ws.data_ptr(),
                                  y.data_ptr(), n, m, n, k, _lib.DTYPE_FP32, _lib.LINEAR_FLAG_TEST_STALL,
                                  _status_word(device).data_ptr(), 20_000_000)
    stream = ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)
    read_status(device)
    assert _lib.load().tmla_linear_int8(ctypes.byref(p), stream) == 0
    torch.cuda.synchronize()
    assert read_status(device) == _lib.STATUS_TIMEOUT
    ref = (xq.double() @ wq.double().T) * xs.double()[:, None] * ws.double()
    missing = torch.isnan(y)
    assert bool(missing[0, 0]) and bool(((y.double() - ref).abs()[~missing] <= ref.abs()[~missing] * 4 * U).all())
    p.flags = 0
    assert _lib.load().tmla_linear_int8(ctypes.byref(p), stream) == 0
    torch.cuda.synchronize()
    assert read_status(device) == 0
    _compare_linear(y, xq, xs, wq, ws)


@pytest.mark.parametrize("m,n,k", [(1, 64, 7211), (10, 2488, 1186), (1, 64, 1150), (16, 2112, 7168), (130, 1000, 4000)])
def test_timed_out_parts_of_a_split_tile(device, m, n, k):
    """A cluster whose first CTA gives up: the parts that the others send to it, and it to them, are late or never
    come.  The next call, launched right behind, runs on the same SMs and is exact, time after time."""
    import ctypes

    from triton_mla import _lib
    from triton_mla.kernel import _status_word

    g = _gen(device, 12)
    xq, wq = _int8(m, k, g, device), _int8(n, k, g, device)
    xs, ws = torch.rand(m, generator=g, device=device), torch.rand(n, generator=g, device=device)
    y, y2 = torch.empty(m, n, device=device), torch.empty(m, n, device=device)
    args = [xq.data_ptr(), xq.stride(0), xs.data_ptr(), wq.data_ptr(), wq.stride(0), ws.data_ptr()]
    stalled = _lib.TmlaLinearInt8Params(*args, y.data_ptr(), n, m, n, k, _lib.DTYPE_FP32, _lib.LINEAR_FLAG_TEST_STALL,
                                        _status_word(device).data_ptr(), 300_000)
    whole = _lib.TmlaLinearInt8Params(*args, y2.data_ptr(), n, m, n, k, _lib.DTYPE_FP32, 0, None, 0)
    stream = ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)
    read_status(device)
    for _ in range(20):
        y2.zero_()
        assert _lib.load().tmla_linear_int8(ctypes.byref(stalled), stream) == 0
        assert _lib.load().tmla_linear_int8(ctypes.byref(whole), stream) == 0
        torch.cuda.synchronize()
        assert read_status(device) == _lib.STATUS_TIMEOUT
        _compare_linear(y2, xq, xs, wq, ws)


@pytest.mark.parametrize("m,n,k", [(1, 64, 7211), (16, 2112, 7168), (300, 520, 1024), (5, 40, 99)])
def test_linear_int8_scales_without_a_value(device, m, n, k):
    """A token or channel whose scale is infinite or NaN (a row without one) has no finite product, in split tiles, in
    whole ones and in rows of y off 16-byte boundaries; the others are exact."""
    g = _gen(device, 41)
    xq, wq = _int8(m, k, g, device), _int8(n, k, g, device)
    xs, ws = torch.rand(m, generator=g, device=device) + 0.01, torch.rand(n, generator=g, device=device) + 0.01
    for dtype in DTYPES:
        want = layer_ops.linear_int8(xq, xs, wq, ws, dtype)
        bad_x, bad_w = xs.clone(), ws.clone()
        bad_x[m - 1], bad_w[1], bad_w[n - 1] = float("nan"), float("inf"), float("nan")
        assert bool(torch.isnan(layer_ops.linear_int8(xq, bad_x, wq, ws, dtype)[m - 1]).all())
        if m > 1:
            assert torch.equal(layer_ops.linear_int8(xq, bad_x, wq, ws, dtype)[: m - 1], want[: m - 1])
        y = layer_ops.linear_int8(xq, xs, wq, bad_w, dtype)
        assert not bool(torch.isfinite(y[:, [1, n - 1]]).any())
        assert torch.equal(y[:, 2:n - 1], want[:, 2:n - 1]) and torch.equal(y[:, 0], want[:, 0])
    assert read_status(device) == 0


def test_an_in_place_residual_under_torch_compile(device):
    def f(x, r, w):
        q, s, h = layer_ops.rms_norm_int8(x, w, residual=r, residual_out=r)
        return q, s, h + 1

    g = _gen(device, 42)
    x, r = (torch.randn(5, 200, generator=g, device=device).to(torch.bfloat16) for _ in range(2))
    w = torch.ones(200, device=device, dtype=torch.bfloat16)
    r1, r2 = r.clone(), r.clone()
    got, want = torch.compile(f, fullgraph=True, backend="aot_eager")(x, r1, w), f(x, r2, w)
    assert torch.equal(r1, r2) and torch.equal(r1, x + r)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_of_another_device_than_the_current_one(device):
    other = torch.device("cuda", 1)
    g = _gen(other, 43)
    x = torch.randn(9, 1001, generator=g, device=other)
    w = torch.ones(1001, device=other)
    wq, ws = layer_ops.quantize_int8(torch.randn(70, 1001, generator=g, device=other))
    with torch.cuda.device(0):
        q, s, h = layer_ops.rms_norm_int8(x, w, residual=x)
        y = layer_ops.linear_int8(q, s, wq, ws, torch.float32)
        assert torch.cuda.current_device() == 0
    assert {t.device for t in (q, s, h, y)} == {other}
    torch.cuda.synchronize(other)
    _compare_linear(y, q, s, wq, ws)
    assert read_status(other) == 0
