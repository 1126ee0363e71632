"""8-bit serving operators (``ops/int8.py``, ``csrc/int8.hip``): the oracle against the formulas in 64 bits (CPU), the
kernels against the same (GPU), refusals, layouts, streams and graphs.

Error bounds used below (u = 2^-24, half a step of fp32):

* a code: ``x * 127 / top`` is made with one rounded division, so it is off by at most 127 u before it is rounded;
* a scale: one rounded division;
* the norm: squares of one sign are summed by at most 8 chunks of 8 elements a thread, 6 + 4 steps across threads (rows
  longer than 32768: one partial sum of K / 1024 elements a thread), the root halves that error and about 8 roundings
  follow: at most (64 + 16 + 24) / 2 + 12 = 64 u = 2^-18 of each value for the lengths tested here;
* the product: the integer sum is rounded once to fp32, multiplied twice, the bias added: 3 u of the product and one u of
  the result (4 and 2 are allowed); tanh adds at most 5 steps of fp32; the output type's own half step comes last.
"""
import math

import pytest
import torch

from d4pg_pytorch_amd import ops
from d4pg_pytorch_amd.ops import ref

U = 2.0 ** -24
NORM = 2.0 ** -18
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
#: smallest half step: below the normal range a rounding is off by a constant
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(*shape, seed=0):
    return torch.randn(*shape, generator=_gen(seed))


def _codes(rows, K, device, seed, garbage=True, offset=0):
    """Random codes [rows, K] whose padding bytes hold anything, and scales."""
    g = _gen(seed)
    kp = (K + 15) // 16 * 16
    buf = torch.randint(-127, 128, (rows, kp), generator=g, dtype=torch.int8) if garbage else torch.zeros(rows, kp, dtype=torch.int8)
    buf[:, :K] = torch.randint(-127, 128, (rows, K), generator=g, dtype=torch.int8)
    return buf.to(device)[:, :K], (torch.rand(rows, generator=g) * 0.02 + 1e-3).to(device)


def _check_codes(q, scale, y, rel):
    """``q``, ``scale`` against the 64-bit rows ``y`` whose own error is at most ``rel`` of each value."""
    q, scale, y = q.double().cpu(), scale.double().cpu(), y.double().cpu()
    top = y.abs().amax(1)
    assert torch.all((scale - top / 127).abs() <= (rel + 2 * U) * top / 127 + 2.0 ** -149)
    v = torch.where(top[:, None] > 0, y * 127 / torch.where(top > 0, top, 1.0)[:, None], 0.0)
    off = (q - v).abs() - 0.5 - 127 * (2 * rel + 2 * U)
    assert torch.all(off <= 0), f"a code is off by {off.max().item() + 0.5}"
    assert torch.all(q.abs() <= 127)


# ---------------------------------------------------------------------------------------------------- quantize_rows
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 2), (1, 7), (5, 8), (2, 9), (4, 15), (3, 16), (2, 17), (257, 24), (4, 111), (3, 400),
                                 (2, 512), (2, 513), (2, 1024), (3, 1111), (2, 2048), (2, 2049), (1, 4096), (2, 4099),
                                 (2, 8192), (2, 8200), (1, 16384), (2, 16391), (1, 32768)])
def test_quantize_rows(M, K, dtype, device):
    x = (_randn(M, K, seed=M * 31 + K) * torch.exp(2 * _randn(M, 1, seed=5))).to(dtype).to(device)
    q, scale = ops.quantize_rows(x)
    assert q.dtype == torch.int8 and q.shape == (M, K) and scale.dtype == torch.float32 and scale.shape == (M,)
    _check_codes(q, scale, x, 0.0)
    assert q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0 or M == 1


@pytest.mark.parametrize("device", DEVICES)
def test_quantize_rows_beyond_the_registers(device):
    x = _randn(2, 70001, seed=3).to(device)
    q, scale = ops.quantize_rows(x)
    _check_codes(q, scale, x, 0.0)


@pytest.mark.parametrize("device", DEVICES)
def test_quantize_padding_is_zero_and_neighbours_stay(device):
    q, _ = ops.quantize_rows(_randn(6, 21).to(device))
    assert q.stride() == (32, 1) and torch.all(torch.as_strided(q, (6, 32), (32, 1))[:, 21:] == 0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("K", [5, 40, 700, 3000, 9000])
def test_quantize_rows_that_are_not_ordinary(K, device):
    x = _randn(9, K, seed=K)
    x[0] = 0.0
    x[1, K // 2] = math.nan
    x[2, 0] = math.inf
    x[3, K - 1] = -math.inf
    x[4] *= 1e-38
    x[5] = 0.0
    x[5, K - 1] = 2.0 ** -149                       # the smallest number there is
    x[6] = torch.finfo(torch.float32).max
    x[7] = -0.0
    x[8] = 0.0
    x[8, 0], x[8, 1] = 254.0, 1.0                    # exactly half a code: to the even one
    q, scale = ops.quantize_rows(x.to(device))
    q, scale = q.cpu(), scale.cpu()
    for r in (0, 7):
        assert scale[r] == 0 and torch.all(q[r] == 0)
    for r in (1, 2, 3):
        assert torch.isnan(scale[r]) and torch.all(q[r] == 0)
    assert q[5, K - 1] == 127
    assert q[8, 0] == 127 and q[8, 1] == 0
    _check_codes(q[[4, 6]], scale[[4, 6]], x[[4, 6]], 0.0)
    back = ops.dequantize_rows(q.to(device), scale.to(device)).cpu()
    assert torch.isnan(back[1:4]).all() and torch.all(back[0] == 0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_other_layouts(dtype, device):
    base = _randn(40, 90, seed=8).to(dtype).to(device)
    for x in (base[:, 3:50], base[::2, 1:], base.t(), base[5:6].expand(4, 90), base.view(4, 10, 90)[:, :, ::2],
              base.view(5, 8, 90), base[0], base[:, 7:8]):
        q, scale = ops.quantize_rows(x)
        assert q.shape == x.shape and scale.shape == x.shape[:-1]
        _check_codes(q.reshape(-1, x.shape[-1]), scale.reshape(-1), x.reshape(-1, x.shape[-1]), 0.0)


# -------------------------------------------------------------------------------------------------- dequantize_rows
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (7, 3), (3, 8), (2, 17), (300, 24), (5, 400), (3, 2047), (2, 5000)])
def test_dequantize_rows(M, K, dtype, device):
    q, scale = _codes(M, K, device, seed=M + K)
    out = ops.dequantize_rows(q, scale, dtype)
    assert out.dtype == dtype and out.shape == (M, K)
    want = q.double() * scale.double()[:, None]
    assert torch.all((out.double() - want).abs() <= (U + HALF[dtype]) * 1.01 * want.abs() + TINY[dtype])
    # other layouts: shifted, transposed, strided
    for p, s in ((q[:, K // 2:], scale), (q.t().contiguous().t(), scale), (q[::2], scale[::2])):
        got = ops.dequantize_rows(p, s, dtype)
        want = p.double() * s.double()[:, None]
        assert torch.all((got.double() - want).abs() <= (U + HALF[dtype]) * 1.01 * want.abs() + TINY[dtype])


# ------------------------------------------------------------------------------------------------ add_rms_norm_int8
def _norm64(x, weight, residual, eps):
    h = x.double() if residual is None else x.double() + residual.double()
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    return h, y if weight is None else y * weight.double()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,add,wtype", [(1, 1, True, "same"), (2, 5, False, None), (3, 8, True, "fp32"), (130, 24, True, "same"),
                                           (5, 111, False, "same"), (4, 400, True, "same"), (2, 513, True, None),
                                           (3, 1111, False, "fp32"), (1, 2048, True, "same"), (2, 4096, True, "same"),
                                           (2, 4103, True, "fp32"), (2, 8192, False, "same"), (2, 16384, True, "same"),
                                           (1, 20001, True, "same"), (33, 128, True, "fp32"), (19, 129, True, None), (300, 250, True, "same"),
                                           (257, 5003, True, "same"), (300, 9001, False, "fp32"), (2, 33001, True, "fp32"), (2, 40008, True, None)])
def test_add_rms_norm_int8(M, K, add, wtype, dtype, device):
    x = _randn(M, K, seed=K).to(dtype).to(device)
    r = (3 * _randn(M, K, seed=K + 1)).to(dtype).to(device) if add else None
    w = None if wtype is None else (1 + 0.3 * _randn(K, seed=2)).to(torch.float32 if wtype == "fp32" else dtype).to(device)
    q, scale, h = ops.add_rms_norm_int8(x, w, r, 1e-5)
    h64, y64 = _norm64(x, w, r, 1e-5)
    _check_codes(q, scale, y64, NORM)
    if add:
        assert h.dtype == dtype and h.shape == (M, K)
        assert torch.all((h.double() - h64).abs() <= (U + HALF[dtype]) * 1.01 * h64.abs() + TINY[dtype])
    else:
        assert h is x


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("K", [6, 200, 3001, 40000])
def test_norm_rows_that_are_not_ordinary(K, device):
    """Squares that leave fp32, rows of zeros, non-finite rows; with and without an added eps."""
    x = _randn(8, K, seed=K)
    x[0] = 0.0
    x[1, K // 3] = math.nan
    x[2, K - 1] = math.inf
    x[3] *= 1e25
    x[4] *= 1e-25
    x[5] *= 1e30
    x[6] *= 1e-39
    for eps in (1e-6, 0.0):
        q, scale, _ = ops.add_rms_norm_int8(x.to(device), None, None, eps)
        q, scale = q.cpu(), scale.cpu()
        assert scale[0] == 0 and torch.all(q[0] == 0)
        assert torch.isnan(scale[1:3]).all() and torch.all(q[1:3] == 0)
        rows = [3, 5, 7] + ([4, 6] if eps == 0.0 else [4])
        _check_codes(q[rows], scale[rows], _norm64(x, None, None, eps)[1][rows], NORM)
    # a sum that leaves the type: h is rounded like any other value, the norm is of the sum itself
    big = torch.full((1, K), 40000.0).half().to(device)
    q, scale, h = ops.add_rms_norm_int8(big, None, big)
    assert torch.isinf(h).all() and torch.all(q == 127)


@pytest.mark.parametrize("device", DEVICES)
def test_norm_other_layouts(device):
    base = _randn(24, 70, seed=1).bfloat16().to(device)
    other = _randn(70, 24, seed=2).bfloat16().to(device)
    w = torch.stack([1 + 0.1 * _randn(70, seed=3)] * 2, 1).to(device)[:, 0]
    for x, r in ((base, other.t()), (base.view(2, 12, 70), base.view(2, 12, 70)), (base[::3], base[1::3]),
                 (base[3:4].expand(24, 70), base), (base[0], base[1])):
        q, scale, h = ops.add_rms_norm_int8(x, w, r)
        h64, y64 = _norm64(x.reshape(-1, 70), w, r.reshape(-1, 70), 1e-6)
        assert h.shape == x.shape and q.shape == x.shape and scale.shape == x.shape[:-1]
        _check_codes(q.reshape(-1, 70), scale.reshape(-1), y64, NORM)
        assert torch.all((h.reshape(-1, 70).double() - h64).abs() <= HALF[torch.bfloat16] * 1.01 * h64.abs())


# ------------------------------------------------------------------------------------------------------- linear_int8
def _linear64(q, scale, w, ws, b, act):
    p = (q.double() @ w.double().t().contiguous()) * scale.double()[:, None] * ws.double()
    y = p if b is None else p + b.double()
    return p, {"none": y, "relu": y.clamp_min(0), "tanh": torch.tanh(y)}[act]


def _check_linear(y, q, scale, w, ws, b, act, dtype):
    p, want = _linear64(q, scale, w, ws, b, act)
    raw = want.abs() if act == "none" else want.abs() + (0 if b is None else b.double().abs()) + p.abs() * 0
    tol = 4 * U * p.abs() + 2 * U * raw + (10 * U * want.abs() if act == "tanh" else 0) + HALF[dtype] * 1.01 * want.abs() + TINY[dtype]
    if act != "none":      # the sum before the activation is rounded too
        tol = tol + 2 * U * (p.abs() + (0 if b is None else b.double().abs()))
    bad = (y.double() - want).abs() > tol
    assert y.dtype == dtype and y.shape == want.shape and not bad.any(), f"{int(bad.sum())} of {bad.numel()} values"


@pytest.mark.gpu
def test_tanh_over_its_whole_range():
    """One column: the sum times its scale is the argument itself.  5 steps of fp32 are allowed (10 u)."""
    v = torch.cat([torch.linspace(-12, 12, 200001), torch.logspace(-30, 4, 50001), -torch.logspace(-30, 4, 50001), torch.linspace(-0.6, 0.6, 100001),
                   torch.tensor([0.0, 0.5, -0.5, 1e-40, -1e-40, 3e38, math.inf, -math.inf, math.nan])]).cuda()
    one = torch.ones(v.numel(), 1, dtype=torch.int8, device="cuda")
    y = ops.linear_int8(one, v, one[:1], torch.ones(1, device="cuda"), None, "tanh")[:, 0]
    want = torch.tanh(v.double())
    assert torch.isnan(y[-1]) and torch.all((y[:-1].double() - want[:-1]).abs() <= 10 * U * want[:-1].abs() + 2.0 ** -149)
    assert torch.all(y[:-1].abs() <= 1)


SHAPES = [(1, 1, 1), (1, 3, 15), (2, 4, 16), (1, 400, 400), (3, 5, 17), (16, 16, 64), (17, 33, 65), (1, 50, 1000), (5, 17, 127),
          (31, 31, 129), (64, 51, 400), (65, 64, 256), (128, 128, 128), (129, 130, 131), (256, 400, 400), (300, 7, 2001),
          (7, 300, 2001), (257, 513, 640), (500, 260, 1111), (2, 4096, 1024), (1030, 1025, 385), (40, 2050, 96)]
#: one shape at least for every tile size and row kernel, all with ragged edges
GPU_SHAPES = [(3585, 3333, 300), (2300, 1700, 1300), (1793, 1665, 700), (700, 900, 5000), (150, 4000, 4100), (130, 4090, 1100), (1000, 1030, 1023),
          (16, 12300, 200), (3, 12289, 70), (9, 3000, 4100), (30, 7000, 333), (31, 20000, 50), (60, 3100, 77), (900, 300, 1000), (17, 330, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", GPU_SHAPES)
def test_linear_int8_by_every_kernel(M, N, K):
    _linear_case(M, N, K, "cuda")


#: large tiles with a long and a short K; few rows and many columns, at both sides of 16, 32, 64 and 128 rows
WIDE_SHAPES = [(1800, 1700, 2050), (2200, 2300, 150), (1, 18500, 2049), (16, 18500, 2100), (17, 18500, 2049), (32, 17000, 2100), (33, 18500, 2049),
               (64, 33000, 40), (65, 33000, 40), (65, 18500, 2049), (128, 49300, 40), (129, 49300, 40), (3, 66000, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", WIDE_SHAPES)
def test_linear_int8_with_many_columns(M, N, K):
    _linear_case(M, N, K, "cuda")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_int8(M, N, K, device):
    _linear_case(M, N, K, device)


def _linear_case(M, N, K, device):
    q, scale = _codes(M, K, device, seed=M + 3 * N + 7 * K)
    w, ws = _codes(N, K, device, seed=K)
    b = _randn(N, seed=4).to(device)
    for i, (act, dtype) in enumerate([("none", torch.float32), ("relu", torch.bfloat16), ("tanh", torch.float16),
                                      ("tanh", torch.float32)]):
        bias = b if i % 2 == 0 else None
        sc = scale if act != "tanh" else scale * 0.05
        y = ops.linear_int8(q, sc, w, ws, bias, act, dtype)
        _check_linear(y, q, sc, w, ws, bias, act, dtype)


@pytest.mark.parametrize("device", DEVICES)
def test_linear_int8_sums_are_exact(device):
    """The largest sums of every sign, to the last unit, with scales that change nothing."""
    for K in (1040, 4097):
        q = torch.full((3, K), 127, dtype=torch.int8)
        q[1], q[2] = -128, -127
        w = torch.full((5, K), -128, dtype=torch.int8)
        w[1], w[2, ::2], w[3, K - 1] = 127, 127, 1
        q, w = q.to(device), w.to(device)
        y = ops.linear_int8(q, torch.ones(3, device=device), w, torch.ones(5, device=device))
        assert torch.equal(y.double(), (q.double() @ w.double().t().contiguous()).float().double())


@pytest.mark.parametrize("device", DEVICES)
def test_linear_int8_other_layouts(device):
    M, N, K = 33, 41, 100
    big, s = _codes(80, 230, device, seed=1)
    wbig, ws = _codes(90, 230, device, seed=2)
    wt = wbig.t()
    want = None
    for q, w in ((big[:M, :K], wbig[:N, :K]), (big[:M, 3:3 + K], wbig[:N, 16:16 + K]), (big[::2][:M, :K], wbig[::2][:N, :K]),
                 (big[4:5, :K].expand(M, K), wbig[:N, :K]), (big[:M, ::2][:, :K], wt.t()[:N, 1:1 + K]),
                 (big.t()[:K, :M].t(), wt[:K, :N].t())):
        y = ops.linear_int8(q, s[:M], w, ws[:N])
        _check_linear(y, q, s[:M], w, ws[:N], None, "none", torch.float32)
    q3 = big[:32, :K].reshape(2, 16, K)
    y = ops.linear_int8(q3, s[:32].view(2, 16), wbig[:N, :K], ws[:N])
    assert y.shape == (2, 16, N) and want is None
    assert torch.equal(y.view(32, N), ops.linear_int8(big[:32, :K], s[:32], wbig[:N, :K], ws[:N]))
    one = ops.linear_int8(big[0, :K], s[0], wbig[:N, :K], ws[:N])
    assert one.shape == (N,) and torch.equal(one, y[0, 0])
    # scales and biases of other types and strides
    b = torch.stack([_randn(N, seed=9)] * 2, 1).to(device)
    y = ops.linear_int8(big[:M, :K], s[:M].double(), wbig[:N, :K], ws[:N], b[:, 1].half())
    _check_linear(y, big[:M, :K], s[:M], wbig[:N, :K], ws[:N], b[:, 1].half(), "none", torch.float32)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_that_are_not_finite_stay_so_through_the_product(device):
    x = _randn(4, 40, seed=3)
    x[1, 7], x[2, 0] = math.nan, math.inf
    w, ws = ops.quantize_rows(_randn(6, 40, seed=4).to(device))
    for act in ("none", "relu", "tanh"):
        y = ops.linear_int8(*ops.quantize_rows(x.to(device)), w, ws, None, act)
        assert torch.isnan(y[1:3]).all() and torch.isfinite(y[[0, 3]]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_nothing_to_do(device):
    q, s = _codes(3, 20, device, 1)
    w, ws = _codes(4, 20, device, 2)
    assert ops.linear_int8(q[:0], s[:0], w, ws).shape == (0, 4)
    assert ops.linear_int8(q, s, w[:0], ws[:0]).shape == (3, 0)
    assert ops.quantize_rows(torch.zeros(0, 7, device=device))[0].shape == (0, 7)
    assert ops.dequantize_rows(q[:0], s[:0]).shape == (0, 20)
    z = torch.zeros(2, 0, 5, device=device)
    assert [t.shape for t in ops.add_rms_norm_int8(z, None, z)] == [(2, 0, 5), (2, 0), (2, 0, 5)]


# -------------------------------------------------------------------------------------------------------- refusals
@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    d = dict(device=device)
    x, q, s = torch.zeros(2, 8, **d), torch.zeros(2, 8, dtype=torch.int8, **d), torch.ones(2, **d)
    w, ws = torch.zeros(3, 8, dtype=torch.int8, **d), torch.ones(3, **d)
    with pytest.raises(TypeError):
        ops.quantize_rows(x.double())
    with pytest.raises(TypeError):
        ops.quantize_rows(q)
    for bad in (torch.zeros(2, 0, **d), torch.zeros((), **d)):
        with pytest.raises(ValueError):
            ops.quantize_rows(bad)
        with pytest.raises(ValueError):
            ops.add_rms_norm_int8(bad)
    with pytest.raises(TypeError):
        ops.dequantize_rows(x, s)
    with pytest.raises(TypeError):
        ops.dequantize_rows(q, s, torch.float64)
    with pytest.raises(ValueError):
        ops.dequantize_rows(q, torch.ones(3, **d))
    with pytest.raises(TypeError):
        ops.add_rms_norm_int8(x.double())
    for kw in (dict(residual=x[:1]), dict(residual=x.half()), dict(weight=torch.ones(7, **d)), dict(weight=torch.ones(1, 8, **d)),
               dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf)):
        with pytest.raises(ValueError):
            ops.add_rms_norm_int8(x, **kw)
    with pytest.raises(TypeError):
        ops.add_rms_norm_int8(x, torch.ones(8, dtype=torch.int32, **d))
    for args, err in (((x, s, w, ws), TypeError), ((q, s, x, ws), TypeError), ((q, s[:1], w, ws), ValueError),
                      ((q, s, w, ws[:2]), ValueError), ((q, s, w[:, :7], ws), ValueError), ((q, s, w[0], ws), ValueError),
                      ((q, s, w, ws, ws[:2]), ValueError), ((q, s, w, ws, ws.long()), TypeError), ((q, s.long(), w, ws), TypeError),
                      ((q, s, w, ws, None, "gelu"), ValueError), ((q, s, w, ws, None, "none", torch.int8), TypeError),
                      ((q[:, :0], s, w[:, :0], ws), ValueError)):
        with pytest.raises(err):
            ops.linear_int8(*args)
    long_q = torch.zeros(1, 131072, dtype=torch.int8, **d)
    with pytest.raises(ValueError, match="32 bits"):
        ops.linear_int8(long_q, s[:1], long_q, s[:1])
    one = torch.zeros(1, **d)
    for shape in ((1 << 31, 1), (1, 1 << 31)):
        with pytest.raises(ValueError, match="2.31"):
            ops.quantize_rows(one.expand(*shape))
    with pytest.raises(ValueError, match="2.29"):
        ops.linear_int8(q[:, :1], s, one.to(torch.int8).expand((1 << 29) + 1, 1), one.expand((1 << 29) + 1))
    with pytest.raises(ValueError):
        ops.mlp3_int8(x, ((w, ws, None),) * 2)
    with pytest.raises(ValueError):
        ops.mlp3_int8(x, ((w, ws, None),) * 3, "gelu")


@pytest.mark.gpu
def test_refusal_of_mixed_devices():
    q, s = _codes(2, 8, "cuda", 1)
    w, ws = _codes(3, 8, "cpu", 2)
    for args in ((q, s, w, ws), (q, s.cpu(), w.cuda(), ws.cuda()), (q, s, w.cuda(), ws), (q, s, w.cuda(), ws.cuda(), ws)):
        with pytest.raises(ValueError, match="is on"):
            ops.linear_int8(*args)
    x = torch.zeros(2, 8, device="cuda")
    for kw in (dict(residual=x.cpu()), dict(weight=torch.ones(8))):
        with pytest.raises(ValueError, match="is on"):
            ops.add_rms_norm_int8(x, **kw)


# ------------------------------------------------------------------------------------------------- together, as used
def _layers(dims, device, seed=0, bias=True):
    out = []
    for i, (n, k) in enumerate(dims):
        w, ws = ops.quantize_rows((_randn(n, k, seed=seed + i) / math.sqrt(k)).to(device))
        out.append((w, ws, (0.1 * _randn(n, seed=seed + 50 + i)).to(device) if bias else None))
    return tuple(out)


def _mlp64(x, layers, final):
    """The formulas in 64 bits, rounding to codes included."""
    h = x.double()
    for i, (w, ws, b) in enumerate(layers):
        top = h.abs().amax(1, keepdim=True)
        step = top / 127
        hq = torch.where(top > 0, torch.round(h / torch.where(top > 0, step, 1.0)) * step, 0.0)
        h = hq @ (w.double() * ws.double()[:, None]).t().contiguous()
        if b is not None:
            h = h + b.double()
        if i < 2:
            h = h.clamp_min(0)
    return {"none": h, "relu": h.clamp_min(0), "tanh": torch.tanh(h), "softmax": torch.softmax(h, 1)}[final]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B,S,H,A,final", [(1, 24, 400, 4, "tanh"), (1, 3, 64, 1, "none"), (7, 111, 400, 8, "tanh"), (300, 17, 256, 6, "relu"),
                                           (256, 28, 1024, 51, "softmax"), (33, 5, 77, 3, "tanh"), (600, 111, 2048, 8, "tanh")])
def test_mlp3_int8(B, S, H, A, final, device):
    """A hidden value that lies at the border of two codes may take either: one step of the row (top / 127) in one of H
    inputs.  Weights of size 1 / sqrt(H) pass on a step of at most ~3 / sqrt(H) x top / 127; two of those per output
    are allowed for, on values of order one."""
    x = _randn(B, S, seed=B).to(device)
    layers = _layers(((H, S), (H, H), (A, H)), device, seed=H, bias=B != 7)
    y = ops.mlp3_int8(x, layers, final)
    want = _mlp64(x, layers, final)
    assert y.shape == (B, A) and y.dtype == torch.float32
    border = 2 * (4.0 / math.sqrt(H)) * (4.0 / 127)
    off = (y.double() - want).abs()
    assert off.max() <= border
    assert (off > 1e-4).double().mean() <= 0.05         # and hardly any value is
    assert ops.mlp3_int8(x.reshape(1, B, S), layers, final, torch.bfloat16).shape == (1, B, A)


@pytest.mark.gpu
@pytest.mark.parametrize("B,dims", [(1, (24, 400, 400, 4)), (5, (3, 64, 64, 1)), (17, (111, 128, 130, 51)), (33, (8, 256, 256, 2)), (40, (376, 300, 77, 300)),
                                    (2049, (17, 400, 400, 6)), (2100, (111, 1024, 1024, 8)), (31, (2048, 40, 2048, 2048)), (2200, (9, 2000, 1500, 33)),
                                    (3, (5, 2100, 2100, 3)), (4, (2500, 64, 64, 2)), (1, (1, 1, 1, 1)), (9, (63, 65, 16, 17)), (16, (64, 144, 129, 128))])
def test_mlp3_int8_is_the_layers_one_by_one(B, dims):
    """One launch or seven: the same values to the last bit, for every way columns and rows are dealt out."""
    x = _randn(B, dims[0], seed=B).cuda()
    x[0] = 0.0
    if B > 2:
        x[1, dims[0] // 2] = math.nan
    layers = _layers([(dims[i + 1], dims[i]) for i in range(3)], "cuda", seed=B, bias=B % 2 == 0)
    for final, dtype, xt in (("tanh", torch.float32, torch.float32), ("none", torch.bfloat16, torch.bfloat16), ("relu", torch.float16, torch.float16)):
        h = x.to(xt)
        want = h
        for i, (w, ws, b) in enumerate(layers):
            want = ops.linear_int8(*ops.quantize_rows(want), w, ws, b, "relu" if i < 2 else final, torch.float32 if i < 2 else dtype)
        got = ops.mlp3_int8(h, layers, final, dtype)
        assert got.dtype == dtype and torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
        assert B <= 2 or torch.isnan(got[1]).all()
    strided = torch.zeros(B, 2 * dims[0] + 3, device="cuda")
    strided[:, 1:1 + 2 * dims[0]:2] = x
    view = strided[:, 1:1 + dims[0]]
    want = ops.mlp3_int8(view.contiguous(), layers)
    assert torch.equal(torch.nan_to_num(ops.mlp3_int8(view, layers)), torch.nan_to_num(want))


@pytest.mark.parametrize("device", DEVICES)
def test_a_residual_block_of_them(device):
    """norm -> product -> norm of the sum -> product, as a residual network calls them, against fp64 layers without any
    8-bit step: the codes' own error (half a step of 1 / 127 of the largest value per element) is what is left."""
    B, D = 19, 320
    x = _randn(B, D, seed=1).bfloat16().to(device)
    g = (1 + 0.1 * _randn(D, seed=2)).bfloat16().to(device)
    w1, w2 = (_randn(D, D, seed=s).to(device) / math.sqrt(D) for s in (3, 4))
    p1, s1 = ops.quantize_rows(w1)
    p2, s2 = ops.quantize_rows(w2)
    q, s, h = ops.add_rms_norm_int8(x, g)
    y = ops.linear_int8(q, s, p1, s1, None, "relu", torch.bfloat16)
    q, s, h = ops.add_rms_norm_int8(y, g, h)
    y = ops.linear_int8(q, s, p2, s2, dtype=torch.bfloat16)
    h64 = x.double()
    y64 = (_norm64(h64, g, None, 1e-6)[1] @ w1.double().t().contiguous()).clamp_min(0)
    h64, n64 = _norm64(y64, g, h64, 1e-6)
    y64 = n64 @ w2.double().t().contiguous()
    # a step is at most 4.5 sigma / 127, its error uniform: 0.0102 sigma a value on both sides, twice over, plus bf16
    assert (h.double() - h64).norm() <= 0.03 * h64.norm()
    assert (y.double() - y64).norm() <= 0.05 * y64.norm()


class _Declines:
    """A binding that leaves everything to the Python way."""

    def __getattr__(self, name):
        return lambda *args: None


@pytest.mark.gpu
def test_the_binding_and_the_python_way_agree(monkeypatch):
    from d4pg_pytorch_amd.ops import int8
    x, r = _randn(70, 333, seed=1).cuda(), _randn(70, 333, seed=2).cuda()
    g = _randn(333, seed=3).cuda()
    narrow = _layers(((130, 333), (130, 130), (9, 130)), "cuda")
    wide = _layers(((1300, 333), (40, 1300), (9, 40)), "cuda", bias=False)

    def everything():
        q, s, h = ops.add_rms_norm_int8(x, g, r, 1e-5)
        p, t, same = ops.add_rms_norm_int8(x.half(), eps=0)
        c, u = ops.quantize_rows(x.bfloat16())
        w, ws, b = narrow[0]
        return (q, s, h, p, t, same, c, u, ops.dequantize_rows(c, u, torch.float16), ops.linear_int8(q, s, w, ws, b, "tanh", torch.bfloat16),
                ops.mlp3_int8(x, narrow, "tanh"), ops.mlp3_int8(x, wide, "relu", torch.float16), ops.mlp3_int8(x, narrow, "softmax"))

    fast = everything()
    with torch.inference_mode():
        again = everything()
    monkeypatch.setattr(int8, "_plain", _Declines())
    slow = everything()
    for a, b, c in zip(fast, slow, again):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride()
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
def test_calls_from_several_threads_on_streams_of_their_own():
    import threading
    layers = _layers(((256, 100), (256, 256), (5, 256)), "cuda")
    xs = [_randn(300, 100, seed=i).cuda() for i in range(4)]
    want = [ops.mlp3_int8(x, layers, "tanh") for x in xs]
    lin = [ops.linear_int8(*ops.quantize_rows(x), *layers[0]) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                y = ops.mlp3_int8(xs[i], layers, "tanh")
                z = ops.linear_int8(*ops.quantize_rows(xs[i]), *layers[0])
                if not (torch.equal(y, want[i]) and torch.equal(z, lin[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not bad


@pytest.mark.gpu
def test_more_rows_than_one_launch_holds():
    """64 threads a row: 2^26 rows are 2^32 threads, which is one too many for a launch; offsets pass 32 bits too."""
    M = (1 << 26) + 70
    x = torch.arange(M, device="cuda", dtype=torch.float32).remainder_(251.0).sub_(125.0)[:, None]
    q, scale = ops.quantize_rows(x)
    assert torch.equal(q, (x.sign() * 127).to(torch.int8))
    assert torch.all((scale.double() - x[:, 0].abs().double() / 127).abs() <= scale.double() * U)
    back = ops.dequantize_rows(q, scale, torch.bfloat16)
    assert torch.equal(back, (q.float() * scale[:, None]).bfloat16())
    del back
    w, ws = _codes(1, 1, "cuda", 3)
    y = ops.linear_int8(q, scale, w, ws)
    assert torch.equal(y, (q.float() * w.float()) * scale[:, None] * ws)


@pytest.mark.gpu
def test_on_another_stream_and_captured():
    x = _randn(65, 200, seed=1).cuda()
    r = _randn(65, 200, seed=2).cuda()
    layers = _layers(((130, 200), (130, 130), (9, 130)), "cuda")
    w, ws, b = layers[0]

    def chain():
        q, s, h = ops.add_rms_norm_int8(x, None, r)
        return (h, ops.dequantize_rows(q, s, torch.bfloat16), ops.linear_int8(q, s, w, ws, b, "relu"), ops.mlp3_int8(x, layers, "tanh"))

    want = chain()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = chain()
    for i in range(4):
        x.copy_(_randn(65, 200, seed=10 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        assert all(torch.equal(a, c) for a, c in zip(got, chain()))


@pytest.mark.gpu
@pytest.mark.parametrize("S,A,Hd,E", [(24, 4, 400, 16), (111, 8, 1024, 300), (3, 1, 2400, 5)])
def test_a_gpu_agent_acts_on_8_bit_codes(S, A, Hd, E):
    """The agent's policy is ``mlp3_int8`` on codes of its parameters, whichever way these arrive, and stays near the
    fp32 policy: three layers of codes are off by about 1 % of a layer's values each."""
    import numpy as np

    from d4pg_pytorch_amd.actors.gpu_actor import GpuActor
    from d4pg_pytorch_amd.models.nets import ActorPolicy, init_net_
    pol = ActorPolicy(S, A, Hd)
    init_net_(pol.view, 0.05, _gen(3))
    ga = GpuActor(S, A, Hd, max_batch=E, action_scale=1.5, precision="int8")
    x = _randn(E, S, seed=4)
    zero = ga.act(x.numpy())
    assert zero.shape == (E, A) and not zero.any()                  # parameters of zeros
    ga.load_flat(pol.flat.numpy())
    got = ga.act(x.numpy())
    layers = [(*ops.quantize_rows(w.cuda()), b.cuda()) for w, b in zip(pol.view.weights, pol.view.biases)]
    assert np.array_equal(got, (1.5 * ops.mlp3_int8(x.cuda(), layers, "tanh")).cpu().numpy())
    want = 1.5 * pol.act(x).numpy()
    assert np.linalg.norm(got - want) <= 0.05 * np.linalg.norm(want)
    init_net_(pol.view, 0.05, _gen(9))
    ga.load_state_dict(pol.state_dict())
    assert np.linalg.norm(ga.act(x.numpy()) - 1.5 * pol.act(x).numpy()) <= 0.05 * np.linalg.norm(want)
    assert np.array_equal(ga.act(x[0].numpy())[0], ga.act(x.numpy())[0])
    with pytest.raises(ValueError):
        GpuActor(S, A, Hd, precision="int4")


@pytest.mark.gpu
@pytest.mark.parametrize("Hd", [64, 1100])
def test_a_captured_policy_follows_new_parameters(Hd):
    from d4pg_pytorch_amd.actors.gpu_actor import GpuActor
    from d4pg_pytorch_amd.models.nets import ActorPolicy, init_net_
    S, A, E = 11, 3, 5
    pol = ActorPolicy(S, A, Hd)
    init_net_(pol.view, 0.05, _gen(3))
    ga = GpuActor(S, A, Hd, max_batch=E, precision="int8")
    ga.load_flat(pol.flat.numpy())
    places = [t.data_ptr() for layer in ga.codes for t in layer]
    obs, out = _randn(E, S, seed=4).cuda(), torch.zeros(E, A, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ga.act_device(obs, out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ga.act_device(obs, out)
    seen = []
    for seed in (5, 6, 7):
        init_net_(pol.view, 0.05, _gen(seed))
        ga.load_flat(pol.flat.numpy())
        assert places == [t.data_ptr() for layer in ga.codes for t in layer]
        graph.replay()
        got = out.clone()
        fresh = [(*ops.quantize_rows(w.cuda()), b.cuda()) for w, b in zip(pol.view.weights, pol.view.biases)]
        assert torch.equal(got, ops.mlp3_int8(obs, fresh, "tanh"))
        seen.append(got)
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_the_agents_precision_is_a_config_key():
    from d4pg_pytorch_amd.config import ConfigError, default_config
    assert default_config(env="Pendulum-v0")["policy_precision"] == "fp32"
    assert default_config(env="Pendulum-v0", policy_precision="int8")["policy_precision"] == "int8"
    with pytest.raises(ConfigError):
        default_config(env="Pendulum-v0", policy_precision="fp8")


@pytest.mark.gpu
def test_the_config_key_reaches_the_agent():
    from d4pg_pytorch_amd.actors.agent import make_policy
    from d4pg_pytorch_amd.config import default_config
    cfg = default_config(env="Pendulum-v0", policy_precision="int8", dense_size=64)
    assert make_policy(cfg, "cuda").precision == "int8" and make_policy(cfg, "cuda").launches_per_act == 2
    assert make_policy(dict(cfg, policy_precision="fp32"), "cuda").precision == "fp32"


def test_parameters_that_want_gradients_are_served_without():
    lin = torch.nn.Linear(12, 5)
    w, ws = ops.quantize_rows(lin.weight)
    q, s = ops.quantize_rows(torch.randn(3, 12, requires_grad=True))
    y = ops.linear_int8(q, s, w, ws, lin.bias)
    assert not y.requires_grad and not ws.requires_grad
    assert ref.linear_int8 is not None


# ------------------------------------------------------------------------------------------------------ C entry points
def test_the_library_refuses_what_its_kernels_cannot_read():
    """Launch descriptors with bad sizes, strides or alignment are turned away before any launch (no GPU needed)."""
    import ctypes as C

    from d4pg_pytorch_amd.ops import hip as H
    lib = H.lib()

    def product(**kw):
        a = H.LinearInt8Args()
        a.q, a.scale, a.w, a.wscale, a.out = 4096, 4096, 8192, 8192, 8192
        a.ld_q, a.ld_w, a.ld_out, a.M, a.N, a.K = 32, 32, 4, 4, 4, 20
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.d4pg_linear_int8(C.byref(a), None)

    for kw in (dict(M=0), dict(N=0), dict(N=(1 << 29) + 1), dict(K=0), dict(K=131072), dict(q=None), dict(w=None), dict(scale=None), dict(wscale=None),
               dict(out=None), dict(ld_q=40), dict(ld_w=24), dict(ld_q=16), dict(ld_w=16), dict(ld_out=3), dict(q=4104), dict(w=8193),
               dict(dtype=3), dict(dtype=-1), dict(act=3), dict(act=-1)):
        assert product(**kw) < 0, kw

    def rows(**kw):
        a = H.QuantRowsArgs()
        a.x, a.q, a.scale, a.M, a.K, a.ld_x, a.ld_q, a.wdtype = 4096, 8192, 4096, 2, 20, 20, 32, H.F_NONE
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.d4pg_quant_rows(C.byref(a), None)

    for kw in (dict(M=0), dict(K=0), dict(M=1 << 31), dict(x=None), dict(q=None), dict(scale=None), dict(ld_q=31), dict(ld_q=16),
               dict(ld_q=48), dict(q=8200), dict(wdtype=0, norm=1), dict(wdtype=3, weight=4096, norm=1), dict(residual=4096), dict(dtype=3)):
        assert rows(**kw) < 0, kw

    a = H.DequantRowsArgs()
    assert lib.d4pg_dequant_rows(C.byref(a), None) < 0
