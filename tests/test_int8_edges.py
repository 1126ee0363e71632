"""8-bit serving operators (``ops/int8.py``, ``csrc/int8.hip``) at borders of their arithmetic, their dispatch and their
calls.  Bounds as in ``test_int8.py``, whose helpers these tests use."""
import math

import pytest
import torch

from d4pg_pytorch_amd import ops
from test_int8 import DEVICES, NORM, _check_codes, _norm64, _randn


# --------------------------------------------------------------------------------------------- the norm's two branches
@pytest.mark.parametrize("device", DEVICES)
def test_norm_whose_sum_of_squares_is_at_the_end_of_fp32(device):
    """By one order of additions the sum of these squares is the largest fp32 number, by another it is infinite: the
    threads of the row have to agree on one."""
    x = torch.zeros(1, 128)
    x[0, 0], x[0, 32], x[0, 64], x[0, 96] = (float.fromhex(v) for v in ("0x1.000004p+63", "0x1.fffffep+62", "0x1p+63", "0x1.fffff6p+62"))
    q, scale, _ = ops.add_rms_norm_int8(x.to(device))
    assert q[0, ::32].tolist() == [127] * 4
    _check_codes(q, scale, _norm64(x, None, None, 1e-6)[1], NORM)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("K", [9, 77, 128, 250, 400, 3001])
def test_norm_around_the_smallest_plain_mean_square(K, device):
    """Rows whose mean square passes 2^-80 in steps of the last place."""
    base = _randn(60, K, seed=K).double()
    base = base * (2.0 ** -40 / base.square().mean(1, keepdim=True).sqrt())
    x = torch.cat([base * (1 + j * 2.0 ** -25) for j in range(-12, 13)]).float()
    q, scale, _ = ops.add_rms_norm_int8(x.to(device), eps=0.0)
    _check_codes(q, scale, _norm64(x, None, None, 0.0)[1], NORM)


# ------------------------------------------------------------------------------------------- views whose sign is pending
@pytest.mark.parametrize("device", DEVICES)
def test_views_whose_sign_is_pending(device):
    """``torch._neg_view(t)`` holds ``t`` in memory and reads as ``-t``; so does the imaginary part of a conjugate."""
    def pending(t):
        view = torch._neg_view(t)
        assert view.is_neg()
        return view

    x, r, g = (_randn(*shape, seed=i).to(device) for i, shape in enumerate(((5, 40), (5, 40), (40,))))
    z = torch.complex(x[:, :1], r[:, :1]).conj().imag
    assert z.is_neg() and z.shape == (5, 1)

    def same(a, b):
        assert all(torch.equal(s, t) for s, t in zip(a, b))

    same(ops.quantize_rows(pending(x)), ops.quantize_rows(-x))
    same(ops.quantize_rows(z), ops.quantize_rows(-r[:, :1]))
    same(ops.add_rms_norm_int8(pending(x), pending(g), pending(r)), ops.add_rms_norm_int8(-x, -g, -r))
    same(ops.add_rms_norm_int8(x, pending(g)), ops.add_rms_norm_int8(x, -g))
    q, s = ops.quantize_rows(x)
    w, ws = ops.quantize_rows(_randn(7, 40, seed=5).to(device))
    b = _randn(7, seed=6).to(device)
    same([ops.dequantize_rows(pending(q), pending(s))], [ops.dequantize_rows(-q, -s)])
    for args in ((pending(q), s, w, ws, b), (q, pending(s), w, ws, b), (q, s, pending(w), ws, b), (q, s, w, pending(ws), b),
                 (q, s, w, ws, pending(b))):
        same([ops.linear_int8(*args)], [ops.linear_int8(*(a.resolve_neg() for a in args))])
    layers = [(*ops.quantize_rows(_randn(n, k, seed=n).to(device)), _randn(n, seed=k).to(device)) for n, k in ((16, 40), (16, 16), (3, 16))]
    same([ops.mlp3_int8(pending(x), layers)], [ops.mlp3_int8(-x, layers)])
    turned = [(w, pending(-ws), pending(-b)) for w, ws, b in layers]
    same([ops.mlp3_int8(x, turned)], [ops.mlp3_int8(x, layers)])


# ---------------------------------------------------------------------------------------------- the ends of eps's range
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("K", [1, 40, 700, 40000])
def test_norm_with_an_eps_at_the_ends_of_fp32(K, device):
    """``mean + eps`` may pass the largest fp32 number though both are finite; ``eps`` below 2^-150 is nothing."""
    top = torch.finfo(torch.float32).max
    x = torch.cat([_randn(2, K, seed=K), 1e19 / math.sqrt(K) * _randn(2, K, seed=1), 1e-30 * _randn(2, K, seed=2)])
    for eps in (top, 3.3e38, 2.0 ** -149, 2.0 ** -126):
        q, scale, _ = ops.add_rms_norm_int8(x.to(device), eps=eps)
        rows = [0, 1, 4, 5] if eps < 1 else [0, 1, 2, 3]
        _check_codes(q[rows], scale[rows], _norm64(x[rows], None, None, eps)[1], NORM)
    q, scale, _ = ops.add_rms_norm_int8(x.to(device), eps=1e-50)
    _check_codes(q, scale, _norm64(x, None, None, 0.0)[1], NORM)


@pytest.mark.parametrize("device", DEVICES)
def test_refusal_of_an_eps_that_fp32_does_not_hold(device):
    x = _randn(2, 8).to(device)
    for eps in (3.5e38, 1e300, 10.0 ** 60, -1e-30, -1e-60, -math.inf):
        with pytest.raises(ValueError, match="eps"):
            ops.add_rms_norm_int8(x, eps=eps)


# ------------------------------------------------------------------------------------------------- codes, to the last one
def _codes_of(x):
    """Codes of rows of whole numbers ``x`` [M, K] (int64, below 2^24), in whole numbers throughout."""
    top = x.abs().amax(1, keepdim=True)
    doubled = 254 * x.abs()                       # of 2 top: code = floor((254 |x| + top) / (2 top)), a half to the even one
    k = (doubled + top) // (2 * top)
    half = (doubled + top) % (2 * top) == 0
    k = k - (half & (k % 2 == 1)).long()
    return x.sign() * k


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shift", [-149, -126, -90, -63, -62, -40, 0, 40, 62, 63, 100, 103])
def test_halves_go_to_the_even_code(shift, device):
    """Rows 2 x 127 m with every half there is, (2 k + 1) m, and its neighbours; and a / 2, which is 63.5 codes of any a."""
    m = torch.tensor([1, 2, 3, 5, 7, 9, 11, 100, 333, 1023, 1025, 4099, 20011, 33023, 66047])[:, None]
    halves = (2 * torch.arange(0, 127)[None] + 1) * m
    x = torch.cat([254 * m, halves, -halves, halves + 1, 1 - halves, halves - 1], 1)
    assert int(x.abs().max()) < 1 << 24
    values = (x.double() * 2.0 ** shift).float()
    assert torch.equal(values.double(), x.double() * 2.0 ** shift)
    q, scale = ops.quantize_rows(values.to(device))
    assert torch.equal(q.cpu().long(), _codes_of(x))
    assert torch.equal(scale.cpu(), values[:, 0] / 127)
    a = torch.randint(1, 1 << 23, (500, 1), generator=torch.Generator().manual_seed(3)) * 2
    x = torch.cat([a, a // 2, -(a // 2)], 1)
    q, _ = ops.quantize_rows((x.double() * 2.0 ** shift).float().to(device))
    assert torch.equal(q.cpu(), torch.tensor([127, 64, -64], dtype=torch.int8).expand(500, 3))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,most", [(torch.bfloat16, 256), (torch.float16, 2048), (torch.float32, 1 << 24)])
@pytest.mark.parametrize("K", [33, 500, 5000])
def test_codes_of_whole_numbers(K, dtype, most, device):
    """Every code of rows that the type holds exactly.  An fp32 quotient within 2^-18 of a half, but not on it, may be
    rounded onto it: such places (at most 254 x 2^-18 x 2 of the values) are left out, for 16-bit types there are none."""
    x = torch.randint(-most, most + 1, (64, K), generator=torch.Generator().manual_seed(K))
    q, _ = ops.quantize_rows(x.to(dtype).to(device))
    want = _codes_of(x)
    v = x.double() * 127 / x.abs().amax(1, keepdim=True).double()
    off = (v - v.floor() - 0.5).abs()
    skip = (off > 0) & (off < 2.0 ** -18)
    assert dtype == torch.float32 or not skip.any()
    assert torch.equal(torch.where(skip, want, q.cpu().long()), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_both_devices_make_the_same_codes(dtype):
    x = (_randn(300, 700, seed=1) * torch.exp(20 * _randn(300, 1, seed=2)).clamp(1e-3, 1e3)).to(dtype)
    for a, b in zip(ops.quantize_rows(x), ops.quantize_rows(x.cuda())):
        assert torch.equal(a, b.cpu())


# ------------------------------------------------------------------------------------------------------ tanh in 32 bits
@pytest.mark.gpu
def test_tanh_of_fp32_results_is_within_two_units_of_the_last_place():
    """One column: the sum times its scale is the argument itself, so all of the error is the function's.  Division and
    exponential of full precision leave at most 1.4 units; two are allowed, and as much through the policy's last layer."""
    v = torch.cat([torch.linspace(0.25, 1.25, 1 << 20), torch.linspace(1.25, 10, 1 << 18)]).cuda()
    v = torch.cat([v, -v])
    one = torch.ones(v.numel(), 1, dtype=torch.int8, device="cuda")
    want = torch.tanh(v.double())
    unit = torch.ldexp(torch.ones_like(want), torch.frexp(want).exponent - 24)
    y = ops.linear_int8(one, v, one[:1], torch.ones(1, device="cuda"), None, "tanh")[:, 0]
    assert torch.all((y.double() - want).abs() <= 2 * unit)
    x = v[: 1 << 20: 16, None].clone()
    eye = (torch.ones(1, 1, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"), None)
    y = ops.mlp3_int8(x, (eye, eye, eye), "tanh")[:, 0]
    h = ops.mlp3_int8(x, (eye, eye, eye))[:, 0].double()
    unit = torch.ldexp(torch.ones_like(h), torch.frexp(torch.tanh(h)).exponent - 24)
    assert torch.all((y.double() - torch.tanh(h)).abs() <= 2 * unit)


# ------------------------------------------------------------------------------------ where the agents' key does not reach
def test_the_precision_key_is_refused_where_it_would_do_nothing():
    from d4pg_pytorch_amd.actors.gpu_rollout import DeviceRollout
    from d4pg_pytorch_amd.config import ConfigError, default_config
    from d4pg_pytorch_amd.utils.learning import GreedyEvaluator
    for kw in (dict(gpu_rollout_envs=64), dict(device="cpu"), dict(device="cpu", agent_device="cpu"), dict(exploiter_device="cpu")):
        with pytest.raises(ConfigError, match="policy_precision"):
            default_config(env="Pendulum-v0", policy_precision="int8", **kw)
    for kw in (dict(), dict(device="cpu", agent_device="cuda"), dict(exploiter_device="cuda:0", agent_device="cpu")):
        assert default_config(env="Pendulum-v0", policy_precision="int8", **kw)["policy_precision"] == "int8"
    cfg = dict(default_config(env="Pendulum-v0"), policy_precision="int8")
    with pytest.raises(ValueError, match="policy_precision"):
        DeviceRollout(cfg, None, None)
    with pytest.raises(ValueError, match="policy_precision"):
        GreedyEvaluator(cfg, 4, "cpu", 1)


# ---------------------------------------------------------------------------------------------------- what entries return
def _policy(M, dims, device="cuda"):
    """A launch descriptor of ``mlp3_int8`` and what it points to."""
    from d4pg_pytorch_amd.ops import hip as H
    a = H.Mlp3Int8Args()
    x, out = _randn(M, dims[0], seed=1).to(device), torch.empty(M, dims[3], device=device)
    layers = [(*ops.quantize_rows(_randn(dims[i + 1], dims[i], seed=i).to(device)), _randn(dims[i + 1], seed=i).to(device)) for i in range(3)]
    for i, (w, s, b) in enumerate(layers):
        a.w[i], a.wscale[i], a.bias[i], a.ld_w[i] = w.data_ptr(), s.data_ptr(), b.data_ptr(), w.stride(0)
    a.x, a.ld_x, a.out, a.ld_out, a.M, a.width[:] = x.data_ptr(), dims[0], out.data_ptr(), dims[3], M, dims
    return a, x, layers, out


def test_a_policy_outside_the_one_launch_is_told_from_an_error():
    """The code for it is no ``hipError_t`` (those are positive); nothing is launched, so no GPU is needed."""
    import ctypes as C

    from d4pg_pytorch_amd.ops import hip as H
    for dims in ([2100, 64, 64, 2], [16, 1025, 64, 2], [16, 64, 64, 1030], [2000, 1024, 1024, 120]):
        a, *held = _policy(3, dims, "cpu")
        assert H.lib().d4pg_mlp3_int8(C.byref(a), None) == H.NOT_TAKEN < 0, dims


def test_a_policy_of_too_many_columns_is_refused():
    """Numbers of columns that leave 32 bits when they are rounded up to tiles; nothing is launched."""
    import ctypes as C

    from d4pg_pytorch_amd.ops import hip as H
    a, *held = _policy(3, [16, 64, 64, 4], "cpu")
    for width in ((1 << 31) - 1, (1 << 31) - 20, (1 << 29) + 1):
        a.width[3] = a.ld_out = width
        assert H.lib().d4pg_mlp3_int8(C.byref(a), None) == -1


@pytest.mark.gpu
def test_an_error_left_by_another_call_is_not_taken_for_an_operators_own():
    import ctypes as C
    import os

    from d4pg_pytorch_amd import build
    from d4pg_pytorch_amd.ops import hip as H
    hip = C.CDLL(os.path.join(build.torch_lib_dir(), "libamdhip64.so"))
    a, x, layers, out = _policy(5, [24, 64, 64, 3])
    want = ops.mlp3_int8(x, layers)
    q, s = ops.quantize_rows(x)
    w, ws, _ = layers[0]
    buf, y, v = torch.empty(5, 32, dtype=torch.int8, device="cuda"), torch.empty(5, 64, device="cuda"), torch.empty(5, 24, device="cuda")
    codes = H.QuantRowsArgs(x.data_ptr(), None, None, None, buf.data_ptr(), s.data_ptr(), 5, 24, 24, 0, 0, 32, 0, H.F_NONE, 0, 0.0)
    product = H.LinearInt8Args(q.data_ptr(), s.data_ptr(), w.data_ptr(), ws.data_ptr(), None, y.data_ptr(), 32, 32, 64, 5, 64, 24, 0, 0, 0)
    values = H.DequantRowsArgs(q.data_ptr(), s.data_ptr(), v.data_ptr(), 5, 24, 32, 0, 0)
    torch.cuda.synchronize()
    got = {}
    for name, args in (("d4pg_mlp3_int8", a), ("d4pg_quant_rows", codes), ("d4pg_linear_int8", product), ("d4pg_dequant_rows", values)):
        assert hip.hipGetDevice(None) == 1                # hipErrorInvalidValue: refused on the host, left pending
        got[name] = H.launch_on(name, args, 0)
        hip.hipGetLastError()
    assert got == dict.fromkeys(got, 0)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(buf[:, :24], q)
    assert torch.equal(y, ops.linear_int8(q, s, w, ws)) and torch.equal(v, ops.dequantize_rows(q, s))


@pytest.mark.gpu
def test_a_launch_that_hip_refuses_raises_and_is_not_tried_again():
    """Entries that return a ``hipError_t`` (nothing reaches the GPU here) in the place of the library's."""
    import ctypes as C

    from d4pg_pytorch_amd.ops import hip as H
    x = _randn(4, 20, seed=1).cuda()
    q, s = ops.quantize_rows(x)
    layers = [(*ops.quantize_rows(_randn(4, k, seed=k).cuda()), None) for k in (20, 4, 4)]
    calls, codes = [], [0]

    @C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_void_p)
    def entry(args, stream):
        calls.append(args)
        return codes[0]

    binding = H.int8_binding()
    real = [C.cast(getattr(H.lib(), name), C.c_void_p).value for name in ("d4pg_quant_rows", "d4pg_dequant_rows", "d4pg_linear_int8", "d4pg_mlp3_int8")]
    try:
        binding.bind(*[C.cast(entry, C.c_void_p).value] * 4)
        for code in (1, 719):
            codes[0] = code
            for call in (lambda: ops.quantize_rows(x), lambda: ops.add_rms_norm_int8(x), lambda: ops.dequantize_rows(q, s),
                         lambda: ops.linear_int8(q, s, q, s), lambda: ops.mlp3_int8(x, layers)):
                calls.clear()
                with pytest.raises(RuntimeError, match=f"failed with code {code}"):
                    call()
                assert len(calls) == 1
    finally:
        binding.bind(*real)
    assert torch.equal(ops.quantize_rows(x)[0], q)


# ------------------------------------------------------------------------------------- more rows than one launch may hold
def _launches(call):
    """Kernel launches of ``call`` (0 is what it returns), which then run once."""
    from d4pg_pytorch_amd.ops import hip as H
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        rc = call(torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    n = H.graph_kernel_nodes(graph)
    graph.instantiate()
    graph.replay()
    torch.cuda.synchronize()
    return n


@pytest.mark.gpu
@pytest.mark.parametrize("M,K", [(1000, 40), (1000, 128), (999, 250), (1000, 500), (300, 1000), (300, 2000), (90, 4000), (30, 5001),
                                 (300, 5001), (300, 9001), (30, 20000), (9, 40001)])
def test_rows_of_several_launches(M, K):
    """Every row kernel with a limit of 4096 threads a launch: the same bits as in one launch, the rows' ends included."""
    import ctypes as C

    from d4pg_pytorch_amd.ops import hip as H
    kp = (K + 15) // 16 * 16
    for dtype, code in ((torch.bfloat16, H.F_BF16), (torch.float32, H.F_FP32)):
        x, r, g = (_randn(*shape, seed=i).to(dtype).cuda() for i, shape in enumerate(((M, K + 3), (M, K), (K,))))
        x = x[:, 2:2 + K]
        for norm in (0, 1):
            want = ops.add_rms_norm_int8(x, g, r) if norm else ops.quantize_rows(x)
            q, s, h = torch.full((M, kp), 99, dtype=torch.int8, device="cuda"), torch.full((M,), -1.0, device="cuda"), torch.zeros_like(r)
            a = H.QuantRowsArgs(x.data_ptr(), None, None, None, q.data_ptr(), s.data_ptr(), M, K, K + 3, 0, 0, kp, code, H.F_NONE, 0, 0.0)
            if norm:
                a.residual, a.weight, a.h, a.ld_r, a.ld_h = r.data_ptr(), g.data_ptr(), h.data_ptr(), K, K
                a.wdtype, a.norm, a.eps = code, 1, 1e-6
            assert _launches(lambda stream: H.lib().d4pg_quant_rows_in(C.byref(a), 4096, stream)) > 1
            assert torch.equal(q[:, :K], want[0]) and not q[:, K:].any() and torch.equal(s, want[1])
            assert not norm or torch.equal(h, want[2])


@pytest.mark.gpu
@pytest.mark.parametrize("M,K", [(3000, 1), (2999, 9), (777, 100), (20, 5001)])
def test_values_of_several_launches(M, K):
    import ctypes as C

    from d4pg_pytorch_amd.ops import hip as H
    q, s = ops.quantize_rows(_randn(M, K, seed=K).cuda())
    for dtype, code in ((torch.float32, H.F_FP32), (torch.float16, H.F_FP16)):
        out = torch.full((M, K), 7.0, dtype=dtype, device="cuda")
        a = H.DequantRowsArgs(q.data_ptr(), s.data_ptr(), out.data_ptr(), M, K, q.stride(0), code, 0)
        assert _launches(lambda stream: H.lib().d4pg_dequant_rows_in(C.byref(a), 1024, stream)) > 1
        assert torch.equal(out, ops.dequantize_rows(q, s, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,threads", [(500, 950, 333, 16384), (777, 130, 2001, 3000), (2300, 1700, 130, 40000), (513, 1, 1, 1024),
                                           (1000, 70, 4100, 60000), (33, 3000, 50, 50000)])
def test_products_of_several_launches(M, N, K, threads):
    import ctypes as C

    from d4pg_pytorch_amd.ops import hip as H
    q, s = ops.quantize_rows(_randn(M, K, seed=1).cuda())
    w, ws = ops.quantize_rows(_randn(N, K, seed=2).cuda())
    b = _randn(N, seed=3).cuda()
    for dtype, code in ((torch.float32, H.F_FP32), (torch.bfloat16, H.F_BF16)):
        out = torch.full((M + 1, N), 7.0, dtype=dtype, device="cuda")
        a = H.LinearInt8Args(q.data_ptr(), s.data_ptr(), w.data_ptr(), ws.data_ptr(), b.data_ptr(), out.data_ptr(), q.stride(0), w.stride(0), N,
                             M, N, K, H.ACT_RELU, code, 0)
        assert _launches(lambda stream: H.lib().d4pg_linear_int8_in(C.byref(a), threads, stream)) > 1
        assert torch.equal(out[:M], ops.linear_int8(q, s, w, ws, b, "relu", dtype)) and torch.all(out[M] == 7)


@pytest.mark.gpu
def test_more_rows_than_the_real_limit():
    """16 threads a row: 2^28 rows of one column are 2^32 threads.  The rows are one in memory, so that codes, scales and
    what checks them are all there is (4 GB of codes, one of scales)."""
    M = (1 << 28) + 70
    x = torch.full((1, 1), -3.0, device="cuda").expand(M, 1)
    q, s = ops.quantize_rows(x)
    want = torch.tensor(3.0) / 127
    for part in range(0, M, 1 << 26):
        assert torch.all(q[part:part + (1 << 26)] == -127) and torch.all(s[part:part + (1 << 26)] == want.item())


def test_limits_a_launch_cannot_have_are_refused():
    import ctypes as C

    from d4pg_pytorch_amd.ops import hip as H
    lib = H.lib()
    for limit in (0, 1023, -1, 1 << 32):
        assert lib.d4pg_quant_rows_in(C.byref(H.QuantRowsArgs()), limit, None) == -8
        assert lib.d4pg_dequant_rows_in(C.byref(H.DequantRowsArgs()), limit, None) == -8
        assert lib.d4pg_linear_int8_in(C.byref(H.LinearInt8Args()), limit, None) == -8
    assert lib.d4pg_linear_int8_in(C.byref(H.LinearInt8Args()), 1024, None) == -1


# --------------------------------------------------------------------- kernels of the dispatch that no other test reaches
@pytest.mark.gpu
@pytest.mark.parametrize("B,dims", [(4097, (24, 400, 400, 4)), (4131, (17, 256, 250, 129)), (4100, (100, 130, 77, 256)), (4127, (33, 60, 512, 9)),
                                    (4112, (200, 500, 300, 500)), (4133, (111, 1024, 1024, 8)), (4099, (64, 1000, 90, 1024)), (8209, (5, 128, 1024, 1)),
                                    (4105, (3, 16, 128, 65)), (4098, (700, 1024, 1024, 1024))])
def test_mlp3_int8_by_32_rows_a_workgroup(B, dims):
    """More than 4096 states: the kernels that take 32 rows at a time, with ragged ends, wide and narrow layers in every
    place, and rows that are not finite in both halves of 16; to the last bit as the layers one by one."""
    x = _randn(B, dims[0], seed=B).cuda()
    x[20, dims[0] // 2], x[5, 0], x[B - 1, 0], x[17] = math.nan, math.inf, -math.inf, 0.0
    layers = []
    for i in range(3):
        bias = 0.1 * _randn(dims[i + 1], seed=i).cuda() if (B + i) % 2 else None
        layers.append((*ops.quantize_rows((_randn(dims[i + 1], dims[i], seed=B + i) / math.sqrt(dims[i])).cuda()), bias))
    for final, dtype, xt in (("tanh", torch.float32, torch.float32), ("none", torch.bfloat16, torch.bfloat16), ("relu", torch.float16, torch.float16)):
        want = x.to(xt)
        for i, (w, ws, b) in enumerate(layers):
            want = ops.linear_int8(*ops.quantize_rows(want), w, ws, b, "relu" if i < 2 else final, torch.float32 if i < 2 else dtype)
        got = ops.mlp3_int8(x.to(xt), layers, final, dtype)
        assert torch.isnan(got[[5, 20, B - 1]]).all() and torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(500, 950, 333), (1900, 250, 1111), (127, 4000, 40), (1500, 200, 1000), (33, 16000, 30)])
def test_linear_int8_between_the_row_kernels_and_the_tiles(M, N, K):
    """Fewer than 128 tiles of 64 x 64, more than 1536 of 16 x 16 (``linear_int8_rows_kernel<4, 2, 8, 2>``), and around it."""
    from test_int8 import _linear_case
    _linear_case(M, N, K, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", [(300, 5003), (300, 8200), (257, 9001), (1000, 4104), (256, 5003), (256, 16384), (257, 16384)])
def test_quantize_long_rows_of_many(M, K, dtype):
    x = (_randn(M, K, seed=M + K) * torch.exp(2 * _randn(M, 1, seed=5))).to(dtype).cuda()
    x[3, K - 1], x[4] = math.nan, 0.0
    q, scale = ops.quantize_rows(x)
    assert torch.isnan(scale[3]) and not q[3].any() and scale[4] == 0 and not q[4].any()
    rows = [i for i in range(M) if i not in (3, 4)]
    _check_codes(q[rows], scale[rows], x[rows], 0.0)


@pytest.mark.gpu
def test_threads_on_streams_of_their_own_all_come_to_their_end():
    """Four threads, each on its own stream: what goes wrong in one is seen, and each has made all of its calls."""
    import threading
    layers = [(*ops.quantize_rows((_randn(n, k, seed=n + k) / math.sqrt(k)).cuda()), None) for n, k in ((256, 100), (256, 256), (5, 256))]
    xs = [_randn(300, 100, seed=i).cuda() for i in range(4)]
    want = [(*ops.add_rms_norm_int8(x, None, x), ops.mlp3_int8(x, layers, "tanh"), ops.linear_int8(*ops.quantize_rows(x), *layers[0])) for x in xs]
    torch.cuda.synchronize()
    done, wrong = [0] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    x = xs[i]
                    got = (*ops.add_rms_norm_int8(x, None, x), ops.mlp3_int8(x, layers, "tanh"), ops.linear_int8(*ops.quantize_rows(x), *layers[0]))
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(f"thread {i}: other values")
                    done[i] += 1
        except BaseException as e:                      # noqa: BLE001
            wrong.append(f"thread {i}: {e!r}")

    threads = [threading.Thread(target=work, args=(i,), daemon=True) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong and done == [50] * 4 and not any(t.is_alive() for t in threads)


# ------------------------------------------------------------------------------------------------ launches, as they are told
@pytest.mark.gpu
@pytest.mark.parametrize("M,dims", [(1, (24, 400, 400, 4)), (3, (111, 1024, 1024, 8)), (3, (64, 1024, 1024, 120)), (4097, (64, 1024, 1024, 120)),
                                    (2, (961, 16, 16, 128)), (2, (960, 16, 16, 128)), (2, (2048, 64, 64, 2)), (2, (3, 1025, 64, 2)), (5, (8, 64, 64, 1025))])
def test_the_policys_launches_are_told_as_they_are(M, dims):
    from d4pg_pytorch_amd.ops import hip as H
    x = _randn(M, dims[0], seed=1).cuda()
    layers = [(*ops.quantize_rows(_randn(dims[i + 1], dims[i], seed=i).cuda()), None) for i in range(3)]
    ops.mlp3_int8(x, layers)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        ops.mlp3_int8(x, layers)
    assert H.graph_kernel_nodes(graph) == H.lib().d4pg_mlp3_int8_launches(M, *dims)


@pytest.mark.gpu
@pytest.mark.parametrize("S,Hd,A,E", [(24, 400, 4, 16), (64, 1024, 120, 8), (64, 1024, 120, 4097), (3, 1100, 1, 2)])
def test_an_agent_tells_its_launches_as_they_are(S, Hd, A, E):
    from d4pg_pytorch_amd.actors.gpu_actor import GpuActor
    from d4pg_pytorch_amd.ops import hip as H
    ga = GpuActor(S, A, Hd, max_batch=E, precision="int8")
    obs = _randn(E, S, seed=1).cuda()
    ga.act_device(obs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        ga.act_device(obs)
    assert H.graph_kernel_nodes(graph) == ga.launches_per_act


@pytest.mark.parametrize("device", DEVICES)
def test_what_requires_gradients_afterwards(device):
    x = _randn(3, 20, seed=1).to(device).requires_grad_()
    q, s, h = ops.add_rms_norm_int8(x, x.detach()[0].clone().requires_grad_(), x)
    assert not any(t.requires_grad for t in (q, s, h, ops.dequantize_rows(q, s), ops.linear_int8(q, s, q, s, x[0, :3])))
    q, s, h = ops.add_rms_norm_int8(x)
    assert h is x and h.requires_grad and not s.requires_grad


# ------------------------------------------------------------------------------------------------ offsets beyond 32 bits
@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(66000, 33000, 48), (66000, 40, 33000), (40, 66000, 33000), (3, 66000, 33000)])
def test_products_whose_offsets_pass_32_bits(M, N, K):
    """More than 2^31 results, activations' codes or weights' codes; rows and columns of both ends against 64 bits."""
    def codes(rows, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        kp = (K + 15) // 16 * 16
        q = torch.randint(-127, 128, (rows, kp), generator=g, device="cuda", dtype=torch.int8)
        return q[:, :K], torch.rand(rows, generator=g, device="cuda") * 0.01 + 1e-3

    q, s = codes(M, 1)
    w, ws = codes(N, 2)
    y = ops.linear_int8(q, s, w, ws, None, "none", torch.bfloat16)
    m = torch.unique(torch.cat([torch.arange(0, min(M, 40)), torch.arange(max(M - 40, 0), M)])).cuda()
    n = torch.unique(torch.cat([torch.arange(0, min(N, 40)), torch.arange(max(N - 40, 0), N)])).cuda()
    want = (q[m].double() @ w[n].double().t().contiguous()) * s[m].double()[:, None] * ws[n].double()
    got = y[m][:, n].double()
    assert torch.all((got - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * want.abs() + 1e-30)


@pytest.mark.gpu
def test_rows_whose_offsets_pass_32_bits():
    M, K = 33, (1 << 26) + 8
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[:, 5], x[:, K - 1] = 2.0, -1.0
    q, s = ops.quantize_rows(x)
    assert torch.all(q[:, 5] == 127) and torch.all(q[:, K - 1] == -64) and torch.all(q.to(torch.int16).abs().sum(1, dtype=torch.int64) == 191)
    back = ops.dequantize_rows(q, s, torch.bfloat16)
    assert torch.all(back[:, 5] == 2.0) and torch.all(back[:, K - 2] == 0) and torch.all(back[:, K - 1] == (-64 * (torch.tensor(2.0) / 127)).bfloat16().item())
    p, t, h = ops.add_rms_norm_int8(x, None, x)
    assert torch.equal(h[-1], x[-1] * 2) and torch.equal(p[-1], q[-1])
