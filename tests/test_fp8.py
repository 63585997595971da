"""The 8-bit operators (quantize_fp8, rmsnorm_fp8, silu_mul_fp8, linear_fp8) against their formulas
in 64 bits, and their refusals.

Tolerances, with u = 2^-24 (half a step of fp32):
- scales: the roundings of the fp32 steps that form them, counted per operator;
- quantized values: e4m3 of the 64-bit quotient y / s moved down and up by the relative error d
  that fp32 leaves in it; the kernel's value lies between the two, so any value is exact unless the
  quotient is within d of the middle between two e4m3 numbers;
- products: fp32 accumulation with truncation, a step of 2^-23 of the group's sum of |x w| for each
  of its 128 terms and 4 instructions, then u for each group, split and scale factor, then the
  output's own half step.
"""
from __future__ import annotations

import ctypes
from fractions import Fraction

import pytest
import torch

U = 2.0 ** -24
FLOOR = 2.0 ** -100
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
F8 = torch.float8_e4m3fn


def _ops():
    from specb200 import ops

    return ops


def _lib():
    from specb200 import _ffi

    return _ffi.lib()


def _rand(seed, *shape, dtype=F32, spread=0.8):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(spread * torch.randn(shape[-1], generator=g))
    return x.to(DEV, dtype)


def _amax(y, block_rows=1):
    """Largest |y| of each group of 128 columns x block_rows rows, of fp64 rows [M, K]."""
    m, k = y.shape
    y = torch.nn.functional.pad(y.abs(), (0, -k % 128, 0, -m % block_rows))
    return y.reshape(y.shape[0] // block_rows, block_rows, -1, 128).amax(dim=(1, 3))


def _spread(s, m, k, block_rows=1):
    """Scales [blocks, groups] as one per element [M, K]."""
    return s.repeat_interleave(block_rows, 0)[:m].repeat_interleave(128, 1)[:, :k]


def _check_quantized(q, s, y64, d, s_tol, block_rows=1):
    """q, s as the quantization of the exact rows y64; d: relative error of y / s in fp32."""
    m, k = y64.shape
    want = _amax(y64, block_rows).clamp_min(FLOOR) / 448
    assert s.dtype == F32 and s.shape == want.shape
    assert ((s.double() - want).abs() <= s_tol * want).all()
    t = y64 / _spread(want, m, k, block_rows)
    a, b = (t * (1 - d)).to(F8).float(), (t * (1 + d)).to(F8).float()
    got = q.float()
    assert q.dtype == F8 and got.shape == t.shape
    assert ((got >= torch.minimum(a, b)) & (got <= torch.maximum(a, b))).all()


def _operands(seed, m, n, k):
    """Random e4m3 operands with scales of their own, independent of the engine's quantizers."""
    g = torch.Generator().manual_seed(seed)
    groups = -(-k // 128)

    def rows(r):
        held = torch.zeros(r, (k + 15) // 16 * 16, dtype=torch.uint8)
        held[:, :k] = (torch.randn(r, k, generator=g) * 60).clamp(-448, 448).to(F8).view(torch.uint8)
        return held.to(DEV).view(F8)[:, :k]

    x, w = rows(m), rows(n)
    xs = torch.exp(torch.randn(m, groups, generator=g)).to(DEV) * 1e-2
    ws = torch.exp(torch.randn(-(-n // 128), groups, generator=g)).to(DEV) * 1e-3
    return x, xs, w, ws


def _product64(x, xs, w, ws):
    """(y, sum of |terms|) in fp64."""
    m, k = x.shape
    n = w.shape[0]
    a = x.double() * _spread(xs.double(), m, k)
    b = w.double() * _spread(ws.double(), n, k, 128)
    return a @ b.T, a.abs() @ b.abs().T


def _check_product(y, x, xs, w, ws, out_f32):
    want, mag = _product64(x, xs, w, ws)
    groups = xs.shape[-1]
    tol = mag * (132 * 2.0 ** -23 + (groups + 8 + 3) * U)
    if not out_f32:
        tol = tol + (want.abs() + tol) * 2.0 ** -8
    assert y.dtype == (F32 if out_f32 else BF16) and y.shape == want.shape
    err = (y.double() - want).abs()
    assert (err <= tol).all(), f"worst error / tolerance {(err / tol.clamp_min(1e-300)).max().item():.3g}"


# ---------------------------------------------------------------- refusals, on the host
def _buf(nbytes=4096, offset=0):
    """A host address that the argument checks may look at (the calls below are refused before any launch)."""
    raw = (ctypes.c_char * (nbytes + 64))()
    base = (ctypes.addressof(raw) + 15) // 16 * 16
    return raw, base + offset


def test_quantize_refuses_bad_arguments_on_the_host():
    from specb200 import _ffi

    lib = _lib()
    keep, p = _buf()
    ok = dict(dtype=_ffi.BF16, x=p, ldx=64, M=2, K=64, rows=1, q=p, ldq=64, s=p)
    call = lambda **k: lib.specb200_quantize_fp8(*{**ok, **k}.values(), None)  # noqa: E731
    for bad in (dict(M=-1), dict(K=0), dict(ldx=63), dict(ldq=63), dict(rows=2), dict(rows=64), dict(x=None),
                dict(q=None), dict(s=None)):
        assert call(**bad) == _ffi.ERR_ARG, bad
        assert b"quantize_fp8" in lib.specb200_last_error()
    assert call(dtype=2) == _ffi.ERR_UNSUPPORTED
    assert call(M=0, x=None, q=None, s=None) == _ffi.OK
    assert call(M=2 ** 31 - 1, K=2 ** 30, ldx=2 ** 30, ldq=2 ** 30) == _ffi.ERR_ARG


def test_rmsnorm_refuses_bad_arguments_on_the_host():
    from specb200 import _ffi

    lib = _lib()
    keep, p = _buf()
    ok = dict(dtype=_ffi.F32, x=p, ldx=64, d=p, ldd=64, w=p, M=2, H=64, eps=1e-5, h=p, ldh=64, q=p, ldq=64, s=p)
    call = lambda **k: lib.specb200_rmsnorm_fp8(*{**ok, **k}.values(), None)  # noqa: E731
    for bad in (dict(M=-1), dict(H=0), dict(ldx=63), dict(ldd=63), dict(ldh=63), dict(ldq=63), dict(x=None),
                dict(w=None), dict(h=None), dict(q=None), dict(s=None)):
        assert call(**bad) == _ffi.ERR_ARG, bad
    assert call(dtype=7) == _ffi.ERR_UNSUPPORTED
    assert call(H=32769, ldx=40000, ldd=40000, ldh=40000, ldq=40000) == _ffi.ERR_UNSUPPORTED
    assert call(M=0) == _ffi.OK


def test_silu_mul_refuses_bad_arguments_on_the_host():
    from specb200 import _ffi

    lib = _lib()
    keep, p = _buf()
    ok = dict(dtype=_ffi.BF16, x=p, ld=128, M=2, I=64, packed=0, q=p, ldq=64, s=p)
    call = lambda **k: lib.specb200_silu_mul_fp8(*{**ok, **k}.values(), None)  # noqa: E731
    for bad in (dict(M=-1), dict(I=0), dict(ld=127), dict(ldq=63), dict(packed=1, I=32), dict(x=None), dict(q=None),
                dict(s=None)):
        assert call(**bad) == _ffi.ERR_ARG, bad
    assert call(dtype=-1) == _ffi.ERR_UNSUPPORTED
    assert call(M=0) == _ffi.OK


def test_linear_refuses_bad_arguments_on_the_host():
    from specb200 import _ffi

    lib = _lib()
    keep, p = _buf()
    ok = dict(x=p, ldx=64, xs=p, w=p, ldw=64, ws=p, M=2, N=16, K=64, f32=0, y=p, ldy=16, status=None)
    call = lambda **k: lib.specb200_linear_fp8(*{**ok, **k}.values(), None)  # noqa: E731
    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(ldx=48), dict(ldw=48), dict(ldx=72), dict(ldw=72), dict(ldy=15),
                dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(y=None), dict(x=p + 8), dict(w=p + 1)):
        assert call(**bad) == _ffi.ERR_ARG, bad
        assert b"linear_fp8" in lib.specb200_last_error()
    assert call(M=0) == _ffi.OK


def test_pointers_off_their_elements_are_refused_on_the_host():
    """Kernels read single elements at the ends of rows: a pointer between two of them would be a misaligned access."""
    from specb200 import _ffi

    lib = _lib()
    keep, p = _buf()

    def refused(call, ok, **bad):
        assert call(*{**ok, **bad}.values(), None) == _ffi.ERR_ARG, bad
        assert b"boundary of its elements" in lib.specb200_last_error(), bad

    for dtype, off in ((_ffi.BF16, 1), (_ffi.F32, 2)):
        ok = dict(dtype=dtype, x=p, ldx=64, M=2, K=64, rows=1, q=p, ldq=64, s=p)
        for bad in (dict(x=p + off), dict(s=p + 2)):
            refused(lib.specb200_quantize_fp8, ok, **bad)
            refused(lib.specb200_quantize_fp8, ok, rows=128, **bad)
        ok = dict(dtype=dtype, x=p, ldx=64, d=p, ldd=64, w=p, M=2, H=64, eps=1e-5, h=p, ldh=64, q=p, ldq=64, s=p)
        for bad in (dict(x=p + off), dict(d=p + off), dict(w=p + off), dict(h=p + off), dict(s=p + 1)):
            refused(lib.specb200_rmsnorm_fp8, ok, **bad)
        ok = dict(dtype=dtype, x=p, ld=128, M=2, I=64, packed=0, q=p, ldq=64, s=p)
        for bad in (dict(x=p + off), dict(s=p + 2)):
            refused(lib.specb200_silu_mul_fp8, ok, **bad)
    ok = dict(x=p, ldx=64, xs=p, w=p, ldw=64, ws=p, M=2, N=16, K=64, f32=0, y=p, ldy=16, status=None)
    for bad in (dict(xs=p + 2), dict(ws=p + 1), dict(y=p + 1), dict(f32=1, y=p + 2), dict(status=p + 2)):
        refused(lib.specb200_linear_fp8, ok, **bad)


def test_a_residual_in_place_has_its_own_pitch():
    from specb200 import _ffi

    lib = _lib()
    keep, p = _buf()
    ok = dict(dtype=_ffi.BF16, x=p, ldx=64, d=p + 256, ldd=72, w=p, M=2, H=64, eps=1e-5, h=p, ldh=72, q=p, ldq=64, s=p)
    for change in ({}, dict(h=p + 256, ldh=64)):
        assert lib.specb200_rmsnorm_fp8(*{**ok, **change}.values(), None) == _ffi.ERR_ARG
        assert b"row pitch" in lib.specb200_last_error()


def test_host_tensors_are_refused():
    x = torch.zeros(2, 64)
    for call in (lambda o: o.quantize_fp8(x), lambda o: o.rmsnorm_fp8(x, x[0], 1e-5), lambda o: o.silu_mul_fp8(x),
                 lambda o: o.linear_fp8(x.to(F8), x, x.to(F8), x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call(_ops())


def test_the_extension_module_is_built_again_for_another_torch(monkeypatch, tmp_path):
    """It uses torch's C++ classes: one that was built for another torch is neither taken for up to date nor loaded."""
    from specb200 import _ffi, build

    runs = []

    def run(cmd, what, verbose):
        runs.append(cmd)
        build.Path(cmd[cmd.index("-o") + 1]).write_bytes(b"built")

    monkeypatch.setattr(build, "_run", run)
    monkeypatch.setattr(build, "TORCH_OPS", tmp_path / "_torch_ops.so")
    for want in (1, 1):
        build.build_torch_ops()
        assert len(runs) == want
    (tmp_path / "_torch_ops.stamp").unlink()  # a module of unknown origin
    build.build_torch_ops()
    assert len(runs) == 2
    module = _ffi.torch_ops()
    assert module.target == build.torch_ops_target()
    monkeypatch.setattr(torch, "__version__", "2.99.0")
    build.build_torch_ops()
    build.build_torch_ops()
    assert len(runs) == 3 and any("2.99.0" in arg for arg in runs[-1])
    with pytest.raises(RuntimeError, match="build it again"):
        _ffi.torch_ops()
    monkeypatch.delattr(module, "target")  # a module from before it said so
    with pytest.raises(RuntimeError, match="unknown torch"):
        _ffi.torch_ops()
    monkeypatch.setattr(build.shutil, "which", lambda name: None)
    with pytest.raises(RuntimeError, match="g\\+\\+ not found"):
        build.build_torch_ops(force=True)


def test_negated_views_are_refused():
    """The imaginary part of a conjugate holds its values with the other sign in memory."""
    x, neg = torch.zeros(2, 64), torch.zeros(2, 1, dtype=torch.complex64).conj().imag
    for call in (lambda o: o.quantize_fp8(neg), lambda o: o.rmsnorm_fp8(neg, neg[0], 1e-5),
                 lambda o: o.rmsnorm_fp8(x, x[0], 1e-5, delta=neg), lambda o: o.silu_mul_fp8(neg),
                 lambda o: o.linear_fp8(x.to(F8), neg, x.to(F8), x)):
        with pytest.raises(ValueError, match="resolve_neg"):
            call(_ops())


@pytest.mark.gpu
def test_wrappers_refuse_mismatched_tensors():
    ops = _ops()
    x = torch.zeros(4, 256, device=DEV, dtype=BF16)
    with pytest.raises(NotImplementedError):
        ops.quantize_fp8(x.half())
    with pytest.raises(ValueError):
        ops.quantize_fp8(x, block_rows=2)
    with pytest.raises(ValueError):
        ops.quantize_fp8(x.view(2, 2, 256), block_rows=128)
    with pytest.raises(ValueError):
        ops.quantize_fp8(x[:, :0])
    with pytest.raises(ValueError):
        ops.rmsnorm_fp8(x, x[0, :128], 1e-5)
    with pytest.raises(ValueError):
        ops.rmsnorm_fp8(x, x[0].float(), 1e-5)
    with pytest.raises(ValueError):
        ops.rmsnorm_fp8(x, x[0], 1e-5, delta=x[:2])
    with pytest.raises(ValueError):
        ops.rmsnorm_fp8(x, x[0].cpu(), 1e-5)
    with pytest.raises(NotImplementedError):
        ops.rmsnorm_fp8(torch.zeros(1, 32776, device=DEV), torch.ones(32776, device=DEV), 1e-5)
    with pytest.raises(ValueError):
        ops.silu_mul_fp8(x[:, :255])
    with pytest.raises(ValueError):
        ops.silu_mul_fp8(x[:, :192], packed=True)
    q, s = ops.quantize_fp8(x)
    w, ws = ops.quantize_fp8(torch.zeros(130, 256, device=DEV, dtype=BF16), block_rows=128)
    for bad in ((x, s, w, ws), (q, s, x, ws), (q[:, :128], s, w, ws), (q, s[:, :1], w, ws), (q, s, w, ws[:1]),
                (q, s.double(), w, ws), (q, s, w, ws.bfloat16()), (q, s.cpu(), w, ws), (q, s, w[0], ws)):
        with pytest.raises(ValueError):
            ops.linear_fp8(*bad)


# ---------------------------------------------------------------- quantize
SIZES = [(1, 1), (1, 16), (3, 127), (5, 128), (7, 129), (130, 576), (257, 2048), (129, 1000), (1, 8192)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("m,k", SIZES)
def test_quantize(m, k, block_rows, dtype):
    x = _rand(m * 7 + k, m, k, dtype=dtype)
    q, s = _ops().quantize_fp8(x, block_rows=block_rows)
    _check_quantized(q, s, x.double(), d=4 * U, s_tol=2 * U, block_rows=block_rows)  # 448/amax, product; amax/448


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_of_views(block_rows, dtype):
    """Columns of a wider matrix (rows off any 16-byte boundary), every other row, a transposed view."""
    wide = _rand(1, 60, 700, dtype=dtype)
    for x in (wide[:, 1:301], wide[:, 8:264], wide[::2, 3:200], wide.t(), wide[0:1, 5:600]):
        q, s = _ops().quantize_fp8(x, block_rows=block_rows)
        _check_quantized(q, s, x.double(), d=4 * U, s_tol=2 * U, block_rows=block_rows)


@pytest.mark.gpu
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_edge_values(block_rows):
    """Groups of zeros, of values below the floor, near fp32's ends, and groups that hold a NaN or an infinity."""
    x = _rand(2, 4, 128 * 7)
    x[:, 0:128] = 0
    x[:, 128:256] *= 1e-33
    x[:, 256:384] *= 1e-38
    x[:, 384:512] *= 1e36
    x[2, 512] = float("nan")
    x[1, 640] = float("inf")
    q, s = _ops().quantize_fp8(x, block_rows=block_rows)
    keep = [0, 1, 2, 3, 6]
    cols = torch.cat([torch.arange(g * 128, g * 128 + 128) for g in keep]).to(DEV)
    _check_quantized(q.float()[:, cols].to(F8), s[:, keep], x[:, cols].double(), d=4 * U, s_tol=2 * U,
                     block_rows=block_rows)
    qn, qi = q.float()[:, 512:640], q.float()[:, 640:768]
    rows_n = [2] if block_rows == 1 else [0, 1, 2, 3]
    rows_i = [1] if block_rows == 1 else [0, 1, 2, 3]
    assert qn[rows_n].isnan().all() and s[rows_n if block_rows == 1 else 0, 4].isnan().all()
    assert torch.isinf(s[rows_i if block_rows == 1 else 0, 5]).all() and qi[1, 0].isnan()
    rest = qi[rows_i].clone()
    rest[rows_i.index(1), 0] = 0
    assert (rest == 0).all()


def _fp32(v):
    """The fp32 number nearest to a positive fraction, ties to even, and half a step there (no underflow)."""
    e = v.numerator.bit_length() - v.denominator.bit_length()
    if Fraction(2) ** e > v:
        e -= 1
    step = Fraction(2) ** (e - 23)
    return round(v / step) * step, step / 2


def test_quotients_of_bf16_values_keep_off_the_middle_of_two_fp32_numbers():
    """x / s with s = amax / 448 rounded to fp32, over all bf16 mantissas of x and amax (powers of two change
    nothing): whatever is within 2^-41 of the quotient, relatively, rounds as the quotient does. The bf16
    quantizer forms it to 2^-42 before the rounding."""
    for amax in range(128, 256):
        s, _ = _fp32(Fraction(amax, 448))
        for x in range(128, 256):
            quotient = x / s
            nearest, half = _fp32(quotient)
            assert half - abs(quotient - nearest) > quotient * Fraction(1, 2 ** 41), (x, amax)


def test_scales_are_quotients_by_448():
    """amax hi + amax lo with hi + lo = 1 / 448 to 2^-51: amax / 448 is no nearer than 2^-28 of itself to the
    middle of two fp32 numbers, because the distance is a multiple of 1 / 14 of a step."""
    for amax in list(range(2 ** 23, 2 ** 24, 9973)) + list(range(2 ** 24 - 64, 2 ** 24)):
        quotient = Fraction(amax, 448)
        nearest, half = _fp32(quotient)
        assert half - abs(quotient - nearest) >= half / 7 > quotient * Fraction(1, 2 ** 28)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("m,k,start", [(321, 2048, 0), (300, 1000, 0), (130, 301, 3), (1, 127, 1)])
def test_quantize_divides_by_the_scale_it_returns(m, k, start, block_rows, dtype):
    """Bit for bit s = max(max |x|, 2^-100) / 448 and q = e4m3(x / s) in fp32, from rows on 16-byte boundaries and
    off them: ordinary values, whole numbers (whose quotients lie between two e4m3 numbers but for the
    scale's rounding), columns below the floor and beyond 1e30, zeros of both signs, a NaN and an infinity."""
    wide = _rand(m + k, m, k + start, dtype=dtype)
    whole = torch.randint(-300, 301, (m, k + start), generator=torch.Generator().manual_seed(m)).to(DEV, dtype)
    far = wide.clone()
    for i, factor in enumerate((1e-38, 1e-33, 2.0 ** -64, 1e-12, 1e12, 2.0 ** 60, 1e30)):
        far[:, 128 * i:128 * (i + 1)] *= factor
    far[:, ::5] = 0
    far[:, 2::10] = -0.0
    odd = wide.clone()
    odd[m // 2, k // 2] = float("nan")
    odd[m // 3, 0] = float("-inf")
    for held in (wide, whole, far, odd):
        x = held[:, start:]
        q, s = _ops().quantize_fp8(x, block_rows=block_rows)
        f = torch.nn.functional.pad(x.float().abs(), (0, -k % 128, 0, -m % block_rows))
        # in 64 bits, then rounded: torch multiplies fp32 CUDA tensors by 1 / 448 where it is asked to divide by a number
        want = (f.reshape(f.shape[0] // block_rows, block_rows, -1, 128).amax(dim=(1, 3)).clamp_min(FLOOR).double() / 448).float()
        assert torch.equal(s.view(torch.int32)[~s.isnan()], want.view(torch.int32)[~want.isnan()])
        assert torch.equal(s.isnan(), want.isnan())
        quotient = (x.float() / _spread(want, m, k, block_rows)).to(F8)
        nan = quotient.float().isnan()
        assert torch.equal(q.float().isnan(), nan)
        assert torch.equal(q.contiguous().view(torch.uint8)[~nan], quotient.view(torch.uint8)[~nan])


@pytest.mark.gpu
def test_rows_of_leading_dimensions():
    ops = _ops()
    x = _rand(3, 2, 3, 200, dtype=BF16)
    q, s = ops.quantize_fp8(x)
    q2, s2 = ops.quantize_fp8(x.view(6, 200))
    assert q.shape == (2, 3, 200) and s.shape == (2, 3, 2)
    assert torch.equal(q.float().view(6, 200), q2.float()) and torch.equal(s.view(6, 2), s2)
    q1, s1 = ops.quantize_fp8(x[0, 0])
    assert torch.equal(q1.float(), q2.float()[0]) and torch.equal(s1, s2[0])
    w, ws = ops.quantize_fp8(_rand(4, 96, 200, dtype=BF16), block_rows=128)
    y = ops.linear_fp8(q, s, w, ws)
    assert y.shape == (2, 3, 96) and torch.equal(y.view(6, 96), ops.linear_fp8(q2, s2, w, ws))
    assert torch.equal(ops.linear_fp8(q1, s1, w, ws), y[0, 0])


@pytest.mark.gpu
def test_no_rows():
    ops = _ops()
    x = torch.zeros(0, 200, device=DEV, dtype=BF16)
    q, s = ops.quantize_fp8(x)
    assert q.shape == (0, 200) and s.shape == (0, 2)
    w, ws = ops.quantize_fp8(_rand(4, 96, 200, dtype=BF16), block_rows=128)
    assert ops.linear_fp8(q, s, w, ws).shape == (0, 96)
    q, s, h = ops.rmsnorm_fp8(x, x.new_ones(200), 1e-5, delta=x)
    assert q.shape == (0, 200) and s.shape == (0, 2) and h.shape == (0, 200)
    q, s = ops.silu_mul_fp8(x)
    assert q.shape == (0, 100) and s.shape == (0, 1)
    q, s = ops.quantize_fp8(torch.zeros(2, 0, 64, device=DEV))
    assert q.shape == (2, 0, 64) and s.shape == (2, 0, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["rows", "blocks", "norm", "silu"])
def test_nothing_is_written_outside_the_rows(op):
    """Through the C ABI into buffers with a pitch and a frame of their own, at an odd offset."""
    from specb200 import _ffi

    lib = _lib()
    m, k, pitch = 5, 201, 230
    x = _rand(5, m, 2 * k, dtype=BF16)
    weight = _rand(6, k, dtype=BF16)
    q = torch.full((m + 2, pitch), 0x55, dtype=torch.uint8, device=DEV)
    blocks = 1 if op == "blocks" else m
    s = torch.full((blocks + 2, 2), -7.0, device=DEV)
    h = torch.full((m + 2, pitch), 3.0, dtype=BF16, device=DEV)
    qp, sp, hp = q[1].data_ptr() + 3, s[1].data_ptr(), h[1].data_ptr() + 2 * 5
    st = torch.cuda.current_stream().cuda_stream
    if op in ("rows", "blocks"):
        rc = lib.specb200_quantize_fp8(_ffi.BF16, x.data_ptr(), 2 * k, m, k, 1 if op == "rows" else 128, qp, pitch, sp, st)
    elif op == "norm":
        rc = lib.specb200_rmsnorm_fp8(_ffi.BF16, x.data_ptr(), 2 * k, x.data_ptr() + 2 * k, 2 * k, weight.data_ptr(), m, k,
                                      1e-5, hp, pitch, qp, pitch, sp, st)
    else:
        rc = lib.specb200_silu_mul_fp8(_ffi.BF16, x.data_ptr(), 2 * k, m, k, 0, qp, pitch, sp, st)
    assert rc == 0, lib.specb200_last_error()
    flat = q.flatten()
    inside = torch.zeros_like(flat, dtype=torch.bool)
    for r in range(m):
        inside[pitch + 3 + r * pitch: pitch + 3 + r * pitch + k] = True
    assert (flat[~inside] == 0x55).all() and (flat[inside] != 0x55).any()
    assert (s[0] == -7).all() and (s[blocks + 1] == -7).all() and (s[1:blocks + 1] > 0).all()
    if op == "norm":
        flat = h.flatten()
        inside = torch.zeros_like(flat, dtype=torch.bool)
        for r in range(m):
            inside[pitch + 5 + r * pitch: pitch + 5 + r * pitch + k] = True
        assert (flat[~inside] == 3).all()
        assert torch.equal(flat[inside].view(m, k), (x[:, :k].float() + x[:, k:].float()).to(BF16))


# ---------------------------------------------------------------- RMSNorm
# The sum of squares: at most 16 in a chain, 4 chunks, 3 shuffles and 64 octets in 4 chains of 16 and their
# join, so 41 roundings (69 allowed); half of that in 1 / rms, then the mean, the sum with eps, the
# root, the quotient, w h, (w h) r and / 448.
NORM_S = (69 / 2 + 7) * U


def _norm64(h, weight, eps):
    h = h.double()
    return h * (h.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.double()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("delta", [False, True])
@pytest.mark.parametrize("m,k", SIZES + [(3, 8200), (2, 16392), (2, 32768), (700, 64)])
def test_rmsnorm(m, k, delta, dtype):
    x = _rand(m + 3 * k, m, k, dtype=dtype)
    weight = (1 + 0.3 * _rand(k, k, spread=0.0)).to(dtype)
    d = _rand(m + k, m, k, dtype=dtype) if delta else None
    out = _ops().rmsnorm_fp8(x, weight, 1e-5, delta=d)
    h = x
    if delta:
        h = (x.float() + d.float()).to(dtype)
        assert torch.equal(out[2], h)
    assert len(out) == (3 if delta else 2)
    _check_quantized(out[0], out[1], _norm64(h, weight, 1e-5), d=4 * U, s_tol=NORM_S)  # w h, 448 / max, product


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rmsnorm_of_views_and_in_place(dtype):
    from specb200 import _ffi

    lib = _lib()
    wide = _rand(7, 20, 900, dtype=dtype)
    weight = _rand(8, 300, dtype=dtype)
    for x, d in ((wide[:, 1:301], wide[:, 401:701]), (wide[::2, 16:316], wide[::2, 320:620])):
        q, s, h = _ops().rmsnorm_fp8(x, weight, 1e-6, delta=d)
        want = (x.float() + d.float()).to(dtype)
        assert torch.equal(h, want)
        _check_quantized(q, s, _norm64(want, weight, 1e-6), d=4 * U, s_tol=NORM_S)
    # the residual stream updated in its place (h = x)
    m, k = 6, 300
    x, d = wide[:m, :k].contiguous(), wide[:m, 400:400 + k].contiguous()
    q, s, h = _ops().rmsnorm_fp8(x, weight, 1e-6, delta=d)
    q2, s2 = torch.empty(m, k, dtype=torch.uint8, device=DEV), torch.empty_like(s)
    rc = lib.specb200_rmsnorm_fp8(_ffi.BF16 if dtype == BF16 else _ffi.F32, x.data_ptr(), k, d.data_ptr(), k,
                                  weight.data_ptr(), m, k, 1e-6, x.data_ptr(), k, q2.data_ptr(), k, s2.data_ptr(),
                                  torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(x, h) and torch.equal(s2, s) and torch.equal(q2, q.contiguous().view(torch.uint8))


# more rows than the grid takes at once, with a ragged last round: loads ahead (one group per octet), several rows
# per CTA on and off the 16-byte boundaries (teams that meet inside a warp), two and four groups per octet
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k", [(5000, 2048), (14001, 576), (9001, 129), (20001, 301), (1500, 4104), (1300, 4105), (700, 8201),
                                 (3, 8201), (2, 32767), (40000, 64)])
def test_rmsnorm_walks_over_its_rows(m, k, dtype):
    from specb200 import _ffi

    ops, lib = _ops(), _lib()
    x, d = _rand(m + k, m, k, dtype=dtype), _rand(m + k + 1, m, k, dtype=dtype)
    weight = (1 + 0.3 * _rand(k, k, spread=0.0)).to(dtype)
    q, s = ops.rmsnorm_fp8(x, weight, 1e-5)
    _check_quantized(q, s, _norm64(x, weight, 1e-5), d=4 * U, s_tol=NORM_S)
    q, s, h = ops.rmsnorm_fp8(x, weight, 1e-5, delta=d)
    assert torch.equal(h, (x.float() + d.float()).to(dtype))
    _check_quantized(q, s, _norm64(h, weight, 1e-5), d=4 * U, s_tol=NORM_S)
    # the same in the place of x and of delta, through the C ABI and into dense rows
    for place in (0, 1):
        x2, d2 = x.clone(), d.clone()
        h2 = d2 if place else x2
        q2, s2 = torch.empty(m, k, dtype=torch.uint8, device=DEV), torch.empty_like(s)
        rc = lib.specb200_rmsnorm_fp8(_ffi.BF16 if dtype == BF16 else _ffi.F32, x2.data_ptr(), k, d2.data_ptr(), k,
                                      weight.data_ptr(), m, k, 1e-5, h2.data_ptr(), k, q2.data_ptr(), k, s2.data_ptr(),
                                      torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(h2, h) and torch.equal(s2, s) and torch.equal(q2.view(F8).float(), q.float())


@pytest.mark.gpu
def test_one_row_in_place_with_any_pitch():
    from specb200 import _ffi

    x, d, weight = (_rand(i, 64, dtype=BF16) for i in (20, 21, 22))
    want = _ops().rmsnorm_fp8(x, weight, 1e-5, delta=d)
    q, s = torch.empty(64, dtype=torch.uint8, device=DEV), torch.empty_like(want[1])
    rc = _lib().specb200_rmsnorm_fp8(_ffi.BF16, x.data_ptr(), 64, d.data_ptr(), 72, weight.data_ptr(), 1, 64, 1e-5,
                                     x.data_ptr(), 100, q.data_ptr(), 64, s.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(x, want[2]) and torch.equal(s, want[1]) and torch.equal(q.view(F8).float(), want[0].float())


@pytest.mark.gpu
def test_rmsnorm_edge_rows():
    """A row of zeros, rows so small that eps decides, groups under the floor, weights of zero, and
    rows that hold a NaN or an infinity: each keeps to itself."""
    k = 400
    x = _rand(9, 8, k)
    x[0] = 0
    x[1] *= 1e-20
    x[2, :128] *= 1e-36
    x[3, :128] = 0
    x[4, 7] = float("nan")
    x[5, 7] = float("inf")
    x[6] *= 1e15
    weight = _rand(10, k)
    weight[128:256] = 0
    q, s = _ops().rmsnorm_fp8(x, weight, 1e-5)
    ok = [0, 1, 2, 3, 6, 7]
    _check_quantized(q.float()[ok].to(F8), s[ok], _norm64(x[ok], weight, 1e-5), d=NORM_S + 4 * U, s_tol=NORM_S)
    assert s[4].isnan().all() and q.float()[4].isnan().all()
    # 1 / rms is zero: finite elements give zero, the infinite one NaN
    assert s[5, 0].isnan() and q.float()[5, :128].isnan().all() and (q.float()[5, 128:] == 0).all()


# ---------------------------------------------------------------- SiLU * up
# The exponent -g log2(e) carries the constant's and the product's rounding, 2 |g| u in the
# exponential (gates beyond 90 give 0 or g u), the exponential itself 4 u (2^-22); then the sum, the
# reciprocal (2 u) and two products: y is off by at most (2 |g| + 9) u. The scale adds its division; the
# quotient y / s has that error twice, 448 / amax and the product.
def _silu_tol(g):
    y = (2 * min(g.abs().max().item(), 90.0) + 9) * U
    return {"d": 2 * y + 2 * U, "s_tol": y + 2 * U}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("m,k", [(1, 64), (5, 128), (3, 192), (130, 576), (257, 2048), (1, 8192)])
def test_silu_mul(m, k, packed, dtype):
    x = _rand(m * 11 + k, m, 2 * k, dtype=dtype, spread=0.3)
    q, s = _ops().silu_mul_fp8(x, packed=packed)
    if packed:
        g, u = (v.reshape(m, k).double() for v in x.view(m, k // 64, 2, 64).unbind(2))
    else:
        g, u = x[:, :k].double(), x[:, k:].double()
    _check_quantized(q, s, g * torch.sigmoid(g) * u, **_silu_tol(g))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_silu_mul_odd_widths_and_views(dtype):
    wide = _rand(12, 40, 1000, dtype=dtype, spread=0.3)
    for x in (wide[:, :2], wide[:, 1:255], wide[::2, 8:408], wide[:7, 3:997]):
        q, s = _ops().silu_mul_fp8(x)
        k = x.shape[1] // 2
        g, u = x[:, :k].double(), x[:, k:].double()
        _check_quantized(q, s, g * torch.sigmoid(g) * u, **_silu_tol(g))
    x = wide[::3, 5:5 + 256]
    q, s = _ops().silu_mul_fp8(x, packed=True)
    g, u = (v.reshape(x.shape[0], 128).double() for v in x.reshape(x.shape[0], 2, 2, 64).unbind(2))
    _check_quantized(q, s, g * torch.sigmoid(g) * u, **_silu_tol(g))


@pytest.mark.gpu
def test_silu_mul_far_gates():
    """Gates whose exponential overflows or vanishes, and NaN."""
    g = torch.tensor([-1e4, -200.0, -88.0, -50.0, 0.0, 50.0, 88.0, 200.0, 1e4], device=DEV)
    x = torch.cat([g, torch.full_like(g, 2.0)])[None]
    q, s = _ops().silu_mul_fp8(x)
    _check_quantized(q, s, (g.double() * torch.sigmoid(g.double()) * 2)[None], **_silu_tol(g))
    # a sweep over where the exponential overflows, one positive gate in each group
    g = torch.linspace(-300.0, -80.0, 128 * 40, device=DEV).view(40, 128).contiguous()
    g[:, 64] = 3.0
    q, s = _ops().silu_mul_fp8(torch.cat([g, torch.full_like(g, 2.0)], 1))
    _check_quantized(q, s, g.double() * torch.sigmoid(g.double()) * 2, **_silu_tol(g))
    x[0, 3] = float("nan")
    q, s = _ops().silu_mul_fp8(x)
    assert s.isnan().all() and q.float().isnan().all()


# Below -87: e^(g/2) to 4 u (2 ulp) twice, four products and the half steps of the fp32 gate and up themselves, which
# are exact; subnormal halves (below -174.7) keep at least 20 bits down to -177. 16 u with those, 2^-18.
def _check_far(x, k, packed=False):
    q, s = _ops().silu_mul_fp8(x, packed=packed)
    g, u = x.view(x.shape[0], k // 64, 2, 64).unbind(2) if packed else (x[:, :k], x[:, k:])
    g, u = g.reshape(-1, k).double(), u.reshape(-1, k).double()
    y = g * u / (1 + torch.exp(-g))
    far = 2 * U * g.abs().max().item() + 16 * U if (g > -87).any() else 16 * U
    far = max(far, 2.0 ** -18) if (g < -174).any() else far
    _check_quantized(q, s, y, d=2 * far + 2 * U, s_tol=far + 2 * U)
    return q


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("packed", [False, True])
def test_silu_mul_gates_whose_sigmoid_leaves_fp32(dtype, packed):
    """Groups that hold nothing but far gates, with `up` values large enough to lift them above the floor: around
    -87 .. -89, where a rounded-off reciprocal is zero first, and on to where no fp32 `up` lifts them."""
    k = 1024
    for lo, hi, up in ((-88.7, -87.36, 1e8), (-90.0, -85.0, 1e12), (-104.0, -80.0, 1e20), (-150.0, -100.0, 1e37),
                       (-176.0, -150.0, 3e38), (-177.0, -60.0, 1e37)):
        g = torch.linspace(lo, hi, 3 * k, device=DEV).view(3, k)
        u = up * (1 - 0.3 * torch.rand(3, k, generator=torch.Generator().manual_seed(3)).to(DEV))
        x = torch.stack([v.view(3, k // 64, 64) for v in (g, u)], 2).reshape(3, 2 * k) if packed else torch.cat([g, u], 1)
        q = _check_far(x.to(dtype).contiguous(), k, packed)
        assert (q.float() != 0).any(), (lo, hi)
    # gates beyond any range, and the formula's values for infinite ones
    g = torch.full((1, 128), -1e4, device=DEV)
    q, s = _ops().silu_mul_fp8(torch.cat([g, torch.full_like(g, 3e38)], 1).to(dtype))
    assert (q.float() == 0).all() and (s == FLOOR / 448).all()
    g[0, 3] = float("-inf")
    q, s = _ops().silu_mul_fp8(torch.cat([g, torch.full_like(g, 2.0)], 1).to(dtype))
    assert s.isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,starts", [(BF16, range(8)), (F32, range(4))])
@pytest.mark.parametrize("k,pitch", [(301, 301), (5, 5), (130, 134), (2049, 2051), (5002, 5002)])
def test_rows_on_any_boundary(k, pitch, dtype, starts):
    """Rows that start anywhere in a 16-byte unit, the first and last ones at the ends of their memory: the
    same bits as from aligned rows, and the residual stream updated in its place with nothing around it touched."""
    from specb200 import _ffi

    ops, m = _ops(), 9
    code, stream = _ffi.BF16 if dtype == BF16 else _ffi.F32, torch.cuda.current_stream().cuda_stream
    x, d, weight = _rand(13, m, k, dtype=dtype), _rand(14, m, k, dtype=dtype), _rand(15, k, dtype=dtype)

    def aligned(t):
        held = torch.zeros(t.shape[0], (t.shape[1] + 15) // 16 * 16, dtype=dtype, device=DEV)
        held[:, :t.shape[1]] = t
        return held[:, :t.shape[1]]

    def placed(t, start):
        flat = torch.full(((m - 1) * pitch + k + start,), float("nan"), dtype=dtype, device=DEV)
        view = flat.as_strided((m, k), (pitch, 1), start)
        view.copy_(t)
        return view

    def same(got, want):
        assert len(got) == len(want)
        for g, w in zip(got, want):
            assert torch.equal(g.float(), w.float())

    want_rows, want_blocks = ops.quantize_fp8(aligned(x)), ops.quantize_fp8(aligned(x), block_rows=128)
    want_norm = ops.rmsnorm_fp8(aligned(x), weight, 1e-5, delta=aligned(d))
    want_plain = ops.rmsnorm_fp8(aligned(x), weight, 1e-5)
    assert torch.equal(want_norm[2], (x.float() + d.float()).to(dtype))
    half = k // 2
    for start in starts:
        v = placed(x, start)
        same(ops.quantize_fp8(v), want_rows)
        same(ops.quantize_fp8(v, block_rows=128), want_blocks)
        same(ops.rmsnorm_fp8(v, weight, 1e-5, delta=placed(d, (start * 3) % len(starts))), want_norm)
        same(ops.rmsnorm_fp8(v, placed(weight[None].expand(m, k), start)[1], 1e-5), want_plain)
        g, u = v[:, :half].double(), v[:, half:2 * half].double()
        q, s = ops.silu_mul_fp8(v[:, :2 * half])
        _check_quantized(q, s, g * torch.sigmoid(g) * u, **_silu_tol(g))
        # h in x's place inside a frame, through the C ABI
        frame = torch.full((m * pitch + 40,), 7.0, dtype=dtype, device=DEV)
        at = 16 + start
        h = frame.as_strided((m, k), (pitch, 1), at)
        h.copy_(x)
        q2, s2 = torch.empty(m, k, dtype=torch.uint8, device=DEV), torch.empty_like(want_norm[1])
        rc = _lib().specb200_rmsnorm_fp8(code, h.data_ptr(), pitch, d.data_ptr(), k, weight.data_ptr(), m, k, 1e-5,
                                         h.data_ptr(), pitch, q2.data_ptr(), k, s2.data_ptr(), stream)
        assert rc == 0
        same((q2.view(F8), s2, h), want_norm)
        outside = torch.ones_like(frame, dtype=torch.bool)
        outside.as_strided((m, k), (pitch, 1), at).fill_(False)
        assert (frame[outside] == 7).all()


# ---------------------------------------------------------------- linear
LINEAR = [(1, 1, 1), (1, 16, 16), (1, 128, 128), (2, 130, 129), (5, 960, 576), (8, 256, 2048), (9, 6144, 2048),
          (33, 2048, 8192), (16, 500, 4096), (17, 500, 4096), (15, 40000, 256), (64, 1000, 1000), (127, 300, 200), (128, 128, 640), (129, 257, 384), (320, 2048, 1024),
          (513, 1024, 300), (1000, 1536, 576), (2049, 4100, 520), (3000, 5000, 130)]


@pytest.mark.gpu
@pytest.mark.parametrize("out_f32", [False, True])
@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear(m, n, k, out_f32):
    x, xs, w, ws = _operands(m + n + k, m, n, k)
    y = _ops().linear_fp8(x, xs, w, ws, out_f32=out_f32)
    _check_product(y, x, xs, w, ws, out_f32)


@pytest.mark.gpu
def test_linear_of_views():
    """Rows off the 16-byte boundaries (copied), a column block of a wider matrix, strided scales."""
    ops = _ops()
    x, xs, w, ws = _operands(21, 40, 300, 512)
    y = ops.linear_fp8(x, xs, w, ws, out_f32=True)
    odd = torch.zeros(40, 515, dtype=torch.uint8, device=DEV).view(F8)
    odd.view(torch.uint8)[:, 3:] = x.view(torch.uint8)
    assert torch.equal(ops.linear_fp8(odd[:, 3:], xs, w, ws, out_f32=True), y)
    wide = torch.zeros(300, 1024, dtype=torch.uint8, device=DEV).view(F8)
    wide.view(torch.uint8)[:, 256:768] = w.view(torch.uint8)
    assert torch.equal(ops.linear_fp8(x, xs, wide[:, 256:768], ws, out_f32=True), y)
    assert torch.equal(ops.linear_fp8(x, xs.t().contiguous().t(), w, ws.t().contiguous().t(), out_f32=True), y)
    one = ops.linear_fp8(odd[5:6, 3:], xs[5:6], w, ws, out_f32=True)
    assert torch.equal(one, ops.linear_fp8(x[5:6].contiguous(), xs[5:6], w, ws, out_f32=True))


@pytest.mark.gpu
@pytest.mark.parametrize("k,n", [(300, 1001), (256, 640), (77, 3)])
def test_outputs_start_on_16_byte_boundaries(k, n):
    """Rows of every output start on them, dense where their length allows it; leading dimensions merge as
    those of a dense tensor, and each output is the next call's input as it is."""
    ops = _ops()
    x, d = _rand(16, 2, 3, k, dtype=BF16), _rand(17, 2, 3, k, dtype=BF16)
    q, s, h = ops.rmsnorm_fp8(x, _rand(18, k, dtype=BF16), 1e-5, delta=d)
    w, ws = ops.quantize_fp8(_rand(19, n, k, dtype=BF16), block_rows=128)
    y = ops.linear_fp8(q, s, w, ws)
    y32 = ops.linear_fp8(q, s, w, ws, out_f32=True)
    for t in (q, h, w, y, y32):
        assert t.stride(-1) == 1 and (t.stride(-2) * t.element_size()) % 16 == 0 and t.data_ptr() % 16 == 0
        assert t.is_contiguous() == (t.shape[-1] * t.element_size() % 16 == 0)
    for t in (q, h, y, y32):
        assert t.view(6, t.shape[-1]).stride(0) == t.stride(1) and t.stride(0) == 3 * t.stride(1)
    assert torch.equal(h, (x.float() + d.float()).bfloat16())
    _check_product(y.view(6, n), q.view(6, k), s.view(6, -1), w, ws, False)
    _check_product(y32.view(6, n), q.view(6, k), s.view(6, -1), w, ws, True)
    again = ops.quantize_fp8(y)
    dense = ops.quantize_fp8(y.contiguous())
    assert torch.equal(again[0].float(), dense[0].float()) and torch.equal(again[1], dense[1])


@pytest.mark.gpu
def test_linear_output_pitch_and_frame():
    """Through the C ABI: an output with a pitch of its own (odd: scalar stores) keeps what lies around it."""
    lib = _lib()
    for m, n, k, pitch in ((5, 200, 256, 207), (130, 96, 128, 104), (40, 333, 2048, 340), (40, 333, 2048, 344),
                           (3, 77, 4096, 80), (300, 8002, 128, 8008), (300, 8001, 130, 8003)):
        x, xs, w, ws = _operands(m, m, n, k)
        for f32 in (0, 1):
            y = torch.full((m + 2, pitch), 9.0, dtype=F32 if f32 else BF16, device=DEV)
            status = torch.full((1,), 77, dtype=torch.int32, device=DEV)
            rc = lib.specb200_linear_fp8(x.data_ptr(), x.stride(0), xs.data_ptr(), w.data_ptr(), w.stride(0), ws.data_ptr(),
                                         m, n, k, f32, y[1].data_ptr(), pitch, status.data_ptr(),
                                         torch.cuda.current_stream().cuda_stream)
            assert rc == 0 and int(status) == 0
            assert (y[0] == 9).all() and (y[-1] == 9).all() and (y[:, n:] == 9).all()
            _check_product(y[1:-1, :n], x, xs, w, ws, bool(f32))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3, 300, 2048), (200, 384, 256)])
def test_linear_keeps_nan_to_its_row(m, n, k):
    """A NaN activation or scale reaches its own token, a NaN weight its own feature, and no others."""
    ops = _ops()
    x, xs, w, ws = _operands(31, m, n, k)
    clean = ops.linear_fp8(x, xs, w, ws, out_f32=True)
    x.view(torch.uint8)[1, 5] = 0x7F
    w.view(torch.uint8)[17, 9] = 0xFF
    xs[2, 1] = float("nan")
    y = ops.linear_fp8(x, xs, w, ws, out_f32=True)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[1] = bad[2] = True
    bad[:, 17] = True
    assert y[bad].isnan().all() and torch.equal(y[~bad], clean[~bad])


@pytest.mark.gpu
def test_linear_is_the_same_every_time_and_in_any_batch():
    """Bit for bit: repeated, and with the other tokens of the call taken away where the plan is the same."""
    ops = _ops()
    x, xs, w, ws = _operands(41, 7, 2048, 8192)
    y = ops.linear_fp8(x, xs, w, ws)
    for _ in range(5):
        assert torch.equal(ops.linear_fp8(x, xs, w, ws), y)
    assert torch.equal(ops.linear_fp8(x[2:5], xs[2:5], w, ws), y[2:5])


# one shape for each way a product is split over CTAs: up to 16 tokens (odd number of groups, K split in
# four, two tiles per SM), one tile per SM, K split in two and four, two tiles per SM, pairs with a
# partial last wave, pairs with an odd number of groups
PLANS = [(9, 900, 1152), (16, 2048, 8192), (5, 25600, 640), (17, 2048, 2048), (40, 900, 512), (300, 2048, 4096), (3, 2048, 2048), (128, 25600, 256), (700, 12000, 256), (2000, 5000, 384)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", PLANS)
def test_linear_repeats_bit_for_bit(m, n, k):
    """Back to back without a wait in between, so that each call starts while the last one ends."""
    ops = _ops()
    x, xs, w, ws = _operands(m + n, m, n, k)
    first = ops.linear_fp8(x, xs, w, ws, out_f32=True)
    _check_product(first, x, xs, w, ws, True)
    again = [ops.linear_fp8(x, xs, w, ws, out_f32=True, check=False) for _ in range(30)]
    assert all(torch.equal(y, first) for y in again)


# products of two CTAs per SM whose groups go round the ring of stages, the scales' slots and the TMEM buffers
# several times: up to 16 tokens and more, odd numbers of groups, a short last group, a short last tile
@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(16, 25600, 2048), (5, 20000, 1160), (1, 19001, 4999), (24, 25600, 2048),
                                   (100, 19100, 1160), (128, 25600, 1024), (33, 19201, 2900)])
def test_linear_on_shared_sms_goes_round_its_rings(m, n, k):
    ops = _ops()
    x, xs, w, ws = _operands(m + n + k, m, n, k)
    first = ops.linear_fp8(x, xs, w, ws, out_f32=True)
    _check_product(first, x, xs, w, ws, True)
    again = [ops.linear_fp8(x, xs, w, ws, out_f32=True, check=False) for _ in range(10)]
    assert all(torch.equal(y, first) for y in again)
    assert torch.equal(ops.linear_fp8(x, xs, w, ws), first.bfloat16())


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """More than 2^31 elements in the inputs and the outputs; the last rows are compared."""
    ops = _ops()
    m, k, tail = 70_000, 32_768, 40
    x = torch.zeros(m, k, dtype=BF16, device=DEV)
    x[-tail:] = _rand(80, tail, k, dtype=BF16)
    q, s = ops.quantize_fp8(x)
    _check_quantized(q[-tail:], s[-tail:], x[-tail:].double(), d=4 * U, s_tol=2 * U)
    del q, s
    weight = torch.ones(k, dtype=BF16, device=DEV)
    q, s, h = ops.rmsnorm_fp8(x, weight, 1e-5, delta=x)
    assert torch.equal(h[-tail:], x[-tail:] + x[-tail:])
    _check_quantized(q[-tail:], s[-tail:], _norm64(h[-tail:], weight, 1e-5), d=4 * U, s_tol=NORM_S)
    del q, s, h
    q, s = ops.silu_mul_fp8(x)
    g, u = x[-tail:, : k // 2].double(), x[-tail:, k // 2:].double()
    _check_quantized(q[-tail:], s[-tail:], g * torch.sigmoid(g) * u, **_silu_tol(g))
    del q, s, x
    xq, xs, w, ws = _operands(81, m, k, 48)
    y = ops.linear_fp8(xq, xs, w, ws)
    _check_product(y[-tail:], xq[-tail:], xs[-tail:], w, ws, False)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3, 2048, 2048), (16, 19200, 256), (60, 1024, 2048), (300, 9000, 256)])
def test_weights_written_by_the_kernel_in_front(m, n, k):
    """One weight buffer, quantized anew right in front of each product, eagerly and in a graph: a kernel that
    starts early must not see what lay there before."""
    from specb200 import _ffi

    ops, lib = _ops(), _lib()
    x, xs = ops.quantize_fp8(_rand(90, m, k, dtype=BF16))
    source = [_rand(91 + i, n, k, dtype=BF16) for i in range(3)]
    want = [ops.linear_fp8(x, xs, *ops.quantize_fp8(w, block_rows=128)) for w in source]
    w, ws = ops.quantize_fp8(source[0], block_rows=128)
    got = torch.zeros(12, m, n, dtype=BF16, device=DEV)

    def run():
        stream = torch.cuda.current_stream().cuda_stream
        for i in range(12):
            rc = lib.specb200_quantize_fp8(_ffi.BF16, source[i % 3].data_ptr(), k, n, k, 128, w.data_ptr(), k,
                                           ws.data_ptr(), stream)
            assert rc == 0
            rc = lib.specb200_linear_fp8(x.data_ptr(), x.stride(0), xs.data_ptr(), w.data_ptr(), k, ws.data_ptr(), m, n, k,
                                         0, got[i].data_ptr(), n, None, stream)
            assert rc == 0

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for call in (run, graph.replay, graph.replay):
        got.zero_()
        call()
        torch.cuda.synchronize()
        for i in range(12):
            assert torch.equal(got[i], want[i % 3])


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,f32,with_status", [
    (5, 200, 256, 1, True), (3, 300, 2048, 0, False), (16, 19000, 128, 0, True), (40, 200, 256, 0, True),
    (40, 333, 4096, 1, False), (20, 19100, 128, 0, True), (300, 9001, 256, 0, True), (2000, 5000, 128, 1, False)])
def test_linear_whose_waits_run_out(m, n, k, f32, with_status):
    """Every kind of product (few tokens, single, split and shared SMs, pairs over one and three tiles) without any
    operand: each wait gives up by itself, all outputs are NaN whether or not a status word is given, nothing
    around them is touched, and the next call is right."""
    from specb200 import _ffi

    ops, lib = _ops(), _lib()
    x, xs, w, ws = _operands(5, m, n, k)
    y = torch.full((m + 2, n + 3), 9.0, dtype=F32 if f32 else BF16, device=DEV)
    status = torch.full((1,), 77, dtype=torch.int32, device=DEV)
    rc = lib.specb200_linear_fp8_wait_probe(x.data_ptr(), x.stride(0), xs.data_ptr(), w.data_ptr(), w.stride(0), ws.data_ptr(),
                                            m, n, k, f32, y[1].data_ptr(), n + 3, status.data_ptr() if with_status else None,
                                            torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert y[1:-1, :n].isnan().all()
    assert (y[0] == 9).all() and (y[-1] == 9).all() and (y[:, n:] == 9).all()
    assert int(status) == (_ffi.ERR_TIMEOUT if with_status else 77)
    _check_product(ops.linear_fp8(x, xs, w, ws, out_f32=bool(f32)), x, xs, w, ws, bool(f32))


@pytest.mark.gpu
def test_a_long_chain_of_products():
    """Products of the longest K back to back, each 0.44 s on one cluster: later ones start beside the earlier ones, and
    the time for which they wait for those (more than a wait's limit of 2 s) is no reason to give up."""
    lib = _lib()
    k = 2 ** 30
    x = torch.zeros(1, k, dtype=torch.uint8, device=DEV)
    x[0, torch.randperm(k // 1024, generator=torch.Generator().manual_seed(1))[:1000].to(DEV) * 1024 + 77] = 0x38  # 1.0
    w = torch.full((1, k), 0x38, dtype=torch.uint8, device=DEV)
    scales = torch.ones(1, k // 128, device=DEV)
    y = torch.full((9, 4), -7.0, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    for row in y:
        rc = lib.specb200_linear_fp8(x.data_ptr(), k, scales.data_ptr(), w.data_ptr(), k, scales.data_ptr(), 1, 1, k, 1,
                                     row.data_ptr(), 4, None, stream)
        assert rc == 0
    assert (y[:, 0] == 1000).all() and (y[:, 1:] == -7).all()


@pytest.mark.gpu
def test_kernels_that_hold_tensor_memory_take_turns():
    """Short products of every kind (all of their groups fit the rings) and bf16 ones back to back in changing orders,
    eagerly and in a graph: whichever starts beside which, each gets its accumulators and its result."""
    from specb200 import _ffi

    ops, lib = _ops(), _lib()
    shapes = [(5, 2048, 512), (16, 25600, 128), (100, 900, 384), (64, 25600, 256), (300, 9000, 256), (3, 2048, 2048)]
    held = [_operands(70 + i, *s) for i, s in enumerate(shapes)]
    want = [ops.linear_fp8(*h) for h in held]
    x, w = _rand(71, 40, 512, dtype=BF16), _rand(72, 4096, 512, dtype=BF16)
    want.append(ops.linear(x, w))
    ws = torch.empty(max(16, lib.specb200_linear_workspace_bytes(40, 4096, 512)), dtype=torch.uint8, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    orders = [torch.randperm(7, generator=torch.Generator().manual_seed(i)).tolist() for i in range(8)]

    def run():
        out = []
        for i in (i for order in orders for i in order):
            if i < 6:
                out.append((i, ops.linear_fp8(*held[i], check=False)))
                continue
            y = torch.empty_like(want[6])
            rc = lib.specb200_linear(_ffi.BF16, w.data_ptr(), x.data_ptr(), 40, 4096, 512, 0, y.data_ptr(), ws.data_ptr(),
                                     ws.numel(), status.data_ptr(), torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            out.append((i, y))
        return out

    for i, y in run():
        assert torch.equal(y, want[i]), shapes[i] if i < 6 else "bf16"
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for i, y in out:
        assert torch.equal(y, want[i])
    assert int(status) == 0


@pytest.mark.gpu
def test_capture_with_a_status_word():
    """Through the C ABI, whose call clears the status word in front of the kernel."""
    lib = _lib()
    x, xs, w, ws = _operands(82, 9, 640, 512)
    y, status = torch.zeros(9, 640, dtype=BF16, device=DEV), torch.full((1,), 5, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            rc = lib.specb200_linear_fp8(x.data_ptr(), x.stride(0), xs.data_ptr(), w.data_ptr(), w.stride(0), ws.data_ptr(),
                                         9, 640, 512, 0, y.data_ptr(), 640, status.data_ptr(),
                                         torch.cuda.current_stream().cuda_stream)
            assert rc == 0
    for _ in range(2):
        y.zero_()
        status.fill_(5)
        graph.replay()
        assert int(status) == 0
        _check_product(y, x, xs, w, ws, False)


@pytest.mark.gpu
def test_streams_and_graphs_do_not_share_state():
    """Two streams that overlap, and two captured graphs replayed at once, give each call's own results."""
    ops = _ops()
    cases = [_operands(50 + i, m, n, k) for i, (m, n, k) in enumerate([(5, 2048, 8192), (700, 12000, 256)])]
    want = [ops.linear_fp8(*c) for c in cases]
    acts = [_rand(60 + i, 50, 2048, dtype=BF16) for i in range(2)]
    weight = torch.ones(2048, dtype=BF16, device=DEV)
    norm = [ops.rmsnorm_fp8(a, weight, 1e-5, delta=a) for a in acts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((ops.linear_fp8(*cases[i], check=False), ops.rmsnorm_fp8(acts[i], weight, 1e-5, delta=acts[i])))
    torch.cuda.synchronize()
    same = lambda a, b: all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, b))  # noqa: E731
    for i in range(2):
        for y, n in got[i]:
            assert torch.equal(y, want[i]) and same(n, norm[i])
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.linear_fp8(*cases[i], check=False)
            n = ops.rmsnorm_fp8(acts[i], weight, 1e-5, delta=acts[i])
        graphs.append((g, y, n))
    for _ in range(3):
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i, (_, y, n) in enumerate(graphs):
        assert torch.equal(y, want[i]) and same(n, norm[i])


# ---------------------------------------------------------------- together
@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 5, 160])
def test_a_layer_of_8_bit_linears(tokens):
    """A Llama layer's linears from 8-bit weights, with the engine's attention between them: every
    step against its formula on the inputs it was given."""
    ops = _ops()
    hidden, heads, kv_heads, d, inter = 576, 9, 3, 64, 1024
    qkv_n = (heads + 2 * kv_heads) * d
    w = {name: ops.quantize_fp8((0.05 * _rand(i, *shape, spread=0.0)).to(BF16), block_rows=128)
         for i, (name, shape) in enumerate([("qkv", (qkv_n, hidden)), ("o", (hidden, heads * d)),
                                            ("gate_up", (2 * inter, hidden)), ("down", (hidden, inter))])}
    ones = torch.ones(hidden, dtype=BF16, device=DEV)
    x = _rand(70, tokens, hidden, dtype=BF16, spread=0.3)

    def linear(q, s, name, out_f32=False):
        y = ops.linear_fp8(q, s, *w[name], out_f32=out_f32)
        _check_product(y, q, s, *w[name], out_f32)
        return y

    q, s = ops.rmsnorm_fp8(x, ones, 1e-5)
    _check_quantized(q, s, _norm64(x, ones, 1e-5), d=4 * U, s_tol=NORM_S)
    qkv = linear(q, s, "qkv")
    block = 16
    nblocks = -(-tokens // block)
    k_pool = torch.zeros(nblocks * block, kv_heads, d, dtype=BF16, device=DEV)
    v_pool = torch.zeros_like(k_pool)
    parts = qkv.view(tokens, heads + 2 * kv_heads, d)
    k_pool[:tokens], v_pool[:tokens] = parts[:, heads:heads + kv_heads], parts[:, heads + kv_heads:]
    table = torch.arange(nblocks, dtype=torch.int32, device=DEV)[None]
    zero, new = (torch.tensor([v], dtype=torch.int32, device=DEV) for v in (0, tokens))
    att = ops.attention(parts[None, :, :heads].contiguous(), k_pool, v_pool, table, block, zero, new, d ** -0.5, tokens)
    att = att.reshape(tokens, heads * d)
    qa, sa = ops.quantize_fp8(att)
    _check_quantized(qa, sa, att.double(), d=4 * U, s_tol=2 * U)
    o = linear(qa, sa, "o")
    q, s, h = ops.rmsnorm_fp8(x, ones, 1e-5, delta=o)
    assert torch.equal(h, (x.float() + o.float()).to(BF16))
    _check_quantized(q, s, _norm64(h, ones, 1e-5), d=4 * U, s_tol=NORM_S)
    gu = linear(q, s, "gate_up")
    q, s = ops.silu_mul_fp8(gu, packed=True)
    g, u = (v.reshape(tokens, inter).double() for v in gu.view(tokens, inter // 64, 2, 64).unbind(2))
    _check_quantized(q, s, g * torch.sigmoid(g) * u, **_silu_tol(g))
    down = linear(q, s, "down")
    assert (h + down).isfinite().all()
