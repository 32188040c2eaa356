"""mkb_proj_i8 against the product in 64 bits, where the integer sums are exact.

Tolerances: the sum is an exact integer; turning it into fp32, the two scales and the bias are one rounding each (half a
step, u = 2^-24): at most 4 u |product| + u |y|. An activation's derivative is at most 1.13; the fp32 forms add a few u of
their own, taken as 2^-20 of max(|argument|, 1). For bf16 outputs the GELU's tanh may come from the SFU (absolute error
2^-10.9, times |v| / 2), and the rounding itself is 2^-8 of the value."""

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _case(cuda, M, N, K, seed):
    import torch

    g = torch.Generator().manual_seed(seed)

    def i8(r):  # rows 16 bytes apart with something else between them
        b = torch.full((r, -(-K // 16) * 16 + 16), 77, dtype=torch.int8)
        b[:, :K] = torch.randint(-128, 128, (r, K), generator=g, dtype=torch.int8)
        return b.to(cuda)[:, :K]

    xs = (torch.rand(M, generator=g) * 0.02 + 1e-3).to(cuda)
    ws = (torch.rand(N, generator=g) * 0.002 + 1e-4).to(cuda)
    return i8(M), xs, i8(N), ws, torch.randn(N, generator=g).to(cuda)


def _act64(v, act):
    import torch

    if act == 1:
        return 0.5 * v * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3)))
    if act == 2:
        return v * torch.sigmoid(v)
    if act == 3:
        return v * torch.sigmoid(1.702 * v)
    if act == 4:
        return 0.5 * v * (1 + torch.erf(v / 2 ** 0.5))
    return v


def _check(out, x, xs, w, ws, bias, act):
    import torch

    D = torch.float64
    p = (x.to(D) @ w.to(D).T) * xs.to(D)[:, None] * ws.to(D)
    v = p + (bias.to(D) if bias is not None else 0)
    ref = _act64(v, act)
    err = 1.13 * (4 * U * p.abs() + U * v.abs())
    bf16 = out.dtype == torch.bfloat16
    if act:
        err = err + 2.0 ** -20 * v.abs().clamp(min=1)
    if bf16:
        err = err + 2.0 ** -8 * ref.abs() + (0.5 * v.abs() * 2.0 ** -10.9 if act == 1 else 0)
    bad = (out.to(D) - ref).abs() > err
    assert not bool(bad.any()), ((out.to(D) - ref).abs().max(), bad.nonzero()[:4])


SHAPES = [(1, 1, 1), (1, 32, 64), (1, 1000, 3000), (2, 33, 100), (5, 257, 1291), (8, 640, 640), (9, 96, 2048), (16, 129, 127),
          (17, 256, 4096), (33, 320, 77), (64, 512, 512), (77, 1280, 1280), (127, 127, 127), (128, 128, 128), (129, 255, 129),
          (200, 1280, 5120), (300, 3072, 768), (513, 2304, 768), (1000, 520, 1040), (1, 48, 131071), (20, 40, 20000)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("f32", [False, True])
def test_proj_i8(cuda, M, N, K, f32):
    import mkimage

    c = _case(cuda, M, N, K, M + N + K)
    x, xs, w, ws, b = c
    out = mkimage.ops.proj_i8(x, xs, w, ws, bias=b, out_f32=f32)
    assert mkimage.ops.check_kernels() == 0
    _check(out, x, xs, w, ws, b, 0)


@pytest.mark.parametrize("M,N,K", [(1, 96, 256), (3, 130, 200), (70, 200, 320), (150, 384, 512), (600, 777, 256)])
@pytest.mark.parametrize("act", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("f32", [False, True])
def test_activations_without_and_with_bias(cuda, M, N, K, act, f32):
    import mkimage

    x, xs, w, ws, b = _case(cuda, M, N, K, act + M)
    for bias in (None, b):
        out = mkimage.ops.proj_i8(x, xs, w, ws, bias=bias, act=act, out_f32=f32)
        _check(out, x, xs, w, ws, bias, act)
    assert mkimage.ops.check_kernels() == 0


@pytest.mark.parametrize("M,N,K", [(8192, 1280, 640), (4097, 1283, 1100), (2304, 6144, 1024), (700, 9216, 768)])
def test_large(cuda, M, N, K):
    import mkimage

    x, xs, w, ws, b = _case(cuda, M, N, K, 3)
    out = mkimage.ops.proj_i8(x, xs, w, ws, bias=b, act=1)
    assert mkimage.ops.check_kernels() == 0
    _check(out, x, xs, w, ws, b, 1)


@pytest.mark.parametrize("M", [1, 4, 40, 300])
def test_largest_sums_are_exact(cuda, M):
    """Every factor -128 and the longest K: the sum is 128 * 128 * 131071, just inside 32 bits."""
    import torch
    import mkimage

    K = 131071
    x = torch.full((M, K + 1), -128, dtype=torch.int8, device=cuda)[:, :K]
    w = torch.full((40, K + 1), -128, dtype=torch.int8, device=cuda)[:, :K]
    out = mkimage.ops.proj_i8(x, torch.ones(M, device=cuda), w, torch.ones(40, device=cuda), out_f32=True)
    assert bool((out == float(128 * 128 * K)).all())


# Few tiles over a long K: tiles of 16 to 64 tokens, K in one to eight parts.
@pytest.mark.parametrize("M,N,K", [(132, 1056, 6784), (192, 288, 9600), (191, 290, 9408), (500, 512, 8192), (194, 1568, 11072),
                                   (40, 2048, 8192), (300, 100, 12300), (60, 128, 12288), (30, 20000, 512), (13, 1664, 8192)])
@pytest.mark.parametrize("f32", [False, True])
def test_parts_of_a_long_k(cuda, M, N, K, f32):
    import torch
    import mkimage

    x, xs, w, ws, b = _case(cuda, M, N, K, M + N)
    buf = torch.full((M + 2, N + 3), 5.0, dtype=torch.float32 if f32 else torch.bfloat16, device=cuda)
    out = buf[1:M + 1, 1:N + 1]
    mkimage.ops.proj_i8(x, xs, w, ws, bias=b, act=2, out=out)
    assert mkimage.ops.check_kernels() == 0
    _check(out, x, xs, w, ws, b, 2)
    out.fill_(5)
    assert bool((buf == 5).all())


# Tiles of 160, 160, 192, 192, 128 and 256 columns on 148 SMs, whole and cut.
@pytest.mark.parametrize("M,N", [(2000, 2560), (2000, 2467), (700, 8192), (705, 8101), (1030, 1500), (8000, 777)])
@pytest.mark.parametrize("f32", [False, True])
def test_widths_of_tiles(cuda, M, N, f32):
    """Outputs that TMA can address and ones that it cannot, inside a buffer whose other values stay."""
    import torch
    import mkimage

    x, xs, w, ws, b = _case(cuda, M, N, 300, M + N)
    for off, ld in ((0, (N + 63) // 32 * 32), (3, N + 8 - N % 2)):
        buf = torch.full((M + 2, ld), 5.0, dtype=torch.float32 if f32 else torch.bfloat16, device=cuda)
        out = buf[1:M + 1, off:off + N]
        mkimage.ops.proj_i8(x, xs, w, ws, bias=b, out=out)
        _check(out, x, xs, w, ws, b, 0)
        assert bool((buf[0] == 5).all() and (buf[M + 1] == 5).all() and (buf[:, :off] == 5).all() and
                    (buf[:, off + N:] == 5).all())
    assert mkimage.ops.check_kernels() == 0


@pytest.mark.parametrize("M", [2, 30, 200, 2000])
def test_guards_and_strided_output(cuda, M):
    """Only [M][N] of a wider, longer output is written, at an unaligned place as well."""
    import torch
    import mkimage

    x, xs, w, ws, b = _case(cuda, M, 300, 400, 9)
    for off in (0, 1, 8):
        for t in (torch.float32, torch.bfloat16):
            buf = torch.full((M + 2, 340), 5.0, dtype=t, device=cuda)
            out = buf[1:M + 1, off:off + 300]
            mkimage.ops.proj_i8(x, xs, w, ws, bias=b, out=out)
            _check(out, x, xs, w, ws, b, 0)
            assert bool((buf[0] == 5).all() and (buf[M + 1] == 5).all() and (buf[:, :off] == 5).all() and
                        (buf[:, off + 300:] == 5).all())
    assert mkimage.ops.check_kernels() == 0


def test_same_rows_whatever_the_batch(cuda):
    """Integer sums do not depend on how the work is split: a row's result is the same in any call."""
    import torch
    import mkimage

    x, xs, w, ws, b = _case(cuda, 700, 512, 2000, 4)
    ops = mkimage.ops
    full = ops.proj_i8(x, xs, w, ws, bias=b, out_f32=True)
    for m in (1, 7, 60, 260):
        assert torch.equal(ops.proj_i8(x[:m], xs[:m], w, ws, bias=b, out_f32=True), full[:m])


def test_nan_scale_marks_its_row(cuda):
    import torch
    import mkimage

    x, xs, w, ws, b = _case(cuda, 20, 64, 64, 4)
    xs[3] = float("nan")
    out = mkimage.ops.proj_i8(x, xs, w, ws, bias=b)
    assert bool(torch.isnan(out[3]).all()) and bool(torch.isfinite(out[torch.arange(20) != 3]).all())


@pytest.mark.parametrize("M", [2, 160])
def test_offsets_past_32_bits(cuda, M):
    import torch
    import mkimage

    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    x, xs, w, ws, b = _case(cuda, M, 64, 256, 4)
    far = -(-(2 ** 31 + 64) // (M - 1) // 16) * 16 + 16
    yb = torch.empty(far * (M - 1) + 64, dtype=torch.bfloat16, device=cuda)
    xb = torch.empty(far * (M - 1) + 256, dtype=torch.int8, device=cuda)
    xf, y = xb.as_strided((M, 256), (far, 1)), yb.as_strided((M, 64), (far, 1))
    xf.copy_(x)
    mkimage.ops.proj_i8(xf, xs, w, ws, bias=b, out=y)
    assert torch.equal(y, mkimage.ops.proj_i8(x, xs, w, ws, bias=b))
    assert mkimage.ops.check_kernels() == 0
