"""Ends of the quantised block's ranges: the negative tail of the projections' GELU, steps at the small end of fp32, a gate's
tanh on both sides of its two forms, a few query rows of as many key heads as fill the GPU, a pair of CTAs whose
load never comes, outputs in their operands' places. u = 2^-24, half a step of fp32."""

import math

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


# One row and few rows, tiles of CTA pairs with one and several rounds.
@pytest.mark.parametrize("M,N", [(1, 3000), (2, 3001), (7, 3000), (300, 12000), (2000, 6001)])
@pytest.mark.parametrize("f32", [False, True])
def test_gelu_tanh_keeps_its_negative_tail(cuda, M, N, f32):
    """gelu(v) = v / (1 + e^-2u) with u = 0.798 (v + 0.0447 v^3), relative to the value however small it is.

    x is zero, so v is the bias. u is off by 5 u of itself (its terms have one sign: two constants, three roundings), which moves
    e^-2u by 10 |u| u; the exponential adds (2 + 1.18 * 2 |u|) ulp = (4 + 4.8 |u|) u, the sum 1 u, the division 2 ulp = 4 u:
    (9 + 15 |u|) u in all. bf16 adds 2^-8 of the value. A quotient by more than 2^126 may be 0: 16 / 2^126."""
    import torch
    import mkimage

    K = 640
    v = torch.linspace(-13, 4, N, device=cuda)
    x = torch.zeros(M, K, dtype=torch.int8, device=cuda)
    w = torch.ones(N, K, dtype=torch.int8, device=cuda)
    out = mkimage.ops.proj_i8(x, torch.ones(M, device=cuda), w, torch.ones(N, device=cuda), bias=v, act=mkimage.ops.ACT_GELU_TANH,
                              out_f32=f32)
    assert mkimage.ops.check_kernels() == 0
    v = v.double()
    u = math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
    ref = v * torch.sigmoid(2 * u)
    tol = (9 + 15 * u.abs()) * U * ref.abs() + 2.0 ** -122
    if not f32:
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * ref.abs()
    err = (out.double() - ref).abs()
    good = bool((err <= tol).all())
    assert good, float((err / ref.abs()).max())


def test_quantize_rows_at_the_smallest_steps(cuda):
    """Steps in [2^-126, 2^-125), where half a step may be no fp32 number: quotients on and next to every border."""
    import torch
    import mkimage

    g = torch.Generator().manual_seed(5)
    low = 127 * 2.0 ** -126
    tops = torch.cat([torch.tensor([low], dtype=torch.float64), low * (1 + torch.rand(200, generator=g, dtype=torch.float64)),
                      torch.tensor([2 * low, 2.3 * low], dtype=torch.float64)]).float()
    step = (tops / torch.tensor(127.0)).double()
    k = torch.arange(-127, 127, dtype=torch.float64) + 0.5
    at = (k[None] * step[:, None]).float()
    inf = torch.full_like(at, math.inf)
    x = torch.cat([tops[:, None], at, torch.nextafter(at, inf), torch.nextafter(at, -inf)], 1)
    x = torch.minimum(torch.maximum(x, -tops[:, None]), tops[:, None])
    want = (x.double() / step[:, None]).round()
    assert int((step * 2.0 ** 149).long().remainder(2).sum()) > 50  # odd significands are among them
    for pad in (0, 1):  # single values, vectors of four
        n = x.shape[1] + pad
        q, got = mkimage.ops.quantize_rows(torch.cat([x, x[:, 1:2]], 1)[:, :n].to(cuda))
        wrong = int((q.double().cpu() != torch.cat([want, want[:, 1:2]], 1)[:, :n]).sum())
        same = torch.equal(got.double().cpu(), step)
        assert wrong == 0 and same


@pytest.mark.parametrize("n", [12288, 5001])
def test_gate_tanh_on_both_sides_of_its_forms(cuda, n):
    """x = 0 and y = 1, so the residual that comes out is tanh(gate) alone.

    Below 0.4 a series x + x^3 p(x^2): what it leaves out is under 2^-27 of x there, x^3 p is under 0.06 of x with roundings of
    4 u of itself, the last sum is one more: 1.5 u. From 0.4 on 1 - t, t = 2 / (e^2a + 1): the exponential is off by
    (2 + 1.18 * 2 a) ulp = (4 + 4.8 a) u of itself, the sum by 1 u, the division by 2 ulp = 4 u, the difference by 1 u of the
    result, one more u for the product with y and the sum with x."""
    import torch
    import mkimage

    a = torch.cat([torch.linspace(0, 0.42, n // 2), torch.linspace(0.35, 0.45, n // 4), torch.linspace(0.4, 12, n - n // 2 - n // 4)])
    for sign in (1, -1):
        gate = (sign * a).to(cuda)
        out = torch.empty(1, n, device=cuda)
        mkimage.ops.gate_add_norm(torch.zeros(1, n, device=cuda), torch.ones(1, n, device=cuda), gate=gate, tanh_gate=True,
                                  x_out=out, out_type=mkimage.ops.OUT_NONE)
        g = gate.double()
        ref, t = torch.tanh(g), 2 / (torch.exp(2 * g.abs()) + 1)
        tol = torch.where(g.abs() < 0.4 + 1e-6, 1.5 * U * ref.abs(), torch.zeros_like(g))
        big = ((9 + 4.8 * g.abs()) * t + 2 * ref.abs()) * U
        tol = torch.where(g.abs() >= 0.4 - 1e-6, torch.maximum(tol, big), tol)
        err = (out[0].double() - ref).abs()
        good = bool((err <= tol).all())
        assert good, (float((err - tol).max()), float(g[(err - tol).argmax()]))


@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,d", [(4, 148, 37, 1, 512, 128), (4, 148, 37, 1, 512, 64), (4, 30, 30, 4, 400, 128),
                                             (4, 111, 37, 1, 300, 128), (4, 74, 37, 1, 512, 128), (5, 60, 60, 1, 700, 64)])
def test_few_rows_of_many_key_heads(cuda, B, H, Hkv, Lq, Lk, d):
    """Key heads for one, two and three CTAs an SM. Weights and sums are fp32 here, so 2^-11 of sum p|v| / sum p covers the
    scores' and the exponentials' errors, and the bf16 output is 2^-8 of the value; a sample without keys is zeros."""
    import torch
    import mkimage

    g = torch.Generator().manual_seed(H + Lk)
    q, k, v = (torch.randn(B, h, n, d, generator=g).to(torch.bfloat16).to(cuda) for h, n in ((H, Lq), (Hkv, Lk), (Hkv, Lk)))
    lens = torch.tensor([Lk, 0, Lk // 3, 1, Lk - 1][:B], dtype=torch.int32, device=cuda)
    got = mkimage.ops.cross_attention(q, k, v, key_len=lens).reshape(B, Lq, H, d).double()
    assert mkimage.ops.check_kernels() == 0
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            assert int((got[b] != 0).sum()) == 0
            continue
        kk, vv = (t[b, :, :n].double().repeat_interleave(H // Hkv, 0) for t in (k, v))
        p = torch.softmax(q[b].double() @ kk.transpose(1, 2) / math.sqrt(d), -1)
        ref, mag = (p @ vv).transpose(0, 1), (p @ vv.abs()).transpose(0, 1)
        good = bool(((got[b] - ref).abs() <= 2.0 ** -11 * mag + 2.0 ** -8 * ref.abs()).all())
        assert good, b


@pytest.mark.parametrize("rows,n", [(5, 640), (700, 1283), (900, 2048)])
def test_an_output_in_the_place_of_its_operand(cuda, rows, n):
    """y's rows become the norm (bf16), x's rows too where there is no branch or where x_out is elsewhere (fp32): the same bits
    as with memory of its own."""
    import torch
    import mkimage

    ops = mkimage.ops
    g = torch.Generator().manual_seed(n)
    x, y = torch.randn(rows, n, generator=g).to(cuda), torch.randn(rows, n, generator=g).to(torch.bfloat16).to(cuda)
    args = dict(y_norm=1, x_norm=2, rows_per_sample=rows // 2)
    xo = torch.empty_like(x)
    want = ops.gate_add_norm(x, y, x_out=xo, **args)
    x1, y1 = x.clone(), y.clone()
    assert torch.equal(ops.gate_add_norm(x1, y1, out=y1, **args), want) and torch.equal(x1, xo)
    want = ops.gate_add_norm(x, y, x_out=xo, out_type=ops.OUT_F32, **args)
    x1, x2 = x.clone(), torch.empty_like(x)
    assert torch.equal(ops.gate_add_norm(x1, y, x_out=x2, out=x1, out_type=ops.OUT_F32, **args), want) and torch.equal(x2, xo)
    yf = y.float()
    want = ops.gate_add_norm(x, yf, x_out=xo, **args)
    y1 = yf.clone()
    assert torch.equal(ops.gate_add_norm(x, y1, x_out=y1, **args), want) and torch.equal(y1, xo)
    want = ops.gate_add_norm(x, x_norm=1, out_type=ops.OUT_F32)
    x1 = x.clone()
    assert torch.equal(ops.gate_add_norm(x1, x_norm=1, out=x1, out_type=ops.OUT_F32), want)


def test_a_stalled_pair_gives_up_and_the_context_survives(cuda):
    """A pair whose first CTA never loads its half of the first stage: the roles' 2 s waits run out, so does the wait for the
    loads in flight, and the kernel returns; the other pairs' rows are right, and so is the next call."""
    import ctypes
    import time

    import torch
    import mkimage

    M, N, K = 1024, 512, 2048
    g = torch.Generator().manual_seed(8)
    x, w = (torch.randint(-128, 128, (r, K), generator=g, dtype=torch.int8).to(cuda) for r in (M, N))
    xs, ws = torch.ones(M, device=cuda), torch.ones(N, device=cuda)
    y = torch.zeros(M, N, device=cuda)
    ref = (x.double() @ w.double().T).float()
    assert mkimage.ops.check_kernels() == 0
    t0 = time.time()
    p = [t.data_ptr() for t in (x, xs, w, ws, y)]
    mkimage.check(mkimage.lib.mkb_selftest_stalled_proj_i8(p[0], K, p[1], p[2], K, p[3], p[4], N, M, N, K, None))
    bits = ctypes.c_uint32()
    code = mkimage.lib.mkb_check_kernels(ctypes.byref(bits))  # synchronises: the kernel has returned by now
    elapsed = time.time() - t0
    assert code == 4 and bits.value & 15 and bits.value & 16, (code, hex(bits.value))
    assert 3 < elapsed < 30, elapsed
    right = (y == ref).all(1)
    assert int(right.sum()) >= M // 2  # the first pair's tile, 256 rows, is not among them
    assert mkimage.ops.check_kernels() == 0
    assert torch.equal(mkimage.ops.proj_i8(x, xs, w, ws, out_f32=True), ref) and mkimage.ops.check_kernels() == 0
