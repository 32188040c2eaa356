"""mkb_gate_add_norm and mkb_quantize_rows against their formulas in 64 bits.

Tolerances, from the roundings alone (u = 2^-24, half a step of fp32). A sum of n fp32 values here goes through at most
24 sequential additions, 5 of a warp and 16 of the block, so it is off by at most 48 u of the sum of magnitudes. With
z = (t - mean) / std that makes the standardised value wrong by at most 48 u (|z| + mean|t| / std) (the square root
halves the variance's part, rsqrt and the products add a few u); TERM below is 64 u for it. A gate's tanh adds 2 u, every product and sum half
a step. bf16 outputs add 2^-8 of the value. Whole numbers may differ by one where the quotient is within the fp32 error
of a border, and are equal for a given row: quantize_rows decides the quotient exactly."""

import pytest

pytestmark = pytest.mark.gpu

TERM = 64 * 2.0 ** -24
U = 2.0 ** -24


def _norm64(t, kind, eps):
    """(value, error bound per element) of a norm of fp64 rows whose elements are exact."""
    import torch

    if kind == 0:
        return t, torch.zeros_like(t)
    mean = t.mean(1, keepdim=True) if kind == 2 else torch.zeros_like(t[:, :1])
    c = t - mean
    std = (c.square().mean(1, keepdim=True) + eps).sqrt()
    z = c / std
    off = t.abs().mean(1, keepdim=True) / std if kind == 2 else torch.zeros_like(std)
    return z, TERM * (z.abs() + off)


def _through_norm(err, t, kind, eps):
    """How far a norm's value moves when its input row is off by `err` (elementwise bound), to first order."""
    import torch

    if kind == 0:
        return err
    mean = t.mean(1, keepdim=True) if kind == 2 else torch.zeros_like(t[:, :1])
    std = ((t - mean).square().mean(1, keepdim=True) + eps).sqrt()
    z = (t - mean) / std
    return err / std + err.mean(1, keepdim=True) / std + z.abs() * (z.abs() * err).mean(1, keepdim=True) / std


def _case(cuda, rows, n, seed, y_f32, vec_samples, shift_x=0.1):
    import torch

    g = torch.Generator().manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g).to(cuda)

    y = r(rows, n) * 3 + 0.2
    return dict(x=2 * r(rows, n) + shift_x, y=y if y_f32 else y.to(torch.bfloat16), yw=1 + 0.1 * r(n), xw=1 + 0.1 * r(n),
                gate=0.5 * r(vec_samples, n), scale=0.3 * r(vec_samples, n), shift=0.3 * r(vec_samples, n))


def _check(ops, c, per, y_norm, x_norm, tanh, mod, out_type, eps=1e-6, in_place=False):
    import torch

    D = torch.float64
    rows, n = c["x"].shape
    at = torch.arange(rows, device=c["x"].device) // per
    x0 = c["x"].clone()
    x_in = c["x"].clone() if in_place else c["x"]
    x_out = None if in_place else torch.full_like(c["x"], 7.0)
    got = ops.gate_add_norm(x_in, c["y"], y_norm=y_norm, y_weight=c["yw"] if y_norm else None, gate=c["gate"],
                            tanh_gate=tanh, x_norm=x_norm, x_weight=c["xw"], scale=c["scale"] if mod else None,
                            shift=c["shift"] if mod else None, rows_per_sample=per, eps=eps, x_out=x_out,
                            out_type=out_type) if out_type != ops.OUT_NONE else ops.gate_add_norm(
        x_in, c["y"], y_norm=y_norm, y_weight=c["yw"] if y_norm else None, gate=c["gate"], tanh_gate=tanh,
        rows_per_sample=per, eps=eps, x_out=x_out, out_type=out_type)
    x_got = (x_in if in_place else x_out).to(D)
    if not in_place:
        assert torch.equal(c["x"], x0)
    z, e = _norm64(c["y"].to(D), y_norm, eps)
    w = c["yw"].to(D) if y_norm else torch.ones(n, dtype=D, device=x0.device)
    g = c["gate"].to(D)[at]
    g = g.tanh() if tanh else g
    x = x0.to(D) + g * z * w
    ex = (g * w).abs() * (e + 6 * U * z.abs()) + 2 * U * x.abs()
    assert ((x_got - x).abs() <= ex).all()
    if out_type == ops.OUT_NONE:
        assert got is None
        return
    h, eh = _norm64(x, x_norm, eps)
    eh = eh + _through_norm(ex, x, x_norm, eps)
    f = c["xw"].to(D).expand(rows, n)
    f = f * (1 + c["scale"].to(D)[at]) if mod else f
    b = c["shift"].to(D)[at] if mod else torch.zeros_like(h)
    ref = h * f + b
    # The product with (1 + scale) is taken as h + h * scale: half a step of each part.
    eh = f.abs() * eh + 6 * U * (h * c["xw"].to(D)).abs() * (1 + c["scale"].to(D)[at].abs() if mod else 1) + 2 * U * ref.abs()
    if out_type == ops.OUT_I8:
        q, step = got
        top, etop = ref.abs().amax(1), eh.amax(1)
        assert ((step.to(D) - top / 127).abs() <= etop / 127 + 2 * U * step.to(D)).all()
        # Half a step, plus the value's own error.
        assert ((q.to(D) * step.to(D)[:, None] - ref).abs() <= 0.5 * step.to(D)[:, None] * (1 + 1e-6) + eh + etop[:, None]).all()
        assert int(q.abs().max()) <= 127 and bool((q.abs().amax(1) == 127).all())
    else:
        err = eh + (2.0 ** -8 * ref.abs() if out_type == ops.OUT_BF16 else 0)
        assert ((got.to(D) - ref).abs() <= err).all()


@pytest.mark.parametrize("rows,n", [(1, 1), (3, 5), (2, 31), (7, 64), (33, 640), (5, 1283), (130, 1280), (9, 3072), (3, 5120),
                                    (2, 12288), (4, 12287)])
@pytest.mark.parametrize("y_norm,x_norm", [(1, 1), (2, 2), (0, 1), (1, 0)])
@pytest.mark.parametrize("out", ["bf16", "f32", "i8"])
def test_gate_add_norm(cuda, rows, n, y_norm, x_norm, out):
    import mkimage

    ops = mkimage.ops
    per = max(1, rows // 2)  # an uneven last sample where rows is odd
    c = _case(cuda, rows, n, rows * n, y_f32=n % 2 == 1, vec_samples=-(-rows // per))
    kind = dict(bf16=ops.OUT_BF16, f32=ops.OUT_F32, i8=ops.OUT_I8)[out]
    _check(ops, c, per, y_norm, x_norm, tanh=(y_norm == 1), mod=(out != "f32"), out_type=kind)


@pytest.mark.parametrize("rows,n,samples", [(1000, 640, 3), (2100, 3072, 2), (900, 1283, 7), (5000, 96, 1), (700, 6144, 2),
                                             (400, 6400, 2), (301, 4099, 301), (800, 12288, 5)])
@pytest.mark.parametrize("out", ["bf16", "i8", "none"])
def test_runs_of_rows(cuda, rows, n, samples, out):
    """Rows enough that a block walks several of one sample, with short last runs and samples; in place as well. Outputs
    with no norm at all take one barrier a row or none."""
    import mkimage

    ops = mkimage.ops
    per = -(-rows // samples)
    c = _case(cuda, rows, n, rows + n, False, -(-rows // per))
    kind = dict(bf16=ops.OUT_BF16, i8=ops.OUT_I8, none=ops.OUT_NONE)[out]
    for y_norm, x_norm in ((1, 1), (0, 2), (0, 0)):
        _check(ops, c, per, y_norm, x_norm, tanh=y_norm == 1, mod=True, out_type=kind, in_place=y_norm == 1)


@pytest.mark.parametrize("n", [4000, 4040, 4043, 4044, 4056, 4093, 4096, 4097, 4100])
@pytest.mark.parametrize("off", [0, 1])
def test_widths_around_48_kb_of_vectors(cuda, n, off):
    """Three vectors of 4096 values fill the shared memory that a launch has without asking, with aligned rows, odd ones and
    ones that begin differently."""
    import torch
    import mkimage

    ops = mkimage.ops
    for rows in (3, 500):
        c = _case(cuda, rows, n, n, False, 1)
        y = torch.empty(rows * n + 8, dtype=torch.bfloat16, device=cuda)[off:off + rows * n].view(rows, n)
        c["y"] = y.copy_(c["y"])
        _check(ops, c, rows, 1, 1, True, True, ops.OUT_BF16)


@pytest.mark.parametrize("rows,n,per", [(7, 131, 1), (1001, 131, 2), (1001, 1283, 3), (1003, 131, 5), (2501, 333, 6), (999, 4099, 4)])
def test_odd_rows_of_short_samples(cuda, rows, n, per):
    """Samples of fewer rows than the four that runs of odd rows start at, and a few more."""
    import mkimage

    ops = mkimage.ops
    c = _case(cuda, rows, n, rows + n, False, -(-rows // per))
    _check(ops, c, per, 1, 2, True, True, ops.OUT_BF16)
    _check(ops, c, per, 0, 1, False, True, ops.OUT_I8, in_place=True)


@pytest.mark.parametrize("off_x,off_y,off_o", [(1, 1, 1), (1, 1, 2), (3, 3, 0), (2, 1, 1), (0, 2, 0)])
@pytest.mark.parametrize("rows,n,ld", [(5, 129, 131), (700, 1283, 1283 + 8), (900, 640, 641), (420, 5111, 5119), (40, 12288, 12289)])
@pytest.mark.parametrize("out", ["bf16", "f32", "i8"])
def test_rows_at_any_place(cuda, off_x, off_y, off_o, rows, n, ld, out):
    """x, y and out at their own places in wider rows, alike and not, against the same call on rows of their own; nothing
    outside the rows is written. The sums' order may differ: 2 TERM of the standardised values, whose size is below 12 here,
    through factors below 3, and a rounding of the output; a whole number may differ by one."""
    import torch
    import mkimage

    ops = mkimage.ops
    kind, dtype = dict(bf16=(ops.OUT_BF16, torch.bfloat16), f32=(ops.OUT_F32, torch.float32), i8=(ops.OUT_I8, torch.int8))[out]
    per = -(-rows // 2)
    c = _case(cuda, rows, n, n + off_x, False, 2)

    def at(t, off):
        buf = torch.full((rows * ld + 16,), 3, device=cuda, dtype=t)
        return buf, buf[off:off + rows * ld].view(rows, ld)[:, :n]

    (xb, x), (yb, y), (ob, o) = at(torch.float32, off_x), at(torch.bfloat16, off_y), at(dtype, off_o)
    x.copy_(c["x"])
    y.copy_(c["y"])
    rx, step = c["x"].clone(), torch.empty(rows, device=cuda) if out == "i8" else None
    args = dict(y_norm=1, y_weight=c["yw"], gate=c["gate"], x_norm=2, x_weight=c["xw"], scale=c["scale"], shift=c["shift"],
                rows_per_sample=per, out_type=kind)
    ref = ops.gate_add_norm(rx, c["y"], **args)
    ops.gate_add_norm(x, y, out=o, out_scale=step, **args)
    assert ((x - rx).abs() <= 2 * TERM * 12 * 3 + 4 * U * rx.abs()).all()
    if out == "i8":
        assert ((step - ref[1]).abs() <= 1e-4 * ref[1]).all() and int((o.int() - ref[0].int()).abs().max()) <= 1
    else:
        err = 1e-3 + (2.0 ** -7 * ref.float().abs() if out == "bf16" else 0)
        assert ((o.float() - ref.float()).abs() <= err).all()
    for buf, rows_of in ((xb, x), (ob, o)):
        rows_of.fill_(3)
        assert bool((buf == 3).all())


def test_in_place_no_output_and_no_branch(cuda):
    import torch
    import mkimage

    ops = mkimage.ops
    c = _case(cuda, 70, 256, 5, False, 2)
    _check(ops, c, 35, 1, 1, True, True, ops.OUT_BF16, in_place=True)
    x = c["x"].clone()
    assert ops.gate_add_norm(x, c["y"], gate=c["gate"], rows_per_sample=35, out_type=ops.OUT_NONE) is None
    at = torch.arange(70, device=cuda) // 35
    ref = c["x"].double() + c["gate"].double()[at] * c["y"].double()
    assert ((x.double() - ref).abs() <= 2 * U * (ref.abs() + c["x"].abs())).all()
    # Without a branch the residual stays and only its norm comes out.
    h = ops.gate_add_norm(x, x_norm=ops.NORM_RMS, x_weight=c["xw"], out_type=ops.OUT_F32)
    ref = x.double() / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt() * c["xw"].double()
    assert ((h.double() - ref).abs() <= (TERM + 4 * U) * ref.abs()).all()


def test_large_mean_keeps_the_layer_norm(cuda):
    """Rows with a mean of 1000 deviations: squares about zero would lose the variance in fp32."""
    import mkimage

    ops = mkimage.ops
    c = _case(cuda, 6, 1024, 8, True, 1, shift_x=2000.0)
    c["y"] += 3000.0
    _check(ops, c, 6, 2, 2, False, True, ops.OUT_F32)


def test_strides_and_guard_rows(cuda):
    """Strided rows of wider buffers, at 16-byte and at odd offsets; nothing outside the rows is written."""
    import torch
    import mkimage

    ops = mkimage.ops
    for off, n in ((0, 512), (3, 512), (4, 510)):
        c = _case(cuda, 20, n, 11, False, 1)
        wide = lambda t: torch.full((22, n + 24), 3.0, device=cuda, dtype=t)  # noqa: E731
        xb, yb, ob = wide(torch.float32), wide(torch.bfloat16), wide(torch.bfloat16)
        x, y, o = (t[1:21, off:off + n] for t in (xb, yb, ob))
        x.copy_(c["x"])
        y.copy_(c["y"])
        ref_x = c["x"].clone()
        ref = ops.gate_add_norm(ref_x, c["y"].clone(), y_norm=1, x_norm=2, gate=c["gate"], scale=c["scale"])
        ops.gate_add_norm(x, y, y_norm=1, x_norm=2, gate=c["gate"], scale=c["scale"], out=o)
        assert ((x - ref_x).abs() <= 1e-5 * (1 + ref_x.abs())).all()  # another order of the sums
        assert ((o.float() - ref.float()).abs() <= 2.0 ** -7 * ref.float().abs() + 1e-4).all()
        for t in (xb, ob):
            inside = torch.zeros_like(t, dtype=torch.bool)
            inside[1:21, off:off + n] = True
            assert bool((t[~inside] == 3.0).all())


def test_nan_and_inf_rows_stay_in_their_rows(cuda):
    import torch
    import mkimage

    ops = mkimage.ops
    c = _case(cuda, 8, 320, 13, False, 1)
    y = c["y"].clone()
    y[2, 7], y[5, 100] = float("nan"), float("inf")
    q, step = ops.gate_add_norm(c["x"].clone(), y, y_norm=1, x_norm=1, out_type=ops.OUT_I8)
    good = [0, 1, 3, 4, 6, 7]
    assert bool(torch.isfinite(step[good]).all()) and bool(torch.isnan(step[[2, 5]]).all())
    assert int(q[[2, 5]].abs().max()) == 0


def _quant64(x):
    import torch

    x = x.double()
    top = x.abs().amax(1)
    step = (top.float() / torch.full_like(top.float(), 127.0))
    step = torch.where(step < torch.finfo(torch.float32).tiny, torch.zeros_like(step), step)
    q = (x / step.double()[:, None]).round()
    return torch.where(step[:, None] > 0, q, torch.zeros_like(q)).to(torch.int8), step


@pytest.mark.parametrize("rows,n", [(1, 1), (3, 7), (2, 64), (77, 1280), (5, 1283), (2, 5000), (3, 16384), (2, 16388), (2, 20001)])
@pytest.mark.parametrize("f32", [False, True])
def test_quantize_rows_is_exact(cuda, rows, n, f32):
    import torch
    import mkimage

    g = torch.Generator().manual_seed(rows + n)
    x = (torch.randn(rows, n, generator=g) * torch.rand(rows, 1, generator=g)).to(cuda)
    x = x if f32 else x.to(torch.bfloat16)
    q, step = mkimage.ops.quantize_rows(x)
    rq, rstep = _quant64(x)
    assert torch.equal(step, rstep) and torch.equal(q, rq)
    assert q.stride(0) % 16 == 0


@pytest.mark.parametrize("rows,n", [(9000, 640), (5000, 333), (3001, 8192), (2500, 5120), (1500, 5001)])
@pytest.mark.parametrize("f32", [False, True])
def test_quantize_many_rows(cuda, rows, n, f32):
    """More rows than blocks that run at once, strided, a NaN among them; what lies between the rows stays."""
    import torch
    import mkimage

    g = torch.Generator().manual_seed(rows + n)
    x = torch.randn(rows, n + 8, generator=g)
    x = (x * torch.rand(rows, 1, generator=g)).to(cuda).to(torch.float32 if f32 else torch.bfloat16)[:, :n]
    x[rows // 2, 3] = float("nan")
    buf = torch.full((rows, (n + 31) // 16 * 16), 99, dtype=torch.int8, device=cuda)
    step = torch.empty(rows, device=cuda)
    mkimage.ops.quantize_rows(x, buf[:, :n], step)
    fine = torch.arange(rows, device=cuda) != rows // 2
    rq, rstep = _quant64(x[fine])
    assert torch.equal(step[fine], rstep) and torch.equal(buf[:, :n][fine], rq) and bool((buf[:, n:] == 99).all())
    assert bool(torch.isnan(step[rows // 2])) and int(buf[rows // 2, :n].abs().max()) == 0


def test_quantize_rows_borders(cuda):
    """Quotients on and next to a border of two whole numbers, rows of zeros, tiny rows, infinities and NaN."""
    import torch
    import mkimage

    k = torch.arange(-127, 127, dtype=torch.float64) + 0.5
    rows = []
    for top in (127.0, 254.0, 1.0, 3.7, 1e-30, 2.0 ** 100):
        step = (torch.tensor(top, dtype=torch.float32) / torch.tensor(127.0)).double()
        at = (k * step).float()
        rows.append(torch.cat([torch.tensor([top]), at, torch.nextafter(at, at + 1e30), torch.nextafter(at, at - 1e30)]))
    x = torch.stack(rows).to(cuda)
    x = x.clamp(min=-x[:, :1], max=x[:, :1])
    q, step = mkimage.ops.quantize_rows(x)
    rq, rstep = _quant64(x)
    assert torch.equal(step, rstep) and torch.equal(q, rq)
    z = torch.zeros(5, 40, device=cuda)
    z[1, 3], z[2, 3], z[3, 4], z[4, 5] = 1e-39, float("inf"), float("nan"), -float("inf")
    q, step = mkimage.ops.quantize_rows(z)
    assert int(q.abs().max()) == 0 and step[0] == 0 and step[1] == 0 and bool(torch.isnan(step[2:]).all())


def test_offsets_past_32_bits(cuda):
    """Two rows 2^31 + 64 elements apart: 64-bit row offsets in every operand."""
    import torch
    import mkimage

    ops = mkimage.ops
    far, n = 2 ** 31 + 64, 256
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    c = _case(cuda, 2, n, 21, False, 1)
    xb = torch.empty(far + n, device=cuda)
    yb = torch.empty(far + n, device=cuda, dtype=torch.bfloat16)
    qb = torch.empty(far + n, device=cuda, dtype=torch.int8)
    x, y, q = (t.as_strided((2, n), (far, 1)) for t in (xb, yb, qb))
    x.copy_(c["x"])
    y.copy_(c["y"])
    ref_x = c["x"].clone()
    rq, rs = ops.gate_add_norm(ref_x, c["y"], y_norm=1, x_norm=1, gate=c["gate"], out_type=ops.OUT_I8)
    s = torch.empty(2, device=cuda)
    ops.gate_add_norm(x, y, y_norm=1, x_norm=1, gate=c["gate"], out=q, out_scale=s, out_type=ops.OUT_I8)
    assert torch.equal(x, ref_x) and torch.equal(q, rq) and torch.equal(s, rs)
    q.zero_()
    ops.quantize_rows(y, q, s)
    rq, rs = ops.quantize_rows(c["y"])
    assert torch.equal(q, rq) and torch.equal(s, rs)
