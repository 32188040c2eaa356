"""Refusals of the quantised block's entry points (quantize_rows, proj_i8, gate_add_norm, cross_attention): every bad
argument is an error code with a message before any device work. CPU only; the pointers are never read."""

import pytest

import mkimage

P = 1 << 20  # an aligned address that nothing dereferences


def _refused(fn, args, word):
    assert fn(*args) == 1
    assert word in mkimage.lib.mkb_last_error().decode()


def _with(base, **changes):
    d = dict(base)
    d.update(changes)
    return list(d.values())


QUANT = dict(x=P, ldx=64, x_f32=0, q=P, ldq=64, scale=P, rows=4, n=64, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(x=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"), (dict(n=0), "n <="), (dict(rows=-1), "rows"),
    (dict(ldx=63), "ldx"), (dict(ldq=63), "ldq"), (dict(x=P + 1), "misaligned"), (dict(x=P + 2, x_f32=1), "misaligned"),
    (dict(scale=P + 2), "misaligned"), (dict(n=1 << 25, ldx=1 << 25, ldq=1 << 25), "2^24")])
def test_quantize_rows_refuses(change, word):
    _refused(mkimage.lib.mkb_quantize_rows, _with(QUANT, **change), word)


PROJ = dict(x=P, ldx=64, xs=P, w=P, ldw=64, ws=P, bias=None, y=P, ldy=32, M=4, N=32, K=64, act=0, f32=0, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(x=None), "null"), (dict(xs=None), "null"), (dict(w=None), "null"), (dict(ws=None), "null"),
    (dict(y=None), "null"), (dict(act=5), "activation"), (dict(act=-1), "activation"), (dict(K=0), "K"),
    (dict(K=131072, ldx=131072, ldw=131072), "131071"), (dict(N=0), "N > 0"), (dict(M=-1), "M >= 0"),
    (dict(ldx=72), "16"), (dict(ldw=40), "16"), (dict(ldx=48), "ldx"), (dict(ldy=31), "ldy"), (dict(x=P + 8), "alignment"),
    (dict(w=P + 8), "alignment"), (dict(y=P + 1), "alignment"), (dict(y=P + 2, f32=1), "alignment"),
    (dict(bias=P + 1), "alignment"), (dict(M=(1 << 31) - 1, N=1 << 20, ldy=1 << 20), "2^30 output tiles"),
    (dict(M=1, N=(1 << 31) - 1, ldy=1 << 31), "N <= 2^30"), (dict(M=(1 << 31) - 1), "N <= 2^30")])
def test_proj_i8_refuses(change, word):
    _refused(mkimage.lib.mkb_proj_i8, _with(PROJ, **change), word)


NORM = dict(x=P, ldx=64, xo=P, ldxo=64, y=P, ldy=64, y_f32=0, y_norm=1, yw=None, gate=None, gs=0, tanh=0, x_norm=1,
            xw=None, scale=None, shift=None, ms=0, rps=4, eps=1e-6, out=P, ldo=64, out_type=1, osc=None, rows=4, n=64,
            stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(x=None, xo=P), "null"), (dict(xo=None), "null"), (dict(out=None), "null"), (dict(n=12289, ldx=12289), "12288"),
    (dict(n=0), "n <="), (dict(rps=0), "rows_per_sample"), (dict(y_norm=3), "unknown"), (dict(x_norm=-1), "unknown"),
    (dict(out_type=4), "unknown"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(y=None), "without y"),
    (dict(y=None, y_norm=0, gate=P), "without y"), (dict(y=None, y_norm=0, xo=2 * P), "without y"),
    (dict(y=None, y_norm=0, out_type=0, x_norm=0), "nothing"), (dict(out_type=0), "without an output"),
    (dict(ldx=63), "leading"), (dict(ldxo=60), "leading"), (dict(ldy=60), "leading"), (dict(ldo=60), "leading"),
    (dict(ldxo=128), "in place"), (dict(gs=-1), "negative"), (dict(out_type=3), "out_scale"), (dict(osc=P), "out_scale"),
    (dict(x=P + 2, xo=P + 2), "misaligned"), (dict(y=P + 1), "misaligned"), (dict(gate=P + 1), "misaligned"),
    (dict(out=P + 1), "misaligned")])
def test_gate_add_norm_refuses(change, word):
    _refused(mkimage.lib.mkb_gate_add_norm, _with(NORM, **change), word)


CROSS = dict(q=P, qr=64, qh=640, qs=6400, k=P, kr=64, kh=640, ks=6400, v=P, vr=64, vh=640, vs=6400, o=P, o_r=64, oh=640,
             os=6400, B=2, H=4, Hkv=2, Lq=10, Lk=10, d=64, key_len=None, key_mask=None, ms=0, scale=0.0, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(o=None), "null"),
    (dict(Hkv=3), "multiple of Hkv"), (dict(H=0), "Hkv"), (dict(Lq=-1), "Lq"), (dict(Lk=-1), "Lk"), (dict(d=96), "64 or 128"),
    (dict(B=1 << 20, H=1 << 12, Hkv=1), "too many"), (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"), (dict(qr=68), "multiples of 8"), (dict(kh=-8), "multiples of 8"),
    (dict(vs=12), "multiples of 8"), (dict(kr=0), "multiples of 8"), (dict(qr=56), "multiples of 8"),
    (dict(oh=0), "own rows"), (dict(os=0), "own rows"), (dict(q=P + 8), "alignment"), (dict(o=P + 2), "alignment"),
    (dict(key_len=P + 2), "alignment"), (dict(key_mask=P, ms=9), "mask rows"), (dict(key_mask=P, ms=-1), "mask rows")])
def test_cross_attention_refuses(change, word):
    _refused(mkimage.lib.mkb_cross_attention, _with(CROSS, **change), word)


def test_nothing_to_do_is_no_error():
    lib = mkimage.lib
    assert lib.mkb_quantize_rows(*_with(QUANT, rows=0, x=None)) == 0
    assert lib.mkb_proj_i8(*_with(PROJ, M=0, x=None)) == 0
    assert lib.mkb_gate_add_norm(*_with(NORM, rows=0, x=None)) == 0
    assert lib.mkb_cross_attention(*_with(CROSS, B=0, q=None)) == 0
    assert lib.mkb_cross_attention(*_with(CROSS, Lq=0, q=None)) == 0


def test_python_checks_refuse():
    import torch

    ops, bf = mkimage.ops, torch.bfloat16
    f = torch.zeros
    i8 = dict(dtype=torch.int8)
    bad = [
        lambda: ops.quantize_rows(f(4, 64)),  # not on a GPU
        lambda: ops.quantize_rows(f(4, 64, dtype=torch.float16)),
        lambda: ops.quantize_rows(f(4)),
        lambda: ops.proj_i8(f(4, 64, **i8), f(4), f(8, 48, **i8), f(8)),
        lambda: ops.proj_i8(f(4, 64), f(4), f(8, 64, **i8), f(8)),
        lambda: ops.gate_add_norm(f(4, 64, dtype=bf)),
        lambda: ops.gate_add_norm(f(4, 64), f(4, 64, dtype=torch.float16)),
        lambda: ops.cross_attention(f(1, 2, 3, 64), f(2, 2, 3, 64), f(2, 2, 3, 64)),
        lambda: ops.cross_attention(f(1, 2, 3, 64, dtype=bf), f(1, 2, 3, 64, dtype=bf), f(1, 2, 4, 64, dtype=bf)),
    ]
    for call in bad:
        with pytest.raises(mkimage.MkbError):
            call()


@pytest.mark.parametrize("change", [
    dict(out=P, xo=P, out_type=2), dict(out=2 * P, xo=2 * P, out_type=1), dict(out=P, xo=2 * P, out_type=1, y=4 * P),
    dict(out=P, xo=2 * P, out_type=2, ldo=72, y=4 * P), dict(out=4 * P, xo=2 * P, out_type=2, y=4 * P),
    dict(out=4 * P, xo=2 * P, out_type=3, osc=P, y=4 * P), dict(out=4 * P, xo=2 * P, out_type=1, ldo=72, y=4 * P),
    dict(out=P, y=None, y_norm=0, xo=None, out_type=1)])
def test_gate_add_norm_refuses_an_output_over_its_operands(change):
    """An output over x_out, or over x or y in another type or at another distance of rows."""
    _refused(mkimage.lib.mkb_gate_add_norm, _with(NORM, **change), "memory of its own")


@pytest.mark.parametrize("change", [dict(xo=4 * P, y=4 * P), dict(xo=4 * P, y=4 * P, y_f32=1, ldy=72)])
def test_gate_add_norm_refuses_a_residual_over_the_branch(change):
    """x_out over a bf16 y, or over an fp32 one at another distance of rows."""
    _refused(mkimage.lib.mkb_gate_add_norm, _with(NORM, **change), "memory of its own")
