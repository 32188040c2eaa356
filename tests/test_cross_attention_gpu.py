"""mkb_cross_attention against softmax attention in 64 bits.

Tolerance per element, from the roundings: the weights p are rounded to bf16 before they meet v (2^-8 of each), so the
output is off by at most 2^-8 sum p|v| / sum p; 2^s from the SFU or a cubic is off by 7.5e-5 < 2^-13 in every weight, in
numerator and sum (twice that); scores come from fp32 sums of d products, each off by d 2^-24 of sum |q||k| scale,
which moves a weight by as much; a result put together from parts is fp32; the bf16 output is 2^-8 of the value. TOL is
2^-8 + 2^-11 on sum p|v| / sum p, plus 2^-8 |o|."""

import math

import pytest

pytestmark = pytest.mark.gpu


def _heads(cuda, g, B, H, L, d, layout="head", scale=1.0):
    import torch

    if layout == "token":
        t = torch.randn(B, L, H, d, generator=g).mul_(scale).to(torch.bfloat16).to(cuda).transpose(1, 2)
    else:
        t = torch.randn(B, H, L, d, generator=g).mul_(scale).to(torch.bfloat16).to(cuda)
    return t


def _ref(q, k, v, key_len, key_mask, scale):
    import torch

    D = torch.float64
    B, H, Lq, d = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    out = torch.zeros(B, Lq, H, d, dtype=D, device=q.device)
    mag = torch.zeros_like(out)
    for b in range(B):
        see = torch.ones(Lk, dtype=torch.bool, device=q.device)
        if key_len is not None:
            see[max(0, min(Lk, int(key_len[b]))):] = False
        if key_mask is not None:
            see &= key_mask[b].bool()
        if not bool(see.any()):
            continue
        kk = k[b][:, see].to(D).repeat_interleave(H // Hkv, 0)
        vv = v[b][:, see].to(D).repeat_interleave(H // Hkv, 0)
        p = torch.softmax(q[b].to(D) @ kk.transpose(1, 2) * scale, -1)
        out[b] = (p @ vv).transpose(0, 1)
        mag[b] = (p @ vv.abs()).transpose(0, 1)
    return out, mag


def _check(q, k, v, key_len=None, key_mask=None, scale=None, out=None):
    import torch
    import mkimage

    ops = mkimage.ops
    got = ops.cross_attention(q, k, v, key_len=key_len, key_mask=key_mask, scale=scale, out=out)
    assert ops.check_kernels() == 0
    B, H, Lq, d = q.shape
    ref, mag = _ref(q, k, v, key_len, key_mask, scale or 1 / math.sqrt(d))
    err = (got.reshape(B, Lq, H, d).to(torch.float64) - ref).abs()
    tol = (2.0 ** -8 + 2.0 ** -11) * mag + 2.0 ** -8 * ref.abs()
    assert bool((err <= tol).all()), (float((err - tol).max()), (err > tol).nonzero()[:4])
    return got


@pytest.mark.parametrize("B,H,Hkv,Lq,Lk", [
    (1, 1, 1, 1, 1), (1, 2, 2, 1, 77), (2, 3, 3, 5, 16), (2, 4, 2, 127, 77), (1, 3, 1, 128, 128), (2, 2, 1, 129, 129),
    (1, 2, 2, 256, 300), (1, 2, 2, 257, 512), (3, 4, 4, 300, 31), (2, 10, 10, 1000, 77), (1, 4, 1, 700, 1000),
    (1, 1, 1, 1, 4096), (2, 4, 4, 1, 5000), (1, 8, 2, 3, 2049), (1, 2, 2, 64, 3333), (4, 24, 24, 260, 130),
    (2, 8, 4, 1, 700), (2, 3, 1, 1, 300), (1, 3, 3, 128, 8000), (1, 3, 3, 256, 8000), (2, 3, 3, 255, 257), (3, 20, 20, 1100, 77),
    (2, 12, 12, 800, 600)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("layout", ["head", "token"])
def test_full_keys(cuda, B, H, Hkv, Lq, Lk, d, layout):
    import torch

    g = torch.Generator().manual_seed(Lq * 7 + Lk)
    _check(_heads(cuda, g, B, H, Lq, d, layout, 1.5), _heads(cuda, g, B, Hkv, Lk, d, layout), _heads(cuda, g, B, Hkv, Lk, d, layout))


@pytest.mark.parametrize("Lq,Lk", [(1, 200), (40, 77), (257, 333), (600, 512), (1, 3000), (2, 3000), (100, 2500), (200, 2500),
                                   (1300, 300)])
@pytest.mark.parametrize("d", [64, 128])
def test_key_lengths_and_masks(cuda, Lq, Lk, d):
    """Each sample its own keys: none, one, all; holes, a first tile without keys, the last key alone."""
    import torch

    B, H, Hkv = 6, 4, 2
    g = torch.Generator().manual_seed(Lk)
    q, k, v = _heads(cuda, g, B, H, Lq, d), _heads(cuda, g, B, Hkv, Lk, d), _heads(cuda, g, B, Hkv, Lk, d, "token")
    lens = torch.tensor([0, 1, Lk, Lk // 2, Lk + 9, -4], dtype=torch.int32, device=cuda)
    got = _check(q, k, v, key_len=lens)
    assert int((got[[0, 5]] != 0).sum()) == 0
    mask = torch.rand(B, Lk, generator=g) < 0.7
    mask[0] = False
    mask[1] = False
    mask[1, Lk - 1] = True
    mask[2, :150] = False
    mask[3] = False
    mask[3, ::17] = True
    mask = mask.to(cuda)
    _check(q, k, v, key_mask=mask)
    lens = torch.tensor([Lk, Lk, Lk, Lk // 2, 1, 0], dtype=torch.int32, device=cuda)
    _check(q, k, v, key_len=lens, key_mask=mask)
    wide = torch.zeros(B, Lk + 13, dtype=torch.uint8, device=cuda)  # rows further apart, at odd addresses, any nonzero byte
    wide[:, 5:5 + Lk] = mask.to(torch.uint8) * 200
    _check(q, k, v, key_len=lens, key_mask=wide[:, 5:5 + Lk])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("Lq,Lk", [(1, 300), (200, 77), (520, 400), (1, 4000), (3, 200), (60, 1700), (180, 1700)])
def test_nothing_hidden_reaches_the_result(cuda, d, Lq, Lk):
    """NaN and infinities in masked and cut-off keys and values, and behind them in memory, change no bit."""
    import torch
    import mkimage

    B, H = 3, 2
    g = torch.Generator().manual_seed(2)
    q = _heads(cuda, g, B, H, Lq, d)
    kb, vb = _heads(cuda, g, B, H, Lk + 40, d), _heads(cuda, g, B, H, Lk + 40, d)
    lens = torch.tensor([Lk // 3, Lk, 5], dtype=torch.int32, device=cuda)
    mask = (torch.rand(B, Lk, generator=g) < 0.6).to(cuda)
    mask[:, 0] = True
    ops = mkimage.ops
    want = _check(q, kb[:, :, :Lk], vb[:, :, :Lk], key_len=lens, key_mask=mask).clone()
    hidden = ~mask | (torch.arange(Lk, device=cuda)[None] >= lens[:, None])
    hidden = torch.cat([hidden, torch.ones(B, 40, dtype=torch.bool, device=cuda)], 1)
    for bad in (float("nan"), float("inf"), -float("inf"), 3e38):
        k2 = torch.where(hidden[:, None, :, None], torch.full_like(kb, bad), kb)
        v2 = torch.where(hidden[:, None, :, None], torch.full_like(vb, bad), vb)
        got = ops.cross_attention(q, k2[:, :, :Lk], v2[:, :, :Lk], key_len=lens, key_mask=mask)
        assert torch.equal(got, want), bad
    assert ops.check_kernels() == 0


def test_a_visible_nan_is_seen(cuda):
    import torch
    import mkimage

    g = torch.Generator().manual_seed(2)
    q, k, v = (_heads(cuda, g, 2, 2, 150, 64) for _ in range(3))
    v[0, 1, 3, 7] = float("nan")
    out = mkimage.ops.cross_attention(q, k, v).reshape(2, 150, 2, 64)
    assert bool(torch.isnan(out[0, :, 1, 7]).all())
    out[0, :, 1, 7] = 0
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("d", [64, 128])
def test_sharp_and_flat_scores(cuda, d):
    """Scores that grow along the keys by far more than the rescaling threshold, and all-equal ones."""
    import torch

    g = torch.Generator().manual_seed(4)
    B, H, Lq, Lk = 1, 2, 130, 700
    q, k, v = _heads(cuda, g, B, H, Lq, d), _heads(cuda, g, B, H, Lk, d), _heads(cuda, g, B, H, Lk, d)
    ramp = torch.linspace(0, 6, Lk, device=cuda)[None, None, :, None]
    _check(q.abs(), (k.abs() * 0.1 + ramp).to(torch.bfloat16), v)
    _check(q.abs(), (k.abs() * 0.1 - 20 + ramp).to(torch.bfloat16), v)
    _check(torch.zeros_like(q), k, v)
    _check(q, k, v, scale=1e-6)
    _check(q, k, v, scale=0.9)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("Lq", [1, 100, 300])
def test_strided_views_shared_keys_and_guards(cuda, d, Lq):
    """q, k, v as slices of one packed projection, a batch that shares one set of keys, an output inside a larger
    buffer whose other elements stay."""
    import torch
    import mkimage

    g = torch.Generator().manual_seed(6)
    B, H, Lk = 3, 4, 90
    packed = torch.randn(B, max(Lq, Lk), 3, H, d, generator=g).to(torch.bfloat16).to(cuda)
    q = packed[:, :Lq, 0].transpose(1, 2)
    k, v = (packed[:1, :Lk, i].transpose(1, 2).expand(B, -1, -1, -1) for i in (1, 2))
    buf = torch.full((B, Lq + 3, H * d + 64), 9.0, dtype=torch.bfloat16, device=cuda)
    out = buf[:, 1:Lq + 1, 32:32 + H * d]
    _check(q, k, v, out=out)
    inside = torch.zeros_like(buf, dtype=torch.bool)
    inside[:, 1:Lq + 1, 32:32 + H * d] = True
    assert bool((buf[~inside] == 9).all())
    lens = torch.tensor([0, 90, 0], dtype=torch.int32, device=cuda)
    hm = torch.full((B, H, Lq, d), 9.0, dtype=torch.bfloat16, device=cuda)  # head-major output
    _check(q, k, v, key_len=lens, out=hm.transpose(1, 2))
    one = mkimage.ops.cross_attention(q, k[:, :1], v[:, :1])  # one key head for all
    assert torch.equal(one, mkimage.ops.cross_attention(q, k[:, :1].expand(-1, H, -1, -1), v[:, :1].expand(-1, H, -1, -1)))


def test_no_keys_at_all(cuda):
    import torch
    import mkimage

    q = torch.randn(2, 3, 50, 64, device=cuda).to(torch.bfloat16)
    k = torch.empty(2, 3, 0, 64, device=cuda, dtype=torch.bfloat16)
    out = torch.full((2, 50, 192), 4.0, device=cuda, dtype=torch.bfloat16)
    mkimage.ops.cross_attention(q, k, k, out=out)
    assert int((out != 0).sum()) == 0


@pytest.mark.parametrize("Lq", [1, 300])
def test_offsets_past_32_bits(cuda, Lq):
    """Samples more than 2^31 elements apart in q, k, v and out."""
    import torch
    import mkimage

    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    g = torch.Generator().manual_seed(6)
    B, H, Lk, d = 2, 2, 140, 64
    far = 2 ** 31 + 1024
    q, k, v = _heads(cuda, g, B, H, Lq, d), _heads(cuda, g, B, H, Lk, d), _heads(cuda, g, B, H, Lk, d)

    def spread(t):
        buf = torch.empty(far + t[0].numel(), dtype=torch.bfloat16, device=cuda)
        s = buf.as_strided(t.shape, (far, t.stride(1), t.stride(2), 1))
        s.copy_(t)
        return s

    want = mkimage.ops.cross_attention(q, k, v)
    buf = torch.empty(far + want[0].numel(), dtype=torch.bfloat16, device=cuda)
    out = buf.as_strided(want.shape, (far, want.stride(1), 1))
    mkimage.ops.cross_attention(spread(q), spread(k), spread(v), out=out)
    assert torch.equal(out, want) and mkimage.ops.check_kernels() == 0
