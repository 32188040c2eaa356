"""Runtime operations on torch CUDA tensors, each one call into the C ABI (include/mkb_image.h, part 1)."""

import ctypes

from ._lib import lib, check, stream_ptr, MkbError

ACT_NONE, ACT_GELU_TANH, ACT_SILU, ACT_QUICK_GELU, ACT_GELU_ERF = 0, 1, 2, 3, 4


def _p(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def proj(x, w, bias=None, act=ACT_NONE, out=None, out_f32=False):
    """y = act(x @ w.T + bias); x [M][K] bf16, w [N][K] bf16, bias fp32 [N]."""
    import torch

    M, K = x.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty(M, N, device=x.device, dtype=torch.float32 if out_f32 else torch.bfloat16)
    check(lib.mkb_proj(_p(x), x.stride(0), _p(w), w.stride(0), _p(bias), _p(out), out.stride(0), M, N, K, act,
                       int(out_f32), stream_ptr()))
    return out


def proj_gate_add(x, w, resid, gate, bias=None, rows_per_sample=None, tanh_gate=False):
    """resid += g(gate[row // rows_per_sample]) * (x @ w.T + bias), in place; gate [samples][N] fp32."""
    M, K = x.shape
    N = w.shape[0]
    rps = rows_per_sample or M
    check(lib.mkb_proj_gate_add(_p(x), x.stride(0), _p(w), w.stride(0), _p(bias), _p(resid), resid.stride(0),
                                _p(gate), gate.stride(0) if gate.dim() > 1 else 0, rps, int(tanh_gate), M, N, K,
                                stream_ptr()))
    return resid


def proj_qkv_heads(x, w, bias, norm_q, norm_k, rope, qh, kh, vh, rows_per_sample, pos_offset, eps=1e-6):
    """Fused QKV projection into head-major q/k/v [samples][heads][L][128] (bf16)."""
    M, K = x.shape
    heads, L = qh.shape[1], qh.shape[2]
    check(lib.mkb_proj_qkv_heads(_p(x), x.stride(0), _p(w), w.stride(0), _p(bias), _p(norm_q), _p(norm_k), _p(rope),
                                 _p(qh), _p(kh), _p(vh), heads, L, rows_per_sample, pos_offset, eps, M, K,
                                 stream_ptr()))


def proj_swiglu(x, w_interleaved, bias=None, out=None):
    """silu(gate) * up from a gate/up-interleaved weight (see swiglu_interleave)."""
    import torch

    M, K = x.shape
    N = w_interleaved.shape[0]
    if out is None:
        out = torch.empty(M, N // 2, device=x.device, dtype=torch.bfloat16)
    check(lib.mkb_proj_swiglu(_p(x), x.stride(0), _p(w_interleaved), w_interleaved.stride(0), _p(bias), _p(out),
                              out.stride(0), M, N, K, stream_ptr()))
    return out


def swiglu_interleave_block():
    return lib.mkb_swiglu_interleave()


def check_kernels():
    bits = ctypes.c_uint32(0)
    check(lib.mkb_check_kernels(ctypes.byref(bits)))
    return bits.value


MASK_NONE, MASK_COND_CAUSAL = 0, 1


def attention(q, k, v, out0, out1, split, Lq=None, Lk=None, q_pos0=0, mask=MASK_NONE, cond_len=0):
    """Flash attention over head-major q [B][H][Lq_rows][d], k/v [B][H][Lk_rows][d] (d 64 or 128); rows routed into out0
    (joint positions < split) and out1 (see mkb_attention)."""
    B, H, Lq_rows, hd = q.shape
    Lk_rows = k.shape[2]
    Lq = Lq or Lq_rows
    Lk = Lk or Lk_rows
    rows0 = out0.shape[0] // B if out0 is not None else 0
    rows1 = out1.shape[0] // B
    check(lib.mkb_attention(_p(q), Lq, Lq_rows, _p(k), _p(v), Lk, Lk_rows, B, H, hd, q_pos0, mask, cond_len, split,
                            _p(out0), out0.stride(0) if out0 is not None else 0, rows0, _p(out1), out1.stride(0),
                            rows1, stream_ptr()))


def attention_kv_shards(q, k, v, out0, out1, split, Lk, kv_shard_rows, kv_plane_stride, Lq=None, q_pos0=0,
                        mask=MASK_NONE, cond_len=0):
    """attention() with keys and values in shards of kv_shard_rows rows: k and v are [planes][kv_shard_rows][d] and
    key row j of head bh is row j % kv_shard_rows of plane (j // kv_shard_rows) * kv_plane_stride + bh (see
    mkb_attention_kv_shards)."""
    B, H, Lq_rows, hd = q.shape
    Lq = Lq or Lq_rows
    rows0 = out0.shape[0] // B if out0 is not None else 0
    rows1 = out1.shape[0] // B
    check(lib.mkb_attention_kv_shards(_p(q), Lq, Lq_rows, _p(k), _p(v), Lk, Lk, B, H, hd, q_pos0, mask, cond_len,
                                      split, _p(out0), out0.stride(0) if out0 is not None else 0, rows0, _p(out1),
                                      out1.stride(0), rows1, kv_shard_rows, kv_plane_stride, stream_ptr()))


def attention_kv_arriving(q, k, v, out0, out1, split, Lk, kv_shard_rows, kv_plane_stride, own_shard, shard_ready,
                          shard_expect, Lq=None, q_pos0=0):
    """attention_kv_shards() where shard own_shard is complete and every other shard g is read only once the int64
    device flag shard_ready[g] >= shard_expect[0] (see mkb_attention_kv_arriving)."""
    B, H, Lq_rows, hd = q.shape
    Lq = Lq or Lq_rows
    rows0 = out0.shape[0] // B if out0 is not None else 0
    rows1 = out1.shape[0] // B
    check(lib.mkb_attention_kv_arriving(_p(q), Lq, Lq_rows, _p(k), _p(v), Lk, Lk, B, H, hd, q_pos0, MASK_NONE, 0,
                                        split, _p(out0), out0.stride(0) if out0 is not None else 0, rows0, _p(out1),
                                        out1.stride(0), rows1, kv_shard_rows, kv_plane_stride, own_shard,
                                        _p(shard_ready), _p(shard_expect), stream_ptr()))


def attention_wide(qkv, d, n=None, q_col=0, k_col=None, v_col=None, out=None):
    """Single-head attention at head dim 256 / 512 over rows of qkv [n][ld] holding q, k, v side by side (see
    mkb_attention_wide); returns out [n][d] bf16."""
    import torch

    n = n or qkv.shape[0]
    k_col = d if k_col is None else k_col
    v_col = 2 * d if v_col is None else v_col
    if out is None:
        out = torch.empty(n, d, device=qkv.device, dtype=torch.bfloat16)
    check(lib.mkb_attention_wide(_p(qkv), qkv.stride(0), n, d, q_col, k_col, v_col, _p(out), out.stride(0),
                                 stream_ptr()))
    return out


def proj_add(x, w, bias=None, addvec=None, rows_per_sample=None, resid=None, out=None, out_f32=True):
    """y = x @ w.T + bias + addvec[row // rows_per_sample] + resid (fp32 or bf16 out; resid may be out)."""
    import torch

    M, K = x.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty(M, N, device=x.device, dtype=torch.float32 if out_f32 else torch.bfloat16)
    check(lib.mkb_proj_add(_p(x), x.stride(0), _p(w), w.stride(0), _p(bias), _p(addvec),
                           addvec.stride(0) if addvec is not None and addvec.dim() > 1 else 0, rows_per_sample or M,
                           _p(resid), resid.stride(0) if resid is not None else 0, _p(out), out.stride(0),
                           int(out_f32), M, N, K, stream_ptr()))
    return out


def proj_heads(x, w, bias, qh, kh, vh, part0, D, rows_per_sample, pos_offset):
    """Scatter x @ w.T + bias into head-major q/k/v [samples][heads][L][head_dim] (no norm)."""
    M, K = x.shape
    N = w.shape[0]
    ref = next(t for t in (qh, kh, vh) if t is not None)
    L, hd = ref.shape[2], ref.shape[3]
    check(lib.mkb_proj_heads(_p(x), x.stride(0), _p(w), w.stride(0), _p(bias), _p(qh), _p(kh), _p(vh), part0, D, hd,
                             L, rows_per_sample, pos_offset, M, N, K, stream_ptr()))


def proj_geglu(x, w_interleaved, bias=None, out=None):
    import torch

    M, K = x.shape
    N = w_interleaved.shape[0]
    if out is None:
        out = torch.empty(M, N // 2, device=x.device, dtype=torch.bfloat16)
    check(lib.mkb_proj_geglu(_p(x), x.stride(0), _p(w_interleaved), w_interleaved.stride(0), _p(bias), _p(out),
                             out.stride(0), M, N, K, stream_ptr()))
    return out


def conv2d(x, w, taps=9, stride=1, bias=None, addvec=None, resid=None, out=None, out_f32=True):
    """x: channels-last bf16 [B][H][W][C]; w: bf16 [Cout][taps * C]; returns [B][Ho][Wo][Cout]."""
    import torch

    B, H, W, C = x.shape
    Cout = w.shape[0]
    Ho = (H - 1) // stride + 1 if taps == 9 else H
    Wo = (W - 1) // stride + 1 if taps == 9 else W
    if out is None:
        out = torch.empty(B, Ho, Wo, Cout, device=x.device, dtype=torch.float32 if out_f32 else torch.bfloat16)
    check(lib.mkb_conv2d(_p(x), B, H, W, C, _p(w), Cout, taps, stride, _p(bias), _p(addvec),
                         addvec.stride(0) if addvec is not None else 0, _p(resid), Cout if resid is not None else 0,
                         _p(out), Cout, int(out_f32), stream_ptr()))
    return out


def ln_modulate(x, mod, shift=None, eps=1e-6, split=0, mod_stride=0, mod_off=0, out=None):
    """bf16 LayerNorm(x) * (1 + scale) (+ shift) of fp32 rows x [rows][n]; row r's scale is
    mod.flatten()[(r < split ? mod_stride : 0) + mod_off + i] (see mkb_ln_modulate)."""
    import torch

    rows, n = x.shape
    if out is None:
        out = torch.empty(rows, n, device=x.device, dtype=torch.bfloat16)
    check(lib.mkb_ln_modulate(_p(x), _p(mod), _p(shift), _p(out), rows, n, eps, split, mod_stride, mod_off,
                              stream_ptr()))
    return out


def group_norm(x, gamma, beta, groups=32, eps=1e-5, silu=False, out=None):
    """x: fp32 channels-last [B][HW][C] (any shape with that memory order); returns bf16 of the same shape."""
    import torch

    B, C = x.shape[0], x.shape[-1]
    HW = x.numel() // (B * C)
    ws_bytes = lib.mkb_group_norm_workspace_size(B, HW, C, groups)
    ws = torch.empty(max(ws_bytes, 16) // 4 + 1, device=x.device, dtype=torch.float32)
    if out is None:
        out = torch.empty(x.shape, device=x.device, dtype=torch.bfloat16)
    check(lib.mkb_group_norm(_p(x), _p(out), _p(gamma), _p(beta), B, HW, C, groups, eps, int(silu), _p(ws),
                             ws.numel() * 4, stream_ptr()))
    return out


NORM_NONE, NORM_RMS, NORM_LAYER = 0, 1, 2
OUT_NONE, OUT_BF16, OUT_F32, OUT_I8 = 0, 1, 2, 3


# torch and the two calls every launch needs of it, looked up once: a call of these operators costs the host about as much as
# its launch, so their checks are written for few steps (and outputs made by empty_strided: 1.8 us, empty takes 2.5). A call for
# another device than the current one is made again with that device current; launches go to the device's current stream.
torch = None
_current_device = _raw_stream = None


def _load():
    global torch, _current_device, _raw_stream
    import torch as t

    torch, _current_device, _raw_stream = t, t._C._cuda_getDevice, t._C._cuda_getCurrentRawStream
    return t


def _fail(what):
    raise MkbError(1, what)


def _same_device(name, dev, *tensors):
    """The given tensors live on CUDA device `dev`."""
    if dev < 0:
        _fail(f"{name}: tensors must be CUDA tensors")
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _fail(f"{name}: a tensor is on {t.device}, not on cuda:{dev}")


def _row_stride(t, n):
    """Elements between the rows of a 2-D tensor of n columns (a single row may come with any stride)."""
    s = t.stride(0)
    return s if s >= n else n if t.shape[0] <= 1 else s


def _vector(t, n, f32, what):
    if t.dtype is not f32 or t.shape != (n,) or (n > 1 and not t.is_contiguous()):
        _fail(what)


def quantize_rows(x, q=None, scale=None):
    """(q, scale): rows of x [rows][n] (bf16 or fp32) as int8 with an fp32 step max|row| / 127 each, so that q * scale
    is x to half a step (see mkb_quantize_rows). q's rows are 16 bytes aligned, as proj_i8 wants them."""
    t = torch or _load()
    f32 = x.dtype is t.float32
    if x.dim() != 2 or not (f32 or x.dtype is t.bfloat16):
        _fail("quantize_rows: x must be 2-D bf16 or fp32")
    rows, n = x.shape
    ldx, step = x.stride()
    if n == 0 or (step != 1 and n > 1):
        _fail("quantize_rows: the values of a row must be contiguous, one at least")
    dev = x.get_device()
    _same_device("quantize_rows", dev, q, scale)
    if _current_device() != dev:
        with t.cuda.device(dev):
            return quantize_rows(x, q, scale)
    if q is None:
        ldq = (n + 15) & ~15
        q = t.empty_strided((rows, n), (ldq, 1), device=x.device, dtype=t.int8)
    else:
        if q.shape != x.shape or q.dtype is not t.int8 or (n > 1 and q.stride(1) != 1):
            _fail("quantize_rows: q must be int8 rows of x's shape")
        ldq = _row_stride(q, n)
    if scale is None:
        scale = t.empty_strided((rows,), (1,), device=x.device, dtype=t.float32)
    else:
        _vector(scale, rows, t.float32, "quantize_rows: scale must be contiguous fp32 [rows]")
    code = lib.mkb_quantize_rows(x.data_ptr(), ldx if rows > 1 else n, f32, q.data_ptr(), ldq, scale.data_ptr(), rows, n,
                                 _raw_stream(dev))
    if code:
        check(code)
    return q, scale


def proj_i8(x, x_scale, w, w_scale, bias=None, act=ACT_NONE, out=None, out_f32=False):
    """y = act(x_scale[:, None] * w_scale * (x @ w.T) + bias): x [M][K] and w [N][K] int8 with rows 16 bytes aligned
    (quantize_rows makes such rows), scales fp32, exact integer sums (see mkb_proj_i8)."""
    t = torch or _load()
    f32 = t.float32
    if x.dtype is not t.int8 or w.dtype is not t.int8 or x.dim() != 2 or w.dim() != 2:
        _fail("proj_i8: x [M][K] and w [N][K] must be int8")
    M, K = x.shape
    N, Kw = w.shape
    if K != Kw:
        _fail("proj_i8: x [M][K] and w [N][K] must have rows of one length")
    ldx, sx = x.stride()
    ldw, sw = w.stride()
    if K > 1 and (sx != 1 or sw != 1):
        _fail("proj_i8: the values of a row must be contiguous")
    if x_scale.dtype is not f32 or w_scale.dtype is not f32 or x_scale.shape != (M,) or w_scale.shape != (N,) or \
            not (x_scale.is_contiguous() and w_scale.is_contiguous()):
        _fail("proj_i8: the scales must be contiguous fp32 vectors, one value a row of x or w")
    if bias is not None:
        _vector(bias, N, f32, "proj_i8: bias must be contiguous fp32 [N]")
    dev = x.get_device()
    _same_device("proj_i8", dev, x_scale, w, w_scale, bias, out)
    if _current_device() != dev:
        with t.cuda.device(dev):
            return proj_i8(x, x_scale, w, w_scale, bias, act, out, out_f32)
    if out is None:
        out = t.empty_strided((M, N), (N, 1), device=x.device, dtype=f32 if out_f32 else t.bfloat16)
        ldy = N
    else:
        out_f32 = out.dtype is f32
        if out.shape != (M, N) or not (out_f32 or out.dtype is t.bfloat16) or (N > 1 and out.stride(1) != 1):
            _fail("proj_i8: out must be [M][N] fp32 or bf16 with contiguous rows")
        ldy = _row_stride(out, N)
    code = lib.mkb_proj_i8(x.data_ptr(), ldx if M > 1 else (K + 15) & ~15, x_scale.data_ptr(), w.data_ptr(),
                           ldw if N > 1 else (K + 15) & ~15, w_scale.data_ptr(), None if bias is None else bias.data_ptr(),
                           out.data_ptr(), ldy, M, N, K, act, out_f32, _raw_stream(dev))
    if code:
        check(code)
    return out


def gate_add_norm(x, y=None, y_norm=NORM_NONE, y_weight=None, gate=None, tanh_gate=False, x_norm=NORM_RMS, x_weight=None,
                  scale=None, shift=None, rows_per_sample=None, eps=1e-6, x_out=None, out=None, out_scale=None,
                  out_type=OUT_BF16):
    """The end of a block's branch and the start of the next in one pass (see mkb_gate_add_norm):

        x  += g(gate) * norm_y(y) * y_weight            (into x_out when it is given)
        out = norm_x(x) * x_weight * (1 + scale) + shift

    x [rows][n] fp32, y bf16 or fp32; gate, scale, shift [samples][n] (or [n]) of the sample row // rows_per_sample.
    Returns out as out_type says: bf16, fp32, (int8 rows, steps) or None."""
    t = torch or _load()
    f32 = t.float32
    if x.dim() != 2 or x.dtype is not f32:
        _fail("gate_add_norm: x must be 2-D fp32")
    shape = x.shape
    rows, n = shape
    rps = rows_per_sample or max(rows, 1)
    samples = -(-rows // rps)

    def rows_of(a, dtype):
        if a.shape == shape and a.dtype is dtype:
            ld, step = a.stride()
            if step == 1 or n <= 1:
                return ld if rows > 1 else max(ld, n)
        _fail("gate_add_norm: x, x_out, y and out must be [rows][n] of their types with contiguous rows")

    def per_sample(a):
        size, ld = a.shape, a.stride()
        if a.dtype is not f32 or not size or size[-1] != n or (ld[-1] != 1 and n > 1) or \
                (len(size) > 1 and size != (samples, n) and size != (1, n)):
            _fail("gate_add_norm: gate, scale and shift must be fp32 [n] or [samples][n]")
        return ld[0] if len(size) > 1 and size[0] > 1 else 0

    dev = x.get_device()
    _same_device("gate_add_norm", dev, y, y_weight, gate, x_weight, scale, shift, x_out, out, out_scale)
    if _current_device() != dev:
        with t.cuda.device(dev):
            return gate_add_norm(x, y, y_norm, y_weight, gate, tanh_gate, x_norm, x_weight, scale, shift, rows_per_sample, eps,
                                 x_out, out, out_scale, out_type)
    ldx = rows_of(x, f32)
    if x_out is None:
        x_out, ldxo = x, ldx
    else:
        ldxo = rows_of(x_out, f32)
    ldy, y_f32 = 0, False
    if y is not None:
        y_f32 = y.dtype is f32
        ldy = rows_of(y, f32 if y_f32 else t.bfloat16)
    if out_type == OUT_NONE:
        if out is not None:
            _fail("gate_add_norm: out without an out_type")
        x_norm, ldo = NORM_NONE, 0
    else:
        dtype = t.bfloat16 if out_type == OUT_BF16 else f32 if out_type == OUT_F32 else t.int8
        if out is not None:
            ldo = rows_of(out, dtype)
        else:
            ldo = (n + 15) & ~15 if out_type == OUT_I8 else n
            out = t.empty_strided(shape, (ldo, 1), device=x.device, dtype=dtype)
    if out_type == OUT_I8:
        if out_scale is None:
            out_scale = t.empty_strided((rows,), (1,), device=x.device, dtype=f32)
        else:
            _vector(out_scale, rows, f32, "gate_add_norm: out_scale must be contiguous fp32 [rows]")
    elif out_scale is not None:
        _fail("gate_add_norm: out_scale goes with 8-bit outputs alone")
    if y_weight is not None:
        _vector(y_weight, n, f32, "gate_add_norm: weights must be contiguous fp32 [n]")
    if x_weight is not None:
        _vector(x_weight, n, f32, "gate_add_norm: weights must be contiguous fp32 [n]")
    gate_stride = 0 if gate is None else per_sample(gate)
    mod_stride = 0 if scale is None else per_sample(scale)
    if shift is not None:
        shift_stride = per_sample(shift)
        if scale is None:
            mod_stride = shift_stride
        elif shift_stride != mod_stride and samples > 1:
            _fail("gate_add_norm: scale and shift must have the same strides")
    code = lib.mkb_gate_add_norm(
        x.data_ptr(), ldx, x_out.data_ptr(), ldxo, None if y is None else y.data_ptr(), ldy, y_f32, y_norm,
        None if y_weight is None else y_weight.data_ptr(), None if gate is None else gate.data_ptr(), gate_stride, tanh_gate,
        x_norm, None if x_weight is None else x_weight.data_ptr(), None if scale is None else scale.data_ptr(),
        None if shift is None else shift.data_ptr(), mod_stride, rps, eps, None if out is None else out.data_ptr(), ldo,
        out_type, None if out_scale is None else out_scale.data_ptr(), rows, n, _raw_stream(dev))
    if code:
        check(code)
    return (out, out_scale) if out_type == OUT_I8 else out


def cross_attention(q, k, v, key_len=None, key_mask=None, scale=None, out=None):
    """Attention of q [B][H][Lq][d] to another stream's k, v [B][Hkv][Lk][d] (bf16, d 64 or 128, any strides with
    contiguous heads: permuted token-major projections as well as head-major ones), over each sample's first key_len[b]
    keys that key_mask [B][Lk] (bool) leaves (see mkb_cross_attention). Returns out [B][Lq][H * d] (given: any
    [B][Lq][H][d] or [B][Lq][H * d] bf16)."""
    t = torch or _load()
    bf16 = t.bfloat16
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        _fail("cross_attention: q must be [B][H][Lq][d], k and v [B][Hkv][Lk][d]")
    B, H, Lq, d = q.shape
    Bk, Hkv, Lk, dk = k.shape
    if Bk != B or dk != d:
        _fail("cross_attention: q must be [B][H][Lq][d], k and v [B][Hkv][Lk][d]")
    dev = q.get_device()
    _same_device("cross_attention", dev, k, v, out, key_len, key_mask)
    if _current_device() != dev:
        with t.cuda.device(dev):
            return cross_attention(q, k, v, key_len, key_mask, scale, out)
    o_last = 1
    if out is None:
        o_row, o_head, o_sample = H * d, d, Lq * H * d
        out = t.empty_strided((B, Lq, o_row), (o_sample, o_row, 1), device=q.device, dtype=bf16)
    elif out.shape == (B, Lq, H * d):
        o_sample, o_row, o_last = out.stride()
        o_head = d
    elif out.shape == (B, Lq, H, d):
        o_sample, o_row, o_head, o_last = out.stride()
    else:
        _fail("cross_attention: out must be [B][Lq][H * d]")
    q_sample, q_head, q_row, q_last = q.stride()
    k_sample, k_head, k_row, k_last = k.stride()
    v_sample, v_head, v_row, v_last = v.stride()
    if not (q_last == k_last == v_last == o_last == 1) or not (q.dtype is bf16 and k.dtype is bf16 and v.dtype is bf16 and
                                                              out.dtype is bf16):
        _fail("cross_attention: tensors must be bf16 with contiguous heads")
    if key_len is not None and (key_len.dtype is not t.int32 or key_len.shape != (B,) or not key_len.is_contiguous()):
        _fail("cross_attention: key_len must be contiguous int32 [B]")
    mask_stride = 0
    if key_mask is not None:
        if key_mask.shape != (B, Lk) or key_mask.dtype not in (t.bool, t.uint8) or (Lk > 1 and key_mask.stride(1) != 1):
            _fail("cross_attention: key_mask must be bool [B][Lk]")
        mask_stride = key_mask.stride(0)
    if scale is not None and not scale > 0:
        _fail("cross_attention: the scale must be positive")
    code = lib.mkb_cross_attention(
        q.data_ptr(), q_row, q_head, q_sample, k.data_ptr(), k_row, k_head, k_sample, v.data_ptr(), v_row, v_head, v_sample,
        out.data_ptr(), o_row, o_head, o_sample, B, H, Hkv, Lq, Lk, d, None if key_len is None else key_len.data_ptr(),
        None if key_mask is None else key_mask.data_ptr(), mask_stride, scale or 0.0, _raw_stream(dev))
    if code:
        check(code)
    return out
