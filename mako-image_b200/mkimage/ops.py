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


def _need(ok, what):
    if not ok:
        raise MkbError(1, what)


def _on(name, device, **tensors):
    """Every given tensor lives on the CUDA device `device`."""
    for k, t in tensors.items():
        _need(t is None or t.device == device, f"{name}: {k} is on {getattr(t, 'device', None)}, not on {device}")
    _need(device.type == "cuda", f"{name}: tensors must be CUDA tensors")


def _launch(fn, device, *args):
    """fn(*args, stream) on the tensors' device and its current stream, whatever device is current."""
    import torch

    if torch.cuda.current_device() == device.index:
        return check(fn(*args, stream_ptr()))
    with torch.cuda.device(device):
        return check(fn(*args, stream_ptr()))


def _row_stride(t):
    """Elements between rows of a 2-D tensor (a single row may come with any stride)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _rows_i8(rows, n, device):
    import torch

    return torch.empty(rows, -(-n // 16) * 16, device=device, dtype=torch.int8)[:, :n]


def quantize_rows(x, q=None, scale=None):
    """(q, scale): rows of x [rows][n] (bf16 or fp32) as int8 with an fp32 step max|row| / 127 each, so that q * scale
    is x to half a step (see mkb_quantize_rows). q's rows are 16 bytes aligned, as proj_i8 wants them."""
    import torch

    _need(x.dim() == 2 and x.dtype in (torch.bfloat16, torch.float32), "quantize_rows: x must be 2-D bf16 or fp32")
    rows, n = x.shape
    if q is None:
        q = _rows_i8(rows, n, x.device)
    if scale is None:
        scale = torch.empty(rows, device=x.device, dtype=torch.float32)
    _on("quantize_rows", x.device, x=x, q=q, scale=scale)
    _need(n > 0 and x.stride(1) == 1 or n == 1, "quantize_rows: the values of a row must be contiguous")
    _need(q.shape == x.shape and q.dtype == torch.int8 and (q.stride(1) == 1 or n == 1),
          "quantize_rows: q must be int8 rows of x's shape")
    _need(scale.shape == (rows,) and scale.dtype == torch.float32 and scale.is_contiguous(),
          "quantize_rows: scale must be contiguous fp32 [rows]")
    _launch(lib.mkb_quantize_rows, x.device, _p(x), _row_stride(x), int(x.dtype == torch.float32), _p(q),
            _row_stride(q), _p(scale), rows, n)
    return q, scale


def proj_i8(x, x_scale, w, w_scale, bias=None, act=ACT_NONE, out=None, out_f32=False):
    """y = act(x_scale[:, None] * w_scale * (x @ w.T) + bias): x [M][K] and w [N][K] int8 with rows 16 bytes aligned
    (quantize_rows makes such rows), scales fp32, exact integer sums (see mkb_proj_i8)."""
    import torch

    _need(x.dim() == 2 and w.dim() == 2 and x.dtype == torch.int8 and w.dtype == torch.int8 and
          x.shape[1] == w.shape[1], "proj_i8: x [M][K] and w [N][K] must be int8")
    M, K = x.shape
    N = w.shape[0]
    if out is None:
        out = torch.empty(M, N, device=x.device, dtype=torch.float32 if out_f32 else torch.bfloat16)
    _on("proj_i8", x.device, x=x, x_scale=x_scale, w=w, w_scale=w_scale, bias=bias, out=out)
    for t in (x, w, out):
        _need(t.stride(1) == 1 or t.shape[1] == 1, "proj_i8: the values of a row must be contiguous")
    _need(out.shape == (M, N) and out.dtype in (torch.float32, torch.bfloat16), "proj_i8: out must be [M][N] fp32 or bf16")
    for t, n in ((x_scale, M), (w_scale, N), (bias, N)):
        _need(t is None or (t.shape == (n,) and t.dtype == torch.float32 and t.is_contiguous()),
              "proj_i8: scales and bias must be contiguous fp32 vectors, one value a row of x or w")
    ldx, ldw = (t.stride(0) if t.shape[0] > 1 else -(-max(t.stride(0), K) // 16) * 16 for t in (x, w))
    _launch(lib.mkb_proj_i8, x.device, _p(x), ldx, _p(x_scale), _p(w), ldw, _p(w_scale), _p(bias), _p(out),
            _row_stride(out), M, N, K, act, int(out.dtype == torch.float32))
    return out


def gate_add_norm(x, y=None, y_norm=NORM_NONE, y_weight=None, gate=None, tanh_gate=False, x_norm=NORM_RMS, x_weight=None,
                  scale=None, shift=None, rows_per_sample=None, eps=1e-6, x_out=None, out=None, out_scale=None,
                  out_type=OUT_BF16):
    """The end of a block's branch and the start of the next in one pass (see mkb_gate_add_norm):

        x  += g(gate) * norm_y(y) * y_weight            (into x_out when it is given)
        out = norm_x(x) * x_weight * (1 + scale) + shift

    x [rows][n] fp32, y bf16 or fp32; gate, scale, shift [samples][n] (or [n]) of the sample row // rows_per_sample.
    Returns out as out_type says: bf16, fp32, (int8 rows, steps) or None."""
    import torch

    f32 = torch.float32
    _need(x.dim() == 2 and x.dtype == f32, "gate_add_norm: x must be 2-D fp32")
    rows, n = x.shape
    rps = rows_per_sample or max(rows, 1)
    samples = -(-rows // rps)
    if x_out is None:
        x_out = x
    if out_type == OUT_I8:
        if out is None:
            out = _rows_i8(rows, n, x.device)
        if out_scale is None:
            out_scale = torch.empty(rows, device=x.device, dtype=f32)
    elif out_type != OUT_NONE and out is None:
        out = torch.empty(rows, n, device=x.device, dtype=f32 if out_type == OUT_F32 else torch.bfloat16)
    _on("gate_add_norm", x.device, x=x, y=y, y_weight=y_weight, gate=gate, x_weight=x_weight, scale=scale, shift=shift,
        x_out=x_out, out=out, out_scale=out_scale)
    want = {OUT_BF16: torch.bfloat16, OUT_F32: f32, OUT_I8: torch.int8}.get(out_type)
    _need(x_out.dtype == f32 and (y is None or y.dtype in (f32, torch.bfloat16)) and
          (out is None) == (want is None) and (out is None or out.dtype == want), "gate_add_norm: wrong type")
    for t in (x, x_out, y, out):
        _need(t is None or (t.shape == x.shape and (n == 1 or t.stride(1) == 1)),
              "gate_add_norm: x, x_out, y and out must be [rows][n] with contiguous rows")
    for t in (y_weight, x_weight):
        _need(t is None or (t.shape == (n,) and t.dtype == f32 and t.is_contiguous()),
              "gate_add_norm: weights must be contiguous fp32 [n]")
    for t in (gate, scale, shift):
        _need(t is None or (t.dtype == f32 and t.shape[-1] == n and t.stride(-1) == 1 and
                            (t.dim() == 1 or (t.dim() == 2 and t.shape[0] in (1, samples) or rows == 0))),
              "gate_add_norm: gate, scale and shift must be fp32 [n] or [samples][n]")
    _need(out_scale is None or (out_type == OUT_I8 and out_scale.shape == (rows,) and out_scale.dtype == f32 and
                                out_scale.is_contiguous()), "gate_add_norm: out_scale must be contiguous fp32 [rows]")

    def per_sample(t):
        return t.stride(0) if t is not None and t.dim() == 2 and t.shape[0] > 1 else 0

    _need(scale is None or shift is None or samples <= 1 or per_sample(scale) == per_sample(shift),
          "gate_add_norm: scale and shift must have the same strides")
    _launch(lib.mkb_gate_add_norm, x.device, _p(x), _row_stride(x), _p(x_out), _row_stride(x_out), _p(y),
            _row_stride(y) if y is not None else 0, int(y is not None and y.dtype == f32), y_norm, _p(y_weight),
            _p(gate), per_sample(gate), int(tanh_gate), x_norm if out_type != OUT_NONE else NORM_NONE, _p(x_weight),
            _p(scale), _p(shift), per_sample(scale if scale is not None else shift), rps, eps, _p(out),
            _row_stride(out) if out is not None else 0, out_type, _p(out_scale), rows, n)
    return (out, out_scale) if out_type == OUT_I8 else out


def cross_attention(q, k, v, key_len=None, key_mask=None, scale=None, out=None):
    """Attention of q [B][H][Lq][d] to another stream's k, v [B][Hkv][Lk][d] (bf16, d 64 or 128, any strides with
    contiguous heads: permuted token-major projections as well as head-major ones), over each sample's first key_len[b]
    keys that key_mask [B][Lk] (bool) leaves (see mkb_cross_attention). Returns out [B][Lq][H * d] (given: any
    [B][Lq][H][d] or [B][Lq][H * d] bf16)."""
    import torch

    _need(q.dim() == 4 and k.dim() == 4 and v.shape == k.shape and q.shape[0] == k.shape[0] and q.shape[3] == k.shape[3],
          "cross_attention: q must be [B][H][Lq][d], k and v [B][Hkv][Lk][d]")
    B, H, Lq, d = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    if out is None:
        out = torch.empty(B, Lq, H * d, device=q.device, dtype=torch.bfloat16)
    _need(tuple(out.shape) in ((B, Lq, H * d), (B, Lq, H, d)), "cross_attention: out must be [B][Lq][H * d]")
    heads = (out.stride(0), out.stride(2) if out.dim() == 4 else d, out.stride(1))
    _on("cross_attention", q.device, q=q, k=k, v=v, out=out, key_len=key_len, key_mask=key_mask)
    for t in (q, k, v, out):
        _need(t.dtype == torch.bfloat16 and t.stride(-1) == 1, "cross_attention: tensors must be bf16 with contiguous heads")
    _need(key_len is None or (key_len.shape == (B,) and key_len.dtype == torch.int32 and key_len.is_contiguous()),
          "cross_attention: key_len must be contiguous int32 [B]")
    _need(key_mask is None or (key_mask.shape == (B, Lk) and key_mask.dtype in (torch.bool, torch.uint8) and
                               (key_mask.stride(1) == 1 or Lk <= 1)), "cross_attention: key_mask must be bool [B][Lk]")
    _need(scale is None or scale > 0, "cross_attention: the scale must be positive")
    _launch(lib.mkb_cross_attention, q.device, _p(q), q.stride(2), q.stride(1), q.stride(0), _p(k), k.stride(2),
            k.stride(1), k.stride(0), _p(v), v.stride(2), v.stride(1), v.stride(0), _p(out), heads[2], heads[1],
            heads[0], B, H, Hkv, Lq, Lk, d, _p(key_len), _p(key_mask),
            key_mask.stride(0) if key_mask is not None else 0, scale or 0.0)
    return out
