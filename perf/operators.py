"""The operators of a quantised prompt-conditioned block, as cases that can be timed and compared: the gated residual
add between two norms (ops.gate_add_norm), the product of 8-bit integers with a scale for each token and each channel
(ops.quantize_rows + ops.proj_i8), and attention from image tokens to an encoder's states of another length
(ops.cross_attention).

A case is a dict of plain values. prepare() makes what a program holds before the call, run() makes one pass: with
`own` false in elementary torch operations in fp32, with `own` true through the framework's public entry points."""

import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _ops():
    if "mkimage" not in sys.modules:
        sys.path.insert(0, os.path.join(ROOT, "mako-image_b200"))
    import mkimage

    return mkimage.ops


# ------------------------------------------------------------------------------------------------------- the cases

def _norm(name, rows, n, y_norm, x_norm, y_f32, tanh, mod, out, samples):
    return dict(name=name, op="gate_add_norm", rows=rows, n=n, y_norm=y_norm, x_norm=x_norm, y_f32=y_f32, tanh=tanh,
                mod=mod, out=out, samples=samples)


def _proj(name, M, N, K, act, bias, x_f32, out_f32):
    return dict(name=name, op="proj_i8", M=M, N=N, K=K, act=act, bias=bias, x_f32=x_f32, out_f32=out_f32)


def _cross(name, B, H, Hkv, Lq, Lk, d, lens, mask, token_major):
    return dict(name=name, op="cross_attention", B=B, H=H, Hkv=Hkv, Lq=Lq, Lk=Lk, d=d, lens=lens, mask=mask,
                token_major=token_major)


def listed():
    return [
        # One 77-token prompt chunk for cond and uncond at the SDXL width: a call where latency is all that counts.
        _norm("norm_prompt", 154, 1280, "rms", "rms", False, False, False, "bf16", 2),
        # The denoiser's text and image rows of a CFG pair at 1024^2, feeding an int8 projection.
        _norm("norm_block_i8", 8704, 3072, "rms", "rms", False, True, True, "i8", 2),
        # An odd width and row count, LayerNorms, an fp32 branch: nothing is aligned to vectors.
        _norm("norm_odd", 4099, 1283, "layer", "layer", True, False, True, "bf16", 1),
        # The modulation vector of one sample: a single token through a wide matrix.
        _proj("proj_one_token", 1, 18432, 3072, "silu", True, True, True),
        # A prompt's tokens through an attention output projection.
        _proj("proj_prompt", 77, 1280, 1280, "none", True, False, True),
        # The text rows' q, k, v projection.
        _proj("proj_text_qkv", 512, 9216, 3072, "none", True, False, False),
        # The image rows' feed-forward projection of a CFG pair at 1024^2.
        _proj("proj_ffn_up", 8192, 12288, 3072, "gelu_tanh", True, False, False),
        # The way back at an odd number of rows.
        _proj("proj_ffn_down_odd", 4097, 1280, 5120, "none", False, False, True),
        # The UNet's 64^2 level over one 77-token chunk: few keys, many queries.
        _cross("cross_unet", 2, 10, 10, 4096, 77, 64, "full", False, False),
        # Image tokens of four samples over prompts of different lengths, one of them dropped (no key at all).
        _cross("cross_prompts", 4, 24, 24, 4096, 512, 128, "ragged", True, True),
        # Shared key heads, odd lengths.
        _cross("cross_shared", 3, 16, 4, 257, 333, 128, "ragged", False, True),
        # One pooled query over every image token.
        _cross("cross_pool", 2, 24, 24, 1, 4096, 128, "full", False, False),
    ]


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["gate_add_norm", "proj_i8", "cross_attention"])
    if op == "gate_add_norm":
        n = _log(rng, 64, 6144)
        if rng.random() < 0.6:
            n = max(64, n // 64 * 64)
        rows = _log(rng, 1, min(17408, 8704 * 3072 // n))
        return dict(op=op, rows=rows, n=n, y_norm=rng.choice(["none", "rms", "layer"]),
                    x_norm=rng.choice(["rms", "layer"]), y_f32=rng.random() < 0.3, tanh=rng.random() < 0.5,
                    mod=rng.random() < 0.7, out=rng.choice(["bf16", "i8", "f32"]), samples=rng.choice([1, 2, 3]))
    if op == "proj_i8":
        K, N = _log(rng, 64, 12288), _log(rng, 32, 12288)
        if rng.random() < 0.7:
            K, N = max(64, K // 64 * 64), max(32, N // 32 * 32)
        M = _log(rng, 1, min(8192, 8192 * 12288 * 3072 // (N * K)))
        return dict(op=op, M=M, N=N, K=K, act=rng.choice(["none", "silu", "gelu_tanh"]),
                    bias=rng.random() < 0.7, x_f32=rng.random() < 0.3, out_f32=rng.random() < 0.4)
    d = rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 4, 8, 10, 12])
    H = Hkv * rng.choice([1, 1, 2])
    Lq = _log(rng, 1, 4096)
    Lk = _log(rng, 1, min(8192, max(512, 1 << 21 // max(1, Lq))))
    return dict(op=op, B=rng.choice([1, 2, 3, 4]), H=H, Hkv=Hkv, Lq=Lq, Lk=Lk, d=d,
                lens=rng.choice(["full", "ragged"]), mask=rng.random() < 0.4, token_major=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------------- the inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _samples(c):
    per = -(-c["rows"] // c["samples"])  # the last sample may be shorter
    return -(-c["rows"] // per), per


def _lens(c):
    """Keys of each sample: the first sample's prompt fills its row, the last of three or more has none."""
    if c["lens"] == "full":
        return [c["Lk"]] * c["B"]
    share = [1.0, 0.3, 0.76, 0.52][: c["B"]]
    if c["B"] >= 3:
        share[-1] = 0.0
    return [math.ceil(f * c["Lk"]) for f in share]


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["op"] == "gate_add_norm":
        rows, n = c["rows"], c["n"]
        ns, per = _samples(c)
        s = dict(c=c, per=per)
        s["x"] = 2.0 * _randn(g, rows, n) + 0.1
        y = _randn(g, rows, n) * 3.0 + 0.2
        s["y"] = y if c["y_f32"] else y.to(torch.bfloat16)
        s["y_weight"] = 1.0 + 0.1 * _randn(g, n) if c["y_norm"] != "none" else None
        s["x_weight"] = 1.0 + 0.1 * _randn(g, n)
        s["gate"] = 0.5 * _randn(g, ns, n)
        s["scale"] = 0.3 * _randn(g, ns, n) if c["mod"] else None
        s["shift"] = 0.3 * _randn(g, ns, n) if c["mod"] else None
        s["x_out"] = torch.empty_like(s["x"])
        return s
    if c["op"] == "proj_i8":
        M, N, K = c["M"], c["N"], c["K"]
        s = dict(c=c)
        x = _randn(g, M, K) * (0.5 + torch.rand(M, 1, device="cuda", generator=g))
        s["x"] = x if c["x_f32"] else x.to(torch.bfloat16)
        w = 0.02 * _randn(g, N, K)
        w_scale = w.abs().amax(1) / 127
        q = torch.zeros(N, -(-K // 16) * 16, dtype=torch.int8, device="cuda")[:, :K]  # rows 16 bytes apart
        q.copy_((w / w_scale[:, None]).round().clamp(-127, 127))
        s["w"], s["w_scale"] = q, w_scale
        s["bias"] = 0.1 * _randn(g, N) if c["bias"] else None
        return s
    B, H, Hkv, Lq, Lk, d = (c[k] for k in ("B", "H", "Hkv", "Lq", "Lk", "d"))
    s = dict(c=c)

    def heads(h, L):
        if c["token_major"]:  # as a projection leaves its rows
            return _randn(g, B, L, h, d).to(torch.bfloat16).transpose(1, 2)
        return _randn(g, B, h, L, d).to(torch.bfloat16)

    s["q"], s["k"], s["v"] = heads(H, Lq), heads(Hkv, Lk), heads(Hkv, Lk)
    s["q"] = s["q"] * 1.5  # scores a little sharper than unit variance
    s["key_len"] = s["key_mask"] = None
    if c["lens"] == "ragged":
        s["key_len"] = torch.tensor(_lens(c), dtype=torch.int32, device="cuda")
    if c["mask"]:  # tokens left out of a prompt
        s["key_mask"] = torch.rand(B, Lk, device="cuda", generator=g) < 0.9
    return s


# ------------------------------------------------------------------------------------------------------- one pass

def _plain_norm(t, kind, eps):
    if kind == "none":
        return t
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps)


def _per_row(s, t):
    return torch.repeat_interleave(t, s["per"], 0)[: s["c"]["rows"]]


def _plain_quant(t):
    """Whole numbers as fp32 and the fp32 step: a quotient next to the border of two of them is decided in 64 bits."""
    amax = t.abs().amax(-1, keepdim=True)
    scale = amax / torch.full_like(amax, 127.0)
    q = (t.double() / scale.double()).round()
    return torch.where(scale > 0, q, torch.zeros_like(q)).float(), scale


def _plain_gate_add_norm(s):
    c = s["c"]
    b = _plain_norm(s["y"].float(), c["y_norm"], 1e-6)
    if s["y_weight"] is not None:
        b = b * s["y_weight"]
    gate = torch.tanh(s["gate"]) if c["tanh"] else s["gate"]
    x = s["x"] + _per_row(s, gate) * b
    h = _plain_norm(x, c["x_norm"], 1e-6) * s["x_weight"]
    if s["scale"] is not None:
        h = h * (1.0 + _per_row(s, s["scale"])) + _per_row(s, s["shift"])
    if c["out"] == "i8":
        q, scale = _plain_quant(h)
        return dict(x=x, h=(q * scale).to(torch.bfloat16), h_scale=scale[:, 0])
    return dict(x=x, h=h if c["out"] == "f32" else h.to(torch.bfloat16))


def _plain_act(t, act):
    if act == "silu":
        return t / (1.0 + torch.exp(-t))
    if act == "gelu_tanh":
        return 0.5 * t * (1.0 + torch.tanh(0.7978845608028654 * (t + 0.044715 * t * t * t)))
    return t


def _plain_proj_i8(s):
    c = s["c"]
    q, scale = _plain_quant(s["x"].float())
    y = torch.matmul(q, s["w"].float().t()) * scale * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    y = _plain_act(y, c["act"])
    return y if c["out_f32"] else y.to(torch.bfloat16)


def _visible(s):
    """[B][Lk] truth values: the keys that a sample's queries see."""
    c = s["c"]
    see = torch.ones(c["B"], c["Lk"], dtype=torch.bool, device="cuda")
    if s["key_len"] is not None:
        see = see & (torch.arange(c["Lk"], device="cuda")[None] < s["key_len"][:, None])
    if s["key_mask"] is not None:
        see = see & s["key_mask"]
    return see


def _plain_cross_attention(s):
    c = s["c"]
    see = _visible(s)[:, None, None, None]
    q = s["q"].float().reshape(c["B"], c["Hkv"], c["H"] // c["Hkv"], c["Lq"], c["d"])
    k, v = s["k"].float()[:, :, None], s["v"].float()[:, :, None]
    p = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(c["d"]))
    p = p.masked_fill(~see, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.reshape(c["B"], c["H"], c["Lq"], c["d"]).transpose(1, 2)
    return o.reshape(c["B"], c["Lq"], c["H"] * c["d"]).to(torch.bfloat16)


def run(state):
    s = state
    c = s["c"]
    op = c["op"]
    if not own:
        if op == "gate_add_norm":
            return _plain_gate_add_norm(s)
        return _plain_proj_i8(s) if op == "proj_i8" else _plain_cross_attention(s)
    ops = _ops()
    if op == "gate_add_norm":
        kinds = dict(none=ops.NORM_NONE, rms=ops.NORM_RMS, layer=ops.NORM_LAYER)
        outs = dict(bf16=ops.OUT_BF16, f32=ops.OUT_F32, i8=ops.OUT_I8)
        h = ops.gate_add_norm(s["x"], s["y"], y_norm=kinds[c["y_norm"]], y_weight=s["y_weight"], gate=s["gate"],
                              tanh_gate=c["tanh"], x_norm=kinds[c["x_norm"]], x_weight=s["x_weight"],
                              scale=s["scale"], shift=s["shift"], rows_per_sample=s["per"], eps=1e-6,
                              x_out=s["x_out"], out_type=outs[c["out"]])
        if c["out"] == "i8":
            q, scale = h
            values = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
            torch.mul(q, scale[:, None], out=values)
            return dict(x=s["x_out"], h=values, h_scale=scale)
        return dict(x=s["x_out"], h=h)
    if op == "proj_i8":
        acts = dict(none=ops.ACT_NONE, silu=ops.ACT_SILU, gelu_tanh=ops.ACT_GELU_TANH)
        q, scale = ops.quantize_rows(s["x"])
        return ops.proj_i8(q, scale, s["w"], s["w_scale"], bias=s["bias"], act=acts[c["act"]], out_f32=c["out_f32"])
    return ops.cross_attention(s["q"], s["k"], s["v"], key_len=s["key_len"], key_mask=s["key_mask"])


# ------------------------------------------------------------------------------------------------------- what it takes

def work(case):
    c = case
    if c["op"] == "gate_add_norm":
        e = c["rows"] * c["n"]
        out = {"bf16": 2, "f32": 4, "i8": 1}[c["out"]]
        vectors = c["n"] * (1 + (c["y_norm"] != "none") + _samples(c)[0] * (1 + 2 * c["mod"]))
        return dict(bytes=e * (4 + 4 + (4 if c["y_f32"] else 2) + out) + 4 * vectors, flops=12 * e)
    if c["op"] == "proj_i8":
        M, N, K = c["M"], c["N"], c["K"]
        moved = M * K * (4 if c["x_f32"] else 2) + N * K + M * N * (4 if c["out_f32"] else 2) + 4 * N * (1 + c["bias"])
        return dict(bytes=moved, flops=2 * M * N * K)
    lens = _lens(c)
    keys = sum(lens)
    seen = 0.9 * keys if c["mask"] else keys
    q = c["H"] * c["Lq"] * c["d"]  # of one sample; a sample without keys needs only its zeros written
    moved = q * (sum(n > 0 for n in lens) + c["B"]) + 2 * c["Hkv"] * c["d"] * seen
    return dict(bytes=2 * moved + c["B"] * 4 * (c["lens"] != "full") + keys * c["mask"],
                flops=4 * q * seen)


# ------------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    c, s = case, prepare(case, seed)
    D = torch.float64

    def quant64(t):  # the step is an fp32 number by definition
        step = (t.abs().max(dim=1, keepdim=True).values / 127).float().to(D)
        return torch.nan_to_num(t / step).round(), step

    if c["op"] == "gate_add_norm":
        def standard(t, kind):
            if kind == "rms":
                return t / ((t * t).sum(1, keepdim=True) / c["n"] + 1e-6).sqrt()
            if kind == "layer":
                mean = t.sum(1, keepdim=True) / c["n"]
                return (t - mean) / (((t - mean) ** 2).sum(1, keepdim=True) / c["n"] + 1e-6).sqrt()
            return t

        at = torch.arange(c["rows"], device="cuda") // s["per"]
        y = standard(s["y"].to(D), c["y_norm"])
        if c["y_norm"] != "none":
            y = y * s["y_weight"].to(D)
        gate = s["gate"].to(D)[at]
        x = s["x"].to(D) + (gate.tanh() if c["tanh"] else gate) * y
        h = standard(x, c["x_norm"]) * s["x_weight"].to(D)
        if c["mod"]:
            h = h + h * s["scale"].to(D)[at] + s["shift"].to(D)[at]
        if c["out"] == "i8":
            q, step = quant64(h)
            return dict(x=x, h=q * step, h_scale=step.flatten())
        return dict(x=x, h=h)
    if c["op"] == "proj_i8":
        q, step = quant64(s["x"].to(D))
        y = (q @ s["w"].to(D).T) * (step * s["w_scale"].to(D)[None])
        if c["bias"]:
            y += s["bias"].to(D)
        if c["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif c["act"] == "gelu_tanh":
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        return y
    out = torch.zeros(c["B"], c["Lq"], c["H"], c["d"], dtype=D, device="cuda")
    group = c["H"] // c["Hkv"]
    for b in range(c["B"]):
        keys = torch.ones(c["Lk"], dtype=torch.bool, device="cuda")
        if c["mask"]:
            keys &= s["key_mask"][b]
        if c["lens"] == "ragged":
            keys[int(s["key_len"][b]):] = False
        if not bool(keys.any()):
            continue
        for h in range(c["H"]):
            k, v = (s[t][b, h // group][keys].to(D) for t in ("k", "v"))
            out[b, :, h] = torch.softmax(s["q"][b, h].to(D) @ k.T / c["d"] ** 0.5, -1) @ v
    return out.reshape(c["B"], c["Lq"], c["H"] * c["d"])
