"""The operators of a quantised block together, as a program uses them: residual norms around a cross-attention branch and a
feed-forward branch whose projections are 8-bit integers, against the same block in 64 bits on the same integers; eager,
on a side stream and captured into a graph."""

import pytest

pytestmark = pytest.mark.gpu


def _block(cuda, B, N, S, D, H, F):
    import torch
    import mkimage

    ops, g = mkimage.ops, torch.Generator().manual_seed(B * N + S)

    def r(*s):
        return torch.randn(*s, generator=g).to(cuda)

    p = dict(B=B, N=N, S=S, D=D, H=H, F=F)
    for name, rows, cols in (("q", D, D), ("k", D, D), ("v", D, D), ("o", D, D), ("up", F, D), ("down", D, F)):
        p[name] = ops.quantize_rows(0.05 * r(rows, cols))
        p[name + "_b"] = 0.1 * r(rows)
    for name in ("w0", "w1", "w2", "w3", "w4"):
        p[name] = 1 + 0.1 * r(D)
    for name in ("g0", "g1", "sc0", "sc1"):
        p[name] = 0.3 * r(B, D)
    p["ctx"] = r(B * S, D).to(torch.bfloat16)
    p["lens"] = torch.tensor(([S, S // 2, 0] * B)[:B], dtype=torch.int32, device=cuda)
    return p, r(B * N, D)


def _run(p, x):
    """x is updated in place; returns the last norm's output."""
    import mkimage

    ops = mkimage.ops
    B, N, S, D, H = (p[k] for k in ("B", "N", "S", "D", "H"))
    d = D // H
    heads = lambda t, L: t.reshape(B, L, H, d).transpose(1, 2)  # noqa: E731
    a = ops.gate_add_norm(x, x_norm=ops.NORM_RMS, x_weight=p["w0"], scale=p["sc0"], rows_per_sample=N,
                          out_type=ops.OUT_I8)
    c = ops.quantize_rows(p["ctx"])
    q = ops.proj_i8(*a, *p["q"], bias=p["q_b"])
    k, v = (ops.proj_i8(*c, *p[n], bias=p[n + "_b"]) for n in "kv")
    o = ops.cross_attention(heads(q, N), heads(k, S), heads(v, S), key_len=p["lens"]).reshape(B * N, D)
    y = ops.proj_i8(*ops.quantize_rows(o), *p["o"], bias=p["o_b"])
    a = ops.gate_add_norm(x, y, y_norm=ops.NORM_RMS, y_weight=p["w1"], gate=p["g0"], tanh_gate=True,
                          x_norm=ops.NORM_RMS, x_weight=p["w2"], scale=p["sc1"], rows_per_sample=N, out_type=ops.OUT_I8)
    u = ops.proj_i8(*a, *p["up"], bias=p["up_b"], act=ops.ACT_GELU_TANH)
    y = ops.proj_i8(*ops.quantize_rows(u), *p["down"], bias=p["down_b"], out_f32=True)
    return ops.gate_add_norm(x, y, y_norm=ops.NORM_LAYER, y_weight=p["w3"], gate=p["g1"], x_norm=ops.NORM_RMS,
                             x_weight=p["w4"], rows_per_sample=N)


def _run64(p, x):
    import torch

    D64 = torch.float64
    B, N, S, D, H = (p[k] for k in ("B", "N", "S", "D", "H"))
    P = {k: t.to(D64) for k, t in p.items() if torch.is_tensor(t) and t.is_floating_point()}
    rms = lambda t: t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
    row = lambda t: t.repeat_interleave(N, 0)  # noqa: E731
    mat = lambda n: p[n][0].to(D64) * p[n][1].to(D64)[:, None]  # noqa: E731

    def quant(t):
        step = t.abs().amax(-1, keepdim=True) / 127
        return torch.nan_to_num((t / step).round() * step)

    lin = lambda t, n: quant(t) @ mat(n).T + P[n + "_b"]  # noqa: E731
    x = x.to(D64)
    heads = lambda t, L: t.reshape(B, L, H, D // H).transpose(1, 2)  # noqa: E731
    h = rms(x) * P["w0"] * (1 + row(P["sc0"]))
    q, k, v = heads(lin(h, "q"), N), heads(lin(P["ctx"], "k"), S), heads(lin(P["ctx"], "v"), S)
    s = q @ k.transpose(-1, -2) / (D // H) ** 0.5
    hide = torch.arange(S, device=x.device)[None] >= p["lens"][:, None]
    a = torch.nan_to_num(torch.softmax(s.masked_fill(hide[:, None, None], -torch.inf), -1))
    y = lin((a @ v).transpose(1, 2).reshape(B * N, D), "o")
    x = x + row(P["g0"]).tanh() * rms(y) * P["w1"]
    u = torch.nn.functional.gelu(lin(rms(x) * P["w2"] * (1 + row(P["sc1"])), "up"), approximate="tanh")
    y = lin(u, "down")
    y = (y - y.mean(-1, keepdim=True)) / (y.var(-1, unbiased=False, keepdim=True) + 1e-6).sqrt()
    x = x + row(P["g1"]) * y * P["w3"]
    return x, rms(x) * P["w4"]


@pytest.mark.parametrize("B,N,S,D,H,F", [(1, 1, 7, 256, 2, 512), (3, 100, 77, 640, 10, 2560), (2, 1024, 300, 1280, 10, 5120)])
def test_block(cuda, B, N, S, D, H, F):
    """bf16 and 8-bit roundings add up over the two branches: each is 2^-8 of its value or half a step of about 1/127 of
    a row's top (an rms error of 0.29 / 127 * 4 = 2^-6.8 of the row's rms for values that reach four deviations), five of
    them in a chain and as many of bf16: sqrt(5) * 2^-6.8 + sqrt(5) * 2^-9 < 0.03 relative in a branch that is about a
    third of the stream. Against the 64-bit block that quantises at the same places only the quotients that change sides
    of a border count, so 0.03 is far above what is left and far below a wrong operand."""
    import torch
    import mkimage

    p, x = _block(cuda, B, N, S, D, H, F)
    want_x, want_h = _run64(p, x)
    got_x = x.clone()
    got_h = _run(p, got_x)
    assert mkimage.ops.check_kernels() == 0
    for got, want in ((got_x, want_x), (got_h, want_h)):
        assert float((got.double() - want).norm() / want.norm()) < 0.03
    # A side stream, then a graph replayed on new contents of the same buffers: the same bits.
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x2 = x.clone()
        h2 = _run(p, x2)
    s.synchronize()
    assert torch.equal(x2, got_x) and torch.equal(h2, got_h)
    xg = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hg = _run(p, xg)
    for _ in range(2):
        xg.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(xg, got_x) and torch.equal(hg, got_h)


def test_first_calls_inside_a_capture(cuda, tmp_path):
    """A process whose first call of each operator is captured: nothing they set up for themselves breaks the capture."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import sys; sys.path.insert(0, {pkg!r})
import torch, mkimage
ops = mkimage.ops
x = torch.randn(200, 256, device="cuda"); w = torch.randint(-127, 128, (384, 256), device="cuda", dtype=torch.int8)
ws = torch.rand(384, device="cuda"); kv = torch.randn(2, 4, 77, 64, device="cuda").bfloat16()
q = torch.randn(2, 4, 300, 64, device="cuda").bfloat16()
def run():
    a = ops.gate_add_norm(x, out_type=ops.OUT_I8)
    return ops.proj_i8(*a, w, ws), ops.proj_i8(a[0][:2], a[1][:2], w, ws), ops.cross_attention(q, kv, kv), \\
        ops.cross_attention(q[:, :, :1], kv, kv), ops.quantize_rows(x)
g = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(g):
    a = run()
g.replay()
b = run()
torch.cuda.synchronize()
flat = lambda t: [v for e in t for v in (e if isinstance(e, tuple) else (e,))]
assert all(torch.equal(u, v) for u, v in zip(flat(a), flat(b)))
assert ops.check_kernels() == 0
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code.format(pkg=os.path.join(root, "mako-image_b200"))], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_two_streams_at_once(cuda):
    """Two blocks in flight on two streams at the same time: nothing is shared between the calls."""
    import torch

    cases = [_block(cuda, 2, 700, 77, 640, 10, 2560), _block(cuda, 1, 900, 333, 1280, 10, 2560)]
    want = []
    for p, x in cases:
        xi = x.clone()
        want.append((_run(p, xi), xi))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    xs = [[x.clone() for _ in range(8)] for _, x in cases]
    got = [[], []]
    torch.cuda.synchronize()
    for i in range(8):
        for j, (p, _) in enumerate(cases):
            with torch.cuda.stream(streams[j]):
                got[j].append(_run(p, xs[j][i]))
    torch.cuda.synchronize()
    for j in range(2):
        for i in range(8):
            assert torch.equal(got[j][i], want[j][0]) and torch.equal(xs[j][i], want[j][1])


def test_another_device_than_the_current_one(cuda):
    """Tensors of device 1 while device 0 is current (needs two GPUs), and a mix of devices is refused."""
    import torch
    import mkimage

    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    p, x = _block(torch.device("cuda:1"), 1, 300, 77, 256, 2, 512)
    a = x.clone()
    h = _run(p, a)
    with torch.cuda.device(1):
        b = x.clone()
        assert torch.equal(_run(p, b), h) and torch.equal(a, b)
    with pytest.raises(mkimage.MkbError):
        mkimage.ops.quantize_rows(x, scale=torch.empty(300, device="cuda:0"))


def test_a_call_for_another_device_is_made_again_there(cuda, monkeypatch):
    """With the current device reported as another one at first, each operator runs once more under the tensors' device and
    gives what it gives otherwise."""
    import torch
    import mkimage

    ops = mkimage.ops
    g = torch.Generator().manual_seed(5)
    x = torch.randn(20, 64, generator=g).to(cuda)
    y = torch.randn(20, 64, generator=g).to(cuda).to(torch.bfloat16)
    q = torch.randn(2, 3, 20, 64, generator=g).to(cuda).to(torch.bfloat16)
    lens = torch.tensor([20, 7], dtype=torch.int32, device=cuda)

    def all_of_them():
        i8, step = ops.quantize_rows(x)
        x_out = torch.empty_like(x)
        n8, n_step = ops.gate_add_norm(x, y, y_norm=ops.NORM_RMS, gate=x[:1], x_norm=ops.NORM_LAYER, scale=x[:1], shift=x[:1],
                                       x_out=x_out, out_type=ops.OUT_I8)
        return [i8, step, x_out, n8, n_step, ops.proj_i8(i8, step, n8, n_step, bias=step, out_f32=True),
                ops.cross_attention(q, q, q, key_len=lens, scale=0.2)]

    want = all_of_them()
    real, calls = ops._current_device, []
    monkeypatch.setattr(ops, "_current_device", lambda: calls.append(1) or (real() if len(calls) % 2 == 0 else real() + 1))
    got = all_of_them()
    assert len(calls) == 8
    assert all(torch.equal(a, b) for a, b in zip(want, got))
