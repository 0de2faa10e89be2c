"""The operators of a recurrent low-bit layer as a serving program calls them, through the public
entry points of ``matmulfreellmcpu_amd.Engine``, beside their plain forms in torch.

  norm  the residual's addition, the RMS norm and the next product's int8 codes with a scale a row
  w4    products with 4-bit weights that have a scale (and perhaps a zero point) per group of a row
  conv  the short causal convolution over each channel, with the inputs carried between calls
  scan  the selective state space scan, with its state carried between calls

The widths are the engine's own (hidden 1024, 2048 and 2560, intermediate 2816, 5632 and 6912,
vocabulary 32000), and odd ones. Activations have a few channels that are far larger than the
others; a scan's steps and decays are spread as such a layer starts out.

torch is imported before the engine's library so that both use one HIP runtime.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "int8": torch.int8}


def listed():
    return [
        # one token's row before a product, the smallest call
        dict(name="norm_f32_1x2048", kind="norm", type="f32", rows=1, cols=2048),
        # a prompt's rows in 16 bits at the widest model's width
        dict(name="norm_bf16_2048x2560", kind="norm", type="bf16", rows=2048, cols=2560),
        # one token through the MLP's gate and up matrix
        dict(name="w4_f32_1x2048x11264", kind="w4", type="f32", rows=1, K=2048, N=11264, group=128, zeros=False),
        # a serving step's int8 rows through the MLP's down matrix
        dict(name="w4_int8_24x6912x2560", kind="w4", type="int8", rows=24, K=6912, N=2560, group=64, zeros=True),
        # a ragged batch through a layer whose sizes fit no tile
        dict(name="w4_bf16_100x1031x1333", kind="w4", type="bf16", rows=100, K=1031, N=1333, group=32, zeros=True),
        # a prompt through the MLP's gate and up matrix
        dict(name="w4_f32_2048x2048x11264", kind="w4", type="f32", rows=2048, K=2048, N=11264, group=128, zeros=False),
        # a server's step: 64 streams of one token each
        dict(name="conv_f32_64_streams", kind="conv", type="f32", rows=64, seqs=64, D=2048, width=4),
        # ragged prompts prefilled together
        dict(name="conv_bf16_2500x5120", kind="conv", type="bf16", rows=2500, seqs=7, D=5120, width=4),
        # one stream's token
        dict(name="scan_f32_1_stream", kind="scan", type="f32", rows=1, seqs=1, D=2048, N=16),
        # a server's step: 64 streams of one token each
        dict(name="scan_bf16_64_streams", kind="scan", type="bf16", rows=64, seqs=64, D=5120, N=16),
        # one long prompt
        dict(name="scan_f32_2048x4096", kind="scan", type="f32", rows=2048, seqs=1, D=4096, N=16),
        # ragged prompts of an odd width with a large state
        dict(name="scan_bf16_1000x1111", kind="scan", type="bf16", rows=1000, seqs=5, D=1111, N=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "w4", "w4", "conv", "scan", "scan"])
    kind_of = rng.choice(["f32", "bf16", "f16"])
    if kind == "norm":
        return dict(kind=kind, type=kind_of, rows=_log(rng, 1, 4096), cols=_log(rng, 64, 8192))
    if kind == "w4":
        K, N = _log(rng, 64, 6912), _log(rng, 64, 16384)
        most = min(2048, 2048 * 2048 * 11264 // (K * N))
        return dict(kind=kind, type=rng.choice(["f32", "bf16", "f16", "int8"]), rows=_log(rng, 1, most), K=K, N=N,
                    group=rng.choice([32, 64, 128, 0]), zeros=rng.random() < 0.5)
    seqs = _log(rng, 1, 64)
    rows = seqs if rng.random() < 0.3 else seqs * _log(rng, 1, 2048) + rng.randint(0, 3)
    if kind == "conv":
        D = _log(rng, 64, 5120)
        rows = max(seqs, min(rows, 2500 * 5120 // D))
        return dict(kind=kind, type=kind_of, rows=rows, seqs=seqs, D=D, width=rng.randint(2, 5))
    N, D = rng.choice([4, 8, 16, 16, 16, 24, 64]), _log(rng, 64, 5120)
    rows = max(seqs, min(rows, 2048, 2048 * 4096 * 16 // (D * N)))
    return dict(kind=kind, type=kind_of, rows=rows, seqs=seqs, D=D, N=N)


def _lens(case):
    """The case's sequence lengths: one row each where rows == seqs, else cut at places of their own."""
    rows, seqs = case["rows"], case["seqs"]
    if rows == seqs:
        return [1] * seqs
    cuts = sorted(random.Random(rows * 1000 + seqs).sample(range(1, rows), seqs - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [rows])]


def _groups(case):
    """(group size, groups of a row): group 0 is the whole row."""
    g = case["group"] or case["K"]
    return g, -(-case["K"] // g)


# ---- inputs ---------------------------------------------------------------------------------


class State:
    pass


def _inputs(case, seed):
    """The case's inputs on the GPU, by name."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t, kind = {}, TYPES[case["type"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    def activations(rows, cols):  # a few channels are far larger than the others
        return randn(rows, cols) * (1.0 + 15.0 * (uniform(cols) < 0.004))

    if case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        t["x"], t["res"] = (randn(rows, cols) * 0.5).to(kind), (activations(rows, cols) * 2.0).to(kind)
        t["w"] = 1.0 + 0.1 * randn(cols)
    elif case["kind"] == "w4":
        rows, K, N = case["rows"], case["K"], case["N"]
        size, n = _groups(case)
        # codes as a quantiser leaves them: bell-shaped around the zero point
        t["zeros"] = (8.0 + 1.5 * randn(N, n)).round().clamp(0, 15).to(torch.uint8) if case["zeros"] else None
        at = t["zeros"][:, torch.arange(K, device="cuda") // size].float() if case["zeros"] else 8.0
        q = (at + 2.7 * randn(N, K)).round().clamp(0, 15).to(torch.uint8)
        if K % 2:
            q = torch.cat([q, q.new_zeros(N, 1)], 1)
        t["codes"] = q[:, 0::2] | (q[:, 1::2] << 4)  # two a byte, the even column's in the low half
        t["scales"] = (0.02 / 2.7 * (0.7 + 0.6 * uniform(N, n))).to(torch.float16)
        if kind == torch.int8:
            t["x"] = (activations(rows, K) * 24.0).round().clamp(-127, 127).to(kind)
            t["xs"] = 0.02 + 0.03 * uniform(rows)
        else:
            t["x"] = activations(rows, K).to(kind)
    elif case["kind"] == "conv":
        rows, D, W = case["rows"], case["D"], case["width"]
        t["xz"] = activations(rows, 2 * D).to(kind)  # one projection's output: the inputs and the gates
        t["w"], t["bias"] = randn(D, W) / math.sqrt(W), 0.1 * randn(D)
        t["state"] = activations(case["seqs"], (W - 1) * D).to(kind).float().reshape(case["seqs"], W - 1, D)
    else:
        rows, D, N = case["rows"], case["D"], case["N"]
        t["u"] = torch.nn.functional.silu(activations(rows, D)).to(kind)
        t["xz"] = randn(rows, 2 * D).to(kind)  # the gates are its second half
        t["R"] = D // 16
        t["proj"] = randn(rows, t["R"] + 2 * N).to(kind)  # one projection's output: dt's inputs, B, C
        t["dt"] = (0.7 * randn(rows, D)).to(kind)
        step = torch.exp(math.log(1e-3) + uniform(D) * math.log(100.0))  # steps between 0.001 and 0.1
        t["dt_bias"] = step + torch.log(-torch.expm1(-step))
        t["A"] = -torch.arange(1, N + 1, device="cuda") * torch.exp(0.1 * randn(D, N))
        t["skip"] = 1.0 + 0.1 * randn(D)
        t["state"] = 0.3 * randn(case["seqs"], N, D)
    return t


def prepare(case, seed):
    s = State()
    s.case, s.kind, t = case, case["kind"], _inputs(case, seed)
    s.__dict__.update(t)
    rows = case["rows"]

    def new(*shape, dtype=torch.float32):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    if own:
        import matmulfreellmcpu_amd as mmf
        s.eng = mmf.Engine(0)
        s.type = {"f32": mmf.F32, "bf16": mmf.BF16, "f16": mmf.F16, "int8": mmf.I8}[case["type"]]
        s.stream = torch.cuda.ExternalStream(s.eng.stream)  # the engine has a stream of its own
        if s.kind == "norm":
            s.h, s.codes, s.scales = torch.empty_like(s.x), new(*s.x.shape, dtype=torch.int8), new(rows)
            s.values = new(*s.x.shape)
        elif s.kind == "w4":  # the weights are laid out once, from the file's arrays
            s.w4 = s.eng.register_w4(s.codes.cpu().numpy(), s.scales.cpu().numpy(),
                                     None if s.zeros is None else s.zeros.cpu().numpy(), K=case["K"],
                                     group=case["group"])
            s.out_type = mmf.F32 if case["type"] == "int8" else s.type
            s.out = new(rows, case["N"], dtype=torch.float32 if case["type"] == "int8" else s.x.dtype)
        else:
            s.out = new(rows, case["D"], dtype=TYPES[case["type"]])
    if s.kind in ("conv", "scan"):
        s.lens = _lens(case)
        s.x, s.z = s.xz[:, :case["D"]], s.xz[:, case["D"]:]
    if s.kind == "scan":
        s.B, s.C = s.proj[:, s.R:s.R + case["N"]], s.proj[:, s.R + case["N"]:]
    torch.cuda.synchronize()
    return s


# ---- one pass -------------------------------------------------------------------------------


def run(s):
    c = s.case
    if own:
        e = s.eng
        if s.kind == "norm":
            e.add_rmsnorm_q8(s.codes, s.scales, s.x, s.w, c["rows"], c["cols"], res=s.res, h=s.h, eps=EPS, dtype=s.type)
            with torch.cuda.stream(s.stream):  # the values that the codes stand for
                torch.mul(s.codes, s.scales[:, None], out=s.values)
            return {"h": s.h, "values": s.values, "scales": s.scales}
        if s.kind == "w4":
            e.w4_linear(s.w4, s.x, s.out, c["rows"], dtype=s.type, out_dtype=s.out_type,
                        scales=s.xs if c["type"] == "int8" else None)
            return {"out": s.out}
        if s.kind == "conv":
            e.short_conv(s.out, s.x, s.w, c["rows"], c["D"], c["width"], bias=s.bias, state=s.state, lens=s.lens,
                         silu=True, dtype=s.type, ldx=2 * c["D"])
            return {"out": s.out, "state": s.state}
        e.selective_scan(s.out, s.u, s.dt, s.A, s.B, s.C, c["rows"], c["D"], c["N"], skip=s.skip, z=s.z,
                         dt_bias=s.dt_bias, state=s.state, lens=s.lens, softplus=True, dtype=s.type,
                         ldb=s.proj.shape[1], ldc=s.proj.shape[1], ldz=2 * c["D"])
        return {"out": s.out, "state": s.state}
    return {"norm": _plain_norm, "w4": _plain_w4, "conv": _plain_conv, "scan": _plain_scan}[s.kind](s)


# ---- the plain forms ------------------------------------------------------------------------


def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _plain_norm(s):
    """The codes are taken in 64 bits: a value between two codes goes by its last bits."""
    h = s.x.float() + s.res.float()
    y = h.double()
    y = y / torch.sqrt((y * y).mean(1, keepdim=True) + EPS) * s.w.double()
    top = y.abs().amax(1, keepdim=True).clamp(min=1e-5)
    codes = torch.round(y * (127.0 / top))
    scales = (top / 127.0).float()
    return {"h": h.to(s.x.dtype), "values": codes.float() * scales, "scales": scales[:, 0]}


def _plain_w4(s):
    c = s.case
    size, n = _groups(c)
    q = torch.stack([s.codes & 15, s.codes >> 4], 2).reshape(c["N"], -1)[:, :c["K"]].float()
    at = torch.arange(c["K"], device="cuda") // size
    w = (q - (s.zeros.float()[:, at] if c["zeros"] else 8.0)) * s.scales.float()[:, at]
    out = s.x.float() @ w.t()
    return {"out": out * s.xs[:, None] if c["type"] == "int8" else out.to(s.x.dtype)}


def _places(s):
    """(sequence, place in it) of each packed row, the sequences' lengths and first rows."""
    lens = torch.tensor(s.lens, device="cuda")
    first = torch.cumsum(lens, 0) - lens
    seq = torch.repeat_interleave(torch.arange(len(s.lens), device="cuda"), lens, output_size=s.case["rows"])
    return seq, torch.arange(s.case["rows"], device="cuda") - first[seq], lens, first


def _plain_conv(s):
    c = s.case
    W, D = c["width"], c["D"]
    seq, place, lens, first = _places(s)
    x = torch.cat([s.state.reshape(-1, D), s.x.float()])  # the carried inputs of all sequences, then the rows
    base = len(s.lens) * (W - 1)

    def row(seq, place):  # where a sequence's input of this place stands: places below 0 are carried ones
        return torch.where(place < 0, seq * (W - 1) + place + W - 1, base + first[seq] + place)

    taps = torch.arange(W, device="cuda")
    at = row(seq[:, None], place[:, None] + taps - (W - 1))
    out = (x[at] * s.w.t()).sum(1) + s.bias
    every = torch.arange(len(s.lens), device="cuda")[:, None]
    s.state.copy_(x[row(every, lens[:, None] + taps[:W - 1] - (W - 1))])
    return {"out": _silu(out).to(s.x.dtype), "state": s.state}


def _plain_scan(s):
    """h_t = a_t h_(t-1) + b_t over all rows at once, by doubling: after the pass of step k, (a, b) of a
    row stand for the last 2k steps up to it. A sequence's first row takes its carried state and a = 0."""
    D, N = s.case["D"], s.case["N"]
    seq, place, lens, first = _places(s)
    u, dt = s.u.float(), s.dt.float() + s.dt_bias
    dt = dt.clamp(min=0) + torch.log1p(torch.exp(-dt.abs()))
    a = torch.exp(dt[:, None] * s.A.t())  # [rows, N, D]
    b = (dt * u)[:, None] * s.B.float()[:, :, None]
    b[first] += a[first] * s.state
    a[first] = 0
    k = 1
    while k < max(s.lens):
        b[k:] += a[k:] * b[:-k].clone()
        a[k:] *= a[:-k].clone()
        k *= 2
    y = (b * s.C.float()[:, :, None]).sum(1) + s.skip * u
    s.state.copy_(b[first + lens - 1])
    return {"out": (y * _silu(s.z.float())).to(s.u.dtype), "state": s.state}


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    """Inputs and outputs once, at the bytes that their types have; 4-bit weights at half a byte. A
    scan's step is counted as 7 operations a state element: the decay, its exponential, the update and the sum."""
    r, b = case["rows"], {"f32": 4, "bf16": 2, "f16": 2, "int8": 1}[case["type"]]
    if case["kind"] == "norm":  # x, the residual, h | the values, the scales, w
        return {"bytes": r * case["cols"] * (3.0 * b + 4.0) + 4.0 * (r + case["cols"]), "flops": 10.0 * r * case["cols"]}
    if case["kind"] == "w4":
        K, N, n = case["K"], case["N"], _groups(case)[1]
        weights = N * K / 2 + N * n * (2.5 if case["zeros"] else 2.0)
        rows = r * K * b + r * N * (4 if b == 1 else b) + (4 * r if b == 1 else 0)
        return {"bytes": weights + rows, "flops": 2.0 * r * K * N}
    D, seqs = case["D"], case["seqs"]
    if case["kind"] == "conv":
        W = case["width"]
        return {"bytes": 2.0 * b * r * D + 8.0 * seqs * (W - 1) * D + 4.0 * D * (W + 1), "flops": (2.0 * W + 5) * r * D}
    N = case["N"]
    return {"bytes": 4.0 * b * r * D + 2.0 * b * r * N + 8.0 * seqs * N * D + 4.0 * D * (N + 2),
            "flops": (7.0 * N + 12) * r * D}


# ---- the same in 64 bits --------------------------------------------------------------------


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "norm":
        h = t["x"].double() + t["res"].double()
        y = torch.nn.functional.rms_norm(h, h.shape[1:], t["w"].double(), EPS)
        scales = torch.clamp(torch.linalg.vector_norm(y, float("inf"), dim=1), min=1e-5) / 127
        return {"h": h, "values": torch.round(y / scales[:, None]) * scales[:, None], "scales": scales}
    if case["kind"] == "w4":
        K, N = case["K"], case["N"]
        size, n = _groups(case)
        q = torch.empty(N, 2 * t["codes"].shape[1], dtype=torch.float64, device="cuda")
        q[:, 0::2], q[:, 1::2] = t["codes"] % 16, t["codes"] // 16
        x = t["x"].double()
        out = torch.zeros(x.shape[0], N, dtype=torch.float64, device="cuda")
        for g in range(n):  # group by group, the scale after the sum
            k = slice(g * size, min(K, (g + 1) * size))
            z = t["zeros"][:, g].double() if case["zeros"] else 8.0
            out += (x[:, k] @ q[:, k].t() - x[:, k].sum(1, keepdim=True) * z) * t["scales"][:, g].double()
        return {"out": out * t["xs"].double()[:, None] if case["type"] == "int8" else out}
    D, lens, out, states = case["D"], _lens(case), [], []
    if case["kind"] == "conv":
        x, w, W = t["xz"][:, :D].double(), t["w"].double(), case["width"]
        for state, rows in zip(t["state"].double(), torch.split(x, lens)):
            ext = torch.cat([state, rows])
            y = (ext.unfold(0, W, 1) * w).sum(-1) + t["bias"].double()
            out.append(y * torch.sigmoid(y))
            states.append(ext[ext.shape[0] - (W - 1):])
        return {"out": torch.cat(out), "state": torch.stack(states)}
    N, R = case["N"], t["R"]
    u, z = t["u"].double(), t["xz"][:, D:].double()
    B, C = t["proj"][:, R:R + N].double(), t["proj"][:, R + N:].double()
    dt = torch.logaddexp(t["dt"].double() + t["dt_bias"].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    A, h, y = t["A"].double().t(), t["state"].double(), torch.empty_like(u)
    first = np.cumsum(lens) - lens
    for p in range(max(lens)):  # step by step, all sequences that are still running together
        live = [i for i, n in enumerate(lens) if n > p]
        r = torch.as_tensor([int(first[i]) + p for i in live], device="cuda")
        at = torch.as_tensor(live, device="cuda")
        h[at] = torch.exp(dt[r][:, None] * A) * h[at] + (dt[r] * u[r])[:, None] * B[r][:, :, None]
        y[r] = (h[at] * C[r][:, :, None]).sum(1)
    return {"out": (y + t["skip"].double() * u) * z * torch.sigmoid(z), "state": h}
