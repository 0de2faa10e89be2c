"""Operators of a layer with 8-bit weights and linear attention, and of what its logits say, as a serving
program calls them through the public entry points of ``matmulfreellmcpu_amd.Engine``, beside their plain
forms in torch.

  w8        products of int8 rows, with a scale a row, and int8 weights, with a scale an output channel
  attention linear attention with a decay for each head, its state carried between calls
  block     a block's output through its norm, gate and residual scale onto the residual, then the next
            block's norm with its int8 codes
  logprobs  log probabilities of given tokens, the distribution's entropy and its most likely tokens

The widths are the engine's own (hidden 1024, 2048 and 2560 as heads of 128, intermediate 2816, 5632 and
6912, vocabulary 32000), and odd ones. Activations have a few channels that are far larger than the others;
decays reach from a few rows to thousands.

torch is imported before the engine's library so that both use one HIP runtime.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token through the MLP's gate and up matrix, the smallest of the products
        dict(name="w8_bf16_1x2048x11264", kind="w8", type="bf16", rows=1, K=2048, N=11264, bias=False),
        # a serving step's rows through the MLP's down matrix
        dict(name="w8_f32_24x6912x2560", kind="w8", type="f32", rows=24, K=6912, N=2560, bias=True),
        # a ragged batch through a layer whose sizes fit no tile
        dict(name="w8_f16_100x1031x1333", kind="w8", type="f16", rows=100, K=1031, N=1333, bias=True),
        # a prompt through the MLP's gate and up matrix
        dict(name="w8_bf16_2048x2048x11264", kind="w8", type="bf16", rows=2048, K=2048, N=11264, bias=False),
        # one stream's token
        dict(name="attention_f32_1_stream", kind="attention", type="f32", rows=1, seqs=1, H=16, q=16, k=16, v=16,
             Dk=128, Dv=128, gates=False),
        # a server's step: 64 streams of one token each
        dict(name="attention_bf16_64_streams", kind="attention", type="bf16", rows=64, seqs=64, H=20, q=20, k=20, v=20,
             Dk=128, Dv=128, gates=True),
        # one long prompt
        dict(name="attention_bf16_2048x2048", kind="attention", type="bf16", rows=2048, seqs=1, H=16, q=16, k=16, v=16,
             Dk=128, Dv=128, gates=True),
        # ragged prompts of odd heads that share their queries and keys
        dict(name="attention_f32_1000x777", kind="attention", type="f32", rows=1000, seqs=5, H=7, q=1, k=1, v=7,
             Dk=72, Dv=111, gates=True),
        # one token's row between two blocks, the smallest call
        dict(name="block_f32_1x2048", kind="block", type="f32", rows=1, cols=2048, gate="none", post=True, pre=True),
        # a prompt's rows in 16 bits at the widest model's width
        dict(name="block_bf16_2048x2560", kind="block", type="bf16", rows=2048, cols=2560, gate="silu", post=True, pre=True),
        # the next token's distribution
        dict(name="logprobs_f32_1x32000", kind="logprobs", type="f32", rows=1, V=32000, top=20, temperature=1.0),
        # a prompt's tokens scored
        dict(name="logprobs_bf16_2048x32000", kind="logprobs", type="bf16", rows=2048, V=32000, top=5, temperature=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["w8", "w8", "attention", "attention", "block", "logprobs"])
    kind_of = rng.choice(["f32", "bf16", "f16"])
    if kind == "w8":
        K, N = _log(rng, 64, 6912), _log(rng, 64, 16384)
        most = min(2048, 2048 * 2048 * 11264 // (K * N))
        return dict(kind=kind, type=kind_of, rows=_log(rng, 1, most), K=K, N=N, bias=rng.random() < 0.5)
    if kind == "block":
        return dict(kind=kind, type=kind_of, rows=_log(rng, 1, 2048), cols=_log(rng, 64, 8192),
                    gate=rng.choice(["none", "plain", "sigmoid", "silu"]), post=rng.random() < 0.8, pre=rng.random() < 0.8)
    if kind == "logprobs":
        V = _log(rng, 256, 200000)
        return dict(kind=kind, type=kind_of, rows=_log(rng, 1, min(2048, 32_000_000 // V)), V=V, top=rng.randint(0, 20),
                    temperature=rng.choice([1.0, 1.0, 0.7, 1.5]))
    seqs = _log(rng, 1, 64)
    rows = seqs if rng.random() < 0.3 else seqs * _log(rng, 1, 2048) + rng.randint(0, 3)
    H = rng.choice([1, 2, 4, 7, 8, 12, 16, 16])
    share = lambda: rng.choice([H, H, H, 1])  # noqa: E731  (heads of a tensor: its own, or one for all)
    Dk, Dv = rng.choice([64, 128, 128, _log(rng, 16, 256)]), rng.choice([64, 128, 128, _log(rng, 16, 256)])
    rows = max(seqs, min(rows, 2048, 2048 * 16 * 128 * 128 // (H * Dk * Dv)))
    return dict(kind=kind, type=kind_of, rows=rows, seqs=seqs, H=H, q=share(), k=share(), v=share(), Dk=Dk, Dv=Dv,
                gates=rng.random() < 0.5)


def _lens(case):
    """The case's sequence lengths: one row each where rows == seqs, else cut at places of their own."""
    rows, seqs = case["rows"], case["seqs"]
    if rows == seqs:
        return [1] * seqs
    cuts = sorted(random.Random(rows * 1000 + seqs).sample(range(1, rows), seqs - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [rows])]


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

    if case["kind"] == "w8":
        rows, K, N = case["rows"], case["K"], case["N"]
        t["codes"] = (randn(N, K) * 33.0).round().clamp(-127, 127).to(torch.int8)  # bell-shaped, as a quantiser leaves them
        t["ws"] = (0.02 / 33.0) * (0.7 + 0.6 * uniform(N))
        t["x"] = (activations(rows, K) * 24.0).round().clamp(-127, 127).to(torch.int8)
        t["xs"] = 0.02 + 0.03 * uniform(rows)
        t["bias"] = 0.1 * randn(N) if case["bias"] else None
    elif case["kind"] == "attention":
        rows, H, Dk, Dv = case["rows"], case["H"], case["Dk"], case["Dv"]
        nq, nk, nv = case["q"] * Dk, case["k"] * Dk, case["v"] * Dv
        t["qkv"] = randn(rows, nq + nk + nv).to(kind)  # one projection's output: queries, keys, values
        t["q"], t["k"], t["v"] = t["qkv"][:, :nq], t["qkv"][:, nq:nq + nk], t["qkv"][:, nq + nk:]
        t["decay"] = torch.log1p(-torch.exp2(-2.0 - 8.0 * uniform(H)))  # heads that forget over 4 rows, and over 1024
        t["gates"] = torch.nn.functional.logsigmoid(3.0 + randn(rows, H)) if case["gates"] else None
        t["state"] = 3.0 * randn(case["seqs"], H, Dk, Dv)
        t["scale"] = Dk ** -0.5
    elif case["kind"] == "block":
        rows, cols = case["rows"], case["cols"]
        t["b"], t["x"] = (randn(rows, cols) * 0.5).to(kind), (activations(rows, cols) * 2.0).to(kind)
        t["gate"] = randn(rows, cols).to(kind) if case["gate"] != "none" else None
        t["post"] = 1.0 + 0.1 * randn(cols) if case["post"] else None
        t["pre"] = 1.0 + 0.1 * randn(cols) if case["pre"] else None
        t["channels"] = 0.5 + 0.05 * randn(cols)  # the residual scale of each channel
        t["scale"] = 0.7
    else:
        rows, V = case["rows"], case["V"]
        x = 2.5 * randn(rows, V) - 1.5 * torch.log1p(torch.arange(V, device="cuda") / 50.0)  # frequent tokens stand first
        x[::3] = torch.where(uniform(V) < 0.02, float("-inf"), x[::3])  # rows with tokens that may not come
        x[:, V // 3] = x[:, V // 3].clamp(min=-20.0)
        t["x"] = x.to(kind)
        p = t["x"].float() - torch.log(-torch.log(uniform(rows, V).clamp(1e-7, 1.0 - 1e-7)))
        t["ids"] = p.argmax(1)  # tokens drawn from the distribution
    return t


def prepare(case, seed):
    s = State()
    s.case, s.kind, t = case, case["kind"], _inputs(case, seed)
    s.__dict__.update(t)
    rows = case["rows"]

    def new(*shape, dtype=torch.float32):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    if s.kind == "attention":
        s.lens = _lens(case)
    if own:
        import matmulfreellmcpu_amd as mmf
        s.eng = mmf.Engine(0)
        s.stream = torch.cuda.ExternalStream(s.eng.stream)  # the engine has a stream of its own
        kind = TYPES[case["type"]]
        if s.kind == "w8":  # the weights are laid out once, from the file's arrays
            s.w8 = s.eng.register_w8(s.codes.cpu().numpy(), s.ws.cpu().numpy())
            s.out = new(rows, case["N"], dtype=kind)
        elif s.kind == "attention":
            s.out = new(rows, case["H"] * case["Dv"], dtype=kind)
        elif s.kind == "block":
            s.act = {"none": mmf.ACT_NONE, "plain": mmf.ACT_NONE, "sigmoid": mmf.ACT_SIGMOID, "silu": mmf.ACT_SILU}[case["gate"]]
            s.h, s.codes, s.scales = torch.empty_like(s.x), new(rows, case["cols"], dtype=torch.int8), new(rows)
            s.values = new(rows, case["cols"])
        else:
            s.logprobs, s.entropy = new(rows), new(rows)
            s.top_ids = new(rows, case["top"], dtype=torch.int64)
            s.top_logprobs = new(rows, case["top"])
    torch.cuda.synchronize()
    return s


# ---- one pass -------------------------------------------------------------------------------


def run(s):
    c = s.case
    if own:
        e = s.eng
        if s.kind == "w8":
            e.w8_linear(s.w8, s.x, s.xs, s.out, c["rows"], bias=s.bias)
            return {"out": s.out}
        if s.kind == "attention":
            n = s.qkv.shape[1]
            e.decay_attention(s.out, s.q, s.k, s.v, c["rows"], c["H"], c["Dk"], c["Dv"], decay=s.decay, gates=s.gates,
                              state=s.state, lens=s.lens, q_heads=c["q"], k_heads=c["k"], v_heads=c["v"], scale=s.scale,
                              ldq=n, ldk=n, ldv=n)
            return {"out": s.out, "state": s.state}
        if s.kind == "block":
            e.block_norm_q8(s.codes, s.scales, s.b, c["rows"], c["cols"], x=s.x, gate=s.gate, act=s.act, w_post=s.post,
                            w_pre=s.pre, channels=s.channels, scale=s.scale, h=s.h, eps=EPS)
            with torch.cuda.stream(s.stream):  # the values that the codes stand for
                torch.mul(s.codes, s.scales[:, None], out=s.values)
            return {"h": s.h, "values": s.values, "scales": s.scales}
        e.token_logprobs(s.x, c["rows"], c["V"], ids=s.ids, logprobs=s.logprobs, entropy=s.entropy, top=c["top"],
                         top_ids=s.top_ids, top_logprobs=s.top_logprobs, temperature=c["temperature"])
        return {"logprobs": s.logprobs, "entropy": s.entropy, "top_ids": s.top_ids, "top_logprobs": s.top_logprobs}
    return {"w8": _plain_w8, "attention": _plain_attention, "block": _plain_block, "logprobs": _plain_logprobs}[s.kind](s)


# ---- the plain forms ------------------------------------------------------------------------


def _plain_w8(s):
    out = (s.x.float() @ s.codes.float().t()) * s.xs[:, None] * s.ws
    return {"out": (out + s.bias if s.case["bias"] else out).to(TYPES[s.case["type"]])}


def _plain_attention(s):
    """All pairs of rows at once. Log decays are summed in 64 bits: what counts are differences of long sums."""
    c = s.case
    H, Dk, Dv, rows, seqs = c["H"], c["Dk"], c["Dv"], c["rows"], c["seqs"]
    lens = torch.tensor(s.lens, device="cuda")
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), lens, output_size=rows)
    first = torch.cumsum(lens, 0) - lens

    def heads(x, n, D):  # [H, rows, D]
        return x.float().reshape(rows, n, D).repeat_interleave(H // n, 1).transpose(0, 1).contiguous()

    q, k, v = heads(s.q, c["q"], Dk) * s.scale, heads(s.k, c["k"], Dk), heads(s.v, c["v"], Dv)
    a = s.decay.double() + (s.gates.double() if c["gates"] else torch.zeros(rows, 1, device="cuda", dtype=torch.float64))
    up = torch.cumsum(a, 0)  # [rows, H]: up to each row
    before = up - a  # up to the row before
    start, end = before[first], up[first + lens - 1]
    at = torch.arange(rows, device="cuda")
    sees = (seq[:, None] == seq) & (at[:, None] >= at)
    g = up.t()
    w = torch.where(sees, torch.exp((g[:, :, None] - g[:, None, :]).clamp(max=0.0)).float(), 0.0)
    w *= q @ k.transpose(1, 2).contiguous()
    out = w @ v
    mine = (seq[:, None] == torch.arange(seqs, device="cuda")).float()  # [rows, seqs]
    since = torch.exp(up - start[seq]).float().t()  # [H, rows]
    till = torch.exp(end[seq] - up).float().t()
    state = s.state.transpose(0, 1).reshape(H, seqs * Dk, Dv)
    out += ((q * since[:, :, None])[:, :, None, :] * mine[None, :, :, None]).reshape(H, rows, seqs * Dk) @ state
    kept = ((k * till[:, :, None])[:, :, None, :] * mine[None, :, :, None]).reshape(H, rows, seqs * Dk)
    new = (kept.transpose(1, 2).contiguous() @ v).reshape(H, seqs, Dk, Dv).transpose(0, 1)
    s.state.copy_(s.state * torch.exp(end - start).float()[:, :, None, None] + new)
    return {"out": out.transpose(0, 1).reshape(rows, H * Dv).to(s.qkv.dtype), "state": s.state}


def _plain_block(s):
    """The codes are taken in 64 bits, of the sum in 32: a value between two codes goes by its last bits."""
    c = s.case
    p = s.b.double()
    if c["post"]:
        p = p / torch.sqrt((p * p).mean(1, keepdim=True) + EPS) * s.post.double()
    if c["gate"] != "none":
        g = s.gate.double()
        p = p * {"plain": lambda: g, "sigmoid": lambda: 1.0 / (1.0 + torch.exp(-g)), "silu": lambda: g / (1.0 + torch.exp(-g))}[c["gate"]]()
    h = (s.x.double() + p * s.channels.double() * np.float32(s.scale).item()).float()
    y = h.double()
    if c["pre"]:
        y = y / torch.sqrt((y * y).mean(1, keepdim=True) + EPS) * s.pre.double()
    top = y.abs().amax(1, keepdim=True).clamp(min=1e-5)
    codes = torch.round(y * (127.0 / top))
    scales = (top / 127.0).float()
    return {"h": h.to(s.b.dtype), "values": codes.float() * scales, "scales": scales[:, 0]}


def _plain_logprobs(s):
    c = s.case
    x = s.x.float()
    order = torch.sort(x, dim=1, descending=True, stable=True)  # equal ones by their index
    z = (x - order.values[:, :1]) * (1.0 / c["temperature"])
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    log = torch.log(total)
    entropy = log[:, 0] - (torch.where(e > 0, z, 0.0) * e).sum(1) / total[:, 0]
    lp = z - log
    ids = order.indices[:, :c["top"]].contiguous()
    return {"logprobs": lp.gather(1, s.ids[:, None])[:, 0], "entropy": entropy, "top_ids": ids, "top_logprobs": lp.gather(1, ids)}


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    """Inputs and outputs once, at the bytes that their types have. Attention's step is counted as the
    update of the state and the sum over it."""
    r, b = case["rows"], {"f32": 4, "bf16": 2, "f16": 2}[case["type"]]
    if case["kind"] == "w8":
        K, N = case["K"], case["N"]
        return {"bytes": N * K + r * K + b * r * N + 4.0 * (r + N * (2 if case["bias"] else 1)), "flops": 2.0 * r * K * N}
    if case["kind"] == "attention":
        H, Dk, Dv = case["H"], case["Dk"], case["Dv"]
        rows = b * r * (case["q"] * Dk + case["k"] * Dk + case["v"] * Dv + H * Dv) + (4.0 * r * H if case["gates"] else 0.0)
        return {"bytes": rows + 8.0 * case["seqs"] * H * Dk * Dv, "flops": 4.0 * r * H * Dk * Dv}
    if case["kind"] == "block":  # b, x, the gate, h | the values, the scales, the weights
        n = 3.0 + (case["gate"] != "none")
        return {"bytes": r * case["cols"] * (n * b + 4.0) + 4.0 * (r + 3 * case["cols"]), "flops": 25.0 * r * case["cols"]}
    return {"bytes": r * (float(b) * case["V"] + 16.0 + 12.0 * case["top"]), "flops": 6.0 * r * case["V"]}


# ---- the same in 64 bits --------------------------------------------------------------------


def exact(case, seed):
    t, r = _inputs(case, seed), case["rows"]
    if case["kind"] == "w8":
        out = torch.nn.functional.linear(t["x"].double() * t["xs"].double()[:, None],
                                         t["codes"].double() * t["ws"].double()[:, None])
        return {"out": out if t["bias"] is None else out + t["bias"].double()}
    if case["kind"] == "attention":  # step by step, all sequences that are still running together
        H, Dk, Dv, lens = case["H"], case["Dk"], case["Dv"], _lens(case)
        q, k, v = (torch.stack([t[n].double().reshape(r, case[n], D)[:, h * case[n] // H] for h in range(H)], 1)
                   for n, D in (("q", Dk), ("k", Dk), ("v", Dv)))
        keep = torch.exp(t["decay"].double().expand(r, H) + (t["gates"].double() if case["gates"] else 0.0))
        state, out = t["state"].double(), torch.empty(r, H, Dv, dtype=torch.float64, device="cuda")
        first = np.cumsum(lens) - lens
        for p in range(max(lens)):
            live = [i for i, n in enumerate(lens) if n > p]
            row = torch.as_tensor([int(first[i]) + p for i in live], device="cuda")
            at = torch.as_tensor(live, device="cuda")
            now = state[at] * keep[row][:, :, None, None] + k[row][:, :, :, None] * v[row][:, :, None, :]
            state[at] = now
            out[row] = (q[row][:, :, :, None] * now).sum(2) * t["scale"]
        return {"out": out.reshape(r, H * Dv), "state": state}
    if case["kind"] == "block":
        h = t["b"].double()
        if case["post"]:
            h = torch.nn.functional.rms_norm(h, h.shape[1:], t["post"].double(), EPS)
        if case["gate"] != "none":
            g = t["gate"].double()
            h = h * {"plain": torch.Tensor.clone, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu}[case["gate"]](g)
        h = t["x"].double() + h * t["channels"].double() * float(np.float32(t["scale"]))
        y = h.float().double()
        if case["pre"]:
            y = torch.nn.functional.rms_norm(y, y.shape[1:], t["pre"].double(), EPS)
        scales = torch.clamp(torch.linalg.vector_norm(y, float("inf"), dim=1), min=1e-5) / 127
        return {"h": h, "values": torch.round(y / scales[:, None]) * scales[:, None], "scales": scales}
    lp = torch.log_softmax(t["x"].double() / case["temperature"], 1)
    entropy = torch.special.entr(torch.exp(lp)).sum(1)
    ids = torch.argsort(t["x"], dim=1, descending=True, stable=True)[:, :case["top"]]
    return {"logprobs": lp[torch.arange(r, device="cuda"), t["ids"]], "entropy": entropy, "top_ids": ids,
            "top_logprobs": torch.take_along_dim(lp, ids, 1)}
