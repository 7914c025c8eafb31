"""Cases for the operators that keep activations in 8 bits between the forward and the backward pass.

An 8-bit activation is a pair: `q`, e4m3 values [rows][D], and `scale`, one power of two per row and block of 32 columns,
held as the byte of its exponent (2^(byte - 127)).  The exponent k of a block is the smallest whole number with
amax <= 448 * 2^k, in [-117, 119], so no value saturates and every value is exact in BF16.

    add_norm    residual add + RMSNorm, the normalised rows also in 8 bits            (forward)
    norm_bwd    the norm's input gradient from those 8 bits, added to the residual's  (backward)
    store, load any BF16 activation into 8 bits and back
    swiglu_fwd  silu(gate) * up, gate and up also in 8 bits                           (forward)
    swiglu_bwd  d_gate, d_up and the product again, from 8 bits                       (backward)
    grad        an adapter's gradient, a sum over tokens, from an 8-bit input         (backward)
"""
import math

import torch
import torch.nn.functional as F

own = False

EPS = 1e-6
BLOCK = 32


def listed():
    return [
        # one short prompt through the 0.5B configuration: launch latency
        {"name": "add_norm 256x896", "op": "add_norm", "rows": 256, "D": 896, "delta": True},
        # a micro-batch of 4 x 4096 tokens of the 7B configuration
        {"name": "add_norm 16384x3584", "op": "add_norm", "rows": 16384, "D": 3584, "delta": True},
        # a ragged batch at 1.5B shapes
        {"name": "norm_bwd 4099x1536", "op": "norm_bwd", "rows": 4099, "D": 1536},
        {"name": "norm_bwd 16384x3584", "op": "norm_bwd", "rows": 16384, "D": 3584},
        # the attention output of a 7B layer kept for the backward pass
        {"name": "store 16384x3584", "op": "store", "rows": 16384, "D": 3584},
        # the normed input of a ragged 0.5B batch widened again, with the norm's weight
        {"name": "load 8191x904", "op": "load", "rows": 8191, "D": 904, "col": True},
        # the feed-forward block of a 7B layer
        {"name": "swiglu_fwd 16384x18944", "op": "swiglu_fwd", "rows": 16384, "D": 18944},
        {"name": "swiglu_bwd 333x4864", "op": "swiglu_bwd", "rows": 333, "D": 4864},
        {"name": "swiglu_bwd 16384x18944", "op": "swiglu_bwd", "rows": 16384, "D": 18944},
        # q, k and v adapters of rank 16 in one pass over their common input, 0.5B, 8 x 1024 tokens
        {"name": "grad 8192x896 r48", "op": "grad", "rows": 8192, "D": 896, "M": 48, "col": True},
        # rank 64 on the down projection, 1.5B, 4 x 2048 tokens
        {"name": "grad 8192x8960 r64", "op": "grad", "rows": 8192, "D": 8960, "M": 64, "col": False},
        # rank 16 on the down projection, 7B, 4 x 4096 tokens
        {"name": "grad 16384x18944 r16", "op": "grad", "rows": 16384, "D": 18944, "M": 16, "col": False},
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["add_norm", "norm_bwd", "store", "load", "swiglu_fwd", "swiglu_bwd", "grad"])
    wide = op in ("swiglu_fwd", "swiglu_bwd", "grad")
    case = {"op": op, "rows": log_int(1, 16384), "D": 8 * log_int(8, 2368 if wide else 1024)}
    if op == "add_norm":
        case["delta"] = rng.random() < 0.75
    if op in ("load", "grad"):
        case["col"] = rng.random() < 0.5
    if op == "grad":
        case["M"] = 8 * rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 24])
        # no more work than rank 16 on the largest projection
        case["rows"] = max(1, min(case["rows"], 16384 * 18944 * 16 // (case["D"] * case["M"])))
    return case


# ── inputs ──────────────────────────────────────────────────────────────────

def _activations(gen, rows, D, size=1.0, padded=True):
    """BF16 rows as a decoder layer has them: tokens of unlike size, a few channels far above the rest, some padded rows."""
    x = torch.randn(rows, D, generator=gen, device="cuda", dtype=torch.bfloat16)
    token = torch.randn(rows, 1, generator=gen, device="cuda").mul_(0.5).exp_().mul_(size)
    channel = torch.randn(1, D, generator=gen, device="cuda").mul_(0.3).exp_()
    channel[:, torch.randint(0, D, (max(1, D // 256),), generator=gen, device="cuda")] *= 24.0
    if padded and rows >= 64:
        token[torch.randint(0, rows, (rows // 64,), generator=gen, device="cuda")] = 0.0
    return x.mul_(token.bfloat16()).mul_(channel.bfloat16())


def _weight(gen, D):
    return torch.randn(D, generator=gen, device="cuda").mul_(0.1).add_(1.0).bfloat16()


def _gradient(gen, rows, D, size):
    token = torch.randn(rows, 1, generator=gen, device="cuda").exp_().mul_(size).bfloat16()
    return torch.randn(rows, D, generator=gen, device="cuda", dtype=torch.bfloat16).mul_(token)


def _held(x):
    """An activation in 8 bits, as bytes."""
    q, scale = _pack(x.float())
    return q.view(torch.uint8), scale.view(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, rows, D = case["op"], case["rows"], case["D"]
    nb = -(-D // BLOCK)
    dev = {"device": "cuda"}
    s = {"op": op, "rows": rows, "D": D}

    def bf16(*shape):
        return torch.empty(*shape, dtype=torch.bfloat16, **dev)

    def held():
        return torch.empty(rows, D, dtype=torch.uint8, **dev), torch.empty(rows, nb, dtype=torch.uint8, **dev)

    if op == "add_norm":
        s["x"] = _activations(gen, rows, D, 4.0, padded=False)
        s["delta"] = _activations(gen, rows, D, 0.5, padded=False) if case["delta"] else None
        s["w"] = _weight(gen, D)
        s["res"] = bf16(rows, D) if case["delta"] else None      # without a delta the residual stays where it is
        s["y"], s["rstd"] = bf16(rows, D), torch.empty(rows, **dev)
        s["q"], s["scale"] = held()
    elif op == "norm_bwd":
        x = _activations(gen, rows, D, 4.0, padded=False).float()
        s["rstd"] = 1.0 / torch.sqrt(x.square().mean(-1) + EPS)
        s["q"], s["scale"] = _held(x * s["rstd"][:, None])
        s["w"], s["dy"] = _weight(gen, D), _gradient(gen, rows, D, 1e-3)
        s["add"], s["dx"] = _gradient(gen, rows, D, 1e-3), bf16(rows, D)
    elif op == "store":
        s["x"] = _activations(gen, rows, D)
        s["q"], s["scale"] = held()
    elif op == "load":
        s["q"], s["scale"] = _held(_activations(gen, rows, D))
        s["col"], s["out"] = _weight(gen, D) if case["col"] else None, bf16(rows, D)
    elif op == "swiglu_fwd":
        s["gate"], s["up"], s["act"] = _activations(gen, rows, D), _activations(gen, rows, D), bf16(rows, D)
        s["gate_q"], s["gate_scale"] = held()
        s["up_q"], s["up_scale"] = held()
    elif op == "swiglu_bwd":
        s["gate_q"], s["gate_scale"] = _held(_activations(gen, rows, D))
        s["up_q"], s["up_scale"] = _held(_activations(gen, rows, D))
        s["dout"] = _gradient(gen, rows, D, 1e-3)
        s["dgate"], s["dup"], s["act"] = bf16(rows, D), bf16(rows, D), bf16(rows, D)
    else:
        s["q"], s["scale"] = _held(_activations(gen, rows, D))
        s["col"] = _weight(gen, D) if case["col"] else None
        s["dh"], s["M"] = _gradient(gen, rows, case["M"], 1e-3), case["M"]
        s["alpha"], s["gA"] = 1.0, torch.empty(case["M"], D, **dev)
    return s


# ── plain forms ─────────────────────────────────────────────────────────────

def _pack(v):
    """FP32 [rows, D] into (e4m3 values, E8M0 scales)."""
    rows, D = v.shape
    n = -(-D // BLOCK)
    b = F.pad(v, (0, n * BLOCK - D)).view(rows, n, BLOCK)
    amax = b.abs().amax(-1)
    m, e = torch.frexp(amax)                                 # amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    k = torch.where(m > 0.875, e - 8, e - 9).clamp(-117, 119)
    k = torch.where(amax == 0, torch.full_like(k, -117), k).to(torch.int32)
    inverse = ((127 - k) << 23).view(torch.float32)          # 2^-k
    q = (b * inverse[..., None]).view(rows, n * BLOCK)[:, :D].contiguous().to(torch.float8_e4m3fn)
    return q, (k + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _widen(q, scale):
    """The FP32 values that bytes of e4m3 and of exponents stand for."""
    rows, D = q.shape
    step = (scale.to(torch.int32) << 23).view(torch.float32)
    return q.view(torch.float8_e4m3fn).float() * step.repeat_interleave(BLOCK, dim=1)[:, :D]


def _plain(s):
    op = s["op"]
    if op == "add_norm":
        res = s["x"] if s["delta"] is None else (s["x"].float() + s["delta"].float()).bfloat16()
        r = res.float()
        rstd = 1.0 / torch.sqrt(r.square().mean(-1) + EPS)
        n = r * rstd[:, None]
        q, scale = _pack(n)
        return {"res": None if s["delta"] is None else res, "y": (n * s["w"].float()).bfloat16(), "q": q, "scale": scale, "rstd": rstd}
    if op == "norm_bwd":
        n = _widen(s["q"], s["scale"])
        g = s["dy"].float() * s["w"].float()
        mean = (g * n).mean(-1, keepdim=True)
        return {"dx": (s["add"].float() + s["rstd"][:, None] * (g - n * mean)).bfloat16()}
    if op == "store":
        q, scale = _pack(s["x"].float())
        return {"q": q, "scale": scale}
    if op == "load":
        v = _widen(s["q"], s["scale"])
        return {"out": (v if s["col"] is None else v * s["col"].float()).bfloat16()}
    if op == "swiglu_fwd":
        g, u = s["gate"].float(), s["up"].float()
        gate_q, gate_scale = _pack(g)
        up_q, up_scale = _pack(u)
        return {"act": (g / (1.0 + torch.exp(-g)) * u).bfloat16(), "gate_q": gate_q, "gate_scale": gate_scale, "up_q": up_q, "up_scale": up_scale}
    if op == "swiglu_bwd":
        g, u, d = _widen(s["gate_q"], s["gate_scale"]), _widen(s["up_q"], s["up_scale"]), s["dout"].float()
        sig = 1.0 / (1.0 + torch.exp(-g))
        return {"dgate": (d * u * sig * (1.0 + g * (1.0 - sig))).bfloat16(), "dup": (d * g * sig).bfloat16(), "act": (g * sig * u).bfloat16()}
    v = _widen(s["q"], s["scale"])
    c = s["alpha"] * torch.matmul(s["dh"].float().t(), v)
    return {"gA": c if s["col"] is None else c * s["col"].float()}


# ── the framework's operators ───────────────────────────────────────────────

_ctx = None


def _own(s):
    global _ctx
    from tensor_adapt_b200 import Context, ptr, stream_ptr
    if _ctx is None:
        _ctx = Context(torch.cuda.current_device())
    op, rows, D, st = s["op"], s["rows"], s["D"], stream_ptr()

    def values(name):
        return s[name + "q"].view(torch.float8_e4m3fn), s[name + "scale"].view(torch.float8_e8m0fnu)

    if op == "add_norm":
        _ctx.call("ta_add_rms_norm_q8_fwd", ptr(s["x"]), ptr(s["delta"]), ptr(s["w"]), ptr(s["res"]), ptr(s["y"]), ptr(s["q"]),
                  ptr(s["scale"]), ptr(s["rstd"]), rows, D, EPS, st)
        q, scale = values("")
        return {"res": s["res"], "y": s["y"], "q": q, "scale": scale, "rstd": s["rstd"]}
    if op == "norm_bwd":
        _ctx.call("ta_rms_norm_q8_bwd", ptr(s["dy"]), ptr(s["q"]), ptr(s["scale"]), ptr(s["w"]), ptr(s["rstd"]), ptr(s["dx"]),
                  ptr(s["add"]), rows, D, st)
        return {"dx": s["dx"]}
    if op == "store":
        _ctx.call("ta_q8_store", ptr(s["x"]), ptr(s["q"]), ptr(s["scale"]), rows, D, st)
        q, scale = values("")
        return {"q": q, "scale": scale}
    if op == "load":
        _ctx.call("ta_q8_load", ptr(s["q"]), ptr(s["scale"]), ptr(s["col"]), ptr(s["out"]), rows, D, st)
        return {"out": s["out"]}
    if op == "swiglu_fwd":
        _ctx.call("ta_silu_mul_q8_fwd", ptr(s["gate"]), ptr(s["up"]), ptr(s["act"]), ptr(s["gate_q"]), ptr(s["gate_scale"]),
                  ptr(s["up_q"]), ptr(s["up_scale"]), rows, D, st)
        gate_q, gate_scale = values("gate_")
        up_q, up_scale = values("up_")
        return {"act": s["act"], "gate_q": gate_q, "gate_scale": gate_scale, "up_q": up_q, "up_scale": up_scale}
    if op == "swiglu_bwd":
        _ctx.call("ta_silu_mul_q8_bwd", ptr(s["dout"]), ptr(s["gate_q"]), ptr(s["gate_scale"]), ptr(s["up_q"]), ptr(s["up_scale"]),
                  ptr(s["dgate"]), ptr(s["dup"]), ptr(s["act"]), rows, D, st)
        return {"dgate": s["dgate"], "dup": s["dup"], "act": s["act"]}
    _ctx.call("ta_gemm_tokens_q8_f32", s["M"], D, rows, s["alpha"], ptr(s["dh"]), s["M"], ptr(s["q"]), ptr(s["scale"]), ptr(s["col"]),
              ptr(s["gA"]), D, 0, st)
    return {"gA": s["gA"]}


def run(state):
    return _own(state) if own else _plain(state)


# ── the definition in 64 bits ───────────────────────────────────────────────

def _round_to(v, mantissa, lowest):
    """To the nearest value of `mantissa` bits behind the point, ties to even; below 2^lowest in steps of 2^(lowest - mantissa)."""
    exponent = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** (lowest - 60))))
    exponent = torch.where(torch.exp2(exponent) > v.abs(), exponent - 1, exponent)
    exponent = torch.where(torch.exp2(exponent + 1) <= v.abs(), exponent + 1, exponent)
    step = torch.exp2(exponent.clamp_min(lowest) - mantissa)
    return torch.round(v / step) * step


def _exact_pack(v):
    rows, D = v.shape
    n = -(-D // BLOCK)
    full = torch.zeros(rows, n * BLOCK, dtype=torch.float64, device=v.device)
    full[:, :D] = v
    full = full.view(rows, n, BLOCK)
    amax = full.abs().max(dim=-1).values
    k = torch.ceil(torch.log2(amax.clamp_min(2.0 ** -200) / 448.0))
    k = torch.where(amax > 448.0 * torch.exp2(k), k + 1, k)
    k = torch.where(amax <= 448.0 * torch.exp2(k - 1), k - 1, k).clamp(-117, 119)
    scale = torch.exp2(k)
    q = _round_to(full / scale[..., None], 3, -6).reshape(rows, n * BLOCK)[:, :D]
    return q, scale


_E4M3 = [(-1.0) ** (b >> 7) * (2.0 ** ((b >> 3 & 15) - 7) * (1 + (b & 7) / 8) if b >> 3 & 15 else (b & 7) * 2.0 ** -9) for b in range(256)]


def _exact_widen(q, scale):
    table = torch.tensor(_E4M3, dtype=torch.float64, device=q.device)
    block = torch.arange(q.shape[1], device=q.device) // BLOCK
    return table[q.long()] * torch.exp2(scale.double() - 127)[:, block]


def _exact_rows(op, s, at):
    """The rows `at` (a slice) of an operator that works row by row."""
    def take(name):
        return s[name][at].double()

    if op == "add_norm":
        r = take("x") if s["delta"] is None else _round_to(take("x") + take("delta"), 7, -126)
        rstd = (r.pow(2).sum(-1) / r.shape[1] + EPS).rsqrt()
        n = r * rstd[:, None]
        q, scale = _exact_pack(n)
        return {"res": None if s["delta"] is None else r, "y": n * s["w"].double(), "q": q, "scale": scale, "rstd": rstd}
    if op == "norm_bwd":
        n, rstd = _exact_widen(s["q"][at], s["scale"][at]), take("rstd")[:, None]
        g = take("dy") * s["w"].double()
        return {"dx": take("add") + rstd * g - n * (rstd * (g * n).sum(-1, keepdim=True) / n.shape[1])}
    if op == "store":
        q, scale = _exact_pack(take("x"))
        return {"q": q, "scale": scale}
    if op == "load":
        v = _exact_widen(s["q"][at], s["scale"][at])
        return {"out": v if s["col"] is None else v * s["col"].double()}
    if op == "swiglu_fwd":
        g, u = take("gate"), take("up")
        gate_q, gate_scale = _exact_pack(g)
        up_q, up_scale = _exact_pack(u)
        return {"act": g * torch.sigmoid(g) * u, "gate_q": gate_q, "gate_scale": gate_scale, "up_q": up_q, "up_scale": up_scale}
    g, u = _exact_widen(s["gate_q"][at], s["gate_scale"][at]), _exact_widen(s["up_q"][at], s["up_scale"][at])
    d, sig = take("dout"), torch.sigmoid(g)
    return {"dgate": d * u * (sig + g * sig * torch.sigmoid(-g)), "dup": d * g * sig, "act": g * sig * u}


def exact(case, seed):
    s = prepare(case, seed)
    op, rows, D = case["op"], case["rows"], case["D"]
    chunk = max(1, (1 << 25) // D)
    if op == "grad":
        total = torch.zeros(case["M"], D, dtype=torch.float64, device="cuda")
        for at in range(0, rows, chunk):
            part = slice(at, min(rows, at + chunk))
            total += s["dh"][part].double().t() @ _exact_widen(s["q"][part], s["scale"][part])
        return {"gA": s["alpha"] * total * (1.0 if s["col"] is None else s["col"].double())}
    parts = [_exact_rows(op, s, slice(at, min(rows, at + chunk))) for at in range(0, rows, chunk)]
    return {name: None if parts[0][name] is None else torch.cat([p[name] for p in parts]) for name in parts[0]}


# ── what a pass cannot do without ───────────────────────────────────────────

def work(case):
    op, rows, D = case["op"], case["rows"], case["D"]
    n, nb = rows * D, rows * -(-D // BLOCK)
    held = n + nb
    if op == "add_norm":
        return {"bytes": (8 if case["delta"] else 6) * n + held + 2 * D + 4 * rows, "flops": 8 * n}
    if op == "norm_bwd":
        return {"bytes": 6 * n + held + 2 * D + 4 * rows, "flops": 9 * n}
    if op == "store":
        return {"bytes": 2 * n + held, "flops": 2 * n}
    if op == "load":
        return {"bytes": 2 * n + held + (2 * D if case["col"] else 0), "flops": 2 * n}
    if op == "swiglu_fwd":
        return {"bytes": 6 * n + 2 * held, "flops": 10 * n}
    if op == "swiglu_bwd":
        return {"bytes": 8 * n + 2 * held, "flops": 16 * n}
    M = case["M"]
    return {"bytes": held + 2 * rows * M + 4 * M * D + (2 * D if case["col"] else 0), "flops": 2 * n * M}
