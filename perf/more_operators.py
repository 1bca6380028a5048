"""Performance cases of the expert layer over 4-bit weights and of the dense gated block.

Rows in 4 bits: blocks of 32 neighbouring columns share a power of two, and
each value is held beside it as an e2m1 float (0, 0.5, 1, 1.5, 2, 3, 4 or 6
and a sign), two to a byte.  Four kinds of work, each through the entry points
that a serving or training program calls:

* ``hold``: rows are written in 4 bits and read back (weights as they are
  loaded, or rows kept);
* ``grouped``: the product of ragged row groups with one 4-bit weight matrix
  per group, the rows in 8 or in 4 bits;
* ``layer``: the whole expert layer over weights in 4 bits (serving);
* ``ffn``: the gated feed-forward block that every token passes, beside the
  routed experts or in their place: forward alone, or with its gradients.

The layer shapes are those of ``placemoe_amd/workloads.py`` and, in drawn
cases, others between them.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK, GROUP = 32, 512  # columns that share an exponent; columns whose 16 exponents lie together
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(name, **fields):
    return dict(fields, name=name) if name else fields


def _hold(name, G, R, N, dtype="bf16"):
    """G matrices of R rows of N columns."""
    return _case(name, op="hold", G=G, R=R, N=N, dtype=dtype)


def _grouped(name, G, M, N, K, a, spread, dtype="bf16"):
    """M rows over G groups (`spread`: the sigma of the log of a group's share), in `a` bits."""
    return _case(name, op="grouped", G=G, M=M, N=N, K=K, a=a, spread=spread, dtype=dtype)


def _layer(name, T, H, I, E, C, K, S, dtype="bf16"):
    return _case(name, op="layer", T=T, H=H, I=I, E=E, C=C, K=K, S=S, dtype=dtype)


def _ffn(name, T, H, I, act, train, dtype="bf16"):
    return _case(name, op="ffn", T=T, H=H, I=I, act=act, train=train, dtype=dtype)


def listed():
    return [
        # An odd number of fp16 rows of odd width.
        _hold("hold-1531-odd", 1, 1531, 1411, "fp16"),
        # Weights as they are loaded: gate and up rows of the 16 copies of one rank of a large model.
        _hold("hold-weights-16", 16, 4096, 7168),
        # fc1 of one decode step, rows in 8 bits: 4-5 per copy, bound by the weights.
        _grouped("grouped-decode-768", 160, 768, 1536, 2048, 8, 0.5),
        # Ragged groups with widths that end inside every tile, fp16 results.
        _grouped("grouped-ragged-2500", 12, 2500, 1000, 1120, 4, 1.0, "fp16"),
        # fc1 of one expert-parallel rank of a large model, everything in 4 bits.
        _grouped("grouped-ep-rank-65536", 16, 65536, 4096, 7168, 4, 0.3),
        # One token through the layer: latency.
        _layer("layer-token", 1, 2048, 768, 128, 160, 8, 8),
        # One decode step of a loaded server with replicated hot experts.
        _layer("layer-decode-96", 96, 2048, 768, 128, 160, 8, 8),
        # Prefill of long prompts.
        _layer("layer-prefill-8192", 8192, 2048, 768, 128, 160, 8, 8),
        # The block beside the experts of a large model, one token.
        _ffn("ffn-token", 1, 7168, 2048, "silu", False),
        # An odd number of fp16 tokens through a narrow block, with gradients.
        _ffn("ffn-train-1531", 1531, 1416, 1000, "gelu_tanh", True, "fp16"),
        # The block beside 128 small experts: small weights, many tokens.
        _ffn("ffn-train-16384", 16384, 2048, 768, "silu", True),
        # The block beside the experts of a large model, a training step's tokens.
        _ffn("ffn-train-8192", 8192, 7168, 2048, "silu", True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ranges; none costs more than the largest of its kind."""
    op = rng.choice(["hold", "grouped", "layer", "ffn", "ffn"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    while True:
        if op == "hold":
            case = _hold("", rng.choice([1, 1, 4, 16]), _log_int(rng, 1, 65536), _log_int(rng, 32, 8192), dtype)
            if case["G"] * case["R"] * case["N"] <= 16 * 4096 * 7168:
                return case
        elif op == "grouped":
            case = _grouped("", rng.randint(1, 160), _log_int(rng, 1, 65536), 8 * _log_int(rng, 4, 512), 32 * _log_int(rng, 2, 224),
                            rng.choice([4, 8]), rng.choice([0.0, 0.3, 0.5, 1.0]), dtype)
            if case["G"] * case["N"] * case["K"] <= 16 * 4096 * 7168 and case["M"] * case["N"] * case["K"] <= 65536 * 4096 * 7168 // 4:
                return case
        elif op == "layer":
            E = rng.choice([8, 16, 32, 64, 128])
            C, K = E + rng.randint(0, E // 2), rng.choice([1, 2, 4, 6, 8])
            H, I, T = 32 * _log_int(rng, 8, 224), 32 * _log_int(rng, 4, 88), _log_int(rng, 1, 16384)
            if K <= E // 2 and C * H * I <= 160 * 2048 * 768 and T * K * H * I <= 65536 * 2048 * 768 and T * K * (H + I) <= 65536 * 2816:
                return _layer("", T, H, I, E, C, K, rng.choice([1, 4, 8]), dtype)
        else:
            case = _ffn("", _log_int(rng, 1, 16384), 8 * _log_int(rng, 8, 896), 8 * _log_int(rng, 8, 512),
                        rng.choice(["silu", "gelu_tanh", "quick_gelu"]), rng.random() < 0.6, dtype)
            if case["T"] * case["H"] * case["I"] <= 8192 * 7168 * 2048:
                return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(gen, shape, dtype):
    """About N(0, 1), with the few loud columns that hidden states have and a silent row in 64."""
    x = torch.randn(shape, generator=gen, device="cuda")
    col = torch.rand(shape[-1], generator=gen, device="cuda")
    x *= torch.where(col < 0.01, 20.0, 1.0)
    x *= (torch.rand((*shape[:-1], 1), generator=gen, device="cuda") > 1 / 64).float()
    return x.to(dtype)


def _blocks(x):
    """Rows [..., R, N] as [..., R, B * 16, 32], padded with zeros to whole groups, and each block's largest magnitude."""
    *lead, R, N = x.shape
    B = -(-N // GROUP)
    x = torch.nn.functional.pad(x.float(), (0, B * GROUP - N)).view(*lead, R, B * 16, BLOCK)
    return x, x.abs().amax(-1, keepdim=True)


def _bytes(e):
    """Exponents [..., R, B * 16, 1] as they are held: [..., B, R, 16], e + 127."""
    *lead, R, n, _ = e.shape
    return (e + 127).to(torch.uint8).view(*lead, R, n // 16, 16).transpose(-3, -2).contiguous()


def _pack8(x):
    """(codes, exponent bytes) of rows in e4m3: each block's power of two is the
    smallest at which its largest value lies within 448."""
    N = x.shape[-1]
    x, most = _blocks(x)
    m, e = torch.frexp(most)  # most = m * 2^e, m in [0.5, 1)
    e = torch.where(most == 0, 0, (e - 9 + (m > 0.875).int()).clamp(-127, 127))
    codes = torch.ldexp(x, -e).to(torch.float8_e4m3fn).flatten(-2)[..., :N].contiguous()
    return codes, _bytes(e)


def _pack4(x):
    """(codes, exponent bytes) of rows in e2m1: each block's power of two is the
    smallest at which its largest value lies below 7, so that it rounds to 6 at
    most; nearest level, ties to the even code; the even column in a byte's low half."""
    N = x.shape[-1]
    x, most = _blocks(x)
    m, e = torch.frexp(most)
    e = torch.where(most == 0, 0, (e - 3 + (m >= 0.875).int()).clamp(-127, 127))
    y = torch.ldexp(x, -e).flatten(-2)[..., : N + N % 2]
    a = y.abs()
    code = 8 * (y < 0).to(torch.uint8)
    for border, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += a >= border if up else a > border
    return (code[..., 0::2] + 16 * code[..., 1::2]).contiguous(), _bytes(e)


def _units(scales, N, to=torch.float32):
    """The powers of two beside N columns, as exponents [..., R, N]."""
    *lead, B, R, _ = scales.shape
    e = scales.transpose(-3, -2).reshape(*lead, R, B * 16).to(torch.int32) - 127
    return e.repeat_interleave(BLOCK, -1)[..., :N]


def _unpack8(codes, scales):
    return torch.ldexp(codes.float(), _units(scales, codes.shape[-1]))


def _unpack4(codes, scales, N):
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :N]
    return torch.ldexp(level[both.int()], _units(scales, N))


def _weights(gen, shape, dtype, std=0.02):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def prepare(case, seed):
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    s = dict(case=case, dtype=dtype)
    if case["op"] == "hold":
        shape = (case["G"], case["R"], case["N"]) if case["G"] > 1 else (case["R"], case["N"])
        s["x"] = _weights(gen, shape, dtype) if case["G"] > 1 else _activations(gen, shape, dtype)
    elif case["op"] == "grouped":
        G, M, N, K = case["G"], case["M"], case["N"], case["K"]
        share = torch.exp(case["spread"] * torch.randn(G, generator=gen, device="cuda"))
        counts = torch.bincount(torch.multinomial(share, M, replacement=True, generator=gen), minlength=G)
        s["offsets"] = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32)
        s["most"] = int(counts.max())
        s["a"] = (_pack8 if case["a"] == 8 else _pack4)(_activations(gen, (M, K), dtype))
        s["b"] = _pack4(_weights(gen, (G, N, K), dtype))
    elif case["op"] == "layer":
        T, H, I, E, C, K, S = (case[k] for k in ("T", "H", "I", "E", "C", "K", "S"))
        s["hidden"] = _activations(gen, (T, H), dtype)
        logits = torch.randn((T, E), generator=gen, device="cuda") + 0.5 * torch.randn(E, generator=gen, device="cuda")
        w, s["selected"] = torch.topk(torch.softmax(logits, -1), K)
        s["weights"] = (w / w.sum(-1, keepdim=True)).to(dtype)
        # experts 0 .. C-E-1 have a second copy; sources take turns
        source, expert = torch.arange(S, device="cuda").view(S, 1), torch.arange(E, device="cuda").view(1, E)
        s["mapping"] = torch.where((expert < C - E) & (source % 2 == 1), E + expert, expert).contiguous()
        s["sources"] = torch.randint(0, S, (T,), generator=gen, device="cuda")
        s["fc1"] = _pack4(_weights(gen, (C, 2 * I, H), dtype))
        s["fc2"] = _pack4(_weights(gen, (C, H, I), dtype))
        copies = s["mapping"][s["sources"].view(-1, 1), s["selected"]]
        s["most"] = int(torch.bincount(copies.reshape(-1), minlength=C).max())
    else:
        T, H, I = case["T"], case["H"], case["I"]
        s["x"] = _activations(gen, (T, H), dtype)
        s["gate_up"] = _weights(gen, (2 * I, H), dtype, 1 / math.sqrt(H))
        s["down"] = _weights(gen, (H, I), dtype, 1 / math.sqrt(I))
        if case["train"]:
            s["dout"] = (0.1 * torch.randn((T, H), generator=gen, device="cuda")).to(dtype)
            for name in ("x", "gate_up", "down"):
                s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _spread(group, G):
    """For rows of the groups `group` [A]: each one's place within its group."""
    order = torch.argsort(group, stable=True)
    start = torch.nn.functional.pad(torch.bincount(group, minlength=G).cumsum(0), (1, 0))[:-1]
    place = torch.empty_like(order)
    place[order] = torch.arange(group.numel(), device=group.device) - start[group[order]]
    return place


def _products(rows, group, place, weights, most):
    """rows[r] @ weights[group[r]]^T, over groups padded to `most` rows."""
    G = weights.shape[0]
    padded = rows.new_zeros(G, most, rows.shape[1])
    padded[group, place] = rows
    return torch.bmm(padded, weights.transpose(1, 2))[group, place]


# act(g) = g * sigmoid(g * (a + b g^2)); tanh(z) = 2 sigmoid(2 z) - 1 makes the second of the tanh form of GELU
GATES = {"silu": (1.0, 0.0), "gelu_tanh": (2 * math.sqrt(2 / math.pi), 2 * math.sqrt(2 / math.pi) * 0.044715), "quick_gelu": (1.702, 0.0)}


def _plain_ffn(s):
    case, dtype = s["case"], s["dtype"]
    a, b = GATES[case["act"]]
    x, w1, w2 = (s[n].detach().float() for n in ("x", "gate_up", "down"))
    g, u = (x @ w1.t()).chunk(2, -1)
    sig = 1 / (1 + torch.exp(-g * (a + b * g * g)))
    h = g * sig * u
    out = (h @ w2.t()).to(dtype)
    if not case["train"]:
        return out
    d = s["dout"].float()
    dh = d @ w2
    slope = sig + g * sig * (1 - sig) * (a + 3 * b * g * g)
    dgu = torch.cat((dh * u * slope, dh * g * sig), -1)
    return out, (dgu @ w1).to(dtype), (dgu.t() @ x).to(dtype), (d.t() @ h).to(dtype)


def _plain(s):
    case, dtype = s["case"], s["dtype"]
    if case["op"] == "hold":
        return _unpack4(*_pack4(s["x"]), case["N"]).to(dtype)
    if case["op"] == "grouped":
        rows = torch.arange(case["M"], device="cuda")
        group = torch.searchsorted(s["offsets"][1:].long(), rows, right=True)
        place = rows - s["offsets"].long()[group]
        a = _unpack8(*s["a"]) if case["a"] == 8 else _unpack4(*s["a"], case["K"])
        return _products(a, group, place, _unpack4(*s["b"], case["K"]), s["most"]).to(dtype)
    if case["op"] == "ffn":
        return _plain_ffn(s)
    copy = s["mapping"][s["sources"].view(-1, 1), s["selected"]].reshape(-1)
    place = _spread(copy, case["C"])
    x = _unpack8(*_pack8(s["hidden"])).repeat_interleave(case["K"], 0)
    g, u = _products(x, copy, place, _unpack4(*s["fc1"], case["H"]), s["most"]).chunk(2, -1)
    act = g / (1 + torch.exp(-g)) * u * s["weights"].float().view(-1, 1)
    y = _products(_unpack8(*_pack8(act)), copy, place, _unpack4(*s["fc2"], case["I"]), s["most"])
    return y.view(case["T"], case["K"], case["H"]).sum(1).to(dtype)


def run(state):
    if not own:
        return _plain(state)
    import placemoe_amd
    from placemoe_amd import rows4, rows8

    s, case, dtype = state, state["case"], state["dtype"]
    if case["op"] == "hold":
        return rows4.dequantize_rows4(rows4.quantize_rows4(s["x"]))
    if case["op"] == "grouped":
        a = rows8.Rows8(*s["a"], dtype) if case["a"] == 8 else rows4.Rows4(*s["a"], case["K"], dtype)
        return rows4.group_gemm_nt_rows4(a, rows4.Rows4(*s["b"], case["K"], dtype), s["offsets"])
    if case["op"] == "ffn":
        if not case["train"]:
            with torch.no_grad():
                return placemoe_amd.gated_ffn(s["x"], s["gate_up"], s["down"], activation=case["act"])
        out = placemoe_amd.gated_ffn(s["x"], s["gate_up"], s["down"], activation=case["act"])
        return out.detach(), *torch.autograd.grad(out, (s["x"], s["gate_up"], s["down"]), s["dout"])
    experts = rows4.Experts4(rows4.Rows4(*s["fc1"], case["H"], dtype), rows4.Rows4(*s["fc2"], case["I"], dtype))
    return rows4.expert_layer_rows4(s["hidden"], s["weights"], s["selected"], experts, mapping=s["mapping"], sources=s["sources"])


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------


def _exact_round(x, bits):
    """Rows in 64 bits, rounded to what 8 or 4 bits hold: in each block of 32
    columns to four significant bits, at least 2^-9 of the block's power of two
    apart (8), or to two, at least half of it apart (4); ties to even."""
    *lead, N = x.shape
    v = torch.nn.functional.pad(x, (0, -N % BLOCK)).reshape(*lead, -1, BLOCK)
    most = v.abs().amax(-1, keepdim=True)
    held = (lambda e: most <= 448.0 * torch.exp2(e)) if bits == 8 else (lambda e: most < 7.0 * torch.exp2(e))
    # the smallest e that holds the block, by log2 and then by comparison
    e = torch.where(most > 0, torch.ceil(torch.log2(torch.where(most > 0, most, 1.0) / (448.0 if bits == 8 else 7.0))), 0.0)
    e = torch.where(held(e), e, e + 1)
    e = torch.where((most > 0) & held(e - 1), e - 1, e).clamp(-127, 127)
    unit = torch.exp2(e)
    v = v / unit
    digits, least = (3, 2.0**-9) if bits == 8 else (1, 0.5)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - digits).clamp_min(least)
    return (torch.round(v / step) * step * unit).reshape(*lead, -1)[..., :N]


def _exact_values(codes, scales, bits, N):
    """What codes [R, ...] and exponent bytes [B, R, 16] stand for, in 64 bits."""
    col = torch.arange(N, device=codes.device)
    unit = torch.exp2(scales[col // GROUP, :, col // BLOCK % 16].t().double() - 127)  # the indexed columns come first
    if bits == 8:
        return codes.double() * unit
    half = codes[:, col // 2].int() >> (4 * (col % 2).int()) & 15
    k = half & 7
    size = torch.where(k < 2, 0.5 * k.double(), torch.exp2((k // 2 - 1).double()) * (1 + 0.5 * (k % 2).double()))
    return torch.where(half >= 8, -size, size) * unit


def _exact_products(rows, copy, weights, N):
    """rows[r] @ weights[copy[r]]^T, copy by copy."""
    out = rows.new_zeros(rows.shape[0], weights[0].shape[-2])
    for c in range(weights[0].shape[0]):
        at = torch.nonzero(copy == c).view(-1)
        if at.numel():
            out[at] = rows[at] @ _exact_values(weights[0][c], weights[1][c], 4, N).t()
    return out


def _exact_ffn(s):
    I = s["case"]["I"]
    x, w1, w2 = (s[n].detach().double() for n in ("x", "gate_up", "down"))
    g, u = x @ w1[:I].t(), x @ w1[I:].t()
    if s["case"]["act"] == "gelu_tanh":
        root = math.sqrt(2 / math.pi)
        t = torch.tanh(root * (g + 0.044715 * g**3))
        act = 0.5 * g * (1 + t)
        slope = 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * root * (1 + 3 * 0.044715 * g * g)
    else:
        k = 1.0 if s["case"]["act"] == "silu" else 1.702
        act = g * torch.sigmoid(k * g)
        slope = torch.sigmoid(k * g) * (1 + k * g * torch.sigmoid(-k * g))
    out = (act * u) @ w2.t()
    if not s["case"]["train"]:
        return out
    d = s["dout"].double()
    dh = d @ w2
    dg, du = dh * u * slope, dh * act
    return out, dg @ w1[:I] + du @ w1[I:], torch.cat((dg.t() @ x, du.t() @ x)), d.t() @ (act * u)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "hold":
        return _exact_round(s["x"].double(), 4)
    if case["op"] == "grouped":
        counts = (s["offsets"][1:] - s["offsets"][:-1]).long()
        copy = torch.repeat_interleave(torch.arange(case["G"], device="cuda"), counts)
        return _exact_products(_exact_values(*s["a"], case["a"], case["K"]), copy, s["b"], case["K"])
    if case["op"] == "ffn":
        return _exact_ffn(s)
    T, K, I = case["T"], case["K"], case["I"]
    copy = s["mapping"][s["sources"][:, None].expand(T, K), s["selected"]].reshape(-1)
    x = _exact_round(s["hidden"].double(), 8)[torch.arange(T * K, device="cuda") // K]
    gu = _exact_products(x, copy, s["fc1"], case["H"])
    act = gu[:, :I] * torch.sigmoid(gu[:, :I]) * gu[:, I:] * s["weights"].double().reshape(-1, 1)
    y = _exact_products(_exact_round(act, 8), copy, s["fc2"], I)
    return y.reshape(T, K, -1).sum(1)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def _held(rows, n, bits):
    """Bytes of rows in 8 or 4 bits with their exponents."""
    return rows * -(-n * bits // 8) + rows * 16 * -(-n // GROUP)


def work(case):
    if case["op"] == "hold":
        n = case["G"] * case["R"]
        return {"bytes": 4 * n * case["N"] + 2 * _held(n, case["N"], 4), "flops": 4 * n * case["N"]}
    if case["op"] == "grouped":
        G, M, N, K = case["G"], case["M"], case["N"], case["K"]
        active = G * (1 - (1 - 1 / G) ** M)  # groups with rows, if all were alike
        return {"bytes": _held(M, K, case["a"]) + active * _held(N, K, 4) + 2 * M * N, "flops": 2 * M * N * K}
    if case["op"] == "layer":
        T, H, I, C, K = (case[k] for k in ("T", "H", "I", "C", "K"))
        A = T * K
        active = C * (1 - (1 - 1 / C) ** A)
        return {"bytes": 4 * T * H + 10 * A + active * (_held(2 * I, H, 4) + _held(H, I, 4)), "flops": 6 * A * H * I}
    T, H, I = case["T"], case["H"], case["I"]
    if case["train"]:
        return {"bytes": 8 * T * H + 12 * H * I, "flops": 18 * T * H * I}
    return {"bytes": 4 * T * H + 6 * H * I, "flops": 6 * T * H * I}
