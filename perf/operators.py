"""Operators of a decoder block with local attention, each through the call that a model makes of it, on one GPU.

op "rotary"     queries and keys turned by the angles of their positions (``FO.rotary``)
op "attention"  causal attention over a window of recent keys and the first few (``FO.window_attention``)
op "mlp"        gated feed-forward block, silu(x Wg) * (x Wu) Wd (``FO.gated_mlp``)

``train`` cases run forward and backward and return the output and every gradient.  Where ``own`` is false the operators are
computed from elementary torch operations in 32 bits (angles in 64) and rounded once at the end.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One new token for each of eight sequences at far-apart positions: bound by the launch.
        dict(name="rotary-token", op="rotary", batch=8, seq=1, heads=16, kv_heads=4, hd=128, rot=128, layout="half", scaling="none",
             far=32000, dtype="bf16", train=False),
        # The 1.3 B GPT's sequences and heads in training.
        dict(name="rotary-train", op="rotary", batch=4, seq=2048, heads=16, kv_heads=16, hd=128, rot=128, layout="interleaved",
             scaling="none", far=0, dtype="bf16", train=True),
        # Ragged sequences, a part of each narrow head turned, fp32.
        dict(name="rotary-part", op="rotary", batch=3, seq=701, heads=12, kv_heads=4, hd=80, rot=32, layout="half", scaling="linear",
             far=1000, dtype="fp32", train=True),
        # The 13 B model's heads over one long context whose frequencies are stretched.
        dict(name="rotary-long", op="rotary", batch=1, seq=32768, heads=40, kv_heads=40, hd=128, rot=128, layout="half",
             scaling="yarn", far=0, dtype="bf16", train=True),
        # The next token of eight scored sequences, keys shared by four heads each.
        dict(name="attention-token", op="attention", batch=8, sq=1, sk=2000, heads=16, kv_heads=4, hd=128, window=1024, sinks=4,
             train=False),
        # Scoring a ragged piece behind a long prefix under a wide window.
        dict(name="attention-score", op="attention", batch=2, sq=501, sk=8192, heads=16, kv_heads=16, hd=128, window=4096, sinks=64,
             train=False),
        # Training at the 1.3 B GPT's sizes with a narrow window.
        dict(name="attention-train", op="attention", batch=4, sq=2048, sk=2048, heads=16, kv_heads=16, hd=128, window=512, sinks=4,
             train=True),
        # Sizes that fit no tile, narrow heads, three of them to a key head.
        dict(name="attention-ragged", op="attention", batch=3, sq=1537, sk=1537, heads=12, kv_heads=4, hd=64, window=200, sinks=1,
             train=True),
        # One long context in training.
        dict(name="attention-long", op="attention", batch=1, sq=32768, sk=32768, heads=16, kv_heads=4, hd=128, window=2048, sinks=4,
             train=True),
        # A few tokens through the block: bound by reading the weights.
        dict(name="mlp-token", op="mlp", tokens=8, d=2048, ff=8192, train=False),
        # Ragged sizes in training.
        dict(name="mlp-ragged", op="mlp", tokens=1111, d=1032, ff=2744, train=True),
        # The 13 B model's block over two sequences.
        dict(name="mlp-wide", op="mlp", tokens=4096, d=5120, ff=13824, train=True),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of ``step`` spread evenly over the logarithm of [lo, hi]."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["rotary", "attention", "attention", "mlp"])
    train = rng.random() < 0.6
    while True:
        kv = rng.choice([1, 2, 3, 4, 5, 8, 16, 20, 40])
        heads = kv * rng.choice([1, 1, 2, 3, 4, 8])
        if heads > 40:
            continue
        if op == "rotary":
            hd = rng.choice([64, 80, 96, 128])
            c = dict(op=op, batch=_log(rng, 1, 32), seq=_log(rng, 1, 32768), heads=heads, kv_heads=kv, hd=hd,
                     rot=rng.choice([hd, hd, hd // 2, 32]), layout=rng.choice(["half", "interleaved"]),
                     scaling=rng.choice(["none", "linear", "ntk", "yarn"]), far=rng.choice([0, _log(rng, 1, 500000)]),
                     dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), train=train)
            if work(c)["bytes"] <= work(listed()[3])["bytes"]:
                return c
        elif op == "attention":
            # in training a query sees two keys at least: beside a single one q and k have no gradient but rounding
            sk = _log(rng, 2 if train else 1, 32768)
            same = train or rng.random() < 0.5
            c = dict(op=op, batch=_log(rng, 1, 16), sq=sk if same else _log(rng, 1, sk), sk=sk, heads=heads, kv_heads=kv,
                     hd=rng.choice([64, 128]), window=_log(rng, 2 if train else 1, 4096), sinks=rng.choice([0, 1, 4, 4, rng.randint(5, 200)]), train=train)
            scores = c["batch"] * heads * c["sq"] * (min(c["window"], sk) + c["sinks"] + 256)
            if work(c)["flops"] <= work(listed()[8])["flops"] and scores <= 16 * 32768 * 2560:
                return c
        else:
            c = dict(op=op, tokens=_log(rng, 1, 8192), d=_log(rng, 64, 5120, 8), ff=_log(rng, 64, 13824, 8), train=train)
            if work(c)["flops"] <= work(listed()[11])["flops"]:
                return c


# ------------------------------------------------------------------------------------------------------------- inputs
def _frequencies(rot, scaling):
    """Angles a position turns each pair by, float64, and the factor on the result.  linear: positions squeezed eightfold; ntk: the
    base grows instead; yarn: pairs that turn often inside 4096 positions stay, slow ones are squeezed, a ramp between."""
    k = torch.arange(0, rot, 2, dtype=torch.float64)
    base, factor = 10000.0, 8.0
    if scaling == "ntk":
        base = base * factor ** (rot / max(rot - 2, 1))
    f = base ** (-k / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        turns = 4096 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1 - keep)
        return f, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, scale=1.0, grad=False):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype).requires_grad_(grad)

    train = case["train"]
    state = {"case": case}
    if case["op"] == "rotary":
        B, S, H, Hkv, hd = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["hd"]
        dt = TYPES[case["dtype"]]
        # q and k lie side by side in the projection of the token, with v behind them
        qkv = normal(B, S, H + 2 * Hkv, hd, dtype=dt)
        state["q"] = qkv[:, :, :H].detach().requires_grad_(train)
        state["k"] = qkv[:, :, H:H + Hkv].detach().requires_grad_(train)
        start = torch.randint(0, case["far"] + 1, (B, 1), device=DEV, generator=g)
        state["positions"] = start + torch.arange(S, device=DEV)
        f, state["magnitude"] = _frequencies(case["rot"], case["scaling"])
        state["freqs"] = f.to(DEV)
        if train:
            state["dq"], state["dk"] = normal(B, S, H, hd, dtype=dt), normal(B, S, Hkv, hd, dtype=dt)
    elif case["op"] == "attention":
        B, Sq, Sk, H, Hkv, hd = (case[n] for n in ("batch", "sq", "sk", "heads", "kv_heads", "hd"))
        state["q"] = normal(B, Sq, H, hd, grad=train)
        state["k"], state["v"] = normal(B, Sk, Hkv, hd, grad=train), normal(B, Sk, Hkv, hd, grad=train)
        if train:
            state["do"] = normal(B, Sq, H, hd)
    else:
        T, D, F = case["tokens"], case["d"], case["ff"]
        state["x"] = normal(T, D, grad=train)
        state["w_gate_up"] = normal(2 * F, D, scale=0.02, grad=train)
        state["w_down"] = normal(D, F, scale=0.02, grad=train)
        if train:
            state["dy"] = normal(T, D)
    return state


# ------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    op, train = state["case"]["op"], state["case"]["train"]
    if op == "rotary":
        ins, douts = ("q", "k"), ("dq", "dk")
        outs = (_own_rotary if own else _plain_rotary)(state)
    elif op == "attention":
        ins, douts = ("q", "k", "v"), ("do",)
        outs = (_own_attention if own else _plain_attention)(state)
    else:
        ins, douts = ("x", "w_gate_up", "w_down"), ("dy",)
        outs = (_own_mlp if own else _plain_mlp)(state)
    if not train:
        return [o.detach() for o in outs]
    grads = torch.autograd.grad(outs, [state[n] for n in ins], [state[n] for n in douts])
    return [o.detach() for o in outs] + list(grads)


def _own_rotary(s):
    from rtp_b200.ops import functional as FO
    return FO.rotary(s["q"], s["k"], s["positions"], s["freqs"], layout=s["case"]["layout"], magnitude=s["magnitude"])


def _own_attention(s):
    from rtp_b200.ops import functional as FO
    return (FO.window_attention(s["q"], s["k"], s["v"], s["case"]["window"], sinks=s["case"]["sinks"]),)


def _own_mlp(s):
    from rtp_b200.ops import functional as FO
    return (FO.gated_mlp(s["x"], s["w_gate_up"], s["w_down"]),)


def _plain_rotary(s):
    rot, half_layout = s["case"]["rot"], s["case"]["layout"] == "half"
    angle = s["positions"].double()[..., None] * s["freqs"]
    cos = (angle.cos() * s["magnitude"]).float()[:, :, None]
    sin = (angle.sin() * s["magnitude"]).float()[:, :, None]

    def turn(x):
        y = x.float()
        t = y[..., :rot]
        if half_layout:
            a, b = t[..., :rot // 2], t[..., rot // 2:]
            t = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
        else:
            a, b = t[..., 0::2], t[..., 1::2]
            t = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
        return torch.cat([t, y[..., rot:]], dim=-1).to(x.dtype)

    return turn(s["q"]), turn(s["k"])


def _plain_attention(s):
    """Blocks of queries, each against the keys that one of its queries can see and the first few."""
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    B, Sq, H, hd = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    G, W, sinks = H // Hkv, min(s["case"]["window"], Sk), min(s["case"]["sinks"], Sk)
    block = min(256, Sq)
    n = -(-Sq // block)
    dev = q.device
    pos = (torch.arange(n * block, device=dev) + (Sk - Sq)).clamp(max=Sk - 1).view(n, block, 1)
    near = torch.arange(block + W - 1, device=dev) + (torch.arange(n, device=dev) * block + (Sk - Sq) - W + 1)[:, None]
    first = torch.arange(sinks, device=dev).expand(n, sinks)
    sees_near = (near[:, None] >= 0) & (near[:, None] <= pos) & (near[:, None] > pos - W)
    sees = torch.cat([sees_near, first[:, None] <= pos - W], dim=-1)                  # [n, block, keys]
    keys = torch.cat([near.clamp(0, Sk - 1), first], dim=-1)
    kk = k[:, keys].permute(0, 3, 1, 2, 4)                                            # [B, Hkv, n, keys, hd]
    vv = v[:, keys].permute(0, 3, 1, 2, 4)
    qq = torch.cat([q, q.new_zeros(B, n * block - Sq, H, hd)], dim=1)
    qq = qq.view(B, n, block, Hkv, G, hd).permute(0, 3, 1, 4, 2, 5).reshape(B, Hkv, n, G * block, hd)
    scores = (qq @ kk.transpose(-1, -2) * hd ** -0.5).view(B, Hkv, n, G, block, -1)
    scores = scores.masked_fill(~sees[:, None], float("-inf"))
    e = (scores - scores.amax(-1, keepdim=True).detach()).exp()
    p = (e / e.sum(-1, keepdim=True)).view(B, Hkv, n, G * block, -1)
    o = (p @ vv).view(B, Hkv, n, G, block, hd).permute(0, 2, 4, 1, 3, 5).reshape(B, n * block, H, hd)
    return (o[:, :Sq].to(s["q"].dtype),)


def _plain_mlp(s):
    x, wgu, wd = s["x"].float(), s["w_gate_up"].float(), s["w_down"].float()
    gu = x @ wgu.t()
    F = wd.shape[1]
    g, u = gu[:, :F], gu[:, F:]
    return ((g * torch.sigmoid(g) * u @ wd.t()).to(s["x"].dtype),)


# ------------------------------------------------------------------------------------------------------------- work
def _pairs(case):
    """(query, key) pairs of one head that see each other."""
    Sq, Sk, W, sinks = case["sq"], case["sk"], case["window"], case["sinks"]

    def upto(n, cap):                 # sum of min(p, cap) for p = 1 .. n
        m = min(n, cap)
        return m * (m + 1) // 2 + (n - m) * cap if n > 0 else 0

    first = Sk - Sq                   # the first query's position; query i sees p = first + i + 1 keys before masks
    near = upto(Sk, W) - upto(first, W)
    far = (upto(Sk - W, sinks) - upto(first - W, sinks)) if sinks else 0
    return near + far


def work(case):
    train = case["train"]
    if case["op"] == "rotary":
        size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
        tokens = case["batch"] * case["seq"]
        once = 2 * tokens * (case["heads"] + case["kv_heads"]) * case["hd"] * size + 8 * tokens
        flops = 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rot"]
        return {"bytes": once * (2 if train else 1), "flops": flops * (2 if train else 1)}
    if case["op"] == "attention":
        q = 2 * case["batch"] * case["sq"] * case["heads"] * case["hd"]
        seen = case["sk"]
        if case["sq"] < case["sk"]:   # keys before the first query's window that are no sinks are not read
            seen = min(case["sk"], case["sq"] + case["window"] - 1 + case["sinks"])
        kv = 4 * case["batch"] * seen * case["kv_heads"] * case["hd"]
        flops = 4 * case["batch"] * case["heads"] * case["hd"] * _pairs(case)
        if train:                     # q, k, v, do in, o, dq, dk, dv out; five products behind the two of the forward
            return {"bytes": 4 * q + 2 * kv, "flops": flops * 3.5}
        return {"bytes": 2 * q + kv, "flops": flops}
    T, D, F = case["tokens"], case["d"], case["ff"]
    acts, weights, flops = 2 * T * D, 6 * D * F, 6 * T * D * F
    if train:
        return {"bytes": 4 * acts + 2 * weights, "flops": 3 * flops}
    return {"bytes": 2 * acts + weights, "flops": flops}


# ------------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "attention": _exact_attention, "mlp": _exact_mlp}[case["op"]](case, s)


def _exact_rotary(case, s):
    rot, m = case["rot"], s["magnitude"]
    pairs = torch.arange(rot // 2, device=DEV)
    one, two = (pairs, pairs + rot // 2) if case["layout"] == "half" else (2 * pairs, 2 * pairs + 1)
    turn = torch.polar(torch.full((), m, dtype=torch.float64, device=DEV), s["positions"].double()[:, :, None, None] * s["freqs"])

    def turned(x, by):
        y = x.double()
        z = torch.complex(y[..., one], y[..., two]) * by
        y[..., one], y[..., two] = z.real, z.imag
        return y

    outs = [turned(s["q"], turn), turned(s["k"], turn)]
    if case["train"]:
        outs += [turned(s["dq"], turn.conj()), turned(s["dk"], turn.conj())]
    return outs


def _exact_attention(case, s):
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    B, Sq, H, hd = q.shape
    Sk, G, W, sinks = k.shape[1], H // k.shape[2], case["window"], case["sinks"]
    scale = 1.0 / math.sqrt(hd)
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for a in range(0, Sq, 512):
        z = min(a + 512, Sq)
        lo = max(0, a + Sk - Sq - W + 1)
        cols = torch.arange(lo, z + Sk - Sq, device=DEV)
        if min(sinks, lo):
            cols = torch.cat([torch.arange(min(sinks, lo), device=DEV), cols])
        at = torch.arange(a + Sk - Sq, z + Sk - Sq, device=DEV)[:, None]
        hidden = (cols > at) | ((at - cols >= W) & (cols >= sinks))
        for h in range(H):
            qh, kh, vh = q[:, a:z, h], k[:, cols, h // G], v[:, cols, h // G]
            p = torch.einsum("bid,bjd->bij", qh, kh).mul_(scale).masked_fill_(hidden, -math.inf).softmax(-1)
            oh = p @ vh
            out[:, a:z, h] = oh
            if case["train"]:
                g = s["do"][:, a:z, h].double()
                dv[:, cols, h // G] += p.transpose(1, 2) @ g
                ds = (g @ vh.transpose(1, 2) - (g * oh).sum(-1, keepdim=True)) * p * scale
                dq[:, a:z, h] = ds @ kh
                dk[:, cols, h // G] += ds.transpose(1, 2) @ qh
    return [out, dq, dk, dv] if case["train"] else [out]


def _exact_mlp(case, s):
    x, w, wd = s["x"].double(), s["w_gate_up"].double(), s["w_down"].double()
    F = case["ff"]
    g, u = torch.nn.functional.linear(x, w[:F]), torch.nn.functional.linear(x, w[F:])
    sig = 1.0 / (1.0 + torch.exp(-g))
    h = g * sig * u
    y = torch.nn.functional.linear(h, wd)
    if not case["train"]:
        return [y]
    dy = s["dy"].double()
    dh = dy @ wd
    dg, du = dh * u * (sig + g * sig * (1 - sig)), dh * g * sig
    d_gu = torch.cat([dg, du], dim=1)
    return [y, d_gu @ w, d_gu.t() @ x, dy.t() @ h]
