"""The operators of the encoder's transformer layers as cases that can be timed and checked.

Between the embedding and the pooled vector an encoder mixes its tokens: queries and keys are rotated by
their positions, attention runs over each sequence, and a gated feed-forward block follows.  A case is one
operator on one size:

  rotary        queries and keys (all heads of both in one tensor) turned by their positions
  rotary_train  the same and its backward pass
  attn          attention of every token over its own sequence, packed or padded, full or causal
  attn_train    the same and its backward pass
  gated         act(x Wg^T) * (x Wu^T)
  gated_train   the same and its backward pass: gradients of x and both weights

``run`` computes them in plain torch where ``own`` is false, and through ``trident_amd.encoder``
where it is true.  Sizes are generic ones and those of the indexes' vectors (96, 100, 128, 960
dimensions).
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
BASE = 10000.0
TRAINED = 2048       # positions that the scaled rotary frequencies were trained on
LOW, HIGH = 1.0, 32.0  # turns over TRAINED between which a frequency goes from scaled to its own
ACTIVATIONS = ("silu", "gelu", "gelu_tanh")


# ---------------------------------------------------------------------------------------------
# cases


def listed():
    return [
        # one query's tokens at serving time: 12 + 12 heads; latency counts
        dict(name="rotary_query", op="rotary", T=16, H=24, D=64, R=64, style="half", factor=1.0, start=0, dtype="bf16"),
        # a batch of passages while a corpus is encoded
        dict(name="rotary_corpus", op="rotary", T=131072, H=24, D=64, R=64, style="half", factor=1.0, start=0,
             dtype="bf16"),
        # far positions of a long document, half of each head, scaled frequencies, forward and backward
        dict(name="rotary_train_long", op="rotary_train", T=16385, H=40, D=128, R=64, style="interleaved", factor=8.0,
             start=1_000_003, dtype="f32"),
        # one query's tokens: latency counts
        dict(name="attn_query", op="attn", layout="packed", n=1, L=16, Hq=12, Hkv=12, D=64, causal=False, dtype="bf16"),
        # a padded batch of passages while a corpus is encoded
        dict(name="attn_corpus", op="attn", layout="padded", n=512, L=256, Hq=12, Hkv=12, D=64, causal=False,
             dtype="bf16"),
        # a long document among short ones, grouped heads, causal as in encoders made from decoders
        dict(name="attn_long", op="attn", layout="packed", n=4, L=16384, Hq=32, Hkv=8, D=128, causal=True,
             dtype="bf16"),
        # a training batch of passages of all lengths, packed
        dict(name="attn_train_batch", op="attn_train", layout="packed", n=64, L=2048, Hq=12, Hkv=4, D=64, causal=False,
             dtype="f16"),
        # a small float32 step: lengths from one token on, a head that fills no tile
        dict(name="attn_train_ragged", op="attn_train", layout="packed", n=17, L=777, Hq=6, Hkv=2, D=80, causal=True,
             dtype="f32"),
        # one query's vector: the weights are read for one row
        dict(name="gated_query", op="gated", M=1, N=2560, K=960, act="silu", dtype="bf16"),
        # a batch of a corpus
        dict(name="gated_corpus", op="gated", M=16384, N=4096, K=1024, act="gelu_tanh", dtype="bf16"),
        # a training step's tokens
        dict(name="gated_train_batch", op="gated_train", M=16384, N=4096, K=1024, act="silu", dtype="bf16"),
        # nothing round, float32
        dict(name="gated_train_ragged", op="gated_train", M=1237, N=777, K=333, act="gelu", dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the listed ones' ranges, no dearer than the largest of its operator: 1 to 131,072
    tokens, sequences of 1 to 16,384 of them, heads of 16 to 128 dimensions, 1 to 32 heads in groups of
    1 to 8, products of 1 to 16,384 rows by weights of 64 to 8,192 rows and columns."""
    op = rng.choice(["rotary", "rotary_train", "attn", "attn", "attn", "attn_train", "attn_train", "attn_train",
                     "gated", "gated", "gated_train", "gated_train"])
    dtype = rng.choice(["f32", "bf16", "bf16", "bf16", "f16"])
    if op in ("rotary", "rotary_train"):
        D = rng.choice([16, 32, 64, 80, 96, 100, 128, 128])
        H = rng.randint(1, 48)
        T = min(_log_int(rng, 1, 131_072), max(1, 131_072 * 24 * 64 * 2 // (H * D * BYTES[dtype])))
        return dict(op=op, T=T, H=H, D=D, R=rng.choice([D, D, D // 4 * 2]), style=rng.choice(["half", "interleaved"]),
                    factor=rng.choice([1.0, 1.0, 4.0, 8.0]), start=rng.choice([0, 0, _log_int(rng, 100, 2_000_000)]),
                    dtype=dtype)
    if op in ("attn", "attn_train"):
        D = rng.choice([16, 32, 64, 64, 64, 80, 96, 128, 128])
        Hkv = rng.randint(1, 12)
        Hq = Hkv * rng.choice([1, 1, 2, 3, 4, 8])
        while Hq > 32:
            Hq -= Hkv
        layout, L = rng.choice(["packed", "packed", "padded"]), _log_int(rng, 1, 16_384)
        n = _log_int(rng, 1, 1024)
        # pairs of tokens and elements, no more than attn_long's or a training batch's
        pairs = 2e10 if op == "attn" else 1e9
        pairs = min(pairs, 2e9 if op == "attn" else 2e8) if dtype == "f32" else pairs
        L = max(1, min(L, int(math.sqrt(pairs * 64 / (D * Hq)))))
        n = max(1, min(n, int(pairs * 64 / (D * Hq * L * L)), int(1e8 / (D * Hq * L))))
        return dict(op=op, layout=layout, n=n, L=L, Hq=Hq, Hkv=Hkv, D=D, causal=rng.random() < 0.5, dtype=dtype)
    M, N, K = _log_int(rng, 1, 16_384), _log_int(rng, 64, 8192), _log_int(rng, 64, 8192)
    if rng.random() < 0.6:
        N, K = max(64, N // 64 * 64), max(64, K // 64 * 64)
    M = max(1, min(M, 16384 * 4096 * 1024 // (N * K * (4 if dtype == "f32" else 1))))
    return dict(op=op, M=M, N=N, K=K, act=rng.choice(ACTIVATIONS), dtype=dtype)


def _lengths(case):
    """Tokens of each sequence.  Padded: between half and all of its slots, one empty where there are
    many.  Packed: the longest first, the others of all lengths below it."""
    n, L = case["n"], case["L"]
    if case["layout"] == "padded":
        return [0 if b == 7 else L - (7919 * b + 3) % (L // 2 + 1) for b in range(n)]
    return [L if b == 0 else max(1, (L * ((7919 * b) % 97 + 1)) // 97 - b % 2) for b in range(n)]


def work(case):
    op, es = case["op"], BYTES[case["dtype"]]
    if op in ("rotary", "rotary_train"):
        n = case["T"] * case["H"] * case["D"]
        passes = 2 if op == "rotary_train" else 1
        return {"bytes": passes * 2 * n * es + 8 * case["T"], "flops": passes * 3 * n}
    if op in ("attn", "attn_train"):
        lens = _lengths(case)
        tokens, d = sum(lens), case["D"]
        pairs = sum(m * (m + 1) // 2 if case["causal"] else m * m for m in lens)
        q, kv = tokens * case["Hq"] * d * es, tokens * case["Hkv"] * d * es
        flops = 4 * pairs * d * case["Hq"]
        if op == "attn":
            return {"bytes": 2 * q + 2 * kv, "flops": flops}
        return {"bytes": 4 * q + 4 * kv, "flops": flops * 7 // 2}  # q, grad, out, dq; k, v, dk, dv
    M, N, K = case["M"], case["N"], case["K"]
    forward = {"bytes": (M * K + 2 * N * K + M * N) * es, "flops": 4 * M * N * K}
    if op == "gated":
        return forward
    return {"bytes": forward["bytes"] + (M * K + 2 * N * K + M * N) * es, "flops": 12 * M * N * K}


# ---------------------------------------------------------------------------------------------
# inputs


def _frequencies(R, factor):
    """Radians a position for each pair of columns; scaled for contexts `factor` times those trained on:
    a frequency that turns less than LOW times over TRAINED positions is divided by the factor, one that
    turns more than HIGH times stays, between them by the share of the way."""
    f = [BASE ** (-2.0 * i / R) for i in range(R // 2)]
    if factor != 1.0:
        for i, w in enumerate(f):
            keep = min(1.0, max(0.0, (TRAINED * w / (2 * math.pi) - LOW) / (HIGH - LOW)))
            f[i] = w * keep + w / factor * (1.0 - keep)
    return f


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 31)
    op, dt = case["op"], TYPES[case["dtype"]]

    def rand(*shape, by=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * by).to(dt)

    if op in ("rotary", "rotary_train"):
        T, H, D = case["T"], case["H"], case["D"]
        # sequences of up to 512 tokens next to one another, or one that begins at `start`
        positions = torch.arange(T, device=DEV) + case["start"] if case["start"] else torch.arange(T, device=DEV) % 509
        s = dict(op=op, x=rand(T, H, D), positions=positions, style=case["style"],
                 frequencies=torch.tensor(_frequencies(case["R"], case["factor"]), dtype=torch.float64, device=DEV))
        if case["factor"] != 1.0:
            s["amplitude"] = 0.1 * math.log(case["factor"]) + 1.0
        if op == "rotary_train":
            s["grad"] = rand(T, H, D, by=1e-2)
        return s
    if op in ("attn", "attn_train"):
        lens = _lengths(case)
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        lead = (case["n"], case["L"]) if case["layout"] == "padded" else (sum(lens),)
        qkv = rand(*lead, Hq + 2 * Hkv, D)  # one projection's result, cut into the three
        s = dict(op=op, q=qkv[..., :Hq, :], k=qkv[..., Hq:Hq + Hkv, :], v=qkv[..., Hq + Hkv:, :], lens=lens,
                 causal=case["causal"], scale=1.0 / math.sqrt(D))
        if case["layout"] == "padded":
            s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        else:
            s["offsets"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
        if op == "attn_train":
            s["grad"] = rand(*lead, Hq, D, by=1e-2)
        return s
    M, N, K = case["M"], case["N"], case["K"]
    s = dict(op=op, x=rand(M, K), wg=rand(N, K, by=1 / math.sqrt(K)), wu=rand(N, K, by=1 / math.sqrt(K)),
             act=case["act"])
    if op == "gated_train":
        s["grad"] = rand(M, N, by=1e-2)
    return s


# ---------------------------------------------------------------------------------------------
# one pass


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from trident_amd import encoder
    op = s["op"]
    if op in ("rotary", "rotary_train"):
        how = dict(positions=s["positions"], interleaved=s["style"] == "interleaved", amplitude=s.get("amplitude", 1.0))
        y = encoder.rotary(s["x"], s["frequencies"], **how)
        if op == "rotary":
            return y
        return dict(y=y, dx=encoder.rotary(s["grad"], s["frequencies"], inverse=True, **how))
    if op in ("attn", "attn_train"):
        how = dict(offsets=s.get("offsets"), lengths=s.get("lengths"), causal=s["causal"], scale=s["scale"])
        if op == "attn":
            return encoder.attention(s["q"], s["k"], s["v"], **how)
        out, lse = encoder.attention_forward(s["q"], s["k"], s["v"], **how)
        dq, dk, dv = encoder.attention_grad(s["grad"], s["q"], s["k"], s["v"], out, lse, **how)
        return dict(out=out, dq=dq, dk=dk, dv=dv)
    if op == "gated":
        return encoder.gated_linear(s["x"], s["wg"], s["wu"], activation=s["act"])
    h, gate, up = encoder.gated_linear_forward(s["x"], s["wg"], s["wu"], activation=s["act"])
    dx, dwg, dwu = encoder.gated_linear_grad(s["grad"], s["x"], s["wg"], s["wu"], gate, up, activation=s["act"])
    return dict(h=h, dx=dx, dwg=dwg, dwu=dwu)


def _run_plain(s):
    op = s["op"]
    if op in ("rotary", "rotary_train"):
        y = _rotary_plain(s, s["x"], 1.0)
        return y if op == "rotary" else dict(y=y, dx=_rotary_plain(s, s["grad"], -1.0))
    if op in ("attn", "attn_train"):
        return _attention_plain(s)
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    a, slope = _activation_plain(s["act"], g, op == "gated_train")
    dt = s["x"].dtype
    if op == "gated":
        return (a * u).to(dt)
    dh = s["grad"].float()
    dg, du = dh * u * slope, dh * a
    return dict(h=(a * u).to(dt), dx=(dg @ wg + du @ wu).to(dt), dwg=(dg.t() @ x).to(dt), dwu=(du.t() @ x).to(dt))


def _rotary_plain(s, x, sign):
    f = s["frequencies"]
    t = s["positions"].double()[:, None, None] * f
    R, a = 2 * f.numel(), s.get("amplitude", 1.0)
    c, n = (a * torch.cos(t)).float(), (a * sign * torch.sin(t)).float()
    y = x.float()
    turned, rest = y[..., :R], y[..., R:]
    if s["style"] == "interleaved":
        x0, x1 = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((x0 * c - x1 * n, x0 * n + x1 * c), -1).flatten(-2)
    else:
        x0, x1 = turned[..., :R // 2], turned[..., R // 2:]
        turned = torch.cat((x0 * c - x1 * n, x0 * n + x1 * c), -1)
    return torch.cat((turned, rest), -1).to(x.dtype)


def _activation_plain(act, g, slope):
    """(act(g), act'(g) where it is asked for)"""
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-g))
        return g * p, p * (1.0 + g * (1.0 - p)) if slope else None
    if act == "gelu":
        p = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * p, p + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2 * math.pi)) if slope else None
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g * g * g))
    a = 0.5 * g * (1.0 + t)
    return a, 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g) if slope else None


def _attention_plain(s):
    train = s["op"] == "attn_train"
    names = ("out", "dq", "dk", "dv") if train else ("out",)
    like = dict(out=s["q"], dq=s["q"], dk=s["k"], dv=s["v"])
    res = {n: torch.zeros(like[n].shape, dtype=like[n].dtype, device=DEV) for n in names}
    Hq, Hkv = s["q"].shape[-2], s["k"].shape[-2]
    G, at = Hq // Hkv, 0
    for b, m in enumerate(s["lens"]):
        rows = (b, slice(0, m)) if "lengths" in s else (slice(at, at + m),)
        at += m
        if m == 0:
            continue
        later = torch.ones((m, m), dtype=torch.bool, device=DEV).triu_(1) if s["causal"] else None
        step = max(1, int(2 ** 28 / (m * m * G)))  # kv heads at a time: 1 GB of scores
        for h in range(0, Hkv, step):
            kv, qs = slice(h, min(h + step, Hkv)), slice(h * G, min(h + step, Hkv) * G)

            def heads(t, which):  # [heads, tokens, D]
                return t[rows][:, which].float().transpose(0, 1)

            q = heads(s["q"], qs).reshape(-1, G * m, s["q"].shape[-1])
            k, v = heads(s["k"], kv), heads(s["v"], kv).contiguous()
            scores = (torch.bmm(q, k.transpose(1, 2).contiguous()) * s["scale"]).view(-1, G, m, m)
            if later is not None:
                scores.masked_fill_(later, -math.inf)
            p = torch.exp(scores - scores.amax(-1, keepdim=True))
            p = (p / p.sum(-1, keepdim=True)).view(-1, G * m, m)
            del scores
            o = torch.bmm(p, v)

            def put(name, t, which):
                res[name][rows][:, which] = t.reshape(-1, m, t.shape[-1]).transpose(0, 1).to(res[name].dtype)

            put("out", o, qs)
            if train:
                do = heads(s["grad"], qs).reshape(-1, G * m, q.shape[-1])
                put("dv", torch.bmm(p.transpose(1, 2).contiguous(), do), kv)
                dp = torch.bmm(do, v.transpose(1, 2).contiguous())
                ds = p * (dp - (do * o).sum(-1, keepdim=True)) * s["scale"]
                put("dq", torch.bmm(ds, k.contiguous()), qs)
                put("dk", torch.bmm(ds.transpose(1, 2).contiguous(), q), kv)
    return res if train else res["out"]


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op, f64 = s["op"], torch.float64
    if op in ("rotary", "rotary_train"):
        turn = torch.polar(torch.full_like(s["frequencies"], s.get("amplitude", 1.0)).expand(case["T"], -1),
                           torch.outer(s["positions"].to(f64), s["frequencies"]))[:, None, :]

        def rotated(x, turn):
            y = x.to(f64)
            R = case["R"]
            part = y[..., :R].unflatten(-1, (R // 2, 2) if case["style"] == "interleaved" else (2, R // 2))
            pair = -1 if case["style"] == "interleaved" else -2
            z = torch.complex(part.select(pair, 0), part.select(pair, 1)) * turn
            y[..., :R] = torch.stack((z.real, z.imag), pair).flatten(-2)
            return y

        y = rotated(s["x"], turn)
        return y if op == "rotary" else dict(y=y, dx=rotated(s["grad"], turn.conj()))
    if op in ("attn", "attn_train"):
        return _exact_attention(s, case)
    x, wg, wu = (s[n].to(f64).requires_grad_(op == "gated_train") for n in ("x", "wg", "wu"))
    with torch.enable_grad():
        g = torch.nn.functional.linear(x, wg)
        a = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
             "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[s["act"]](g)
        h = a * torch.nn.functional.linear(x, wu)
        if op == "gated":
            return h.detach()
        dx, dwg, dwu = torch.autograd.grad(h, (x, wg, wu), s["grad"].to(f64))
    return dict(h=h.detach(), dx=dx, dwg=dwg, dwu=dwu)


def _exact_attention(s, case):
    f64 = torch.float64
    train, G = s["op"] == "attn_train", case["Hq"] // case["Hkv"]
    out = torch.zeros(s["q"].shape, dtype=f64, device=DEV)
    dq = torch.zeros_like(out)
    dk, dv = torch.zeros((2, *s["k"].shape), dtype=f64, device=DEV)
    first = 0
    for b, m in enumerate(s["lens"]):
        rows = (b, slice(0, m)) if case["layout"] == "padded" else (slice(first, first + m),)
        first += m
        for h in range(case["Hq"] if m else 0):
            k, v = s["k"][rows][:, h // G].to(f64), s["v"][rows][:, h // G].to(f64)
            for a in range(0, m, 4096):  # so many queries at a time
                e = min(m, a + 4096)
                keys = e if case["causal"] else m
                q = s["q"][rows][a:e, h].to(f64)
                x = torch.mm(q, k[:keys].t()) * s["scale"]
                if case["causal"]:
                    x += torch.full((e - a, keys), -math.inf, dtype=f64, device=DEV).triu(a + 1)
                p = torch.softmax(x, 1)
                o = torch.mm(p, v[:keys])
                out[rows][a:e, h] = o
                if train:
                    do = s["grad"][rows][a:e, h].to(f64)
                    ds = p * (torch.mm(do, v[:keys].t()) - torch.einsum("id,id->i", do, o)[:, None]) * s["scale"]
                    dv[rows][:keys, h // G] += torch.mm(p.t(), do)
                    dk[rows][:keys, h // G] += torch.mm(ds.t(), q)
                    dq[rows][a:e, h] = torch.mm(ds, k[:keys])
    return dict(out=out, dq=dq, dk=dk, dv=dv) if train else out
