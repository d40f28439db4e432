"""The encoder's operators as cases that can be timed and checked.

The encoder makes the vectors that an index holds: tokens are looked up in a table, normalised and
projected; the table and the weights are trained with AdamW.  A case is one operator on one size:

  embed       rows of a table for a padded batch of token ids, scaled
  embed_grad  the table's gradient from the gradient of those rows
  norm        layer norm of a batch of vectors (no gradient kept)
  norm_train  layer norm and its backward pass: gradients of the vectors, the weight and the bias
  adamw       one optimizer step over a list of tensors, states in 32 or 8 bits
  linear      the projection of a batch by a weight held in 8-bit floating point, one power-of-two
              scale for each row and 128 of its columns, the batch quantised the same way in the call

``run`` computes them in plain torch where ``own`` is false, and through ``trident_amd.encoder``
where it is true.  Sizes are those of the indexes' vectors (96, 100, 128, 960 dimensions) and generic
ones between and above them.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 256          # elements of an optimizer state that share a scale
BETA1, BETA2, EPS, DECAY, LR, STEP = 0.9, 0.999, 1e-8, 0.01, 3e-4, 17  # STEP: the step being taken


# ---------------------------------------------------------------------------------------------
# cases


def listed():
    return [
        # one query's tokens at serving time: latency counts
        dict(name="embed_query", op="embed", V=32768, D=128, B=1, L=16, dtype="bf16", ids=64),
        # a batch of passages while a corpus is encoded
        dict(name="embed_corpus", op="embed", V=65536, D=960, B=512, L=256, dtype="bf16", ids=64),
        # a small training step on a small model, ragged
        dict(name="embed_grad_step", op="embed_grad", V=32768, D=128, B=64, L=37, dtype="f32", ids=64),
        # a large training step; frequent tokens have thousands of rows each
        dict(name="embed_grad_batch", op="embed_grad", V=65536, D=768, B=1024, L=128, dtype="bf16", ids=64),
        # one query's vector at serving time
        dict(name="norm_query", op="norm", rows=1, D=960, dtype="f32"),
        # the tokens of a training batch, forward and backward
        dict(name="norm_train_batch", op="norm_train", rows=131072, D=768, dtype="bf16"),
        # the small tensors of an encoder: norms, biases, projections of odd sizes
        dict(name="adamw_small", op="adamw", tensors=26, largest=100_000, dtype="f32", grad="f32", bits=32),
        # an encoder with its table, gradients from a mixed-precision backward pass
        dict(name="adamw_table", op="adamw", tensors=14, largest=50_331_648, dtype="f32", grad="bf16", bits=32),
        # the same with both moments in 8 bits
        dict(name="adamw_table8", op="adamw", tensors=14, largest=50_331_648, dtype="f32", grad="f32", bits=8),
        # one query's vector through the projection: the weight is read for one row
        dict(name="linear_query", op="linear", M=1, N=1024, K=960, dtype="bf16"),
        # nothing round: rows, columns, and a last block of K that is not whole
        dict(name="linear_ragged", op="linear", M=1237, N=777, K=1000, dtype="f32"),
        # a batch of a corpus through a wide projection
        dict(name="linear_corpus", op="linear", M=8192, N=4096, K=4096, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the listed ones' ranges, no dearer than the largest of its operator: 1 to
    131,072 tokens or rows, tables of 1,000 to 131,072 rows, vectors of 33 to 2,048 dimensions,
    1 to 40 tensors of up to 50 million elements, products of 1 to 8,192 rows."""
    op = rng.choice(["embed", "embed_grad", "embed_grad", "norm", "norm_train", "norm_train", "adamw", "adamw",
                     "linear", "linear", "linear"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    D = rng.choice([33, 64, 96, 100, 128, 200, 256, 333, 384, 500, 512, 768, 960, 1024, 2048, _log_int(rng, 33, 2048)])
    if op in ("embed", "embed_grad"):
        n = _log_int(rng, 1, 131_072)
        L = max(1, min(n, _log_int(rng, 1, 512)))
        V = _log_int(rng, 1000, 131_072)
        if op == "embed":  # bytes written at most those of embed_corpus
            n = min(n, 512 * 256 * 960 * 2 // (D * BYTES[dtype]))
        else:              # bytes read and written at most those of embed_grad_batch
            V = min(V, 65536 * 768 * 2 // (D * BYTES[dtype]))
            n = min(n, 131_072 * 768 * 2 // (D * BYTES[dtype]))
        return dict(op=op, V=V, D=D, B=max(1, n // L), L=L, dtype=dtype, ids=rng.choice([32, 64, 64]))
    if op in ("norm", "norm_train"):
        rows = min(_log_int(rng, 1, 131_072), 131_072 * 768 * 2 // (D * BYTES[dtype]))
        return dict(op=op, rows=rows, D=D, dtype=dtype)
    if op == "adamw":
        return dict(op=op, tensors=rng.randint(1, 40), largest=_log_int(rng, 500, 50_000_000),
                    dtype=rng.choice(["f32", "f32", "bf16"]), grad=rng.choice(["f32", "bf16", "f16"]),
                    bits=rng.choice([32, 8]))
    M, N, K = _log_int(rng, 1, 8192), _log_int(rng, 64, 8192), _log_int(rng, 64, 8192)
    if rng.random() < 0.5:
        N, K = max(64, N // 128 * 128), max(64, K // 128 * 128)
    M = max(1, min(M, 8192 * 4096 * 4096 // (N * K)))
    return dict(op=op, M=M, N=N, K=K, dtype=dtype)


def _sizes(case):
    """Elements of each tensor of an optimizer case: the largest first, then norms, biases and
    projections of falling, mostly odd sizes, all together no more than the largest."""
    n, left, out = case["largest"], case["largest"], [case["largest"]]
    for i in range(1, case["tensors"]):
        s = max(1, n // (4 * i * i + 5) + (0 if i % 3 == 0 else 2 * i + 1))
        s = min(s, max(1, left // 2))
        left -= s
        out.append(s)
    return out


def _lengths(case):
    """Tokens of each sequence of a padded batch, between half and all of its slots."""
    L, B = case["L"], case["B"]
    return [L - (7919 * b + 3) % (L // 2 + 1) for b in range(B)]


def work(case):
    op = case["op"]
    if op in ("embed", "embed_grad"):
        n, D, es = case["B"] * case["L"], case["D"], BYTES[case["dtype"]]
        live = sum(_lengths(case))
        ids = n * (8 if case["ids"] == 64 else 4)
        if op == "embed":
            return {"bytes": min(live, case["V"]) * D * es + ids + n * D * es, "flops": live * D}
        return {"bytes": live * D * es + ids + case["V"] * D * es, "flops": 2 * live * D}
    if op in ("norm", "norm_train"):
        nd, es = case["rows"] * case["D"], BYTES[case["dtype"]]
        if op == "norm":
            return {"bytes": 2 * nd * es + 2 * case["D"] * es, "flops": 8 * nd}
        return {"bytes": 4 * nd * es + 3 * case["D"] * es, "flops": 24 * nd}
    if op == "adamw":
        n = sum(_sizes(case))
        state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8  # the 8-bit states' values come back too
        return {"bytes": n * (2 * BYTES[case["dtype"]] + BYTES[case["grad"]] + state), "flops": 14 * n}
    M, N, K, es = case["M"], case["N"], case["K"], BYTES[case["dtype"]]
    return {"bytes": M * K * es + N * K * (1 + 1 / 128) + N * es + M * N * es, "flops": 2 * M * N * K}


# ---------------------------------------------------------------------------------------------
# inputs


def _rand(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _token_ids(case, g):
    """A padded batch: frequencies fall as one over the rank, as a vocabulary's do; -1 past a
    sequence's end."""
    B, L, V = case["B"], case["L"], case["V"]
    u = torch.rand((B, L), generator=g, device=DEV, dtype=torch.float64)
    ids = (torch.exp(u * math.log(V + 1)).long() - 1).clamp_(0, V - 1)
    lens = torch.tensor(_lengths(case), device=DEV)
    ids[torch.arange(L, device=DEV)[None, :] >= lens[:, None]] = -1
    return ids.to(torch.int64 if case["ids"] == 64 else torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 29)
    op, dt = case["op"], TYPES[case.get("dtype", "f32")]
    if op == "embed":
        w = (0.02 * _rand(g, case["V"], case["D"])).to(dt)
        return dict(op=op, ids=_token_ids(case, g), weight=w, scale=math.sqrt(case["D"]))
    if op == "embed_grad":
        ids = _token_ids(case, g)
        grad = (1e-2 * _rand(g, case["B"], case["L"], case["D"])).to(dt)
        return dict(op=op, ids=ids, grad=grad, rows=case["V"], scale=math.sqrt(case["D"]))
    if op in ("norm", "norm_train"):
        n, D = case["rows"], case["D"]
        x = ((1.0 + torch.rand((n, 1), generator=g, device=DEV)) * _rand(g, n, D) + 0.5 * _rand(g, n, 1)).to(dt)
        s = dict(op=op, x=x, weight=(1.0 + 0.1 * _rand(g, D)).to(dt), bias=(0.1 * _rand(g, D)).to(dt), eps=1e-5)
        if op == "norm_train":
            s["grad"] = (1e-2 * _rand(g, n, D)).to(dt)
        return s
    if op == "adamw":
        gt = TYPES[case["grad"]]
        sizes = _sizes(case)
        params = [(0.02 * _rand(g, n)).to(dt) for n in sizes]
        grads = [(1e-3 * _rand(g, n) * torch.exp(_rand(g, n))).to(gt) for n in sizes]
        # the states are flat: tensor i's begin at a whole block, the gaps hold zeros
        starts, total = [], 0
        for n in sizes:
            starts.append(total)
            total += -(-n // BLOCK) * BLOCK
        slots = torch.cat([torch.arange(a, a + n, device=DEV) for a, n in zip(starts, sizes)])
        m, v = torch.zeros(total, device=DEV), torch.zeros(total, device=DEV)
        m[slots] = 1e-3 * _rand(g, slots.numel())
        v[slots] = (1e-3 * _rand(g, slots.numel())).square() + 1e-9
        s = dict(op=op, bits=case["bits"], params=params, grads=grads, slots=slots, sizes=sizes)
        if case["bits"] == 32:
            s.update(m=m, v=v)
        else:  # as a step before this one left them
            s["m"], s["m_scale"] = _encode_m(m)
            s["v"], s["v_scale"] = _encode_v(v)
        if own:  # the optimizer a program keeps, in the same state
            from trident_amd import encoder
            opt = encoder.AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                                state_bits=case["bits"])
            opt.load_state(STEP - 1, s["m"], s["v"], s.get("m_scale"), s.get("v_scale"))
            s["optimizer"] = opt
        return s
    x = (_rand(g, case["M"], case["K"]) * torch.exp(0.5 * _rand(g, case["M"], 1))).to(dt)
    codes, scales = _quantize(_rand(g, case["N"], case["K"]) / math.sqrt(case["K"]))
    return dict(op=op, x=x, codes=codes, scales=scales, K=case["K"], bias=(0.1 * _rand(g, case["N"])).to(dt))


# ---------------------------------------------------------------------------------------------
# one pass


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from trident_amd import encoder
    op = s["op"]
    if op == "embed":
        return encoder.embedding(s["ids"], s["weight"], scale=s["scale"])
    if op == "embed_grad":
        return encoder.embedding_grad(s["grad"], s["ids"], s["rows"], scale=s["scale"])
    if op == "norm":
        return encoder.layer_norm(s["x"], s["weight"], s["bias"], eps=s["eps"])
    if op == "norm_train":
        y, mean, rstd = encoder.layer_norm_forward(s["x"], s["weight"], s["bias"], eps=s["eps"])
        dx, dw, db = encoder.layer_norm_grad(s["grad"], s["x"], s["weight"], mean, rstd)
        return dict(y=y, dx=dx, dw=dw, db=db)
    if op == "adamw":
        opt = s["optimizer"]
        opt.step_count = STEP - 1  # the same step each pass
        opt.step(s["grads"])
        m, v = opt.state_values()
        return dict(params=s["params"], m=m, v=v)
    # results of 16 bits take the 8-bit matrix instruction's sums, float32 ones float32 sums
    return encoder.fp8_linear(s["x"], encoder.Fp8Blocks(s["codes"], s["scales"], s["K"]), s["bias"],
                              fast_accum=s["x"].dtype != torch.float32)


def _run_plain(s):
    op = s["op"]
    if op == "embed":
        ids = s["ids"].long()
        y = s["weight"][ids.clamp(min=0)].float() * s["scale"]
        return torch.where((ids >= 0)[..., None], y, 0.0).to(s["weight"].dtype)
    if op == "embed_grad":
        ids, D = s["ids"].long().reshape(-1), s["grad"].shape[-1]
        out = torch.zeros((s["rows"] + 1, D), device=DEV)  # the last row takes the empty slots
        out.index_add_(0, torch.where(ids >= 0, ids, s["rows"]), s["grad"].reshape(-1, D).float())
        return (out[:-1] * s["scale"]).to(s["grad"].dtype)
    if op in ("norm", "norm_train"):
        x, w = s["x"].float(), s["weight"].float()
        c = x - x.mean(1, keepdim=True)
        rstd = torch.rsqrt(c.square().mean(1, keepdim=True) + s["eps"])
        h = c * rstd
        y = (h * w + s["bias"].float()).to(s["x"].dtype)
        if op == "norm":
            return y
        dy = s["grad"].float()
        a = dy * w
        dx = rstd * (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True))
        dt = s["x"].dtype
        return dict(y=y, dx=dx.to(dt), dw=(dy * h).sum(0).to(dt), db=dy.sum(0).to(dt))
    if op == "adamw":
        return _adamw_plain(s)
    codes, scales = _quantize(s["x"].float())
    y = _dequantize(codes, scales, s["K"]) @ _dequantize(s["codes"], s["scales"], s["K"]).t()
    return (y + s["bias"].float()).to(s["x"].dtype)


def _adamw_plain(s):
    slots, bits = s["slots"], s["bits"]
    m, v = (s["m"], s["v"]) if bits == 32 else (_decode_m(s["m"], s["m_scale"]), _decode_v(s["v"], s["v_scale"]))
    g, p = torch.zeros_like(m), torch.zeros_like(m)
    g[slots] = torch.cat(s["grads"]).float()
    p[slots] = torch.cat(s["params"]).float()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    denom = torch.sqrt(v) * (1 / math.sqrt(1 - BETA2 ** STEP)) + EPS
    p = p * (1 - LR * DECAY) - (LR / (1 - BETA1 ** STEP)) * (m / denom)
    parts = torch.split(p[slots], s["sizes"])
    _ = [old.copy_(new) for old, new in zip(s["params"], parts)]
    if bits == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return dict(params=s["params"], m=s["m"], v=s["v"])
    s["m"], s["m_scale"] = _encode_m(m)
    s["v"], s["v_scale"] = _encode_v(v)
    return dict(params=s["params"], m=_decode_m(s["m"], s["m_scale"]), v=_decode_v(s["v"], s["v_scale"]))


# The 8-bit states, for blocks of 256 elements: the first moment as sign(c) c^2 times the block's
# largest value over 127^2, the second moment's root as c^2 times the block's largest root over
# 255^2, at least 1 where the moment is not 0.


def _factor(top, levels):
    """What maps a block's largest value to `levels`; 0 for a block without one."""
    return torch.where(top >= 2.0 ** -100, top.reciprocal() * levels, 0.0)


def _encode_m(m):
    b = m.view(-1, BLOCK)
    top = b.abs().amax(1, keepdim=True)
    c = torch.sqrt(b.abs() * _factor(top, 16129.0)).round().clamp(max=127.0)
    scale = torch.where(top >= 2.0 ** -100, top * (1 / 16129), 0.0)
    return torch.where(b < 0, -c, c).to(torch.int8).view(-1), scale.view(-1)


def _decode_m(codes, scale):
    c = codes.view(-1, BLOCK).float()
    return (c * c.abs() * scale[:, None]).view(-1)


def _encode_v(v):
    b = torch.sqrt(v).view(-1, BLOCK)
    top = b.amax(1, keepdim=True)
    c = torch.sqrt(b * _factor(top, 65025.0)).round().clamp(max=255.0)
    c = torch.where((b > 0) & (top >= 2.0 ** -100), c.clamp(min=1.0), c)
    scale = torch.where(top >= 2.0 ** -100, top * (1 / 65025), 0.0)
    return c.to(torch.uint8).view(-1), scale.view(-1)


def _decode_v(codes, scale):
    c = codes.view(-1, BLOCK).float()
    r = c * c * scale[:, None]
    return (r * r).view(-1)


# 8-bit floating point (e4m3) in blocks of 128 columns: the scale is 2^e, the least with the block's
# largest value <= 448 * 2^e, stored as e + 127.  Codes are padded with zeros to whole blocks, rows of
# scales to a multiple of four.


def _power(e):
    return ((e + 127) << 23).view(torch.float32)


def _quantize(x):
    M, K = x.shape
    kb = -(-K // 128)
    b = torch.nn.functional.pad(x, (0, kb * 128 - K)).view(M, kb, 128)
    f, e = torch.frexp(b.abs().amax(2))
    e = torch.where(f == 0, 0, (e - 9 + (f > 0.875).int()).clamp(min=-126)).int()
    codes = (b * _power(-e)[..., None]).to(torch.float8_e4m3fn).view(M, kb * 128)
    scales = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, -kb % 4), value=127)
    return codes, scales


def _dequantize(codes, scales, K):
    M, Kp = codes.shape
    e = scales[:, :Kp // 128].int() - 127
    return (codes.float().view(M, -1, 128) * _power(e)[..., None]).view(M, Kp)[:, :K]


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op, f64 = s["op"], torch.float64
    if op == "embed":
        out = torch.zeros((*s["ids"].shape, case["D"]), dtype=f64, device=DEV)
        live = s["ids"] >= 0
        out[live] = s["weight"].to(f64).index_select(0, s["ids"][live].long()) * s["scale"]
        return out
    if op == "embed_grad":
        live = s["ids"] >= 0
        out = torch.zeros((case["V"], case["D"]), dtype=f64, device=DEV)
        return out.index_add_(0, s["ids"][live].long(), s["grad"][live].to(f64), alpha=s["scale"])
    if op in ("norm", "norm_train"):
        x, w, b = s["x"].to(f64), s["weight"].to(f64), s["bias"].to(f64)
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        sigma = torch.sqrt(var + s["eps"])
        h = (x - mean) / sigma
        y = w * h + b
        if op == "norm":
            return y
        dy = s["grad"].to(f64)
        D = case["D"]
        dh = dy * w
        dx = (D * dh - dh.sum(1, keepdim=True) - h * (dh * h).sum(1, keepdim=True)) / (D * sigma)
        return dict(y=y, dx=dx, dw=torch.einsum("nd,nd->d", dy, h), db=torch.einsum("nd->d", dy))
    if op == "adamw":
        return _exact_adamw(s)
    wq = _exact_blocks(s["codes"].to(f64), s["scales"], case["K"])
    x = s["x"].to(f64)
    K = case["K"]
    out = s["bias"].to(f64).expand(case["M"], case["N"]).clone()
    for k in range(0, K, 128):
        b = x[:, k:k + 128]
        top = b.abs().amax(1, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448.0)).clamp(min=-126))
        q = b / scale
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)  # three bits after the first
        out += (torch.round(q / step) * step * scale) @ wq[:, k:k + 128].t()
    return out


def _exact_blocks(values, scales, K):
    e = scales.to(torch.float64)[:, :values.shape[1] // 128] - 127
    return (values * torch.exp2(e).repeat_interleave(128, dim=1))[:, :K]


def _exact_adamw(s):
    f64 = torch.float64
    T = s["m"].numel()
    if s["bits"] == 32:
        m, v = s["m"].to(f64), s["v"].to(f64)
    else:
        cm, cv = s["m"].to(f64), s["v"].to(f64)
        m = torch.sign(cm) * cm ** 2 * s["m_scale"].to(f64).repeat_interleave(BLOCK)
        v = (cv ** 2 * s["v_scale"].to(f64).repeat_interleave(BLOCK)) ** 2
    params, at = [], 0
    live = torch.zeros(T, dtype=torch.bool, device=DEV)
    for p, g in zip(s["params"], s["grads"]):
        n = p.numel()
        a = slice(at, at + n)
        live[a] = True
        g64 = g.to(f64)
        m[a] = BETA1 * m[a] + (1 - BETA1) * g64
        v[a] = BETA2 * v[a] + (1 - BETA2) * g64 ** 2
        m_hat, v_hat = m[a] / (1 - BETA1 ** STEP), v[a] / (1 - BETA2 ** STEP)
        params.append(p.to(f64) - LR * DECAY * p.to(f64) - LR * m_hat / (torch.sqrt(v_hat) + EPS))
        at += -(-n // BLOCK) * BLOCK
    if s["bits"] == 8:
        blocks = m.view(-1, BLOCK)
        top = blocks.abs().amax(1, keepdim=True)
        unit = torch.where(top > 0, top, 1.0)
        m = (torch.sign(blocks) * torch.round(127 * torch.sqrt(blocks.abs() / unit)) ** 2 * (top / 127 ** 2)).view(-1)
        root = torch.sqrt(v).view(-1, BLOCK)
        top = root.amax(1, keepdim=True)
        unit = torch.where(top > 0, top, 1.0)
        code = torch.round(255 * torch.sqrt(root / unit))
        code = torch.where(root > 0, code.clamp(min=1), code)
        v = ((code ** 2 * (top / 255 ** 2)) ** 2).view(-1)
    return dict(params=params, m=m, v=v)
