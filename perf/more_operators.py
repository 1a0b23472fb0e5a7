"""What a decoder block computes around its attention, as cases with work in them: the norm of
each query and key head with the position rotation, the gated feed-forward block, and the 8-bit
form in which a training step keeps its activations for the backward pass.

``run`` computes a case either in plain torch operations (``own`` false) or by the calls a
user's program makes of ``dsalt_b200`` (``own`` true). Definitions:

* rope: head ``x`` of a token becomes ``n = w * x / sqrt(mean(x^2) + eps)`` (without weights:
  ``n = x``), then its halves ``(a, b)`` become ``(a cos - b sin, b cos + a sin)`` with the
  angles of the token's position.
* ffn: ``y = (act(x Wg^T) * (x Wu^T)) Wd^T`` with ``act`` silu or gelu (by the error function).
* pack: 32 neighbouring values of a row share a scale ``2^(e - 6)``, ``2^e`` the highest power of
  two that is at most their largest magnitude (``e - 6 >= -126``); a value is held as the
  nearest whole number of steps (ties to even), at most 127 of them.
* ffn with ``keep`` 8: the backward pass takes ``x``, ``x Wg^T`` and ``x Wu^T`` as pack holds them.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
GROUP = 32   # values that share a scale
EPS = 1e-6


def listed():
    return [
        # one request's decode step through one layer's feed-forward block: latency
        dict(name="ffn_token", op="ffn", tokens=1, d_model=1024, d_ff=4096, dtype="bf16", act="silu", train=False,
             keep=16),
        # a decode step of 64 requests, the wide model: the weights are read once
        dict(name="ffn_step_64", op="ffn", tokens=64, d_model=2048, d_ff=11008, dtype="bf16", act="silu", train=False,
             keep=16),
        # a few short prompts together, fp16, an odd number of tokens
        dict(name="ffn_prompts_1999", op="ffn", tokens=1999, d_model=768, d_ff=2048, dtype="fp16", act="gelu",
             train=False, keep=16),
        # one long prompt of the wide model
        dict(name="ffn_prompt_32768", op="ffn", tokens=32768, d_model=2048, d_ff=11008, dtype="bf16", act="silu",
             train=False, keep=16),
        # a training step over a pack of 4 x 8192 tokens, activations kept in the input type
        dict(name="ffn_train_4x8192", op="ffn", tokens=32768, d_model=768, d_ff=2048, dtype="bf16", act="silu",
             train=True, keep=16),
        # a training step over one long sequence, activations kept in 8 bits
        dict(name="ffn_train_8bit", op="ffn", tokens=16384, d_model=1024, d_ff=4096, dtype="bf16", act="silu",
             train=True, keep=8),
        # one layer's hidden states put away in 8 bits and read back
        dict(name="pack_32768", op="pack", rows=32768, cols=2048, dtype="bf16"),
        # a ragged micro-batch in fp32, rows that end inside a group
        dict(name="pack_ragged_fp32", op="pack", rows=1013, cols=1000, dtype="fp32"),
        # a decode step of 64 requests, grouped heads: latency
        dict(name="rope_step_64", op="rope", seqs=64, tokens=1, heads=16, kv_heads=2, head_dim=128, dtype="bf16",
             norm=True, fused=True, train=False),
        # one very long prompt, 16 heads of 64
        dict(name="rope_prompt_131072", op="rope", seqs=1, tokens=131072, heads=16, kv_heads=16, head_dim=64,
             dtype="bf16", norm=True, fused=False, train=False),
        # a training step over a pack of 4 x 8192 tokens, 12 heads of 64
        dict(name="rope_train_4x8192", op="rope", seqs=4, tokens=8192, heads=12, kv_heads=12, head_dim=64,
             dtype="bf16", norm=True, fused=False, train=True),
        # training in fp32, grouped heads cut from one projection, sequences of odd length
        dict(name="rope_train_fp32", op="rope", seqs=3, tokens=1111, heads=16, kv_heads=2, head_dim=128, dtype="fp32",
             norm=True, fused=True, train=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "pack", "rope"])
    if op == "ffn":
        d_model, d_ff = rng.choice([(256, 768), (512, 1408), (768, 2048), (1024, 2816), (1024, 4096), (2048, 5504),
                                    (2048, 11008), (8 * rng.randint(8, 96), 8 * rng.randint(8, 256))])
        train = rng.random() < 0.5
        most = 16384 * 1024 * 4096 // (d_model * d_ff) if train else 32768
        return dict(op=op, tokens=_log_uniform(rng, 16 if train else 1, min(32768, most)), d_model=d_model, d_ff=d_ff,
                    dtype=rng.choice(["bf16", "fp16"]), act=rng.choice(["silu", "silu", "gelu"]), train=train,
                    keep=rng.choice([8, 16]) if train else 16)
    if op == "pack":
        cols = rng.choice([768, 1024, 2048, rng.randint(1, 4096)])
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return dict(op=op, rows=_log_uniform(rng, 1, 32768 * 2048 * 2 // (cols * BYTES[dtype])), cols=cols, dtype=dtype)
    heads, kv_heads, head_dim = rng.choice([(16, 8, 64), (12, 12, 64), (4, 4, 64), (16, 2, 128), (12, 4, 128),
                                            (6, 2, 96), (5, 1, 128), (8, 8, 32), (4, 1, 256)])
    dtype, train = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.5
    seqs = _log_uniform(rng, 1, 64)
    most = 131072 * 2048 // ((heads + kv_heads) * head_dim) // (BYTES[dtype] // 2) // (3 if train else 1)
    return dict(op=op, seqs=seqs, tokens=_log_uniform(rng, 1, min(32768, most // seqs)), heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, norm=rng.random() < 0.75, fused=rng.random() < 0.5,
                train=train)


# ---------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"ffn": _prepare_ffn, "pack": _prepare_pack, "rope": _prepare_rope}[case["op"]](case, g)


def _normal(g, shape, dtype, scale=1.0):
    return torch.empty(shape, device="cuda").normal_(0.0, scale, generator=g).to(dtype)


def _prepare_ffn(case, g):
    T, d, F, dt = case["tokens"], case["d_model"], case["d_ff"], DTYPES[case["dtype"]]
    s = dict(case=case, x=_normal(g, (T, d), dt), w_gate=_normal(g, (F, d), dt, 1.0 / math.sqrt(d)),
             w_up=_normal(g, (F, d), dt, 1.0 / math.sqrt(d)), w_down=_normal(g, (d, F), dt, 1.0 / math.sqrt(F)))
    if case["train"]:
        s["dy"] = _normal(g, (T, d), dt, 0.05)
        for name in ("x", "w_gate", "w_up", "w_down"):
            s[name].requires_grad_(True)
    return s


def _prepare_pack(case, g):
    shape = (case["rows"], case["cols"])
    # hidden states: a few channels are much larger than the others
    x = torch.empty(shape, device="cuda").normal_(generator=g)
    channel = torch.exp(torch.empty(case["cols"], device="cuda").normal_(0.0, 1.0, generator=g))
    return dict(case=case, x=(x * channel).to(DTYPES[case["dtype"]]))


def _prepare_rope(case, g):
    S, L, H, Hk, D, dt = (case[n] for n in ("seqs", "tokens", "heads", "kv_heads", "head_dim", "dtype"))
    dt = DTYPES[dt]
    # the lengths are the case's, whatever the seed: they are the sizes of its tensors
    fixed = torch.Generator().manual_seed(S * 131071 + L)
    lens = torch.randint((L + 1) // 2, L + 1, (S,), generator=fixed) if S > 1 and L > 1 else torch.full((S,), L)
    T = int(lens.sum())
    if L == 1:  # single tokens: far along, each at its own place
        positions = torch.randint(0, 32768, (S,), generator=g, device="cuda", dtype=torch.int32)
    else:
        positions = torch.cat([torch.arange(int(n)) for n in lens]).to(torch.int32).cuda()
    table = max(L, 32768)
    theta = 10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    angles = torch.outer(torch.arange(table, device="cuda", dtype=torch.float64), theta)
    cos, sin = (torch.cat([t, t], 1).float() for t in (angles.cos(), angles.sin()))
    s = dict(case=case, positions=positions, cos=cos, sin=sin, q_weight=None, k_weight=None)
    if case["fused"]:  # queries, keys and values of one projection
        qkv = _normal(g, (T, H + 2 * Hk, D), dt)
        s["q"], s["k"] = qkv[:, :H], qkv[:, H:H + Hk]
    else:
        s["q"], s["k"] = _normal(g, (T, H, D), dt), _normal(g, (T, Hk, D), dt)
    if case["norm"]:
        s["q_weight"], s["k_weight"] = (torch.rand(D, device="cuda", generator=g) + 0.5 for _ in range(2))
    if case["train"]:
        s["dq"], s["dk"] = _normal(g, (T, H, D), dt), _normal(g, (T, Hk, D), dt)
        s["leaves"] = [s[n].detach().requires_grad_(True) for n in ("q", "k")]
        s["q"], s["k"] = s["leaves"]
        if case["norm"]:
            for n in ("q_weight", "k_weight"):
                s["leaves"].append(s[n].requires_grad_(True))
    return s


# ---------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"ffn": _plain_ffn, "pack": _plain_pack, "rope": _plain_rope}[state["case"]["op"]](state)


def _run_own(s):
    import dsalt_b200 as D

    case = s["case"]
    if case["op"] == "pack":
        codes, exps = D.pack8(s["x"])
        return [D.unpack8(codes, exps, s["x"].dtype)]
    if case["op"] == "rope":
        out = D.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], positions=s["positions"], q_weight=s["q_weight"],
                             k_weight=s["k_weight"], eps=EPS)
        if not case["train"]:
            return list(out)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, s["leaves"], (s["dq"], s["dk"])))
    y = D.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], activation=case["act"], keep=f"{case['keep']}bit")
    if not case["train"]:
        return [y]
    return [y.detach()] + list(torch.autograd.grad(y, (s["x"], s["w_gate"], s["w_up"], s["w_down"]), s["dy"]))


def _act(g, act):
    """The activation and its derivative."""
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-g))
        return g * p, p * (1.0 + g * (1.0 - p))
    p = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * p, p + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _held(x):
    """What `x` (32 bits) becomes when it is held in 8 bits."""
    rows, n = x.shape
    pad = -n % GROUP
    b = torch.cat([x, x.new_zeros(rows, pad)], 1).view(rows, -1, GROUP)
    e = (torch.frexp(b.abs().amax(-1, keepdim=True))[1] - 7).clamp(min=-126)
    return ((b * _power(-e)).round().clamp(-127, 127) * _power(e)).view(rows, -1)[:, :n]


def _power(e):
    """2^e, exactly."""
    return ((e + 127) << 23).view(torch.float32)


def _plain_ffn(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu, wd = (s[n].float() for n in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(g, case["act"])
    y = ((a * u) @ wd.T).to(dt)
    if not case["train"]:
        return [y]
    dy = s["dy"].float()
    if case["keep"] == 8:
        x, g, u = _held(x), _held(g), _held(u)
        a, da = _act(g, case["act"])
    dh = dy @ wd
    d_wd = dy.T @ (a * u)
    dg, du = dh * u * da, dh * a
    return [y] + [t.to(dt) for t in (dg @ wg + du @ wu, dg.T @ x, du.T @ x, d_wd)]


def _plain_pack(s):
    return [_held(s["x"].float()).to(s["x"].dtype)]


def _plain_rope(s):
    case, at = s["case"], s["positions"].long()
    half = case["head_dim"] // 2
    cos, sin = s["cos"][at, None, :half], s["sin"][at, None, :half]
    out, grads, w_grads = [], [], []
    for name in ("q", "k"):
        x, w = s[name].float(), s[name + "_weight"]
        n = x
        if w is not None:
            r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            n = w * (x * r)
        a, b = n[..., :half], n[..., half:]
        out.append(torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(s[name].dtype))
        if case["train"]:
            dt = s["d" + name].float()
            a, b = dt[..., :half], dt[..., half:]
            dn = torch.cat([a * cos + b * sin, b * cos - a * sin], -1)
            if w is not None:
                xr = x * r
                w_grads.append((dn * xr).double().sum((0, 1)).float())
                dn = dn * w
                dn = r * (dn - xr * (dn * xr).mean(-1, keepdim=True))
            grads.append(dn.to(s[name].dtype))
    return out + grads + w_grads


# ---------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        return {"ffn": _exact_ffn, "pack": _exact_pack, "rope": _exact_rope}[case["op"]](case, s)


def _steps64(x):
    """The 8-bit form of a 64-bit matrix, group by group of its columns."""
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], GROUP):
        part = x[:, c:c + GROUP]
        top = part.abs().amax(1, keepdim=True)
        e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
        e = torch.where(torch.exp2(e) > top, e - 1, e)          # a logarithm that was rounded up
        e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)      # or down
        step = torch.exp2(torch.where(top > 0, e - 6, -126.0).clamp(min=-126.0))
        out[:, c:c + GROUP] = torch.round(part / step).clamp(-127, 127) * step
    return out


def _exact_ffn(case, s):
    x, wg, wu, wd = (s[n].double() for n in ("x", "w_gate", "w_up", "w_down"))

    def gate(g):
        if case["act"] == "silu":
            p = torch.sigmoid(g)
            return p, p * (1 - p)
        return torch.special.ndtr(g), torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)

    y = torch.empty(x.shape[0], wd.shape[0], device=x.device, dtype=x.dtype)
    if case["train"]:
        dx, d_wg, d_wu, d_wd = torch.empty_like(x), torch.zeros_like(wg), torch.zeros_like(wu), torch.zeros_like(wd)
    for t in range(0, x.shape[0], 4096):
        part = slice(t, t + 4096)
        xs = x[part]
        g, u = torch.mm(xs, wg.t()), torch.mm(xs, wu.t())
        y[part] = torch.mm(g * gate(g)[0] * u, wd.t())
        if case["train"]:
            if case["keep"] == 8:
                xs, g, u = _steps64(xs), _steps64(g), _steps64(u)
            p, dp = gate(g)
            dy = s["dy"][part].double()
            dh = torch.mm(dy, wd)
            dg, du = dh * u * (p + g * dp), dh * g * p
            dx[part] = torch.mm(dg, wg) + torch.mm(du, wu)
            d_wg += torch.mm(dg.t(), xs)
            d_wu += torch.mm(du.t(), xs)
            d_wd += torch.mm(dy.t(), g * p * u)
    return [y, dx, d_wg, d_wu, d_wd] if case["train"] else [y]


def _exact_pack(case, s):
    return [_steps64(s["x"].double())]


def _exact_rope(case, s):
    D = case["head_dim"]
    at = s["positions"].long()
    # a head's halves are the real and imaginary parts of D / 2 numbers, turned by the position's angles
    turn = torch.complex(s["cos"].double()[at, :D // 2], s["sin"].double()[at, :D // 2]).unsqueeze(1)
    out, grads, w_grads = [], [], []
    for name in ("q", "k"):
        x, w = s[name].double(), s[name + "_weight"]
        rms = torch.sqrt(x.square().sum(-1, keepdim=True) / D + EPS) if w is not None else torch.ones_like(x[..., :1])
        weight = w.double() if w is not None else torch.ones(D, device=x.device, dtype=x.dtype)
        unit = x / rms
        n = unit * weight
        z = torch.complex(n[..., :D // 2], n[..., D // 2:]) * turn
        out.append(torch.cat([z.real, z.imag], -1))
        if case["train"]:
            d = s["d" + name].double()
            z = torch.complex(d[..., :D // 2], d[..., D // 2:]) * turn.conj()
            dn = torch.cat([z.real, z.imag], -1)
            if w is not None:
                w_grads.append((dn * unit).sum((0, 1)))
                dn = dn * weight
                dn = (dn - unit * (dn * unit).sum(-1, keepdim=True) / D) / rms
            grads.append(dn)
    return out + grads + w_grads


# ---------------------------------------------------------------------- work
def work(case):
    es = BYTES[case["dtype"]]
    if case["op"] == "ffn":
        T, d, F = case["tokens"], case["d_model"], case["d_ff"]
        if not case["train"]:
            return {"bytes": es * (2 * T * d + 3 * d * F), "flops": 6 * T * d * F}
        # x, y, dy, dx and three weights with their gradients; three products forward, six backward
        return {"bytes": es * (4 * T * d + 6 * d * F), "flops": 18 * T * d * F}
    if case["op"] == "pack":
        n, groups = case["rows"] * case["cols"], case["rows"] * -(-case["cols"] // GROUP)
        return {"bytes": n * (2 * es + 2) + 2 * groups, "flops": 4 * n}
    S, L, H, Hk, D = (case[n] for n in ("seqs", "tokens", "heads", "kv_heads", "head_dim"))
    fixed = torch.Generator().manual_seed(S * 131071 + L)
    lens = torch.randint((L + 1) // 2, L + 1, (S,), generator=fixed) if S > 1 and L > 1 else torch.full((S,), L)
    T = int(lens.sum())
    n = T * (H + Hk) * D
    angles = 4 * D * min(T, 32768 if L == 1 else int(lens.max()))
    # forward: q, k in and out; backward: their gradients in and out and q, k once more
    return {"bytes": es * n * (5 if case["train"] else 2) + angles + 4 * T, "flops": n * (20 if case["train"] else 8)}
