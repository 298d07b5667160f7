"""Work of the operators around the shared products of a layer, as cases that can be timed and checked.

Each case is one pass through public entry points of lastengine_amd.Engine, or the same result in plain torch:

  norm      the residual's addition, RMS norm and int8 activations with a scale per 32 values, for many tokens
  lora      low-rank adapters of many requests beside a shared projection: each token has an adapter of its own, or none
  experts   the products of the experts that a router picked, dense weights, rows grouped by expert
  gradient  the gradients of those products: of their rows and of their weights

Sizes are those of this package's benchmark: hidden 4096 with 14336 (dense), hidden 2048 with 768 and 128 experts of
which a token takes 8 (experts), or between them.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
MOST = 32768 * 1536 * 2048  # products of rows, outputs and inputs in the largest call of the experts
_engine = None


def _eng():
    """The program's one Engine (it loads the code objects)."""
    global _engine
    if _engine is None:
        import lastengine_amd as le
        _engine = le.Engine()
    return _engine


def _ty(name):
    import lastengine_amd as le
    return {"f32": le.F32, "f16": le.F16, "bf16": le.BF16}[name]


# ---------------------------------------------------------------- the cases

def _norm(tokens, cols, x, res=True, normed=True):
    """res: a residual is added first. normed: the normed rows are wanted beside the int8 ones (by a router, an adapter)."""
    return {"kind": "norm", "tokens": tokens, "cols": cols, "x": x, "res": res, "normed": normed}


def _lora(tokens, rows, cols, rank, n_ad, x, w, requests, bare=0.1):
    """requests: in how many runs of consecutive tokens the tokens come, each with an adapter; bare: how many of those have none."""
    return {"kind": "lora", "tokens": tokens, "rows": rows, "cols": cols, "rank": rank, "n_ad": n_ad, "x": x, "w": w, "requests": requests, "bare": bare}


def _experts(kind, tokens, k, n_exp, rows, cols, x, pad=0.0, dw=None):
    """pad: the share of tokens at the end that no expert takes. dw: the type of the weights' gradient."""
    case = {"kind": kind, "tokens": tokens, "k": k, "n_exp": n_exp, "rows": rows, "cols": cols, "x": x, "pad": pad}
    return dict(case, dw=dw or x) if kind == "gradient" else case


def listed():
    return [
        # the smallest call: one decoded token before a dense layer's int8 products; the launch is most of the time
        dict(_norm(1, 4096, "f32", normed=False), name="norm_decode"),
        # a batch of decoding requests before a routed block: the router reads the normed rows
        dict(_norm(37, 2048, "bf16"), name="norm_batch"),
        # a prompt
        dict(_norm(4096, 4096, "f32"), name="norm_prompt"),
        # one decoded token with an adapter beside a quantized projection
        dict(_lora(1, 4096, 4096, 16, 8, "f32", "f16", 1, 0.0), name="lora_decode"),
        # a batch of decoding requests, most with an adapter of their own, beside gate and up
        dict(_lora(61, 28672, 4096, 16, 48, "bf16", "bf16", 61), name="lora_batch"),
        # drafted tokens of a few requests in verify, an odd rank, beside down
        dict(_lora(15, 4096, 14336, 12, 6, "f16", "f16", 3, 0.0), name="lora_verify"),
        # prompts of several requests in one call
        dict(_lora(4096, 4096, 4096, 64, 8, "f32", "bf16", 9), name="lora_prompt"),
        # eight decoded tokens, each with its own eight of 128 experts: gate and up rows
        dict(_experts("experts", 8, 8, 128, 1536, 2048, "bf16"), name="experts_decode"),
        # down over a prompt of odd length, padded at its end
        dict(_experts("experts", 1021, 8, 128, 2048, 768, "f16", 0.1), name="experts_ragged"),
        # gate and up over a long prompt
        dict(_experts("experts", 4096, 8, 128, 1536, 2048, "bf16", 0.1), name="experts_prompt"),
        # training steps: a ragged micro-batch whose rows end anywhere, and a full one
        dict(_experts("gradient", 301, 6, 60, 515, 1001, "f32", 0.1), name="gradient_ragged"),
        dict(_experts("gradient", 4096, 8, 128, 1536, 2048, "bf16", 0.1), name="gradient_full"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "lora", "lora", "experts", "experts", "gradient"])
    x = rng.choice(["f32", "f16", "bf16"])
    if kind == "norm":
        return _norm(_log(rng, 1, 4096), 32 * _log(rng, 4, 128), x, rng.random() < 0.8, rng.random() < 0.6)
    if kind == "lora":
        tokens, n_ad = _log(rng, 1, 4096), _log(rng, 1, 64)
        few = tokens <= 64
        rows, cols = (rng.choice([_log(rng, 64, 28672 if few else 4096), 8 * _log(rng, 8, 3584 if few else 512)]) for _ in range(2))
        rank = rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 64)])
        while rank * n_ad * (rows + cols) > 1 << 26:
            n_ad = max(1, n_ad // 2)
            rows, cols = rows if n_ad > 1 else rows // 2, cols
        return _lora(tokens, rows, cols, rank, n_ad, x, rng.choice([x, x, "f16", "bf16", "f32"]), min(tokens, _log(rng, 1, 64)), rng.choice([0.0, 0.1, 0.5]))
    n_exp = _log(rng, 4, 128)
    k = rng.randint(1, min(8, n_exp))
    rows, cols = (rng.choice([_log(rng, 48, 2048), 8 * _log(rng, 8, 256)]) for _ in range(2))
    most = MOST // (8 if x == "f32" else 1) // (rows * cols * k)
    return _experts(kind, min(_log(rng, 1, 4096), max(1, most)), k, n_exp, rows, cols, x, rng.choice([0.0, 0.0, 0.1, 0.5]), rng.choice([x, "f32"]))


# ---------------------------------------------------------------- inputs

def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * std


def _activations(gen, rows, cols):
    """Unit rows with a few channels that stand out, as the residual stream has them."""
    big = torch.rand(cols, generator=gen, device="cuda") < 0.004
    return _normal(gen, rows, cols) * torch.where(big, 12.0, 1.0)


def _offsets(gen, case):
    """Where each expert's rows begin, from a router whose experts are not equally popular; padding tokens have no expert."""
    n, e, k = case["tokens"], case["n_exp"], case["k"]
    logits = _normal(gen, n, e) + _normal(gen, e, std=0.4)
    idx = torch.sort(logits, dim=-1, descending=True).indices[:n - int(n * case["pad"]), :k]
    counts = torch.bincount(idx.reshape(-1), minlength=e)
    off = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    off[1:] = counts.cumsum(0)
    return off, int(counts.max())


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    kind, n, cols, ty = case["kind"], case["tokens"], case["cols"], DTYPES[case["x"]]
    if kind == "norm":
        s["x"] = (_activations(gen, n, cols) * 3.0).to(ty)
        s["res"] = _normal(gen, n, cols).to(ty) if case["res"] else None
        s["w"] = 1.0 + _normal(gen, cols, std=0.2)
        s["h"] = torch.empty(n, cols, dtype=ty, device="cuda")
        s["o"] = torch.empty(n, cols, dtype=ty, device="cuda") if case["normed"] else None
        s["xq"] = torch.empty(n, cols // 32, 32, dtype=torch.int8, device="cuda")
        s["xd"] = torch.empty(n, cols // 32, dtype=torch.float32, device="cuda")
        return s
    if kind == "lora":
        rows, rank, n_ad, wt = case["rows"], case["rank"], case["n_ad"], DTYPES[case["w"]]
        s["a"] = _normal(gen, n_ad, rank, cols, std=cols ** -0.5).to(wt)
        s["b"] = _normal(gen, n_ad, rows, rank, std=0.05).to(wt)
        s["scale"] = torch.rand(n_ad, generator=gen, device="cuda") * 1.5 + 0.5
        starts = torch.sort(torch.randperm(n, generator=gen, device="cuda")[:case["requests"]]).values
        which = torch.randint(0, n_ad, (case["requests"] + 1,), generator=gen, device="cuda")
        which = torch.where(torch.rand(case["requests"] + 1, generator=gen, device="cuda") < case["bare"], -1, which)
        s["idx"] = which[torch.searchsorted(starts, torch.arange(n, device="cuda"), right=True)].to(torch.int32)
        s["x"] = _activations(gen, n, cols).to(ty)
        s["base"] = _normal(gen, n, rows).to(ty)
        s["y"] = torch.empty(n, rows, dtype=ty, device="cuda")
        return s
    rows, e, n_row = case["rows"], case["n_exp"], n * case["k"]
    s["off"], s["cap"] = _offsets(gen, case)
    s["x"] = _activations(gen, n_row, cols).to(ty)
    if kind == "experts":
        s["w"] = _normal(gen, e, rows, cols, std=0.02).to(ty)
        s["y"] = torch.zeros(n_row, rows, dtype=ty, device="cuda")
        return s
    s["w"] = _normal(gen, e, rows, cols, std=0.02).to(ty)
    s["dy"] = _normal(gen, n_row, rows, std=0.1).to(ty)
    s["dx"] = torch.zeros(n_row, cols, dtype=ty, device="cuda")
    s["dw"] = torch.empty(e, rows, cols, dtype=DTYPES[case["dw"]], device="cuda")
    return s


# ---------------------------------------------------------------- the plain forms

def _plain_norm(s, case):
    """Which code a value gets turns on its last bit: the sum and the first product in 64 bits, the rest in the 32 bits that define it."""
    n, cols = case["tokens"], case["cols"]
    h = s["x"] if s["res"] is None else (s["x"].float() + s["res"].float()).to(s["x"].dtype)
    v = h.double()
    r = 1.0 / torch.sqrt((v * v).sum(-1, keepdim=True) / cols + EPS)
    o = (v * r).float() * s["w"]
    unit = o.reshape(n, cols // 32, 32)
    # a true division, as the scale is defined: torch divides by a plain number through its reciprocal
    d = unit.abs().amax(-1) / torch.full_like(unit[:1, :1, 0], 127.0)
    q = torch.round(unit * torch.where(d > 0, 1.0 / d, 0.0).unsqueeze(-1))
    return h, o.to(h.dtype) if case["normed"] else None, d, q * d.unsqueeze(-1)


def _plain_lora(s, case):
    """All adapters' first products for every token, those of other adapters masked, then all second products."""
    n, n_ad, rank = case["tokens"], case["n_ad"], case["rank"]
    u = s["x"].float() @ s["a"].float().reshape(n_ad * rank, -1).t()
    mine = s["idx"].unsqueeze(-1) == torch.arange(n_ad, device="cuda")
    u = torch.where(mine.unsqueeze(-1), u.reshape(n, n_ad, rank) * s["scale"].reshape(1, n_ad, 1), 0.0)
    b = s["b"].float().transpose(1, 2).reshape(n_ad * rank, -1)
    return (s["base"].float() + u.reshape(n, n_ad * rank) @ b).to(s["base"].dtype)


def _padded(s, case):
    """For each expert the numbers of its rows, up to the most that any has, and which of them there are."""
    off = s["off"].long()
    at = off[:-1, None] + torch.arange(s["cap"], device="cuda")
    return at.clamp(max=case["tokens"] * case["k"] - 1), at < off[1:, None]


def _back(v, at, live, n_row, ty):
    """The padded rows back in their places; zeros in rows of no expert."""
    out = torch.zeros(n_row + 1, v.shape[-1], device="cuda")
    out[torch.where(live, at, n_row)] = v
    return out[:-1].to(ty)


def _plain(s):
    case = s["case"]
    if case["kind"] == "norm":
        return _plain_norm(s, case)
    if case["kind"] == "lora":
        return _plain_lora(s, case)
    n_row, ty = case["tokens"] * case["k"], s["x"].dtype
    at, live = _padded(s, case)
    x = torch.where(live.unsqueeze(-1), s["x"][at].float(), 0.0)
    w = s["w"].float()
    if case["kind"] == "experts":
        return _back(torch.bmm(x, w.transpose(1, 2)), at, live, n_row, ty)
    dy = torch.where(live.unsqueeze(-1), s["dy"][at].float(), 0.0)
    return _back(torch.bmm(dy, w), at, live, n_row, ty), torch.bmm(dy.transpose(1, 2), x).to(s["dw"].dtype)


# ---------------------------------------------------------------- the framework's calls

def _own(s):
    case, eng = s["case"], _eng()
    kind = case["kind"]
    if "ty" not in s:
        s["ty"] = _ty(case["x"])
        if kind == "lora":
            import lastengine_amd as le
            s["adapters"] = le.Adapters(s["a"], s["b"], s["scale"], case["n_ad"], case["rank"], case["rows"], case["cols"])
    ty, n = s["ty"], case["tokens"]
    if kind == "norm":
        eng.add_rms_quant(ty, s["x"], s["res"], s["w"], s["h"], s["o"], s["xq"], s["xd"], None, n, case["cols"], EPS)
        return s["h"], s["o"], s["xd"], s["xq"] * s["xd"].unsqueeze(-1)
    if kind == "lora":
        eng.lora(ty, s["adapters"], s["idx"], s["x"], s["base"], s["y"], n)
        return s["y"]
    shape = (case["n_exp"], n * case["k"], case["rows"], case["cols"])
    if kind == "experts":
        eng.mm_experts(ty, s["w"], s["off"], s["x"], s["y"], *shape)
        return s["y"]
    eng.mm_experts_dx(ty, s["w"], s["off"], s["dy"], s["dx"], *shape)
    eng.mm_experts_dw(ty, s["dy"], s["x"], s["off"], s["dw"], *shape, dw_ty=_ty(case["dw"]))
    return s["dx"], s["dw"]


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind, n, cols, z = case["kind"], case["tokens"], case["cols"], SIZE[case["x"]]
    if kind == "norm":
        # the int8 values are written once, and given back as what they stand for
        return {"bytes": n * cols * (z * (2 + case["res"] + case["normed"]) + 1 + 4) + n * cols // 8 + cols * 4, "flops": 8 * n * cols}
    if kind == "lora":
        rows, rank = case["rows"], case["rank"]
        live = min(case["n_ad"], max(1, round(case["requests"] * (1 - case["bare"]))))
        return {"bytes": live * rank * (rows + cols) * SIZE[case["w"]] + n * (cols + 2 * rows) * z, "flops": 2 * n * rank * (rows + cols)}
    rows, live = case["rows"], (n - int(n * case["pad"])) * case["k"]
    weights = min(case["n_exp"], live) * rows * cols
    if kind == "experts":
        return {"bytes": weights * z + live * (rows + cols) * z, "flops": 2 * live * rows * cols}
    return {"bytes": weights * z + case["n_exp"] * rows * cols * SIZE[case["dw"]] + live * (rows + 2 * cols) * z, "flops": 4 * live * rows * cols}


# ---------------------------------------------------------------- the same from the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    kind = case["kind"]
    if kind == "norm":
        total = s["x"].to(d)
        if s["res"] is not None:
            total = total + s["res"].to(d)
        h = total.to(s["x"].dtype).to(d)  # the norm is of the sum as it is stored
        o = h * torch.rsqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / case["cols"] + EPS) * s["w"].to(d)
        # which code a value gets is defined by the 32-bit steps, not in 64 bits
        return total, o if case["normed"] else None, o.abs().unflatten(1, (-1, 32)).max(2).values / 127, None
    if kind == "lora":
        y = s["base"].to(d).clone()
        for i in sorted(set(s["idx"].tolist()) - {-1}):
            t = torch.nonzero(s["idx"] == i).reshape(-1)
            low = torch.matmul(s["x"][t].to(d), s["a"][i].to(d).t().contiguous())
            y[t] += torch.matmul(low, s["b"][i].to(d).t().contiguous()) * float(s["scale"][i])
        return y
    off, e = s["off"].tolist(), case["n_exp"]
    n_row, rows, cols = case["tokens"] * case["k"], case["rows"], case["cols"]
    if kind == "experts":
        y = torch.zeros(n_row, rows, dtype=d, device="cuda")
        for i in range(e):
            y[off[i]:off[i + 1]] = s["x"][off[i]:off[i + 1]].to(d) @ s["w"][i].to(d).t()
        return y
    dx = torch.zeros(n_row, cols, dtype=d, device="cuda")
    dw = torch.zeros(e, rows, cols, dtype=d, device="cuda")
    for i in range(e):
        part = s["dy"][off[i]:off[i + 1]].to(d)
        dx[off[i]:off[i + 1]] = part @ s["w"][i].to(d)
        dw[i] = part.t() @ s["x"][off[i]:off[i + 1]].to(d)
    return dx, dw
