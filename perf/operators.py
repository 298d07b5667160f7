"""Work of the 4-bit matvec and of the expert-routing operators, as cases that can be timed and checked.

Each case is one pass through public entry points of lastengine_amd.Engine, or the same result in plain torch:

  g4        matrix-vector products with 4-bit codes, a scale (and a zero point) per group: one matrix at one token or a
            few, SwiGLU formed inside the down projection, the experts that a router picked out of a stack
  route     the router: top-k of the expert logits, softmax over the selected
  dispatch  (token, expert) pairs sorted by expert, and the tokens' rows copied to that order
  combine   the expert outputs back in token order, weighted and summed
  gradient  the backward of the routed block: of the weighted sum (rows and weights), of the router and of the copies

Sizes are those of this package's benchmark: hidden 4096 with 14336 (dense), hidden 2048 with 768 and 128 experts of
which a token takes 8 (experts), or between them.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
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

def _g4(rows, cols, group, m, x, scale="f16", zeros=True, swiglu=False, n_mat=1, slots=1, share=1, k=1):
    """group 0: one scale a row. k: the experts of a token, where slots pick from a stack of n_mat matrices."""
    return {"kind": "g4", "rows": rows, "cols": cols, "group": group, "m": m, "x": x, "scale": scale, "zeros": zeros,
            "swiglu": swiglu, "n_mat": n_mat, "slots": slots, "share": share, "k": k}


def listed():
    return [
        # the smallest call: one k or v projection of a decoded token, symmetric codes; the launch is most of the time
        dict(_g4(1024, 2048, 128, 1, "f32", zeros=False), name="g4_kv_projection"),
        # gate and up of a dense layer as one matrix, one token in the type that the layer's norm leaves it in
        dict(_g4(28672, 4096, 128, 1, "bf16"), name="g4_gate_up"),
        # down of the same layer, SwiGLU formed inside, five drafted tokens in verify, small groups
        dict(_g4(4096, 14336, 64, 5, "f32", swiglu=True), name="g4_down_verify"),
        # four decoded tokens, each with its own eight of 128 experts: gate and up rows of the picked experts
        dict(_g4(1536, 2048, 32, 1, "f16", n_mat=128, slots=32, share=8, k=8), name="g4_experts"),
        # the router at a small batch, and over a prompt
        {"name": "route_decode", "kind": "route", "tokens": 8, "n_exp": 128, "k": 8, "x": "f32", "pad": 0.0},
        {"name": "route_prompt", "kind": "route", "tokens": 16384, "n_exp": 128, "k": 8, "x": "f32", "pad": 0.1},
        # a batch of decoding requests, an odd count, some of them padding
        {"name": "dispatch_batch", "kind": "dispatch", "tokens": 37, "n_exp": 128, "k": 8, "cols": 2048, "x": "f32", "pad": 0.2},
        # a prompt, padded at its end
        {"name": "dispatch_prompt", "kind": "dispatch", "tokens": 4096, "n_exp": 128, "k": 8, "cols": 2048, "x": "bf16", "pad": 0.1},
        # the way back: a few tokens, a prompt
        {"name": "combine_decode", "kind": "combine", "tokens": 8, "n_exp": 128, "k": 8, "cols": 2048, "x": "f32", "pad": 0.0},
        {"name": "combine_prompt", "kind": "combine", "tokens": 4096, "n_exp": 128, "k": 8, "cols": 2048, "x": "bf16", "pad": 0.1},
        # training steps: a ragged micro-batch whose rows end anywhere, and a full one
        {"name": "gradient_ragged", "kind": "gradient", "tokens": 301, "n_exp": 60, "k": 6, "cols": 1001, "x": "f32", "pad": 0.1},
        {"name": "gradient_full", "kind": "gradient", "tokens": 4096, "n_exp": 128, "k": 8, "cols": 2048, "x": "bf16", "pad": 0.1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["g4", "g4", "g4", "route", "dispatch", "combine", "gradient"])
    x = rng.choice(["f32", "f16", "bf16"])
    if kind == "g4":
        group = rng.choice([32, 64, 128, 128, 256, 0])
        step = group or 32
        swiglu = rng.random() < 0.25
        experts = rng.random() < 0.35
        cols = max(step, _log(rng, 256, 2048 if experts else 14336) // step * step)
        rows = _log(rng, 64, 1536) if experts else _log(rng, 64, max(256, min(32000, (28672 * 4096) // cols)))
        if not experts:
            return _g4(rows, cols, group, rng.choice([1, 1, 1, rng.randint(2, 16), rng.randint(17, 40)]), x, rng.choice(["f16", "f16", "bf16", "f32"]),
                       rng.random() < 0.6, swiglu)
        n_mat = _log(rng, 4, 128)
        k, tokens = rng.randint(1, min(8, n_mat)), rng.randint(1, 5)
        # gate and up read one row for all of a token's experts, down one row for each of them
        return _g4(rows, cols, group, 1, x, rng.choice(["f16", "bf16"]), rng.random() < 0.6, swiglu, n_mat, tokens * k, 1 if swiglu else k, k)
    n_exp = _log(rng, 4, 256)
    case = {"kind": kind, "tokens": _log(rng, 1, 16384 if kind == "route" else 3000), "n_exp": n_exp, "k": rng.randint(1, min(8, n_exp)), "x": x,
            "pad": rng.choice([0.0, 0.0, 0.1, 0.5])}
    if kind != "route":
        case["cols"] = rng.choice([_log(rng, 64, 2048), _log(rng, 8, 256) * 8])
    return case


# ---------------------------------------------------------------- inputs

def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * std


def _activations(gen, rows, cols):
    """Unit rows with a few channels that stand out, as the residual stream has them."""
    big = torch.rand(cols, generator=gen, device="cuda") < 0.004
    return _normal(gen, rows, cols) * torch.where(big, 12.0, 1.0)


def _routing(gen, case):
    """Logits of a router whose experts are not equally popular; the last tokens are padding (no expert allowed)."""
    n, e = case["tokens"], case["n_exp"]
    logits = _normal(gen, n, e) + _normal(gen, e, std=0.7)
    if case["pad"]:
        logits[n - int(n * case["pad"]):] = float("-inf")
    return logits


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "g4":
        rows, cols, n_mat, slots, m = case["rows"], case["cols"], case["n_mat"], case["slots"], case["m"]
        ng = cols // case["group"] if case["group"] else 1
        # two codes to a byte, the even column in the low half; each the sum of two even draws, so that the middle ones are
        # the common ones, as in a quantized weight
        byte = torch.randint(0, 256, (n_mat, rows, cols // 2), generator=gen, device="cuda", dtype=torch.uint8)
        more = torch.randint(0, 256, (n_mat, rows, cols // 2), generator=gen, device="cuda", dtype=torch.uint8)
        s["codes"] = (byte & 0x77) + (more & 0x77)
        s["scales"] = (torch.exp(_normal(gen, n_mat, rows, ng, std=0.3)) * (0.02 / 3.2)).to(DTYPES[case["scale"]])
        s["zeros"] = torch.randint(5, 11, (n_mat, rows, ng), generator=gen, device="cuda").to(DTYPES[case["scale"]]) if case["zeros"] else None
        a = _activations(gen, -(-slots // case["share"]) * m, cols * (2 if case["swiglu"] else 1))
        s["x"] = a.to(DTYPES[case["x"]])
        s["sel"] = None
        if n_mat > 1:  # each token's experts are distinct; the last slot is of a token that asked for one fewer
            picks = [torch.randperm(n_mat, generator=gen, device="cuda")[:case["k"]] for _ in range(slots // case["k"])]
            s["sel"] = torch.cat(picks).to(torch.int32)
            s["sel"][-1] = -1
        s["out"] = torch.empty(slots, m, rows, dtype=DTYPES[case["x"]], device="cuda")
        return s
    n, k, e = case["tokens"], case["k"], case["n_exp"]
    logits = _routing(gen, case)
    if case["kind"] == "route":
        s["logits"] = logits.to(DTYPES[case["x"]])
        s["idx"] = torch.empty(n, k, dtype=torch.int32, device="cuda")
        s["w"] = torch.empty(n, k, dtype=torch.float32, device="cuda")
        return s
    cols, ty = case["cols"], DTYPES[case["x"]]
    idx, w = _plain_route(logits, k)
    s["idx"] = idx.contiguous()
    s["w"] = w.contiguous()
    if case["kind"] == "dispatch":
        s["x"] = _activations(gen, n, cols).to(ty)
        s["off"] = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
        s["in_idx"], s["out_idx"], s["pos"] = (torch.full((n * k,), -1, dtype=torch.int32, device="cuda") for _ in range(3))
        s["rows"] = torch.zeros(n * k, cols, dtype=ty, device="cuda")
        s["ws"] = torch.empty(4 << 20, dtype=torch.uint8, device="cuda")
        return s
    s["pos"] = _plain_sort(s["idx"], k, e)[3].contiguous()
    s["rows"] = _activations(gen, n * k, cols).to(ty)
    if case["kind"] == "combine":
        s["out"] = torch.empty(n, cols, dtype=ty, device="cuda")
        return s
    s["dout"] = _normal(gen, n, cols, std=0.1).to(ty)
    s["drows_in"] = _normal(gen, n * k, cols, std=0.1).to(ty)  # gradient of the copies that went to the experts
    s["drows"] = torch.zeros(n * k, cols, dtype=ty, device="cuda")
    s["dw"] = torch.empty(n, k, dtype=torch.float32, device="cuda")
    s["dlogits"] = torch.empty(n, e, dtype=torch.float32, device="cuda")
    s["dx"] = torch.empty(n, cols, dtype=ty, device="cuda")
    return s


# ---------------------------------------------------------------- the plain forms

def _plain_g4(s, case):
    rows, cols, m, slots = case["rows"], case["cols"], case["m"], case["slots"]
    group = case["group"] or cols
    sel = s["sel"]
    pick = torch.arange(slots, device="cuda") if sel is None else sel.clamp(0, case["n_mat"] - 1).long()
    code = s["codes"][pick]
    q = torch.stack([code & 15, code >> 4], dim=-1).reshape(slots, rows, cols // group, group).float()
    z = s["zeros"][pick].float().unsqueeze(-1) if s["zeros"] is not None else 8.0
    w = ((q - z) * s["scales"][pick].float().unsqueeze(-1)).reshape(slots, rows, cols)
    x = s["x"].float()
    if case["swiglu"]:
        g, u = x[:, :cols], x[:, cols:]
        x = g / (1.0 + torch.exp(-g)) * u
    x = x.reshape(-1, m, cols)[torch.arange(slots, device="cuda") // case["share"]]
    y = x[0] @ w[0].t() if slots == 1 else (w * x).sum(-1) if m == 1 else (w.unsqueeze(1) * x.unsqueeze(2)).sum(-1)
    y = y.reshape(slots, m, rows)
    if sel is not None:
        y = torch.where(((sel >= 0) & (sel < case["n_mat"]))[:, None, None], y, 0.0)
    return y.to(DTYPES[case["x"]])


def _plain_route(logits, k):
    v = logits.float()
    v = torch.where(torch.isnan(v), float("-inf"), v)
    top, order = torch.sort(v, dim=-1, descending=True, stable=True)
    top, order = top[:, :k], order[:, :k]
    there = top > float("-inf")
    e = torch.where(there, torch.exp(top - torch.where(there[:, :1], top[:, :1], 0.0)), 0.0)
    w = e / torch.where(there[:, :1], e.sum(-1, keepdim=True), 1.0)
    return torch.where(there, order, -1).to(torch.int32), w


def _plain_sort(idx, k, n_exp):
    p = idx.reshape(-1).long()
    key = torch.where((p >= 0) & (p < n_exp), p, n_exp)
    key, order = torch.sort(key, stable=True)
    off = torch.searchsorted(key, torch.arange(n_exp + 1, device="cuda")).to(torch.int32)
    there = key < n_exp
    place = torch.where(there, torch.arange(len(key), device="cuda"), -1)
    pos = torch.empty_like(place)
    pos[order] = place
    return off, torch.where(there, order // k, -1).to(torch.int32), torch.where(there, order, -1).to(torch.int32), pos.to(torch.int32)


def _plain_combine(rows, pos, w, n, k):
    there = (pos >= 0).reshape(n, k, 1)
    y = rows[pos.clamp(min=0).long()].float().reshape(n, k, -1)
    y = torch.where(there, y, 0.0)
    return (y if w is None else y * w.unsqueeze(-1)).sum(1).to(rows.dtype)


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "g4":
        return _plain_g4(s, case)
    if kind == "route":
        return _plain_route(s["logits"], case["k"])
    n, k, e = case["tokens"], case["k"], case["n_exp"]
    if kind == "dispatch":
        off, in_idx, out_idx, pos = _plain_sort(s["idx"], k, e)
        rows = torch.where((in_idx >= 0).unsqueeze(-1), s["x"][in_idx.clamp(min=0).long()], 0.0)
        return off, in_idx, out_idx, pos, rows
    pos, w = s["pos"], s["w"]
    if kind == "combine":
        return _plain_combine(s["rows"], pos, w, n, k)
    there = pos >= 0
    at = pos.clamp(min=0).long()
    each = s["dout"].float().repeat_interleave(k, 0)
    dw = torch.where(there, (each * s["rows"][at].float()).sum(-1), 0.0).reshape(n, k)
    drows = torch.zeros(n * k + 1, each.shape[1], device="cuda")
    drows[torch.where(there, at, n * k)] = each * w.reshape(-1, 1)
    dl = w * (dw - (w * dw).sum(-1, keepdim=True))
    idx = s["idx"].long()
    dlogits = torch.zeros(n, e + 1, device="cuda").scatter_(1, torch.where(idx >= 0, idx, e), dl)[:, :e]
    return drows[:-1].to(s["rows"].dtype), dw, dlogits.contiguous(), _plain_combine(s["drows_in"], pos, None, n, k)


# ---------------------------------------------------------------- the framework's calls

def _own(s):
    case, eng = s["case"], _eng()
    kind = case["kind"]
    if "ty" not in s:
        s["ty"] = _ty(case["x"])
        if kind == "g4":
            import lastengine_amd as le
            s["g4"] = le.G4(s["codes"], s["scales"], s["zeros"], case["rows"], case["cols"], case["group"] or case["cols"], n_mat=case["n_mat"])
    ty = s["ty"]
    if kind == "g4":
        eng.mv_g4(ty, s["g4"], s["x"], s["out"], m=case["m"], slots=case["slots"], share=case["share"], sel=s["sel"], swiglu=case["swiglu"])
        return s["out"]
    n, k, e = case["tokens"], case["k"], case["n_exp"]
    if kind == "route":
        eng.moe_route(ty, s["logits"], n, e, k, s["idx"], s["w"])
        return s["idx"], s["w"]
    cols = case["cols"]
    if kind == "dispatch":
        eng.moe_sort(s["idx"], n, k, e, s["off"], s["in_idx"], s["out_idx"], s["pos"], ws=s["ws"])
        eng.moe_permute(ty, s["x"], s["pos"], n, k, cols, s["rows"], n * k)
        return s["off"], s["in_idx"], s["out_idx"], s["pos"], s["rows"]
    if kind == "combine":
        eng.moe_combine(ty, s["rows"], s["pos"], s["w"], n, k, cols, s["out"], n * k)
        return s["out"]
    eng.moe_combine_bwd(ty, s["dout"], s["rows"], s["pos"], s["w"], n, k, cols, s["drows"], s["dw"], n * k)
    eng.moe_route_bwd(_ty("f32"), s["idx"], s["w"], s["dw"], n, e, k, s["dlogits"])
    eng.moe_combine(ty, s["drows_in"], s["pos"], None, n, k, cols, s["dx"], n * k)
    return s["drows"], s["dw"], s["dlogits"], s["dx"]


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    z = SIZE[case["scale"]] if case["kind"] == "g4" else 0
    if case["kind"] == "g4":
        rows, cols, slots, m = case["rows"], case["cols"], case["slots"], case["m"]
        ng = cols // case["group"] if case["group"] else 1
        one = rows * cols // 2 + rows * ng * z * (2 if case["zeros"] else 1)
        a = -(-slots // case["share"]) * m * cols * (2 if case["swiglu"] else 1)
        return {"bytes": min(slots, case["n_mat"]) * one + (a + slots * m * rows) * SIZE[case["x"]], "flops": 2 * rows * cols * m * slots}
    n, k, e = case["tokens"], case["k"], case["n_exp"]
    if case["kind"] == "route":
        return {"bytes": n * e * SIZE[case["x"]] + n * k * 8, "flops": n * (e * 2 + k * 4)}
    live = (n - int(n * case["pad"])) * k
    row = case["cols"] * SIZE[case["x"]]
    if case["kind"] == "dispatch":
        return {"bytes": n * k * 16 + (e + 1) * 4 + (live // k + live) * row, "flops": 0}
    if case["kind"] == "combine":
        return {"bytes": n * k * 8 + (live + n) * row, "flops": 2 * live * case["cols"]}
    return {"bytes": n * k * 4 * 6 + n * e * 4 + (3 * live + live // k + n) * row, "flops": 4 * live * case["cols"]}


# ---------------------------------------------------------------- the same from the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    kind = case["kind"]
    if kind == "g4":
        m, cols = case["m"], case["cols"]
        out = torch.zeros(case["slots"], m, case["rows"], dtype=d, device="cuda")
        x = s["x"].to(d)
        if case["swiglu"]:
            x = x[:, :cols] * torch.sigmoid(x[:, :cols]) * x[:, cols:]
        picks = list(range(case["slots"])) if s["sel"] is None else s["sel"].tolist()
        for slot, mat in enumerate(picks):
            if mat < 0 or mat >= case["n_mat"]:
                continue
            w = torch.empty(case["rows"], cols, dtype=d, device="cuda")
            byte = s["codes"][mat].to(torch.int32)
            w[:, 0::2] = torch.remainder(byte, 16).to(d)
            w[:, 1::2] = torch.div(byte, 16, rounding_mode="floor").to(d)
            each = case["group"] or cols
            w -= s["zeros"][mat].to(d).repeat_interleave(each, 1) if s["zeros"] is not None else 8
            w *= s["scales"][mat].to(d).repeat_interleave(each, 1)
            at = slot // case["share"] * m
            out[slot] = torch.matmul(w, x[at:at + m].t().contiguous()).t()
        return out
    n, k, e = case["tokens"], case["k"], case["n_exp"]
    if kind == "route":
        left = s["logits"].to(d).clone()
        idx, top = [], []
        for _ in range(k):  # the largest that is left, the first of equals
            best = left.max(1, keepdim=True).values
            first = (left == best).to(torch.uint8).argmax(1, keepdim=True)
            idx.append(first)
            top.append(best)
            left.scatter_(1, first, float("-inf"))
        idx, top = torch.cat(idx, 1), torch.cat(top, 1)
        none = torch.isneginf(top)
        w = torch.softmax(torch.where(none, -1e300, top), 1)
        return torch.where(none, -1, idx).to(torch.int32), torch.where(none, 0.0, w)
    if kind == "dispatch":
        where = s["idx"].reshape(-1)
        lists = [torch.nonzero(where == i).reshape(-1) for i in range(e)]
        order = torch.cat(lists)
        off = torch.tensor([0] + [len(v) for v in lists], device="cuda").cumsum(0).to(torch.int32)
        in_idx, out_idx, pos = (torch.full((n * k,), -1, dtype=torch.int32, device="cuda") for _ in range(3))
        rows = torch.zeros(n * k, case["cols"], dtype=d, device="cuda")
        c = len(order)
        in_idx[:c] = torch.div(order, k, rounding_mode="floor").to(torch.int32)
        out_idx[:c] = order.to(torch.int32)
        pos[order] = torch.arange(c, dtype=torch.int32, device="cuda")
        rows[:c] = s["x"].to(d)[in_idx[:c].long()]
        return off, in_idx, out_idx, pos, rows
    pos = s["pos"].reshape(n, k)

    def back(rows, w):
        total = torch.zeros(n, case["cols"], dtype=d, device="cuda")
        for j in range(k):
            live = torch.nonzero(pos[:, j] >= 0).reshape(-1)
            part = rows[pos[live, j].long()].to(d)
            total[live] += part if w is None else part * w[live, j, None].to(d)
        return total

    if kind == "combine":
        return back(s["rows"], s["w"])
    drows = torch.zeros(n * k, case["cols"], dtype=d, device="cuda")
    dw = torch.zeros(n, k, dtype=d, device="cuda")
    dlogits = torch.zeros(n, e, dtype=d, device="cuda")
    w = s["w"].to(d)
    for j in range(k):
        live = torch.nonzero(pos[:, j] >= 0).reshape(-1)
        at = pos[live, j].long()
        drows[at] = s["dout"][live].to(d) * w[live, j, None]
        dw[live, j] = (s["dout"][live].to(d) * s["rows"][at].to(d)).sum(1)
    mean = (w * dw).sum(1)
    for j in range(k):
        live = torch.nonzero(s["idx"][:, j] >= 0).reshape(-1)
        dlogits[live, s["idx"][live, j].long()] += w[live, j] * (dw[live, j] - mean[live])
    return drows, dw, dlogits, back(s["drows_in"], None)
