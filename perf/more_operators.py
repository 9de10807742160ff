"""Low-rank adapters of many requests beside a shared projection, rotary positions with several axes, and attention for
a batch that shares a long prefix: the calls a user makes, their plain forms, and the cases they are measured on.

The cases stand for serving many requests of one model at once, each with a fine-tuned adapter of its own, behind one
long system prompt or document, with images among the tokens: a layer's projections with their adapters, the q and k
turned by the tokens' time, row and column and appended to the caches, and the attention to the shared and to the own
rows. Widths and head layouts of the 64-layer hybrid decoder (hidden 5120, FFN 17408, 24 q and 4 kv heads of 256, 64
rotated dims) beside generic ones.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bonsai-ternary-fast_b200")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6  # of the per-head norm


def _btf():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import btf_b200

    return btf_b200


def _lora(name, T, requests, adapters, K, Ns, R, x, w, y, base):
    """T rows of some requests, whose adapters are among `adapters`; a projection of each width in Ns (text: it is
    split at the commas)."""
    return {"name": name, "op": "lora", "T": T, "requests": requests, "adapters": adapters, "K": K, "Ns": Ns, "R": R,
            "x": x, "w": w, "y": y, "base": base}


def _rope(name, mode, T, H, HK, D, sections, layout, inter, scaling, factor, base, type, ctx=0):
    return {"name": name, "op": "rope", "mode": mode, "T": T, "H": H, "HK": HK, "D": D, "sections": sections,
            "layout": layout, "inter": inter, "scaling": scaling, "factor": factor, "base": base, "type": type, "ctx": ctx}


def _prefix(name, B, n, P, ctx, H, HK, D, type, ragged):
    return {"name": name, "op": "prefix", "B": B, "n": n, "P": P, "ctx": ctx, "H": H, "HK": HK, "D": D, "type": type,
            "ragged": ragged}


def listed():
    return [
        # one request's new token through the attention's output projection, a small adapter: latency
        _lora("lora_1_o", 1, 1, 4, 6144, "5120", 16, "f32", "bf16", "f32", True),
        # a batch of 48 requests that answer, q, k and v in one call, ranks of up to 64
        _lora("lora_48_qkv", 48, 48, 24, 5120, "6144,1024,1024", 64, "f32", "bf16", "f32", True),
        # 200 rows of drafts, fp16 throughout, odd widths, no base
        _lora("lora_200_odd", 200, 50, 9, 1672, "4091", 24, "f16", "f16", "f16", False),
        # prompts of 11 requests through the FFN's gate, 16-bit
        _lora("lora_6007_gate", 6007, 11, 8, 5120, "17408", 64, "bf16", "bf16", "bf16", True),
        # 8 requests' new tokens behind an image: q/k norm, 64 of 256 dims by time, row and column, to the fp16 caches
        _rope("axes_append_8", "append", 8, 24, 4, 256, "11,11,10", "split", False, "none", 1.0, 1e7, "f16", 64),
        # a prompt with images, the axes take turns over the frequencies, stretched context
        _rope("axes_prompt_9001", "apply", 9001, 32, 8, 128, "24,20,20", "turns", False, "linear", 2.0, 1e6, "bf16"),
        # the gradient of an image encoder's patches: rows and columns with frequencies of their own, fp32
        _rope("axes_grad_16k", "grad", 16384, 16, 16, 80, "20,20", "own", True, "none", 1.0, 1e4, "f32"),
        # a few answers drawn to one prompt: latency
        _prefix("prefix_4_1k", 4, 1, 1000, 70, 24, 4, 256, "f16", True),
        # a batch just forked from its prompt, odd heads
        _prefix("prefix_48_4k", 48, 1, 4099, 5, 20, 5, 96, "bf16", False),
        # drafts of 8 nodes for 16 requests
        _prefix("prefix_16x8_16k", 16, 8, 16384, 1100, 24, 4, 256, "f16", True),
        # a large batch over a long document
        _prefix("prefix_128_64k", 128, 1, 65536, 2000, 32, 8, 128, "bf16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _unnamed(case):
    del case["name"]
    return case


def draw(rng):
    op = rng.choice(["lora", "rope", "prefix"])
    if op == "lora":
        K, R = 8 * _log(rng, 16, 2176), 8 * _log(rng, 1, 16)
        Ns = [_log(rng, 64, 17408) for _ in range(rng.choice([1, 1, 2, 3]))]
        n = min(_log(rng, 1, 64), 600_000_000 // (R * (3 * K + sum(Ns))) + 1)
        w = rng.choice(["f16", "bf16"])
        x = rng.choice(["f32", w])
        y = rng.choice(["f32", w])
        T = _log(rng, 1, max(2, min(8192, 6007 * (5120 + 2 * 17408) * 2 // (K * SIZE[x] + 2 * sum(Ns) * SIZE[y]))))
        return _unnamed(_lora("", T, rng.choice([T, max(1, T // 4), min(T, _log(rng, 1, 64))]), n, K,
                              ",".join(map(str, Ns)), R, x, w, y, rng.random() < 0.7))
    if op == "rope":
        mode = rng.choice(["append", "apply", "grad"])
        HK = rng.choice([1, 2, 4, 5, 8])
        H = HK * rng.choice([1, 2, 3, 4, 6, 7])
        D = rng.choice([64, 72, 80, 96, 100, 128, 160, 192, 256])
        half = rng.choice([D, D, D // 2, D // 4]) // 2
        sections, left = [], half
        for a in range(rng.choice([2, 3, 3, 4]) - 1):
            sections.append(rng.randrange(1, max(2, left // 2)))
            left -= sections[-1]
        sections.append(left)
        kind = rng.choice(["f16", "bf16"] if mode == "append" else ["f16", "bf16", "f32"])
        T = _log(rng, 1, 256) if mode == "append" else _log(rng, 1, 9001 * 40 * 128 * 2 // ((H + HK) * D * SIZE[kind]))
        scaling = rng.choice(["none", "linear", "yarn"])
        return _unnamed(_rope("", mode, T, H, HK, D, ",".join(map(str, sections)), rng.choice(["split", "turns", "own"]),
                              rng.random() < 0.5, scaling, 1.0 if scaling == "none" else rng.choice([1.5, 2.0, 4.0]),
                              rng.choice([1e4, 5e5, 1e6, 1e7]), kind, T + _log(rng, 1, 1000) if mode == "append" else 0))
    HK = rng.choice([1, 2, 4, 5, 8])
    G = rng.choice([1, 2, 3, 4, 6, 8])
    D = rng.choice([64, 80, 96, 128, 192, 256])
    B = _log(rng, 2, 256)
    n = rng.choice([1, 1, rng.randrange(2, 17)])
    P = _log(rng, 1, min(65536, 65536 * 128 * 32 * 128 // (B * n * HK * G * D)))
    ctx = n + _log(rng, 1, max(2, min(4000, 2 ** 28 // (B * HK * D) - n)))
    return _unnamed(_prefix("", B, n, P, ctx, HK * G, HK, D, rng.choice(["f16", "bf16"]), rng.random() < 0.7))


# ---------------------------------------------------------------- inputs
def _randn(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale


def _ints(text):
    return [int(v) for v in text.split(",")]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"lora": _prepare_lora, "rope": _prepare_rope, "prefix": _prepare_prefix}[case["op"]](
        case, np.random.default_rng(seed), g)


def _prepare_lora(c, rng, g):
    T, n, K, R, w = c["T"], c["adapters"], c["K"], c["R"], TYPES[c["w"]]
    s = dict(c)
    # the rows of a request lie together and share its adapter; one request in eight or so has none
    owner = np.sort(rng.integers(0, c["requests"], T))
    which = np.where(rng.random(c["requests"]) < 0.12, -1, rng.integers(0, n, c["requests"]))
    which[owner[0]] = rng.integers(0, n)
    index = which[owner].astype(np.int32)
    rank = rng.choice([r for r in (8, 16, 32, 64, 128, R) if r <= R], n)
    rank[rng.integers(n)] = R
    s["rank"] = rank.tolist()
    s["ranks"] = torch.from_numpy(rank.astype(np.int32)).cuda()
    s["scales"] = torch.from_numpy((rng.choice([16.0, 32.0, 64.0], n) / rank).astype(np.float32)).cuda()
    x = _randn(g, (T, K))
    x[:, torch.randint(K, (max(1, K // 500),), generator=g, device="cuda")] *= 12.0  # the few large channels of a hidden state
    s["xs"] = x.to(TYPES[c["x"]])
    s["a"], s["b"], s["bases"], s["ys"] = [], [], [], []
    for N in _ints(c["Ns"]):
        s["a"].append(_randn(g, (n, R, K), K ** -0.5).to(w))
        s["b"].append(_randn(g, (n, N, R), 0.02).to(w))
        s["bases"].append(_randn(g, (T, N)).to(TYPES[c["y"]]) if c["base"] else None)
        s["ys"].append(torch.empty((T, N), dtype=TYPES[c["y"]], device="cuda"))
    index = torch.from_numpy(index).cuda()
    if own:  # which rows belong to which adapter: a batch's plan serves every layer of a step
        btf = _btf()
        s["plan"] = btf.AdapterPlan(index, n)
        s["segs"] = [btf.AdapterSeg(a, b, y, base) for a, b, y, base in zip(s["a"], s["b"], s["ys"], s["bases"])]
        s["work"] = btf.adapters_work(s["xs"], s["segs"], s["plan"])
    s["rows"] = [(index == a).nonzero()[:, 0] for a in range(n)]
    return s


def _grid_positions(rng, T, axes):
    """Text and images in turn: a text token has one position on every axis; an image's tokens the time of its start
    and their place in its grid."""
    out, at, start = np.zeros((axes, T), dtype=np.int64), 0, int(rng.integers(0, 3000))
    while at < T:
        if rng.random() < 0.5:
            m = min(T - at, int(rng.integers(1, 200)))
            out[:, at: at + m] = start + np.arange(m)
            start += m
        else:
            rows, cols = (int(v) for v in rng.integers(2, 60, 2))
            m = min(T - at, rows * cols)
            cell = np.arange(m)
            out[0, at: at + m] = start
            out[1, at: at + m] = start + cell // cols
            if axes > 2:
                out[2, at: at + m] = start + cell % cols
            start += max(rows, cols)
        at += m
    return torch.from_numpy(out.astype(np.int32))


def _prepare_rope(c, rng, g):
    T, H, HK, D, t = c["T"], c["H"], c["HK"], c["D"], TYPES[c["type"]]
    s = dict(c)
    axes = len(_ints(c["sections"]))
    if c["mode"] == "append":
        # rows of the q projection hold (q, gate) of each head; k and v are projections of their own
        s["q"] = _randn(g, (T, H, 2 * D))[..., :D]
        s["k"], s["v"] = _randn(g, (T, HK, D)), _randn(g, (T, HK, D))
        s["qn"], s["kn"] = 1.2 + _randn(g, (D,), 0.1), 1.2 + _randn(g, (D,), 0.1)
        s["kc"], s["vc"] = (_randn(g, (c["ctx"], HK, D)).to(t) for _ in range(2))
        s["yq"] = torch.empty((T, H, D), dtype=t, device="cuda")
        s["rows"] = torch.from_numpy(rng.permutation(c["ctx"])[:T].astype(np.int32)).cuda()
    else:
        rows = _randn(g, (T, (H + 2 * HK) * D)).to(t)  # a fused projection's rows: q, k and v of a token
        s["q"], s["k"] = (x.unflatten(1, (-1, D)) for x in (rows[:, : H * D], rows[:, H * D: (H + HK) * D]))
        s["yq"], s["yk"] = (torch.empty((T, h, D), dtype=t, device="cuda") for h in (H, HK))
    s["pos"] = _grid_positions(rng, T, axes).cuda()
    if own:  # the plan that a user's program keeps: the frequencies and their axes
        s["table"] = _btf().RopeTable(2 * sum(_ints(c["sections"])), base=c["base"], scaling=c["scaling"],
                                      factor=c["factor"], orig_ctx=4096, interleaved=c["inter"],
                                      sections=_ints(c["sections"]), axes=c["layout"], device="cuda")
    return s


def _parents(rng, n):
    """A drafter's tree: node 0 is the pending token, later nodes hang on a recent or an early one."""
    p = np.full(n, -1, dtype=np.int32)
    for j in range(1, n):
        p[j] = rng.integers(max(0, j - 4), j) if rng.random() < 0.7 else rng.integers(0, j)
    return p


def _prepare_prefix(c, rng, g):
    B, n, P, ctx, H, HK, D, t = c["B"], c["n"], c["P"], c["ctx"], c["H"], c["HK"], c["D"], TYPES[c["type"]]
    s = dict(c)
    s["q"] = _randn(g, (B, n, H, D), 1.5).to(t)
    s["pk"] = _randn(g, (P, HK, D), 1.5).to(t)
    s["pv"] = (_randn(g, (P, HK, D), 0.8) + _randn(g, (HK, D), 0.3)).to(t)
    s["k"] = _randn(g, (B, ctx, HK, D), 1.5).to(t)
    s["v"] = (_randn(g, (B, ctx, HK, D), 0.8) + _randn(g, (HK, D), 0.3)).to(t)
    lens, counts = np.zeros(B), np.full(B, n)
    if c["ragged"]:  # the answers so far
        lens = np.exp(rng.uniform(0, math.log(max(1, ctx - n) + 1), B)).astype(np.int64) - 1
        lens[rng.integers(B)] = ctx - n
        counts = rng.integers(1, n + 1, B)
    s["parents"] = torch.from_numpy(np.stack([_parents(rng, n) for _ in range(B)])).cuda()
    s["lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
    s["counts"] = torch.from_numpy(counts.astype(np.int32)).cuda()
    s["longest"] = int(lens.max()) + n  # the caller knows its longest sequence
    s["out"] = torch.zeros((B, n, H, D), dtype=t, device="cuda")
    if own:
        s["work"] = _btf().prefix_attention_work(s["q"], s["pk"], s["k"])
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return {"lora": _run_lora, "rope": _run_rope, "prefix": _run_prefix}[s["op"]](s)


def _run_lora(s):
    if own:
        return _btf().adapters(s["xs"], s["segs"], s["plan"], ranks=s["ranks"], scales=s["scales"], work=s["work"])
    out = []
    x = s["xs"].float()
    for a, b, base, y in zip(s["a"], s["b"], s["bases"], s["ys"]):
        z = torch.zeros(y.shape, device="cuda") if base is None else base.float().clone()
        for j, rows in enumerate(s["rows"]):
            r = s["rank"][j]
            if rows.numel():
                h = x[rows] @ a[j, :r].float().T
                z.index_add_(0, rows, h @ b[j, :, :r].float().T * s["scales"][j])
        out.append(z.to(y.dtype))
    return out


def _ramp(R, base, f, i):
    """How far pair i is stretched, of R rotated dims."""
    lo, hi = (R * math.log(4096 / (2 * math.pi * b)) / (2 * math.log(base)) for b in (32.0, 1.0))
    lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), R - 1)
    return ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)


def _frequencies(s):
    """Each rotated pair's angle per position and its axis, and the factor on cos and sin."""
    sections, base, f = _ints(s["sections"]), s["base"], s["factor"]
    half = sum(sections)
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    R = torch.full_like(i, 2 * half)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).cuda()
    if s["layout"] == "own":  # the frequencies begin anew with each axis
        first = torch.tensor([sum(sections[:a]) for a in range(len(sections))]).cuda()
        i, R = i - first[axis], 2.0 * torch.tensor(sections).cuda()[axis]
    if s["layout"] == "turns":  # round and round, an axis without pairs left is passed over
        left, order = list(sections), []
        while sum(left):
            for a in range(len(left)):
                if left[a]:
                    left[a] -= 1
                    order.append(a)
        axis = torch.tensor(order).cuda()
    w = base ** (-2 * i / R)
    if s["scaling"] == "linear":
        return w / f, axis, 1.0
    if s["scaling"] == "none":
        return w, axis, 1.0
    ramp = torch.zeros_like(i)
    for size in set(R.tolist()):
        ramp = torch.where(R == size, _ramp(int(size), base, f, i), ramp)
    return w * (1 - ramp) + w / f * ramp, axis, 0.1 * math.log(f) + 1


def _rotate(x, s, cos, sin, to, norm=None):
    R, x = 2 * cos.shape[-1], x.float()
    if norm is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * norm
    r = x[..., :R]
    a, b = (r[..., 0::2], r[..., 1::2]) if s["inter"] else (r[..., : R // 2], r[..., R // 2:])
    a, b = a * cos - b * sin, a * sin + b * cos
    r = torch.stack((a, b), -1).flatten(-2) if s["inter"] else torch.cat((a, b), -1)
    return torch.cat((r, x[..., R:]), -1).to(to)


def _run_rope(s):
    if own:
        btf = _btf()
        if s["mode"] == "append":
            btf.rope([btf.RopeSeg(s["q"], s["yq"], normw=s["qn"]),
                      btf.RopeSeg(s["k"], s["kc"], normw=s["kn"], rows=s["rows"]),
                      btf.RopeSeg(s["v"], s["vc"], rotate=False, rows=s["rows"])], s["table"], s["pos"], eps=EPS)
            return {"q": s["yq"], "k": s["kc"], "v": s["vc"]}
        btf.rope([btf.RopeSeg(s["q"], s["yq"]), btf.RopeSeg(s["k"], s["yk"])], s["table"], s["pos"],
                 inverse=s["mode"] == "grad")
        return {"q": s["yq"], "k": s["yk"]}
    t = TYPES[s["type"]]
    w, axis, m = _frequencies(s)
    angle = (s["pos"].double().T[:, axis] * w)[:, None, :]  # [T][1][pairs]: far positions need 64 bits
    cos, sin = (angle.cos() * m).float(), (angle.sin() * m).float()
    if s["mode"] == "append":
        rows = s["rows"].long()
        s["kc"][rows] = _rotate(s["k"], s, cos, sin, t, s["kn"])
        s["vc"][rows] = s["v"].to(t)
        return {"q": _rotate(s["q"], s, cos, sin, t, s["qn"]), "k": s["kc"], "v": s["vc"]}
    if s["mode"] == "grad":
        sin = -sin
    return {"q": _rotate(s["q"], s, cos, sin, t), "k": _rotate(s["k"], s, cos, sin, t)}


def _run_prefix(s):
    if own:
        return _btf().prefix_attention(s["q"], s["pk"], s["pv"], s["k"], s["v"], s["lens"], s["parents"],
                                       counts=s["counts"], out=s["out"], work=s["work"])
    B, n, H, HK, D, L = s["B"], s["n"], s["H"], s["HK"], s["D"], s["longest"]
    G = H // HK
    parent = s["parents"].long()
    one = torch.zeros((B, n, n + 1), device="cuda").scatter_(2, torch.where(parent < 0, n, parent)[..., None], 1.0)
    see = torch.linalg.matrix_power(one[..., :n] + torch.eye(n, device="cuda"), n) > 0  # itself and its ancestors
    row = torch.arange(L, device="cuda")
    node = row - s["lens"].long()[:, None]  # [B][L]: the node of a row behind the cache
    seen = see.gather(2, node.clamp(0, n - 1)[:, None, :].expand(B, n, L))
    seen = (node < 0)[:, None, :] | (seen & (node < n)[:, None, :])  # [B][n][L]
    q = s["q"].float().unflatten(2, (HK, G)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B][HK][G n][D]
    k, v = (s[x][:, :L].float().permute(0, 2, 1, 3) for x in "kv")
    score = (q @ k.transpose(2, 3) * D ** -0.5).unflatten(2, (G, n))
    score = score.masked_fill_(~seen[:, None, None], -math.inf).flatten(2, 3)
    stacked = q.transpose(0, 1).flatten(1, 2)  # [HK][B G n][D]: every sequence's rows against the shared ones
    pk, pv = (s[x].float().transpose(0, 1) for x in ("pk", "pv"))
    shared = stacked @ pk.transpose(1, 2)
    shared *= D ** -0.5
    back = lambda x: x.unflatten(1, (B, G * n)).transpose(0, 1)  # noqa: E731
    top = torch.maximum(score.amax(-1), back(shared.amax(-1)))
    w = (score - top[..., None]).exp_()
    shared = shared.sub_(top.transpose(0, 1).flatten(1, 2)[..., None]).exp_()
    o = w @ v + back(shared @ pv)
    o = o / (w.sum(-1) + back(shared.sum(-1)))[..., None]
    o = o.unflatten(2, (G, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    there = torch.arange(n, device="cuda") < s["counts"][:, None]
    return torch.where(there[..., None, None], o, 0.0).to(s["q"].dtype)


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"lora": _exact_lora, "rope": _exact_rope, "prefix": _exact_prefix}[case["op"]](s)


def _exact_lora(s):
    out = []
    for a, b, base, y in zip(s["a"], s["b"], s["bases"], s["ys"]):
        z = torch.zeros(y.shape, dtype=torch.float64, device="cuda")
        for j, rows in enumerate(s["rows"]):
            for some in rows.split(1024):
                r = s["rank"][j]
                h = torch.einsum("tk,rk->tr", s["xs"][some].double(), a[j, :r].double())
                z[some] = torch.einsum("tr,nr->tn", h, b[j, :, :r].double()) * s["scales"][j].double()
        if base is not None:
            z += base
        out.append(z)
    return out


def _exact_rope(s):
    sections, factor = _ints(s["sections"]), s["factor"]
    half, mul = sum(sections), 1.0
    left, w, ax = list(sections), np.zeros(half), np.zeros(half, dtype=np.int64)
    turn = -1
    for i in range(half):
        if s["layout"] == "turns":
            turn = (turn + 1) % len(sections)
            while left[turn] == 0:
                turn = (turn + 1) % len(sections)
        else:
            turn = next(a for a in range(len(sections)) if left[a])
        j, R = i, 2 * half
        if s["layout"] == "own":
            j, R = sections[turn] - left[turn], 2 * sections[turn]
        left[turn] -= 1
        ax[i] = turn
        w[i] = math.exp(-2.0 * j / R * math.log(s["base"]))
        if s["scaling"] == "linear":
            w[i] /= factor
        if s["scaling"] == "yarn":
            mul = 1.0 + math.log(factor) / 10.0
            edge = [R * (math.log(4096) - math.log(2 * math.pi * b)) / math.log(s["base"]) / 2 for b in (32.0, 1.0)]
            lo, hi = max(0, math.floor(edge[0])), min(R - 1, math.ceil(edge[1]))
            part = min(1.0, max(0.0, (j - lo) / max(hi - lo, 0.001)))
            w[i] = part * w[i] / factor + (1.0 - part) * w[i]
    turned = s["pos"].double()[torch.from_numpy(ax).cuda()].T * torch.from_numpy(w).cuda()
    unit = torch.polar(torch.full_like(turned, mul), -turned if s["mode"] == "grad" else turned)[:, None]
    R = 2 * half

    def spun(x, norm=None):
        x = x.double()
        if norm is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * norm.double()
        y = x.clone()
        if s["inter"]:
            z = torch.complex(x[..., 0:R:2], x[..., 1:R:2]) * unit
            y[..., 0:R:2], y[..., 1:R:2] = z.real, z.imag
        else:
            z = torch.complex(x[..., :half], x[..., half: R]) * unit
            y[..., :half], y[..., half: R] = z.real, z.imag
        return y

    if s["mode"] != "append":
        return {"q": spun(s["q"]), "k": spun(s["k"])}
    out = {"q": spun(s["q"], s["qn"]), "k": s["kc"].double(), "v": s["vc"].double()}
    out["k"].index_copy_(0, s["rows"].long(), spun(s["k"], s["kn"]))
    out["v"].index_copy_(0, s["rows"].long(), s["v"].double())
    return out


def _exact_prefix(s):
    B, H, HK, D, P = s["B"], s["H"], s["HK"], s["D"], s["P"]
    lens, counts, parents = (s[x].cpu().numpy() for x in ("lens", "counts", "parents"))
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, past = int(counts[b]), int(lens[b])
        mask = np.zeros((n, P + past + n), dtype=bool)
        mask[:, : P + past] = True
        for i in range(n):
            j = i
            while j >= 0:
                mask[i, P + past + j] = True
                j = int(parents[b, j])
        hide = torch.from_numpy(~mask).cuda()
        for h in range(HK):
            k, v = (torch.cat((s["p" + x][:, h], s[x][b, : past + n, h])).double() for x in "kv")
            q = s["q"][b, :n, h * (H // HK): (h + 1) * (H // HK)].double()
            a = torch.einsum("ngd,ld->gnl", q, k) / math.sqrt(D)
            o = torch.softmax(a.masked_fill(hide, -math.inf), -1) @ v
            out[b, :n, h * (H // HK): (h + 1) * (H // HK)] = o.transpose(0, 1)
    return out


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "lora":
        T, K, R, n = c["T"], c["K"], c["R"], c["adapters"]
        used = n * (1 - (1 - 1 / n) ** (0.88 * c["requests"]))  # adapters with a row, as many as are expected
        rank = np.mean([r for r in (8, 16, 32, 64, 128, R) if r <= R])  # their mean rank
        Ns = _ints(c["Ns"])
        weights = used * rank * (len(Ns) * K + sum(Ns)) * 2
        passes = 2 if c["base"] else 1
        return {"bytes": int(T * K * SIZE[c["x"]] + weights + passes * T * sum(Ns) * SIZE[c["y"]] + 4 * T),
                "flops": int(2 * 0.88 * T * rank * (len(Ns) * K + sum(Ns)))}
    if c["op"] == "rope":
        T, H, HK, D, size = c["T"], c["H"], c["HK"], c["D"], SIZE[c["type"]]
        heads = H + (2 if c["mode"] == "append" else 1) * HK
        read = 4 if c["mode"] == "append" else size
        sections = _ints(c["sections"])
        return {"bytes": T * heads * D * (read + size) + T * 4 * len(sections), "flops": T * (H + HK) * 6 * sum(sections)}
    B, n, P, ctx, H, HK, D = c["B"], c["n"], c["P"], c["ctx"], c["H"], c["HK"], c["D"]
    rows, nodes = B * n, B * n
    if c["ragged"]:  # lengths uniform in their logarithm, one of them the longest
        mean = max(1, ctx - n) / math.log(max(1, ctx - n) + 1)
        nodes = B * (n + 1) / 2
        rows = ctx + (B - 1) * mean + nodes
    return {"bytes": int(2 * (P + rows) * HK * D * 2 + 2 * nodes * H * D * 2),
            "flops": int(4 * nodes * H * D * (P + rows / B))}
