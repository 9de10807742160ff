"""Rotary positions, attention for a tree of drafted tokens, and sampling: the calls a user makes, their plain
forms, and the cases they are measured on.

The cases stand for checking drafted tokens against a model's cache: rotate the new tokens' q and k at their
positions and append k and v to the cache, attend from every drafted node to the cache and to its ancestors, and
draw a token from each row of logits. Head layouts, vocabulary and cache length of the 64-layer hybrid decoder
(24 q and 4 kv heads of 256, 64 rotated dims, 248320 tokens, 4096 cached) beside generic ones.
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


def _rope(name, mode, T, H, HK, D, R, inter, scaling, factor, base, type, pos, ctx=0):
    return {"name": name, "op": "rope", "mode": mode, "T": T, "H": H, "HK": HK, "D": D, "R": R, "inter": inter,
            "scaling": scaling, "factor": factor, "base": base, "type": type, "pos": pos, "ctx": ctx}


def _tree(name, B, n, ctx, H, HK, D, type, ragged):
    return {"name": name, "op": "tree", "B": B, "n": n, "ctx": ctx, "H": H, "HK": HK, "D": D, "type": type,
            "ragged": ragged}


def _sample(name, B, V, type, k, p, m):
    return {"name": name, "op": "sample", "B": B, "V": V, "type": type, "top_k": k, "top_p": p, "min_p": m}


def listed():
    return [
        # one new token of the hybrid decoder: q/k norm, 64 of 256 dims rotated, k and v to the fp16 cache
        _rope("rope_append_1", "append", 1, 24, 4, 256, 64, False, "none", 1.0, 1e7, "f16", 1234, 64),
        # a tree of 61 drafted tokens far into a long context, interpolated positions
        _rope("rope_append_61", "append", 61, 32, 8, 128, 128, True, "linear", 4.0, 1e4, "bf16", 120011, 256),
        # a long prompt's q and k, half layout, context stretched by a ramp over the frequencies
        _rope("rope_prompt_16k", "apply", 16384, 32, 8, 128, 128, False, "yarn", 8.0, 1e6, "bf16", 0),
        # the gradient of a training batch, an odd token count and a partly rotated odd head size, fp32
        _rope("rope_grad_7001", "grad", 7001, 20, 20, 80, 40, True, "ntk", 2.0, 1e4, "f32", 0),
        # a single token against a short cache: the latency of serving without drafts
        _tree("tree_1_short", 1, 1, 513, 24, 4, 256, "f16", False),
        # the decoder's own cache, full, and a tree of 16
        _tree("tree_16_4k", 1, 16, 4096, 24, 4, 256, "f16", False),
        # a batch of sequences of unlike lengths with trees of up to 24 nodes
        _tree("tree_24_batch", 16, 24, 8203, 32, 8, 128, "bf16", True),
        # the largest tree over a long context
        _tree("tree_64_128k", 1, 64, 131072, 24, 4, 256, "bf16", False),
        # one answer token: the usual small candidate set
        _sample("sample_1_topk", 1, 248320, "f32", 50, 0.95, 0.0),
        # a nucleus alone, an odd vocabulary
        _sample("sample_7_topp", 7, 128003, "f32", 0, 0.9, 0.0),
        # every row of a large batch, unfiltered but for a floor on the probability
        _sample("sample_64_minp", 64, 248320, "f32", 0, 1.0, 0.02),
        # a batch of a 16-bit head with every filter
        _sample("sample_33_all", 33, 50257, "bf16", 200, 0.9, 0.01),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _unnamed(case):
    del case["name"]
    return case


def draw(rng):
    op = rng.choice(["rope", "tree", "sample"])
    if op == "rope":
        mode = rng.choice(["append", "apply", "grad"])
        HK = rng.choice([1, 2, 4, 5, 8])
        H = HK * rng.choice([1, 2, 3, 4, 6, 7])
        D = rng.choice([64, 72, 80, 96, 100, 128, 160, 192, 256])
        R = rng.choice([D, D, D // 2 // 2 * 2, max(4, D // 4 // 2 * 2)])
        T = _log(rng, 1, 256) if mode == "append" else _log(rng, 1, 16384 * 40 * 128 // ((H + HK) * D))
        ctx = T + _log(rng, 1, 1000) if mode == "append" else 0
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        kind = rng.choice(["f16", "bf16"] if mode == "append" else ["f16", "bf16", "f32"])
        if mode != "append" and kind == "f32":
            T = max(1, T // 2)
        pos = rng.choice([0, _log(rng, 1, 200000)])
        return _unnamed(_rope("", mode, T, H, HK, D, R, rng.random() < 0.5, scaling,
                              1.0 if scaling == "none" else rng.choice([1.5, 2.0, 4.0, 16.0]),
                              rng.choice([1e4, 5e5, 1e6, 1e7]), kind, pos, ctx))
    if op == "tree":
        HK = rng.choice([1, 2, 4, 8])
        G = rng.choice([1, 2, 3, 4, 6, 8])
        D = rng.choice([64, 80, 96, 128, 192, 256])
        B = _log(rng, 1, 32)
        n = rng.choice([1, rng.randrange(2, 65), rng.randrange(2, 65)])
        most = 131072 * 4 * 256 // (B * HK * D)
        most = min(most, 64 * 24 * 131072 * 256 // (B * n * HK * G * D), 131072)
        ctx = n + _log(rng, 1, max(2, most - n))
        return _unnamed(_tree("", B, n, ctx, HK * G, HK, D, rng.choice(["f16", "bf16"]), rng.random() < 0.5))
    V = _log(rng, 1000, 262144)
    B = _log(rng, 1, min(256, 64 * 248320 // V))
    return _unnamed(_sample("", B, V, rng.choice(["f32", "f16", "bf16"]), rng.choice([0, 0, _log(rng, 1, 1000)]),
                            rng.choice([1.0, 0.95, 0.8, 0.5]), rng.choice([0.0, 0.0, 0.05, 0.3])))


# ---------------------------------------------------------------- inputs
def _randn(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"rope": _prepare_rope, "tree": _prepare_tree, "sample": _prepare_sample}[case["op"]](case, seed, g)


def _prepare_rope(c, seed, g):
    T, H, HK, D, t = c["T"], c["H"], c["HK"], c["D"], TYPES[c["type"]]
    s = dict(c)
    pos = torch.arange(c["pos"], c["pos"] + T, dtype=torch.int32)
    if c["mode"] == "append":
        # rows of the q projection hold (q, gate) of each head; k and v are projections of their own
        s["q"] = _randn(g, (T, H, 2 * D))[..., :D]
        s["k"], s["v"] = _randn(g, (T, HK, D)), _randn(g, (T, HK, D))
        s["qn"], s["kn"] = 1.2 + _randn(g, (D,), 0.1), 1.2 + _randn(g, (D,), 0.1)
        s["kc"], s["vc"] = (_randn(g, (c["ctx"], HK, D)).to(t) for _ in range(2))
        s["yq"] = torch.empty((T, H, D), dtype=t, device="cuda")
        s["rows"] = (pos % c["ctx"]).cuda()  # a cache of the last ctx tokens
        if T > 1:  # drafted nodes sit at the depth of their branch
            pos = c["pos"] + torch.from_numpy(_depths(_parents(np.random.default_rng(seed), T))).int()
    else:
        rows = _randn(g, (T, (H + 2 * HK) * D)).to(t)  # a fused projection's rows: q, k and v of a token
        s["q"], s["k"] = (x.unflatten(1, (-1, D)) for x in (rows[:, : H * D], rows[:, H * D: (H + HK) * D]))
        s["yq"], s["yk"] = (torch.empty((T, h, D), dtype=t, device="cuda") for h in (H, HK))
        if c["mode"] == "grad":  # packed sequences: positions start again
            pos = c["pos"] + torch.arange(T, dtype=torch.int32) % max(1, T // 3)
    s["pos"] = pos.cuda()
    if own:  # the plan that a user's program keeps: the frequencies
        btf = _btf()
        s["table"] = btf.RopeTable(c["R"], base=c["base"], scaling=c["scaling"], factor=c["factor"], orig_ctx=4096,
                                   interleaved=c["inter"], device="cuda")
    return s


def _parents(rng, n):
    """A drafter's tree: node 0 is the pending token, later nodes hang on a recent or an early one."""
    p = np.full(n, -1, dtype=np.int32)
    for j in range(1, n):
        p[j] = rng.integers(max(0, j - 4), j) if rng.random() < 0.7 else rng.integers(0, j)
    return p


def _depths(p):
    d = np.zeros(len(p), dtype=np.int64)
    for j in range(len(p)):
        d[j] = 0 if p[j] < 0 else d[p[j]] + 1
    return d


def _prepare_tree(c, seed, g):
    B, n, ctx, H, HK, D, t = c["B"], c["n"], c["ctx"], c["H"], c["HK"], c["D"], TYPES[c["type"]]
    rng = np.random.default_rng(seed)
    s = dict(c)
    s["q"] = _randn(g, (B, n, H, D), 1.5).to(t)
    s["k"] = _randn(g, (B, ctx, HK, D), 1.5).to(t)
    s["v"] = (_randn(g, (B, ctx, HK, D), 0.8) + _randn(g, (HK, D), 0.3)).to(t)
    lens, counts = np.full(B, ctx - n), np.full(B, n)
    if c["ragged"]:
        lens = np.exp(rng.uniform(0, math.log(max(1, ctx - n) + 1), B)).astype(np.int64) - 1
        lens[rng.integers(B)] = ctx - n
        counts = rng.integers(1, n + 1, B)
    s["parents"] = torch.from_numpy(np.stack([_parents(rng, n) for _ in range(B)])).cuda()
    s["lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
    s["counts"] = torch.from_numpy(counts.astype(np.int32)).cuda()
    s["rows"] = int(lens.max()) + n  # the caller knows its longest sequence
    s["out"] = torch.zeros((B, n, H, D), dtype=t, device="cuda")
    if own:
        s["work"] = _btf().tree_attention_work(s["q"], s["k"])
    return s


def _prepare_sample(c, seed, g):
    B, V, t = c["B"], c["V"], TYPES[c["type"]]
    x = _randn(g, (B, V), 2.2)
    hot = torch.randint(V, (B, 40), generator=g, device="cuda")
    x.scatter_add_(1, hot, torch.rand((B, 40), generator=g, device="cuda") * 9.0)  # the candidates of a trained head
    rng = np.random.default_rng(seed)
    temp = rng.choice([0.0, 0.6, 0.7, 0.8, 1.0, 1.2], B, p=[0.1, 0.2, 0.2, 0.2, 0.2, 0.1])
    if B == 1:
        temp[:] = 0.8
    s = dict(c, logits=x.to(t), u=torch.rand(B, generator=g, device="cuda"),
             t=torch.from_numpy(temp.astype(np.float32)).cuda(), k=None, p=None, m=None)
    if c["top_k"]:
        s["k"] = torch.from_numpy(rng.integers(max(1, c["top_k"] // 2), c["top_k"] + 1, B).astype(np.int32)).cuda()
    if c["top_p"] < 1:
        s["p"] = torch.from_numpy(rng.uniform(c["top_p"] - 0.1, c["top_p"], B).astype(np.float32)).cuda()
    if c["min_p"] > 0:
        s["m"] = torch.from_numpy(rng.uniform(c["min_p"] / 2, c["min_p"], B).astype(np.float32)).cuda()
    s["token"] = torch.empty(B, dtype=torch.int32, device="cuda")
    s["logprob"] = torch.empty(B, dtype=torch.float32, device="cuda")
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return {"rope": _run_rope, "tree": _run_tree, "sample": _run_sample}[s["op"]](s)


def _frequencies(s):
    """Angle per position of each rotated pair, and the factor on cos and sin."""
    R, base, f = s["R"], s["base"], s["factor"]
    i = torch.arange(R // 2, dtype=torch.float64, device="cuda")
    if s["scaling"] == "ntk":
        base = base * f ** (R / (R - 2))
    w = base ** (-2 * i / R)
    if s["scaling"] == "linear":
        w = w / f
    if s["scaling"] != "yarn":
        return w, 1.0
    lo, hi = (R * math.log(4096 / (2 * math.pi * b)) / (2 * math.log(base)) for b in (32.0, 1.0))
    lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), R - 1)
    ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return w * (1 - ramp) + w / f * ramp, 0.1 * math.log(f) + 1


def _rotate(x, s, cos, sin, to, norm=None):
    R, x = s["R"], x.float()
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
    w, m = _frequencies(s)
    angle = (s["pos"].double()[:, None] * w)[:, None, :]  # [T][1][R/2]: far positions need 64 bits
    cos, sin = (angle.cos() * m).float(), (angle.sin() * m).float()
    if s["mode"] == "append":
        rows = s["rows"].long()
        s["kc"][rows] = _rotate(s["k"], s, cos, sin, t, s["kn"])
        s["vc"][rows] = s["v"].to(t)
        return {"q": _rotate(s["q"], s, cos, sin, t, s["qn"]), "k": s["kc"], "v": s["vc"]}
    if s["mode"] == "grad":
        sin = -sin
    return {"q": _rotate(s["q"], s, cos, sin, t), "k": _rotate(s["k"], s, cos, sin, t)}


def _run_tree(s):
    if own:
        return _btf().tree_attention(s["q"], s["k"], s["v"], s["lens"], s["parents"], counts=s["counts"], out=s["out"],
                                     work=s["work"])
    B, n, H, HK, D, L = s["B"], s["n"], s["H"], s["HK"], s["D"], s["rows"]
    parent = s["parents"].long()
    one = torch.zeros((B, n, n + 1), device="cuda").scatter_(2, torch.where(parent < 0, n, parent)[..., None], 1.0)
    see = torch.linalg.matrix_power(one[..., :n] + torch.eye(n, device="cuda"), n) > 0  # itself and its ancestors
    row = torch.arange(L, device="cuda")
    node = row - s["lens"].long()[:, None]  # [B][L]: the node of a row behind the cache
    seen = see.gather(2, node.clamp(0, n - 1)[:, None, :].expand(B, n, L))
    seen = (node < 0)[:, None, :] | (seen & (node < n)[:, None, :])  # [B][n][L]
    q = s["q"].float().unflatten(2, (HK, H // HK)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B][HK][G n][D]
    k, v = (s[x][:, :L].float().permute(0, 2, 1, 3) for x in "kv")
    score = (q @ k.transpose(2, 3) * D ** -0.5).unflatten(2, (H // HK, n))
    score.masked_fill_(~seen[:, None, None], -math.inf)
    w = (score - score.amax(-1, keepdim=True)).exp_()
    o = w.flatten(2, 3) @ v / w.sum(-1).flatten(2, 3)[..., None]
    o = o.unflatten(2, (H // HK, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    there = torch.arange(n, device="cuda") < s["counts"][:, None]
    return torch.where(there[..., None, None], o, 0.0).to(s["q"].dtype)


def _run_sample(s):
    if own:
        return dict(zip(("token", "logprob"), _btf().sample(
            s["logits"], s["u"], temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"], tokens=s["token"],
            logprobs=s["logprob"])))
    V = s["V"]
    greedy = (s["t"] <= 0)[:, None]
    temp = torch.where(greedy, 1.0, s["t"][:, None]).double()
    x, order = s["logits"].float().sort(dim=-1, descending=True, stable=True)
    e = (x.double() - x[:, :1].double()) / temp
    w = e.exp()  # 64 bits: a rounding next to a border would draw another token
    keep = torch.arange(V, device="cuda").expand_as(w) < torch.where(greedy, 1, V)
    if s["k"] is not None:
        keep = keep & (torch.arange(V, device="cuda") < s["k"][:, None])
    if s["p"] is not None:
        before = (w * keep).cumsum(-1) - w * keep
        keep = keep & (before < s["p"].double()[:, None] * (w * keep).sum(-1, keepdim=True))
    if s["m"] is not None:
        keep = keep & (e >= s["m"].double().log()[:, None])
    w = torch.zeros_like(w).scatter_(1, order, w * keep)  # back in the vocabulary's order
    c = w.cumsum(-1)
    z = c[:, -1:]
    token = (c <= s["u"].double()[:, None] * z).sum(-1, keepdim=True)
    return {"token": token[:, 0].int(), "logprob": (w.gather(1, token) / z).log()[:, 0].float()}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "tree": _exact_tree, "sample": _exact_sample}[case["op"]](s)


def _exact_rope(s):
    R, factor = s["R"], s["factor"]
    base = s["base"] * (factor ** (R / (R - 2)) if s["scaling"] == "ntk" else 1.0)
    w = np.array([math.exp(-2.0 * i / R * math.log(base)) for i in range(R // 2)])
    mul = 1.0
    if s["scaling"] == "linear":
        w /= factor
    if s["scaling"] == "yarn":
        mul = 1.0 + math.log(factor) / 10.0
        edge = [R * (math.log(4096) - math.log(2 * math.pi * b)) / math.log(base) / 2 for b in (32.0, 1.0)]
        lo, hi = max(0, math.floor(edge[0])), min(R - 1, math.ceil(edge[1]))
        for i in range(R // 2):
            part = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            w[i] = part * w[i] / factor + (1.0 - part) * w[i]
    turn = torch.outer(s["pos"].double(), torch.from_numpy(w).cuda())
    unit = torch.polar(torch.full_like(turn, mul), -turn if s["mode"] == "grad" else turn)[:, None]

    def spun(x, norm=None):
        x = x.double()
        if norm is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * norm.double()
        y = x.clone()
        if s["inter"]:
            z = torch.complex(x[..., 0:R:2], x[..., 1:R:2]) * unit
            y[..., 0:R:2], y[..., 1:R:2] = z.real, z.imag
        else:
            z = torch.complex(x[..., : R // 2], x[..., R // 2: R]) * unit
            y[..., : R // 2], y[..., R // 2: R] = z.real, z.imag
        return y

    if s["mode"] != "append":
        return {"q": spun(s["q"]), "k": spun(s["k"])}
    out = {"q": spun(s["q"], s["qn"]), "k": s["kc"].double(), "v": s["vc"].double()}
    out["k"].index_copy_(0, s["rows"].long(), spun(s["k"], s["kn"]))
    out["v"].index_copy_(0, s["rows"].long(), s["v"].double())
    return out


def _exact_tree(s):
    B, H, HK, D = s["B"], s["H"], s["HK"], s["D"]
    lens, counts, parents = (s[x].cpu().numpy() for x in ("lens", "counts", "parents"))
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, past = int(counts[b]), int(lens[b])
        mask = np.zeros((n, past + n), dtype=bool)
        mask[:, :past] = True
        for i in range(n):
            j = i
            while j >= 0:
                mask[i, past + j] = True
                j = int(parents[b, j])
        hide = torch.from_numpy(~mask).cuda()
        for h in range(HK):
            k, v = (s[x][b, : past + n, h].double() for x in "kv")
            for head in range(h * (H // HK), (h + 1) * (H // HK)):
                a = torch.matmul(s["q"][b, :n, head].double(), k.T) / math.sqrt(D)
                out[b, :n, head] = torch.softmax(a.masked_fill(hide, -math.inf), -1) @ v
    return out


def _exact_sample(s):
    x, u, temp = s["logits"].float().cpu().numpy().astype(np.float64), s["u"].cpu().numpy(), s["t"].cpu().numpy()
    k, p, m = (None if s[n] is None else s[n].cpu().numpy() for n in "kpm")
    out = np.zeros(s["B"])
    for b in range(s["B"]):
        if temp[b] <= 0:
            continue  # one token, with certainty
        order = np.argsort(-x[b], kind="stable")
        z = (x[b][order] - x[b].max()) / np.float64(temp[b])
        n = len(z) if k is None else min(len(z), int(k[b]))
        w = np.exp(z[:n])
        if p is not None:
            n = min(n, int(np.searchsorted(np.cumsum(w), np.float64(p[b]) * w.sum())) + 1)
        if m is not None:
            n = min(n, int(np.sum(z[:n] >= math.log(m[b]))))
        kept = np.sort(order[:n])
        c = np.cumsum(np.exp((x[b][kept] - x[b].max()) / np.float64(temp[b])))
        t = kept[np.searchsorted(c, np.float64(u[b]) * c[-1], side="right")]
        out[b] = (x[b][t] - x[b].max()) / np.float64(temp[b]) - math.log(c[-1])
    return {"token": None, "logprob": torch.from_numpy(out)}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "rope":
        T, H, HK, D, size = c["T"], c["H"], c["HK"], c["D"], SIZE[c["type"]]
        heads = H + (2 if c["mode"] == "append" else 1) * HK
        read = 4 if c["mode"] == "append" else size
        return {"bytes": T * heads * D * (read + size) + T * 4, "flops": T * (H + HK) * c["R"] * 3}
    if c["op"] == "tree":
        B, n, H, HK, D, ctx = c["B"], c["n"], c["H"], c["HK"], c["D"], c["ctx"]
        rows = B * ctx
        if c["ragged"]:  # lengths uniform in their logarithm, one of them the longest
            mean = max(1, ctx - n) / math.log(max(1, ctx - n) + 1)
            rows = ctx + (B - 1) * (mean + n / 2)
        return {"bytes": 2 * rows * HK * D * 2 + 2 * B * n * H * D * 2, "flops": 4 * n * H * D * rows}
    return {"bytes": c["B"] * (c["V"] * SIZE[c["type"]] + 28), "flops": 4 * c["B"] * c["V"]}
