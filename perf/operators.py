# SPDX-License-Identifier: Apache-2.0
"""Measured calls of the 8-bit integer products and of the expert sort.

A program with int8 weights (one fp32 scale a weight row) and int8 tokens (one
fp32 scale a token) makes these calls: the tokens' quantization, plain or
through SwiGLU; the product of one matrix; the product of every expert's bucket
of rows; the sort of tokens into those buckets; and the weighted way back. The
last two come with their gradients.

Operators ("op" of a case):
  quant      dsv4_hip_quant_i8_dev, dsv4_hip_swiglu_quant_i8_dev
  gemm       dsv4_hip_gemm_i8_dev, from codes or (a: an element type) with the
             tokens' quantization in front of it
  experts    dsv4_hip_gemm_i8_grouped_dev
  permute    dsv4_hip_moe_permute_dev, with grad also its backward pass
  unpermute  dsv4_hip_moe_unpermute_dev, with grad also its backward pass

int8 codes are whole numbers and come back as such, beside their scales.
"""
import importlib
import math

import torch

own = False

DEV = "cuda:0"
LIMIT = 10.0                       # SwiGLU clamp
CHUNK = 1024                       # 1024 products of codes up to 127 sum exactly in fp32
TILE = 32                          # rows of one expert that the plain form multiplies together
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"f32": 0, "bf16": 1, "f16": 2}
WI8 = 5                            # the int8 weight tag of a matrix descriptor

_lib = None


def _own():
    """The package and its initialised library."""
    global _lib
    if _lib is None:
        pkg = importlib.import_module("deepseek-v4-in-c_amd")
        lib = pkg.load()
        lib.check(lib.init(0), "init")
        _lib = pkg, lib
    return _lib


# ------------------------------------------------------------------ cases ----

def listed():
    return [
        # one decode token's hidden state: the smallest call, all latency
        {"name": "token_rows", "op": "quant", "n": 1, "k": 4096, "type": "f32", "act": "none"},
        # gate and up rows of a ragged prompt's routed pairs (701 tokens, six experts each) into the down product's rows
        {"name": "prompt_mid_rows", "op": "quant", "n": 4206, "k": 2048, "type": "bf16", "act": "swiglu"},
        # an attention-sized projection of one decode token, from its bf16 hidden state
        {"name": "token_projection", "op": "gemm", "m": 1, "n": 4096, "k": 4096, "a": "bf16", "out": "bf16"},
        # the query up-projection over a few sequences decoded together
        {"name": "few_tokens_up", "op": "gemm", "m": 5, "n": 32768, "k": 1024, "a": "codes", "out": "f32"},
        # a ragged prompt through the small query down-projection, from fp32 activations
        {"name": "prompt_down_333", "op": "gemm", "m": 333, "n": 1024, "k": 4096, "a": "f32", "out": "f32"},
        # a prompt block through an attention-sized projection
        {"name": "prompt_block_2048", "op": "gemm", "m": 2048, "n": 4096, "k": 4096, "a": "codes", "out": "bf16"},
        # gate projection of the routed experts, a handful of sequences decoded together
        {"name": "batch_experts_7", "op": "experts", "tokens": 7, "topk": 6, "experts": 256, "zipf": 0.0, "n": 2048,
         "k": 4096, "out": "f32"},
        # the same over a long prompt block with uneven routing: the largest call
        {"name": "prompt_experts_4096", "op": "experts", "tokens": 4096, "topk": 6, "experts": 256, "zipf": 1.1,
         "n": 2048, "k": 4096, "out": "bf16"},
        # 64 sequences decoded together, sorted by expert
        {"name": "batch_sort_64", "op": "permute", "tokens": 64, "topk": 6, "experts": 256, "world": 1, "hidden": 4096,
         "type": "bf16", "grad": False},
        # a training step's block of tokens sorted by expert, and the gradient back
        {"name": "train_sort_4096", "op": "permute", "tokens": 4096, "topk": 6, "experts": 256, "world": 1,
         "hidden": 4096, "type": "bf16", "grad": True},
        # the batch's expert outputs weighted, summed and added to the shared expert's
        {"name": "batch_return_64", "op": "unpermute", "tokens": 64, "topk": 6, "experts": 256, "world": 1,
         "hidden": 4096, "type": "f32", "shared": True, "grad": False},
        # a training step's ragged block on one of two devices that share the experts: way back and both gradients
        {"name": "train_return_2803", "op": "unpermute", "tokens": 2803, "topk": 6, "experts": 128, "world": 2,
         "hidden": 4096, "type": "bf16", "shared": False, "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quant", "gemm", "experts", "permute", "unpermute"])
    typ = rng.choice(["f32", "bf16", "f16"])
    if op == "quant":
        k = 16 * _log(rng, 8, 1024)
        return {"op": op, "n": _log(rng, 1, min(8192, (1 << 25) // k)), "k": k, "type": typ,
                "act": rng.choice(["none", "swiglu"])}
    if op == "gemm":
        n, k = _log(rng, 48, 32768), 16 * _log(rng, 8, 512)
        n = min(n, (1 << 26) // k)
        return {"op": op, "m": _log(rng, 1, min(4096, max(2, (1 << 35) // (n * k)))), "n": n, "k": k,
                "a": rng.choice(["codes", "f32", "bf16", "f16"]), "out": typ}
    topk = rng.choice([1, 2, 4, 6, 8])
    if op == "experts":
        e = _log(rng, max(4, topk), 256)
        n, k = _log(rng, 96, 4096), 16 * _log(rng, 16, 256)
        return {"op": op, "tokens": _log(rng, 1, 4096 if n * k < 1 << 22 else 1024), "topk": topk, "experts": e,
                "zipf": rng.choice([0.0, 1.1]), "n": n, "k": k, "out": typ}
    h = 8 * _log(rng, 32, 1024)
    t = _log(rng, 1, max(2, min(8192, (1 << 26) // (h * topk))))
    case = {"op": op, "tokens": t, "topk": topk, "experts": _log(rng, max(4, topk), 384), "world": rng.choice([1, 1, 4]),
            "hidden": h, "type": typ}
    if op == "unpermute":
        case["shared"] = rng.choice([True, False])
    case["grad"] = rng.choice([True, False])
    return case


# ----------------------------------------------------------------- inputs ----

def _tokens(gen, n, k, typ):
    """Hidden states: N(0, 1), a few channels much larger than the rest."""
    x = torch.randn(n, k, device=DEV, generator=gen)
    return x.mul_(1 + 15 * (torch.rand(k, device=DEV, generator=gen) < 0.003)).to(TYPES[typ])


def _codes(x):
    """Codes and scales of rows, for operands that a program already holds quantized."""
    m = x.float().abs().amax(-1, keepdim=True)
    return (x.float() * (127 / m)).round().to(torch.int8), (m / 127).squeeze(-1)


def _routing(gen, c):
    """Distinct experts of each token, int32; those that another device holds are -1."""
    e, all_e = c["experts"], c["experts"] * c.get("world", 1)
    score = -c.get("zipf", 0.0) * torch.arange(1, all_e + 1, device=DEV, dtype=torch.float32).log()
    score = score[torch.randperm(all_e, device=DEV, generator=gen)]
    u = torch.rand(c["tokens"], all_e, device=DEV, generator=gen).clamp_(1e-7, 1 - 1e-6)
    ids = (score - (-u.log()).log()).topk(c["topk"], dim=1).indices
    return torch.where(ids < e, ids, -1).to(torch.int32)


def _sorted(idx, e):
    """(first row of each expert, pair of each row, row of each pair), from sorting the ids; -1 for pairs without."""
    key = torch.where(idx < 0, e, idx).reshape(-1).long()
    order = torch.argsort(key, stable=True)
    count = torch.zeros(e + 1, dtype=torch.long, device=idx.device).scatter_add_(0, key, torch.ones_like(key))
    off = torch.zeros(e + 1, dtype=torch.long, device=idx.device)
    off[1:] = count[:e].cumsum(0)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(order.numel(), device=idx.device)
    return off, order, torch.where(key < e, pos, -1)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": c, "stream": torch.cuda.current_stream().cuda_stream or None}
    op = c["op"]
    if op == "quant":
        s["Q"] = torch.empty(c["n"], c["k"], dtype=torch.int8, device=DEV)
        s["S"] = torch.empty(c["n"], device=DEV)
        if c["act"] == "swiglu":
            s["g"], s["u"] = (_tokens(gen, c["n"], c["k"], c["type"]) for _ in range(2))
        else:
            s["x"] = _tokens(gen, c["n"], c["k"], c["type"])
    elif op == "gemm":
        s["W"], s["Sw"] = _codes(0.02 * torch.randn(c["n"], c["k"], device=DEV, generator=gen))
        if c["a"] == "codes":
            s["Q"], s["S"] = _codes(_tokens(gen, c["m"], c["k"], "f32"))
        else:
            s["x"] = _tokens(gen, c["m"], c["k"], c["a"])
            s["Q"] = torch.empty(c["m"], c["k"], dtype=torch.int8, device=DEV)
            s["S"] = torch.empty(c["m"], device=DEV)
        s["C"] = torch.empty(c["m"], c["n"], dtype=TYPES[c["out"]], device=DEV)
    elif op == "experts":
        e, n, k, r = c["experts"], c["n"], c["k"], c["tokens"] * c["topk"]
        s["W"] = torch.empty(e, n, k, dtype=torch.int8, device=DEV)
        for w in s["W"].split(16):
            w.copy_(torch.randn(w.shape, device=DEV, generator=gen).mul_(31).round_().clamp_(-127, 127))
        s["Sw"] = (0.5 + torch.rand(e, n, device=DEV, generator=gen)) * (0.08 / 127)
        # the descriptors that a loader keeps on the device: w, s, (wdt, rows), (cols, blk_r), (blk_c)
        i = torch.arange(e, device=DEV)
        s["table"] = torch.stack([s["W"].data_ptr() + i * (n * k), s["Sw"].data_ptr() + i * (4 * n),
                                  0 * i + (WI8 + (n << 32)), 0 * i + (k + (1 << 32)), 0 * i + k], 1).contiguous()
        off, order, _ = _sorted(_routing(gen, c), e)
        s["off"], s["row_tok"] = off.to(torch.int32), (order // c["topk"]).to(torch.int32)
        s["Q"], s["S"] = _codes(_tokens(gen, c["tokens"], k, "f32"))
        s["C"] = torch.zeros(r, n, dtype=TYPES[c["out"]], device=DEV)
    else:
        t, h, r, typ = c["tokens"], c["hidden"], c["tokens"] * c["topk"], TYPES[c["type"]]
        s["idx"] = _routing(gen, c)
        if op == "permute":
            s["x"] = _tokens(gen, t, h, c["type"])
            s["off"] = torch.zeros(c["experts"] + 1, dtype=torch.int32, device=DEV)
            s["row_tok"], s["pos"] = (torch.zeros(r, dtype=torch.int32, device=DEV) for _ in range(2))
            s["rows"] = torch.zeros(r, h, dtype=typ, device=DEV)
            if c["grad"]:
                s["drows"], s["dx"] = _tokens(gen, r, h, c["type"]), torch.empty(t, h, dtype=typ, device=DEV)
        else:
            s["pos"] = _sorted(s["idx"], c["experts"])[2].to(torch.int32)
            s["rows"], s["out"] = _tokens(gen, r, h, c["type"]), torch.empty(t, h, dtype=typ, device=DEV)
            s["w"] = torch.rand(t, c["topk"], device=DEV, generator=gen).add_(0.1)
            s["w"].mul_(2.5 / s["w"].sum(1, keepdim=True))
            s["shared"] = _tokens(gen, t, h, c["type"]) if c["shared"] else None
            if c["grad"]:
                s["dout"] = _tokens(gen, t, h, c["type"])
                s["drows"], s["dw"] = torch.zeros(r, h, dtype=typ, device=DEV), torch.empty_like(s["w"])
    return s


# ------------------------------------------------------------ plain forms ----

def _plain_quant(x):
    """In 64 bits: a code next to a border is decided by the exact quotient."""
    m = x.abs().amax(-1, keepdim=True)
    q = (x.double() * 127 / m.double()).round().to(torch.int8)
    return torch.where(m > 0, q, 0), torch.where(m > 0, (m / 127).float(), 1.0).squeeze(-1)


def _plain_swiglu(g, u):
    g, u = g.double().clamp(max=LIMIT), u.double().clamp(-LIMIT, LIMIT)
    return g / (1 + torch.exp(-g)) * u


def _plain_product(a, w):
    """Sums of products of codes over the last axis, a by rows of w: whole numbers, each chunk's exact in fp32."""
    acc = 0
    for k in range(0, a.shape[-1], CHUNK):
        acc = acc + torch.matmul(a[..., k:k + CHUNK].float(), w[..., k:k + CHUNK].float().transpose(-1, -2)).double()
    return acc.float()


def _plain_experts(s, c):
    """Every expert's rows in tiles of TILE, each multiplied by its expert's matrix; rows behind the last stay."""
    r, e = s["C"].shape[0], c["experts"]
    off = s["off"].long()
    tiles = (off[1:] - off[:-1] + TILE - 1) // TILE
    last = tiles.cumsum(0)
    t = torch.arange(r // TILE + min(e, r), device=DEV)
    ex = torch.searchsorted(last, t, right=True).clamp_(max=e - 1)
    row = (off[ex] + (t - last[ex] + tiles[ex]) * TILE)[:, None] + torch.arange(TILE, device=DEV)
    row = torch.where((t < last[-1])[:, None] & (row < off[ex + 1][:, None]), row, r)
    tok = s["row_tok"].long()[row.clamp(max=r - 1)]
    acc = 0
    for k in range(0, c["k"], CHUNK):
        acc = acc + torch.matmul(s["Q"][:, k:k + CHUNK][tok].float(),
                                 s["W"][:, :, k:k + CHUNK][ex].float().transpose(1, 2)).double()
    v = acc.float() * s["S"][tok][..., None] * s["Sw"][ex][:, None, :]
    out = torch.cat([s["C"], s["C"].new_zeros(1, c["n"])])
    out[row] = v.to(out.dtype)
    return out[:r]


def _plain_permute(s, c):
    off, order, pos = _sorted(s["idx"], c["experts"])
    live = torch.arange(order.numel(), device=DEV) < off[-1]
    tok = order // c["topk"]
    out = [torch.where(live[:, None], s["x"][tok], s["rows"]), off.to(torch.int32),
           torch.where(live, tok, s["row_tok"]).to(torch.int32), pos.to(torch.int32)]
    if c["grad"]:
        p = pos.reshape(c["tokens"], c["topk"])
        d = torch.where((p >= 0)[..., None], s["drows"][p.clamp(min=0)].float(), 0.0).sum(1)
        out.append(d.to(s["x"].dtype))
    return out


def _plain_unpermute(s, c):
    p = s["pos"].long().reshape(c["tokens"], c["topk"])
    there = p >= 0
    rows = torch.where(there[..., None], s["rows"][p.clamp(min=0)].float(), 0.0)
    acc = (s["w"][..., None] * rows).sum(1)
    if s["shared"] is not None:
        acc = acc + s["shared"].float()
    out = [acc.to(s["rows"].dtype)]
    if c["grad"]:
        d = s["dout"].float()[:, None]
        r = s["rows"].shape[0]
        drows = torch.cat([s["drows"], s["drows"].new_zeros(1, c["hidden"])])
        drows[torch.where(there, p, r)] = (s["w"][..., None] * d).to(drows.dtype)
        out += [drows[:r], torch.where(there, (d * rows).sum(-1), 0.0)]
    return out


def _plain(s, c):
    op = c["op"]
    if op == "quant":
        return list(_plain_quant(_plain_swiglu(s["g"], s["u"]) if c["act"] == "swiglu" else s["x"].float()))
    if op == "gemm":
        q, sa = (s["Q"], s["S"]) if c["a"] == "codes" else _plain_quant(s["x"].float())
        return [(_plain_product(q, s["W"]) * sa[:, None] * s["Sw"]).to(TYPES[c["out"]])]
    if op == "experts":
        return [_plain_experts(s, c)]
    return _plain_permute(s, c) if op == "permute" else _plain_unpermute(s, c)


# ------------------------------------------------------------ the calls ----

def _calls(s, c):
    pkg, lib = _own()
    st, op = s["stream"], c["op"]
    if op == "quant":
        q, sc = s["Q"], s["S"]
        if c["act"] == "swiglu":
            lib.swiglu_quant_i8_dev(q.data_ptr(), sc.data_ptr(), s["g"].data_ptr(), s["u"].data_ptr(), CODE[c["type"]],
                                    c["k"], c["n"], c["k"], LIMIT, st)
        else:
            lib.quant_i8_dev(q.data_ptr(), sc.data_ptr(), s["x"].data_ptr(), CODE[c["type"]], c["k"], c["n"], c["k"], st)
        return [q, sc]
    if op == "gemm":
        q, sc, out = s["Q"], s["S"], s["C"]
        if c["a"] != "codes":
            lib.quant_i8_dev(q.data_ptr(), sc.data_ptr(), s["x"].data_ptr(), CODE[c["a"]], c["k"], c["m"], c["k"], st)
        w = pkg.qmat(pkg.DSV4_WI8, s["W"].data_ptr(), s["Sw"].data_ptr(), c["n"], c["k"], 1, c["k"])
        lib.gemm_i8_dev(out.data_ptr(), CODE[c["out"]], q.data_ptr(), sc.data_ptr(), c["m"], w, st)
        return [out]
    if op == "experts":
        lib.gemm_i8_grouped_dev(s["C"].data_ptr(), CODE[c["out"]], s["Q"].data_ptr(), s["S"].data_ptr(), c["tokens"],
                                s["row_tok"].data_ptr(), c["tokens"] * c["topk"], s["off"].data_ptr(),
                                s["table"].data_ptr(), c["experts"], c["n"], c["k"], st)
        return [s["C"]]
    typ, t, h = CODE[c["type"]], c["tokens"], c["hidden"]
    if op == "permute":
        lib.moe_permute_dev(s["rows"].data_ptr(), s["off"].data_ptr(), s["row_tok"].data_ptr(), s["pos"].data_ptr(),
                            s["x"].data_ptr(), typ, s["idx"].data_ptr(), t, c["topk"], c["experts"], h, st)
        out = [s["rows"], s["off"], s["row_tok"], s["pos"]]
        if c["grad"]:
            lib.moe_permute_bwd_dev(s["dx"].data_ptr(), s["drows"].data_ptr(), typ, s["pos"].data_ptr(), t, c["topk"], h,
                                    st)
            out.append(s["dx"])
        return out
    sh = s["shared"].data_ptr() if s["shared"] is not None else None
    lib.moe_unpermute_dev(s["out"].data_ptr(), s["rows"].data_ptr(), typ, s["pos"].data_ptr(), s["w"].data_ptr(), sh, t,
                          c["topk"], h, st)
    out = [s["out"]]
    if c["grad"]:
        lib.moe_unpermute_bwd_dev(s["drows"].data_ptr(), s["dw"].data_ptr(), s["dout"].data_ptr(), s["rows"].data_ptr(),
                                  typ, s["pos"].data_ptr(), s["w"].data_ptr(), t, c["topk"], h, st)
        out += [s["drows"], s["dw"]]
    return out


def run(state):
    return _calls(state, state["case"]) if own else _plain(state, state["case"])


# ------------------------------------------------------------------- work ----

def _experts_hit(c):
    """Expected number of experts that some token chooses, from each one's share of the choices."""
    e, a = c["experts"], c.get("zipf", 0.0)
    p = [(i + 1) ** -a for i in range(e)]
    tot = sum(p)
    return sum(1 - (1 - min(1.0, c["topk"] * q / tot)) ** c["tokens"] for q in p)


def work(case):
    c, op = case, case["op"]
    if op == "quant":
        z, el = (2 if c["act"] == "swiglu" else 1), 4 if c["type"] == "f32" else 2
        return {"bytes": c["n"] * c["k"] * (z * el + 1) + 4 * c["n"], "flops": (12 if z == 2 else 4) * c["n"] * c["k"]}
    if op == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        el = {"codes": 1, "f32": 4}.get(c["a"], 2)
        return {"bytes": m * k * el + n * k + 4 * (m + n) + m * n * (4 if c["out"] == "f32" else 2),
                "flops": 2 * m * n * k}
    if op == "experts":
        r, n, k = c["tokens"] * c["topk"], c["n"], c["k"]
        return {"bytes": _experts_hit(c) * n * (k + 4) + c["tokens"] * (k + 4) + r * (n * (4 if c["out"] == "f32" else 2) + 4),
                "flops": 2 * r * n * k}
    el, t, h = 4 if c["type"] == "f32" else 2, c["tokens"], c["hidden"]
    live = t * c["topk"] // c["world"]
    b = (t + live) * h * el + 12 * t * c["topk"]
    if op == "permute":
        return {"bytes": b * (2 if c["grad"] else 1), "flops": live * h if c["grad"] else t}
    b += t * h * el if c["shared"] else 0
    return {"bytes": b + ((t + 2 * live) * h * el + 12 * t * c["topk"] if c["grad"] else 0),
            "flops": (2 + (3 if c["grad"] else 0)) * live * h}


# ------------------------------------------------------------------ exact ----

def _exact_rows(x):
    m = x.abs().max(dim=-1).values
    return m / 127


def exact(case, seed):
    """From each operator's definition in 64 bits, value by value or product by product, not by the plain form's steps."""
    s, c = prepare(case, seed), case
    op = c["op"]
    if op == "quant":
        if c["act"] == "swiglu":
            g, u = s["g"].double(), s["u"].double()
            g = torch.minimum(g, torch.full_like(g, LIMIT))
            u = torch.maximum(torch.minimum(u, torch.full_like(u, LIMIT)), torch.full_like(u, -LIMIT))
            x = g * torch.sigmoid(g) * u
        else:
            x = s["x"].double()
        return [None, _exact_rows(x)]
    if op == "gemm":
        if c["a"] == "codes":
            a = s["Q"].double() * s["S"].double()[:, None]
        else:
            x = s["x"].double()
            a = torch.round(x * 127 / x.abs().max(dim=-1).values[:, None]) * _exact_rows(x)[:, None]
        return [a @ (s["W"].double() * s["Sw"].double()[:, None]).t().contiguous()]
    if op == "experts":
        off, tok = s["off"].tolist(), s["row_tok"].long()
        out = torch.zeros(s["C"].shape, dtype=torch.float64, device=DEV)
        a = s["Q"].double() * s["S"].double()[:, None]
        for e in range(c["experts"]):
            if off[e + 1] > off[e]:
                w = s["W"][e].double() * s["Sw"][e].double()[:, None]
                out[off[e]:off[e + 1]] = a[tok[off[e]:off[e + 1]]] @ w.t().contiguous()
        return [out]
    t, topk = c["tokens"], c["topk"]
    ids = s["idx"].reshape(-1).tolist()
    row, n_of = [-1] * len(ids), 0
    buckets = [[] for _ in range(c["experts"])]
    for p, e in enumerate(ids):
        if e >= 0:
            buckets[e].append(p)
    for b in buckets:
        for p in b:
            row[p] = n_of
            n_of += 1
    at = torch.tensor(row, device=DEV).reshape(t, topk)
    acc = torch.zeros(t, c["hidden"], dtype=torch.float64, device=DEV)
    if op == "permute":
        rows = torch.zeros(t * topk, c["hidden"], dtype=torch.float64, device=DEV)
        for k in range(topk):
            m = at[:, k] >= 0
            rows[at[m, k]] = s["x"][m].double()
            if c["grad"]:
                acc[m] += s["drows"][at[m, k]].double()
        return [rows, None, None, None] + ([acc] if c["grad"] else [])
    drows = torch.zeros(t * topk, c["hidden"], dtype=torch.float64, device=DEV)
    dw = torch.zeros(t, topk, dtype=torch.float64, device=DEV)
    for k in range(topk):
        m = at[:, k] >= 0
        y, w = s["rows"][at[m, k]].double(), s["w"][m, k].double()[:, None]
        acc[m] += w * y
        if c["grad"]:
            d = s["dout"][m].double()
            drows[at[m, k]] = w * d
            dw[m, k] = (d * y).sum(1)
    if s["shared"] is not None:
        acc += s["shared"].double()
    return [acc] + ([drows, dw] if c["grad"] else [])
