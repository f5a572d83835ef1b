# SPDX-License-Identifier: Apache-2.0
"""Measured calls of the microscaled 4-bit products and of the router with groups.

A program that runs experts and projections with both operands in 4 bits (e2m1
codes, one E8M0 scale for 32 values along the sum) makes these calls: the rows'
quantization, plain, through SwiGLU or by columns (the operands of a backward
pass); the product of one matrix; the product of every expert's bucket of rows;
and the router in front of them, softmax or sigmoid scores with a bias for
balance and groups of experts, with its gradient.

Operators ("op" of a case):
  route      dsv4_hip_route_groups_dev, with grad also its backward pass
  quant      dsv4_hip_quant_mxfp4_dev, dsv4_hip_swiglu_quant_mxfp4_dev,
             dsv4_hip_quant_mxfp4_t_dev, decoded by dsv4_hip_dequant_dev
  gemm       dsv4_hip_gemm_mxfp4q_dev, from codes or (a: an element type) with
             the tokens' quantization in front of it
  linear     a projection's forward pass and both gradients from these calls
  experts    dsv4_hip_gemm_mxfp4q_grouped_dev

4-bit rows come back as the values they stand for.
"""
import importlib
import math

import torch

own = False

DEV = "cuda:0"
LIMIT = 10.0                       # SwiGLU clamp
SCALE = 2.5                        # of the routing weights
TILE = 32                          # rows of one expert that the plain form multiplies together
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"f32": 0, "bf16": 1, "f16": 2}
SCORE = {"softmax": 1, "sigmoid": 2}
WFP4 = 3                           # the e2m1 weight tag of a matrix descriptor
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]

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
        # one decode token's gate outputs: the smallest call, all latency
        {"name": "token_route", "op": "route", "n": 1, "experts": 256, "topk": 6, "score": "sigmoid", "bias": True,
         "groups": 8, "kept": 4, "top": 2, "renorm": True, "type": "f32", "grad": False, "aux": False},
        # a ragged prompt routed by softmax without groups
        {"name": "prompt_route_2803", "op": "route", "n": 2803, "experts": 256, "topk": 6, "score": "softmax",
         "bias": False, "groups": 1, "kept": 1, "top": 1, "renorm": False, "type": "bf16", "grad": False, "aux": False},
        # a training step's tokens, with the scores that a balance loss reads and both gradients back
        {"name": "train_route_16384", "op": "route", "n": 16384, "experts": 256, "topk": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "kept": 4, "top": 2, "renorm": True, "type": "f32", "grad": True, "aux": True},
        # one decode token's hidden state
        {"name": "token_rows", "op": "quant", "n": 1, "k": 4096, "type": "f32", "form": "rows"},
        # gate and up rows of a ragged prompt's routed pairs (701 tokens, six experts each) into the down product's rows
        {"name": "prompt_mid_rows", "op": "quant", "n": 4206, "k": 2048, "type": "bf16", "form": "swiglu"},
        # a training step's ragged activations by columns, for the weight gradient
        {"name": "train_columns_2803", "op": "quant", "n": 2803, "k": 4096, "type": "bf16", "form": "columns"},
        # an attention-sized projection of one decode token, from its bf16 hidden state
        {"name": "token_projection", "op": "gemm", "m": 1, "n": 4096, "k": 4096, "a": "bf16", "out": "bf16"},
        # a ragged prompt through the small query down-projection, from fp32 activations
        {"name": "prompt_down_333", "op": "gemm", "m": 333, "n": 1024, "k": 4096, "a": "f32", "out": "f32"},
        # a prompt block through an attention-sized projection
        {"name": "prompt_block_4096", "op": "gemm", "m": 4096, "n": 4096, "k": 4096, "a": "codes", "out": "bf16"},
        # a training step of the query down-projection on a ragged block: forward and both gradients
        {"name": "train_linear_2803", "op": "linear", "m": 2803, "n": 1024, "k": 4096, "type": "bf16"},
        # gate projection of the routed experts, a handful of sequences decoded together
        {"name": "batch_experts_7", "op": "experts", "tokens": 7, "topk": 6, "experts": 256, "zipf": 0.0, "n": 2048,
         "k": 4096, "out": "f32"},
        # the same over a long prompt block with uneven routing: the largest call
        {"name": "prompt_experts_4096", "op": "experts", "tokens": 4096, "topk": 6, "experts": 256, "zipf": 1.1,
         "n": 2048, "k": 4096, "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "quant", "gemm", "linear", "experts"])
    typ = rng.choice(["f32", "bf16", "f16"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        each = _log(rng, 8, 1024 // groups)
        kept, topk = rng.randint(1, groups), rng.choice([1, 2, 4, 6, 8])
        case = {"op": op, "n": _log(rng, 1, min(16384, (1 << 22) // (each * groups))), "experts": each * groups,
                "topk": topk, "score": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.choice([True, False]), "groups": groups, "kept": kept, "top": rng.choice([1, 2]),
                # the one weight of a single expert is a constant when it is renormalised: no gradient to measure
                "renorm": topk > 1 and rng.choice([True, False]), "type": typ, "grad": rng.choice([True, False])}
        return case | {"aux": case["grad"] and rng.choice([True, False])}
    if op == "quant":
        k = 32 * _log(rng, 4, 512)
        return {"op": op, "n": _log(rng, 1, min(8192, (1 << 25) // k)), "k": k, "type": typ,
                "form": rng.choice(["rows", "swiglu", "columns"])}
    if op == "gemm":
        n, k = _log(rng, 48, 32768), 32 * _log(rng, 4, 256)
        n = min(n, (1 << 26) // k)
        return {"op": op, "m": _log(rng, 1, min(4096, max(2, (1 << 35) // (n * k)))), "n": n, "k": k,
                "a": rng.choice(["codes", "f32", "bf16", "f16"]), "out": typ}
    if op == "linear":
        n, k = 32 * _log(rng, 4, 256), 32 * _log(rng, 4, 128)
        return {"op": op, "m": _log(rng, 32, min(4096, (1 << 34) // (n * k))), "n": n, "k": k, "type": typ}
    topk = rng.choice([1, 2, 4, 6, 8])
    e = _log(rng, max(4, topk), 256)
    n, k = _log(rng, 96, 4096), 32 * _log(rng, 8, 128)
    return {"op": op, "tokens": _log(rng, 1, 4096 if n * k < 1 << 22 else 1024), "topk": topk, "experts": e,
            "zipf": rng.choice([0.0, 1.1]), "n": n, "k": k, "out": typ}


# ----------------------------------------------------------------- inputs ----

def _tokens(gen, n, k, typ):
    """Hidden states: N(0, 1), a few channels much larger than the rest."""
    x = torch.randn(n, k, device=DEV, generator=gen)
    return x.mul_(1 + 15 * (torch.rand(k, device=DEV, generator=gen) < 0.003)).to(TYPES[typ])


def _rows_as_held(x):
    """Packed codes and scale bytes of rows, for operands that a program already holds quantized."""
    v, s = _codes(x.double())
    return _pack(v), s


def _pack(code):
    """Two codes a byte, the even element in the low nibble."""
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8)


def _routing(gen, c):
    """Distinct experts of each token."""
    e = c["experts"]
    score = -c["zipf"] * torch.arange(1, e + 1, device=DEV, dtype=torch.float32).log()
    score = score[torch.randperm(e, device=DEV, generator=gen)]
    u = torch.rand(c["tokens"], e, device=DEV, generator=gen).clamp_(1e-7, 1 - 1e-6)
    return (score - (-u.log()).log()).topk(c["topk"], dim=1).indices


def _ceil32(n):
    return (n + 31) // 32 * 32


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": c, "stream": torch.cuda.current_stream().cuda_stream or None}
    op = c["op"]

    def buf(rows, cols):                           # packed codes and scales
        return (torch.empty(rows, cols // 2, dtype=torch.uint8, device=DEV),
                torch.empty(rows, cols // 32, dtype=torch.uint8, device=DEV))

    if op == "route":
        n, e = c["n"], c["experts"]
        s["x"] = (1.5 * torch.randn(n, e, device=DEV, generator=gen)).to(TYPES[c["type"]])
        s["bias"] = 0.05 * torch.randn(e, device=DEV, generator=gen) if c["bias"] else None
        s["idx"] = torch.empty(n, c["topk"], dtype=torch.int32, device=DEV)
        s["w"] = torch.empty(n, c["topk"], device=DEV)
        s["scores"] = torch.empty(n, e, device=DEV) if c["aux"] else None
        if c["grad"]:
            s["dw"] = torch.randn(n, c["topk"], device=DEV, generator=gen)
            s["ds"] = 0.01 * torch.randn(n, e, device=DEV, generator=gen) if c["aux"] else None
            s["dx"] = torch.empty_like(s["x"])
    elif op == "quant":
        n, k = c["n"], c["k"]
        s["x"] = _tokens(gen, n, k, c["type"])
        if c["form"] == "swiglu":
            s["u"] = _tokens(gen, n, k, c["type"])
        rows, cols = (k, _ceil32(n)) if c["form"] == "columns" else (n, k)
        s["Q"], s["S"] = buf(rows, cols)
        s["V"] = torch.empty(rows, cols, device=DEV)
    elif op == "gemm":
        s["W"], s["Sw"] = _rows_as_held(0.02 * torch.randn(c["n"], c["k"], device=DEV, generator=gen))
        if c["a"] == "codes":
            s["Q"], s["S"] = _rows_as_held(_tokens(gen, c["m"], c["k"], "f32"))
        else:
            s["x"] = _tokens(gen, c["m"], c["k"], c["a"])
            s["Q"], s["S"] = buf(c["m"], c["k"])
        s["C"] = torch.empty(c["m"], c["n"], dtype=TYPES[c["out"]], device=DEV)
    elif op == "linear":
        m, n, k, typ = c["m"], c["n"], c["k"], TYPES[c["type"]]
        s["x"], s["dy"] = _tokens(gen, m, k, c["type"]), (0.1 * torch.randn(m, n, device=DEV, generator=gen)).to(typ)
        s["w"] = (0.02 * torch.randn(n, k, device=DEV, generator=gen)).to(typ)
        s["y"], s["dx"] = torch.empty(m, n, dtype=typ, device=DEV), torch.empty(m, k, dtype=typ, device=DEV)
        s["dw"] = torch.empty(n, k, device=DEV)
        s["xq"], s["wq"], s["dyq"] = buf(m, k), buf(n, k), buf(m, n)
        s["xt"], s["wt"], s["dyt"] = buf(k, _ceil32(m)), buf(k, n), buf(n, _ceil32(m))
    else:
        e, n, k, r = c["experts"], c["n"], c["k"], c["tokens"] * c["topk"]
        s["W"], s["Sw"] = buf(e * n, k)
        s["W"], s["Sw"] = s["W"].view(e, n, k // 2), s["Sw"].view(e, n, k // 32)
        for i in range(0, e, 8):
            w = 0.02 * torch.randn(min(8, e - i), n, k, device=DEV, generator=gen)
            s["W"][i:i + 8], s["Sw"][i:i + 8] = _rows_as_held(w)
        # the descriptors that a loader keeps on the device: w, s, (wdt, rows), (cols, blk_r), (blk_c)
        i = torch.arange(e, device=DEV)
        s["table"] = torch.stack([s["W"].data_ptr() + i * (n * k // 2), s["Sw"].data_ptr() + i * (n * k // 32),
                                  0 * i + (WFP4 + (n << 32)), 0 * i + (k + (1 << 32)), 0 * i + 32], 1).contiguous()
        key = _routing(gen, c).reshape(-1)
        count = torch.zeros(e, dtype=torch.long, device=DEV).scatter_add_(0, key, torch.ones_like(key))
        s["off"] = torch.zeros(e + 1, dtype=torch.int32, device=DEV)
        s["off"][1:] = count.cumsum(0)
        s["row_tok"] = (torch.argsort(key, stable=True) // c["topk"]).to(torch.int32)
        s["Q"], s["S"] = _rows_as_held(_tokens(gen, c["tokens"], k, "f32"))
        s["C"] = torch.empty(r, n, dtype=TYPES[c["out"]], device=DEV)
    return s


# ------------------------------------------------------------ plain forms ----

def _two_to(e):
    """2^e in fp64, exactly."""
    return ((e + 1023) << 52).view(torch.float64)


def _codes(x):
    """e2m1 codes [.., k] and E8M0 bytes [.., k / 32] of fp64 rows: values next to a border are decided exactly."""
    b = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    byte = (127 + e - 3 + (m > 0.75).int()).clamp(0, 254)
    byte = torch.where(m > 0, byte, 127)
    v = b * _two_to(127 - byte.long())
    a = v.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code + 8 * torch.signbit(v)
    return code.flatten(-2).to(torch.uint8), byte.squeeze(-1).to(torch.uint8)


def _decode(code, byte):
    """fp32 values of unpacked codes."""
    table = torch.tensor(VALUES + [-v for v in VALUES], device=code.device)
    v = table[code.int()].unflatten(-1, (-1, 32))
    return (v * _two_to(byte.long().unsqueeze(-1) - 127).float()).flatten(-2)


def _unpack(q):
    return torch.stack([q & 15, q >> 4], -1).flatten(-2)


def _plain_swiglu(g, u):
    g, u = g.double().clamp(max=LIMIT), u.double().clamp(-LIMIT, LIMIT)
    return g / (1 + torch.exp(-g)) * u


def _columns(x):
    """Rows of x^T, padded with zeros to whole blocks."""
    pad = torch.zeros(x.shape[1], _ceil32(x.shape[0]), dtype=torch.float64, device=x.device)
    pad[:, :x.shape[0]] = x.double().t()
    return pad


def _rounded(x):
    """The values that x's 4-bit rows stand for."""
    return _decode(*_codes(x.double()))


def _plain_scores(x, kind):
    x = x.double()
    if kind == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _order(v):
    """Places of the largest values first, ties to the lower place."""
    return torch.sort(v, dim=-1, descending=True, stable=True)


def _plain_route(s, c):
    n, e = s["x"].shape
    p = _plain_scores(s["x"], c["score"])
    score = p.float()
    choice = score if s["bias"] is None else score + s["bias"]
    if c["groups"] > 1:
        by = choice.reshape(n, c["groups"], -1)
        best = _order(by)[0][..., :c["top"]].sum(-1)
        kept = _order(best)[1][:, :c["kept"]]
        off = torch.ones(n, c["groups"], dtype=torch.bool, device=DEV).scatter_(1, kept, False)
        choice = by.masked_fill(off[..., None], -math.inf).reshape(n, e)
    idx = _order(choice)[1][:, :c["topk"]]
    got = score.gather(1, idx).double()
    total = got.sum(-1, keepdim=True) if c["renorm"] else torch.ones(n, 1, dtype=torch.float64, device=DEV)
    out = [idx.to(torch.int32), (got * SCALE / total).float()]
    if c["aux"]:
        out.append(score)
    if c["grad"]:
        got = p.gather(1, idx)
        dw = s["dw"].double() * SCALE
        if c["renorm"]:
            total = got.sum(-1, keepdim=True)
            d = (dw - (dw * got).sum(-1, keepdim=True) / total) / total
        else:
            d = dw
        ds = s["ds"].double() if c["aux"] else torch.zeros_like(p)
        ds = ds.scatter_add(1, idx, d)
        dx = p * (1 - p) * ds if c["score"] == "sigmoid" else p * (ds - (p * ds).sum(-1, keepdim=True))
        out.append(dx.to(s["x"].dtype))
    return out


def _plain_experts(s, c):
    """Every expert's rows in tiles of TILE, each multiplied by its expert's matrix."""
    r, e, n, k = s["C"].shape[0], c["experts"], c["n"], c["k"]
    off = s["off"].long()
    tiles = (off[1:] - off[:-1] + TILE - 1) // TILE
    last = tiles.cumsum(0)
    t = torch.arange(r // TILE + min(e, r), device=DEV)
    ex = torch.searchsorted(last, t, right=True).clamp_(max=e - 1)
    row = (off[ex] + (t - last[ex] + tiles[ex]) * TILE)[:, None] + torch.arange(TILE, device=DEV)
    row = torch.where((t < last[-1])[:, None] & (row < off[ex + 1][:, None]), row, r)
    tok = s["row_tok"].long()[row.clamp(max=r - 1)]
    x = _decode(_unpack(s["Q"]), s["S"])[tok]
    chunk = max(1, (1 << 28) // (t.numel() * k))
    acc = []
    for i in range(0, n, chunk):                   # weight rows
        w = _decode(_unpack(s["W"][:, i:i + chunk][ex]), s["Sw"][:, i:i + chunk][ex])
        acc.append(torch.matmul(x, w.transpose(1, 2)))
    out = torch.zeros(r + 1, n, dtype=s["C"].dtype, device=DEV)
    out[row] = torch.cat(acc, -1).to(out.dtype)
    return out[:r]


def _plain(s, c):
    op = c["op"]
    if op == "route":
        return _plain_route(s, c)
    if op == "quant":
        x = s["x"].double()
        if c["form"] == "swiglu":
            x = _plain_swiglu(s["x"], s["u"])
        return [_rounded(_columns(x) if c["form"] == "columns" else x)]
    if op == "gemm":
        a = _decode(_unpack(s["Q"]), s["S"]) if c["a"] == "codes" else _rounded(s["x"])
        return [(a @ _decode(_unpack(s["W"]), s["Sw"]).t()).to(TYPES[c["out"]])]
    if op == "linear":
        typ = TYPES[c["type"]]
        y = _rounded(s["x"]) @ _rounded(s["w"]).t()
        dx = _rounded(s["dy"]) @ _rounded(_columns(s["w"])).t()
        dw = _rounded(_columns(s["dy"])) @ _rounded(_columns(s["x"])).t()
        return [y.to(typ), dx.to(typ), dw]
    return [_plain_experts(s, c)]


# ------------------------------------------------------------ the calls ----

def _calls(s, c):
    pkg, lib = _own()
    st, op = s["stream"], c["op"]

    def ptr(t):
        return t.data_ptr() if t is not None else None

    def mat(q, sc):
        return pkg.qmat(pkg.DSV4_WFP4, ptr(q), ptr(sc), q.shape[0], 2 * q.shape[1], 1, 32)

    if op == "route":
        r = pkg.Router(SCORE[c["score"]], c["experts"], c["topk"], c["groups"], c["kept"], c["top"], int(c["renorm"]), SCALE)
        typ = CODE[c["type"]]
        lib.route_groups_dev(ptr(s["idx"]), ptr(s["w"]), ptr(s["scores"]), ptr(s["x"]), typ, c["n"], ptr(s["bias"]), r, st)
        out = [s["idx"], s["w"]] + ([s["scores"]] if c["aux"] else [])
        if c["grad"]:
            lib.route_groups_bwd_dev(ptr(s["dx"]), ptr(s["dw"]), ptr(s["ds"]), ptr(s["x"]), typ, ptr(s["idx"]), c["n"], r,
                                     st)
            out.append(s["dx"])
        return out
    if op == "quant":
        n, k, typ = c["n"], c["k"], CODE[c["type"]]
        q, sc = s["Q"], s["S"]
        if c["form"] == "swiglu":
            lib.swiglu_quant_mxfp4_dev(ptr(q), ptr(sc), ptr(s["x"]), ptr(s["u"]), typ, k, n, k, LIMIT, st)
        elif c["form"] == "columns":
            lib.quant_mxfp4_t_dev(ptr(q), ptr(sc), ptr(s["x"]), typ, k, n, k, st)
        else:
            lib.quant_mxfp4_dev(ptr(q), ptr(sc), ptr(s["x"]), typ, k, n, k, st)
        lib.dequant_dev(ptr(s["V"]), mat(q, sc), st)
        return [s["V"]]
    if op == "gemm":
        if c["a"] != "codes":
            lib.quant_mxfp4_dev(ptr(s["Q"]), ptr(s["S"]), ptr(s["x"]), CODE[c["a"]], c["k"], c["m"], c["k"], st)
        lib.gemm_mxfp4q_dev(ptr(s["C"]), CODE[c["out"]], ptr(s["Q"]), ptr(s["S"]), c["m"], mat(s["W"], s["Sw"]), st)
        return [s["C"]]
    if op == "linear":
        m, n, k, typ = c["m"], c["n"], c["k"], CODE[c["type"]]
        for to, x, rows, cols in ((s["xq"], s["x"], m, k), (s["wq"], s["w"], n, k), (s["dyq"], s["dy"], m, n)):
            lib.quant_mxfp4_dev(ptr(to[0]), ptr(to[1]), ptr(x), typ, cols, rows, cols, st)
        for to, x, rows, cols in ((s["xt"], s["x"], m, k), (s["wt"], s["w"], n, k), (s["dyt"], s["dy"], m, n)):
            lib.quant_mxfp4_t_dev(ptr(to[0]), ptr(to[1]), ptr(x), typ, cols, rows, cols, st)
        for out, code, a, rows, w in ((s["y"], typ, s["xq"], m, s["wq"]), (s["dx"], typ, s["dyq"], m, s["wt"]),
                                      (s["dw"], 0, s["dyt"], n, s["xt"])):
            lib.gemm_mxfp4q_dev(ptr(out), code, ptr(a[0]), ptr(a[1]), rows, mat(*w), st)
        return [s["y"], s["dx"], s["dw"]]
    lib.gemm_mxfp4q_grouped_dev(ptr(s["C"]), CODE[c["out"]], ptr(s["Q"]), ptr(s["S"]), c["tokens"], ptr(s["row_tok"]),
                                c["tokens"] * c["topk"], ptr(s["off"]), ptr(s["table"]), c["experts"], c["n"], c["k"], st)
    return [s["C"]]


def run(state):
    return _calls(state, state["case"]) if own else _plain(state, state["case"])


# ------------------------------------------------------------------- work ----

def _experts_hit(c):
    """Expected number of experts that some token chooses, from each one's share of the choices."""
    p = [(i + 1) ** -c["zipf"] for i in range(c["experts"])]
    tot = sum(p)
    return sum(1 - (1 - min(1.0, c["topk"] * q / tot)) ** c["tokens"] for q in p)


def _held(elements):
    """Bytes of elements held as codes and scales."""
    return elements / 2 + elements / 32


def work(case):
    c, op = case, case["op"]
    el = 4 if c.get("type") == "f32" else 2
    if op == "route":
        n, e = c["n"], c["experts"]
        b = n * e * el + 8 * n * c["topk"] + (4 * e if c["bias"] else 0) + (4 * n * e if c["aux"] else 0)
        if c["grad"]:
            b += 2 * n * e * el + 8 * n * c["topk"] + (4 * n * e if c["aux"] else 0)
        return {"bytes": b, "flops": n * e * (20 if c["grad"] else 10)}
    if op == "quant":
        n, k, z = c["n"], c["k"], 2 if c["form"] == "swiglu" else 1
        out = k * _ceil32(n) if c["form"] == "columns" else n * k
        return {"bytes": n * k * z * el + _held(out) + 4 * out, "flops": (12 if z == 2 else 4) * n * k}
    if op == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        a = _held(m * k) if c["a"] == "codes" else m * k * (4 if c["a"] == "f32" else 2)
        return {"bytes": a + _held(n * k) + m * n * (4 if c["out"] == "f32" else 2), "flops": 2 * m * n * k}
    if op == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": el * (2 * m * k + 2 * m * n + n * k) + 4 * n * k, "flops": 6 * m * n * k}
    r, n, k = c["tokens"] * c["topk"], c["n"], c["k"]
    return {"bytes": _experts_hit(c) * _held(n * k) + _held(c["tokens"] * k) + r * (n * (4 if c["out"] == "f32" else 2) + 4),
            "flops": 2 * r * n * k}


# ------------------------------------------------------------------ exact ----

def _exact_values(x):
    """The 4-bit values of fp64 rows: the least power of two that keeps a block within 6, then the nearest value."""
    out = torch.empty_like(x)
    power = torch.tensor([2.0 ** e for e in range(-300, 301)], dtype=torch.float64, device=x.device)
    near = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], dtype=torch.float64, device=x.device)
    rows = max(1, (1 << 24) // x.shape[1])
    for i in range(0, x.shape[0], rows):
        b = x[i:i + rows].unflatten(-1, (-1, 32))
        top = b.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(top > 0, top, 6.0) / 6)).long() + 300
        e = torch.where(6 * power[e - 1] >= top, e - 1, e)
        e = torch.where(6 * power[e] < top, e + 1, e)
        step = power[torch.where(top > 0, e, 300).clamp(min=300 - 127)]
        a = b.abs() / step
        best, dist = torch.zeros_like(a), a.clone()
        for v in near[1:]:                         # a value with an even code wins a tie: they come first
            d = (a - v).abs()
            best = torch.where(d < dist, v, best)
            dist = torch.minimum(dist, d)
        out[i:i + rows] = (best * torch.sign(b) * step).flatten(-2)
    return out


def _exact_held(q, s):
    table = torch.tensor(VALUES + [-v for v in VALUES], dtype=torch.float64, device=q.device)
    v = torch.empty(*q.shape[:-1], 2 * q.shape[-1], dtype=torch.float64, device=q.device)
    v[..., 0::2], v[..., 1::2] = table[(q % 16).long()], table[(q // 16).long()]
    power = torch.tensor([2.0 ** (e - 127) for e in range(256)], dtype=torch.float64, device=q.device)
    return v * power[s.long()].repeat_interleave(32, dim=-1)


def _exact_columns(x):
    t = torch.zeros(x.shape[1], -(-x.shape[0] // 32) * 32, dtype=torch.float64, device=x.device)
    t[:, :x.shape[0]] = x.double().transpose(0, 1)
    return _exact_values(t)


def _exact_route(s, c):
    x = s["x"].double()
    n, e = x.shape
    sc = torch.sigmoid(x) if c["score"] == "sigmoid" else torch.softmax(x, -1)
    choice = sc.float() + (s["bias"] if s["bias"] is not None else 0.0)
    place = torch.arange(e, device=DEV).expand(n, e)

    def largest(v, ids):
        """The largest value's place, the lowest among equals, and what it is."""
        m = v.max(-1, keepdim=True).values
        return torch.where(v == m, ids, v.shape[-1]).min(-1).values, m.squeeze(-1)

    if c["groups"] > 1:
        g, per = c["groups"], e // c["groups"]
        best = torch.zeros(n, g, device=DEV)
        for j in range(g):
            v = choice[:, j * per:(j + 1) * per].clone()
            for _ in range(c["top"]):
                at, m = largest(v, place[:, :per])
                best[:, j] += m
                v[torch.arange(n, device=DEV), at] = -math.inf
        allowed = torch.zeros(n, g, dtype=torch.bool, device=DEV)
        for _ in range(c["kept"]):
            at, _m = largest(best, place[:, :g])
            allowed[torch.arange(n, device=DEV), at] = True
            best[torch.arange(n, device=DEV), at] = -math.inf
        choice = torch.where(allowed.repeat_interleave(per, 1), choice, -math.inf)
    idx = []
    for _ in range(c["topk"]):
        at, _m = largest(choice, place)
        idx.append(at)
        choice = choice.clone()
        choice[torch.arange(n, device=DEV), at] = -math.inf
    idx = torch.stack(idx, 1)
    # weights and gradients by differentiation of the definition
    x = x.clone().requires_grad_(True)
    sc = torch.sigmoid(x) if c["score"] == "sigmoid" else torch.softmax(x, -1)
    w = sc.gather(1, idx)
    w = SCALE * (w / w.sum(-1, keepdim=True) if c["renorm"] else w)
    out = [None, w.detach()] + ([sc.detach()] if c["aux"] else [])
    if c["grad"]:
        loss = (w * s["dw"].double()).sum()
        if c["aux"]:
            loss = loss + (sc * s["ds"].double()).sum()
        out.append(torch.autograd.grad(loss, x)[0])
    return out


def exact(case, seed):
    """From each operator's definition in 64 bits, not by the plain form's steps."""
    s, c = prepare(case, seed), case
    op = c["op"]
    if op == "route":
        return _exact_route(s, c)
    if op == "quant":
        x = s["x"].double()
        if c["form"] == "swiglu":
            g, u = torch.minimum(x, torch.full_like(x, LIMIT)), s["u"].double()
            x = g * torch.sigmoid(g) * torch.maximum(torch.minimum(u, torch.full_like(u, LIMIT)), torch.full_like(u, -LIMIT))
        return [_exact_columns(x) if c["form"] == "columns" else _exact_values(x)]
    if op == "gemm":
        a = _exact_held(s["Q"], s["S"]) if c["a"] == "codes" else _exact_values(s["x"].double())
        return [a @ _exact_held(s["W"], s["Sw"]).t().contiguous()]
    if op == "linear":
        y = _exact_values(s["x"].double()) @ _exact_values(s["w"].double()).t().contiguous()
        dx = _exact_values(s["dy"].double()) @ _exact_columns(s["w"]).t().contiguous()
        dw = _exact_columns(s["dy"]) @ _exact_columns(s["x"]).t().contiguous()
        return [y, dx, dw]
    off, tok = s["off"].tolist(), s["row_tok"].long()
    out = torch.zeros(s["C"].shape, dtype=torch.float64, device=DEV)
    a = _exact_held(s["Q"], s["S"])
    for e in range(c["experts"]):
        if off[e + 1] > off[e]:
            w = _exact_held(s["W"][e], s["Sw"][e])
            out[off[e]:off[e + 1]] = a[tok[off[e]:off[e + 1]]] @ w.t().contiguous()
    return [out]
