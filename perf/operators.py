"""What users of the 4-bit and mixture-of-experts operators have them do, as cases that can be timed and checked.

The operators serve transformers whose weights lie on the GPU in microscaled 4-bit floating point (MX4: E2M1 codes, one
power-of-two scale for each 32 values of a row):

    quantize   rows of FP16 or FP32 values to MX4 and back
    product    C = A·Wᵀ, W in MX4, A in FP16 or FP32 (decode and prompts), or A quantised to MX4 on the way ("quantized")
    route      a router's logits to the experts of each token and their weights
    experts    the products of each token's rows with its experts' MX4 weights, gated (SiLU) or joined by the router's weights

    own  listed()  draw(rng)  prepare(case, seed)  run(state)  work(case)  exact(case, seed)
"""
import math
import os
import sys

import torch

own = False

TORCH = {"H": torch.float16, "S": torch.float32}
SIZE = {"H": 2, "S": 4}


def listed():
    return [
        # the activations of 16 sequences decoded together, before a product of two MX4 operands
        {"name": "quantize_step", "op": "quantize", "type": "H", "rows": 16, "K": 4096},
        # the first feed-forward weights of a transformer, quantised when they are loaded, and read back
        {"name": "quantize_weights", "op": "quantize", "type": "S", "rows": 11008, "K": 4096},
        # one sequence decoded: one activation row against resident weights
        {"name": "decode_token", "op": "product", "type": "H", "M": 1, "N": 11008, "K": 4096},
        # 24 sequences decoded together, activations in FP32
        {"name": "decode_batch", "op": "product", "type": "S", "M": 24, "N": 4096, "K": 11008},
        # a prompt of 1000 tokens through the same weights
        {"name": "prompt", "op": "product", "type": "H", "M": 1000, "N": 11008, "K": 4096},
        # long prompts whose activations are quantised too: both operands of the product in 4 bits
        {"name": "prompt_quantized", "op": "quantized", "type": "H", "M": 4096, "N": 11008, "K": 4096},
        # the router of one decoded token
        {"name": "route_token", "op": "route", "type": "S", "T": 1, "E": 64, "k": 8, "score": "softmax", "groups": 1,
         "top_groups": 1, "bias": False, "renorm": True, "scale": 1.0},
        # the router of a long prompt: sigmoid scores, a bias for balance, experts in groups
        {"name": "route_prompt", "op": "route", "type": "S", "T": 8192, "E": 256, "k": 8, "score": "sigmoid", "groups": 8,
         "top_groups": 4, "bias": True, "renorm": True, "scale": 2.5},
        # the first products of one decoded token's experts, gate and up, with the gate's SiLU
        {"name": "experts_token", "op": "experts", "type": "H", "form": "gated", "T": 1, "S": 8, "E": 64, "N": 1536, "K": 4096},
        # the second products of 24 sequences decoded together, joined by the router's weights, in FP32
        {"name": "experts_step", "op": "experts", "type": "S", "form": "joined", "T": 24, "S": 4, "E": 64, "N": 4096, "K": 1536},
        # the first products of a prompt's experts
        {"name": "experts_prompt", "op": "experts", "type": "H", "form": "gated", "T": 2048, "S": 4, "E": 64, "N": 1536, "K": 4096},
        # the second products of a prompt of odd length
        {"name": "experts_join", "op": "experts", "type": "H", "form": "joined", "T": 2047, "S": 4, "E": 64, "N": 4096, "K": 1536},
    ]


# ---------------------------------------------------------------------------------------------------------------
# More cases of the same ranges
# ---------------------------------------------------------------------------------------------------------------
def _spread(rng, lo, hi, step=1):
    """A size spread over the logarithm of [lo, hi], a multiple of `step`."""
    n = round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step) * step
    return min(max(n, -(-lo // step) * step), hi // step * step)


def draw(rng):
    op = rng.choice(("quantize", "product", "product", "product", "quantized", "route", "experts", "experts", "experts"))
    t = rng.choice(("H", "S"))
    if op == "quantize":
        # activations (few rows) and weights (many); any row length
        return {"op": op, "type": t, "rows": _spread(rng, 1, 11008), "K": _spread(rng, 64, 4096, rng.choice((1, 32, 128)))}
    if op in ("product", "quantized"):
        while True:
            # widths of linear layers, in multiples of 32; sometimes (an output head) any number of outputs
            M = _spread(rng, 1, 1000 if op == "product" else 4096)
            N, K = _spread(rng, 512, 11008, 64), _spread(rng, 512, 11008, rng.choice((32, 128)))
            if rng.random() < 0.25:
                N -= rng.randrange(64)
            if M * N * K <= (1000 if op == "product" and t == "H" else 300 if op == "product" else 4096) * 11008 * 4096:
                return {"op": op, "type": t, "M": M, "N": N, "K": K}
    if op == "route":
        score = rng.choice(("softmax", "sigmoid"))
        E = rng.choice((8, 16, 40, 64, 96, 128, 160, 256, 384))
        groups = rng.choice((1, 1, 4, 8)) if E >= 32 else 1
        top = rng.randint(1, groups)
        return {"op": op, "type": t, "T": _spread(rng, 1, 8192), "E": E, "k": rng.randint(1, min(10, E // groups * top)),
                "score": score, "groups": groups, "top_groups": top, "bias": score == "sigmoid" and rng.random() < 0.7,
                "renorm": rng.random() < 0.7, "scale": rng.choice((1.0, 2.5))}
    form = rng.choice(("gated", "joined"))
    E = rng.choice((8, 16, 40, 64))
    wide, narrow = _spread(rng, 1024, 4096, 128), _spread(rng, 256, 2048, rng.choice((32, 64)))
    N, K = (narrow, wide) if form == "gated" else (wide, narrow)
    S, T = rng.randint(1, min(8, E)), _spread(rng, 1, 2048)
    if T * S > (8192 if t == "H" else 2048):
        T = max(1, (8192 if t == "H" else 2048) // S)
    return {"op": op, "type": t, "form": form, "T": T, "S": S, "E": E, "N": N, "K": K}


# ---------------------------------------------------------------------------------------------------------------
# Inputs: from the seed alone
# ---------------------------------------------------------------------------------------------------------------
def _normal(g, *shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale)


def _weights(g, *shape):
    """MX4 weights as a checkpoint holds them: rows of codes, two to a byte (the even one in the low half), and rows of
    scales (exponent + 127), quantised from normal values of a linear layer's size."""
    w = _normal(g, *shape, scale=1 / math.sqrt(shape[-1])).view(*shape[:-1], -1, 32)
    e = torch.frexp(w.abs().amax(-1, keepdim=True))[1] - 3
    codes = torch.bucketize(_e2m1(w * _power(-e)).abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda"))
    codes = (codes.to(torch.uint8) | ((w < 0).to(torch.uint8) << 3)).view(*shape)
    return codes[..., 0::2] | codes[..., 1::2] << 4, (e + 127).to(torch.uint8).squeeze(-1)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, t = case["op"], TORCH[case["type"]]
    if op == "quantize":
        # activations after a norm: normal values, with channels of larger ones
        x = _normal(g, case["rows"], case["K"])
        return {"X": (x * torch.exp(_normal(g, case["K"], scale=0.7))).to(t)}
    if op in ("product", "quantized"):
        codes, scales = _weights(g, case["N"], case["K"])
        return {"A": _normal(g, case["M"], case["K"]).to(t), "codes": codes, "scales": scales}
    if op == "route":
        d = {"logits": _normal(g, case["T"], case["E"], scale=1.5).to(t)}
        if case["bias"]:
            d["bias"] = _normal(g, case["E"], scale=0.1)
        return d
    T, S, E, N, K = (case[k] for k in "TSENK")
    # experts as a router chooses them: some more often than others
    liking = _normal(g, T, E) + _normal(g, E, scale=0.5)
    p, ids = torch.topk(torch.softmax(liking, -1), S)
    gated = case["form"] == "gated"
    # gated: the experts of a token share its row; joined: each has the row that its first products left
    d = {"ids": ids.int(), "X": _normal(g, *((T, K) if gated else (T, S, K))).to(t),
         "cap": int(torch.bincount(ids.flatten(), minlength=E).max())}
    d["codes"], d["scales"] = _weights(g, E, N, K)
    if gated:
        d["gate_codes"], d["gate_scales"] = _weights(g, E, N, K)
    else:
        d["weights"] = p / p.sum(-1, keepdim=True)
    return d


# ---------------------------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------------------------
def _power(e):
    """2^e in FP32 for whole e of -126 to 127."""
    return ((e + 127).int() << 23).view(torch.float32)


def _e2m1(a):
    """The nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, ties to the even code, beyond 6 to 6."""
    m = a.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    return torch.copysign((torch.round(m / step) * step).clamp(max=6.0), a)


def _rounded(x):
    """Rows of x at MX4's precision, in FP32: blocks of 32 share the scale 2^(⌊log2 of the largest⌋ − 2)."""
    rows, K = x.shape
    b = torch.nn.functional.pad(x.float(), (0, -K % 32)).view(rows, -1, 32)
    e = torch.frexp(b.abs().amax(-1, keepdim=True))[1] - 3
    return (_e2m1(b * _power(-e)) * _power(e)).view(rows, -1)[:, :K]


def _values(codes, scales):
    """The FP32 values of MX4 rows."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    c = torch.stack((codes & 15, codes >> 4), -1).view(*scales.shape, 32).int()
    v = torch.cat((table, -table)).index_select(0, c.flatten()).view(c.shape)
    return (v * _power(scales.int() - 127).unsqueeze(-1)).flatten(-2)


def _plain_route(s):
    x, T = s["logits"].float(), s["logits"].shape[0]
    if s["score"] == "sigmoid":
        score = 1 / (1 + torch.exp(-x))
        choice = score + s["bias"] if s["bias"] is not None else score
    else:
        score = torch.exp(x - x.amax(-1, keepdim=True))
        score = score / score.sum(-1, keepdim=True)
        choice = x   # the logits are in the order of their softmax
    if s["groups"] > 1:
        # the groups with the largest sum of two choices (sigmoid) or the largest choice (softmax)
        top = choice.view(T, s["groups"], -1).sort(dim=-1, descending=True)[0]
        of_group = top[..., 0] + top[..., 1] if s["score"] == "sigmoid" else top[..., 0]
        best = of_group.sort(dim=-1, descending=True, stable=True)[1][:, :s["top_groups"]]
        keep = torch.zeros_like(of_group, dtype=torch.bool).scatter_(1, best, True)
        choice = torch.where(keep.repeat_interleave(top.shape[-1], 1), choice, -math.inf)
    ids = choice.sort(dim=-1, descending=True, stable=True)[1][:, :s["k"]]
    w = score.gather(1, ids)
    if s["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return ids.int(), w * s["scale"]


def _plain_experts(s):
    ids, X = s["ids"], s["X"]
    T, S = ids.shape
    used, mine = torch.unique(ids.flatten(), return_inverse=True)
    order = mine.sort(stable=True)[1]                      # slots by expert
    count = torch.zeros_like(used, dtype=torch.int64).scatter_add_(0, mine, torch.ones_like(mine))
    place = torch.empty_like(mine)                         # of a slot among its expert's
    place[order] = torch.arange(T * S, device="cuda") - (count.cumsum(0) - count)[mine[order]]
    rows = (X if X.dim() == 3 else X[:, None].expand(T, S, -1)).float().reshape(T * S, -1)
    padded = torch.zeros((len(used), s["cap"], rows.shape[1]), device="cuda")
    padded[mine, place] = rows

    def product(codes, scales):
        return torch.bmm(padded, _values(codes[used], scales[used]).transpose(1, 2))[mine, place].view(T, S, -1)

    y = product(s["codes"], s["scales"])
    if s["form"] == "gated":
        z = product(s["gate_codes"], s["gate_scales"])
        return (z / (1 + torch.exp(-z)) * y).to(X.dtype)
    return (y * s["weights"].unsqueeze(-1)).sum(1).to(X.dtype)


# ---------------------------------------------------------------------------------------------------------------
# A pass
# ---------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    """What a program holds before the call: operands on the GPU, the weights (for the framework's calls laid out by it
    once) and, there, result buffers that are used again and again."""
    s = {**_inputs(case, seed), **{k: case[k] for k in ("op", "form", "score", "groups", "top_groups", "k", "renorm", "scale") if k in case}}
    s.setdefault("bias", None)
    if not own:
        return s
    sys.path.insert(0, os.path.join(os.getcwd(), "gen9-gpu-blas_amd"))
    import gen9blas
    s["g9"] = gen9blas
    gen9blas.set_nowait(True)   # device operands: calls queue on the library's stream and return
    if "codes" in s:
        s["W"] = gen9blas.mx4_load(s.pop("codes"), s.pop("scales"))
    if "gate_codes" in s:
        s["gate"] = gen9blas.mx4_load(s.pop("gate_codes"), s.pop("gate_scales"))
    op = case["op"]
    if op in ("quantize", "quantized"):
        X = s["X"] if op == "quantize" else s["A"]
        s["Q"] = gen9blas.MX4(*X.shape)
    if op == "quantize":
        s["Y"] = torch.empty(s["X"].shape, device="cuda")
    elif op in ("product", "quantized"):
        s["C"] = torch.empty((case["M"], case["N"]), dtype=s["A"].dtype, device="cuda")
    elif op == "route":
        s["ids"] = torch.empty((case["T"], case["k"]), dtype=torch.int32, device="cuda")
        s["w"] = torch.empty((case["T"], case["k"]), device="cuda")
    else:
        shape = (case["T"], case["S"], case["N"]) if case["form"] == "gated" else (case["T"], case["N"])
        s["C"] = torch.empty(shape, dtype=s["X"].dtype, device="cuda")
    return s


def run(s):
    return _own_run(s, s["g9"]) if own else _plain_run(s)


def _own_run(s, g9):
    op = s["op"]
    if op == "quantize":
        return g9.mx4_dequantize(g9.mx4_quantize(s["X"], out=s["Q"]), out=s["Y"])
    if op == "product":
        return g9.mx4_gemm(s["A"], s["W"], C=s["C"])
    if op == "quantized":
        return g9.mx4_gemm(g9.mx4_quantize(s["A"], out=s["Q"]), s["W"], C=s["C"])
    if op == "route":
        return g9.moe_route(s["logits"], s["k"], bias=s["bias"], score=s["score"], groups=s["groups"],
                            top_groups=s["top_groups"], renorm=s["renorm"], scale=s["scale"], out=(s["ids"], s["w"]))
    return g9.moe_gemm(s["X"], s["ids"], s["W"], gate=s.get("gate"), weights=s.get("weights"), C=s["C"])


def _plain_run(s):
    op = s["op"]
    if op == "quantize":
        return _rounded(s["X"])
    if op in ("product", "quantized"):
        A = s["A"].float() if op == "product" else _rounded(s["A"])
        return (A @ _values(s["codes"], s["scales"]).t()).to(s["A"].dtype)
    return _plain_route(s) if op == "route" else _plain_experts(s)


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def _mx4_bytes(rows, K):
    return rows * (K / 2 + K / 32)


def work(case):
    op, es = case["op"], SIZE[case["type"]]
    if op == "quantize":
        n = case["rows"] * case["K"]
        return {"bytes": es * n + 2 * _mx4_bytes(case["rows"], case["K"]) + 4 * n, "flops": 4.0 * n}
    if op in ("product", "quantized"):
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": es * (M * K + M * N) + _mx4_bytes(N, K), "flops": 2.0 * M * N * K}
    if op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        return {"bytes": es * T * E + 8 * T * k + (4 * E if case["bias"] else 0), "flops": 5.0 * T * E}
    T, S, E, N, K = (case[k] for k in "TSENK")
    pairs = 2 if case["form"] == "gated" else 1
    used = E * (1 - (1 - S / E) ** T)   # experts that some token has, were all equally likely
    rows_in, rows_out = (T, T * S) if case["form"] == "gated" else (T * S, T)
    return {"bytes": es * (rows_in * K + rows_out * N) + pairs * used * _mx4_bytes(N, K) + 8 * T * S, "flops": 2.0 * pairs * T * S * N * K}


# ---------------------------------------------------------------------------------------------------------------
# The same results from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_values(codes, scales):
    both = torch.stack((codes % 16, codes // 16), dim=-1).flatten(-2).long()
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), dtype=torch.float64, device=codes.device)
    return grid[both] * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def _exact_rounded(x):
    rows, K = x.shape
    x = torch.cat((x.double(), x.new_zeros((rows, -K % 32), dtype=torch.float64)), 1).view(rows, -1, 32)
    largest = x.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(largest.clamp(min=2.0 ** -120))) - 2)
    a, q = x.abs() / scale, torch.zeros_like(x)
    for code in range(1, 8):   # the midpoint below a level rounds to the level if its code is even
        mid = (_GRID[code - 1] + _GRID[code]) / 2
        q = torch.where(a >= mid if code % 2 == 0 else a > mid, torch.full_like(q, _GRID[code]), q)
    return (torch.sign(x) * q * scale).view(rows, -1)[:, :K]


def exact(case, seed):
    d, op = _inputs(case, seed), case["op"]
    if op == "quantize":
        return _exact_rounded(d["X"])
    if op in ("product", "quantized"):
        A = d["A"].double() if op == "product" else _exact_rounded(d["A"])
        return torch.mm(A, _exact_values(d["codes"], d["scales"]).t())
    if op == "route":
        x = d["logits"].double()
        p = torch.sigmoid(x) if case["score"] == "sigmoid" else torch.softmax(x, -1)
        choice = p + d["bias"].double() if case["bias"] else p
        G = case["groups"]
        if G > 1:
            per = choice.view(len(x), G, -1)
            of_group = torch.topk(per, 2 if case["score"] == "sigmoid" else 1)[0].sum(-1)
            rank = torch.argsort(torch.argsort(of_group, dim=-1, descending=True, stable=True), dim=-1)
            choice = per.masked_fill((rank >= case["top_groups"]).unsqueeze(-1), -math.inf).flatten(1)
        w = p.gather(1, torch.topk(choice, case["k"])[1])
        return None, (w / w.sum(-1, keepdim=True) if case["renorm"] else w) * case["scale"]
    T, S = d["ids"].shape
    X = d["X"].double().view(T, -1, case["K"]).expand(T, S, case["K"])
    y = torch.zeros((T, S, case["N"]), dtype=torch.float64, device=X.device)
    for e in range(case["E"]):
        t, s = torch.nonzero(d["ids"] == e, as_tuple=True)
        if len(t):
            y[t, s] = X[t, s] @ _exact_values(d["codes"][e], d["scales"][e]).t()
            if case["form"] == "gated":
                z = X[t, s] @ _exact_values(d["gate_codes"][e], d["gate_scales"][e]).t()
                y[t, s] *= z * torch.sigmoid(z)
    return y if case["form"] == "gated" else torch.einsum("tsn,ts->tn", y, d["weights"].double())
