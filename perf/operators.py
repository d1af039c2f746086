"""Cases of the row operators around a mixture of experts: rows sorted by expert and back, their gradients, and matrix
products in 8-bit integers with a scale for each token and channel.

  sort     pairs (token, slot) sorted by expert, and the token rows in that order (elements, or 8-bit codes with scales)
  merge    rows in expert order back to their tokens: weighted sum over the slots; without weights the gradient of `sort`
  grad     the weighted sum's gradients: of the rows and of the weights
  product  rows times one matrix of 8-bit codes (a shared expert's projections)
  experts  rows in expert order times the matrix of each row's expert

Sizes are those of the repository's layer (hidden 2048, 256 experts, top-8, expert intermediate 512) and what lies below
them.  Inputs are synthetic and made on the device from the seed.
"""
from __future__ import annotations

import torch

own = False

D, F, E, K = 2048, 512, 256, 8
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4, "int8": 1}


def _sort(tokens, dtype, *, d=D, experts=E, top_k=K, held=1.0, skew=0.0, out=""):
    """held: share of the experts that this rank has; pairs of the others are not sorted.  out: "int8" for codes."""
    return {"kind": "sort", "tokens": tokens, "dtype": dtype, "out": out or dtype, "d": d, "experts": experts,
            "top_k": top_k, "held": held, "skew": skew}


def _merge(tokens, dtype, *, d=D, experts=E, top_k=K, held=1.0, weights="fp16", base=False, grad=False):
    """weights: their type, or "none"; base: rows that the sum is added to (a shared expert's output)."""
    return {"kind": "grad" if grad else "merge", "tokens": tokens, "dtype": dtype, "d": d, "experts": experts,
            "top_k": top_k, "held": held, "weights": weights, "base": base}


def _product(rows, dtype, k, n, *, out="fp16", gated=False):
    return {"kind": "product", "rows": rows, "dtype": dtype, "k": k, "n": n, "out": out, "gated": gated}


def _experts(tokens, dtype, k, n, *, out="fp16", gated=False, experts=E, top_k=K, skew=0.0):
    return {"kind": "experts", "tokens": tokens, "dtype": dtype, "k": k, "n": n, "out": out, "gated": gated,
            "experts": experts, "top_k": top_k, "skew": skew}


def listed():
    named = [
        # one decoded token to its eight experts: the smallest call, all latency
        ("sort_1token_fp16", _sort(1, "fp16")),
        # a short prompt's rows as 8-bit codes for the product below
        ("sort_201tokens_int8", _sort(201, "fp16", out="int8")),
        # a full chunk of training rows, some experts popular
        ("sort_4096tokens_bf16_skewed", _sort(4096, "bf16", skew=0.8)),
        # a decoded token's expert rows back, added to the shared expert's output
        ("merge_1token_fp16", _merge(1, "fp16", base=True)),
        # a full chunk back to its tokens
        ("merge_4096tokens_bf16", _merge(4096, "bf16", weights="fp32")),
        # the gradient of the sorting, on a rank that has a quarter of the experts
        ("sum_1531tokens_fp32_64of256", _merge(1531, "fp32", weights="none", held=0.25)),
        # the weighted sum's gradients
        ("grad_1531tokens_bf16", _merge(1531, "bf16", weights="fp32", grad=True)),
        # a shared expert's gate and up rows for one decoded token
        ("product_1row_gated", _product(1, "fp16", D, F, gated=True)),
        # the same for a ragged chunk, down projection back to the hidden size
        ("product_1531rows_bf16", _product(1531, "bf16", F, D, out="bf16")),
        # one decoded token through its eight experts' gate and up rows
        ("experts_1token_gated", _experts(1, "fp16", D, F, gated=True)),
        # a short prompt's activations through the experts' down rows
        ("experts_201tokens_down", _experts(201, "fp16", F, D, out="fp32")),
        # a full chunk of sorted codes through the experts' gate and up rows
        ("experts_4096tokens_gated", _experts(4096, "int8", D, F, gated=True)),
    ]
    return [dict(c, name=name) for name, c in named]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("sort", "merge", "grad", "product", "experts", "experts"))
    dtype = rng.choice(("fp16", "bf16", "fp32"))
    experts = _log_int(rng, 8, E)
    top_k = rng.randint(1, K)
    if kind in ("sort", "merge", "grad"):
        tokens, d = _log_int(rng, 1, 4096), _log_int(rng, 48, D)
        held = rng.choice((1.0, 1.0, round(rng.uniform(0.1, 0.9), 2)))
        if kind == "sort":
            return _sort(tokens, dtype, d=d, experts=experts, top_k=top_k, held=held, out=rng.choice(("", "int8")),
                         skew=rng.choice((0.0, round(rng.uniform(0.3, 1.2), 2))))
        weights = rng.choice(("none", "fp16", "fp32", "bf16") if kind == "merge" else ("fp16", "fp32", "bf16"))
        return _merge(tokens, dtype, d=d, experts=experts, top_k=top_k, held=held, weights=weights,
                      base=kind == "merge" and rng.random() < 0.5, grad=kind == "grad")
    k, n = _log_int(rng, 48, D), _log_int(rng, 24, D if kind == "product" else D // 2)
    out, gated = rng.choice(("fp16", "bf16", "fp32")), rng.random() < 0.5
    if kind == "product":
        return _product(_log_int(rng, 1, 4096), dtype, k, n // 2 if gated else n, out=out, gated=gated)
    return _experts(_log_int(rng, 1, 900), rng.choice((dtype, "int8")), k, n // 2 if gated else n, out=out, gated=gated,
                    experts=experts, top_k=top_k, skew=rng.choice((0.0, round(rng.uniform(0.3, 1.0), 2))))


def _stride(n):
    """Codes of a row start on 16-byte boundaries."""
    return -(-n // 16) * 16


def _route(tokens, experts, top_k, skew, gen):
    """Distinct experts of each token, int32 [tokens][top_k]; skew: popularity about as 1 / rank^skew."""
    score = -torch.log(-torch.log(torch.rand((tokens, experts), device="cuda", generator=gen).clamp(1e-12, 1 - 1e-7)))
    rank = torch.randperm(experts, device="cuda", generator=gen).float() + 1.0
    return (score - skew * torch.log(rank)).topk(top_k, dim=1).indices.to(torch.int32)


def _plan(idx, held):
    """position, source, begin of the pairs whose expert is below `held`."""
    flat = idx.reshape(-1).long()
    order = torch.sort(torch.where(flat < held, flat, held), stable=True).indices
    ends = torch.cumsum(torch.bincount(flat.clamp(max=held), minlength=held + 1)[:held], 0)
    begin = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    kept = torch.arange(flat.numel(), device="cuda") < begin[-1]
    source = torch.where(kept, order, -1).to(torch.int32)
    position = torch.empty_like(source)
    position[order] = torch.where(kept, torch.arange(flat.numel(), device="cuda"), -1).to(torch.int32)
    return position.view_as(idx), source, begin


def _codes(rows, n, gen, scale):
    """Codes of normally distributed rows [rows][n] with a scale each, in rows of whole 16-byte pieces."""
    x = torch.randn((rows, n), device="cuda", generator=gen)
    low, high = torch.aminmax(x, dim=1)
    top = torch.maximum(-low, high)
    q = torch.zeros((rows, _stride(n)), dtype=torch.int8, device="cuda")
    q[:, :n] = x.mul_((127.0 / top)[:, None]).round_()
    return q, top * (scale / 127.0)


class State:
    pass


def prepare(case, seed):
    s = State()
    s.case, kind = case, case["kind"]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s.stream = torch.cuda.current_stream()
    normal = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    if kind in ("sort", "merge", "grad"):
        tokens, d, top_k = case["tokens"], case["d"], case["top_k"]
        s.dtype = TYPES[case["dtype"]]
        s.held = max(1, round(case["experts"] * case["held"]))
        s.idx = _route(tokens, case["experts"], top_k, case.get("skew", 0.0), gen)
        if kind == "sort":
            s.x = normal(tokens, d).to(s.dtype)
            int8 = case["out"] == "int8"
            s.position = torch.empty((tokens, top_k), dtype=torch.int32, device="cuda")
            s.source = torch.empty(tokens * top_k, dtype=torch.int32, device="cuda")
            s.begin = torch.empty(s.held + 1, dtype=torch.int32, device="cuda")
            s.rows = torch.zeros((tokens * top_k, _stride(d) if int8 else d), dtype=torch.int8 if int8 else s.dtype, device="cuda")
            s.scales = torch.zeros(tokens * top_k, device="cuda") if int8 else None
            s.workspace = None
            return s
        s.position, _, begin = _plan(s.idx, s.held)
        s.kept = int(begin[-1])
        s.rows = normal(max(1, s.kept), d).to(s.dtype)
        w = torch.softmax(normal(tokens, top_k), dim=1)
        s.w = None if case["weights"] == "none" else w.to(TYPES[case["weights"]])
        s.base = normal(tokens, d).to(s.dtype) if case["base"] else None
        if kind == "merge":
            s.y = torch.empty((tokens, d), dtype=s.dtype, device="cuda")
        else:
            s.dy = normal(tokens, d).to(s.dtype)
            s.drows = torch.zeros_like(s.rows)
            s.dw = torch.empty((tokens, top_k), device="cuda")
        return s
    k, n = case["k"], case["n"]
    channels = 2 * n if case["gated"] else n
    s.experts = case["experts"] if kind == "experts" else 1
    if kind == "experts":
        idx = _route(case["tokens"], s.experts, case["top_k"], case["skew"], gen)
        _, _, s.begin = _plan(idx, s.experts)
        s.count = case["tokens"] * case["top_k"]
        s.most = int((s.begin[1:] - s.begin[:-1]).max())
    else:
        s.begin, s.count, s.most = None, case["rows"], case["rows"]
    if case["dtype"] == "int8":
        s.a, s.a_scales = _codes(s.count, k, gen, 1.0)
    else:
        s.a, s.a_scales = normal(s.count, k).to(TYPES[case["dtype"]]), None
    s.b, scales = _codes(s.experts * channels, k, gen, k ** -0.5)
    s.b, s.b_scales = s.b.view(s.experts, channels, -1), scales.view(s.experts, channels)
    s.out = torch.empty((s.count, n), dtype=TYPES[case["out"]], device="cuda")
    s.workspace = None
    return s


def _quantized(x):
    """Codes (as floats) and scales of rows: s = max / 127, q = rint(x (127 / max)), every step rounded to 32 bits."""
    x = x.float()
    top = x.abs().amax(1, keepdim=True)
    whole = torch.full_like(top, 127.0)
    return torch.where(top > 0, torch.round(x * (whole / top)), 0.0), top / whole


def _run_own(s):
    import nvmai_b200 as nv
    c, kind = s.case, s.case["kind"]
    elem = {"fp16": nv.format.ELEM_F16, "bf16": nv.format.ELEM_BF16, "fp32": nv.format.ELEM_F32, "int8": nv.format.ELEM_I8}
    if kind == "sort":
        if s.workspace is None:       # kept by the program for all its calls of this size
            s.workspace = torch.empty(nv.sort_rows_workspace(c["tokens"], c["top_k"], s.held), dtype=torch.uint8, device="cuda")
        nv.sort_rows(s.idx, c["tokens"], c["top_k"], s.held, s.position, s.source, s.begin, x=s.x, d=c["d"], elem=elem[c["dtype"]],
                     rows=s.rows, rows_elem=elem[c["out"]], rows_stride=s.rows.shape[1], row_scales=s.scales,
                     workspace=s.workspace, workspace_bytes=s.workspace.numel(), stream=s.stream)
        rows = s.rows if s.scales is None else s.rows[:, :c["d"]] * s.scales[:, None]
        return {"position": s.position, "source": s.source, "begin": s.begin, "rows": rows}
    if kind == "merge":
        nv.merge_rows(s.rows, s.kept, s.position, c["tokens"], c["top_k"], c["d"], s.y, elem=elem[c["dtype"]], w=s.w,
                      w_elem=elem.get(c["weights"], nv.format.ELEM_F32), base=s.base, stream=s.stream)
        return {"y": s.y}
    if kind == "grad":
        nv.merge_rows_grad(s.dy, s.rows, s.kept, s.position, s.w, c["tokens"], c["top_k"], c["d"], s.drows, s.dw,
                           elem=elem[c["dtype"]], w_elem=elem[c["weights"]], stream=s.stream)
        return {"drows": s.drows, "dw": s.dw}
    if s.workspace is None:
        size = nv.int8_matmul_workspace(s.count, c["k"], elem[c["dtype"]])
        s.workspace = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
    nv.int8_matmul(s.a, s.b, s.b_scales, s.out, s.count, c["k"], c["n"], a_elem=elem[c["dtype"]], a_stride=s.a.shape[1],
                   a_scales=s.a_scales, b_stride=s.b.shape[2], num_experts=s.experts, expert_begin=s.begin,
                   activation=nv.format.ACT_SILU if c["gated"] else nv.format.ACT_NONE, out_elem=elem[c["out"]],
                   workspace=s.workspace, workspace_bytes=s.workspace.numel(), stream=s.stream)
    return {"out": s.out}


def run(s):
    if own:
        return _run_own(s)
    c, kind = s.case, s.case["kind"]
    if kind == "sort":
        position, source, begin = _plan(s.idx, s.held)
        kept = (source >= 0)[:, None]
        tokens = source.clamp(min=0).long() // c["top_k"]
        if s.scales is None:
            rows = torch.where(kept, s.x[tokens], 0)
        else:
            q, scale = _quantized(s.x)
            rows = torch.where(kept, (q * scale)[tokens], 0.0)
        return {"position": position, "source": source, "begin": begin, "rows": rows}
    if kind in ("merge", "grad"):
        at, kept = s.position.clamp(min=0).long(), s.position >= 0
        if kind == "merge":
            w = kept.float() if s.w is None else torch.where(kept, s.w.float(), 0.0)
            y = (s.rows[at].float() * w[:, :, None]).sum(1)
            return {"y": (y if s.base is None else y + s.base.float()).to(s.dtype)}
        drows = torch.zeros_like(s.rows)
        to = torch.where(kept, at, len(s.rows)).reshape(-1)       # what is not kept goes to a row behind the others
        full = torch.cat([drows, drows[:1]])
        full[to] = (s.dy.float()[:, None, :] * s.w.float()[:, :, None]).to(s.dtype).reshape(-1, c["d"])
        dw = torch.where(kept, (s.rows[at].float() * s.dy.float()[:, None, :]).sum(2), 0.0)
        return {"drows": full[:-1], "dw": dw}
    q, scale = (s.a[:, :c["k"]].float(), s.a_scales[:, None]) if s.a_scales is not None else _quantized(s.a)
    b = s.b[:, :, :c["k"]]
    if s.begin is None:
        acc, b_scales = q @ b[0].float().T, s.b_scales
    else:
        row = torch.arange(s.count, device="cuda")
        expert = torch.searchsorted(s.begin[1:].contiguous(), row.to(torch.int32), right=True)
        if s.count <= s.experts:                 # the matrix of each row's expert
            acc = torch.bmm(b[expert].float(), q[:, :, None])[:, :, 0]
        else:                                    # rows in blocks of their experts, filled up to the longest
            to = expert * s.most + row - s.begin[expert]
            padded = torch.zeros((s.experts * s.most, c["k"]), device="cuda")
            padded[to] = q
            acc = torch.bmm(padded.view(s.experts, s.most, c["k"]), b.float().transpose(1, 2)).flatten(0, 1)[to]
        b_scales = s.b_scales[expert]
    y = acc * scale * b_scales
    if c["gated"]:
        gate, up = y[:, :c["n"]], y[:, c["n"]:]
        y = gate / (1.0 + torch.exp(-gate)) * up
    return {"out": y.to(s.out.dtype)}


def _distinct(tokens, experts, top_k):
    """Experts that have a row, on average, each token taking top_k of them evenly."""
    return experts * (1.0 - (1.0 - top_k / experts) ** tokens)


def work(case):
    kind = case["kind"]
    if kind in ("sort", "merge", "grad"):
        tokens, d, pairs, size = case["tokens"], case["d"], case["tokens"] * case["top_k"], BYTES[case["dtype"]]
        held = max(1, round(case["experts"] * case["held"]))
        kept = pairs * held / case["experts"]
        if kind == "sort":       # indexes and rows in; positions, sources, begins, rows (codes: and their scales) out
            coded = case["out"] == "int8"
            nbytes = 12 * pairs + 4 * (held + 1) + tokens * d * size + kept * (d * BYTES[case["out"]] + (4 if coded else 0))
            return {"bytes": nbytes, "flops": 2 * tokens * d if coded else 0}
        weights = 0 if case["weights"] == "none" else BYTES[case["weights"]]
        if kind == "merge":
            return {"bytes": pairs * (4 + weights) + kept * d * size + (2 if case["base"] else 1) * tokens * d * size,
                    "flops": 2 * kept * d}
        return {"bytes": pairs * (8 + weights) + 2 * kept * d * size + tokens * d * size, "flops": 3 * kept * d}
    k, n = case["k"], case["n"]
    channels = 2 * n if case["gated"] else n
    if kind == "product":
        rows, matrices, extra = case["rows"], 1, 0
    else:
        rows, matrices = case["tokens"] * case["top_k"], _distinct(case["tokens"], case["experts"], case["top_k"])
        extra = 4 * (case["experts"] + 1)
    coded = 4 if case["dtype"] == "int8" else 0
    return {"bytes": extra + rows * (k * BYTES[case["dtype"]] + coded) + matrices * channels * (k + 4) + rows * n * BYTES[case["out"]],
            "flops": 2 * rows * channels * k}


def exact(case, seed):
    """The same in 64 bits from the definitions: positions by counting, sums over one-hot or selected rows, whole-number
    products in double precision.  Codes are the ones that the definition's steps of 32 bits give, its rounding included."""
    s, kind = prepare(case, seed), case["kind"]

    def to32(v):
        return v.to(torch.float32).double()

    def codes(x):
        x = x.double()
        top = x.abs().max(dim=1).values[:, None]
        inverse = to32(127.0 / top)
        q = torch.round(to32(x * inverse))
        return torch.where(top == 0, 0.0, q), to32(top / 127.0)

    if kind == "sort":
        flat = s.idx.flatten().long()
        hot = flat[:, None] == torch.arange(s.held, device="cuda")[None, :]
        total = hot.sum(0)
        begin = torch.zeros(s.held + 1, dtype=torch.int64, device="cuda")
        begin[1:] = total.cumsum(0)
        before = hot.to(torch.int32).cumsum(0)                     # pairs of the expert up to this one
        kept = flat < s.held
        e = flat.clamp(max=s.held - 1)
        position = torch.where(kept, begin[e] + before[torch.arange(flat.numel(), device="cuda"), e] - 1, -1)
        del hot, before
        source = torch.full_like(flat, -1)
        rows = torch.zeros((flat.numel(), case["d"]), dtype=torch.float64, device="cuda")
        pair = torch.arange(flat.numel(), device="cuda")[kept]
        source[position[kept]] = pair
        if case["out"] == "int8":
            q, scale = codes(s.x)
            values = to32(q * scale)
        else:
            values = s.x.double()
        rows[position[kept]] = values[pair // case["top_k"]]
        return {"position": position.to(torch.int32).view_as(s.idx), "source": source.to(torch.int32),
                "begin": begin.to(torch.int32), "rows": rows}
    if kind in ("merge", "grad"):
        kept = s.position >= 0
        w = torch.ones(s.position.shape, dtype=torch.float64, device="cuda") if s.w is None else s.w.double()
        token, slot = kept.nonzero(as_tuple=True)
        at = s.position[token, slot].long()
        if kind == "merge":
            y = torch.zeros((case["tokens"], case["d"]), dtype=torch.float64, device="cuda")
            if s.base is not None:
                y += s.base.double()
            y.index_add_(0, token, s.rows[at].double() * w[token, slot][:, None])
            return {"y": y}
        drows = torch.zeros(s.rows.shape, dtype=torch.float64, device="cuda")
        drows[at] = s.dy[token].double() * w[token, slot][:, None]
        dw = torch.zeros(s.position.shape, dtype=torch.float64, device="cuda")
        dw[token, slot] = torch.einsum("pd,pd->p", s.rows[at].double(), s.dy[token].double())
        return {"drows": drows, "dw": dw}
    k = case["k"]
    q, scale = (s.a[:, :k].double(), s.a_scales.double()[:, None]) if s.a_scales is not None else codes(s.a)
    ends = [0, s.count] if s.begin is None else s.begin.tolist()
    y = torch.empty((s.count, s.b.shape[1]), dtype=torch.float64, device="cuda")
    for e, (first, last) in enumerate(zip(ends[:-1], ends[1:])):
        if last > first:
            y[first:last] = q[first:last] @ s.b[e, :, :k].double().T * scale[first:last] * s.b_scales[e].double()
    if case["gated"]:
        gate, up = y[:, :case["n"]], y[:, case["n"]:]
        y = gate * torch.sigmoid(gate) * up
    return {"out": y}
