"""The dense products beside the packed experts, as a serving program calls them, for timing.

Four operators:

  grouped   ``grouped_linear``: rows grouped by expert times the matrix of their expert, y[i] = x[row(i)] . W[e(i)]^T, groups of any
            size; with ``gather`` the rows are picked out of the token matrix, without it they lie in expert order already
  experts   ``dense_experts``: un-quantised SwiGLU experts of a MoE block for a given top-k selection,
            y[t] = residual[t] + sum_s w[t, s] * Wd[e] . (silu(Wg[e] . x[t]) * (Wu[e] . x[t])),  e = expert of slot s; with
            ``routed`` only the first ``experts`` entries of an id map over ``routed`` ids are held here ("super" experts)
  linear4   ``linear4``: y = x . (scale * (code - 8))^T with 4-bit codes and one fp16 scale for every ``group`` columns of a row
  mlp4      ``dense_mlp4``: a SwiGLU MLP (shared expert) whose three matrices are held in that form, with a per-token sigmoid gate
            where ``gated``, added to a residual

A case is a plain dict; ``prepare`` makes what a program holds before the call, ``run`` is one pass, ``work`` the traffic and
arithmetic no implementation can avoid, ``exact`` the result from the definition in 64 bits.  Shapes are those of the three layer
configurations of this package (2048 hidden; 128 experts of 768, 512 of 512, 64 of 1408 with a shared expert of 2816; 32 query
heads of 128) or generic ones.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # gate and up projections of 64 experts for five sequences being decoded: 30 rows, most experts have none or one
        {"name": "grouped_up_5", "op": "grouped", "experts": 64, "tokens": 5, "top": 6, "k": 2048, "n": 2816, "gather": True,
         "dtype": "fp16", "skew": 0.0},
        # down projection of one chunk of a chunked prefill, rows in expert order, uneven load
        {"name": "grouped_down_777", "op": "grouped", "experts": 128, "tokens": 777, "top": 8, "k": 768, "n": 2048, "gather": False,
         "dtype": "bf16", "skew": 0.8},
        # gate and up projections of a long prefill, Zipf(1.1) load: the largest case
        {"name": "grouped_up_8192", "op": "grouped", "experts": 128, "tokens": 8192, "top": 8, "k": 2048, "n": 1536, "gather": True,
         "dtype": "bf16", "skew": 1.1},
        # a layer whose experts are not quantised, one sequence being decoded
        {"name": "experts_qwen3_1", "op": "experts", "experts": 128, "routed": 128, "tokens": 1, "top": 8, "hidden": 2048, "inter": 768,
         "dtype": "bf16", "skew": 0.0},
        # three un-quantised experts of a layer whose other 509 are packed, decode batch
        {"name": "experts_super_24", "op": "experts", "experts": 3, "routed": 512, "tokens": 24, "top": 10, "hidden": 2048, "inter": 512,
         "dtype": "bf16", "skew": 0.0},
        # the decode batch of the headline number on un-quantised experts
        {"name": "experts_qwen3_64", "op": "experts", "experts": 128, "routed": 128, "tokens": 64, "top": 8, "hidden": 2048, "inter": 768,
         "dtype": "bf16", "skew": 0.0},
        # one evaluation sequence of 2048 fp16 tokens, as the perplexity runs feed it
        {"name": "experts_deepseek_2048", "op": "experts", "experts": 64, "routed": 64, "tokens": 2048, "top": 6, "hidden": 2048,
         "inter": 1408, "dtype": "fp16", "skew": 0.5},
        # query projection of one sequence being decoded: a matrix of 4 MB, launches and host work are what counts
        {"name": "linear4_query_1", "op": "linear4", "tokens": 1, "k": 2048, "n": 4096, "group": 128, "dtype": "bf16"},
        # output projection of a decode batch of 16
        {"name": "linear4_output_16", "op": "linear4", "tokens": 16, "k": 4096, "n": 2048, "group": 64, "dtype": "fp16"},
        # output layer over a vocabulary of odd size, four sequences
        {"name": "linear4_head_4", "op": "linear4", "tokens": 4, "k": 2048, "n": 100003, "group": 128, "dtype": "bf16"},
        # two shared experts of 1408 for five sequences
        {"name": "mlp4_deepseek_5", "op": "mlp4", "tokens": 5, "hidden": 2048, "inter": 2816, "group": 128, "gated": False,
         "dtype": "fp16"},
        # gated shared expert on a chunk of prefill with decode tokens mixed in
        {"name": "mlp4_next_300", "op": "mlp4", "tokens": 300, "hidden": 2048, "inter": 512, "group": 128, "gated": True,
         "dtype": "bf16"},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["grouped", "experts", "experts", "linear4", "linear4", "mlp4"])
    c = {"op": op, "dtype": rng.choice(["bf16", "fp16"])}
    if op == "grouped":
        experts = _log_uniform(rng, 2, 128)
        c.update(experts=experts, tokens=_log_uniform(rng, 1, 8192), top=rng.randint(1, min(8, experts)), k=8 * _log_uniform(rng, 32, 256),
                 n=_log_uniform(rng, 200, 1536), gather=rng.choice([True, False]), skew=round(rng.uniform(0.0, 1.1), 2))
    elif op == "experts":
        routed = _log_uniform(rng, 4, 512)
        experts = rng.choice([routed if routed <= 128 else rng.randint(32, 128), rng.randint(1, min(4, routed))])
        c.update(experts=experts, routed=routed, tokens=_log_uniform(rng, 1, 2048), top=rng.randint(1, min(8, routed)),
                 hidden=8 * _log_uniform(rng, 64, 256), inter=8 * _log_uniform(rng, 16, 128), skew=round(rng.uniform(0.0, 1.1), 2))
    elif op == "linear4":
        c.update(tokens=_log_uniform(rng, 1, 1024), k=_log_uniform(rng, 256, 8192), n=_log_uniform(rng, 256, 16384),
                 group=rng.choice([32, 64, 128]))
    else:
        c.update(tokens=_log_uniform(rng, 1, 2048), hidden=8 * _log_uniform(rng, 64, 512), inter=_log_uniform(rng, 128, 4096),
                 group=rng.choice([32, 64, 128]), gated=rng.choice([True, False]))
    return c


# ---- inputs
def _random(gen, *shape, std=1.0, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device=gen.device).normal_(0.0, std, generator=gen)


def _selection(case, routed, gen):
    """Top-k experts of every token and their weights, fp32 renormalised: Gumbel top-k of a Zipf(skew) law over the experts.  Experts
    that stay un-quantised beside packed ones are those that tokens prefer: their logits are raised."""
    law = -case["skew"] * torch.log(torch.arange(1, routed + 1, dtype=torch.float32, device=gen.device))
    law = law[torch.randperm(routed, generator=gen, device=gen.device)]
    if case.get("experts", routed) < routed:
        law[: case["experts"]] += 1.5
    u = torch.rand(case["tokens"], routed, generator=gen, device=gen.device).clamp_(1e-6, 1.0 - 1e-6)
    logits, idx = torch.topk(law - torch.log(-torch.log(u)), case["top"], dim=-1)
    return idx.to(torch.int32), torch.softmax(logits, dim=-1)


def _grouped_rows(idx, experts):
    """Assignments in expert order: the token of each, and the offset where each expert's begin."""
    order = torch.argsort(idx.reshape(-1).long(), stable=True)
    counts = torch.bincount(idx.reshape(-1).long(), minlength=experts)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=idx.device)
    offsets[1:] = torch.cumsum(counts, 0)
    return (order // idx.shape[1]).to(torch.int32), offsets


def _matrix4(gen, n, k, group):
    """A matrix N(0, 0.02) rounded to the nearest of 16 steps of its group's scale: codes 0 .. 15 standing for -8 .. 7, eight to a
    32-bit word (column 8 j + i in bits 4 i of word j), rows padded to whole 16 bytes with code 8."""
    width, groups = -(-k // 32) * 32, -(-k // group)
    payload = torch.empty(n, width // 8, dtype=torch.int32, device=gen.device)
    scale = torch.empty(n, groups, dtype=torch.float16, device=gen.device)
    shifts = 4 * torch.arange(8, dtype=torch.int64, device=gen.device)
    for r in range(0, n, 16384):
        rows = min(16384, n - r)
        w = torch.zeros(rows, max(width, groups * group), device=gen.device)
        w[:, :k] = _random(gen, rows, k, std=0.02)
        parts = w[:, : groups * group].reshape(rows, groups, group)
        s = (parts.abs().amax(dim=2) / 7.5).clamp_(min=1e-4).half()
        scale[r:r + rows] = s
        codes = torch.zeros_like(w)
        codes[:, : groups * group] = torch.clamp(torch.round(parts / s.float()[:, :, None]), -8, 7).reshape(rows, -1)
        words = ((codes[:, :width].to(torch.int64) + 8).reshape(rows, width // 8, 8) << shifts).sum(dim=2)
        payload[r:r + rows] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    return payload.view(torch.uint32), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, st = DTYPES[case["dtype"]], {"case": case}
    if case["op"] == "grouped":
        idx, _ = _selection(case, case["experts"], gen)
        tok, st["offsets"] = _grouped_rows(idx, case["experts"])
        st["tok"] = tok if case["gather"] else None
        st["x"] = _random(gen, case["tokens"] if case["gather"] else tok.numel(), case["k"], dtype=dtype)
        st["w"] = _random(gen, case["experts"], case["n"], case["k"], std=0.02, dtype=dtype)
    elif case["op"] == "experts":
        st["idx"], st["weight"] = _selection(case, case["routed"], gen)
        st["map"] = None
        if case["experts"] < case["routed"]:
            st["map"] = torch.full((case["routed"],), -1, dtype=torch.int32, device=DEVICE)
            st["map"][: case["experts"]] = torch.arange(case["experts"], dtype=torch.int32, device=DEVICE)
        st["x"] = _random(gen, case["tokens"], case["hidden"], dtype=dtype)
        st["gate_up"] = _random(gen, case["experts"], 2 * case["inter"], case["hidden"], std=0.02, dtype=dtype)
        st["down"] = _random(gen, case["experts"], case["hidden"], case["inter"], std=0.02, dtype=dtype)
        st["residual"] = _random(gen, case["tokens"], case["hidden"], std=0.1, dtype=dtype)
    elif case["op"] == "linear4":
        st["x"] = _random(gen, case["tokens"], case["k"], dtype=dtype)
        st["w"] = _matrix4(gen, case["n"], case["k"], case["group"])
    else:
        st["x"] = _random(gen, case["tokens"], case["hidden"], dtype=dtype)
        st["gate"] = _matrix4(gen, case["inter"], case["hidden"], case["group"])
        st["up"] = _matrix4(gen, case["inter"], case["hidden"], case["group"])
        st["down"] = _matrix4(gen, case["hidden"], case["inter"], case["group"])
        st["token_gate"] = _random(gen, case["hidden"], std=0.02, dtype=torch.float16) if case["gated"] else None
        st["residual"] = _random(gen, case["tokens"], case["hidden"], std=0.1, dtype=dtype)
    return st


# ---- one pass
def _codes4(payload, k):
    """Codes of a packed matrix as fp32 numbers -8 .. 7, [n, k]."""
    shifts = 4 * torch.arange(8, dtype=torch.int32, device=payload.device)
    codes = (payload.view(torch.int32)[:, :, None] >> shifts) & 15
    return codes.reshape(payload.shape[0], -1)[:, :k].float() - 8.0


def _linear4_plain(x, w, group):
    payload, scale = w
    k = x.shape[1]
    return x @ (_codes4(payload, k) * scale.float().repeat_interleave(group, dim=1)[:, :k]).T


def _silu(v):
    return v / (1.0 + torch.exp(-v))


def _by_group(x, offsets, product, width):
    """product(expert, rows) for every expert that has rows; one copy of the offsets to the host."""
    y = torch.empty(x.shape[0], width, dtype=torch.float32, device=x.device)
    ends = offsets.tolist()
    for e in range(len(ends) - 1):
        if ends[e + 1] > ends[e]:
            y[ends[e]:ends[e + 1]] = product(e, x[ends[e]:ends[e + 1]])
    return y


def _grouped_plain(st):
    rows = st["x"] if st["tok"] is None else st["x"][st["tok"].long()]
    return _by_group(rows.float(), st["offsets"], lambda e, r: r @ st["w"][e].float().T, st["w"].shape[1]).to(st["x"].dtype)


def _experts_plain(st):
    inter, held = st["down"].shape[2], st["down"].shape[0]
    local = st["idx"].long() if st["map"] is None else st["map"].long()[st["idx"].long()]
    local = torch.where(local < 0, held, local).reshape(-1)          # what is not held here comes last
    order = torch.argsort(local, stable=True)
    offsets = torch.zeros(held + 1, dtype=torch.int64, device=local.device)
    offsets[1:] = torch.cumsum(torch.bincount(local, minlength=held + 1)[:held], 0)
    tok = order // st["idx"].shape[1]

    def mlp(e, r):
        h = r @ st["gate_up"][e].float().T
        return (_silu(h[:, :inter]) * h[:, inter:]) @ st["down"][e].float().T

    d = _by_group(st["x"].float()[tok], offsets, mlp, st["x"].shape[1]) * st["weight"].reshape(-1)[order, None]
    d = torch.where((local[order] < held)[:, None], d, torch.zeros_like(d))
    y = torch.empty_like(d)
    y[order] = d
    return (st["residual"].float() + y.reshape(*st["idx"].shape, -1).sum(dim=1)).to(st["x"].dtype)


def _mlp4_plain(st, group):
    x = st["x"].float()
    z = _silu(_linear4_plain(x, st["gate"], group)) * _linear4_plain(x, st["up"], group)
    y = _linear4_plain(z, st["down"], group)
    if st["token_gate"] is not None:
        y = y / (1.0 + torch.exp(-(x @ st["token_gate"].float())))[:, None]
    return (st["residual"].float() + y).to(st["x"].dtype)


def run(st):
    op = st["case"]["op"]
    if own:
        from bitsmoe_b200 import layer
        if op == "grouped":
            return layer.grouped_linear(st["x"], st["w"], st["offsets"], token_indices=st["tok"])
        if op == "experts":
            return layer.dense_experts(st["x"], st["idx"], st["weight"], st["gate_up"], st["down"], global_to_local=st["map"],
                                       residual=st["residual"])
        if op == "linear4":
            return layer.linear4(st["x"], *st["w"], group_size=st["case"]["group"])
        return layer.dense_mlp4(st["x"], st["gate"], st["up"], st["down"], group_size=st["case"]["group"],
                                token_gate_weight=st["token_gate"], residual=st["residual"])
    if op == "grouped":
        return _grouped_plain(st)
    if op == "experts":
        return _experts_plain(st)
    if op == "linear4":
        return _linear4_plain(st["x"].float(), st["w"], st["case"]["group"]).to(st["x"].dtype)
    return _mlp4_plain(st, st["case"]["group"])


# ---- what no implementation can avoid
def _held_load(case, routed, held):
    """(assignments to the experts held here, how many of them have any), for one selection of this case's law."""
    idx, _ = _selection(case, routed, torch.Generator(device="cpu").manual_seed(0))
    load = torch.bincount(idx.reshape(-1).long(), minlength=routed)[:held]
    return int(load.sum()), int((load > 0).sum())


def _matrix4_bytes(n, k, group):
    return n * (k / 2 + 2 * -(-k // group))


def work(case):
    t = case["tokens"]
    if case["op"] == "grouped":
        rows, active = _held_load(case, case["experts"], case["experts"])
        read = (t if case["gather"] else rows) * case["k"] * 2 + active * case["n"] * case["k"] * 2
        index = 4 * (case["experts"] + 1) + (4 * rows if case["gather"] else 0)
        return {"bytes": read + index + rows * case["n"] * 2, "flops": 2 * rows * case["n"] * case["k"]}
    if case["op"] == "experts":
        rows, active = _held_load(case, case["routed"], case["experts"])
        weights = active * 3 * case["hidden"] * case["inter"] * 2
        return {"bytes": weights + 3 * t * case["hidden"] * 2 + t * case["top"] * 8, "flops": 6 * rows * case["hidden"] * case["inter"]}
    if case["op"] == "linear4":
        k, n = case["k"], case["n"]
        return {"bytes": _matrix4_bytes(n, k, case["group"]) + 2 * t * (k + n), "flops": 2 * t * k * n}
    h, i, g = case["hidden"], case["inter"], case["group"]
    return {"bytes": 2 * _matrix4_bytes(i, h, g) + _matrix4_bytes(h, i, g) + 3 * t * h * 2 + (2 * h if case["gated"] else 0),
            "flops": 6 * t * h * i + (2 * t * h if case["gated"] else 0)}


# ---- from the definition, in 64 bits
def _dense64(w, k, group):
    """Every column of a packed matrix on its own: nibble c % 8 of word c // 8, times the scale of group c // group."""
    payload, scale = w
    words, out = payload.view(torch.int32).to(torch.int64) & 0xFFFFFFFF, []
    for i in range(8):
        out.append(torch.div(words, 16 ** i, rounding_mode="floor") % 16 - 8)
    codes = torch.stack(out, dim=2).flatten(1)[:, :k].double()
    return codes * scale.double()[:, torch.arange(k, device=codes.device) // group]


def _swiglu64(x, gate, up, down):
    g, u = torch.einsum("tk,nk->tn", x, gate), torch.einsum("tk,nk->tn", x, up)
    return torch.einsum("tn,hn->th", g * torch.sigmoid(g) * u, down)


def exact(case, seed):
    st = prepare(case, seed)
    x = st["x"].double()
    if case["op"] == "grouped":
        at = st["offsets"].cpu().numpy()
        y = torch.zeros(int(at[-1]), case["n"], dtype=torch.float64, device=x.device)
        for e in range(case["experts"]):
            rows = torch.arange(int(at[e]), int(at[e + 1]), device=x.device)
            if rows.numel():
                y[rows] = torch.einsum("tk,nk->tn", x[rows if st["tok"] is None else st["tok"].long()[rows]], st["w"][e].double())
        return y
    if case["op"] == "experts":
        y, i = st["residual"].double(), case["inter"]
        for e in range(case["experts"]):          # the ids held here are the first ones
            tokens, slots = torch.nonzero(st["idx"] == e, as_tuple=True)
            if tokens.numel():
                d = _swiglu64(x[tokens], st["gate_up"][e, :i].double(), st["gate_up"][e, i:].double(), st["down"][e].double())
                y.index_add_(0, tokens, d * st["weight"].double()[tokens, slots, None])
        return y
    if case["op"] == "linear4":
        if case["n"] * case["k"] > 2 ** 26:         # in pieces of the rows
            (p, s), n = st["w"], case["n"]
            return torch.cat([torch.einsum("tk,nk->tn", x, _dense64((p[r:r + 8192], s[r:r + 8192]), case["k"], case["group"]))
                              for r in range(0, n, 8192)], dim=1)
        return torch.einsum("tk,nk->tn", x, _dense64(st["w"], case["k"], case["group"]))
    h, i, g = case["hidden"], case["inter"], case["group"]
    y = _swiglu64(x, _dense64(st["gate"], h, g), _dense64(st["up"], h, g), _dense64(st["down"], i, g))
    if case["gated"]:
        y = y * torch.sigmoid((x * st["token_gate"].double()).sum(dim=1, keepdim=True))
    return st["residual"].double() + y
