"""The feed-forward operators of a decoder layer around the int4 weights, and what they are measured on: a dense linear
layer with bias, activation and residual in its epilogue, and the parts of a layer of experts (router, products
grouped by expert, weighted combination).

A case is a dict of plain values. `kind` says which operator it takes:

  linear   y = bf16(act(x W^T + bias) + residual) for M tokens, W int4 with groups of 128
  experts  y[p] = bf16(act(x[row of p] W_e^T + bias_e)) for the slots p of every expert e: ragged sizes, empty experts
  route    router logits -> the top_k experts of every token, their weights, and the slots sorted by expert
  combine  y[t] = bf16(residual[t] + sum over t's picks of weight * expert output)

W is what the library dequantises to: bf16((q - zero point) * scale). Layers are out_f x in_f ("rows", "cols"); with the
activation "swiglu" the checkpoint's rows are [gate | up] and y has rows / 2 columns. Dense sizes are the model's own
(hidden 5120, MLP 17408, 16384 rows of attention projections); the experts' are generic ones on the same hidden size.
"""
import importlib
import math

import torch

own = False

GROUP = 128
HIDDEN, INTER = 5120, 17408
ACTS = ["none", "silu", "gelu", "gelu_tanh", "swiglu"]


def listed():
    return [
        # Attention output projection of one decode token, into the residual stream: the smallest layer, launch included.
        {"name": "linear M=1 5120x6144", "kind": "linear", "rows": HIDDEN, "cols": 6144, "M": 1, "act": "none", "bias": True, "residual": True},
        # gate|up of a speculative-verify block of 8 drafted tokens and one more.
        {"name": "linear M=9 swiglu", "kind": "linear", "rows": 2 * INTER, "cols": HIDDEN, "M": 9, "act": "swiglu", "bias": False, "residual": False},
        # A short chat turn behind a cached prefix through a widening layer with an activation.
        {"name": "linear M=77 gelu", "kind": "linear", "rows": 16384, "cols": HIDDEN, "M": 77, "act": "gelu_tanh", "bias": True, "residual": False},
        # The down projection of a 4096-token prompt chunk into the residual stream.
        {"name": "linear M=4096 residual", "kind": "linear", "rows": HIDDEN, "cols": INTER, "M": 4096, "act": "none", "bias": False, "residual": True},
        # Decode of one sequence: 8 of 64 experts with one token each, gate|up.
        {"name": "experts T=1 gate|up", "kind": "experts", "E": 64, "top_k": 8, "tokens": 1, "rows": 2048, "cols": HIDDEN, "act": "swiglu", "bias": False, "gather": True},
        # Decode of a batch of 33 sequences: nearly every expert has a few tokens; the down projection, inputs in slot order.
        {"name": "experts T=33 down", "kind": "experts", "E": 64, "top_k": 8, "tokens": 33, "rows": HIDDEN, "cols": 1024, "act": "none", "bias": True, "gather": False},
        # A prompt of 300 tokens: some 37 tokens per expert, ragged.
        {"name": "experts T=300 gate|up", "kind": "experts", "E": 64, "top_k": 8, "tokens": 300, "rows": 2048, "cols": HIDDEN, "act": "swiglu", "bias": False, "gather": True},
        # A 4096-token prompt chunk.
        {"name": "experts T=4096 gate|up", "kind": "experts", "E": 64, "top_k": 8, "tokens": 4096, "rows": 2048, "cols": HIDDEN, "act": "swiglu", "bias": False, "gather": True},
        # Router of one decode token.
        {"name": "route T=1", "kind": "route", "E": 64, "top_k": 8, "tokens": 1, "type": "bf16", "renormalize": True, "padded": 0.0},
        # Router of a prompt chunk over many experts, a tenth of the rows padding.
        {"name": "route T=4096", "kind": "route", "E": 256, "top_k": 8, "tokens": 4096, "type": "fp32", "renormalize": True, "padded": 0.1},
        # One decode token's expert outputs back into the residual stream.
        {"name": "combine T=1", "kind": "combine", "top_k": 8, "tokens": 1, "hidden": HIDDEN, "residual": True, "padded": 0.0},
        # The same for a prompt chunk with a tenth of its rows padding.
        {"name": "combine T=4096", "kind": "combine", "top_k": 8, "tokens": 4096, "hidden": HIDDEN, "residual": True, "padded": 0.1},
    ]


def _log_uniform(rng, lo, hi, step):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    kind = rng.choice(["linear", "linear", "experts", "experts", "route", "combine"])
    tokens = _log_uniform(rng, 1, 4096, 1)
    if kind == "linear":
        rows, cols = _log_uniform(rng, 1024, 2 * INTER, 32), _log_uniform(rng, 1024, INTER, GROUP)
        limit = HIDDEN * INTER * 4096 // (rows * cols)  # no dearer than the largest listed one
        return {"kind": kind, "rows": rows, "cols": cols, "M": max(1, min(tokens, limit)), "act": rng.choice(ACTS),
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    if kind == "route":
        E = _log_uniform(rng, 8, 256, 1)
        return {"kind": kind, "E": E, "top_k": rng.randint(1, min(8, E)), "tokens": tokens, "type": rng.choice(["bf16", "fp32"]),
                "renormalize": rng.random() < 0.5, "padded": rng.choice([0.0, 0.1, 0.3])}
    top_k = rng.randint(1, 8)
    if kind == "combine":
        return {"kind": kind, "top_k": top_k, "tokens": tokens, "hidden": _log_uniform(rng, 1024, HIDDEN, 16),
                "residual": rng.random() < 0.5, "padded": rng.choice([0.0, 0.1])}
    E = _log_uniform(rng, 8, 64, 1)
    act = rng.choice(["swiglu", "none", "silu"])
    rows, cols = _log_uniform(rng, 512, 2048, 32), _log_uniform(rng, 512, HIDDEN, GROUP)
    if act == "none" and rng.random() < 0.7:  # a down projection: few columns, many rows
        rows, cols = _log_uniform(rng, 512, HIDDEN, 32), _log_uniform(rng, 512, 2048, GROUP)
    return {"kind": kind, "E": E, "top_k": top_k, "tokens": tokens, "rows": rows, "cols": cols, "act": act,
            "bias": rng.random() < 0.3, "gather": act != "none"}


# ------------------------------------------------------------------ what a user's program has in hand
class State:
    """Inputs of one case, buffers for its outputs and, for the library's calls, the weights in its containers."""

    def __init__(self, case):
        self.case = case
        self.w = None

    def __del__(self):
        if self.w is not None and torch is not None and torch.cuda is not None:
            torch.cuda.synchronize()
            pkg = _pkg()
            (pkg.experts_free if self.case["kind"] == "experts" else pkg.awq_free)(self.w)


def _pkg():
    return importlib.import_module("qwen38-3090-cuda-server_b200")


def _disk_tensors(gen, rows, cols, batch=()):
    """Seeded tensors in the checkpoint's layout: codes packed eight to a word along the columns, bf16 scales, zero
    points packed eight to a word along the rows."""
    lo, hi = -2 ** 31, 2 ** 31 - 1
    packed = torch.randint(lo, hi, (*batch, rows, cols // 8), dtype=torch.int32, device="cuda", generator=gen)
    scale = (torch.randn((*batch, rows, cols // GROUP), device="cuda", generator=gen).abs() * 0.02 + 1e-4).to(torch.bfloat16)
    zp = torch.randint(lo, hi, (*batch, rows // 8, cols // GROUP), dtype=torch.int32, device="cuda", generator=gen)
    return packed, scale, zp


def _activations(gen, tokens, cols):
    x = torch.randn((tokens, cols), device="cuda", generator=gen)
    x[:, torch.randint(0, cols, (max(1, cols // 512),), device="cuda", generator=gen)] *= 16.0
    return x.to(torch.bfloat16)


def _columns(case):
    return case["rows"] // 2 if case["act"] == "swiglu" else case["rows"]


def _inputs(case, seed):
    """The case's inputs, as tensors on the GPU (the slots' bounds on the host as well, for loops over experts)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = State(case)
    kind = case["kind"]
    if kind == "linear":
        s.disk = _disk_tensors(gen, case["rows"], case["cols"])
        s.x = _activations(gen, case["M"], case["cols"])
        # (outputs have a deviation of about sqrt(cols) * 0.15: bias and residual of that size matter)
        size = 0.15 * math.sqrt(case["cols"])
        s.bias = (torch.randn(case["rows"], device="cuda", generator=gen) * size).to(torch.bfloat16) if case["bias"] else None
        s.residual = (torch.randn((case["M"], _columns(case)), device="cuda", generator=gen) * size).to(torch.bfloat16) if case["residual"] else None
        s.y = torch.zeros((case["M"], _columns(case)), dtype=torch.bfloat16, device="cuda")
    elif kind == "experts":
        E, k, T = case["E"], case["top_k"], case["tokens"]
        s.disk = _disk_tensors(gen, case["rows"], case["cols"], (E,))
        score = torch.randn((T, E), device="cuda", generator=gen) + 0.5 * torch.randn(E, device="cuda", generator=gen)  # some experts are liked more
        picks = score.topk(k, dim=1).indices.flatten()
        order = torch.argsort(picks, stable=True)
        counts = torch.bincount(picks, minlength=E)
        s.offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s.bounds = s.offsets.tolist()
        s.x_rows = (order // k).to(torch.int32) if case["gather"] else None
        s.x = _activations(gen, T if case["gather"] else T * k, case["cols"])
        size = 0.15 * math.sqrt(case["cols"])
        s.bias = (torch.randn((E, case["rows"]), device="cuda", generator=gen) * size).to(torch.bfloat16) if case["bias"] else None
        s.y = torch.zeros((T * k, _columns(case)), dtype=torch.bfloat16, device="cuda")
    elif kind == "route":
        s.logits = torch.randn((case["tokens"], case["E"]), device="cuda", generator=gen) * 2
        s.logits += torch.randn(case["E"], device="cuda", generator=gen)
        # padding: every logit of the row is -inf, the row picks no expert
        s.logits[torch.rand(case["tokens"], device="cuda", generator=gen) < case["padded"]] = -math.inf
        s.logits = s.logits.to(torch.bfloat16 if case["type"] == "bf16" else torch.float32)
    else:
        T, k, H = case["tokens"], case["top_k"], case["hidden"]
        kept = torch.rand(T, device="cuda", generator=gen) >= case["padded"]
        s.weights = torch.rand((T, k), device="cuda", generator=gen).softmax(1) * kept[:, None]
        # every pick of a kept token has a slot of its own, in the order of a random expert assignment
        n = int(kept.sum()) * k
        s.slots = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
        s.slots[kept] = torch.randperm(n, device="cuda", generator=gen, dtype=torch.int32).view(-1, k)
        s.parts = torch.randn((T * k, H), device="cuda", generator=gen).to(torch.bfloat16)
        s.parts[n:] = math.nan  # rows behind the last slot hold anything
        s.residual = _activations(gen, T, H) if case["residual"] else None
        s.y = torch.zeros((T, H), dtype=torch.bfloat16, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        # at load time: weights into the library's containers, buffers of the router
        pkg = _pkg()
        if case["kind"] == "linear":
            s.w = pkg.awq_alloc_fused(case["rows"], case["cols"])
            _repack(pkg, s.w, case, *s.disk)
        elif case["kind"] == "experts":
            s.w = pkg.experts_alloc(case["E"], case["rows"], case["cols"])
            for e in range(case["E"]):
                _repack(pkg, pkg.experts_view(s.w, e), case, *(t[e] for t in s.disk))
        elif case["kind"] == "route":
            s.route = pkg.route_alloc(case["tokens"], case["E"], case["top_k"])
        torch.cuda.synchronize()
    return s


def _repack(pkg, w, case, packed, scale, zp):
    if case["act"] == "swiglu":
        pkg.awq_repack_into_swiglu(w, 0, packed, scale, zp, case["rows"] // 2)
    else:
        pkg.awq_repack_into(w, 0, packed, scale, zp)


# ------------------------------------------------------------------ one pass
def run(s):
    return (_run_own if own else globals()["_plain_" + s.case["kind"]])(s)


def _run_own(s):
    pkg, case = _pkg(), s.case
    if case["kind"] == "linear":
        pkg.linear_epilogue(s.y, s.w, s.x, case["M"], bias=s.bias, activation=_code(pkg, case), residual=s.residual)
        return s.y
    if case["kind"] == "experts":
        pkg.experts_linear(s.y, s.w, s.x, s.offsets, x_rows=s.x_rows, bias=s.bias, activation=_code(pkg, case))
        return s.y
    if case["kind"] == "route":
        r = s.route
        pkg.route(r, s.logits, renormalize=case["renormalize"])
        return r.ids, r.weights, r.offsets, r.slots, r.rows
    pkg.experts_combine(s.y, s.parts, s.slots, s.weights, residual=s.residual)
    return s.y


def _code(pkg, case):
    return {"none": pkg.ACT_NONE, "silu": pkg.ACT_SILU, "gelu": pkg.ACT_GELU, "gelu_tanh": pkg.ACT_GELU_TANH,
            "swiglu": pkg.ACT_SWIGLU}[case["act"]]


def _dequantise(packed, scale, zp):
    """The weights as the library defines them, bf16((q - zp) * s), in fp32."""
    at = torch.arange(0, 32, 4, dtype=torch.int32, device=packed.device)
    q = (packed.unsqueeze(-1) >> at & 15).flatten(-2)
    z = (zp.unsqueeze(-2) >> at[:, None] & 15).flatten(-3, -2)
    rows, cols = q.shape
    w = (q.view(rows, -1, GROUP) - z.unsqueeze(-1)).float() * scale.float().unsqueeze(-1)
    return w.view(rows, cols).to(torch.bfloat16).float()


def _activate(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "swiglu":
        gate, up = v.chunk(2, dim=-1)
        return gate / (1 + torch.exp(-gate)) * up
    return v


def _plain_linear(s):
    v = s.x.float() @ _dequantise(*s.disk).t()
    if s.bias is not None:
        v = v + s.bias.float()
    v = _activate(v, s.case["act"])
    if s.residual is not None:
        v = v + s.residual.float()
    return v.to(torch.bfloat16)


def _plain_experts(s):
    y = torch.zeros_like(s.y)
    x = s.x if s.x_rows is None else s.x[s.x_rows.long()]
    for e, (lo, hi) in enumerate(zip(s.bounds, s.bounds[1:])):
        if lo < hi:
            v = x[lo:hi].float() @ _dequantise(*(t[e] for t in s.disk)).t()
            if s.bias is not None:
                v = v + s.bias[e].float()
            y[lo:hi] = _activate(v, s.case["act"]).to(torch.bfloat16)
    return y


def _plain_route(s):
    k, E = s.case["top_k"], s.case["E"]
    logits = s.logits.float()
    values, ids = torch.sort(logits, dim=1, descending=True, stable=True)  # (ties: the lowest index first)
    top = values[:, :1].nan_to_num(neginf=0.0)
    picked = torch.exp(values[:, :k] - top)
    total = (picked if s.case["renormalize"] else torch.exp(logits - top)).sum(1, keepdim=True)
    real = values[:, :k] > -math.inf
    weights = torch.where(real, picked / total, 0.0)
    ids = torch.where(real, ids[:, :k], -1).to(torch.int32)
    # slots: the picks sorted by expert, within an expert by token; empty picks have none
    flat = torch.where(real, ids, E).flatten()
    order = torch.argsort(flat, stable=True)
    counts = (flat[:, None] == torch.arange(E, device=flat.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    slots = torch.where(real.flatten(), place, -1).to(torch.int32).view(ids.shape)
    rows = torch.where(torch.arange(order.numel(), device=order.device) < offsets[-1], order // k, 0).to(torch.int32)
    return ids, weights, offsets, slots, rows


def _plain_combine(s):
    has = s.slots >= 0
    parts = torch.where(has.unsqueeze(-1), s.parts[s.slots.clamp(min=0).long()].float(), 0.0)
    v = (s.weights.unsqueeze(-1) * parts).sum(1)
    if s.residual is not None:
        v = v + s.residual.float()
    return v.to(torch.bfloat16)


# ------------------------------------------------------------------ what a pass cannot do without
def _weight_bytes(rows, cols):
    """Codes, bf16 scales and four-bit zero points."""
    return rows * cols // 2 + (2 * rows + rows // 2) * (cols // GROUP)


def work(case):
    kind = case["kind"]
    if kind == "linear":
        rows, cols, M = case["rows"], case["cols"], case["M"]
        nbytes = _weight_bytes(rows, cols) + 2 * M * cols + 2 * M * _columns(case) * (2 if case["residual"] else 1) + (2 * rows if case["bias"] else 0)
        return {"bytes": float(nbytes), "flops": 2.0 * M * rows * cols}
    if kind == "experts":
        rows, cols, slots, E = case["rows"], case["cols"], case["tokens"] * case["top_k"], case["E"]
        # experts that at least one token picks (expected, for even odds); an expert that nobody picks is not read
        used = E * (1 - (1 - min(1.0, case["top_k"] / E)) ** case["tokens"])
        nbytes = used * (_weight_bytes(rows, cols) + (2 * rows if case["bias"] else 0)) + 2 * slots * _columns(case) + 4 * (E + 1)
        nbytes += 2 * case["tokens"] * cols + 4 * slots if case["gather"] else 2 * slots * cols
        return {"bytes": float(nbytes), "flops": 2.0 * slots * rows * cols}
    T, k = case["tokens"], case["top_k"]
    if kind == "route":
        nbytes = T * case["E"] * (2 if case["type"] == "bf16" else 4) + 16 * T * k + 4 * (case["E"] + 1)
        return {"bytes": float(nbytes), "flops": 4.0 * T * case["E"]}
    kept = T * (1 - case["padded"])
    nbytes = 2 * kept * k * case["hidden"] + 8 * T * k + 2 * T * case["hidden"] * (2 if case["residual"] else 1)
    return {"bytes": float(nbytes), "flops": 2.0 * kept * k * case["hidden"]}


# ------------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    return globals()["_exact_" + case["kind"]](s, case)


def _weights64(packed, scale, zp):
    rows, words = packed.shape
    w = torch.empty((rows, words * 8), dtype=torch.float64, device=packed.device)
    z = torch.empty((rows, zp.shape[1]), dtype=torch.float64, device=packed.device)
    for i in range(8):  # nibble i: column 8 j + i of the codes, row 8 j + i of the zero points
        w[:, i::8] = (packed // 2 ** (4 * i) % 16).double() if i < 7 else (packed.long() % 2 ** 32 // 2 ** 28).double()
        z[i::8] = (zp.long() % 2 ** 32 // 2 ** (4 * i) % 16).double()
    w -= z.repeat_interleave(GROUP, dim=1)
    w *= scale.double().repeat_interleave(GROUP, dim=1)
    return w.to(torch.bfloat16).double()  # (the product is exact, the rounding is the definition's)


def _layer64(x, disk, bias, act):
    v = x.double() @ _weights64(*disk).T
    if bias is not None:
        v += bias.double()
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * 0.5 * torch.special.erfc(-v / math.sqrt(2.0))
    if act == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    if act == "swiglu":
        half = v.shape[1] // 2
        return v[:, :half] * torch.sigmoid(v[:, :half]) * v[:, half:]
    return v


def _exact_linear(s, case):
    v = _layer64(s.x, s.disk, s.bias, case["act"])
    return v if s.residual is None else v + s.residual.double()


def _exact_experts(s, case):
    y = torch.zeros(s.y.shape, dtype=torch.float64, device="cuda")
    for e in range(case["E"]):
        here = slice(s.bounds[e], s.bounds[e + 1])
        if here.start < here.stop:
            x = s.x[here] if s.x_rows is None else s.x[s.x_rows[here].long()]
            y[here] = _layer64(x, [t[e] for t in s.disk], None if s.bias is None else s.bias[e], case["act"])
    return y


def _exact_route(s, case):
    logits = s.logits.double()
    k, E = case["top_k"], case["E"]
    left = logits.clone()
    ids, weights = [], []
    share = torch.softmax(logits, 1)  # (nan where every logit is -inf)
    for _ in range(k):
        best = left.amax(1, keepdim=True)
        first = (left == best).float().argmax(1, keepdim=True)
        gone = best == -math.inf
        ids.append(torch.where(gone, -1, first))
        weights.append(torch.where(gone, 0.0, share.gather(1, first)))
        left.scatter_(1, first, -math.inf)
    ids, weights = torch.cat(ids, 1), torch.cat(weights, 1)
    if case["renormalize"]:
        weights = torch.where(ids >= 0, weights / weights.sum(1, keepdim=True), 0.0)
    chosen = torch.zeros((case["tokens"], E + 1), dtype=torch.int64, device="cuda").scatter_(1, torch.where(ids < 0, E, ids), 1)[:, :E]
    before = chosen.cumsum(0) - chosen  # earlier tokens with the same expert
    offsets = torch.cat([before.new_zeros(1), chosen.sum(0).cumsum(0)])
    slots = torch.where(ids < 0, -1, offsets[ids.clamp(min=0)] + before.gather(1, ids.clamp(min=0)))
    rows = torch.zeros(case["tokens"] * k + 1, dtype=torch.int64, device="cuda")
    rows[slots.flatten()] = torch.arange(case["tokens"], device="cuda").repeat_interleave(k)  # (slot -1: the extra last entry)
    return ids.int(), weights, offsets.int(), slots.int(), rows[:-1].int()


def _exact_combine(s, case):
    v = torch.zeros(s.y.shape, dtype=torch.float64, device="cuda") if s.residual is None else s.residual.double()
    for j in range(case["top_k"]):
        t = (s.slots[:, j] >= 0).nonzero().flatten()
        v[t] += s.weights[t, j].double().unsqueeze(1) * s.parts[s.slots[t, j].long()].double()
    return v
