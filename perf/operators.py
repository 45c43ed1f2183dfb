"""What the speed of the 4-bit operators is measured on: products with 4-bit weights and group scales, the
conversion of a matrix to them and back, tokens sorted by expert and back, and routed experts with 4-bit weights.

Sizes are those of the released architecture (hidden 4096, experts of 2048 channels, 288 of them or the 36 that one
of eight expert-parallel ranks owns, top-8, a dense MLP of 12288, a vocabulary of 154880) and odd ones beside them.

Kinds of case
  matmul    y[t] = W x[t]: `rows` x `cols` in groups of `group`, `tokens` rows of `dtype`
  quantize  a matrix of `source` (f32, bf16, fp8 with 128 x 128 block scales) to 4 bits, and its values back in FP32
  sort      picks of `tokens` tokens (top-`topk` of 288 experts, `experts` of them here) sorted, the rows gathered, combined
  experts   `tokens` rows through the routed experts: gate, up, clamped SwiGLU, down, weighted sum
"""
import functools
import importlib.util
import os
import sys

import torch

own = False

ALL_EXPERTS = 288
LIMIT = 10.0                # clamp of the SwiGLU
BLOCK = 128                 # FP8 scale blocks
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one token through a matrix of the size of an expert's down projection: the smallest call
        {"name": "matmul_1", "kind": "matmul", "rows": 4096, "cols": 2048, "group": 128, "tokens": 1, "dtype": "f32"},
        # the vocabulary head of one decoded token: the largest stream of weights
        {"name": "head_1", "kind": "matmul", "rows": 154880, "cols": 4096, "group": 128, "tokens": 1, "dtype": "f32"},
        # a few sequences, a matrix whose sizes fit no tile
        {"name": "matmul_7_ragged", "kind": "matmul", "rows": 1003, "cols": 1234, "group": 32, "tokens": 7, "dtype": "bf16"},
        # the dense MLP of a full batch of sequences
        {"name": "matmul_64", "kind": "matmul", "rows": 12288, "cols": 4096, "group": 64, "tokens": 64, "dtype": "f32"},
        # the same of a prompt's pass
        {"name": "matmul_2048", "kind": "matmul", "rows": 12288, "cols": 4096, "group": 128, "tokens": 2048, "dtype": "f32"},
        # one expert matrix of the checkpoint on its way to 4 bits
        {"name": "quantize_fp8", "kind": "quantize", "rows": 2048, "cols": 4096, "group": 32, "source": "fp8"},
        # a dense MLP matrix of a BF16 checkpoint
        {"name": "quantize_bf16", "kind": "quantize", "rows": 12288, "cols": 4096, "group": 128, "source": "bf16"},
        # the picks of a full batch of sequences, all experts here
        {"name": "sort_64", "kind": "sort", "tokens": 64, "topk": 8, "experts": 288, "cols": 4096, "dtype": "f32"},
        # the picks of a prompt's pass on one of eight ranks: most of them are another rank's
        {"name": "sort_2048_rank", "kind": "sort", "tokens": 2048, "topk": 8, "experts": 36, "cols": 4096, "dtype": "bf16"},
        # one decoded token
        {"name": "experts_1", "kind": "experts", "tokens": 1, "topk": 8, "experts": 288, "hidden": 4096, "inter": 2048, "group": 128, "dtype": "f32"},
        # a full batch of sequences: nearly every expert has a token or two
        {"name": "experts_64", "kind": "experts", "tokens": 64, "topk": 8, "experts": 288, "hidden": 4096, "inter": 2048, "group": 128, "dtype": "f32"},
        # a prompt's pass on one of eight ranks: some 57 tokens to an expert
        {"name": "experts_2048_rank", "kind": "experts", "tokens": 2048, "topk": 8, "experts": 36, "hidden": 4096, "inter": 2048, "group": 64, "dtype": "f32"},
    ]


def _log_int(rng, lo, hi):
    return int(min(hi, max(lo, round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("matmul", "matmul", "quantize", "sort", "experts"))
    group, dtype = rng.choice((32, 64, 128)), rng.choice(("f32", "f32", "bf16"))
    if kind == "matmul":
        rows, cols = _log_int(rng, 16, 32768), _log_int(rng, 48, 16384)
        most = max(1, 12288 * 4096 * 2048 // (rows * cols))
        return {"kind": kind, "rows": rows, "cols": cols, "group": group, "tokens": _log_int(rng, 1, min(2048, most)), "dtype": dtype}
    if kind == "quantize":
        rows = _log_int(rng, 64, 16384)
        return {"kind": kind, "rows": rows, "cols": _log_int(rng, 64, min(16384, 12288 * 4096 // rows)), "group": group, "source": rng.choice(("f32", "bf16", "fp8"))}
    experts = rng.choice((36, 288))              # a rank's share: enough tokens that some of their picks are here
    if kind == "sort":
        tokens = _log_int(rng, 32, 2048) if experts == 36 else _log_int(rng, 1, 512)
        return {"kind": kind, "tokens": tokens, "topk": rng.choice((2, 4, 8)), "experts": experts, "cols": rng.choice((4096, _log_int(rng, 64, 4096))), "dtype": dtype}
    hidden, inter = rng.choice(((4096, 2048), (_log_int(rng, 64, 4096), _log_int(rng, 64, 2048))))
    tokens = _log_int(rng, 32, 2048) if experts == 36 else _log_int(rng, 1, 64)
    return {"kind": kind, "tokens": tokens, "topk": rng.choice((4, 8)), "experts": experts, "hidden": hidden, "inter": inter, "group": group, "dtype": dtype}


# ------------------------------------------------------------------ inputs ----
@functools.lru_cache(None)
def _package():
    """The package of the tree in the working folder (its directory name is not an identifier)."""
    path = os.path.join(os.getcwd(), "glm-5.3-flash-in-c_b200")
    spec = importlib.util.spec_from_file_location("glm53f_b200", os.path.join(path, "__init__.py"), submodule_search_locations=[path])
    mod = importlib.util.module_from_spec(spec)
    sys.modules["glm53f_b200"] = mod
    spec.loader.exec_module(mod)
    return mod


def _up(n, m):
    return (n + m - 1) // m * m


def _matrix(g, rows, cols, group, count=None):
    """Codes and scales as a quantized matrix of normal weights (deviation 0.02) has them: codes in a bell around the middle,
    scales of groups a little apart. Rows are padded as the format asks (16 bytes of codes, 8 scales)."""
    shape = (rows,) if count is None else (count, rows)
    pitch, groups = _up(cols, 32) // 2, (cols + group - 1) // group
    dice = lambda: torch.randint(0, 6, shape + (pitch,), generator=g, device="cuda", dtype=torch.uint8)     # noqa: E731
    low, high = dice().add_(dice()).add_(dice()), dice().add_(dice()).add_(dice())
    scales = torch.zeros(shape + (_up(groups, 8),), device="cuda", dtype=torch.bfloat16)
    scales[..., :groups] = 0.0075 * (0.2 * torch.randn(shape + (groups,), generator=g, device="cuda")).exp()
    return {"codes": low | (high << 4), "scales": scales, "rows": rows, "cols": cols, "group": group}


def _activations(g, tokens, cols, dtype):
    """Rows as they come out of a norm: unit deviation, a few channels ten times as large."""
    x = torch.randn((tokens, cols), generator=g, device="cuda")
    x[:, torch.randint(0, cols, (max(1, cols // 500),), generator=g, device="cuda")] *= 10.0
    return x.to(TYPES[dtype])


def _picks(g, tokens, topk, experts):
    """Distinct experts of every token, numbered from the first that is here; -1 where another rank owns one."""
    score = torch.rand((tokens, ALL_EXPERTS), generator=g, device="cuda")
    idx = score.topk(topk, dim=1).indices.to(torch.int32)
    idx = torch.where(idx < experts, idx, -1)
    w = torch.rand((tokens, topk), generator=g, device="cuda") + 0.1
    return idx.contiguous(), 2.5 * w / w.sum(1, keepdim=True)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    kind, s = case["kind"], {"kind": case["kind"]}
    if kind == "matmul":
        s["w"] = _matrix(g, case["rows"], case["cols"], case["group"])
        s["x"] = _activations(g, case["tokens"], case["cols"], case["dtype"])
        s["y"] = torch.empty((case["tokens"], case["rows"]), device="cuda", dtype=s["x"].dtype)
    elif kind == "quantize":
        rows, cols, group = case["rows"], case["cols"], case["group"]
        w = 0.02 * torch.randn((rows, cols), generator=g, device="cuda")
        s["scale"] = None
        if case["source"] == "fp8":
            s["scale"] = 1e-4 * (1.0 + torch.rand((_up(rows, BLOCK) // BLOCK, _up(cols, BLOCK) // BLOCK), generator=g, device="cuda"))
            s["source"] = (w * 5000.0).to(torch.float8_e4m3fn)
        else:
            s["source"] = w.to(TYPES[case["source"]])
        s["w"] = {"codes": torch.zeros((rows, _up(cols, 32) // 2), device="cuda", dtype=torch.uint8),
                  "scales": torch.zeros((rows, _up((cols + group - 1) // group, 8)), device="cuda", dtype=torch.bfloat16),
                  "rows": rows, "cols": cols, "group": group}
        s["y"] = torch.empty((rows, cols), device="cuda")
    else:
        tokens, topk, experts = case["tokens"], case["topk"], case["experts"]
        s["idx"], s["weights"] = _picks(g, tokens, topk, experts)
        s["experts"] = experts
        if kind == "sort":
            s["x"] = _activations(g, tokens, case["cols"], case["dtype"])
            s["order"] = torch.empty(tokens * topk, device="cuda", dtype=torch.int32)
            s["place"] = torch.empty((tokens, topk), device="cuda", dtype=torch.int32)
            s["offsets"] = torch.empty(experts + 1, device="cuda", dtype=torch.int32)
            s["rows"] = torch.zeros((tokens * topk, case["cols"]), device="cuda", dtype=s["x"].dtype)
        else:
            H, I, group = case["hidden"], case["inter"], case["group"]
            s["gate"], s["up"] = (_matrix(g, I, H, group, experts) for _ in range(2))
            s["down"] = _matrix(g, H, I, group, experts)
            s["x"] = _activations(g, tokens, H, case["dtype"])
        s["y"] = torch.empty_like(s["x"])
    if own:                      # the handles and the workspace that a program keeps beside its weights
        p = _package()
        s["handles"] = {n: p.W4(**s[n]) for n in ("w", "gate", "up", "down") if n in s}
        if kind == "matmul":
            n = p.w4_matmul_workspace(s["handles"]["w"], s["x"])
        elif kind == "experts":
            n = p.w4_experts_workspace(*(s["handles"][m] for m in ("gate", "up", "down")), s["x"], s["idx"])
        else:
            n = 0
        s["workspace"] = torch.empty(max(1, n), device="cuda", dtype=torch.uint8)
    return s


# ------------------------------------------------------------------ the operators ----
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    p, h = _package(), s["handles"]
    if s["kind"] == "matmul":
        p.w4_matmul(h["w"], s["x"], s["y"], s["workspace"])
        return s["y"]
    if s["kind"] == "quantize":
        p.w4_quantize(s["source"], h["w"], scale_inv=s["scale"])
        p.w4_dequantize(h["w"], s["y"])
        return s["y"], s["w"]["scales"]
    if s["kind"] == "sort":
        p.expert_sort(s["idx"], s["experts"], s["order"], s["place"], s["offsets"])
        p.expert_gather(s["x"], s["order"], s["offsets"], s["rows"])
        p.expert_combine(s["rows"], s["place"], s["weights"], s["y"])
        return s["order"], s["place"], s["offsets"], s["rows"], s["y"]
    p.w4_experts(h["gate"], h["up"], h["down"], s["x"], s["idx"], s["weights"], LIMIT, s["y"], s["workspace"])
    return s["y"]


def _values(w, picked=None):
    """The FP32 values of a matrix (or of the picked ones of a stack)."""
    codes, scales = (w["codes"], w["scales"]) if picked is None else (w["codes"][picked], w["scales"][picked])
    c = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)[..., :w["cols"]].to(torch.float32).sub_(8.0)
    return c.mul_(scales.to(torch.float32).repeat_interleave(w["group"], dim=-1)[..., :w["cols"]])


def _plain_quantize(s):
    w, group = s["w"], s["w"]["group"]
    rows, cols = w["rows"], w["cols"]
    v = s["source"].to(torch.float32)
    if s["scale"] is not None:
        v = v * s["scale"].repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    groups = (cols + group - 1) // group
    v = torch.nn.functional.pad(v, (0, groups * group - cols)).view(rows, groups, group)
    # 64 bits: quotients next to a border between two roundings must fall on their own side of it
    scale = (v.abs().amax(2).double() / 7.0).to(torch.float32).to(torch.bfloat16)
    q = (v.double() / scale.double()[..., None]).round().clamp(-7.0, 7.0)
    q = torch.where(scale[..., None] == 0, 0.0, q)
    y = (q * scale.double()[..., None]).to(torch.float32).view(rows, -1)[:, :cols]
    return y.contiguous(), torch.nn.functional.pad(scale, (0, w["scales"].shape[1] - groups))


def _plain_sort(s):
    x, idx, E = s["x"], s["idx"], s["experts"]
    T, K = idx.shape
    key = torch.where((idx >= 0) & (idx < E), idx, E).flatten()
    by = torch.argsort(key, stable=True)
    here = key[by] < E
    order = torch.where(here, by, -1).to(torch.int32)
    at = torch.empty_like(by)
    at[by] = torch.arange(T * K, device=x.device)
    place = torch.where(key < E, at, -1).to(torch.int32).view(T, K)
    offsets = (key[None, :] < torch.arange(E + 1, device=x.device)[:, None]).sum(1).to(torch.int32)
    rows = torch.where(here[:, None], x[by // K], 0)
    taken = torch.where(place[..., None] >= 0, rows[place.clamp(min=0).long()].to(torch.float32) * s["weights"][..., None], 0.0)
    return order, place, offsets, rows, taken.sum(1).to(x.dtype)


def _swiglu(gate, up):
    gate, up = gate.clamp(max=LIMIT), up.clamp(-LIMIT, LIMIT)
    return gate / (1.0 + torch.exp(-gate)) * up


def _plain_experts(s):
    x, idx, E = s["x"].to(torch.float32), s["idx"].long(), s["experts"]
    T, K = idx.shape
    here = (idx >= 0) & (idx < E)
    if T * K <= E:               # few picks: each one's expert on its own
        e = idx.clamp(min=0).flatten()
        rows = x.repeat_interleave(K, 0)[..., None]
        h = _swiglu(_values(s["gate"], e) @ rows, _values(s["up"], e) @ rows)
        got = (_values(s["down"], e) @ h).view(T, K, -1)
        return torch.where(here[..., None], got * s["weights"][..., None], 0.0).sum(1).to(s["x"].dtype)
    # many: every expert past all tokens, weighted by what each token gives it
    part = torch.zeros((T, E), device=x.device).scatter_add_(1, idx.clamp(min=0), torch.where(here, s["weights"], 0.0))
    h = _swiglu(x @ _values(s["gate"]).transpose(1, 2), x @ _values(s["up"]).transpose(1, 2))       # [E][T][inter]
    h = torch.where(part.t()[..., None] != 0, h * part.t()[..., None], 0.0)
    return (h @ _values(s["down"]).transpose(1, 2)).sum(0).to(s["x"].dtype)


def _run_plain(s):
    if s["kind"] == "matmul":
        return (s["x"].to(torch.float32) @ _values(s["w"]).t()).to(s["x"].dtype)
    if s["kind"] == "quantize":
        return _plain_quantize(s)
    return _plain_sort(s) if s["kind"] == "sort" else _plain_experts(s)


# ------------------------------------------------------------------ what a pass cannot do without ----
def _matrix_bytes(rows, cols, group):
    return rows * (cols / 2 + 2 * ((cols + group - 1) // group))


def work(case):
    kind, size = case["kind"], {"f32": 4, "bf16": 2, "fp8": 1}
    if kind == "matmul":
        r, c, t = case["rows"], case["cols"], case["tokens"]
        return {"bytes": _matrix_bytes(r, c, case["group"]) + t * (r + c) * size[case["dtype"]], "flops": 2 * r * c * t}
    if kind == "quantize":       # the matrix in, codes and scales out, and in again for their FP32 values
        r, c = case["rows"], case["cols"]
        return {"bytes": r * c * size[case["source"]] + 2 * _matrix_bytes(r, c, case["group"]) + 4 * r * c, "flops": 4 * r * c}
    t, picks, share = case["tokens"], case["tokens"] * case["topk"], case["experts"] / ALL_EXPERTS
    if kind == "sort":           # picks in, order and places out, the rows of the picks that are here written, read and summed
        row = case["cols"] * size[case["dtype"]]
        return {"bytes": 16 * picks + 4 * case["experts"] + 2 * t * row + 2 * picks * share * row, "flops": 2 * picks * share * case["cols"]}
    H, I = case["hidden"], case["inter"]
    used = case["experts"] * (1 - (1 - case["topk"] / ALL_EXPERTS) ** t)        # experts that some token chooses
    each = 2 * _matrix_bytes(I, H, case["group"]) + _matrix_bytes(H, I, case["group"])
    return {"bytes": used * each + 2 * t * H * size[case["dtype"]] + 8 * picks, "flops": 6 * H * I * picks * share}


# ------------------------------------------------------------------ the definition, in 64 bits ----
def _weight64(w, e=None):
    codes, scales = (w["codes"], w["scales"]) if e is None else (w["codes"][e], w["scales"][e])
    out = torch.empty((w["rows"], 2 * codes.shape[1]), device="cuda", dtype=torch.float64)
    out[:, 0::2] = codes.bitwise_and(0x0f)
    out[:, 1::2] = codes.bitwise_right_shift(4)
    column = torch.arange(w["cols"], device="cuda")
    return (out[:, :w["cols"]] - 8) * scales.double().index_select(1, column // w["group"])


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "matmul":
        x = s["x"].double()
        step = 16384             # rows at a time
        out = torch.empty((x.shape[0], case["rows"]), device="cuda", dtype=torch.float64)
        for r in range(0, case["rows"], step):
            part = {**s["w"], "codes": s["w"]["codes"][r:r + step], "scales": s["w"]["scales"][r:r + step], "rows": min(step, case["rows"] - r)}
            out[:, r:r + step] = x.mm(_weight64(part).t())
        return out
    if kind == "quantize":
        v = s["source"].float()
        r, c = torch.arange(case["rows"], device="cuda"), torch.arange(case["cols"], device="cuda")
        if s["scale"] is not None:                  # a weight of the checkpoint is the FP32 product of its code and its block's scale
            v = v * s["scale"][r // BLOCK][:, c // BLOCK]
        v, group = v.double(), case["group"]
        y, scales = torch.zeros_like(v), torch.zeros(s["w"]["scales"].shape, device="cuda", dtype=torch.float64)
        for k, c0 in enumerate(range(0, case["cols"], group)):
            part = v[:, c0:c0 + group]
            sc = (part.abs().max(1).values / 7).float().bfloat16().double()
            scales[:, k] = sc
            q = torch.where(sc[:, None] > 0, torch.round(part / sc[:, None]), torch.zeros_like(part))
            y[:, c0:c0 + group] = torch.minimum(torch.maximum(q, q.new_tensor(-7.0)), q.new_tensor(7.0)) * sc[:, None]
        return y, scales
    idx, w, x = s["idx"].tolist(), s["weights"].double(), s["x"].double()
    T, K, E = case["tokens"], case["topk"], case["experts"]
    of = [[] for _ in range(E)]                     # picks of each expert, in order
    for t, row in enumerate(idx):
        for k, e in enumerate(row):
            if 0 <= e < E:
                of[e].append(t * K + k)
    out = torch.zeros_like(x)
    if kind == "sort":
        order = [p for picks in of for p in picks]
        place, offsets = [-1] * (T * K), [0]
        for i, p in enumerate(order):
            place[p] = i
        for picks in of:
            offsets.append(offsets[-1] + len(picks))
        rows = torch.zeros((T * K, case["cols"]), device="cuda", dtype=torch.float64)
        if order:
            at = torch.tensor(order, device="cuda")
            rows[:len(order)] = x[at // K]
            out.index_add_(0, at // K, rows[:len(order)] * w.flatten()[at][:, None])
        whole = lambda v: torch.tensor(v, dtype=torch.int32)        # noqa: E731
        return whole(order + [-1] * (T * K - len(order))), whole(place).view(T, K), whole(offsets), rows, out
    for e, picks in enumerate(of):
        if picks:
            at = torch.tensor(picks, device="cuda")
            rows = x[at // K]
            gate, up = rows.mm(_weight64(s["gate"], e).t()), rows.mm(_weight64(s["up"], e).t())
            gate, up = gate.minimum(gate.new_tensor(LIMIT)), up.maximum(up.new_tensor(-LIMIT)).minimum(up.new_tensor(LIMIT))
            h = gate * torch.sigmoid(gate) * up
            out.index_add_(0, at // K, h.mm(_weight64(s["down"], e).t()) * w.flatten()[at][:, None])
    return out
