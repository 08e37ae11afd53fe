"""Cases of the 8-bit floating point and mixture-of-experts operators, in plain torch and through the framework.

Three operators of a feed-forward network are measured:

* ``quant``: rows of activations to e4m3 with one fp32 scale for each row and 128 columns;
* ``dense``: y = act(W x + b) on e4m3 operands, x scaled per row and 128 columns, W per block
  of 128 x 128, the result in 32 or 16 bits or again in e4m3 with scales;
* ``moe``: a whole mixture-of-experts layer for up to 32 rows (router, choice of the experts,
  their gated products, and the weighted sum).

``own`` selects which form ``run`` computes.
"""
import math

import torch

own = False

BLOCK = 128
FP8_MAX = 448.0
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _up(n, m):
    return -(-n // m) * m


def _ceil(n, m):
    return -(-n // m)


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one request's activations before a layer of 2048 inputs: launch latency is all there is
        {"name": "quant_row", "op": "quant", "rows": 1, "dim": 2048, "x": "bf16", "pow2": False},
        # a ragged micro-batch of fp32 activations whose last group is short, power-of-two scales
        {"name": "quant_ragged", "op": "quant", "rows": 333, "dim": 1000, "x": "f32", "pow2": True},
        # a stacked batch of wide activations: bound by the memory
        {"name": "quant_stack", "op": "quant", "rows": 8192, "dim": 4096, "x": "bf16", "pow2": False},
        # one request through one hidden layer: the weights are read once
        {"name": "dense_row", "op": "dense", "rows": 1, "m": 2048, "k": 2048, "y": "bf16", "act": "relu", "bias": True},
        # the largest small batch, wide layer, result handed on in e4m3 to the next layer
        {"name": "dense_batch32", "op": "dense", "rows": 32, "m": 4096, "k": 4096, "y": "f8", "act": "gelu",
         "bias": True},
        # sizes that fill no tile and no scale block, 32-bit result
        {"name": "dense_ragged", "op": "dense", "rows": 301, "m": 1000, "k": 1100, "y": "f32", "act": "identity",
         "bias": False},
        # a batch of 256 through a square layer of 2048
        {"name": "dense_batch256", "op": "dense", "rows": 256, "m": 2048, "k": 2048, "y": "bf16", "act": "relu",
         "bias": True},
        # stacked batches: bound by the tensor cores
        {"name": "dense_stack", "op": "dense", "rows": 8192, "m": 4096, "k": 4096, "y": "bf16", "act": "gelu",
         "bias": True},
        # one request through a small layer of few experts: latency
        {"name": "moe_row_small", "op": "moe", "rows": 1, "hidden": 1024, "inter": 512, "experts": 8, "top_k": 2,
         "act": "silu", "gated": True, "w": "bf16", "x": "bf16", "renorm": True},
        # one request through many experts in e4m3 blocks
        {"name": "moe_row_fp8", "op": "moe", "rows": 1, "hidden": 2048, "inter": 1024, "experts": 64, "top_k": 8,
         "act": "silu", "gated": True, "w": "f8", "x": "bf16", "renorm": True},
        # a few requests, int8 experts without a gate, sizes that fill no tile, 32-bit activations
        {"name": "moe_ragged_int8", "op": "moe", "rows": 5, "hidden": 1000, "inter": 344, "experts": 10, "top_k": 3,
         "act": "gelu", "gated": False, "w": "i8", "x": "f32", "renorm": False},
        # the largest small batch: nearly every expert is read
        {"name": "moe_batch32", "op": "moe", "rows": 32, "hidden": 2048, "inter": 1024, "experts": 64, "top_k": 8,
         "act": "silu", "gated": True, "w": "bf16", "x": "bf16", "renorm": True},
    ]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["quant", "dense", "dense", "moe", "moe"])
    if op == "quant":
        while True:
            rows, dim = _log_int(rng, 1, 8192), _log_int(rng, 16, 8192)
            if rows * dim <= 8192 * 4096:
                break
        return {"op": "quant", "rows": rows, "dim": dim, "x": rng.choice(["f32", "bf16", "f16"]),
                "pow2": rng.random() < 0.5}
    if op == "dense":
        while True:
            rows, m, k = _log_int(rng, 1, 8192), _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)
            if rng.random() < 0.5:
                m, k = _up(m, 64), _up(k, 64)
            if rows * m * k <= 8192 * 4096 * 4096:
                break
        return {"op": "dense", "rows": rows, "m": m, "k": k, "y": rng.choice(["f32", "bf16", "f16", "f8"]),
                "act": rng.choice(["identity", "relu", "gelu", "silu"]), "bias": rng.random() < 0.5}
    while True:
        hidden, inter = _log_int(rng, 64, 4096), _log_int(rng, 64, 2048)
        if rng.random() < 0.7:
            hidden, inter = _up(hidden, 64), _up(inter, 64)
        experts = _log_int(rng, 2, 128)
        if experts * hidden * inter <= 64 * 2048 * 1024:
            break
    return {"op": "moe", "rows": _log_int(rng, 1, 32), "hidden": hidden, "inter": inter, "experts": experts,
            "top_k": rng.randint(1, min(8, experts)), "act": rng.choice(["silu", "gelu", "relu"]),
            "gated": rng.random() < 0.7, "w": rng.choice(["bf16", "i8", "f8"]),
            "x": rng.choice(["bf16", "f16", "f32"]), "renorm": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _fp8_rows(x):
    """e4m3 values (in a buffer whose rows start on 16 bytes) and scales of x per row and 128 columns."""
    r, k = x.shape
    kb, ld = _ceil(k, BLOCK), _up(k, 16)
    p = torch.zeros(r, kb * BLOCK, device=x.device)
    p[:, :k] = x
    p = p.view(r, kb, BLOCK)
    s = (p.abs().amax(2) / FP8_MAX).clamp_min(1e-30)
    q = torch.zeros(r, ld, dtype=torch.float8_e4m3fn, device=x.device)
    q.view(torch.uint8)[:, :k] = (p / s[:, :, None]).view(r, -1)[:, :k].to(torch.float8_e4m3fn).view(torch.uint8)
    return q, s


def _fp8_blocks(w):
    """e4m3 values and scales of w [..., m, k] per block of 128 x 128 (w is padded for the scales alone)."""
    *lead, m, k = w.shape
    mb, kb = _ceil(m, BLOCK), _ceil(k, BLOCK)
    s = torch.empty(*lead, mb, kb, device=w.device)
    q = torch.zeros(*lead, m, k, dtype=torch.uint8, device=w.device)
    for i in range(mb):
        for j in range(kb):
            c = w[..., i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK].float()
            t = (c.abs().amax((-1, -2)) / FP8_MAX).clamp_min(1e-30)
            s[..., i, j] = t
            q[..., i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] = \
                (c / t[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return q.view(torch.float8_e4m3fn), s


def _expert_weights(g, e, m, k, kind):
    w = torch.empty(e, m, k, dtype=torch.bfloat16, device="cuda").normal_(0.0, k ** -0.5, generator=g)
    if kind == "bf16":
        return w, None
    if kind == "i8":
        f = w.float()
        s = f.abs().amax(2) / 127.0
        return torch.round(f / s[:, :, None]).clamp(-127, 127).to(torch.int8), s
    return _fp8_blocks(w)


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    if case["op"] == "quant":
        r, d = case["rows"], case["dim"]
        x = torch.randn(r, d, device="cuda", generator=g)
        # activations have channels that are far larger than the others, and dead groups
        x *= torch.exp(1.5 * torch.randn(d, device="cuda", generator=g))
        if d > BLOCK:
            x[:: 7, :BLOCK] = 0
        st["x"] = x.to(DT[case["x"]])
        st["q"] = torch.zeros(r, _up(d, 16), dtype=torch.float8_e4m3fn, device="cuda")
        st["s"] = torch.zeros(r, _ceil(d, BLOCK), device="cuda")
    elif case["op"] == "dense":
        r, m, k = case["rows"], case["m"], case["k"]
        st["x"], st["sx"] = _fp8_rows(torch.randn(r, k, device="cuda", generator=g))
        w = torch.randn(m, _up(k, 16), device="cuda", generator=g) * k ** -0.5
        w[:, k:] = 0
        st["w"], st["sw"] = _fp8_blocks(w)
        st["sw"] = st["sw"][:, :_ceil(k, BLOCK)].contiguous()
        st["b"] = 0.1 * torch.randn(m, device="cuda", generator=g) if case["bias"] else None
        if case["y"] == "f8":
            st["y"] = torch.zeros(r, _up(m, 16), dtype=torch.float8_e4m3fn, device="cuda")
            st["sy"] = torch.zeros(r, _ceil(m, BLOCK), device="cuda")
        else:
            st["y"] = torch.zeros(r, m, dtype=DT[case["y"]], device="cuda")
    else:
        t, h, f, e, k = case["rows"], case["hidden"], case["inter"], case["experts"], case["top_k"]
        st["x"] = torch.randn(t, h, device="cuda", generator=g).to(DT[case["x"]])
        st["router"] = (1.5 * torch.randn(e, h, device="cuda", generator=g) * h ** -0.5).to(torch.bfloat16)
        st["gate"], st["gate_s"] = _expert_weights(g, e, f, h, case["w"])
        st["up"], st["up_s"] = _expert_weights(g, e, f, h, case["w"]) if case["gated"] else (None, None)
        st["down"], st["down_s"] = _expert_weights(g, e, h, f, case["w"])
        st["y"] = torch.zeros(t, h, dtype=DT[case["x"]], device="cuda")
        st["ids"] = torch.zeros(t, k, dtype=torch.int32, device="cuda")
        st["probs"] = torch.zeros(t, k, device="cuda")
    if own:
        _prepare_own(case, st)
    return st


def _prepare_own(case, st):
    """What a program of this framework keeps beside its tensors: the description and the workspace."""
    import low_latency_inference_gpu_b200 as ll

    st["act"] = {"identity": ll.ACT_IDENTITY, "relu": ll.ACT_RELU, "gelu": ll.ACT_GELU,
                 "silu": ll.ACT_SILU}[case.get("act", "identity")]
    types = {"f32": ll.T_F32, "bf16": ll.T_BF16, "f16": ll.T_F16, "f8": ll.T_F8}
    if case["op"] == "quant":
        st["type"] = types[case["x"]]
    elif case["op"] == "dense":
        st["type"] = types[case["y"]]
    else:
        st["moe"] = ll.MoE(hidden=case["hidden"], inter=case["inter"], n_experts=case["experts"],
                           top_k=case["top_k"], act=st["act"], gated=case["gated"],
                           wtype={"bf16": ll.W_BF16, "i8": ll.W_I8, "f8": ll.W_F8}[case["w"]],
                           x_type=types[case["x"]], router_type=ll.T_BF16, renormalize=case["renorm"])
        ptr = lambda v: 0 if v is None else v.data_ptr()  # noqa: E731
        st["weights"] = ll.MoEWeights(router=ptr(st["router"]), gate=ptr(st["gate"]), up=ptr(st["up"]),
                                      down=ptr(st["down"]), gate_scale=ptr(st["gate_s"]),
                                      up_scale=ptr(st["up_s"]), down_scale=ptr(st["down_s"]))
        st["work"] = torch.zeros(ll.moe_workspace_bytes(st["moe"], case["rows"]), dtype=torch.uint8, device="cuda")


# ---------------------------------------------------------------- the plain form
def _act(v, act):
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * 0.5 ** 0.5))
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _round_e4m3(t):
    """t (64 bits) to the nearest e4m3 value, ties to even, values past the largest to the largest."""
    a = t.abs().clamp_max(FP8_MAX)
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return (torch.sign(t) * (torch.round(a / step) * step).clamp_max(FP8_MAX)).to(torch.float32).to(torch.float8_e4m3fn)


def _quant_plain(x, pow2):
    r, d = x.shape
    g = _ceil(d, BLOCK)
    p = torch.zeros(r, g * BLOCK, dtype=torch.float32, device=x.device)
    p[:, :d] = x.float()
    p = p.view(r, g, BLOCK)
    amax = p.abs().amax(2)
    # 64 bits here, rounded once: the scale decides on which side of a border a quotient falls
    s = (amax.double() / FP8_MAX).float()
    if pow2:
        m, e = torch.frexp(s.double())
        s = torch.where(amax > 0, torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e)), 0.0).float()
    # 64 bits here: a quotient next to the border of two e4m3 values
    t = p.double() / torch.where(s > 0, s, torch.ones_like(s)).double()[:, :, None]
    return _round_e4m3(t.view(r, -1)[:, :d]), s


def _dequant_rows(q, s, k):
    return q[:, :k].float() * s.repeat_interleave(BLOCK, 1)[:, :k]


def _dequant(w, s, m, k):
    """32-bit values of expert or layer weights [..., m, k] in any of their types."""
    f = w.float()
    if s is None:
        return f
    if w.dtype == torch.int8:
        return f * s[..., None]
    return f * s.repeat_interleave(BLOCK, -2)[..., :m, :].repeat_interleave(BLOCK, -1)[..., :k]


def _run_plain(st):
    c = st["case"]
    if c["op"] == "quant":
        return _quant_plain(st["x"], c["pow2"])
    if c["op"] == "dense":
        m, k = c["m"], c["k"]
        y = _dequant_rows(st["x"], st["sx"], k) @ _dequant(st["w"][:, :k], st["sw"], m, k).t()
        if st["b"] is not None:
            y = y + st["b"]
        y = _act(y, c["act"])
        return _quant_plain(y, False) if c["y"] == "f8" else y.to(DT[c["y"]])
    t, h, f, e, k = c["rows"], c["hidden"], c["inter"], c["experts"], c["top_k"]
    x = st["x"].float()
    logits = x @ st["router"].float().t()
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :k]
    w = torch.gather(p, 1, ids)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    if t * k <= e:  # few rows: their experts alone, gathered
        pick = lambda v: None if v is None else v.view(torch.uint8)[ids].view(v.dtype) if v.dtype == torch.float8_e4m3fn else v[ids]  # noqa: E731,E501
        wg = _dequant(pick(st["gate"]), pick(st["gate_s"]), f, h)
        a = _act((wg @ x[:, None, :, None])[..., 0], c["act"])
        if c["gated"]:
            a = a * (_dequant(pick(st["up"]), pick(st["up_s"]), f, h) @ x[:, None, :, None])[..., 0]
        y = (_dequant(pick(st["down"]), pick(st["down_s"]), h, f) @ a[..., None])[..., 0]
        y = (w[:, :, None] * y).sum(1)
    else:  # nearly every expert has a row: all of them, those that a row did not pick with weight 0
        a = _act(x @ _dequant(st["gate"], st["gate_s"], f, h).transpose(1, 2), c["act"])
        if c["gated"]:
            a = a * (x @ _dequant(st["up"], st["up_s"], f, h).transpose(1, 2))
        y = a @ _dequant(st["down"], st["down_s"], h, f).transpose(1, 2)
        full = torch.zeros(t, e, device=x.device).scatter_(1, ids, w)
        y = (full.t()[:, :, None] * y).sum(0)
    return {"y": y.to(DT[c["x"]]), "ids": ids.int(), "probs": w}


# ---------------------------------------------------------------- the framework's calls
def _run_own(st):
    import low_latency_inference_gpu_b200 as ll

    c = st["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "quant":
        q, s = st["q"], st["s"]
        ll.quantize_fp8(st["x"].data_ptr(), st["type"], c["rows"], c["dim"], q.data_ptr(), s.data_ptr(),
                        ldq=q.stride(0), pow2=c["pow2"], stream=stream)
        return q[:, :c["dim"]], s
    if c["op"] == "dense":
        y, f8 = st["y"], c["y"] == "f8"
        ll.dense_fp8(st["w"].data_ptr(), st["sw"].data_ptr(), st["b"].data_ptr() if c["bias"] else 0,
                     st["x"].data_ptr(), st["sx"].data_ptr(), y.data_ptr(), c["rows"], c["m"], c["k"],
                     act=st["act"], y_type=st["type"], sy_ptr=st["sy"].data_ptr() if f8 else 0,
                     ldw=st["w"].stride(0), ldx=st["x"].stride(0), ldy=y.stride(0), stream=stream)
        return (y[:, :c["m"]], st["sy"]) if f8 else y
    ll.moe_forward(st["moe"], st["weights"], st["x"].data_ptr(), st["y"].data_ptr(), c["rows"],
                   st["work"].data_ptr(), st["work"].numel(), ids_ptr=st["ids"].data_ptr(),
                   probs_ptr=st["probs"].data_ptr(), stream=stream)
    return {"y": st["y"], "ids": st["ids"], "probs": st["probs"]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1, "f8": 1}


def work(case):
    if case["op"] == "quant":
        r, d = case["rows"], case["dim"]
        return {"bytes": r * d * (SIZE[case["x"]] + 1) + 4 * r * _ceil(d, BLOCK), "flops": 3 * r * d}
    if case["op"] == "dense":
        r, m, k = case["rows"], case["m"], case["k"]
        kb, mb = _ceil(k, BLOCK), _ceil(m, BLOCK)
        b = r * k + m * k + 4 * (r * kb + mb * kb) + (4 * m if case["bias"] else 0) + r * m * SIZE[case["y"]]
        return {"bytes": b + (4 * r * mb if case["y"] == "f8" else 0), "flops": 2 * r * m * k}
    t, h, f, e, k = case["rows"], case["hidden"], case["inter"], case["experts"], case["top_k"]
    mats = 3 if case["gated"] else 2
    used = e * (1.0 - (1.0 - k / e) ** t)  # experts that a row picked, rows choosing evenly
    b = used * mats * h * f * SIZE[case["w"]] + 2 * e * h + 2 * t * h * SIZE[case["x"]] + 8 * t * k
    return {"bytes": b, "flops": 2 * t * h * e + 2 * t * k * mats * h * f}


# ---------------------------------------------------------------- the definition in 64 bits
def _e4m3_table(device):
    codes = torch.arange(127, dtype=torch.uint8, device=device)  # 0 .. 448, rising
    return codes.view(torch.float8_e4m3fn).double()


def _nearest_e4m3(t):
    """The table's value nearest to |t|; a value half way goes to the even code."""
    table = _e4m3_table(t.device)
    a = t.abs().clamp_max(FP8_MAX)
    hi = torch.searchsorted(table, a.contiguous()).clamp(1, 126)
    lo = hi - 1
    down, up = a - table[lo], table[hi] - a
    code = torch.where(down < up, lo, torch.where(up < down, hi, lo + lo % 2))
    return torch.copysign(table[code], t)


def _quant_exact(v, pow2):
    r, d = v.shape
    q, s = torch.empty_like(v), torch.empty(r, _ceil(d, BLOCK), dtype=torch.float64, device=v.device)
    for j in range(s.shape[1]):
        x = v[:, j * BLOCK:(j + 1) * BLOCK]
        amax = x.abs().max(1).values
        t = (amax / FP8_MAX).float().double()
        if pow2:
            t = torch.where(amax > 0, 2.0 ** torch.ceil(torch.log2(t)), t)
        s[:, j] = t
        q[:, j * BLOCK:(j + 1) * BLOCK] = _nearest_e4m3(x / torch.where(t > 0, t, 1.0)[:, None])
    return q, s


def _act64(v, act):
    if act == "relu":
        return v.clamp_min(0.0)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "silu":
        return v * torch.special.expit(v)
    return v


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "quant":
        return _quant_exact(st["x"].double(), case["pow2"])
    if case["op"] == "dense":
        r, m, k = case["rows"], case["m"], case["k"]
        y = torch.zeros(r, m, dtype=torch.float64, device="cuda")
        for j in range(_ceil(k, BLOCK)):  # a block of 128 at a time
            lo, hi = j * BLOCK, min(k, (j + 1) * BLOCK)
            part = st["x"][:, lo:hi].double() @ st["w"][:, lo:hi].double().t()
            col = st["sw"][:, j].double()[torch.arange(m, device="cuda") // BLOCK]
            y += part * st["sx"][:, j].double()[:, None] * col
        if st["b"] is not None:
            y += st["b"].double()
        y = _act64(y, case["act"])
        return _quant_exact(y, False) if case["y"] == "f8" else y
    t, h, f, k = case["rows"], case["hidden"], case["inter"], case["top_k"]
    x = st["x"].double()
    logits = x @ st["router"].double().t()
    order = torch.argsort(-logits, dim=1, stable=True)[:, :k]
    lse = torch.logsumexp(logits if not case["renorm"] else torch.gather(logits, 1, order), 1)
    w = torch.exp(torch.gather(logits, 1, order) - lse[:, None])

    def full(name, i, m, n):
        q, s = st[name][i].double(), st[name + "_s"]
        if s is None:
            return q
        s = s[i].double()
        if case["w"] == "i8":
            return q * s[:, None]
        return q * s[torch.arange(m, device="cuda") // BLOCK][:, torch.arange(n, device="cuda") // BLOCK]

    y = torch.zeros(t, h, dtype=torch.float64, device="cuda")
    for i in torch.unique(order).tolist():
        rows, slot = torch.nonzero(order == i, as_tuple=True)
        a = _act64(x[rows] @ full("gate", i, f, h).t(), case["act"])
        if case["gated"]:
            a = a * (x[rows] @ full("up", i, f, h).t())
        y.index_add_(0, rows, w[rows, slot][:, None] * (a @ full("down", i, h, f).t()))
    return {"y": y, "ids": order.int(), "probs": w}
