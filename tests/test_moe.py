"""ll_moe_forward, a mixture-of-experts layer for a few rows, against numpy in 64 bits (B200).

Tolerances, per output, from the sums of magnitudes (A_v = sum |a| |b| of each product v):
  * every weight and every bf16 term of x is exact in the tensor instruction, whose fp32 sums are
    off by at most 2^-23 of a partial sum (<= A) per addition; a product over K columns makes
    NS K additions (NS = 1, 2, 3 bf16 terms for bf16, fp16, fp32 x) and at most 40 more (warps,
    blocks' scales, splits): |v - exact| <= A (NS K + 40) 2^-23.
  * the router (bf16 or 3 terms, so NS is 3 NS): logits off by t_l; a softmax weight is off by a
    factor within exp(+-2 t_l), and 2^-19 for exp and the sum of up to 256 terms.
  * act has slope <= 1.13 and is evaluated to 2^-20 of |v|; the product with up adds 2^-23; the
    activation is kept with 16 bits (2^-16) for 16-bit x, 23 (2^-22) for fp32.
  * the result is rounded by half a step: 2^-8 bf16, 2^-11 fp16.
The picked experts must be a top_k up to t_l: any expert left out has a logit at most 2 t_l above
one that was picked; the reference continues with the device's choice.
"""
import dataclasses

import numpy as np
import pytest

import low_latency_inference_gpu_b200 as ll
from test_fp8 import F8, act64, decode, dequant_blocks, dequant_rows, dev, quantize_rows, t_dtype, up

U = 2.0 ** -23
ROUND = {ll.T_F32: 2.0 ** -23, ll.T_BF16: 2.0 ** -8, ll.T_F16: 2.0 ** -11}


def desc(**kw):
    d = dict(hidden=64, inter=32, n_experts=4, top_k=2)
    d.update(kw)
    return ll.MoE(**d)


# ---------------------------------------------------------------- refusals (host)
def refused(fn, code, *a, **kw):
    with pytest.raises(ll.LLError) as e:
        fn(*a, **kw)
    assert e.value.code == code
    return str(e.value)


@pytest.mark.parametrize("bad", [
    dict(hidden=0), dict(inter=0), dict(hidden=65537), dict(n_experts=0), dict(n_experts=257), dict(top_k=0),
    dict(top_k=5), dict(n_experts=64, top_k=17), dict(act=4), dict(act=-1), dict(wtype=ll.W_F32), dict(wtype=4),
    dict(x_type=ll.T_F8), dict(router_type=ll.T_F16), dict(router_type=ll.T_F8)])
def test_refuses_descriptions(bad):
    refused(ll.moe_workspace_bytes, ll.LL_ERR_BAD_DESC, desc(**bad), 1)
    w = ll.MoEWeights(16, 16, 16, 16, 16, 16, 16)
    refused(ll.moe_forward, ll.LL_ERR_BAD_DESC, desc(**bad), w, 16, 16, 1, 256, 1 << 20)


def test_refuses_arguments():
    m, big = desc(), 1 << 20
    w = ll.MoEWeights(16, 16, 16, 16)
    bad = ll.LL_ERR_INVALID_ARG
    for rows in (-1, ll.MOE_MAX_ROWS + 1):
        refused(ll.moe_workspace_bytes, bad, m, rows)
        refused(ll.moe_forward, bad, m, w, 16, 16, rows, 256, big)
    refused(ll.moe_forward, bad, m, w, 0, 16, 1, 256, big)
    refused(ll.moe_forward, bad, m, w, 16, 0, 1, 256, big)
    refused(ll.moe_forward, bad, m, w, 16, 16, 1, 0, big)
    refused(ll.moe_forward, bad, m, w, 16, 16, 1, 256, big, ldx=63)
    refused(ll.moe_forward, bad, m, w, 16, 16, 1, 256, big, ldy=63)
    assert "workspace" in refused(ll.moe_forward, bad, m, w, 16, 16, 1, 256, ll.moe_workspace_bytes(m, 1) - 1)
    for name in ("router", "gate", "up", "down"):
        refused(ll.moe_forward, bad, m, dataclasses.replace(w, **{name: 0}), 16, 16, 1, 256, big)
    for t in (ll.W_I8, ll.W_F8):
        refused(ll.moe_forward, bad, desc(wtype=t), w, 16, 16, 1, 256, big)
    ll.moe_forward(m, w, 0, 0, 0, 0, 0)  # no rows: nothing to do


def test_workspace_grows_with_rows_and_covers_every_pair():
    for x_type, planes in ((ll.T_BF16, 2), (ll.T_F16, 2), (ll.T_F32, 3)):
        m = desc(inter=333, top_k=3, x_type=x_type)
        sizes = [ll.moe_workspace_bytes(m, r) for r in range(ll.MOE_MAX_ROWS + 1)]
        assert all(a <= b for a, b in zip(sizes, sizes[1:]))
        assert sizes[-1] >= 32 * 3 * (333 * 2 * planes + 8)


# ---------------------------------------------------------------- device
class Layer:
    def __init__(self, m: ll.MoE, rows, seed=1, router_scale=2.0, pad_x=0, pad_y=0, shift=0):
        import torch

        self.m, self.rows, self.torch = m, rows, torch
        e, h, f = m.n_experts, m.hidden, m.inter
        self.ldx, self.ldy = h + pad_x, h + pad_y
        x = ll.fill_normal(rows * h, 0.0, 1.0, seed).reshape(rows, h)
        xb = torch.full((shift + rows * self.ldx,), 5.0, device="cuda", dtype=t_dtype(m.x_type))
        self.xv = xb[shift:].view(rows, self.ldx)
        self.xv[:, :h] = dev(x).to(t_dtype(m.x_type))
        self.x = self.xv[:, :h].double().cpu().numpy()
        r = ll.fill_normal(e * h, 0.0, router_scale * h ** -0.5, seed + 1).reshape(e, h)
        self.d = {"router": dev(r).to(t_dtype(m.router_type))}
        self.r = self.d["router"].double().cpu().numpy()
        self.w = {}
        for i, (name, a, b) in enumerate((("gate", f, h), ("up", f, h), ("down", h, f))):
            if name == "up" and not m.gated:
                continue
            mats = [ll.fill_normal(a * b, 0.0, b ** -0.5, seed + 10 + 3 * j + i).reshape(a, b) for j in range(e)]
            if m.wtype == ll.W_BF16:
                t = dev(np.stack(mats)).to(torch.bfloat16)
                self.d[name], self.w[name] = t, t.double().cpu().numpy()
            elif m.wtype == ll.W_I8:
                q, s = zip(*[ll.quantize_int8_rows(v) for v in mats])
                self.d[name], self.d[name + "_scale"] = dev(np.stack(q)), dev(np.stack(s))
                self.w[name] = np.stack(q).astype(np.float64) * np.stack(s).astype(np.float64)[:, :, None]
            else:
                q, s = zip(*[ll.quantize_fp8_blocks(v) for v in mats])
                self.d[name], self.d[name + "_scale"] = dev(np.stack(q)), dev(np.stack(s))
                self.w[name] = np.stack([dequant_blocks(*v) for v in zip(q, s)])
        self.weights = ll.MoEWeights(**{n: self.d[n].data_ptr() if n in self.d else 0
                                        for n in ("router", "gate", "up", "down", "gate_scale", "up_scale",
                                                  "down_scale")})
        self.buffers()

    def buffers(self):
        t = self.torch
        n = ll.moe_workspace_bytes(self.m, self.rows)
        self.work = t.full((n,), 0xFF, dtype=t.uint8, device="cuda")  # NaN wherever it is read unwritten
        self.y = t.full((self.rows + 1, self.ldy), 99.0, device="cuda", dtype=t_dtype(self.m.x_type))
        self.ids = t.full((self.rows, self.m.top_k), -1, dtype=t.int32, device="cuda")
        self.probs = t.full((self.rows, self.m.top_k), -1.0, device="cuda")

    def run(self, stream=None):
        st = (stream or self.torch.cuda.current_stream()).cuda_stream
        ll.moe_forward(self.m, self.weights, self.xv.data_ptr(), self.y.data_ptr(), self.rows, self.work.data_ptr(),
                       self.work.numel(), ids_ptr=self.ids.data_ptr(), probs_ptr=self.probs.data_ptr(), ldx=self.ldx,
                       ldy=self.ldy, stream=st)

    def check(self):
        m, x = self.m, self.x
        ns = {ll.T_BF16: 1, ll.T_F16: 2, ll.T_F32: 3}[m.x_type]
        ids, probs = self.ids.cpu().numpy(), self.probs.double().cpu().numpy()
        h, f, k = m.hidden, m.inter, m.top_k
        got = self.y.double().cpu().numpy()
        assert np.all(got[self.rows:] == 99) and np.all(got[:, h:] == 99)
        logits = x @ self.r.T
        tl = (np.abs(x) @ np.abs(self.r).T) * (3 * ns * h + 40) * U
        for i in range(self.rows):
            order = ids[i]
            assert len(set(order)) == k and order.min() >= 0 and order.max() < m.n_experts
            t = 2 * tl[i].max()
            l = logits[i]
            rest = np.delete(l, order)
            assert np.all(np.diff(l[order]) <= t) and (rest.size == 0 or rest.max() <= l[order].min() + t)
            p = np.exp(l - l.max())
            p /= p.sum()
            w = p[order] / (p[order].sum() if m.renormalize else 1.0)
            assert np.all(np.abs(probs[i] - w) <= w * (np.expm1(2 * t) + 2.0 ** -19))
            y, tol = np.zeros(h), np.zeros(h)
            for j, e in enumerate(order):
                g = x[i] @ self.w["gate"][e].T
                tg = (np.abs(x[i]) @ np.abs(self.w["gate"][e]).T) * (ns * h + 40) * U
                a = act64(g, m.act)
                ta = 1.13 * tg + 2.0 ** -20 * np.abs(g)
                if m.gated:
                    u = x[i] @ self.w["up"][e].T
                    tu = (np.abs(x[i]) @ np.abs(self.w["up"][e]).T) * (ns * h + 40) * U
                    ta = ta * (np.abs(u) + tu) + np.abs(a) * tu
                    a = a * u
                    ta = ta + np.abs(a) * U
                ta = ta + np.abs(a) * (2.0 ** -22 if m.x_type == ll.T_F32 else 2.0 ** -16)
                d = np.abs(self.w["down"][e])
                nsh = 3 if m.x_type == ll.T_F32 else 2
                y += w[j] * (self.w["down"][e] @ a)
                tol += w[j] * (d @ ta + (d @ (np.abs(a) + ta)) * ((nsh * f + 40) * U + np.expm1(2 * t) + 2.0 ** -19))
            tol = tol * 1.01 + np.abs(y) * ROUND[m.x_type] + 2.0 ** -25
            worst = np.max(np.abs(got[i, :h] - y) - tol)
            assert worst <= 0, (i, worst)


CASES = [
    # rows, hidden, inter, experts, top_k, gated, renorm, act, router_type, pads
    (1, 64, 64, 1, 1, True, True, ll.ACT_SILU, ll.T_BF16, 0),
    (1, 256, 128, 8, 2, True, True, ll.ACT_SILU, ll.T_BF16, 0),
    (1, 2048, 512, 16, 8, True, False, ll.ACT_SILU, ll.T_F32, 0),
    (2, 100, 36, 5, 3, False, False, ll.ACT_GELU, ll.T_BF16, 4),
    (3, 129, 65, 7, 7, True, True, ll.ACT_RELU, ll.T_F32, 1),
    (7, 1000, 344, 10, 3, False, True, ll.ACT_GELU, ll.T_BF16, 0),
    (8, 640, 1032, 20, 4, True, True, ll.ACT_SILU, ll.T_BF16, 8),
    (9, 512, 256, 2, 1, True, True, ll.ACT_IDENTITY, ll.T_BF16, 0),
    (16, 257, 129, 33, 16, False, False, ll.ACT_SILU, ll.T_BF16, 3),
    (32, 384, 200, 40, 8, True, True, ll.ACT_SILU, ll.T_F32, 0),
    (32, 64, 16, 256, 2, True, True, ll.ACT_SILU, ll.T_BF16, 0),
    (31, 1040, 528, 3, 3, True, True, ll.ACT_GELU, ll.T_BF16, 0),
]


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("wtype", [ll.W_BF16, ll.W_I8, ll.W_F8])
@pytest.mark.parametrize("x_type", [ll.T_BF16, ll.T_F16, ll.T_F32])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_moe(wtype, x_type, case):
    rows, h, f, e, k, gated, renorm, act, rt, pad = CASES[case]
    m = ll.MoE(h, f, e, k, act, gated, wtype, x_type, rt, renorm)
    layer = Layer(m, rows, seed=case + 1, pad_x=pad, pad_y=2 * pad, shift=pad % 2)
    layer.run()
    ll.ops_check()
    layer.check()


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("wtype,x_type", [(ll.W_BF16, ll.T_BF16), (ll.W_F8, ll.T_F32), (ll.W_I8, ll.T_F16)])
@pytest.mark.parametrize("rows,hidden,inter,experts,top_k,gated", [
    (8, 4096, 72, 4, 2, True),     # few rows whose x fits no shared memory
    (2, 72, 9000, 3, 3, True),     # nor their activations
    (1, 48, 24, 256, 16, False),   # one row, the most experts and picks
    (1, 65536, 8, 2, 1, True),     # the widest rows
    (1, 8, 65536, 2, 2, False),
    (1, 1, 1, 1, 1, True),
    (32, 1, 1, 3, 2, False),
])
def test_borders(wtype, x_type, rows, hidden, inter, experts, top_k, gated):
    layer = Layer(ll.MoE(hidden, inter, experts, top_k, gated=gated, wtype=wtype, x_type=x_type), rows, seed=3)
    layer.run()
    ll.ops_check()
    layer.check()


@pytest.mark.gpu
@pytest.mark.timeout(300)
def test_ties_go_to_the_lower_index():
    m = ll.MoE(128, 64, 12, 5)
    layer = Layer(m, 4)
    layer.d["router"][:] = layer.d["router"][0]
    layer.d["router"][9] += layer.d["router"][0]  # twice the others' logit: first or last
    layer.run()
    ids = layer.ids.cpu().numpy()
    l = layer.x @ layer.r[0]
    for i in range(4):
        assert ids[i].tolist() == ([9, 0, 1, 2, 3] if l[i] > 0 else [0, 1, 2, 3, 4])
    assert np.all(np.isfinite(layer.y.float().cpu().numpy()))


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("wtype", [ll.W_BF16, ll.W_F8])
def test_special_values_stay_in_their_rows(wtype):
    m = ll.MoE(256, 128, 8, 2, wtype=wtype)
    clean, layer = Layer(m, 6), Layer(m, 6)
    clean.run()
    layer.xv[2, 7] = float("nan")
    layer.xv[4, 9] = float("inf")
    layer.run()
    ll.ops_check()
    y, want = layer.y.float().cpu().numpy()[:6], clean.y.float().cpu().numpy()[:6]
    assert np.isnan(y[2]).all() and not np.isfinite(y[4]).any()
    keep = [0, 1, 3, 5]
    assert np.array_equal(y[keep], want[keep])  # and the others do not move by a bit
    ids = layer.ids.cpu().numpy()
    assert ids.min() >= 0 and ids.max() < 8 and all(len(set(r)) == 2 for r in ids)


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows", [1, 12])
def test_nan_weights_of_an_expert_reach_the_rows_that_picked_it(rows):
    m = ll.MoE(256, 384, 4, 1, wtype=ll.W_F8)
    layer = Layer(m, rows, router_scale=8.0)
    layer.run()
    ids = layer.ids.cpu().numpy()[:, 0]
    clean = layer.y.float().cpu().numpy()[:rows]
    e = int(ids[0])
    layer.d["down"][e, 33, 200] = 0xFF  # one output channel
    layer.run()
    y = layer.y.float().cpu().numpy()[:rows]
    hit = np.zeros_like(y, bool)
    hit[ids == e, 33] = True
    assert np.isnan(y[hit]).all() and np.array_equal(y[~hit], clean[~hit])
    layer.d["gate"][e, 70, 5] = 0x7F    # one activation, so every output channel
    layer.run()
    y = layer.y.float().cpu().numpy()[:rows]
    assert np.isnan(y[ids == e]).all() and np.array_equal(y[ids != e], clean[ids != e])


@pytest.mark.gpu
@pytest.mark.timeout(300)
def test_every_e4m3_code_counts_exactly():
    # gate weights that run through all codes, subnormal ones too, against a one-hot x: the activation is the
    # weight itself; down is the identity, so y is the code's value times the scales
    import torch

    h = f = 256
    m = ll.MoE(h, f, 1, 1, act=ll.ACT_IDENTITY, gated=False, wtype=ll.W_F8, x_type=ll.T_F32)
    layer = Layer(m, 2)
    codes = np.arange(256, dtype=np.uint8)
    codes[[0x7F, 0xFF]] = 0
    gate = np.zeros((1, f, h), np.uint8)
    gate[0, :, 3], gate[0, :, 200] = codes, codes
    down = np.zeros((1, h, f), np.uint8)
    down[0, np.arange(h), np.arange(f)] = 0x38  # 1
    layer.d["gate"].copy_(dev(gate))
    layer.d["down"].copy_(dev(down))
    layer.d["gate_scale"].fill_(0.5)
    layer.d["down_scale"].fill_(2.0)
    layer.xv.zero_()
    layer.xv[0, 3] = 1.0
    layer.xv[1, 200] = 1.0
    layer.run()
    y = layer.y.cpu().numpy()[:2]
    assert np.array_equal(y[0], decode(codes).astype(np.float32)) and np.array_equal(y[1], y[0])


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows", [1, 20])
def test_repeats_bit_for_bit_on_streams_and_in_graphs(rows):
    import torch

    m = ll.MoE(512, 320, 16, 4, wtype=ll.W_F8)
    a, b = Layer(m, rows, seed=2), Layer(m, rows, seed=50)
    a.run(), b.run()
    torch.cuda.synchronize()
    ya, yb = a.y.clone(), b.y.clone()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):  # two calls at once, each with its own workspace
        a.run(s1), b.run(s2)
    torch.cuda.synchronize()
    assert torch.equal(a.y, ya) and torch.equal(b.y, yb)
    for _ in range(10):  # one after another through one workspace
        b.work = a.work
        a.run(), b.run()
    assert torch.equal(a.y, ya) and torch.equal(b.y, yb)
    b.buffers()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        a.run()
    with torch.cuda.graph(gb):
        b.run()
        b.run()
    for _ in range(5):
        a.y.zero_(), b.y.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            ga.replay()
        with torch.cuda.stream(s2):
            gb.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.y[:rows], ya[:rows]) and torch.equal(b.y[:rows], yb[:rows])
    a.xv.copy_(b.xv)  # a replay reads x anew: other experts
    ga.replay()
    torch.cuda.synchronize()
    a.x = b.x
    a.y[rows:] = 99
    a.check()
    ll.ops_check()


@pytest.mark.gpu
@pytest.mark.timeout(300)
def test_refuses_memory_of_the_host():
    import torch

    layer = Layer(ll.MoE(64, 32, 4, 2), 2)
    host = torch.zeros(2, 64, dtype=torch.bfloat16)
    a = (layer.m, layer.weights, layer.xv.data_ptr(), layer.y.data_ptr(), 2, layer.work.data_ptr(), layer.work.numel())
    for i in (2, 3, 5):
        args = list(a)
        args[i] = host.data_ptr() // 256 * 256
        assert "current device" in refused(ll.moe_forward, ll.LL_ERR_INVALID_ARG, *args)
    args = list(a)
    args[5] += 16
    assert "aligned" in refused(ll.moe_forward, ll.LL_ERR_INVALID_ARG, *args)


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows", [1, 6, 32])
def test_a_layer_of_experts_and_an_output_layer(rows):
    """moe (e4m3 experts) -> quantise -> dense (e4m3): each step against 64 bits on the device's own input."""
    import torch

    m = ll.MoE(384, 256, 12, 3, wtype=ll.W_F8, x_type=ll.T_BF16)
    layer = Layer(m, rows, seed=5)
    W = ll.fill_normal(96 * 384, 0.0, 384 ** -0.5, 77).reshape(96, 384)
    wq, sw = ll.quantize_fp8_blocks(W)
    dw, dsw = dev(wq), dev(sw)
    q = torch.zeros(rows, 384, dtype=torch.uint8, device="cuda")
    s = torch.zeros(rows, 3, device="cuda")
    out = torch.zeros(rows, 96, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    layer.run()
    ll.quantize_fp8(layer.y.data_ptr(), ll.T_BF16, rows, 384, q.data_ptr(), s.data_ptr(), ldx=layer.ldy, stream=st)
    ll.dense_fp8(dw.data_ptr(), dsw.data_ptr(), 0, q.data_ptr(), s.data_ptr(), out.data_ptr(), rows, 96, 384, stream=st)
    ll.ops_check(st)
    layer.check()
    qn, sn = quantize_rows(layer.y[:rows].float().cpu().numpy())
    assert np.array_equal(decode(q.cpu().numpy()), decode(qn)) and np.array_equal(s.cpu().numpy(), sn)
    x, w = dequant_rows(qn, sn), dequant_blocks(wq, sw)
    tol = (np.abs(x) @ np.abs(w).T) * (128 + 3 + 11) * U
    assert np.all(np.abs(out.cpu().numpy() - x @ w.T) <= tol)


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows,wtype,x_type", [(1, ll.W_BF16, ll.T_BF16), (4, ll.W_F8, ll.T_F16), (32, ll.W_I8, ll.T_F32)])
def test_layers_in_a_row_write_over_their_input(rows, wtype, x_type):
    """A chain of layers, each with y = x and one workspace: a launch that sets itself up beside the one before
    it reads what that one wrote, eager and captured (the same results as with a synchronise after each)."""
    import torch

    m = ll.MoE(256, 128, 16, 2, wtype=wtype, x_type=x_type)
    layers = [Layer(m, rows, seed=20 + 40 * i) for i in range(3)]
    x = layers[0].xv
    first = x.clone()
    for l in layers:
        l.xv, l.y, l.work = x, x, layers[0].work

    def chain(wait):
        x.copy_(first)
        seen = []
        for _ in range(2):
            for l in layers:
                l.run()
                if wait:
                    torch.cuda.synchronize()
                seen.append((l.ids.clone(), x.clone()))
        return seen

    want = chain(True)
    assert torch.isfinite(x).all() and not torch.equal(x, first)
    for _ in range(5):
        for a, b in zip(want, chain(False)):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x.copy_(first)
        for _ in range(2):
            for l in layers:
                l.run()
    for _ in range(5):
        g.replay()
        assert torch.equal(x, want[-1][1])
    ll.ops_check()


def test_the_limit_of_waits_is_bounded():
    refused(ll.ops_set_wait_limit, ll.LL_ERR_INVALID_ARG, 60_000_000_001)
    ll.ops_set_wait_limit()


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows,hidden,inter,experts,top_k,wtype,x_type", [
    (1, 256, 128, 8, 2, ll.W_BF16, ll.T_BF16),     # bulk copies in both kernels: the up kernel's first wait gives up
    (1, 1024, 512, 8, 2, ll.W_F8, ll.T_BF16),
    (3, 512, 96, 4, 2, ll.W_I8, ll.T_F32),
    (32, 384, 512, 40, 8, ll.W_BF16, ll.T_F16),    # in the down kernel alone
])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(rows, hidden, inter, experts, top_k, wtype, x_type):
    # with a limit of 0 every wait gives up with its copies in flight: they land before the kernel ends, the
    # status says so, and the calls behind it on the same stream are as ever
    import torch

    layer = Layer(ll.MoE(hidden, inter, experts, top_k, wtype=wtype, x_type=x_type), rows, seed=5)
    layer.run()
    ll.ops_check()
    layer.check()
    want = layer.y.clone()
    for _ in range(3):
        ll.ops_set_wait_limit(0)
        try:
            layer.run()
        finally:
            ll.ops_set_wait_limit()
        layer.run()
        with pytest.raises(ll.LLError) as e:
            ll.ops_check()
        assert e.value.code == ll.LL_ERR_DEVICE_FAULT
        assert torch.equal(layer.y, want)
        ll.ops_check()


@pytest.mark.gpu
@pytest.mark.timeout(300)
def test_rows_that_start_on_no_16_bytes_wait_for_no_barrier():
    layer = Layer(ll.MoE(129, 65, 7, 3, x_type=ll.T_F32), 3, seed=6)
    ll.ops_set_wait_limit(0)
    try:
        layer.run()
    finally:
        ll.ops_set_wait_limit()
    ll.ops_check()
    layer.check()


def within_relative_bounds(layer):
    """Run a layer of one expert (so that its weight is 1): the bounds of the module's head, relative to the sums of
    magnitudes, without its absolute share."""
    layer.x = layer.xv[:, :layer.m.hidden].double().cpu().numpy()
    layer.run()
    ll.ops_check()
    m, rows, x_type, act = layer.m, layer.rows, layer.m.x_type, layer.m.act
    h, f, gated = m.hidden, m.inter, m.gated
    ns, nsh = (3, 3) if x_type == ll.T_F32 else (1, 2)
    w = {n: layer.w[n][0] for n in layer.w}
    x = layer.x
    g, tg = x @ w["gate"].T, (np.abs(x) @ np.abs(w["gate"]).T) * (ns * h + 40) * U
    a, ta = act64(g, act), 1.13 * tg + 2.0 ** -20 * np.abs(g)
    if gated:
        u, tu = x @ w["up"].T, (np.abs(x) @ np.abs(w["up"]).T) * (ns * h + 40) * U
        ta = ta * (np.abs(u) + tu) + np.abs(a) * tu
        a = a * u
        ta = ta + np.abs(a) * U
    ta = ta + np.abs(a) * (2.0 ** -22 if nsh == 3 else 2.0 ** -16)
    d = np.abs(w["down"])
    y = a @ w["down"].T
    tol = ta @ d.T + ((np.abs(a) + ta) @ d.T) * ((nsh * f + 40) * U + 2.0 ** -19)
    tol = tol * 1.01 + np.abs(y) * ROUND[x_type]
    off = np.abs(layer.y[:rows].double().cpu().numpy() - y)
    assert np.all(off <= tol), np.max(off / tol)


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("wtype", [ll.W_F8, ll.W_I8])
@pytest.mark.parametrize("x_type", [ll.T_F32, ll.T_BF16])
@pytest.mark.parametrize("rows", [1, 12])
@pytest.mark.parametrize("scale,gated", [(1e-8, True), (2.0 ** -36, True), (2.0 ** -75, False), (2.0 ** 60, False)])
def test_small_and_large_values_keep_their_digits(wtype, x_type, rows, scale, gated):
    # x of 1e-8 makes activations of 2^-54 through a gate and SiLU, of 2^-36 some 2^-72
    h, f = 384, 256
    act = ll.ACT_SILU if gated else ll.ACT_RELU
    layer = Layer(ll.MoE(h, f, 1, 1, act, gated, wtype, x_type, ll.T_BF16), rows, seed=71)
    layer.xv[:, :h] *= scale
    within_relative_bounds(layer)


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows", [1, 9])
def test_the_largest_fp32_values_are_finite(rows):
    # above the largest bf16 number, which the first of their three terms must not exceed
    layer = Layer(ll.MoE(128, 96, 1, 1, ll.ACT_RELU, False, ll.W_BF16, ll.T_F32, ll.T_BF16), rows, seed=81)
    layer.xv.zero_()
    for i in range(rows):
        layer.xv[i, 7 * i] = 3.4e38 if i % 2 else -3.402e38
    within_relative_bounds(layer)


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("wtype", [ll.W_BF16, ll.W_F8])
@pytest.mark.parametrize("rows", [3, 12])
def test_infinities_and_nan_of_fp32_rows_stay_in_their_rows(wtype, rows):
    m = ll.MoE(256, 128, 8, 2, wtype=wtype, x_type=ll.T_F32)
    clean, layer = Layer(m, rows), Layer(m, rows)
    clean.run()
    layer.xv[0, 7] = float("inf")
    layer.xv[2, 9] = float("nan")
    layer.run()
    ll.ops_check()
    y, want = layer.y.cpu().numpy()[:rows], clean.y.cpu().numpy()[:rows]
    assert not np.isfinite(y[[0, 2]]).any()
    keep = np.delete(np.arange(rows), [0, 2])
    assert np.array_equal(y[keep], want[keep])
