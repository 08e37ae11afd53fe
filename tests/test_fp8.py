"""The e4m3 block format: ll_quantize_fp8_blocks (host), ll_quantize_fp8 and ll_dense_fp8 (B200).

The plain implementation is numpy in 64 bits.  Quantised bytes are compared exactly: the
definition (scale = fl32(max / 448), value nearest to x / scale, ties to even) leaves no choice.

Tolerance of the dense layer, per output, from A = sum_k |x_k| |w_k| (dequantised):
  * e4m3 products are exact in fp32; a 128-column block is at most 128 fp32 additions, each off
    by at most one unit 2^-23 of a partial sum <= A;
  * per block the product of the two scales and the fused add are off by 2^-24 each, and the
    sums of at most 8 splits and the bias add another 9: nkb + 11 in units of 2^-23 covers them.
  So |sum - exact| <= A (128 + nkb + 11) 2^-23 (plus the bias' share).  An activation's slope is
  at most 1.13 (gelu) and its own evaluation is good to 2^-20 of max(|v|, result); the result's
  rounding is half a step: 2^-8 bf16, 2^-11 fp16, and for e4m3 2^-4 of the value, or half a step
  of the lowest octave, 2^-10 scales.
"""
import ctypes

import numpy as np
import pytest

import low_latency_inference_gpu_b200 as ll

F8 = ll.F8_BLOCK


def up(n, m):
    return -(-n // m) * m


def e4m3_values():
    """The 127 values of codes 0x00 .. 0x7e."""
    out = np.empty(127)
    for c in range(127):
        e, m = c >> 3, c & 7
        out[c] = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
    return out


TABLE = e4m3_values()


def decode(q):
    q = np.asarray(q, np.uint8)
    mag = np.append(TABLE, np.nan)[q & 0x7F]
    return np.where(q & 0x80, -mag, mag)


def nearest_code(t):
    """Code of the e4m3 value nearest to t (float64), ties to the even code; NaN to 0x7f."""
    a = np.minimum(np.abs(np.nan_to_num(t, nan=0.0, posinf=np.inf, neginf=-np.inf)), 448.0)
    hi = np.clip(np.searchsorted(TABLE, a), 1, 126)
    lo = hi - 1
    d, u = a - TABLE[lo], TABLE[hi] - a
    code = np.where(d < u, lo, np.where(u < d, hi, lo + lo % 2)).astype(np.uint8)
    code = code | np.where(np.signbit(t), 0x80, 0).astype(np.uint8)
    return np.where(np.isnan(t), 0x7F, code).astype(np.uint8)


def quantize_rows(x, pow2=False):
    """(codes [r][d], scales [r][g]) by the definition, x float32."""
    x = np.asarray(x, np.float32)
    r, d = x.shape
    g = -(-d // F8)
    q, s = np.empty((r, d), np.uint8), np.empty((r, g), np.float32)
    for j in range(g):
        c = x[:, j * F8:(j + 1) * F8].astype(np.float64)
        amax = np.nanmax(np.where(np.isnan(c), 0.0, np.abs(c)), axis=1)
        sc = np.where(amax > 0, np.maximum((amax.astype(np.float32) / np.float32(448.0)).astype(np.float32),
                                           np.float32(2.0 ** -126)), np.float32(0)).astype(np.float32)
        if pow2:
            sc = np.where(amax > 0, 2.0 ** np.ceil(np.log2(np.where(sc > 0, sc, 1).astype(np.float64))), 0.0)
            sc = sc.astype(np.float32)
        s[:, j] = sc
        div = np.where(sc > 0, sc, 1).astype(np.float64)[:, None]
        with np.errstate(invalid="ignore"):
            q[:, j * F8:(j + 1) * F8] = nearest_code(c / div)
    return q, s


def dequant_rows(q, s):
    return decode(q) * np.repeat(s.astype(np.float64), F8, 1)[:, :q.shape[1]]


def dequant_blocks(q, s):
    return decode(q) * np.repeat(np.repeat(s.astype(np.float64), F8, 0), F8, 1)[:q.shape[0], :q.shape[1]]


# ---------------------------------------------------------------- host
@pytest.mark.parametrize("m,k", [(1, 1), (128, 128), (130, 257), (64, 1000), (300, 96)])
def test_quantize_blocks_on_the_host(m, k):
    W = ll.fill_normal(m * k, 0.0, 0.05, 3).reshape(m, k)
    W[: m // 3] = 0.0
    q, s = ll.quantize_fp8_blocks(W)
    assert s.shape == (-(-m // F8), -(-k // F8))
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            blk = (slice(i * F8, (i + 1) * F8), slice(j * F8, (j + 1) * F8))
            amax = np.abs(W[blk]).max()
            want = np.float32(amax) / np.float32(448) if amax > 0 else np.float32(1)
            assert s[i, j] == want
            assert np.array_equal(q[blk], nearest_code(W[blk].astype(np.float64) / float(want)))


def test_e4m3_codes_on_the_host():
    # every value, every tie, every neighbour of a tie, both signs: one block whose scale is 1
    mids = (TABLE[:-1] + TABLE[1:]) / 2
    v = np.concatenate([TABLE, mids, mids * (1 + 2.0 ** -20), mids * (1 - 2.0 ** -20)]).astype(np.float32)
    v = np.concatenate([v, -v])
    for i in range(0, v.size, F8 - 1):
        row = np.zeros((1, F8), np.float32)
        part = v[i:i + F8 - 1]
        row[0, :part.size], row[0, -1] = part, 448.0
        q, s = ll.quantize_fp8_blocks(row)
        assert s[0, 0] == 1.0
        assert np.array_equal(q[0], nearest_code(row[0].astype(np.float64)))


def call_refused(fn, *args, **kw):
    with pytest.raises(ll.LLError) as e:
        fn(*args, **kw)
    assert e.value.code == ll.LL_ERR_INVALID_ARG
    return str(e.value)


def test_refusals_before_any_device_is_touched():
    q = dict(x_ptr=16, x_type=ll.T_BF16, rows=1, dim=64, q_ptr=16, s_ptr=16)
    for bad in (dict(x_type=ll.T_F8), dict(rows=-1), dict(dim=0), dict(ldx=63), dict(ldq=63), dict(x_ptr=0),
                dict(q_ptr=0), dict(s_ptr=0), dict(rows=2 ** 30, dim=300)):
        call_refused(ll.quantize_fp8, **{**q, **bad})
    d = dict(W_ptr=16, sw_ptr=16, b_ptr=0, x_ptr=16, sx_ptr=16, y_ptr=16, rows=1, M=64, K=64)
    for bad in (dict(rows=-1), dict(M=0), dict(K=0), dict(K=60), dict(ldw=72), dict(ldx=60), dict(ldy=60),
                dict(act=4), dict(act=-1), dict(y_type=4), dict(y_type=ll.T_F8), dict(W_ptr=0), dict(sw_ptr=0),
                dict(x_ptr=0), dict(sx_ptr=0), dict(y_ptr=0), dict(rows=65535 * 128 + 1)):
        call_refused(ll.dense_fp8, **{**d, **bad})
    ll.quantize_fp8(0, ll.T_F32, 0, 8, 0, 0)  # no rows: nothing to do
    ll.dense_fp8(0, 0, 0, 0, 0, 0, 0, 16, 16)


def test_other_paths_refuse_the_new_types():
    for wtype, act in ((ll.W_F8, ll.ACT_RELU), (ll.W_F32, ll.ACT_SILU)):
        with pytest.raises(ll.LLError):
            ll.plan_net(ll.Net([64, 64], [act], wtype, 1))
    with pytest.raises(ll.LLError):
        ll.batched_plan(ll.Net([64, 64], [ll.ACT_RELU], ll.W_F8, 1))
    with pytest.raises(ll.LLError):
        ll.batched_plan(ll.Net([64, 64], [ll.ACT_SILU], ll.W_BF16, 1))


# ---------------------------------------------------------------- device
gpu = [pytest.mark.gpu, pytest.mark.timeout(300)]


def dev(a, dtype=None):
    import torch

    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def t_dtype(t):
    import torch

    return {ll.T_F32: torch.float32, ll.T_BF16: torch.bfloat16, ll.T_F16: torch.float16, ll.T_F8: torch.uint8}[t]


def run_quantize(x, x_type, pow2=False, pad_x=0, pad_q=0, shift=0):
    """Quantise numpy x through the library; rows pad_x / pad_q wider, the first row `shift` elements in."""
    import torch

    r, d = x.shape
    ldx, ldq = d + pad_x, d + pad_q
    buf = torch.full((shift + r * ldx,), 7.0, device="cuda", dtype=t_dtype(x_type))
    view = buf[shift:].view(r, ldx)
    view[:, :d] = dev(x).to(t_dtype(x_type))
    q = torch.full((shift + r * ldq,), 0xAA, device="cuda", dtype=torch.uint8)
    s = torch.full((r, -(-d // F8)), -1.0, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    ll.quantize_fp8(view.data_ptr(), x_type, r, d, q.data_ptr() + shift, s.data_ptr(), ldx=ldx, ldq=ldq, pow2=pow2,
                    stream=st)
    qn = q.cpu().numpy()
    assert np.all(qn[:shift] == 0xAA)
    qn = qn[shift:].reshape(r, ldq)
    assert np.all(qn[:, d:] == 0xAA)  # nothing beside the rows is written
    return qn[:, :d], s.cpu().numpy(), view[:, :d].float().cpu().numpy()


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("x_type", [ll.T_F32, ll.T_BF16, ll.T_F16])
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("r,d,pad_x,pad_q,shift", [
    (1, 1, 0, 0, 0), (1, 128, 0, 0, 0), (3, 1000, 8, 8, 0), (5, 129, 0, 0, 0), (17, 257, 3, 5, 1), (2, 2048, 0, 0, 0),
    (333, 72, 0, 0, 0), (70, 640, 16, 0, 8)])
def test_quantize_rows(x_type, pow2, r, d, pad_x, pad_q, shift):
    x = ll.fill_normal(r * d, 0.0, 1.0, r + d).reshape(r, d)
    x *= np.exp2(np.arange(d) % 23 - 11).astype(np.float32)
    x[:: 4, : d // 2] = 0.0
    q, s, x = run_quantize(x, x_type, pow2, pad_x, pad_q, shift)
    want_q, want_s = quantize_rows(x, pow2)
    assert np.array_equal(s.view(np.uint32), want_s.view(np.uint32))
    assert np.array_equal(decode(q), decode(want_q))


@pytest.mark.gpu
@pytest.mark.timeout(300)
def test_quantize_ties_and_borders():
    # groups whose quotients are ties or next to one: v = mid * s rounded up, down and to nearest
    rng = np.random.RandomState(5)
    amax = np.exp2(rng.uniform(-20, 20, 400)).astype(np.float32)
    s = (amax / np.float32(448)).astype(np.float32)
    mids = (TABLE[:-1] + TABLE[1:]) / 2
    v = (mids[None, :] * s[:, None].astype(np.float64)).astype(np.float32)
    v = np.nextafter(v, (v * rng.choice([0.5, 1.0, 2.0], v.shape)).astype(np.float32))
    x = np.concatenate([v, amax[:, None], -amax[:, None]], 1)
    assert x.shape[1] == F8
    q, sc, x = run_quantize(x, ll.T_F32)
    want_q, want_s = quantize_rows(x)
    assert np.array_equal(sc, want_s)
    assert np.array_equal(q, want_q)


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("x_type", [ll.T_BF16, ll.T_F16])
def test_quantize_16_bit_ties(x_type):
    # 16-bit quotients are often ties up to the rounding of the scale: every significand against every
    # largest magnitude's (bf16), or a spread of them (fp16), over the octaves of e4m3 and below
    bits = 8 if x_type == ll.T_BF16 else 11
    sig = np.arange(2 ** (bits - 1), 2 ** bits)[:: 1 if bits == 8 else 8].astype(np.float64)
    rows = []
    for a in sig:
        v = (sig[None, :] * np.exp2(-np.arange(0, 20, 3))[:, None]).ravel()
        v = v[v <= a]
        for i in range(0, v.size, F8 - 1):
            g = np.zeros(F8)
            part = v[i:i + F8 - 1]
            g[:part.size], g[-1] = part * np.where(np.arange(part.size) % 2, -1, 1), a
            rows.append(g)
    x = (np.stack(rows) * np.exp2(1 - bits)).astype(np.float32)
    q, s, x = run_quantize(x, x_type)
    want_q, want_s = quantize_rows(x)
    assert np.array_equal(s, want_s)
    assert np.array_equal(decode(q), decode(want_q))


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("pow2", [False, True])
def test_quantize_special_values(pow2):
    x = np.ones((6, 256), np.float32)
    x[0, 3] = np.nan                       # stays in its place
    x[1, 5] = np.inf                       # its group stands for NaN
    x[2, :128] = np.nan
    x[3] = -0.0
    x[4, :128] = 1e-40                     # below every scale: zeros
    x[5, 7] = np.float32(3.4e38)
    q, s, _ = run_quantize(x, ll.T_F32, pow2)
    v = decode(q) * np.repeat(s.astype(np.float64), F8, 1)
    one = lambda t: abs(t - 1.0) <= 2.0 ** -24  # noqa: E731  (448 times the fp32 rounding of 1 / 448, half a step off)
    assert np.isnan(v[0, 3]) and np.isfinite(np.delete(v[0], 3)).all() and one(v[0, 4])
    assert np.isinf(s[1, 0]) and np.isnan(v[1, :128]).all() and np.isfinite(v[1, 128:]).all()
    assert np.isnan(v[2, :128]).all() and np.isfinite(v[2, 128:]).all()
    assert np.all(v[3] == 0) and np.all(s[3] == 0)
    assert np.all(np.abs(v[4, :128]) <= 1e-40 + 2.0 ** -126 * 2.0 ** -9) and one(v[4, 200])
    assert abs(v[5, 7] - 3.4e38) <= 3.4e38 * 2.0 ** -4


def act64(v, act):
    from math import erf

    if act == ll.ACT_RELU:
        return np.maximum(v, 0)
    if act == ll.ACT_GELU:
        return 0.5 * v * (1 + np.vectorize(erf)(v / np.sqrt(2.0)))
    if act == ll.ACT_SILU:
        return v / (1 + np.exp(-v))
    return v


class DenseCase:
    """Operands of one dense layer on the device, and its result in 64 bits with its tolerance."""

    def __init__(self, rows, M, K, bias=True, seed=1, pad=0):
        import torch

        x = ll.fill_normal(rows * K, 0.0, 1.0, seed).reshape(rows, K)
        x *= np.exp2(np.arange(K) // F8 % 5 - 2).astype(np.float32)  # scales that differ by block
        W = ll.fill_normal(M * K, 0.0, K ** -0.5, seed + 1).reshape(M, K)
        W *= np.exp2(np.arange(M) // F8 % 3).astype(np.float32)[:, None]
        self.rows, self.M, self.K = rows, M, K
        self.xq, self.sx = quantize_rows(x)
        self.wq, self.sw = ll.quantize_fp8_blocks(W)
        self.b = ll.fill_uniform(M, -1.0, 1.0, seed + 2) if bias else None
        self.ld = up(K, 16) + pad
        # NaN bytes behind column K: not used
        xp, wp = np.full((rows, self.ld), 0x7F, np.uint8), np.full((M, self.ld), 0x7F, np.uint8)
        xp[:, :K], wp[:, :K] = self.xq, self.wq
        self.d = {"x": dev(xp), "sx": dev(self.sx), "w": dev(wp), "sw": dev(self.sw),
                  "b": dev(self.b) if bias else None}
        self.torch = torch

    def reference(self, act):
        x, w = dequant_rows(self.xq, self.sx), dequant_blocks(self.wq, self.sw)
        b = self.b.astype(np.float64) if self.b is not None else 0.0
        v = x @ w.T + b
        nkb = -(-self.K // F8)
        tol = ((np.abs(x) @ np.abs(w).T) * (128 + nkb + 11) + np.abs(b)) * 2.0 ** -23
        y = act64(v, act)
        if act != ll.ACT_IDENTITY:
            tol = 1.13 * tol + 2.0 ** -20 * np.maximum(np.abs(v), np.abs(y))
        return y, tol

    def run(self, act, y_type, pad_y=0, stream=None, y=None, sy=None):
        t, d = self.torch, self.d
        ldy = self.M + pad_y
        if y is None:
            y = t.full((self.rows + 1, ldy), 99 if y_type == ll.T_F8 else 99.0, device="cuda", dtype=t_dtype(y_type))
            sy = t.full((self.rows, -(-self.M // F8)), -1.0, device="cuda")
        st = (stream or t.cuda.current_stream()).cuda_stream
        ll.dense_fp8(d["w"].data_ptr(), d["sw"].data_ptr(), d["b"].data_ptr() if d["b"] is not None else 0,
                     d["x"].data_ptr(), d["sx"].data_ptr(), y.data_ptr(), self.rows, self.M, self.K, act=act,
                     y_type=y_type, sy_ptr=sy.data_ptr() if y_type == ll.T_F8 else 0, ldw=self.ld, ldx=self.ld,
                     ldy=ldy, stream=st)
        return y, sy

    def check(self, act, y_type, y, sy):
        ref, tol = self.reference(act)
        got = y.cpu().numpy() if y_type in (ll.T_F8, ll.T_F32) else y.float().cpu().numpy()
        # rows behind the last and columns behind M are left as they were
        assert np.all(got[self.rows:] == 99) and np.all(got[:self.rows, self.M:] == 99)
        got = got[:self.rows, :self.M]
        if y_type == ll.T_F8:
            s = sy.cpu().numpy()
            amax = np.stack([np.abs(ref[:, j:j + F8]).max(1) for j in range(0, self.M, F8)], 1)
            tmax = np.stack([tol[:, j:j + F8].max(1) for j in range(0, self.M, F8)], 1)
            assert np.all(np.abs(s * 448.0 - amax) <= tmax + amax * 2.0 ** -22)
            tol = tol * (1 + 2.0 ** -3) + np.abs(ref) * 2.0 ** -4 + np.repeat(s, F8, 1)[:, :self.M] * 2.0 ** -10
            got = dequant_rows(got, s)
        elif y_type != ll.T_F32:
            tol = tol * 1.01 + np.abs(ref) * (2.0 ** -8 if y_type == ll.T_BF16 else 2.0 ** -11) + 2.0 ** -25
        worst = np.max(np.abs(got - ref) - tol)
        assert worst <= 0, (worst, np.max(np.abs(got - ref)))


SHAPES = [(1, 16, 16), (1, 2048, 2048), (2, 128, 128), (7, 130, 260), (16, 64, 1000), (17, 200, 129), (32, 512, 4096),
          (33, 128, 640), (64, 384, 256), (65, 1000, 1100), (128, 257, 300), (129, 256, 512), (300, 520, 400),
          (256, 2048, 2048), (640, 1280, 384),
          # enough tiles of 256 x 256 for the many-row kernel: whole ones, ragged ones, one K block and several
          (1300, 1700, 200), (1280, 2048, 128), (2500, 1030, 700), (9601, 130, 1300)]


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows,M,K", SHAPES)
@pytest.mark.parametrize("y_type", [ll.T_F32, ll.T_BF16, ll.T_F16, ll.T_F8])
def test_dense(rows, M, K, y_type):
    act = [ll.ACT_IDENTITY, ll.ACT_RELU, ll.ACT_GELU, ll.ACT_SILU][(rows + M + y_type) % 4]
    c = DenseCase(rows, M, K, bias=(rows + K) % 3 != 0, seed=rows + M, pad=16 * (rows % 2))
    y, sy = c.run(act, y_type, pad_y=rows % 5)
    ll.ops_check()
    c.check(act, y_type, y, sy)


@pytest.mark.gpu
@pytest.mark.timeout(300)
def test_dense_special_values():
    c = DenseCase(20, 256, 384, bias=False)
    c.d["x"][3, 5] = 0x7F                       # NaN: its row
    c.d["x"][4, :] = 0
    c.d["sx"][6, 1] = float("inf")              # a scale: its row
    c.d["w"][200, 17] = 0x7F                    # NaN: its channel
    y, _ = c.run(ll.ACT_IDENTITY, ll.T_F32)
    y = y.cpu().numpy()[:20]
    bad = np.isnan(y)
    assert bad[3].all() and bad[:, 200].all()
    assert not np.isfinite(y[6]).any()
    rest = np.delete(np.delete(y, [3, 6], 0), 200, 1)
    assert np.isfinite(rest).all() and np.all(np.delete(y[4], 200) == 0)


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("act", [ll.ACT_GELU, ll.ACT_SILU, ll.ACT_RELU])
@pytest.mark.parametrize("y_type", [ll.T_F32, ll.T_BF16, ll.T_F16, ll.T_F8])
def test_dense_many_rows_every_activation(act, y_type):
    c = DenseCase(1290, 2048, 384, seed=31)
    y, sy = c.run(act, y_type)
    ll.ops_check()
    c.check(act, y_type, y, sy)


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("act", [ll.ACT_IDENTITY, ll.ACT_GELU])
@pytest.mark.parametrize("y_type", [ll.T_F32, ll.T_BF16])
def test_dense_many_rows_special_values(act, y_type):
    c = DenseCase(1290, 2048, 384, seed=32)
    plain, _ = c.run(act, y_type)
    plain = plain.float().cpu().numpy()[:1290]
    c.d["x"][3, 5] = 0x7F                       # NaN: its row
    c.d["sx"][700, 1] = float("nan")            # a scale: its row
    c.d["w"][2000, 17] = 0x7F                   # NaN: its channel
    y, _ = c.run(act, y_type)
    y = y.float().cpu().numpy()[:1290]
    assert np.isnan(y[[3, 700]]).all() and np.isnan(y[:, 2000]).all()
    rows, cols = np.delete(np.arange(1290), [3, 700]), np.delete(np.arange(2048), 2000)
    assert np.array_equal(y[np.ix_(rows, cols)], plain[np.ix_(rows, cols)])
    ll.ops_check()


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows", [1, 40, 700, 3500])
def test_dense_repeats_bit_for_bit_on_streams_and_in_graphs(rows):
    import torch

    a, b = DenseCase(rows, 700, 900, seed=3), DenseCase(rows, 700, 900, seed=4)
    ya, _ = a.run(ll.ACT_GELU, ll.T_F32)
    yb, _ = b.run(ll.ACT_GELU, ll.T_F32)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [(a.run(ll.ACT_GELU, ll.T_F32, stream=s1)[0], b.run(ll.ACT_GELU, ll.T_F32, stream=s2)[0])
            for _ in range(8)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, ya) and torch.equal(y, yb) for x, y in outs)
    y, sy = torch.empty_like(ya), None
    y.fill_(99.0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.run(ll.ACT_GELU, ll.T_F32, y=y, sy=torch.empty(1, device="cuda"))
    for _ in range(3):
        y[:rows].zero_()
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ya)
    a.d["x"].copy_(b.d["x"])  # a replay reads the buffers anew
    for name in ("sx", "w", "sw", "b"):
        a.d[name].copy_(b.d[name])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, yb)
    ll.ops_check()


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows", [2, 3500])
def test_dense_behind_copies_and_other_launches(rows):
    # the few-row kernel sets itself up beside the launch before it: what that one writes is seen all the same,
    # behind a copy, a kernel of torch, the quantiser and another dense layer, eager and captured
    import torch

    c = DenseCase(rows, 384, 640, seed=9)
    want, _ = c.run(ll.ACT_IDENTITY, ll.T_F32)
    good = {k: c.d[k].clone() for k in ("x", "sx", "w", "sw", "b")}
    y, sy = want.clone(), torch.empty(1, device="cuda")
    other = DenseCase(5, 128, 256, seed=10)
    oy, _ = other.run(ll.ACT_IDENTITY, ll.T_F32)

    def sequence():
        for k in good:  # copies
            c.d[k].copy_(good[k])
        c.run(ll.ACT_IDENTITY, ll.T_F32, y=y, sy=sy)
        c.d["sx"].mul_(2.0)  # a kernel of torch
        c.run(ll.ACT_IDENTITY, ll.T_F32, y=y, sy=sy)
        c.d["sx"].mul_(0.5)
        other.run(ll.ACT_IDENTITY, ll.T_F32, y=oy, sy=sy)
        c.run(ll.ACT_IDENTITY, ll.T_F32, y=y, sy=sy)

    for _ in range(3):
        for k in ("x", "w", "sx"):
            c.d[k].zero_()
        y[:rows].fill_(-1.0)
        sequence()
        assert torch.equal(y[:rows], want[:rows])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sequence()
    for _ in range(3):
        for k in ("x", "w", "sx"):
            c.d[k].zero_()
        g.replay()
        assert torch.equal(y[:rows], want[:rows])
    ll.ops_check()


@pytest.mark.gpu
@pytest.mark.timeout(300)
def test_silu_in_the_launch_per_layer_kernels():
    M, K = 70, 96
    W = ll.fill_normal(M * K, 0.0, 0.2, 1).reshape(M, K)
    x, b = ll.fill_normal(K, 0.0, 1.0, 2), ll.fill_normal(M, 0.0, 1.0, 3)
    v = W.astype(np.float64) @ x + b
    tol = 1.1 * (np.abs(W) @ np.abs(x) + np.abs(b)) * (K + 2) * 2.0 ** -24 + np.abs(v) * 2.0 ** -20
    dW, dWc, db, dx = dev(W), dev(ll.pack_rm_to_kmajor_padded(W, 96)), dev(ll.pack_bias_padded(b, 96)), dev(x)
    for i in range(2):
        y = dev(np.zeros(M, np.float32))
        if i == 0:
            ll.dense_warp_rm(dW.data_ptr(), db.data_ptr(), dx.data_ptr(), y.data_ptr(), M, K, ll.ACT_SILU)
        else:
            ll.dense_mbyv_packed(dWc.data_ptr(), db.data_ptr(), dx.data_ptr(), y.data_ptr(), M, K, ll.ACT_SILU)
        assert np.all(np.abs(y.cpu().numpy() - v / (1 + np.exp(-v))) <= tol)


@pytest.mark.gpu
@pytest.mark.timeout(300)
def test_refuses_memory_of_the_host():
    import torch

    c = DenseCase(4, 64, 64)
    host = torch.empty(4, 64)
    args = dict(W_ptr=c.d["w"].data_ptr(), sw_ptr=c.d["sw"].data_ptr(), b_ptr=0, x_ptr=c.d["x"].data_ptr(),
                sx_ptr=c.d["sx"].data_ptr(), y_ptr=host.data_ptr(), rows=4, M=64, K=64)
    assert "current device" in call_refused(ll.dense_fp8, **args)
    out = torch.empty(8, 64, device="cuda")
    args["y_ptr"] = out.data_ptr()
    ll.dense_fp8(**args)
    assert "aligned" in call_refused(ll.dense_fp8, **{**args, "x_ptr": c.d["x"].data_ptr() + 4})
    x, q, s = torch.empty(4, 64), torch.empty(4, 64, dtype=torch.uint8, device="cuda"), torch.empty(4, device="cuda")
    assert "current device" in call_refused(ll.quantize_fp8, x.data_ptr(), ll.T_F32, 4, 64, q.data_ptr(), s.data_ptr())


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows", [1, 9, 160])
def test_an_e4m3_net_layer_after_layer(rows):
    """quantise -> dense (e4m3 out) -> dense (fp32 out), as a net of two layers is run, against the
    64-bit layers on the device's own quantised activations (each step has its own tolerance)."""
    import torch

    dims = [300, 512, 200]
    x = ll.fill_normal(rows * dims[0], 0.0, 1.0, 8).reshape(rows, dims[0])
    Ws = [ll.fill_normal(dims[i + 1] * dims[i], 0.0, dims[i] ** -0.5, 9 + i).reshape(dims[i + 1], dims[i])
          for i in range(2)]
    ld0 = up(dims[0], 16)
    dq = torch.zeros(rows, ld0, dtype=torch.uint8, device="cuda")
    ds = torch.zeros(rows, 3, device="cuda")
    dx = dev(x)
    qs = [ll.quantize_fp8_blocks(w) for w in Ws]
    w0 = np.zeros((dims[1], ld0), np.uint8)
    w0[:, :dims[0]] = qs[0][0]
    dw = [dev(w0), dev(qs[1][0])]
    dsw = [dev(q[1]) for q in qs]
    h = torch.zeros(rows, dims[1], dtype=torch.uint8, device="cuda")
    hs = torch.zeros(rows, 4, device="cuda")
    y = torch.zeros(rows, dims[2], device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    ll.quantize_fp8(dx.data_ptr(), ll.T_F32, rows, dims[0], dq.data_ptr(), ds.data_ptr(), ldq=ld0, stream=st)
    ll.dense_fp8(dw[0].data_ptr(), dsw[0].data_ptr(), 0, dq.data_ptr(), ds.data_ptr(), h.data_ptr(), rows, dims[1],
                 dims[0], act=ll.ACT_GELU, y_type=ll.T_F8, sy_ptr=hs.data_ptr(), ldw=ld0, ldx=ld0, stream=st)
    ll.dense_fp8(dw[1].data_ptr(), dsw[1].data_ptr(), 0, h.data_ptr(), hs.data_ptr(), y.data_ptr(), rows, dims[2],
                 dims[1], stream=st)
    ll.ops_check(st)
    xq, xs = quantize_rows(x)
    assert np.array_equal(decode(dq.cpu().numpy()[:, :dims[0]]), decode(xq))
    v = dequant_rows(xq, xs) @ dequant_blocks(*qs[0]).T
    h_ref = act64(v, ll.ACT_GELU)
    h_got = dequant_rows(h.cpu().numpy(), hs.cpu().numpy())
    a = np.abs(dequant_rows(xq, xs)) @ np.abs(dequant_blocks(*qs[0])).T
    tol = a * 2.0 ** -15 + np.abs(h_ref) * (2.0 ** -4 + 2.0 ** -16) + np.repeat(hs.cpu().numpy(), F8, 1) * 2.0 ** -10
    assert np.all(np.abs(h_got - h_ref) <= tol)
    y_ref = h_got @ dequant_blocks(*qs[1]).T
    a = np.abs(h_got) @ np.abs(dequant_blocks(*qs[1])).T
    assert np.all(np.abs(y.cpu().numpy() - y_ref) <= a * (128 + 4 + 11) * 2.0 ** -23)


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows,M", [(1, 4096), (256, 8192)])  # the few-row kernel, the many-row one
@pytest.mark.parametrize("y_type", [ll.T_F32, ll.T_BF16, ll.T_F16])
def test_gelu_keeps_its_digits_for_negative_values(rows, M, y_type):
    # Weights of zero, so that the activation's argument is the bias, exactly.  Bounds relative to the result:
    #   fp32: the exponent -v^2 / 2 has two roundings, 2^-24 of it each, so v^2 2^-23 / 2 in the tail; the rest
    #         (a polynomial's fit and its nine roundings, the approximate quotient and power, three products)
    #         within 6 units 2^-23, which also cover the other half of v^2;
    #   16 bits: the tail is good to 2^-16.5 up to |v| = 6.5 and 2^-14.2 beyond; two more operations add 2^-23;
    #         then half a step of rounding, of fp16's lowest octave 2^-25.
    from math import erfc

    import torch

    v = np.concatenate([np.linspace(-12.5, 8, M - 64), -np.exp2(np.linspace(-30, 3, 64))]).astype(np.float32)
    K = 16
    c = DenseCase(rows, M, K)
    c.d["w"].zero_()
    c.d["b"] = dev(v)
    y, _ = c.run(ll.ACT_GELU, y_type)
    ll.ops_check()
    v = v.astype(np.float64)
    ref = 0.5 * v * np.vectorize(erfc)(v * -np.sqrt(0.5))
    if y_type == ll.T_F32:
        tol = np.abs(ref) * (v * v + 6) * 2.0 ** -23
    else:
        tol = np.abs(ref) * (np.where(np.abs(v) <= 6.5, 2.0 ** -16.5, 2.0 ** -14.2) + 2.0 ** -22) * 1.01
        tol += np.abs(ref) * (2.0 ** -8 if y_type == ll.T_BF16 else 2.0 ** -11) + (y_type == ll.T_F16) * 2.0 ** -25
    got = y[:rows].double().cpu().numpy()
    assert torch.equal(y[0], y[rows - 1])
    off = np.abs(got - ref)
    assert np.all(off <= tol), (v[np.argmax(np.max(off - tol, 0))], np.max(off / np.maximum(tol, 1e-300)))
    big = DenseCase(rows, M, K, bias=False)
    big.d["w"].zero_()
    big.d["b"] = dev(np.full(M, np.inf, np.float32))
    assert np.all(big.run(ll.ACT_GELU, y_type)[0][:rows].float().cpu().numpy() == np.inf)


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows,M,K", [
    (1, 130, 300), (20, 520, 900), (150, 2000, 520), (1100, 1500, 300),  # few rows: tiles of 16, 32 and 128, split or not
    (1290, 2048, 384), (2500, 1030, 700)])                               # many rows
@pytest.mark.parametrize("act", [ll.ACT_IDENTITY, ll.ACT_RELU, ll.ACT_GELU, ll.ACT_SILU])
def test_e4m3_result_is_the_fp32_result_quantised(rows, M, K, act):
    # byte for byte, scales too: the bias spreads the values over the activations' whole range
    import torch

    c = DenseCase(rows, M, K, seed=41)
    c.d["b"] = dev(np.linspace(-13.0, 6.0, M).astype(np.float32)[np.argsort(np.arange(M) * 7919 % M, kind="stable")])
    f, _ = c.run(act, ll.T_F32)
    q, s = c.run(act, ll.T_F8)
    want_q = torch.full_like(q, 99)
    want_s = torch.empty_like(s)
    ll.quantize_fp8(f.data_ptr(), ll.T_F32, rows, M, want_q.data_ptr(), want_s.data_ptr(),
                    stream=torch.cuda.current_stream().cuda_stream)
    ll.ops_check()
    assert torch.equal(s, want_s)
    assert torch.equal(q, want_q)


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows,M,K,y_type", [
    (1, 16, 16, ll.T_F32), (1, 2048, 2048, ll.T_BF16),       # one block; two blocks in each of eight CTAs
    (20, 512, 4096, ll.T_F8), (8, 300, 40000, ll.T_F32),     # as many blocks as stages and more
    (1100, 1500, 1300, ll.T_F32),                            # tiles of 128 rows
    (1290, 2048, 384, ll.T_BF16), (2560, 4096, 1024, ll.T_F8),  # pairs of SMs: within the first stages, and beyond
])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(rows, M, K, y_type):
    # with a limit of 0 every wait gives up: loads and products in flight end before the kernel does, the status
    # says so, and the calls behind it are as ever
    import torch

    c = DenseCase(rows, M, K, seed=51)
    want, want_s = c.run(ll.ACT_RELU, y_type)
    ll.ops_check()
    y, sy = want.clone(), want_s.clone()
    for _ in range(3):
        ll.ops_set_wait_limit(0)
        try:
            c.run(ll.ACT_RELU, y_type, y=y, sy=sy)
        finally:
            ll.ops_set_wait_limit()
        c.run(ll.ACT_RELU, y_type, y=y, sy=sy)
        with pytest.raises(ll.LLError) as e:
            ll.ops_check()
        assert e.value.code == ll.LL_ERR_DEVICE_FAULT
        assert torch.equal(y, want) and torch.equal(sy, want_s)
        ll.ops_check()


@pytest.mark.gpu
@pytest.mark.timeout(300)
def test_every_stream_and_thread_is_told_of_a_failure():
    # a failure on stream b: the check of stream a takes nothing from b's, whichever comes first, nor from
    # another thread's; each is told once
    import threading

    import torch

    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    c = DenseCase(3, 128, 256, seed=61)
    y, sy = c.run(ll.ACT_RELU, ll.T_F32)
    torch.cuda.synchronize()

    def told(stream):
        try:
            ll.ops_check(stream.cuda_stream)
            return False
        except ll.LLError as e:
            assert e.code == ll.LL_ERR_DEVICE_FAULT
            return True

    def elsewhere(stream):
        out = []
        t = threading.Thread(target=lambda: out.extend((told(stream), told(stream))))
        t.start()
        t.join()
        return out

    for first, second in ((a, b), (b, a)):
        ll.ops_set_wait_limit(0)
        try:
            c.run(ll.ACT_RELU, ll.T_F32, stream=b, y=y, sy=sy)
        finally:
            ll.ops_set_wait_limit()
        b.synchronize()
        assert told(first)
        assert told(second)
        assert elsewhere(b) == [True, False]
        assert not told(first) and not told(second)
    assert told(torch.cuda.default_stream()) and not told(torch.cuda.default_stream())


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("x_type", [ll.T_F32, ll.T_BF16])
def test_quantize_ties_of_the_smallest_scales(x_type):
    # groups whose scale is 2^-126 or little more: what separates a quotient from a border of two e4m3 values is
    # below fp32's smallest number there, and still decides
    rows = []
    mids = (TABLE[:-1] + TABLE[1:]) / 2
    if x_type == ll.T_F32:
        sig = np.concatenate([1 + np.arange(1, 40) * 2.0 ** -23, np.linspace(1.0, 2.0, 25)])
        for e in (-126, -125, -120, -110, -66, -60):
            for g in sig:
                s = np.float32(g * 2.0 ** e)
                amax = np.float32(448.0 * s)
                s = np.float32(amax / np.float32(448))
                v = (mids * np.float64(s)).astype(np.float32)
                v = np.concatenate([np.nextafter(v[:42], np.float32(0)), v[42:84], np.nextafter(v[84:], np.float32(1))])
                rows.append(np.concatenate([v, [amax, -amax]]))
    else:
        for k in range(1, 37):  # the scales that are exact in 16 bits
            for e in range(-126 - 5, -112):
                s = k * 2.0 ** e
                if s < 2.0 ** -126:
                    continue
                v = (mids * s).astype(np.float32)
                u = v.view(np.uint32)
                u += 0x7FFF + ((u >> 16) & 1)
                u &= np.uint32(0xFFFF0000)
                rows.append(np.concatenate([v, [448 * s, -448 * s]]))
    x = np.stack(rows).astype(np.float32)
    assert x.shape[1] == F8
    q, s, x = run_quantize(x, x_type)
    want_q, want_s = quantize_rows(x)
    assert np.array_equal(s, want_s)
    assert np.array_equal(decode(q), decode(want_q))


@pytest.mark.gpu
@pytest.mark.timeout(300)
@pytest.mark.parametrize("rows,M,K", [(17, 12300, 200), (32, 14336, 256), (100, 12288, 144)])
@pytest.mark.parametrize("y_type", [ll.T_BF16, ll.T_F8])
def test_dense_wide_layers_of_few_rows(rows, M, K, y_type):
    # tiles of 128 rows of which most do not exist
    c = DenseCase(rows, M, K, seed=91)
    y, sy = c.run(ll.ACT_GELU, y_type, pad_y=4)
    ll.ops_check()
    c.check(ll.ACT_GELU, y_type, y, sy)
