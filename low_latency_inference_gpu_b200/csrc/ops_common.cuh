// Shared by the stateless operators (fp8_quant.cu, dense_fp8.cu, moe.cu): element types,
// the e4m3 rounding, checks of device pointers, and the device status word.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "common.h"
#include "tc_layer.cuh"

namespace llk {

constexpr int kF8Block = LL_F8_BLOCK;   // columns (and weight rows) that share one scale
constexpr float kF8Max = 448.0f;        // largest e4m3 value
constexpr float kF8SmallScale = 0x1p-60f;  // v - s times an e4m3 border may be subnormal well below this
constexpr int kOpsMaxDevices = 64;
// Bound on every device-side wait of the stateless operators (ll_ops_set_wait_limit changes it), and the longest
// that a CTA which gave up stays for its own copies and products in flight: independent of the first.
constexpr unsigned long long kOpsWaitNs = 1000ull * 1000 * 1000, kOpsMaxWaitNs = 60 * kOpsWaitNs;
constexpr unsigned long long kOpsDrainNs = 2000ull * 1000 * 1000;

__host__ __device__ constexpr int type_bytes(int t)
{
    return t == LL_T_F32 ? 4 : t == LL_T_F8 ? 1 : 2;
}

// Coefficients of Q below, from the eighth power down.
__host__ __device__ constexpr float gelu_ratio(int k)
{
    constexpr float c[9] = {-2.912588469e-02f, 1.438723275e-01f, -2.555047497e-01f, 1.589294961e-01f, -2.293727501e-02f,
                            1.054329923e-01f,  1.198524239e-01f, 1.398590840e-01f,  1.396215697e-01f};
    return c[k];
}

// GELU, v Phi(v), with the digits of the normal tail: 1 + erf(v / sqrt 2) cancels for negative v and leaves
// none of them from -5.5 on.  Phi(-a) = exp(-a^2 / 2) t Q(t), t = 1 / (1 + 0.35 a) (the form of Hastings,
// Approximations for Digital Computers, 1955; Q fitted on a <= 13.5 for the least largest relative error).
// Off by (v^2 + 6) 2^-23 of the result at most: the exponent's two roundings, and 2^-21 for the rest.  Side by
// side in ll_dense_fp8, 8192 x 4096 x 4096 with an fp32 result: 169 us, with erfcf 204, with erff 174.
__device__ __forceinline__ float ops_gelu(float v)
{
    const float a = fminf(fabsf(v), 13.5f);  // the exponential is 0 there
    float t, e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(a, 0.35f, 1.0f)));
    float r = gelu_ratio(0);
#pragma unroll
    for (int k = 1; k < 9; ++k)
        r = fmaf(r, t, gelu_ratio(k));
    r = __fmul_rn(r, t);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(__fmul_rn(a, a), -0.72134752044448170f)));
    return v > 0.0f ? fmaf(-__fmul_rn(a, r), e, v) : __fmul_rn(__fmul_rn(v, r), e);
}

__device__ __forceinline__ float ops_act(float v, int act)
{
    if (act == LL_ACT_RELU)
        return v > 0.0f ? v : 0.0f;
    if (act == LL_ACT_GELU)
        return ops_gelu(v);
    if (act == LL_ACT_SILU)
        return v / __fadd_rn(1.0f, expf(-v));  // no step is fused with another one, wherever this is compiled
    return v;
}

// Coefficients of log2 Phi(-a), from the tenth power down.
__host__ __device__ constexpr float gelu_tail(int k)
{
    constexpr float c[11] = {4.106086714e-11f, -4.780448844e-09f, 2.251157347e-07f, -5.900948207e-06f, 9.810118466e-05f,
                             -1.111293283e-03f, 9.013057538e-03f, -5.472723828e-02f, -4.578987302e-01f, -1.151406366e+00f,
                             -9.999885429e-01f};
    return c[k];
}
constexpr float kGeluClamp = 13.25f;  // from 12.95 on the power of two is below fp32's normal numbers: 0

// The activations for results that are rounded to 16 bits, where that rounding takes up to 2^-8 (bf16) or
// 2^-11 (fp16) of the result, at a third of the instructions:
//   gelu  v Phi(v), Phi(-a) = 2^P(a): the logarithm of the normal tail is smooth, so a polynomial of degree
//         10, fitted on [0, 13.25] for the least largest error (fit and fp32 evaluation), gives the tail to
//         2^-16.5 of itself up to a = 6.5 and to 2^-14.2 beyond, where only bf16 has numbers for it.
//         Results below 2^-122 become 0.
//   silu  with the approximate exponential and quotient: 2^-16 of the result; those below 2^-119 become 0.
__device__ __forceinline__ float ops_act_fast(float v, int act)
{
    if (act == LL_ACT_GELU) {
        const float b = fminf(fabsf(v), kGeluClamp);
        float r = gelu_tail(0);
#pragma unroll
        for (int k = 1; k < 11; ++k)
            r = fmaf(r, b, gelu_tail(k));
        float tail;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(tail) : "f"(r));
        return v * (v > 0.0f ? 1.0f - tail : tail);
    }
    if (act == LL_ACT_SILU)
        return __fdividef(v, 1.0f + __expf(-v));
    return ops_act(v, act);
}

// Two fp32 values in a register pair.
__device__ __forceinline__ uint64_t f2_pack(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 f2_unpack(uint64_t v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// gelu of ops_act_fast, N values in pairs: the same steps in fewer instructions.  8192 x 4096 x 4096 of
// ll_dense_fp8 with a bf16 result takes 151 us with it (142 with relu).
template <int N>
__device__ __forceinline__ void ops_gelu_fast(float (&v)[N])
{
    uint64_t b[N / 2], r[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        b[i] = f2_pack(fminf(fabsf(v[2 * i]), kGeluClamp), fminf(fabsf(v[2 * i + 1]), kGeluClamp));
        r[i] = f2_pack(gelu_tail(0), gelu_tail(0));
    }
#pragma unroll
    for (int k = 1; k < 11; ++k) {
        const uint64_t ck = f2_pack(gelu_tail(k), gelu_tail(k));
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
            r[i] = f2_fma(r[i], b[i], ck);
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float2 q = f2_unpack(r[i]);
        float2 t;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t.x) : "f"(q.x));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t.y) : "f"(q.y));
        v[2 * i] = v[2 * i] * (v[2 * i] > 0.0f ? 1.0f - t.x : t.x);
        v[2 * i + 1] = v[2 * i + 1] * (v[2 * i + 1] > 0.0f ? 1.0f - t.y : t.y);
    }
}

// Bounded waits on a barrier of this CTA, by one thread or a whole warp.  Most end within the first
// looks, which read no timer and keep the loop short.  A bound of 0 gives up without a look.
__device__ __forceinline__ bool ops_try_wait(uint32_t bar, uint32_t parity)
{
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0u;
}

// status: how many waits ran out, never reset, and the role of the last one (llh::ops_status_words).
__device__ __forceinline__ void ops_give_up(volatile uint32_t *fail, unsigned *status, uint32_t role)
{
    *fail = 1u;
    atomicExch(status + 1, role);
    atomicAdd(status, 1u);
}

__device__ __forceinline__ bool ops_wait(uint32_t bar, uint32_t parity, unsigned long long bound_ns,
                                         volatile uint32_t *fail, unsigned *status, uint32_t role)
{
    uint64_t t0 = 0;
#pragma unroll 1
    for (uint32_t it = 1; bound_ns != 0; ++it) {
        if (ops_try_wait(bar, parity))
            return true;
        if ((it & 63u) == 0) {
            if (*fail)  // another role of the CTA gave up
                return false;
            const uint64_t now = globaltimer();
            if (t0 == 0)
                t0 = now;
            else if (now - t0 > bound_ns)
                break;
        }
    }
    ops_give_up(fail, status, role);
    return false;
}

// Every lane looks for itself (so that what the phase guards is visible to each) and the verdict is the warp's.
__device__ __forceinline__ bool ops_wait_warp(uint32_t bar, uint32_t parity, unsigned long long bound_ns,
                                              volatile uint32_t *fail, unsigned *status, uint32_t role)
{
    uint64_t t0 = 0;
#pragma unroll 1
    for (uint32_t it = 1; bound_ns != 0; ++it) {
        if (__all_sync(0xffffffffu, ops_try_wait(bar, parity)))
            return true;
        if ((it & 63u) == 0) {
            if (__any_sync(0xffffffffu, *fail != 0u))
                return false;
            const uint64_t now = globaltimer();
            if (t0 == 0)
                t0 = now;
            else if (__any_sync(0xffffffffu, now - t0 > bound_ns))
                break;
        }
    }
    if ((threadIdx.x & 31) == 0)
        ops_give_up(fail, status, role);
    return false;
}

// What a CTA that gave up still waits for: phase `parity` of `bar`, until kOpsDrainNs after t0.
__device__ __forceinline__ void ops_drain(uint32_t bar, uint32_t parity, uint64_t t0)
{
    while (!mbar_try_wait(bar, parity) && globaltimer() - t0 < kOpsDrainNs) {
    }
}

// One lane of a converged warp, the same one every time: true there.  With the warp converged around it the
// compiler keeps addresses and descriptors in uniform registers.
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0u;
}

// ---- e4m3 ----

// Two fp32 values to e4m3 (nearest, ties to even, beyond the largest to the largest), lo in bits 0..7.
__device__ __forceinline__ uint32_t f32x2_to_e4m3(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// The value of an e4m3 code without sign (exact).
__device__ __forceinline__ float e4m3_value(uint32_t code)
{
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)code));
    return __low2float(*reinterpret_cast<const __half2 *>(&h));
}

// Of two neighbouring e4m3 codes (one byte each, of v's sign) the one nearest to the exact quotient v / s:
// the sign of |v| - border * s, one fused operation, says on which side of the border (5 significant
// bits, exact) the quotient lies; a tie goes to the even code.  Of a small scale both are lifted by a power of
// two: among fp32's subnormal numbers the difference would be rounded to 0.
__device__ __forceinline__ uint32_t nearer_e4m3(float v, float s, uint32_t a, uint32_t b)
{
    const uint32_t lo = min(a, b) & 0x7fu, hi = max(a, b) & 0x7fu, sign = a & 0x80u;
    const float border = 0.5f * (e4m3_value(lo) + e4m3_value(hi));
    const float lift = s < kF8SmallScale ? 1.0f / kF8SmallScale : 1.0f;
    const float side = fmaf(-border, s * lift, fabsf(v) * lift);
    return sign | (side > 0.0f ? hi : side < 0.0f ? lo : lo + (lo & 1u));
}

// The e4m3 codes of v0 / s and v1 / s where a border lies between a and b.  Rare, so by a call: in line its copies for
// each of 128 values weighed on the many-row dense layer's store (8192 x 4096 x 4096 with GELU and an e4m3 result 384 us
// with them, 321 without).
static __device__ __noinline__ uint32_t near_border_e4m3(float v0, float v1, float s, uint32_t a, uint32_t b)
{
    uint32_t o = a;
    if ((a ^ b) & 0xffu)
        o = (o & 0xff00u) | nearer_e4m3(v0, s, a & 0xffu, b & 0xffu);
    if ((a ^ b) & 0xff00u)
        o = (o & 0xffu) | (nearer_e4m3(v1, s, a >> 8, b >> 8) << 8);
    return o;
}

// e4m3 of v0 / s and v1 / s given inv = 1 / s to 2^-23.  The quotient lies between v times inv (1 + 2^-21)
// and v times inv (1 - 2^-21), each rounded; where both are one e4m3 value that is the answer.
// Else a border lies between, and the exact side is decided in a few operations.
__device__ __forceinline__ uint32_t quot_e4m3(float v0, float v1, float s, float inv)
{
    const float up = inv * (1.0f + 0x1p-21f), down = inv * (1.0f - 0x1p-21f);
    const uint32_t a = f32x2_to_e4m3(v0 * up, v1 * up);
    const uint32_t b = f32x2_to_e4m3(v0 * down, v1 * down);
    if (a == b)
        return a;
    return near_border_e4m3(v0, v1, s, a, b);
}

// The scale of a group whose largest magnitude is amax: amax / 448, or the next power of two at
// or above it; at least 2^-126 so that its reciprocal is finite; 0 for an all-zero group.
__device__ __forceinline__ void e4m3_scale(float amax, bool pow2, float &s, float &inv)
{
    if (!(amax > 0.0f)) {
        s = 0.0f;
        inv = 0.0f;
        return;
    }
    const float q = fmaxf(__fdiv_rn(amax, kF8Max), 0x1p-126f);
    if (pow2) {
        const uint32_t u = __float_as_uint(q);
        const uint32_t e = (u >> 23) + ((u & 0x7fffffu) != 0u);
        s = __uint_as_float(e << 23);
        inv = e >= 254u ? 0.0f : __uint_as_float((254u - e) << 23);
    } else {
        s = q;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(q));
    }
}

// Four fp32 values of one group as four e4m3 bytes.
__device__ __forceinline__ uint32_t group_e4m3x4(const float *v, bool pow2, float s, float inv)
{
    if (pow2 || s == 0.0f)  // the product is the quotient (a power of two; zeros and NaN)
        return f32x2_to_e4m3(v[0] * inv, v[1] * inv) | (f32x2_to_e4m3(v[2] * inv, v[3] * inv) << 16);
    return quot_e4m3(v[0], v[1], s, inv) | (quot_e4m3(v[2], v[3], s, inv) << 16);
}

}  // namespace llk

namespace llh {

// Device words in which a stateless operator's kernel counts the bounded waits that ran out, and notes the role
// of the last one (one pair per GPU, never reset; read by ll_ops_check).  Looked up once per device.
int ops_status_words(int *device, unsigned **words);

// The bound of device-side waits that calls from now on take.
unsigned long long ops_wait_ns();

// LL_OK when p is memory of the current device (managed memory included), aligned to `align` bytes.
int check_device_ptr(const char *op, const char *what, const void *p, int device, size_t align);

}  // namespace llh

#define LL_TRY(call)         \
    do {                     \
        int _rc = (call);    \
        if (_rc != LL_OK)    \
            return _rc;      \
    } while (0)
