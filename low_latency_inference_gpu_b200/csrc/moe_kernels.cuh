// A mixture-of-experts layer for up to LL_MOE_MAX_ROWS rows in two kernels (no counterpart in the
// reference, whose net is one dense chain).
//
//   logits = Wr x;  the top_k experts of each row (ties: lowest index) with weights w from softmax
//   a[r, j] = act(Wg_e x_r) * (Wu_e x_r)          (gated; else act(Wg_e x_r)),  e = expert j of row r
//   y_r     = sum_j w[r, j] Wd_e a[r, j]
//
// With few rows the layer reads the picked experts' weights once and does little else, so both
// kernels stream weight rows from memory through a ring in shared memory (bulk copies, 1 KB of
// each of 16 rows per stage; one warp copies, eight compute) and multiply them on the warp-level
// bf16 tensor instruction with 16 weight rows as M and 8 of the expert's rows of x as N.  A
// tcgen05 tile (M = 128) would need each expert's rows padded to a full tile and int8 / e4m3
// weights widened in tensor memory; at these widths the memory is the bound and the warp-level
// instruction is at a few per cent of its rate.
//
// Precision: weights are exact in bf16 (int8 and e4m3 too; their scales multiply fp32 sums).  x
// and the activations a are split into bf16 terms that add up to the value: x in bf16 one, fp16
// two (exact), fp32 three (exact); a two (16 bits, below the rounding of a 16-bit y) or three
// for an fp32 layer.  All sums are fp32.
//
// Kernel 1 (clusters of 8 CTAs): every cluster computes all logits, each CTA over an eighth of the
// columns, exchanged through distributed shared memory; then each CTA picks the experts and takes
// its share of the (expert, channels) tiles: 8 gate rows and the 8 up rows of the same channels
// (so the product of the two is taken in the thread that holds both).
// Kernel 2: each CTA owns up to 16 output channels and walks all picked experts' rows of Wd for
// them; every warp keeps its own partial outputs, added in warp order at the end.
// No atomics on floating-point values: results repeat bit for bit.
#pragma once
#include "ops_common.cuh"
#include "tc_layer.cuh"

namespace llk {

constexpr int kMoeThreads = 288;        // warps 0..7 compute, warp 8 copies
constexpr int kMoeWarps = 8;
constexpr int kMoeCluster = 8;          // kernel 1
constexpr int kMoeSegment = 1024;       // bytes of a weight row per stage: 128 per computing warp
constexpr int kMoePitch = kMoeSegment + 64;  // 64 mod 128: the 8 rows that a quarter warp reads do not collide
constexpr int kMoeStage = 16 * kMoePitch;
constexpr int kMoeMaxStages = 12;
constexpr int kMoeMaxPairs = LL_MOE_MAX_ROWS * LL_MOE_MAX_TOPK;

struct MoeParams {
    const void *x;
    long long ldx;
    void *y;
    long long ldy;
    int rows, hidden, inter, experts, top_k, act, gated, renorm, x_type;
    const void *router;
    int router_f32, router_vec, x_vec;  // *_vec: rows start on 16 bytes
    const uint8_t *wg, *wu, *wd;
    const float *sg, *su, *sd;
    int up_ring, down_ring;             // weight rows start on 16 bytes and are multiples of 16 bytes long
    int *ids;                           // workspace [rows][top_k]
    float *probs;
    int *user_ids;                      // or nullptr
    float *user_probs;
    __nv_bfloat16 *hid;                 // workspace: planes [rows * top_k][hid_ld]
    long long hid_plane;
    int hid_ld;
    int stages;                         // of the ring
    unsigned *status;
    unsigned long long wait_ns;
};

// ---- shared memory after the ring (byte offsets; the ring is at 0) ----
struct MoeSmem {
    int bars, pairs, ids, probs, mask, act_e, act_off, misc, logits, part, red, total;
};

__host__ __device__ inline int moe_up16(int v)
{
    return (v + 15) & ~15;
}

__host__ __device__ inline MoeSmem moe_smem(const MoeParams &p, bool up, int nt)
{
    MoeSmem s;
    int o = p.stages * kMoeStage;
    const int n = p.rows * p.top_k;
    s.bars = o, o += moe_up16(16 * kMoeMaxStages);
    s.misc = o, o += 16;  // fail flag, number of picked experts
    s.pairs = o, o += moe_up16(2 * n);
    s.ids = o, o += moe_up16(4 * n);
    s.probs = o, o += moe_up16(4 * n);
    s.mask = o, o += moe_up16(4 * p.experts);
    s.act_e = o, o += moe_up16(2 * (p.experts < n ? p.experts : n));
    s.act_off = o, o += moe_up16(2 * ((p.experts < n ? p.experts : n) + 1));
    s.logits = s.part = 0;
    if (up) {
        const int mt = (p.experts + 15) / 16, ksub = mt >= kMoeWarps ? 1 : kMoeWarps / mt;
        const int tp = (p.rows + 7) / 8 * 8;
        s.logits = o, o += moe_up16(4 * p.rows * p.experts);
        s.part = o, o += 4 * ksub * mt * 16 * tp;
        s.red = o, o += 2 * kMoeWarps * nt * 32 * 16;
    } else {
        s.red = o, o += kMoeWarps * p.rows * 16 * 4;
    }
    s.total = o;
    return s;
}

// ---- bf16 terms ----
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ float2 unpack_bf16(uint32_t w)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// (a, b) as NS packed bf16 terms each; an infinity or NaN keeps its first term alone.
template <int NS>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&w)[NS])
{
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        w[s] = pack_bf16(a, b);
        if (s + 1 < NS) {
            const float2 h = unpack_bf16(w[s]);
            a = fabsf(h.x) <= 3.4e38f ? a - h.x : 0.0f;
            b = fabsf(h.y) <= 3.4e38f ? b - h.y : 0.0f;
        }
    }
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Weight types: EP values in 16 bytes; widen() gives them as EP / 2 packed bf16 pairs, exact.
template <int WT>
struct MoeW;

template <>
struct MoeW<LL_W_BF16> {
    static constexpr int BYTES = 2, EP = 8;
    static __device__ __forceinline__ void widen(const uint4 &v, uint32_t (&o)[4])
    {
        o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
    }
};

template <>
struct MoeW<LL_W_I8> {
    static constexpr int BYTES = 1, EP = 16;
    static __device__ __forceinline__ void widen(const uint4 &v, uint32_t (&o)[8])
    {
        i8x4_to_bf16x4(v.x, o[0], o[1]);
        i8x4_to_bf16x4(v.y, o[2], o[3]);
        i8x4_to_bf16x4(v.z, o[4], o[5]);
        i8x4_to_bf16x4(v.w, o[6], o[7]);
    }
};

template <>
struct MoeW<LL_W_F8> {
    static constexpr int BYTES = 1, EP = 16;
    static __device__ __forceinline__ uint32_t pair(uint32_t two)
    {
        uint32_t h;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
        return pack_bf16(f.x, f.y);
    }
    static __device__ __forceinline__ void widen(const uint4 &v, uint32_t (&o)[8])
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[2 * i] = pair(w[i] & 0xffffu);
            o[2 * i + 1] = pair(w[i] >> 16);
        }
    }
};

// The first n values of 16 bytes at p (n <= 0: none), the others zero; any alignment.
template <int BYTES>
__device__ __forceinline__ uint4 load_some(const uint8_t *p, int n)
{
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16 / BYTES; ++i)
        if (i < n) {
            const uint32_t v = BYTES == 1 ? (uint32_t)p[i] : (uint32_t) reinterpret_cast<const uint16_t *>(p)[i];
            w[i * BYTES / 4] |= v << (8 * (i * BYTES % 4));
        }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// EP consecutive values of a row of x as NS packed bf16 terms: n of them exist (n <= 0: none).
template <int XT>
struct MoeX {
    static constexpr int NS = XT == LL_T_BF16 ? 1 : XT == LL_T_F16 ? 2 : 3;
    static constexpr int BYTES = XT == LL_T_F32 ? 4 : 2;

    template <int EP>
    static __device__ __forceinline__ void load(const uint8_t *row, int k, int n, bool vec, uint32_t (&w)[NS][EP / 2])
    {
        const uint8_t *p = row + (size_t)k * BYTES;
        if (vec && n >= EP) {
#pragma unroll
            for (int i = 0; i < EP * BYTES / 16; ++i) {
                const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p) + i);
                take<EP>(v, i, w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < EP * BYTES / 16; ++i) {
                const int have = n - i * (16 / BYTES);
                uint4 v;
                if constexpr (BYTES == 4) {
                    const uint32_t *q = reinterpret_cast<const uint32_t *>(p) + 4 * i;
                    v.x = have > 0 ? __ldg(q) : 0u;
                    v.y = have > 1 ? __ldg(q + 1) : 0u;
                    v.z = have > 2 ? __ldg(q + 2) : 0u;
                    v.w = have > 3 ? __ldg(q + 3) : 0u;
                } else {
                    v = load_some<2>(p + 16 * i, have);
                }
                take<EP>(v, i, w);
            }
        }
    }

    // The i-th 16 bytes of the values into their places.
    template <int EP>
    static __device__ __forceinline__ void take(const uint4 &v, int i, uint32_t (&w)[NS][EP / 2])
    {
        if constexpr (XT == LL_T_BF16) {
            w[0][4 * i] = v.x, w[0][4 * i + 1] = v.y, w[0][4 * i + 2] = v.z, w[0][4 * i + 3] = v.w;
        } else if constexpr (XT == LL_T_F16) {
            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[j]));
                uint32_t t[NS];
                split_pair<NS>(f.x, f.y, t);
#pragma unroll
                for (int s = 0; s < NS; ++s)
                    w[s][4 * i + j] = t[s];
            }
        } else {
            uint32_t t[NS];
            split_pair<NS>(__uint_as_float(v.x), __uint_as_float(v.y), t);
#pragma unroll
            for (int s = 0; s < NS; ++s)
                w[s][2 * i] = t[s];
            split_pair<NS>(__uint_as_float(v.z), __uint_as_float(v.w), t);
#pragma unroll
            for (int s = 0; s < NS; ++s)
                w[s][2 * i + 1] = t[s];
        }
    }
};

// ---- the lists of picked experts, from the ids in shared memory (all threads; rows <= 32) ----
// act_e[a] = a-th picked expert (rising), its rows are pairs[act_off[a] .. act_off[a + 1]),
// pair = row | slot << 8, rows rising.
__device__ __forceinline__ void moe_lists(const MoeParams &p, uint8_t *smem, const MoeSmem &L)
{
    const int n = p.rows * p.top_k;
    const int *ids = reinterpret_cast<const int *>(smem + L.ids);
    uint32_t *mask = reinterpret_cast<uint32_t *>(smem + L.mask);
    uint16_t *act_e = reinterpret_cast<uint16_t *>(smem + L.act_e);
    uint16_t *act_off = reinterpret_cast<uint16_t *>(smem + L.act_off);
    uint16_t *pairs = reinterpret_cast<uint16_t *>(smem + L.pairs);
    uint32_t *misc = reinterpret_cast<uint32_t *>(smem + L.misc);
    for (int e = threadIdx.x; e < p.experts; e += blockDim.x)
        mask[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x)
        atomicOr(&mask[ids[i]], 1u << (i / p.top_k));
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int a0 = 0, off0 = 0;
        for (int e0 = 0; e0 < p.experts; e0 += 32) {
            const int e = e0 + lane;
            const uint32_t m = e < p.experts ? mask[e] : 0u;
            const uint32_t on = __ballot_sync(0xffffffffu, m != 0u);
            int sum = __popc(m);  // inclusive prefix sum over the lanes
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d)
                    sum += v;
            }
            if (m != 0u) {
                const int a = a0 + __popc(on & ((1u << lane) - 1u));
                act_e[a] = (uint16_t)e;
                act_off[a] = (uint16_t)(off0 + sum - __popc(m));
            }
            a0 += __popc(on);
            off0 += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) {
            act_off[a0] = (uint16_t)off0;
            misc[1] = (uint32_t)a0;
        }
    }
    __syncthreads();
    const int na = (int)misc[1];
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int row = i / p.top_k, slot = i - row * p.top_k, e = ids[i];
        int lo = 0, hi = na - 1;  // the place of e among the picked
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (act_e[mid] < e)
                lo = mid + 1;
            else
                hi = mid;
        }
        pairs[act_off[lo] + __popc(mask[e] & ((1u << row) - 1u))] = (uint16_t)(row | slot << 8);
    }
    __syncthreads();
}

// ---- the ring ----
struct MoeRing {
    uint32_t base, bars;
    int stages;
    __device__ __forceinline__ uint32_t full(int s) const
    {
        return bars + 16u * (uint32_t)s;
    }
    __device__ __forceinline__ uint32_t empty(int s) const
    {
        return bars + 16u * (uint32_t)s + 8u;
    }
};

__device__ __forceinline__ void moe_ring_init(const MoeRing &r)
{
    for (int s = 0; s < r.stages; ++s) {
        mbar_init(r.full(s), 1);
        mbar_init(r.empty(s), kMoeWarps);
    }
    fence_mbar_init_cluster();
}

// The copying warp's part for one set of 16 rows: their segments one after another.  `src` is this
// lane's row (lanes 0..15; nullptr: no such row), `bytes` its length.  `it` counts stages.
__device__ __forceinline__ bool moe_copy_rows(const MoeParams &p, const MoeRing &r, const uint8_t *src, int bytes,
                                              int n_rows, uint32_t &it, volatile uint32_t *fail)
{
    const int lane = threadIdx.x & 31;
    for (int o = 0; o < bytes; o += kMoeSegment, ++it) {
        const int s = (int)(it % (uint32_t)r.stages);
        const uint32_t lap = it / (uint32_t)r.stages;
        const int len = min(kMoeSegment, bytes - o);
        if (lap > 0 && !tc_wait_warp(r.empty(s), (lap - 1) & 1, p.wait_ns, fail, p.status, 1))
            return false;
        if (lane == 0)
            mbar_arrive_expect_tx(r.full(s), (uint32_t)(len * n_rows));
        __syncwarp();
        if (src)
            bulk_g2s(r.base + (uint32_t)(s * kMoeStage + lane * kMoePitch), src + o, (uint32_t)len, r.full(s));
    }
    return true;
}

// Waits for the loads of the last stages: nothing is in flight when the CTA leaves.
__device__ __forceinline__ void moe_drain(const MoeParams &p, const MoeRing &r, uint32_t it)
{
    const uint32_t n = min(it, (uint32_t)r.stages);
    for (uint32_t j = it - n; j < it; ++j) {
        const uint64_t t0 = globaltimer();
        while (!mbar_try_wait(r.full((int)(j % (uint32_t)r.stages)), (j / (uint32_t)r.stages) & 1) &&
               globaltimer() - t0 < p.wait_ns) {
        }
    }
}

// One warp's 128 bytes of each of 16 weight rows against the n-tiles of x: acc += W x.
// r0 / r1: this thread's rows g and g + 8 at the warp's bytes (shared or global memory); k0: their
// first column; K: columns of the row; wvec: 16-byte loads allowed; load_x(nt, k, n, words).
template <int WT, int NS, int NT, class LoadX>
__device__ __forceinline__ void moe_step(float (&acc)[NT][4], const uint8_t *r0, const uint8_t *r1, bool wvec, int k0,
                                         int K, int ntc, LoadX load_x)
{
    using W = MoeW<WT>;
    constexpr int EP = W::EP;
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int pc = 0; pc < 2; ++pc) {
        const int ko = pc * 4 * EP + t * EP;  // this thread's values within the step
        const int n = K - (k0 + ko);
        uint4 v0, v1;
        if (wvec && n >= EP) {
            v0 = *reinterpret_cast<const uint4 *>(r0 + ko * W::BYTES);
            v1 = *reinterpret_cast<const uint4 *>(r1 + ko * W::BYTES);
        } else {
            v0 = load_some<W::BYTES>(r0 + ko * W::BYTES, n);
            v1 = load_some<W::BYTES>(r1 + ko * W::BYTES, n);
        }
        uint32_t a0[EP / 2], a1[EP / 2];
        W::widen(v0, a0);
        W::widen(v1, a1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt < ntc) {
                uint32_t b[NS][EP / 2];
                load_x(nt, k0 + ko, n, b);
#pragma unroll
                for (int j = 0; j < EP / 4; ++j)
#pragma unroll
                    for (int s = 0; s < NS; ++s)
                        mma_bf16(acc[nt], a0[2 * j], a1[2 * j], a0[2 * j + 1], a1[2 * j + 1], b[s][2 * j],
                                 b[s][2 * j + 1]);
            }
        }
    }
}

// Sum over a whole set of 16 rows: this warp takes bytes 128 w .. 128 w + 127 of every segment.
// Through the ring (row pointers unused) or straight from global memory.  e4m3: sc0 / sc1 are the
// scales of the thread's rows g and g + 8 by 128-column block.
template <int WT, int NS, int NT, class LoadX>
__device__ __forceinline__ bool moe_rows(const MoeParams &p, const MoeRing &r, const uint8_t *smem, bool ring,
                                         const uint8_t *g0, const uint8_t *g1, int K, const float *sc0,
                                         const float *sc1, int ntc, uint32_t &it, bool ok, volatile uint32_t *fail,
                                         float (&acc)[NT][4], LoadX load_x)
{
    using W = MoeW<WT>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    constexpr int KSEG = kMoeSegment / W::BYTES, KW = 128 / W::BYTES;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            acc[nt][i] = 0.0f;
    for (int kseg = 0; kseg < K; kseg += KSEG, ++it) {
        const int k0 = kseg + warp * KW;
        const uint8_t *r0 = g0 + (size_t)k0 * W::BYTES, *r1 = g1 + (size_t)k0 * W::BYTES;
        int s = 0;
        if (ring) {
            s = (int)(it % (uint32_t)r.stages);
            r0 = smem + s * kMoeStage + g * kMoePitch + warp * 128;
            r1 = r0 + 8 * kMoePitch;
            if (ok)
                ok = tc_wait_warp(r.full(s), (it / (uint32_t)r.stages) & 1, p.wait_ns, fail, p.status, 2);
        }
        if (ok && k0 < K) {
            if constexpr (WT == LL_W_F8) {
                float part[NT][4] = {};
                const float f0 = __ldg(sc0 + k0 / kF8Block), f1 = __ldg(sc1 + k0 / kF8Block);
                moe_step<WT, NS, NT>(part, r0, r1, ring, k0, K, ntc, load_x);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    acc[nt][0] = fmaf(part[nt][0], f0, acc[nt][0]);
                    acc[nt][1] = fmaf(part[nt][1], f0, acc[nt][1]);
                    acc[nt][2] = fmaf(part[nt][2], f1, acc[nt][2]);
                    acc[nt][3] = fmaf(part[nt][3], f1, acc[nt][3]);
                }
            } else {
                moe_step<WT, NS, NT>(acc, r0, r1, ring, k0, K, ntc, load_x);
            }
        }
        if (ring) {
            __syncwarp();
            if (lane == 0)
                mbar_arrive_local(r.empty(s));
        }
    }
    return ok;
}

__device__ __forceinline__ void moe_bar()
{
    asm volatile("bar.sync 1, 256;" ::: "memory");  // the computing warps
}

// ---- router: logits of every (row, expert), by the whole cluster ----
template <int XT, int NT>
__device__ __forceinline__ void moe_logits(const MoeParams &p, uint8_t *smem, const MoeSmem &L)
{
    using X = MoeX<XT>;
    constexpr int EP = 8, KS = 64;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int mt_n = (p.experts + 15) / 16, ksub = mt_n >= kMoeWarps ? 1 : kMoeWarps / mt_n;
    const int tp = (p.rows + 7) / 8 * 8, ntc = tp / 8, H = p.hidden;
    const int rank = (int)cluster_ctarank();
    float *part = reinterpret_cast<float *>(smem + L.part);
    const int steps = (H + KS - 1) / KS, slices = kMoeCluster * ksub;
    const int esz = p.router_f32 ? 4 : 2;
    if (warp < kMoeWarps) {
        for (int u = warp; u < mt_n * ksub; u += kMoeWarps) {
            const int mt = u / ksub, ks = u - mt * ksub, sl = rank * ksub + ks;
            const uint8_t *w0 = static_cast<const uint8_t *>(p.router) +
                                (size_t)min(mt * 16 + g, p.experts - 1) * H * esz;
            const uint8_t *w1 = static_cast<const uint8_t *>(p.router) +
                                (size_t)min(mt * 16 + g + 8, p.experts - 1) * H * esz;
            float acc[NT][4] = {};
            for (int st = sl * steps / slices; st < (sl + 1) * steps / slices; ++st) {
#pragma unroll
                for (int pc = 0; pc < 2; ++pc) {
                    const int k = st * KS + pc * 32 + t * EP, n = H - k;
                    uint32_t a0[3][EP / 2], a1[3][EP / 2];
                    if (p.router_f32) {
                        MoeX<LL_T_F32>::load<EP>(w0, k, n, p.router_vec, a0);
                        MoeX<LL_T_F32>::load<EP>(w1, k, n, p.router_vec, a1);
                    } else {
                        MoeX<LL_T_BF16>::load<EP>(w0, k, n, p.router_vec,
                                                  reinterpret_cast<uint32_t(&)[1][EP / 2]>(a0[0]));
                        MoeX<LL_T_BF16>::load<EP>(w1, k, n, p.router_vec,
                                                  reinterpret_cast<uint32_t(&)[1][EP / 2]>(a1[0]));
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        if (nt < ntc) {
                            uint32_t b[X::NS][EP / 2];
                            const int row = min(nt * 8 + g, p.rows - 1);
                            X::template load<EP>(static_cast<const uint8_t *>(p.x) + (size_t)row * p.ldx * X::BYTES, k,
                                                 n, p.x_vec, b);
#pragma unroll
                            for (int ra = 0; ra < 3; ++ra)
                                if (ra == 0 || p.router_f32) {
#pragma unroll
                                    for (int s = 0; s < X::NS; ++s)
#pragma unroll
                                        for (int j = 0; j < EP / 4; ++j)
                                            mma_bf16(acc[nt], a0[ra][2 * j], a1[ra][2 * j], a0[ra][2 * j + 1],
                                                     a1[ra][2 * j + 1], b[s][2 * j], b[s][2 * j + 1]);
                                }
                        }
                }
            }
            float *o = part + (size_t)(ks * mt_n + mt) * 16 * tp;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                if (nt < ntc) {
                    const int c = nt * 8 + 2 * t;
                    o[g * tp + c] = acc[nt][0];
                    o[g * tp + c + 1] = acc[nt][1];
                    o[(g + 8) * tp + c] = acc[nt][2];
                    o[(g + 8) * tp + c + 1] = acc[nt][3];
                }
        }
    }
    __syncwarp();
    cluster_sync();
    float *logits = reinterpret_cast<float *>(smem + L.logits);
    const uint32_t pa = smem_u32(part);
    for (int i = tid; i < p.rows * p.experts; i += kMoeThreads) {
        const int row = i / p.experts, e = i - row * p.experts;
        float v = 0.0f;
        for (int ks = 0; ks < ksub; ++ks) {
            const uint32_t at = pa + (uint32_t)((ks * mt_n * 16 + e) * tp + row) * 4u;
            float q[kMoeCluster];
#pragma unroll
            for (int r = 0; r < kMoeCluster; ++r)
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(q[r]) : "r"(mapa(at, (uint32_t)r)) : "memory");
#pragma unroll
            for (int r = 0; r < kMoeCluster; ++r)
                v += q[r];
        }
        logits[row * p.experts + e] = v;
    }
    // the peers' partial sums are read; matched by the wait at the kernel's end
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    __syncthreads();
}

// A float as an unsigned number of the same order, NaN lowest; never 0.
__device__ __forceinline__ uint32_t order_key(float v)
{
    const uint32_t u = __float_as_uint(v);
    if (v != v)
        return 1u;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);  // -inf: 0x007fffff
}

// ---- the top_k experts of each row and their weights (one warp per row) ----
__device__ __forceinline__ void moe_pick(const MoeParams &p, uint8_t *smem, const MoeSmem &L)
{
    constexpr int PER = LL_MOE_MAX_EXPERTS / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *ids = reinterpret_cast<int *>(smem + L.ids);
    float *probs = reinterpret_cast<float *>(smem + L.probs);
    for (int row = warp; row < p.rows; row += kMoeThreads / 32) {
        const float *lg = reinterpret_cast<const float *>(smem + L.logits) + row * p.experts;
        uint32_t key[PER];
        float l[PER];
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane + 32 * i;
            l[i] = e < p.experts ? lg[e] : -INFINITY;
            key[i] = e < p.experts ? order_key(l[i]) : 0u;
            top = fmaxf(top, l[i]);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1)
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        float sum = 0.0f;
        if (!p.renorm) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (lane + 32 * i < p.experts)
                    sum += expf(l[i] - top);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1)
                sum += __shfl_xor_sync(0xffffffffu, sum, off);
        }
        float mine = 0.0f;  // lane j: exp of the j-th picked logit
        for (int j = 0; j < p.top_k; ++j) {
            uint32_t best = 0u;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                best = max(best, key[i]);
            best = __reduce_max_sync(0xffffffffu, best);
            uint32_t at = 0xffffffffu;
#pragma unroll
            for (int i = PER - 1; i >= 0; --i)
                if (key[i] == best && key[i] != 0u)
                    at = (uint32_t)(lane + 32 * i);
            at = __reduce_min_sync(0xffffffffu, at);
            const float ex = expf(lg[at] - top);
            if (lane == j)
                mine = ex;
            if (p.renorm)
                sum += ex;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (at == (uint32_t)(lane + 32 * i))
                    key[i] = 0u;
            if (lane == 0)
                ids[row * p.top_k + j] = (int)at;
        }
        if (lane < p.top_k)
            probs[row * p.top_k + lane] = mine / sum;
    }
    __syncthreads();
}

// ---- kernel 1: router, choice, and the activations of the picked experts ----
template <int WT, int XT, int NT>
__global__ void __launch_bounds__(kMoeThreads, 1) ll_moe_up_kernel(const __grid_constant__ MoeParams p)
{
    using W = MoeW<WT>;
    using X = MoeX<XT>;
    constexpr int NSH = XT == LL_T_F32 ? 3 : 2;  // bf16 terms of an activation
    extern __shared__ __align__(128) uint8_t moe_smem_raw[];
    uint8_t *smem = moe_smem_raw;
    const MoeSmem L = moe_smem(p, true, NT);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint32_t *misc = reinterpret_cast<uint32_t *>(smem + L.misc);
    volatile uint32_t *fail = misc;
    const MoeRing ring = {smem_u32(smem), smem_u32(smem + L.bars), p.stages};
    if (tid == 0) {
        misc[0] = 0;
        moe_ring_init(ring);
    }
    griddep_wait();
    griddep_launch_dependents();
    __syncthreads();
    moe_logits<XT, NT>(p, smem, L);
    moe_pick(p, smem, L);
    const int n_pairs = p.rows * p.top_k;
    if (blockIdx.x == 0) {
        for (int i = tid; i < n_pairs; i += kMoeThreads) {
            const int id = reinterpret_cast<const int *>(smem + L.ids)[i];
            const float w = reinterpret_cast<const float *>(smem + L.probs)[i];
            p.ids[i] = id;
            p.probs[i] = w;
            if (p.user_ids)
                p.user_ids[i] = id;
            if (p.user_probs)
                p.user_probs[i] = w;
        }
    }
    moe_lists(p, smem, L);
    const uint16_t *act_e = reinterpret_cast<const uint16_t *>(smem + L.act_e);
    const uint16_t *act_off = reinterpret_cast<const uint16_t *>(smem + L.act_off);
    const uint16_t *pairs = reinterpret_cast<const uint16_t *>(smem + L.pairs);
    const int na = (int)misc[1], F = p.inter, H = p.hidden;

    // Tiles of ch channels (at most 8 gated, 16 not), as many rounds over the CTAs as the widest tile
    // needs and ch as small as keeps that number, so that the CTAs' shares are even.
    const int ch_max = p.gated ? 8 : 16, G = (int)gridDim.x;
    const int rounds = (int)(((long long)na * F + (long long)ch_max * G - 1) / ((long long)ch_max * G));
    int ch = min(ch_max, max(1, (int)(((long long)na * F + (long long)rounds * G - 1) / ((long long)rounds * G))));
    while (ch < ch_max && (long long)na * ((F + ch - 1) / ch) > (long long)rounds * G)
        ++ch;
    const int per_e = (F + ch - 1) / ch;
    const long long total = (long long)na * per_e;
    const int lo = (int)(total * blockIdx.x / G), hi = (int)(total * (blockIdx.x + 1) / G);
    const size_t row_bytes = (size_t)H * W::BYTES;
    // weight row r of a tile (nullptr: none), and its channel
    auto row_at = [&](int a, int f0, int r, int &f) -> const uint8_t * {
        const bool up = p.gated && r >= 8;
        const int i = up ? r - 8 : r;
        f = f0 + i;
        if (i >= ch || f >= F)
            return nullptr;
        return (up ? p.wu : p.wg) + ((size_t)act_e[a] * F + f) * row_bytes;
    };
    uint32_t it = 0;
    if (warp == kMoeWarps) {
        if (p.up_ring) {
            for (int tile = lo; tile < hi; ++tile) {
                const int a = tile / per_e, f0 = (tile - a * per_e) * ch;
                int f;
                const uint8_t *src = lane < 16 ? row_at(a, f0, lane, f) : nullptr;
                const int n_rows = __popc(__ballot_sync(0xffffffffu, src != nullptr));
                if (!moe_copy_rows(p, ring, src, (int)row_bytes, n_rows, it, fail))
                    break;
            }
            if (lane == 0)
                moe_drain(p, ring, it);
        }
    } else {
        bool ok = true;
        int buf = 0;
        for (int tile = lo; tile < hi; ++tile, buf ^= 1) {
            const int a = tile / per_e, f0 = (tile - a * per_e) * ch, e = act_e[a];
            const int pos0 = act_off[a], cnt = act_off[a + 1] - pos0, ntc = (cnt + 7) >> 3;
            const uint8_t *xrow[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                xrow[nt] = static_cast<const uint8_t *>(p.x) +
                           (size_t)(pairs[pos0 + min(nt * 8 + g, cnt - 1)] & 0xff) * p.ldx * X::BYTES;
            // rows past the tile's end: any row of the tile (their sums are not used)
            int fa, fb;
            const uint8_t *g0 = row_at(a, f0, g, fa), *g1 = row_at(a, f0, g + 8, fb);
            const uint8_t *first = row_at(a, f0, 0, fb);
            const int c0 = g0 ? f0 + g : f0;
            const int c1 = p.gated ? c0 : (g1 ? f0 + g + 8 : f0);
            g0 = g0 ? g0 : first;
            g1 = g1 ? g1 : first;
            const float *sc0 = nullptr, *sc1 = nullptr;
            if constexpr (WT == LL_W_F8) {
                const int kb = (H + kF8Block - 1) / kF8Block, fb_n = (F + kF8Block - 1) / kF8Block;
                sc0 = p.sg + ((size_t)e * fb_n + c0 / kF8Block) * kb;
                sc1 = (p.gated ? p.su : p.sg) + ((size_t)e * fb_n + c1 / kF8Block) * kb;
            }
            float acc[NT][4];
            ok = moe_rows<WT, X::NS, NT>(p, ring, smem, p.up_ring != 0, g0, g1, H, sc0, sc1, ntc, it, ok, fail, acc,
                                         [&](int nt, int k, int n, uint32_t(&b)[X::NS][W::EP / 2]) {
                                             X::template load<W::EP>(xrow[nt], k, n, p.x_vec, b);
                                         });
            float4 *red = reinterpret_cast<float4 *>(smem + L.red) + buf * (kMoeWarps * NT * 32);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                if (nt < ntc)
                    red[(warp * NT + nt) * 32 + lane] = make_float4(acc[nt][0], acc[nt][1], acc[nt][2], acc[nt][3]);
            moe_bar();
            if (ok && warp < ntc) {  // warp nt: the n-tile's sums over the warps, in their order
                float4 v = red[warp * 32 + lane];
#pragma unroll
                for (int w = 1; w < kMoeWarps; ++w) {
                    const float4 q = red[(w * NT + warp) * 32 + lane];
                    v.x += q.x, v.y += q.y, v.z += q.z, v.w += q.w;
                }
                if constexpr (WT == LL_W_I8) {
                    const float q0 = __ldg(p.sg + (size_t)e * F + c0);
                    const float q1 = __ldg((p.gated ? p.su : p.sg) + (size_t)e * F + c1);
                    v.x *= q0, v.y *= q0, v.z *= q1, v.w *= q1;
                }
                const int c = warp * 8 + 2 * t;  // columns c and c + 1 of the expert's rows
                auto put = [&](int col, int f, float val) {
                    __nv_bfloat16 *h = p.hid + (size_t)(pos0 + col) * p.hid_ld + f;
                    uint32_t w[NSH];
                    split_pair<NSH>(val, 0.0f, w);
#pragma unroll
                    for (int s = 0; s < NSH; ++s)
                        h[(size_t)s * p.hid_plane] = __ushort_as_bfloat16((unsigned short)(w[s] & 0xffffu));
                };
                if (p.gated) {
                    if (g < ch && f0 + g < F) {
                        if (c < cnt)
                            put(c, f0 + g, ops_act(v.x, p.act) * v.z);
                        if (c + 1 < cnt)
                            put(c + 1, f0 + g, ops_act(v.y, p.act) * v.w);
                    }
                } else {
                    if (g < ch && f0 + g < F) {
                        if (c < cnt)
                            put(c, f0 + g, ops_act(v.x, p.act));
                        if (c + 1 < cnt)
                            put(c + 1, f0 + g, ops_act(v.y, p.act));
                    }
                    if (g + 8 < ch && f0 + g + 8 < F) {
                        if (c < cnt)
                            put(c, f0 + g + 8, ops_act(v.z, p.act));
                        if (c + 1 < cnt)
                            put(c + 1, f0 + g + 8, ops_act(v.w, p.act));
                    }
                }
            }
        }
    }
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- kernel 2: down projection and the weighted sum ----
template <int WT, int NSH, int NT>
__global__ void __launch_bounds__(kMoeThreads, 1) ll_moe_down_kernel(const __grid_constant__ MoeParams p)
{
    using W = MoeW<WT>;
    extern __shared__ __align__(128) uint8_t moe_smem_raw[];
    uint8_t *smem = moe_smem_raw;
    const MoeSmem L = moe_smem(p, false, NT);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint32_t *misc = reinterpret_cast<uint32_t *>(smem + L.misc);
    volatile uint32_t *fail = misc;
    const MoeRing ring = {smem_u32(smem), smem_u32(smem + L.bars), p.stages};
    if (tid == 0) {
        misc[0] = 0;
        moe_ring_init(ring);
    }
    float *part = reinterpret_cast<float *>(smem + L.red);  // [warp][row][16 channels]
    for (int i = tid; i < kMoeWarps * p.rows * 16; i += kMoeThreads)
        part[i] = 0.0f;
    griddep_wait();
    int *ids = reinterpret_cast<int *>(smem + L.ids);
    float *probs = reinterpret_cast<float *>(smem + L.probs);
    for (int i = tid; i < p.rows * p.top_k; i += kMoeThreads) {
        ids[i] = __ldcg(p.ids + i);
        probs[i] = __ldcg(p.probs + i);
    }
    __syncthreads();
    moe_lists(p, smem, L);
    const uint16_t *act_e = reinterpret_cast<const uint16_t *>(smem + L.act_e);
    const uint16_t *act_off = reinterpret_cast<const uint16_t *>(smem + L.act_off);
    const uint16_t *pairs = reinterpret_cast<const uint16_t *>(smem + L.pairs);
    const int na = (int)misc[1], F = p.inter, H = p.hidden, G = (int)gridDim.x;
    const int rounds = (H + 16 * G - 1) / (16 * G), R = (H + rounds * G - 1) / (rounds * G);
    const size_t row_bytes = (size_t)F * W::BYTES;
    uint32_t it = 0;
    if (warp == kMoeWarps) {
        if (p.down_ring) {
            bool ok = true;
            for (int n0 = (int)blockIdx.x * R; n0 < H && ok; n0 += G * R) {
                const int n_rows = min(R, H - n0);
                for (int a = 0; a < na && ok; ++a) {
                    const uint8_t *src =
                        lane < n_rows ? p.wd + ((size_t)act_e[a] * H + n0 + lane) * row_bytes : nullptr;
                    ok = moe_copy_rows(p, ring, src, (int)row_bytes, n_rows, it, fail);
                }
            }
            if (lane == 0)
                moe_drain(p, ring, it);
        }
    } else {
        bool ok = true;
        float *mine = part + warp * p.rows * 16;
        for (int n0 = (int)blockIdx.x * R; n0 < H; n0 += G * R) {
            const int n_rows = min(R, H - n0);
            const int c0 = n0 + min(g, n_rows - 1), c1 = n0 + min(g + 8, n_rows - 1);
            for (int a = 0; a < na; ++a) {
                const int e = act_e[a], pos0 = act_off[a], cnt = act_off[a + 1] - pos0, ntc = (cnt + 7) >> 3;
                const __nv_bfloat16 *hrow[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    hrow[nt] = p.hid + (size_t)(pos0 + min(nt * 8 + g, cnt - 1)) * p.hid_ld;
                const uint8_t *g0 = p.wd + ((size_t)e * H + c0) * row_bytes, *g1 = p.wd + ((size_t)e * H + c1) * row_bytes;
                const float *sc0 = nullptr, *sc1 = nullptr;
                if constexpr (WT == LL_W_F8) {
                    const int kb = (F + kF8Block - 1) / kF8Block, hb = (H + kF8Block - 1) / kF8Block;
                    sc0 = p.sd + ((size_t)e * hb + c0 / kF8Block) * kb;
                    sc1 = p.sd + ((size_t)e * hb + c1 / kF8Block) * kb;
                }
                float acc[NT][4];
                ok = moe_rows<WT, NSH, NT>(
                    p, ring, smem, p.down_ring != 0, g0, g1, F, sc0, sc1, ntc, it, ok, fail, acc,
                    [&](int nt, int k, int n, uint32_t(&b)[NSH][W::EP / 2]) {
#pragma unroll
                        for (int s = 0; s < NSH; ++s) {
                            const __nv_bfloat16 *q = hrow[nt] + (size_t)s * p.hid_plane + k;
#pragma unroll
                            for (int i = 0; i < W::EP / 8; ++i) {
                                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                                if (n >= 8 * (i + 1)) {
                                    v = __ldcg(reinterpret_cast<const uint4 *>(q) + i);
                                } else if (n > 8 * i) {  // the row's last values
                                    uint32_t h[4] = {0, 0, 0, 0};
#pragma unroll
                                    for (int j = 0; j < 8; ++j)
                                        if (8 * i + j < n)
                                            h[j / 2] |= (uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(q) +
                                                                         8 * i + j)
                                                        << (16 * (j & 1));
                                    v = make_uint4(h[0], h[1], h[2], h[3]);
                                }
                                b[s][4 * i] = v.x, b[s][4 * i + 1] = v.y, b[s][4 * i + 2] = v.z, b[s][4 * i + 3] = v.w;
                            }
                        }
                    });
                if constexpr (WT == LL_W_I8) {
                    const float q0 = __ldg(p.sd + (size_t)e * H + c0), q1 = __ldg(p.sd + (size_t)e * H + c1);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        acc[nt][0] *= q0, acc[nt][1] *= q0, acc[nt][2] *= q1, acc[nt][3] *= q1;
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int c = nt * 8 + 2 * t + j;
                        if (c < cnt) {
                            const int pr = pairs[pos0 + c], row = pr & 0xff;
                            const float w = probs[row * p.top_k + (pr >> 8)];
                            mine[row * 16 + g] = fmaf(w, acc[nt][j], mine[row * 16 + g]);
                            mine[row * 16 + g + 8] = fmaf(w, acc[nt][2 + j], mine[row * 16 + g + 8]);
                        }
                    }
                __syncwarp();  // another lane may add to the same place for the next expert
            }
            moe_bar();
            for (int i = tid; i < p.rows * 16; i += kMoeWarps * 32) {
                const int row = i >> 4, r = i & 15;
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < kMoeWarps; ++w) {
                    v += part[w * p.rows * 16 + i];
                    part[w * p.rows * 16 + i] = 0.0f;
                }
                if (ok && r < n_rows) {
                    const size_t o = (size_t)row * p.ldy + n0 + r;
                    if (p.x_type == LL_T_F32)
                        static_cast<float *>(p.y)[o] = v;
                    else if (p.x_type == LL_T_BF16)
                        static_cast<__nv_bfloat16 *>(p.y)[o] = __float2bfloat16_rn(v);
                    else
                        static_cast<__half *>(p.y)[o] = __float2half_rn(v);
                }
            }
            moe_bar();
        }
    }
}

// Launches both kernels for one weight type (moe_bf16.cu, moe_i8.cu, moe_f8.cu).
int launch_moe_bf16(MoeParams &p, int device, cudaStream_t st);
int launch_moe_i8(MoeParams &p, int device, cudaStream_t st);
int launch_moe_f8(MoeParams &p, int device, cudaStream_t st);

constexpr int kMoeSmemCap = 226 * 1024;

// One kernel with its own dynamic shared memory; `cluster` CTAs per cluster (0: none).
inline int moe_launch(const void *fn, bool *ready, MoeParams &p, int smem, int grid, int cluster, bool dependent,
                      int device, cudaStream_t st)
{
    if (!__atomic_load_n(&ready[device], __ATOMIC_ACQUIRE)) {
        LL_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMoeSmemCap));
        __atomic_store_n(&ready[device], true, __ATOMIC_RELEASE);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kMoeThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (cluster) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = (unsigned)cluster;
        at[n].val.clusterDim.y = 1;
        at[n].val.clusterDim.z = 1;
        ++n;
    }
    if (dependent) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = at;
    cfg.numAttrs = (unsigned)n;
    void *args[] = {&p};
    LL_CUDA_TRY(cudaLaunchKernelExC(&cfg, fn, args));
    return LL_OK;
}

// Clusters of kernel 1 that the device holds at once, one CTA per SM.
inline int moe_clusters(const void *fn, int *n)
{
    LL_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMoeSmemCap));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kMoeCluster);
    cfg.blockDim = dim3(kMoeThreads);
    cfg.dynamicSmemBytes = kMoeSmemCap;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = kMoeCluster;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    LL_CUDA_TRY(cudaOccupancyMaxActiveClusters(n, fn, &cfg));
    if (*n < 1) {
        llh::set_error("ll_moe_forward: the device holds no cluster of %d CTAs", kMoeCluster);
        return LL_ERR_CUDA;
    }
    return LL_OK;
}

template <int WT, int XT, int NT>
int launch_moe_typed(MoeParams &p, int device, cudaStream_t st)
{
    static bool up_ready[kOpsMaxDevices], down_ready[kOpsMaxDevices];
    static int sm_count[kOpsMaxDevices], cluster_count[kOpsMaxDevices];
    constexpr int NSH = XT == LL_T_F32 ? 3 : 2;
    int sms = __atomic_load_n(&sm_count[device], __ATOMIC_ACQUIRE);
    if (sms == 0) {
        LL_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
        __atomic_store_n(&sm_count[device], sms, __ATOMIC_RELEASE);
    }
    p.stages = 0;
    const int rest_up = moe_smem(p, true, NT).total, rest_down = moe_smem(p, false, NT).total;
    p.stages = std::min(kMoeMaxStages, (kMoeSmemCap - rest_up) / kMoeStage);
    if (p.stages < 2) {
        llh::set_error("ll_moe_forward: the router of %d experts x %d rows leaves no shared memory", p.experts, p.rows);
        return LL_ERR_BAD_DESC;
    }
    // one wave of clusters: a GPC whose SMs are not a multiple of 8 leaves some out
    int clusters = __atomic_load_n(&cluster_count[device], __ATOMIC_ACQUIRE);
    if (clusters == 0) {
        LL_TRY(moe_clusters(reinterpret_cast<const void *>(&ll_moe_up_kernel<WT, XT, NT>), &clusters));
        __atomic_store_n(&cluster_count[device], clusters, __ATOMIC_RELEASE);
    }
    const int grid_up = clusters * kMoeCluster;
    LL_TRY(moe_launch(reinterpret_cast<const void *>(&ll_moe_up_kernel<WT, XT, NT>), up_ready, p,
                      moe_smem(p, true, NT).total, grid_up, kMoeCluster, false, device, st));
    p.stages = std::min(kMoeMaxStages, (kMoeSmemCap - rest_down) / kMoeStage);
    const int grid_down = std::min(sms, p.hidden);
    return moe_launch(reinterpret_cast<const void *>(&ll_moe_down_kernel<WT, NSH, NT>), down_ready, p,
                      moe_smem(p, false, NT).total, grid_down, 0, true, device, st);
}

template <int WT>
int launch_moe(MoeParams &p, int device, cudaStream_t st)
{
    const bool few = p.rows <= 8;
    switch (p.x_type) {
    case LL_T_BF16:
        return few ? launch_moe_typed<WT, LL_T_BF16, 1>(p, device, st) : launch_moe_typed<WT, LL_T_BF16, 4>(p, device, st);
    case LL_T_F16:
        return few ? launch_moe_typed<WT, LL_T_F16, 1>(p, device, st) : launch_moe_typed<WT, LL_T_F16, 4>(p, device, st);
    default:
        return few ? launch_moe_typed<WT, LL_T_F32, 1>(p, device, st) : launch_moe_typed<WT, LL_T_F32, 4>(p, device, st);
    }
}

}  // namespace llk
