// A mixture-of-experts layer for up to LL_MOE_MAX_ROWS rows in two kernels (no counterpart in the
// reference, whose net is one dense chain).
//
//   logits = Wr x;  the top_k experts of each row (ties: lowest index) with weights w from softmax
//   a[r, j] = act(Wg_e x_r) * (Wu_e x_r)          (gated; else act(Wg_e x_r)),  e = expert j of row r
//   y_r     = sum_j w[r, j] Wd_e a[r, j]
//
// With few rows the layer reads the picked experts' weights once and does little else, so both
// kernels stream weight rows from memory and multiply them on the warp-level bf16 tensor
// instruction with 16 weight rows as M and 8 of the expert's rows of x as N.  A tcgen05 tile
// (M = 128) would need each expert's rows padded to a full tile and int8 / e4m3 weights widened in
// tensor memory; at these widths the memory is the bound and the warp-level instruction is at a
// few per cent of its rate.
// Every warp works alone: it takes whole tiles (up to 16 weight rows, all columns), copies their
// rows into a ring of its own (asynchronous copies, two stages of 256 bytes of each row, refilled as
// soon as a stage is read) and keeps the tile's sums in registers.  Nothing is handed from warp to
// warp on the way, so the warps drift apart and cover each other's latencies.  For up to 8 rows two
// warps share a tile, half of its columns each, as there are few tiles then.
// Measured back to back, both kernels: 32 rows, 8 of 64 gated experts 2048 -> 1024 in bf16 (794 MB of
// weights) 185 us, 4.3 TB/s, with one layer again and again, and 260 us, 3.1 TB/s, with three layers in turn, in
// a graph as in calls: short copies (256 bytes of a row) all over 2.4 GB.  The same with e4m3 experts 421 us
// (three layers): x and the sums of four n-tiles beside the widened weights spill.  One row, 8 of 64 e4m3
// experts (50 MB) 31 us and 2 of 8 bf16 experts 1024 -> 512 15 us, of which kernel 1 spends 7 to 10 on
// logits and choice before its first weight arrives: latency.
//
// Precision: weights are exact in bf16 (int8 and e4m3 too; their scales multiply fp32 sums).  x
// and the activations a are split into bf16 terms that add up to the value: x in bf16 one, fp16
// two (exact), fp32 three (exact); a two (16 bits, below the rounding of a 16-bit y) or three
// for an fp32 layer.  All sums are fp32.
//
// Kernel 1 (clusters of 4 CTAs): every cluster computes all logits, each CTA over a quarter of the
// columns, exchanged through distributed shared memory; then each CTA picks the experts and takes
// its share of the (expert, channels) tiles: 8 gate rows and the 8 up rows of the same channels
// (so the product of the two is taken in the thread that holds both).
// Kernel 2: each CTA owns up to 16 output channels and walks all picked experts' rows of Wd for
// them; every warp keeps its own partial outputs, added in warp order at the end.
// No atomics on floating-point values: results repeat bit for bit.
#pragma once
#include <type_traits>

#include "ops_common.cuh"
#include "tc_layer.cuh"

namespace llk {

constexpr int kMoeWarps = 16;
constexpr int kMoeThreads = 32 * kMoeWarps;
constexpr int kMoeStages = 2;           // stages of a warp's ring
// Warps that share a tile, each with a part of the columns: for up to 8 rows, where a T-row layer has few
// tiles (one row of 8 experts of 1024 channels: 7 per SM), two; for more rows one.
__host__ __device__ constexpr int moe_team(int nt)
{
    return nt == 1 ? 2 : 1;
}
constexpr int kMoeCluster = 4;          // kernel 1
constexpr int kMoeStage = 5120;         // bytes of a ring stage: 16 rows of 256 + 64, or fewer longer ones
constexpr int kMoeRing = kMoeWarps * kMoeStages * kMoeStage;

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
    int up_grain, down_grain;           // weight rows start on and are multiples of so many bytes (1 .. 16)
    int *ids;                           // workspace [rows][top_k]
    float *probs;
    int *user_ids;                      // or nullptr
    float *user_probs;
    __nv_bfloat16 *hid;                 // workspace: planes [rows * top_k][hid_ld]
    long long hid_plane;
    int hid_ld;
    unsigned *status;
    unsigned long long wait_ns;
};

// ---- shared memory (byte offsets) ----
// The warps' rings from 0; kernel 1's logits lie in the same place, read before the rings fill.
struct MoeSmem {
    int bars, pairs, ids, probs, mask, act_e, act_off, misc, logits, part, team, x, total;
};

__host__ __device__ inline int moe_up16(int v)
{
    return (v + 15) & ~15;
}

__host__ __device__ inline MoeSmem moe_smem(const MoeParams &p, bool up)
{
    MoeSmem s;
    const int n = p.rows * p.top_k, picked = p.experts < n ? p.experts : n;
    int o = kMoeRing;
    s.bars = o, o += 8 * kMoeWarps * kMoeStages;
    s.misc = o, o += 16;  // number of picked experts, fail flag
    s.pairs = o, o += moe_up16(2 * n);
    s.ids = o, o += moe_up16(4 * n);
    s.probs = o, o += moe_up16(4 * n);
    s.mask = o, o += moe_up16(4 * p.experts);
    s.act_e = o, o += moe_up16(2 * picked);
    s.act_off = o, o += moe_up16(2 * (picked + 1));
    s.logits = 0;
    s.part = moe_up16(4 * p.rows * p.experts);  // kernel 1: at most 32 + 64 KB with the logits
    s.team = o, o += up ? kMoeWarps * 512 : 0;  // a team's sums on their way, two tiles'
    if (!up)
        s.part = o, o += kMoeWarps * p.rows * 16 * 4;
    s.x = o;  // the rows of x (kernel 2: the activations) where they are staged
    s.total = o;
    return s;
}
static_assert(4 * LL_MOE_MAX_ROWS * LL_MOE_MAX_EXPERTS * 2 <= kMoeRing, "logits and their parts fit the rings' place");

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

// The same, but at most the largest bf16 number: also for an infinity, whose second term is then infinite.
__device__ __forceinline__ uint32_t pack_bf16_finite(float lo, float hi)
{
    uint32_t w;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}

// (a, b) as NS packed bf16 terms each.  Three terms are an fp32 value exactly (from 2^-110 on: bf16's numbers end
// at 2^-133); two are the nearest value of 16 bits, and an infinity or NaN keeps its first term alone.
template <int NS>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&w)[NS])
{
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        w[s] = NS == 3 && s == 0 ? pack_bf16_finite(a, b) : pack_bf16(a, b);
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
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Weight types: EP values in 16 bytes; widen() gives them as EP / 2 packed bf16 pairs times UNIT
// (exact).  PERM: of every four values the pairs are (0, 2) and (1, 3), and x follows.
constexpr float kMoeF8Up = 0x1p64f, kMoeF8Back = 0x1p56f;  // 0x1p120f together

template <int WT>
struct MoeW;

template <>
struct MoeW<LL_W_BF16> {
    static constexpr int BYTES = 2, EP = 8;
    static constexpr bool PERM = false;
    static __device__ __forceinline__ void widen(const uint4 &v, uint32_t (&o)[4], uint32_t &)
    {
        o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
    }
};

template <>
struct MoeW<LL_W_I8> {
    static constexpr int BYTES = 1, EP = 16;
    static constexpr bool PERM = false;
    // A byte b = m - 128 s (s its sign bit, m the rest): bf16 0x43mm is 128 + m and 0x4300 | 128 s is
    // 128 + 128 s, so their difference, exact, is b.
    static __device__ __forceinline__ uint32_t pair(uint32_t w, uint32_t sel)
    {
        const uint32_t p = prmt(w, 0x43434343u, sel);
        return bf16x2_sub(p & 0xff7fff7fu, p & 0xff80ff80u);
    }
    static __device__ __forceinline__ void widen(const uint4 &v, uint32_t (&o)[8], uint32_t &)
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[2 * i] = pair(w[i], 0x4140u);
            o[2 * i + 1] = pair(w[i], 0x4342u);
        }
    }
};

template <>
struct MoeW<LL_W_F8> {
    static constexpr int BYTES = 1, EP = 16;
    static constexpr bool PERM = true;
    // Sign, exponent and significand moved to their bf16 places are the value times 2^-120 (the
    // exponents' biases differ by 120; e4m3's subnormals become bf16's).  x is multiplied by
    // kMoeF8Up = 2^64 beforehand, so a block's sum carries 2^-56 and is multiplied by kMoeF8Back on its
    // way to the others: x below 2^64 does not overflow in bf16, and sums from 2^-70 on are fp32's
    // normal numbers.  7 operations for 4 values, where the conversion instructions run at a fraction
    // of the rate.  NaN (0x7f) would read as 480: `nan` collects a mark (bit 7 of a byte) for it, and the
    // row's sums become NaN at the tile's end.
    static __device__ __forceinline__ void widen(const uint4 &v, uint32_t (&o)[8], uint32_t &nan)
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[2 * i] = ((w[i] << 8) & 0x80008000u) | ((w[i] << 4) & 0x07f007f0u);  // bytes 0 and 2
            o[2 * i + 1] = (w[i] & 0x80008000u) | ((w[i] >> 4) & 0x07f007f0u);     // bytes 1 and 3
            nan |= (w[i] & 0x7f7f7f7fu) + 0x01010101u;
        }
    }
};

// (v0, v1), (v2, v3) -> (v0, v2), (v1, v3)
__device__ __forceinline__ void moe_permute(uint32_t &a, uint32_t &b)
{
    const uint32_t lo = prmt(a, b, 0x5410u), hi = prmt(a, b, 0x7632u);
    a = lo;
    b = hi;
}

constexpr int moe_terms(int x_type)
{
    return x_type == LL_T_BF16 ? 1 : x_type == LL_T_F16 ? 2 : 3;
}

// Rows of x in global memory: EP consecutive values as RAW 16-byte words, and those as NS packed
// bf16 terms.
template <int XT>
struct MoeX {
    static constexpr int NS = moe_terms(XT);
    static constexpr int BYTES = XT == LL_T_F32 ? 4 : 2;
    static constexpr bool GLOBAL = true;
    template <int EP>
    static constexpr int RAW = EP * BYTES / 16;

    const uint8_t *base;
    size_t row_bytes;
    int cols;
    bool vec;  // rows start on 16 bytes

    // A thread's place in a row: pieces of EP values, 4 EP apart, from column k + t EP on.
    struct At {
        const uint8_t *row;
        int k;
    };
    template <int EP>
    __device__ __forceinline__ At at(uint32_t row, int k) const
    {
        return {base + row * row_bytes, k + (int)(threadIdx.x & 3) * EP};
    }
    template <int EP>
    __device__ __forceinline__ void piece(const At &a, int i, uint4 (&v)[RAW<EP>]) const
    {
        load<EP>(a.row, a.k + i * 4 * EP, v);
    }
    template <int EP>
    static __device__ __forceinline__ void next(At &a, int pieces)
    {
        a.k += pieces * 4 * EP;
    }

    // Values k .. k + EP - 1 of a row, zero from column `cols` on.
    template <int EP>
    __device__ __forceinline__ void load(const uint8_t *row, int k, uint4 (&v)[RAW<EP>]) const
    {
        const uint8_t *p = row + (size_t)k * BYTES;
        const int n = cols - k;
        if (vec && n >= EP) {
#pragma unroll
            for (int i = 0; i < RAW<EP>; ++i)
                v[i] = reinterpret_cast<const uint4 *>(p)[i];
        } else {
#pragma unroll 1
            for (int i = 0; i < RAW<EP>; ++i) {
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 16 / BYTES; ++j)
                    if (i * (16 / BYTES) + j < n) {
                        const uint32_t one = BYTES == 4
                                                 ? reinterpret_cast<const uint32_t *>(p)[4 * i + j]
                                                 : (uint32_t)reinterpret_cast<const uint16_t *>(p)[8 * i + j];
                        w[j * BYTES / 4] |= one << (8 * (j * BYTES % 4));
                    }
                const uint4 t = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
                for (int j = 0; j < RAW<EP>; ++j)  // v is kept in registers: no index that is not known
                    if (j == i)
                        v[j] = t;
            }
        }
    }

    template <int EP, bool PERM>
    static __device__ __forceinline__ void terms(const uint4 (&v)[RAW<EP>], uint32_t (&w)[NS][EP / 2])
    {
        const float up = PERM ? kMoeF8Up : 1.0f;
#pragma unroll
        for (int i = 0; i < RAW<EP>; ++i) {
            const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            if constexpr (BYTES == 4) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t t[NS];
                    split_pair<NS>(__uint_as_float(u[2 * j]) * up, __uint_as_float(u[2 * j + 1]) * up, t);
#pragma unroll
                    for (int s = 0; s < NS; ++s)
                        w[s][2 * i + j] = t[s];
                }
            } else if constexpr (XT == LL_T_BF16) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[0][4 * i + j] = u[j];
                    if constexpr (PERM)  // 0x5f80: 2^64
                        asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(w[0][4 * i + j]) : "r"(0x5f805f80u));
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[j]));
                    uint32_t t[NS];
                    split_pair<NS>(f.x * up, f.y * up, t);
#pragma unroll
                    for (int s = 0; s < NS; ++s)
                        w[s][4 * i + j] = t[s];
                }
            }
        }
        if constexpr (PERM)
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int j = 0; j < EP / 2; j += 2)
                    moe_permute(w[s][j], w[s][j + 1]);
    }
};

// Rows of bf16 terms, ready for the tensor instruction: planes of rows, zero behind the last column.
// SMEM: x staged in shared memory by kernel 1; else the activations in the workspace, written by
// kernel 1 while kernel 2 may already be resident, so read past L1.
template <int NSP, bool SMEM>
struct MoeTerms {
    static constexpr int NS = NSP;
    static constexpr bool GLOBAL = !SMEM;
    template <int EP>
    static constexpr int RAW = NSP * EP / 8;

    const uint8_t *base;
    size_t plane;  // bytes
    uint32_t pitch;

    struct At {
        const uint8_t *p;
    };
    template <int EP>
    __device__ __forceinline__ At at(uint32_t row, int k) const
    {
        return {base + (size_t)row * pitch + (size_t)(k + (int)(threadIdx.x & 3) * EP) * 2};
    }
    template <int EP>
    __device__ __forceinline__ void piece(const At &a, int j, uint4 (&v)[RAW<EP>]) const
    {
#pragma unroll
        for (int s = 0; s < NSP; ++s) {
            const uint4 *q = reinterpret_cast<const uint4 *>(a.p + s * plane + j * (8 * EP));
#pragma unroll
            for (int i = 0; i < EP / 8; ++i)
                v[s * (EP / 8) + i] = SMEM ? q[i] : __ldcg(q + i);
        }
    }
    template <int EP>
    static __device__ __forceinline__ void next(At &a, int pieces)
    {
        a.p += pieces * (8 * EP);
    }

    template <int EP, bool PERM>
    static __device__ __forceinline__ void terms(const uint4 (&v)[RAW<EP>], uint32_t (&w)[NSP][EP / 2])
    {
#pragma unroll
        for (int s = 0; s < NSP; ++s)
#pragma unroll
            for (int i = 0; i < EP / 8; ++i) {
                const uint4 t = v[s * (EP / 8) + i];
                w[s][4 * i] = t.x, w[s][4 * i + 1] = t.y, w[s][4 * i + 2] = t.z, w[s][4 * i + 3] = t.w;
            }
    }
};

// Columns of a row of terms: whole steps of 256 bytes of weights.
__host__ __device__ constexpr int moe_cols(int cols, int wbytes)
{
    return (cols + 256 / wbytes - 1) / (256 / wbytes) * (256 / wbytes);
}

// Bytes between rows of x in shared memory (8-bit types: the 16-byte pieces that a quarter of the
// warp reads are 32 bytes apart in a row and 16 from row to row; bf16: 16 and 64).
__host__ __device__ constexpr int moe_x_pitch(int cols, int wbytes)
{
    return 2 * moe_cols(cols, wbytes) + (wbytes == 1 ? 16 : 64);
}

// ---- the lists of picked experts, from the ids in shared memory (all threads; rows <= 32) ----
// act_e[a] = a-th picked expert (rising, but for one row by its weight), its rows are pairs[act_off[a] .. act_off[a + 1]),
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
    if (p.rows == 1) {  // the picked experts as they are
        const int i = threadIdx.x;
        if (i < n) {
            act_e[i] = (uint16_t)ids[i];
            pairs[i] = (uint16_t)(i << 8);
        }
        if (i <= n)
            act_off[i] = (uint16_t)i;
        if (i == 0)
            misc[0] = (uint32_t)n;
        __syncthreads();
        return;
    }
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
            misc[0] = (uint32_t)a0;
        }
    }
    __syncthreads();
    const int na = (int)misc[0];
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

// ---- a warp's ring of weight rows ----
// BYTES to shared memory, the first n of them from src, the others zero.
template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void *src, int n)
{
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n)
                     : "memory");
}

// A segment of a tile's rows (see MoeRing) in pieces of 16 bytes, 16 pieces (a half warp) of one row at a
// time; zeros for rows that do not exist and from byte `end` of a row on.
template <int GRAIN>
__device__ __forceinline__ void moe_copy(uint32_t dst, int rows, int m, int half, int have, const uint8_t *s0,
                                         const uint8_t *s1, int row_bytes, int off, int end)
{
    const int lane = threadIdx.x & 31, pl = (lane & 15) * 16, pitch = (256 << m) + 64;
    dst += (uint32_t)pl;
    constexpr int UN = GRAIN == 16 ? 2 : 1;
#pragma unroll UN
    for (int c = lane >> 4; c < rows << m; c += 2) {
        const int r = c >> m, sub = (c - (r << m)) << 8, at = off + pl + sub;
        const int h = r < half ? r : r - half;
        const int n = h < have ? min(16, max(0, end - at)) : 0;
        const uint8_t *src = n > 0 ? (r < half ? s0 : s1) + (size_t)h * (size_t)row_bytes + at : s0;
        const uint32_t d = dst + (uint32_t)(r * pitch + sub);
        if constexpr (GRAIN == 16) {
            cp_async<16>(d, src, n);
        } else if constexpr (GRAIN >= 4) {
#pragma unroll
            for (int i = 0; i < 16; i += GRAIN)
                cp_async<GRAIN>(d + i, n > i ? src + i : s0, n > i ? GRAIN : 0);
        } else {  // rows on odd addresses: by value
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < n)
                    w[i / 4] |= (uint32_t)src[i] << (8 * (i % 4));
            st_shared_v4(d, make_uint4(w[0], w[1], w[2], w[3]));
        }
    }
}

// n whole segments (nothing of them behind a row's end), one row or two half rows at a time: four
// instructions a copy.  m = 0 takes an even n.
__device__ __forceinline__ void moe_copy_whole(uint32_t dst, int n, int m, const uint8_t *src, int row_bytes)
{
    const int lane = threadIdx.x & 31, hw = lane >> 4, pl = (lane & 15) * 16, pitch = (256 << m) + 64;
    src += pl;
    dst += (uint32_t)pl;
    if (m == 0) {
        src += (size_t)hw * (size_t)row_bytes;
        dst += (uint32_t)(hw * pitch);
#pragma unroll 4
        for (int i = 0; i < n; i += 2, src += 2 * (size_t)row_bytes, dst += 2u * (uint32_t)pitch)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    } else {
        src += hw * 256;
        dst += (uint32_t)(hw * 256);
        for (int i = 0; i < n; ++i, src += (size_t)row_bytes, dst += (uint32_t)pitch)
#pragma unroll 2
            for (int j = 0; j < 256 << m; j += 512)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + (uint32_t)j), "l"(src + j) : "memory");
    }
}

// Rows that do not start on 16 bytes, or end within the segment: out of the way of the others' instructions.
static __device__ __noinline__ void moe_copy_small(int grain, uint32_t dst, int rows, int m, int half, int have,
                                                   const uint8_t *s0, const uint8_t *s1, int row_bytes, int off, int end)
{
    if (grain >= 16)
        moe_copy<16>(dst, rows, m, half, have, s0, s1, row_bytes, off, end);
    else if (grain >= 8)
        moe_copy<8>(dst, rows, m, half, have, s0, s1, row_bytes, off, end);
    else if (grain >= 4)
        moe_copy<4>(dst, rows, m, half, have, s0, s1, row_bytes, off, end);
    else
        moe_copy<1>(dst, rows, m, half, have, s0, s1, row_bytes, off, end);
}

// Tiles of `rows` rows come in segments of 256 << m bytes per row, m as large as 16 rows' 256 bytes
// allow (a pitch of 64 mod 128 bytes, so that the 8 rows that a quarter of the warp reads do not
// collide); what lies behind a row's end is zero up to a whole step.  The warp issues its tiles'
// segments in order, kMoeStages ahead: bulk copies on a barrier per stage for up to 4 rows, else one
// group of 16-byte (or smaller) copies per segment, empty ones past the last, so that the count of
// groups tells which has landed.
struct MoeRing {
    uint32_t base, bars;  // shared-memory addresses of this warp's stages and of a barrier for each
    uint32_t laps;        // of each stage's barrier, the phase that its next wait is for (a bit)
    uint32_t out;         // stages whose bulk copies were issued and not yet waited for (a bit)
    bool ok;              // no wait has run out; from then on nothing is issued or waited for
    bool bulk;            // up to 4 rows: bulk copies (a lane's takes 12 instructions, whatever its length)
    int rows, m, grain;
    int q, n;       // next tile to be copied, number of tiles
    int slot, off, row_bytes;
    int step0, step1, begin, end;  // the steps and the bytes of a row that are this warp's
    const uint8_t *s0, *s1;  // first row of tile q, and first of its second half (rows half ..)
    int half, have;          // rows that exist: i < have, half + i < half + have

    __device__ __forceinline__ int seg() const
    {
        return 256 << m;
    }
    __device__ __forceinline__ int pitch() const
    {
        return seg() + 64;
    }
    __device__ __forceinline__ void shape(int r)
    {
        rows = r;
        m = r > 8 ? 0 : r > 4 ? 1 : r > 2 ? 2 : r > 1 ? 3 : 4;
    }

    // This warp's part of the columns: the i-th of TEAM, whole steps of 256 bytes.
    template <int TEAM>
    __device__ __forceinline__ void part(int bytes, int i)
    {
        row_bytes = bytes;
        const int steps = (bytes + 255) >> 8, first = (steps + TEAM - 1) / TEAM;
        step0 = min(steps, i * first);
        step1 = min(steps, (i + 1) * first);
        begin = off = step0 << 8;
        end = min(bytes, step1 << 8);
        if (step0 == step1)
            n = 0;
    }

    template <class TileAt>
    __device__ __forceinline__ void feed(TileAt tile_at)
    {
        if (q < n && ok) {
            if (off == begin)
                tile_at(q, s0, s1, half, have);
            const uint32_t dst = base + (uint32_t)(slot * kMoeStage);
            if (bulk) {
                // a row's segment per lane; a barrier of the stage counts the bytes
                const int lane = threadIdx.x & 31, h = lane < half ? lane : lane - half, len = min(seg(), end - off);
                const bool mine = lane < rows && h < have;
                const int n_rows = __popc(__ballot_sync(0xffffffffu, mine));
                const uint32_t bar = bars + 8u * (uint32_t)slot, d = dst + (uint32_t)(lane * pitch());
                if (lane == 0)
                    mbar_arrive_expect_tx(bar, (uint32_t)(len * n_rows));
                out |= 1u << slot;
                __syncwarp();
                if (mine)
                    bulk_g2s(d, (lane < half ? s0 : s1) + (size_t)h * (size_t)row_bytes + off, (uint32_t)len, bar);
                if (len & 255) {  // behind a row's last byte: zeros up to a whole step
                    for (int i = len; lane < rows && i < ((len + 255) & ~255); i += 16)
                        st_shared_v4(d + (uint32_t)i, make_uint4(0u, 0u, 0u, 0u));
                    fence_proxy_async_shared();  // before a later segment's copy to the same place
                }
            } else if (grain >= 16 && have >= half && off + seg() <= end && (m > 0 || (half & 1) == 0)) {
                moe_copy_whole(dst, half, m, s0 + off, row_bytes);
                if (rows > half)
                    moe_copy_whole(dst + (uint32_t)(half * pitch()), half, m, s1 + off, row_bytes);
            } else {
                moe_copy_small(grain, dst, rows, m, half, have, s0, s1, row_bytes, off, end);
            }
            slot = slot + 1 == kMoeStages ? 0 : slot + 1;
            off += seg();
            if (off >= end) {
                off = begin;
                ++q;
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // The segment in stage `at` has landed, for the whole warp.
    __device__ __forceinline__ void wait(const MoeParams &p, int at, volatile uint32_t *fail)
    {
        if (bulk) {
            if (ok) {
                ok = ops_wait_warp(bars + 8u * (uint32_t)at, (laps >> at) & 1u, p.wait_ns, fail, p.status, 6);
                if (ok) {
                    laps ^= 1u << at;
                    out &= ~(1u << at);
                }
            }
        } else {
            asm volatile("cp.async.wait_group %0;" ::"n"(kMoeStages - 1) : "memory");
        }
        __syncwarp();
    }

    // After a wait that ran out: what is still on its way lands (or kOpsDrainNs pass) before the shared memory
    // is given back.
    __device__ __forceinline__ void drain() const
    {
        if (ok || (threadIdx.x & 31) != 0)
            return;
        const uint64_t t0 = globaltimer();
        for (int i = 0; i < kMoeStages; ++i)
            if ((out >> i) & 1u)
                ops_drain(bars + 8u * (uint32_t)i, (laps >> i) & 1u, t0);
    }
};

// This warp's ring (its stages are part of `stages`), barriers initialised; the caller synchronises.
__device__ __forceinline__ MoeRing moe_ring(uint8_t *smem, const MoeSmem &L)
{
    const int warp = threadIdx.x >> 5;
    MoeRing r = {};
    r.base = smem_u32(smem) + (uint32_t)(warp * kMoeStages * kMoeStage);
    r.bars = smem_u32(smem + L.bars) + (uint32_t)(warp * kMoeStages * 8);
    r.ok = true;
    if ((threadIdx.x & 31) == 0) {
        for (int i = 0; i < kMoeStages; ++i)
            mbar_init(r.bars + 8u * (uint32_t)i, 1);
        fence_mbar_init_cluster();
    }
    if (threadIdx.x == 0)
        *reinterpret_cast<uint32_t *>(smem + L.misc + 4) = 0;
    return r;
}

// One tile: acc = (its rows) . x over this warp's columns, in steps of 128 bytes of every row, two at a
// time (segments and x are zero up to a whole pair).  i0 / i1: places of this thread's rows g and
// g + 8 in a stage; sc0 / sc1: their e4m3 scales by 128-column block.  Refills the ring as it goes.
// The sums run on in the tensor instruction's accumulators, except that an e4m3 block's (its
// scale) and an fp32 layer's (the instruction cuts off where fp32 would round) are added in fp32.
// The loop is kept short: with 16 warps at different places in it, a body of 24 KB of code
// waited for instructions half of the time.  NT: n-tiles that are computed (of NTA that have room);
// an expert with up to 8 rows, nearly every one, takes the copy with NT = 1: in the other one the
// instructions of the n-tiles that it lacks would be issued all the same, switched off one by one.
template <int WT, int NT, int NTA, class Src, class TileAt>
__device__ __forceinline__ void moe_tile(const MoeParams &p, MoeRing &r, volatile uint32_t *fail, const uint8_t *stages,
                                         int &slot, TileAt tile_at, int i0, int i1, int K, const float *sc0,
                                         const float *sc1, int ntc, const Src &src, const uint32_t (&xrow)[NTA],
                                         float (&out)[NTA][4])
{
    using W = MoeW<WT>;
    constexpr int EP = W::EP, RAW = Src::template RAW<EP>, KS = 128 / W::BYTES, NS = Src::NS;
    // x from global memory is loaded a step ahead where the registers allow (2 x 32)
    constexpr bool PRE = Src::GLOBAL && 2 * RAW * 4 <= 32;
    constexpr bool FRESH = WT == LL_W_F8 || NS == 3;
    constexpr float back = WT == LL_W_F8 ? kMoeF8Back : 1.0f;
    const int t = threadIdx.x & 3, last = (K + kF8Block - 1) / kF8Block - 1;
    uint4 ba[PRE ? 2 : 1][RAW], bb[PRE ? 2 : 1][RAW];
    float fa0 = 1.0f, fa1 = 1.0f, fb0 = 1.0f, fb1 = 1.0f;  // e4m3: scales of rows g and g + 8
    uint32_t nan0 = 0, nan1 = 0;
    float acc[NT][4];
    typename Src::At x[NT], ahead;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
        x[nt] = src.template at<EP>(xrow[nt], 2 * r.step0 * KS);
    ahead = x[0];
    int blk = 2 * r.step0;
    auto load_step = [&](uint4(&to)[PRE ? 2 : 1][RAW], float &f0, float &f1) {
        if constexpr (PRE) {
            src.template piece<EP>(ahead, 0, to[0]);
            src.template piece<EP>(ahead, 1, to[1]);
            Src::template next<EP>(ahead, 2);
        }
        if constexpr (WT == LL_W_F8) {
            f0 = sc0[min(blk, last)];
            f1 = sc1[min(blk, last)];
            ++blk;
        }
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            acc[nt][i] = 0.0f;
    // d: the products of the first terms of x, e: those of the others (FRESH; else the same sums)
    auto products = [&](float(&d)[NT][4], float(&e)[NT][4], const uint8_t *r0, const uint8_t *r1,
                        const uint4(&b)[PRE ? 2 : 1][RAW]) {
#pragma unroll
        for (int pc = 0; pc < 2; ++pc) {
            uint32_t a0[EP / 2], a1[EP / 2];
            W::widen(*reinterpret_cast<const uint4 *>(r0 + 64 * pc), a0, nan0);
            W::widen(*reinterpret_cast<const uint4 *>(r1 + 64 * pc), a1, nan1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (NT == 1 || nt < ntc) {
                    uint32_t w[NS][EP / 2];
                    if (PRE && nt == 0) {
                        Src::template terms<EP, W::PERM>(b[pc * PRE], w);
                    } else {
                        uint4 v[RAW];
                        src.template piece<EP>(x[nt], pc, v);
                        Src::template terms<EP, W::PERM>(v, w);
                    }
#pragma unroll
                    for (int j = 0; j < EP / 4; ++j)
#pragma unroll
                        for (int s = 0; s < NS; ++s)
                            mma_bf16(s == 0 ? d[nt] : e[nt], a0[2 * j], a1[2 * j], a0[2 * j + 1], a1[2 * j + 1],
                                     w[s][2 * j], w[s][2 * j + 1]);
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            Src::template next<EP>(x[nt], 2);
    };
    auto step = [&](const uint8_t *r0, const uint8_t *r1, const uint4(&b)[PRE ? 2 : 1][RAW], float f0, float f1) {
        if constexpr (NS == 3) {
            // fp32: the large products apart from the small ones, so that fewer cuts fall on the large sums
            float d[NT][4] = {}, e[NT][4] = {};
            products(d, e, r0, r1, b);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                acc[nt][0] = fmaf((d[nt][0] + e[nt][0]) * back, f0, acc[nt][0]);
                acc[nt][1] = fmaf((d[nt][1] + e[nt][1]) * back, f0, acc[nt][1]);
                acc[nt][2] = fmaf((d[nt][2] + e[nt][2]) * back, f1, acc[nt][2]);
                acc[nt][3] = fmaf((d[nt][3] + e[nt][3]) * back, f1, acc[nt][3]);
            }
        } else if constexpr (FRESH) {
            float d[NT][4] = {};
            products(d, d, r0, r1, b);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                acc[nt][0] = fmaf(d[nt][0] * back, f0, acc[nt][0]);
                acc[nt][1] = fmaf(d[nt][1] * back, f0, acc[nt][1]);
                acc[nt][2] = fmaf(d[nt][2] * back, f1, acc[nt][2]);
                acc[nt][3] = fmaf(d[nt][3] * back, f1, acc[nt][3]);
            }
        } else {
            products(acc, acc, r0, r1, b);
        }
    };
    int st = r.step0;
    if (st < r.step1)
        load_step(ba, fa0, fa1);
    while (st < r.step1) {
        const uint8_t *at = stages + slot * kMoeStage + t * 16;
        const uint8_t *r0 = at + i0 * r.pitch(), *r1 = at + i1 * r.pitch();
        const int end = min(r.step1, st + (1 << r.m));
        r.wait(p, slot, fail);
#pragma unroll 1
        for (; st < end; ++st) {
            load_step(bb, fb0, fb1);  // on its way while the step before is computed
            step(r0, r1, ba, fa0, fa1);
            if (st + 1 < r.step1)
                load_step(ba, fa0, fa1);
            step(r0 + 128, r1 + 128, bb, fb0, fb1);
            r0 += 256;
            r1 += 256;
        }
        __syncwarp();  // every lane has read the stage
        slot = slot + 1 == kMoeStages ? 0 : slot + 1;
        r.feed(tile_at);
    }
    if constexpr (WT == LL_W_F8) {
        float s0 = 1.0f, s1 = 1.0f;
        const uint32_t lanes = 0xfu << (threadIdx.x & 28);  // the four threads of a row
        if (__ballot_sync(0xffffffffu, nan0 & 0x80808080u) & lanes)
            s0 = __uint_as_float(0x7fc00000u);
        if (__ballot_sync(0xffffffffu, nan1 & 0x80808080u) & lanes)
            s1 = __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            acc[nt][0] *= s0, acc[nt][1] *= s0, acc[nt][2] *= s1, acc[nt][3] *= s1;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            out[nt][i] = acc[nt][i];
}

// This thread's pieces of the router's rows e0 and e1 (columns k0 .. k0 + 63) as bf16 terms.
template <int RT, int NR>
__device__ __forceinline__ void moe_router_step(const MoeParams &p, uint32_t e0, uint32_t e1, int k0, uint32_t (&a0)[2][NR][4],
                                                uint32_t (&a1)[2][NR][4])
{
    using R = MoeX<RT>;
    const R src = {static_cast<const uint8_t *>(p.router), (size_t)p.hidden * R::BYTES, p.hidden, p.router_vec != 0};
    const int t = threadIdx.x & 3;
    uint4 v[2][2][R::template RAW<8>];
#pragma unroll
    for (int pc = 0; pc < 2; ++pc) {
        const int k = k0 + pc * 32 + t * 8;
        src.template load<8>(src.base + e0 * src.row_bytes, k, v[pc][0]);
        src.template load<8>(src.base + e1 * src.row_bytes, k, v[pc][1]);
    }
#pragma unroll
    for (int pc = 0; pc < 2; ++pc) {
        uint32_t w[2][NR][4];
        R::template terms<8, false>(v[pc][0], w[0]);
        R::template terms<8, false>(v[pc][1], w[1]);
#pragma unroll
        for (int s = 0; s < NR; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a0[pc][s][j] = w[0][s][j];
                a1[pc][s][j] = w[1][s][j];
            }
    }
}

// ---- router: logits of every (row, expert), by the whole cluster ----
// A warp takes 16 experts x 8 rows over a part of the columns.  One such product in the code, however many
// rows there are, and its loop not unrolled: its first pass waits for every instruction of it to come from
// memory (32 rows of 64 experts 2048 x 1024: 229 us unrolled twice, 225 not; one row of 8: 16.2, 15.7).
template <int XT, class Meanwhile>
__device__ __forceinline__ void moe_logits(const MoeParams &p, uint8_t *smem, const MoeSmem &L, Meanwhile meanwhile)
{
    using X = MoeX<XT>;
    constexpr int EP = 8, KS = 64;
    const int tid = threadIdx.x, warp = tid >> 5, g = (tid & 31) >> 2, t = tid & 3;
    constexpr int WARPS = kMoeWarps;
    const int tp = (p.rows + 7) / 8 * 8, ntc = tp / 8, H = p.hidden;
    const int mt_n = (p.experts + 15) / 16, units = mt_n * ntc, ksub = units >= WARPS ? 1 : WARPS / units;
    const int rank = (int)cluster_ctarank();
    float *part = reinterpret_cast<float *>(smem + L.part);
    const int steps = (H + KS - 1) / KS, slices = kMoeCluster * ksub;
    const X src = {static_cast<const uint8_t *>(p.x), (size_t)p.ldx * X::BYTES, H, p.x_vec != 0};
    // one copy for each type of the router, of which a launch fetches one
    auto products = [&](auto type) {
        constexpr int RT = decltype(type)::value, NR = RT == LL_T_F32 ? 3 : 1;
        for (int u = warp; u < units * ksub; u += WARPS) {
            const int ks = u / units, v = u - ks * units, mt = v / ntc, nt = v - mt * ntc, sl = rank * ksub + ks;
            const uint32_t e0 = (uint32_t)min(mt * 16 + g, p.experts - 1), e1 = (uint32_t)min(mt * 16 + g + 8, p.experts - 1);
            const uint8_t *row = src.base + (size_t)min(nt * 8 + g, p.rows - 1) * src.row_bytes;
            float acc[4] = {};
#pragma unroll 1
            for (int st = sl * steps / slices; st < (sl + 1) * steps / slices; ++st) {
                uint4 xb[2][X::template RAW<EP>];
#pragma unroll
                for (int pc = 0; pc < 2; ++pc)
                    src.template load<EP>(row, st * KS + pc * 32 + t * EP, xb[pc]);
                uint32_t a0[2][NR][EP / 2], a1[2][NR][EP / 2];
                moe_router_step<RT, NR>(p, e0, e1, st * KS, a0, a1);
                float part4[4] = {};  // each step from zero, then added in fp32
#pragma unroll
                for (int pc = 0; pc < 2; ++pc) {
                    uint32_t b[X::NS][EP / 2];
                    X::template terms<EP, false>(xb[pc], b);
#pragma unroll
                    for (int ra = 0; ra < NR; ++ra)
#pragma unroll
                        for (int s = 0; s < X::NS; ++s)
#pragma unroll
                            for (int j = 0; j < EP / 4; ++j)
                                mma_bf16(part4, a0[pc][ra][2 * j], a1[pc][ra][2 * j], a0[pc][ra][2 * j + 1],
                                         a1[pc][ra][2 * j + 1], b[s][2 * j], b[s][2 * j + 1]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[i] += part4[i];
            }
            float *o = part + (size_t)(ks * mt_n + mt) * 16 * tp + nt * 8 + 2 * t;
            o[g * tp] = acc[0];
            o[g * tp + 1] = acc[1];
            o[(g + 8) * tp] = acc[2];
            o[(g + 8) * tp + 1] = acc[3];
        }
    };
    if (p.router_f32)
        products(std::integral_constant<int, LL_T_F32>());
    else
        products(std::integral_constant<int, LL_T_BF16>());
    const int stride = mt_n * 16 * tp;
    if (ksub > 1) {  // this CTA's parts first: the peers then read one word of each CTA
        __syncthreads();
        for (int i = tid; i < stride; i += 32 * WARPS) {
            float v = part[i];
            for (int ks = 1; ks < ksub; ++ks)
                v += part[ks * stride + i];
            part[i] = v;
        }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    meanwhile();  // while the others come
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    float *logits = reinterpret_cast<float *>(smem + L.logits);
    const uint32_t pa = smem_u32(part);
    const int n_out = p.rows * p.experts;
    for (int i = tid; i < n_out; i += 32 * WARPS) {
        // consecutive threads: consecutive rows of an expert where there are several, so consecutive words
        const int e = i / p.rows, row = i - e * p.rows;
        const uint32_t at = pa + (uint32_t)(e * tp + row) * 4u;
        float q[kMoeCluster], v = 0.0f;
#pragma unroll
        for (int r = 0; r < kMoeCluster; ++r)
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(q[r]) : "r"(mapa(at, (uint32_t)r)) : "memory");
#pragma unroll
        for (int r = 0; r < kMoeCluster; ++r)
            v += q[r];
        logits[row * p.experts + e] = v;
    }
    // the peers' partial sums are read; matched by the wait before the rings fill
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
// PER experts per lane.  COUNT: an expert's place is counted, 64 steps that wait for nothing (a row alone);
// else the largest is taken top_k times, fewer instructions where every warp has rows in turn.
template <int PER, bool COUNT>
__device__ __forceinline__ void moe_pick(const MoeParams &p, uint8_t *smem, const MoeSmem &L)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *ids = reinterpret_cast<int *>(smem + L.ids);
    float *probs = reinterpret_cast<float *>(smem + L.probs);
    for (int row = warp; row < p.rows; row += (int)blockDim.x / 32) {
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
        uint32_t mine = 0;  // lane j: the j-th picked expert
        if constexpr (COUNT) {
            static_assert(PER <= 2, "two keys per lane");
            // an expert's place is the number of experts before it: by logit, of equal ones by index
            int place[PER] = {};
#pragma unroll 8
            for (int e = 0; e < p.experts; ++e) {
                const uint32_t k = __shfl_sync(0xffffffffu, PER == 2 && e >= 32 ? key[PER - 1] : key[0], e & 31);
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    place[i] += k > key[i] || (k == key[i] && e < lane + 32 * i) ? 1 : 0;
            }
            uint32_t *slots = reinterpret_cast<uint32_t *>(ids + row * p.top_k);
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (lane + 32 * i < p.experts && place[i] < p.top_k)
                    slots[place[i]] = (uint32_t)(lane + 32 * i);
            __syncwarp();
            mine = lane < p.top_k ? slots[lane] : 0u;
        } else {
#pragma unroll 1
            for (int j = 0; j < p.top_k; ++j) {
                uint32_t best = 0u, at = 0xffffffffu;
#pragma unroll
                for (int i = PER - 1; i >= 0; --i)
                    if (key[i] >= best && key[i] != 0u) {  // of equal keys the lowest index
                        best = key[i];
                        at = (uint32_t)(lane + 32 * i);
                    }
                const uint32_t top_key = __reduce_max_sync(0xffffffffu, best);
                at = __reduce_min_sync(0xffffffffu, best == top_key ? at : 0xffffffffu);
                if (lane == j)
                    mine = at;
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (at == (uint32_t)(lane + 32 * i))
                        key[i] = 0u;
            }
        }
        const float ex = lane < p.top_k ? expf(lg[mine] - top) : 0.0f;
        if (p.renorm) {
            sum = ex;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1)
                sum += __shfl_xor_sync(0xffffffffu, sum, off);
        }
        if (lane < p.top_k) {
            ids[row * p.top_k + lane] = (int)mine;
            probs[row * p.top_k + lane] = ex / sum;
        }
    }
    __syncthreads();
}

// Kernel 1: the rows of x as planes of bf16 terms in shared memory, zero behind the last column.
template <int WT, int XT>
__device__ __forceinline__ void moe_stage_x(const MoeParams &p, uint8_t *to)
{
    using W = MoeW<WT>;
    using X = MoeX<XT>;
    const int pitch = moe_x_pitch(p.hidden, W::BYTES), chunks = moe_cols(p.hidden, W::BYTES) / 8;
    const X src = {static_cast<const uint8_t *>(p.x), (size_t)p.ldx * X::BYTES, p.hidden, p.x_vec != 0};
    for (int i = threadIdx.x; i < p.rows * chunks; i += (int)blockDim.x) {
        const int row = i / chunks, c = i - row * chunks;
        uint4 v[X::template RAW<8>];
        src.template load<8>(src.base + (size_t)row * src.row_bytes, c * 8, v);
        uint32_t w[X::NS][4];
        X::template terms<8, W::PERM>(v, w);
#pragma unroll
        for (int s = 0; s < X::NS; ++s)
            *reinterpret_cast<uint4 *>(to + (size_t)(s * p.rows + row) * pitch + c * 16) =
                make_uint4(w[s][0], w[s][1], w[s][2], w[s][3]);
    }
}

// ---- kernel 1: router, choice, and the activations of the picked experts ----
// NT n-tiles of 8 rows; STAGED: x in shared memory (else it is read from global memory as it goes).
template <int WT, int XT, int NT, bool STAGED>
__global__ void __launch_bounds__(kMoeThreads, 1) ll_moe_up_kernel(const __grid_constant__ MoeParams p)
{
    using W = MoeW<WT>;
    using X = MoeX<XT>;
    constexpr int NSH = XT == LL_T_F32 ? 3 : 2;  // bf16 terms of an activation
    extern __shared__ __align__(128) uint8_t moe_smem_raw[];
    uint8_t *smem = moe_smem_raw;
    constexpr int TEAM = moe_team(NT), TEAMS = kMoeWarps / TEAM;
    const MoeSmem L = moe_smem(p, true);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    volatile uint32_t *misc = reinterpret_cast<volatile uint32_t *>(smem + L.misc);
    MoeRing ring = moe_ring(smem, L);
    // What the launches before wrote is read from here on, by plain loads: those for data that stays as it is
    // for a whole kernel may return what was there at its start.
    griddep_wait();
    griddep_launch_dependents();
    moe_logits<XT>(p, smem, L, [&] {
        if constexpr (STAGED)
            moe_stage_x<WT, XT>(p, smem + L.x);
    });
    if (p.experts <= 64)
        moe_pick<2, NT == 1>(p, smem, L);
    else
        moe_pick<LL_MOE_MAX_EXPERTS / 32, false>(p, smem, L);
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
    const int na = (int)misc[0], F = p.inter, H = p.hidden;

    // Tiles of ch channels (at most 8 gated, 16 not): as many rounds over the warps as the widest tile
    // needs, and ch as small as keeps that number, so that the warps' shares are even.
    const int ch_max = p.gated ? 8 : 16, G = (int)gridDim.x * TEAMS, me = (int)blockIdx.x * TEAMS + warp / TEAM;
    const int all = na * F;  // at most LL_MOE_MAX_ROWS LL_MOE_MAX_TOPK LL_MOE_MAX_DIM = 2^25
    const int slots = (all + ch_max * G - 1) / (ch_max * G) * G;
    int ch = min(ch_max, (all + slots - 1) / slots);
    int per_e = (F + ch - 1) / ch;
    if (ch < ch_max && na * per_e > slots) {  // every expert's last tile is short
        ++ch;
        per_e = (F + ch - 1) / ch;
    }
    const int total = na * per_e, base = total / G, rest = total - base * G;
    const int lo = me * base + min(me, rest), hi = lo + base + (me < rest ? 1 : 0);
    const size_t row_bytes = (size_t)H * W::BYTES;
    // Rows of a tile's stage: its gate rows, then (gated) the up rows of the same channels.
    auto tile_at = [&](int q, const uint8_t *&s0, const uint8_t *&s1, int &half, int &have) {
        const int tile = lo + q, a = tile / per_e, f0 = (tile - a * per_e) * ch;
        const size_t at = ((size_t)act_e[a] * F + f0) * row_bytes;
        s0 = p.wg + at;
        s1 = p.wu + (p.gated ? at : 0);
        half = ch;
        have = min(ch, F - f0);
    };
    const uint8_t *stages = smem + warp * (kMoeStages * kMoeStage);
    ring.shape(p.gated ? 2 * ch : ch);
    ring.grain = p.up_grain;
    ring.bulk = ring.grain >= 16 && ring.rows <= 4;
    ring.n = hi - lo;
    ring.part<TEAM>((int)row_bytes, warp % TEAM);
    // the rings' place still holds the logits' parts: the cluster's CTAs have read them
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    fence_proxy_async_shared();
    for (int s = 0; s < kMoeStages; ++s)
        ring.feed(tile_at);
    using Src = std::conditional_t<STAGED, MoeTerms<X::NS, true>, X>;
    Src src;
    if constexpr (STAGED) {
        const int pitch = moe_x_pitch(H, W::BYTES);
        src = {smem + L.x, (size_t)p.rows * (size_t)pitch, (uint32_t)pitch};
    } else {
        src = {static_cast<const uint8_t *>(p.x), (size_t)p.ldx * X::BYTES, H, p.x_vec != 0};
    }
    int slot = 0;
    for (int tile = lo; tile < hi; ++tile) {
        const int a = tile / per_e, f0 = (tile - a * per_e) * ch, e = act_e[a];
        const int pos0 = act_off[a], cnt = act_off[a + 1] - pos0, ntc = (cnt + 7) >> 3;
        uint32_t xrow[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            xrow[nt] = pairs[pos0 + min(nt * 8 + g, cnt - 1)] & 0xffu;
        // rows past the tile's end: its last one again (their sums are not used)
        const int chs = min(ch, F - f0), i0 = min(g, chs - 1);
        const int c0 = f0 + i0, c1 = p.gated ? c0 : f0 + min(g + 8, chs - 1);
        const int i1 = p.gated ? ch + i0 : c1 - f0;
        const float *sc0 = nullptr, *sc1 = nullptr;
        if constexpr (WT == LL_W_F8) {
            const int kb = (H + kF8Block - 1) / kF8Block, fb = (F + kF8Block - 1) / kF8Block;
            sc0 = p.sg + ((size_t)e * fb + c0 / kF8Block) * kb;
            sc1 = (p.gated ? p.su : p.sg) + ((size_t)e * fb + c1 / kF8Block) * kb;
        }
        float acc[NT][4];
        if (NT == 1 || ntc == 1)
            moe_tile<WT, 1, NT>(p, ring, misc + 1, stages, slot, tile_at, i0, i1, H, sc0, sc1, 1, src, xrow, acc);
        else
            moe_tile<WT, NT, NT>(p, ring, misc + 1, stages, slot, tile_at, i0, i1, H, sc0, sc1, ntc, src, xrow, acc);
        if constexpr (TEAM == 2) {  // the second warp's sums to the first (NT is 1)
            float4 *sums = reinterpret_cast<float4 *>(smem + L.team) + ((warp & ~1) + ((tile - lo) & 1)) * 32 + lane;
            if (warp & 1)
                *sums = make_float4(acc[0][0], acc[0][1], acc[0][2], acc[0][3]);
            asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp >> 1)) : "memory");
            if (warp & 1)
                continue;
            const float4 q = *sums;
            acc[0][0] += q.x, acc[0][1] += q.y, acc[0][2] += q.z, acc[0][3] += q.w;
        }
        float q0 = 1.0f, q1 = 1.0f;
        if constexpr (WT == LL_W_I8) {
            q0 = p.sg[(size_t)e * F + c0];
            q1 = (p.gated ? p.su : p.sg)[(size_t)e * F + c1];
        }
        // An activation into its planes, in the order that kernel 2 wants; behind the last one zeros up
        // to a whole step.
        auto put = [&](int col, int f, float val) {
            const int at = W::PERM ? (f & ~3) | ((f & 1) << 1) | ((f >> 1) & 1) : f;
            __nv_bfloat16 *h = p.hid + (size_t)(pos0 + col) * p.hid_ld + at;
            uint32_t w[NSH];
            split_pair<NSH>(W::PERM ? val * kMoeF8Up : val, 0.0f, w);
#pragma unroll
            for (int s = 0; s < NSH; ++s)
                h[(size_t)s * p.hid_plane] = __ushort_as_bfloat16((unsigned short)(w[s] & 0xffffu));
        };
        if (f0 + ch >= F)
            for (int i = lane; i < cnt * (p.hid_ld - F); i += 32)
                put(i / (p.hid_ld - F), F + i % (p.hid_ld - F), 0.0f);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt >= ntc)
                break;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = nt * 8 + 2 * t + j;  // column: one of the expert's rows of x
                const float v0 = acc[nt][j] * q0, v1 = acc[nt][2 + j] * q1;
                if (c < cnt && g < chs)
                    put(c, f0 + g, p.gated ? ops_act(v0, p.act) * v1 : ops_act(v0, p.act));
                if (!p.gated && c < cnt && g + 8 < chs)
                    put(c, f0 + g + 8, ops_act(v1, p.act));
            }
        }
    }
    ring.drain();
}

// ---- kernel 2: down projection and the weighted sum ----
// STAGED: the activations (all rows of all picked experts) in shared memory, else read from L2 as it goes.
template <int WT, int NSH, int NT, bool STAGED>
__global__ void __launch_bounds__(kMoeThreads, 1) ll_moe_down_kernel(const __grid_constant__ MoeParams p)
{
    using W = MoeW<WT>;
    extern __shared__ __align__(128) uint8_t moe_smem_raw[];
    uint8_t *smem = moe_smem_raw;
    constexpr int TEAM = moe_team(NT), TEAMS = kMoeWarps / TEAM;
    const MoeSmem L = moe_smem(p, false);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    volatile uint32_t *misc = reinterpret_cast<volatile uint32_t *>(smem + L.misc);
    MoeRing ring = moe_ring(smem, L);
    float *part = reinterpret_cast<float *>(smem + L.part);  // [warp][row][16 channels]
    for (int i = tid; i < kMoeWarps * p.rows * 16; i += kMoeThreads)
        part[i] = 0.0f;
    griddep_wait();
    griddep_launch_dependents();
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
    const int na = (int)misc[0], F = p.inter, H = p.hidden, G = (int)gridDim.x;
    const int rounds = (H + 16 * G - 1) / (16 * G), R = (H + rounds * G - 1) / (rounds * G);
    const size_t row_bytes = (size_t)F * W::BYTES;
    // The CTA's R channels and the picked experts are shared out over the warps as (expert, rs
    // channels), rs as large as leaves every warp something to do.
    int rs = R;
    while (rs > 1 && (R + rs - 1) / rs * na < TEAMS)
        rs = (rs + 1) / 2;
    const int subs = (R + rs - 1) / rs, units = subs * na;
    const int team = warp / TEAM, mine_n = units > team ? (units - team + TEAMS - 1) / TEAMS : 0;  // of this team, per item
    const int first = (int)blockIdx.x * R, items = first < H ? (H - first + G * R - 1) / (G * R) : 0;
    auto tile_at = [&](int q, const uint8_t *&s0, const uint8_t *&s1, int &half, int &have) {
        const int item = q / mine_n, u = team + (q - item * mine_n) * TEAMS;
        const int a = u / subs, r = (u - a * subs) * rs, n = first + item * G * R + r;
        s0 = s1 = p.wd + ((size_t)act_e[a] * H + min(n, H - 1)) * row_bytes;
        half = rs;
        have = min(min(rs, R - r), H - n);
    };
    const uint8_t *stages = smem + warp * (kMoeStages * kMoeStage);
    ring.shape(rs);
    ring.grain = p.down_grain;
    ring.bulk = ring.grain >= 16 && ring.rows <= 4;
    ring.n = items * mine_n;
    ring.part<TEAM>((int)row_bytes, warp % TEAM);
    for (int s = 0; s < kMoeStages; ++s)
        ring.feed(tile_at);
    MoeTerms<NSH, STAGED> src;
    if constexpr (STAGED) {
        const int pitch = moe_x_pitch(F, W::BYTES), chunks = p.hid_ld / 8, n = p.rows * p.top_k;
        for (int i = tid; i < NSH * n * chunks; i += kMoeThreads) {
            const int row = i / chunks, c = i - row * chunks, s = row / n;  // rows of all planes
            *reinterpret_cast<uint4 *>(smem + L.x + (size_t)row * pitch + c * 16) =
                __ldcg(reinterpret_cast<const uint4 *>(p.hid + (size_t)s * p.hid_plane + (size_t)(row - s * n) * p.hid_ld) + c);
        }
        __syncthreads();
        src = {smem + L.x, (size_t)n * (size_t)pitch, (uint32_t)pitch};
    } else {
        src = {reinterpret_cast<const uint8_t *>(p.hid), (size_t)p.hid_plane * 2, (uint32_t)p.hid_ld * 2u};
    }
    int slot = 0;
    float *mine = part + warp * p.rows * 16;
    for (int item = 0; item < items; ++item) {
        const int n0 = first + item * G * R, n_rows = min(R, H - n0);
        for (int u = team; u < units; u += TEAMS) {
            const int a = u / subs, rr = (u - a * subs) * rs;
            const int e = act_e[a], pos0 = act_off[a], cnt = act_off[a + 1] - pos0, ntc = (cnt + 7) >> 3;
            uint32_t hrow[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                hrow[nt] = (uint32_t)(pos0 + min(nt * 8 + g, cnt - 1));
            // rows past the end: the last one again (their sums are not used; none at all: row n0)
            const int last = max(0, min(rs, n_rows - rr) - 1), i0 = min(g, last), i1 = min(g + 8, last);
            const int c0 = min(n0 + rr + i0, H - 1), c1 = min(n0 + rr + i1, H - 1);
            const float *sc0 = nullptr, *sc1 = nullptr;
            if constexpr (WT == LL_W_F8) {
                const int kb = (F + kF8Block - 1) / kF8Block, hb = (H + kF8Block - 1) / kF8Block;
                sc0 = p.sd + ((size_t)e * hb + c0 / kF8Block) * kb;
                sc1 = p.sd + ((size_t)e * hb + c1 / kF8Block) * kb;
            }
            float acc[NT][4];
            if (NT == 1 || ntc == 1)
                moe_tile<WT, 1, NT>(p, ring, misc + 1, stages, slot, tile_at, i0, i1, F, sc0, sc1, 1, src, hrow, acc);
            else
                moe_tile<WT, NT, NT>(p, ring, misc + 1, stages, slot, tile_at, i0, i1, F, sc0, sc1, ntc, src, hrow, acc);
            float q0 = 1.0f, q1 = 1.0f;
            if constexpr (WT == LL_W_I8) {
                q0 = p.sd[(size_t)e * H + c0];
                q1 = p.sd[(size_t)e * H + c1];
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (nt >= ntc)
                    break;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int c = nt * 8 + 2 * t + j;
                    if (c < cnt) {
                        const int pr = pairs[pos0 + c], row = pr & 0xff;
                        const float w = probs[row * p.top_k + (pr >> 8)];
                        if (g < min(rs, n_rows - rr))
                            mine[row * 16 + rr + g] = fmaf(w, acc[nt][j] * q0, mine[row * 16 + rr + g]);
                        if (g + 8 < min(rs, n_rows - rr))
                            mine[row * 16 + rr + g + 8] = fmaf(w, acc[nt][2 + j] * q1, mine[row * 16 + rr + g + 8]);
                    }
                }
            }
            __syncwarp();  // another lane may add to the same place for the next expert
        }
        __syncthreads();
        for (int i = tid; i < p.rows * 16; i += kMoeThreads) {
            const int row = i >> 4, r = i & 15;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kMoeWarps; ++w) {
                v += part[w * p.rows * 16 + i];
                part[w * p.rows * 16 + i] = 0.0f;
            }
            if (misc[1] == 0 && r < n_rows) {
                const size_t o = (size_t)row * p.ldy + n0 + r;
                if (p.x_type == LL_T_F32)
                    static_cast<float *>(p.y)[o] = v;
                else if (p.x_type == LL_T_BF16)
                    static_cast<__nv_bfloat16 *>(p.y)[o] = __float2bfloat16_rn(v);
                else
                    static_cast<__half *>(p.y)[o] = __float2half_rn(v);
            }
        }
        __syncthreads();
    }
    ring.drain();
}

// Launches both kernels for one weight type (moe_bf16.cu, moe_i8.cu, moe_f8.cu).
int launch_moe_bf16(MoeParams &p, int device, cudaStream_t st);
int launch_moe_i8(MoeParams &p, int device, cudaStream_t st);
int launch_moe_f8(MoeParams &p, int device, cudaStream_t st);

constexpr int kMoeSmemCap = 226 * 1024;

template <int WT, int XT>
int moe_x_bytes(const MoeParams &p)
{
    const long long b = (long long)moe_terms(XT) * p.rows * moe_x_pitch(p.hidden, MoeW<WT>::BYTES);
    return (int)std::min<long long>(b, 1 << 24);
}

// One kernel with its own dynamic shared memory; `cluster` CTAs per cluster (0: none).
inline int moe_launch(const void *fn, bool *ready, MoeParams &p, int smem, int grid, int cluster, int device,
                      cudaStream_t st)
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
    // its CTAs may take their places as the launch before it leaves, and wait there for its end
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
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

template <int WT, int XT, int NT, bool STAGED>
int launch_moe_typed(MoeParams &p, int device, cudaStream_t st)
{
    static bool up_ready[kOpsMaxDevices], down_ready[2][kOpsMaxDevices];
    static int sm_count[kOpsMaxDevices], cluster_count[kOpsMaxDevices];
    constexpr int NSH = XT == LL_T_F32 ? 3 : 2;
    const void *up = reinterpret_cast<const void *>(&ll_moe_up_kernel<WT, XT, NT, STAGED>);
    const long long staged_h = moe_smem(p, false).total +
                               (long long)NSH * p.rows * p.top_k * moe_x_pitch(p.inter, MoeW<WT>::BYTES);
    const bool stage_h = NT == 1 && staged_h <= kMoeSmemCap;
    const void *down = stage_h ? reinterpret_cast<const void *>(&ll_moe_down_kernel<WT, NSH, NT, NT == 1>)
                               : reinterpret_cast<const void *>(&ll_moe_down_kernel<WT, NSH, NT, false>);
    int sms = __atomic_load_n(&sm_count[device], __ATOMIC_ACQUIRE);
    if (sms == 0) {
        LL_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
        __atomic_store_n(&sm_count[device], sms, __ATOMIC_RELEASE);
    }
    // one wave of clusters: a GPC whose SMs are not a multiple of the cluster leaves some out
    int clusters = __atomic_load_n(&cluster_count[device], __ATOMIC_ACQUIRE);
    if (clusters == 0) {
        LL_TRY(moe_clusters(up, &clusters));
        __atomic_store_n(&cluster_count[device], clusters, __ATOMIC_RELEASE);
    }
    LL_TRY(moe_launch(up, up_ready, p, moe_smem(p, true).total + (STAGED ? moe_x_bytes<WT, XT>(p) : 0),
                      clusters * kMoeCluster, kMoeCluster, device, st));
    return moe_launch(down, down_ready[stage_h], p, stage_h ? (int)staged_h : moe_smem(p, false).total,
                      std::min(sms, p.hidden), 0, device, st);
}

// Up to 8 rows whose terms fit beside the rings take the kernel that stages x.
template <int WT, int XT>
int launch_moe_rows(MoeParams &p, int device, cudaStream_t st)
{
    if (p.rows <= 8 && moe_smem(p, true).total + moe_x_bytes<WT, XT>(p) <= kMoeSmemCap)
        return launch_moe_typed<WT, XT, 1, true>(p, device, st);
    return launch_moe_typed<WT, XT, 4, false>(p, device, st);
}

template <int WT>
int launch_moe(MoeParams &p, int device, cudaStream_t st)
{
    switch (p.x_type) {
    case LL_T_BF16:
        return launch_moe_rows<WT, LL_T_BF16>(p, device, st);
    case LL_T_F16:
        return launch_moe_rows<WT, LL_T_F16>(p, device, st);
    default:
        return launch_moe_rows<WT, LL_T_F32>(p, device, st);
    }
}

}  // namespace llk
