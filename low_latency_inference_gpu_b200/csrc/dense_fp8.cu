// ll_dense_fp8: y = act(W x + b) on e4m3 operands (no counterpart in the reference, whose dense
// layers are fp32: include/ll/dense_warp.cuh:33-90; the layer contract is the same).
//
//   y[r, m] = act( sum_kb sx[r, kb] sw[m / 128, kb] ( sum_{k in kb} x[r, k] W[m, k] ) + b[m] )
//
// with kb the 128-column blocks of K.  A block's products are summed by the tensor cores
// (tcgen05.mma kind::f8f6f4, fp32 accumulator in TMEM), started afresh for every block; the
// block's two scales multiply the sum on its way into a second accumulator in registers.
#include <algorithm>
#include <cstring>

#include "ops_common.cuh"
#include "tc_layer.cuh"
#include "tc_swap2.cuh"
#include "tmap.h"

namespace llk {

struct DenseF8Params {
    CUtensorMap tm_w;   // e4m3 [M][K], box {128, 128}, 128-byte swizzle
    CUtensorMap tm_x;   // e4m3 [rows][K], box {128, NT}, 128-byte swizzle
    const float *sw;    // [ceil(M / 128)][nkb]
    const float *sx;    // [rows][nkb]
    const float *bias;  // [M] or nullptr
    void *y;
    float *sy;          // [rows][ceil(M / 128)] (e4m3 output)
    long long ldy;
    int rows, M, nkb, kb_split;  // kb_split: K blocks per CTA of the cluster
    int act, y_type, y_vec;      // y_vec: 4 consecutive outputs may be stored at once
    unsigned *status;
    unsigned long long wait_ns;
};

// Instruction descriptor, kind::f8f6f4: A = B = e4m3, D = fp32, both K-major, M = 128, N = n.
__host__ __device__ constexpr uint32_t tc_idesc_e4m3(int n)
{
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ void tc_mma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 32 lanes x 16 consecutive fp32 columns, waited for.
__device__ __forceinline__ void tc_ld_16cols(uint32_t taddr, float (&v)[16])
{
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i)
        v[i] = __uint_as_float(r[i]);
}

// Four consecutive outputs of row `row` from channel m on; a warp holds one row's 128 channels of
// one tile (lane l: 4 l ..), so the e4m3 output's group maximum is a warp reduction.
__device__ __forceinline__ void store_y4(const DenseF8Params &p, long long row, int m, float (&v)[4], int mtile)
{
    const int have = p.M - m;  // <= 0: past the last channel
    if (p.y_type == LL_T_F8) {
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < have)
                amax = fmaxf(amax, fabsf(v[i]));
#pragma unroll
        for (int off = 16; off > 0; off >>= 1)
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        float s, inv;
        e4m3_scale(amax, false, s, inv);
        const uint32_t o = group_e4m3x4(v, false, s, inv);
        uint8_t *q = static_cast<uint8_t *>(p.y) + row * p.ldy + m;
        if (have >= 4 && p.y_vec) {
            *reinterpret_cast<uint32_t *>(q) = o;
        } else {
            for (int i = 0; i < 4; ++i)
                if (i < have)
                    q[i] = (uint8_t)(o >> (8 * i));
        }
        if ((threadIdx.x & 31) == 0)
            p.sy[row * ((p.M + kF8Block - 1) / kF8Block) + mtile] = s;
    } else if (p.y_type == LL_T_F32) {
        float *q = static_cast<float *>(p.y) + row * p.ldy + m;
        if (have >= 4 && p.y_vec) {
            *reinterpret_cast<float4 *>(q) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            for (int i = 0; i < 4; ++i)
                if (i < have)
                    q[i] = v[i];
        }
    } else {
        uint16_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            h[i] = p.y_type == LL_T_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v[i]))
                                         : __half_as_ushort(__float2half_rn(v[i]));
        uint16_t *q = static_cast<uint16_t *>(p.y) + row * p.ldy + m;
        if (have >= 4 && p.y_vec) {
            *reinterpret_cast<uint2 *>(q) =
                make_uint2((uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16));
        } else {
            for (int i = 0; i < 4; ++i)
                if (i < have)
                    q[i] = h[i];
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Few rows: D[128 channels x NT rows] = W tile . X^T, so a weight tile is the MMA's A operand and
// few rows are a narrow N.  The K blocks of a tile are split over the CTAs of one cluster (grid z);
// each CTA sends the sums of every row to the CTA that owns the row (rank = row mod splits), through
// distributed shared memory, and the owner adds them in rank order.  Latency is what counts here:
//   * up to 8 accumulators in tensor memory, so that the MMAs of all K blocks of a CTA are issued
//     as their operands land and wait for nobody;
//   * 4 stages of 18 KB at 16 rows, so that two CTAs fit an SM and the next launch's set-up
//     (barriers, tensor memory, tensor maps) runs beside this one's end (programmatic dependent launch).
// Back to back in a graph: 1 x 2048 x 2048 4.0 us, 32 x 4096 x 4096 with e4m3 output 6.7 (16.8 MB of weights, 2.5
// TB/s), 256 x 2048 x 2048 7.8.
//   warp 0     TMA producer (W box 16 KB + X box NT * 128 B per K block)
//   warp 1     TMEM allocation; one lane issues the MMAs
//   warps 2-5  lane = channel: TMEM -> registers, times the block's scales
//   all        sums of this CTA's rows, bias, activation, store
constexpr int kDsThreads = 192;
constexpr int kDsScaleKb = 8;  // K blocks whose scales are staged at once

template <int NT>
struct DsSmem {
    static constexpr int WB = 128 * kF8Block;
    static constexpr int XB = NT * kF8Block;
    static constexpr int STAGE = WB + XB;
    static constexpr int STAGES = NT <= 32 ? 4 : 5;
    static constexpr int ACC = NT <= 32 ? 8 : 4;                   // accumulators
    static constexpr uint32_t TMEM_COLS = ACC * NT;                // 128, 256 or 512
    static constexpr int OFF_SC = STAGES * STAGE;                  // sx * sw: [4 warps][kDsScaleKb][NT] fp32
    static constexpr int OFF_PART = NT <= 32 ? OFF_SC + 4 * kDsScaleKb * NT * 4 : 0;  // [NT][128] fp32
    // full[S], empty[S], accfull[A], accempty[A], done
    static constexpr int OFF_BAR = OFF_SC + 4 * kDsScaleKb * NT * 4 + (NT <= 32 ? NT * 512 : 0);
    static constexpr int N_BAR = 2 * STAGES + 2 * ACC + 1;
    static constexpr int OFF_MISC = OFF_BAR + 8 * N_BAR;           // tmem base, fail flag
    static constexpr int ALLOC = OFF_MISC + 16 + 1024;
    // NT <= 32: a place of its own for the received sums; else in the ring, once the whole cluster has
    // read its last stage
    static constexpr bool OWN_PART = NT <= 32;
    static_assert(OWN_PART || NT * 512 <= STAGES * STAGE, "the sums fit the ring");
    static_assert(ALLOC <= 227 * 1024, "shared memory");
    // CTAs that fit an SM together find tensor memory together: a cluster never holds some of it while
    // another one waits for it on the next SM.
    static_assert(2 * TMEM_COLS <= 512 || 2 * ALLOC > 227 * 1024, "tensor memory for the CTAs that fit");
    static_assert(3 * ALLOC > 227 * 1024, "at most two CTAs fit");
};

__device__ __forceinline__ void cluster_arrive()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}

__device__ __forceinline__ void cluster_wait()
{
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t cluster_addr)
{
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
    return v;
}

__device__ __forceinline__ void st_cluster_f32(uint32_t cluster_addr, float v)
{
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}

// The sums of the rows of this CTA (row c of the tile at slot c / SPLITS, rank r's share at [slot][r]).
template <int NT, int SPLITS>
__device__ __forceinline__ void ds_finish(const DenseF8Params &p, const float *part, long long t0, int rank, int mtile)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, m = mtile * 128 + 4 * lane;
    float bias[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        bias[i] = p.bias && m + i < p.M ? p.bias[m + i] : 0.0f;
    const int mine = (int)min((long long)(NT - rank + SPLITS - 1) / SPLITS,
                              (p.rows - t0 - rank + SPLITS - 1) / SPLITS);  // rows c = rank + SPLITS slot that exist
    for (int slot = warp; slot < mine; slot += kDsThreads / 32) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < SPLITS; ++r) {
            const float4 q = *reinterpret_cast<const float4 *>(part + (slot * SPLITS + r) * 128 + 4 * lane);
            v[0] += q.x, v[1] += q.y, v[2] += q.z, v[3] += q.w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] += bias[i];
            v[i] = ops_act(v[i], p.act);
        }
        store_y4(p, t0 + rank + SPLITS * slot, m, v, mtile);
    }
}

template <int NT>
__global__ void __launch_bounds__(kDsThreads, 1) ll_dense_fp8_kernel(const __grid_constant__ DenseF8Params p)
{
    using L = DsSmem<NT>;
    constexpr int S = L::STAGES, A = L::ACC;
    extern __shared__ uint8_t ds_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(ds_smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t *misc = reinterpret_cast<uint32_t *>(smem + L::OFF_MISC);
    volatile uint32_t *fail = misc + 1;
    float *s_sc = reinterpret_cast<float *>(smem + L::OFF_SC);
    float *s_part = reinterpret_cast<float *>(smem + L::OFF_PART);
    auto bar = [&](int i) { return sbase + (uint32_t)L::OFF_BAR + 8u * (uint32_t)i; };
    auto b_full = [&](int s) { return bar(s); };
    auto b_empty = [&](int s) { return bar(S + s); };
    auto b_accf = [&](int b) { return bar(2 * S + b); };
    auto b_acce = [&](int b) { return bar(2 * S + A + b); };
    const uint32_t b_done = bar(2 * S + 2 * A);

    const int splits = (int)gridDim.z, rank = (int)blockIdx.z;  // the cluster is the z extent
    const int mtile = blockIdx.x, m0 = mtile * 128;
    const long long t0 = (long long)blockIdx.y * NT;
    const int kb0 = rank * p.kb_split, nkb = max(0, min(p.kb_split, p.nkb - kb0));

    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(b_full(s), 1);
            mbar_init(b_empty(s), 1);
        }
        for (int b = 0; b < A; ++b) {
            mbar_init(b_accf(b), 1);
            mbar_init(b_acce(b), 4);
        }
        mbar_init(b_done, 1);
        misc[1] = 0;
        fence_mbar_init_cluster();
        prefetch_tmap(&p.tm_w);
        prefetch_tmap(&p.tm_x);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         sbase + (uint32_t)L::OFF_MISC),
                     "r"(L::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = misc[0];
    // Operands, scales and outputs belong to the launches before until here; so they are read by plain loads,
    // not by those for data that stays as it is for a whole kernel.
    griddep_wait();
    griddep_launch_dependents();
    if (splits > 1 && L::OWN_PART)
        cluster_arrive();  // this CTA runs: its shared memory may be written to

    int issued = 0;  // producer: K blocks whose loads were started
    if (warp == 0) {
        if (lane == 0) {
            for (int j = 0; j < nkb; ++j) {
                const int s = j % S;
                if (j >= S && !ops_wait(b_empty(s), ((j / S) - 1) & 1, p.wait_ns, fail, p.status, 1))
                    break;
                mbar_arrive_expect_tx(b_full(s), L::STAGE);
                tma_load_2d(sbase + s * L::STAGE, &p.tm_w, (kb0 + j) * kF8Block, m0, b_full(s));
                tma_load_2d(sbase + s * L::STAGE + L::WB, &p.tm_x, (kb0 + j) * kF8Block, (int)t0, b_full(s));
                issued = j + 1;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        constexpr uint32_t idesc = tc_idesc_e4m3(NT);
        const uint64_t da = sw128_kmajor_desc(sbase), db = sw128_kmajor_desc(sbase + L::WB);
        const bool one = elect_one();
        for (int j = 0; j < nkb; ++j) {
            const int s = j % S, b = j % A;
            if ((j >= A && !ops_wait_warp(b_acce(b), ((j / A) - 1) & 1, p.wait_ns, fail, p.status, 2)) ||
                !ops_wait_warp(b_full(s), (j / S) & 1, p.wait_ns, fail, p.status, 3))
                break;
            tc_fence_after();
            if (one) {
                const uint64_t off = (uint64_t)(s * (L::STAGE >> 4));
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    tc_mma_f8(tmem + (uint32_t)(b * NT), da + off + 2 * kk, db + off + 2 * kk, idesc, kk != 0);
                tc_commit(b_empty(s));
                tc_commit(b_accf(b));
            }
            __syncwarp();
        }
        if (one)
            tc_commit(b_done);
        __syncwarp();
    } else {
        const int quad = warp & 3, chan = 32 * quad + lane;
        float *w_sc = s_sc + quad * (kDsScaleKb * NT);
        const float *sw = p.sw + (size_t)mtile * p.nkb + kb0;
        float acc[NT];
#pragma unroll
        for (int c = 0; c < NT; ++c)
            acc[c] = 0.0f;
        bool ok = true;
        for (int j = 0; j < nkb; ++j) {
            if (j % kDsScaleKb == 0) {  // the next blocks' scales, a copy per warp: no warp waits for another
                const int n = min(kDsScaleKb, nkb - j);
                float f[kDsScaleKb];
#pragma unroll
                for (int jj = 0; jj < kDsScaleKb; ++jj)
                    f[jj] = jj < n ? sw[j + jj] : 0.0f;
                __syncwarp();
#pragma unroll
                for (int c0 = 0; c0 < NT; c0 += 32) {  // a row's blocks per lane, all loads at once
                    const int c = c0 + lane;
                    const long long row = t0 + c;
                    const float *px = p.sx + row * p.nkb + kb0 + j;
                    float v[kDsScaleKb];
#pragma unroll
                    for (int jj = 0; jj < kDsScaleKb; ++jj)
                        v[jj] = c < NT && row < p.rows && jj < n ? px[jj] : 0.0f;
                    if (c < NT)
#pragma unroll
                        for (int jj = 0; jj < kDsScaleKb; ++jj)
                            w_sc[jj * NT + c] = v[jj] * f[jj];
                }
                __syncwarp();
            }
            const int b = j % A;
            ok = ops_wait_warp(b_accf(b), (j / A) & 1, p.wait_ns, fail, p.status, 4);
            if (!ok)
                break;
            tc_fence_after();
            const float *sc = w_sc + (j % kDsScaleKb) * NT;
#pragma unroll
            for (int c0 = 0; c0 < NT; c0 += 16) {
                float v[16];
                tc_ld_16cols(tmem + ((uint32_t)(32 * quad) << 16) + (uint32_t)(b * NT + c0), v);
#pragma unroll
                for (int c = 0; c < 16; c += 4) {
                    const float4 f = *reinterpret_cast<const float4 *>(sc + c0 + c);
                    acc[c0 + c] = fmaf(v[c], f.x, acc[c0 + c]);
                    acc[c0 + c + 1] = fmaf(v[c + 1], f.y, acc[c0 + c + 1]);
                    acc[c0 + c + 2] = fmaf(v[c + 2], f.z, acc[c0 + c + 2]);
                    acc[c0 + c + 3] = fmaf(v[c + 3], f.w, acc[c0 + c + 3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive_local(b_acce(b));
        }
        // every MMA of this CTA has read its stage
        ops_wait_warp(b_done, 0, p.wait_ns, fail, p.status, 5);
        if (splits > 1) {
            if (!L::OWN_PART)
                cluster_arrive();  // its ring may be written to
            cluster_wait();
        }
        // row c's sums of this CTA to the owner's [c / splits][rank]
        const uint32_t part = smem_u32(s_part) + (uint32_t)chan * 4u;
        if (splits == 1) {
#pragma unroll
            for (int c = 0; c < NT; ++c)
                s_part[c * 128 + chan] = acc[c];
        } else {
            const int log2 = 31 - __clz(splits), mask = splits - 1;
#pragma unroll
            for (int c = 0; c < NT; ++c)
                st_cluster_f32(mapa(part + (uint32_t)((((c >> log2) << log2) + rank) * 512), (uint32_t)(c & mask)), acc[c]);
        }
    }
    __syncwarp();
    if (splits > 1 && warp < 2) {  // the producers' part of the barrier that the others have passed
        if (!L::OWN_PART)
            cluster_arrive();
        cluster_wait();
    }
    tc_fence_before();
    if (splits > 1) {
        cluster_arrive();  // this CTA's sums are with their owners
        cluster_wait();
    } else {
        __syncthreads();
    }
    // Every role has ended, so nobody gives up any more.  A CTA in which one did has loads and MMAs in flight: they
    // end before its shared and tensor memory are given back.
    if (*fail) {
        const uint64_t w0 = globaltimer();
        if (warp == 0 && lane == 0)
            for (int j = max(0, issued - S); j < issued; ++j)
                ops_drain(b_full(j % S), (j / S) & 1, w0);
        if (warp == 1 && lane == 0)
            ops_drain(b_done, 0, w0);
        __syncwarp();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::TMEM_COLS)
                     : "memory");
    }
    if (*fail == 0) {
        if (splits == 1)
            ds_finish<NT, 1>(p, s_part, t0, rank, mtile);
        else if (splits == 2)
            ds_finish<NT, 2>(p, s_part, t0, rank, mtile);
        else if (splits == 4)
            ds_finish<NT, 4>(p, s_part, t0, rank, mtile);
        else
            ds_finish<NT, 8>(p, s_part, t0, rank, mtile);
    }
}

// ---------------------------------------------------------------------------------------------
// Many rows: D[256 rows x 256 channels] = X tile . W tile^T on pairs of SMs (cta_group::2, one
// persistent cluster of two CTAs per pair), lane = row, 128 rows per CTA.  Each CTA loads its
// rows of x and half of the tile's channels; the 2-SM instruction reads the other half from the
// peer, so an SM's shared memory takes in 32 KB and gives 32 KB per K block of 512 tensor cycles,
// just its 128 bytes a cycle (a 128 x 256 tile of one SM wants 192).
// 8192 x 4096 x 4096 with GELU, back to back in a graph: bf16 output 151 us, 1820 TFLOP/s (171 called in a row for
// 70 ms, under the power cap), fp32 161, e4m3 320, whose group maxima and roundings of 128 values per thread spill.
// Of a bf16 output at 156 us the loop without the store took 125, the instructions and loads alone 91, which
// twice the measured bf16 rate would do in 82.
// The loads from TMEM follow each other without a pause, across blocks too, each beside the multiply-adds of
// the 32 columns before it (all of a block's loads and then its last sums: 167).
// A K block's way out is 32 K values per CTA from TMEM and as many multiply-adds by the block's
// scales (one factor per thread: sx of its row times sw of its 128 channels), beside the tensor
// cores' work on the next block.
//   warp 0      TMA producer (x box 16 KB + W box 16 KB per K block, 5 stages)
//   warp 1      TMEM allocation (all 512 columns, two accumulators); in CTA 0 one thread issues the MMAs
//   warps 4-11  warps 4-7 channels 0..127 of the tile, warps 8-11 the other 128: 128 sums per
//               thread in registers; at a tile's end bias, activation and a staged store
constexpr int kDlThreads = 384;
constexpr int kDlM = 128, kDlN = 256, kDlStages = 5;         // rows per CTA, channels per pair
constexpr int kDlStage = (kDlM + kDlN / 2) * kF8Block;
constexpr int kDlOut = 32 * 256;                             // staging of a warp: 32 rows of 64 fp32 values
constexpr int kDlOffOut = kDlStages * kDlStage;
constexpr int kDlOffBar = kDlOffOut + 8 * kDlOut;            // full[S], empty[S], accfull[2], accempty[2], done
constexpr int kDlOffMisc = kDlOffBar + 8 * (2 * kDlStages + 5);
constexpr int kDlAlloc = kDlOffMisc + 16 + 1024;
static_assert(kDlAlloc <= 227 * 1024, "shared memory");

// Instruction descriptor of the pair: M = 256 (128 per CTA), N = n.
__host__ __device__ constexpr uint32_t tc_idesc_e4m3_pair(int n)
{
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
}

__device__ __forceinline__ void tc_mma_f8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                               uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 2-D tensor load of this CTA's tile whose completion bytes go to an mbarrier of the pair (cluster
// address: CTA 0's barrier); no multicast.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *tm, int x, int y, uint32_t cluster_bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(cluster_bar)
        : "memory");
}

// 32 lanes x 32 consecutive fp32 columns; the wait is separate.
__device__ __forceinline__ void tc_ld_32cols_async(uint32_t taddr, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}

// Waits for the loads into r: the registers are operands, so that no use of them moves before the wait.
__device__ __forceinline__ void tc_wait_ld_32(uint32_t (&r)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// acc += v * s for 32 columns.
__device__ __forceinline__ void fma_32cols(float *acc, const uint32_t (&v)[32], float s)
{
#pragma unroll
    for (int i = 0; i < 32; ++i)
        acc[i] = fmaf(__uint_as_float(v[i]), s, acc[i]);
}

// The warp's 32 rows x 64 columns (thread = row, in registers) through its staging tile (16-byte pieces,
// piece j of row r at j ^ (r & 7) within its 128 bytes), so that 8 lanes hold a row's 64 values, 8
// each: there bias and activation are applied and the results stored, 16 bytes a lane for a
// 16-bit type, or (e4m3) put back for the threads' group maxima.  The activation runs here, on 8
// values at a time, and not on the 128 registers: one copy of its code, where one per register
// would stream tens of KB through the instruction cache.
template <int YT, int ACT>
__device__ __forceinline__ void dl_store_64cols(const DenseF8Params &p, uint8_t *out, float *acc, long long row0, int c0)
{
    // an e4m3 result is the fp32 one, quantised: the same activation, so that the two agree in every byte
    constexpr bool HALF = YT == LL_T_BF16 || YT == LL_T_F16;
    const int lane = threadIdx.x & 31, j = lane & 7, c = c0 + 8 * j, have = p.M - c;
    auto piece = [&](int r, int i) {  // 16 pieces of a row: two stretches of 8
        return reinterpret_cast<float4 *>(out + r * 256 + (i >> 3) * 128 + (((i ^ r) & 7) << 4));
    };
#pragma unroll
    for (int i = 0; i < 16; ++i)
        *piece(lane, i) = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
    float bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
        bias[e] = p.bias && e < have ? __ldg(p.bias + c + e) : 0.0f;
    __syncwarp();
    const long long left = p.rows - row0;  // rows of the tile that exist
    if (have >= 8 && (YT == LL_T_F8 || p.y_vec)) {
        constexpr int ESZ = YT == LL_T_F32 ? 4 : 2;
        uint8_t *y = static_cast<uint8_t *>(p.y) + ((row0 + (lane >> 3)) * p.ldy + c) * ESZ;
#pragma unroll 4
        for (int i = 0; i < 8; ++i, y += 4 * p.ldy * ESZ) {
            const int r = 4 * i + (lane >> 3);
            const float4 q0 = *piece(r, 2 * j), q1 = *piece(r, 2 * j + 1);
            float v[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] += bias[e];
            if constexpr (HALF && ACT == LL_ACT_GELU) {
                ops_gelu_fast(v);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] = HALF ? ops_act_fast(v[e], ACT) : ops_act(v[e], ACT);
            }
            if constexpr (YT == LL_T_F8) {
                *piece(r, 2 * j) = make_float4(v[0], v[1], v[2], v[3]);
                *piece(r, 2 * j + 1) = make_float4(v[4], v[5], v[6], v[7]);
            } else if constexpr (YT == LL_T_F32) {
                if (r < left) {
                    reinterpret_cast<float4 *>(y)[0] = make_float4(v[0], v[1], v[2], v[3]);
                    reinterpret_cast<float4 *>(y)[1] = make_float4(v[4], v[5], v[6], v[7]);
                }
            } else {
                uint32_t h[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (YT == LL_T_BF16) {
                        const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
                        h[e] = *reinterpret_cast<const uint32_t *>(&t);
                    } else {
                        const __half2 t = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
                        h[e] = *reinterpret_cast<const uint32_t *>(&t);
                    }
                }
                if (r < left)
                    *reinterpret_cast<uint4 *>(y) = make_uint4(h[0], h[1], h[2], h[3]);
            }
        }
    } else {  // the last channels, or rows that do not start on 16 bytes: value by value
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 3);
#pragma unroll 1
            for (int e = 0; e < 8; ++e) {
                float *at = reinterpret_cast<float *>(piece(r, 2 * j + (e >> 2))) + (e & 3);
                float v = *at + (p.bias && e < have ? __ldg(p.bias + c + e) : 0.0f);
                v = HALF ? ops_act_fast(v, ACT) : ops_act(v, ACT);
                const long long o = (row0 + r) * p.ldy + c + e;
                if constexpr (YT == LL_T_F8) {
                    *at = e < have ? v : 0.0f;
                } else if (r < left && e < have) {
                    if constexpr (YT == LL_T_F32)
                        static_cast<float *>(p.y)[o] = v;
                    else if constexpr (YT == LL_T_BF16)
                        static_cast<__nv_bfloat16 *>(p.y)[o] = __float2bfloat16_rn(v);
                    else
                        static_cast<__half *>(p.y)[o] = __float2half_rn(v);
                }
            }
        }
    }
    __syncwarp();
    if constexpr (YT == LL_T_F8) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float4 q = *piece(lane, i);
            acc[4 * i] = q.x, acc[4 * i + 1] = q.y, acc[4 * i + 2] = q.z, acc[4 * i + 3] = q.w;
        }
        __syncwarp();
    }
}

// The same rows' 128 columns as e4m3: a thread has a whole group, so its scale is the thread's own.
__device__ __forceinline__ void dl_store_e4m3(const DenseF8Params &p, uint8_t *out, const float (&acc)[128],
                                              long long row0, int c0)
{
    const int lane = threadIdx.x & 31, mblocks = (p.M + kF8Block - 1) / kF8Block;
    float amax = 0.0f, s, inv;
#pragma unroll
    for (int i = 0; i < 128; ++i)
        amax = fmaxf(amax, fabsf(acc[i]));  // columns past M are zero
    e4m3_scale(amax, false, s, inv);
    if (row0 + lane < p.rows)
        p.sy[(row0 + lane) * mblocks + c0 / kF8Block] = s;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        *reinterpret_cast<uint4 *>(out + lane * 128 + ((i ^ (lane & 7)) << 4)) =
            make_uint4(group_e4m3x4(acc + 16 * i, false, s, inv), group_e4m3x4(acc + 16 * i + 4, false, s, inv),
                       group_e4m3x4(acc + 16 * i + 8, false, s, inv), group_e4m3x4(acc + 16 * i + 12, false, s, inv));
    __syncwarp();
#pragma unroll 2
    for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3), j = lane & 7, have = p.M - (c0 + 16 * j);
        const uint8_t *at = out + r * 128 + ((j ^ (r & 7)) << 4);
        if (row0 + r < p.rows && have > 0) {
            uint8_t *y = static_cast<uint8_t *>(p.y) + (row0 + r) * p.ldy + c0 + 16 * j;
            if (p.y_vec && have >= 16) {
                *reinterpret_cast<uint4 *>(y) = *reinterpret_cast<const uint4 *>(at);
            } else {
                for (int e = 0; e < min(16, have); ++e)
                    y[e] = at[e];
            }
        }
    }
    __syncwarp();
}

template <int YT, int ACT>
__device__ __forceinline__ void dl_store_act(const DenseF8Params &p, uint8_t *out, float (&acc)[128], long long row0,
                                             int c0)
{
    dl_store_64cols<YT, ACT>(p, out, acc, row0, c0);
    if (c0 + 64 < p.M)
        dl_store_64cols<YT, ACT>(p, out, acc + 64, row0, c0 + 64);
    if constexpr (YT == LL_T_F8) {
        if (c0 + 64 >= p.M)
#pragma unroll
            for (int i = 64; i < 128; ++i)
                acc[i] = 0.0f;
        dl_store_e4m3(p, out, acc, row0, c0);
    }
}

template <int YT>
__device__ __forceinline__ void dl_store(const DenseF8Params &p, uint8_t *out, float (&acc)[128], long long row0, int c0)
{
    if (p.act == LL_ACT_RELU)
        dl_store_act<YT, LL_ACT_RELU>(p, out, acc, row0, c0);
    else if (p.act == LL_ACT_GELU)
        dl_store_act<YT, LL_ACT_GELU>(p, out, acc, row0, c0);
    else if (p.act == LL_ACT_SILU)
        dl_store_act<YT, LL_ACT_SILU>(p, out, acc, row0, c0);
    else
        dl_store_act<YT, LL_ACT_IDENTITY>(p, out, acc, row0, c0);
}

template <int YT>
__global__ void __launch_bounds__(kDlThreads, 1) ll_dense_fp8_large_kernel(const __grid_constant__ DenseF8Params p)
{
    constexpr int S = kDlStages;
    extern __shared__ uint8_t dl_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(dl_smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t *misc = reinterpret_cast<uint32_t *>(smem + kDlOffMisc);
    volatile uint32_t *fail = misc + 1;
    auto bar = [&](int i) { return sbase + (uint32_t)kDlOffBar + 8u * (uint32_t)i; };
    auto b_full = [&](int s) { return bar(s); };
    auto b_empty = [&](int s) { return bar(S + s); };
    auto b_accf = [&](int b) { return bar(2 * S + b); };
    auto b_acce = [&](int b) { return bar(2 * S + 2 + b); };
    const uint32_t b_done = bar(2 * S + 4);
    const uint32_t rank = cluster_ctarank();  // the pair is the cluster
    const bool lead = rank == 0u;
    const int pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1;
    const int mt_n = (p.rows + 2 * kDlM - 1) / (2 * kDlM), nt_n = (p.M + kDlN - 1) / kDlN, tiles = mt_n * nt_n;
    // Tiles in bands of 8 row tiles, rows fastest: pairs that run at once share rows of W and of x in L2.
    auto tile_at = [&](int tile, int &mt, int &nt) {
        const int band = tile / (8 * nt_n), first = band * 8, in = tile - band * 8 * nt_n;
        const int h = min(8, mt_n - first);
        nt = in / h;
        mt = first + in - nt * h;
    };

    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(b_full(s), 1);
            mbar_init(b_empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(b_accf(b), 1);
            mbar_init(b_acce(b), 16);  // CTA 0's: eight warps of each CTA
        }
        mbar_init(b_done, 1);
        misc[1] = 0;
        fence_mbar_init_cluster();
        prefetch_tmap(&p.tm_w);
        prefetch_tmap(&p.tm_x);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         sbase + (uint32_t)kDlOffMisc),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers are initialised and their tensor memory allocated
    tc_fence_after();
    const uint32_t tmem = misc[0];

    if (warp < 4) {
        // 384 threads were launched with 168 registers each: 256 x 224 + 128 x 56 is just that
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        int issued = 0;  // producer: K blocks whose loads were started
        auto load = [&](int s, int mt, int nt, int kb) {
            if (lead)
                mbar_arrive_expect_tx(b_full(s), 2 * kDlStage);  // both CTAs' loads land on this barrier
            const uint32_t full = mapa(b_full(s), 0u);
            tma_load_2d_pair(sbase + s * kDlStage, &p.tm_x, kb * kF8Block, (2 * mt + (int)rank) * kDlM, full);
            tma_load_2d_pair(sbase + s * kDlStage + kDlM * kF8Block, &p.tm_w, kb * kF8Block,
                             nt * kDlN + (int)rank * (kDlN / 2), full);
        };
        if (warp == 0) {
            if (lane == 0) {
                bool ok = true;
                for (int tile = pair; tile < tiles && ok; tile += pairs) {
                    int mt, nt;
                    tile_at(tile, mt, nt);
                    for (int kb = 0; kb < p.nkb; ++kb) {
                        const int s = issued % S;
                        if (issued >= S &&
                            !ops_wait(b_empty(s), ((issued / S) - 1) & 1, p.wait_ns, fail, p.status, 1)) {
                            ok = false;
                            break;
                        }
                        load(s, mt, nt, kb);
                        ++issued;
                    }
                }
                misc[2] = (uint32_t)issued;
            }
            __syncwarp();
        } else if (warp == 1) {
            if (lead) {  // the whole warp, so that the loop runs on uniform registers; one lane issues
                constexpr uint32_t idesc = tc_idesc_e4m3_pair(kDlN);
                const uint64_t dx = sw128_kmajor_desc(sbase), dw = sw128_kmajor_desc(sbase + kDlM * kF8Block);
                const int mine = tiles > pair ? (tiles - pair + pairs - 1) / pairs : 0, total = mine * p.nkb;
                const bool one = elect_one();
                uint32_t s = 0, s_lap = 0;   // stage, and its phase
                uint32_t b = 0, b_lap = 1;   // accumulator; a fresh barrier counts as just emptied
                bool ok = true;
                for (int g = 0; g < total; ++g) {
                    ok = ops_wait_warp(b_acce((int)b), b_lap, p.wait_ns, fail, p.status, 2) &&
                         ops_wait_warp(b_full((int)s), s_lap, p.wait_ns, fail, p.status, 3);
                    if (!ok)
                        break;
                    tc_fence_after();
                    if (one) {
                        const uint64_t ax = dx + (uint64_t)(s * (kDlStage >> 4)), aw = dw + (uint64_t)(s * (kDlStage >> 4));
                        const uint32_t acc = tmem + b * kDlN;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            tc_mma_f8_pair(acc, ax + 2 * kk, aw + 2 * kk, idesc, kk != 0);
                        tc_commit_both(b_empty((int)s));
                        tc_commit_both(b_accf((int)b));
                    }
                    __syncwarp();
                    if (++s == S) {
                        s = 0;
                        s_lap ^= 1u;
                    }
                    b ^= 1u;
                    b_lap ^= b == 0u ? 1u : 0u;
                }
                if (one)
                    tc_commit_both(b_done);
                __syncwarp();
            }
        }
        tc_fence_before();
        cluster_sync();  // every role of both CTAs has ended: nobody gives up any more
        if (warp == 0 && lane == 0) {
            const uint32_t peer = mapa(sbase + (uint32_t)kDlOffMisc, rank ^ 1u);
            if (*fail || ld_cluster_u32(peer + 4u)) {
                // The loads in flight land before the shared memory is given back.  CTA 0's barriers count both
                // CTAs' bytes, so a CTA that stopped earlier than its peer first issues what it is behind:
                // at most S blocks, each into a stage whose last MMAs had released the peer.
                const int n = max(issued, (int)ld_cluster_u32(peer + 8u));
                for (; issued < n; ++issued) {
                    const int t = issued / p.nkb;
                    int mt, nt;
                    tile_at(pair + t * pairs, mt, nt);
                    load(issued % S, mt, nt, issued - t * p.nkb);
                }
                const uint64_t w0 = globaltimer();
                for (int j = max(0, n - S); lead && j < n; ++j)
                    ops_drain(b_full(j % S), (j / S) & 1, w0);
            }
        }
        if (warp == 1 && lane == 0)
            ops_drain(b_done, 0, globaltimer());
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int quad = warp & 3, half = (warp - 4) >> 2, mblocks = (p.M + kF8Block - 1) / kF8Block;
        const uint32_t tq = tmem + ((uint32_t)(32 * quad) << 16) + (uint32_t)(half * 128);
        const bool s_vec = p.nkb % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.sx) | reinterpret_cast<uintptr_t>(p.sw)) & 15) == 0;
        uint8_t *out = smem + kDlOffOut + (warp - 4) * kDlOut;
        int g = 0;
        bool ok = true;
        for (int tile = pair; tile < tiles && ok; tile += pairs) {
            int mt, nt;
            tile_at(tile, mt, nt);
            const long long row0 = ((long long)mt * 2 + rank) * kDlM + 32 * quad;
            const int c0 = nt * kDlN + half * 128, block = c0 / kF8Block;
            const float *sx = p.sx + min(row0 + lane, (long long)p.rows - 1) * p.nkb;
            const float *sw = p.sw + (size_t)min(block, mblocks - 1) * p.nkb;
            float acc[128];
#pragma unroll
            for (int i = 0; i < 128; ++i)
                acc[i] = 0.0f;
            // the scales of four K blocks, and those of the next four on their way (multiplied when they
            // are needed).  A warp's 32 rows are 32 lines: one 16-byte load where the rows allow it
            // instead of four, each of which would hold the load unit for 32 cycles.
            float f[4], fx[4], fw[4];
            auto load_scales = [&](int kb) {
                if (s_vec) {
                    const float4 a = kb < p.nkb ? __ldg(reinterpret_cast<const float4 *>(sx + kb)) : make_float4(0, 0, 0, 0);
                    const float4 c = kb < p.nkb ? __ldg(reinterpret_cast<const float4 *>(sw + kb)) : make_float4(0, 0, 0, 0);
                    fx[0] = a.x, fx[1] = a.y, fx[2] = a.z, fx[3] = a.w;
                    fw[0] = c.x, fw[1] = c.y, fw[2] = c.z, fw[3] = c.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        fx[i] = kb + i < p.nkb ? __ldg(sx + kb + i) : 0.0f;
                        fw[i] = kb + i < p.nkb ? __ldg(sw + kb + i) : 0.0f;
                    }
                }
            };
            load_scales(0);
            uint32_t v0[32], v1[32];
#pragma unroll
            for (int i = 0; i < 32; ++i)
                v1[i] = 0u;
            float late = 0.0f;
            for (int kb0 = 0; kb0 < p.nkb && ok; kb0 += 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    f[i] = fx[i] * fw[i];
                load_scales(kb0 + 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (kb0 + i >= p.nkb)
                        break;
                    const int b = g & 1;
                    ok = ops_wait_warp(b_accf(b), (g / 2) & 1, p.wait_ns, fail, p.status, 4);
                    if (!ok)
                        break;
                    ++g;
                    tc_fence_after();
                    const float s = f[i];
                    const uint32_t at = tq + (uint32_t)(b * kDlN);
                    tc_ld_32cols_async(at, v0);
                    fma_32cols(acc + 96, v1, late);
                    tc_wait_ld_32(v0);
                    tc_ld_32cols_async(at + 32, v1);
                    fma_32cols(acc, v0, s);
                    tc_wait_ld_32(v1);
                    tc_ld_32cols_async(at + 64, v0);
                    fma_32cols(acc + 32, v1, s);
                    tc_wait_ld_32(v0);
                    tc_ld_32cols_async(at + 96, v1);
                    fma_32cols(acc + 64, v0, s);
                    tc_wait_ld_32(v1);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (lead)
                            mbar_arrive_local(b_acce(b));
                        else
                            mbar_arrive_remote_cta(mapa(b_acce(b), 0u));
                    }
                    late = s;
                }
            }
            fma_32cols(acc + 96, v1, late);
            if (ok && c0 < p.M)
                dl_store<YT>(p, out, acc, row0, c0);
        }
        tc_fence_before();
        cluster_sync();  // with the other warps' above
    }
    cluster_sync();  // the pair's MMAs are complete in both CTAs, and nobody arrives at the peer any more
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace llk

namespace {

using namespace llk;

bool f8_map(CUtensorMap *m, const void *base, int k, long long rows, long long ld, int box_rows)
{
    auto fn = llh::encode_fn();
    if (!fn)
        return false;
    cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {(cuuint32_t)kF8Block, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NT>
int launch_few(const DenseF8Params &p, int splits, int device, cudaStream_t st)
{
    static bool ready[kOpsMaxDevices];
    const void *fn = reinterpret_cast<const void *>(&ll_dense_fp8_kernel<NT>);
    if (!__atomic_load_n(&ready[device], __ATOMIC_ACQUIRE)) {
        LL_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, DsSmem<NT>::ALLOC));
        __atomic_store_n(&ready[device], true, __ATOMIC_RELEASE);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((p.M + 127) / 128), (unsigned)((p.rows + NT - 1) / NT), (unsigned)splits);
    cfg.blockDim = dim3(kDsThreads);
    cfg.dynamicSmemBytes = (size_t)DsSmem<NT>::ALLOC;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = (unsigned)splits;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    void *args[] = {const_cast<DenseF8Params *>(&p)};
    LL_CUDA_TRY(cudaLaunchKernelExC(&cfg, fn, args));
    return LL_OK;
}

template <int YT>
int launch_many(const DenseF8Params &p, int device, cudaStream_t st)
{
    static int sm_count[kOpsMaxDevices];
    const void *fn = reinterpret_cast<const void *>(&ll_dense_fp8_large_kernel<YT>);
    int sms = __atomic_load_n(&sm_count[device], __ATOMIC_ACQUIRE);
    if (sms == 0) {
        LL_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kDlAlloc));
        LL_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
        __atomic_store_n(&sm_count[device], sms, __ATOMIC_RELEASE);
    }
    const long long tiles = (long long)((p.rows + 2 * kDlM - 1) / (2 * kDlM)) * ((p.M + kDlN - 1) / kDlN);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2u * (unsigned)std::min<long long>(tiles, sms / 2));
    cfg.blockDim = dim3(kDlThreads);
    cfg.dynamicSmemBytes = kDlAlloc;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    void *args[] = {const_cast<DenseF8Params *>(&p)};
    LL_CUDA_TRY(cudaLaunchKernelExC(&cfg, fn, args));
    return LL_OK;
}

}  // namespace

extern "C" int ll_dense_fp8(const uint8_t *d_W, const float *d_sw, const float *d_b, const uint8_t *d_x,
                            const float *d_sx, void *d_y, float *d_sy, int y_type, int rows, int M, int K, int64_t ldw,
                            int64_t ldx, int64_t ldy, int act, void *stream)
{
    static const char op[] = "ll_dense_fp8";
    if (ldw == 0)
        ldw = K;
    if (ldx == 0)
        ldx = K;
    if (ldy == 0)
        ldy = M;
    if (rows < 0 || M < 1 || K < 1 || M > (1 << 24) || K > (1 << 24) || ldw < K || ldx < K || ldy < M ||
        ldw % 16 != 0 || ldx % 16 != 0 || ldw >= (1ll << 40) || ldx >= (1ll << 40)) {
        llh::set_error("%s: invalid sizes (rows=%d M=%d K=%d ldw=%lld ldx=%lld ldy=%lld; the rows of W and x start on "
                       "16 bytes)",
                       op, rows, M, K, (long long)ldw, (long long)ldx, (long long)ldy);
        return LL_ERR_INVALID_ARG;
    }
    if (act < LL_ACT_IDENTITY || act > LL_ACT_SILU || y_type < LL_T_F32 || y_type > LL_T_F8) {
        llh::set_error("%s: unknown activation %d or output type %d", op, act, y_type);
        return LL_ERR_INVALID_ARG;
    }
    if (rows > 65535 * 128) {
        llh::set_error("%s: at most %d rows in one call (rows=%d)", op, 65535 * 128, rows);
        return LL_ERR_INVALID_ARG;
    }
    if (rows == 0)
        return LL_OK;
    if (!d_W || !d_sw || !d_x || !d_sx || !d_y || (y_type == LL_T_F8 && !d_sy)) {
        llh::set_error("%s: null pointer (an e4m3 output needs its scales' address too)", op);
        return LL_ERR_INVALID_ARG;
    }
    int dev = 0;
    unsigned *status = nullptr;
    LL_TRY(llh::ops_status_words(&dev, &status));
    LL_TRY(llh::check_device_ptr(op, "W", d_W, dev, 16));
    LL_TRY(llh::check_device_ptr(op, "the scales of W", d_sw, dev, 4));
    LL_TRY(llh::check_device_ptr(op, "x", d_x, dev, 16));
    LL_TRY(llh::check_device_ptr(op, "the scales of x", d_sx, dev, 4));
    LL_TRY(llh::check_device_ptr(op, "y", d_y, dev, (size_t)type_bytes(y_type)));
    if (d_b)
        LL_TRY(llh::check_device_ptr(op, "b", d_b, dev, 4));
    if (y_type == LL_T_F8)
        LL_TRY(llh::check_device_ptr(op, "the scales of y", d_sy, dev, 4));

    DenseF8Params p;
    p.sw = d_sw;
    p.sx = d_sx;
    p.bias = d_b;
    p.y = d_y;
    p.sy = d_sy;
    p.ldy = ldy;
    p.rows = rows;
    p.M = M;
    p.nkb = (K + kF8Block - 1) / kF8Block;
    p.act = act;
    p.y_type = y_type;
    const int v4 = 4 * type_bytes(y_type);  // bytes of four outputs
    p.y_vec = (ldy % 4 == 0 && (reinterpret_cast<uintptr_t>(d_y) % v4) == 0) ? 1 : 0;
    p.status = status;
    p.wait_ns = llh::ops_wait_ns();
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Which kernel, measured in a graph on B200 (us; many-row kernel / few-row kernel at its best):
    //   32 tiles of 256 x 256 and more: 1024 x 2048 x 1024 12.6 / 13.2, 512 x 4096 x 4096 26 / 33,
    //   768 x 4096 x 4096 27 / 57; fewer leave too many SMs idle: 256 x 4096 x 4096 25.5 / 19.9.
    // Rows per tile of the few-row kernel: 32 (16 for up to 16 rows); 128 once those tiles alone fill
    // the SMs: 1500 x 900 x 900 13.7 against 15.2 at 32, 256 x 2048 x 2048 9.6 against 8.1 at 32.
    const long long large_tiles = (long long)((rows + 2 * kDlM - 1) / (2 * kDlM)) * ((M + kDlN - 1) / kDlN);
    const bool many = rows > 128 && large_tiles >= 32;
    const long long mtiles = (M + 127) / 128;
    const int nt = many ? kDlM : rows <= 16 ? 16 : mtiles * ((rows + 127) / 128) >= 96 ? 128 : 32;
    if (!f8_map(&p.tm_w, d_W, K, M, ldw, 128) || !f8_map(&p.tm_x, d_x, K, rows, ldx, nt)) {
        llh::set_error("%s: the tensor maps could not be encoded", op);
        return LL_ERR_CUDA;
    }
    if (many) {
        p.y_vec = ((ldy * type_bytes(y_type)) % 16 == 0 && (reinterpret_cast<uintptr_t>(d_y) & 15) == 0) ? 1 : 0;
        return y_type == LL_T_F32    ? launch_many<LL_T_F32>(p, dev, st)
               : y_type == LL_T_BF16 ? launch_many<LL_T_BF16>(p, dev, st)
               : y_type == LL_T_F16  ? launch_many<LL_T_F16>(p, dev, st)
                                     : launch_many<LL_T_F8>(p, dev, st);
    }
    // Splits of K (CTAs of a cluster): up to one CTA per SM with two K blocks each, or two small CTAs per SM
    // with four blocks each (64 x 4096 x 4096: 8.3 us at 256 CTAs, 9.3 at 128); not 8 splits for that, whose
    // exchange costs more than the shorter sums save (200 x 640 x 8192: 12.5 us at 280 CTAs, 10.3 at 140).
    const long long tiles = mtiles * ((rows + nt - 1) / nt);
    int splits = 1;
    while (splits < 8 && ((tiles * splits * 2 <= 148 && p.nkb >= splits * 4) ||
                          (tiles * splits * 2 <= 296 && splits <= 2 && nt <= 32 && p.nkb >= splits * 8)))
        splits *= 2;
    p.kb_split = (p.nkb + splits - 1) / splits;
    switch (nt) {
    case 16:
        return launch_few<16>(p, splits, dev, st);
    case 32:
        return launch_few<32>(p, splits, dev, st);
    default:
        return launch_few<128>(p, splits, dev, st);
    }
}
