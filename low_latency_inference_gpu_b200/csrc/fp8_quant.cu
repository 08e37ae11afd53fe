// ll_quantize_fp8: rows of activations to e4m3 with one fp32 scale per row and 128 columns,
// the input format of ll_dense_fp8 (no counterpart in the reference, which is fp32 only).
//
//   amax = max |x[r, 128 g .. 128 g + 127]|,  s = amax / 448 (or the power of two at or above),
//   q = e4m3 nearest to x / s.
//
// One pass: 8 lanes hold a group in registers (16 values each), agree on amax by three
// shuffles, and write 16 bytes each.  Bound by memory for many rows, by the launch for few.
#include "ops_common.cuh"

namespace llk {

constexpr int kQtThreads = 256;
constexpr int kQtLanes = 8;                           // lanes per group
constexpr int kQtPer = kF8Block / kQtLanes;           // values per lane
constexpr int kQtGroups = kQtThreads / kQtLanes;      // groups per block and step

// n / d for n < 2^31 by one multiplication: m = floor(2^(31+l) / d) + 1 with 2^l >= d.
struct FastDiv {
    uint32_t d, shift;
    uint64_t m;
};

inline FastDiv fast_div(uint32_t d)
{
    uint32_t l = 0;
    while ((1ull << l) < d)
        ++l;
    return {d, 31 + l, (1ull << (31 + l)) / d + 1};
}

__device__ __forceinline__ float to_f32(float v)
{
    return v;
}
__device__ __forceinline__ float to_f32(__nv_bfloat16 v)
{
    return __bfloat162float(v);
}
__device__ __forceinline__ float to_f32(__half v)
{
    return __half2float(v);
}

__device__ __forceinline__ void load_all(const float *p, float (&v)[kQtPer])
{
#pragma unroll
    for (int j = 0; j < kQtPer / 4; ++j) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(p) + j);
        v[4 * j] = a.x, v[4 * j + 1] = a.y, v[4 * j + 2] = a.z, v[4 * j + 3] = a.w;
    }
}

template <typename T>
__device__ __forceinline__ void load_all(const T *p, float (&v)[kQtPer])
{
#pragma unroll
    for (int j = 0; j < kQtPer / 8; ++j) {
        const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p) + j);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const T *h = reinterpret_cast<const T *>(&w[i]);
            v[8 * j + 2 * i] = to_f32(h[0]);
            v[8 * j + 2 * i + 1] = to_f32(h[1]);
        }
    }
}

// Four values of a 16-bit type as four e4m3 bytes, without a slow path.  v and amax have at most 11
// significant bits, a border of two e4m3 values 5, so v * 448 / amax is either on a border or at
// least 2^-17 (relative) away from it; v / s differs from it by the rounding of s alone, one
// factor for the whole group within 2^-24.  So where s is not exact, a factor of 1 +- 2^-20
// towards the side on which that rounding puts the quotients decides the ties and changes nothing
// else; where it is, one correction step makes the quotient exact.  (Not for scales below kF8SmallScale, whose
// residuals would be fp32's subnormal numbers: those groups go the way of fp32 values.)
struct Scale16 {
    float s, inv, by;  // by: the reciprocal with the group's factor
    bool exact;
};

__device__ __forceinline__ Scale16 scale16(float amax, float s, float inv)
{
    const float d = fmaf(-kF8Max, s, amax);  // exact: s is amax / 448 to 2^-24
    const bool exact = d == 0.0f;
    return {s, inv, exact ? inv : inv * (d > 0.0f ? 1.0f + 0x1p-20f : 1.0f - 0x1p-20f), exact};
}

__device__ __forceinline__ uint32_t e4m3x4_of16(const float *v, const Scale16 &g)
{
    float t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        t[i] = v[i] * g.by;
    if (g.exact)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            t[i] = fmaf(fmaf(-t[i], g.s, v[i]), g.inv, t[i]);
    return f32x2_to_e4m3(t[0], t[1]) | (f32x2_to_e4m3(t[2], t[3]) << 16);
}

// VEC: every row of x and of q starts on 16 bytes.
// 8192 x 4096 bf16 (101 MB): 19.3 us, 5.2 TB/s, 80 % of the measured copy rate; fp32 (169 MB): 25.9 us, 99 %; one row
// of 2048: the launch.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kQtThreads) ll_quantize_fp8_kernel(const T *__restrict__ x, long long ldx, int dim,
                                                                     uint32_t n_groups, FastDiv per_row,
                                                                     uint8_t *__restrict__ q, long long ldq,
                                                                     float *__restrict__ s, bool pow2)
{
    griddep_launch_dependents();  // a dense layer behind this launch sets itself up meanwhile
    const uint32_t g = blockIdx.x * kQtGroups + threadIdx.x / kQtLanes;
    const uint32_t row = (uint32_t)(((uint64_t)g * per_row.m) >> per_row.shift);
    const int col = (int)(g - row * per_row.d) * kF8Block + (threadIdx.x % kQtLanes) * kQtPer;
    const int have = g < n_groups ? min(kQtPer, dim - col) : 0;  // <= 0: nothing of the row is left here
    const T *px = x + (size_t)row * (size_t)ldx + col;
    float v[kQtPer];
    if (VEC && have == kQtPer) {
        load_all(px, v);
    } else {
#pragma unroll
        for (int i = 0; i < kQtPer; ++i)
            v[i] = i < have ? to_f32(px[i]) : 0.0f;
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kQtPer; ++i)
        amax = fmaxf(amax, fabsf(v[i]));
#pragma unroll
    for (int off = kQtLanes / 2; off > 0; off >>= 1)
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    float sc, inv;
    e4m3_scale(amax, pow2, sc, inv);
    uint32_t o[kQtPer / 4];
    if (sizeof(T) == 2 && !pow2 && !(sc < kF8SmallScale && sc != 0.0f)) {
        const Scale16 f = scale16(amax, sc, inv);
#pragma unroll
        for (int i = 0; i < kQtPer / 4; ++i)
            o[i] = e4m3x4_of16(v + 4 * i, f);
    } else {
#pragma unroll
        for (int i = 0; i < kQtPer / 4; ++i)
            o[i] = group_e4m3x4(v + 4 * i, pow2, sc, inv);
    }
    if (have <= 0)
        return;
    uint8_t *pq = q + (size_t)row * (size_t)ldq + col;
    if (VEC && have == kQtPer) {
        *reinterpret_cast<uint4 *>(pq) = make_uint4(o[0], o[1], o[2], o[3]);
    } else {
#pragma unroll
        for (int i = 0; i < kQtPer; ++i)
            if (i < have)
                pq[i] = (uint8_t)(o[i / 4] >> (8 * (i % 4)));
    }
    if (threadIdx.x % kQtLanes == 0)
        s[g] = sc;
}

template <typename T>
void launch_quantize(const void *x, long long ldx, int rows, int dim, bool pow2, uint8_t *q, long long ldq, float *s,
                     cudaStream_t st)
{
    const uint32_t per_row = (uint32_t)((dim + kF8Block - 1) / kF8Block), n = (uint32_t)rows * per_row;
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * (long long)sizeof(T)) % 16 == 0 &&
                     (reinterpret_cast<uintptr_t>(q) & 15) == 0 && ldq % 16 == 0;
    const dim3 grid((n + kQtGroups - 1) / kQtGroups);
    const FastDiv fd = fast_div(per_row);
    if (vec)
        ll_quantize_fp8_kernel<T, true><<<grid, kQtThreads, 0, st>>>((const T *)x, ldx, dim, n, fd, q, ldq, s, pow2);
    else
        ll_quantize_fp8_kernel<T, false><<<grid, kQtThreads, 0, st>>>((const T *)x, ldx, dim, n, fd, q, ldq, s, pow2);
}

__device__ unsigned g_ops_status[2];  // see llh::ops_status_words

}  // namespace llk

namespace llh {

int ops_status_words(int *device, unsigned **words)
{
    static unsigned *at[llk::kOpsMaxDevices];  // racing first calls store the same address
    LL_CUDA_TRY(cudaGetDevice(device));
    if (*device < 0 || *device >= llk::kOpsMaxDevices) {
        set_error("device index %d out of range", *device);
        return LL_ERR_INVALID_ARG;
    }
    unsigned *p = __atomic_load_n(&at[*device], __ATOMIC_ACQUIRE);
    if (!p) {
        void *v = nullptr;
        LL_CUDA_TRY(cudaGetSymbolAddress(&v, llk::g_ops_status));
        p = static_cast<unsigned *>(v);
        __atomic_store_n(&at[*device], p, __ATOMIC_RELEASE);
    }
    *words = p;
    return LL_OK;
}

static unsigned long long g_wait_ns = llk::kOpsWaitNs;

unsigned long long ops_wait_ns()
{
    return __atomic_load_n(&g_wait_ns, __ATOMIC_RELAXED);
}

int check_device_ptr(const char *op, const char *what, const void *p, int device, size_t align)
{
    if ((reinterpret_cast<uintptr_t>(p) & (align - 1)) != 0) {
        set_error("%s: %s must be aligned to %zu bytes", op, what, align);
        return LL_ERR_INVALID_ARG;
    }
    cudaPointerAttributes a;
    LL_CUDA_TRY(cudaPointerGetAttributes(&a, p));
    if ((a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) ||
        (a.type == cudaMemoryTypeDevice && a.device != device)) {
        set_error("%s: %s is not memory of the current device (%d)", op, what, device);
        return LL_ERR_INVALID_ARG;
    }
    return LL_OK;
}

}  // namespace llh

extern "C" {

int ll_quantize_fp8(const void *d_x, int x_type, int rows, int dim, int64_t ldx, int pow2_scales, uint8_t *d_q,
                    int64_t ldq, float *d_s, void *stream)
{
    static const char op[] = "ll_quantize_fp8";
    if (x_type != LL_T_F32 && x_type != LL_T_BF16 && x_type != LL_T_F16) {
        llh::set_error("%s: x must be fp32, bf16 or fp16 (type %d)", op, x_type);
        return LL_ERR_INVALID_ARG;
    }
    if (ldx == 0)
        ldx = dim;
    if (ldq == 0)
        ldq = dim;
    if (rows < 0 || dim < 1 || dim > (1 << 30) || ldx < dim || ldq < dim || (pow2_scales != 0 && pow2_scales != 1)) {
        llh::set_error("%s: invalid arguments (rows=%d dim=%d ldx=%lld ldq=%lld pow2_scales=%d)", op, rows, dim,
                       (long long)ldx, (long long)ldq, pow2_scales);
        return LL_ERR_INVALID_ARG;
    }
    if ((int64_t)rows * ((dim + LL_F8_BLOCK - 1) / LL_F8_BLOCK) > INT32_MAX - 64) {
        llh::set_error("%s: %d rows of %d have more than 2^31 groups", op, rows, dim);
        return LL_ERR_INVALID_ARG;
    }
    if (rows == 0)
        return LL_OK;
    if (!d_x || !d_q || !d_s) {
        llh::set_error("%s: null pointer", op);
        return LL_ERR_INVALID_ARG;
    }
    int dev = 0;
    LL_CUDA_TRY(cudaGetDevice(&dev));
    LL_TRY(llh::check_device_ptr(op, "x", d_x, dev, (size_t)llk::type_bytes(x_type)));
    LL_TRY(llh::check_device_ptr(op, "q", d_q, dev, 1));
    LL_TRY(llh::check_device_ptr(op, "s", d_s, dev, 4));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (x_type == LL_T_F32)
        llk::launch_quantize<float>(d_x, ldx, rows, dim, pow2_scales != 0, d_q, ldq, d_s, st);
    else if (x_type == LL_T_BF16)
        llk::launch_quantize<__nv_bfloat16>(d_x, ldx, rows, dim, pow2_scales != 0, d_q, ldq, d_s, st);
    else
        llk::launch_quantize<__half>(d_x, ldx, rows, dim, pow2_scales != 0, d_q, ldq, d_s, st);
    LL_CUDA_TRY(cudaGetLastError());
    return LL_OK;
}

int ll_ops_set_wait_limit(uint64_t ns)
{
    if (ns > llk::kOpsMaxWaitNs) {
        llh::set_error("ll_ops_set_wait_limit: at most %llu ns (%llu)", llk::kOpsMaxWaitNs, (unsigned long long)ns);
        return LL_ERR_INVALID_ARG;
    }
    __atomic_store_n(&llh::g_wait_ns, (unsigned long long)ns, __ATOMIC_RELAXED);
    return LL_OK;
}

int ll_ops_check(void *stream)
{
    // The device's count is never reset, so that no check takes a failure from another one; what each has told its
    // caller is kept here, per thread, stream and device, once there is something to tell.
    struct Told {
        void *stream;
        int device;
        unsigned failures;
    };
    constexpr int kTold = 64;  // of more streams than these the oldest is told again
    static thread_local Told told[kTold];
    static thread_local unsigned n_told;

    int dev = 0;
    unsigned *words = nullptr, now[2] = {0, 0};
    LL_TRY(llh::ops_status_words(&dev, &words));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    LL_CUDA_TRY(cudaMemcpyAsync(now, words, sizeof(now), cudaMemcpyDeviceToHost, st));
    LL_CUDA_TRY(cudaStreamSynchronize(st));
    if (now[0] == 0)
        return LL_OK;
    Told *t = nullptr;
    for (unsigned i = 0; i < kTold && i < n_told && !t; ++i)
        if (told[i].stream == stream && told[i].device == dev)
            t = &told[i];
    if (t && t->failures == now[0])
        return LL_OK;
    if (!t)
        t = &told[n_told++ % kTold];
    *t = {stream, dev, now[0]};
    llh::set_error("a device-side wait of ll_dense_fp8 or ll_moe_forward ran out (%u in all, the last in role %u)", now[0],
                   now[1]);
    return LL_ERR_DEVICE_FAULT;
}

}  // extern "C"
