// ll_quantize_fp8: rows of activations to e4m3 with one fp32 scale per row and 128 columns,
// the input format of ll_dense_fp8 (no counterpart in the reference, which is fp32 only).
//
//   amax = max |x[r, 128 g .. 128 g + 127]|,  s = amax / 448 (or the power of two at or above),
//   q = e4m3 nearest to x / s.
//
// One pass: 16 lanes hold a group in registers (8 values each), agree on amax by four
// shuffles, and write 8 bytes each.  Bound by memory for many rows, by the launch for few.
#include "ops_common.cuh"

namespace llk {

constexpr int kQtThreads = 256;
constexpr int kQtLanes = 16;                          // lanes per group
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

__device__ __forceinline__ void load8(const float *p, float (&v)[kQtPer])
{
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[kQtPer])
{
    const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const T *h = reinterpret_cast<const T *>(&w[i]);
        v[2 * i] = to_f32(h[0]);
        v[2 * i + 1] = to_f32(h[1]);
    }
}

// VEC: every row of x starts on 16 bytes and every row of q on 8.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kQtThreads) ll_quantize_fp8_kernel(const T *__restrict__ x, long long ldx, int dim,
                                                                     uint32_t n_groups, FastDiv per_row,
                                                                     uint8_t *__restrict__ q, long long ldq,
                                                                     float *__restrict__ s, bool pow2)
{
    const uint32_t g = blockIdx.x * kQtGroups + threadIdx.x / kQtLanes;
    const uint32_t row = (uint32_t)(((uint64_t)g * per_row.m) >> per_row.shift);
    const int col = (int)(g - row * per_row.d) * kF8Block + (threadIdx.x % kQtLanes) * kQtPer;
    const int have = g < n_groups ? min(kQtPer, dim - col) : 0;  // <= 0: nothing of the row is left here
    const T *px = x + (size_t)row * (size_t)ldx + col;
    float v[kQtPer];
    if (VEC && have == kQtPer) {
        load8(px, v);
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
    const uint2 o = make_uint2(group_e4m3x4(v, pow2, sc, inv), group_e4m3x4(v + 4, pow2, sc, inv));
    if (have <= 0)
        return;
    uint8_t *pq = q + (size_t)row * (size_t)ldq + col;
    if (VEC && have == kQtPer) {
        *reinterpret_cast<uint2 *>(pq) = o;
    } else {
#pragma unroll
        for (int i = 0; i < kQtPer; ++i)
            if (i < have)
                pq[i] = (uint8_t)((i < 4 ? o.x >> (8 * i) : o.y >> (8 * (i - 4))) & 0xffu);
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
                     (reinterpret_cast<uintptr_t>(q) & 7) == 0 && ldq % 8 == 0;
    const dim3 grid((n + kQtGroups - 1) / kQtGroups);
    const FastDiv fd = fast_div(per_row);
    if (vec)
        ll_quantize_fp8_kernel<T, true><<<grid, kQtThreads, 0, st>>>((const T *)x, ldx, dim, n, fd, q, ldq, s, pow2);
    else
        ll_quantize_fp8_kernel<T, false><<<grid, kQtThreads, 0, st>>>((const T *)x, ldx, dim, n, fd, q, ldq, s, pow2);
}

__device__ unsigned g_ops_status;  // see llh::ops_status_word

}  // namespace llk

namespace llh {

int ops_status_word(int *device, unsigned **word)
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
    *word = p;
    return LL_OK;
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

int ll_ops_check(void *stream)
{
    int dev = 0;
    unsigned *word = nullptr, v = 0;
    LL_TRY(llh::ops_status_word(&dev, &word));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    LL_CUDA_TRY(cudaMemcpyAsync(&v, word, sizeof(v), cudaMemcpyDeviceToHost, st));
    LL_CUDA_TRY(cudaStreamSynchronize(st));
    if (v == 0)
        return LL_OK;
    LL_CUDA_TRY(cudaMemsetAsync(word, 0, sizeof(v), st));
    LL_CUDA_TRY(cudaStreamSynchronize(st));
    llh::set_error("a device-side wait of ll_dense_fp8 or ll_moe_forward ran out (role %u)", (v >> 8) & 0xffu);
    return LL_ERR_DEVICE_FAULT;
}

}  // extern "C"
