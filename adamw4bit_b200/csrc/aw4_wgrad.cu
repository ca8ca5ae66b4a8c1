// aw4_wgrad.cu -- weight gradient of a projection whose input is an 8-bit checkpoint.
//
// dW_g[n][k] = sum over the rows t of group g of dy[t][n] v[t][k], v the
// checkpoint's values.  Group g holds rows [offsets[g], offsets[g + 1]); an
// empty group's gradient is zero.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/adamw4bit_b200.h"
#include "aw4_act8.cuh"
#include "aw4_host.h"

namespace aw4 {

constexpr int kWgTile = 64, kWgRows = 16;

// A block of 256 threads holds a 64 x 64 tile, 4 x 4 sums a thread.
template <int DT, int OT>
__global__ void __launch_bounds__(256)
weight_grad_kernel(const void* __restrict__ dy, int64_t ld, int64_t rows, int n, const uint8_t* __restrict__ codes,
                   const uint8_t* __restrict__ scales, int k, uint32_t blocks, const int32_t* __restrict__ offsets,
                   void* __restrict__ out, bool accumulate) {
    __shared__ float a[kWgRows][kWgTile], b[kWgRows][kWgTile];
    const int g = blockIdx.z;
    const int n0 = blockIdx.x * kWgTile, k0 = blockIdx.y * kWgTile;
    int64_t first = 0, last = rows;
    if (offsets) {
        first = max((int64_t)0, min(rows, (int64_t)offsets[g]));
        last = max(first, min(rows, (int64_t)offsets[g + 1]));
    }
    const int tn = threadIdx.x / 16 * 4, tk = threadIdx.x % 16 * 4;
    float acc[4][4] = {};
    for (int64_t t0 = first; t0 < last; t0 += kWgRows) {
        for (int i = threadIdx.x; i < kWgRows * kWgTile; i += 256) {
            const int r = i / kWgTile, c = i % kWgTile;
            const int64_t t = t0 + r;
            a[r][c] = t < last && n0 + c < n ? Elem<DT>::load1(dy, t * ld + n0 + c) : 0.0f;
            b[r][c] = t < last && k0 + c < k
                          ? (float)(int8_t)codes[t * blocks * 32 + k0 + c] * a8_scale(scales[t * blocks + (k0 + c) / 32])
                          : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kWgRows; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(a[r][tn + i], b[r][tk + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j)
            if (n0 + tn + i < n && k0 + tk + j < k) {
                const int64_t at = ((int64_t)g * n + n0 + tn + i) * k + k0 + tk + j;
                Elem<OT>::store1(out, at, accumulate ? Elem<OT>::load1(out, at) + acc[i][j] : acc[i][j]);
            }
}

}  // namespace aw4

using namespace aw4;

extern "C" uint64_t aw4_weight_grad_workspace(int64_t rows, int64_t n, int64_t k, int64_t groups, int32_t device) {
    (void)rows; (void)n; (void)k; (void)groups; (void)device;
    return 0;
}

extern "C" int32_t aw4_weight_grad(const void* dy, int32_t dtype, int64_t rows, int64_t n, int64_t ld,
                                   const uint8_t* codes, const uint8_t* scales, int64_t k, const int32_t* offsets,
                                   int64_t groups, void* out, int32_t out_dtype, int32_t accumulate,
                                   void* workspace, int64_t workspace_bytes, int32_t* status, int32_t device,
                                   void* stream) {
    if (dtype != AW4_BF16 && dtype != AW4_F16)
        return fail(AW4_ERR_UNSUPPORTED, "aw4_weight_grad: gradients are bf16 or f16, not dtype %d", dtype);
    if (out_dtype != dtype && out_dtype != AW4_F32)
        return fail(AW4_ERR_UNSUPPORTED, "aw4_weight_grad: output dtype %d", out_dtype);
    if (rows < 0 || n < 0 || k < 0 || groups < 1 || (!offsets && groups != 1))
        return fail(AW4_ERR_INVALID, "aw4_weight_grad: bad size");
    if (rows > 0x7fffffff || n > 1 << 20 || k > 1 << 20 || groups > 65535)
        return fail(AW4_ERR_UNSUPPORTED, "aw4_weight_grad: size above the kernel's");
    if (n == 0 || k == 0) return AW4_OK;
    if (!out || (rows && (!dy || !codes || !scales || (uintptr_t)codes % 16)))
        return fail(AW4_ERR_INVALID, "aw4_weight_grad: null or misaligned buffer");
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(AW4_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    const dim3 grid((unsigned)((n + kWgTile - 1) / kWgTile), (unsigned)((k + kWgTile - 1) / kWgTile), (unsigned)groups);
    const uint32_t blocks = (uint32_t)((k + kA8Block - 1) / kA8Block);
    cudaStream_t s = (cudaStream_t)stream;
    auto go = [&](auto dt, auto ot) {
        weight_grad_kernel<dt.value, ot.value><<<grid, 256, 0, s>>>(dy, ld, rows, (int)n, codes, scales, (int)k,
                                                                   blocks, offsets, out, accumulate != 0);
    };
    using std::integral_constant;
    if (dtype == AW4_BF16) {
        if (out_dtype == AW4_F32) go(integral_constant<int, AW4_BF16>(), integral_constant<int, AW4_F32>());
        else go(integral_constant<int, AW4_BF16>(), integral_constant<int, AW4_BF16>());
    } else {
        if (out_dtype == AW4_F32) go(integral_constant<int, AW4_F16>(), integral_constant<int, AW4_F32>());
        else go(integral_constant<int, AW4_F16>(), integral_constant<int, AW4_F16>());
    }
    note_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? AW4_OK : fail(AW4_ERR_CUDA, "weight_grad launch: %s", cudaGetErrorString(e));
}
