// aw4_route.cu -- expert router: softmax, top-k, per-expert counts and the balance loss, with gradients.
//
// For a row of logits l over E experts, p = softmax(l).  The k largest logits
// are chosen (ties to the lowest index, a NaN above every number, -inf never),
// w_j = p of the j-th choice, divided by the sum of the chosen p where
// renormalized.  With n valid rows
//
//     balance = sum_e share_e mean_e,  share_e = E counts_e / (k n),  mean_e = sum of p_e over valid rows / n
//
// and, for dB = d loss / d balance and t_j = w_j (dw_j - [renormalize] sum_i w_i dw_i),
//
//     dl_e = p_e (share_e dB / n - K) + sum_{j: choice j = e} t_j
//     K = sum_e p_e share_e dB / n + [not renormalize] sum_j w_j dw_j
//
// A row that is not valid, or whose logits are all -inf, takes no part:
// choices -1, weights 0, gradient 0, no count.
//
// Counts are integers; the sums of p go through registers, then blocks'
// partial sums, then one block, each in a fixed order, so a repeated call
// gives the same bits.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/adamw4bit_b200.h"
#include "aw4_act8.cuh"
#include "aw4_host.h"

namespace aw4 {

constexpr int kRouteThreads = 256;
constexpr int kRouteMaxK = 32;

// Logits as integers whose order is that of the numbers, -0 = +0, NaN on top.
__device__ __forceinline__ uint32_t order_key(float l) {
    uint32_t u = __float_as_uint(l);
    if (l != l) return 0xffffffffu;
    if (l == 0.0f) u = 0;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;

// A row belongs to L lanes; lane i holds experts [8 i, 8 i + 8) and, where V > 8, those 8 L further on.
template <int DT, int L, int V>
__device__ __forceinline__ void load_logits(const RowsIn& logits, int64_t row, int lane, int experts, bool in,
                                            float l[V]) {
#pragma unroll
    for (int c = 0; c < V / 8; ++c) {
        const int at = (c * L + lane) * 8;
        float v[8];
        widen8<DT>(load_raw8<DT>(logits, in ? row : 0, at, in ? experts : 0), v);
#pragma unroll
        for (int i = 0; i < 8; ++i) l[c * 8 + i] = in && at + i < experts ? v[i] : -INFINITY;
    }
}

template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = L / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int DT, int L, int V>
__global__ void __launch_bounds__(kRouteThreads)
route_forward_kernel(const RowsIn logits, int64_t rows, int experts, int k,
                     const uint8_t* __restrict__ valid, bool renormalize, float* __restrict__ weights,
                     int32_t* __restrict__ chosen, float2* __restrict__ stats, float* __restrict__ psum,
                     int32_t* __restrict__ pcount) {
    constexpr int kRows = kRouteThreads / L;
    extern __shared__ int32_t smem[];
    int32_t* count = smem;                                        // [experts + 1], the last: valid rows
    float* sums = reinterpret_cast<float*>(smem + experts + 1);   // [experts]
    for (int i = threadIdx.x; i <= experts; i += kRouteThreads) count[i] = 0;
    for (int i = threadIdx.x; i < experts; i += kRouteThreads) sums[i] = 0.0f;
    __syncthreads();
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    float acc[V] = {};
    const int64_t tiles = (rows + kRows - 1) / kRows;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t row = tile * kRows + group;
        const bool in = row < rows;
        bool ok = in && (!valid || valid[row]);
        float l[V];
        load_logits<DT, L, V>(logits, row, lane, experts, ok, l);
        uint32_t key[V];
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = order_key(l[i]);
        float top = 0.0f, total = 0.0f, denominator = 0.0f;
        for (int j = 0; j < k; ++j) {
            // the largest key left, and the lowest index that has it
            uint32_t best = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) best = max(best, key[i]);
#pragma unroll
            for (int o = L / 2; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
            int at = 0x7fffffff;
#pragma unroll
            for (int i = V - 1; i >= 0; --i)
                if (key[i] == best) at = (i / 8 * L + lane) * 8 + i % 8;
#pragma unroll
            for (int o = L / 2; o; o >>= 1) at = min(at, __shfl_xor_sync(0xffffffffu, at, o));
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (at == (i / 8 * L + lane) * 8 + i % 8) key[i] = 0;
            const bool some = best > kKeyNegInf;
            if (j == 0) {
                ok = ok && some;
                top = key_value(best);
                float part = 0.0f;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    l[i] = ok ? expf(l[i] - top) : 0.0f;
                    part += l[i];
                }
                total = lanes_sum<L>(part);
            }
            const bool take = ok && some;
            const float w = take ? expf(key_value(best) - top) : 0.0f;
            denominator += w;
            if (in && lane == 0) {
                weights[row * k + j] = w;
                chosen[row * k + j] = take ? at : -1;
                if (take) atomicAdd(&count[at], 1);
            }
        }
        const float inv = ok ? 1.0f / total : 0.0f;
        if (in && lane == 0) {
            stats[row] = make_float2(top, inv);
            if (ok) atomicAdd(&count[experts], 1);
            const float scale = !ok ? 0.0f : renormalize ? 1.0f / denominator : inv;
            for (int j = 0; j < k; ++j) weights[row * k + j] *= scale;
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (ok) acc[i] = __fmaf_rn(l[i], inv, acc[i]);
    }
    // groups of the warp, then the warps in turn
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int o = 16; o >= L; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    for (int w = 0; w < kRouteThreads / 32; ++w) {
        __syncthreads();
        if ((int)(threadIdx.x >> 5) == w && (threadIdx.x & 31) < L)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int e = (i / 8 * L + lane) * 8 + i % 8;
                if (e < experts) sums[e] += acc[i];
            }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < experts; i += kRouteThreads) psum[(int64_t)blockIdx.x * experts + i] = sums[i];
    for (int i = threadIdx.x; i <= experts; i += kRouteThreads)
        pcount[(int64_t)blockIdx.x * (experts + 1) + i] = count[i];
}

// One block: counts, the number of valid rows and the balance loss.
__global__ void __launch_bounds__(1024)
route_finish_kernel(const float* __restrict__ psum, const int32_t* __restrict__ pcount, int parts, int experts,
                    int k, int32_t* __restrict__ counts, float* __restrict__ balance) {
    __shared__ float warp_part[32];
    __shared__ int valid_rows;
    float mine = 0.0f;
    for (int e = threadIdx.x; e <= experts; e += 1024) {
        int c = 0;
        for (int p = 0; p < parts; ++p) c += pcount[(int64_t)p * (experts + 1) + e];
        counts[e] = c;
        if (e == experts) {
            valid_rows = c;
        } else {
            float s = 0.0f;
            for (int p = 0; p < parts; ++p) s += psum[(int64_t)p * experts + e];
            mine = __fmaf_rn((float)c, s, mine);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        float s = 0.0f;
        for (int i = 0; i < 32; ++i) s += warp_part[i];
        const float n = (float)valid_rows;
        *balance = valid_rows ? s * ((float)experts / (float)k) / n / n : 0.0f;
    }
}

template <int DT, int L, int V>
__global__ void __launch_bounds__(kRouteThreads)
route_backward_kernel(const RowsIn logits, int64_t rows, int experts, int k,
                      bool renormalize, const float* __restrict__ weights, const int32_t* __restrict__ chosen,
                      const float2* __restrict__ stats, const int32_t* __restrict__ counts,
                      const float* __restrict__ dweights, const float* __restrict__ dbalance,
                      const RowsOut dlogits) {
    constexpr int kRows = kRouteThreads / L;
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    const float n = fmaxf((float)counts[experts], 1.0f);
    const float unit = dbalance ? *dbalance * ((float)experts / (float)k) / n / n : 0.0f;
    float share[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = (i / 8 * L + lane) * 8 + i % 8;
        share[i] = e < experts ? (float)counts[e] * unit : 0.0f;
    }
    const int64_t tiles = (rows + kRows - 1) / kRows;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t row = tile * kRows + group;
        const bool in = row < rows;
        const float2 st = in ? stats[row] : make_float2(0.0f, 0.0f);
        const bool ok = st.y != 0.0f;             // a NaN row is a valid one
        float l[V];
        load_logits<DT, L, V>(logits, row, lane, experts, ok, l);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            l[i] = ok ? expf(l[i] - st.x) * st.y : 0.0f;
            sum = __fmaf_rn(l[i], share[i], sum);
        }
        sum = lanes_sum<L>(sum);
        float inner = 0.0f;
        if (dweights && ok)
            for (int j = 0; j < k; ++j) inner = __fmaf_rn(weights[row * k + j], dweights[row * k + j], inner);
        const float off = renormalize ? sum : sum + inner, back = renormalize ? inner : 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) l[i] *= share[i] - off;
        if (dweights && ok)
            for (int j = 0; j < k; ++j) {
                const int at = chosen[row * k + j];
                const float t = weights[row * k + j] * (dweights[row * k + j] - back);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (at == (i / 8 * L + lane) * 8 + i % 8) l[i] += t;
            }
        if (in)
#pragma unroll
            for (int c = 0; c < V / 8; ++c)
                store_raw8<DT>(dlogits, row, (c * L + lane) * 8, experts, narrow8<DT>(l + c * 8));
    }
}

// Lanes of a row: the fewest that hold eight logits each, a whole warp from 256 experts on.
template <typename F>
static int32_t route_shape(int experts, F f) {
    using std::integral_constant;
    if (experts <= 8) return f(integral_constant<int, 1>(), integral_constant<int, 8>());
    if (experts <= 16) return f(integral_constant<int, 2>(), integral_constant<int, 8>());
    if (experts <= 32) return f(integral_constant<int, 4>(), integral_constant<int, 8>());
    if (experts <= 64) return f(integral_constant<int, 8>(), integral_constant<int, 8>());
    if (experts <= 128) return f(integral_constant<int, 16>(), integral_constant<int, 8>());
    if (experts <= 256) return f(integral_constant<int, 32>(), integral_constant<int, 8>());
    if (experts <= 512) return f(integral_constant<int, 32>(), integral_constant<int, 16>());
    return f(integral_constant<int, 32>(), integral_constant<int, 32>());
}

template <typename F>
static int32_t route_by_dtype(int dtype, F f) {
    using std::integral_constant;
    if (dtype == AW4_F32) return f(integral_constant<int, AW4_F32>());
    if (dtype == AW4_BF16) return f(integral_constant<int, AW4_BF16>());
    return f(integral_constant<int, AW4_F16>());
}

static int32_t check_route(const char* what, int dtype, int64_t rows, int64_t experts, int32_t k) {
    if (dtype < AW4_F32 || dtype > AW4_F16) return fail(AW4_ERR_INVALID, "%s: bad dtype %d", what, dtype);
    if (rows < 0 || experts < 1) return fail(AW4_ERR_INVALID, "%s: bad size", what);
    if (rows > 0x7fffffff) return fail(AW4_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows", what);
    if (experts > AW4_ROUTE_MAX_EXPERTS)
        return fail(AW4_ERR_UNSUPPORTED, "%s: more than %d experts", what, AW4_ROUTE_MAX_EXPERTS);
    if (k < 1 || k > kRouteMaxK || k > experts)
        return fail(AW4_ERR_INVALID, "%s: k = %d of %d experts", what, k, (int)experts);
    return AW4_OK;
}

static int route_lanes(int experts) {
    int lanes = 1;
    while (lanes < 32 && lanes * 8 < experts) lanes *= 2;
    return lanes;
}

static int route_grid(int device, int64_t rows, int experts) {
    const int per = kRouteThreads / route_lanes(experts);
    return (int)std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, (int64_t)sm_count(device) * 2));
}

static bool route_vec(const void* p, int64_t ld, int dtype) {
    return (uintptr_t)p % 16 == 0 && ld * (dtype == AW4_F32 ? 4 : 2) % 16 == 0;
}

static RowsIn route_rows(const void* p, int64_t rows, int experts, int64_t ld, int dtype) {
    const char* base = static_cast<const char*>(p);
    return {base, base + ((rows - 1) * ld + experts) * (dtype == AW4_F32 ? 4 : 2), ld, route_vec(p, ld, dtype)};
}

}  // namespace aw4

using namespace aw4;

extern "C" uint64_t aw4_route_forward_workspace(int64_t rows, int32_t experts, int32_t device) {
    if (rows <= 0 || experts < 1 || experts > AW4_ROUTE_MAX_EXPERTS) return 0;
    return (uint64_t)route_grid(device, rows, experts) * (2 * experts + 1) * 4;
}

extern "C" int32_t aw4_route_forward(const void* logits, int32_t dtype, int64_t rows, int32_t experts, int64_t ld,
                                     int32_t k, const uint8_t* valid, int32_t renormalize, float* weights,
                                     int32_t* chosen, float* stats, int32_t* counts, float* balance,
                                     void* workspace, int64_t workspace_bytes, int32_t device, void* stream) {
    if (const int32_t rc = check_route("aw4_route_forward", dtype, rows, experts, k)) return rc;
    if (!counts || !balance) return fail(AW4_ERR_INVALID, "aw4_route_forward: null buffer");
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(AW4_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    cudaStream_t s = (cudaStream_t)stream;
    if (rows == 0) {
        cudaError_t e = cudaMemsetAsync(counts, 0, (experts + 1) * 4, s);
        if (e == cudaSuccess) e = cudaMemsetAsync(balance, 0, 4, s);
        return e == cudaSuccess ? AW4_OK : fail(AW4_ERR_CUDA, "route_forward: %s", cudaGetErrorString(e));
    }
    if (!logits || !weights || !chosen || !stats || (uintptr_t)stats % 8)
        return fail(AW4_ERR_INVALID, "aw4_route_forward: null or misaligned buffer");
    const int grid = route_grid(device, rows, experts);
    if (!workspace || workspace_bytes < (int64_t)grid * (2 * experts + 1) * 4)
        return fail(AW4_ERR_INVALID, "aw4_route_forward: workspace of %lld bytes is too small",
                    (long long)workspace_bytes);
    float* psum = static_cast<float*>(workspace);
    int32_t* pcount = reinterpret_cast<int32_t*>(psum + (int64_t)grid * experts);
    const int32_t rc = route_by_dtype(dtype, [&](auto dt) {
        return route_shape(experts, [&](auto lanes, auto v) {
            route_forward_kernel<dt.value, lanes.value, v.value>
                <<<grid, kRouteThreads, (2 * experts + 1) * 4, s>>>(
                    route_rows(logits, rows, experts, ld, dtype), rows, experts, k, valid, renormalize != 0, weights,
                    chosen, reinterpret_cast<float2*>(stats), psum, pcount);
            note_launch();
            const cudaError_t e = cudaGetLastError();
            return e == cudaSuccess ? AW4_OK
                                    : fail(AW4_ERR_CUDA, "route_forward launch: %s", cudaGetErrorString(e));
        });
    });
    if (rc) return rc;
    route_finish_kernel<<<1, 1024, 0, s>>>(psum, pcount, grid, experts, k, counts, balance);
    note_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? AW4_OK : fail(AW4_ERR_CUDA, "route_finish launch: %s", cudaGetErrorString(e));
}

extern "C" int32_t aw4_route_backward(const void* logits, int32_t dtype, int64_t rows, int32_t experts, int64_t ld,
                                      int32_t k, int32_t renormalize, const float* weights, const int32_t* chosen,
                                      const float* stats, const int32_t* counts, const float* dweights,
                                      const float* dbalance, void* dlogits, int32_t device, void* stream) {
    if (const int32_t rc = check_route("aw4_route_backward", dtype, rows, experts, k)) return rc;
    if (rows == 0) return AW4_OK;
    if (!logits || !weights || !chosen || !stats || !counts || !dlogits || (uintptr_t)stats % 8)
        return fail(AW4_ERR_INVALID, "aw4_route_backward: null or misaligned buffer");
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(AW4_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    return route_by_dtype(dtype, [&](auto dt) {
        return route_shape(experts, [&](auto lanes, auto v) {
            const int per = kRouteThreads / lanes.value;
            const int grid = (int)std::min<int64_t>((rows + per - 1) / per, (int64_t)sm_count(device) * 8);
            route_backward_kernel<dt.value, lanes.value, v.value>
                <<<grid, kRouteThreads, 0, (cudaStream_t)stream>>>(
                    route_rows(logits, rows, experts, ld, dtype), rows, experts, k, renormalize != 0, weights, chosen,
                    reinterpret_cast<const float2*>(stats), counts, dweights, dbalance,
                    RowsOut{static_cast<char*>(dlogits), experts, route_vec(dlogits, experts, dtype)});
            note_launch();
            const cudaError_t e = cudaGetLastError();
            return e == cudaSuccess ? AW4_OK
                                    : fail(AW4_ERR_CUDA, "route_backward launch: %s", cudaGetErrorString(e));
        });
    });
}
