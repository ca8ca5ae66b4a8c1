// aw4_act8.cu -- 8-bit activation checkpoints and the elementwise backward passes that read them.
//
// Every kernel here is one pass over its inputs, bound by HBM.  Warps walk
// runs of kChunks * 32 chunks of eight values; loads of a run are issued
// before the first is used.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/adamw4bit_b200.h"
#include "aw4_act8.cuh"
#include "aw4_host.h"

namespace aw4 {

constexpr int kA8Threads = 256;
constexpr int kChunks = 4;                      // chunks of eight values per lane in flight
constexpr int kRun = 32 * kChunks;              // chunks per warp and turn

// Writes the scale bytes of a run: lane i holds block i's.
__device__ __forceinline__ void store_scales(uint8_t* scales, int64_t unit0, int64_t blocks,
                                             const int b[kChunks], int lane) {
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        const int got = __shfl_sync(0xffffffffu, b[j], (lane & 7) * 4);
        if ((lane >> 3) == j) mine = got;
    }
    const int64_t blk = (unit0 >> 2) + lane;
    if (blk < blocks) scales[blk] = (uint8_t)mine;
}

template <int DT>
__global__ void __launch_bounds__(kA8Threads)
act8_quantize_kernel(const void* __restrict__ x, int64_t rows, int cols, int64_t ld, uint32_t per_row,
                     bool vec, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int lane = threadIdx.x & 31;
    const int64_t units = rows * per_row;
    const int64_t warps = (int64_t)gridDim.x * (kA8Threads / 32);
    for (int64_t w = (int64_t)blockIdx.x * (kA8Threads / 32) + (threadIdx.x >> 5); w * kRun < units;
         w += warps) {
        const int64_t unit0 = w * kRun;
        const RunAt run = run_at(unit0, per_row);
        Raw8<DT> raw[kChunks];
        bool in[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const ChunkAt c = chunk_at(run, j * 32 + lane, per_row, rows);
            in[j] = c.in;
            raw[j] = load_raw8<DT>(x, c.row * ld, c.col, c.in ? cols : 0, vec);
        }
        int b[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            float v[8];
            widen8<DT>(raw[j], v);
            b[j] = a8_scale_byte<DT>(v);
            if (in[j])
                *reinterpret_cast<uint2*>(codes + (unit0 + j * 32 + lane) * 8) = a8_encode8(v, b[j]);
        }
        store_scales(scales, unit0, units >> 2, b, lane);
    }
}

template <int DT>
__global__ void __launch_bounds__(kA8Threads)
act8_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                       int64_t rows, int cols, uint32_t per_row, void* __restrict__ out, int64_t ld,
                       bool vec) {
    const int lane = threadIdx.x & 31;
    const int64_t units = rows * per_row;
    const int64_t warps = (int64_t)gridDim.x * (kA8Threads / 32);
    for (int64_t w = (int64_t)blockIdx.x * (kA8Threads / 32) + (threadIdx.x >> 5); w * kRun < units;
         w += warps) {
        const int64_t unit0 = w * kRun;
        const RunAt run = run_at(unit0, per_row);
        uint2 q[kChunks];
        int b[kChunks];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const int64_t u = unit0 + j * 32 + lane;
            if (u < units) {
                q[j] = __ldcs(reinterpret_cast<const uint2*>(codes + u * 8));
                b[j] = scales[u >> 2];
            }
        }
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const ChunkAt c = chunk_at(run, j * 32 + lane, per_row, rows);
            if (!c.in) continue;
            float v[8];
            a8_decode8(q[j], a8_scale(b[j]), v);
            store_raw8<DT>(out, c.row * ld, c.col, cols, vec, narrow8<DT>(v));
        }
    }
}

// ---------------------------------------------------------------------------
// gated activation: h = g sigmoid(g) u
// ---------------------------------------------------------------------------

// exp to a few units in the last place of float32 either way; the 16-bit
// types take the hardware exponential and reciprocal, far below their rounding.
template <int DT>
__device__ __forceinline__ float sigmoid(float g) {
    if constexpr (DT == AW4_F32) return 1.0f / (1.0f + expf(-g));
    else return __frcp_rn(1.0f + __expf(-g));
}

template <int DT, bool EMIT>
__global__ void __launch_bounds__(kA8Threads)
swiglu_forward_kernel(const void* __restrict__ gate, const void* __restrict__ up, int64_t rows, int cols,
                      int64_t ld_gate, int64_t ld_up, uint32_t per_row, bool vec, void* __restrict__ h,
                      int64_t ld_h, bool vec_h, uint8_t* __restrict__ gcodes, uint8_t* __restrict__ gscales,
                      uint8_t* __restrict__ ucodes, uint8_t* __restrict__ uscales,
                      uint8_t* __restrict__ hcodes, uint8_t* __restrict__ hscales) {
    constexpr int kC = 2, kR = 32 * kC;
    const int lane = threadIdx.x & 31;
    const int64_t units = rows * per_row;
    const int64_t warps = (int64_t)gridDim.x * (kA8Threads / 32);
    for (int64_t w = (int64_t)blockIdx.x * (kA8Threads / 32) + (threadIdx.x >> 5); w * kR < units; w += warps) {
        const int64_t unit0 = w * kR;
        const RunAt run = run_at(unit0, per_row);
        Raw8<DT> rg[kC], ru[kC];
        ChunkAt at[kC];
#pragma unroll
        for (int j = 0; j < kC; ++j) {
            at[j] = chunk_at(run, j * 32 + lane, per_row, rows);
            rg[j] = load_raw8<DT>(gate, at[j].row * ld_gate, at[j].col, at[j].in ? cols : 0, vec);
            ru[j] = load_raw8<DT>(up, at[j].row * ld_up, at[j].col, at[j].in ? cols : 0, vec);
        }
#pragma unroll
        for (int j = 0; j < kC; ++j) {
            const int64_t u = unit0 + j * 32 + lane;
            float g[8], p[8], y[8];
            widen8<DT>(rg[j], g);
            widen8<DT>(ru[j], p);
            const int bg = a8_scale_byte<DT>(g), bu = a8_scale_byte<DT>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = g[i] * sigmoid<DT>(g[i]) * p[i];
            const Raw8<DT> r = narrow8<DT>(y);
            int bh = 0;
            if constexpr (EMIT) {       // the checkpoint of h is that of its rounded values
                widen8<DT>(r, y);
                bh = a8_scale_byte<DT>(y);
            }
            if (at[j].in) {
                *reinterpret_cast<uint2*>(gcodes + u * 8) = a8_encode8(g, bg);
                *reinterpret_cast<uint2*>(ucodes + u * 8) = a8_encode8(p, bu);
                store_raw8<DT>(h, at[j].row * ld_h, at[j].col, cols, vec_h, r);
                if constexpr (EMIT) *reinterpret_cast<uint2*>(hcodes + u * 8) = a8_encode8(y, bh);
                if ((lane & 3) == 0) {
                    gscales[u >> 2] = (uint8_t)bg;
                    uscales[u >> 2] = (uint8_t)bu;
                    if constexpr (EMIT) hscales[u >> 2] = (uint8_t)bh;
                }
            }
        }
    }
}

template <int DT>
__global__ void __launch_bounds__(kA8Threads)
swiglu_backward_kernel(const void* __restrict__ dh, int64_t rows, int cols, int64_t ld_dh, uint32_t per_row,
                       bool vec, const uint8_t* __restrict__ gcodes, const uint8_t* __restrict__ gscales,
                       const uint8_t* __restrict__ ucodes, const uint8_t* __restrict__ uscales,
                       void* __restrict__ dgate, void* __restrict__ dup, int64_t ld_out, bool vec_out) {
    constexpr int kC = 2, kR = 32 * kC;
    const int lane = threadIdx.x & 31;
    const int64_t units = rows * per_row;
    const int64_t warps = (int64_t)gridDim.x * (kA8Threads / 32);
    for (int64_t w = (int64_t)blockIdx.x * (kA8Threads / 32) + (threadIdx.x >> 5); w * kR < units; w += warps) {
        const int64_t unit0 = w * kR;
        const RunAt run = run_at(unit0, per_row);
        Raw8<DT> rd[kC];
        uint2 qg[kC], qu[kC];
        int bg[kC], bu[kC];
        ChunkAt at[kC];
#pragma unroll
        for (int j = 0; j < kC; ++j) {
            const int64_t u = unit0 + j * 32 + lane;
            at[j] = chunk_at(run, j * 32 + lane, per_row, rows);
            if (!at[j].in) continue;
            rd[j] = load_raw8<DT>(dh, at[j].row * ld_dh, at[j].col, cols, vec);
            qg[j] = __ldcs(reinterpret_cast<const uint2*>(gcodes + u * 8));
            qu[j] = __ldcs(reinterpret_cast<const uint2*>(ucodes + u * 8));
            bg[j] = gscales[u >> 2];
            bu[j] = uscales[u >> 2];
        }
#pragma unroll
        for (int j = 0; j < kC; ++j) {
            if (!at[j].in) continue;
            float d[8], g[8], p[8];
            widen8<DT>(rd[j], d);
            a8_decode8(qg[j], a8_scale(bg[j]), g);
            a8_decode8(qu[j], a8_scale(bu[j]), p);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float s = sigmoid<DT>(g[i]);
                const float gs = g[i] * s;
                p[i] = d[i] * p[i] * __fmaf_rn(gs, 1.0f - s, s);
                g[i] = d[i] * gs;
            }
            store_raw8<DT>(dgate, at[j].row * ld_out, at[j].col, cols, vec_out, narrow8<DT>(p));
            store_raw8<DT>(dup, at[j].row * ld_out, at[j].col, cols, vec_out, narrow8<DT>(g));
        }
    }
}

// ---------------------------------------------------------------------------
// RMS norm: y = x r w, r = (mean(x^2) + eps)^-1/2
// ---------------------------------------------------------------------------

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the NT threads that share a row; NT == 32: a warp per row.
// `slot` alternates so that one barrier per sum is enough.
template <int NT>
__device__ __forceinline__ float row_sum(float v, float (*part)[32], int slot) {
    v = warp_sum(v);
    if constexpr (NT == 32) {
        return v;
    } else {
        if ((threadIdx.x & 31) == 0) part[slot][threadIdx.x >> 5] = v;
        __syncthreads();
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) s += part[slot][i];
        return s;
    }
}

__device__ __forceinline__ float load_weight(const void* w, int dtype, int col, int cols) {
    if (col >= cols) return 0.0f;
    if (dtype == AW4_F32) return Elem<AW4_F32>::load1(w, col);
    if (dtype == AW4_BF16) return Elem<AW4_BF16>::load1(w, col);
    return Elem<AW4_F16>::load1(w, col);
}

// A row belongs to NT threads that hold V chunks of eight values each.
template <int DT, int NT, int V>
__global__ void __launch_bounds__(NT == 32 ? 256 : NT)
rms_norm_forward_kernel(const void* __restrict__ x, int64_t rows, int cols, int64_t ld, uint32_t per_row,
                        bool vec, const void* __restrict__ w, int w_dtype, float eps, void* __restrict__ y,
                        bool vec_y, float* __restrict__ rstd, uint8_t* __restrict__ codes,
                        uint8_t* __restrict__ scales, uint8_t* __restrict__ ycodes,
                        uint8_t* __restrict__ yscales) {
    __shared__ float part[2][32];
    constexpr int kRows = NT == 32 ? 8 : 1;
    const int t = NT == 32 ? (threadIdx.x & 31) : threadIdx.x;
    int slot = 0;
    for (int64_t row = (int64_t)blockIdx.x * kRows + (NT == 32 ? threadIdx.x >> 5 : 0); row < rows;
         row += (int64_t)gridDim.x * kRows, slot ^= 1) {
        Raw8<DT> raw[V];
#pragma unroll
        for (int j = 0; j < V; ++j) raw[j] = load_raw8<DT>(x, row * ld, (j * NT + t) * 8, cols, vec);
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float v[8];
            widen8<DT>(raw[j], v);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __fmaf_rn(v[i], v[i], ss);
        }
        const float r = 1.0f / sqrtf(row_sum<NT>(ss, part, slot) / (float)cols + eps);
        if (t == 0) rstd[row] = r;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t u = j * NT + t;
            const int col = (int)u * 8;
            float v[8], o[8];
            widen8<DT>(raw[j], v);
            const int b = a8_scale_byte<DT>(v);
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = v[i] * r * load_weight(w, w_dtype, col + i, cols);
            const Raw8<DT> ry = narrow8<DT>(o);
            int by = 0;
            if (ycodes) {               // the checkpoint of y is that of its rounded values
                widen8<DT>(ry, o);
                by = a8_scale_byte<DT>(o);
            }
            if (u < per_row) {
                const int64_t at = row * per_row + u;
                *reinterpret_cast<uint2*>(codes + at * 8) = a8_encode8(v, b);
                if ((t & 3) == 0) scales[at >> 2] = (uint8_t)b;
                store_raw8<DT>(y, row * cols, col, cols, vec_y, ry);
                if (ycodes) {
                    *reinterpret_cast<uint2*>(ycodes + at * 8) = a8_encode8(o, by);
                    if ((t & 3) == 0) yscales[at >> 2] = (uint8_t)by;
                }
            }
        }
    }
}

// dx = r (w dy) - v r^3 mean(v w dy); each block leaves its rows' sum of
// dy v r in partial[blockIdx.x][cols].
template <int DT, int NT, int V>
__global__ void __launch_bounds__(NT == 32 ? 256 : NT)
rms_norm_backward_kernel(const void* __restrict__ dy, int64_t rows, int cols, int64_t ld, uint32_t per_row,
                         bool vec, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                         const float* __restrict__ rstd, const void* __restrict__ w, int w_dtype,
                         void* __restrict__ dx, bool vec_dx, float* __restrict__ partial) {
    __shared__ float part[2][32];
    constexpr int kRows = NT == 32 ? 8 : 1;
    const int t = NT == 32 ? (threadIdx.x & 31) : threadIdx.x;
    float acc[V][8] = {};
    int slot = 0;
    for (int64_t row = (int64_t)blockIdx.x * kRows + (NT == 32 ? threadIdx.x >> 5 : 0); row < rows;
         row += (int64_t)gridDim.x * kRows, slot ^= 1) {
        Raw8<DT> raw[V];
        uint2 q[V];
        int b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t u = j * NT + t;
            const int64_t at = row * per_row + u;
            raw[j] = load_raw8<DT>(dy, row * ld, (int)u * 8, cols, vec);
            q[j] = u < per_row ? __ldcs(reinterpret_cast<const uint2*>(codes + at * 8)) : make_uint2(0, 0);
            b[j] = u < per_row ? scales[at >> 2] : 1;
        }
        const float r = rstd[row];
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float d[8], v[8];
            widen8<DT>(raw[j], d);
            a8_decode8(q[j], a8_scale(b[j]), v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int col = (j * NT + t) * 8 + i;
                const float dv = col < cols ? d[i] * v[i] : 0.0f;
                dot = __fmaf_rn(dv, load_weight(w, w_dtype, col, cols), dot);
                acc[j][i] = __fmaf_rn(dv, r, acc[j][i]);
            }
        }
        const float k = r * r * r * (row_sum<NT>(dot, part, slot) / (float)cols);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t u = j * NT + t;
            float d[8], v[8];
            widen8<DT>(raw[j], d);
            a8_decode8(q[j], a8_scale(b[j]), v);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                d[i] = __fmaf_rn(r * load_weight(w, w_dtype, (int)u * 8 + i, cols), d[i], -(v[i] * k));
            if (u < per_row) store_raw8<DT>(dx, row * cols, (int)u * 8, cols, vec_dx, narrow8<DT>(d));
        }
    }
    if constexpr (NT == 32) {
        // the block's eight warps hold the same columns: added in their order
        __shared__ float sums[V * 256];
        for (int i = threadIdx.x; i < V * 256; i += 256) sums[i] = 0.0f;
        for (int wi = 0; wi < 8; ++wi) {
            __syncthreads();
            if ((int)(threadIdx.x >> 5) == wi)
#pragma unroll
                for (int j = 0; j < V; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sums[(j * 32 + t) * 8 + i] += acc[j][i];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < cols; i += 256) partial[(int64_t)blockIdx.x * cols + i] = sums[i];
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int col = (j * NT + t) * 8 + i;
                if (col < cols) partial[(int64_t)blockIdx.x * cols + col] = acc[j][i];
            }
    }
}

// Column sums of partial[parts][cols], in a fixed order: 32 threads share a column.
template <int DT>
__global__ void __launch_bounds__(1024)
column_sum_kernel(const float* __restrict__ partial, int parts, int cols, void* __restrict__ out) {
    __shared__ float s[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x;
    float v = 0.0f;
    if (c < cols)
        for (int p = threadIdx.y; p < parts; p += 32) v += partial[(int64_t)p * cols + c];
    s[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    v = warp_sum(s[threadIdx.x][threadIdx.y]);
    const int col = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && col < cols) Elem<DT>::store1(out, col, v);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

static int sm_count(int device) {
    int sms = 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms <= 0)
        sms = 1;
    return sms;
}

static bool known_dtype(int dtype) { return dtype >= AW4_F32 && dtype <= AW4_F16; }
static int size_of(int dtype) { return dtype == AW4_F32 ? 4 : 2; }

// Whether whole chunks of eight values of every row start on 16 bytes.
static bool vec_ok(const void* p, int64_t ld, int dtype) {
    return (uintptr_t)p % 16 == 0 && (ld * size_of(dtype)) % 16 == 0;
}

static int32_t check_matrix(const char* what, int dtype, int64_t rows, int64_t cols) {
    if (!known_dtype(dtype)) return fail(AW4_ERR_INVALID, "%s: bad dtype %d", what, dtype);
    if (rows < 0 || cols < 0) return fail(AW4_ERR_INVALID, "%s: negative size", what);
    if (cols > (int64_t)1 << 30) return fail(AW4_ERR_UNSUPPORTED, "%s: rows of more than 2^30 values", what);
    return AW4_OK;
}

static int32_t launched(const char* what) {
    note_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? AW4_OK : fail(AW4_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

static uint32_t chunks_per_row(int64_t cols) { return (uint32_t)((cols + kA8Block - 1) / kA8Block * 4); }

static int run_grid(int device, int64_t units, int run) {
    const int64_t per_block = (int64_t)run * (kA8Threads / 32);
    return (int)std::max<int64_t>(1, std::min<int64_t>((units + per_block - 1) / per_block,
                                                       (int64_t)sm_count(device) * 64));
}

// Rows' threads and chunks: the fewest threads whose chunks cover the row.
// Up to 1024 columns a warp holds a row and needs no barrier.
template <typename F>
static int32_t norm_shape(int64_t cols, F f) {
    if (cols <= 256) return f(std::integral_constant<int, 32>(), std::integral_constant<int, 1>());
    if (cols <= 512) return f(std::integral_constant<int, 32>(), std::integral_constant<int, 2>());
    if (cols <= 1024) return f(std::integral_constant<int, 32>(), std::integral_constant<int, 4>());
    if (cols <= 2048) return f(std::integral_constant<int, 128>(), std::integral_constant<int, 2>());
    if (cols <= 4096) return f(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
    if (cols <= 8192) return f(std::integral_constant<int, 512>(), std::integral_constant<int, 2>());
    return f(std::integral_constant<int, 512>(), std::integral_constant<int, 4>());
}

template <typename F>
static int32_t by_dtype(int dtype, F f) {
    if (dtype == AW4_F32) return f(std::integral_constant<int, AW4_F32>());
    if (dtype == AW4_BF16) return f(std::integral_constant<int, AW4_BF16>());
    return f(std::integral_constant<int, AW4_F16>());
}

constexpr int64_t kNormCols = 16384;

// Blocks of the backward kernel, and so rows of its partial sums.
static int norm_backward_grid(int device, int64_t rows, int64_t cols) {
    const int64_t per_block = cols <= 1024 ? 8 : 1;
    const int per_sm = cols <= 2048 ? 4 : cols <= 4096 ? 3 : 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>((rows + per_block - 1) / per_block,
                                                       (int64_t)sm_count(device) * per_sm));
}

}  // namespace aw4

using namespace aw4;

extern "C" int32_t aw4_act8_quantize(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t ld,
                                     uint8_t* codes, uint8_t* scales, int32_t device, void* stream) {
    if (const int32_t rc = check_matrix("aw4_act8_quantize", dtype, rows, cols)) return rc;
    if (rows == 0 || cols == 0) return AW4_OK;
    if (!x || !codes || !scales || (uintptr_t)codes % 16)
        return fail(AW4_ERR_INVALID, "aw4_act8_quantize: null or misaligned buffer");
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(AW4_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    const uint32_t per_row = chunks_per_row(cols);
    return by_dtype(dtype, [&](auto dt) {
        act8_quantize_kernel<dt.value><<<run_grid(device, rows * per_row, kRun), kA8Threads, 0,
                                         (cudaStream_t)stream>>>(x, rows, (int)cols, ld, per_row,
                                                                 vec_ok(x, ld, dtype), codes, scales);
        return launched("act8_quantize");
    });
}

extern "C" int32_t aw4_act8_dequantize(const uint8_t* codes, const uint8_t* scales, int32_t dtype,
                                       int64_t rows, int64_t cols, void* out, int64_t ld, int32_t device,
                                       void* stream) {
    if (const int32_t rc = check_matrix("aw4_act8_dequantize", dtype, rows, cols)) return rc;
    if (rows == 0 || cols == 0) return AW4_OK;
    if (!codes || !scales || !out || (uintptr_t)codes % 16)
        return fail(AW4_ERR_INVALID, "aw4_act8_dequantize: null or misaligned buffer");
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(AW4_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    const uint32_t per_row = chunks_per_row(cols);
    return by_dtype(dtype, [&](auto dt) {
        act8_dequantize_kernel<dt.value><<<run_grid(device, rows * per_row, kRun), kA8Threads, 0,
                                           (cudaStream_t)stream>>>(codes, scales, rows, (int)cols, per_row,
                                                                   out, ld, vec_ok(out, ld, dtype));
        return launched("act8_dequantize");
    });
}

extern "C" int32_t aw4_swiglu_forward(const void* gate, const void* up, int32_t dtype, int64_t rows,
                                      int64_t cols, int64_t ld_gate, int64_t ld_up, void* h,
                                      uint8_t* gcodes, uint8_t* gscales, uint8_t* ucodes, uint8_t* uscales,
                                      uint8_t* hcodes, uint8_t* hscales, int32_t device, void* stream) {
    if (const int32_t rc = check_matrix("aw4_swiglu_forward", dtype, rows, cols)) return rc;
    if (rows == 0 || cols == 0) return AW4_OK;
    if (!gate || !up || !h || !gcodes || !gscales || !ucodes || !uscales || !hcodes != !hscales ||
        ((uintptr_t)gcodes | (uintptr_t)ucodes | (uintptr_t)hcodes) % 16)
        return fail(AW4_ERR_INVALID, "aw4_swiglu_forward: null or misaligned buffer");
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(AW4_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    const uint32_t per_row = chunks_per_row(cols);
    const bool vec = vec_ok(gate, ld_gate, dtype) && vec_ok(up, ld_up, dtype);
    const int grid = run_grid(device, rows * per_row, 64);
    return by_dtype(dtype, [&](auto dt) {
        if (hcodes)
            swiglu_forward_kernel<dt.value, true><<<grid, kA8Threads, 0, (cudaStream_t)stream>>>(
                gate, up, rows, (int)cols, ld_gate, ld_up, per_row, vec, h, cols, vec_ok(h, cols, dtype),
                gcodes, gscales, ucodes, uscales, hcodes, hscales);
        else
            swiglu_forward_kernel<dt.value, false><<<grid, kA8Threads, 0, (cudaStream_t)stream>>>(
                gate, up, rows, (int)cols, ld_gate, ld_up, per_row, vec, h, cols, vec_ok(h, cols, dtype),
                gcodes, gscales, ucodes, uscales, nullptr, nullptr);
        return launched("swiglu_forward");
    });
}

extern "C" int32_t aw4_swiglu_backward(const void* dh, int32_t dtype, int64_t rows, int64_t cols,
                                       int64_t ld_dh, const uint8_t* gcodes, const uint8_t* gscales,
                                       const uint8_t* ucodes, const uint8_t* uscales, void* dgate, void* dup,
                                       int64_t ld_out, int32_t device, void* stream) {
    if (const int32_t rc = check_matrix("aw4_swiglu_backward", dtype, rows, cols)) return rc;
    if (rows == 0 || cols == 0) return AW4_OK;
    if (!dh || !gcodes || !gscales || !ucodes || !uscales || !dgate || !dup ||
        ((uintptr_t)gcodes | (uintptr_t)ucodes) % 16)
        return fail(AW4_ERR_INVALID, "aw4_swiglu_backward: null or misaligned buffer");
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(AW4_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    const uint32_t per_row = chunks_per_row(cols);
    return by_dtype(dtype, [&](auto dt) {
        swiglu_backward_kernel<dt.value><<<run_grid(device, rows * per_row, 64), kA8Threads, 0,
                                           (cudaStream_t)stream>>>(
            dh, rows, (int)cols, ld_dh, per_row, vec_ok(dh, ld_dh, dtype), gcodes, gscales, ucodes, uscales,
            dgate, dup, ld_out, vec_ok(dgate, ld_out, dtype) && vec_ok(dup, ld_out, dtype));
        return launched("swiglu_backward");
    });
}

extern "C" int32_t aw4_rms_norm_forward(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t ld,
                                        const void* weight, int32_t weight_dtype, float eps, void* y,
                                        float* rstd, uint8_t* codes, uint8_t* scales, uint8_t* ycodes,
                                        uint8_t* yscales, int32_t device, void* stream) {
    if (const int32_t rc = check_matrix("aw4_rms_norm_forward", dtype, rows, cols)) return rc;
    if (!known_dtype(weight_dtype))
        return fail(AW4_ERR_INVALID, "aw4_rms_norm_forward: bad weight dtype %d", weight_dtype);
    if (cols > kNormCols)
        return fail(AW4_ERR_UNSUPPORTED, "aw4_rms_norm_forward: rows of more than %d values", (int)kNormCols);
    if (rows == 0 || cols == 0) return AW4_OK;
    if (!x || !weight || !y || !rstd || !codes || !scales || !ycodes != !yscales ||
        ((uintptr_t)codes | (uintptr_t)ycodes) % 16)
        return fail(AW4_ERR_INVALID, "aw4_rms_norm_forward: null or misaligned buffer");
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(AW4_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    const uint32_t per_row = chunks_per_row(cols);
    return by_dtype(dtype, [&](auto dt) {
        return norm_shape(cols, [&](auto nt, auto v) {
            constexpr int kRows = nt.value == 32 ? 8 : 1;
            const int grid = (int)std::min<int64_t>((rows + kRows - 1) / kRows, (int64_t)sm_count(device) * 64);
            rms_norm_forward_kernel<dt.value, nt.value, v.value>
                <<<grid, nt.value == 32 ? 256 : nt.value, 0, (cudaStream_t)stream>>>(
                    x, rows, (int)cols, ld, per_row, vec_ok(x, ld, dtype), weight, weight_dtype, eps, y,
                    vec_ok(y, cols, dtype), rstd, codes, scales, ycodes, yscales);
            return launched("rms_norm_forward");
        });
    });
}

extern "C" uint64_t aw4_rms_norm_backward_workspace(int64_t rows, int64_t cols, int32_t device) {
    if (rows <= 0 || cols <= 0 || cols > kNormCols) return 0;
    return (uint64_t)norm_backward_grid(device, rows, cols) * cols * sizeof(float);
}

extern "C" int32_t aw4_rms_norm_backward(const void* dy, int32_t dtype, int64_t rows, int64_t cols, int64_t ld,
                                         const uint8_t* codes, const uint8_t* scales, const float* rstd,
                                         const void* weight, int32_t weight_dtype, void* dx, void* dweight,
                                         float* workspace, int64_t workspace_bytes, int32_t device,
                                         void* stream) {
    if (const int32_t rc = check_matrix("aw4_rms_norm_backward", dtype, rows, cols)) return rc;
    if (!known_dtype(weight_dtype))
        return fail(AW4_ERR_INVALID, "aw4_rms_norm_backward: bad weight dtype %d", weight_dtype);
    if (cols > kNormCols)
        return fail(AW4_ERR_UNSUPPORTED, "aw4_rms_norm_backward: rows of more than %d values", (int)kNormCols);
    if (cols == 0) return AW4_OK;
    if (!dweight) return fail(AW4_ERR_INVALID, "aw4_rms_norm_backward: null buffer");
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(AW4_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    cudaStream_t s = (cudaStream_t)stream;
    if (rows == 0) {
        const cudaError_t e = cudaMemsetAsync(dweight, 0, cols * size_of(weight_dtype), s);
        return e == cudaSuccess ? AW4_OK
                                : fail(AW4_ERR_CUDA, "rms_norm_backward: %s", cudaGetErrorString(e));
    }
    if (!dy || !codes || !scales || !rstd || !weight || !dx || (uintptr_t)codes % 16)
        return fail(AW4_ERR_INVALID, "aw4_rms_norm_backward: null or misaligned buffer");
    const int grid = norm_backward_grid(device, rows, cols);
    if (!workspace || workspace_bytes < (int64_t)grid * cols * (int64_t)sizeof(float))
        return fail(AW4_ERR_INVALID, "aw4_rms_norm_backward: workspace of %lld bytes is too small",
                    (long long)workspace_bytes);
    const uint32_t per_row = chunks_per_row(cols);
    const int32_t rc = by_dtype(dtype, [&](auto dt) {
        return norm_shape(cols, [&](auto nt, auto v) {
            rms_norm_backward_kernel<dt.value, nt.value, v.value>
                <<<grid, nt.value == 32 ? 256 : nt.value, 0, s>>>(
                    dy, rows, (int)cols, ld, per_row, vec_ok(dy, ld, dtype), codes, scales, rstd, weight,
                    weight_dtype, dx, vec_ok(dx, cols, dtype), workspace);
            return launched("rms_norm_backward");
        });
    });
    if (rc) return rc;
    return by_dtype(weight_dtype, [&](auto wt) {
        column_sum_kernel<wt.value><<<(int)((cols + 31) / 32), dim3(32, 32), 0, s>>>(workspace, grid, (int)cols,
                                                                                    dweight);
        return launched("column_sum");
    });
}
