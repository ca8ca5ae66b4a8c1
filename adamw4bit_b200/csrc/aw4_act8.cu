// aw4_act8.cu -- 8-bit activation checkpoints and the elementwise backward passes that read them.
//
// Every kernel here is one pass over its inputs, bound by HBM.  A warp takes
// a run of 32 * k chunks of eight values; the run's loads are issued before the
// first is used.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/adamw4bit_b200.h"
#include "aw4_act8.cuh"
#include "aw4_host.h"

namespace aw4 {

constexpr int kA8Threads = 256;
constexpr int kChunks = 4;                      // chunks of eight values per lane in flight
constexpr int kRun = 32 * kChunks;              // chunks of a warp

// Writes the scale bytes of a run, 32 blocks, together.
__device__ __forceinline__ void store_scales(uint8_t* scales, int64_t unit0, int64_t blocks,
                                             const A8Block b[kChunks], int lane) {
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        const int got = __shfl_sync(0xffffffffu, b[j].byte, (lane & 7) * 4);
        if ((lane >> 3) == j) mine = got;
    }
    const int64_t blk = (unit0 >> 2) + lane;
    if (blk < blocks) scales[blk] = (uint8_t)mine;
}

// The first chunk of this thread's warp.
__device__ __forceinline__ int64_t warp_run(int run) {
    return ((int64_t)blockIdx.x * (kA8Threads / 32) + (threadIdx.x >> 5)) * run;
}

// A lane reads 16 bytes of bf16 and writes 8 of codes; 32 blocks' exponents leave a warp together.  Bound by
// HBM: 8192 x 14336 bf16 in 55 to 60 us over several chips, 6.0 to 6.5 TB/s (72 us with a capped grid whose warps had one run or two).
template <int DT, bool WHOLE>
__global__ void __launch_bounds__(kA8Threads)
act8_quantize_kernel(const RowsIn x, int64_t rows, int cols, uint32_t per_row, uint8_t* __restrict__ codes,
                     uint8_t* __restrict__ scales) {
    const int lane = threadIdx.x & 31;
    const int64_t units = rows * per_row, unit0 = warp_run(kRun);
    if (unit0 >= units) return;
    const RunAt run = run_at(unit0, per_row);
    Raw8<DT> raw[kChunks];
    bool in[kChunks];
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        const ChunkAt c = chunk_at(run, j * 32 + lane, per_row, rows);
        in[j] = c.in;
        raw[j] = load_raw8<DT, WHOLE>(x, c.in ? c.row : 0, c.col, c.in ? cols : 0);
    }
    A8Block b[kChunks];
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        float v[8];
        widen8<DT>(raw[j], v);
        b[j] = a8_block<DT>(raw[j]);
        const uint2 q = a8_encode8(v, b[j]);
        if (in[j]) *reinterpret_cast<uint2*>(codes + (unit0 + j * 32 + lane) * 8) = q;
    }
    store_scales(scales, unit0, units >> 2, b, lane);
}

// Bound by HBM: 8192 x 14336 bf16 in 52 us, 6.9 TB/s.
template <int DT, bool WHOLE>
__global__ void __launch_bounds__(kA8Threads)
act8_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows,
                       int cols, uint32_t per_row, const RowsOut out) {
    const int lane = threadIdx.x & 31;
    const int64_t units = rows * per_row, unit0 = warp_run(kRun);
    if (unit0 >= units) return;
    const RunAt run = run_at(unit0, per_row);
    uint2 q[kChunks];
    int b[kChunks];
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        const int64_t u = unit0 + j * 32 + lane;
        q[j] = make_uint2(0, 0);
        b[j] = 1;
        if (u < units) {
            q[j] = __ldcs(reinterpret_cast<const uint2*>(codes + u * 8));
            b[j] = scales[u >> 2];
        }
    }
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        const ChunkAt c = chunk_at(run, j * 32 + lane, per_row, rows);
        float v[8];
        a8_decode8(q[j], a8_scale(b[j]), v);
        store_raw8_warp<DT, WHOLE, true>(out, c.row, c.col, cols, c.in, narrow8<DT>(v));
    }
}

// ---------------------------------------------------------------------------
// gated activation: h = g sigmoid(g) u
// ---------------------------------------------------------------------------

// float32 takes expf and a division: a few units in the last place, 0 once exp(-g) is above float32 (g < -88.7).  The
// 16-bit types take the hardware's exponential and reciprocal: off by (8 + 1.25 |g|) 2^-24 of the value, 0 from g < -87.4 on,
// both far below their rounding.
template <int DT>
__device__ __forceinline__ float sigmoid(float g) {
    if constexpr (DT == AW4_F32) {
        return 1.0f / (1.0f + expf(-g));
    } else {
        float e, r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.44269504f));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
        return r;
    }
}

// Chunks in flight: two forward (153 us at 8192 x 14336 bf16; 164 with one, 157 with four), one backward (145 us;
// 167 with two, 205 with four).
constexpr int kGluForward = 2, kGluBackward = 1;

// Reads g and u, writes h and both checkpoints (EMIT: and that of h).  Bound by HBM: 8192 x 14336 bf16 in 153 us,
// 6.2 TB/s.
template <int DT, bool WHOLE, bool EMIT>
__global__ void __launch_bounds__(kA8Threads)
swiglu_forward_kernel(const RowsIn gate, const RowsIn up, int64_t rows, int cols, uint32_t per_row,
                      const RowsOut h, uint8_t* __restrict__ gcodes, uint8_t* __restrict__ gscales,
                      uint8_t* __restrict__ ucodes, uint8_t* __restrict__ uscales,
                      uint8_t* __restrict__ hcodes, uint8_t* __restrict__ hscales) {
    const int lane = threadIdx.x & 31;
    const int64_t units = rows * per_row, unit0 = warp_run(32 * kGluForward);
    if (unit0 >= units) return;
    const RunAt run = run_at(unit0, per_row);
    Raw8<DT> rg[kGluForward], ru[kGluForward];
    ChunkAt at[kGluForward];
#pragma unroll
    for (int j = 0; j < kGluForward; ++j) {
        at[j] = chunk_at(run, j * 32 + lane, per_row, rows);
        rg[j] = load_raw8<DT, WHOLE>(gate, at[j].in ? at[j].row : 0, at[j].col, at[j].in ? cols : 0);
        ru[j] = load_raw8<DT, WHOLE>(up, at[j].in ? at[j].row : 0, at[j].col, at[j].in ? cols : 0);
    }
#pragma unroll
    for (int j = 0; j < kGluForward; ++j) {
        const int64_t u = unit0 + j * 32 + lane;
        float g[8], p[8], y[8];
        widen8<DT>(rg[j], g);
        widen8<DT>(ru[j], p);
        const A8Block bg = a8_block<DT>(rg[j]), bu = a8_block<DT>(ru[j]);
        const uint2 qg = a8_encode8(g, bg), qu = a8_encode8(p, bu);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = sigmoid<DT>(g[i]);
        vmul8(y, y, g);
        vmul8(y, y, p);
        const Raw8<DT> r = narrow8<DT>(y);
        A8Block bh = {0, 0.0f};
        uint2 qh = make_uint2(0, 0);
        if constexpr (EMIT) {       // the checkpoint of h is that of its rounded values
            widen8<DT>(r, y);
            bh = a8_block<DT>(r);
            qh = a8_encode8(y, bh);
        }
        store_raw8_warp<DT, WHOLE>(h, at[j].row, at[j].col, cols, at[j].in, r);
        if (!at[j].in) continue;
        *reinterpret_cast<uint2*>(gcodes + u * 8) = qg;
        *reinterpret_cast<uint2*>(ucodes + u * 8) = qu;
        if constexpr (EMIT) *reinterpret_cast<uint2*>(hcodes + u * 8) = qh;
        if ((lane & 3) == 0) {
            gscales[u >> 2] = (uint8_t)bg.byte;
            uscales[u >> 2] = (uint8_t)bu.byte;
            if constexpr (EMIT) hscales[u >> 2] = (uint8_t)bh.byte;
        }
    }
}

// dg = dh u (s + g s (1 - s)), du = dh g s, s = sigmoid(g), g and u from their checkpoints.  Bound by HBM:
// 8192 x 14336 bf16 in 145 us, 6.5 TB/s.
template <int DT, bool WHOLE>
__global__ void __launch_bounds__(kA8Threads)
swiglu_backward_kernel(const RowsIn dh, int64_t rows, int cols, uint32_t per_row,
                       const uint8_t* __restrict__ gcodes, const uint8_t* __restrict__ gscales,
                       const uint8_t* __restrict__ ucodes, const uint8_t* __restrict__ uscales,
                       const RowsOut dgate, const RowsOut dup) {
    const int lane = threadIdx.x & 31;
    const int64_t units = rows * per_row, unit0 = warp_run(32 * kGluBackward);
    if (unit0 >= units) return;
    const RunAt run = run_at(unit0, per_row);
    Raw8<DT> rd[kGluBackward];
    uint2 qg[kGluBackward], qu[kGluBackward];
    int bg[kGluBackward], bu[kGluBackward];
    ChunkAt at[kGluBackward];
#pragma unroll
    for (int j = 0; j < kGluBackward; ++j) {
        const int64_t u = unit0 + j * 32 + lane;
        at[j] = chunk_at(run, j * 32 + lane, per_row, rows);
        rd[j] = {};
        qg[j] = qu[j] = make_uint2(0, 0);
        bg[j] = bu[j] = 1;
        if (!at[j].in) continue;
        rd[j] = load_raw8<DT, WHOLE>(dh, at[j].row, at[j].col, cols);
        qg[j] = __ldcs(reinterpret_cast<const uint2*>(gcodes + u * 8));
        qu[j] = __ldcs(reinterpret_cast<const uint2*>(ucodes + u * 8));
        bg[j] = gscales[u >> 2];
        bu[j] = uscales[u >> 2];
    }
#pragma unroll
    for (int j = 0; j < kGluBackward; ++j) {
        float d[8], g[8], p[8], s[8], f[8];
        widen8<DT>(rd[j], d);
        a8_decode8(qg[j], a8_scale(bg[j]), g);
        a8_decode8(qu[j], a8_scale(bu[j]), p);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            s[i] = sigmoid<DT>(g[i]);
            f[i] = 1.0f - s[i];
        }
        vmul8(g, g, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = __fmaf_rn(g[i], f[i], s[i]);
        vmul8(p, p, d);
        vmul8(p, p, s);
        vmul8(g, g, d);
        store_raw8_warp<DT, WHOLE>(dgate, at[j].row, at[j].col, cols, at[j].in, narrow8<DT>(p));
        store_raw8_warp<DT, WHOLE>(dup, at[j].row, at[j].col, cols, at[j].in, narrow8<DT>(g));
    }
}

// ---------------------------------------------------------------------------
// RMS norm: y = x r w, r = (mean(x^2) + eps)^-1/2
// ---------------------------------------------------------------------------
//
// A row belongs to NT threads that hold V chunks of eight values each; up to a warp
// no barrier, and a warp has 32 / NT rows.  Blocks stay and walk the rows, the next row's loads on
// their way while one is worked on.  The weight waits in shared memory, and the
// backward kernel keeps its columns' sum of dy v r in registers over all its rows.
// Two chunks a thread: a row's own cost, the sum over its threads, is then half of
// what one chunk a thread pays (forward 73 us at 16384 x 4096 bf16 with one).

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the NT threads that share a row.  `slot` alternates so that one
// barrier per sum is enough.
template <int NT>
__device__ __forceinline__ float row_sum(float v, float (*part)[NT < 64 ? 1 : NT / 32], int slot) {
    if constexpr (NT <= 32) {
#pragma unroll
        for (int o = NT / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    } else {
        v = warp_sum(v);
        if ((threadIdx.x & 31) == 0) part[slot][threadIdx.x >> 5] = v;
        __syncthreads();
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) s += part[slot][i];
        return s;
    }
}

// 1 / sqrt(x): the hardware's estimate and one step of Newton's method for a positive normal x.
__device__ __forceinline__ float inv_sqrt(float x) {
    if (!(x >= 1.17549435e-38f && x < INFINITY)) return 1.0f / sqrtf(x);
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return __fmaf_rn(0.5f * r, __fmaf_rn(-x * r, r, 1.0f), r);
}

// A thread's chunks of the weight as float32 in shared memory, zeros behind the
// last column: the first halves of all chunks, then the second, so that a warp
// reads whole lines.  A thread reads what it wrote: no barrier.
template <int NT, int V>
__device__ __forceinline__ void stage_weight(const void* w, int dtype, int cols, int t, float4* s) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int u = j * NT + t, col = u * 8;
        float v[8];
        const char* p = static_cast<const char*>(w) + (int64_t)col * (dtype == AW4_F32 ? 4 : 2);
        if (col + 8 <= cols && (uintptr_t)p % 16 == 0) {
            if (dtype == AW4_F32) Elem<AW4_F32>::load8(w, col, v);
            else if (dtype == AW4_BF16) Elem<AW4_BF16>::load8(w, col, v);
            else Elem<AW4_F16>::load8(w, col, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = 0.0f;
                if (col + i < cols)
                    v[i] = dtype == AW4_F32    ? Elem<AW4_F32>::load1(w, col + i)
                           : dtype == AW4_BF16 ? Elem<AW4_BF16>::load1(w, col + i)
                                               : Elem<AW4_F16>::load1(w, col + i);
            }
        }
        s[u] = make_float4(v[0], v[1], v[2], v[3]);
        s[NT * V + u] = make_float4(v[4], v[5], v[6], v[7]);
    }
}
__device__ __forceinline__ void weight8(const float4* s, int chunks, int u, float v[8]) {
    const float4 a = s[u], b = s[chunks + u];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

constexpr int kNormWarps = 4;       // warps of a block where rows belong to warps, at most

// Blocks resident on an SM for that many threads of it.
template <int NT>
constexpr int norm_blocks(int threads) {
    return NT <= 32 ? threads / (32 * kNormWarps) : NT < threads ? threads / NT : 1;
}

// Which rows a thread works on: `first` and every `step` behind it, as long as `warp_first` of its warp (of its
// block, where a row has more) is one; t: the thread's place in the row.
template <int NT>
struct NormWalk {
    int64_t first, warp_first, step;
    int t;
    __device__ __forceinline__ NormWalk() {
        constexpr int kRows = NT < 32 ? 32 / NT : 1;
        const int warps = NT <= 32 ? blockDim.x >> 5 : 1, warp = NT <= 32 ? threadIdx.x >> 5 : 0;
        step = (int64_t)gridDim.x * warps * kRows;
        warp_first = ((int64_t)blockIdx.x * warps + warp) * kRows;
        first = warp_first + (NT < 32 ? (threadIdx.x & 31) / NT : 0);
        t = threadIdx.x % NT;
    }
};
// Forward: 1024 threads of an SM at 64 registers (55 us at 16384 x 4096 bf16; 58 with 768, 64 with 512).
// Backward: 768 at 85 (61 us; 66 with 512, 103 with 1024, where its sums spill); 512 where what a thread has of
// the next row is larger, in float32 and in the two chunks of a warp's row (2047 x 1531 float32: 14 us, 17 with 768).
// Rows of more than 8192 values off 16 bytes, or 12288, need 1024 threads and spill all the same: 84 to 152 bytes a thread
// are read back a row in 16 bits, 152 to 252 in float32 (4096 x 16384 bf16 in 134 us, 3.0 TB/s).
constexpr int kNormForward = 1024, kNormBackwardMost = 768;
template <int DT, int NT, int V>
constexpr int kNormBackward = DT == AW4_F32 || (NT == 32 && V == 2) ? 512 : kNormBackwardMost;

// Bound by HBM: 16384 x 4096 bf16 in 55 us, 6.2 TB/s.
template <int DT, int NT, int V, bool WHOLE>
__global__ void __launch_bounds__(NT <= 32 ? 32 * kNormWarps : NT, norm_blocks<NT>(kNormForward))
rms_norm_forward_kernel(const RowsIn x, int64_t rows, int cols, float inv_cols, int per_row,
                        const void* __restrict__ w, int w_dtype, float eps, const RowsOut y,
                        float* __restrict__ rstd, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                        uint8_t* __restrict__ ycodes, uint8_t* __restrict__ yscales) {
    __shared__ float part[2][NT < 64 ? 1 : NT / 32];
    extern __shared__ float4 weight_s[];
    constexpr int kChunks8 = NT * V;
    const NormWalk<NT> walk;
    const int t = walk.t;
    const int64_t step = walk.step;
    int64_t row = walk.first;
    Raw8<DT> raw[V];
    if (row < rows)
#pragma unroll
        for (int j = 0; j < V; ++j) raw[j] = load_raw8<DT, WHOLE>(x, row, (j * NT + t) * 8, cols);
    stage_weight<NT, V>(w, w_dtype, cols, t, weight_s);
    int slot = 0;
    for (int64_t at_row = walk.warp_first; at_row < rows; at_row += step, row += step, slot ^= 1) {
        const bool live = NT >= 32 || row < rows;
        Raw8<DT> next[V];
        if (row + step < rows)
#pragma unroll
            for (int j = 0; j < V; ++j) next[j] = load_raw8<DT, WHOLE>(x, row + step, (j * NT + t) * 8, cols);
        f2 ss = pk2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float v[8];
            widen8<DT>(raw[j], v);
#pragma unroll
            for (int i = 0; i < 8; i += 2) ss = f2_fma(pk2(v[i], v[i + 1]), pk2(v[i], v[i + 1]), ss);
        }
        float s0, s1;
        upk2(ss, s0, s1);
        const float r = inv_sqrt(__fmaf_rn(row_sum<NT>(s0 + s1, part, slot), inv_cols, eps));
        if (t == 0 && live) rstd[row] = r;
        uint8_t* code_row = codes + row * per_row * 8;
        uint8_t* scale_row = scales + (row * per_row >> 2);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int u = j * NT + t;
            float v[8], o[8], wv[8];
            widen8<DT>(raw[j], v);
            const A8Block b = a8_block<DT>(raw[j]);
            const uint2 q = a8_encode8(v, b);
            weight8(weight_s, kChunks8, u, wv);
            vmuls8(o, v, r);
            vmul8(o, o, wv);
            const Raw8<DT> ry = narrow8<DT>(o);
            A8Block by = {0, 0.0f};
            uint2 qy = make_uint2(0, 0);
            if (ycodes) {               // the checkpoint of y is that of its rounded values
                widen8<DT>(ry, o);
                by = a8_block<DT>(ry);
                qy = a8_encode8(o, by);
            }
            store_raw8_warp<DT, WHOLE>(y, row, u * 8, cols, u < per_row && live, ry);
            if (u < per_row && live) {
                *reinterpret_cast<uint2*>(code_row + u * 8) = q;
                if ((t & 3) == 0) scale_row[u >> 2] = (uint8_t)b.byte;
                if (ycodes) {
                    *reinterpret_cast<uint2*>(ycodes + row * per_row * 8 + u * 8) = qy;
                    if ((t & 3) == 0) yscales[(row * per_row + u) >> 2] = (uint8_t)by.byte;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) raw[j] = next[j];
    }
}

// What a thread has of a row of the backward pass.
template <int DT, int V>
struct NormRow {
    Raw8<DT> dy[V];
    uint2 q[V];
    int b[V];
    float r;
};

template <int DT, int NT, int V, bool WHOLE>
__device__ __forceinline__ void load_norm_row(NormRow<DT, V>& n, const RowsIn& dy, int64_t row, int t, int cols,
                                              int per_row, const uint8_t* codes, const uint8_t* scales,
                                              const float* rstd) {
    const uint8_t* code_row = codes + row * per_row * 8;
    const uint8_t* scale_row = scales + (row * per_row >> 2);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int u = j * NT + t;
        n.dy[j] = load_raw8<DT, WHOLE>(dy, row, u * 8, cols);
        n.q[j] = make_uint2(0, 0);
        n.b[j] = 1;
        if (u < per_row) {
            n.q[j] = __ldcs(reinterpret_cast<const uint2*>(code_row + u * 8));
            n.b[j] = scale_row[u >> 2];
        }
    }
    n.r = rstd[row];
}

// dx = r (w dy) - v r^3 mean(v w dy); each block leaves its rows' sum of
// dy v r in partial[blockIdx.x][cols].  16384 x 4096 bf16 in 61 us, 5.5 TB/s: between HBM and the
// latency of a row's sum.
template <int DT, int NT, int V, bool WHOLE>
__global__ void __launch_bounds__(NT <= 32 ? 32 * kNormWarps : NT, norm_blocks<NT>(kNormBackward<DT, NT, V>))
rms_norm_backward_kernel(const RowsIn dy, int64_t rows, int cols, float inv_cols, int per_row,
                         const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                         const float* __restrict__ rstd, const void* __restrict__ w, int w_dtype,
                         const RowsOut dx, float* __restrict__ partial) {
    __shared__ float part[2][NT < 64 ? 1 : NT / 32];
    extern __shared__ float4 weight_s[];
    constexpr int kChunks8 = NT * V;
    const NormWalk<NT> walk;
    const int t = walk.t;
    const int64_t step = walk.step;
    int64_t row = walk.first;
    float acc[V][8];
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[j][i] = 0.0f;
    NormRow<DT, V> now = {};
    if (row < rows) load_norm_row<DT, NT, V, WHOLE>(now, dy, row, t, cols, per_row, codes, scales, rstd);
    stage_weight<NT, V>(w, w_dtype, cols, t, weight_s);
    int slot = 0;
    for (int64_t at_row = walk.warp_first; at_row < rows; at_row += step, row += step, slot ^= 1) {
        const bool live = NT >= 32 || row < rows;
        NormRow<DT, V> next;
        if (NT < 32) next = {};                 // a warp's last rows may not be there: zeros add nothing
        if (row + step < rows)
            load_norm_row<DT, NT, V, WHOLE>(next, dy, row + step, t, cols, per_row, codes, scales, rstd);
        const float r = now.r;
        f2 dot2 = pk2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float d[8], v[8], wv[8];
            widen8<DT>(now.dy[j], d);
            a8_decode8(now.q[j], a8_scale(now.b[j]), v);
            vmul8(d, d, v);             // behind the last column 0, or NaN in a block that has made the row's NaN anyway
            weight8(weight_s, kChunks8, j * NT + t, wv);
#pragma unroll
            for (int i = 0; i < 8; i += 2) dot2 = f2_fma(pk2(d[i], d[i + 1]), pk2(wv[i], wv[i + 1]), dot2);
            vfmas8(acc[j], r, d, acc[j]);
        }
        float d0, d1;
        upk2(dot2, d0, d1);
        // r by r: r^3 alone is beyond float32's normal numbers where r is beyond 2^-42 or 2^42
        const float k = r * (r * (r * (row_sum<NT>(d0 + d1, part, slot) * inv_cols)));
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int u = j * NT + t;
            float d[8], v[8], wv[8];
            widen8<DT>(now.dy[j], d);
            a8_decode8(now.q[j], a8_scale(now.b[j]), v);
            weight8(weight_s, kChunks8, u, wv);
            vmul8(d, d, wv);
            vmuls8(d, d, r);
            vfmas8(d, -k, v, d);
            store_raw8_warp<DT, WHOLE>(dx, row, u * 8, cols, u < per_row && live, narrow8<DT>(d));
        }
        now = next;
    }
    if constexpr (NT <= 32) {
        // the warp's rows and then the block's warps hold the same columns: added in their order
        __shared__ float sums[V * NT * 8];
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int o = 16; o >= NT; o >>= 1) acc[j][i] += __shfl_xor_sync(0xffffffffu, acc[j][i], o);
        for (int wi = 0; wi < (int)(blockDim.x >> 5); ++wi) {
            if ((int)(threadIdx.x >> 5) == wi && (threadIdx.x & 31) < NT)
#pragma unroll
                for (int j = 0; j < V; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float& s = sums[(j * NT + t) * 8 + i];
                        s = wi ? s + acc[j][i] : acc[j][i];
                    }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < cols; i += blockDim.x) partial[(int64_t)blockIdx.x * cols + i] = sums[i];
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

// Column sums of partial[parts][cols], in a fixed order: a block has eight columns (whole sectors), 32 threads
// share a column.  444 x 4096 in 7 us from HBM, 5 us behind the kernel above: latency.
constexpr int kSumCols = 8;

template <int DT>
__global__ void __launch_bounds__(32 * kSumCols)
column_sum_kernel(const float* __restrict__ partial, int parts, int cols, void* __restrict__ out) {
    __shared__ float s[kSumCols][33];
    const int c = threadIdx.x % kSumCols, r = threadIdx.x / kSumCols, col = blockIdx.x * kSumCols + c;
    float v = 0.0f;
    if (col < cols)
#pragma unroll 8
        for (int p = r; p < parts; p += 32) v += partial[(int64_t)p * cols + col];
    s[c][r] = v;
    __syncthreads();
    const int mine = blockIdx.x * kSumCols + (threadIdx.x >> 5);
    v = warp_sum(s[threadIdx.x >> 5][threadIdx.x & 31]);
    if ((threadIdx.x & 31) == 0 && mine < cols) Elem<DT>::store1(out, mine, v);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

static bool known_dtype(int dtype) { return dtype >= AW4_F32 && dtype <= AW4_F16; }
static int size_of(int dtype) { return dtype == AW4_F32 ? 4 : 2; }

static int32_t check_matrix(const char* what, int dtype, int64_t rows, int64_t cols) {
    if (!known_dtype(dtype)) return fail(AW4_ERR_INVALID, "%s: bad dtype %d", what, dtype);
    if (rows < 0 || cols < 0) return fail(AW4_ERR_INVALID, "%s: negative size", what);
    if (cols > (int64_t)1 << 30) return fail(AW4_ERR_UNSUPPORTED, "%s: rows of more than 2^30 values", what);
    if (rows && cols > ((int64_t)1 << 40) / rows)
        return fail(AW4_ERR_UNSUPPORTED, "%s: more than 2^40 values", what);
    return AW4_OK;
}

static int32_t launched(const char* what) {
    note_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? AW4_OK : fail(AW4_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

static uint32_t chunks_per_row(int64_t cols) { return (uint32_t)((cols + kA8Block - 1) / kA8Block * 4); }

static unsigned run_grid(int64_t units, int run) {
    const int64_t per_block = (int64_t)run * (kA8Threads / 32);
    return (unsigned)((units + per_block - 1) / per_block);
}

static RowsIn rows_in(const void* p, int64_t rows, int64_t cols, int64_t ld, int dtype) {
    const char* base = static_cast<const char*>(p);
    return {base, base + ((rows - 1) * ld + cols) * size_of(dtype), ld, rows_on(p, ld, dtype, 16)};
}
static RowsOut rows_out(void* p, int64_t ld, int dtype) { return {static_cast<char*>(p), ld, rows_on(p, ld, dtype, 16)}; }

// A row's threads and chunks of eight.  Rows of whole vectors have more widths to choose from, so that
// few threads are idle (5120 columns bf16, 2^26 values: 172 us with 512 threads a row, 125 with 320).
template <bool WHOLE, typename F>
static int32_t norm_shape(int64_t cols, F f) {
    using std::integral_constant;
    if (cols <= 64) return f(integral_constant<int, 8>(), integral_constant<int, 1>());
    if (cols <= 128) return f(integral_constant<int, 16>(), integral_constant<int, 1>());
    if (cols <= 256) return f(integral_constant<int, 32>(), integral_constant<int, 1>());
    if (cols <= 512) return f(integral_constant<int, 32>(), integral_constant<int, 2>());
    if (cols <= 1024) return f(integral_constant<int, 64>(), integral_constant<int, 2>());
    if constexpr (WHOLE)
        if (cols <= 1536) return f(integral_constant<int, 96>(), integral_constant<int, 2>());
    if (cols <= 2048) return f(integral_constant<int, 128>(), integral_constant<int, 2>());
    if constexpr (WHOLE)
        if (cols <= 2560) return f(integral_constant<int, 160>(), integral_constant<int, 2>());
    if (cols <= 4096) return f(integral_constant<int, 256>(), integral_constant<int, 2>());
    if constexpr (WHOLE) {
        if (cols <= 5120) return f(integral_constant<int, 320>(), integral_constant<int, 2>());
        if (cols <= 6144) return f(integral_constant<int, 384>(), integral_constant<int, 2>());
        if (cols <= 7168) return f(integral_constant<int, 448>(), integral_constant<int, 2>());
    }
    if (cols <= 8192) return f(integral_constant<int, 512>(), integral_constant<int, 2>());
    if constexpr (WHOLE)
        if (cols <= 12288) return f(integral_constant<int, 768>(), integral_constant<int, 2>());
    return f(integral_constant<int, 1024>(), integral_constant<int, 2>());
}

template <typename F>
static int32_t by_dtype(int dtype, F f) {
    if (dtype == AW4_F32) return f(std::integral_constant<int, AW4_F32>());
    if (dtype == AW4_BF16) return f(std::integral_constant<int, AW4_BF16>());
    return f(std::integral_constant<int, AW4_F16>());
}

// f(dtype, whether all of the call's rows are whole vectors)
template <typename F>
static int32_t by_form(int dtype, bool whole, F f) {
    return by_dtype(dtype, [&](auto dt) { return whole ? f(dt, std::true_type()) : f(dt, std::false_type()); });
}

constexpr int64_t kNormCols = 16384;

// Where rows belong to warps: the warps that have rows, and how many a block has of them, one for each SM's
// share of few.
template <int NT>
static int64_t norm_units(int64_t rows) {
    return NT < 32 ? (rows + 32 / NT - 1) / (32 / NT) : rows;
}
template <int NT>
static int norm_warps(int device, int64_t rows) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(kNormWarps, norm_units<NT>(rows) / sm_count(device)));
}

// Resident blocks, or as many as have a row: of the backward kernel also the rows of its partial sums.
template <int NT>
static int norm_grid(int device, int64_t rows, int threads) {
    const int held = NT <= 32 ? norm_warps<NT>(device, rows) : 1;
    const int resident = NT <= 32 ? threads / (32 * held) : norm_blocks<NT>(threads);
    return (int)std::min<int64_t>((norm_units<NT>(rows) + held - 1) / held, (int64_t)sm_count(device) * resident);
}
template <int NT>
static int norm_threads(int device, int64_t rows) {
    return NT <= 32 ? 32 * norm_warps<NT>(device, rows) : NT;
}

template <typename K>
static int32_t norm_smem(K kernel, int bytes) {
    if (bytes <= 32 * 1024) return AW4_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return e == cudaSuccess ? (int32_t)AW4_OK : fail(AW4_ERR_CUDA, "rms_norm: %s", cudaGetErrorString(e));
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
    const RowsIn in = rows_in(x, rows, cols, ld, dtype);
    return by_form(dtype, rows_whole(x, ld, cols, dtype), [&](auto dt, auto whole) {
        act8_quantize_kernel<dt.value, whole.value>
            <<<run_grid(rows * per_row, kRun), kA8Threads, 0, (cudaStream_t)stream>>>(in, rows, (int)cols, per_row,
                                                                                     codes, scales);
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
    const RowsOut to = rows_out(out, ld, dtype);
    return by_form(dtype, rows_whole(out, ld, cols, dtype), [&](auto dt, auto whole) {
        act8_dequantize_kernel<dt.value, whole.value>
            <<<run_grid(rows * per_row, kRun), kA8Threads, 0, (cudaStream_t)stream>>>(codes, scales, rows, (int)cols,
                                                                                     per_row, to);
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
    const RowsIn g = rows_in(gate, rows, cols, ld_gate, dtype), u = rows_in(up, rows, cols, ld_up, dtype);
    const RowsOut o = rows_out(h, cols, dtype);
    const unsigned grid = run_grid(rows * per_row, 32 * kGluForward);
    const bool all_whole = rows_whole(gate, ld_gate, cols, dtype) && rows_whole(up, ld_up, cols, dtype) &&
                           rows_whole(h, cols, cols, dtype);
    return by_form(dtype, all_whole, [&](auto dt, auto whole) {
        if (hcodes)
            swiglu_forward_kernel<dt.value, whole.value, true><<<grid, kA8Threads, 0, (cudaStream_t)stream>>>(
                g, u, rows, (int)cols, per_row, o, gcodes, gscales, ucodes, uscales, hcodes, hscales);
        else
            swiglu_forward_kernel<dt.value, whole.value, false><<<grid, kA8Threads, 0, (cudaStream_t)stream>>>(
                g, u, rows, (int)cols, per_row, o, gcodes, gscales, ucodes, uscales, nullptr, nullptr);
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
    const RowsIn in = rows_in(dh, rows, cols, ld_dh, dtype);
    const RowsOut dg = rows_out(dgate, ld_out, dtype), du = rows_out(dup, ld_out, dtype);
    const bool all_whole = rows_whole(dh, ld_dh, cols, dtype) && rows_whole(dgate, ld_out, cols, dtype) &&
                           rows_whole(dup, ld_out, cols, dtype);
    return by_form(dtype, all_whole, [&](auto dt, auto whole) {
        swiglu_backward_kernel<dt.value, whole.value>
            <<<run_grid(rows * per_row, 32 * kGluBackward), kA8Threads, 0, (cudaStream_t)stream>>>(
                in, rows, (int)cols, per_row, gcodes, gscales, ucodes, uscales, dg, du);
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
    const RowsIn in = rows_in(x, rows, cols, ld, dtype);
    const RowsOut out = rows_out(y, cols, dtype);
    const bool all_whole = rows_whole(x, ld, cols, dtype) && rows_whole(y, cols, cols, dtype);
    return by_form(dtype, all_whole, [&](auto dt, auto whole) {
        return norm_shape<whole.value>(cols, [&](auto nt, auto v) {
            auto kernel = rms_norm_forward_kernel<dt.value, nt.value, v.value, whole.value>;
            const int bytes = nt.value * v.value * 32;
            if (const int32_t rc = norm_smem(kernel, bytes)) return rc;
            kernel<<<norm_grid<nt.value>(device, rows, kNormForward), norm_threads<nt.value>(device, rows), bytes,
                     (cudaStream_t)stream>>>(in, rows, (int)cols, 1.0f / (float)cols, (int)per_row, weight,
                                             weight_dtype, eps, out, rstd, codes, scales, ycodes, yscales);
            return launched("rms_norm_forward");
        });
    });
}

extern "C" uint64_t aw4_rms_norm_backward_workspace(int64_t rows, int64_t cols, int32_t device) {
    if (rows <= 0 || cols <= 0 || cols > kNormCols) return 0;
    int grid = 0;
    auto most = [&](auto nt, auto) {
        grid = std::max(grid, norm_grid<nt.value>(device, rows, kNormBackwardMost));
        return (int32_t)AW4_OK;
    };
    norm_shape<true>(cols, most);
    norm_shape<false>(cols, most);
    return (uint64_t)grid * cols * sizeof(float);
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
    if (!workspace || workspace_bytes < (int64_t)aw4_rms_norm_backward_workspace(rows, cols, device))
        return fail(AW4_ERR_INVALID, "aw4_rms_norm_backward: workspace of %lld bytes is too small",
                    (long long)workspace_bytes);
    const uint32_t per_row = chunks_per_row(cols);
    int grid = 0;
    const RowsIn in = rows_in(dy, rows, cols, ld, dtype);
    const RowsOut out = rows_out(dx, cols, dtype);
    const bool all_whole = rows_whole(dy, ld, cols, dtype) && rows_whole(dx, cols, cols, dtype);
    const int32_t rc = by_form(dtype, all_whole, [&](auto dt, auto whole) {
        return norm_shape<whole.value>(cols, [&](auto nt, auto v) {
            auto kernel = rms_norm_backward_kernel<dt.value, nt.value, v.value, whole.value>;
            const int bytes = nt.value * v.value * 32;
            if (const int32_t rc = norm_smem(kernel, bytes)) return rc;
            grid = norm_grid<nt.value>(device, rows, kNormBackward<dt.value, nt.value, v.value>);
            kernel<<<grid, norm_threads<nt.value>(device, rows), bytes, s>>>(
                in, rows, (int)cols, 1.0f / (float)cols, (int)per_row, codes, scales, rstd, weight, weight_dtype,
                out, workspace);
            return launched("rms_norm_backward");
        });
    });
    if (rc) return rc;
    return by_dtype(weight_dtype, [&](auto wt) {
        column_sum_kernel<wt.value><<<(int)((cols + kSumCols - 1) / kSumCols), 32 * kSumCols, 0, s>>>(
            workspace, grid, (int)cols, dweight);
        return launched("column_sum");
    });
}
