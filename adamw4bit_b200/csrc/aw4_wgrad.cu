// aw4_wgrad.cu -- weight gradient of a projection whose input is an 8-bit checkpoint.
//
// dW_g[n][k] = sum over the rows t of group g of dy[t][n] v[t][k], v the
// checkpoint's values.  Group g holds rows [offsets[g], offsets[g + 1]); an
// empty group's gradient is zero.
//
// A pair of blocks holds a 512 x 256 tile of dW in tensor memory (two 256 x 256
// accumulators, 128 rows of each in a block: all 512 columns) and walks the rows 64
// at a time.  In each block:
//
//   warp 16      bulk tensor copies of its dy [64][256] and codes [64][128], four stages
//   warps 0-15   codes * 2^e -> 16-bit values in shared memory, four buffers, two groups
//                of warps taking turns.  A lane owns a block of 32 codes of one row
//   warp 17      (first block) tcgen05.mma for the pair, both operands with the row
//                index as the inner dimension
//   warps 18-19  (second block) tell the first that a group's values are there
//   warps 0-15   accumulators -> dW, or a float32 partial tile
//
// The values of the second block are written by its threads and read for a product that the first
// block issues: its arrivals release, and the wait for them acquires, over the pair.  A warp of its own for each group's
// arrivals keeps that release (most of a microsecond) out of the conversion: 8192 x 14336 x 4096 in 734 us, 751 with one such warp
// for both groups, 770 with an arrival of every converting warp.
//
// A pair, because shared memory bounds a single block: for 256 x 256 x 64 its tensor
// core reads 96 KB of operands, and copies and conversion move 96 KB more, 1536
// cycles at 128 bytes a cycle for 1024 cycles of products.  A pair's tensor cores share
// the values, so that a block moves 128 KB in the same 1024 cycles.
//
// q * 2^e is exact in bf16 and f16, so the products are those of dy and the
// checkpoint's own values, summed in float32.
//
// Rows behind a group's last are zeroed in both operands (a NaN of the next
// group must not meet a zero).
//
// Bound by the tensor cores at the power limit and by the way from values to product: 8192 x 14336 x 4096 bf16 in 730 us,
// 1317 TFLOP/s (cuBLAS on bf16 values 629 us; 839 and 708 us in a loop of seconds, where both clock down).  A step of 64 rows takes 0.83 us for 1024 cycles of products.
//
// Work split: whole tiles go round the pairs, n-tiles outermost so that
// pairs that run together share dy and codes in L2; the last wave and what
// does not fill one are cut by row steps, so that every pair gets the same
// number of steps whatever the groups' sizes.  A tile that is cut leaves float32
// partial tiles, added in the order of their rows by a second kernel: the same bits
// on every run.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/adamw4bit_b200.h"
#include "aw4_act8.cuh"
#include "aw4_host.h"
#include "aw4_tc.cuh"

namespace aw4 {

constexpr int kWgTileN = 512, kWgTileK = 256;   // a pair's tile
constexpr int kWgRows = 64;                     // rows of a step
constexpr int kWgStages = 4, kWgBuffers = 4;    // even: see the converting warps
constexpr int kWgConvert = 512;                 // threads that convert and write out, in two groups
constexpr int kWgThreads = kWgConvert + 128;
constexpr int kWgCopy = kWgConvert / 32, kWgProduct = kWgCopy + 1, kWgTell = kWgProduct + 1;   // warps
constexpr int kWgBox = kWgRows * 128;           // a copied box: 64 lines of 128 bytes
constexpr int kWgDyBytes = 4 * kWgBox;          // a block's 2 x 128 columns of dy
constexpr int kWgCodeBytes = kWgBox;            // its 128 codes of each row
constexpr int kWgValBytes = 2 * kWgBox;         // ... and their values
constexpr int kWgMaxPairs = 128;
constexpr int kWgMaxCut = 2 * kWgMaxPairs;      // cut tiles: less than two for each pair

struct WgSegment {
    int tile;         // over all groups
    int first, last;  // row steps [first, last) of the tile
    int slot;         // partial tile, or -1: the whole tile, written to dW
};

// What a partial slot holds, for the kernel that adds the parts.
struct WgSlot {
    int tile;   // -1: nothing
    int ends;   // 1: the tile's last part
};

struct WgParams {
    int64_t rows;
    int n, k;
    int n_tiles, k_tiles;
    int groups;
    uint32_t blocks;            // exponent blocks of a row
    const uint8_t* scales;
    const int32_t* offsets;
    void* out;
    bool accumulate, vec_out;
    float* partial;
    WgSlot* slots;              // null: no tile is cut
    int32_t* status;
    uint64_t wait_ns;           // limit of a wait
};

struct WgShared {
    alignas(8) uint64_t full[kWgStages], empty[kWgStages], ready[kWgBuffers], done[kWgBuffers], acc_full, acc_empty,
        out_done, drain;
    uint32_t tmem;
    int gave_up;
    int whole;                  // whole tiles of this pair
    int first_cut, cuts;        // its cut tiles, and where the first begins and the last ends
    int first_step, last_step;
    int64_t part[3][kWgThreads / 32];
};

constexpr int kWgSmem =
    1024 + kWgStages * (kWgDyBytes + kWgCodeBytes) + kWgBuffers * kWgValBytes + (int)sizeof(WgShared);
static_assert(kWgSmem <= 227 * 1024, "shared memory of a block");
static_assert(kWgConvert / 32 * 2048 <= kWgBuffers * kWgValBytes, "2 KB for each warp that writes out");
static_assert(kWgStages % 2 == 0 && kWgBuffers % 2 == 0, "a stage or buffer belongs to one group of warps");
static_assert(kWgMaxCut <= kWgThreads, "a thread for each cut tile");

__device__ __forceinline__ void wg_group(const WgParams& p, int g, int64_t& first, int64_t& last) {
    first = 0;
    last = p.rows;
    if (p.offsets) {
        first = max((int64_t)0, min(p.rows, (int64_t)p.offsets[g]));
        last = max(first, min(p.rows, (int64_t)p.offsets[g + 1]));
    }
}

// Row steps of a tile of group g; an empty group has one, of which no row counts.
__device__ __forceinline__ int wg_steps(const WgParams& p, int g) {
    int64_t first, last;
    wg_group(p, g, first, last);
    return max(1, (int)((last - first + kWgRows - 1) / kWgRows));
}

// Sum over the block, for every thread; `slot` names scratch of its own.
__device__ __forceinline__ int64_t wg_block_sum(int64_t v, int64_t* part) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < kWgThreads / 32; ++i) v += part[i];
    __syncthreads();
    return v;
}

// Cutting evens the pairs' steps and costs the parts' way through memory and the second kernel, about as much
// as this many steps: 4096 x 4096 x 4096, 128 tiles of 64 steps, takes 145 us cut over 74 pairs and 123 us as
// two whole tiles on each of 64; 8192 x 14336 x 4096, 448 tiles of 128 steps, 732 us cut and 769 us in seven
// rounds; 2048 x 768 x 768, 6 tiles of 32 steps, 35 us cut and 38 us whole.
constexpr int kWgCutSteps = 24;

// This pair's segments.  Tiles [cut, tiles) are laid end to end as row steps; a pair
// takes as many as it lacks to the average of all pairs.  A thread looks at one pair, then at one cut tile.  Where
// whole tiles alone leave no pair more than kWgCutSteps above the average, none is cut.
__device__ __noinline__ void wg_schedule(const WgParams& p, WgShared& s, int pair, int pairs, bool writes) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per_group = p.n_tiles * p.k_tiles;
    const int tiles = per_group * p.groups;
    if (tid == 0) {
        s.whole = (tiles - pair + pairs - 1) / pairs;  // none is cut
        s.cuts = 0;
    }
    if (!p.slots) {
        __syncthreads();
        return;
    }
    const int whole = max(0, tiles / pairs - 1);       // whole tiles of every pair
    const int cut = whole * pairs;
    int64_t load = 0;
    if (tid < pairs) {
        if (p.offsets) {
#pragma unroll 8
            for (int w = 0; w < whole; ++w) load += wg_steps(p, (w * pairs + tid) / per_group);
        } else {
            load = (int64_t)whole * wg_steps(p, 0);
        }
    }
    const int steps = cut + tid < tiles ? wg_steps(p, (cut + tid) / per_group) : 0;
    const int64_t rest = wg_block_sum(steps, s.part[0]);
    const int64_t target = (wg_block_sum(load, s.part[1]) + rest + pairs - 1) / pairs;
    if (writes && tid < 2) p.slots[2 * pair + tid] = {-1, 0};
    int64_t uncut = load;
    for (int t = cut + tid; tid < pairs && t < tiles; t += pairs) uncut += wg_steps(p, t / per_group);
    if (!wg_block_sum(tid < pairs && uncut - target > kWgCutSteps, s.part[0])) return;
    const int64_t lack = tid < pairs ? max((int64_t)0, target - load) : 0;
    const int64_t from = min(rest, wg_block_sum(tid < pair ? lack : 0, s.part[0]));
    const int64_t to = min(rest, from + wg_block_sum(tid == pair ? lack : 0, s.part[1]));
    // where this thread's tile begins
    int64_t at = steps;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += v;
    }
    if (lane == 31) s.part[2][warp] = at;
    __syncthreads();
    at -= steps;
    for (int i = 0; i < warp; ++i) at += s.part[2][i];
    const int64_t a = max(from, at), b = min(to, at + steps);
    if (a < b) {
        const int first = (int)(a - at), last = (int)(b - at);
        const int slot = first > 0 ? 2 * pair : last < steps ? 2 * pair + 1 : -1;
        atomicAdd(&s.cuts, 1);
        if (at <= from) {                              // the pair's first tile
            s.first_cut = cut + tid;
            s.first_step = first;
        }
        if (at + steps >= to) s.last_step = last;      // its last
        if (writes && slot >= 0) p.slots[slot] = {cut + tid, last == steps};
    }
    if (tid == 0) s.whole = whole;
    __syncthreads();
}

__device__ __forceinline__ WgSegment wg_segment(const WgParams& p, const WgShared& s, int i, int pair, int pairs) {
    const bool cut = i >= s.whole;
    const int c = i - s.whole;
    const int tile = cut ? s.first_cut + c : i * pairs + pair;
    const int steps = wg_steps(p, tile / (p.n_tiles * p.k_tiles));
    WgSegment g = {tile, 0, steps, -1};
    if (cut && c == 0) g.first = s.first_step;
    if (cut && c == s.cuts - 1) g.last = s.last_step;
    if (g.first > 0) g.slot = 2 * pair;
    else if (g.last < steps) g.slot = 2 * pair + 1;
    return g;
}

struct WgTile {
    int g, n0, k0;
    int64_t first, last;
    int half;         // columns of k that a block converts: the product has twice as many
};

__device__ __forceinline__ WgTile wg_tile(const WgParams& p, int tile) {
    WgTile t;
    const int per_group = p.n_tiles * p.k_tiles;
    t.g = tile / per_group;
    const int in = tile - t.g * per_group;
    t.n0 = in / p.k_tiles * kWgTileN;
    t.k0 = in % p.k_tiles * kWgTileK;
    wg_group(p, t.g, t.first, t.last);
    t.half = p.k - t.k0 > 128 ? 128 : 64;
    return t;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == AW4_BF16) {
        return pack_bf16x2(a, b);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// 2^e twice, in the operand's type; 0 for a row that does not count.
template <int DT>
__device__ __forceinline__ uint32_t wg_scale2(int byte, bool live) {
    uint32_t h;
    if constexpr (DT == AW4_BF16) {
        h = byte == kA8Nan ? 0x7fc0u : (uint32_t)byte << 7;
    } else {
        const int e = byte - 127;             // down to -24: below -14 a subnormal
        h = byte == kA8Nan ? 0x7e00u : e >= -14 ? (uint32_t)(e + 15) << 10 : 1u << (e + 24);
    }
    return live ? h * 0x10001u : 0u;
}

// q * 2^e of four codes, two and two; every step is exact.
//   bf16  the code's low seven bits behind 0x43 are 128 + (q mod 128), its sign bit alone 128 or
//         256: their difference is q
//   f16   q + 128 behind 0x64 is 1152 + q
template <int DT>
__device__ __forceinline__ uint2 wg_values4(uint32_t w, uint32_t s2) {
    uint2 r;
    if constexpr (DT == AW4_BF16) {
        const __nv_bfloat162 s = *reinterpret_cast<const __nv_bfloat162*>(&s2);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t t = __byte_perm(w, 0x43434343u, i ? 0x4342 : 0x4140);
            const uint32_t x = t & 0xff7fff7fu, y = t & 0xff80ff80u;
            const __nv_bfloat162 v = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x),
                                                     *reinterpret_cast<const __nv_bfloat162*>(&y)), s);
            (i ? r.y : r.x) = *reinterpret_cast<const uint32_t*>(&v);
        }
    } else {
        const __half2 s = *reinterpret_cast<const __half2*>(&s2);
        const __half2 off = __float2half2_rn(1152.0f);
        w ^= 0x80808080u;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t t = __byte_perm(w, 0x64646464u, i ? 0x4342 : 0x4140);
            const __half2 v = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&t), off), s);
            (i ? r.y : r.x) = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    return r;
}

// Block j of 32 codes of row r of the step, to 16-bit values.  A quarter of a
// warp has two rows and four blocks: the order of a block's halves, and the
// swizzle, put its eight accesses on different banks.
template <int DT>
__device__ __forceinline__ void wg_convert(const char* codes, char* operand, int r, int j, uint32_t s2) {
    char* line = operand + (j >> 1) * kWgBox + r * 128;
    const int swz = r & 7, to = (j & 1) * 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int h = i ^ (j >> 1);
        const uint4 w = *reinterpret_cast<const uint4*>(codes + r * 128 + (((2 * j + h) ^ swz) << 4));
        const uint2 a = wg_values4<DT>(w.x, s2), b = wg_values4<DT>(w.y, s2);
        const uint2 c = wg_values4<DT>(w.z, s2), d = wg_values4<DT>(w.w, s2);
        *reinterpret_cast<uint4*>(line + (((to + 2 * h) ^ swz) << 4)) = make_uint4(a.x, a.y, b.x, b.y);
        *reinterpret_cast<uint4*>(line + (((to + 2 * h + 1) ^ swz) << 4)) = make_uint4(c.x, c.y, d.x, d.y);
    }
}

// 32 lines of 64 bytes, a line a lane, turned in the warp's shared memory on
// their way out: 16 float32 sums of a row of dW (FROM32), or 32 values rounded already.  Line r is row
// first_row + r of dW, from column k on.  Where rows are on 16 bytes four lanes store a line in
// vectors; else, and where sums are added to what is there, a warp stores consecutive values.
template <int OT, bool FROM32>
__device__ __forceinline__ void wg_store_lines(const WgParams& p, char* stage, int64_t first_row, int rows, int k,
                                               const uint32_t v[16]) {
    const int lane = threadIdx.x & 31;
    constexpr bool kVectors = !FROM32 || OT == AW4_F32;
    constexpr int kLine = FROM32 ? 16 : 32, kValue = FROM32 ? 4 : 2;       // values of a line, bytes of one
    auto at = [&](int r, int byte) { return stage + r * 64 + (((byte >> 4) ^ ((r >> 1) & 3)) << 4) + (byte & 15); };
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c)
        *reinterpret_cast<uint4*>(at(lane, c * 16)) = make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
    __syncwarp();
    if (kVectors && p.vec_out && !p.accumulate && k + kLine <= p.k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + (lane >> 2);
            if (r < rows)
                __stcs(reinterpret_cast<uint4*>(static_cast<char*>(p.out) + ((first_row + r) * p.k + k) * kValue +
                                                (lane & 3) * 16),
                       *reinterpret_cast<const uint4*>(at(r, (lane & 3) * 16)));
        }
        return;
    }
    const int col = lane % kLine;
    if (k + col >= p.k) return;
    const int end = min(rows, 32);
#pragma unroll 4
    for (int r = lane / kLine; r < end; r += 32 / kLine) {
        const int64_t to = (first_row + r) * p.k + k + col;
        if constexpr (FROM32) {
            const float f = *reinterpret_cast<const float*>(at(r, col * 4));
            Elem<OT>::store1(p.out, to, p.accumulate ? Elem<OT>::load1(p.out, to) + f : f);
        } else {
            static_cast<uint16_t*>(p.out)[to] = *reinterpret_cast<const uint16_t*>(at(r, col * 2));
        }
    }
}

// A partial tile keeps four columns of all its rows together, so that a warp, a row a lane, writes and
// reads whole lines.  Four sums at row `row` and column `col` of the tile:
__device__ __forceinline__ float4* wg_partial(const WgParams& p, int slot, int row, int col) {
    return reinterpret_cast<float4*>(p.partial) + ((int64_t)slot * (kWgTileK / 4) + col / 4) * kWgTileN + row;
}

// Of a converting warp that has given up a wait before tile `from`: NaN in its place of that and of the tiles behind
// it, so that what is missing shows in the result, which a replayed graph or a program that does not look at the status
// may use.  Not through shared memory, where products in flight may read.
template <int OT>
__device__ __noinline__ void wg_no_numbers(const WgParams& p, const WgShared& s, int from, int pair, int pairs, int side) {
    const float nan = __uint_as_float(0x7fc00000u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row_in = ((warp >> 2) & 1) * 256 + side * 128 + (warp & 3) * 32 + lane;
    for (int i = from; i < s.whole + s.cuts; ++i) {
        const WgSegment seg = wg_segment(p, s, i, pair, pairs);
        const WgTile t = wg_tile(p, seg.tile);
        const int n = t.n0 + row_in, end = min((warp >> 3) * 128 + 128, p.k - t.k0);
        if (n >= p.n) continue;
        for (int col = (warp >> 3) * 128; col < end; ++col) {
            if (seg.slot < 0) Elem<OT>::store1(p.out, ((int64_t)t.g * p.n + n) * p.k + t.k0 + col, nan);
            else if (col % 4 == 0) *wg_partial(p, seg.slot, row_in, col) = make_float4(nan, nan, nan, nan);
        }
    }
}

template <int DT, int OT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWgThreads, 1)
weight_grad_kernel(const __grid_constant__ CUtensorMap dy_map, const __grid_constant__ CUtensorMap code_map,
                   const WgParams p) {
    extern __shared__ char raw_smem[];
    char* base = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
    char* dy_s = base;
    char* code_s = dy_s + kWgStages * kWgDyBytes;
    char* val_s = code_s + kWgStages * kWgCodeBytes;
    WgShared& s = *reinterpret_cast<WgShared*>(val_s + kWgBuffers * kWgValBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int side = block_in_pair();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kWgStages; ++i) {
            bar_init(smem_addr(&s.full[i]), 1);
            bar_init(smem_addr(&s.empty[i]), 1);
        }
        for (int i = 0; i < kWgBuffers; ++i) {
            bar_init(smem_addr(&s.ready[i]), kWgConvert / 64 + (side == 0));   // a group; the second block's word
            bar_init(smem_addr(&s.done[i]), 1);
        }
        bar_init(smem_addr(&s.acc_full), 1);
        bar_init(smem_addr(&s.acc_empty), 2 * kWgConvert / 32);
        bar_init(smem_addr(&s.out_done), kWgConvert / 32);
        bar_init(smem_addr(&s.drain), 1);
        s.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWgProduct) tmem_alloc(smem_addr(&s.tmem), 512);
    wg_schedule(p, s, pair, pairs, side == 0);
    tc_fence_before();
    pair_sync();
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    const int segments = s.whole + s.cuts;
    volatile int* gave_up = &s.gave_up;

    if (warp == kWgCopy) {
        if (lane == 0) {
            tma_prefetch_map(&dy_map);
            tma_prefetch_map(&code_map);
            uint32_t c = 0;
            bool ok = true;
            for (int i = 0; ok && i < segments; ++i) {
                const WgSegment seg = wg_segment(p, s, i, pair, pairs);
                const WgTile t = wg_tile(p, seg.tile);
                const int n1 = t.n0 + side * 128, k1 = t.k0 + side * t.half;
                // boxes that begin inside the matrices; what lies behind reads as zero or
                // is multiplied into sums that nobody stores
                bool in[4];
                uint32_t bytes = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    in[b] = n1 + (b >> 1) * 256 + (b & 1) * 64 < p.n;
                    bytes += in[b] ? kWgBox : 0;
                }
                const bool codes_in = k1 < (int)(p.blocks * kA8Block);
                bytes += codes_in ? kWgBox : 0;
                for (int step = seg.first; step < seg.last; ++step, ++c) {
                    const int st = c % kWgStages;
                    ok = bar_wait(smem_addr(&s.empty[st]), ((c / kWgStages) & 1) ^ 1, gave_up, p.wait_ns);
                    if (!ok) break;
                    const uint32_t bar = smem_addr(&s.full[st]);
                    const int row = (int)(t.first + (int64_t)step * kWgRows);
                    bar_expect(bar, bytes);
                    if (codes_in) tma_load_2d(smem_addr(code_s + st * kWgCodeBytes), &code_map, k1, row, bar);
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        if (in[b])
                            tma_load_2d(smem_addr(dy_s + st * kWgDyBytes + b * kWgBox), &dy_map,
                                        n1 + (b >> 1) * 256 + (b & 1) * 64, row, bar);
                }
            }
            if (!ok)   // copies in flight land before the block leaves
                for (uint32_t j = c < kWgStages ? 0 : c - kWgStages; j < c; ++j)
                    bar_drain(smem_addr(&s.full[j % kWgStages]), (j / kWgStages) & 1);
        }
        __syncwarp();
    } else if (warp == kWgProduct) {
        if (lane == 0 && side == 0) {
            uint32_t c = 0, buf = 0, turn = 0;
            bool ok = true;
            for (int i = 0; ok && i < segments; ++i) {
                const WgSegment seg = wg_segment(p, s, i, pair, pairs);
                const WgTile t = wg_tile(p, seg.tile);
                const uint32_t idesc = tc_idesc(DT == AW4_BF16, 2 * t.half);
                const bool two = t.n0 + 256 < p.n;
                ok = bar_wait<kWaitPairRelaxed>(smem_addr(&s.acc_empty), (i & 1) ^ 1, gave_up, p.wait_ns);
                for (int step = seg.first; ok && step < seg.last; ++step, ++c) {
                    const int st = c % kWgStages;
                    ok = bar_wait(smem_addr(&s.full[st]), (c / kWgStages) & 1, gave_up, p.wait_ns) &&
                         bar_wait<kWaitPair>(smem_addr(&s.ready[buf]), turn, gave_up, p.wait_ns);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t dy_a = smem_addr(dy_s + st * kWgDyBytes);
                    const uint32_t val_a = smem_addr(val_s + buf * kWgValBytes);
#pragma unroll
                    for (int j = 0; j < kWgRows / 16; ++j) {
                        const uint64_t vd = tc_desc(val_a + j * 2048, kWgBox);
                        const uint32_t add = step > seg.first || j > 0;
                        tc_mma_f16(tmem, tc_desc(dy_a + j * 2048, kWgBox), vd, idesc, add);
                        if (two) tc_mma_f16(tmem + 256, tc_desc(dy_a + 2 * kWgBox + j * 2048, kWgBox), vd, idesc, add);
                    }
                    tc_commit(smem_addr(&s.empty[st]));
                    tc_commit(smem_addr(&s.done[buf]));
                    if (++buf == kWgBuffers) {
                        buf = 0;
                        turn ^= 1;
                    }
                }
                if (ok) tc_commit(smem_addr(&s.acc_full));
            }
            if (!ok) {   // products in flight end before the tensor memory goes
                tc_commit(smem_addr(&s.drain));
                bar_drain(smem_addr(&s.drain), 0);
            }
        }
        __syncwarp();
    } else if (warp >= kWgTell) {
        if (lane == 0 && side == 1) {
            const uint32_t group = warp - kWgTell;
            uint32_t c = 0, buf = 0, turn = 0;
            bool ok = true;
            for (int i = 0; ok && i < segments; ++i) {
                const WgSegment seg = wg_segment(p, s, i, pair, pairs);
                for (int step = seg.first; step < seg.last; ++step, ++c) {
                    if ((c & 1) == group) {
                        ok = bar_wait(smem_addr(&s.ready[buf]), turn, gave_up, p.wait_ns);
                        if (!ok) break;
                        bar_arrive_pair_release(in_first_block(smem_addr(&s.ready[buf])));
                    }
                    if (++buf == kWgBuffers) {
                        buf = 0;
                        turn ^= 1;
                    }
                }
            }
        }
        __syncwarp();
    } else {
        // Converts the steps of its parity.  Stages and buffers are even in number, so each is of one
        // group, which sees every turn of its barriers: parity alone tells one turn from the next.
        const int group = warp >> 3;
        const int r = (warp & 7) * 8 + (lane >> 2), j = lane & 3;
        uint32_t c = 0, buf = 0, turn = 0;
        bool ok = true;
        int i = 0;
        for (; i < segments; ++i) {
            const WgSegment seg = wg_segment(p, s, i, pair, pairs);
            const WgTile t = wg_tile(p, seg.tile);
            const uint32_t block = (t.k0 + side * t.half) / kA8Block + j;
            const bool cols = j * kA8Block < t.half && block < p.blocks;
            // the exponent of this group's next step is on its way while one is converted
            const int skip = (c & 1) ^ group;
            int64_t row = t.first + (int64_t)(seg.first + skip) * kWgRows + r;
            const int64_t end = min(t.last, t.first + (int64_t)seg.last * kWgRows);
            const uint8_t* scale = p.scales + row * p.blocks + block;
            int byte = cols && row < end ? *scale : 1;
            // the values' buffers also turn the last tile's sums on their way out
            if (i > 0) ok = __all_sync(0xffffffffu, bar_wait(smem_addr(&s.out_done), (i - 1) & 1, gave_up, p.wait_ns));
            if (!ok) break;
            for (int step = seg.first; step < seg.last; ++step, ++c) {
                if ((c & 1) == group) {
                    const int st = c % kWgStages;
                    const bool live = row < t.last;
                    row += 2 * kWgRows;
                    scale += 2 * kWgRows * p.blocks;
                    const int next = cols && row < end ? *scale : 1;
                    ok = bar_wait(smem_addr(&s.full[st]), (c / kWgStages) & 1, gave_up, p.wait_ns) &&
                         bar_wait(smem_addr(&s.done[buf]), turn ^ 1, gave_up, p.wait_ns);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    if (cols)
                        wg_convert<DT>(code_s + st * kWgCodeBytes, val_s + buf * kWgValBytes, r, j,
                                       wg_scale2<DT>(byte, live));
                    if (!live) {   // the row belongs to the next group
                        char* line = dy_s + st * kWgDyBytes + j * kWgBox + r * 128;
#pragma unroll
                        for (int h = 0; h < 8; ++h)
                            *reinterpret_cast<uint4*>(line + h * 16) = make_uint4(0, 0, 0, 0);
                    }
                    byte = next;
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) bar_arrive(smem_addr(&s.ready[buf]));
                }
                if (++buf == kWgBuffers) {
                    buf = 0;
                    turn ^= 1;
                }
            }
            if (!ok) break;
            ok = __all_sync(0xffffffffu, bar_wait(smem_addr(&s.acc_full), i & 1, gave_up, p.wait_ns));
            if (!ok) break;
            tc_fence_after();
            // four warps for the 128 rows that this block has of each accumulator; the groups
            // take half the columns each
            const int acc = (warp >> 2) & 1;
            const int row_in = acc * 256 + side * 128 + (warp & 3) * 32 + lane;
            const int n = t.n0 + row_in;
            const uint32_t from = tmem + ((uint32_t)(warp & 3) << 21) + acc * 256;
            const int k_end = min(group * 128 + 128, p.k - t.k0);
            const int64_t first_row = (int64_t)t.g * p.n + n - lane;
            // no product reads the values any more, and none are written before out_done
            char* stage = val_s + warp * 2048;
            if (n - lane < p.n)
                for (int col = group * 128; col < k_end; col += 32) {
                    uint32_t v[32];
                    tmem_load32(from + col, v);
                    tmem_load_wait();
                    if (seg.slot >= 0) {
                        float4* o = wg_partial(p, seg.slot, row_in, col);
#pragma unroll
                        for (int q = 0; q < 8; ++q)
                            if (n < p.n)
                                o[q * kWgTileN] = make_float4(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1]),
                                                              __uint_as_float(v[4 * q + 2]),
                                                              __uint_as_float(v[4 * q + 3]));
                    } else if (OT == AW4_F32 || p.accumulate) {
                        wg_store_lines<OT, true>(p, stage, first_row, p.n - n + lane, t.k0 + col, v);
                        wg_store_lines<OT, true>(p, stage, first_row, p.n - n + lane, t.k0 + col + 16, v + 16);
                    } else {
                        uint32_t h[16];
#pragma unroll
                        for (int q = 0; q < 16; ++q)
                            h[q] = pack2<OT>(__uint_as_float(v[2 * q]), __uint_as_float(v[2 * q + 1]));
                        wg_store_lines<OT, false>(p, stage, first_row, p.n - n + lane, t.k0 + col, h);
                    }
                }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                bar_arrive(smem_addr(&s.out_done));
                bar_arrive_pair_relaxed(in_first_block(smem_addr(&s.acc_empty)));
            }
        }
        if (!ok) wg_no_numbers<OT>(p, s, i, pair, pairs, side);
    }
    // neither block leaves while the other's products or arrivals may reach it
    tc_fence_before();
    __syncwarp();
    pair_sync();
    tc_fence_after();
    if (warp == kWgProduct) tmem_free(tmem, 512);
    if (threadIdx.x == 0 && s.gave_up && p.status) *reinterpret_cast<volatile int32_t*>(p.status) = 1;
}

// Adds the parts of each cut tile, in the order of their rows.  Block (b, i): the tile whose first part
// pair b left, rows [32 i, 32 i + 32).
// 74 cut tiles of 512 x 256, two parts each, in 18 us from HBM.
constexpr int kWgSlice = 32;

template <int OT>
__global__ void __launch_bounds__(256)
weight_grad_join_kernel(const WgParams p, int pairs) {
    const WgSlot head = p.slots[2 * blockIdx.x + 1];
    if (head.tile < 0) return;
    const WgTile t = wg_tile(p, head.tile);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row0 = blockIdx.y * kWgSlice;
    if (t.n0 + row0 >= p.n) return;
    __shared__ float tile[kWgSlice][kWgTileK + 4];
    const bool row_in = t.n0 + row0 + lane < p.n;
    float4 acc[8] = {};
    for (int b = blockIdx.x; b < pairs; ++b) {
        const WgSlot slot = b == (int)blockIdx.x ? head : p.slots[2 * b];
        if (slot.tile != head.tile) continue;
        const int at = b == (int)blockIdx.x ? 2 * b + 1 : 2 * b;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int col = (q * 8 + warp) * 4;
            if (row_in && t.k0 + col < p.k) {
                const float4 f = __ldcg(wg_partial(p, at, row0 + lane, col));
                acc[q].x += f.x;
                acc[q].y += f.y;
                acc[q].z += f.z;
                acc[q].w += f.w;
            }
        }
        if (slot.ends) break;
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) *reinterpret_cast<float4*>(&tile[lane][(q * 8 + warp) * 4]) = acc[q];
    __syncthreads();
    const RowsOut out = {static_cast<char*>(p.out), p.k, p.vec_out};
    const RowsIn old = {out.base, out.base + (int64_t)p.groups * p.n * p.k * Elem<OT>::kBytes, p.k, p.vec_out};
    for (int r = warp; r < kWgSlice && t.n0 + row0 + r < p.n; r += 8) {
        const int64_t row = (int64_t)t.g * p.n + t.n0 + row0 + r;
        const int at = t.k0 + lane * 8;
        if (at >= p.k) continue;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = tile[r][lane * 8 + i];
        if (p.accumulate) {
            float o[8];
            widen8<OT>(load_raw8<OT, false>(old, row, at, p.k), o);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] += o[i];
        }
        store_raw8<OT, false>(out, row, at, p.k, narrow8<OT>(f));
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

static std::atomic<uint64_t> g_wait_ns{kWaitNs};

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// A matrix of rows lines, copied in boxes of 128 bytes x 64 rows with the 128-byte swizzle.
static bool encode_rows(CUtensorMap* map, CUtensorMapDataType type, int size, const void* base, int64_t cols,
                        int64_t rows, int64_t row_bytes) {
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)kWgRows};
    const cuuint32_t step[2] = {1, 1};
    return encode_tiled()(map, type, 2, const_cast<void*>(base), dims, strides, box, step,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int64_t wg_tiles(int64_t n, int64_t k) {
    return (n + kWgTileN - 1) / kWgTileN * ((k + kWgTileK - 1) / kWgTileK);
}

// How a call is split: pairs of blocks, at most one on each two SMs, and whether tiles may be cut.  One group's
// tiles have all as many steps, and the rule of kWgCutSteps is applied here; groups' steps are known on the
// device only.  Where tiles may be cut, a pair has at least kWgMinSteps steps on average.
constexpr int64_t kWgMinSteps = 4;

struct WgPlan {
    int pairs;
    bool cuts;
};

static WgPlan wg_plan(int device, int64_t rows, int64_t n, int64_t k, int64_t groups) {
    const int64_t most = std::min<int64_t>(std::max(1, sm_count(device) / 2), kWgMaxPairs);
    const int64_t tiles = wg_tiles(n, k) * groups;
    const int64_t steps = (rows + kWgRows - 1) / kWgRows;
    if (groups == 1) {
        const int64_t rounds = (tiles + most - 1) / most;
        if (rounds * steps - tiles * steps / most <= kWgCutSteps)
            return {(int)((tiles + rounds - 1) / rounds), false};
    }
    const int64_t all = std::max(groups, steps) * wg_tiles(n, k);
    return {(int)std::max<int64_t>(1, std::min(most, std::max(tiles, all / kWgMinSteps))), true};
}

static uint64_t wg_workspace(const WgPlan& plan) {
    if (!plan.cuts) return 0;
    return (uint64_t)plan.pairs * 2 * (sizeof(WgSlot) + (uint64_t)kWgTileN * kWgTileK * sizeof(float));
}

}  // namespace aw4

using namespace aw4;

extern "C" int32_t aw4_set_wait_limit(uint64_t ns) {
    g_wait_ns.store(std::min(ns, kWaitNs), std::memory_order_relaxed);
    return AW4_OK;
}

extern "C" uint64_t aw4_weight_grad_workspace(int64_t rows, int64_t n, int64_t k, int64_t groups, int32_t device) {
    if (rows <= 0 || n <= 0 || k <= 0 || groups < 1) return 0;
    return wg_workspace(wg_plan(device, rows, n, k, groups));
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
    if (rows > 0x7fffff00 || n > 1 << 20 || k > 1 << 20 || groups > 65535 ||
        wg_tiles(n, k) * groups > 0x7fffff00)
        return fail(AW4_ERR_UNSUPPORTED, "aw4_weight_grad: size above the kernel's");
    if (n == 0 || k == 0) return AW4_OK;
    if (!out || (uintptr_t)out % (out_dtype == AW4_F32 ? 4 : 2))
        return fail(AW4_ERR_INVALID, "aw4_weight_grad: null or misaligned output");
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(AW4_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    cudaStream_t s = (cudaStream_t)stream;
    const int64_t size = out_dtype == AW4_F32 ? 4 : 2;
    if (rows == 0) {
        const cudaError_t e = accumulate ? cudaSuccess : cudaMemsetAsync(out, 0, groups * n * k * size, s);
        return e == cudaSuccess ? AW4_OK : fail(AW4_ERR_CUDA, "weight_grad: %s", cudaGetErrorString(e));
    }
    if (!dy || !codes || !scales || (uintptr_t)codes % 16 || (uintptr_t)dy % 16 || ld < n || ld * 2 % 16)
        return fail(AW4_ERR_INVALID, "aw4_weight_grad: null buffer, or rows not on 16 bytes");
    const WgPlan plan = wg_plan(device, rows, n, k, groups);
    const int pairs = plan.pairs;
    if (plan.cuts &&
        (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < (int64_t)wg_workspace(plan)))
        return fail(AW4_ERR_INVALID, "aw4_weight_grad: workspace of %lld bytes is too small or misaligned",
                    (long long)workspace_bytes);
    if (!encode_tiled()) return fail(AW4_ERR_CUDA, "aw4_weight_grad: the driver has no cuTensorMapEncodeTiled");
    WgParams p;
    p.rows = rows;
    p.n = (int)n;
    p.k = (int)k;
    p.n_tiles = (int)((n + kWgTileN - 1) / kWgTileN);
    p.k_tiles = (int)((k + kWgTileK - 1) / kWgTileK);
    p.groups = (int)groups;
    p.blocks = (uint32_t)((k + kA8Block - 1) / kA8Block);
    p.scales = scales;
    p.offsets = offsets;
    p.out = out;
    p.accumulate = accumulate != 0;
    p.vec_out = (uintptr_t)out % 16 == 0 && k * size % 16 == 0;
    p.partial = static_cast<float*>(workspace);
    p.slots = plan.cuts ? reinterpret_cast<WgSlot*>(p.partial + (int64_t)pairs * 2 * kWgTileN * kWgTileK) : nullptr;
    p.status = status;
    p.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
    CUtensorMap dy_map, code_map;
    if (!encode_rows(&dy_map, dtype == AW4_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                     dy, n, rows, ld * 2) ||
        !encode_rows(&code_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, (int64_t)p.blocks * kA8Block, rows,
                     (int64_t)p.blocks * kA8Block))
        return fail(AW4_ERR_CUDA, "aw4_weight_grad: tensor map refused");
    auto go = [&](auto dt, auto ot) -> int32_t {
        auto kernel = weight_grad_kernel<dt.value, ot.value>;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kWgSmem);
        if (e != cudaSuccess) return fail(AW4_ERR_CUDA, "weight_grad: %s", cudaGetErrorString(e));
        kernel<<<2 * pairs, kWgThreads, kWgSmem, s>>>(dy_map, code_map, p);
        note_launch();
        e = cudaGetLastError();
        if (e != cudaSuccess) return fail(AW4_ERR_CUDA, "weight_grad launch: %s", cudaGetErrorString(e));
        if (!plan.cuts) return AW4_OK;
        weight_grad_join_kernel<ot.value><<<dim3(pairs, kWgTileN / kWgSlice), 256, 0, s>>>(p, pairs);
        note_launch();
        e = cudaGetLastError();
        return e == cudaSuccess ? AW4_OK : fail(AW4_ERR_CUDA, "weight_grad_join launch: %s", cudaGetErrorString(e));
    };
    using std::integral_constant;
    if (dtype == AW4_BF16)
        return out_dtype == AW4_F32 ? go(integral_constant<int, AW4_BF16>(), integral_constant<int, AW4_F32>())
                                    : go(integral_constant<int, AW4_BF16>(), integral_constant<int, AW4_BF16>());
    return out_dtype == AW4_F32 ? go(integral_constant<int, AW4_F16>(), integral_constant<int, AW4_F32>())
                                : go(integral_constant<int, AW4_F16>(), integral_constant<int, AW4_F16>());
}
