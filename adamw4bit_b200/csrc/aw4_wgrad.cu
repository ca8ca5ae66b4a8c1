// aw4_wgrad.cu -- weight gradient of a projection whose input is an 8-bit checkpoint.
//
// dW_g[n][k] = sum over the rows t of group g of dy[t][n] v[t][k], v the
// checkpoint's values.  Group g holds rows [offsets[g], offsets[g + 1]); an
// empty group's gradient is zero.
//
// A block holds a 256 x 256 tile of dW in tensor memory (two 128 x 256
// accumulators, all 512 columns) and walks the rows 64 at a time:
//
//   warp 8      bulk tensor copies of dy [64][256] and of the codes [64][256] bytes, three stages
//   warps 0-7   codes * 2^e -> 16-bit values in shared memory, two buffers.  A lane owns
//               64 values of one row, a 128-byte line of the operand: reads and
//               writes of a warp then cover all banks under the 128-byte swizzle
//   warp 9      tcgen05.mma, both operands with the row index as the inner dimension
//   warps 0-7   accumulators -> dW, or a float32 partial tile
//
// q * 2^e is exact in bf16 and f16, so the products are those of dy and the
// checkpoint's own values, summed in float32.
//
// Rows behind a group's last are zeroed in both operands (a NaN of the next
// group must not meet a zero).
//
// Work split: whole tiles go round the blocks, n-tiles outermost so that
// blocks that run together share dy and codes in L2; the last wave and what
// does not fill one are cut by row steps, so that every block gets the same
// number of steps whatever the groups' sizes.  A tile that is cut leaves float32
// partial tiles, added in the order of their rows by a second kernel: the same bits
// on every run.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/adamw4bit_b200.h"
#include "aw4_act8.cuh"
#include "aw4_host.h"
#include "aw4_tc.cuh"

namespace aw4 {

constexpr int kWgTile = 256;                 // n and k of a tile
constexpr int kWgRows = 64;                  // rows of a step
constexpr int kWgStages = 3;
constexpr int kWgConvert = 256;              // threads that convert and write out
constexpr int kWgThreads = kWgConvert + 64;
constexpr int kWgDyBytes = kWgRows * kWgTile * 2;
constexpr int kWgCodeBytes = kWgRows * kWgTile;
constexpr int kWgBox = kWgRows * 128;        // a copied box: 64 lines of 128 bytes
constexpr int kWgMaxBlocks = 256;            // the schedule's scan gives a thread to each block
constexpr int kWgSegments = 2 * kWgMaxBlocks + 2;

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
    WgSlot* slots;
    int32_t* status;
};

struct WgShared {
    alignas(8) uint64_t full[kWgStages], empty[kWgStages], ready[2], done[2], acc_full, acc_empty, drain;
    uint32_t tmem;
    int gave_up;
    int segments;
    int whole;                  // whole tiles of this block
    int64_t scan[kWgMaxBlocks];
    WgSegment list[kWgSegments];
};

constexpr int kWgSmem = 1024 + kWgStages * (kWgDyBytes + kWgCodeBytes) + 2 * kWgDyBytes + (int)sizeof(WgShared);

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

// This block's segments of the cut tiles.  Tiles [cut, tiles) are laid end to end as
// row steps; block b takes as many as it lacks to the average of all blocks.
__device__ void wg_schedule(const WgParams& p, WgShared& s) {
    const int tid = threadIdx.x;
    const int per_group = p.n_tiles * p.k_tiles;
    const int tiles = per_group * p.groups;
    const int blocks = gridDim.x;
    const int whole = max(0, tiles / blocks - 1);      // whole tiles of every block
    const int cut = whole * blocks;
    int64_t mine = 0;
    if (tid < blocks) {
        if (p.offsets)
            for (int w = 0; w < whole; ++w) mine += wg_steps(p, (w * blocks + tid) / per_group);
        else
            mine = (int64_t)whole * wg_steps(p, 0);
    }
    if (tid < kWgMaxBlocks) s.scan[tid] = mine;
    __syncthreads();
    if (tid == 0) {
        int64_t load = 0, rest = 0;
        for (int b = 0; b < blocks; ++b) load += s.scan[b];
        for (int t = cut; t < tiles;) {
            const int g = t / per_group, end = min(tiles, (g + 1) * per_group);
            rest += (int64_t)(end - t) * wg_steps(p, g);
            t = end;
        }
        const int64_t target = (load + rest + blocks - 1) / blocks;
        int64_t from = 0;
        for (int b = 0; b < (int)blockIdx.x; ++b) from += max((int64_t)0, target - s.scan[b]);
        int64_t to = from + max((int64_t)0, target - s.scan[blockIdx.x]);
        from = min(from, rest);
        to = min(to, rest);
        int count = 0;
        WgSlot first_slot = {-1, 0}, last_slot = {-1, 0};
        int64_t at = 0;
        for (int t = cut; from < to && t < tiles && at < to;) {
            const int g = t / per_group, end = min(tiles, (g + 1) * per_group);
            const int steps = wg_steps(p, g);
            const int64_t group_end = at + (int64_t)(end - t) * steps;
            if (group_end > from) {
                if (from > at) {
                    const int skip = (int)((from - at) / steps);
                    t += skip;
                    at += (int64_t)skip * steps;
                }
                for (; t < end && at < to && count < kWgSegments; ++t, at += steps) {
                    const int a = (int)max((int64_t)0, from - at), b = (int)min((int64_t)steps, to - at);
                    int slot = -1;
                    if (a > 0) {
                        slot = 2 * blockIdx.x;
                        first_slot = {t, b == steps};
                    } else if (b < steps) {
                        slot = 2 * blockIdx.x + 1;
                        last_slot = {t, 0};
                    }
                    s.list[count++] = {t, a, b, slot};
                }
            }
            at = group_end;
            t = end;
        }
        s.segments = count;
        s.whole = whole;
        p.slots[2 * blockIdx.x] = first_slot;
        p.slots[2 * blockIdx.x + 1] = last_slot;
    }
    __syncthreads();
}

__device__ __forceinline__ WgSegment wg_segment(const WgParams& p, const WgShared& s, int i) {
    if (i >= s.whole) return s.list[i - s.whole];
    const int tile = i * gridDim.x + blockIdx.x;
    return {tile, 0, wg_steps(p, tile / (p.n_tiles * p.k_tiles)), -1};
}

struct WgTile {
    int g, n0, k0;
    int64_t first, last;
    int dy_boxes, code_boxes;   // boxes of 64 columns of dy, of 128 of the codes
};

__device__ __forceinline__ WgTile wg_tile(const WgParams& p, int tile) {
    WgTile t;
    const int per_group = p.n_tiles * p.k_tiles;
    t.g = tile / per_group;
    const int in = tile - t.g * per_group;
    t.n0 = in / p.k_tiles * kWgTile;
    t.k0 = in % p.k_tiles * kWgTile;
    wg_group(p, t.g, t.first, t.last);
    t.dy_boxes = min(4, (p.n - t.n0 + 63) / 64);
    t.code_boxes = min(2, (p.k - t.k0 + 127) / 128);
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

// 64 codes of row r, columns [64 c, 64 c + 64) of the step, to 16-bit values.
template <int DT>
__device__ __forceinline__ void wg_convert(const char* codes, char* operand, int r, int c, int b0, int b1,
                                           bool live) {
    char* line = operand + c * kWgBox + r * 128;
    const int swz = r & 7;
    if (!live) {
#pragma unroll
        for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(line + j * 16) = make_uint4(0, 0, 0, 0);
        return;
    }
    const char* src = codes + (c >> 1) * kWgBox + r * 128;
    const float s[2] = {a8_scale(b0), a8_scale(b1)};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint4 w = *reinterpret_cast<const uint4*>(src + ((((c & 1) * 4 + j) ^ swz) << 4));
        const uint32_t q[4] = {w.x, w.y, w.z, w.w};
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v[4];
            a8_decode4(q[i], s[j >> 1], v);
            o[2 * i] = pack2<DT>(v[0], v[1]);
            o[2 * i + 1] = pack2<DT>(v[2], v[3]);
        }
        *reinterpret_cast<uint4*>(line + (((2 * j) ^ swz) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(line + (((2 * j + 1) ^ swz) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
    }
}

// 32 sums of one row of dW.
template <int OT>
__device__ __forceinline__ void wg_store(const WgParams& p, int64_t row_off, int k, const uint32_t v[32]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int at = k + c * 8;
        if (at >= p.k) return;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(v[c * 8 + i]);
        if (p.accumulate) {
            float o[8];
            widen8<OT>(load_raw8<OT>(p.out, row_off, at, p.k, p.vec_out), o);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] += o[i];
        }
        store_raw8<OT>(p.out, row_off, at, p.k, p.vec_out, narrow8<OT>(f));
    }
}

template <int DT, int OT>
__global__ void __launch_bounds__(kWgThreads, 1)
weight_grad_kernel(const __grid_constant__ CUtensorMap dy_map, const __grid_constant__ CUtensorMap code_map,
                   const WgParams p) {
    extern __shared__ char raw_smem[];
    char* base = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
    char* dy_s = base;
    char* code_s = dy_s + kWgStages * kWgDyBytes;
    char* val_s = code_s + kWgStages * kWgCodeBytes;
    WgShared& s = *reinterpret_cast<WgShared*>(val_s + 2 * kWgDyBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kWgStages; ++i) {
            bar_init(smem_addr(&s.full[i]), 1);
            bar_init(smem_addr(&s.empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(smem_addr(&s.ready[i]), kWgConvert / 32);
            bar_init(smem_addr(&s.done[i]), 1);
        }
        bar_init(smem_addr(&s.acc_full), 1);
        bar_init(smem_addr(&s.acc_empty), kWgConvert / 32);
        bar_init(smem_addr(&s.drain), 1);
        s.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) tmem_alloc(smem_addr(&s.tmem), 512);
    wg_schedule(p, s);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    const int segments = s.whole + s.segments;
    volatile int* gave_up = &s.gave_up;

    if (warp == 8) {
        if (lane == 0) {
            tma_prefetch_map(&dy_map);
            tma_prefetch_map(&code_map);
            uint32_t c = 0;
            bool ok = true;
            for (int i = 0; ok && i < segments; ++i) {
                const WgSegment seg = wg_segment(p, s, i);
                const WgTile t = wg_tile(p, seg.tile);
                const uint32_t bytes = (t.dy_boxes + t.code_boxes) * kWgBox;
                for (int step = seg.first; step < seg.last; ++step, ++c) {
                    const int st = c % kWgStages;
                    ok = bar_wait(smem_addr(&s.empty[st]), ((c / kWgStages) & 1) ^ 1, gave_up);
                    if (!ok) break;
                    const uint32_t bar = smem_addr(&s.full[st]);
                    const int row = (int)(t.first + (int64_t)step * kWgRows);
                    bar_expect(bar, bytes);
                    for (int b = 0; b < t.dy_boxes; ++b)
                        tma_load_2d(smem_addr(dy_s + st * kWgDyBytes + b * kWgBox), &dy_map, t.n0 + b * 64, row, bar);
                    for (int b = 0; b < t.code_boxes; ++b)
                        tma_load_2d(smem_addr(code_s + st * kWgCodeBytes + b * kWgBox), &code_map, t.k0 + b * 128,
                                    row, bar);
                }
            }
            if (!ok)   // copies in flight land before the block leaves
                for (uint32_t j = c < kWgStages ? 0 : c - kWgStages; j < c; ++j)
                    bar_drain(smem_addr(&s.full[j % kWgStages]), (j / kWgStages) & 1);
        }
        __syncwarp();
    } else if (warp == 9) {
        if (lane == 0) {
            uint32_t c = 0;
            bool ok = true;
            for (int i = 0; ok && i < segments; ++i) {
                const WgSegment seg = wg_segment(p, s, i);
                const WgTile t = wg_tile(p, seg.tile);
                const uint32_t idesc = tc_idesc(DT == AW4_BF16, min(kWgTile, (p.k - t.k0 + 15) / 16 * 16));
                const bool two = t.dy_boxes > 2;
                ok = bar_wait(smem_addr(&s.acc_empty), (i & 1) ^ 1, gave_up);
                for (int step = seg.first; ok && step < seg.last; ++step, ++c) {
                    const int st = c % kWgStages, b = c & 1;
                    ok = bar_wait(smem_addr(&s.ready[b]), (c >> 1) & 1, gave_up) &&
                         bar_wait(smem_addr(&s.full[st]), (c / kWgStages) & 1, gave_up);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t dy_a = smem_addr(dy_s + st * kWgDyBytes);
                    const uint32_t val_a = smem_addr(val_s + b * kWgDyBytes);
#pragma unroll
                    for (int j = 0; j < kWgRows / 16; ++j) {
                        const uint64_t vd = tc_desc(val_a + j * 2048, kWgBox);
                        const uint32_t add = step > seg.first || j > 0;
                        tc_mma_f16(tmem, tc_desc(dy_a + j * 2048, kWgBox), vd, idesc, add);
                        if (two) tc_mma_f16(tmem + 256, tc_desc(dy_a + 2 * kWgBox + j * 2048, kWgBox), vd, idesc, add);
                    }
                    tc_commit(smem_addr(&s.empty[st]));
                    tc_commit(smem_addr(&s.done[b]));
                }
                if (ok) tc_commit(smem_addr(&s.acc_full));
            }
            if (!ok) {   // products in flight end before the tensor memory goes
                tc_commit(smem_addr(&s.drain));
                bar_drain(smem_addr(&s.drain), 0);
            }
        }
        __syncwarp();
    } else {
        const int r = threadIdx.x & 63, chunk = threadIdx.x >> 6;
        uint32_t c = 0;
        bool ok = true;
        for (int i = 0; ok && i < segments; ++i) {
            const WgSegment seg = wg_segment(p, s, i);
            const WgTile t = wg_tile(p, seg.tile);
            const uint32_t block = t.k0 / kA8Block + chunk * 2;
            const bool cols = chunk < t.code_boxes * 2 && block < p.blocks;
            const bool second = block + 1 < p.blocks;
            const int64_t row0 = t.first + (int64_t)seg.first * kWgRows + r;
            // exponent bytes of the next step are on their way while this one is converted
            int b0 = 1, b1 = 1;
            if (cols && row0 < t.last) {
                b0 = p.scales[row0 * p.blocks + block];
                if (second) b1 = p.scales[row0 * p.blocks + block + 1];
            }
            for (int step = seg.first; step < seg.last; ++step, ++c) {
                const int st = c % kWgStages, b = c & 1;
                const int64_t row = t.first + (int64_t)step * kWgRows + r;
                const bool live = row < t.last;
                int nb0 = 1, nb1 = 1;
                if (cols && step + 1 < seg.last && row + kWgRows < t.last) {
                    nb0 = p.scales[(row + kWgRows) * p.blocks + block];
                    if (second) nb1 = p.scales[(row + kWgRows) * p.blocks + block + 1];
                }
                ok = bar_wait(smem_addr(&s.full[st]), (c / kWgStages) & 1, gave_up) &&
                     bar_wait(smem_addr(&s.done[b]), ((c >> 1) & 1) ^ 1, gave_up);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (cols) wg_convert<DT>(code_s + st * kWgCodeBytes, val_s + b * kWgDyBytes, r, chunk, b0, b1, live);
                if (!live) {   // the row belongs to the next group
                    char* line = dy_s + st * kWgDyBytes + chunk * kWgBox + r * 128;
#pragma unroll
                    for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(line + j * 16) = make_uint4(0, 0, 0, 0);
                }
                b0 = nb0;
                b1 = nb1;
                fence_async_smem();
                __syncwarp();
                if (lane == 0) bar_arrive(smem_addr(&s.ready[b]));
            }
            if (!ok) break;
            ok = __all_sync(0xffffffffu, bar_wait(smem_addr(&s.acc_full), i & 1, gave_up));
            if (!ok) break;
            tc_fence_after();
            // warps 0-3: rows 0-127 of the tile, warps 4-7: rows 128-255
            const int row_in = (warp >> 2) * 128 + (warp & 3) * 32 + lane;
            const int n = t.n0 + row_in;
            const uint32_t from = tmem + ((uint32_t)(warp & 3) << 21) + (warp >> 2) * 256;
            const int k_end = min(kWgTile, p.k - t.k0);
            if (t.n0 + (warp >> 2) * 128 < p.n)
                for (int col = 0; col < k_end; col += 32) {
                    uint32_t v[32];
                    tmem_load32(from + col, v);
                    tmem_load_wait();
                    if (n < p.n) {
                        if (seg.slot < 0) {
                            wg_store<OT>(p, ((int64_t)t.g * p.n + n) * p.k, t.k0 + col, v);
                        } else {
                            float4* o = reinterpret_cast<float4*>(
                                p.partial + ((int64_t)seg.slot * kWgTile + row_in) * kWgTile + col);
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                o[j] = make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]),
                                                   __uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3]));
                        }
                    }
                }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(smem_addr(&s.acc_empty));
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) tmem_free(tmem, 512);
    if (threadIdx.x == 0 && s.gave_up && p.status) *reinterpret_cast<volatile int32_t*>(p.status) = 1;
}

// Adds the parts of each cut tile, in the order of their rows.  Block (b, i): the tile whose first part
// block b of the main kernel left, rows [16 i, 16 i + 16).
constexpr int kWgSliceRows = 16;

template <int OT>
__global__ void __launch_bounds__(256)
weight_grad_join_kernel(const WgParams p, int main_blocks) {
    const WgSlot head = p.slots[2 * blockIdx.x + 1];
    if (head.tile < 0) return;
    const WgTile t = wg_tile(p, head.tile);
    const int row_in = blockIdx.y * kWgSliceRows + threadIdx.x / 16;
    const int n = t.n0 + row_in;
    if (n >= p.n) return;
    float acc[16];
    const int c0 = threadIdx.x % 16 * 8;       // columns [c0, c0 + 8) and 128 further
    for (int b = blockIdx.x; b < main_blocks; ++b) {
        const WgSlot slot = b == (int)blockIdx.x ? head : p.slots[2 * b];
        if (slot.tile != head.tile) continue;
        const float* src = p.partial + ((int64_t)(b == (int)blockIdx.x ? 2 * b + 1 : 2 * b) * kWgTile + row_in) * kWgTile;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int col = c0 + (h >> 1) * 128 + (h & 1) * 4;
            const float4 f = t.k0 + col < p.k ? __ldcg(reinterpret_cast<const float4*>(src + col))
                                              : make_float4(0, 0, 0, 0);
            const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[h * 4 + i] = b == (int)blockIdx.x ? v[i] : acc[h * 4 + i] + v[i];
        }
        if (slot.ends) break;
    }
    const int64_t row_off = ((int64_t)t.g * p.n + n) * p.k;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int at = t.k0 + c0 + h * 128;
        if (at >= p.k) break;
        if (p.accumulate) {
            float o[8];
            widen8<OT>(load_raw8<OT>(p.out, row_off, at, p.k, p.vec_out), o);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[h * 8 + i] += o[i];
        }
        store_raw8<OT>(p.out, row_off, at, p.k, p.vec_out, narrow8<OT>(acc + h * 8));
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

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

// Blocks: one for each tile, more where few tiles have many rows (kWgMinSteps steps a block at least), at
// most one on each SM.  With groups only their average is known here.
constexpr int64_t kWgMinSteps = 4;

static int wg_grid(int device, int64_t rows, int64_t n, int64_t k, int64_t groups) {
    int sms = 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms <= 0) sms = 1;
    const int64_t tiles = (n + kWgTile - 1) / kWgTile * ((k + kWgTile - 1) / kWgTile);
    const int64_t steps = std::max<int64_t>(groups, (rows + kWgRows - 1) / kWgRows) * tiles;
    const int64_t want = std::max(tiles * groups, steps / kWgMinSteps);
    return (int)std::max<int64_t>(1, std::min<int64_t>({want, sms, kWgMaxBlocks}));
}

static uint64_t wg_workspace(int blocks) {
    return (uint64_t)blocks * 2 * (sizeof(WgSlot) + (uint64_t)kWgTile * kWgTile * sizeof(float));
}

}  // namespace aw4

using namespace aw4;

extern "C" uint64_t aw4_weight_grad_workspace(int64_t rows, int64_t n, int64_t k, int64_t groups, int32_t device) {
    if (rows <= 0 || n <= 0 || k <= 0 || groups < 1) return 0;
    return wg_workspace(wg_grid(device, rows, n, k, groups));
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
        (n + kWgTile - 1) / kWgTile * ((k + kWgTile - 1) / kWgTile) * groups > 0x7fffff00)
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
    const int grid = wg_grid(device, rows, n, k, groups);
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < (int64_t)wg_workspace(grid))
        return fail(AW4_ERR_INVALID, "aw4_weight_grad: workspace of %lld bytes is too small or misaligned",
                    (long long)workspace_bytes);
    if (!encode_tiled()) return fail(AW4_ERR_CUDA, "aw4_weight_grad: the driver has no cuTensorMapEncodeTiled");
    WgParams p;
    p.rows = rows;
    p.n = (int)n;
    p.k = (int)k;
    p.n_tiles = (int)((n + kWgTile - 1) / kWgTile);
    p.k_tiles = (int)((k + kWgTile - 1) / kWgTile);
    p.groups = (int)groups;
    p.blocks = (uint32_t)((k + kA8Block - 1) / kA8Block);
    p.scales = scales;
    p.offsets = offsets;
    p.out = out;
    p.accumulate = accumulate != 0;
    p.vec_out = (uintptr_t)out % 16 == 0 && k * size % 16 == 0;
    p.partial = static_cast<float*>(workspace);
    p.slots = reinterpret_cast<WgSlot*>(p.partial + (int64_t)grid * 2 * kWgTile * kWgTile);
    p.status = status;
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
        kernel<<<grid, kWgThreads, kWgSmem, s>>>(dy_map, code_map, p);
        note_launch();
        e = cudaGetLastError();
        if (e != cudaSuccess) return fail(AW4_ERR_CUDA, "weight_grad launch: %s", cudaGetErrorString(e));
        // without groups the host knows that blocks with whole tiles leave no parts
        const int64_t tiles = (int64_t)p.n_tiles * p.k_tiles;
        if (!offsets && tiles % grid == 0) return AW4_OK;
        weight_grad_join_kernel<ot.value><<<dim3(grid, kWgTile / kWgSliceRows), 256, 0, s>>>(p, grid);
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
