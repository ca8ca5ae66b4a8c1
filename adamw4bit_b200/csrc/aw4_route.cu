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
// Counts are integers; the sums of p go through registers and shared memory in
// a fixed order, then as whole numbers from block to block, so a repeated
// call gives the same bits.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/adamw4bit_b200.h"
#include "aw4_act8.cuh"
#include "aw4_host.h"

namespace aw4 {

constexpr int kRouteMaxK = 32;

// A row belongs to L lanes; lane i holds experts [8 i, 8 i + 8) and, where V > 8, those 8 L further on.
template <int L>
__device__ __forceinline__ int expert_of(int lane, int i) {
    return (i / 8 * L + lane) * 8 + i % 8;
}

template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = L / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int L>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    // a whole warp's in one instruction (16384 x 1024 bf16, k = 8: 35.2 us by shuffles, 31.8)
    if constexpr (L == 32) {
        v = __reduce_max_sync(0xffffffffu, v);
    } else {
#pragma unroll
        for (int o = L / 2; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    return v;
}

// exp(l - top).  The difference comes first: products of logits near the type's limits would overflow.
// FULL: to the last bit or two of float32, for float32 logits and for the weights, which are float32 whatever the logits are.
// Else the hardware's exponential, 2^-22 of the value and 1.25 * 2^-24 |l - top| of it, in the sums and 16-bit gradients of 16-bit
// logits: in a sum the terms far from the top are small, and a gradient's rounding is coarser.  65536 x 128 float32, k = 8: forward
// 34.9 us and backward 18.5 in full, 33.7 and 14.5 with the hardware's.
template <bool FULL>
__device__ __forceinline__ float exp_from(float l, float top) {
    if constexpr (FULL) {
        return expf(l - top);
    } else {
        float r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"((l - top) * 1.44269504f));
        return r;
    }
}

// Sorts eight words, the largest first (Batcher's odd-even merge).
template <typename K>
__device__ __forceinline__ void sort8(K key[8]) {
    constexpr int kA[19] = {0, 2, 4, 6, 0, 1, 4, 5, 1, 5, 0, 1, 2, 3, 2, 3, 1, 3, 5};
    constexpr int kB[19] = {1, 3, 5, 7, 2, 3, 6, 7, 2, 6, 4, 5, 6, 7, 4, 5, 2, 4, 6};
#pragma unroll
    for (int i = 0; i < 19; ++i) {
        const K a = key[kA[i]], b = key[kB[i]];
        key[kA[i]] = a > b ? a : b;
        key[kB[i]] = a > b ? b : a;
    }
}

// Takes a row's logits from the largest down.  A key holds a logit's order as an unsigned integer (-0 = +0, NaN on
// top) above its index counted down, so keys are all different and the largest is also the lowest
// index's: one word for 16-bit logits, two for float32.  None is 0.
// Each eight of a lane are sorted once and wait in shared memory; a lane holds its lists' largest, and the
// list that had the row's takes its next.
template <int DT, int L, int V>
struct Picker {
    using Key = std::conditional_t<DT == AW4_F32, unsigned long long, uint32_t>;
    static constexpr int kLists = V / 8, kShared = V * (int)sizeof(Key) / 4;      // words of shared memory a thread
    Key head[kLists];
    Key* rest[kLists];      // the next of the list's keys, 0 behind them
    int stride;

    __device__ __forceinline__ Picker(const Raw8<DT> raw[kLists], int lane, uint32_t* shared, int threads) {
        stride = threads;
#pragma unroll
        for (int c = 0; c < kLists; ++c) {
            Key key[8];
            keys(raw[c], 0xffffu - expert_of<L>(lane, c * 8), key);
            sort8(key);
            rest[c] = reinterpret_cast<Key*>(shared) + c * 8 * threads + threadIdx.x;
            head[c] = key[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) rest[c][(i - 1) * stride] = key[i];
            rest[c][7 * stride] = 0;
        }
    }
    // low: what the first one's index counts down to
    static __device__ __forceinline__ void keys(const Raw8<DT>& raw, uint32_t low, Key key[8]) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(raw.w);
        if constexpr (DT == AW4_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float z = __uint_as_float(w[i]) + 0.0f;                     // -0 + 0 = +0
                const uint32_t u = __float_as_uint(z);
                const uint32_t k = z != z ? 0xffffffffu : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
                key[i] = (unsigned long long)k << 32 | (low - i);
            }
        } else {
            // two logits at once; their sums with 0 turn -0 to +0 and a NaN to 0x7fff, the largest of all
            uint32_t two = low | (low - 1) << 16;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t u;
                if constexpr (DT == AW4_BF16) asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(u) : "r"(w[i]), "r"(0));
                else asm("add.rn.f16x2 %0, %1, %2;" : "=r"(u) : "r"(w[i]), "r"(0));
                uint32_t negative;      // all ones in the half of a number with a sign
                asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(negative) : "r"(u));
                const uint32_t k = u ^ (negative | 0x80008000u);
                key[2 * i] = __byte_perm(two, k, 0x5410);
                key[2 * i + 1] = __byte_perm(two, k, 0x7632);
                two -= 0x00020002u;
            }
        }
    }
    __device__ __forceinline__ Key next() {
        Key mine = head[0];
#pragma unroll
        for (int c = 1; c < kLists; ++c) mine = mine > head[c] ? mine : head[c];
        Key best;
        if constexpr (DT == AW4_F32) {
            const uint32_t top = lanes_max<L>((uint32_t)(mine >> 32));
            best = (unsigned long long)top << 32 | lanes_max<L>((uint32_t)(mine >> 32) == top ? (uint32_t)mine : 0u);
        } else {
            best = lanes_max<L>(mine);
        }
#pragma unroll
        for (int c = 0; c < kLists; ++c)
            if (head[c] == best) {
                head[c] = *rest[c];
                rest[c] += stride;
            }
        return best;
    }
    // whether it is above -inf
    static __device__ __forceinline__ bool some(Key best) {
        if constexpr (DT == AW4_F32) return (uint32_t)(best >> 32) > 0x007fffffu;
        else return (best >> 16) > (DT == AW4_BF16 ? 0x007fu : 0x03ffu);
    }
    static __device__ __forceinline__ int expert(Key best) { return (int)(0xffffu - ((uint32_t)best & 0xffffu)); }
    static __device__ __forceinline__ float value(Key best) {
        if constexpr (DT == AW4_F32) {
            const uint32_t k = (uint32_t)(best >> 32);
            if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
            return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
        } else {
            const uint32_t top = best >> 16;
            if (top == 0xffffu) return __uint_as_float(0x7fc00000u);
            const uint32_t u = (top & 0x8000u) ? top & 0x7fffu : ~top & 0xffffu;
            return DT == AW4_BF16 ? __uint_as_float(u << 16) : __half2float(__ushort_as_half((unsigned short)u));
        }
    }
};

// A row's logits as loaded.  WHOLE: rows of V L experts on 16 bytes.
template <int DT, int L, int V, bool WHOLE>
struct RowLogits {
    Raw8<DT> raw[V / 8];
    // p: where the row has the first of this lane's logits
    __device__ __forceinline__ void load(const RowsIn& logits, const char* p, int lane, int experts, bool in) {
#pragma unroll
        for (int c = 0; c < V / 8; ++c)
            raw[c] = load_raw8_at<DT, WHOLE>(logits, p + c * L * 8 * Elem<DT>::kBytes, (c * L + lane) * 8, in ? experts : 0);
    }
    // -inf in the place of those that take no part
    __device__ __forceinline__ void mask(int lane, int experts, bool in) {
        constexpr uint32_t kNegInf = DT == AW4_F32 ? 0xff800000u : DT == AW4_BF16 ? 0xff80u : 0xfc00u;
#pragma unroll
        for (int c = 0; c < V / 8; ++c) {
            uint32_t* w = reinterpret_cast<uint32_t*>(raw[c].w);
            const int have = !in ? 0 : WHOLE ? 8 : experts - expert_of<L>(lane, c * 8);
            if constexpr (DT == AW4_F32) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (have <= (WHOLE ? 0 : i)) w[i] = kNegInf;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (have <= (WHOLE ? 0 : 2 * i)) w[i] = kNegInf << 16 | kNegInf;
                    if constexpr (!WHOLE)
                        if (have == 2 * i + 1) w[i] = __byte_perm(w[i], kNegInf, 0x5410);
                }
            }
        }
    }
    __device__ __forceinline__ void widen(float l[V]) const {
#pragma unroll
        for (int c = 0; c < V / 8; ++c) widen8<DT>(raw[c], l + c * 8);
    }
};

// One pass over the logits, a row to L lanes, so that selections and sums are shuffles.  Bound by
// instructions (sort and selections half of them): 65536 x 128, k = 8, in 20 us in bf16 (22.6 a call with the clearing of
// the totals) and 34.9 in float32, where the bytes would take 4 and 6.  Blocks of T threads stay, their sums over rows in
// registers: one an SM with as many threads as registers allow, or two to four of 256 where those would leave SMs without a
// row (48 x 8: 4.5 us for 6.5).  Float32 from 33 experts on spills: 28 to 100 bytes a thread up to 128, 160 to 188 up to
// 256, 4 to 12 up to 512, 40 to 84 above (65536 x 256, k = 8, in 57 us).
constexpr int kRouteFew = 256;
template <int V>
constexpr int kRouteMost = V == 8 ? 1024 : V == 16 ? 768 : 512;

// What the blocks of a call add up, zero before it.  The sums of p are whole
// numbers of 2^-32, so that the order of the additions does not matter; a
// block's sum that is no number is counted instead.
struct RouteTotals {
    unsigned arrived;
    int valid_rows, not_numbers, pad;
    // then unsigned long long sum[experts], int count[experts]
};
constexpr float kRouteUnit = 4294967296.0f;

__host__ __device__ constexpr int64_t route_totals_bytes(int experts) {
    return (int64_t)sizeof(RouteTotals) + 12 * (int64_t)experts;
}

// Words of shared memory in front of a forward block's counts.
template <int DT, int L, int V, int T>
__host__ __device__ constexpr int route_work_words(int k) {
    using P = Picker<DT, L, V>;
    const int rows = P::kShared * T + T / L * k * ((int)sizeof(typename P::Key) / 4), sums = T / 32 * V * L;
    return rows > sums ? rows : sums;
}

template <int DT, int L, int V, bool WHOLE, int T>
__global__ void __launch_bounds__(T, kRouteMost<V> / T)
route_forward_kernel(const RowsIn logits, int64_t rows, int experts, int k, const uint8_t* __restrict__ valid,
                     bool renormalize, float* __restrict__ weights, int32_t* __restrict__ chosen,
                     float2* __restrict__ stats, RouteTotals* __restrict__ totals, int32_t* __restrict__ counts,
                     int32_t* __restrict__ valid_rows, float* __restrict__ balance) {
    constexpr int kThreads = T, kRows = kThreads / L;
    using P = Picker<DT, L, V>;
    using Key = typename P::Key;
    // the lists and choices of the rows in work, later the warps' sums, and behind them the counts
    extern __shared__ __align__(16) uint32_t work[];
    __shared__ float scratch[kThreads / 32];
    __shared__ int is_last;
    int32_t* count = reinterpret_cast<int32_t*>(work) + route_work_words<DT, L, V, T>(k);      // [experts + 1], the last: valid rows
    for (int i = threadIdx.x; i <= experts; i += kThreads) count[i] = 0;
    __syncthreads();
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    Key* my_key = reinterpret_cast<Key*>(work + P::kShared * kThreads) + group * k;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    const int64_t step = (int64_t)gridDim.x * kRows;
    int64_t row = (int64_t)blockIdx.x * kRows + group;
    // the next row's logits are on their way while one is worked on
    RowLogits<DT, L, V, WHOLE> now;
    uint8_t now_valid = 1;
    const char* from = logits.base + (row * logits.ld + lane * 8) * Elem<DT>::kBytes;
    const int64_t from_step = step * logits.ld * Elem<DT>::kBytes, k_step = step * k;
    now.load(logits, from, lane, experts, row < rows);
    if (valid && row < rows) now_valid = valid[row];
    int64_t picks_at = row * k;
    for (int64_t base = (int64_t)blockIdx.x * kRows; base < rows;
         base += step, row += step, picks_at += k_step) {
        const bool in = row < rows;
        bool ok = in && now_valid;
        float l[V];
        now.mask(lane, experts, ok);
        now.widen(l);
        P picker(now.raw, lane, work, kThreads);
        from += from_step;
        now.load(logits, from, lane, experts, row + step < rows);
        if (valid && row + step < rows) now_valid = valid[row + step];
        // The k largest, kept by the lanes in turn: a lane's first in registers, any further ones in shared
        // memory.
        const Key first = picker.next();
        Key mine_key = first;
        const int few = min(k, L);
#pragma unroll 2
        for (int j = 1; j < few; ++j) {
            const Key best = picker.next();
            mine_key = lane == j ? best : mine_key;
        }
        for (int j = few; j < k; ++j) {
            const Key best = picker.next();
            if (lane == j % L) my_key[j] = best;
        }
        ok = ok && P::some(first);
        const float top = P::value(first);
        float part = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            l[i] = exp_from<DT == AW4_F32>(l[i], top);
            part += l[i];
        }
        const float total = lanes_sum<L>(part);
        const float inv = ok ? 1.0f / total : 0.0f;
        if (ok)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = __fmaf_rn(l[i], inv, acc[i]);
        const bool take = ok && lane < few && P::some(mine_key);
        const float mine_w = take ? exp_from<true>(P::value(mine_key), top) : 0.0f;
        float scale = inv;
        if (renormalize) {
            float chosen_sum = mine_w;
            for (int j = lane + L; j < k; j += L)
                if (ok && P::some(my_key[j])) chosen_sum += exp_from<true>(P::value(my_key[j]), top);
            chosen_sum = lanes_sum<L>(chosen_sum);
            scale = ok ? 1.0f / chosen_sum : 0.0f;
        }
        if (in) {
            if (lane == 0) {
                stats[row] = make_float2(top, inv);
                if (ok) atomicAdd(&count[experts], 1);
            }
            if (lane < few) {
                const int e = take ? P::expert(mine_key) : -1;
                weights[picks_at + lane] = mine_w * scale;
                chosen[picks_at + lane] = e;
                if (take) atomicAdd(&count[e], 1);
            }
            for (int j = lane + L; j < k; j += L) {
                const bool more = ok && P::some(my_key[j]);
                const int e = more ? P::expert(my_key[j]) : -1;
                weights[picks_at + j] = more ? exp_from<true>(P::value(my_key[j]), top) * scale : 0.0f;
                chosen[picks_at + j] = e;
                if (more) atomicAdd(&count[e], 1);
            }
        }
    }
    // groups of the warp, then the warps in turn
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int o = 16; o >= L; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    __syncthreads();
    float* warp_sums = reinterpret_cast<float*>(work);       // [kThreads / 32][V L]: the choices are out
    if ((threadIdx.x & 31) < L)
#pragma unroll
        for (int i = 0; i < V; ++i) warp_sums[(threadIdx.x >> 5) * (V * L) + expert_of<L>(lane, i)] = acc[i];
    __syncthreads();
    unsigned long long* sum_t = reinterpret_cast<unsigned long long*>(totals + 1);
    int* count_t = reinterpret_cast<int*>(sum_t + experts);
    const bool alone = gridDim.x == 1;
    float mine = 0.0f;
    for (int e = threadIdx.x; e < experts; e += kThreads) {
        float s = 0.0f;
#pragma unroll 8
        for (int w = 0; w < kThreads / 32; ++w) s += warp_sums[w * (V * L) + e];
        if (alone) {
            counts[e] = count[e];
            mine = __fmaf_rn((float)count[e], s, mine);
        } else {
            if (count[e]) atomicAdd(&count_t[e], count[e]);
            if (s == s) atomicAdd(&sum_t[e], (unsigned long long)(s * kRouteUnit));
            else atomicAdd(&totals->not_numbers, 1);
        }
    }
    int n = count[experts], bad = 0;
    if (!alone) {
        if (threadIdx.x == 0 && n) atomicAdd(&totals->valid_rows, n);
        // the block that arrives last has every block's additions before it
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) is_last = atomicAdd(&totals->arrived, 1u) == gridDim.x - 1;
        __syncthreads();
        if (!is_last) return;
        __threadfence();
        n = __ldcg(&totals->valid_rows);
        bad = __ldcg(&totals->not_numbers);
        for (int e = threadIdx.x; e < experts; e += kThreads) {
            const int c = __ldcg(&count_t[e]);
            counts[e] = c;
            mine = __fmaf_rn((float)c, (float)__ldcg(&sum_t[e]) / kRouteUnit, mine);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        float s = bad ? __uint_as_float(0x7fc00000u) : 0.0f;
        for (int i = 0; i < kThreads / 32; ++i) s += scratch[i];
        *balance = n ? s * ((float)experts / (float)k) / (float)n / (float)n : 0.0f;
        *valid_rows = n;
    }
}

// One pass: logits, statistics and choices in, the gradient out.  65536 x 128 bf16, k = 8, in 14 us (float32 18.5);
// instructions, then HBM (5 us).  Rows that are not whole vectors spill 28 to 44 bytes a thread at 64 registers, float32
// rows of more than 512 experts 76 to 116.
constexpr int kRouteBackThreads = 256;
template <int V>
constexpr int kRouteBackBlocks = V == 8 ? 4 : 2;        // resident on an SM

template <int DT, int L, int V, bool WHOLE>
__global__ void __launch_bounds__(kRouteBackThreads, kRouteBackBlocks<V>)
route_backward_kernel(const RowsIn logits, int64_t rows, int experts, int k, bool renormalize,
                      const float* __restrict__ weights, const int32_t* __restrict__ chosen,
                      const float2* __restrict__ stats, const int32_t* __restrict__ counts,
                      const int32_t* __restrict__ valid_rows, const float* __restrict__ dweights, const float* __restrict__ dbalance,
                      const RowsOut dlogits) {
    constexpr int kRows = kRouteBackThreads / L;
    // t_j at its expert's place, zero elsewhere: written and cleared by the lanes that have the choices
    __shared__ __align__(16) float place[kRows][V * L];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    float* mine = place[group];
#pragma unroll
    for (int i = 0; i < V; ++i) mine[expert_of<L>(lane, i)] = 0.0f;
    __syncwarp();
    const float n = fmaxf((float)*valid_rows, 1.0f);
    const float unit = dbalance ? *dbalance * ((float)experts / (float)k) / n / n : 0.0f;
    float share[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = expert_of<L>(lane, i);
        share[i] = e < experts ? (float)counts[e] * unit : 0.0f;
    }
    const int64_t step = (int64_t)gridDim.x * kRows;
    int64_t row = (int64_t)blockIdx.x * kRows + group;
    // The next row is on its way while one is worked on: its logits, its statistics and a
    // lane's first choice.
    RowLogits<DT, L, V, WHOLE> now;
    float2 now_st;
    int now_at;
    float now_w, now_d;
    const char* from = logits.base + (row * logits.ld + lane * 8) * Elem<DT>::kBytes;
    const int64_t from_step = step * logits.ld * Elem<DT>::kBytes, k_step = step * k;
    char* to = dlogits.base + (row * experts + lane * 8) * Elem<DT>::kBytes;
    const int64_t to_step = step * experts * Elem<DT>::kBytes;
    int64_t picks_at = row * k;
    auto fetch = [&](int64_t r, int64_t picks_r) {
        const bool in = r < rows;
        now.load(logits, from, lane, experts, in);
        now_st = in ? stats[r] : make_float2(0.0f, 0.0f);
        now_at = -1;
        now_w = now_d = 0.0f;
        if (in && dweights && lane < k) {
            now_at = chosen[picks_r + lane];
            now_w = weights[picks_r + lane];
            now_d = dweights[picks_r + lane];
        }
    };
    fetch(row, picks_at);
    for (int64_t base = (int64_t)blockIdx.x * kRows; base < rows;
         base += step, row += step, picks_at += k_step, to += to_step) {
        const bool in = row < rows;
        const float2 st = now_st;
        const bool ok = st.y != 0.0f;             // a NaN row is a valid one
        const int picks = dweights && in ? k : 0;
        const int at = now_at;
        const float w = now_w, d = now_d;
        float l[V];
        now.mask(lane, experts, ok);
        now.widen(l);
        from += from_step;
        fetch(row + step, picks_at + k_step);
        // up to L choices a lane has one, the one that came with the logits
        const bool few = k <= L;
        float inner = at >= 0 ? w * d : 0.0f;
        if (!few)
            for (int j = lane + L; j < picks; j += L)
                if (chosen[picks_at + j] >= 0) inner = __fmaf_rn(weights[picks_at + j], dweights[picks_at + j], inner);
        inner = lanes_sum<L>(inner);
        const float back = renormalize ? inner : 0.0f;
        if (at >= 0) mine[at] = w * (d - back);
        if (!few)
            for (int j = lane + L; j < picks; j += L) {
                const int e = chosen[picks_at + j];
                if (e >= 0) mine[e] = weights[picks_at + j] * (dweights[picks_at + j] - back);
            }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            l[i] = ok ? exp_from<DT == AW4_F32>(l[i], st.x) * st.y : 0.0f;
            sum = __fmaf_rn(l[i], share[i], sum);
        }
        sum = lanes_sum<L>(sum);
        const float off = renormalize ? sum : sum + inner;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < V; ++i) l[i] = __fmaf_rn(l[i], share[i] - off, mine[expert_of<L>(lane, i)]);
        __syncwarp();
        if (at >= 0) mine[at] = 0.0f;
        if (!few)
            for (int j = lane + L; j < picks; j += L) {
                const int e = chosen[picks_at + j];
                if (e >= 0) mine[e] = 0.0f;
            }
        if (in)
#pragma unroll
            for (int c = 0; c < V / 8; ++c)
                store_raw8_at<DT, WHOLE>(dlogits, to + c * L * 8 * Elem<DT>::kBytes, (c * L + lane) * 8, experts,
                                  narrow8<DT>(l + c * 8));
        __syncwarp();
    }
}

// Lanes of a row in the forward kernel.  Fewer lanes with more logits each make a warp's selections serve more rows (65536
// rows in bf16: 128 experts by 8 lanes 22.5 us, by 16 26.7, by 4 28.8; 256 by 8 30.5, by 16 35.0, by 32
// 37.1; 64 by 4 16.6, by 8 18.1), until a row's logits and sums fill the registers; from 257 experts on a whole
// warp has its maximum in one instruction (16384 x 512: 21 us, by 16 lanes 25).  Measured with k = 8.
constexpr int route_lanes(int experts) {
    return experts <= 8 ? 1 : experts <= 16 ? 2 : experts <= 64 ? 4 : experts <= 256 ? 8 : 32;
}
template <int E, typename F>
static int32_t route_lanes_shape(F f) {
    constexpr int kLanes = route_lanes(E);
    return f(std::integral_constant<int, kLanes>(), std::integral_constant<int, E / kLanes>());
}
template <typename F>
static int32_t route_shape_forward(int experts, F f) {
    if (experts <= 8) return route_lanes_shape<8>(f);
    if (experts <= 16) return route_lanes_shape<16>(f);
    if (experts <= 32) return route_lanes_shape<32>(f);
    if (experts <= 64) return route_lanes_shape<64>(f);
    if (experts <= 128) return route_lanes_shape<128>(f);
    if (experts <= 256) return route_lanes_shape<256>(f);
    if (experts <= 512) return route_lanes_shape<512>(f);
    return route_lanes_shape<1024>(f);
}

// Lanes of a row in the backward kernel: the fewest that hold eight logits each, up to a whole warp.
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

template <typename F>
static int32_t route_form(bool whole, F f) {
    return whole ? f(std::true_type()) : f(std::false_type());
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

static int route_most(int experts) {
    int values = 8;
    while (values * route_lanes(experts) < experts) values *= 2;
    return values == 8 ? kRouteMost<8> : values == 16 ? kRouteMost<16> : kRouteMost<32>;
}
// Threads of the forward kernel's blocks, and blocks: as many as have a row, at most one an SM (of 256 threads two to four).
static int route_threads(int device, int64_t rows, int experts) {
    const int most = route_most(experts);
    return rows * route_lanes(experts) / most < sm_count(device) ? kRouteFew : most;
}
static int route_grid(int device, int64_t rows, int experts) {
    const int threads = route_threads(device, rows, experts), per = threads / route_lanes(experts);
    const int64_t resident = (int64_t)sm_count(device) * (threads == kRouteFew ? route_most(experts) / kRouteFew : 1);
    return (int)std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, resident));
}

static RowsIn route_rows(const void* p, int64_t rows, int experts, int64_t ld, int dtype) {
    const char* base = static_cast<const char*>(p);
    return {base, base + ((rows - 1) * ld + experts) * (dtype == AW4_F32 ? 4 : 2), ld, rows_on(p, ld, dtype, 16)};
}

}  // namespace aw4

using namespace aw4;

extern "C" uint64_t aw4_route_forward_workspace(int64_t rows, int32_t experts, int32_t device) {
    if (rows <= 0 || experts < 1 || experts > AW4_ROUTE_MAX_EXPERTS) return 0;
    return route_grid(device, rows, experts) == 1 ? 0 : (uint64_t)route_totals_bytes(experts);
}

extern "C" int32_t aw4_route_forward(const void* logits, int32_t dtype, int64_t rows, int32_t experts, int64_t ld,
                                     int32_t k, const uint8_t* valid, int32_t renormalize, float* weights,
                                     int32_t* chosen, float* stats, int32_t* counts, int32_t* valid_rows,
                                     float* balance, void* workspace, int64_t workspace_bytes, int32_t device,
                                     void* stream) {
    if (const int32_t rc = check_route("aw4_route_forward", dtype, rows, experts, k)) return rc;
    if (!counts || !valid_rows || !balance) return fail(AW4_ERR_INVALID, "aw4_route_forward: null buffer");
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(AW4_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    cudaStream_t s = (cudaStream_t)stream;
    if (rows == 0) {
        cudaError_t e = cudaMemsetAsync(counts, 0, experts * 4, s);
        if (e == cudaSuccess) e = cudaMemsetAsync(valid_rows, 0, 4, s);
        if (e == cudaSuccess) e = cudaMemsetAsync(balance, 0, 4, s);
        return e == cudaSuccess ? AW4_OK : fail(AW4_ERR_CUDA, "route_forward: %s", cudaGetErrorString(e));
    }
    if (!logits || !weights || !chosen || !stats || (uintptr_t)stats % 8)
        return fail(AW4_ERR_INVALID, "aw4_route_forward: null or misaligned buffer");
    const int grid = route_grid(device, rows, experts);
    if (grid > 1) {
        if (!workspace || (uintptr_t)workspace % 8 || workspace_bytes < route_totals_bytes(experts))
            return fail(AW4_ERR_INVALID, "aw4_route_forward: workspace of %lld bytes is too small or misaligned",
                        (long long)workspace_bytes);
        const cudaError_t e = cudaMemsetAsync(workspace, 0, route_totals_bytes(experts), s);
        if (e != cudaSuccess) return fail(AW4_ERR_CUDA, "route_forward: %s", cudaGetErrorString(e));
    }
    return route_by_dtype(dtype, [&](auto dt) {
        return route_shape_forward(experts, [&](auto lanes, auto v) {
            const RowsIn in = route_rows(logits, rows, experts, ld, dtype);
            const bool all_whole = rows_whole(logits, ld, experts, dtype) && experts == lanes.value * v.value;
            return route_form(all_whole, [&](auto whole) {
                auto go = [&](auto threads) -> int32_t {
                    constexpr int kThreads = threads.value;
                    auto kernel = route_forward_kernel<dt.value, lanes.value, v.value, whole.value, kThreads>;
                    const int bytes = (route_work_words<dt.value, lanes.value, v.value, kThreads>(k) + experts + 1) * 4;
                    if (bytes > 40 * 1024) {
                        const cudaError_t e =
                            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
                        if (e != cudaSuccess) return fail(AW4_ERR_CUDA, "route_forward: %s", cudaGetErrorString(e));
                    }
                    kernel<<<grid, kThreads, bytes, s>>>(in, rows, experts, k, valid, renormalize != 0, weights, chosen,
                                                         reinterpret_cast<float2*>(stats),
                                                         static_cast<RouteTotals*>(workspace), counts, valid_rows,
                                                         balance);
                    note_launch();
                    const cudaError_t e = cudaGetLastError();
                    return e == cudaSuccess ? (int32_t)AW4_OK
                                            : fail(AW4_ERR_CUDA, "route_forward launch: %s", cudaGetErrorString(e));
                };
                if (route_threads(device, rows, experts) == kRouteFew)
                    return go(std::integral_constant<int, kRouteFew>());
                return go(std::integral_constant<int, kRouteMost<v.value>>());
            });
        });
    });
}

extern "C" int32_t aw4_route_backward(const void* logits, int32_t dtype, int64_t rows, int32_t experts, int64_t ld,
                                      int32_t k, int32_t renormalize, const float* weights, const int32_t* chosen,
                                      const float* stats, const int32_t* counts, const int32_t* valid_rows,
                                      const float* dweights, const float* dbalance, void* dlogits, int32_t device,
                                      void* stream) {
    if (const int32_t rc = check_route("aw4_route_backward", dtype, rows, experts, k)) return rc;
    if (rows == 0) return AW4_OK;
    if (!logits || !weights || !chosen || !stats || !counts || !valid_rows || !dlogits || (uintptr_t)stats % 8)
        return fail(AW4_ERR_INVALID, "aw4_route_backward: null or misaligned buffer");
    DeviceGuard guard(device);
    if (!guard.ok()) return fail(AW4_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    return route_by_dtype(dtype, [&](auto dt) {
        return route_shape(experts, [&](auto lanes, auto v) {
            const int per = kRouteBackThreads / lanes.value;
            const int grid = (int)std::min<int64_t>((rows + per - 1) / per,
                                                   (int64_t)sm_count(device) * kRouteBackBlocks<v.value>);
            const RowsIn in = route_rows(logits, rows, experts, ld, dtype);
            const RowsOut out = {static_cast<char*>(dlogits), experts, rows_on(dlogits, experts, dtype, 16)};
            return route_form(rows_whole(logits, ld, experts, dtype) && rows_whole(dlogits, experts, experts, dtype) &&
                                           experts == lanes.value * v.value, [&](auto whole) {
            route_backward_kernel<dt.value, lanes.value, v.value, whole.value>
                <<<grid, kRouteBackThreads, 0, (cudaStream_t)stream>>>(
                    in, rows, experts, k, renormalize != 0, weights, chosen, reinterpret_cast<const float2*>(stats),
                    counts, valid_rows, dweights, dbalance, out);
            note_launch();
            const cudaError_t e = cudaGetLastError();
            return e == cudaSuccess ? (int32_t)AW4_OK
                                    : fail(AW4_ERR_CUDA, "route_backward launch: %s", cudaGetErrorString(e));
            });
        });
    });
}
