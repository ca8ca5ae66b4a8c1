// aw4_act8.cuh -- the 8-bit activation checkpoint: format, encode and decode.
//
// A row of `cols` values is cut into blocks of 32.  A block keeps one byte,
// e + 127, and 32 two's complement bytes q that stand for q * 2^e:
//
//     e = max(floor(log2(max |x|)) - 6, e_min)      q = clamp(rn(x * 2^-e), -127, 127)
//
// so the largest magnitude takes 64..127 steps of 2^e.  A power of two needs
// no division, x * 2^-e is exact, and q * 2^e has at most seven significant
// bits: it is a bf16 or f16 value, and a tensor core multiplies it without any
// rounding beyond the checkpoint's own.  e_min keeps q * 2^e a normal float32 (-126), and
// for float16 a multiple of its smallest step (-24).  Byte 255 marks a block
// that held an infinity or a NaN: it reads back as NaN, since no whole number
// stands for either.
//
// Memory: codes[rows][pitch], pitch = cols rounded up to 32 with zeros behind
// the last column; scales[rows][pitch / 32].  Eight values belong to a lane,
// so a block is four neighbouring lanes.
#pragma once

#include "aw4_device.cuh"

namespace aw4 {

constexpr int kA8Block = 32;     // values per exponent
constexpr int kA8Nan = 255;      // scale byte of a block that is not finite

// Smallest scale byte: e_min + 127.
template <int DT>
constexpr int kA8MinByte = DT == AW4_F16 ? 103 : 1;

// Eight values as loaded, so that several loads are in flight before the first is used.
template <int DT>
struct Raw8 {
    uint4 w[Elem<DT>::kBytes / 2];
};

// Rows of a matrix in memory.  `vec`: every row starts on 16 bytes.  Kernels come in two
// forms: WHOLE where all their matrices' rows are whole chunks of eight that start on a chunk's size (16 bytes, 32 in
// float32), so that an access is one vector and the code for the others is not in the way (router
// backward: 400 instructions a row without).
struct RowsIn {
    const char* base;
    const char* end;      // behind the last value
    int64_t ld;           // values from row to row
    bool vec;
};
struct RowsOut {
    char* base;
    int64_t ld;
    bool vec;
};

inline bool rows_on(const void* p, int64_t ld, int dtype, int bytes) {
    return (uintptr_t)p % bytes == 0 && ld * (dtype == AW4_F32 ? 4 : 2) % bytes == 0;
}
// Whether a matrix can take the WHOLE form.
inline bool rows_whole(const void* p, int64_t ld, int64_t cols, int dtype) {
    return cols % 8 == 0 && rows_on(p, ld, dtype, dtype == AW4_F32 ? 32 : 16);
}

// Values [col, col + 8) of the row that has its column `col` at p; zeros from `cols` on.
template <int DT, bool WHOLE>
__device__ __forceinline__ Raw8<DT> load_raw8_at(const RowsIn& m, const char* p, int col, int cols) {
    constexpr int kSize = Elem<DT>::kBytes, kWords = kSize * 2;
    Raw8<DT> r;
    if constexpr (WHOLE && DT == AW4_F32) {
        uint32_t* v = reinterpret_cast<uint32_t*>(r.w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0;
        if (col < cols)
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                         : "l"(p));
        return r;
    } else if constexpr (WHOLE) {
        r.w[0] = col < cols ? __ldcs(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
        return r;
    }
    uint32_t* w = reinterpret_cast<uint32_t*>(r.w);
    if (col + 8 <= cols) {
        if (m.vec) {
#pragma unroll
            for (int i = 0; i < kSize / 2; ++i) r.w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
            return r;
        }
        // the aligned words around them, where those lie inside the matrix, shifted into place
        const char* q = reinterpret_cast<const char*>((uintptr_t)p & ~(uintptr_t)15);
        constexpr int kLoads = kSize / 2 + 1;
        if (q >= m.base && q + 16 * kLoads <= m.end) {
            uint32_t v[4 * kLoads];
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(q) + i);
            const uint32_t at = (uint32_t)(p - q);
            if (at & 8)
#pragma unroll
                for (int i = 0; i + 2 < 4 * kLoads; ++i) v[i] = v[i + 2];
            if (at & 4)
#pragma unroll
                for (int i = 0; i + 1 < 4 * kLoads; ++i) v[i] = v[i + 1];
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                w[i] = kSize == 2 && (at & 2) ? __funnelshift_r(v[i], v[i + 1], 16) : v[i];
            return r;
        }
    }
    if constexpr (DT == AW4_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = col + i < cols ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = col + 2 * i < cols ? reinterpret_cast<const uint16_t*>(p)[2 * i] : 0u;
            const uint32_t hi = col + 2 * i + 1 < cols ? reinterpret_cast<const uint16_t*>(p)[2 * i + 1] : 0u;
            w[i] = lo | (hi << 16);
        }
    }
    return r;
}

template <int DT, bool WHOLE>
__device__ __forceinline__ Raw8<DT> load_raw8(const RowsIn& m, int64_t row, int col, int cols) {
    return load_raw8_at<DT, WHOLE>(m, m.base + (row * m.ld + col) * Elem<DT>::kBytes, col, cols);
}

template <int DT, bool WHOLE>
__device__ __forceinline__ void store_raw8_at(const RowsOut& m, char* p, int col, int cols, const Raw8<DT>& r) {
    constexpr int kSize = Elem<DT>::kBytes;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
    if constexpr (WHOLE && DT == AW4_F32) {
        if (col < cols)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                         ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
        return;
    } else if constexpr (WHOLE) {
        if (col < cols) __stcs(reinterpret_cast<uint4*>(p), r.w[0]);
        return;
    }
    if (col + 8 <= cols) {
        if (m.vec) {
#pragma unroll
            for (int i = 0; i < kSize / 2; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, r.w[i]);
            return;
        }
        if constexpr (DT == AW4_F32) {
            // the one aligned group of four words among the eight, the others by themselves
            const int head = (int)((16 - ((uintptr_t)p & 15)) & 15) >> 2;
            uint32_t v[7];
#pragma unroll
            for (int i = 0; i < 7; ++i) v[i] = w[i];
            if (head & 2)
#pragma unroll
                for (int i = 0; i < 5; ++i) v[i] = v[i + 2];
            if (head & 1)
#pragma unroll
                for (int i = 0; i < 6; ++i) v[i] = v[i + 1];
            uint32_t* o = reinterpret_cast<uint32_t*>(p);
            *reinterpret_cast<uint4*>(o + head) = make_uint4(v[0], v[1], v[2], v[3]);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < head || i >= head + 4) o[i] = w[i];
        } else if ((uintptr_t)p & 2) {
            uint16_t* o = reinterpret_cast<uint16_t*>(p);
            o[0] = (uint16_t)w[0];
#pragma unroll
            for (int i = 0; i < 3; ++i)
                *reinterpret_cast<uint32_t*>(o + 1 + 2 * i) = __funnelshift_r(w[i], w[i + 1], 16);
            o[7] = (uint16_t)(w[3] >> 16);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(p)[i] = w[i];
        }
        return;
    }
    if constexpr (DT == AW4_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < cols) reinterpret_cast<uint32_t*>(p)[i] = w[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < cols) reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(w[i / 2] >> (16 * (i % 2)));
    }
}

template <int DT>
__device__ __forceinline__ void widen8(const Raw8<DT>& r, float v[8]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
    if constexpr (DT == AW4_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    } else if constexpr (DT == AW4_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = bf16_lo(w[i]);
            v[2 * i + 1] = bf16_hi(w[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

// The eight values rounded to the element type, as words.
template <int DT>
__device__ __forceinline__ Raw8<DT> narrow8(const float v[8]) {
    Raw8<DT> r;
    uint32_t* w = reinterpret_cast<uint32_t*>(r.w);
    if constexpr (DT == AW4_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
    } else if constexpr (DT == AW4_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    return r;
}

template <int DT, bool WHOLE>
__device__ __forceinline__ void store_raw8(const RowsOut& m, int64_t row, int col, int cols, const Raw8<DT>& r) {
    store_raw8_at<DT, WHOLE>(m, m.base + (row * m.ld + col) * Elem<DT>::kBytes, col, cols, r);
}

// The same by a whole warp, lanes with `in` storing.  Where its lanes hold consecutive whole chunks of a row
// that starts off 16 bytes, each takes what it lacks to whole aligned vectors from the next lane (TURN).  In
// float32 that pays everywhere (8192 x 8191 read back and forth 220 -> 135 us), in 16 bits where a
// kernel does little else (118 -> 104 us; gated activation 276 -> 305).
template <int DT, bool WHOLE, bool TURN = DT == AW4_F32>
__device__ __forceinline__ void store_raw8_warp(const RowsOut& m, int64_t row, int col, int cols, bool in,
                                                const Raw8<DT>& r) {
    constexpr int kSize = Elem<DT>::kBytes, kWords = 2 * kSize;
    if constexpr (WHOLE) {
        if (in) store_raw8<DT, true>(m, row, col, cols, r);
    } else if constexpr (!TURN) {
        if (in) store_raw8<DT, false>(m, row, col, cols, r);
    } else {
        const int lane = threadIdx.x & 31;
        char* p = m.base + (row * m.ld + col) * kSize;
        const char* first = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, (unsigned long long)p, 0));
        if (m.vec || !__all_sync(0xffffffffu, in && col + 8 <= cols && p == first + lane * 8 * kSize)) {
            if (in) store_raw8_at<DT, false>(m, p, col, cols, r);
            return;
        }
        const int head = (int)((16 - ((uintptr_t)p & 15)) & 15);       // bytes before the first aligned vector
        const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
        uint32_t v[kWords + 4];
#pragma unroll
        for (int i = 0; i < kWords; ++i) v[i] = w[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[kWords + i] = __shfl_down_sync(0xffffffffu, w[i], 1);
        if (head & 8)
#pragma unroll
            for (int i = 0; i + 2 < kWords + 4; ++i) v[i] = v[i + 2];
        if (head & 4)
#pragma unroll
            for (int i = 0; i + 1 < kWords + 4; ++i) v[i] = v[i + 1];
        if (kSize == 2 && (head & 2))
#pragma unroll
            for (int i = 0; i < kWords; ++i) v[i] = __funnelshift_r(v[i], v[i + 1], 16);
        if (lane < 31 || head == 0)
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i)
                __stcs(reinterpret_cast<uint4*>(p + head) + i,
                       make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
        // the first lane's values before its first vector, the last lane's behind it
        if (head && (lane == 0 || lane == 31))
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (lane == 0 ? i * kSize < head : i * kSize >= head) {
                    if constexpr (DT == AW4_F32) reinterpret_cast<uint32_t*>(p)[i] = w[i];
                    else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(w[i / 2] >> (16 * (i % 2)));
                }
    }
}

// Larger magnitude of two words' values (its sign is not meaningful); a NaN is above every number.
template <int DT>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (DT == AW4_F32) asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else if constexpr (DT == AW4_BF16) asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

struct A8Block {
    int byte;       // e + 127, or kA8Nan
    float most;     // largest magnitude
};

// The exponent of a block whose four lanes hold eight values each.
template <int DT>
__device__ __forceinline__ A8Block a8_block(const Raw8<DT>& r) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
    constexpr int kWords = Elem<DT>::kBytes * 2;
    uint32_t m = larger<DT>(w[0], w[1]);
#pragma unroll
    for (int i = 2; i < kWords; ++i) m = larger<DT>(m, w[i]);
    m = larger<DT>(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = larger<DT>(m, __shfl_xor_sync(0xffffffffu, m, 2));
    if constexpr (DT == AW4_F32) {
        m &= 0x7fffffffu;
    } else {
        m &= 0x7fff7fffu;
        m = max(m & 0xffffu, m >> 16);             // as integers, like the magnitudes
        if constexpr (DT == AW4_BF16) m <<= 16;
        else m = __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
    }
    const int field = (int)(m >> 23);              // floor(log2) + 127; 255: not finite
    return {field == 255 ? kA8Nan : max(field - 6, kA8MinByte<DT>), __uint_as_float(m)};
}

// The eight codes.  Adding 1.5 * 2^23 leaves rn(x * 2^-e), ties to even, in
// the low bits of the sum.  Only a block whose largest magnitude is 127.5 steps or
// more rounds to 128: the warp looks once whether it has one.
__device__ __forceinline__ uint2 a8_encode8(const float v[8], const A8Block& b) {
    const float inv = __uint_as_float(b.byte == kA8Nan ? 0u : (uint32_t)(254 - b.byte) << 23);
    const f2 inv2 = pk2(inv, inv), magic = pk2(12582912.0f, 12582912.0f);
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) upk2(f2_fma(pk2(v[i], v[i + 1]), inv2, magic), t[i], t[i + 1]);
    if (__any_sync(0xffffffffu, b.most * inv >= 127.5f))
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = fminf(fmaxf(t[i], 12582912.0f - 127.0f), 12582912.0f + 127.0f);
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(t[i]);
    uint2 r;
    r.x = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
    r.y = __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410);
    return r;
}

__device__ __forceinline__ float a8_scale(int b) {
    return __uint_as_float(b == kA8Nan ? 0x7fc00000u : (uint32_t)b << 23);
}

// q * 2^e of eight codes.  q + 128 in the low bits of 2^23 is the float
// 2^23 + 128 + q; the subtraction (a product by one and a sum) and the product are exact.
__device__ __forceinline__ void a8_decode8(uint2 w, float s, float v[8]) {
    const f2 one = pk2(1.0f, 1.0f), off = pk2(-8388736.0f, -8388736.0f), ss = pk2(s, s);
    const uint32_t u[2] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float a = __uint_as_float(__byte_perm(u[i / 4], 0x4b000000u, 0x7540 + i % 4));
        const float b = __uint_as_float(__byte_perm(u[i / 4], 0x4b000000u, 0x7541 + i % 4));
        upk2(f2_mul(f2_fma(pk2(a, b), one, off), ss), v[i], v[i + 1]);
    }
}

// Where a lane's chunk of eight values lies: chunk `unit` of the
// rows' chunks laid end to end, `per_row` of them in a row.
struct ChunkAt {
    int64_t row;
    int col;       // first column
    bool in;
};

// The first chunk of a warp's run, split once by a division that all lanes share.
struct RunAt {
    int64_t row;
    uint32_t rem;
};

__device__ __forceinline__ RunAt run_at(int64_t unit, uint32_t per_row) {
    RunAt r;
    if ((unit >> 32) == 0) {
        r.row = (uint32_t)unit / per_row;
        r.rem = (uint32_t)unit % per_row;
    } else {
        r.row = unit / per_row;
        r.rem = (uint32_t)(unit % per_row);
    }
    return r;
}

__device__ __forceinline__ ChunkAt chunk_at(const RunAt& r, uint32_t off, uint32_t per_row,
                                            int64_t rows) {
    ChunkAt c;
    uint32_t k = r.rem + off;
    c.row = r.row;
    if (k >= per_row) {
        const uint32_t over = k / per_row;
        c.row += over;
        k -= over * per_row;
    }
    c.col = (int)(k * 8);
    c.in = c.row < rows;
    return c;
}

}  // namespace aw4
