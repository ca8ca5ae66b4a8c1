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

// Values [col, col + 8) of a row at `base`; zeros from `cols` on.  `vec`: the
// row starts on 16 bytes, so that whole chunks are vector loads.
template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw8(const void* base, int64_t row_off, int col, int cols,
                                              bool vec) {
    Raw8<DT> r;
    if (vec && col + 8 <= cols) {
        const char* p = static_cast<const char*>(base) + (row_off + col) * Elem<DT>::kBytes;
#pragma unroll
        for (int i = 0; i < Elem<DT>::kBytes / 2; ++i)
            r.w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    } else {
        uint32_t* w = reinterpret_cast<uint32_t*>(r.w);
        if constexpr (DT == AW4_F32) {
            const uint32_t* p = static_cast<const uint32_t*>(base) + row_off;
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = col + i < cols ? p[col + i] : 0u;
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(base) + row_off;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = col + 2 * i < cols ? p[col + 2 * i] : 0u;
                const uint32_t hi = col + 2 * i + 1 < cols ? p[col + 2 * i + 1] : 0u;
                w[i] = lo | (hi << 16);
            }
        }
    }
    return r;
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

template <int DT>
__device__ __forceinline__ void store_raw8(void* base, int64_t row_off, int col, int cols, bool vec,
                                           const Raw8<DT>& r) {
    if (vec && col + 8 <= cols) {
        char* p = static_cast<char*>(base) + (row_off + col) * Elem<DT>::kBytes;
#pragma unroll
        for (int i = 0; i < Elem<DT>::kBytes / 2; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, r.w[i]);
    } else {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
        if constexpr (DT == AW4_F32) {
            uint32_t* p = static_cast<uint32_t*>(base) + row_off;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (col + i < cols) p[col + i] = w[i];
        } else {
            uint16_t* p = static_cast<uint16_t*>(base) + row_off;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (col + i < cols) p[col + i] = (uint16_t)(w[i / 2] >> (16 * (i % 2)));
        }
    }
}

// Scale byte of a block whose four lanes hold eight values each.  The maximum
// is taken over magnitude bits as integers, where a NaN is above every number.
template <int DT>
__device__ __forceinline__ int a8_scale_byte(const float v[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const int field = (int)(m >> 23);                       // floor(log2) + 127; 255: not finite
    return field == 255 ? kA8Nan : max(field - 6, kA8MinByte<DT>);
}

// The eight codes under scale byte b.  Adding 1.5 * 2^23 leaves rn(x * 2^-e),
// ties to even, in the low bits of the sum.
__device__ __forceinline__ uint2 a8_encode8(const float v[8], int b) {
    const float inv = __uint_as_float(b == kA8Nan ? 0u : (uint32_t)(254 - b) << 23);
    uint32_t t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float s = __fmaf_rn(v[i], inv, 12582912.0f);
        t[i] = __float_as_uint(fminf(fmaxf(s, 12582912.0f - 127.0f), 12582912.0f + 127.0f));
    }
    uint2 r;
    r.x = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
    r.y = __byte_perm(__byte_perm(t[4], t[5], 0x0040), __byte_perm(t[6], t[7], 0x0040), 0x5410);
    return r;
}

__device__ __forceinline__ float a8_scale(int b) {
    return __uint_as_float(b == kA8Nan ? 0x7fc00000u : (uint32_t)b << 23);
}

// q * 2^e of four codes.  q + 128 in the low bits of 2^23 is the float
// 2^23 + 128 + q; the subtraction and the product are both exact.
__device__ __forceinline__ void a8_decode4(uint32_t w, float s, float v[4]) {
    w ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540 + i)) - 8388736.0f) * s;
}

__device__ __forceinline__ void a8_decode8(uint2 w, float s, float v[8]) {
    a8_decode4(w.x, s, v);
    a8_decode4(w.y, s, v + 4);
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
