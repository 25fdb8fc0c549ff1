// Operand tiles of the 16-bit matrix instructions for the context operators (attention, gated feed-forward).
//
// One product form serves every element type: v_mfma_f32_32x32x16_{bf16,f16}, fp32 accumulation (lane l of the C tile holds column
// l & 31 and rows 8 (r >> 2) + 4 (l >> 5) + (r & 3), r = 0..15; an A or B operand is eight consecutive k at 8 (l >> 5) of row l & 31).
//   bf16, fp16   one plane: the value itself.
//   fp32         three bf16 planes, x = hi + mid + lo (8 significant bits each, exact to 24), and the six products hi.hi, hi.mid,
//                mid.hi, mid.mid, hi.lo, lo.hi.  hi is cut off (to nearest, the largest values would become infinite), mid rounded to
//                nearest: lo has either sign and is below 2^-16 |x|, so the three dropped products are below 2^-22 |a b| and average
//                to zero (with mid cut off, too: 2^-21, always towards zero, 0.7 x 2^-24 on average).  Six passes of the 16-bit pipe cost 6/16 of the fp32 matrix instruction's time (2.5 against 0.157 PFLOP/s).
//                A non-finite fp32 value gives non-finite results (its residual planes are NaN).
// Values are kept as raw 16-bit lanes (short vectors) and cast at the instruction.
#pragma once
#include <hip/hip_runtime.h>

#include "common.h"

namespace eq {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float pf32x2 __attribute__((ext_vector_type(2)));
typedef float pf32x4 __attribute__((ext_vector_type(4)));
typedef float pf32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 pbf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 pbf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 pf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 pf16x8 __attribute__((ext_vector_type(8)));

enum { kF32 = EQUIGSPR_F32, kBF16 = EQUIGSPR_BF16, kF16 = EQUIGSPR_F16 };

template <int T> struct Num;
template <> struct Num<kF32> { using type = float; static constexpr int planes = 3; };
template <> struct Num<kBF16> { using type = __bf16; static constexpr int planes = 1; };
template <> struct Num<kF16> { using type = _Float16; static constexpr int planes = 1; };

// eight values on their way from memory to a tile
template <int T> struct Raw8 { s16x8 v; };
template <> struct Raw8<kF32> { pf32x4 v[2]; };

// one operand: eight values of every plane
template <int T> struct Op8 { s16x8 p[Num<T>::planes]; };

template <int T>
__device__ __forceinline__ pf32x16 mfma32(s16x8 a, s16x8 b, pf32x16 c) {
    if constexpr (T == kF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(pf16x8, a), __builtin_bit_cast(pf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pbf16x8, a), __builtin_bit_cast(pbf16x8, b), c, 0, 0, 0);
}

// acc += A B with all planes (the small products first)
template <int T>
__device__ __forceinline__ void mma(pf32x16& acc, const Op8<T>& a, const Op8<T>& b) {
    if constexpr (T == kF32) {
        acc = mfma32<T>(a.p[2], b.p[0], acc);
        acc = mfma32<T>(a.p[0], b.p[2], acc);
        acc = mfma32<T>(a.p[1], b.p[1], acc);
        acc = mfma32<T>(a.p[1], b.p[0], acc);
        acc = mfma32<T>(a.p[0], b.p[1], acc);
    }
    acc = mfma32<T>(a.p[0], b.p[0], acc);
}

// two fp32 -> the planes' packed 16-bit pairs.  fp32: hi + mid + lo is the value exactly.
template <int T>
__device__ __forceinline__ void split2(float x, float y, unsigned (&out)[Num<T>::planes]) {
    if constexpr (T == kF32) {
        const unsigned ux = __float_as_uint(x), uy = __float_as_uint(y);
        out[0] = __builtin_amdgcn_perm(uy, ux, 0x07060302u);
        const float rx = x - __uint_as_float(ux & 0xffff0000u), ry = y - __uint_as_float(uy & 0xffff0000u);
        out[1] = __builtin_bit_cast(unsigned, __builtin_convertvector((pf32x2){rx, ry}, pbf16x2));
        const float sx = rx - __uint_as_float(out[1] << 16), sy = ry - __uint_as_float(out[1] & 0xffff0000u);
        out[2] = __builtin_amdgcn_perm(__float_as_uint(sy), __float_as_uint(sx), 0x07060302u);
    } else if constexpr (T == kBF16) {
        out[0] = __builtin_bit_cast(unsigned, __builtin_convertvector((pf32x2){x, y}, pbf16x2));
    } else {
        out[0] = __builtin_bit_cast(unsigned, __builtin_convertvector((pf32x2){x, y}, pf16x2));
    }
}

template <int T>
__device__ __forceinline__ Op8<T> pack8(const float (&x)[8]) {
    u32x4 w[Num<T>::planes];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        unsigned o[Num<T>::planes];
        split2<T>(x[2 * i], x[2 * i + 1], o);
#pragma unroll
        for (int p = 0; p < Num<T>::planes; ++p) w[p][i] = o[p];
    }
    Op8<T> r;
#pragma unroll
    for (int p = 0; p < Num<T>::planes; ++p) r.p[p] = __builtin_bit_cast(s16x8, w[p]);
    return r;
}

// what the rounding of pack8 dropped, as an operand of the same 16-bit type
template <int T>
__device__ __forceinline__ Op8<T> pack8_rest(const float (&x)[8]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i] - (float)(typename Num<T>::type)x[i];
    return pack8<T>(r);
}

template <int T>
__device__ __forceinline__ Op8<T> planes_of(const Raw8<T>& raw) {
    if constexpr (T == kF32) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = raw.v[i >> 2][i & 3];
        return pack8<T>(x);
    } else {
        Op8<T> r;
        r.p[0] = raw.v;
        return r;
    }
}

template <int T>
__device__ __forceinline__ float raw_float(const Raw8<T>& raw, int i) {
    if constexpr (T == kF32) return raw.v[i >> 2][i & 3];
    else return (float)__builtin_bit_cast(typename Num<T>::type, (short)raw.v[i]);
}

template <int T>
__device__ __forceinline__ Raw8<T> raw_zero() {
    Raw8<T> r;
    if constexpr (T == kF32) r.v[0] = r.v[1] = (pf32x4){0.f, 0.f, 0.f, 0.f};
    else r.v = (s16x8){0, 0, 0, 0, 0, 0, 0, 0};
    return r;
}

// Memory accesses of 16 bytes on addresses that are only aligned to their element: gfx950 takes them (a parameter inside a flat block,
// a head of odd width), at the cost of an extra cycle where a line is crossed.
typedef pf32x4 pf32x4_u __attribute__((aligned(4)));
typedef s16x8 s16x8_u __attribute__((aligned(2)));
typedef s16x4 s16x4_u __attribute__((aligned(2)));

// eight values at row + col of a row of `width` values; those at or behind the end are zero.  The row's last eight values are loaded for a
// chunk that crosses the end, and moved down (one load for every lane; value by value, the edge tiles of odd sizes took three times as
// long as the others).
template <int T>
__device__ __forceinline__ Raw8<T> load8(const typename Num<T>::type* row, int col, int width) {
    Raw8<T> r;
    if (width >= 8) {
        const int start = min(col, width - 8), move = col - start;
        if constexpr (T == kF32) {
            r.v[0] = *reinterpret_cast<const pf32x4_u*>(row + start);
            r.v[1] = *reinterpret_cast<const pf32x4_u*>(row + start + 4);
            if (move > 0) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = r.v[i >> 2][i & 3];
#pragma unroll
                for (int k = 0; k < 3; ++k)
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = move & (1 << k) ? (i + (1 << k) < 8 ? x[i + (1 << k)] : 0.f) : x[i];
#pragma unroll
                for (int i = 0; i < 8; ++i) r.v[i >> 2][i & 3] = move < 8 ? x[i] : 0.f;
            }
        } else {
            r.v = *reinterpret_cast<const s16x8_u*>(row + start);
            if (move > 0) {
                typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
                const u64x2 w = __builtin_bit_cast(u64x2, r.v);
                const int bits = 16 * (move & 3);
                u64x2 o = {bits ? (w[0] >> bits) | (w[1] << (64 - bits)) : w[0], w[1] >> bits};
                if (move >= 4) o = (u64x2){o[1], 0};
                if (move >= 8) o = (u64x2){0, 0};
                r.v = __builtin_bit_cast(s16x8, o);
            }
        }
    } else {
        r = raw_zero<T>();
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (col + i < width) {
                if constexpr (T == kF32) r.v[i >> 2][i & 3] = row[col + i];
                else r.v[i] = __builtin_bit_cast(short, row[col + i]);
            }
    }
    return r;
}

// the same value by value behind the last whole chunk: fewer registers (the large feed-forward tiles have none to spare)
template <int T>
__device__ __forceinline__ Raw8<T> load8_small(const typename Num<T>::type* row, int col, int width) {
    Raw8<T> r;
    if (col + 8 <= width) return load8<T>(row + col, 0, 8);
    r = raw_zero<T>();
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (col + i < width) {
            if constexpr (T == kF32) r.v[i >> 2][i & 3] = row[col + i];
            else r.v[i] = __builtin_bit_cast(short, row[col + i]);
        }
    return r;
}

// A tile of rows of W 16-bit values in LDS.  The rows' stride is padded so that the 16 rows of a ds_read_b128 group start in 16 different
// bank quads; the four rows of a transposed read then overlap two-fold, which costs a cycle.  (An XOR swizzle has neither conflict but an
// address register per k-step: in the kernels' keys' gradients at W = 128 that was the difference between one and two waves per SIMD.)
template <int W>
struct Tile {
    static_assert(W == 32 || W == 64 || W == 128 || W == 256, "tile width");
    static constexpr int kStride = W == 32 ? 40 : W == 64 ? 72 : W == 128 ? 152 : 280;
    // values of a tile of `rows` rows
    __host__ __device__ static constexpr int size(int rows) { return rows * kStride; }
    // offset (in 16-bit values) of chunk c of row r
    __device__ static __forceinline__ int at(int r, int c) { return r * kStride + c * 8; }
    // eight consecutive values of one row
    __device__ static __forceinline__ s16x8 row8(const short* t, int r, int c) { return *reinterpret_cast<const s16x8*>(t + at(r, c)); }
    // transposed: lane l receives the values of rows r0 .. r0 + 3 in column col0 + (l & 15); r0 % 4 == 0, col0 % 16 == 0 (both may
    // differ between the four groups of 16 lanes).  Lane i of a group fetches eight bytes of row r0 + (i >> 2).
    __device__ static __forceinline__ s16x4 col4(const short* t, int r0, int col0, int lane) {
        const int i = lane & 15, r = r0 + (i >> 2), c = col0 + 4 * (i & 3);
        const short* a = t + at(r, c >> 3) + (c & 4);
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a);
    }
};

__device__ __forceinline__ s16x8 join8(s16x4 a, s16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// blocks are dealt to the eight XCDs in turn: give every XCD a contiguous run of logical blocks, so that neighbours share its L2
__device__ __forceinline__ int xcd_block(int id, int n) {
    const int x = id & 7, per = n >> 3, rem = n & 7;
    return x * per + (x < rem ? x : rem) + (id >> 3);
}

template <int T>
__device__ __forceinline__ void store_value(typename Num<T>::type* p, float v) { *p = (typename Num<T>::type)v; }

// the first n of four consecutive values, the rest zero
template <int T>
__device__ __forceinline__ void load4(const typename Num<T>::type* p, int n, float (&v)[4]) {
    if (n >= 4) {
        if constexpr (T == kF32) {
            const pf32x4 r = *reinterpret_cast<const pf32x4_u*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = r[i];
        } else {
            const s16x4 r = *reinterpret_cast<const s16x4_u*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (float)__builtin_bit_cast(typename Num<T>::type, (short)r[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < n ? (float)p[i] : 0.f;
    }
}

// the first n of four consecutive values
template <int T>
__device__ __forceinline__ void store4(typename Num<T>::type* p, const float (&v)[4], int n) {
    if (n >= 4) {
        if constexpr (T == kF32) {
            *reinterpret_cast<pf32x4_u*>(p) = (pf32x4){v[0], v[1], v[2], v[3]};
        } else {
            unsigned a[1], b[1];
            split2<T>(v[0], v[1], a);
            split2<T>(v[2], v[3], b);
            *reinterpret_cast<s16x4_u*>(p) = __builtin_bit_cast(s16x4, make_uint2(a[0], b[0]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < n) store_value<T>(p + i, v[i]);
    }
}

// eight consecutive values, of which the first n exist
template <int T>
__device__ __forceinline__ void load8f(const typename Num<T>::type* p, int n, float (&v)[8]) {
    const Raw8<T> r = load8<T>(p, 0, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = raw_float<T>(r, i);
}
template <int T>
__device__ __forceinline__ void store8(typename Num<T>::type* p, const float (&v)[8], int n) {
    if constexpr (T != kF32) {
        if (n >= 8) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                unsigned o[1];
                split2<T>(v[2 * i], v[2 * i + 1], o);
                w[i] = o[0];
            }
            *reinterpret_cast<s16x8_u*>(p) = __builtin_bit_cast(s16x8, w);
            return;
        }
    }
    float a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] = v[i]; b[i] = v[4 + i]; }
    store4<T>(p, a, n);
    if (n > 4) store4<T>(p + 4, b, n - 4);
}

}  // namespace eq
