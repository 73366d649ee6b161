// Device code shared by the kernels on 4-bit weights and 8-bit activations: the 8-bit codes of a row
// and the integer products with packed weights.
//
// The codes of a group are round(y / s) with s = max |y| / 127.  A quotient that lies next to a half
// goes to either side by the last bit of y, and y hangs on the order in which its row's squares were
// added.  So that the codes are a function of the row alone, whatever the launch, the squares are added, and y / s
// is formed, in 64 bits: v_fma_f64 runs at the rate of v_fma_f32 here, and a row's memory traffic takes longer.
#pragma once
#include "common.h"

namespace itts {
namespace q4 {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 16, kTileCols = 128, kTileBytes = 1024;
constexpr int kElems = 8;  // consecutive columns that a lane holds

// ------------------------------------------------------------------ 64-bit values across lanes
__device__ __forceinline__ double join64(float lo, float hi) { return __hiloint2double(__float_as_int(hi), __float_as_int(lo)); }
__device__ __forceinline__ float lo64(double v) { return __int_as_float(__double2loint(v)); }
__device__ __forceinline__ float hi64(double v) { return __int_as_float(__double2hiint(v)); }
__device__ __forceinline__ double lane_x1(double v) { return join64(itts::lane_x1(lo64(v)), itts::lane_x1(hi64(v))); }
__device__ __forceinline__ double lane_x2(double v) { return join64(itts::lane_x2(lo64(v)), itts::lane_x2(hi64(v))); }
__device__ __forceinline__ double lane_x4(double v) { return join64(itts::lane_x4(lo64(v)), itts::lane_x4(hi64(v))); }
__device__ __forceinline__ double lane_x8(double v) { return join64(itts::lane_x8(lo64(v)), itts::lane_x8(hi64(v))); }
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int d = 32; d > 8; d >>= 1) v += __shfl_xor(v, d);
    v += lane_x8(v);
    v += lane_x4(v);
    v += lane_x2(v);
    return v + lane_x1(v);
}
// The larger, NaN if one is.
__device__ __forceinline__ double max_nan(double a, double b) { return a > b || a != a ? a : b; }
// Over the G / 8 lanes that hold a group.
template <int G>
__device__ __forceinline__ double group_max64(double v) {
    v = max_nan(v, lane_x1(v));
    v = max_nan(v, lane_x2(v));
    if constexpr (G >= 64) v = max_nan(v, lane_x4(v));
    if constexpr (G >= 128) v = max_nan(v, lane_x8(v));
    return v;
}

// ------------------------------------------------------------------ element types
template <class T>
__device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }
// To the nearest, halves to even.  The empty asm keeps v a number in FP32: without it the compiler may
// fuse the product or sum that gives v into the conversion to FP16 (v_fma_mixlo_f16), here and not there.
template <class T>
__device__ __forceinline__ T from_float(float v) {
    if constexpr (sizeof(T) == 2) asm("" : "+v"(v));
    return static_cast<T>(v);
}

template <class T>
struct alignas(sizeof(T) * kElems) Pack8 {
    T v[kElems];
};
template <class T>
struct alignas(16) Part16 {
    T v[16 / sizeof(T)];
};

// Eight elements from column c of a row of `cols`, zeros behind its end.  VEC: the row is 16-byte
// aligned and a multiple of eight columns long.
template <bool VEC, class T>
__device__ __forceinline__ void load8(const T* row, int64_t c, int64_t cols, float (&out)[kElems]) {
    if constexpr (VEC) {
        constexpr int P = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < kElems; ++i) out[i] = 0.0f;
        if (c < cols) {
#pragma unroll
            for (int k = 0; k < kElems / P; ++k) {
                const Part16<T> p = *reinterpret_cast<const Part16<T>*>(row + c + k * P);
#pragma unroll
                for (int i = 0; i < P; ++i) out[k * P + i] = to_float(p.v[i]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kElems; ++i) out[i] = c + i < cols ? to_float(row[c + i]) : 0.0f;
    }
}
template <bool VEC, class T>
__device__ __forceinline__ void store8(T* row, int64_t c, int64_t cols, const float (&in)[kElems]) {
    if constexpr (VEC) {
        constexpr int P = 16 / sizeof(T);
        if (c < cols) {
#pragma unroll
            for (int k = 0; k < kElems / P; ++k) {
                Part16<T> p;
#pragma unroll
                for (int i = 0; i < P; ++i) p.v[i] = from_float<T>(in[k * P + i]);
                *reinterpret_cast<Part16<T>*>(row + c + k * P) = p;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kElems; ++i)
            if (c + i < cols) row[c + i] = from_float<T>(in[i]);
    }
}

// ------------------------------------------------------------------ 8-bit codes
// The codes and the scale of this lane's group, of which it holds the eight values z[i] * inv (z = x or
// h * weight, exact in 64 bits; inv = 1 or the row's 1 / rms).  inside: the group begins before the row's end.
template <int G>
__device__ __forceinline__ float group_codes(const double (&z)[kElems], double inv, bool inside, int8_t (&code)[kElems]) {
    double top = 0.0, bad = 0.0;
#pragma unroll
    for (int i = 0; i < kElems; ++i) {
        top = fmax(top, fabs(z[i]));    // (leaves NaN out)
        bad = fma(z[i], 0.0, bad);      // NaN if z[i] is not finite
    }
    top = group_max64<G>(top + bad);
    float s = static_cast<float>(top * inv / 127.0);
    if (!(s <= 3.402823466e38f)) s = __uint_as_float(0x7fc00000u);
    if (!inside) s = 0.0f;  // (inv may be infinite or NaN)
    const double c = inv / static_cast<double>(s);
#pragma unroll
    for (int i = 0; i < kElems; ++i) {
        double t = z[i] * c;
        // next to a half the product's rounding could decide: the quotient itself does
        if (fabs(fabs(t - rint(t)) - 0.5) < 1e-9) t = z[i] * inv / static_cast<double>(s);
        const double r = fmin(fmax(rint(t), -127.0), 127.0);
        code[i] = s > 0.0f ? static_cast<int8_t>(static_cast<int>(r)) : int8_t(0);
    }
    return s;
}
__device__ __forceinline__ uint2 pack_codes(const int8_t (&c)[kElems]) {
    uint2 v = make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v.x |= static_cast<uint32_t>(static_cast<uint8_t>(c[i])) << (8 * i);
        v.y |= static_cast<uint32_t>(static_cast<uint8_t>(c[4 + i])) << (8 * i);
    }
    return v;
}

// ------------------------------------------------------------------ products with packed weights
// A lane's 16 bytes of a tile as matrix-instruction operands, 16 times the codes: a code in the high half of a
// byte with zeros below is 16 times itself in two's complement, and 1 / 16 goes into the scale
// (exactly).  lo: columns 64 p + 8 j + i, hi: 64 p + 32 + 8 j + i.
constexpr uint32_t kHigh = 0xf0f0f0f0u;
__device__ __forceinline__ void tile_codes(u32x4 w, int p, uint32_t (&lo)[2], uint32_t (&hi)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        lo[i] = (w[2 * p + i] << 4) & kHigh;
        hi[i] = w[2 * p + i] & kHigh;
    }
}
// A token's codes at the lane's columns of a tile: four pieces of eight, 32 columns apart.
struct TokenCodes {
    uint2 p[4];
};
__device__ __forceinline__ TokenCodes token_codes(const int8_t* row, int lane) {
    TokenCodes x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.p[i] = *reinterpret_cast<const uint2*>(row + 32 * i + 8 * (lane >> 4));
    return x;
}
__device__ __forceinline__ i32x4 mfma64(uint2 xa, uint2 xb, const uint32_t (&lo)[2], const uint32_t (&hi)[2], i32x4 c) {
    const i32x4 a = {static_cast<int>(xa.x), static_cast<int>(xa.y), static_cast<int>(xb.x), static_cast<int>(xb.y)};
    const i32x4 b = {static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(hi[0]), static_cast<int>(hi[1])};
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ long join32(uint32_t a, uint32_t b) { return static_cast<long>(static_cast<uint64_t>(b) << 32 | a); }
__device__ __forceinline__ i32x4 mfma32(uint2 x, const uint32_t (&w)[2], i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x32_i8(join32(x.x, x.y), join32(w[0], w[1]), c, 0, 0, 0);
}

// One tile (128 columns) of 16 tokens times 16 weight rows, f[g] the group's product sum (times 16): the
// instruction holds tokens as its rows, weights as its columns, so lane l ends with weight row
// l % 16 and the four tokens at 4 (l / 16) + r.
template <int G>
__device__ __forceinline__ void tile_product(const TokenCodes& x, u32x4 w, i32x4 (&f)[128 / G]) {
    const i32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        uint32_t lo[2], hi[2];
        tile_codes(w, p, lo, hi);
        if constexpr (G == 32) {
            f[2 * p] = mfma32(x.p[2 * p], lo, zero);
            f[2 * p + 1] = mfma32(x.p[2 * p + 1], hi, zero);
        } else if constexpr (G == 64) {
            f[p] = mfma64(x.p[2 * p], x.p[2 * p + 1], lo, hi, zero);
        } else {
            f[0] = mfma64(x.p[2 * p], x.p[2 * p + 1], lo, hi, p ? f[0] : zero);
        }
    }
}

// BF16 to float, with the 1 / 16 of tile_codes.
__device__ __forceinline__ float weight_scale(uint16_t s) { return bf16_to_f32(s) * 0.0625f; }

__device__ __forceinline__ float silu_mul(float g, float u) { return (g / (1.0f + expf(-g))) * u; }

}  // namespace q4
}  // namespace itts
