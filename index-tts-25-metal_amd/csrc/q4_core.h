// Device code shared by the kernels on 4-bit weights and 8-bit activations: the 8-bit codes of a row
// and the integer products with packed weights.
//
// The codes of a group are round(y / s) with s = max |y| / 127.  A quotient that lies next to a half
// goes to either side by the last bit of y, and y hangs on the order in which its row's squares were
// added.  So that the codes are a function of the row alone, whatever the launch, the squares are added, and y / s
// is formed, in 64 bits: v_fma_f64 runs at the rate of v_fma_f32 here, and a row's memory traffic takes longer.
#pragma once
#include "q4.h"

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
// op of the values of lanes l and l ^ D, in the order of the lanes
template <int D, class F>
__device__ __forceinline__ double pair64(double v, F op) {
    if constexpr (D >= 16) {
        const uint32_t lo = static_cast<uint32_t>(__double2loint(v)), hi = static_cast<uint32_t>(__double2hiint(v));
        if constexpr (D == 32) {
            const auto a = __builtin_amdgcn_permlane32_swap(lo, lo, false, false), b = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
            return op(__hiloint2double(b[0], a[0]), __hiloint2double(b[1], a[1]));
        } else {
            const auto a = __builtin_amdgcn_permlane16_swap(lo, lo, false, false), b = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
            return op(__hiloint2double(b[0], a[0]), __hiloint2double(b[1], a[1]));
        }
    } else if constexpr (D == 8) {
        return op(v, join64(lane_x8(lo64(v)), lane_x8(hi64(v))));
    } else if constexpr (D == 4) {
        return op(v, join64(lane_x4(lo64(v)), lane_x4(hi64(v))));
    } else if constexpr (D == 2) {
        return op(v, join64(lane_x2(lo64(v)), lane_x2(hi64(v))));
    } else {
        return op(v, join64(lane_x1(lo64(v)), lane_x1(hi64(v))));
    }
}
template <int D>
struct Lane {
    static constexpr int value = D;
};
// The value of lane l ^ D.
template <int D>
__device__ __forceinline__ float lane_of(float v) {
    if constexpr (D == 1) return lane_x1(v);
    else if constexpr (D == 2) return lane_x2(v);
    else if constexpr (D == 4) return lane_x4(v);
    else if constexpr (D == 8) return lane_x8(v);
    else {
        static_assert(D == 16, "within 32 lanes");
        return __shfl_xor(v, 16);
    }
}
__device__ __forceinline__ double add64(double a, double b) { return a + b; }
// The larger, NaN if one is.
__device__ __forceinline__ double max64(double a, double b) { return a > b || a != a ? a : b; }

// ------------------------------------------------------------------ a row's squares
// One order for every kernel that keeps a row in registers: four neighbours one after the other, two such sums; of these
// eight-column sums every 64th one after the other, then pairs of those.  (Rows of more than 32768 columns, which only one
// kernel takes, are added a thread's passes first.)
__device__ __forceinline__ double quad_squares(const float* v) {
    double s = static_cast<double>(v[0]) * static_cast<double>(v[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) s = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), s);
    return s;
}
__device__ __forceinline__ double wave_sum64(double s) {
    s = pair64<1>(s, add64);
    s = pair64<2>(s, add64);
    s = pair64<4>(s, add64);
    s = pair64<8>(s, add64);
    s = pair64<16>(s, add64);
    return pair64<32>(s, add64);
}
// Of the eight-column sums in LDS; every lane has the result.
__device__ __forceinline__ double row_squares(const double* eights, int count, int lane) {
    double s = 0.0;
    for (int i = lane; i < count; i += 64) s += eights[i];
    return wave_sum64(s);
}
// 1 / sqrt(v) and 1 / v to a few units of the last place: the instruction's estimate and two Newton steps
// (a correctly rounded quotient and root take ten times the steps, one after the other).
__device__ __forceinline__ double inv_sqrt64(double v) {
    const double e = __builtin_amdgcn_rsq(v);
    double y = e;
#pragma unroll
    for (int i = 0; i < 2; ++i) y = fma(y * 0.5, fma(-v * y, y, 1.0), y);
    return v > 0.0 && v < __builtin_huge_val() ? y : e;
}
__device__ __forceinline__ double inv64(double v) {
    const double e = __builtin_amdgcn_rcp(v);
    double y = e;
#pragma unroll
    for (int i = 0; i < 2; ++i) y = fma(y, fma(-v, y, 1.0), y);
    return y;
}
__device__ __forceinline__ double inv_rms(double squares, const NormArgs& a) {
    return inv_sqrt64(squares * inv64(static_cast<double>(a.cols)) + static_cast<double>(a.eps));
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

template <class T, int N>
struct alignas(sizeof(T) * N) Part {
    T v[N];
};

// Words that are aligned as their elements are: the memory's loads and stores take them at any such address.
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    uint32_t v[N];
};

// E elements from column c of a row of `cols`, as they lie in memory (0 behind the row's end): loads alone, so
// that several rows' are under way at once.  VEC: the row is 16-byte aligned and a multiple of eight columns long;
// others'
// elements come one by one only in the piece that the row's end cuts.  (All of them one by one, inputs from memory: norm of
// 4096 x 5121 BF16 with a residual 132 us, so 80; packing and unpacking 16384 x 5121 139 and 202, so 75 and 88.)
template <int E>
struct Raw {
    uint32_t w[E];  // four bytes an element, or (two-byte types, whole pieces) two elements a word
};
template <int E>
__device__ __forceinline__ bool whole(uint32_t c, uint32_t cols) { return c + E <= cols; }
template <bool VEC, class T, int E>
__device__ __forceinline__ void load_raw(const T* row, uint32_t c, uint32_t cols, Raw<E>& out) {
#pragma unroll
    for (int i = 0; i < E; ++i) out.w[i] = 0;
    if constexpr (VEC) {
        constexpr int words = E * sizeof(T) / 4, P = words < 4 ? words : 4;
        if (c < cols) {
#pragma unroll
            for (int k = 0; k < words / P; ++k) {
                const Part<uint32_t, P> p = reinterpret_cast<const Part<uint32_t, P>*>(row + c)[k];
#pragma unroll
                for (int i = 0; i < P; ++i) out.w[k * P + i] = p.v[i];
            }
        }
    } else if (whole<E>(c, cols)) {
        constexpr int words = E * sizeof(T) / 4, P = words < 4 ? words : 4;
#pragma unroll
        for (int k = 0; k < words / P; ++k) {
            const Loose<T, P> p = reinterpret_cast<const Loose<T, P>*>(row + c)[k];
#pragma unroll
            for (int i = 0; i < P; ++i) out.w[k * P + i] = p.v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (c + i < cols) {
                if constexpr (sizeof(T) == 4) out.w[i] = __builtin_bit_cast(uint32_t, row[c + i]);
                else out.w[i] = __builtin_bit_cast(uint16_t, row[c + i]);
            }
    }
}
template <bool VEC, class T, int E>
__device__ __forceinline__ void floats(const Raw<E>& in, uint32_t c, uint32_t cols, float (&out)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if constexpr (sizeof(T) == 4) {
            out[i] = __uint_as_float(in.w[i]);
        } else {
            const uint32_t w = VEC || whole<E>(c, cols) ? in.w[i / 2] >> (16 * (i & 1)) : in.w[i];
            out[i] = to_float(__builtin_bit_cast(T, static_cast<uint16_t>(w)));
        }
    }
}
template <bool VEC, class T>
__device__ __forceinline__ void store_row(T* row, uint32_t c, uint32_t cols, const float (&in)[kElems]) {
    if constexpr (VEC) {
        constexpr int P = 16 / sizeof(T);
        if (c < cols) {
#pragma unroll
            for (int k = 0; k < kElems / P; ++k) {
                Part<T, P> p;
#pragma unroll
                for (int i = 0; i < P; ++i) p.v[i] = from_float<T>(in[k * P + i]);
                *reinterpret_cast<Part<T, P>*>(row + c + k * P) = p;
            }
        }
    } else if (whole<kElems>(c, cols)) {
        constexpr int P = 16 / sizeof(T);
#pragma unroll
        for (int k = 0; k < kElems / P; ++k) {
            Part<T, P> p;
#pragma unroll
            for (int i = 0; i < P; ++i) p.v[i] = from_float<T>(in[k * P + i]);
            *reinterpret_cast<Loose<T, 4>*>(row + c + k * P) = __builtin_bit_cast(Loose<T, 4>, p);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kElems; ++i)
            if (c + i < cols) row[c + i] = from_float<T>(in[i]);
    }
}

// ------------------------------------------------------------------ 8-bit codes
// Over the lanes that hold a group of `group` columns, E each.
template <int E, class T, class F>
__device__ __forceinline__ T over_group(T v, int group, F step) {
    v = step(Lane<1>(), v);
    v = step(Lane<2>(), v);
    if constexpr (E == 4) v = step(Lane<4>(), v);
    if (group >= 64) {
        v = step(Lane<E == 4 ? 8 : 4>(), v);
        if (group >= 128) v = step(Lane<E == 4 ? 16 : 8>(), v);
    }
    return v;
}
// The codes q (whole numbers) and the scale of this lane's group: y = v * inv, or v * w * inv with `norm`, of which it
// holds E values.  inside: the group begins before the row's end.
// What the scale and a code are is settled in 64 bits, but few values need them.  The scale needs the group's
// largest product exactly: the largest in FP32 plus the largest remainder (exact by fma) of those that
// have it.  A code needs them where its quotient in FP32 lies within 1e-4 of a half (product, reciprocal,
// their products and inv in FP32 are off by at most 127 * 6 * 2^-24 = 4.6e-5).  Groups of zeros, of numbers near the ends of
// FP32's range or with infinities or NaN take the 64-bit way whole.  All in 64 bits took 66 instead of 30 instructions a value.
template <int E>
__device__ __forceinline__ float group_codes(const float (&v)[E], const float (&w)[E], bool norm, double inv, int group, bool inside, float (&q)[E]) {
    auto exact = [&](int i) { return norm ? static_cast<double>(v[i]) * static_cast<double>(w[i]) : static_cast<double>(v[i]); };
    auto larger = [](auto d, float x) { return fmaxf(x, lane_of<decltype(d)::value>(x)); };
    float p[E], top = 0.0f, bad = 0.0f, rest = -INFINITY;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        p[i] = norm ? v[i] * w[i] : v[i];
        top = fmaxf(top, fabsf(p[i]));
        bad = __builtin_fmaf(p[i], 0.0f, bad);  // NaN if p[i] is not finite
    }
    top = over_group<E>(bad == 0.0f ? top : INFINITY, group, larger);
    if (norm) {
#pragma unroll
        for (int i = 0; i < E; ++i) rest = fmaxf(rest, fabsf(p[i]) == top ? __builtin_fmaf(fabsf(v[i]), fabsf(w[i]), -fabsf(p[i])) : -INFINITY);
        rest = over_group<E>(rest, group, larger);
    } else {
        rest = 0.0f;
    }
    float s = static_cast<float>((static_cast<double>(top) + static_cast<double>(rest)) * inv * (1.0 / 127.0));
    if (top >= 1e-25f && top <= 1e38f && s >= 1e-35f && s <= 1e35f && inv <= 1e35) {
        const float cf = static_cast<float>(inv) * __builtin_amdgcn_rcpf(s);
        float off = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float t = p[i] * cf;
            q[i] = rintf(t);
            off = fmaxf(off, fabsf(t - q[i]));
        }
        if (off > 0.4999f) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                // |y| against the half between the two codes next to it, (k + 1 / 2) s, exact in 64 bits
                const double y = fabs(exact(i) * inv);
                const float k = floorf(fabsf(p[i] * cf) - 0.4f);
                const double half = (static_cast<double>(k) + 0.5) * static_cast<double>(s);
                const bool odd = static_cast<int>(k) & 1;
                if (fabsf(fabsf(p[i] * cf) - k - 0.5f) < 0.4f) q[i] = copysignf(y > half || (y == half && odd) ? k + 1.0f : k, p[i]);
            }
        }
        return s;
    }
    double z = 0.0, none = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        z = fmax(z, fabs(exact(i)));       // (leaves NaN out)
        none = fma(exact(i), 0.0, none);   // NaN if it is not finite
    }
    z = over_group<E>(z + none, group, [](auto d, double x) { return pair64<decltype(d)::value>(x, max64); });
    s = static_cast<float>(z * inv * (1.0 / 127.0));
    if (!(s <= 3.402823466e38f)) s = __uint_as_float(0x7fc00000u);
    if (!inside) s = 0.0f;  // (inv may be infinite or NaN)
#pragma unroll
    for (int i = 0; i < E; ++i)
        q[i] = s > 0.0f ? static_cast<float>(fmin(fmax(rint(exact(i) * inv / static_cast<double>(s)), -127.0), 127.0)) : 0.0f;
    return s;
}
// Four codes as bytes: adding 1.5 * 2^23 leaves a small whole number in the low bits.
__device__ __forceinline__ uint32_t four_codes(const float* q) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(q[i] + 12582912.0f);
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    return lo | hi;
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
