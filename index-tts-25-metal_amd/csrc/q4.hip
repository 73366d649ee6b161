// Operators on 4-bit weights and 8-bit activations (include/itts_ops.h): kernels, launchers and C ABI.
#include <algorithm>
#include <stdexcept>
#include <string>

#include "itts_ops.h"
#include "q4.h"
#include "q4_core.h"

namespace itts {
namespace q4 {

// ------------------------------------------------------------------ rows to 8 bits
// One workgroup per row: the row's squares in a first pass (which writes h), its codes in a second one
// that reads h again.
struct RowsArgs {
    NormArgs a;
    int kp;
};

template <class T, class WT, int G, bool NORM, bool VEC>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs ra) {
    const NormArgs& a = ra.a;
    __shared__ double red[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
        const T* res = a.residual ? static_cast<const T*>(a.residual) + r * a.residual_stride : nullptr;
        T* h = a.h_out ? static_cast<T*>(a.h_out) + r * a.h_stride : nullptr;
        auto hidden = [&](int64_t c, float (&v)[kElems]) {
            load8<VEC>(x, c, a.cols, v);
            if (res) {
                float u[kElems];
                load8<VEC>(res, c, a.cols, u);
#pragma unroll
                for (int i = 0; i < kElems; ++i) v[i] = to_float(from_float<T>(v[i] + u[i]));
            }
        };
        double inv = 1.0;
        if constexpr (NORM) {
            double ss = 0.0;
            for (int64_t c = tid * kElems; c < a.cols; c += 256 * kElems) {
                float v[kElems];
                hidden(c, v);
#pragma unroll
                for (int i = 0; i < kElems; ++i) ss = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), ss);
            }
            ss = wave_sum64(ss);
            if (lane == 0) red[wave] = ss;
            __syncthreads();
            ss = (red[0] + red[1]) + (red[2] + red[3]);
            __syncthreads();
            inv = 1.0 / sqrt(ss / static_cast<double>(a.cols) + static_cast<double>(a.eps));
        }
        for (int64_t c = tid * kElems; c < ra.kp; c += 256 * kElems) {
            float v[kElems];
            hidden(c, v);
            if (h) store8<VEC>(h, c, a.cols, v);
            double z[kElems];
            if constexpr (NORM) {
                float w[kElems];
                load8<VEC>(static_cast<const WT*>(a.weight), c, a.cols, w);
#pragma unroll
                for (int i = 0; i < kElems; ++i) z[i] = static_cast<double>(v[i]) * static_cast<double>(w[i]);
            } else {
#pragma unroll
                for (int i = 0; i < kElems; ++i) z[i] = static_cast<double>(v[i]);
            }
            int8_t code[kElems];
            const float s = group_codes<G>(z, inv, c - c % G < a.cols, code);
            *reinterpret_cast<uint2*>(a.q + r * ra.kp + c) = pack_codes(code);
            if (c % G == 0) a.scales[r * (ra.kp / G) + c / G] = s;
            if (a.values) {
#pragma unroll
                for (int i = 0; i < kElems; ++i) v[i] = static_cast<float>(code[i]) * s;
                store8<VEC>(static_cast<T*>(a.values) + r * a.values_stride, c, a.cols, v);
            }
        }
    }
}

// ------------------------------------------------------------------ packing
struct PackArgs {
    const void* w;
    int64_t stride;
    int n, k;
    uint8_t* packed;
    uint16_t* scales;
};

__device__ __forceinline__ float quarter_max(float v) { return xmax16(xmax32(v)); }  // over lanes l, l ^ 16, l ^ 32, l ^ 48

// One wave per tile: lane 16 j + r holds row r's columns 32 b + 8 j .. + 7 of the tile, b < 4.
template <class T, int G, bool VEC>
__global__ __launch_bounds__(256) void pack_kernel(PackArgs a) {
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    const int kb = (a.k + kTileCols - 1) / kTileCols;
    const int64_t tiles = static_cast<int64_t>((a.n + kTileRows - 1) / kTileRows) * kb;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (t >= tiles) return;
    const int64_t row = t / kb * kTileRows + r;
    const int c0 = static_cast<int>(t % kb) * kTileCols + 8 * j;
    const T* src = static_cast<const T*>(a.w) + row * a.stride;
    float v[4][kElems];
#pragma unroll
    for (int b = 0; b < 4; ++b) load8<VEC>(src, c0 + 32 * b, row < a.n ? a.k : 0, v[b]);
    uint32_t out[4] = {0, 0, 0, 0};
    constexpr int B = G / 32, NG = 4 / B;
    uint16_t sc[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        float mx = -INFINITY, mn = -INFINITY, bad = 0.0f;
#pragma unroll
        for (int b = g * B; b < (g + 1) * B; ++b)
#pragma unroll
            for (int i = 0; i < kElems; ++i) {
                mx = fmaxf(mx, v[b][i]);
                mn = fmaxf(mn, -v[b][i]);
                bad = __builtin_fmaf(v[b][i], 0.0f, bad);
            }
        mx = quarter_max(mx);
        mn = quarter_max(mn);
        const float wrong = quarter_max(bad == 0.0f ? 0.0f : 1.0f);
        const __bf16 sb = static_cast<__bf16>(fmaxf(mx / 7.0f, mn / 8.0f));
        float s = static_cast<float>(sb);
        if (wrong != 0.0f || !(fabsf(s) <= 3.402823466e38f)) s = __uint_as_float(0x7fc00000u);
        sc[g] = static_cast<uint16_t>(__float_as_uint(s) >> 16);
#pragma unroll
        for (int b = g * B; b < (g + 1) * B; ++b)
#pragma unroll
            for (int i = 0; i < kElems; ++i) {
                // The quotient is rounded to FP32, which could put it on a half; the remainder, exact
                // (q s has 12 bits and is next to v), tells.  A remainder of s / 2 is a half indeed, and q even.
                float q = rintf(v[b][i] / s);
                const float rem = __builtin_fmaf(-q, s, v[b][i]);
                if (2.0f * fabsf(rem) > s) q += copysignf(1.0f, rem);
                q = fminf(fmaxf(q, -8.0f), 7.0f);
                const int code = s > 0.0f ? static_cast<int>(q) : 0;
                out[2 * (b >> 1) + (i >> 2)] |= (static_cast<uint32_t>(code) & 15u) << (8 * (i & 3) + 4 * (b & 1));
            }
    }
    *reinterpret_cast<u32x4*>(a.packed + t * kTileBytes + lane * 16) = u32x4{out[0], out[1], out[2], out[3]};
    if (j == 0) {
#pragma unroll
        for (int g = 0; g < NG; ++g) a.scales[(t * kTileRows + r) * NG + g] = sc[g];
    }
}

struct UnpackArgs {
    const uint8_t* packed;
    const uint16_t* scales;
    int n, k;
    void* out;
    int64_t stride;
};

template <class T, int G, bool VEC>
__global__ __launch_bounds__(256) void unpack_kernel(UnpackArgs a) {
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4;
    const int kb = (a.k + kTileCols - 1) / kTileCols;
    const int64_t tiles = static_cast<int64_t>((a.n + kTileRows - 1) / kTileRows) * kb;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (t >= tiles) return;
    const int64_t row = t / kb * kTileRows + r;
    if (row >= a.n) return;
    const u32x4 w = *reinterpret_cast<const u32x4*>(a.packed + t * kTileBytes + lane * 16);
    T* dst = static_cast<T*>(a.out) + row * a.stride;
    const int c0 = static_cast<int>(t % kb) * kTileCols + 8 * j;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const float s = bf16_to_f32(a.scales[(t * kTileRows + r) * (128 / G) + 32 * b / G]);
        float v[kElems];
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            const int shift = 8 * (i & 3) + 4 * (b & 1);
            v[i] = static_cast<float>(static_cast<int32_t>(w[2 * (b >> 1) + (i >> 2)] << (28 - shift)) >> 28) * s;
        }
        store8<VEC>(dst, c0 + 32 * b, a.k, v);
    }
}

// ------------------------------------------------------------------ products
// One wave per 16 tokens x 16 weight rows, over all columns.
template <class T, int G, bool SWIGLU>
__global__ __launch_bounds__(256) void matmul_kernel(ProductArgs a) {
    const int lane = threadIdx.x & 63, c = lane & 15, quarter = lane >> 4;
    const int nt = blockIdx.x * 4 + (threadIdx.x >> 6), m0 = blockIdx.y * 16;
    const int kb = (a.k + kTileCols - 1) / kTileCols;
    if (nt * kTileRows >= a.n) return;
    constexpr int NG = 128 / G;
    const int8_t* x = a.q + static_cast<int64_t>(min(m0 + c, a.rows - 1)) * kb * kTileCols;
    const uint8_t* w = a.packed + static_cast<int64_t>(nt) * kb * kTileBytes + lane * 16;
    const uint16_t* ws = a.wscales + (static_cast<int64_t>(nt) * kb * kTileRows + c) * NG;
    const float* xs[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) xs[r] = a.qscales + static_cast<int64_t>(min(m0 + 4 * quarter + r, a.rows - 1)) * kb * NG;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int b = 0; b < kb; ++b) {
        const TokenCodes xc = token_codes(x + b * kTileCols, lane);
        const u32x4 wc = *reinterpret_cast<const u32x4*>(w + static_cast<int64_t>(b) * kTileBytes);
        i32x4 f[NG];
        tile_product<G>(xc, wc, f);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const float s = weight_scale(ws[static_cast<int64_t>(b) * kTileRows * NG + g]);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(static_cast<float>(f[g][r]), xs[r][b * NG + g] * s, acc[r]);
        }
    }
    const int n = nt * kTileRows + c;
    const float bias = a.bias && n < a.n ? a.bias[n] : 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int m = m0 + 4 * quarter + r;
        float v = acc[r] + bias;
        int col = n;
        bool live = m < a.rows && n < a.n;
        if constexpr (SWIGLU) {
            const float u = itts::lane_x1(v);
            v = silu_mul(v, u);
            col = n >> 1;
            live = live && !(n & 1);
        }
        if (live) {
            if (a.residual) v += to_float(static_cast<const T*>(a.residual)[m * a.residual_stride + col]);
            static_cast<T*>(a.out)[m * a.out_stride + col] = from_float<T>(v);
        }
    }
}

// ------------------------------------------------------------------ launchers
namespace {
template <class F>
hipError_t by_type(int dtype, F&& f) {
    if (dtype == ITTS_T_F32) return f(float());
    if (dtype == ITTS_T_BF16) return f(__bf16());
    return f(_Float16());
}
template <int V>
struct Int {
    static constexpr int value = V;
};
template <class F>
hipError_t by_group(int group, F&& f) {
    if (group == 32) return f(Int<32>());
    if (group == 64) return f(Int<64>());
    return f(Int<128>());
}
template <class F>
hipError_t by_bool(bool b, F&& f) {
    return b ? f(Int<1>()) : f(Int<0>());
}
size_t type_size(int dtype) { return dtype == ITTS_T_F32 ? 4 : 2; }
// Rows that load8 and store8 may take 16 bytes at a time.
bool rows_aligned(const void* p, int64_t stride, int dtype) {
    return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * static_cast<int64_t>(type_size(dtype)) % 16 == 0);
}
int pad_cols(int64_t k) { return static_cast<int>((k + kTileCols - 1) / kTileCols * kTileCols); }
}  // namespace

hipError_t launch_rows(const NormArgs& a, hipStream_t s) {
    if (a.rows == 0) return hipSuccess;
    const bool vec = a.cols % kElems == 0 && rows_aligned(a.x, a.x_stride, a.dtype) && rows_aligned(a.residual, a.residual_stride, a.dtype) &&
                     rows_aligned(a.h_out, a.h_stride, a.dtype) && rows_aligned(a.values, a.values_stride, a.dtype) &&
                     rows_aligned(a.weight, 0, a.dtype);
    RowsArgs ra{a, pad_cols(a.cols)};
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(a.rows, 1 << 20)));
    return by_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return by_group(a.group, [&](auto g) {
            return by_bool(vec, [&](auto v) {
                constexpr int G = decltype(g)::value;
                constexpr bool V = decltype(v)::value;
                if (!a.weight) hipLaunchKernelGGL((rows_kernel<T, T, G, false, V>), grid, dim3(256), 0, s, ra);
                else if (a.weight_dtype == a.dtype) hipLaunchKernelGGL((rows_kernel<T, T, G, true, V>), grid, dim3(256), 0, s, ra);
                else hipLaunchKernelGGL((rows_kernel<T, float, G, true, V>), grid, dim3(256), 0, s, ra);
                return hipGetLastError();
            });
        });
    });
}

hipError_t launch_product(const ProductArgs& a, hipStream_t s) {
    if (a.rows == 0) return hipSuccess;
    const dim3 grid((a.n + 63) / 64, (a.rows + 15) / 16);
    return by_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return by_group(a.group, [&](auto g) {
            return by_bool(a.swiglu, [&](auto sw) {
                hipLaunchKernelGGL((matmul_kernel<T, decltype(g)::value, decltype(sw)::value>), grid, dim3(256), 0, s, a);
                return hipGetLastError();
            });
        });
    });
}

hipError_t launch_pack(const void* w, int64_t stride, int dtype, int n, int k, int group, void* packed, void* scales, hipStream_t s) {
    const PackArgs a{w, stride, n, k, static_cast<uint8_t*>(packed), static_cast<uint16_t*>(scales)};
    const bool vec = k % kElems == 0 && rows_aligned(w, stride, dtype);
    const int64_t tiles = static_cast<int64_t>((n + kTileRows - 1) / kTileRows) * (pad_cols(k) / kTileCols);
    const dim3 grid(static_cast<unsigned>((tiles + 3) / 4));
    return by_type(dtype, [&](auto t) {
        return by_group(group, [&](auto g) {
            return by_bool(vec, [&](auto v) {
                hipLaunchKernelGGL((pack_kernel<decltype(t), decltype(g)::value, decltype(v)::value>), grid, dim3(256), 0, s, a);
                return hipGetLastError();
            });
        });
    });
}

hipError_t launch_unpack(const void* packed, const void* scales, int n, int k, int group, int dtype, void* out, int64_t stride, hipStream_t s) {
    const UnpackArgs a{static_cast<const uint8_t*>(packed), static_cast<const uint16_t*>(scales), n, k, out, stride};
    const bool vec = k % kElems == 0 && rows_aligned(out, stride, dtype);
    const int64_t tiles = static_cast<int64_t>((n + kTileRows - 1) / kTileRows) * (pad_cols(k) / kTileCols);
    const dim3 grid(static_cast<unsigned>((tiles + 3) / 4));
    return by_type(dtype, [&](auto t) {
        return by_group(group, [&](auto g) {
            return by_bool(vec, [&](auto v) {
                hipLaunchKernelGGL((unpack_kernel<decltype(t), decltype(g)::value, decltype(v)::value>), grid, dim3(256), 0, s, a);
                return hipGetLastError();
            });
        });
    });
}

}  // namespace q4
}  // namespace itts

// ------------------------------------------------------------------ C ABI
namespace {
using namespace itts::q4;

thread_local std::string g_ops_error;

template <class F>
int ops_guarded(F&& f) {
    try {
        f();
        return ITTS_OK;
    } catch (const std::invalid_argument& e) {
        g_ops_error = e.what();
        return ITTS_EINVAL;
    } catch (const std::exception& e) {
        g_ops_error = e.what();
        return ITTS_ERUNTIME;
    }
}

void need(bool ok, const char* message) {
    if (!ok) throw std::invalid_argument(message);
}
void launched(hipError_t e) {
    if (e != hipSuccess) throw std::runtime_error(std::string("HIP error ") + hipGetErrorString(e));
}
bool type_ok(int32_t t) { return t == ITTS_T_F32 || t == ITTS_T_BF16 || t == ITTS_T_F16; }
bool group_ok(int32_t g) { return g == 32 || g == 64 || g == 128; }
// Sizes up to these keep every index that the kernels form in 32 bits where they use 32, and every grid in range.
constexpr int64_t kMaxRows = int64_t(1) << 30, kMaxN = int64_t(1) << 26, kMaxK = int64_t(1) << 20;
bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
bool aligned_for(const void* p, int32_t dtype) { return aligned(p, dtype == ITTS_T_F32 ? 4 : 2); }

void check_rows(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t cols, int32_t group, const void* values,
                int64_t values_stride, const int8_t* q, const float* scales) {
    need(type_ok(dtype), "Element type is F32, BF16 or F16");
    need(group_ok(group), "Group is 32, 64 or 128 columns");
    need(rows >= 0 && rows <= kMaxRows, "Row count out of range");
    need(cols >= 1 && cols <= kMaxK, "Column count out of range");
    if (rows == 0) return;
    need(x && q && scales, "Missing tensor");
    need(x_stride >= 0 && (!values || rows == 1 || values_stride >= cols), "Row stride out of range");
    need(aligned_for(x, dtype) && aligned_for(values, dtype) && aligned(q, 16) && aligned(scales, 4), "Misaligned tensor");
}

void check_weight(const void* packed, const void* scales, int64_t n, int64_t k, int32_t group) {
    need(group_ok(group), "Group is 32, 64 or 128 columns");
    need(n >= 1 && n <= kMaxN && k >= 1 && k <= kMaxK, "Weight size out of range");
    need(packed && scales, "Missing tensor");
    need(aligned(packed, 16) && aligned(scales, 16), "Misaligned tensor");
}

ProductArgs product_args(int64_t rows, const void* packed, const void* scales, int64_t n, int64_t k, int32_t group, const float* bias,
                         const void* residual, int64_t residual_stride, uint32_t flags, int32_t dtype, void* out, int64_t out_stride) {
    check_weight(packed, scales, n, k, group);
    need(type_ok(dtype), "Element type is F32, BF16 or F16");
    need((flags & ~ITTS_Q4_SWIGLU) == 0, "Unknown flag");
    const bool swiglu = flags & ITTS_Q4_SWIGLU;
    need(!swiglu || n % 2 == 0, "SwiGLU takes pairs of columns");
    need(rows >= 0 && rows <= 16 * 65535, "Row count out of range");
    if (rows != 0) {
        need(out, "Missing tensor");
        need(residual_stride >= 0 && (rows == 1 || out_stride >= (swiglu ? n / 2 : n)), "Row stride out of range");
        need(aligned_for(out, dtype) && aligned_for(residual, dtype) && aligned(bias, 4), "Misaligned tensor");
    }
    ProductArgs p{};
    p.rows = static_cast<int>(rows);
    p.packed = static_cast<const uint8_t*>(packed);
    p.wscales = static_cast<const uint16_t*>(scales);
    p.n = static_cast<int>(n);
    p.k = static_cast<int>(k);
    p.group = group;
    p.bias = bias;
    p.residual = residual;
    p.residual_stride = residual_stride;
    p.swiglu = swiglu;
    p.dtype = dtype;
    p.out = out;
    p.out_stride = out_stride;
    return p;
}

size_t codes_bytes(int64_t rows, int64_t k) { return (static_cast<size_t>(rows) * pad_cols(k) + 255) / 256 * 256; }
}  // namespace

extern "C" {

const char* itts_ops_last_error(void) { return g_ops_error.c_str(); }

int itts_rmsnorm_q8(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight,
                    int32_t weight_dtype, int32_t dtype, int64_t rows, int64_t cols, float eps, int32_t group, void* h_out,
                    int64_t h_stride, void* values, int64_t values_stride, int8_t* q, float* scales, void* stream) {
    return ops_guarded([&] {
        check_rows(x, x_stride, dtype, rows, cols, group, values, values_stride, q, scales);
        need(weight_dtype == dtype || weight_dtype == ITTS_T_F32, "The norm's weight has the rows' type or F32");
        need(eps >= 0.0f, "Negative eps");
        if (rows == 0) return;
        need(weight, "Missing tensor");
        need(residual_stride >= 0 && (!h_out || rows == 1 || h_stride >= cols), "Row stride out of range");
        need(aligned_for(residual, dtype) && aligned_for(h_out, dtype) && aligned_for(weight, weight_dtype), "Misaligned tensor");
        NormArgs a{x, x_stride, residual, residual_stride, weight, weight_dtype, dtype, rows, cols, eps, group, h_out, h_stride, values,
                   values_stride, q, scales};
        launched(launch_rows(a, static_cast<hipStream_t>(stream)));
    });
}

int itts_q8_quantize(const void* x, int64_t x_stride, int32_t dtype, int64_t rows, int64_t cols, int32_t group, void* values,
                     int64_t values_stride, int8_t* q, float* scales, void* stream) {
    return ops_guarded([&] {
        check_rows(x, x_stride, dtype, rows, cols, group, values, values_stride, q, scales);
        if (rows == 0) return;
        NormArgs a{x, x_stride, nullptr, 0, nullptr, dtype, dtype, rows, cols, 0.0f, group, nullptr, 0, values, values_stride, q, scales};
        launched(launch_rows(a, static_cast<hipStream_t>(stream)));
    });
}

size_t itts_q4_packed_bytes(int64_t n, int64_t k) {
    if (n < 1 || n > kMaxN || k < 1 || k > kMaxK) return 0;
    return static_cast<size_t>((n + 15) / 16) * (pad_cols(k) / kTileCols) * kTileBytes;
}

size_t itts_q4_scale_count(int64_t n, int64_t k, int32_t group) {
    return group_ok(group) ? itts_q4_packed_bytes(n, k) / kTileBytes * kTileRows * (128 / group) : 0;
}

int itts_q4_pack(const void* w, int64_t w_stride, int32_t dtype, int64_t n, int64_t k, int32_t group, void* packed, void* scales,
                 void* stream) {
    return ops_guarded([&] {
        check_weight(packed, scales, n, k, group);
        need(type_ok(dtype), "Element type is F32, BF16 or F16");
        need(w, "Missing tensor");
        need(w_stride >= 0, "Row stride out of range");
        need(aligned_for(w, dtype), "Misaligned tensor");
        launched(launch_pack(w, w_stride, dtype, static_cast<int>(n), static_cast<int>(k), group, packed, scales, static_cast<hipStream_t>(stream)));
    });
}

int itts_q4_unpack(const void* packed, const void* scales, int64_t n, int64_t k, int32_t group, int32_t dtype, void* out,
                   int64_t out_stride, void* stream) {
    return ops_guarded([&] {
        check_weight(packed, scales, n, k, group);
        need(type_ok(dtype), "Element type is F32, BF16 or F16");
        need(out, "Missing tensor");
        need(n == 1 || out_stride >= k, "Row stride out of range");
        need(aligned_for(out, dtype), "Misaligned tensor");
        launched(launch_unpack(packed, scales, static_cast<int>(n), static_cast<int>(k), group, dtype, out, out_stride, static_cast<hipStream_t>(stream)));
    });
}

int itts_q4_matmul(const int8_t* q, const float* qscales, int64_t rows, const void* packed, const void* scales, int64_t n, int64_t k,
                   int32_t group, const float* bias, const void* residual, int64_t residual_stride, uint32_t flags, int32_t dtype,
                   void* out, int64_t out_stride, void* stream) {
    return ops_guarded([&] {
        ProductArgs p = product_args(rows, packed, scales, n, k, group, bias, residual, residual_stride, flags, dtype, out, out_stride);
        if (rows == 0) return;
        need(q && qscales, "Missing tensor");
        need(aligned(q, 16) && aligned(qscales, 4), "Misaligned tensor");
        p.q = q;
        p.qscales = qscales;
        launched(launch_product(p, static_cast<hipStream_t>(stream)));
    });
}

size_t itts_q4_linear_workspace(int64_t rows, int64_t n, int64_t k, int32_t group) {
    if (rows < 1 || n < 1 || k < 1 || k > kMaxK || !group_ok(group)) return 0;
    return codes_bytes(rows, k) + static_cast<size_t>(rows) * (pad_cols(k) / group) * sizeof(float);
}

int itts_q4_linear(const void* x, int64_t x_stride, int32_t x_dtype, int64_t rows, const void* norm_weight, int32_t weight_dtype,
                   float eps, const void* packed, const void* scales, int64_t n, int64_t k, int32_t group, const float* bias,
                   const void* residual, int64_t residual_stride, uint32_t flags, int32_t dtype, void* out, int64_t out_stride,
                   void* workspace, size_t workspace_bytes, void* stream) {
    return ops_guarded([&] {
        ProductArgs p = product_args(rows, packed, scales, n, k, group, bias, residual, residual_stride, flags, dtype, out, out_stride);
        need(type_ok(x_dtype), "Element type is F32, BF16 or F16");
        need(!norm_weight || weight_dtype == x_dtype || weight_dtype == ITTS_T_F32, "The norm's weight has the rows' type or F32");
        need(!norm_weight || eps >= 0.0f, "Negative eps");
        if (rows == 0) return;
        need(x, "Missing tensor");
        need(x_stride >= 0, "Row stride out of range");
        need(aligned_for(x, x_dtype) && (!norm_weight || aligned_for(norm_weight, weight_dtype)), "Misaligned tensor");
        const size_t bytes = itts_q4_linear_workspace(rows, n, k, group);
        need(bytes == 0 || (workspace && workspace_bytes >= bytes), "Workspace too small");
        need(aligned(workspace, 256), "Misaligned workspace");
        int8_t* q = static_cast<int8_t*>(workspace);
        float* qs = reinterpret_cast<float*>(q + codes_bytes(rows, k));
        const NormArgs a{x, x_stride, nullptr, 0, norm_weight, weight_dtype, x_dtype, rows, k, eps, group, nullptr, 0, nullptr, 0, q, qs};
        launched(launch_rows(a, static_cast<hipStream_t>(stream)));
        p.q = q;
        p.qscales = qs;
        launched(launch_product(p, static_cast<hipStream_t>(stream)));
    });
}

}  // extern "C"
