// Operators on 4-bit weights and 8-bit activations (include/itts_ops.h): kernels, launchers and C ABI.
#include <algorithm>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "itts_ops.h"
#include "q4.h"
#include "q4_core.h"

namespace itts {
namespace q4 {

// load_raw and floats for a type known at run time.
template <bool VEC, int E>
__device__ __forceinline__ void load_raw_as(const void* row, uint32_t c, uint32_t cols, int dtype, Raw<E>& out) {
    if (dtype == ITTS_T_F32) load_raw<VEC>(static_cast<const float*>(row), c, cols, out);
    else load_raw<VEC>(static_cast<const _Float16*>(row), c, cols, out);
}
template <bool VEC, int E>
__device__ __forceinline__ void floats_as(const Raw<E>& in, uint32_t c, uint32_t cols, int dtype, float (&out)[E]) {
    if (dtype == ITTS_T_F32) floats<VEC, float>(in, c, cols, out);
    else if (dtype == ITTS_T_BF16) floats<VEC, __bf16>(in, c, cols, out);
    else floats<VEC, _Float16>(in, c, cols, out);
}

// Orders a wave's LDS accesses before and after it.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ------------------------------------------------------------------ rows to 8 bits
// Every element is read once: a team of waves owns a row and keeps it in registers between the two passes, CH runs of eight
// columns a lane; the norm's weights are requested with the row.  CH = 0: rows longer than that, by 1024 threads,
// which read h (or x) again.
// What bounds it, on inputs that come from memory: the quantisation of wide aligned rows, memory (4096 x 4096 FP32 16.4 us, a copy's
// rate).  With the norm, the chain of each row, its sums through two barriers and then its codes, which only CH = 1 overlaps with
// the next row's loads: 8192 x 5120 BF16 67 us without and 80 with a residual, where a copy of the same bytes takes 25 and 57; 84 MB of
// `values` beside that, 16 us for a copy, cost 9.  8192 x 1280 FP16 20 us, 2048 x 4096 FP32 15.
struct RowsArgs {
    NormArgs a;
    int kp, waves, shift;  // padded columns; waves of a team; log2 of the group
};
constexpr int kLongThreads = 1024;

template <class T, int CH, bool VEC, bool RES>
__global__ __launch_bounds__(1024) void rows_kernel(RowsArgs ra) {
    const NormArgs& a = ra.a;
    constexpr int N = CH ? CH : 1;
    constexpr int kEights = CH ? 1024 * CH : 1024;
    __shared__ double eights[kEights];
    const int lane = threadIdx.x & 63, waves = ra.waves, teams = blockDim.x / (64 * waves);
    const int team = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6) / waves), tid = threadIdx.x - team * waves * 64;
    const int step = waves * 64 * kElems, passes = CH ? CH : (ra.kp + step - 1) / step;
    const bool norm = a.weight != nullptr;
    double* mine = eights + team * waves * 64 * N;
    Raw<kElems> xr[N], rr[N], wr[N];
    float v[N][kElems];
    // (rows behind the last one count as empty)
    auto width = [&](int64_t r) { return r < a.rows ? static_cast<uint32_t>(a.cols) : 0u; };
    auto fetch = [&](int64_t r, uint32_t c, int i) {
        load_raw<VEC>(static_cast<const T*>(a.x) + r * a.x_stride, c, width(r), xr[i]);
        if constexpr (RES) load_raw<VEC>(static_cast<const T*>(a.residual) + r * a.residual_stride, c, width(r), rr[i]);
    };
    auto hidden = [&](int64_t r, uint32_t c, int i) {
        floats<VEC, T>(xr[i], c, width(r), v[i]);
        if constexpr (RES) {
            float u[kElems];
            floats<VEC, T>(rr[i], c, width(r), u);
#pragma unroll
            for (int e = 0; e < kElems; ++e) v[i][e] = to_float(from_float<T>(v[i][e] + u[e]));
        }
    };
    const int64_t each = static_cast<int64_t>(gridDim.x) * teams;
    int64_t r0 = static_cast<int64_t>(blockIdx.x) * teams;
    // Of one run a lane: the next row's loads are under way while this one is worked on (more do not fit the registers).
    constexpr bool NEXT = CH == 1;
    auto begin = [&](int64_t r) {
#pragma unroll
        for (int i = 0; i < CH; ++i) fetch(r, tid * kElems + i * step, i);
    };
    auto weights = [&] {
        if (norm) {
#pragma unroll
            for (int i = 0; i < CH; ++i) load_raw_as<VEC>(a.weight, tid * kElems + i * step, a.cols, a.weight_dtype, wr[i]);
        }
    };
    if constexpr (NEXT) {
        begin(r0 + team);
        weights();
    }
    for (; r0 < a.rows; r0 += each) {
        const int64_t r = r0 + team;
        const uint32_t cols = width(r);
        T* h = a.h_out ? static_cast<T*>(a.h_out) + r * a.h_stride : nullptr;
        if constexpr (CH > 0) {
            if constexpr (!NEXT) {
                begin(r);
                weights();
            }
#pragma unroll
            for (int i = 0; i < CH; ++i) hidden(r, tid * kElems + i * step, i);
            if constexpr (NEXT) {
                if (r0 + each < a.rows) begin(r + each);
            }
        }
        double inv = 1.0;
        if (norm) {
            if constexpr (CH == 0) {
                double sum = 0.0;
                for (int i = 0; i < passes; ++i) {
                    fetch(r, tid * kElems + i * step, 0);
                    hidden(r, tid * kElems + i * step, 0);
                    sum += quad_squares(v[0]) + quad_squares(v[0] + 4);
                }
                mine[tid] = sum;
            } else {
#pragma unroll
                for (int i = 0; i < CH; ++i) mine[tid + i * waves * 64] = quad_squares(v[i]) + quad_squares(v[i] + 4);
            }
            __syncthreads();
            inv = inv_rms(row_squares(mine, waves * 64 * N, lane), a);  // (zeros behind the row's end)
            __syncthreads();
        }
        auto codes = [&](uint32_t c, int i) {
            if (cols == 0 || c >= static_cast<uint32_t>(ra.kp)) return;  // (whole groups)
            if (h) store_row<VEC>(h, c, cols, v[i]);
            float w[kElems], code[kElems];
            if (norm) floats_as<VEC>(wr[i], c, a.cols, a.weight_dtype, w);
            const float s = group_codes(v[i], w, norm, inv, a.group, (c & -static_cast<uint32_t>(a.group)) < cols, code);
            *reinterpret_cast<uint2*>(a.q + r * ra.kp + c) = make_uint2(four_codes(code), four_codes(code + 4));
            if ((c & (a.group - 1)) == 0) a.scales[r * (ra.kp >> ra.shift) + (c >> ra.shift)] = s;
            if (a.values) {
#pragma unroll
                for (int e = 0; e < kElems; ++e) code[e] *= s;
                store_row<VEC>(static_cast<T*>(a.values) + r * a.values_stride, c, cols, code);
            }
        };
        if constexpr (CH > 0) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                codes(tid * kElems + i * step, i);
                __builtin_amdgcn_sched_barrier(0);  // (runs interleaved took more registers than there are)
            }
        } else {
            for (int i = 0; i < passes; ++i) {
                const uint32_t c = tid * kElems + i * step;
                fetch(r, c, 0);
                if (norm) load_raw_as<VEC>(a.weight, c, a.cols, a.weight_dtype, wr[0]);
                hidden(r, c, 0);
                codes(c, 0);
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

// One workgroup per tile, wave b its columns 32 b .. + 31: lane 16 j + r holds row r's eight from 8 j.  What a group wider than
// 32 columns and a byte's two halves need of other waves goes through LDS.  (One wave per tile, with a true
// quotient a value, took as long for large matrices, at the rate of a copy, but 6.8 us for 2049 x 387 against 4.1.)
template <class T, int G, bool VEC>
__global__ __launch_bounds__(256) void pack_kernel(PackArgs a) {
    __shared__ float tops[4][16];
    __shared__ uint2 halves[4][64];
    const int lane = threadIdx.x & 63, r = lane & 15, j = lane >> 4, b = threadIdx.x >> 6;
    const int kb = (a.k + kTileCols - 1) / kTileCols;
    const int64_t t = blockIdx.x, row = t / kb * kTileRows + r;
    Raw<kElems> raw;
    float v[kElems];
    const uint32_t col = static_cast<uint32_t>(t % kb) * kTileCols + 32 * b + 8 * j, cols = row < a.n ? a.k : 0;
    load_raw<VEC>(static_cast<const T*>(a.w) + row * a.stride, col, cols, raw);
    floats<VEC, T>(raw, col, cols, v);
    // the larger of max w / 7 and -min w / 8, or infinity where a value is not finite
    float mx = -INFINITY, mn = -INFINITY, bad = 0.0f;
#pragma unroll
    for (int i = 0; i < kElems; ++i) {
        mx = fmaxf(mx, v[i]);
        mn = fmaxf(mn, -v[i]);
        bad = __builtin_fmaf(v[i], 0.0f, bad);
    }
    float top = quarter_max(bad == 0.0f ? fmaxf(mx / 7.0f, mn / 8.0f) : INFINITY);
    if constexpr (G > 32) {
        if (j == 0) tops[b][r] = top;
        __syncthreads();
        top = fmaxf(tops[b][r], tops[b ^ 1][r]);
        if constexpr (G > 64) top = fmaxf(top, fmaxf(tops[b ^ 2][r], tops[b ^ 3][r]));
    }
    float s = static_cast<float>(static_cast<__bf16>(top));
    if (!(fabsf(s) <= 3.402823466e38f)) s = __uint_as_float(0x7fc00000u);
    // Codes: v / s by the reciprocal, at most one off; the remainder (exact by fma: q s has 12 bits and is next to v)
    // says whether, and finds the halves, which go to the even one.  Tiny numbers are scaled by 2^64 first.
    const float up = s < 1e-30f ? 18446744073709551616.0f : 1.0f, su = s * up, inv = 1.0f / su;
    uint32_t out[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kElems; ++i) {
        const float vu = v[i] * up;
        float q = rintf(vu * inv);
        const float rem = __builtin_fmaf(-q, su, vu), two = 2.0f * fabsf(rem);
        if (two > su || (two == su && (static_cast<int>(q) & 1))) q += copysignf(1.0f, rem);
        q = fminf(fmaxf(q, -8.0f), 7.0f);
        out[i >> 2] |= (s > 0.0f ? static_cast<uint32_t>(static_cast<int>(q)) & 15u : 0u) << (8 * (i & 3));
    }
    halves[b][lane] = make_uint2(out[0], out[1]);
    constexpr int NG = 128 / G;
    if (j == 0 && b % (G / 32) == 0) a.scales[(t * kTileRows + r) * NG + b / (G / 32)] = static_cast<uint16_t>(__float_as_uint(s) >> 16);
    __syncthreads();
    if (b < 2) {
        const uint2 lo = halves[2 * b][lane], hi = halves[2 * b + 1][lane];
        *reinterpret_cast<uint2*>(a.packed + t * kTileBytes + lane * 16 + 8 * b) = make_uint2(lo.x | hi.x << 4, lo.y | hi.y << 4);
    }
}

struct UnpackArgs {
    const uint8_t* packed;
    const uint16_t* scales;
    int n, k;
    void* out;
    int64_t stride;
};

// One wave per tile.  FP32 rows go through LDS, so that half a wave writes 512 bytes in a row past the caches (85 -> 54 us for
// 16384 x 5120; 74 through them).
template <class T, int G, bool VEC>
__global__ __launch_bounds__(256) void unpack_kernel(UnpackArgs a) {
    constexpr bool STAGED = VEC && sizeof(T) == 4;
    constexpr int kRow = kTileCols + 4;
    __shared__ __align__(16) float staged[STAGED ? 4 * kTileRows * kRow : 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, j = lane >> 4;
    const int kb = (a.k + kTileCols - 1) / kTileCols;
    const int64_t tiles = static_cast<int64_t>((a.n + kTileRows - 1) / kTileRows) * kb;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (t >= tiles) return;
    const int64_t row0 = t / kb * kTileRows, row = row0 + r;
    const u32x4 w = *reinterpret_cast<const u32x4*>(a.packed + t * kTileBytes + lane * 16);
    const int c0 = static_cast<int>(t % kb) * kTileCols;
    float* mine = staged + wave * kTileRows * kRow;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const float s = bf16_to_f32(a.scales[(t * kTileRows + r) * (128 / G) + 32 * b / G]);
        float v[kElems];
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            const int shift = 8 * (i & 3) + 4 * (b & 1);
            v[i] = static_cast<float>(static_cast<int32_t>(w[2 * (b >> 1) + (i >> 2)] << (28 - shift)) >> 28) * s;
        }
        if constexpr (STAGED) {
            float4* at = reinterpret_cast<float4*>(mine + r * kRow + 32 * b + 8 * j);
            at[0] = make_float4(v[0], v[1], v[2], v[3]);
            at[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            store_row<VEC>(static_cast<T*>(a.out) + row * a.stride, c0 + 32 * b + 8 * j, row < a.n ? a.k : 0, v);
        }
    }
    if constexpr (STAGED) {
        wave_sync();
        const int col = 4 * (lane & 31);
#pragma unroll
        for (int i = 0; i < kTileRows / 2; ++i) {
            const int rr = 2 * i + (lane >> 5);
            const f32x4 v = *reinterpret_cast<const f32x4*>(mine + rr * kRow + col);
            if (row0 + rr < a.n && c0 + col < a.k)
                __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + (row0 + rr) * a.stride + c0 + col));
        }
    }
}

// ------------------------------------------------------------------ products
__device__ __forceinline__ float load_as(const void* p, int64_t i, int dtype) {
    if (dtype == ITTS_T_F32) return static_cast<const float*>(p)[i];
    if (dtype == ITTS_T_BF16) return to_float(static_cast<const __bf16*>(p)[i]);
    return to_float(static_cast<const _Float16*>(p)[i]);
}
__device__ __forceinline__ void store_as(void* p, int64_t i, int dtype, float v) {
    if (dtype == ITTS_T_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == ITTS_T_BF16) static_cast<__bf16*>(p)[i] = from_float<__bf16>(v);
    else static_cast<_Float16*>(p)[i] = from_float<_Float16>(v);
}
// What a product adds to the sum of token m and weight row n, read ahead of it.
struct Added {
    float bias, residual;
};
__device__ __forceinline__ Added added(const ProductArgs& a, int m, int n) {
    Added e{0.0f, 0.0f};
    if (m < a.rows && n < a.n) {
        if (a.bias) e.bias = a.bias[n];
        if (a.residual) e.residual = load_as(a.residual, m * a.residual_stride + (a.swiglu ? n >> 1 : n), a.dtype);
    }
    return e;
}
// The last steps of a product's sum.  Lanes next to each other hold weight rows next to each other; all
// lanes of the wave take part.
__device__ __forceinline__ void finish(const ProductArgs& a, int m, int n, float v, const Added& e) {
    v += e.bias;
    int col = n;
    bool live = m < a.rows && n < a.n;
    if (a.swiglu) {
        v = silu_mul(v, itts::lane_x1(v));
        col = n >> 1;
        live = live && !(n & 1);
    }
    if (a.residual) v += e.residual;
    if (live) store_as(a.out, m * a.out_stride + col, a.dtype, v);
}

// The same for eight weight rows from n, a multiple of eight, at once.  Rows that are not 16-byte aligned are written in the
// same pieces but for their ends (2048 x 10241 x 1280 to FP16 with a residual: 56 us; one by one 96; 10240: 52).
template <class T, int N>
__device__ __forceinline__ void finish_row(const ProductArgs& a, int m, int col, int cols, float (&v)[N]) {
    T* out = static_cast<T*>(a.out) + m * a.out_stride + col;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + m * a.residual_stride + col : nullptr;
    struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Piece {
        T v[N * sizeof(T) < 16 ? N : 16 / sizeof(T)];
    };
    constexpr int P = sizeof(Piece) / sizeof(T);
    if (a.wide && col + N <= cols) {
#pragma unroll
        for (int k = 0; k < N / P; ++k) {
            Piece o;
            if (res) {
                const Piece r = reinterpret_cast<const Piece*>(res)[k];
#pragma unroll
                for (int i = 0; i < P; ++i) v[k * P + i] += to_float(r.v[i]);
            }
#pragma unroll
            for (int i = 0; i < P; ++i) o.v[i] = from_float<T>(v[k * P + i]);
            reinterpret_cast<Piece*>(out)[k] = o;
        }
    } else if (col + N <= cols) {
        constexpr int W = sizeof(Piece) / 4;
#pragma unroll
        for (int k = 0; k < N / P; ++k) {
            Piece o;
            if (res) {
                const Piece r = __builtin_bit_cast(Piece, reinterpret_cast<const Loose<T, W>*>(res)[k]);
#pragma unroll
                for (int i = 0; i < P; ++i) v[k * P + i] += to_float(r.v[i]);
            }
#pragma unroll
            for (int i = 0; i < P; ++i) o.v[i] = from_float<T>(v[k * P + i]);
            reinterpret_cast<Loose<T, W>*>(out)[k] = __builtin_bit_cast(Loose<T, W>, o);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col + i < cols) out[i] = from_float<T>(res ? v[i] + to_float(res[i]) : v[i]);
    }
}
template <int N>
__device__ __forceinline__ void finish_typed(const ProductArgs& a, int m, int col, int cols, float (&v)[N]) {
    if (a.dtype == ITTS_T_F32) finish_row<float, N>(a, m, col, cols, v);
    else if (a.dtype == ITTS_T_BF16) finish_row<__bf16, N>(a, m, col, cols, v);
    else finish_row<_Float16, N>(a, m, col, cols, v);
}
__device__ __forceinline__ void finish8(const ProductArgs& a, int m, int n, float (&v)[kElems]) {
    if (m >= a.rows || n >= a.n) return;
    if (a.bias) {
#pragma unroll
        for (int i = 0; i < kElems; ++i) v[i] += a.bias[min(n + i, a.n - 1)];
    }
    if (a.swiglu) {
        float u[kElems / 2];
#pragma unroll
        for (int i = 0; i < kElems / 2; ++i) u[i] = silu_mul(v[2 * i], v[2 * i + 1]);
        finish_typed(a, m, n >> 1, a.n >> 1, u);
    } else {
        finish_typed(a, m, n, a.n, v);
    }
}

// The largest of a tile's 16 sums (token 0: lanes 0 to 15), the first of equal ones; of NaN and -inf alone: -inf, row 0.
__device__ __forceinline__ void tile_best(float2* best, int tile, int tiles, float v, int n, int lane) {
    float i = __int_as_float(n);
    if (!(v > -INFINITY)) v = -INFINITY, i = __int_as_float(0);
    auto take = [&](float ov, float oi) {
        if (ov > v || (ov == v && __float_as_int(oi) < __float_as_int(i))) v = ov, i = oi;
    };
    take(itts::lane_x8(v), itts::lane_x8(i));
    take(itts::lane_x4(v), itts::lane_x4(i));
    take(itts::lane_x2(v), itts::lane_x2(i));
    take(itts::lane_x1(v), itts::lane_x1(i));
    if (lane == 0 && tile < tiles) best[tile] = make_float2(v, i);
}

// Up to four tokens: bound by the weights' bytes and, for small matrices, by latency.  A workgroup owns NT
// tile rows (16 weight rows each) and all columns; its waves take every W-th tile of 128 columns, U at a
// time, with all loads of a turn requested before their first use, and add their sums through LDS in
// wave order.  W hangs on k alone, so a token's result does not depend on the other tokens.
// The instruction's token rows 4 i hold token i: lane l then ends with token l / 16 in its first register, and
// the other three are not scaled, which is most of the vector work.
// FUSED: one token as a float row.  Every workgroup norms it and forms its codes in LDS, with its first
// turn's weights already under way: one launch instead of two, 6.4 -> 4.2 us for one row x 4096 x 1024.
// (Four rows by every workgroup took longer than a launch of their own: 14.8 us against 8.4 for 4 x 10240 x 1280.)
constexpr int kFewWaves = 8, kFewTokens = 4, kFusedCols = 16384;
// Where the tokens come from: codes; a float row; or a decode step's attention, in parts over splits of the cache.
enum : int { kFromCodes = 0, kFromRow = 1, kFromParts = 2 };
constexpr uint32_t kSplitRows = 64;  // cache rows a split
constexpr int kFewRow = kTileCols + 8;  // four rows' pieces lie in different banks
template <int G, int NT, int U, int FROM>
__global__ __launch_bounds__(64 * kFewWaves) void few_kernel(FewArgs fa) {
    constexpr bool FUSED = FROM != kFromCodes;
    const ProductArgs& a = fa.p;
    // (asked for first, waited for once the first loads are under way)
    const uint32_t active = fa.active ? *fa.active : 1u;
    constexpr int NG = 128 / G;
    // codes by blocks of 128 columns: [block][token][136 bytes], and scales [block][token][NG]; all blocks
    // of one token (FUSED), or those of a wave's turn
    constexpr int kBlocks = FUSED ? kFusedCols / kTileCols : kFewWaves * U * kFewTokens;
    __shared__ __align__(16) uint8_t codes[kBlocks * kFewRow];
    __shared__ float scales[kBlocks * NG];
    __shared__ float sums[kFewWaves * NT * 64];
    __shared__ double squares[FROM == kFromRow ? kFusedCols / kElems : 1];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, quarter = lane >> 4;
    const int W = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kb = (a.k + kTileCols - 1) / kTileCols, tiles = (a.n + kTileRows - 1) / kTileRows;
    const int rows = a.rows, mine = min(c >> 2, rows - 1), scaled = min(quarter, rows - 1);  // (c & 3 > 0: whatever)

    u32x4 wc[U][NT];
    uint16_t sc[U][NT][NG];
    auto weights = [&](int run, int b0) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int64_t row = static_cast<int64_t>(min(run * NT + i, tiles - 1)) * kb;
            const uint8_t* w = a.packed + row * kTileBytes + lane * 16;
            const uint16_t* ws = a.wscales + (row * kTileRows + c) * NG;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t b = min(b0 + u * W, kb - 1);
                wc[u][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(w + b * kTileBytes));
#pragma unroll
                for (int g = 0; g < NG; ++g) sc[u][i][g] = ws[b * kTileRows * NG + g];
            }
        }
    };
    if constexpr (FUSED) weights(blockIdx.x, wave);
    if constexpr (FROM == kFromParts) {
        // Four columns a thread, half a wave a head.  Its lanes hold the splits' largest scores and sums, two each, and
        // form the splits' weights at once; the first splits' values are asked for before their number is known.
        constexpr int TURN = 8;
        const uint32_t cached = *fa.cached;
        for (int p = tid; p < kb * 32; p += blockDim.x) {
            const int head = p >> 5, l = p & 31;
            auto v_at = [&](int s) { return *reinterpret_cast<const float4*>(fa.parts + (static_cast<size_t>(s) * kb + head) * kTileCols + l * 4); };
            const float2* ml = reinterpret_cast<const float2*>(fa.part_ml) + head;
            float2 a0 = ml[l * kb], a1 = ml[(l + 32) * kb];
            float4 v[TURN];
#pragma unroll
            for (int s = 0; s < TURN; ++s) v[s] = v_at(s);
            if (!active) return;
            const int splits = static_cast<int>(cached / kSplitRows) + 1;
            if (l >= splits) a0 = make_float2(-INFINITY, 0.0f);
            if (l + 32 >= splits) a1 = make_float2(-INFINITY, 0.0f);
            auto over_half = [](float x, auto op) {
                x = op(x, lane_of<1>(x));
                x = op(x, lane_of<2>(x));
                x = op(x, lane_of<4>(x));
                x = op(x, lane_of<8>(x));
                return op(x, lane_of<16>(x));
            };
            const float top = over_half(fmaxf(a0.x, a1.x), [](float x, float y) { return fmaxf(x, y); });
            const float w0 = expf(a0.x - top), w1 = expf(a1.x - top);
            const float den = over_half(__builtin_fmaf(w1, a1.y, w0 * a0.y), [](float x, float y) { return x + y; });
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f}, none[4] = {1.0f, 1.0f, 1.0f, 1.0f};
            for (int s0 = 0; s0 < splits; s0 += TURN) {
                float4 x[TURN];
#pragma unroll
                for (int s = 0; s < TURN; ++s) x[s] = v[s];
                if (s0 + TURN < splits) {
#pragma unroll
                    for (int s = 0; s < TURN; ++s) v[s] = v_at(min(s0 + TURN + s, splits - 1));
                }
#pragma unroll
                for (int s = 0; s < TURN; ++s) {
                    if (s0 + s >= splits) break;
                    const float w = __shfl(s0 < 32 ? w0 : w1, (lane & 32) | ((s0 + s) & 31));
                    sum[0] = __builtin_fmaf(w, x[s].x, sum[0]);
                    sum[1] = __builtin_fmaf(w, x[s].y, sum[1]);
                    sum[2] = __builtin_fmaf(w, x[s].z, sum[2]);
                    sum[3] = __builtin_fmaf(w, x[s].w, sum[3]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] /= den;
            float code[4];
            const float s = group_codes(sum, none, false, 1.0, G, true, code);
            *reinterpret_cast<uint32_t*>(codes + head * kFewRow + (p & 31) * 4) = four_codes(code);
            if (p * 4 % G == 0) scales[p * 4 / G] = s;
        }
        __syncthreads();
    }
    if constexpr (FROM == kFromRow) {
        const NormArgs& r = fa.rows;
        const int T = blockDim.x, quads = kb * 32;
        const int64_t first = fa.token ? *fa.token : 0;
        const uint8_t* row = static_cast<const uint8_t*>(r.x) + first * r.x_stride * (r.dtype == ITTS_T_F32 ? 4 : 2);
        // four columns a thread, half a wave a block; the first two turns stay in registers between the passes
        constexpr int KEEP = 2;
        Raw<4> x0[KEEP], w0[KEEP];
        float v0[KEEP][4], g0[KEEP][4];
        auto request = [&](int p, Raw<4>& v, Raw<4>& g) {
            if (fa.vec) {
                load_raw_as<true>(row, p * 4, a.k, r.dtype, v);
                if (r.weight) load_raw_as<true>(r.weight, p * 4, a.k, r.weight_dtype, g);
            } else {
                load_raw_as<false>(row, p * 4, a.k, r.dtype, v);
                if (r.weight) load_raw_as<false>(r.weight, p * 4, a.k, r.weight_dtype, g);
            }
        };
        auto convert = [&](int p, const Raw<4>& vr, const Raw<4>& gr, float (&v)[4], float (&g)[4]) {
            if (fa.vec) {
                floats_as<true>(vr, p * 4, a.k, r.dtype, v);
                if (r.weight) floats_as<true>(gr, p * 4, a.k, r.weight_dtype, g);
            } else {
                floats_as<false>(vr, p * 4, a.k, r.dtype, v);
                if (r.weight) floats_as<false>(gr, p * 4, a.k, r.weight_dtype, g);
            }
        };
        auto fetch = [&](int p, float (&v)[4], float (&g)[4]) {
            Raw<4> vr, gr;
            request(p, vr, gr);
            convert(p, vr, gr, v, g);
        };
        auto norm = [&](int p, const float (&v)[4]) {
            const double s = pair64<1>(quad_squares(v), add64);
            if ((p & 1) == 0) squares[p >> 1] = s;
        };
        double inv = 1.0;
        auto quantise = [&](int p, const float (&v)[4], const float (&g)[4]) {
            const int col = p * 4;
            if (fa.h_out && blockIdx.x == 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < a.k) fa.h_out[col + e] = v[e];
            }
            float code[4];
            const float s = group_codes(v, g, r.weight != nullptr, inv, G, col - col % G < a.k, code);
            *reinterpret_cast<uint32_t*>(codes + (p >> 5) * kFewRow + (p & 31) * 4) = four_codes(code);
            if (col % G == 0) scales[col / G] = s;
        };
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            if (tid + i * T < quads) request(tid + i * T, x0[i], w0[i]);
        if (!active) return;
#pragma unroll
        for (int i = 0; i < KEEP; ++i) convert(tid + i * T, x0[i], w0[i], v0[i], g0[i]);
        if (r.weight) {
#pragma unroll
            for (int i = 0; i < KEEP; ++i)
                if (tid + i * T < quads) norm(tid + i * T, v0[i]);
            for (int p = tid + KEEP * T; p < quads; p += T) {
                float v[4], g[4];
                fetch(p, v, g);
                norm(p, v);
            }
            __syncthreads();
            if (wave * 64 < quads) inv = inv_rms(row_squares(squares, kb * (kTileCols / kElems), lane), r);
        }
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            if (tid + i * T < quads) quantise(tid + i * T, v0[i], g0[i]);
        for (int p = tid + KEEP * T; p < quads; p += T) {
            float v[4], g[4];
            fetch(p, v, g);
            quantise(p, v, g);
        }
        __syncthreads();
    }
    if (!active) return;
    // the wave's own places for a turn's codes and scales, which whole cache lines bring there
    const int own = wave * U * kFewTokens, piece = lane & 7, token_c = min(lane >> 3, rows - 1);
    const int8_t* xg = FUSED ? nullptr : a.q + static_cast<int64_t>(token_c) * kb * kTileCols + 16 * piece;
    const float* sg = FUSED ? nullptr : a.qscales + static_cast<int64_t>(min(lane / NG, rows - 1)) * kb * NG + lane % NG;

    {
        const int run = blockIdx.x;
        float acc[NT] = {};
        for (int b0 = wave; b0 < kb; b0 += W * U) {
            if (!FUSED || b0 != wave) weights(run, b0);
            if constexpr (!FUSED) {
                u32x4 xr[U];
                float sr[U];
                if (lane < 8 * kFewTokens) {
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int b = min(b0 + u * W, kb - 1);
                        xr[u] = *reinterpret_cast<const u32x4*>(xg + b * kTileCols);
                        sr[u] = lane < kFewTokens * NG ? sg[b * NG] : 0.0f;
                    }
                    wave_sync();
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        uint8_t* at = codes + (own + u * kFewTokens + (lane >> 3)) * kFewRow + 16 * piece;
                        *reinterpret_cast<uint2*>(at) = make_uint2(xr[u][0], xr[u][1]);
                        *reinterpret_cast<uint2*>(at + 8) = make_uint2(xr[u][2], xr[u][3]);
                        if (lane < kFewTokens * NG) scales[(own + u * kFewTokens) * NG + lane] = sr[u];
                    }
                }
                wave_sync();
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int b = b0 + u * W;
                if (b >= kb) break;
                const int at = FUSED ? b : own + u * kFewTokens;
                const TokenCodes xc = token_codes(reinterpret_cast<const int8_t*>(codes) + (at + mine) * kFewRow, lane);
                float xs[NG];
#pragma unroll
                for (int g = 0; g < NG; ++g) xs[g] = scales[(at + scaled) * NG + g];
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    i32x4 f[NG];
                    tile_product<G>(xc, wc[u][i], f);
#pragma unroll
                    for (int g = 0; g < NG; ++g) acc[i] = __builtin_fmaf(static_cast<float>(f[g][0]), xs[g] * weight_scale(sc[u][i][g]), acc[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) sums[(wave * NT + i) * 64 + lane] = acc[i];
        __syncthreads();
        for (int i = wave; i < NT; i += W) {
            const int n = (run * NT + i) * kTileRows + c;
            const Added e = added(a, quarter, n);
            float v = 0.0f;
            for (int k = 0; k < W; ++k) v += sums[(k * NT + i) * 64 + lane];
            finish(a, quarter, n, v, e);
            if (fa.best) tile_best(fa.best, run * NT + i, tiles, n < a.n ? v : -INFINITY, n, lane);
        }
    }
}

// 5 to 16 tokens: as few_kernel, with the same sums.  A wave's codes of a tile of columns (16 rows of 128
// bytes) and their scales go through LDS of its own, whole cache lines at a time: as operands straight from
// memory, 8 bytes a lane from 16 rows, they took longer than the weights (18.7 -> 8.7 us for 16 x 10240 x 5120).
constexpr int kCodeRow16 = kTileCols + 8;  // 16 rows' pieces of 8 bytes lie in 32 different banks
template <int G, int NT, int U>
__global__ __launch_bounds__(64 * kFewWaves) void batch_kernel(ProductArgs a) {
    constexpr int NG = 128 / G, kStage = 16 * kCodeRow16 + NG * 16 * 4, S = NT * 4;
    constexpr int kSums = kFewWaves * S * 256, kCodes = kFewWaves * kStage;
    __shared__ __align__(16) uint8_t lds[kSums > kCodes ? kSums : kCodes];
    const int lane = threadIdx.x & 63, c = lane & 15, quarter = lane >> 4;
    const int W = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kb = (a.k + kTileCols - 1) / kTileCols, nt0 = blockIdx.x * NT, tiles = (a.n + kTileRows - 1) / kTileRows;
    uint8_t* mine = lds + wave * kStage;
    float* sums = reinterpret_cast<float*>(lds);

    const int8_t* xg[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) xg[i] = a.q + static_cast<int64_t>(min(8 * i + (lane >> 3), a.rows - 1)) * kb * kTileCols + 16 * (lane & 7);
    const int token_g = lane / NG, g_of = lane % NG;  // lanes under 16 NG fetch a scale each
    const float* sg = a.qscales + static_cast<int64_t>(min(token_g, a.rows - 1)) * kb * NG + g_of;
    const uint8_t* w[NT];
    const uint16_t* ws[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int64_t row = static_cast<int64_t>(min(nt0 + i, tiles - 1)) * kb;
        w[i] = a.packed + row * kTileBytes + lane * 16;
        ws[i] = a.wscales + (row * kTileRows + c) * NG;
    }
    float acc[NT][4] = {};
    for (int b0 = wave; b0 < kb; b0 += W * U) {
        u32x4 xr[U][2], wr[U][NT];
        float sr[U];
        uint16_t wsr[U][NT][NG];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = min(b0 + u * W, kb - 1);
#pragma unroll
            for (int i = 0; i < 2; ++i) xr[u][i] = *reinterpret_cast<const u32x4*>(xg[i] + b * kTileCols);
            sr[u] = lane < 16 * NG ? sg[b * NG] : 0.0f;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                wr[u][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(w[i] + static_cast<int64_t>(b) * kTileBytes));
#pragma unroll
                for (int g = 0; g < NG; ++g) wsr[u][i][g] = ws[i][static_cast<int64_t>(b) * kTileRows * NG + g];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (b0 + u * W >= kb) break;
            wave_sync();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint8_t* at = mine + (8 * i + (lane >> 3)) * kCodeRow16 + 16 * (lane & 7);
                *reinterpret_cast<uint2*>(at) = make_uint2(xr[u][i][0], xr[u][i][1]);
                *reinterpret_cast<uint2*>(at + 8) = make_uint2(xr[u][i][2], xr[u][i][3]);
            }
            if (lane < 16 * NG) *reinterpret_cast<float*>(mine + 16 * kCodeRow16 + (g_of * 16 + token_g) * 4) = sr[u];
            wave_sync();
            const TokenCodes xc = token_codes(reinterpret_cast<const int8_t*>(mine) + c * kCodeRow16, lane);
            float xs[NG][4];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float4 v = *reinterpret_cast<const float4*>(mine + 16 * kCodeRow16 + (g * 16 + 4 * quarter) * 4);
                xs[g][0] = v.x, xs[g][1] = v.y, xs[g][2] = v.z, xs[g][3] = v.w;
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                i32x4 f[NG];
                tile_product<G>(xc, wr[u][i], f);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const float s = weight_scale(wsr[u][i][g]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][r] = __builtin_fmaf(static_cast<float>(f[g][r]), xs[g][r] * s, acc[i][r]);
                }
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < S; ++s) sums[(wave * S + s) * 64 + lane] = acc[s / 4][s % 4];
    __syncthreads();
    for (int s = wave; s < S; s += W) {
        const int m = 4 * quarter + s % 4, n = (nt0 + s / 4) * kTileRows + c;
        const Added e = added(a, m, n);
        float v = 0.0f;
        for (int k = 0; k < W; ++k) v += sums[(k * S + s) * 64 + lane];
        finish(a, m, n, v, e);
    }
}

// More than 16 tokens: bound by the scaling, in this schedule.  Every group's 32-bit sums take a conversion, the product of
// the two scales and a multiply-add a value in the vector units: at 2048 x 10240 x 5120 in groups of 128 a block of 32 x 32
// and a group costs about 270 cycles of those and 140 of matrix instructions, and runs in 430 (162 us; SwiGLU 166, in groups
// of 64 216, of 32 312), as if the two came one after the other.  The machine does not ask for that: 32 v_fma_f32 beside four
// v_mfma_i32_32x32x32_i8 take 191 cycles where apart they take 142 and 139.  The outer product of scales as a matrix
// instruction of its own took 171 us, the last block of a turn scaled beside the next turn's products 163 (and 174 became
// 247 in blocks of 128 x 128).
// A workgroup owns 32 WM MT tokens x 32 WN NT weight rows.  WM x WN waves share a tile of codes staged through LDS;
// weights go from memory to registers, in the order of the instruction's operand; the next turn's loads are under way while
// this one's are multiplied.  WK such groups of waves take every WK-th tile of columns and add their sums through LDS in order.
// v_mfma_i32_32x32x32_i8, not 16x16x64: the same operands give twice the products, and four waves
// of a SIMD ran them at 35 cycles each against 29 for half the work.
// The instruction takes 16 consecutive columns from each half of the wave: 64 p + 32 b + 16 h + 0..15 for
// lane half h, which in a packed tile are the low (b = 0) or high halves of the bytes at 8 p of the lanes of j = 2 h
// and 2 h + 1.  It leaves weight row l % 32 and tokens 8 (r / 4) + 4 (l / 32) + r % 4 in lane l's registers r.
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
constexpr int kCodeRow = kTileCols + 16;  // eight rows' pieces of 16 bytes lie in 32 different banks
template <int G, int WM, int WN, int WK, int MT, int NT>
struct TilesLds {
    static constexpr int kTokens = WM * MT * 32, kStage = kTokens * (kCodeRow + 128 / G * 4);
    static constexpr int kSums = WK > 1 ? WK * WM * WN * MT * NT * 4096 : WM * WN * 32 * (NT * 32 + 4) * 4;
    static constexpr int kBytes = 2 * WK * kStage > kSums ? 2 * WK * kStage : kSums;
};
template <int G, int WM, int WN, int WK, int MT, int NT>
__global__ __launch_bounds__(64 * WM * WN * WK) void tiles_kernel(ProductArgs a) {
    using Lds = TilesLds<G, WM, WN, WK, MT, NT>;
    __shared__ __align__(16) uint8_t lds[Lds::kBytes];
    constexpr int NG = 128 / G, BM = Lds::kTokens, BN = WN * NT * 32, TG = 64 * WM * WN;
    constexpr int CH = BM * 8 / TG, SC = (BM * NG + TG - 1) / TG;
    static_assert(BM * 8 % TG == 0, "whole pieces of 16 codes a thread");
    const int lane = threadIdx.x & 63, c = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wk = wave / (WM * WN), wmn = wave % (WM * WN), wm = wmn / WN, wn = wmn % WN, tg = threadIdx.x - wk * TG;
    const int kb = (a.k + kTileCols - 1) / kTileCols, tiles = (a.n + kTileRows - 1) / kTileRows;
    const int mblocks = (a.rows + BM - 1) / BM;
    const int m0 = blockIdx.x % mblocks * BM, n0 = blockIdx.x / mblocks * BN;

    // places relative to the block's first row, in 32 bits: loads take a uniform address and these
    const int64_t row_bytes = static_cast<int64_t>(kb) * kTileCols, tile_bytes = static_cast<int64_t>(kb) * kTileBytes;
    const int8_t* const x0 = a.q + m0 * row_bytes;
    const float* const s0 = a.qscales + static_cast<int64_t>(m0) * kb * NG;
    const uint8_t* const w0 = a.packed + n0 / 16 * tile_bytes;
    const uint16_t* const ws0 = a.wscales + static_cast<int64_t>(n0 / 16) * kb * kTileRows * NG;
    uint32_t xo[CH], so[SC], wo[NT], wso[NT];
    int xl[CH], sl[SC];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int p = i * TG + tg, r = p >> 3, q = p & 7;
        xo[i] = static_cast<uint32_t>(min(r, a.rows - 1 - m0)) * static_cast<uint32_t>(row_bytes) + 16 * q;
        xl[i] = r * kCodeRow + 16 * q;
    }
#pragma unroll
    for (int i = 0; i < SC; ++i) {
        const int p = min(i * TG + tg, BM * NG - 1), r = p / NG, g = p % NG;
        so[i] = static_cast<uint32_t>(min(r, a.rows - 1 - m0)) * static_cast<uint32_t>(kb * NG) + g;
        sl[i] = BM * kCodeRow + (g * BM + r) * 4;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const uint32_t tile = static_cast<uint32_t>(min((wn * NT + i) * 2 + (c >> 4), tiles - 1 - n0 / 16));
        wo[i] = tile * static_cast<uint32_t>(tile_bytes) + (32 * half + (c & 15)) * 16;
        wso[i] = (tile * static_cast<uint32_t>(kb) * kTileRows + (c & 15)) * NG;
    }
    u32x4 xr[CH], wr[NT][2];
    float sr[SC];
    uint16_t wsr[NT][NG];
    auto fetch = [&](int step) {
        const int b = min(step * WK + wk, kb - 1);
        const int8_t* const xb = x0 + b * kTileCols;
        const float* const sb = s0 + b * NG;
        const uint8_t* const wb = w0 + static_cast<int64_t>(b) * kTileBytes;
        const uint16_t* const wsb = ws0 + static_cast<int64_t>(b) * kTileRows * NG;
#pragma unroll
        for (int i = 0; i < CH; ++i) xr[i] = *reinterpret_cast<const u32x4*>(xb + xo[i]);
#pragma unroll
        for (int i = 0; i < SC; ++i) sr[i] = sb[so[i]];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            wr[i][0] = *reinterpret_cast<const u32x4*>(wb + wo[i]);
            wr[i][1] = *reinterpret_cast<const u32x4*>(wb + wo[i] + 256);
#pragma unroll
            for (int g = 0; g < NG; ++g) wsr[i][g] = wsb[wso[i] + g];
        }
    };
    auto stage = [&](int step) {
        uint8_t* at = lds + (2 * wk + (step & 1)) * Lds::kStage;
#pragma unroll
        for (int i = 0; i < CH; ++i) *reinterpret_cast<u32x4*>(at + xl[i]) = xr[i];
#pragma unroll
        for (int i = 0; i < SC; ++i) *reinterpret_cast<float*>(at + sl[i]) = sr[i];
    };
    float acc[NT][MT][16] = {};
    const int steps = (kb + WK - 1) / WK;
    fetch(0);
    stage(0);
    for (int step = 0; step < steps; ++step) {
        u32x4 wc[NT][2];
        float sc[NT][NG];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            wc[i][0] = wr[i][0];
            wc[i][1] = wr[i][1];
#pragma unroll
            for (int g = 0; g < NG; ++g) sc[i][g] = weight_scale(wsr[i][g]);
        }
        __syncthreads();
        if (step + 1 < steps) fetch(step + 1);
        if (step * WK + wk < kb) {
            const uint8_t* at = lds + (2 * wk + (step & 1)) * Lds::kStage;
            i32x4 xc[MT][4];
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int q = 0; q < 4; ++q) xc[t][q] = *reinterpret_cast<const i32x4*>(at + ((wm * MT + t) * 32 + c) * kCodeRow + 32 * q + 16 * half);
            // the tokens' scales, ahead of their use where they fit the registers
            const uint8_t* xs = at + BM * kCodeRow + (wm * MT * 32 + 4 * half) * 4;
            constexpr bool AHEAD = NG == 1 && MT <= 2;
            auto token_scales = [&](int t, int g, int q) { return *reinterpret_cast<const float4*>(xs + (g * BM + t * 32 + 8 * q) * 4); };
            float4 xa[AHEAD ? MT * NG : 1][4];
            if constexpr (AHEAD) {
#pragma unroll
                for (int j = 0; j < MT * NG; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) xa[j][q] = token_scales(j / NG, j % NG, q);
            }
            // the products of one block of 32 x 32 and group are under way while those of the one before are scaled
            i32x16 f[2];
            auto multiply = [&](int i, int t, int g, i32x16& to) {
                const i32x16 zero = {};
                constexpr int Q = G / 32;
#pragma unroll
                for (int q = g * Q; q < (g + 1) * Q; ++q) {
                    const int p = q >> 1;
                    i32x4 wq;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t v = wc[i][e >> 1][2 * p + (e & 1)];
                        wq[e] = static_cast<int>((q & 1 ? v : v << 4) & kHigh);
                    }
                    to = __builtin_amdgcn_mfma_i32_32x32x32_i8(xc[t][q], wq, q == g * Q ? zero : to, 0, 0, 0);
                }
            };
            auto scale = [&](int i, int t, int g, const i32x16& from) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 v = AHEAD ? xa[AHEAD ? t * NG + g : 0][q] : token_scales(t, g, q);
                    const float x4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        acc[i][t][4 * q + r] = __builtin_fmaf(static_cast<float>(from[4 * q + r]), x4[r] * sc[i][g], acc[i][t][4 * q + r]);
                }
            };
#pragma unroll
            for (int j = 0; j < NT * MT * NG; ++j) {
                multiply(j / (MT * NG), j / NG % MT, j % NG, f[j & 1]);
                if (j > 0) scale((j - 1) / (MT * NG), (j - 1) / NG % MT, (j - 1) % NG, f[(j - 1) & 1]);
            }
            scale(NT - 1, MT - 1, NG - 1, f[(NT * MT * NG - 1) & 1]);
        }
        if (step + 1 < steps) stage(step + 1);
    }
    __syncthreads();
    if constexpr (WK == 1) {
        // thirty-two tokens at a time through LDS, so that a lane has eight columns of one token
        constexpr int BW = NT * 32, LR = BW / 8;  // columns of the wave, lanes a token
        float* mine = reinterpret_cast<float*>(lds) + wave * (32 * (BW + 4));
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) mine[(8 * (r >> 2) + 4 * half + (r & 3)) * (BW + 4) + i * 32 + c] = acc[i][t][r];
            wave_sync();
            for (int r0 = 0; r0 < 32; r0 += 64 / LR) {
                const int r = r0 + lane / LR, col = lane % LR * 8;
                float v[kElems];
#pragma unroll
                for (int e = 0; e < kElems; ++e) v[e] = mine[r * (BW + 4) + col + e];
                finish8(a, m0 + (wm * MT + t) * 32 + r, n0 + wn * BW + col, v);
            }
            wave_sync();
        }
    } else {
        constexpr int S = NT * MT * 16;
        float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int s = 0; s < S; ++s) sums[(wave * S + s) * 64 + lane] = acc[s / (MT * 16)][s / 16 % MT][s % 16];
        __syncthreads();
        for (int j = wave; j < WM * WN * S; j += WM * WN * WK) {
            const int o = j / S, s = j % S, r = s % 16;
            const int m = m0 + (o / WN * MT + s / 16 % MT) * 32 + 8 * (r >> 2) + 4 * half + (r & 3), n = n0 + (o % WN * NT + s / (MT * 16)) * 32 + c;
            const Added e = added(a, m, n);
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < WK; ++k) v += sums[((k * WM * WN + o) * S + s) * 64 + lane];
            finish(a, m, n, v, e);
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
// Rows that load_raw and store_row may take 16 bytes at a time.
bool rows_aligned(const void* p, int64_t stride, int dtype) {
    return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * static_cast<int64_t>(type_size(dtype)) % 16 == 0);
}
int pad_cols(int64_t k) { return static_cast<int>((k + kTileCols - 1) / kTileCols * kTileCols); }
}  // namespace

constexpr int kFewRows = 512;
constexpr int kRowGroups = 1024;  // workgroups that are resident together, about: each goes through several rows

hipError_t launch_rows(const NormArgs& a, hipStream_t s) {
    if (a.rows == 0) return hipSuccess;
    const bool vec = a.cols % kElems == 0 && rows_aligned(a.x, a.x_stride, a.dtype) && rows_aligned(a.residual, a.residual_stride, a.dtype) &&
                     rows_aligned(a.h_out, a.h_stride, a.dtype) && rows_aligned(a.values, a.values_stride, a.dtype) &&
                     rows_aligned(a.weight, 0, a.dtype);
    // Waves a row takes with one run of 512 columns each.  Few rows: as many (up to 16), for their latency.  Many
    // rows: one, two or four waves and up to four runs each, whose loads are under way at once; and teams that
    // fill workgroups of four waves, or a multiple: of five waves a SIMD got two in every workgroup, and 8192 x
    // 5120 took 118 us instead of 81.
    const int kp = pad_cols(a.cols), all = (kp + 511) / 512;
    const bool few = all <= 16 && a.rows <= kFewRows;
    const int waves = few ? all : all == 1 ? 1 : all <= 4 ? (all + 1) / 2 : all <= 16 ? 4 : all <= 32 ? 8 : 16;
    const int ch = few ? 1 : all <= 64 ? (all + waves - 1) / waves : 0;
    const int teams = waves >= 4 ? 1 : 4 / waves;
    const RowsArgs ra{a, kp, waves, a.group == 32 ? 5 : a.group == 64 ? 6 : 7};
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((a.rows + teams - 1) / teams, kRowGroups))), block(64 * waves * teams);
    return by_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return by_bool(vec, [&](auto v) {
            return by_bool(a.residual != nullptr, [&](auto res) {
                constexpr bool V = decltype(v)::value, R = decltype(res)::value;
                if (ch == 1) hipLaunchKernelGGL((rows_kernel<T, 1, V, R>), grid, block, 0, s, ra);
                else if (ch == 2) hipLaunchKernelGGL((rows_kernel<T, 2, V, R>), grid, block, 0, s, ra);
                else if (ch == 3) hipLaunchKernelGGL((rows_kernel<T, 3, V, R>), grid, block, 0, s, ra);
                else if (ch == 4) hipLaunchKernelGGL((rows_kernel<T, 4, V, R>), grid, block, 0, s, ra);
                else hipLaunchKernelGGL((rows_kernel<T, 0, V, R>), grid, block, 0, s, ra);
                return hipGetLastError();
            });
        });
    });
}

namespace {
// Matrices of so many rows take four tile rows a workgroup, which then reads the codes once for the four and has more loads
// under way; fewer rows leave too few workgroups for that.  Measured (us with one and with four tile rows):
//   1 row: 16384 x 1024 3.9 4.3; 32768 x 512 4.1 4.4, x 1024 6.0 5.5, x 2048 8.1 8.0, x 5120 16.3 16.8; 151936 x 512 10.6 8.8,
//     x 1024 18.8 14.2, x 2048 26.2 26.6, x 5120 60.1 60.7; 4 rows: four against one within 3% of that
//   5 rows: 10240 x 1024 4.0 4.3, x 5120 8.5 8.3; 16384 x 1024 4.3 4.6, x 5120 10.7 9.4, x 8192 14.9 14.8; 65536 x 5120 35 28
//   16 rows: 8192 x 5120 8.0 8.8; 10240 x 1024 4.1 4.5, x 5120 10.2 9.0; 16384 x 1024 4.6 4.7, x 5120 13.3 9.8, x 8192 19.0 14.5
constexpr int kFewWide = 32768, kBatchWide = 16384;

// Tiles of columns that a wave takes in a turn, of `each` in all: those that leave the fewest of its last turn
// idle, the more the better.
int turn_tiles(int each) {
    int u = 1;
    for (int k = 2; k <= std::min(each, 5); ++k)
        if ((each + k - 1) / k * k <= (each + u - 1) / u * u || u == 1) u = k;
    return u;
}

template <int G, int NT, int U, int FROM>
hipError_t launch_few(const FewArgs& a, int waves, hipStream_t s) {
    const int tiles = (a.p.n + kTileRows - 1) / kTileRows;
    hipLaunchKernelGGL((few_kernel<G, NT, U, FROM>), dim3((tiles + NT - 1) / NT), dim3(64 * waves), 0, s, a);
    return hipGetLastError();
}
template <int G, int FROM>
hipError_t few_rows(const FewArgs& a, hipStream_t s) {
    const int kb = pad_cols(a.p.k) / kTileCols, waves = std::min(kb, kFewWaves), each = (kb + waves - 1) / waves;
    if constexpr (FROM == kFromCodes) {
        if (a.p.n >= kFewWide) return each == 1 ? launch_few<G, 4, 1, FROM>(a, waves, s) : launch_few<G, 4, 2, FROM>(a, waves, s);
    }
    switch (turn_tiles(each)) {
        case 1: return launch_few<G, 1, 1, FROM>(a, waves, s);
        case 2: return launch_few<G, 1, 2, FROM>(a, waves, s);
        case 3: return launch_few<G, 1, 3, FROM>(a, waves, s);
        case 4: return launch_few<G, 1, 4, FROM>(a, waves, s);
        default: return launch_few<G, 1, 5, FROM>(a, waves, s);
    }
}
template <int G, int NT, int U>
hipError_t launch_batch(const ProductArgs& a, int waves, hipStream_t s) {
    const int tiles = (a.n + kTileRows - 1) / kTileRows;
    hipLaunchKernelGGL((batch_kernel<G, NT, U>), dim3((tiles + NT - 1) / NT), dim3(64 * waves), 0, s, a);
    return hipGetLastError();
}
template <int G>
hipError_t batch_rows(const ProductArgs& a, hipStream_t s) {
    const int kb = pad_cols(a.k) / kTileCols, waves = std::min(kb, kFewWaves), each = (kb + waves - 1) / waves;
    if (a.n >= kBatchWide) return launch_batch<G, 4, 1>(a, waves, s);
    switch (turn_tiles(each)) {
        case 1: return launch_batch<G, 1, 1>(a, waves, s);
        case 2: return launch_batch<G, 1, 2>(a, waves, s);
        case 3: return launch_batch<G, 1, 3>(a, waves, s);
        case 4: return launch_batch<G, 1, 4>(a, waves, s);
        default: return launch_batch<G, 1, 5>(a, waves, s);
    }
}
template <int G, int WM, int WN, int WK, int MT, int NT>
hipError_t launch_tiles(const ProductArgs& a, hipStream_t s) {
    const int mb = (a.rows + WM * MT * 32 - 1) / (WM * MT * 32), nb = (a.n + WN * NT * 32 - 1) / (WN * NT * 32);
    hipLaunchKernelGGL((tiles_kernel<G, WM, WN, WK, MT, NT>), dim3(static_cast<unsigned>(mb) * nb), dim3(64 * WM * WN * WK), 0, s, a);
    return hipGetLastError();
}
template <int G>
hipError_t product(const ProductArgs& a, hipStream_t s) {
    if (a.rows <= kFewTokens) return few_rows<G, kFromCodes>(FewArgs{a}, s);
    if (a.rows <= 16) return batch_rows<G>(a, s);
    // Workgroups of 64 x 128 (one wave 64 x 32: the fewest LDS and memory reads a product) where two a CU come of
    // them; else of 64 x 64, nearly as many; else smaller blocks whose waves share the columns, for the latency of
    // their turns.  Measured (us; 64 x 128, 64 x 64, 32 x 64 by 4, 32 x 32 by 8): 1024 x 4096 x 4096 33 39 - -;
    // 512 x 6144 x 1024 12.6 12.1 - -; 155 x 10240 x 1280 12.0 10.5 13.6 -; 256 x 4096 x 4096 in groups of 64 34 26
    // 16.8 -; 64 x 10240 x 5120 - - 15.3 16.9; 64 x 1024 x 2048 - - 6.3 4.9; 32 x 151936 x 1024 (32 x 128) 23 - 29 36.
    const auto blocks = [&](int bm, int bn) { return static_cast<int64_t>((a.rows + bm - 1) / bm) * ((a.n + bn - 1) / bn); };
    if (a.rows <= 32 && blocks(32, 128) >= 512) return launch_tiles<G, 1, 4, 1, 1, 1>(a, s);
    if (blocks(64, 128) >= 512) return launch_tiles<G, 1, 4, 1, 2, 1>(a, s);
    if (blocks(64, 64) >= 448) return launch_tiles<G, 2, 2, 1, 1, 1>(a, s);
    if (blocks(32, 32) <= 512) return launch_tiles<G, 1, 1, 8, 1, 1>(a, s);
    return launch_tiles<G, 1, 2, 4, 1, 1>(a, s);
}
}  // namespace

hipError_t launch_product(const ProductArgs& given, hipStream_t s) {
    if (given.rows == 0) return hipSuccess;
    ProductArgs a = given;
    a.wide = rows_aligned(a.out, a.out_stride, a.dtype) && rows_aligned(a.residual, a.residual_stride, a.dtype);
    return by_group(a.group, [&](auto g) { return product<decltype(g)::value>(a, s); });
}

// A row that every workgroup norms for itself: not for more workgroups than are resident together (four a CU).
bool linear_is_fused(int64_t rows, int64_t n, int64_t k) { return rows == 1 && n <= 1024 * kTileRows && k <= kFusedCols; }

hipError_t launch_few(const FewArgs& a, hipStream_t s) {
    return by_group(a.p.group, [&](auto g) { return few_rows<decltype(g)::value, kFromCodes>(a, s); });
}

hipError_t launch_fused(const FewArgs& given, hipStream_t s) {
    FewArgs a = given;
    a.vec = a.p.k % kElems == 0 && rows_aligned(a.rows.x, a.rows.x_stride, a.rows.dtype) && rows_aligned(a.rows.weight, 0, a.rows.dtype);
    return by_group(a.p.group, [&](auto g) { return few_rows<decltype(g)::value, kFromRow>(a, s); });
}

// (turns of two tiles: those of the decoder's 16 heads, two a wave)
hipError_t launch_merged(const FewArgs& a, hipStream_t s) { return launch_few<128, 1, 2, kFromParts>(a, std::min(pad_cols(a.p.k) / kTileCols, kFewWaves), s); }

hipError_t launch_linear(const ProductArgs& product, const NormArgs& rows, hipStream_t s) {
    if (product.rows == 0) return hipSuccess;
    if (linear_is_fused(product.rows, product.n, product.k)) return launch_fused(FewArgs{product, rows}, s);
    const hipError_t e = launch_rows(rows, s);
    if (e != hipSuccess) return e;
    ProductArgs p = product;
    p.q = rows.q;
    p.qscales = rows.scales;
    return launch_product(p, s);
}

hipError_t launch_pack(const void* w, int64_t stride, int dtype, int n, int k, int group, void* packed, void* scales, hipStream_t s) {
    const PackArgs a{w, stride, n, k, static_cast<uint8_t*>(packed), static_cast<uint16_t*>(scales)};
    const bool vec = k % kElems == 0 && rows_aligned(w, stride, dtype);
    const int64_t tiles = static_cast<int64_t>((n + kTileRows - 1) / kTileRows) * (pad_cols(k) / kTileCols);
    const dim3 grid(static_cast<unsigned>(tiles));
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
    } catch (...) {
        g_ops_error = "Unknown failure";
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
constexpr int64_t kMaxResults = int64_t(1) << 36;
// A workgroup of 256 a tile: fewer than 2^32 threads, the most that a launch takes.
constexpr size_t kMaxPacked = size_t(kTileBytes) << 23;
bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
bool aligned_for(const void* p, int32_t dtype) { return aligned(p, dtype == ITTS_T_F32 ? 4 : 2); }

// A matrix in memory: rows of `width` bytes, `step` bytes apart.
struct Span {
    const void* at;
    int64_t rows, width, step;
    Span(const void* p, int64_t r, int64_t cols, int64_t stride, int32_t dtype) : at(p), rows(r), width(cols * static_cast<int64_t>(type_size(dtype))), step(width) {
        if (r <= 1) return;
        need(!p || stride <= (int64_t(1) << 56) / (4 * r), "Row stride out of range");
        step = p ? stride * static_cast<int64_t>(type_size(dtype)) : width;
    }
    Span(const void* p, size_t bytes) : at(p), rows(1), width(static_cast<int64_t>(bytes)), step(width) {}
    bool same(const Span& o) const { return at == o.at && step == o.step; }
    // Whether the two share a byte (or, with different steps, might): columns of one wider matrix do not.
    bool meets(const Span& o) const {
        if (!at || !o.at) return false;
        const int64_t a = static_cast<int64_t>(reinterpret_cast<uintptr_t>(at)), b = static_cast<int64_t>(reinterpret_cast<uintptr_t>(o.at));
        if (a + (rows - 1) * step + width <= b || b + (o.rows - 1) * o.step + o.width <= a) return false;
        if (rows == 1 && o.rows == 1) return true;
        const int64_t s = rows > 1 ? step : o.step;
        if ((o.rows > 1 && o.step != s) || s < width || s < o.width) return true;
        const int64_t d = ((b - a) % s + s) % s;  // where o's rows begin in this one's
        return d < width || d + o.width > s;
    }
    void apart(std::initializer_list<Span> others) const {
        for (const Span& o : others) need(!meets(o), "Output overlaps an input or another output");
    }
};

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
    const int64_t kp = pad_cols(cols);
    const Span xs(x, rows, cols, x_stride, dtype), vs(values, rows, cols, values_stride, dtype), qs(q, static_cast<size_t>(rows * kp)),
        ss(scales, static_cast<size_t>(rows * (kp / group)) * sizeof(float));
    vs.apart({xs, qs, ss});
    qs.apart({xs, ss});
    ss.apart({xs});
}

void check_weight(const void* packed, const void* scales, int64_t n, int64_t k, int32_t group) {
    need(group_ok(group), "Group is 32, 64 or 128 columns");
    need(n >= 1 && n <= kMaxN && k >= 1 && k <= kMaxK, "Weight size out of range");
    need(packed && scales, "Missing tensor");
    need(aligned(packed, 16) && aligned(scales, 16), "Misaligned tensor");
}

Span packed_span(const void* packed, int64_t n, int64_t k) { return {packed, itts_q4_packed_bytes(n, k)}; }
Span scales_span(const void* scales, int64_t n, int64_t k, int32_t group) { return {scales, itts_q4_scale_count(n, k, group) * 2}; }
Span out_span(const ProductArgs& p) { return {p.out, p.rows, p.swiglu ? p.n / 2 : p.n, p.out_stride, p.dtype}; }

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
        need(rows * n <= kMaxResults, "Too many results");
        const int64_t cols = swiglu ? n / 2 : n;
        const Span os(out, rows, cols, out_stride, dtype), rs(residual, rows, cols, residual_stride, dtype);
        need(os.same(rs) || !os.meets(rs), "Output overlaps an input");
        os.apart({packed_span(packed, n, k), scales_span(scales, n, k, group), Span(bias, static_cast<size_t>(n) * sizeof(float))});
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
        const Span xs(x, rows, cols, x_stride, dtype), rs(residual, rows, cols, residual_stride, dtype), hs(h_out, rows, cols, h_stride, dtype),
            vs(values, rows, cols, values_stride, dtype);
        const Span ws(weight, static_cast<size_t>(cols) * type_size(weight_dtype)), qs(q, static_cast<size_t>(rows * pad_cols(cols))),
            ss(scales, static_cast<size_t>(rows * (pad_cols(cols) / group)) * sizeof(float));
        need((hs.same(xs) || !hs.meets(xs)) && (hs.same(rs) || !hs.meets(rs)), "Output overlaps an input");
        hs.apart({vs, qs, ss, ws});
        vs.apart({rs, ws});
        qs.apart({rs, ws});
        ss.apart({rs, ws});
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
        need(itts_q4_packed_bytes(n, k) <= kMaxPacked, "Weight too large");
        const Span ps = packed_span(packed, n, k), ss = scales_span(scales, n, k, group), ws(w, n, k, w_stride, dtype);
        ps.apart({ss, ws});
        ss.apart({ws});
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
        need(itts_q4_packed_bytes(n, k) <= kMaxPacked, "Weight too large");
        Span(out, n, k, out_stride, dtype).apart({packed_span(packed, n, k), scales_span(scales, n, k, group)});
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
        const int64_t kp = pad_cols(k);
        out_span(p).apart({Span(q, static_cast<size_t>(rows * kp)), Span(qscales, static_cast<size_t>(rows * (kp / group)) * sizeof(float))});
        launched(launch_product(p, static_cast<hipStream_t>(stream)));
    });
}

size_t itts_q4_linear_workspace(int64_t rows, int64_t n, int64_t k, int32_t group) {
    if (rows < 1 || n < 1 || k < 1 || k > kMaxK || !group_ok(group) || linear_is_fused(rows, n, k)) return 0;
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
        // (workgroups that norm the row for themselves read x while others write out)
        const Span xs(x, rows, k, x_stride, x_dtype), ns(norm_weight, static_cast<size_t>(k) * type_size(weight_dtype)), os = out_span(p);
        os.apart({xs, ns});
        const size_t bytes = itts_q4_linear_workspace(rows, n, k, group);
        need(bytes == 0 || (workspace && workspace_bytes >= bytes), "Workspace too small");
        need(aligned(workspace, 256), "Misaligned workspace");
        if (bytes)
            Span(workspace, bytes).apart({xs, ns, os, packed_span(packed, n, k), scales_span(scales, n, k, group), Span(bias, static_cast<size_t>(n) * sizeof(float)),
                                          Span(residual, rows, p.swiglu ? n / 2 : n, residual_stride, dtype)});
        int8_t* q = static_cast<int8_t*>(workspace);
        float* qs = bytes ? reinterpret_cast<float*>(q + codes_bytes(rows, k)) : nullptr;
        const NormArgs r{x, x_stride, nullptr, 0, norm_weight, weight_dtype, x_dtype, rows, k, eps, group, nullptr, 0, nullptr, 0, q, qs};
        launched(launch_linear(p, r, static_cast<hipStream_t>(stream)));
    });
}

}  // extern "C"
