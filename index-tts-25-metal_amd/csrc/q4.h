// Launch arguments and launchers of the kernels on 4-bit weights and 8-bit activations (q4.hip).
// The formats are those of include/itts_ops.h, whose entry points check what is assumed here.
#pragma once
#include "common.h"

namespace itts {
namespace q4 {

struct NormArgs {
    const void* x;
    int64_t x_stride;
    const void* residual;  // or null
    int64_t residual_stride;
    const void* weight;    // null: no norm
    int weight_dtype, dtype;
    int64_t rows, cols;
    float eps;
    int group;
    void* h_out;           // or null
    int64_t h_stride;
    void* values;          // or null
    int64_t values_stride;
    int8_t* q;
    float* scales;
};
hipError_t launch_rows(const NormArgs& a, hipStream_t s);

struct ProductArgs {
    const int8_t* q;
    const float* qscales;
    int rows;
    const uint8_t* packed;
    const uint16_t* wscales;
    int n, k, group;
    const float* bias;     // or null
    const void* residual;  // or null
    int64_t residual_stride;
    bool swiglu;
    int dtype;
    void* out;
    int64_t out_stride;
    bool wide;             // set by launch_product: rows of out and residual are 16-byte aligned
};
hipError_t launch_product(const ProductArgs& a, hipStream_t s);

// A product of up to four rows, or (launch_fused) the norm or quantisation of one row and its product, with what a
// decode step adds to them.
struct FewArgs {
    ProductArgs p;           // (launch_fused: without q, qscales)
    NormArgs rows;           // launch_fused: x, x_stride, weight, weight_dtype, dtype, cols, eps
    const uint32_t* active;  // or null: the launch does nothing where it is 0
    const uint32_t* token;   // or null: x is row *token of a matrix (launch_fused)
    float* h_out;            // or null: receives x's row in F32 (launch_fused)
    float2* best;            // or null: per 16 weight rows the largest sum of row 0 and its index
    const float* parts;      // launch_merged: attention over splits of 64 cache rows, [split][k / 128 heads][128], weighted sums
    const float* part_ml;    //   [split][heads][2]: the largest score and the sum of exp(score - largest); both hold 64 splits
    const uint32_t* cached;  //   cache rows before this step's: cached / 64 + 1 splits count
    bool vec;                // set by launch_fused
};
hipError_t launch_few(const FewArgs& a, hipStream_t s);
// launch_fused for a decode step's attention output, whose splits it merges: x[128 h + d] = sum over splits of w_s parts[s][h][d] /
// sum of w_s ml[s][h][1], w_s = exp(ml[s][h][0] - their largest).  k a multiple of 128, group 128.
hipError_t launch_merged(const FewArgs& a, hipStream_t s);
bool linear_is_fused(int64_t rows, int64_t n, int64_t k);
hipError_t launch_fused(const FewArgs& a, hipStream_t s);
// Norm (or quantisation) and product: fused, or through rows.q and rows.scales.
hipError_t launch_linear(const ProductArgs& p, const NormArgs& rows, hipStream_t s);

hipError_t launch_pack(const void* w, int64_t stride, int dtype, int n, int k, int group, void* packed, void* scales, hipStream_t s);
hipError_t launch_unpack(const void* packed, const void* scales, int n, int k, int group, int dtype, void* out, int64_t stride, hipStream_t s);

}  // namespace q4
}  // namespace itts
