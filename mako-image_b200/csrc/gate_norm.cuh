// The row kernels of a quantised block: the gated residual add between a branch's output norm and the next branch's
// input norm in one pass, and rows to 8-bit integers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace mkb {

enum NormKind : int { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };
enum RowOut : int { kOutNone = 0, kOutBf16 = 1, kOutF32 = 2, kOutI8 = 3 };

// x_out = x + g(gate) * (N_y(y) * y_weight); out = N_x(x_out) * x_weight * (1 + scale) + shift. Null vectors are left
// out. gate, scale and shift are those of sample row / rows_per_sample.
struct GateNormArgs {
    const float* x;
    long ldx;
    float* x_out;
    long ldxo;
    const void* y;  // null: no residual, x_out is x
    long ldy;
    int y_f32, y_norm, x_norm, tanh_gate;
    const float* y_weight;
    const float* gate;
    long gate_stride;
    const float* x_weight;
    const float* scale;
    const float* shift;
    long mod_stride;
    long rows_per_sample;
    float eps;
    void* out;
    long ldo;
    int out_type;
    float* out_scale;  // kOutI8: a step per row
    long rows;
    int n;
};
constexpr int kGateNormMaxWidth = 12288;  // 512 threads, 24 values each
cudaError_t gate_norm(const GateNormArgs& a, cudaStream_t st);

struct QuantRowsArgs {
    const void* x;  // bf16, or fp32 with x_f32
    long ldx;
    int x_f32;
    int8_t* q;
    long ldq;
    float* scale;
    long rows;
    int n;
};
cudaError_t quantize_rows(const QuantRowsArgs& a, cudaStream_t st);

}  // namespace mkb
